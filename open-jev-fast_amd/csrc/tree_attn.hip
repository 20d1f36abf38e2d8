// Attention of drafted tokens over a paged cache.
//
// Sequence b has n = q_ptr[b + 1] - q_ptr[b] drafted tokens (rows) and ctx[b] tokens before them; its cache position p
// lies in page table[b][p / page] at place p % page, and drafted token j at position ctx[b] + j. A row sees the positions
// below ctx[b] and those drafted tokens whose bit is set in its bits (without bits: its predecessors and itself).
//   s_p = scale q . k_p,  m = max s_p,  out = sum exp(s_p - m) v_p / sum exp(s_p - m),  lse = m + log sum exp(s_p - m)
// over the positions seen; a row that sees nothing gives zeros and lse = -inf.
#include "ojx_internal.h"

namespace ojx {

namespace {

template <bool FP8>
__device__ __forceinline__ float cache_value(const void* c, const float* s, int64_t row, int D, int d) {
  if (FP8) {
    const uint8_t* p = static_cast<const uint8_t*>(c) + row * D + d;
    return __builtin_amdgcn_cvt_f32_fp8(*p, 0) * s[row];
  }
  return bf2f(static_cast<const uint16_t*>(c)[row * D + d]);
}

// One workgroup of four waves per (row, query head); wave w takes positions w, w + 4, ..; a lane holds D / 64 dims.
template <int D, bool FP8>
__global__ void __launch_bounds__(256) tree_attn_k(TreeParams p) {
  constexpr int E = D / 64;
  const int64_t n = blockIdx.x / p.HQ;
  const int h = blockIdx.x - (int)(n * p.HQ), hk = h / (p.HQ / p.HKV);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t b = -1, first = 0, end = 0;
  for (int i = 0; i < p.B; ++i) {
    const int64_t x = min(max((int64_t)p.q_ptr[i], (int64_t)0), p.N), y = min(max((int64_t)p.q_ptr[i + 1], x), p.N);
    if (n >= x && n < y) {
      b = i;
      first = x;
      end = y;
    }
  }
  float q[E], acc[E], m = -INFINITY, l = 0.f;
  for (int e = 0; e < E; ++e) {
    q[e] = bf2f(p.q[((int64_t)h * p.N + n) * D + lane * E + e]);
    acc[e] = 0.f;
  }
  if (b >= 0) {
    const int64_t ctx = max(p.ctx[b], 0);
    const int64_t total = min(ctx + (end - first), p.max_pages * p.page);
    for (int64_t pos = wave; pos < total; pos += 4) {
      const int64_t j = pos - ctx;
      if (j >= 0) {
        const bool sees = p.bits == nullptr ? j <= n - first
                                            : j < 64LL * p.words && ((p.bits[n * p.words + j / 64] >> (j % 64)) & 1);
        if (!sees) continue;
      }
      const int page = p.table[b * p.max_pages + pos / p.page];
      if (page < 0 || page >= p.pages) continue;
      const int64_t row = ((int64_t)page * p.HKV + hk) * p.page + pos % p.page;
      float s = 0.f;
      for (int e = 0; e < E; ++e) s += q[e] * cache_value<FP8>(p.kc, p.ks, row, D, lane * E + e);
      s = wave_sum64(s) * p.scale;
      const float t = fmaxf(m, s), a = m == -INFINITY ? 0.f : expf(m - t), w = expf(s - t);
      l = l * a + w;
      for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + w * cache_value<FP8>(p.vc, p.vs, row, D, lane * E + e);
      m = t;
    }
  }
  __shared__ float sm[4], sl[4], so[4][D];
  for (int e = 0; e < E; ++e) so[wave][lane * E + e] = acc[e];
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
  __syncthreads();
  float mm = -INFINITY, ll = 0.f, f[4];
  for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sm[w]);
  for (int w = 0; w < 4; ++w) {
    f[w] = sm[w] == -INFINITY ? 0.f : expf(sm[w] - mm);
    ll += f[w] * sl[w];
  }
  if (threadIdx.x < D) {
    float o = 0.f;
    for (int w = 0; w < 4; ++w) o += f[w] * so[w][threadIdx.x];
    p.out[(n * p.HQ + h) * D + threadIdx.x] = (uint16_t)f2bf(ll == 0.f ? 0.f : o / ll);
  }
  if (p.lse != nullptr && threadIdx.x == 0) p.lse[n * p.HQ + h] = ll == 0.f ? -INFINITY : mm + logf(ll);
}

}  // namespace

hipError_t launch_tree_attn(const TreeParams& p, int D, bool fp8, hipStream_t st) {
  const auto kernel = D == 256 ? (fp8 ? tree_attn_k<256, true> : tree_attn_k<256, false>)
                               : (fp8 ? tree_attn_k<128, true> : tree_attn_k<128, false>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)(p.N * p.HQ)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

// Linear attention (linattn.hip) around drafted tokens: a tree of them on a state that stays as it is, and a state taken
// forward over the tokens that were kept.
//
// A drafted token i follows another row of its sequence, or the sequence's state S0 itself. With A(i) its ancestors and G_i
// the sum of g over them and itself,
//   u_i = beta_i (v_i - e^(G_i) S0^T k_i - sum_{j in A(i)} e^(G_i - G_j) (k_j . k_i) u_j)     (without the delta rule u = v)
//   o_i = scale (e^(G_i) S0^T q_i + sum_{j in A(i) or j = i} e^(G_i - G_j) (k_j . q_i) u_j)
// which is the recurrence along each path from the state, with no state but S0 ever written down.
#include "gemm_common.h"

#include <algorithm>

namespace ojx {

namespace {

constexpr int kHD = 128;

__device__ __forceinline__ void load16(const uint16_t* p, float (&x)[16]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = bf2f(w[i] & 0xffffu);
    x[2 * i + 1] = bf2f(w[i] >> 16);
  }
}

// Thread t of 256 has value dims 4 (t % 32) .. + 3 of key dims 16 (t / 32) .. + 15. Sums over the key dims: two groups of a
// wave by a lane swap, the four waves through LDS (red: [4][32][NF + 3] floats, not in use by an earlier sum), in wave order.
template <int NF>
__device__ __forceinline__ void add_groups(float (&f)[NF], float* red) {
  constexpr int LD = NF + 3;
  const int wave = threadIdx.x >> 6, c = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < NF; ++i) f[i] += __shfl_xor(f[i], 32);
  if ((threadIdx.x & 32) == 0)
#pragma unroll
    for (int i = 0; i < NF; ++i) red[(wave * 32 + c) * LD + i] = f[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NF; ++i) {
    f[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) f[i] += red[(w * 32 + c) * LD + i];
  }
}

__device__ __forceinline__ void store4(uint16_t* o, float a, float b, float c, float d) {
  *reinterpret_cast<uint2*>(o) = make_uint2(pack2(a, b), pack2(c, d));
}

// Row by row, any tree: each row's ancestors from its parent upwards, their u from the workspace.
template <bool DELTA>
__global__ void __launch_bounds__(256) lintree_rows_k(LinTreeParams p) {
  __shared__ float red[4 * 32 * 12];
  const int64_t b = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(b * p.HV), hk = h / (p.HV / p.HK);
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  if (b == p.B) {  // rows of no sequence
    int lo, hi;
    seq_span(p.q_ptr, p.B, p.N, lo, hi);
    for (int64_t r = rg; r < p.N; r += 8)
      if (r < lo || r >= hi) *reinterpret_cast<uint2*>(p.o + (r * p.HV + h) * kHD + c * 4) = make_uint2(0u, 0u);
    return;
  }
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int64_t slot = p.slot[b];
  if (slot < 0 || slot >= p.slots) {
    const uint32_t x = slot < 0 ? 0u : 0x7fc07fc0u;
    for (int i = rg; i < at.n; i += 8)
      *reinterpret_cast<uint2*>(p.o + ((int64_t)(at.first + i) * p.HV + h) * kHD + c * 4) = make_uint2(x, x);
    return;
  }
  const float* const st = p.state + (slot * p.HV + h) * (kHD * kHD) + rg * 16 * kHD + c * 4;
  float4 s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const float4*>(st + i * kHD);
  for (int i = 0; i < at.n; ++i) {
    const int64_t row = at.first + i;
    float k[16], q[16], f[9];
    load16(p.k + (row * p.HK + hk) * kHD + rg * 16, k);
    load16(p.q + (row * p.HK + hk) * kHD + rg * 16, q);
#pragma unroll
    for (int x = 0; x < 9; ++x) f[x] = 0.f;
    // ancestors from the nearest on: the decay between them and this row grows with every one
    float fade = expf(p.g[row * p.HV + h]);
    int j = p.parents == nullptr ? i - 1 : p.parents[row];
    for (int below = i; j >= 0 && j < below;) {
      const int64_t a = at.first + j;
      float y[16], dk = 0.f, dq = 0.f;
      load16(p.k + (a * p.HK + hk) * kHD + rg * 16, y);
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        dk += y[x] * k[x];
        dq += y[x] * q[x];
      }
      const float4 u = *reinterpret_cast<const float4*>(p.u + (a * p.HV + h) * kHD + c * 4);
      dk *= fade;
      dq *= fade;
      f[0] += dk * u.x;
      f[1] += dk * u.y;
      f[2] += dk * u.z;
      f[3] += dk * u.w;
      f[4] += dq * u.x;
      f[5] += dq * u.y;
      f[6] += dq * u.z;
      f[7] += dq * u.w;
      fade *= expf(p.g[a * p.HV + h]);
      below = j;
      j = p.parents == nullptr ? j - 1 : p.parents[a];
    }
    float sk[4] = {}, sq[4] = {};
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      sk[0] += s[x].x * k[x];
      sk[1] += s[x].y * k[x];
      sk[2] += s[x].z * k[x];
      sk[3] += s[x].w * k[x];
      sq[0] += s[x].x * q[x];
      sq[1] += s[x].y * q[x];
      sq[2] += s[x].z * q[x];
      sq[3] += s[x].w * q[x];
      f[8] += q[x] * k[x];
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      f[x] += fade * sk[x];
      f[4 + x] += fade * sq[x];
    }
    add_groups(f, red);
    const uint2 vw = *reinterpret_cast<const uint2*>(p.v + (row * p.HV + h) * kHD + c * 4);
    float u[4] = {bf2f(vw.x & 0xffffu), bf2f(vw.x >> 16), bf2f(vw.y & 0xffffu), bf2f(vw.y >> 16)};
    if (DELTA) {
      const float beta = bf2f(p.beta[row * p.HV + h]);
#pragma unroll
      for (int x = 0; x < 4; ++x) u[x] = beta * (u[x] - f[x]);
    }
    if (rg == 0) {
      *reinterpret_cast<float4*>(p.u + (row * p.HV + h) * kHD + c * 4) = make_float4(u[0], u[1], u[2], u[3]);
      store4(p.o + (row * p.HV + h) * kHD + c * 4, p.scale * (f[4] + f[8] * u[0]), p.scale * (f[5] + f[8] * u[1]),
             p.scale * (f[6] + f[8] * u[2]), p.scale * (f[7] + f[8] * u[3]));
    }
    __syncthreads();
  }
}

// The kept tokens of sequence b, rows path[0 .. count - 1] of its own, through its state one after the other.
template <bool DELTA>
__global__ void __launch_bounds__(256) linattn_keep_k(LinTreeParams p) {
  __shared__ float red[2][4 * 32 * 7];
  const int64_t b = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(b * p.HV), hk = h / (p.HV / p.HK);
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = min(at.n, p.count[b]);
  const int64_t slot = p.slot[b];
  // A slot belongs to the first sequence that names it: two workgroups that update one state would race.
  bool twice = slot < 0 || slot >= p.slots;
  for (int64_t i = threadIdx.x; i < b; i += 256) twice |= p.slot[i] == slot;
  if (__syncthreads_or(twice) || n <= 0) return;
  float* const st = p.state + (slot * p.HV + h) * (kHD * kHD) + rg * 16 * kHD + c * 4;
  float4 s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const float4*>(st + i * kHD);
  for (int i = 0, turn = 0; i < n; ++i) {
    const int r = p.path[at.first + i];
    if (r < 0 || r >= at.n) continue;  // the same for the whole workgroup
    const int64_t row = at.first + r;
    float k[16], f[4] = {};
    load16(p.k + (row * p.HK + hk) * kHD + rg * 16, k);
    const uint2 vw = *reinterpret_cast<const uint2*>(p.v + (row * p.HV + h) * kHD + c * 4);
    const float a = expf(p.g[row * p.HV + h]);
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      s[x].x *= a;
      s[x].y *= a;
      s[x].z *= a;
      s[x].w *= a;
    }
    float u[4] = {bf2f(vw.x & 0xffffu), bf2f(vw.x >> 16), bf2f(vw.y & 0xffffu), bf2f(vw.y >> 16)};
    if (DELTA) {
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        f[0] += s[x].x * k[x];
        f[1] += s[x].y * k[x];
        f[2] += s[x].z * k[x];
        f[3] += s[x].w * k[x];
      }
      add_groups(f, red[turn]);
      turn ^= 1;
      const float beta = bf2f(p.beta[row * p.HV + h]);
#pragma unroll
      for (int x = 0; x < 4; ++x) u[x] = beta * (u[x] - f[x]);
    }
#pragma unroll
    for (int x = 0; x < 16; ++x) {
      s[x].x += k[x] * u[0];
      s[x].y += k[x] * u[1];
      s[x].z += k[x] * u[2];
      s[x].w += k[x] * u[3];
    }
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(st + i * kHD) = s[i];
}

}  // namespace

hipError_t launch_linattn_tree(const LinTreeParams& p, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? lintree_rows_k<true> : lintree_rows_k<false>,
                     dim3((unsigned)((p.B + 1LL) * p.HV)), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_linattn_keep(const LinTreeParams& p, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_keep_k<true> : linattn_keep_k<false>, dim3((unsigned)((int64_t)p.B * p.HV)),
                     dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

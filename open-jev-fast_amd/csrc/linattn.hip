// Linear attention with a decay for each head, over whole sequences (prompts) and for single tokens.
//
// A value head carries a state S [128 (key dims), 128 (value dims)]; token t has a key k, a query q, a value v, the
// logarithm g of its decay and, with the delta rule, a strength beta:
//   S <- e^g S;  u = beta (v - S^T k)  (without the delta rule u = v);  S <- S + k u^T;  o = scale S^T q
// Value head h reads key head h / (HV / HK).
#include "ojx_internal.h"

namespace ojx {

namespace {

constexpr int kHD = 128;

// Thread t of 256 holds value dims 4 (t % 32) .. + 3 of key dims 16 (t / 32) .. + 15. A token needs three sums over the
// key dims, S^T k, S^T q (both of the decayed state) and q . k, since the new state's S^T q is the decayed state's plus
// (q . k) u: they are added over the eight groups of threads in one go, two groups in a wave by a lane swap and the four
// waves through LDS, in wave order.
struct Token {
  float4 sk, sq;
  float qk;
};

__device__ __forceinline__ void token_sums(const float4 (&s)[16], const float (&k)[16], const float (&q)[16], Token& t) {
  t.sk = t.sq = make_float4(0.f, 0.f, 0.f, 0.f);
  t.qk = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    t.sk.x += s[i].x * k[i];
    t.sk.y += s[i].y * k[i];
    t.sk.z += s[i].z * k[i];
    t.sk.w += s[i].w * k[i];
    t.sq.x += s[i].x * q[i];
    t.sq.y += s[i].y * q[i];
    t.sq.z += s[i].z * q[i];
    t.sq.w += s[i].w * q[i];
    t.qk += q[i] * k[i];
  }
}

// red: [4][32][12] floats, not in use by an earlier token of any thread
__device__ __forceinline__ void add_groups(Token& t, float* red) {
  const int wave = threadIdx.x >> 6, c = threadIdx.x & 31;
  float* const f = reinterpret_cast<float*>(&t);
#pragma unroll
  for (int i = 0; i < 9; ++i) f[i] += __shfl_xor(f[i], 32);
  float* const r = red + (wave * 32 + c) * 12;
  if ((threadIdx.x & 32) == 0) {
    *reinterpret_cast<float4*>(r) = t.sk;
    *reinterpret_cast<float4*>(r + 4) = t.sq;
    r[8] = t.qk;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 9; ++i) f[i] = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w)
#pragma unroll
    for (int i = 0; i < 9; ++i) f[i] += red[(w * 32 + c) * 12 + i];
}

__device__ __forceinline__ void load16(const uint16_t* p, float (&x)[16]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p), b = *reinterpret_cast<const uint4*>(p + 8);
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    x[2 * i] = bf2f(w[i] & 0xffffu);
    x[2 * i + 1] = bf2f(w[i] >> 16);
  }
}

// One token through the state that the workgroup holds; the thread's four outputs.
template <bool DELTA>
__device__ __forceinline__ void one_token(const LinParams& p, int64_t row, int h, int hk, float4 (&s)[16], float* red,
                                          uint16_t* o) {
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  float k[16], q[16];
  load16(p.k + (row * p.HK + hk) * kHD + rg * 16, k);
  load16(p.q + (row * p.HK + hk) * kHD + rg * 16, q);
  const uint2 vw = *reinterpret_cast<const uint2*>(p.v + (row * p.HV + h) * kHD + c * 4);
  const float a = expf(p.g[row * p.HV + h]);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i].x *= a;
    s[i].y *= a;
    s[i].z *= a;
    s[i].w *= a;
  }
  Token t;
  token_sums(s, k, q, t);
  add_groups(t, red);
  float4 u = make_float4(bf2f(vw.x & 0xffffu), bf2f(vw.x >> 16), bf2f(vw.y & 0xffffu), bf2f(vw.y >> 16));
  if (DELTA) {
    const float b = bf2f(p.beta[row * p.HV + h]);
    u = make_float4(b * (u.x - t.sk.x), b * (u.y - t.sk.y), b * (u.z - t.sk.z), b * (u.w - t.sk.w));
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    s[i].x += k[i] * u.x;
    s[i].y += k[i] * u.y;
    s[i].z += k[i] * u.z;
    s[i].w += k[i] * u.w;
  }
  if (rg == 0)
    *reinterpret_cast<uint2*>(o + (row * p.HV + h) * kHD + c * 4) =
        make_uint2(pack2(p.scale * (t.sq.x + t.qk * u.x), p.scale * (t.sq.y + t.qk * u.y)),
                   pack2(p.scale * (t.sq.z + t.qk * u.z), p.scale * (t.sq.w + t.qk * u.w)));
}

// One workgroup per (row, value head).
template <bool DELTA>
__global__ void __launch_bounds__(256) linattn_step_k(LinParams p, float* state, const int32_t* __restrict__ slot) {
  __shared__ float red[4 * 32 * 12];
  const int64_t row = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(row * p.HV), hk = h / (p.HV / p.HK);
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const int64_t at = slot[row];
  // A slot belongs to the first row that names it: two workgroups that update one state would race.
  bool twice = at >= p.slots;
  for (int64_t i = threadIdx.x; i < row; i += 256) twice |= slot[i] == at;
  twice = at >= 0 && __syncthreads_or(twice);
  if (at < 0 || twice) {
    if (rg == 0) {
      const uint32_t x = at < 0 ? 0u : 0x7fc07fc0u;
      *reinterpret_cast<uint2*>(p.o + (row * p.HV + h) * kHD + c * 4) = make_uint2(x, x);
    }
    return;
  }
  float* const st = state + (at * p.HV + h) * (kHD * kHD) + rg * 16 * kHD + c * 4;
  float4 s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const float4*>(st + i * kHD);
  one_token<DELTA>(p, row, h, hk, s, red, p.o);
#pragma unroll
  for (int i = 0; i < 16; ++i) *reinterpret_cast<float4*>(st + i * kHD) = s[i];
}

// One workgroup per (sequence, value head), token after token; the workgroups behind the last sequence write zeros to the
// rows of no sequence.
template <bool DELTA>
__global__ void __launch_bounds__(256) linattn_prompt_k(LinParams p) {
  __shared__ float red[2][4 * 32 * 12];
  const int64_t sq = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(sq * p.HV), hk = h / (p.HV / p.HK);
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const auto ptr = [&](int64_t i) { return min(max((int64_t)p.seq_ptr[i], (int64_t)0), p.R); };
  if (sq == p.S) {
    const int64_t x = ptr(0), y = max(ptr(p.S), x);
    for (int64_t r = rg; r < x + (p.R - y); r += 8)
      *reinterpret_cast<uint2*>(p.o + ((r < x ? r : y + r - x) * p.HV + h) * kHD + c * 4) = make_uint2(0u, 0u);
    return;
  }
  float4 s[16];
  int64_t at = -1;
  if (p.state != nullptr) at = p.src != nullptr ? (int64_t)p.src[sq] : sq;
  const float fill = at >= p.slots ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    s[i] = at >= 0 && at < p.slots
               ? *reinterpret_cast<const float4*>(p.state + (at * p.HV + h) * (kHD * kHD) + (rg * 16 + i) * kHD + c * 4)
               : make_float4(fill, fill, fill, fill);
  const int64_t x = ptr(sq), y = max(ptr(sq + 1), x);
  for (int64_t r = x; r < y; ++r) one_token<DELTA>(p, r, h, hk, s, red[r & 1], p.o);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    *reinterpret_cast<float4*>(p.state_out + (sq * p.HV + h) * (kHD * kHD) + (rg * 16 + i) * kHD + c * 4) = s[i];
}

}  // namespace

hipError_t launch_linattn_step(const LinParams& p, float* state, const int32_t* slot, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_step_k<true> : linattn_step_k<false>, dim3((unsigned)(p.R * p.HV)),
                     dim3(256), 0, st, p, state, slot);
  return hipGetLastError();
}

hipError_t launch_linattn_prompt(const LinParams& p, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_prompt_k<true> : linattn_prompt_k<false>,
                     dim3((unsigned)((p.S + 1) * p.HV)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

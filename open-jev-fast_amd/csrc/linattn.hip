// Linear attention with a decay for each head, over whole sequences (prompts) and for single tokens.
//
// A value head carries a state S [128 (key dims), 128 (value dims)]; token t has a key k, a query q, a value v, the
// logarithm g of its decay and, with the delta rule, a strength beta:
//   S <- e^g S;  u = beta (v - S^T k)  (without the delta rule u = v);  S <- S + k u^T;  o = scale S^T q
// Value head h reads key head h / (HV / HK).
#include "gemm_common.h"

#include <algorithm>
#include <atomic>
#include <cstddef>

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

// One workgroup per (row, value head). What bounds it: the states, read and written once (64 rows of 48 heads, 403 MB:
// 82.7 us, 4.9 TB/s, where a large copy reaches 5.2); for one row the chain of a state's load, three sums and its store, 5 us.
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

// ------------------------------------------------------------------------------------------------------------- prompts
// A chunk of C = 64 tokens at once. With G_i the sum of g up to token i of the chunk and S0 the state before it,
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  P_ij = e^(G_i - G_j) q_i . k_j (j <= i),  T = (I + A)^-1 diag(beta),
//   X = V - diag(e^G) K S0,  U = T X,
//   O = scale (diag(e^G) Q S0 + P U),  S = e^(G_C) S0 + K^T diag(e^(G_C - G)) U;
// without the delta rule U = V. T and P need no state: linattn_chunk_k makes, for all chunks at once, scale P T and
// diag(e^(G_C - G)) T, the two products in which T is used. linattn_prompt_k then goes through a sequence's chunks in order.
//
// Precision. The states are fp32, and so is what makes them: a factor that is not a bf16 input (S0, X, U, the products with
// T) enters the products that make states as three bf16 pieces, which hold all of an fp32, and leave out what is 2^-24 of
// the result. The states come out 1e-7 off 64 bits, relative to their norm, after 288 tokens as after 16384 (torch's fp32
// products: 1.2e-7; with two pieces: 5e-6, and 637 us for 16384 tokens in place of 758, 163 for 16 x 539 in place of 190).
// Outputs are rounded to bf16, half a step of 2^-8: what only they meet (S0 with Q, P T, X with P T) enters in two pieces.
// Differences of G are taken in 64 bits before they are rounded: after a long decay G is large, and its fp32 steps would
// show in e^(G_i - G_j).
// A chunk with a value that is not finite, or a decay above 1, goes token by token (the same recurrence), so that nothing
// reaches the tokens before it: in the products a zero above the diagonal times NaN would.

constexpr int kChunk = 64;
constexpr float kMinDecay = -200.f;  // e^-200 is 0 in fp32: -infinity does no worse, and differences of sums stay numbers

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(4))) const int32_t* const_ints;

// Rows t0 .. t0 + cnt - 1 of one head of x [R, heads, 128] as a buffer: rows behind them read as zeros, and what is stored
// there goes nowhere, without a branch.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_rows(const void* x, int64_t t0, int cnt, int heads, int h) {
  return make_rsrc(static_cast<const uint16_t*>(x) + (t0 * heads + h) * kHD, ((int64_t)(cnt - 1) * heads + 1) * kHD * 2);
}

// What a chunk of a head leaves for linattn_prompt_k, in the order in which it goes to LDS. The matrices are A operands of
// 16 x 32 products, one lane's 8 values after the other, piece by piece: operand (it, ks) covers tokens 16 it .. + 15 against
// tokens 32 ks .. + 31, the latter in the order in which a lane holds the other factor: 4 of the first 16, 4 of the
// second. Those above the diagonal are left out: (0, 0), (1, 0), (2, 0), (2, 1), (3, 0), (3, 1) are here.
struct ChunkWork {
  float from[kChunk], out[kChunk], to[kChunk];  // e^G, scale e^G, e^(G_C - G)
  float all;                                    // e^(G_C)
  int32_t odd;                                  // token by token
  int32_t pad[62];
  uint16_t P[2][6][64][8];                      // scale P T (without the delta rule scale P)
  uint16_t T[3][6][64][8];                      // diag(to) T; the delta rule's last part
};
static_assert(offsetof(ChunkWork, P) == 1024, "whole 1-KB pieces");
constexpr int chunk_bytes(bool delta) { return delta ? (int)sizeof(ChunkWork) : (int)offsetof(ChunkWork, T); }
__device__ __forceinline__ constexpr int frag(int it, int ks) { return it < 2 ? it : 2 * it - 2 + ks; }

__device__ __forceinline__ int seq_chunks(int, int n) { return (n + kChunk - 1) / kChunk; }

// x and y less a pair of bf16.
__device__ __forceinline__ void less_pair(float& x, float& y, uint32_t pair) {
  x -= __uint_as_float(pair << 16);
  y -= __uint_as_float(pair & 0xffff0000u);
}
// bf16 pieces of 8 values: hi + lo is x to 16 bits, with low all of an fp32's 24.
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& lo, bf16x8& low) {
  uint32_t h[4], l[4], m[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
    h[i] = cvt_pk2(x, y);
    less_pair(x, y, h[i]);
    l[i] = cvt_pk2(x, y);
    less_pair(x, y, l[i]);
    m[i] = cvt_pk2(x, y);
  }
  hi = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
  lo = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
  low = __builtin_bit_cast(bf16x8, make_uint4(m[0], m[1], m[2], m[3]));
}
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& lo) {
  bf16x8 low;  // not asked for, not computed
  split8(a, b, hi, lo, low);
}
__device__ __forceinline__ f32x4 widen(bf16x4 x) {
  const uint2 v = __builtin_bit_cast(uint2, x);
  return f32x4{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16),
               __uint_as_float(v.y & 0xffff0000u)};
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// 16-byte piece x of a row r of K or Q lies at x ^ swizzle(r) in LDS: the reads of 16 rows' pieces, and the transposing ones
// of 4 pieces of 8 rows, then spread over the banks.
__device__ __forceinline__ constexpr int swizzle(int r) { return (r & 7) << 1 | (r >> 3 & 1); }

// The sum of x over the lanes up to and including this one, in 64 bits, by lane shifts within rows of 16 and the rows' last
// lanes handed on (a lane outside reads as zero).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0u, (uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0u, (uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double scan64(double x) {
  x = dpp_add<0x111, 0xf>(x);  // row_shr 1, 2, 4, 8
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // row_bcast 15 to rows 1 and 3, 31 to rows 2 and 3
  x = dpp_add<0x143, 0xc>(x);
  return x;
}
// The largest magnitude of bf16 bits, two at a time.
__device__ __forceinline__ uint32_t top2(uint32_t top, uint32_t x) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top),
                                                                __builtin_bit_cast(u16x2, x & 0x7fff7fffu)));
}
__device__ __forceinline__ uint32_t top8(uint32_t top, bf16x8 x) {
  const uint4 u = __builtin_bit_cast(uint4, x);
  return top2(top2(top2(top2(top, u.x), u.y), u.z), u.w);
}
__device__ __forceinline__ bool odd_top(uint32_t top) { return (top & 0xffffu) >= 0x7f80u || top >= 0x7f800000u; }

// T and P of one chunk and value head; wave w has the tokens 16 w .. + 15 as rows.
//   * k . k and q . k on bf16 MFMA from the rows as they lie in memory;
//   * (I + A)^-1 in blocks of 16: the diagonal ones by forward substitution, a column a lane; then block column w by wave
//     w, T_iw = -T_ii (sum_k A_ik T_kw), on fp32 MFMA (16x16x4), whose B operand is the accumulator of the product before
//     when the contraction runs in its order; P T likewise.
// LDS holds the ten lower blocks of each matrix, rows of 20 floats (so that 16 rows' 16-byte reads meet every bank once).
// What bounds it: the chain of one chunk (loads, scan, substitution, up to 19 block products on one wave), so what counts
// is how many workgroups a CU holds: four, by LDS and registers (16384 tokens of 48 heads: 160 us; with two 206 against 155
// before; MFMAs busy 16-19% of the time, waves waiting half of theirs). A single round of them takes 11 us: 288 tokens.
template <bool DELTA>
__global__ void __launch_bounds__(256, 4) linattn_chunk_k(LinParams p) {
  constexpr int LD = 20, BLK = 16 * LD;
  const auto lower = [](int i, int k) { return (i * (i + 1) / 2 + k) * BLK; };
  __shared__ __attribute__((aligned(16))) float mem[DELTA ? 24 * BLK : 64 * 64];
  float* const Pb = mem;              // ten blocks
  float* const Ab = mem + 10 * BLK;   // ten blocks
  float* const Db = mem + 20 * BLK;   // four
  uint8_t* const Kb = reinterpret_cast<uint8_t*>(mem);  // before them: the chunk's rows of K
  __shared__ double Gs[4][64];  // every wave's own
  __shared__ float to_end[64];
  __shared__ int odd_at;
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t chunk = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(chunk * p.HV), hk = h / (p.HV / p.HK);
  SeqPlace at;
  if (!seq_find(p.seq_ptr, p.S, p.R, seq_chunks, [=](int, int upto) { return upto > (int)chunk; }, at)) return;
  const int t0 = at.first + ((int)chunk - at.before) * kChunk, cnt = min(kChunk, at.first + at.n - t0);
  ChunkWork* const out = reinterpret_cast<ChunkWork*>(p.work + (chunk * p.HV + h) * (int64_t)chunk_bytes(DELTA));

  const __amdgpu_buffer_rsrc_t kr = head_rows(p.k, t0, cnt, p.HK, hk), qr = head_rows(p.q, t0, cnt, p.HK, hk);
  bf16x8 ka[4], qa[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    const uint32_t x = (uint32_t)(w * 16 + c) * (p.HK * kHD * 2) + s * 64 + g * 16;
    ka[s] = __builtin_bit_cast(bf16x8, bload(kr, x));
    qa[s] = __builtin_bit_cast(bf16x8, bload(qr, x));
  }
  // a token a lane: decays, to base two, and strengths; tokens behind the end add nothing
  const int64_t tok = (int64_t)(t0 + min(lane, cnt - 1)) * p.HV + h;
  float gv = p.g[tok], beta = DELTA ? bf2f(p.beta[tok]) : 0.f;
  if (lane >= cnt) gv = beta = 0.f;
  bool odd = !(gv <= 0.f) || !(fabsf(beta) < INFINITY);
  gv = gv < kMinDecay ? kMinDecay : gv;
  const double G = scan64((double)gv * 1.4426950408889634074);
  Gs[w][lane] = G;
  if (w == 0) {
    const double last = Gs[0][63];
    to_end[lane] = __builtin_amdgcn_exp2f((float)(last - G));
    if (lane == 0) odd_at = 0;
  }
  uint32_t top = 0;
  int koff[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    koff[s] = c * 256 + ((s * 4 + g) ^ swizzle(c)) * 16;
    *reinterpret_cast<bf16x8*>(Kb + w * 4096 + koff[s]) = ka[s];
    top = top8(top8(top, ka[s]), qa[s]);
  }
  odd |= odd_top(top);
  __syncthreads();
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    kk[jt] = qk[jt] = f32x4{};
    if (jt > w) continue;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8 kb = *reinterpret_cast<const bf16x8*>(Kb + jt * 4096 + koff[s]);
      if (DELTA) kk[jt] = mfma(ka[s], kb, kk[jt]);
      qk[jt] = mfma(qa[s], kb, qk[jt]);
    }
  }
  __syncthreads();  // K has been read

  double Gi[4];
  float bi[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    Gi[r] = Gs[w][w * 16 + g * 4 + r];
    bi[r] = DELTA ? __shfl(beta, w * 16 + g * 4 + r) : 0.f;
  }
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    if (jt > w) continue;
    const double Gj = Gs[w][jt * 16 + c];
    f32x4 a;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = w * 16 + g * 4 + r, j = jt * 16 + c;
      const float e = j <= i ? __builtin_amdgcn_exp2f((float)(Gi[r] - Gj)) : 0.f;
      Pb[lower(w, jt) + (g * 4 + r) * LD + c] = j <= i ? e * qk[jt][r] : 0.f;
      a[r] = DELTA && j < i ? bi[r] * (e * kk[jt][r]) : 0.f;
      if (DELTA && jt < w) Ab[lower(w, jt) + (g * 4 + r) * LD + c] = a[r];
    }
    if (DELTA && jt == w) *reinterpret_cast<f32x4*>(Db + w * BLK + c * LD + g * 4) = a;  // columns of A as rows
  }
  if (DELTA) {
    // column c of the diagonal block's inverse: a row known, its multiples leave the rows below
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = i == c ? 1.f : 0.f;
#pragma unroll
    for (int i = 0; i < 15; ++i)
#pragma unroll
      for (int q = (i + 1) / 4; q < 4; ++q) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(Db + w * BLK + i * LD + q * 4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (q * 4 + r > i) x[q * 4 + r] -= a[r] * x[i];
      }
    if (g == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) Ab[lower(w, w) + i * LD + c] = x[i];
    __syncthreads();
    f32x4 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = f32x4{};
      if (i == w) {
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i][r] = Ab[lower(i, i) + (g * 4 + r) * LD + c];
      } else if (i > w) {
        f32x4 sum{}, neg{};
#pragma unroll
        for (int k = 0; k < i; ++k) {
          if (k < w) continue;
          const f32x4 a = *reinterpret_cast<const f32x4*>(Ab + lower(i, k) + c * LD + g * 4);
#pragma unroll
          for (int s = 0; s < 4; ++s) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], t[k][s], sum, 0, 0, 0);
        }
        const f32x4 a = *reinterpret_cast<const f32x4*>(Ab + lower(i, i) + c * LD + g * 4);
#pragma unroll
        for (int s = 0; s < 4; ++s) neg = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], sum[s], neg, 0, 0, 0);
        t[i] = -neg;
      }
    }
    // P T and diag(to) T, block column w
    const float bj = __shfl(beta, w * 16 + c);
    f32x4 pt[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] *= bj;
      pt[i] = f32x4{};
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k < w) continue;
#pragma unroll
      for (int i = k; i < 4; ++i) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(Pb + lower(i, k) + c * LD + g * 4);
#pragma unroll
        for (int s = 0; s < 4; ++s) pt[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], t[k][s], pt[i], 0, 0, 0);
      }
    }
    __syncthreads();  // A, P and the diagonal blocks have been read
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i < w) continue;
      const f32x4 e = *reinterpret_cast<const f32x4*>(to_end + i * 16 + g * 4);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        odd |= !(fabsf(t[i][r]) + fabsf(pt[i][r]) < INFINITY);
        Ab[lower(i, w) + (g * 4 + r) * LD + c] = t[i][r] * e[r];
        Pb[lower(i, w) + (g * 4 + r) * LD + c] = pt[i][r];
      }
    }
  }
  if (!DELTA) __syncthreads();
  if (__any(odd) && lane == 0) atomicOr(&odd_at, 1);
  __syncthreads();
  // operands: row w, the tokens of two tiles; the one above the diagonal is zeros
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (ks > (w >> 1)) continue;
    const bool both = 2 * ks + 1 <= w;
    const int x = lower(w, 2 * ks) + c * LD + g * 4, y = both ? lower(w, 2 * ks + 1) + c * LD + g * 4 : x;
    const float on = both ? p.scale : 0.f;
    bf16x8 hi, lo;
    split8(*reinterpret_cast<const f32x4*>(Pb + x) * p.scale, *reinterpret_cast<const f32x4*>(Pb + y) * on, hi, lo);
    *reinterpret_cast<bf16x8*>(out->P[0][frag(w, ks)][lane]) = hi;
    *reinterpret_cast<bf16x8*>(out->P[1][frag(w, ks)][lane]) = lo;
    if (DELTA) {
      bf16x8 low;
      split8(*reinterpret_cast<const f32x4*>(Ab + x), *reinterpret_cast<const f32x4*>(Ab + y) * (both ? 1.f : 0.f), hi, lo, low);
      *reinterpret_cast<bf16x8*>(out->T[0][frag(w, ks)][lane]) = hi;
      *reinterpret_cast<bf16x8*>(out->T[1][frag(w, ks)][lane]) = lo;
      *reinterpret_cast<bf16x8*>(out->T[2][frag(w, ks)][lane]) = low;
    }
  }
  if (w != 0) return;
  const float e = __builtin_amdgcn_exp2f((float)G);
  out->from[lane] = e;
  out->out[lane] = p.scale * e;
  out->to[lane] = to_end[lane];
  if (lane == 63) {
    out->all = e;
    out->odd = odd_at;
  }
}

// Zeros in value head h of the rows of no sequence.
__device__ __forceinline__ void zero_rows(const LinParams& p, int h) {
  int lo, hi;
  seq_span(p.seq_ptr, p.S, p.R, lo, hi);
  for (int64_t r = threadIdx.x >> 4; r < lo + (p.R - hi); r += blockDim.x >> 4)
    *reinterpret_cast<uint4*>(p.o + ((r < lo ? r : r - lo + hi) * p.HV + h) * kHD + (threadIdx.x & 15) * 8) =
        make_uint4(0u, 0u, 0u, 0u);
}

// The chunks of one sequence and value head in order. A slice is 16 value dims of the state with all 128 key dims: 8
// accumulators, d of them with key dims key_dim(d, g) .. + 3 in the lanes (c, g) of value dim c. Two of them together are
// then the B operand of K S0 and Q S0 for 32 key dims in order, and nothing of the state, of X or of U has to change its
// lane. A workgroup takes two slices with two waves each:
//   * the slice's first wave has the state: X, U, the new state. This is the chain that bounds a long sequence (a chunk's
//     products wait for each other, and the next chunk for this one), so nothing else is on it;
//   * the second has the rest: the outputs, from the pieces of S0 and X that the first hands over through LDS, and the DMAs.
// K, Q, V and the chunk's matrices come to LDS one chunk ahead. K^T and V's columns are read transposed from the rows (16
// lanes get 4 rows x 16 columns column by column, the columns in any groups of 4). Two barriers a chunk: S0's pieces and
// the stage are there; X's pieces are there.
__device__ __forceinline__ constexpr int key_dim(int d, int g) { return (d >> 1) * 32 + g * 8 + (d & 1) * 4; }

// x = the 64 rows at `rows` (aoff: a lane's place in a row of 16 for key dims 32 s ..) times the state's pieces, sp[0] the
// largest; the others are summed apart, so that only sp[0]'s sums round at the size of the result. Products on one
// accumulator follow each other with others between them: one waits for the one before on its accumulator twice as long as
// it occupies the unit.
template <int PIECES>
__device__ __forceinline__ void rows_times(const uint8_t* rows, const int (&aoff)[4], const bf16x8 (&sp)[PIECES][4],
                                           f32x4 (&x)[4]) {
  f32x4 rest[4];
#pragma unroll
  for (int it = 0; it < 4; ++it) x[it] = rest[it] = f32x4{};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    bf16x8 a[4];
#pragma unroll
    for (int it = 0; it < 4; ++it) a[it] = *reinterpret_cast<const bf16x8*>(rows + it * 4096 + aoff[s]);
#pragma unroll
    for (int part = 0; part < PIECES; ++part)
#pragma unroll
      for (int it = 0; it < 4; ++it) {
        f32x4& to = PIECES > 2 && part > 0 ? rest[it] : x[it];
        to = mfma(a[it], sp[part][s], to);
      }
  }
#pragma unroll
  for (int it = 0; it < 4; ++it)
    if (PIECES > 2) x[it] += rest[it];
}

// x += P b for the outputs, P a chunk's lower triangular matrix in two pieces, b in two (lo lo is left out) or, exact, in one.
template <bool TWO, int PIECES>
__device__ __forceinline__ void lower_times(const uint16_t (&m)[2][6][64][8], int lane, const bf16x8 (&b)[PIECES][2],
                                            f32x4 (&x)[4]) {
#pragma unroll
  for (int part = 0; part < 2; ++part)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      bf16x8 a[4];
#pragma unroll
      for (int it = 2 * k; it < 4; ++it) a[it] = *reinterpret_cast<const bf16x8*>(m[part][frag(it, k)][lane]);
#pragma unroll
      for (int piece = 0; piece < (TWO && part == 0 ? 2 : 1); ++piece)
#pragma unroll
        for (int it = 2 * k; it < 4; ++it) x[it] = mfma(a[it], b[piece][k], x[it]);
    }
}

// u = T X, both in three pieces: the products of pieces down to 2^-16 of the largest, that one summed apart from the others.
__device__ __forceinline__ void strengths_times(const uint16_t (&T)[3][6][64][8], int lane, const bf16x8 (&xp)[3][2],
                                                f32x4 (&u)[4]) {
  f32x4 rest[4];
#pragma unroll
  for (int it = 0; it < 4; ++it) u[it] = rest[it] = f32x4{};
#pragma unroll
  for (int part = 0; part < 3; ++part)
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      bf16x8 a[4];
#pragma unroll
      for (int it = 2 * k; it < 4; ++it) a[it] = *reinterpret_cast<const bf16x8*>(T[part][frag(it, k)][lane]);
#pragma unroll
      for (int piece = 0; piece < 3 - part; ++piece)
#pragma unroll
        for (int it = 2 * k; it < 4; ++it) {
          f32x4& to = part + piece > 0 ? rest[it] : u[it];
          to = mfma(a[it], xp[piece][k], to);
        }
    }
#pragma unroll
  for (int it = 0; it < 4; ++it) u[it] += rest[it];
}

// The state that sequence sq starts from: value dim dv, this lane's key dims.
__device__ __forceinline__ void load_state(const LinParams& p, int64_t sq, int h, int g, int dv, f32x4 (&st)[8]) {
  int64_t at = -1;
  if (p.state != nullptr) at = p.src != nullptr ? (int64_t)p.src[sq] : sq;
  if (at >= 0 && at < p.slots) {
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) st[d][r] = p.state[(at * p.HV + h) * (kHD * kHD) + (key_dim(d, g) + r) * kHD + dv];
  } else {
    const float fill = at >= p.slots ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) st[d] = f32x4{fill, fill, fill, fill};
  }
}
__device__ __forceinline__ void store_state(const LinParams& p, int64_t sq, int h, int g, int dv, const f32x4 (&st)[8]) {
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      p.state_out[(sq * p.HV + h) * (kHD * kHD) + (key_dim(d, g) + r) * kHD + dv] = st[d][r];
}

// cnt tokens from row t0 one by one, K and Q from LDS: state and outputs.
template <bool DELTA>
__device__ __forceinline__ void by_tokens(const LinParams& p, const uint8_t* krows, const uint8_t* qrows, int64_t t0, int cnt,
                                          int h, int g, int dv, f32x4 (&st)[8]) {
#pragma unroll 1
  for (int t = 0; t < cnt; ++t) {
    const int64_t row = (t0 + t) * p.HV + h;
    const float a = expf(p.g[row]), b = DELTA ? bf2f(p.beta[row]) : 1.f;
    bf16x4 k[8], q[8];
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      const int at = t * 256 + (((d >> 1) * 4 + g) ^ swizzle(t & 15)) * 16 + (d & 1) * 8;
      k[d] = *reinterpret_cast<const bf16x4*>(krows + at);
      q[d] = *reinterpret_cast<const bf16x4*>(qrows + at);
    }
    float u = bf2f(p.v[row * kHD + dv]), x = 0.f, o = 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      st[d] *= a;
#pragma unroll
      for (int r = 0; r < 4; ++r) x += st[d][r] * (float)k[d][r];
    }
    x += __shfl_xor(x, 16);
    x += __shfl_xor(x, 32);
    if (DELTA) u = b * (u - x);
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        st[d][r] += (float)k[d][r] * u;
        o += st[d][r] * (float)q[d][r];
      }
    o += __shfl_xor(o, 16);
    o += __shfl_xor(o, 32);
    if (g == 0) p.o[row * kHD + dv] = (uint16_t)f2bf(p.scale * o);
  }
}

// A chunk's outputs in value dim dv; rows: its rows of head h.
__device__ __forceinline__ void store_out(const LinParams& p, __amdgpu_buffer_rsrc_t rows, int g, int dv,
                                          const f32x4 (&x)[4]) {
#pragma unroll
  for (int it = 0; it < 4; ++it)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      __builtin_amdgcn_raw_buffer_store_b16((uint16_t)f2bf(x[it][r]), rows,
                                            (uint32_t)(it * 16 + g * 4 + r) * (p.HV * kHD * 2) + dv * 2, 0, 0);
}

__device__ __forceinline__ bf16x8 join(bf16x4 a, bf16x4 b) {
  return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ __forceinline__ bool odd_values(const bf16x4 (&v)[4]) {  // one of them is not finite
  uint32_t top = 0;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const uint2 x = __builtin_bit_cast(uint2, v[it]);
    top = top2(top2(top, x.x), x.y);
  }
  return odd_top(top);
}

// Every wave's LDS reads of the stage before are done, and what its own wait has seen land is there for all; global loads
// and DMAs stay in flight.
__device__ __forceinline__ void stage_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Few sequences: four workgroups a sequence and value head, each of two slices of 16 value dims, and for each slice a wave
// with the state in its accumulators and a wave for the outputs and the DMAs, which works a chunk behind: the chain of a
// chunk's products that need the state is all that the chunks wait for.
// What bounds it: that chain, 2.4 us a chunk (16384 tokens of 48 heads: 600 us; with two pieces a factor 509, and over 800
// with all of a slice in one wave): products that wait for each other, and the splits between them; MFMAs are busy 19% of the
// time.
template <bool DELTA>
__global__ void __launch_bounds__(256, 1) linattn_prompt_k(LinParams p) {
  constexpr int SL = 4;                  // workgroups of a head
  constexpr int VB = 64;                 // bytes of a V row: the workgroup's 32 value dims
  constexpr int WB = chunk_bytes(DELTA);
  constexpr int KO = WB, QO = KO + kChunk * 256, VO = QO + kChunk * 256, STAGE = VO + kChunk * VB;
  constexpr int SO = 2 * STAGE, XO = SO + 2 * 8192, FO = XO + 2 * 4096;  // handed over: S0's pieces, X's, token by token
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), slice = wave & 1;
  // Workgroups go to the eight XCDs in turn. Of 32, the four of a head are eight apart: one L2 serves them (16384 tokens, with
  // two pieces a factor: 682 -> 638 us, 1369 -> 459 MB read; with three 516 MB), and the heads still take the XCDs in turn,
  // so that sequences of unlike lengths share them
  const uint32_t b = blockIdx.x, whole = (uint32_t)p.S * p.HV / 8 * (8 * SL);
  const uint32_t wg = b < whole ? (b / (8 * SL) * 8 + b % 8) * SL + b / 8 % SL : b;
  const int64_t sq = wg / (p.HV * SL);
  const int hs = wg - (int)(sq * p.HV * SL), h = hs / SL, hk = h / (p.HV / p.HK);
  if (sq == p.S) {
    if (hs % SL == 0) zero_rows(p, h);
    return;
  }
  SeqPlace place;
  if (!seq_find(p.seq_ptr, p.S, p.R, seq_chunks, [=](int i, int) { return i == (int)sq; }, place)) return;
  const int first = place.first, n = place.n;
  const int chunks = seq_chunks(0, n);
  const int dv0 = (hs % SL) * 32, dv = dv0 + slice * 16 + c;
  // LDS offsets of this lane: rows c of K and Q, key dims 32 s .. + 31; its slice's pieces of S0 and X
  int aoff[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) aoff[s] = c * 256 + ((s * 4 + g) ^ swizzle(c)) * 16;
  bf16x8* const s0 = reinterpret_cast<bf16x8*>(smem + SO + slice * 8192) + lane;
  bf16x8* const x0 = reinterpret_cast<bf16x8*>(smem + XO + slice * 4096) + lane;
  int32_t* const by_token = reinterpret_cast<int32_t*>(smem + FO) + slice;

  if (wave >= 2) {
    // ------------------------------------------------------------------------------------------ DMAs and outputs
    const int64_t next_work = (int64_t)p.HV * WB;
    const uint8_t* const work = p.work + ((int64_t)place.before * p.HV + h) * (int64_t)WB;
    uint32_t koff[4];  // rows 4 i + g of 16
#pragma unroll
    for (int i = 0; i < 4; ++i) koff[i] = (uint32_t)(4 * i + g) * (p.HK * kHD * 2) + (c ^ swizzle(4 * i + g)) * 16;
    const uint32_t voff = (uint32_t)(lane >> 2) * (p.HV * kHD * 2) + (lane & 3) * 16;
    // quarter i of the chunk that begins at token t: 16 rows of K, Q and V, a part of the matrices, between the two waves
    const auto fetch = [&](int i, int t, uint8_t* stage) {
      const int cnt = min(kChunk, n - t);
      const __amdgpu_buffer_rsrc_t kr = head_rows(p.k, first + t, cnt, p.HK, hk);
      const __amdgpu_buffer_rsrc_t qr = head_rows(p.q, first + t, cnt, p.HK, hk);
      const __amdgpu_buffer_rsrc_t vr = make_rsrc(p.v + ((int64_t)(first + t) * p.HV + h) * kHD + dv0,
                                                  ((int64_t)(cnt - 1) * p.HV * kHD + 32) * 2);
      const __amdgpu_buffer_rsrc_t wr = make_rsrc(work + (int64_t)(t / kChunk) * next_work, WB);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = (uint32_t)(i * 16) * (p.HK * kHD * 2) + koff[j];
        dma16(slice == 0 ? kr : qr, stage + (slice == 0 ? KO : QO) + i * 4096 + j * 1024, at);
      }
      if (slice == (i & 1)) dma16(vr, stage + VO + i * 1024, (uint32_t)(i * 16) * (p.HV * kHD * 2) + voff);
      constexpr int PW = (WB / 1024 + 1) / 2;  // pieces of the matrices a wave
#pragma unroll
      for (int j = i; j < PW; j += 4) {
        const int at = min(j * 2 + slice, WB / 1024 - 1) * 1024;  // past the last piece: that one again
        dma16(wr, stage + at, at + lane * 16);
      }
    };
    if (chunks > 0)
#pragma unroll
      for (int i = 0; i < 4; ++i) fetch(i, 0, smem);
    for (int ch = 0; ch < chunks; ++ch) {
      const int t0 = ch * kChunk, cnt = min(kChunk, n - t0);
      const uint8_t* const stage = smem + (ch & 1) * STAGE;
      const ChunkWork& cw = *reinterpret_cast<const ChunkWork*>(stage);
      if (ch > 0)
        wait_vmcnt<16>();  // all but the last chunk's output stores
      else
        wait_vmcnt<0>();
      stage_barrier();
      const bool more = ch + 1 < chunks;
      uint8_t* const other = smem + ((ch + 1) & 1) * STAGE;
      bf16x8 sp[2][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        sp[0][s] = s0[(2 * s) * 64];
        sp[1][s] = s0[(2 * s + 1) * 64];
      }
      // the next chunk's DMAs, in two lots: all at once they would hold up the wave
      if (more) {
        fetch(0, t0 + kChunk, other);
        fetch(1, t0 + kChunk, other);
      }
      f32x4 x[4];
      rows_times(stage + QO, aoff, sp, x);
#pragma unroll
      for (int it = 0; it < 4; ++it) x[it] *= *reinterpret_cast<const f32x4*>(cw.out + it * 16 + g * 4);
      if (more) {
        fetch(2, t0 + kChunk, other);
        fetch(3, t0 + kChunk, other);
      }
      stage_barrier();
      if (*by_token != 0) {  // the first wave writes the outputs
        wait_vmcnt<0>();
        continue;
      }
      bf16x8 xp[2][2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        xp[0][k] = x0[(2 * k) * 64];
        if (DELTA) xp[1][k] = x0[(2 * k + 1) * 64];
      }
      lower_times<DELTA>(cw.P, lane, xp, x);
      store_out(p, head_rows(p.o, first + t0, cnt, p.HV, h), g, dv, x);
    }
    return;
  }

  // -------------------------------------------------------------------------------------------------- the state
  f32x4 st[8];
  load_state(p, sq, h, g, dv, st);
  int toff[4];  // K's rows read transposed, key dims 32 s .. + 31
  const int trow = g * 4 + (c >> 2);
#pragma unroll
  for (int s = 0; s < 4; ++s) toff[s] = KO + trow * 256 + ((s * 4 + (c & 3)) ^ swizzle(trow)) * 16;
  const int vtoff = VO + trow * VB + slice * 32 + (c & 3) * 8;
  // Every step is taken in halves, so that one half's conversions run behind the other's products; products on one
  // accumulator are two apart (one waits for the one before it twice as long as it occupies the unit); what the second part
  // of a chunk reads from LDS is read in the first.
  bf16x8 sp[3][4];
  const auto split_state = [&](int s) { split8(st[2 * s], st[2 * s + 1], sp[0][s], sp[1][s], sp[2][s]); };
#pragma unroll
  for (int s = 0; s < 4; ++s) split_state(s);
  for (int ch = 0; ch < chunks; ++ch) {
    const int t0 = ch * kChunk, cnt = min(kChunk, n - t0);
    const uint8_t* const stage = smem + (ch & 1) * STAGE;
    const ChunkWork& cw = *reinterpret_cast<const ChunkWork*>(stage);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      s0[(2 * s) * 64] = sp[0][s];
      s0[(2 * s + 1) * 64] = sp[1][s];
    }
    stage_barrier();
    const auto tr = [](const uint8_t* a) {
      return __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)a);
    };
    // The order of the reads from LDS is fixed (sched_barrier): each goes out while the products before its use run.
    f32x4 x[4], from[4], to[4];
    bf16x8 ka[2][4][2], T[3][6];
    bf16x4 vt[4], kt[8][4];  // V's columns (X's accumulators' places); K^T: accumulator d's key dims, tokens 16 t + 4 g ..
    if (DELTA) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            ka[half][s][e] = *reinterpret_cast<const bf16x8*>(stage + KO + half * 8192 + e * 4096 + aoff[s]);
    }
    const auto keys_times_state = [&](int half) {
      f32x4 sum[2][2]{};  // the largest piece's products, the others'
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int part = 0; part < 3; ++part)
#pragma unroll
          for (int e = 0; e < 2; ++e) sum[part > 0][e] = mfma(ka[half][s][e], sp[part][s], sum[part > 0][e]);
#pragma unroll
      for (int e = 0; e < 2; ++e) x[2 * half + e] = sum[0][e] + sum[1][e];
    };
    __builtin_amdgcn_sched_barrier(0);
    if (DELTA) keys_times_state(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int it = 0; it < 4; ++it) {
      vt[it] = tr(stage + vtoff + it * 16 * VB);
      if (DELTA)
        from[it] = *reinterpret_cast<const f32x4*>(cw.from + it * 16 + g * 4);
      else
        to[it] = *reinterpret_cast<const f32x4*>(cw.to + it * 16 + g * 4);
    }
    const int odd = cw.odd;
    const float all = cw.all;
    __builtin_amdgcn_sched_barrier(0);
    if (DELTA) keys_times_state(1);
    __builtin_amdgcn_sched_barrier(0);
    if (DELTA) {
#pragma unroll
      for (int f = 0; f < 6; ++f)
#pragma unroll
        for (int part = 0; part < 3; ++part) T[part][f] = *reinterpret_cast<const bf16x8*>(cw.T[part][f][lane]);
      }
    __builtin_amdgcn_sched_barrier(0);
    const bool slow = __any(odd != 0 || odd_values(vt));
    if (lane == 0) *by_token = slow;
    if (slow) {
      stage_barrier();
      by_tokens<DELTA>(p, stage + KO, stage + QO, first + t0, cnt, h, g, dv, st);
#pragma unroll
      for (int s = 0; s < 4; ++s) split_state(s);
      continue;
    }

    bf16x8 xp[3][2];  // X, or V itself
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (DELTA) {
#pragma unroll
        for (int it = 2 * k; it < 2 * k + 2; ++it) {
          x[it] = widen(vt[it]) - from[it] * x[it];
        }
        split8(x[2 * k], x[2 * k + 1], xp[0][k], xp[1][k], xp[2][k]);
        x0[(2 * k + 1) * 64] = xp[1][k];
      } else {
        xp[0][k] = join(vt[2 * k], vt[2 * k + 1]);
      }
      x0[(2 * k) * 64] = xp[0][k];
    }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        kt[2 * s][t] = tr(stage + toff[s] + t * 4096);
        kt[2 * s + 1][t] = tr(stage + toff[s] + t * 4096 + 8);
      }
    __builtin_amdgcn_sched_barrier(0);
    stage_barrier();
    // U, decayed to the chunk's end
    f32x4 u[4];
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if (DELTA) {
        f32x4 sum[2][2]{};  // the product of the largest pieces, those down to 2^-16 of it
#pragma unroll
        for (int k = 0; k <= half; ++k)
#pragma unroll
          for (int part = 0; part < 3; ++part)
#pragma unroll
            for (int piece = 0; piece < 3 - part; ++piece)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                sum[part + piece > 0][e] = mfma(T[part][frag(2 * half + e, k)], xp[piece][k], sum[part + piece > 0][e]);
#pragma unroll
        for (int e = 0; e < 2; ++e) u[2 * half + e] = sum[0][e] + sum[1][e];
      } else {
        u[2 * half] = to[2 * half] * widen(vt[2 * half]);
        u[2 * half + 1] = to[2 * half + 1] * widen(vt[2 * half + 1]);
      }
    // the state: what the chunk adds is summed by itself, so that the state rounds once a chunk
    f32x4 add[8];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      bf16x8 up[3];
      split8(u[2 * k], u[2 * k + 1], up[0], up[1], up[2]);
#pragma unroll
      for (int d = 0; d < 8; d += 2) {
        const bf16x8 a = join(kt[d][2 * k], kt[d][2 * k + 1]), b = join(kt[d + 1][2 * k], kt[d + 1][2 * k + 1]);
        if (k == 0) add[d] = add[d + 1] = f32x4{};
#pragma unroll
        for (int part = 2; part >= 0; --part) {
          add[d] = mfma(a, up[part], add[d]);
          add[d + 1] = mfma(b, up[part], add[d + 1]);
        }
        if (k == 0) continue;
        st[d] = st[d] * all + add[d];
        st[d + 1] = st[d + 1] * all + add[d + 1];
        if (d >= 2) split_state(d / 2 - 1);
      }
    }
    split_state(3);
  }
  store_state(p, sq, h, g, dv, st);
}

// Many sequences: a workgroup of eight waves per sequence and value head, each with one slice and all of its work, so that
// two waves a SIMD fill each other's gaps and what they share is loaded once a head: 16 sequences of up to 539 tokens, 48
// heads, 151 us in this kernel (237 with slices as above), MFMAs busy 33%, 260 MB of memory, the chunks' matrices (31 KB
// each) about half of them. (Here the waves that read K^T and V transposed have DMAs in flight, and the builtin makes the
// compiler wait for those: the reads are written out, with the wait for themselves in the same block, so that the registers
// are filled when it ends.)
template <int X0, int X1, int X2, int X3>
__device__ __forceinline__ void tr_read4(const uint8_t* pa, bf16x4 (&a)[4]) {
  const uint32_t x = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)pa;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %4 offset:%5\n\t"
      "ds_read_b64_tr_b16 %1, %4 offset:%6\n\t"
      "ds_read_b64_tr_b16 %2, %4 offset:%7\n\t"
      "ds_read_b64_tr_b16 %3, %4 offset:%8\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3])
      : "v"(x), "n"(X0), "n"(X1), "n"(X2), "n"(X3)
      : "memory");
}
template <int X0, int X1, int X2, int X3>
__device__ __forceinline__ void tr_read8(const uint8_t* pa, const uint8_t* pb, bf16x4 (&a)[4], bf16x4 (&b)[4]) {
  const uint32_t x = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)pa;
  const uint32_t y = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)pb;
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%10\n\t"
      "ds_read_b64_tr_b16 %1, %8 offset:%11\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %3, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %4, %9 offset:%10\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%11\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %7, %9 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(a[0]), "=&v"(a[1]), "=&v"(a[2]), "=&v"(a[3]), "=&v"(b[0]), "=&v"(b[1]), "=&v"(b[2]), "=&v"(b[3])
      : "v"(x), "v"(y), "n"(X0), "n"(X1), "n"(X2), "n"(X3)
      : "memory");
}

template <bool DELTA>
__global__ void __launch_bounds__(512, 1) linattn_many_k(LinParams p) {
  constexpr int WB = chunk_bytes(DELTA);
  constexpr int KO = WB, QO = KO + kChunk * 256, VO = QO + kChunk * 256, STAGE = VO + kChunk * 256;
  extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // the value heads of a key head on one XCD, as above (with two pieces a factor: the call 163 -> 161 us, this kernel 176 ->
  // 128 MB read; with three 142 MB)
  const uint32_t b = blockIdx.x, per = p.HV / p.HK, whole = (uint32_t)p.S * p.HK / 8 * (8 * per);
  const uint32_t wg = b < whole ? (b / (8 * per) * 8 + b % 8) * per + b / 8 % per : b;
  const int64_t sq = wg / p.HV;
  const int h = wg - (int)(sq * p.HV), hk = h / per;
  if (sq == p.S) return zero_rows(p, h);
  SeqPlace place;
  if (!seq_find(p.seq_ptr, p.S, p.R, seq_chunks, [=](int i, int) { return i == (int)sq; }, place)) return;
  const int first = place.first, n = place.n;
  const int chunks = seq_chunks(0, n);
  const int dv = wave * 16 + c;

  // a chunk to an LDS stage: this wave's 8 rows of K, Q and V, its part of the chunk's matrices, in two halves
  const uint8_t* const work = p.work + ((int64_t)place.before * p.HV + h) * (int64_t)WB;
  const int64_t next_work = (int64_t)p.HV * WB;
  uint32_t koff[2], voff[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = wave * 8 + 4 * i + g;
    koff[i] = (uint32_t)r * (p.HK * kHD * 2) + (c ^ swizzle(r & 15)) * 16;
    voff[i] = (uint32_t)r * (p.HV * kHD * 2) + (c ^ swizzle(r & 15)) * 16;
  }
  const auto fetch = [&](int i, int t, uint8_t* stage) {
    const int cnt = min(kChunk, n - t);
    const __amdgpu_buffer_rsrc_t kr = head_rows(p.k, first + t, cnt, p.HK, hk);
    const __amdgpu_buffer_rsrc_t qr = head_rows(p.q, first + t, cnt, p.HK, hk);
    const __amdgpu_buffer_rsrc_t vr = head_rows(p.v, first + t, cnt, p.HV, h);
    const __amdgpu_buffer_rsrc_t wr = make_rsrc(work + (int64_t)(t / kChunk) * next_work, WB);
    dma16(kr, stage + KO + wave * 2048 + i * 1024, koff[i]);
    dma16(qr, stage + QO + wave * 2048 + i * 1024, koff[i]);
    dma16(vr, stage + VO + wave * 2048 + i * 1024, voff[i]);
#pragma unroll
    for (int j = i; j < (WB / 1024 + 7) / 8; j += 2) {
      const int at = min(j * 8 + wave, WB / 1024 - 1) * 1024;  // past the last piece: that one again
      dma16(wr, stage + at, at + lane * 16);
    }
  };
  if (chunks > 0) {
    fetch(0, 0, smem);
    fetch(1, 0, smem);
  }
  f32x4 st[8];
  load_state(p, sq, h, g, dv, st);

  // LDS offsets of this lane: rows c of K and Q, key dims 32 s .. + 31; the same of K's rows, and V's, read transposed
  int aoff[4], toff[4];
  const int trow = g * 4 + (c >> 2);
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    aoff[s] = c * 256 + ((s * 4 + g) ^ swizzle(c)) * 16;
    toff[s] = KO + trow * 256 + ((s * 4 + (c & 3)) ^ swizzle(trow)) * 16;
  }
  const int vtoff = VO + trow * 256 + ((wave * 2 + (c >> 1 & 1)) ^ swizzle(trow)) * 16 + (c & 1) * 8;

  // vmcnt(0), as the compiler knows it: the state is there, and no wait for it, which would take the DMAs along, is left
  // for the loop
  __builtin_amdgcn_s_waitcnt(0x0f70);
  for (int ch = 0; ch < chunks; ++ch) {
    const int t0 = ch * kChunk, cnt = min(kChunk, n - t0);
    const uint8_t* const stage = smem + (ch & 1) * STAGE;
    const ChunkWork& cw = *reinterpret_cast<const ChunkWork*>(stage);
    if (ch > 0) wait_vmcnt<16>();  // all but the last chunk's output stores
    stage_barrier();               // the stage has landed, and every wave is done with the other one
    const bool more = ch + 1 < chunks;
    uint8_t* const other = smem + ((ch + 1) & 1) * STAGE;
    if (more) fetch(0, t0 + kChunk, other);
    bf16x4 vt[4];  // V's columns: X's accumulators' places, and its B operand
    tr_read4<0, 4096, 8192, 12288>(stage + vtoff, vt);
    if (__any(cw.odd != 0 || odd_values(vt))) {
      if (more) fetch(1, t0 + kChunk, other);
      by_tokens<DELTA>(p, stage + KO, stage + QO, first + t0, cnt, h, g, dv, st);
      wait_vmcnt<0>();
      continue;
    }
    bf16x8 sp[2][4];  // the state before the chunk, for the outputs
    if (more) fetch(1, t0 + kChunk, other);
    bf16x8 xp[3][2];  // X, or V itself
    if (DELTA) {
      f32x4 x[4];
      bf16x8 all3[3][4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        split8(st[2 * s], st[2 * s + 1], all3[0][s], all3[1][s], all3[2][s]);
        sp[0][s] = all3[0][s];
        sp[1][s] = all3[1][s];
      }
      rows_times(stage + KO, aoff, all3, x);
#pragma unroll
      for (int it = 0; it < 4; ++it)
        x[it] = widen(vt[it]) - *reinterpret_cast<const f32x4*>(cw.from + it * 16 + g * 4) * x[it];
#pragma unroll
      for (int k = 0; k < 2; ++k) split8(x[2 * k], x[2 * k + 1], xp[0][k], xp[1][k], xp[2][k]);
    } else {
#pragma unroll
      for (int s = 0; s < 4; ++s) split8(st[2 * s], st[2 * s + 1], sp[0][s], sp[1][s]);
#pragma unroll
      for (int k = 0; k < 2; ++k) xp[0][k] = join(vt[2 * k], vt[2 * k + 1]);
    }
    // U, decayed to the chunk's end, and the state
    bf16x8 up[3][2];
    {
      f32x4 u[4];
      if (DELTA)
        strengths_times(cw.T, lane, xp, u);
      else
#pragma unroll
        for (int it = 0; it < 4; ++it) u[it] = *reinterpret_cast<const f32x4*>(cw.to + it * 16 + g * 4) * widen(vt[it]);
#pragma unroll
      for (int k = 0; k < 2; ++k) split8(u[2 * k], u[2 * k + 1], up[0][k], up[1][k], up[2][k]);
    }
    const float all = cw.all;
#pragma unroll
    for (int d = 0; d < 8; d += 4) {
      bf16x4 kt[4][4];  // key dims of d .. d + 3, tokens 16 t + 4 g ..
      tr_read8<0, 4096, 8192, 12288>(stage + toff[d / 2], stage + toff[d / 2] + 8, kt[0], kt[1]);
      tr_read8<0, 4096, 8192, 12288>(stage + toff[d / 2 + 1], stage + toff[d / 2 + 1] + 8, kt[2], kt[3]);
      f32x4 add[4]{};  // by itself, so that the state rounds once a chunk
#pragma unroll
      for (int part = 2; part >= 0; --part)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) add[e] = mfma(join(kt[e][2 * k], kt[e][2 * k + 1]), up[part][k], add[e]);
#pragma unroll
      for (int e = 0; e < 4; ++e) st[d + e] = st[d + e] * all + add[e];
    }
    f32x4 x[4];
    rows_times(stage + QO, aoff, sp, x);
#pragma unroll
    for (int it = 0; it < 4; ++it) x[it] *= *reinterpret_cast<const f32x4*>(cw.out + it * 16 + g * 4);
    lower_times<DELTA>(cw.P, lane, xp, x);
    store_out(p, head_rows(p.o, first + t0, cnt, p.HV, h), g, dv, x);
  }
  store_state(p, sq, h, g, dv, st);
}

constexpr int many_lds(bool delta) { return 2 * (chunk_bytes(delta) + kChunk * 768); }
// Sequences times value heads up to which the workgroups of two slices run (four of them a head). Calls of 48-head sequences,
// with slices and with eight waves a head: 500 tokens each, one sequence 37 and 58 us, two 59 and 59, three 84 and 66, six
// 143 and 127; 4096 tokens each, one 203 and 367, two 386 and 416, three 570 and 459, six 985 and 932. (Three of unlike
// lengths, 4096 and less: 396 and 427.)
constexpr int64_t kFew = 96;
constexpr int prompt_lds(bool delta) { return 2 * (chunk_bytes(delta) + kChunk * (512 + 64)) + 2 * (8192 + 4096) + 16; }

}  // namespace

hipError_t launch_linattn_step(const LinParams& p, float* state, const int32_t* slot, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_step_k<true> : linattn_step_k<false>, dim3((unsigned)(p.R * p.HV)),
                     dim3(256), 0, st, p, state, slot);
  return hipGetLastError();
}

int64_t linattn_chunks(int64_t R, int64_t S) { return R / kChunk + std::min(R, S); }

int64_t linattn_work_bytes(int64_t R, int64_t S, int HV, bool delta) {
  return linattn_chunks(R, S) * HV * (int64_t)chunk_bytes(delta);
}

hipError_t launch_linattn_prompt(const LinParams& p, hipStream_t st) {
  const bool delta = p.beta != nullptr;
  const int64_t chunks = linattn_chunks(p.R, p.S);
  // a launch has fewer than 2^32 threads
  const int64_t per = ((1LL << 24) - 1) / p.HV;
  if (chunks > per) return hipErrorInvalidValue;
  if (chunks > 0) {
    hipLaunchKernelGGL(delta ? linattn_chunk_k<true> : linattn_chunk_k<false>, dim3((unsigned)(chunks * p.HV)), dim3(256),
                       0, st, p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
  }
  const bool many = p.S * p.HV > kFew;
  const auto kernel = many ? (delta ? linattn_many_k<true> : linattn_many_k<false>)
                           : (delta ? linattn_prompt_k<true> : linattn_prompt_k<false>);
  const int lds = many ? many_lds(delta) : prompt_lds(delta);
  // once for each device and kernel; a second thread that comes meanwhile sets the same again
  static std::atomic<bool> set[64][4];
  int dev = 0;
  hipError_t err = hipGetDevice(&dev);
  if (err != hipSuccess) return err;
  std::atomic<bool>* const done = dev >= 0 && dev < 64 ? &set[dev][2 * many + delta] : nullptr;
  if (done == nullptr || !done->load(std::memory_order_acquire)) {
    err = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (err != hipSuccess) return err;
    if (done != nullptr) done->store(true, std::memory_order_release);
  }
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.S + 1) * p.HV * (many ? 1 : 4))), dim3(many ? 512 : 256), lds, st, p);
  return hipGetLastError();
}

}  // namespace ojx

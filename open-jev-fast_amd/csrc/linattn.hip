// Linear attention with a decay for each head, over whole sequences (prompts) and for single tokens.
//
// A value head carries a state S [128 (key dims), 128 (value dims)]; token t has a key k, a query q, a value v, the
// logarithm g of its decay and, with the delta rule, a strength beta:
//   S <- e^g S;  u = beta (v - S^T k)  (without the delta rule u = v);  S <- S + k u^T;  o = scale S^T q
// Value head h reads key head h / (HV / HK).
#include "ojx_internal.h"

#include <algorithm>
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

// ------------------------------------------------------------------------------------------------------------- prompts
// A chunk of C = 64 tokens at once. With G_i the sum of g up to token i of the chunk and S0 the state before it,
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j (j < i),  P_ij = e^(G_i - G_j) q_i . k_j (j <= i),  T = (I + A)^-1 diag(beta),
//   U = T (V - diag(e^G) K S0)  (without the delta rule U = V),
//   O = scale (diag(e^G) Q S0 + P U),  S = e^(G_C) S0 + K^T diag(e^(G_C - G)) U.
// T and P need no state: linattn_chunk_k makes them for all chunks at once. linattn_prompt_k then goes through a
// sequence's chunks in order.
//
// Precision. The states are fp32, and so is what makes them: a factor that is not a bf16 input (S0, T, U, V - ..) enters
// its products as two bf16 pieces, hi + lo, which keep 16 bits and more (K and Q are bf16 already; hi lo and lo hi are
// taken, lo lo is not). Differences of G are taken in 64 bits before they are rounded: after a long decay G is large, and
// its fp32 steps would show in e^(G_i - G_j). Outputs are rounded to bf16, so what only they need is taken in bf16: S0 for
// Q S0, P and U for P U.
// A chunk with a value that is not finite, or a decay above 1, goes token by token (the same recurrence), so that nothing
// reaches the tokens before it: in the products a zero above the diagonal times NaN would.

constexpr int kChunk = 64;
constexpr float kMinDecay = -200.f;  // e^-200 is 0 in fp32: -infinity does no worse, and differences of sums stay numbers

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// What a chunk of a head leaves for linattn_prompt_k: A operands of 16 x 32 products, one lane's 8 values after the other.
// The operand (it, ks) covers tokens 16 it .. + 15 against tokens 32 ks .. + 31, the latter in the order in which a lane
// holds the other factor: 4 of the first 16, 4 of the second. Those above the diagonal are left out: (0, 0), (1, 0),
// (2, 0), (2, 1), (3, 0), (3, 1).
struct ChunkWork {
  uint16_t P[6][64][8];
  float from[kChunk], to[kChunk];  // e^G, e^(G_C - G)
  float all;                       // e^(G_C)
  int32_t odd;                     // token by token
  int32_t pad[2];
  uint16_t T[2][6][64][8];         // hi, lo; the delta rule's last part
};
constexpr int64_t kPlainBytes = (int64_t)offsetof(ChunkWork, T);
__host__ __device__ constexpr int64_t chunk_bytes(bool delta) { return delta ? (int64_t)sizeof(ChunkWork) : kPlainBytes; }
__device__ __forceinline__ constexpr int frag(int it, int ks) { return it < 2 ? it : 2 * it - 2 + ks; }

__device__ __forceinline__ int seq_chunks(int n) { return (n + kChunk - 1) / kChunk; }

// Two bf16 pieces of 8 values: x = hi + lo to 16 bits.
__device__ __forceinline__ void split8(const f32x4& a, const f32x4& b, bf16x8& hi, bf16x8& lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x = i < 2 ? a[2 * i] : b[2 * i - 4], y = i < 2 ? a[2 * i + 1] : b[2 * i - 3];
    h[i] = pack2(x, y);
    l[i] = pack2(x - __uint_as_float(h[i] << 16), y - __uint_as_float(h[i] & 0xffff0000u));
  }
  hi = __builtin_bit_cast(bf16x8, make_uint4(h[0], h[1], h[2], h[3]));
  lo = __builtin_bit_cast(bf16x8, make_uint4(l[0], l[1], l[2], l[3]));
}
__device__ __forceinline__ bf16x8 round8(const f32x4& a, const f32x4& b) {
  return __builtin_bit_cast(bf16x8, make_uint4(pack2(a[0], a[1]), pack2(a[2], a[3]), pack2(b[0], b[1]), pack2(b[2], b[3])));
}
__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ bool odd8(bf16x8 x) {  // one of them is not finite
  const uint4 u = __builtin_bit_cast(uint4, x);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  bool r = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (w[i] & 0x7f80u) == 0x7f80u || (w[i] & 0x7f800000u) == 0x7f800000u;
  return r;
}

// T and P of one chunk and value head; wave w has the tokens 16 w .. + 15 as rows.
//   * k . k and q . k on bf16 MFMA from the rows as they lie in memory;
//   * (I + A)^-1 in blocks of 16: the diagonal ones by forward substitution, a column a lane; then block column w by wave
//     w, T_iw = -T_ii (sum_k A_ik T_kw), on fp32 MFMA (16x16x4), whose B operand is the accumulator of the product before
//     when the contraction runs in its order.
template <bool DELTA>
__global__ void __launch_bounds__(256) linattn_chunk_k(LinParams p) {
  constexpr int LD = 68;  // LDS row of 64 floats
  __shared__ __attribute__((aligned(16))) float Pt[64 * LD], At[DELTA ? 64 * LD : 1], Tt[DELTA ? 64 * LD : 1];
  __shared__ int odd_at[4];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t chunk = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(chunk * p.HV), hk = h / (p.HV / p.HK);
  SeqPlace at;
  if (!seq_find(p.seq_ptr, p.S, p.R, seq_chunks, [=](int, int upto) { return upto > (int)chunk; }, at)) return;
  const int t0 = at.first + ((int)chunk - at.before) * kChunk, cnt = min(kChunk, at.first + at.n - t0);
  ChunkWork* const out = reinterpret_cast<ChunkWork*>(p.work + (chunk * p.HV + h) * chunk_bytes(DELTA));

  // a token a lane: decays and strengths; tokens behind the end add nothing
  const bool on = lane < cnt;
  float gv = on ? p.g[(int64_t)(t0 + lane) * p.HV + h] : 0.f;
  const float beta = DELTA && on ? bf2f(p.beta[(int64_t)(t0 + lane) * p.HV + h]) : 0.f;
  bool odd = !(gv <= 0.f) || !(fabsf(beta) < INFINITY);
  gv = gv < kMinDecay ? kMinDecay : gv;
  double G = gv;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double t = __shfl_up(G, o);
    if (lane >= o) G += t;
  }

  const auto rows = [&](const uint16_t* x, int tile, int s) {
    const int t = tile * 16 + c;
    return t < cnt ? *reinterpret_cast<const bf16x8*>(x + ((int64_t)(t0 + t) * p.HK + hk) * kHD + s * 32 + g * 8)
                   : bf16x8{};
  };
  bf16x8 ka[4], qa[4];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    ka[s] = rows(p.k, w, s);
    qa[s] = rows(p.q, w, s);
    odd |= odd8(ka[s]) || odd8(qa[s]);
  }
  double Gi[4];
  float bi[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    Gi[r] = __shfl(G, w * 16 + g * 4 + r);
    bi[r] = __shfl(beta, w * 16 + g * 4 + r);
  }
#pragma unroll
  for (int jt = 0; jt < 4; ++jt) {
    if (jt > w) {  // the operands of a pair of tiles reach one tile above the diagonal
      if (jt == (w | 1))
#pragma unroll
        for (int r = 0; r < 4; ++r) Pt[(w * 16 + g * 4 + r) * LD + jt * 16 + c] = 0.f;
      continue;
    }
    f32x4 kk{}, qk{};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8 kb = rows(p.k, jt, s);
      if (DELTA) kk = mfma(ka[s], kb, kk);
      qk = mfma(qa[s], kb, qk);
    }
    const double Gj = __shfl(G, jt * 16 + c);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = w * 16 + g * 4 + r, j = jt * 16 + c;
      const float e = j <= i ? expf((float)(Gi[r] - Gj)) : 0.f;
      Pt[i * LD + j] = j <= i ? e * qk[r] : 0.f;
      if (DELTA) At[i * LD + j] = j < i ? bi[r] * (e * kk[r]) : 0.f;
    }
  }
  if (DELTA) {
    // column c of the diagonal block's inverse
    float x[16];
    const float* const blk = At + w * 16 * LD + w * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float a = i == c ? 1.f : 0.f;
#pragma unroll
      for (int m = 0; m < i; ++m) a -= blk[i * LD + m] * x[m];
      x[i] = a;
    }
    if (g == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) Tt[(w * 16 + i) * LD + w * 16 + c] = x[i];
    __syncthreads();
    f32x4 t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = f32x4{};
      if (i == w) {
#pragma unroll
        for (int r = 0; r < 4; ++r) t[i][r] = Tt[(i * 16 + g * 4 + r) * LD + i * 16 + c];
      } else if (i > w) {
        f32x4 sum{}, neg{};
#pragma unroll
        for (int k = 0; k < i; ++k) {
          if (k < w) continue;
          const f32x4 a = *reinterpret_cast<const f32x4*>(At + (i * 16 + c) * LD + k * 16 + g * 4);
#pragma unroll
          for (int s = 0; s < 4; ++s) sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], t[k][s], sum, 0, 0, 0);
        }
        const f32x4 a = *reinterpret_cast<const f32x4*>(Tt + (i * 16 + c) * LD + i * 16 + g * 4);
#pragma unroll
        for (int s = 0; s < 4; ++s) neg = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], sum[s], neg, 0, 0, 0);
        t[i] = -neg;
      }
    }
    const float bj = __shfl(beta, w * 16 + c);
    __syncthreads();  // the diagonal blocks have been read
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float v = t[i][r] * bj;
        odd |= !(fabsf(v) < INFINITY);
        Tt[(i * 16 + g * 4 + r) * LD + w * 16 + c] = v;
      }
  }
  if (lane == 0) odd_at[w] = 0;
  if (__any(odd) && lane == 0) odd_at[w] = 1;
  __syncthreads();
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (ks > (w >> 1)) continue;
    const int at = (w * 16 + c) * LD + ks * 32 + g * 4;
    const f32x4 a = *reinterpret_cast<const f32x4*>(Pt + at), b = *reinterpret_cast<const f32x4*>(Pt + at + 16);
    *reinterpret_cast<bf16x8*>(out->P[frag(w, ks)][lane]) = round8(a, b);
    if (DELTA) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(Tt + at), y = *reinterpret_cast<const f32x4*>(Tt + at + 16);
      bf16x8 hi, lo;
      split8(x, y, hi, lo);
      *reinterpret_cast<bf16x8*>(out->T[0][frag(w, ks)][lane]) = hi;
      *reinterpret_cast<bf16x8*>(out->T[1][frag(w, ks)][lane]) = lo;
    }
  }
  if (w != 0) return;
  const double last = __shfl(G, 63);
  out->from[lane] = expf((float)G);
  out->to[lane] = expf((float)(last - G));
  if (lane == 0) {
    out->all = expf((float)last);
    out->odd = odd_at[0] | odd_at[1] | odd_at[2] | odd_at[3];
  }
}

// The chunks of one sequence and value head in order. A wave has 16 CT value dims of the state, all 128 key dims: 8 CT
// accumulators, lane (c, g) holding key dims 16 d + 4 g .. + 3 of value dim c. As the B operand of K S0 and Q S0 that is the
// contraction in the order 4 of one 16, 4 of the next, so K and Q come as two 8-byte pieces, and nothing of the state, of
// U or of V - .. ever leaves its lane: the waves share only K and Q, through LDS, and meet once a chunk. K^T comes from
// the same LDS rows by transposing reads. Every operand of the next chunk is loaded where the present one's has been used.
template <bool DELTA, int CT>
__global__ void __launch_bounds__(256, 1) linattn_prompt_k(LinParams p) {
  constexpr int LD = kHD + 8;  // LDS row
  __shared__ __attribute__((aligned(16))) uint16_t kq[2][2][kChunk * LD];
  constexpr int SL = 2 / CT;  // workgroups of a head
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t sq = blockIdx.x / (p.HV * SL);
  const int hs = blockIdx.x - (int)(sq * p.HV * SL), h = hs / SL, hk = h / (p.HV / p.HK);
  if (sq == p.S) {  // the rows of no sequence
    int lo, hi;
    seq_span(p.seq_ptr, p.S, p.R, lo, hi);
    for (int64_t r = threadIdx.x >> 4; r < lo + (p.R - hi) && hs % SL == 0; r += 16)
      *reinterpret_cast<uint4*>(p.o + ((r < lo ? r : r - lo + hi) * p.HV + h) * kHD + (threadIdx.x & 15) * 8) =
          make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  SeqPlace place;
  if (!seq_find(p.seq_ptr, p.S, p.R, seq_chunks, [=](int i, int) { return i == (int)sq; }, place)) return;
  const int first = place.first, n = place.n;
  const int chunks = seq_chunks(n);
  const int dv = ((hs % SL) * 4 + wave) * 16 * CT + c;  // + 16 ct

  f32x4 st[8][CT];
  {
    int64_t at = -1;
    if (p.state != nullptr) at = p.src != nullptr ? (int64_t)p.src[sq] : sq;
    const bool have = at >= 0 && at < p.slots;
    const float fill = at >= p.slots ? __uint_as_float(0x7fc00000u) : 0.f;
#pragma unroll
    for (int d = 0; d < 8; ++d)
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          st[d][ct][r] =
              have ? p.state[(at * p.HV + h) * (kHD * kHD) + (d * 16 + g * 4 + r) * kHD + dv + ct * 16] : fill;
  }
  const uint8_t* work = p.work + ((int64_t)place.before * p.HV + h) * chunk_bytes(DELTA);
  const int64_t next_work = p.HV * chunk_bytes(DELTA);

  // K and Q rows of a chunk: 16-byte pieces, zeros behind the sequence's end
  uint4 kx[4], qx[4];
  const auto load_kq = [&](int t) {  // first token of the chunk
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int piece = i * 256 + threadIdx.x, r = t + (piece >> 4);
      const int64_t at = ((int64_t)(first + r) * p.HK + hk) * kHD + (piece & 15) * 8;
      kx[i] = r < n ? *reinterpret_cast<const uint4*>(p.k + at) : make_uint4(0u, 0u, 0u, 0u);
      qx[i] = r < n ? *reinterpret_cast<const uint4*>(p.q + at) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  const auto store_kq = [&](int half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int piece = i * 256 + threadIdx.x, at = (piece >> 4) * LD + (piece & 15) * 8;
      *reinterpret_cast<uint4*>(kq[half][0] + at) = kx[i];
      *reinterpret_cast<uint4*>(kq[half][1] + at) = qx[i];
    }
  };
  uint32_t vx[4][4][CT];
  const auto load_v = [&](int t) {
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const int tk = t + it * 16 + g * 4 + r;
          vx[it][r][ct] = tk < n ? p.v[((int64_t)(first + tk) * p.HV + h) * kHD + dv + ct * 16] : 0u;
        }
  };
  bf16x8 T[2][6], P[6];
  f32x4 from[4], to[4];
  float all = 0.f;
  int odd = 0;
  const auto cw = [&](const uint8_t* at) { return reinterpret_cast<const ChunkWork*>(at); };
  const auto load_T = [&](const ChunkWork* x) {
    if (DELTA)
#pragma unroll
      for (int f = 0; f < 6; ++f) {
        T[0][f] = *reinterpret_cast<const bf16x8*>(x->T[0][f][lane]);
        T[1][f] = *reinterpret_cast<const bf16x8*>(x->T[1][f][lane]);
      }
  };
  const auto load_P = [&](const ChunkWork* x) {
#pragma unroll
    for (int f = 0; f < 6; ++f) P[f] = *reinterpret_cast<const bf16x8*>(x->P[f][lane]);
#pragma unroll
    for (int it = 0; it < 4; ++it) from[it] = *reinterpret_cast<const f32x4*>(x->from + it * 16 + g * 4);
  };
  const auto load_to = [&](const ChunkWork* x) {
#pragma unroll
    for (int it = 0; it < 4; ++it) to[it] = *reinterpret_cast<const f32x4*>(x->to + it * 16 + g * 4);
    all = x->all;
    odd = x->odd;
  };

  if (chunks > 0) {
    load_kq(0);
    load_v(0);
    load_T(cw(work));
    load_P(cw(work));
    load_to(cw(work));
    store_kq(0);
  }
  for (int ch = 0; ch < chunks; ++ch) {
    const int t0 = ch * kChunk, half = ch & 1, cnt = min(kChunk, n - t0);
    const bool more = ch + 1 < chunks;
    const ChunkWork* const next = cw(work + next_work);
    const uint16_t* const kl = kq[half][0];
    const uint16_t* const ql = kq[half][1];
    __syncthreads();
    if (more) load_kq(t0 + kChunk);
    bool slow = odd != 0;
#pragma unroll
    for (int it = 0; it < 4; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) slow |= (vx[it][r][ct] & 0x7f80u) == 0x7f80u;
    if (__any(slow)) {
      for (int t = 0; t < cnt; ++t) {
        const int64_t row = (int64_t)(first + t0 + t) * p.HV + h;
        const float a = expf(p.g[row]), b = DELTA ? bf2f(p.beta[row]) : 1.f;
        bf16x4 kt[8], qt[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          kt[d] = *reinterpret_cast<const bf16x4*>(kl + t * LD + d * 16 + g * 4);
          qt[d] = *reinterpret_cast<const bf16x4*>(ql + t * LD + d * 16 + g * 4);
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          float u = bf2f(p.v[row * kHD + dv + ct * 16]), x = 0.f, o = 0.f;
#pragma unroll
          for (int d = 0; d < 8; ++d) {
            st[d][ct] *= a;
#pragma unroll
            for (int r = 0; r < 4; ++r) x += st[d][ct][r] * (float)kt[d][r];
          }
          x += __shfl_xor(x, 16);
          x += __shfl_xor(x, 32);
          if (DELTA) u = b * (u - x);
#pragma unroll
          for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              st[d][ct][r] += (float)kt[d][r] * u;
              o += st[d][ct][r] * (float)qt[d][r];
            }
          o += __shfl_xor(o, 16);
          o += __shfl_xor(o, 32);
          if (g == 0) p.o[row * kHD + dv + ct * 16] = (uint16_t)f2bf(p.scale * o);
        }
      }
      if (more) {
        load_v(t0 + kChunk);
        load_T(next);
        load_P(next);
        load_to(next);
      }
    } else {
      bf16x8 sh[4][CT], sl[4][CT];
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) split8(st[2 * s][ct], st[2 * s + 1][ct], sh[s][ct], sl[s][ct]);
      f32x4 ks[4][CT], qs[4][CT];
#pragma unroll
      for (int it = 0; it < 4; ++it) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) ks[it][ct] = qs[it][ct] = f32x4{};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int at = (it * 16 + c) * LD + s * 32 + g * 4;
          if (DELTA) {
            const bf16x8 a = __builtin_shufflevector(*reinterpret_cast<const bf16x4*>(kl + at),
                                                     *reinterpret_cast<const bf16x4*>(kl + at + 16), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) {
              ks[it][ct] = mfma(a, sh[s][ct], ks[it][ct]);
              ks[it][ct] = mfma(a, sl[s][ct], ks[it][ct]);
            }
          }
          const bf16x8 b = __builtin_shufflevector(*reinterpret_cast<const bf16x4*>(ql + at),
                                                   *reinterpret_cast<const bf16x4*>(ql + at + 16), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) qs[it][ct] = mfma(b, sh[s][ct], qs[it][ct]);
        }
      }
      f32x4 u[4][CT];
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = bf2f(vx[it][r][ct]);
            u[it][ct][r] = DELTA ? v - from[it][r] * ks[it][ct][r] : v;
          }
      if (more) load_v(t0 + kChunk);
      if (DELTA) {
        bf16x8 rh[2][CT], rl[2][CT];
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) split8(u[2 * k][ct], u[2 * k + 1][ct], rh[k][ct], rl[k][ct]);
#pragma unroll
        for (int it = 0; it < 4; ++it)
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            f32x4 x{};
#pragma unroll
            for (int k = 0; k <= it / 2; ++k) {
              x = mfma(T[0][frag(it, k)], rh[k][ct], x);
              x = mfma(T[0][frag(it, k)], rl[k][ct], x);
              x = mfma(T[1][frag(it, k)], rh[k][ct], x);
            }
            u[it][ct] = x;
          }
        if (more) load_T(next);
      }
      // the state
      bf16x8 uh[2][CT], ul[2][CT], ub[2][CT];
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          ub[k][ct] = round8(u[2 * k][ct], u[2 * k + 1][ct]);
          split8(u[2 * k][ct] * to[2 * k], u[2 * k + 1][ct] * to[2 * k + 1], uh[k][ct], ul[k][ct]);
        }
      const uint16_t* const kt = kl + (g * 4 + (c >> 2)) * LD + (c & 3) * 4;
#pragma unroll
      for (int d = 0; d < 8; ++d) {
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) st[d][ct] *= all;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (__attribute__((address_space(3))) bf16x4*)(kt + k * 32 * LD + d * 16));
          const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
              (__attribute__((address_space(3))) bf16x4*)(kt + (k * 32 + 16) * LD + d * 16));
          const bf16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) {
            st[d][ct] = mfma(a, uh[k][ct], st[d][ct]);
            st[d][ct] = mfma(a, ul[k][ct], st[d][ct]);
          }
        }
      }
      // the outputs
#pragma unroll
      for (int it = 0; it < 4; ++it)
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          f32x4 x = qs[it][ct] * from[it];
#pragma unroll
          for (int k = 0; k <= it / 2; ++k) x = mfma(P[frag(it, k)], ub[k][ct], x);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int tk = it * 16 + g * 4 + r;
            if (tk < cnt)
              p.o[((int64_t)(first + t0 + tk) * p.HV + h) * kHD + dv + ct * 16] = (uint16_t)f2bf(p.scale * x[r]);
          }
        }
      if (more) {
        load_P(next);
        load_to(next);
      }
    }
    if (more) store_kq(half ^ 1);
    work += next_work;
  }
#pragma unroll
  for (int d = 0; d < 8; ++d)
#pragma unroll
    for (int ct = 0; ct < CT; ++ct)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        p.state_out[(sq * p.HV + h) * (kHD * kHD) + (d * 16 + g * 4 + r) * kHD + dv + ct * 16] = st[d][ct][r];
}

}  // namespace

hipError_t launch_linattn_step(const LinParams& p, float* state, const int32_t* slot, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_step_k<true> : linattn_step_k<false>, dim3((unsigned)(p.R * p.HV)),
                     dim3(256), 0, st, p, state, slot);
  return hipGetLastError();
}

int64_t linattn_chunks(int64_t R, int64_t S) { return R / kChunk + std::min(R, S); }

int64_t linattn_work_bytes(int64_t R, int64_t S, int HV, bool delta) {
  return linattn_chunks(R, S) * HV * chunk_bytes(delta);
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
  const bool wide = p.S * p.HV >= 256;
  const auto kernel = delta ? (wide ? linattn_prompt_k<true, 2> : linattn_prompt_k<true, 1>)
                            : (wide ? linattn_prompt_k<false, 2> : linattn_prompt_k<false, 1>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)((p.S + 1) * p.HV * (wide ? 1 : 2))), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

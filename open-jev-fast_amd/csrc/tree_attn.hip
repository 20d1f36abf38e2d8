// Attention of drafted tokens over a paged cache.
//
// Sequence b has n = q_ptr[b + 1] - q_ptr[b] drafted tokens (rows) and ctx[b] tokens before them; its cache position p
// lies in page table[b][p / page] at place p % page, and drafted token j at position ctx[b] + j. A row sees the positions
// below ctx[b] and those drafted tokens whose bit is set in its bits (without bits: its predecessors and itself).
//   s_p = scale q . k_p,  m = max s_p,  out = sum exp(s_p - m) v_p / sum exp(s_p - m),  lse = m + log sum exp(s_p - m)
// over the positions seen; a row that sees nothing gives zeros and lse = -inf.
//
// Work layout. The G = HQ / HKV query heads of a kv head read the same keys, so their rows (token, head) are packed: a
// workgroup takes a block of 16 CT packed rows of one sequence and kv head and a part of the positions. Its four waves
// take the part's units of 32 positions in turn and are independent until the end:
//   * S^T = K Q^T on 16x16x32 MFMA: the K rows are the A operand, straight from the cache into registers (a lane's 16
//     bytes are 8 bf16 or 16 e4m3 values of one key; the e4m3 form orders the contraction accordingly, for Q too), Q stays
//     in registers. A lane then holds one row's scores of 4 positions of each 16.
//   * the softmax runs per lane: the maximum needs two shuffles, the sum none until the end, and the reference maximum
//     only moves when it has grown by 2^8 (the weights stay below 2^8, well inside fp32 and bf16), so that the outputs are
//     rarely rescaled;
//   * O^T += V^T P^T: P^T is the B operand as the lane holds it, with the contraction in the order 4 of the first 16
//     positions, 4 of the second; V^T comes from the wave's own LDS rows by transposing reads (ds_read_b64_tr_b16: 16
//     lanes get 4 x 16 elements column by column), rows padded by 32 bytes so that the reads spread over the banks.
// The loads of the next unit, keys and values, go into the registers that the present unit has just left and arrive
// behind its products. P is rounded to bf16 as every operand of these products is (half a step, 2^-8 of each weight); the
// sum of the weights and the outputs are fp32.
// Units in which a row may not see every position (drafted ones, the sequence's end, pages outside the cache) also mask,
// take the values of places that nobody sees as zeros and, where a value is not finite, add position by position, so that
// a NaN reaches the rows that see it and no other.
// Where sequences and row blocks are few, the positions are split over more workgroups, whose sums a second launch joins.
#include "gemm_common.h"

#include <algorithm>

namespace ojx {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(4))) const int32_t* const_ints;  // read-only: scalar loads

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;  // the reference maximum follows when it is this far behind, base two

// Zeros (and lse -inf) for kv head hk's heads of the rows before the first sequence and behind the last.
__device__ __forceinline__ void zero_rows(const TreeParams& p, int hk, int D) {
  int lo, hi;
  seq_span(p.q_ptr, p.B, p.N, lo, hi);
  const int G = p.HQ / p.HKV, per = G * D / 8;
  const int64_t rows = lo + p.N - hi;
  for (int64_t t = threadIdx.x; t < rows * per; t += blockDim.x) {
    const int64_t i = t / per, n = i < lo ? i : i - lo + hi;
    const int c = (int)(t - i * per);
    *reinterpret_cast<uint4*>(p.out + (n * p.HQ + hk * G) * D + c * 8) = make_uint4(0u, 0u, 0u, 0u);
    if (p.lse != nullptr && c < G) p.lse[n * p.HQ + hk * G + c] = -INFINITY;
  }
}

__device__ __forceinline__ uint32_t cvt_fp8x2(int x, bool hi) {  // two e4m3 values as bf16: exact
  const bf16x2 r = hi ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true)
                      : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false);
  return __builtin_bit_cast(uint32_t, r);
}
__device__ __forceinline__ uint4 cvt_fp8x8(uint32_t a, uint32_t b) {
  return make_uint4(cvt_fp8x2(a, false), cvt_fp8x2(a, true), cvt_fp8x2(b, false), cvt_fp8x2(b, true));
}
__device__ __forceinline__ bool odd2(uint32_t x) {  // either bf16 of x is not finite
  return (x & 0x7f80u) == 0x7f80u || (x & 0x7f800000u) == 0x7f800000u;
}

// Positions p0 .. p0 + 31 of those that a row of drafted index i sees, as bits; w: its words.
__device__ __forceinline__ uint32_t seen32(const TreeParams& p, const int64_t* w, int i, int64_t j0) {
  if (j0 <= -32) return ~0u;
  if (w == nullptr) {
    const int64_t c = i - j0 + 1;
    return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1;
  }
  if (j0 < 0) return ((uint32_t)w[0] << -j0) | ((1u << -j0) - 1);
  const int64_t at = j0 >> 6;
  const int sh = (int)(j0 & 63);
  if (at >= p.words) return 0u;
  uint64_t x = (uint64_t)w[at] >> sh;
  if (sh > 32 && at + 1 < p.words) x |= (uint64_t)w[at + 1] << (64 - sh);
  return (uint32_t)x;
}

// The packed rows that a lane's columns stand for: row0 + 16 ct + lane % 16.
template <int CT>
struct Rows {
  int tok[CT], head[CT];
  bool live[CT];
  const int64_t* words[CT];
  __device__ __forceinline__ Rows(const TreeParams& p, int row0, int rows, int first, int hk) {
    const int G = p.HQ / p.HKV;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int r = row0 + ct * 16 + (threadIdx.x & 15);
      live[ct] = r < rows;
      tok[ct] = live[ct] ? r / G : 0;
      head[ct] = hk * G + (live[ct] ? r - tok[ct] * G : 0);
      words[ct] = p.bits != nullptr ? p.bits + (int64_t)(first + tok[ct]) * p.words : nullptr;
    }
  }
};

// Q as the B operand; an e4m3 cache's 16-byte pieces of a key order the contraction.
template <int D, bool FP8, int CT>
__device__ __forceinline__ void load_q(const TreeParams& p, const Rows<CT>& w, int first, bool paired,
                                       bf16x8 (&qf)[CT][D / 32]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const uint16_t* src = p.q + ((int64_t)w.head[ct] * p.N + first + w.tok[ct]) * D;
#pragma unroll
    for (int f = 0; f < D / 32; ++f) {
      const int d = paired ? (f >> 1) * 64 + g * 16 + (f & 1) * 8 : f * 32 + g * 8;
      qf[ct][f] = *reinterpret_cast<const bf16x8*>(src + d);  // a column without a row repeats the first one's
    }
  }
}

// One workgroup's part of the positions.
struct Part {
  int b, first, n, row0, rows, hk, split, u0, u1;
  int64_t ctx, total;
  // false: nothing to do. Blocks and parts of a launch are numbered row block, part, kv head, the last fastest.
  __device__ __forceinline__ bool find(const TreeParams& p, int R, int D, int step) {
    const int groups = p.HKV * p.splits;
    const int rb = blockIdx.x / groups, at = blockIdx.x - rb * groups;
    split = at / p.HKV;
    hk = at - split * p.HKV;
    if (rb == 0 && split == 0) zero_rows(p, hk, D);
    const int G = p.HQ / p.HKV;
    SeqPlace at_seq;
    if (!seq_find(
            p.q_ptr, p.B, p.N, [=](int m) { return (m * G + R - 1) / R; }, [=](int, int upto) { return upto > rb; }, at_seq))
      return false;
    b = at_seq.seq;
    first = at_seq.first;
    n = at_seq.n;
    row0 = (rb - at_seq.before) * R;
    rows = n * G;
    ctx = max(p.ctx[b], 0);
    total = p.pages > 0 ? min(ctx + n, p.max_pages * p.page) : 0;
    const int units = (int)((total + 31) >> 5);
    const int part = max(step, ((units + p.splits - 1) / p.splits + step - 1) / step * step);
    u0 = min(units, split * part);
    u1 = min(units, u0 + part);
    return true;
  }
  __device__ __forceinline__ int64_t head_row(const TreeParams& p, int row) const {  // (row, head) of a packed row
    const int G = p.HQ / p.HKV, tk = row / G;
    return (int64_t)(first + tk) * p.HQ + hk * G + (row - tk * G);
  }
  // An empty part of a short sequence has no sums: its rows say so.
  __device__ __forceinline__ void no_sums(const TreeParams& p, int R) const {
    for (int r = row0 + threadIdx.x; r < min(rows, row0 + R); r += blockDim.x)
      p.ml[head_row(p, r) * p.splits + split] = make_float2(-INFINITY, 0.f);
  }
};

// Row of the cache where the 16 positions of tile t begin, or -1 where there is none.
struct Table {
  const_ints at;
  int64_t max_pages, pages;
  int tiles, page, HKV, hk;
  uint32_t inv;
  __device__ __forceinline__ Table(const TreeParams& p, const Part& w)
      : at((const_ints)(uintptr_t)(p.table + (int64_t)w.b * p.max_pages)), max_pages(p.max_pages), pages(p.pages),
        tiles(p.page >> 4), page(p.page), HKV(p.HKV), hk(w.hk), inv(p.tiles_inv) {}
  __device__ __forceinline__ int64_t row(int t) const {
    int i = t;  // t / tiles
    if (tiles > 1) {
      i = (int)(((uint64_t)(uint32_t)t * inv) >> 32);  // or one more
      if (i * tiles > t) --i;
    }
    if (i >= max_pages) return -1;
    const int pg = at[i];
    return pg >= 0 && pg < pages ? ((int64_t)pg * HKV + hk) * page + (t - i * tiles) * 16 : -1;
  }
};

// Scores of 32 positions -> weights (the B operand of the outputs' product, and for the rare path as they are), with the
// rows' reference maxima, sums and outputs brought up to date. edge: `there` and the rows' bits say what is seen.
template <bool FP8, int DT, int CT>
__device__ __forceinline__ void soft_weights(const TreeParams& p, const Rows<CT>& rw, const f32x4 (&s)[2][CT], float f2,
                                             const f32x4 (&kq)[2], const f32x4 (&vq)[2], bool edge, uint32_t there,
                                             int64_t j0, float (&m)[CT], float (&l)[CT], f32x4 (&acc)[DT][CT],
                                             float (&w)[CT][8], bf16x8 (&pf)[CT]) {
  const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    uint32_t see = ~0u;
    if (edge) see = (rw.live[ct] ? there & seen32(p, rw.words[ct], rw.tok[ct], j0) : 0u) >> (g * 4);
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      float v = s[i >> 2][ct][i & 3] * f2;
      if (FP8) v *= kq[i >> 2][i & 3];
      if (edge && !(see >> ((i >> 2) * 16 + (i & 3)) & 1)) v = -INFINITY;
      w[ct][i] = v;
      top = fmaxf(top, v);
    }
    top = fmaxf(top, __shfl_xor(top, 16));
    top = fmaxf(top, __shfl_xor(top, 32));
    const bool up = top > m[ct] + kSlack;
    if (__any(up)) {
      const float a = up ? __builtin_amdgcn_exp2f(m[ct] - top) : 1.f;
      if (up) m[ct] = top;
      l[ct] *= a;
#pragma unroll
      for (int d = 0; d < DT; ++d) acc[d][ct] *= a;
    }
    const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = __builtin_amdgcn_exp2f(w[ct][i] - ref);
      l[ct] += e;
      w[ct][i] = e;
      if (FP8) w[ct][i] = edge && !(see >> ((i >> 2) * 16 + (i & 3)) & 1) ? 0.f : e * vq[i >> 2][i & 3];
    }
    pf[ct] = __builtin_bit_cast(bf16x8, make_uint4(cvt_pk2(w[ct][0], w[ct][1]), cvt_pk2(w[ct][2], w[ct][3]),
                                                   cvt_pk2(w[ct][4], w[ct][5]), cvt_pk2(w[ct][6], w[ct][7])));
  }
}

// O^T += V^T P^T over 32 positions from LDS rows of RS values; one by one where a value is not finite, so that a weight of
// zero takes nothing.
template <int RS, int DT, int CT>
__device__ __forceinline__ void add_values(const uint16_t* vl, const float (&w)[CT][8], const bf16x8 (&pf)[CT], bool odd,
                                           f32x4 (&acc)[DT][CT]) {
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  if (odd) {
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      const int slot = (key >> 4) * 4 + (key & 3), from = ((key >> 2) & 3) * 16 + c;
      float wk[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        float y = w[ct][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) y = slot == i ? w[ct][i] : y;
        wk[ct] = __shfl(y, from);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float v = bf2f(vl[key * RS + d * 16 + g * 4 + r]);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[d][ct][r] += wk[ct] == 0.f ? 0.f : wk[ct] * v;
        }
    }
    return;
  }
  const uint16_t* const at = vl + (g * 4 + (c >> 2)) * RS + (c & 3) * 4;
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const bf16x4 lo =
        __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(at + d * 16));
    const bf16x4 hi =
        __builtin_amdgcn_ds_read_tr16_b64_v4bf16((__attribute__((address_space(3))) bf16x4*)(at + 16 * RS + d * 16));
    const bf16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) acc[d][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pf[ct], acc[d][ct], 0, 0, 0);
  }
}

// Which of the 32 positions from p0 exist: below the sequence's end, in pages of the cache.
__device__ __forceinline__ uint32_t existing(int64_t left, bool ok0, bool ok1) {
  return (left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1) & ((ok0 ? 0xffffu : 0u) | (ok1 ? 0xffff0000u : 0u));
}

// Few rows: 16 packed rows a workgroup, its four waves take the part's units in turn.
template <int D, bool FP8>
__global__ void __launch_bounds__(256, 1) tree_narrow_k(TreeParams p) {
  constexpr int R = 16, KF = D / 32, DT = D / 16, RB = D * (FP8 ? 1 : 2);  // RB: bytes of a cache row
  constexpr int RS = D + 16;                                 // LDS row of values, in bf16
  constexpr int KL = RB / 64;                                // 16-byte loads of a key
  constexpr int VR = RB / 16;                                // lanes of a value row
  constexpr int VK = 64 / VR, VL = 32 / VK;                  // keys a load, loads of 32 keys
  constexpr int XS = D + 4;                                  // row of the waves' exchange, in floats
  __shared__ __attribute__((aligned(16))) uint16_t vbuf[4 * 32 * RS];
  __shared__ float sm[4][R], sl[4][R];
  static_assert(sizeof(vbuf) >= 4 * R * XS * 4, "the exchange of sums reuses the value rows");

  Part w;
  if (!w.find(p, R, D, 4)) return;
  if (p.splits > 1 && w.u0 >= w.u1) return w.no_sums(p, R);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<1> rw(p, w.row0, w.rows, w.first, w.hk);
  const Table table(p, w);
  bf16x8 qf[1][KF];
  load_q<D, FP8, 1>(p, rw, w.first, FP8, qf);

  uint4 kx[2][KL], vx[VL];
  f32x4 ks[2], vs[2];
  bool ok[2];
  const auto load = [&](int u) {
    int64_t row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      row[t] = table.row(2 * u + t);
      ok[t] = row[t] >= 0;
      row[t] = max(row[t], (int64_t)0);  // any row of the cache: its values are not used
      const uint8_t* kb = static_cast<const uint8_t*>(p.kc) + row[t] * RB;
#pragma unroll
      for (int f = 0; f < KL; ++f) kx[t][f] = *reinterpret_cast<const uint4*>(kb + c * RB + f * 64 + g * 16);
      if (FP8) {
        ks[t] = *reinterpret_cast<const f32x4*>(p.ks + row[t] + g * 4);
        vs[t] = *reinterpret_cast<const f32x4*>(p.vs + row[t] + g * 4);
      }
    }
#pragma unroll
    for (int i = 0; i < VL; ++i)
      vx[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.vc) + row[i / (VL / 2)] * RB +
                                              (i % (VL / 2)) * 1024 + lane * 16);
  };

  const float f2 = p.scale * kLog2e;
  f32x4 acc[DT][1];
  float m[1] = {-INFINITY}, l[1] = {0.f};
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d][0] = f32x4{};
  uint16_t* const vl = vbuf + wave * 32 * RS;

  int u = w.u0 + wave;
  if (u < w.u1) load(u);
  for (; u < w.u1; u += 4) {
    f32x4 s[2][1];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t][0] = f32x4{};
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        const uint4 x = kx[t][FP8 ? f >> 1 : f];
        const bf16x8 a = __builtin_bit_cast(bf16x8, !FP8 ? x : f & 1 ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y));
        s[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[0][f], s[t][0], 0, 0, 0);
      }
    }
    const int64_t p0 = (int64_t)u * 32;
    const bool edge = !(ok[0] && ok[1]) || p0 + 32 > min(w.ctx, w.total);
    const uint32_t there = existing(w.total - p0, ok[0], ok[1]);
    bool odd = false;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = i * VK + lane / VR;
      uint4* const dst = reinterpret_cast<uint4*>(vl + key * RS + (lane % VR) * (FP8 ? 16 : 8));
#pragma unroll
      for (int h = 0; h < (FP8 ? 2 : 1); ++h) {
        uint4 x = vx[i];
        if (FP8) x = h ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y);
        if (edge) {
          if (!(there >> key & 1)) x = make_uint4(0u, 0u, 0u, 0u);
          odd |= odd2(x.x) || odd2(x.y) || odd2(x.z) || odd2(x.w);
        }
        dst[h] = x;
      }
    }
    f32x4 kq[2], vq[2];
    if (FP8)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        kq[t] = ks[t];
        vq[t] = vs[t];
      }
    if (u + 4 < w.u1) load(u + 4);
    float wt[1][8];
    bf16x8 pf[1];
    soft_weights<FP8, DT, 1>(p, rw, s, f2, kq, vq, edge, there, p0 - w.ctx, m, l, acc, wt, pf);
    add_values<RS, DT, 1>(vl, wt, pf, edge && __any(odd), acc);
  }

  // the four waves' sums, each brought to the largest reference
  l[0] += __shfl_xor(l[0], 16);
  l[0] += __shfl_xor(l[0], 32);
  if (g == 0) {
    sm[wave][c] = m[0];
    sl[wave][c] = l[0];
  }
  __syncthreads();
  const float all = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c]));
  const float mine = m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[0] - all);
  float* const swap = reinterpret_cast<float*>(vbuf);
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(swap + (wave * R + c) * XS + d * 16 + g * 4) = acc[d][0] * mine;
  __syncthreads();
  const int r = threadIdx.x >> 4, row = w.row0 + r;
  if (row >= w.rows) return;
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = fmaxf(top, sm[k][r]);
#pragma unroll
  for (int k = 0; k < 4; ++k)  // a wave without a reference has a sum only where every score was NaN
    sum += sm[k][r] == -INFINITY ? sl[k][r] : sl[k][r] * __builtin_amdgcn_exp2f(sm[k][r] - top);
  const int64_t nh = w.head_row(p, row), i = nh * p.splits + w.split;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int q = 0; q < D / 64; ++q) {
    const int d = q * 64 + (threadIdx.x & 15) * 4;
    f32x4 o{};
#pragma unroll
    for (int k = 0; k < 4; ++k) o += *reinterpret_cast<const f32x4*>(swap + (k * R + r) * XS + d);
    if (p.splits > 1)
      *reinterpret_cast<f32x4*>(p.part + i * D + d) = o;
    else
      *reinterpret_cast<uint2*>(p.out + nh * D + d) = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
  }
  if ((threadIdx.x & 15) != 0) return;
  if (p.splits > 1)
    p.ml[i] = make_float2(top, sum);
  else if (p.lse != nullptr)
    p.lse[nh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// More rows: 16 CT packed rows a workgroup, 128 positions at a time. A wave takes 32 of the positions for the scores, with
// their keys straight from the cache as in the narrow kernel, and a quarter of the dims for the outputs, with that quarter
// of the 128 values in LDS rows of its own: keys and values are read once a workgroup, however many rows it has. What the
// waves exchange is the weights (a lane's eight are the B operand for its 32 positions as they are) and the maxima. The
// steps of two lots overlap, so that one barrier a lot is enough: behind it a wave
//   adds the values of lot i - 1 with the weights of all four waves,
//   takes lot i's maxima, brings its sums to a new reference where one has grown, makes its weights of lot i,
//   makes its scores of lot i + 1 and leaves their maxima.
// All waves see the same maxima and so hold the same references.
template <int D, bool FP8, int CT>
__global__ void __launch_bounds__(256, 1) tree_wide_k(TreeParams p) {
  constexpr int R = 16 * CT, KF = D / 32, RB = D * (FP8 ? 1 : 2);  // RB: bytes of a cache row
  constexpr int DS = D / 4, DT = DS / 16;                          // dims of a wave
  constexpr int VS = DS + 16;                                      // LDS row of values, in bf16
  constexpr int KL = RB / 64;                                      // 16-byte loads of a key
  constexpr int VR = RB / 64, VK = 64 / VR, VL = 128 / VK;         // lanes of a value row's quarter, rows a load, loads
  __shared__ __attribute__((aligned(16))) uint16_t vbuf[4][128 * VS];
  __shared__ __attribute__((aligned(16))) uint4 pbuf[2][4][CT][64];
  __shared__ float sm[2][4][R], sl[4][R];

  Part w;
  if (!w.find(p, R, D, 4)) return;
  if (p.splits > 1 && w.u0 >= w.u1) return w.no_sums(p, R);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Rows<CT> rw(p, w.row0, w.rows, w.first, w.hk);
  const Table table(p, w);
  bf16x8 qf[CT][KF];
  load_q<D, FP8, CT>(p, rw, w.first, FP8, qf);

  // keys of unit u (32 positions) and values of the lot that begins there; which of their tiles of 16 are in the cache
  uint4 kx[2][KL], vx[VL];
  f32x4 ks[2], vs[2];
  const auto load_k = [&](int u) -> int {
    int ok = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int64_t r = table.row(2 * u + t), row = max(r, (int64_t)0);  // any row of the cache: it is not used
      ok |= (r >= 0) << t;
      const uint8_t* kb = static_cast<const uint8_t*>(p.kc) + row * RB;
#pragma unroll
      for (int f = 0; f < KL; ++f) kx[t][f] = *reinterpret_cast<const uint4*>(kb + c * RB + f * 64 + g * 16);
      if (FP8) {
        ks[t] = *reinterpret_cast<const f32x4*>(p.ks + row + g * 4);
        vs[t] = *reinterpret_cast<const f32x4*>(p.vs + row + g * 4);
      }
    }
    return ok;
  };
  const auto load_v = [&](int u) -> int {
    int64_t row[8];
    int ok = 0;
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int64_t r = table.row(2 * u + t);
      row[t] = max(r, (int64_t)0);
      ok |= (r >= 0) << t;
    }
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = lane / VR;  // of this load's VK
      int64_t at;
      if constexpr (VK == 32)
        at = (key >= 16 ? row[2 * i + 1] : row[2 * i]) + (key & 15);
      else
        at = row[i * VK / 16] + (i * VK) % 16 + key;
      vx[i] = *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p.vc) + at * RB + wave * (RB / 4) + (lane % VR) * 16);
    }
    return ok;
  };
  const int64_t plain = min(w.ctx, w.total);  // positions below are seen by every row, if they are in the cache

  const float f2 = p.scale * kLog2e;
  f32x4 acc[DT][CT], s[2][CT], vq[2];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d][ct] = f32x4{};
  }
  bool edge_s = false;  // of the scores in s
  // scores of the loaded unit u, masked, to base two; their maxima to sm[half]
  const auto scores = [&](int u, int ok, int half) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[t][ct] = f32x4{};
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        const uint4 x = kx[t][FP8 ? f >> 1 : f];
        const bf16x8 a = __builtin_bit_cast(bf16x8, !FP8 ? x : f & 1 ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y));
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[t][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[ct][f], s[t][ct], 0, 0, 0);
      }
    }
    const int64_t p0 = (int64_t)u * 32;
    edge_s = ok != 3 || p0 + 32 > plain;
    const uint32_t there = edge_s ? existing(w.total - p0, ok & 1, ok >> 1) : ~0u;
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float top = -INFINITY;
      uint32_t see = ~0u;
      if (edge_s) see = (rw.live[ct] ? there & seen32(p, rw.words[ct], rw.tok[ct], p0 - w.ctx) : 0u) >> (g * 4);
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[t][ct] *= f2;
        if (FP8) s[t][ct] *= ks[t];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (edge_s && !(see >> (t * 16 + r) & 1)) s[t][ct][r] = -INFINITY;
          top = fmaxf(top, s[t][ct][r]);
        }
      }
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      if (g == 0) sm[half][wave][ct * 16 + c] = top;
    }
    if (FP8) {
      vq[0] = vs[0];
      vq[1] = vs[1];
    }
  };
  // weights of the scores in s, with the maxima in sm[half], to pbuf[half]
  const auto weights = [&](int half) {
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      const int r = ct * 16 + c;
      const float top = fmaxf(fmaxf(sm[half][0][r], sm[half][1][r]), fmaxf(sm[half][2][r], sm[half][3][r]));
      const bool up = top > m[ct] + kSlack;
      if (__any(up)) {
        const float a = up ? __builtin_amdgcn_exp2f(m[ct] - top) : 1.f;
        if (up) m[ct] = top;
        l[ct] *= a;
#pragma unroll
        for (int d = 0; d < DT; ++d) acc[d][ct] *= a;
      }
      const float ref = m[ct] == -INFINITY ? 0.f : m[ct];
      float e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = s[i >> 2][ct][i & 3];
        e[i] = __builtin_amdgcn_exp2f(x - ref);
        l[ct] += e[i];
        if (FP8) e[i] = edge_s && x == -INFINITY ? 0.f : e[i] * vq[i >> 2][i & 3];
      }
      pbuf[half][wave][ct][lane] =
          make_uint4(cvt_pk2(e[0], e[1]), cvt_pk2(e[2], e[3]), cvt_pk2(e[4], e[5]), cvt_pk2(e[6], e[7]));
    }
  };
  uint16_t* const vl = vbuf[wave];
  // the loaded values of the lot that begins at unit u to LDS, zeros where there is no position; whether one is not finite
  const auto store_v = [&](int u, int ok) -> bool {
    const int64_t p0 = (int64_t)u * 32;
    const bool edge = ok != 255 || p0 + 128 > plain;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < VL; ++i) {
      const int key = i * VK + lane / VR;
      uint4* const dst = reinterpret_cast<uint4*>(vl + key * VS + (lane % VR) * (FP8 ? 16 : 8));
#pragma unroll
      for (int h = 0; h < (FP8 ? 2 : 1); ++h) {
        uint4 x = vx[i];
        if (FP8) x = h ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y);
        if (edge) {
          if (!(ok >> (key >> 4) & 1) || p0 + key >= w.total) x = make_uint4(0u, 0u, 0u, 0u);
          odd |= odd2(x.x) || odd2(x.y) || odd2(x.z) || odd2(x.w);
        }
        dst[h] = x;
      }
    }
    return edge && __any(odd);
  };
  const auto add_lot = [&](int half, bool odd) {
    if (odd) {  // one by one, so that a weight of zero takes nothing
#pragma unroll 1
      for (int key = 0; key < 128; ++key) {
        const int from = ((key >> 2) & 3) * 16 + c, at = (key >> 4 & 1) * 4 + (key & 3);
        float wk[CT];
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          wk[ct] = bf2f(reinterpret_cast<const uint16_t*>(&pbuf[half][key >> 5][ct][from])[at]);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float v = bf2f(vl[key * VS + d * 16 + g * 4 + r]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct) acc[d][ct][r] += wk[ct] == 0.f ? 0.f : wk[ct] * v;
          }
      }
      return;
    }
    const uint16_t* const at = vl + (g * 4 + (c >> 2)) * VS + (c & 3) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      bf16x8 pf[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) pf[ct] = __builtin_bit_cast(bf16x8, pbuf[half][k][ct][lane]);
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const bf16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(at + k * 32 * VS + d * 16));
        const bf16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4bf16(
            (__attribute__((address_space(3))) bf16x4*)(at + (k * 32 + 16) * VS + d * 16));
        const bf16x8 a = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int ct = 0; ct < CT; ++ct)
          acc[d][ct] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pf[ct], acc[d][ct], 0, 0, 0);
      }
    }
  };

  const int lots = (w.u1 - w.u0 + 3) >> 2;
  int kok = 0, vok = 0;
  bool odd = false;
  if (lots > 0) {
    kok = load_k(w.u0 + wave);
    vok = load_v(w.u0);
    scores(w.u0 + wave, kok, 0);
    if (lots > 1) kok = load_k(w.u0 + 4 + wave);
  }
  for (int i = 0; i < lots; ++i) {
    const int u = w.u0 + 4 * i, half = i & 1;
    lds_barrier();
    if (i > 0) add_lot(half ^ 1, odd);
    odd = store_v(u, vok);
    if (i + 1 < lots) vok = load_v(u + 4);
    weights(half);
    if (i + 1 < lots) {
      scores(u + 4 + wave, kok, half ^ 1);
      if (i + 2 < lots) kok = load_k(u + 8 + wave);
    }
  }
  lds_barrier();
  if (lots > 0) add_lot((lots - 1) & 1, odd);

#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16);
    l[ct] += __shfl_xor(l[ct], 32);
    if (g == 0) sl[wave][ct * 16 + c] = l[ct];
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (!rw.live[ct]) continue;
    const int r = ct * 16 + c;
    const float sum = (sl[0][r] + sl[1][r]) + (sl[2][r] + sl[3][r]), inv = sum == 0.f ? 0.f : 1.f / sum;
    const int64_t nh = (int64_t)(w.first + rw.tok[ct]) * p.HQ + rw.head[ct], i = nh * p.splits + w.split;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 o = acc[d][ct];
      const int at = wave * DS + d * 16 + g * 4;
      if (p.splits > 1)
        *reinterpret_cast<f32x4*>(p.part + i * D + at) = o;
      else
        *reinterpret_cast<uint2*>(p.out + nh * D + at) = make_uint2(cvt_pk2(o[0] * inv, o[1] * inv), cvt_pk2(o[2] * inv, o[3] * inv));
    }
    if (g != 0 || wave != 0) continue;
    if (p.splits > 1)
      p.ml[i] = make_float2(m[ct], sum);
    else if (p.lse != nullptr)
      p.lse[nh] = sum == 0.f ? -INFINITY : (m[ct] + log2f(sum)) * kLn2;
  }
}

// Joins the parts of a row: one wave per (row, head), 4 D / 256 dims a lane.
template <int D>
__global__ void __launch_bounds__(256) tree_join_k(TreeParams p) {
  constexpr int E = D / 64;
  const int64_t nh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (nh >= p.N * p.HQ) return;
  const int64_t row = nh / p.HQ;
  int lo, hi;
  seq_span(p.q_ptr, p.B, p.N, lo, hi);
  if (row < lo || row >= hi) return;  // of no sequence: it has its zeros
  const float2* const ml = p.ml + nh * p.splits;
  float top = -INFINITY, sum = 0.f, o[E] = {};
  for (int s = 0; s < p.splits; ++s) top = fmaxf(top, ml[s].x);
  for (int s = 0; s < p.splits; ++s) {
    const float2 x = ml[s];
    if (x.x == -INFINITY && x.y == 0.f) continue;  // nothing seen there; an empty part has no sums either
    const float f = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - top);
    sum += f * x.y;
    const float* const src = p.part + (nh * p.splits + s) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * src[e];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* const dst = reinterpret_cast<uint32_t*>(p.out + nh * D + lane * E);
#pragma unroll
  for (int e = 0; e < E; e += 2) dst[e / 2] = pack2(o[e] * inv, o[e + 1] * inv);
  if (lane == 0 && p.lse != nullptr) p.lse[nh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

}  // namespace

TreePlan tree_plan(int64_t N, int B, int HQ, int HKV, int D, int64_t max_pages, int page) {
  TreePlan t{};
  const int64_t G = HQ / HKV, seqs = std::max<int64_t>(1, std::min<int64_t>(B, N)), mean = (N * G + seqs - 1) / seqs;
  t.rows = mean <= 16 ? 16 : mean <= 32 ? 32 : 64;
  // an upper bound of sum ceil(n_b G / rows) over the sequences with rows, which are `seqs` at most
  t.blocks = (N * G + seqs * (t.rows - 1)) / t.rows;
  const int64_t units = (max_pages * page + 31) / 32, base = t.blocks * HKV;
  t.splits = std::max<int64_t>(1, std::min<int64_t>((512 + base - 1) / base, std::min<int64_t>(units / 8, 64)));
  return t;
}

template <int D, bool FP8>
static void (*tree_kernel(int rows))(TreeParams) {
  return rows == 16 ? tree_narrow_k<D, FP8> : rows == 32 ? tree_wide_k<D, FP8, 2> : tree_wide_k<D, FP8, 4>;
}

hipError_t launch_tree_attn(const TreeParams& p, const TreePlan& t, int D, bool fp8, hipStream_t st) {
  const auto kernel = D == 256 ? (fp8 ? tree_kernel<256, true>(t.rows) : tree_kernel<256, false>(t.rows))
                               : (fp8 ? tree_kernel<128, true>(t.rows) : tree_kernel<128, false>(t.rows));
  hipLaunchKernelGGL(kernel, dim3((unsigned)(t.blocks * p.HKV * t.splits)), dim3(256), 0, st, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || t.splits == 1) return err;
  hipLaunchKernelGGL(D == 256 ? tree_join_k<256> : tree_join_k<128>, dim3((unsigned)((p.N * p.HQ + 3) / 4)), dim3(256),
                     0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

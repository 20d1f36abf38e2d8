// Attention of drafted tokens over a paged cache.
//
// Sequence b has n = q_ptr[b + 1] - q_ptr[b] drafted tokens (rows) and ctx[b] tokens before them; its cache position p
// lies in page table[b][p / page] at place p % page, and drafted token j at position ctx[b] + j. A row sees the positions
// below ctx[b] and those drafted tokens whose bit is set in its bits (without bits: its predecessors and itself).
//   s_p = scale q . k_p,  m = max s_p,  out = sum exp(s_p - m) v_p / sum exp(s_p - m),  lse = m + log sum exp(s_p - m)
// over the positions seen; a row that sees nothing gives zeros and lse = -inf.
//
// Work layout. The G = HQ / HKV query heads of a kv head read the same keys, so their rows (token, head) are packed, and a
// workgroup takes a block of packed rows of one sequence and kv head and a part of the positions, in units of 32:
//   * S^T = K Q^T on 16x16x32 MFMA, K rows as the A operand, Q in registers as B. A lane then holds one row's scores of 4
//     positions of each 16.
//   * the softmax runs per lane: the maximum needs two lane swaps, the sum none until the end, and the reference maximum
//     only moves when it has grown by 2^8 (the weights stay below 2^8, well inside fp32 and bf16), so that the outputs are
//     rarely rescaled;
//   * O^T += V^T P^T: P^T is the B operand as the lane holds it, with the contraction in the order 4 of the first 16
//     positions, 4 of the second; V^T comes from LDS rows by transposing reads (ds_read_b64_tr_b16: 16 lanes get 4 x 16
//     elements column by column).
// P is rounded to bf16 as every operand of these products is (half a step, 2^-8 of each weight): outputs are up to a fourth
// further off than their own rounding alone; the sum of the weights and the outputs are fp32. e4m3 keys and values become bf16, which is exact; a position's scales go into its score and weight.
// Units in which a row may not see every position (drafted ones, the sequence's end, pages outside the cache) also mask,
// take the values of places that nobody sees as zeros and keep values that are not finite apart, so that a NaN reaches the
// rows that see it and no other.
// The positions are split over workgroups so that one round of them fills the GPU; a second launch joins the parts.
//
// Three sizes of row blocks, by the mean packed rows of a sequence (tree_plan). Times of tree_attn, D = 256, four kv heads
// of six query heads, three caches in turn, bf16 / e4m3, in blocks of 16, 64 and 128 rows:
//   16 sequences of  1 over 4096 ( 6 rows):  57 /  36,   58 /  45,  60 /  70 us -> 16
//                    4           (24 rows):  65 /  43,   60 /  47,  62 /  72    -> 64
//                    8           (48 rows): 101 /  67,   62 /  49,  65 /  75    -> 64
//                   12           (72 rows): 180 / 124,   78 /  81,  67 /  78    -> 128
//   4 sequences of  64 over 8192 (384 rows): 310 / 214, 134 / 145,  85 / 107    -> 128
// An e4m3 cache is half the bytes, but its values become bf16 on their way to LDS: faster than bf16 up to 48 rows or so a
// sequence (64 x 1 over 4096: 104 and 188 us, 64 x 4: 139 and 187), slower from 72 on.
// What bounds them now: a single row block of a bf16 cache, its stream (64 x 4 over 4096: 187 us, 5.8 TB/s); else the steps
// of a wave between barriers: in the 16 x 12 case of up to 8192 (e4m3, 69 us) MFMAs are busy 10% of the time, waves wait
// for memory and barriers 40% and to issue 21% of theirs; in the 4 x 64 case of up to 16384 (bf16, 78 us) 21, 35 and 31%.
// Reading operands further ahead than the loops do changes neither. A chain of 2048 rows over nothing takes 258 / 305 us:
// each of its row blocks runs the whole sequence's units, and all of them as edges.
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
    if (c >= G) continue;
    if (p.lse != nullptr) p.lse[n * p.HQ + hk * G + c] = -INFINITY;
    if (p.target > 0) p.joins[n * p.HQ + hk * G + c] = make_uint2(0u, 0u);
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
template <bool FP8>
__device__ __forceinline__ uint4 half_piece(uint4 x, int e) {  // 8 values of a 16-byte piece as bf16: the only, or half e
  return !FP8 ? x : e ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y);
}
__device__ __forceinline__ bool odd2(uint32_t x) {  // either bf16 of x is not finite
  return ((x & 0x7f80u) == 0x7f80u) | ((x & 0x7f800000u) == 0x7f800000u);
}
__device__ __forceinline__ uint32_t even2(uint32_t x) {  // with zeros for those
  x = (x & 0x7f80u) == 0x7f80u ? x & 0xffff0000u : x;
  return (x & 0x7f800000u) == 0x7f800000u ? x & 0xffffu : x;
}

// Positions p0 .. p0 + 31 of those that a row of drafted index i sees, as bits; w: its words.
__device__ __forceinline__ uint32_t seen32(const TreeParams& p, const int64_t* w, int i, int j0) {
  if (j0 <= -32) return ~0u;
  if (w == nullptr) {
    const int c = i - j0 + 1;
    return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1;
  }
  if (j0 < 0) return ((uint32_t)w[0] << -j0) | ((1u << -j0) - 1);
  const int at = j0 >> 6, sh = j0 & 63;
  if (at >= p.words) return 0u;
  uint64_t x = (uint64_t)w[at] >> sh;
  if (sh > 32 && at + 1 < p.words) x |= (uint64_t)w[at + 1] << (64 - sh);
  return (uint32_t)x;
}

// The packed row that a lane's column stands for: row0 + lane % 16 (column).
struct Row {
  int tok, head;
  bool live;
  const int64_t* words;
  __device__ __forceinline__ Row(const TreeParams& p, int row0, int rows, int first, int hk, int column) {
    const int G = p.HQ / p.HKV, r = row0 + column;
    live = r < rows;
    tok = live ? r / G : 0;
    head = hk * G + (live ? r - tok * G : 0);
    words = p.bits != nullptr ? p.bits + (int64_t)(first + tok) * p.words : nullptr;
  }
};

// Q as the B operand; an e4m3 cache's 16-byte pieces of a key order the contraction (paired).
template <int D>
__device__ __forceinline__ void load_q(const TreeParams& p, const Row& w, int first, bool paired, bf16x8 (&qf)[D / 32]) {
  const int g = (threadIdx.x & 63) >> 4;
  const uint16_t* src = p.q + ((int64_t)w.head * p.N + first + w.tok) * D;
#pragma unroll
  for (int f = 0; f < D / 32; ++f) {
    const int d = paired ? (f >> 1) * 64 + g * 16 + (f & 1) * 8 : f * 32 + g * 8;
    qf[f] = *reinterpret_cast<const bf16x8*>(src + d);  // a column without a row repeats the first one's
  }
}

// One workgroup's share: a row block of R packed rows of a sequence and a part of the sequence's units of 32 positions.
// Work is shared out by the lengths as they are on the device: a sequence of u units has ceil(u / L) parts of equal length
// for each of its row blocks. With up to 64 sequences and no more row blocks, nb, than workgroups run at once (p.target, of
// a kv head), L is the least that makes p.target parts at most, found in steps of a sixteenth from the mean on: one round
// of workgroups, all about as long (16 x 12 over up to 8192, e4m3: 77 us with the L below, 69 this way; equal lengths
// are level). With more, L is `total` units over all row blocks by max(p.target - nb, nb / 4), so that there are
// max(p.target, nb + nb / 4) parts at most and the longest sequences do not come last and alone. No part has fewer than
// p.least units unless its sequence has.
struct Part {
  int b, first, n, row0, rows, hk, parts, u0, u1;
  uint32_t slot;  // of the part's first row in the workspace; a row's parts lie HKV R slots apart
  int ctx, total;  // positions before the drafted ones; all of them that the table can hold
  // false: nothing to do. Shares are numbered sequence, row block, part; the kv head is the fastest of a launch. Parts
  // begin at multiples of step.
  __device__ __forceinline__ bool find(const TreeParams& p, int R, int D, int step) {
    const int lane = threadIdx.x & 63, share = blockIdx.x / p.HKV, G = p.HQ / p.HKV;
    hk = blockIdx.x - share * p.HKV;
    if (share == 0) zero_rows(p, hk, D);
    const int64_t most = p.pages > 0 ? p.max_pages * p.page : 0;
    const auto units = [=](int i, int n) {
      return n > 0 ? (int)((min(max((int64_t)p.ctx[i], (int64_t)0) + n, most) + 31) >> 5) : 0;
    };
    const auto blocks = [=](int n) { return (n * G + R - 1) / R; };
    int L = 0x7fffffff;
    const auto cut = [&](int u) { return max(1, (int)(((uint32_t)u + (uint32_t)L - 1) / (uint32_t)L)); };
    if (p.target > 0) {
      int64_t all = 0;
      int nb = 0, carry = 0, bl = 0, un = 0;  // bl, un: row blocks and units of a lane's sequence
      for (int64_t base = 0; base < p.B; base += 64) {
        const int64_t i = base + lane;
        const int x = max(carry, wave_scan_max(seq_bound(p.q_ptr, min(i, (int64_t)p.B), p.N)));
        const int e = max(x, seq_bound(p.q_ptr, min(i + 1, (int64_t)p.B), p.N));
        bl = blocks(e - x);
        un = units((int)min(i, (int64_t)p.B - 1), e - x);
        all += (int64_t)bl * un;
        nb += bl;
        carry = __builtin_amdgcn_readlane(e, 63);
      }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        all += __shfl_xor(all, o);
        nb += __shfl_xor(nb, o);
      }
      const bool search = p.B <= 64 && nb <= p.target;
      const int by = search ? p.target : max(max(p.target - nb, nb / 4), 1);
      L = (int)min((max((all + by - 1) / by, (int64_t)p.least) + step - 1) / step * step, (int64_t)(1 << 27));
      if (search)  // ends: with L as long as the longest sequence there are nb parts
        while (L < (1 << 27) && __builtin_amdgcn_readlane(wave_scan_sum(bl * cut(un)), 63) > p.target)
          L += ((L >> 4) / step + 1) * step;
    }
    SeqPlace at;
    if (!seq_find(
            p.q_ptr, p.B, p.N,
            [=](int i, int m) { return blocks(m) * cut(units((int)min((int64_t)i, (int64_t)p.B - 1), m)); },
            [=](int, int upto) { return upto > share; }, at))
      return false;
    b = __builtin_amdgcn_readfirstlane(at.seq);
    first = at.first;
    n = at.n;
    rows = n * G;
    ctx = max(p.ctx[b], 0);
    total = (int)min((int64_t)ctx + n, most);
    const int u = units(b, n);
    parts = __builtin_amdgcn_readfirstlane(cut(u));
    const int k = share - at.before, rb = k / parts, part = k - rb * parts;
    const int len = ((u + parts - 1) / parts + step - 1) / step * step;  // at most L: none is empty
    row0 = rb * R;
    u0 = min(u, part * len);
    u1 = min(u, u0 + len);
    slot = (uint32_t)blockIdx.x * R;
    if (p.target > 0 && part == 0)  // what joins the rows' parts
      for (int r = row0 + threadIdx.x; r < min(rows, row0 + R); r += blockDim.x)
        p.joins[head_row(p, r)] = make_uint2(slot + r - row0, parts);
    return true;
  }
  __device__ __forceinline__ int64_t head_row(const TreeParams& p, int row) const {  // (row, head) of a packed row
    const int G = p.HQ / p.HKV, tk = row / G;
    return (int64_t)(first + tk) * p.HQ + hk * G + (row - tk * G);
  }
};

// Where in the cache the 16 positions of a tile are (a sequence with positions has pages).
struct Table {
  const_ints at;
  int max_pages, tiles, page, HKV, hk;
  uint32_t inv, pages;
  __device__ __forceinline__ Table(const TreeParams& p, const Part& w)
      : at((const_ints)(uintptr_t)(p.table + (int64_t)w.b * p.max_pages)), max_pages((int)p.max_pages), tiles(p.page >> 4),
        page(p.page), HKV(p.HKV), hk(w.hk), inv(p.tiles_inv), pages((uint32_t)p.pages) {}
  __device__ __forceinline__ int index(int t) const {  // t / tiles
    const int i = (int)(((uint64_t)(uint32_t)t * inv) >> 32);  // or one less
    return i + ((i + 1) * tiles <= t);
  }
  // the page of tile t, without a branch: a tile behind the table reads its last entry
  __device__ __forceinline__ int entry(int t) const { return at[min(index(t), max_pages - 1)]; }
  __device__ __forceinline__ bool ok(int t, int pg) const { return (index(t) < max_pages) & ((uint32_t)pg < pages); }
  // the row, given that entry; where there is none, any row of the cache (it is not used)
  __device__ __forceinline__ int64_t row(int t, int pg) const {
    return ((int64_t)(ok(t, pg) ? pg : 0) * HKV + hk) * page + (t - index(t) * tiles) * 16;
  }
};

// The largest of lanes l, l ^ 16, l ^ 32, l ^ 48, by swaps of rows of 16 and halves of 32: no trip through LDS.
__device__ __forceinline__ float quarters_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t v = __float_as_uint(fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1])));
  const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// Scaled scores of 32 positions, base two, -> weights (the B operand of the outputs' product), with the rows' reference
// maxima, sums and outputs brought up to date. edge: seen() says which of the positions the row sees.
template <bool FP8, int DT, typename Scale, typename Seen>
__device__ __forceinline__ void soft_weights(const f32x4 (&s)[2], Scale vscale, bool edge, Seen seen, float& m, float& l,
                                             f32x4 (&acc)[DT], bf16x8& pf) {
  float w[8];
  const int g = (threadIdx.x & 63) >> 4;
  uint32_t see = ~0u;
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = s[i >> 2][i & 3];
  if (edge) {
    see = seen() >> (g * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = see >> ((i >> 2) * 16 + (i & 3)) & 1 ? w[i] : -INFINITY;
  }
  float top = w[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) top = fmaxf(top, w[i]);
  top = quarters_max(top);
  const bool up = top > m + kSlack;
  if (__any(up)) {
    const float a = up ? __builtin_amdgcn_exp2f(m - top) : 1.f;
    if (up) m = top;
    l *= a;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] *= a;
  }
  const float ref = m == -INFINITY ? 0.f : m;
  f32x4 vq[2];
  if (FP8) {
    vq[0] = vscale(0);
    vq[1] = vscale(1);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    w[i] = __builtin_amdgcn_exp2f(w[i] - ref);
    l += w[i];
    if (FP8) w[i] *= vq[i >> 2][i & 3];
  }
  if (FP8 && edge)  // a scale that nobody sees may be anything
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = see >> ((i >> 2) * 16 + (i & 3)) & 1 ? w[i] : 0.f;
  pf = __builtin_bit_cast(bf16x8, make_uint4(cvt_pk2(w[0], w[1]), cvt_pk2(w[2], w[3]), cvt_pk2(w[4], w[5]), cvt_pk2(w[6], w[7])));
}

// One of a row's 32 weights, from the lane that holds it.
__device__ __forceinline__ float weight_of(bf16x8 pf, int key) {
  const int slot = (key >> 4) * 4 + (key & 3), from = ((key >> 2) & 3) * 16 + (threadIdx.x & 15);
  const uint4 y = __builtin_bit_cast(uint4, pf);
  const uint32_t z = slot < 2 ? y.x : slot < 4 ? y.y : slot < 6 ? y.z : y.w;
  return bf2f((uint32_t)__shfl((int)(slot & 1 ? z >> 16 : z & 0xffffu), from));
}

// O^T += V^T P^T over 32 positions from LDS rows of RS values; one by one where a value is not finite, so that a row takes
// nothing from a position that it does not see (seen() gives those that it does). From one that it sees, a value that is not
// finite goes in whatever the weight, also where that is too small for fp32: an infinity keeps its sign.
template <int RS, int DT, typename Seen>
__device__ __forceinline__ void add_values(const uint16_t* vl, bf16x8 pf, bool odd, Seen seen, f32x4 (&acc)[DT]) {
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  if (odd) {
    const uint32_t see = seen();
#pragma unroll 1
    for (int key = 0; key < 32; ++key) {
      const float wk = weight_of(pf, key);
      const bool on = see >> key & 1;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float x = bf2f(vl[key * RS + d * 16 + g * 4 + r]);
          acc[d][r] += !on ? 0.f : wk == 0.f && !(fabsf(x) < INFINITY) ? x : wk * x;
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
    acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pf, acc[d], 0, 0, 0);
  }
}

// Which of the 32 positions from p0 exist: below the sequence's end, in pages of the cache.
__device__ __forceinline__ uint32_t existing(int left, bool ok0, bool ok1) {
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
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Row rw(p, w.row0, w.rows, w.first, w.hk, c);
  const Table table(p, w);
  bf16x8 qf[KF];
  load_q<D>(p, rw, w.first, FP8, qf);

  uint4 kx[2][KL], vx[VL];
  f32x4 ks[2], vs[2];
  bool ok[2];
  const auto load = [&](int u) {
    int64_t row[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int pg = table.entry(2 * u + t);
      ok[t] = table.ok(2 * u + t, pg);
      row[t] = table.row(2 * u + t, pg);
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
  const int full = min(w.ctx, w.total) >> 5;  // units below are seen by every row, if they are in the cache
  f32x4 acc[DT];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d] = f32x4{};
  uint16_t* const vl = vbuf + wave * 32 * RS;

  int u = w.u0 + wave;
  if (u < w.u1) load(u);
  for (; u < w.u1; u += 4) {
    f32x4 s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] = f32x4{};
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        const uint4 x = kx[t][FP8 ? f >> 1 : f];
        const bf16x8 a = __builtin_bit_cast(bf16x8, !FP8 ? x : f & 1 ? cvt_fp8x8(x.z, x.w) : cvt_fp8x8(x.x, x.y));
        s[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qf[f], s[t], 0, 0, 0);
      }
    }
    const int p0 = u * 32;
    const bool edge = !(ok[0] && ok[1]) || u >= full;
    const uint32_t there = existing(w.total - p0, ok[0], ok[1]);
    bool odd = false;
    const auto piece = [&](int i, int h) {
      return !FP8 ? vx[i] : h ? cvt_fp8x8(vx[i].z, vx[i].w) : cvt_fp8x8(vx[i].x, vx[i].y);
    };
    uint4* const dst = reinterpret_cast<uint4*>(vl + lane / VR * RS + (lane % VR) * (FP8 ? 16 : 8));
    constexpr int STEP = VK * RS / 8;  // from one load's rows to the next's
    if (!edge) {
#pragma unroll
      for (int i = 0; i < VL; ++i)
#pragma unroll
        for (int h = 0; h < (FP8 ? 2 : 1); ++h) dst[i * STEP + h] = piece(i, h);
    } else {
#pragma unroll
      for (int i = 0; i < VL; ++i)
#pragma unroll
        for (int h = 0; h < (FP8 ? 2 : 1); ++h) {
          const uint4 x = there >> (i * VK + lane / VR) & 1 ? piece(i, h) : make_uint4(0u, 0u, 0u, 0u);
          odd |= odd2(x.x) | odd2(x.y) | odd2(x.z) | odd2(x.w);
          dst[i * STEP + h] = x;
        }
    }
    f32x4 vq[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      s[t] *= f2;
      if (FP8) {
        s[t] *= ks[t];
        vq[t] = vs[t];
      }
    }
    if (u + 4 < w.u1) load(u + 4);
    bf16x8 pf;
    const auto seen = [&] { return rw.live ? there & seen32(p, rw.words, rw.tok, p0 - w.ctx) : 0u; };
    soft_weights<FP8, DT>(s, [&](int t) { return vq[t]; }, edge, seen, m, l, acc, pf);
    add_values<RS, DT>(vl, pf, edge && __any(odd), seen, acc);
  }

  // the four waves' sums, each brought to the largest reference
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (g == 0) {
    sm[wave][c] = m;
    sl[wave][c] = l;
  }
  __syncthreads();
  const float all = fmaxf(fmaxf(sm[0][c], sm[1][c]), fmaxf(sm[2][c], sm[3][c]));
  const float mine = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - all);
  float* const swap = reinterpret_cast<float*>(vbuf);
#pragma unroll
  for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(swap + (wave * R + c) * XS + d * 16 + g * 4) = acc[d] * mine;
  __syncthreads();
  const int r = threadIdx.x >> 4, row = w.row0 + r;
  if (row >= w.rows) return;
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) top = fmaxf(top, sm[k][r]);
#pragma unroll
  for (int k = 0; k < 4; ++k)  // a wave without a reference has a sum only where every score was NaN
    sum += sm[k][r] == -INFINITY ? sl[k][r] : sl[k][r] * __builtin_amdgcn_exp2f(sm[k][r] - top);
  const int64_t nh = w.head_row(p, row), i = w.slot + r;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int q = 0; q < D / 64; ++q) {
    const int d = q * 64 + (threadIdx.x & 15) * 4;
    f32x4 o{};
#pragma unroll
    for (int k = 0; k < 4; ++k) o += *reinterpret_cast<const f32x4*>(swap + (k * R + r) * XS + d);
    if (w.parts > 1)
      *reinterpret_cast<f32x4*>(p.part + i * D + d) = o;
    else
      *reinterpret_cast<uint2*>(p.out + nh * D + d) = make_uint2(pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv));
  }
  if ((threadIdx.x & 15) != 0) return;
  if (w.parts > 1)
    p.ml[i] = make_float2(top, sum);
  else if (p.lse != nullptr)
    p.lse[nh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

// Values of 4 tiles of 16 dims as the A operand (lo: the first 16 of 32 positions, hi: the others) from LDS. Written out
// with the wait in the same block, because the builtin makes the compiler wait for the DMAs in flight, too.
template <int LO, int HI>
__device__ __forceinline__ void values4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, bf16x4 (&lo)[4], bf16x4 (&hi)[4]) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8 offset:%12\n\t"
      "ds_read_b64_tr_b16 %4, %8 offset:%13\n\t"
      "ds_read_b64_tr_b16 %1, %9 offset:%12\n\t"
      "ds_read_b64_tr_b16 %5, %9 offset:%13\n\t"
      "ds_read_b64_tr_b16 %2, %10 offset:%12\n\t"
      "ds_read_b64_tr_b16 %6, %10 offset:%13\n\t"
      "ds_read_b64_tr_b16 %3, %11 offset:%12\n\t"
      "ds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(lo[0]), "=&v"(lo[1]), "=&v"(lo[2]), "=&v"(lo[3]), "=&v"(hi[0]), "=&v"(hi[1]), "=&v"(hi[2]), "=&v"(hi[3])
      : "v"(a0), "v"(a1), "v"(a2), "v"(a3), "n"(LO), "n"(HI)
      : "memory");
}

// The lane, in a way that keeps what is made of it from being kept over a loop: there, every register is the outputs'.
__device__ __forceinline__ int lane_anew() {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));
  return lane & 63;  // known not to be negative: shifts, not divisions
}

// Many rows: 64 CT packed rows a workgroup of eight waves. Four of them take every other unit of 32 positions of the part,
// the other four the units between; a wave has 16 CT of the rows, and brings 8 of its unit's rows of keys and of values to
// LDS for its four. At the end the two sums of each row are joined through LDS, so that one part goes to memory (with four
// waves a workgroup and two workgroups a CU: 16 x 16 over 4096 75 us where this takes 67, 4 x 64 of up to 16384 78 and 77).
// Rows are not padded: the 16-byte chunk j of key r lies at place j ^ r % 8 of its row, the pair of chunks j of value r at
// j ^ r % 8, which spreads both kinds of reads over the banks. A bf16 cache's unit is fetched by LDS DMA
// (each lane fetches the chunk that belongs where the DMA puts it) an iteration ahead; an e4m3 cache's goes through
// registers, where it becomes bf16: fetched an iteration before it is stored where there are registers for it (EARLY),
// else keys and values in turn through the same ones. A unit that is an edge goes through registers, too, with zeros for
// values that are not finite; what those add to the rows that see them is an infinity or a NaN whatever the weight, and is
// added at the end.
// The main loop has no register to spare at D = 256, CT = 2 (128 for the outputs, 64 for Q), and a wait for a reload from
// scratch memory waits for the DMAs before it (4 x 64 over 16384, with 45 registers in scratch: 262 us). Hence lane_anew,
// the scores' operands one step ahead and no more, and QL.
template <int D, bool FP8, int CT>
__global__ void __launch_bounds__(512, 2) tree_wide_k(TreeParams p) {
  constexpr int R = 64 * CT, KF = D / 32, DT = D / 16, SB = D * (FP8 ? 1 : 2), RB = D * 2;  // bytes of a row: cache, LDS
  constexpr int PR = SB / 16, RL = 64 / PR, PL = 8 / RL;  // 16-byte pieces of a row, rows a wave's load takes, loads of 8 rows
  constexpr int TILE = 32 * RB;
  constexpr bool EARLY = FP8 && CT * D < 512;
  // steps of the last 16 rows' Q that stay in LDS, as many as a workgroup has room for: with them 155 KB of the CU's 160
  // (16 x 12 over 4096, 72 rows each: 87 us with none, 85 with two, 79 with three; 4 x 64 over 8192: 114, 110, 106)
  constexpr int QL = FP8 && !EARLY ? 3 : 0;
  __shared__ __attribute__((aligned(1024))) uint8_t bufs[2][2][2][TILE];  // of each four waves, two of keys and values
  __shared__ __attribute__((aligned(16))) float scs[2][2][2][32];
  __shared__ float2 sums[2][R];
  __shared__ __attribute__((aligned(16))) uint4 qbuf[QL > 0 ? QL : 1][QL > 0 ? 512 : 1];
  __shared__ int odd_any;

  Part w;
  if (!w.find(p, R, D, 1)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 3, four = __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  auto& buf = bufs[four];
  auto& sc = scs[four];
  const int wrow = w.row0 + wave * 16 * CT;
  const Table table(p, w);
  const int full = min(w.ctx, w.total) >> 5;  // units below are seen by every row, if they are in the cache
  bf16x8 qf[CT][KF];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
    load_q<D>(p, Row(p, wrow + ct * 16, w.rows, w.first, w.hk, threadIdx.x & 15), w.first, false, qf[ct]);

#pragma unroll
  for (int f = 0; f < QL; ++f) qbuf[f][threadIdx.x] = __builtin_bit_cast(uint4, qf[CT - 1][KF - QL + f]);
  struct Pieces {
    uint4 at[PL];
    float scale;
  };
  // this wave's row of a unit, and whether the unit's first 16 positions, and the others, are in the cache
  int64_t row = 0;
  bool in0 = false, in1 = false;
  const auto rows_of = [&](int u, int page0, int page1) {
    in0 = table.ok(2 * u, page0);
    in1 = table.ok(2 * u + 1, page1);
    row = table.row(2 * u + (wave >> 1), wave >> 1 ? page1 : page0);
  };
  int e0 = 0, e1 = 0;  // the next unit's table entries, fetched an iteration before they are looked at
  const auto entries_of = [&](int u) {
    e0 = table.entry(2 * u);
    e1 = table.entry(2 * u + 1);
  };
  const auto is_edge = [&](int u, bool ok) { return !ok || u >= full; };
  const auto dma = [&](int h) {  // rows_of()'s rows to half h
    const int lane = lane_anew(), sub = lane / PR, pc = lane % PR;  // row and piece of a lane in a load
    const auto kr = make_rsrc(static_cast<const uint8_t*>(p.kc) + row * SB, 16 * SB);
    const auto vr = make_rsrc(static_cast<const uint8_t*>(p.vc) + row * SB, 16 * SB);
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int r = i * RL + sub, at = ((wave & 1) * 8 + r) * SB;
      dma16(kr, &buf[h][0][(wave * 8 + i * RL) * RB], at + (pc ^ r) * 16);
      dma16(vr, &buf[h][1][(wave * 8 + i * RL) * RB], at + (pc ^ r * 2) * 16);
    }
  };
  // rows_of()'s rows of keys or of values to registers
  const auto fetch = [&](const void* cache, const float* scales, Pieces& x) {
    const int lane = lane_anew(), sub = lane / PR, pc = lane % PR;
    const auto rs = make_rsrc(static_cast<const uint8_t*>(cache) + row * SB, 16 * SB);
#pragma unroll
    for (int i = 0; i < PL; ++i) x.at[i] = bload(rs, ((wave & 1) * 8 + i * RL + sub) * SB + pc * 16);
    if (FP8) x.scale = scales[row + (wave & 1) * 8 + (lane & 7)];
  };
  const auto store_keys = [&](const Pieces& x, int h) {  // and from there to half h
    const int lane = lane_anew(), sub = lane / PR, pc = lane % PR;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int r = i * RL + sub;
      uint8_t* const to = &buf[h][0][(wave * 8 + r) * RB];
#pragma unroll
      for (int e = 0; e < (FP8 ? 2 : 1); ++e)
        *reinterpret_cast<uint4*>(to + ((FP8 ? pc * 2 + e : pc) ^ r) * 16) = half_piece<FP8>(x.at[i], e);
    }
    if (FP8) sc[h][0][wave * 8 + (lane & 7)] = x.scale;  // the same from eight lanes
  };
  // zeros for values that are not there or not finite
  const auto store_values = [&](const Pieces& x, int u, int h, bool ok0, bool ok1) {
    const int lane = lane_anew(), sub = lane / PR, pc = lane % PR;
    const bool edge = is_edge(u, ok0 && ok1);
    const uint32_t there = existing(w.total - u * 32, ok0, ok1) >> wave * 8;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < PL; ++i) {
      const int r = i * RL + sub;
      uint8_t* const to = &buf[h][1][(wave * 8 + r) * RB];
#pragma unroll
      for (int e = 0; e < (FP8 ? 2 : 1); ++e) {
        uint4 y = half_piece<FP8>(x.at[i], e);
        if (edge) {
          if (!(there >> r & 1)) y = make_uint4(0u, 0u, 0u, 0u);
          odd |= odd2(y.x) | odd2(y.y) | odd2(y.z) | odd2(y.w);
          y = make_uint4(even2(y.x), even2(y.y), even2(y.z), even2(y.w));
        }
        *reinterpret_cast<uint4*>(to + ((FP8 ? pc * 2 + e : pc) ^ r * 2) * 16) = y;
      }
    }
    if (FP8) sc[h][1][wave * 8 + (lane & 7)] = x.scale;
    if (edge && __any(odd)) odd_any = 1;
  };

  const float f2 = p.scale * kLog2e;
  f32x4 acc[CT][DT];
  float m[CT], l[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    m[ct] = -INFINITY;
    l[ct] = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[ct][d] = f32x4{};
  }
  if (threadIdx.x == 0) odd_any = 0;
  __syncthreads();
  const int ua = w.u0 + four;  // the four waves' units: every other one
  bool ok0 = false, ok1 = false;  // of the unit at hand
  if (ua < w.u1) {
    entries_of(ua);
    rows_of(ua, e0, e1);
    entries_of(ua + 2);
    ok0 = in0;
    ok1 = in1;
    if (FP8 || is_edge(ua, ok0 && ok1)) {
      Pieces x, y;
      fetch(p.kc, p.ks, x);
      fetch(p.vc, p.vs, y);
      store_keys(x, 0);
      store_values(y, ua, 0, ok0, ok1);
    } else {
      dma(0);
    }
  }
  Pieces nk, nv;  // EARLY: the next unit's, fetched an iteration before they are stored
  const auto fetch_early = [&](int u) {
    if (!EARLY || u >= w.u1) return;
    rows_of(u, e0, e1);
    entries_of(u + 2);
    fetch(p.kc, p.ks, nk);
    fetch(p.vc, p.vs, nv);
  };
  __builtin_amdgcn_s_waitcnt(0x0f70);  // Q is there: else the loop waits for it, and so for the loads behind it, each time
  fetch_early(ua + 2);
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)&bufs[0][0][0][0];
  const int rounds = (w.u1 - w.u0 + 1) >> 1;  // of all eight waves
  for (int i = 0; i < rounds; ++i) {
    const int u = ua + 2 * i, h = i & 1;
    if (!FP8) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's rows are there
    lds_barrier();
    const bool more = u + 2 < w.u1;
    if (!EARLY) {
      rows_of(u + 2, e0, e1);
      entries_of(u + 4);
    }
    const bool ok2 = in0, ok3 = in1;
    Pieces next;
    if (EARLY) {
      if (more) {
        store_keys(nk, h ^ 1);
        store_values(nv, u + 2, h ^ 1, ok2, ok3);
      }
      fetch_early(u + 4);
    } else if (FP8) {
      if (more) fetch(p.kc, p.ks, next);
    } else if (more) {
      if (is_edge(u + 2, ok2 && ok3)) {
        Pieces x, y;
        fetch(p.kc, p.ks, x);
        fetch(p.vc, p.vs, y);
        store_keys(x, h ^ 1);
        store_values(y, u + 2, h ^ 1, ok2, ok3);
        __builtin_amdgcn_s_waitcnt(0x0f70);  // said here: else the compiler waits behind the DMAs of the other path, too
      } else {
        dma(h ^ 1);
      }
    }
    const bool live = wrow < w.rows && u < w.u1;
    f32x4 s[CT][2];
    if (live) {
      const int lane = lane_anew(), g = lane >> 4, c = lane & 15;
      const uint8_t* const kl = &buf[h][0][c * RB + (g ^ (c & 7)) * 16];
      const uint8_t* const kl4 = &buf[h][0][c * RB + (g ^ 4 ^ (c & 7)) * 16];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) s[ct][0] = s[ct][1] = f32x4{};
      bf16x8 a[2][2];
      const auto keys = [&](int f) {
        const uint8_t* const at = (f & 1 ? kl4 : kl) + (f >> 1) * 128;
        a[f & 1][0] = *reinterpret_cast<const bf16x8*>(at);
        a[f & 1][1] = *reinterpret_cast<const bf16x8*>(at + 16 * RB);
      };
      keys(0);
#pragma unroll
      for (int f = 0; f < KF; ++f) {
        if (f + 1 < KF) keys(f + 1);
        bf16x8 ql;
        if (f >= KF - QL) ql = __builtin_bit_cast(bf16x8, qbuf[QL > 0 ? f - (KF - QL) : 0][four * 256 + wave * 64 + lane]);
        __builtin_amdgcn_sched_barrier(0);  // one step ahead: more would take the outputs' registers
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
          const bf16x8 b = ct == CT - 1 && f >= KF - QL ? ql : qf[ct][f];
          s[ct][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[f & 1][0], b, s[ct][0], 0, 0, 0);
          s[ct][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[f & 1][1], b, s[ct][1], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const f32x4 kq = FP8 ? *reinterpret_cast<const f32x4*>(&sc[h][0][t * 16 + g * 4]) * f2 : f32x4{} + f2;
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) s[ct][t] *= kq;
      }
    }
    if (FP8 && !EARLY && more) {  // the next unit's values take the registers that its keys leave
      store_keys(next, h ^ 1);
      fetch(p.vc, p.vs, next);
    }
    if (live) {
      const int lane = lane_anew(), g = lane >> 4, c = lane & 15, vrow = g * 4 + (c >> 2);
      const int p0 = u * 32;
      const bool edge = is_edge(u, ok0 && ok1);
      bf16x8 pf[CT];
#pragma unroll
      for (int ct = 0; ct < CT; ++ct)
        soft_weights<FP8, DT>(
            s[ct], [&](int t) { return *reinterpret_cast<const f32x4*>(&sc[h][1][t * 16 + g * 4]); }, edge,
            [&] {
              const Row rw(p, wrow + ct * 16, w.rows, w.first, w.hk, lane_anew() & 15);
              return rw.live ? existing(w.total - p0, ok0, ok1) & seen32(p, rw.words, rw.tok, p0 - w.ctx) : 0u;
            },
            m[ct], l[ct], acc[ct], pf[ct]);
      const uint32_t at = lds + (four * 4 + h * 2 + 1) * TILE + vrow * RB + (vrow & 7) * 32 + (c & 3) * 8;
#pragma unroll
      for (int d0 = 0; d0 < DT; d0 += 4) {
        bf16x4 lo[4], hi[4];
        const uint32_t b = at ^ (d0 & 7) * 32;
        if (d0 < 8)
          values4<0, 16 * RB>(b, b ^ 32, b ^ 64, b ^ 96, lo, hi);
        else
          values4<256, 16 * RB + 256>(b, b ^ 32, b ^ 64, b ^ 96, lo, hi);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bf16x8 a = __builtin_shufflevector(lo[i], hi[i], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
          for (int ct = 0; ct < CT; ++ct)
            acc[ct][d0 + i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pf[ct], acc[ct][d0 + i], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (FP8 && !EARLY && more) store_values(next, u + 2, h ^ 1, ok2, ok3);
    ok0 = ok2;
    ok1 = ok3;
  }

  // each four waves leave half of the dims to the others and join the other half of both sums
  constexpr int HT = DT / 2;
  const int lane = lane_anew(), g = lane >> 4, c = lane & 15;
  lds_barrier();
  f32x4* const give = reinterpret_cast<f32x4*>(&bufs[0][0][0][0]) + (four * 4 + wave) * CT * HT * 64 + lane;
  const f32x4* const take = reinterpret_cast<const f32x4*>(&bufs[0][0][0][0]) + ((four ^ 1) * 4 + wave) * CT * HT * 64 + lane;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    l[ct] += __shfl_xor(l[ct], 16);
    l[ct] += __shfl_xor(l[ct], 32);
    if (g == 0) sums[four][(wave * CT + ct) * 16 + c] = make_float2(m[ct], l[ct]);
#pragma unroll
    for (int d = 0; d < HT; ++d) give[(ct * HT + d) * 64] = four ? acc[ct][d] : acc[ct][d + HT];
  }
  __syncthreads();
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const Row rw(p, wrow + ct * 16, w.rows, w.first, w.hk, c);
    if (!rw.live) continue;
    const float2 other = sums[four ^ 1][(wave * CT + ct) * 16 + c];
    const float top = fmaxf(m[ct], other.x);
    // four waves without a reference have a sum only where every score was NaN
    const float fa = m[ct] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[ct] - top);
    const float fb = other.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(other.x - top);
    const float sum = four ? other.y * fb + l[ct] * fa : l[ct] * fa + other.y * fb;  // the same on both sides
    const int64_t nh = (int64_t)(w.first + rw.tok) * p.HQ + rw.head, i = w.slot + (wave * CT + ct) * 16 + c;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int d = 0; d < HT; ++d) {
      const f32x4 mine = four ? acc[ct][d + HT] : acc[ct][d];
      const f32x4 o = mine * fa + take[(ct * HT + d) * 64] * fb;
      const int at = (four * HT + d) * 16 + g * 4;
      if (w.parts > 1)
        *reinterpret_cast<f32x4*>(p.part + i * D + at) = o;
      else
        *reinterpret_cast<uint2*>(p.out + nh * D + at) = make_uint2(cvt_pk2(o[0] * inv, o[1] * inv), cvt_pk2(o[2] * inv, o[3] * inv));
    }
    if (g != 0 || four != 0) continue;
    if (w.parts > 1)
      p.ml[i] = make_float2(top, sum);
    else if (p.lse != nullptr)
      p.lse[nh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * kLn2;
  }

  if (odd_any == 0) return;
#pragma unroll 1
  for (int ct = 0; ct < CT; ++ct) {
    const Row rw(p, wrow + ct * 16, w.rows, w.first, w.hk, c);
    if (!rw.live) continue;
    const int64_t nh = (int64_t)(w.first + rw.tok) * p.HQ + rw.head;
#pragma unroll 1
    for (int u = w.u0; u < w.u1; ++u) {
      entries_of(u);
      rows_of(u, e0, e1);
      if (!is_edge(u, in0 && in1)) continue;
      const int p0 = u * 32;
      const uint32_t see = existing(w.total - p0, in0, in1) & seen32(p, rw.words, rw.tok, p0 - w.ctx);
#pragma unroll 1
      for (int key = 0; key < 32; ++key) {
        if (!(see >> key & 1)) continue;
        const int64_t v = (table.row(2 * u + (key >> 4), key >> 4 ? e1 : e0) + (key & 15)) * D;
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) {
          const int d = (four * HT + (i >> 2)) * 16 + g * 4 + (i & 3);  // what this lane has written
          const float x = FP8 ? bf2f(cvt_fp8x2(static_cast<const uint8_t*>(p.vc)[v + d], false) & 0xffffu)
                              : bf2f(static_cast<const uint16_t*>(p.vc)[v + d]);
          if (fabsf(x) < INFINITY) continue;
          if (w.parts > 1)
            p.part[(int64_t)(w.slot + (wave * CT + ct) * 16 + c) * D + d] += x;
          else
            p.out[nh * D + d] = (uint16_t)f2bf(bf2f(p.out[nh * D + d]) + x);
        }
      }
    }
  }
}

// Joins the parts of a row: one wave per (row, head), 4 D / 256 dims a lane.
template <int D>
__global__ void __launch_bounds__(256) tree_join_k(TreeParams p, int R) {
  constexpr int E = D / 64;
  const int64_t nh = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  if (nh >= p.N * p.HQ) return;
  const uint2 at = p.joins[nh];
  const int parts = (int)at.y;
  if (parts < 2) return;  // done, or of no sequence
  const int64_t step = (int64_t)p.HKV * R;
  const float2* const ml = p.ml + at.x;
  const float* const src = p.part + (int64_t)at.x * D + lane * E;
  float top = -INFINITY, sum = 0.f, o[E] = {};
  for (int s = lane; s < parts; s += 64) top = fmaxf(top, ml[s * step].x);
#pragma unroll
  for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
  for (int s0 = 0; s0 < parts; s0 += 64) {
    const float2 x = s0 + lane < parts ? ml[(s0 + lane) * step] : make_float2(top, 0.f);
    // a part without a maximum has zeros, or NaN where every score was
    const float f = x.x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(x.x - top);
    sum += f * x.y;
#pragma unroll 4
    for (int s = 0; s < min(parts - s0, 64); ++s) {
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(f), s));
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += w * src[(s0 + s) * step * D + e];
    }
  }
  sum = wave_sum64(sum);
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
  t.rows = mean <= 16 ? 16 : mean <= 64 ? 64 : 128;  // times on both sides: at the top of this file
  // an upper bound of sum ceil(n_b G / rows) over the sequences with rows, which are `seqs` at most
  const int64_t blocks = (N * G + seqs * (t.rows - 1)) / t.rows, units = (max_pages * page + 31) / 32;
  t.least = t.rows == 16 ? 4 : 8;  // a unit for each wave; as much work as the start of a part
  const int64_t at_once = t.rows == 128 ? 256 : 256 * 256 / D;  // workgroups that the GPU holds
  t.target = units > t.least ? std::max<int64_t>(1, at_once / HKV) : 0;
  t.shares = t.target == 0 ? blocks
                           : std::min<int64_t>(std::max<int64_t>(t.target, blocks + blocks / 4 + 1),
                                               blocks * ((units + t.least - 1) / t.least));
  t.slots = t.target == 0 ? 0 : t.shares * HKV * t.rows;
  return t;
}

template <int D, bool FP8>
static void (*tree_kernel(int rows))(TreeParams) {
  return rows == 16 ? tree_narrow_k<D, FP8> : rows == 64 ? tree_wide_k<D, FP8, 1> : tree_wide_k<D, FP8, 2>;
}

hipError_t launch_tree_attn(const TreeParams& p, const TreePlan& t, int D, bool fp8, hipStream_t st) {
  const auto kernel = D == 256 ? (fp8 ? tree_kernel<256, true>(t.rows) : tree_kernel<256, false>(t.rows))
                               : (fp8 ? tree_kernel<128, true>(t.rows) : tree_kernel<128, false>(t.rows));
  hipLaunchKernelGGL(kernel, dim3((unsigned)(t.shares * p.HKV)), dim3(t.rows == 16 ? 256 : 512), 0, st, p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || t.target == 0) return err;
  hipLaunchKernelGGL(D == 256 ? tree_join_k<256> : tree_join_k<128>, dim3((unsigned)((p.N * p.HQ + 3) / 4)), dim3(256),
                     0, st, p, t.rows);
  return hipGetLastError();
}

}  // namespace ojx

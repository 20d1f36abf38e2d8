// Verification of drafted tokens against the target's distributions, with random numbers that the caller gives.
//
// Row j of a sequence carries the logits of what follows token j; row 0 is the last token, which stands, the others were
// drafted, each behind the row that it follows. With p = softmax(logits / T) of the current row (first row 0), its children
// are looked at in order. What is left of p after a rejections is
//   w = max(p - a q, 0), t = sum w   (a = 0 and t = 1 at first; a grows by t with every rejection),
// q being the distribution that the children were drawn from: the recursion w <- max(w / t - q, 0) in closed form. Without
// q a drafted token was certain: w = p less the rejected tokens. Child x with the random number u is accepted if u q(x) t <
// w(x) (q(x) = 1 without q), and becomes the current row. When no child is left, the next token is the first i with w_0 + ..
// + w_i > u_0 t.
//
// All of it is computed in 64 bits: a vocabulary has some 10^5 borders between tokens, and with sums that are off by 2^-24
// one draw in a hundred would fall on the wrong side of one.
//
//   draft_chunks_k  a workgroup per chunk of a row: its largest logit, where it is, and the sum of the exponentials below it
//   draft_rows_k    a wave per row: those put together; p and q of the row's token under the row that it follows
//   draft_sums_k    once for each of the first rejections: a workgroup per chunk of a sequence walks over the rows up to that
//                   rejection, all it needs being in draft_rows_k's few numbers, and sums w over the chunk
//   draft_next_k    a workgroup per sequence: the whole walk, the accepted rows, the next token
// The two in the middle are launched with q and more than a few chunks; otherwise draft_next_k does their work.
//
// What bounds it: 64 sequences of up to 12 rows of 131072 bf16 logits (71 million, 142 MB) with a draft model's probabilities
// take 108 to 112 us. The chunks are 55 to 60 of them, the vector unit's: 20 operations a logit, issued 80% of the time, where
// memory would allow 27 us. Each launch of draft_sums_k is 4 us with nothing to do, 7 with a few sequences left and 14 with all
// of them (50 MB); draft_rows_k 5, draft_next_k 9: latency. Few rows are latency alone: 17 us for 6 rows of 32000 in two launches.
#include "ojx_internal.h"

#include <algorithm>

namespace ojx {

struct DraftChunk {
  float top;    // the largest logit; NaN where one is NaN or +infinity
  int32_t at;   // its first place (temperature 0)
  double sum;   // of exp((x - top) / T)
};
struct DraftRow {
  float top;
  int32_t at;
  double sum;
  double p, q;       // of the row's token, in the row above it; p < 0: no such row
  int32_t above, ok; // the row above in the sequence, or -1; ok: the row has a distribution
  int64_t token;
};

struct DraftWalk {
  int j, cur, count, rejections;  // the next row to look at, the current one, accepted so far
  double a, t;                    // without q a = 1 says that t has to be summed
  int first, n;                   // the sequence's rows, its temperature
  float temp, pad;
};

namespace {

constexpr int kPiece = 8192;  // logits of a chunk
constexpr int kSumThreads = 512;  // of a chunk of draft_sums_k (the largest case 109 us, 112 with 256, 114 with 1024)

__device__ __forceinline__ float value(const uint16_t* p) { return bf2f(*p); }
__device__ __forceinline__ float value(const float* p) { return *p; }
__device__ __forceinline__ void unpack(uint4 x, float (&f)[8]) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = bf2f(w[i] & 0xffffu);
    f[2 * i + 1] = bf2f(w[i] >> 16);
  }
}
__device__ __forceinline__ void unpack(uint4 x, float (&f)[4]) {
  f[0] = __uint_as_float(x.x);
  f[1] = __uint_as_float(x.y);
  f[2] = __uint_as_float(x.z);
  f[3] = __uint_as_float(x.w);
}

// Eight places of a row from place e on; places outside [0, V) read as `none`. Rows need no alignment: what lies whole in
// the row and is aligned goes by 16 bytes.
template <typename T>
__device__ __forceinline__ void eight(const T* row, int64_t e, int64_t V, float none, float (&f)[8]) {
  constexpr int W = 16 / sizeof(T);
  const T* const p = row + e;
  if (e >= 0 && e + 8 <= V && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < 8 / W; ++i) {
      float x[W];
      unpack(reinterpret_cast<const uint4*>(p)[i], x);
#pragma unroll
      for (int j = 0; j < W; ++j) f[i * W + j] = x[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = e + i >= 0 && e + i < V ? value(p + i) : none;
  }
}
// The same, still packed.
template <typename T>
struct Raw {
  uint4 x[sizeof(T) / 2];
};
__device__ __forceinline__ void pack(const float (&f)[8], Raw<uint16_t>& r) {  // exact: they come from bf16
  r.x[0] = make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
}
__device__ __forceinline__ void pack(const float (&f)[8], Raw<float>& r) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    r.x[i] = make_uint4(__float_as_uint(f[4 * i]), __float_as_uint(f[4 * i + 1]), __float_as_uint(f[4 * i + 2]),
                        __float_as_uint(f[4 * i + 3]));
}
template <typename T>
__device__ __forceinline__ Raw<T> eight_raw(const T* row, int64_t e, int64_t V) {
  Raw<T> r;
  const T* const p = row + e;
  if (e >= 0 && e + 8 <= V && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.x[i] = reinterpret_cast<const uint4*>(p)[i];
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = e + i >= 0 && e + i < V ? value(p + i) : -INFINITY;
    pack(f, r);
  }
  return r;
}
__device__ __forceinline__ void open(const Raw<uint16_t>& r, float (&f)[8]) { unpack(r.x[0], f); }
__device__ __forceinline__ void open(const Raw<float>& r, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float x[4];
    unpack(r.x[i], x);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[i * 4 + j] = x[j];
  }
}
// Places of a row are taken from its first 16-byte border on: this many before the row's own first place.
template <typename T>
__device__ __forceinline__ int lead(const T* row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}

// The temperature of sequence b; 0: the first largest logit is certain.
__device__ __forceinline__ float temperature(const DraftParams& p, int b) {
  const float t = p.temp == nullptr ? 1.f : p.temp[b];
  return t > 0.f ? t : 0.f;
}
// 2^f for |f| <= 1/2, 3.2e-16 off at most beside the roundings, as much as one and a half of them: a polynomial of degree 10,
// interpolated at Chebyshev's nodes, its first coefficient 1 (degree 9: 3.8e-14, degree 8: 1.1e-12 and two operations of 16 a
// logit less: 108 us in place of 112 for the largest case. A caller who is promised 64 bits gets them).
__device__ __forceinline__ double exp2_part(double f) {
  double x = 0x1.e6063f7217bc6p-28;
  x = fma(x, f, 0x1.b675bca4eeebbp-24);
  x = fma(x, f, 0x1.62bfd47773353p-20);
  x = fma(x, f, 0x1.ffcb54062e698p-17);
  x = fma(x, f, 0x1.430913096fd9fp-13);
  x = fma(x, f, 0x1.5d87fe9d7a584p-10);
  x = fma(x, f, 0x1.3b2ab6fba1ddap-7);
  x = fma(x, f, 0x1.c6b08d703ce49p-5);
  x = fma(x, f, 0x1.ebfbdff82c598p-3);
  x = fma(x, f, 0x1.62e42fefa3a19p-1);
  return fma(x, f, 1.0);
}
constexpr double kRound = 0x1.8p52;  // added and taken off again: rounds to a whole number, whose low bits it leaves in the sum
__device__ __forceinline__ double times_exp2(double x, double rounded) {
  return __hiloint2double(__double2hiint(x) + (int)((uint32_t)__double2loint(rounded) << 20), __double2loint(x));
}
// 2^y for y <= 1/2; 2^-1000 where y is below -1000 or NaN.
__device__ __forceinline__ double exp2_down(double y) {
  y = fmax(y, -1000.0);
  const double t = y + kRound;
  return times_exp2(exp2_part(y - (t - kRound)), t);
}

// exp((x - top) / T) = 2^((x - top) c), c = 1 / (T log 2). In the loops over whole rows it is made as 2^(x c - k), k the
// whole number next to top c, times `rest` = 2^(k - top c): 16 operations a logit instead of 19, where the library's
// exponential would be 40 (the largest case makes 71 million of them, and is bound by them). `plain` says that the sizes do
// not allow it. A logit of -infinity counts as 2^-990 there, next to nothing.
struct Scale {
  double c, top, bias, rest;
  float least;  // logits below it count as this
  bool plain;
};
__device__ __forceinline__ Scale scale_of(float temp, float top) {
  Scale s;
  s.c = 0x1.71547652b82fep+0 / (double)temp;
  s.top = top;
  const double y = s.top * s.c, k = (y + kRound) - kRound;
  s.bias = kRound - k;
  s.rest = exp2_part(-fma(s.top, s.c, -k));
  s.least = (float)((k - 990.0) / s.c);
  s.plain = !(fabs(y) < 0x1p23) || !(s.least > -INFINITY);
  return s;
}
// Without `rest`; not where `plain`.
__device__ __forceinline__ double weight_part(float x, const Scale& s) {
  const double v = __builtin_elementwise_maximum(x, s.least), t = fma(v, s.c, s.bias);
  return times_exp2(exp2_part(fma(v, s.c, -(t - s.bias))), t);
}
__device__ __forceinline__ double weight(float x, const Scale& s) { return exp2_down(((double)x - s.top) * s.c); }
__device__ __forceinline__ double weight_or_none(float x, const Scale& s) {
  const double y = ((double)x - s.top) * s.c;
  return y > -1000.0 ? exp2_down(y) : 0.0;
}

// Sum of x over the lanes up to and including this one: by lane shifts within rows of 16, and the rows' last lanes handed on
// (a lane outside reads as zero).
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_add(double x) {
  const int lo = __builtin_amdgcn_update_dpp(0, __double2loint(x), CTRL, ROWS, 0xf, false);
  const int hi = __builtin_amdgcn_update_dpp(0, __double2hiint(x), CTRL, ROWS, 0xf, false);
  return x + __hiloint2double(hi, lo);
}
__device__ __forceinline__ double wave_upto(double x) {
  x = dpp_add<0x111, 0xf>(x);
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);
  return dpp_add<0x143, 0xc>(x);
}
__device__ __forceinline__ double lane_of(double x, int l) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), l), __builtin_amdgcn_readlane(__double2loint(x), l));
}
__device__ __forceinline__ double wave_add(double x) { return lane_of(wave_upto(x), 63); }
// Sum over the workgroup, in wave order; red: 16 doubles.
__device__ __forceinline__ double block_add(double x, double* red) {
  x = wave_add(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = 0.0;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) t += red[w];
  return t;
}

// Where row r belongs: its sequence, or -1.
__device__ __forceinline__ int owner(const DraftParams& p, int64_t r, SeqPlace& at) {
  const int lo = seq_bound(p.q_ptr, 0, p.N);
  if (r < lo) return -1;
  return seq_find(p.q_ptr, p.B, p.N, [](int, int n) { return n; }, [=](int, int upto) { return lo + upto > r; }, at) ? at.seq
                                                                                                              : -1;
}

// `each` chunks of a row for a workgroup, the next one's logits on their way while one is summed. (Workgroups of 512 and 1024
// threads, with 16 and 8 logits a thread in place of 32: 6% and 29% more time for the largest case.)
template <typename T>
__global__ void __launch_bounds__(256) draft_chunks_k(DraftParams p, int each, int groups) {
  __shared__ float tops[4], temp;
  __shared__ int32_t ats[4];
  __shared__ int some;
  __shared__ double red[16];
  const int64_t r = blockIdx.x / (uint32_t)groups;
  const int first = (blockIdx.x - (int)(r * groups)) * each, last = min(first + each, p.chunks), wave = threadIdx.x >> 6;
  const T* const row = static_cast<const T*>(p.logits) + r * p.ldl;
  const int64_t e = (int64_t)threadIdx.x * 8 - lead(row);
  Raw<T> raw[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) raw[i] = eight_raw(row, e + (int64_t)first * kPiece + i * 2048, p.V);
  if (wave == 0) {
    SeqPlace place;
    const int b = owner(p, r, place);
    if (threadIdx.x == 0) {
      some = b >= 0;
      temp = b >= 0 ? temperature(p, b) : 0.f;
    }
  }
  __syncthreads();
  if (!some) return;
  const float t = temp;
  for (int chunk = first; chunk < last; ++chunk) {
    float x[4][8];
#pragma unroll
    for (int i = 0; i < 4; ++i) open(raw[i], x[i]);
    if (chunk + 1 < last)
#pragma unroll
      for (int i = 0; i < 4; ++i) raw[i] = eight_raw(row, e + (int64_t)(chunk + 1) * kPiece + i * 2048, p.V);
    float top = -INFINITY;  // NaN where one is
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) top = __builtin_elementwise_maximum(top, x[i][j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) tops[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) top = __builtin_elementwise_maximum(top, tops[i]);
    const bool odd = !(top < INFINITY);
    DraftChunk out{odd ? __uint_as_float(0x7fc00000u) : top, 0, 0.0};
    if (t == 0.f) {  // the same for all threads
      int32_t at = 0x7fffffff;
#pragma unroll
      for (int i = 3; i >= 0; --i)
#pragma unroll
        for (int j = 7; j >= 0; --j)
          if (x[i][j] == top) at = (int32_t)(e + (int64_t)chunk * kPiece + i * 2048 + j);
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
      if ((threadIdx.x & 63) == 0) ats[wave] = at;
      __syncthreads();
      out.at = min(min(ats[0], ats[1]), min(ats[2], ats[3]));
      out.sum = 1.0;
      __syncthreads();  // before the next chunk's
    } else {
      const Scale sc = scale_of(t, top);
      double s = 0.0;
      if (top > -INFINITY && !odd) {
        if (!sc.plain) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += weight_part(x[i][j], sc);
          s *= sc.rest;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) s += weight(x[i][j], sc);
        }
      }
      out.sum = block_add(s, red);
    }
    if (threadIdx.x == 0) p.parts[r * p.chunks + chunk] = out;
  }
}

// A row's chunks put together; the whole wave calls.
__device__ __forceinline__ void row_total(const DraftParams& p, int64_t r, float t, float& top, int32_t& at, double& sum) {
  const int lane = threadIdx.x & 63;
  const DraftChunk* const parts = p.parts + r * p.chunks;
  top = -INFINITY;
  bool odd = false;
  for (int c = lane; c < p.chunks; c += 64) {
    const float x = parts[c].top;
    odd |= !(x < INFINITY);
    top = fmaxf(top, x);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  at = 0x7fffffff;
  sum = 0.0;
  const Scale sc = scale_of(t > 0.f ? t : 1.f, top);
  for (int c = lane; c < p.chunks; c += 64) {
    if (t == 0.f && parts[c].top == top) at = min(at, parts[c].at);
    if (t > 0.f) sum += parts[c].sum * weight(parts[c].top, sc);  // the sum is 0 where the largest is -infinity
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
  sum = t > 0.f ? wave_add(sum) : 1.0;
  if (__any(odd)) top = __uint_as_float(0x7fc00000u);
}

// What the walk has to know of row j of a sequence; the whole wave calls.
template <typename T, typename Q, bool PROBS>
__device__ __forceinline__ void row_info(const DraftParams& p, int64_t first, int j, float t) {
  const int lane = threadIdx.x & 63;
  const int64_t r = first + j;
  DraftRow out{};
  int above = p.parents == nullptr ? j - 1 : p.parents[r];
  out.token = p.tokens[r];
  if (above < 0 || above >= j) above = -1;
  row_total(p, r, t, out.top, out.at, out.sum);
  out.ok = out.top > -INFINITY;  // not NaN
  out.above = above;
  out.p = -1.0;
  out.q = 1.0;
  if (above >= 0) {
    const int64_t a = first + above;
    const bool in = out.token >= 0 && out.token < p.V;
    const int64_t token = in ? out.token : 0;
    const float x = value(static_cast<const T*>(p.logits) + a * p.ldl + token);
    const float q = PROBS ? value(static_cast<const Q*>(p.probs) + a * p.ldp + token) : 0.f;
    float top;
    int32_t at;
    double sum;
    row_total(p, a, t, top, at, sum);
    // without q a token that an earlier child has too is gone with that one
    bool gone = !in;
    if (p.parents != nullptr && (!PROBS || t == 0.f)) {
      for (int i = above + 1 + lane; i < j; i += 64)
        gone |= p.parents[first + i] == above && p.tokens[first + i] == out.token;
      gone = __any(gone);
    }
    if (top > -INFINITY) {
      out.p = 0.0;
      if (!gone) {
        if (t == 0.f)
          out.p = out.token == at ? 1.0 : 0.0;
        else
          out.p = weight_or_none(x, scale_of(t, top)) / sum;
      }
      if (PROBS && t > 0.f) out.q = in && q > 0.f ? (double)q : 0.0;
    }
  }
  if (lane == 0) p.rows[r] = out;
}

template <typename T, typename Q>
__global__ void __launch_bounds__(256) draft_rows_k(DraftParams p) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.N) return;
  SeqPlace place;
  const int b = owner(p, r, place);
  if (b >= 0) row_info<T, Q, true>(p, place.first, (int)(r - place.first), temperature(p, b));
}

// Where the walk over a sequence's rows stands.
using Walk = DraftWalk;

// Without q what is left is one less the rejected tokens' shares, as long as that is more than this; where more digits than three
// have cancelled it is summed, should another token be tested (a = 1: it has to be).
constexpr double kCancelled = 1e-3;

// On to the next rejection with q or test with a sum that has to be made (true: what is left has to be summed before the walk
// can go on), or to the end; the whole wave calls, with the walk the same in all lanes. write(i, j): row j is the i-th accepted.
template <bool PROBS, typename Write>
__device__ __forceinline__ bool walk_on(const DraftParams& p, Walk& w, Write write) {
  const int lane = threadIdx.x & 63;
  for (int base = w.j & ~63; base < w.n; base += 64) {
    const int mine = min(base + lane, w.n - 1);
    const DraftRow* const row = p.rows + w.first + mine;
    const int above = row->above;
    const double rp = row->p, rq = row->q, u = p.u[w.first + mine];
    for (; w.j < min(base + 64, w.n); ++w.j) {
      const int l = w.j - base;
      if (__builtin_amdgcn_readlane(above, l) != w.cur) continue;
      const double x = lane_of(rp, l), q = lane_of(rq, l), v = lane_of(u, l);
      if (x < 0.0) continue;
      if (!PROBS && w.a > 0.0) return true;
      const double left = PROBS && w.temp > 0.f && w.a > 0.0 ? fmax(x - w.a * q, 0.0) : x;
      if (v * q * w.t < left) {
        write(w.count, w.j);
        ++w.count;
        w.cur = w.j;
        w.a = 0.0;
        w.t = 1.0;
      } else if (PROBS && w.temp > 0.f) {
        w.a += w.t;
        ++w.rejections;
        ++w.j;
        return true;
      } else {
        ++w.rejections;
        if (w.temp > 0.f && x > 0.0) {
          w.t -= x;
          w.a = w.t < kCancelled ? 1.0 : 0.0;
        }
      }
    }
  }
  return false;
}

// What is left of a row's distribution at eight places: p in units of the largest logit's (unit 1), or with q as it is.
template <typename T, typename Q, bool PROBS>
__device__ __forceinline__ void left_of(const DraftParams& p, int64_t r, int64_t e, Scale sc, double unit, double a,
                                        double (&w)[8]) {
  float x[8], q[8];
  eight(static_cast<const T*>(p.logits) + r * p.ldl, e, p.V, -INFINITY, x);
  if (PROBS && a > 0.0) eight(static_cast<const Q*>(p.probs) + r * p.ldp, e, p.V, 0.f, q);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = weight_or_none(x[i], sc) * unit;
  if (PROBS && a > 0.0)
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = q[i] > 0.f ? fmax(w[i] - a * (double)q[i], 0.0) : w[i];
}

// The sum after rejection i of sequence b, from draft_sums_k; the whole wave calls.
__device__ __forceinline__ double known_sum(const DraftParams& p, int b, int i) {
  double x = 0.0;
  for (int c = threadIdx.x & 63; c < p.chunks; c += 64) x += p.sums[((int64_t)i * p.B + b) * p.chunks + c];
  return wave_add(x);
}

// The sum of what is left with q at 8 E places, `step` apart by eights; not where sc is plain.
template <typename T, typename Q, int E>
__device__ __forceinline__ double left_sum(const DraftParams& p, int64_t r, int64_t e, int64_t step, const Scale& sc,
                                           double unit, double a) {
  float l[E][8], q[E][8];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    eight(static_cast<const T*>(p.logits) + r * p.ldl, e + i * step, p.V, -INFINITY, l[i]);
    eight(static_cast<const Q*>(p.probs) + r * p.ldp, e + i * step, p.V, 0.f, q[i]);
  }
  // a logit of -infinity counts for 2^-990 in weight_part: nothing may be left of it
  const double part = unit * sc.rest, none = 0x1p-980 * part;
  double x = 0.0;
#pragma unroll
  for (int i = 0; i < E; ++i)
#pragma unroll
    for (int k = 0; k < 8; ++k)
      x += fmax(weight_part(l[i][k], sc) * part - (q[i][k] > 0.f ? a * (double)q[i][k] : none), 0.0);
  return x;
}

// Rejection number `round`. Chunk 0's workgroup leaves where the walk stands (rejections = round + 1: at this rejection;
// fewer: it is over) and the rows accepted on the way.
template <typename T, typename Q, int THREADS>
__global__ void __launch_bounds__(THREADS) draft_sums_k(DraftParams p, int round) {
  __shared__ double red[16];
  __shared__ Walk held;
  const int b = blockIdx.x / (uint32_t)p.chunks, chunk = blockIdx.x - b * p.chunks, lane = threadIdx.x & 63;
  DraftWalk* const walks = p.walks + (int64_t)round * p.B;
  if (threadIdx.x < 64) {
    Walk w{1, 0, 1, 0, 0.0, 1.0};
    if (round == 0) {
      SeqPlace s;
      w.temp = temperature(p, b);
      if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == b; }, s)) s.n = 0;
      w.first = s.first;
      w.n = s.n;
    } else {
      w = walks[b - p.B];
    }
    if (w.rejections == round) {
      if (round > 0) w.t = known_sum(p, b, round - 1);
      walk_on<true>(p, w, [&](int i, int j) {
        if (chunk == 0 && lane == 0) p.path[w.first + i] = j;
      });
      if (w.temp == 0.f) w.rejections = 0;  // these need no sums
    }
    if (lane == 0) {
      held = w;
      if (chunk == 0) walks[b] = w;
    }
  }
  __syncthreads();
  const Walk w = held;
  if (w.rejections <= round) return;
  const int64_t r = w.first + w.cur;
  const Scale sc = scale_of(w.temp, p.rows[r].top);
  const double unit = 1.0 / p.rows[r].sum;
  const T* const row = static_cast<const T*>(p.logits) + r * p.ldl;
  const int64_t e = (int64_t)chunk * kPiece - lead(row) + threadIdx.x * 8;
  double x = 0.0;
  if (sc.plain) {
    for (int i = 0; i < kPiece; i += THREADS * 8) {
      double left[8];
      left_of<T, Q, true>(p, r, e + i, sc, unit, w.a, left);
#pragma unroll
      for (int k = 0; k < 8; ++k) x += left[k];
    }
  } else {
    x = left_sum<T, Q, kPiece / THREADS / 8>(p, r, e, THREADS * 8, sc, unit, w.a);
  }
  x = block_add(x, red);
  if (threadIdx.x == 0) p.sums[((int64_t)round * p.B + b) * p.chunks + chunk] = x;
}

// Dynamic LDS: chunks doubles, what is left in each chunk. The workgroup after the last sequence's has the rows of none.
template <typename T, typename Q, bool PROBS>
__global__ void __launch_bounds__(1024) draft_next_k(DraftParams p) {
  extern __shared__ double chunk_left[];
  __shared__ double red[4][16], tail[16];
  __shared__ Walk held;
  __shared__ int need, pick;
  __shared__ double level;
  __shared__ int first_hit[16], last_some[16];
  const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (b == p.B) {
    int lo, hi;
    seq_span(p.q_ptr, p.B, p.N, lo, hi);
    for (int64_t r = threadIdx.x; r < p.N; r += 1024)
      if (r < lo || r >= hi) p.path[r] = -1;
    return;
  }
  // from the start, or from the last rejection that draft_sums_k was launched for, if there were so many
  Walk w{1, 0, 1, 0, 0.0, 1.0};
  if (PROBS && p.rounds > 0) {
    w = p.walks[(int64_t)(p.rounds - 1) * p.B + b];
  } else {
    SeqPlace s;
    w.temp = temperature(p, b);
    if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == b; }, s)) return;
    w.first = s.first;
    w.n = s.n;
  }
  const int64_t first = w.first;
  const int n = w.n;
  const float t = w.temp;
  if (n == 0) {
    if (threadIdx.x == 0) {
      p.count[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  if (!PROBS || p.rounds == 0) {
    for (int j = wave; j < n; j += 16) row_info<T, Q, PROBS>(p, first, j, t);
    __syncthreads();
  }

  // what is left in four chunks, to all threads; without the tokens of the row's children before row `upto`, all of them
  // rejected
  const auto chunk_sums = [&](int64_t r, const Scale& sc, double unit, double a, int c0, int many, int upto) {
    const int64_t e0 = (int64_t)c0 * kPiece - lead(static_cast<const T*>(p.logits) + r * p.ldl) + threadIdx.x * 8;
    double sum[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      sum[k] = 0.0;
      if (k >= many) continue;
      const int64_t e = e0 + (int64_t)k * kPiece;
      if (PROBS && !sc.plain) {
        sum[k] = wave_add(left_sum<T, Q, 1>(p, r, e, 0, sc, unit, a));
        continue;
      }
      double w[8];
      left_of<T, Q, PROBS>(p, r, e, sc, unit, a, w);
      if (!PROBS)
        for (int j = (int)(r - first) + 1; j < upto; ++j) {
          const int64_t x = p.rows[first + j].token - e;
          if (p.rows[first + j].above == (int)(r - first) && x >= 0 && x < 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = i == (int)x ? 0.0 : w[i];
        }
#pragma unroll
      for (int i = 0; i < 8; ++i) sum[k] += w[i];
      sum[k] = wave_add(sum[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (lane == 0) red[k][wave] = sum[k];
    __syncthreads();
    double all = 0.0;
    for (int k = 0; k < many; ++k) {
      double x = 0.0;
      for (int v = 0; v < 16; ++v) x += red[k][v];
      if (threadIdx.x == 0) chunk_left[c0 + k] = x;
      all += x;
    }
    return all;
  };

  if (PROBS && w.rejections == p.rounds && p.rounds > 0 && wave == 0) w.t = known_sum(p, b, p.rounds - 1);
  if (threadIdx.x == 0) p.path[first] = 0;
  while (true) {
    if (wave == 0) {
      const bool more = walk_on<PROBS>(p, w, [&](int i, int j) {
        if (lane == 0) p.path[first + i] = j;
      });
      if (lane == 0) {
        held = w;
        need = more;
      }
    }
    __syncthreads();
    w = held;
    const bool more = need;
    __syncthreads();
    if (!more) break;
    // with q a rejection beyond the ones that draft_sums_k was launched for
    const int64_t r = first + w.cur;
    const Scale sc = scale_of(t, p.rows[r].top);
    const double unit = 1.0 / p.rows[r].sum;
    w.t = 0.0;
    for (int c = 0; c < p.chunks; c += 4) w.t += chunk_sums(r, sc, unit, w.a, c, min(4, p.chunks - c), w.j);
    if (!PROBS) w.a = 0.0;
  }
  for (int i = w.count + threadIdx.x; i < n; i += 1024) p.path[first + i] = -1;
  const int64_t r = first + w.cur;
  const DraftRow row = p.rows[r];
  if (!row.ok || t == 0.f) {
    if (threadIdx.x == 0) {
      p.count[b] = w.count;
      p.next[b] = row.ok ? row.at : -1;
    }
    return;
  }
  // what is left in each chunk, in probabilities with q, otherwise in units of the largest logit's
  const Scale sc = scale_of(t, row.top);
  const double unit = PROBS ? 1.0 / row.sum : 1.0;
  double a = w.a;
  const auto whole = [&]() {
    for (int c = threadIdx.x; c < p.chunks; c += 1024) {
      const DraftChunk x = p.parts[r * p.chunks + c];
      chunk_left[c] = x.sum * weight_or_none(x.top, sc) * unit;
    }
    __syncthreads();
  };
  bool less = false;
  if (PROBS && a > 0.0) {
    if (w.rejections <= p.rounds)  // else they are there from the walk
      for (int c = threadIdx.x; c < p.chunks; c += 1024)
        chunk_left[c] = p.sums[((int64_t)(w.rejections - 1) * p.B + b) * p.chunks + c];
    __syncthreads();
  } else {
    whole();
    if (!PROBS) {
      // less the children's tokens; a chunk of which little is left (cancelled digits) is summed again without them
      if (wave == 0) {
        const int ahead = lead(static_cast<const T*>(p.logits) + r * p.ldl);
        bool some = false;
        for (int j0 = w.cur + 1; j0 < n; j0 += 64) {
          const DraftRow* const child = p.rows + first + min(j0 + lane, n - 1);
          const double x = j0 + lane < n && child->above == w.cur ? child->p : 0.0;
          const int c = x > 0.0 ? (int)((child->token + ahead) / kPiece) : 0;
          for (unsigned long long m = __ballot(x > 0.0); m != 0; m &= m - 1) {
            const int l = __builtin_ctzll(m), at = __builtin_amdgcn_readlane(c, l);
            const double before = chunk_left[at], after = before - lane_of(x, l) * row.sum;
            some = true;
            if (lane == 0) chunk_left[at] = before < 0.0 || after < kCancelled * before ? -1.0 : after;
          }
        }
        if (lane == 0) need = some;
      }
      __syncthreads();
      less = need;
      if (less)
        for (int c = 0; c < p.chunks; ++c) {
          if (chunk_left[c] >= 0.0) continue;  // the same for the whole workgroup: written before the barriers above
          chunk_sums(r, sc, unit, a, c, 1, n);
          __syncthreads();
        }
    }
  }
  int at = -1;
  for (int again = 0; again < 2; ++again) {
    // the chunk in which the sum passes its share; the last one that has anything where none does
    if (wave == 0) {
      double all = 0.0;
      for (int c0 = 0; c0 < p.chunks; c0 += 64) all += wave_add(c0 + lane < p.chunks ? chunk_left[c0 + lane] : 0.0);
      const double share = (double)p.u[first] * all;
      double before = 0.0, pick_before = 0.0;
      int c = -1;
      for (int c0 = 0; c0 < p.chunks; c0 += 64) {
        const double x = c0 + lane < p.chunks ? chunk_left[c0 + lane] : 0.0, upto = wave_upto(x);
        const unsigned long long some = __ballot(x > 0.0), hit = __ballot(x > 0.0 && before + upto > share);
        if (some != 0) {
          const int l = hit != 0 ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some);
          c = c0 + l;
          pick_before = before + (lane_of(upto, l) - lane_of(x, l));
        }
        if (hit != 0) break;
        before += lane_of(upto, 63);
      }
      if (lane == 0) {
        pick = c;
        level = share - pick_before;
      }
    }
    __syncthreads();
    const int c = pick;
    if (c >= 0) {
      const int64_t e = (int64_t)c * kPiece - lead(static_cast<const T*>(p.logits) + r * p.ldl) + threadIdx.x * 8;
      double x[8];
      left_of<T, Q, PROBS>(p, r, e, sc, unit, a, x);
      if (less)
        for (int j = w.cur + 1; j < n; ++j) {
          const int64_t k = p.rows[first + j].token - e;
          if (p.rows[first + j].above == w.cur && k >= 0 && k < 8)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = i == (int)k ? 0.0 : x[i];
        }
      double mine = 0.0;
#pragma unroll
      for (int i = 0; i < 8; ++i) mine += x[i];
      // the sum of the places before this thread's
      const double upto = wave_upto(mine);
      if (lane == 63) tail[wave] = upto;
      __syncthreads();
      double before = upto - mine;
      for (int v = 0; v < wave; ++v) before += tail[v];
      int hit = -1, some = -1;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        before += x[i];
        if (x[i] > 0.0) {
          some = (int)e + i;
          if (before > level && hit < 0) hit = (int)e + i;
        }
      }
      // the first place of the first wave that has one, else the last place with anything
      const unsigned long long hits = __ballot(hit >= 0), somes = __ballot(some >= 0);
      hit = __builtin_amdgcn_readlane(hit, hits != 0 ? __builtin_ctzll(hits) : 0);
      some = __builtin_amdgcn_readlane(some, somes != 0 ? 63 - __builtin_clzll(somes) : 0);
      if (lane == 0) {
        first_hit[wave] = hit;
        last_some[wave] = some;
      }
      __syncthreads();
      for (int v = 0; v < 16; ++v)
        if (last_some[v] >= 0) at = last_some[v];
      for (int v = 15; v >= 0; --v)
        if (first_hit[v] >= 0) at = first_hit[v];
    }
    if (at >= 0) break;  // the same for all threads
    // nothing left: the row's own distribution
    a = 0.0;
    less = false;
    __syncthreads();
    whole();
  }
  if (threadIdx.x == 0) {
    p.count[b] = w.count;
    p.next[b] = at;
  }
}

}  // namespace

int64_t draft_chunks(int64_t V) { return (V + 7 + kPiece - 1) / kPiece; }

// Rejections of a sequence whose sums are launches of their own. In a line of tokens nothing follows a rejection but the next
// token. A few chunks are summed by one workgroup sooner than by other launches: with them and without, trees of 64 x 6 rows
// take 43 and 33 us for 2 chunks, 46 and 44 for 4, 52 and 63 for 5; of one sequence of 6, 28 and 17, 32 and 27, 30 and 22 (33 and
// 34 for 7); lines of 64 x 6 29 and 26, 33 and 34, 35 and 38. Without rows there is no walk to leave.
static int draft_rounds(int64_t N, int64_t B, int64_t V, bool probs, bool tree) {
  return !probs || N == 0 || B == 0 || draft_chunks(V) <= 4 ? 0 : tree ? kDraftRounds : 1;
}

int64_t draft_work_bytes(int64_t N, int64_t B, int64_t V, bool probs) {
  const int64_t c = draft_chunks(V), rounds = draft_rounds(N, B, V, probs, true);
  return N * c * (int64_t)sizeof(DraftChunk) + N * (int64_t)sizeof(DraftRow) + rounds * B * (c * 8 + (int64_t)sizeof(DraftWalk));
}

hipError_t launch_verify(DraftParams p, bool f32, bool probs_f32, uint8_t* work, hipStream_t st) {
  p.chunks = (int)draft_chunks(p.V);
  p.rounds = draft_rounds(p.N, p.B, p.V, p.probs != nullptr, p.parents != nullptr);
  p.parts = reinterpret_cast<DraftChunk*>(work);
  p.rows = reinterpret_cast<DraftRow*>(p.parts + p.N * p.chunks);
  p.walks = reinterpret_cast<DraftWalk*>(p.rows + p.N);
  p.sums = reinterpret_cast<double*>(p.walks + p.rounds * p.B);
  const dim3 wide(256), rows((unsigned)((p.N + 3) / 4));
  if (p.N > 0) {
    // two chunks a workgroup where there are enough of them for the chip twice over: 50 us in place of 53 in the largest case
    const int each = p.N * p.chunks >= 8192 ? 2 : 1, groups = (p.chunks + each - 1) / each;
    hipLaunchKernelGGL(f32 ? draft_chunks_k<float> : draft_chunks_k<uint16_t>, dim3((unsigned)(p.N * groups)), wide, 0, st, p,
                       each, groups);
  }
  if (p.rounds > 0) {
    const auto rows_k = probs_f32 ? (f32 ? draft_rows_k<float, float> : draft_rows_k<uint16_t, float>)
                                  : (f32 ? draft_rows_k<float, uint16_t> : draft_rows_k<uint16_t, uint16_t>);
    const auto sums_k = probs_f32 ? (f32 ? draft_sums_k<float, float, kSumThreads> : draft_sums_k<uint16_t, float, kSumThreads>)
                                  : (f32 ? draft_sums_k<float, uint16_t, kSumThreads> : draft_sums_k<uint16_t, uint16_t, kSumThreads>);
    hipLaunchKernelGGL(rows_k, rows, wide, 0, st, p);
    for (int i = 0; i < p.rounds; ++i)
      hipLaunchKernelGGL(sums_k, dim3((unsigned)(p.B * p.chunks)), dim3(kSumThreads), 0, st, p, i);
  }
  const auto next_k = p.probs == nullptr ? (f32 ? draft_next_k<float, float, false> : draft_next_k<uint16_t, float, false>)
                      : probs_f32 ? (f32 ? draft_next_k<float, float, true> : draft_next_k<uint16_t, float, true>)
                                  : (f32 ? draft_next_k<float, uint16_t, true> : draft_next_k<uint16_t, uint16_t, true>);
  hipLaunchKernelGGL(next_k, dim3((unsigned)(p.B + 1)), dim3(1024), p.chunks * 8, st, p);
  return hipGetLastError();
}

}  // namespace ojx

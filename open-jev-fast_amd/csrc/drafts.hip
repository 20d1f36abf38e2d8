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
//   draft_sums_k    (with q, once for each of the first rejections) a workgroup per chunk of a sequence: walks over the rows
//                   up to that rejection, all it needs being in draft_rows_k's few numbers, and sums w over the chunk
//   draft_next_k    a workgroup per sequence: the whole walk, the accepted rows, the next token
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

namespace {

constexpr int kPiece = 8192;  // logits of a chunk

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
// exp((x - top) / T), rt = 1 / T
__device__ __forceinline__ double weight(float x, float top, double rt) {
  return x == -INFINITY ? 0.0 : exp(((double)x - (double)top) * rt);
}

__device__ __forceinline__ double wave_add(double x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
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

template <typename T>
__global__ void __launch_bounds__(256) draft_chunks_k(DraftParams p) {
  __shared__ float tops[4];
  __shared__ int32_t ats[4];
  __shared__ double red[16];
  const int64_t r = blockIdx.x / (uint32_t)p.chunks;
  const int chunk = blockIdx.x - (int)(r * p.chunks), wave = threadIdx.x >> 6;
  const T* const row = static_cast<const T*>(p.logits) + r * p.ldl;
  const int64_t e0 = (int64_t)chunk * kPiece - lead(row);
  float x[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i) eight(row, e0 + (i * 256 + threadIdx.x) * 8, p.V, -INFINITY, x[i]);
  SeqPlace place;
  const int b = owner(p, r, place);
  if (b < 0) return;
  const float t = temperature(p, b);
  float top = -INFINITY;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      top = fmaxf(top, x[i][j]);
      odd |= !(x[i][j] < INFINITY);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if ((threadIdx.x & 63) == 0) tops[wave] = top;
  odd = __syncthreads_or(odd);
  top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  DraftChunk out{odd ? __uint_as_float(0x7fc00000u) : top, 0, 0.0};
  if (t == 0.f) {  // the same for all threads
    int32_t at = 0x7fffffff;
#pragma unroll
    for (int i = 3; i >= 0; --i)
#pragma unroll
      for (int j = 7; j >= 0; --j)
        if (x[i][j] == top) at = (int32_t)(e0 + (i * 256 + threadIdx.x) * 8 + j);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
    if ((threadIdx.x & 63) == 0) ats[wave] = at;
    __syncthreads();
    out.at = min(min(ats[0], ats[1]), min(ats[2], ats[3]));
    out.sum = 1.0;
  } else {
    const double rt = 1.0 / (double)t;
    double s = 0.0;
    if (top > -INFINITY && !odd)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) s += weight(x[i][j], top, rt);
    out.sum = block_add(s, red);
  }
  if (threadIdx.x == 0) p.parts[r * p.chunks + chunk] = out;
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
  const double rt = t > 0.f ? 1.0 / (double)t : 0.0;
  for (int c = lane; c < p.chunks; c += 64) {
    if (t == 0.f && parts[c].top == top) at = min(at, parts[c].at);
    if (t > 0.f && parts[c].top > -INFINITY) sum += parts[c].sum * exp(((double)parts[c].top - (double)top) * rt);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) at = min(at, __shfl_xor(at, o));
  sum = t > 0.f ? wave_add(sum) : 1.0;
  if (__any(odd)) top = __uint_as_float(0x7fc00000u);
}

template <typename T, typename Q, bool PROBS>
__global__ void __launch_bounds__(256) draft_rows_k(DraftParams p) {
  const int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= p.N) return;
  const int lane = threadIdx.x & 63;
  SeqPlace place;
  const int b = owner(p, r, place);
  if (b < 0) {
    if (lane == 0) p.path[r] = -1;
    return;
  }
  const float t = temperature(p, b);
  const int j = (int)(r - place.first);
  DraftRow out{};
  row_total(p, r, t, out.top, out.at, out.sum);
  out.ok = out.top > -INFINITY;  // not NaN
  out.token = p.tokens[r];
  int above = p.parents == nullptr ? j - 1 : p.parents[r];
  if (above < 0 || above >= j) above = -1;
  out.above = above;
  out.p = -1.0;
  out.q = 1.0;
  if (above >= 0) {
    const int64_t a = place.first + above;
    float top;
    int32_t at;
    double sum;
    row_total(p, a, t, top, at, sum);
    const bool in = out.token >= 0 && out.token < p.V;
    // without q a token that an earlier child has too is gone with that one
    bool gone = !in;
    if (!PROBS || t == 0.f)
      for (int i = above + 1 + lane; i < j; i += 64)
        gone |= (p.parents == nullptr ? i - 1 : p.parents[place.first + i]) == above && p.tokens[place.first + i] == out.token;
    gone = __any(gone);
    if (top > -INFINITY) {
      out.p = 0.0;
      if (!gone) {
        if (t == 0.f)
          out.p = out.token == at ? 1.0 : 0.0;
        else
          out.p = weight(value(static_cast<const T*>(p.logits) + a * p.ldl + out.token), top, 1.0 / (double)t) / sum;
      }
      if (PROBS && t > 0.f) {
        out.q = in ? value(static_cast<const Q*>(p.probs) + a * p.ldp + out.token) : 0.f;
        if (!(out.q > 0.0)) out.q = 0.0;
      }
    }
  }
  if (lane == 0) p.rows[r] = out;
}

// Where the walk over a sequence's rows stands.
struct Walk {
  int j, cur, count, rejections;
  double a, t;
};

// On to the next rejection whose sum of what is left is not known (true), or to the end (false); the whole wave calls, with
// the walk the same in all lanes. sum(i) is the sum after rejection i; known says how many there are. write(i, j): row j is
// the i-th accepted.
template <bool PROBS, typename Sum, typename Write>
__device__ __forceinline__ bool walk_on(const DraftParams& p, const SeqPlace& s, float temp, Walk& w, int known, Sum sum,
                                        Write write) {
  const int lane = threadIdx.x & 63;
  for (int base = w.j & ~63; base < s.n; base += 64) {
    const int mine = min(base + lane, s.n - 1);
    const DraftRow* const row = p.rows + s.first + mine;
    const int above = row->above;
    const double rp = row->p, rq = row->q, u = p.u[s.first + mine];
    for (; w.j < min(base + 64, s.n); ++w.j) {
      const int l = w.j - base;
      if (__builtin_amdgcn_readlane(above, l) != w.cur) continue;
      const double x = __shfl(rp, l), q = __shfl(rq, l), v = __shfl(u, l);
      if (x < 0.0) continue;
      const double left = PROBS && temp > 0.f ? (w.a > 0.0 ? fmax(x - w.a * q, 0.0) : x) : x;
      if (v * q * w.t < left) {
        write(w.count, w.j);
        ++w.count;
        w.cur = w.j;
        w.a = 0.0;
        w.t = 1.0;
      } else if (PROBS && temp > 0.f) {
        w.a += w.t;
        ++w.rejections;
        if (w.rejections > known) {
          ++w.j;
          return true;
        }
        w.t = sum(w.rejections - 1);
      } else {
        ++w.rejections;
        if (temp > 0.f) w.t -= x;
      }
    }
  }
  return false;
}

// What is left of a row's distribution at eight places: p in units of the largest logit's (scale 1), or with q as it is.
template <typename T, typename Q, bool PROBS>
__device__ __forceinline__ void left_of(const DraftParams& p, int64_t r, int64_t e, float top, double rt, double scale,
                                        double a, double (&w)[8]) {
  float x[8];
  eight(static_cast<const T*>(p.logits) + r * p.ldl, e, p.V, -INFINITY, x);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = weight(x[i], top, rt) * scale;
  if (PROBS && a > 0.0) {
    float q[8];
    eight(static_cast<const Q*>(p.probs) + r * p.ldp, e, p.V, 0.f, q);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = q[i] > 0.f ? fmax(w[i] - a * (double)q[i], 0.0) : w[i];
  }
}

template <typename T, typename Q>
__global__ void __launch_bounds__(256) draft_sums_k(DraftParams p, int round) {
  __shared__ double red[16];
  __shared__ Walk held;
  __shared__ int stop;
  const int b = blockIdx.x / (uint32_t)p.chunks, chunk = blockIdx.x - b * p.chunks;
  SeqPlace s;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == b; }, s)) return;
  const float t = temperature(p, b);
  if (s.n == 0 || t == 0.f) return;
  if (threadIdx.x < 64) {
    Walk w{1, 0, 1, 0, 0.0, 1.0};
    const auto sum = [&](int i) {
      double x = 0.0;
      for (int c = threadIdx.x; c < p.chunks; c += 64) x += p.sums[((int64_t)i * p.B + b) * p.chunks + c];
      return wave_add(x);
    };
    const bool here = walk_on<true>(p, s, t, w, round, sum, [](int, int) {});
    if (threadIdx.x == 0) {
      held = w;
      stop = !here;
    }
  }
  __syncthreads();
  if (stop) return;
  const int64_t r = s.first + held.cur;
  const DraftRow row = p.rows[r];
  const double rt = 1.0 / (double)t, scale = 1.0 / row.sum;
  const int64_t e0 = (int64_t)chunk * kPiece - lead(static_cast<const T*>(p.logits) + r * p.ldl);
  double x = 0.0;
  for (int i = 0; i < 4; ++i) {
    double w[8];
    left_of<T, Q, true>(p, r, e0 + (i * 256 + threadIdx.x) * 8, row.top, rt, scale, held.a, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) x += w[k];
  }
  x = block_add(x, red);
  if (threadIdx.x == 0) p.sums[((int64_t)round * p.B + b) * p.chunks + chunk] = x;
}

// Dynamic LDS: chunks doubles, what is left in each chunk.
template <typename T, typename Q, bool PROBS>
__global__ void __launch_bounds__(1024) draft_next_k(DraftParams p) {
  extern __shared__ double chunk_left[];
  __shared__ double red[16], tail[16];
  __shared__ Walk held;
  __shared__ int need, pick;
  __shared__ double level;
  __shared__ int64_t found, last;
  const int b = blockIdx.x;
  SeqPlace s;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == b; }, s)) return;
  if (s.n == 0) {
    if (threadIdx.x == 0) {
      p.count[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  const float t = temperature(p, b);
  const double rt = t > 0.f ? 1.0 / (double)t : 0.0;
  // what is left in one chunk, to all threads; without q less the children's tokens, all of them rejected
  const auto chunk_sum = [&](int64_t r, const DraftRow& row, double scale, double a, int chunk, bool less) {
    const int64_t e = (int64_t)chunk * kPiece - lead(static_cast<const T*>(p.logits) + r * p.ldl) + threadIdx.x * 8;
    double w[8];
    left_of<T, Q, PROBS>(p, r, e, row.top, rt, scale, a, w);
    if (less)
      for (int j = (int)(r - s.first) + 1; j < s.n; ++j) {
        const int64_t x = p.rows[s.first + j].token - e;
        if (p.rows[s.first + j].above == (int)(r - s.first) && x >= 0 && x < 8)
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = i == (int)x ? 0.0 : w[i];
      }
    double x = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) x += w[i];
    return block_add(x, red);
  };

  Walk w{1, 0, 1, 0, 0.0, 1.0};
  const auto known_sum = [&](int i) {
    double x = 0.0;
    for (int c = threadIdx.x & 63; c < p.chunks; c += 64) x += p.sums[((int64_t)i * p.B + b) * p.chunks + c];
    return wave_add(x);
  };
  int known = PROBS ? p.rounds : 0;
  bool fresh = false;  // chunk_left holds the last rejection's sums
  if (threadIdx.x == 0) p.path[s.first] = 0;
  while (true) {
    if (threadIdx.x < 64) {
      const bool more = walk_on<PROBS>(p, s, t, w, known, known_sum, [&](int i, int j) {
        if (threadIdx.x == 0) p.path[s.first + i] = j;
      });
      if (threadIdx.x == 0) {
        held = w;
        need = more;
      }
    }
    __syncthreads();
    w = held;
    const bool more = need;
    __syncthreads();
    if (!more) break;
    // a rejection beyond the ones summed by the whole chip
    const int64_t r = s.first + w.cur;
    const DraftRow row = p.rows[r];
    double all = 0.0;
    for (int c = 0; c < p.chunks; ++c) {
      const double x = chunk_sum(r, row, 1.0 / row.sum, w.a, c, false);
      if (threadIdx.x == 0) chunk_left[c] = x;
      all += x;
    }
    w.t = all;
    known = w.rejections;
    fresh = true;
    __syncthreads();
  }
  for (int i = w.count + threadIdx.x; i < s.n; i += 1024) p.path[s.first + i] = -1;
  const int64_t r = s.first + w.cur;
  const DraftRow row = p.rows[r];
  if (!row.ok || t == 0.f) {
    if (threadIdx.x == 0) {
      p.count[b] = w.count;
      p.next[b] = row.ok ? row.at : -1;
    }
    return;
  }
  // what is left in each chunk, in probabilities with q, otherwise in units of the largest logit's
  double scale = PROBS ? 1.0 / row.sum : 1.0, a = w.a;
  const bool rejected = PROBS ? a > 0.0 : w.rejections > 0;
  const auto whole = [&]() {
    for (int c = threadIdx.x; c < p.chunks; c += 1024) {
      const DraftChunk x = p.parts[r * p.chunks + c];
      chunk_left[c] = x.top > -INFINITY ? x.sum * exp(((double)x.top - (double)row.top) * rt) * scale : 0.0;
    }
    __syncthreads();
  };
  bool less = false;
  if (PROBS && rejected) {
    if (!fresh || w.rejections <= p.rounds)
      for (int c = threadIdx.x; c < p.chunks; c += 1024)
        chunk_left[c] = p.sums[((int64_t)(w.rejections - 1) * p.B + b) * p.chunks + c];
    __syncthreads();
  } else {
    whole();
    if (!PROBS) {
      // the chunks of the children's tokens again without them; each once
      const int first = lead(static_cast<const T*>(p.logits) + r * p.ldl);
      for (int j = w.cur + 1; j < s.n; ++j) {
        const DraftRow child = p.rows[s.first + j];
        if (child.above != w.cur || child.token < 0 || child.token >= p.V) continue;
        less = true;
        const int c = (int)((child.token + first) / kPiece);
        const double x = chunk_sum(r, row, scale, a, c, true);
        if (threadIdx.x == 0) chunk_left[c] = x;
        __syncthreads();
      }
    }
  }
  for (int again = 0; again < 2; ++again) {
    // the chunk in which the sum passes its share; the last one that has anything where none does
    if (threadIdx.x == 0) {
      double all = 0.0;
      for (int c = 0; c < p.chunks; ++c) all += chunk_left[c];
      const double share = (double)p.u[s.first] * all;
      double before = 0.0;
      int at = -1, any = -1;
      double at_any = 0.0;
      for (int c = 0; c < p.chunks; ++c) {
        if (!(chunk_left[c] > 0.0)) continue;
        any = c;
        at_any = before;
        if (before + chunk_left[c] > share) {
          at = c;
          break;
        }
        before += chunk_left[c];
      }
      pick = at >= 0 ? at : any;
      level = share - (at >= 0 ? before : at_any);
      found = 0x7fffffffffffffff;
      last = -1;
    }
    __syncthreads();
    if (pick >= 0) break;
    // nothing left: the row's own distribution
    a = 0.0;
    less = false;
    __syncthreads();
    whole();
  }
  if (pick >= 0) {
    const int64_t e = (int64_t)pick * kPiece - lead(static_cast<const T*>(p.logits) + r * p.ldl) + threadIdx.x * 8;
    double x[8];
    left_of<T, Q, PROBS>(p, r, e, row.top, rt, scale, a, x);
    if (less)
      for (int j = w.cur + 1; j < s.n; ++j) {
        const int64_t k = p.rows[s.first + j].token - e;
        if (p.rows[s.first + j].above == w.cur && k >= 0 && k < 8)
#pragma unroll
          for (int i = 0; i < 8; ++i) x[i] = i == (int)k ? 0.0 : x[i];
      }
    double mine = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) mine += x[i];
    // the sum of the places before this thread's
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const double y = __shfl_up(upto, o);
      if ((threadIdx.x & 63) >= o) upto += y;
    }
    if ((threadIdx.x & 63) == 63) tail[threadIdx.x >> 6] = upto;
    __syncthreads();
    double before = upto - mine;
    for (int v = 0; v < (int)(threadIdx.x >> 6); ++v) before += tail[v];
    int64_t hit = 0x7fffffffffffffff, some = -1;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      before += x[i];
      if (x[i] > 0.0) {
        some = e + i;
        if (before > level && hit == 0x7fffffffffffffff) hit = e + i;
      }
    }
    if (hit != 0x7fffffffffffffff) atomicMin(reinterpret_cast<long long*>(&found), (long long)hit);
    if (some >= 0) atomicMax(reinterpret_cast<long long*>(&last), (long long)some);
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    p.count[b] = w.count;
    p.next[b] = found != 0x7fffffffffffffff ? found : last;
  }
}

}  // namespace

int64_t draft_chunks(int64_t V) { return (V + 7 + kPiece - 1) / kPiece; }

int64_t draft_work_bytes(int64_t N, int64_t B, int64_t V, bool probs) {
  const int64_t c = draft_chunks(V);
  return N * c * (int64_t)sizeof(DraftChunk) + N * (int64_t)sizeof(DraftRow) + (probs ? kDraftRounds * B * c * 8 : 0);
}

hipError_t launch_verify(DraftParams p, bool f32, bool probs_f32, uint8_t* work, hipStream_t st) {
  p.chunks = (int)draft_chunks(p.V);
  // in a line of tokens nothing follows a rejection but the next token
  p.rounds = p.probs == nullptr ? 0 : p.parents != nullptr ? kDraftRounds : 1;
  p.parts = reinterpret_cast<DraftChunk*>(work);
  p.rows = reinterpret_cast<DraftRow*>(p.parts + p.N * p.chunks);
  p.sums = reinterpret_cast<double*>(p.rows + p.N);
  const dim3 wide(256), parts((unsigned)(p.N * p.chunks)), rows((unsigned)((p.N + 3) / 4));
  if (p.N > 0) {
    hipLaunchKernelGGL(f32 ? draft_chunks_k<float> : draft_chunks_k<uint16_t>, parts, wide, 0, st, p);
    const auto rows_k = p.probs == nullptr ? (f32 ? draft_rows_k<float, float, false> : draft_rows_k<uint16_t, float, false>)
                        : probs_f32 ? (f32 ? draft_rows_k<float, float, true> : draft_rows_k<uint16_t, float, true>)
                                    : (f32 ? draft_rows_k<float, uint16_t, true> : draft_rows_k<uint16_t, uint16_t, true>);
    hipLaunchKernelGGL(rows_k, rows, wide, 0, st, p);
  }
  if (p.B == 0) return hipGetLastError();
  const auto sums_k = probs_f32 ? (f32 ? draft_sums_k<float, float> : draft_sums_k<uint16_t, float>)
                                : (f32 ? draft_sums_k<float, uint16_t> : draft_sums_k<uint16_t, uint16_t>);
  for (int i = 0; i < p.rounds; ++i)
    hipLaunchKernelGGL(sums_k, dim3((unsigned)(p.B * p.chunks)), wide, 0, st, p, i);
  const auto next_k = p.probs == nullptr ? (f32 ? draft_next_k<float, float, false> : draft_next_k<uint16_t, float, false>)
                      : probs_f32 ? (f32 ? draft_next_k<float, float, true> : draft_next_k<uint16_t, float, true>)
                                  : (f32 ? draft_next_k<float, uint16_t, true> : draft_next_k<uint16_t, uint16_t, true>);
  hipLaunchKernelGGL(next_k, dim3((unsigned)p.B), dim3(1024), p.chunks * 8, st, p);
  return hipGetLastError();
}

}  // namespace ojx

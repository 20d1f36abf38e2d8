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

// Row by row, any tree: each row's ancestors from its parent upwards, their u from the workspace. The whole workgroup calls;
// red: [4][32][12] floats.
template <bool DELTA>
__device__ __forceinline__ void by_rows(const LinTreeParams& p, const SeqPlace& at, int64_t slot, int h, int hk, float* red) {
  const int c = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const float* const st = p.state + (slot * p.HV + h) * (kHD * kHD) + rg * 16 * kHD + c * 4;
  float4 s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = *reinterpret_cast<const float4*>(st + i * kHD);
#pragma unroll 1
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
#pragma unroll 1
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

constexpr int kTree = 64;  // rows that a sequence may have to be taken at once

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// c += a b of 16 x 16 matrices in fp32. Lane (g, c) holds the rows 4 g .. + 3 of column c of a product; four such values are
// the B operand of the next one as they are, and the A operand of the matrix transposed, when the contraction takes the rows
// in the order r, 4 + r, 8 + r, 12 + r. So `at` is a transposed.
__device__ __forceinline__ f32x4 times(const f32x4& at, const f32x4& b, f32x4 c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(at[r], b[r], c, 0, 0, 0);
  return c;
}
// Is (row, col) in the lower left part of a pair of blocks of `size`?
__device__ __forceinline__ bool joins(int row, int col, int size) {
  return (row / size & 1) == 1 && (col / size & 1) == 0 && row / (2 * size) == col / (2 * size);
}
// The transposed inverse of I + a, a strictly lower triangular, at = a transposed: inverses of blocks of 1, 2, 4, 8 joined
// two by two, T <- T - T a T with a's part below the diagonal blocks, T kept both ways.
__device__ __forceinline__ f32x4 inverse(const f32x4& a, const f32x4& at, int g, int c) {
  f32x4 t, tt;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = 4 * g + r;
    t[r] = (i == c ? 1.f : 0.f) - (joins(i, c, 1) ? a[r] : 0.f);
    tt[r] = (i == c ? 1.f : 0.f) - (joins(c, i, 1) ? at[r] : 0.f);
  }
#pragma unroll
  for (int size = 2; size <= 8; size *= 2) {
    f32x4 m;
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = joins(c, 4 * g + r, size) ? at[r] : 0.f;
    const f32x4 w = times(m, t, f32x4{});
    const f32x4 down = size < 8 ? times(tt, w, f32x4{}) : f32x4{};
    tt -= times(w, tt, f32x4{});
    t -= down;
  }
  return tt;
}

// x and y in two bf16 pieces each: hi + lo is x to 16 bits.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  hi = cvt_pk2(x, y);
  lo = cvt_pk2(x - __uint_as_float(hi << 16), y - __uint_as_float(hi & 0xffff0000u));
}

// A sequence's rows at once, in blocks of 16 (a block's rows are tokens, its columns value dims; with two value dims, 2 c and
// 2 c + 1 of the wave's 32, for each lane): with
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  and  P_ij = e^(G_i - G_j) q_i . k_j  for the ancestors j of i (in P also i itself),
//   X = diag(beta) (V - diag(e^G) K S0),  U = (I + A)^-1 X,  O = scale (diag(e^G) Q S0 + P U),
// block row after block row. S0 enters as two bf16 pieces (what it makes is rounded to bf16 in the end), everything else in
// fp32. A product with a zero in place of a row that is no ancestor is only right for finite numbers: where a U is not finite
// or a decay is above 1, the head goes row by row instead.
template <bool DELTA>
__global__ void __launch_bounds__(256, 2) lintree_k(LinTreeParams p) {
  __shared__ float red[4 * 32 * 12];
  __shared__ double sums[4][kTree];      // every wave's own
  __shared__ uint64_t seen[4][kTree];
  __shared__ float strength[4][kTree];
  const int64_t b = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(b * p.HV), hk = h / (p.HV / p.HK);
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (b == p.B) {  // rows of no sequence
    int lo, hi;
    seq_span(p.q_ptr, p.B, p.N, lo, hi);
    for (int64_t r = threadIdx.x >> 5; r < p.N; r += 8)
      if (r < lo || r >= hi)
        *reinterpret_cast<uint2*>(p.o + (r * p.HV + h) * kHD + (threadIdx.x & 31) * 4) = make_uint2(0u, 0u);
    return;
  }
  const int64_t slot = p.slot[b];
  const bool there = slot >= 0 && slot < p.slots;
  const int dv = w * 32 + c * 2;
  float2 st[4][8];  // key dims 32 s + 8 g + j
  if (there) {
    const float* const from = p.state + (slot * p.HV + h) * (kHD * kHD) + g * 8 * kHD + dv;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) st[s][j] = *reinterpret_cast<const float2*>(from + (s * 32 + j) * kHD);
  }
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = at.n;
  if (n == 0) return;
  if (!there) {
    const uint32_t x = slot < 0 ? 0u : 0x7fc07fc0u;
    for (int i = threadIdx.x >> 5; i < n; i += 8)
      *reinterpret_cast<uint2*>(p.o + ((int64_t)(at.first + i) * p.HV + h) * kHD + (threadIdx.x & 31) * 4) = make_uint2(x, x);
    return;
  }
  if (n > kTree) {
    by_rows<DELTA>(p, at, slot, h, hk, red);
    return;
  }

  // a row a lane: its ancestors and itself, and the sum of their decays (to base two, in 64 bits: differences of long sums
  // are taken), by jumps of 1, 2, 4 .. rows up the tree
  bool odd = false;
  {
    const int64_t row = at.first + min(lane, n - 1);
    const float gate = p.g[row * p.HV + h], beta = DELTA ? bf2f(p.beta[row * p.HV + h]) : 1.f;
    int up = p.parents == nullptr ? lane - 1 : p.parents[row];
    if (up < 0 || up >= lane || lane >= n) up = -1;
    odd = !(gate <= 0.f) || !(fabsf(beta) < INFINITY);
    // e^-200 is 0 in fp32: -infinity does no worse, and differences of sums stay numbers
    double G = lane < n ? (double)fmaxf(gate, -200.f) * 0x1.71547652b82fep+0 : 0.0;
    uint64_t path = lane < n ? 1ull << lane : 0ull;
    while (__any(up >= 0)) {
      const int from = up < 0 ? lane : up;
      const double more = __shfl(G, from);
      const uint64_t rest = __shfl((unsigned long long)path, from);
      const int next = __shfl(up, from);
      if (up >= 0) {
        G += more;
        path |= rest;
        up = next;
      }
    }
    sums[w][lane] = G;
    seen[w][lane] = path;
    strength[w][lane] = beta;
  }
  // the state's pieces
  bf16x8 hi[4][2], lo[4][2];
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    uint32_t ph[2][4], pl[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      split2(st[s][2 * j].x, st[s][2 * j + 1].x, ph[0][j], pl[0][j]);
      split2(st[s][2 * j].y, st[s][2 * j + 1].y, ph[1][j], pl[1][j]);
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      hi[s][f] = __builtin_bit_cast(bf16x8, make_uint4(ph[f][0], ph[f][1], ph[f][2], ph[f][3]));
      lo[s][f] = __builtin_bit_cast(bf16x8, make_uint4(pl[f][0], pl[f][1], pl[f][2], pl[f][3]));
    }
  }
  const auto operand = [&](const uint16_t* x, int block, int s) {  // row 16 block + c, dims 32 s + 8 g .. + 7
    const int64_t row = at.first + min(block * 16 + c, n - 1);
    return *reinterpret_cast<const bf16x8*>(x + (row * p.HK + hk) * kHD + s * 32 + g * 8);
  };

  f32x4 u[4][2];
#pragma unroll
  for (int I = 0; I < 4; ++I) {
    if (I * 16 >= n) break;
    bf16x8 kf[4], qf[4];
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      kf[s] = operand(p.k, I, s);
      qf[s] = operand(p.q, I, s);
    }
    uint32_t vw[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = at.first + min(I * 16 + g * 4 + r, n - 1);
      vw[r] = *reinterpret_cast<const uint32_t*>(p.v + (row * p.HV + h) * kHD + dv);
    }
    f32x4 x[2] = {}, o[2] = {};
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if (DELTA) {
          x[f] = mfma(kf[s], hi[s][f], x[f]);
          x[f] = mfma(kf[s], lo[s][f], x[f]);
        }
        o[f] = mfma(qf[s], hi[s][f], o[f]);
        o[f] = mfma(qf[s], lo[s][f], o[f]);
      }
    // this lane's rows of the block as rows of X and O: 16 I + 4 g + r; as columns of the transposed matrices: 16 I + c
    float since[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = I * 16 + g * 4 + r;
      since[r] = __builtin_amdgcn_exp2f((float)sums[w][i]);
      const float beta = strength[w][i];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float v = f == 0 ? __uint_as_float(vw[r] << 16) : __uint_as_float(vw[r] & 0xffff0000u);
        x[f][r] = i < n ? (DELTA ? beta * (v - since[r] * x[f][r]) : v) : 0.f;
        o[f][r] *= since[r];
      }
    }
    const double Gc = sums[w][I * 16 + c];
    const uint64_t path = seen[w][I * 16 + c];
    const float beta = strength[w][I * 16 + c];
#pragma unroll
    for (int J = 0; J < I; ++J) {
      f32x4 kk = {}, qk = {};
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bf16x8 kj = operand(p.k, J, s);
        if (DELTA) kk = mfma(kj, kf[s], kk);
        qk = mfma(kj, qf[s], qk);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = J * 16 + g * 4 + r;
        const bool in = path >> j & 1;
        const float fade = in ? __builtin_amdgcn_exp2f((float)(Gc - sums[w][j])) : 0.f;
        kk[r] = in ? -beta * fade * kk[r] : 0.f;
        qk[r] = in ? fade * qk[r] : 0.f;
      }
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if (DELTA) x[f] = times(kk, u[J][f], x[f]);
        o[f] = times(qk, u[J][f], o[f]);
      }
    }
    f32x4 kk = {}, qk = {}, a, at_;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if (DELTA) kk = mfma(kf[s], kf[s], kk);
      qk = mfma(kf[s], qf[s], qk);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = I * 16 + g * 4 + r;  // row of the transposed, column c; and row of A, column c
      const bool in = path >> j & 1;
      const float fade = in ? __builtin_amdgcn_exp2f((float)(Gc - sums[w][j])) : 0.f;
      qk[r] = in ? fade * qk[r] : 0.f;
      if (DELTA) {
        at_[r] = in && g * 4 + r != c ? beta * fade * kk[r] : 0.f;
        const bool down = seen[w][j] >> (I * 16 + c) & 1;
        a[r] = down && g * 4 + r != c
                   ? strength[w][j] * __builtin_amdgcn_exp2f((float)(sums[w][j] - Gc)) * kk[r] : 0.f;
      }
    }
    if (DELTA) {
      const f32x4 tt = inverse(a, at_, g, c);
#pragma unroll
      for (int f = 0; f < 2; ++f) u[I][f] = times(tt, x[f], f32x4{});
    } else {
      u[I][0] = x[0];
      u[I][1] = x[1];
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      o[f] = times(qk, u[I][f], o[f]);
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !(fabsf(u[I][f][r]) < INFINITY);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = I * 16 + g * 4 + r;
      if (i < n)
        *reinterpret_cast<uint32_t*>(p.o + ((int64_t)(at.first + i) * p.HV + h) * kHD + dv) =
            cvt_pk2(p.scale * o[0][r], p.scale * o[1][r]);
    }
  }
  if (__syncthreads_or(odd)) by_rows<DELTA>(p, at, slot, h, hk, red);
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
  hipLaunchKernelGGL(p.beta != nullptr ? lintree_k<true> : lintree_k<false>,
                     dim3((unsigned)((p.B + 1LL) * p.HV)), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_linattn_keep(const LinTreeParams& p, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_keep_k<true> : linattn_keep_k<false>, dim3((unsigned)((int64_t)p.B * p.HV)),
                     dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

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

// Row by row, any tree: each row's ancestors from its parent upwards, their u from LDS (near, where there is room for all the
// rows') or the workspace. The whole workgroup calls; red: [4][32][12] floats.
template <bool DELTA, bool NEAR>
__device__ __forceinline__ void by_rows(const LinTreeParams& p, const SeqPlace& at, int64_t slot, int h, int hk, float* red,
                                        float4 (*near)[32]) {
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
      const float4 u = NEAR ? near[j][c] : *reinterpret_cast<const float4*>(p.u + (a * p.HV + h) * kHD + c * 4);
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
      (NEAR ? near[i][c] : *reinterpret_cast<float4*>(p.u + (row * p.HV + h) * kHD + c * 4)) =
          make_float4(u[0], u[1], u[2], u[3]);
      store4(p.o + (row * p.HV + h) * kHD + c * 4, p.scale * (f[4] + f[8] * u[0]), p.scale * (f[5] + f[8] * u[1]),
             p.scale * (f[6] + f[8] * u[2]), p.scale * (f[7] + f[8] * u[3]));
    }
    __syncthreads();
  }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
constexpr int kTree = 64;  // rows that are taken at once
constexpr int kParts = 4;  // as many times as a sequence may have of them

// 16-byte pieces of 16 rows that are read at once spread over the banks.
__device__ __forceinline__ constexpr int swizzle(int r) { return (r & 7) << 1 | (r >> 3 & 1); }

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
// The transposed inverse of I + a, a strictly lower triangular, at = a transposed: inverses of blocks of 1, 2, 4, 8 joined
// two by two, T <- T - T a T with the part of a that joins blocks of this size, T kept both ways. That part is where row and
// column differ in the size's bit and in none above it.
__device__ __forceinline__ f32x4 inverse(const f32x4& a, const f32x4& at, int g, int c) {
  f32x4 t, tt;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int differ = (4 * g + r) ^ c;
    t[r] = differ == 0 ? 1.f : (differ & 15) == 1 ? -a[r] : 0.f;
    tt[r] = differ == 0 ? 1.f : (differ & 15) == 1 ? -at[r] : 0.f;
  }
#pragma unroll
  for (int size = 2; size <= 8; size *= 2) {
    f32x4 m;
#pragma unroll
    for (int r = 0; r < 4; ++r) m[r] = (((4 * g + r) ^ c) & (16 - size)) == size ? at[r] : 0.f;
    const f32x4 w = times(m, t, f32x4{});
    const f32x4 down = size < 8 ? times(tt, w, f32x4{}) : f32x4{};
    tt -= times(w, tt, f32x4{});
    t -= down;
  }
  return tt;
}

// The bf16 pieces next to element e of x and of y, which become what those leave: three pieces are all 24 bits.
__device__ __forceinline__ uint32_t take_piece(f32x2& x, f32x2& y, int e) {
  const uint32_t piece = cvt_pk2(x[e], y[e]);
  x[e] -= __uint_as_float(piece << 16);
  y[e] -= __uint_as_float(piece & 0xffff0000u);
  return piece;
}

// LDS reads and writes of all waves are done; global loads stay in flight.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// What a head's workgroup has in LDS.
struct TreeShared {
  f32x4 mats[19][64];
  bf16x8 rows[2][kTree][16];  // K and Q, piece x of a row r at x ^ swizzle(r)
  double sums[kTree];         // every wave writes the same there
  uint64_t seen[kTree];
  float strength[kTree];
};
static_assert(sizeof(TreeShared::mats) >= 4 * 32 * 12 * 4 && sizeof(TreeShared::rows) == kTree * 32 * sizeof(float4),
              "by_rows' sums and u");

// What parts of a long sequence leave to the later ones, for each row and head: the decays' sum, the ancestors 64 to a word.
struct TreeLeft {
  double sum;
  uint64_t seen[kParts];
};

// Up to 64 rows of a sequence at once, those from row s0 on, in blocks of 16 (a block's rows are tokens, its columns value
// dims; with two value dims, 2 c and 2 c + 1 of the wave's 32, for each lane): with
//   A_ij = beta_i e^(G_i - G_j) k_i . k_j  and  P_ij = e^(G_i - G_j) q_i . k_j  for the ancestors j of i (in P also i itself),
//   X = diag(beta) (V - diag(e^G) K S0),  U = (I + A)^-1 X,  O = scale (diag(e^G) Q S0 + P U),
// block row after block row. S0 enters as three bf16 pieces, all its 24 bits (two, 17 bits: 48 us in place of 50 for the 64
// sequences below, but outputs in which key dims cancel are 2^-17 of those off), everything else in fp32. A product with a zero
// in place of a row that is no ancestor is only right for finite numbers: where a U or an O is not finite (a state's pieces have
// no infinity) or a decay is above 1 (true), the head goes row by row instead.
// Loads come back in the order in which they were made, so the rows' go first: while the state is on its way the four waves
// make the blocks of A, P and the inverses of A's diagonal ones, each once, and hand them to each other in LDS as the operands
// that they are. LONG: the rows before s0 have left their U and TreeLeft in the workspace (a thread reads back the U that it
// wrote), and these rows leave theirs.
template <bool DELTA, bool LONG>
__device__ __forceinline__ bool tree_part(const LinTreeParams& p, TreeShared& lds, int64_t first, int s0, int n, int64_t slot,
                                          int h, int hk) {
  auto& mats = lds.mats;
  auto& rows = lds.rows;
  auto& sums = lds.sums;
  auto& seen = lds.seen;
  auto& strength = lds.strength;
  int lane = threadIdx.x & 63;
  if (LONG) asm volatile("" : "+v"(lane));  // a part computes its addresses anew: there are no registers to keep them over a loop
  const int g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t at = first + s0;
  const int dv = w * 32 + c * 2, blocks = (n + 15) >> 4;
  float gate, beta;
  int up;
  bf16x8 kf[4], qf[4];  // a piece a thread of each block's rows of K and Q
  uint32_t vw[4][4];    // this lane's values of rows 16 I + 4 g + r
  {
    const int64_t row = at + min(lane, n - 1);
    gate = p.g[row * p.HV + h];
    beta = DELTA ? bf2f(p.beta[row * p.HV + h]) : 1.f;
    up = p.parents == nullptr ? s0 + lane - 1 : p.parents[row];
  }
#pragma unroll
  for (int I = 0; I < 4; ++I)
    if (I < blocks) {
      const int64_t row = at + min(I * 16 + ((int)threadIdx.x >> 4), n - 1);
      const int64_t from = (row * p.HK + hk) * kHD + c * 8;
      kf[I] = *reinterpret_cast<const bf16x8*>(p.k + from);
      qf[I] = *reinterpret_cast<const bf16x8*>(p.q + from);
    }
  // the last block's values come behind the state's first parts: there are no registers to have both (with them spilled, 62 us
  // for 64 sequences of 12 rows in place of 50)
  constexpr int kEarly = DELTA && !LONG ? 3 : 4;
  const auto load_v = [&](int I) {
    if (I < blocks)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int64_t row = at + min(I * 16 + g * 4 + r, n - 1);
        vw[I][r] = *reinterpret_cast<const uint32_t*>(p.v + (row * p.HV + h) * kHD + dv);
      }
  };
#pragma unroll
  for (int I = 0; I < kEarly; ++I) load_v(I);
  asm volatile("" ::: "memory");  // the state's loads stay behind
  f32x2 st[4][8];                 // key dims 32 s + 8 g + j
  {
    const float* const from = p.state + (slot * p.HV + h) * (kHD * kHD) + g * 8 * kHD + dv;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) st[s][j] = *reinterpret_cast<const f32x2*>(from + (s * 32 + j) * kHD);
  }
  asm volatile("" ::: "memory");

  // a row a lane: its ancestors and itself, and the sum of their decays (to base two, in 64 bits: differences of long sums
  // are taken), by jumps of 1, 2, 4 .. rows up the tree; `above`: the row before s0 that it hangs on
  bool odd = !(gate <= 0.f) || !(fabsf(beta) < INFINITY);
  uint64_t before[kParts - 1] = {};
  TreeLeft* const left = reinterpret_cast<TreeLeft*>(p.u + p.N * p.HV * kHD);
  {
    if (up < 0 || up >= s0 + lane || lane >= n) up = -1;
    int above = up < s0 ? up : -1;
    up = up < s0 ? -1 : up - s0;
    // e^-200 is 0 in fp32: -infinity does no worse, and differences of sums stay numbers
    double G = lane < n ? (double)fmaxf(gate, -200.f) * 0x1.71547652b82fep+0 : 0.0;
    uint64_t path = lane < n ? 1ull << lane : 0ull;
    while (__any(up >= 0)) {
      const int from = up < 0 ? lane : up;
      const double more = __shfl(G, from);
      const uint64_t rest = __shfl((unsigned long long)path, from);
      const int next = __shfl(up, from), last = LONG ? __shfl(above, from) : -1;
      if (up >= 0) {
        G += more;
        path |= rest;
        up = next;
        above = last;
      }
    }
    if (LONG) {
      if (above >= 0) {
        const TreeLeft& l = left[(first + above) * p.HV + h];
        G += l.sum;
#pragma unroll
        for (int m = 0; m < kParts - 1; ++m) before[m] = l.seen[m];
      }
      if (w == 0 && lane < n) {
        TreeLeft& l = left[(at + lane) * p.HV + h];
        l.sum = G;
#pragma unroll
        for (int m = 0; m < kParts; ++m)
          l.seen[m] = m * kTree == s0 ? path : m < kParts - 1 && m * kTree < s0 ? before[m] : 0ull;
      }
    }
    sums[lane] = G;
    seen[lane] = path;
    strength[lane] = beta;
  }
#pragma unroll
  for (int I = 0; I < 4; ++I)
    if (I < blocks) {
      const int r = w * 4 + g, x = c ^ swizzle(r);
      rows[0][I * 16 + r][x] = kf[I];
      rows[1][I * 16 + r][x] = qf[I];
    }
  lds_barrier();
  const auto operand = [&](int which, int block, int s) {  // row 16 block + c, dims 32 s + 8 g .. + 7
    return rows[which][block * 16 + c][(s * 4 + g) ^ swizzle(c)];
  };
  const auto fade = [&](double from, double to) { return __builtin_amdgcn_exp2f((float)(from - to)); };

  // mats: the transposed inverses of the diagonal blocks 0 .. 2, the blocks' P transposed 3 .. 6; below the diagonal -A
  // transposed 7 .. 12 and P transposed 13 .. 18. Wave w has diagonal block w and the pairs w and w + 4 of the six others.
  // The fourth inverse stays with its wave until the rows' place is free: with 1 KB less, three workgroups fit a CU.
  f32x4 fourth = {};
#pragma unroll
  for (int turn = 0; turn < 3; ++turn) {
    // pairs (1, 0), (2, 0), (2, 1), (3, 0), (3, 1), (3, 2)
    const int pair = turn == 2 ? w + 4 : w, I = turn == 0 ? w : pair == 0 ? 1 : pair <= 2 ? 2 : 3;
    const int J = turn == 0 ? w : pair == 0 ? 0 : pair <= 2 ? pair - 1 : pair - 3;
    if (I >= blocks || (turn > 0 && pair > 5)) continue;  // the same for the wave
    const int i = I * 16 + c;
    const uint64_t path = seen[i];
    const double Gi = sums[i];
    f32x4 kk = {}, qk = {};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const bf16x8 kj = operand(0, J, s);
      if (DELTA) kk = mfma(kj, turn == 0 ? kj : operand(0, I, s), kk);
      qk = mfma(kj, operand(1, I, s), qk);
    }
    f32x4 a, down;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = J * 16 + g * 4 + r;
      const bool in = path >> j & 1;
      const float e = in ? fade(Gi, sums[j]) : 0.f;
      qk[r] = in ? e * qk[r] : 0.f;
      if (DELTA) {
        a[r] = in && i != j ? strength[i] * e * kk[r] : 0.f;
        // the block itself, from the other side (its products are symmetric)
        if (turn == 0) down[r] = i != j && (seen[j] >> i & 1) ? strength[j] * fade(sums[j], Gi) * kk[r] : 0.f;
      }
    }
    mats[turn == 0 ? 3 + w : 13 + pair][lane] = qk;
    if (DELTA) {
      const f32x4 x = turn == 0 ? inverse(down, a, g, c) : -a;
      if (turn == 0 && w == 3)
        fourth = x;
      else
        mats[turn == 0 ? w : 7 + pair][lane] = x;
    }
  }
  lds_barrier();

  // K S0 and Q S0
  f32x4 u[4][2], o[4][2];
#pragma unroll
  for (int I = 0; I < 4; ++I)
#pragma unroll
    for (int f = 0; f < 2; ++f) u[I][f] = o[I][f] = f32x4{};
#pragma unroll
  for (int s = 0; s < 4; ++s) {
    if (s == 2 && kEarly < 4) {
      asm volatile("" ::: "memory");
      load_v(3);
      asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      bf16x8 piece[3];
#pragma unroll
      for (int x = 0; x < 3; ++x) {
        uint32_t at[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) at[j] = take_piece(st[s][2 * j], st[s][2 * j + 1], f);
        piece[x] = __builtin_bit_cast(bf16x8, make_uint4(at[0], at[1], at[2], at[3]));
      }
#pragma unroll
      for (int I = 0; I < 4; ++I) {
        if (I >= blocks) break;
        const bf16x8 ki = operand(0, I, s), qi = operand(1, I, s);
#pragma unroll
        for (int x = 0; x < 3; ++x) {
          if (DELTA) u[I][f] = mfma(ki, piece[x], u[I][f]);
          o[I][f] = mfma(qi, piece[x], o[I][f]);
        }
      }
    }
  }
  // X in place of K S0, Q S0 decayed
#pragma unroll
  for (int I = 0; I < 4; ++I) {
    if (I >= blocks) break;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = I * 16 + g * 4 + r;
      const float since = __builtin_amdgcn_exp2f((float)sums[i]), by = strength[i];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        const float v = __uint_as_float(f == 0 ? vw[I][r] << 16 : vw[I][r] & 0xffff0000u);
        u[I][f][r] = i < n ? (DELTA ? by * (v - since * u[I][f][r]) : v) : 0.f;
        o[I][f][r] *= since;
      }
    }
  }
  f32x4* const late = reinterpret_cast<f32x4*>(rows);

#pragma unroll
  for (int I = 0; I < 4; ++I) {
    if (I >= blocks) break;
    // the rows before s0, 16 at a time
    if (LONG)
#pragma unroll 1
      for (int j0 = 0; j0 < s0; j0 += 16) {
        asm volatile("" ::: "memory");  // LDS is read where it is needed: there are no registers to hold its rows
        const uint64_t word = j0 < kTree ? before[0] : j0 < 2 * kTree ? before[1] : before[2];
        const uint64_t path = __shfl((unsigned long long)word, I * 16 + c) >> (j0 & (kTree - 1));
        f32x4 kk = {}, qk = {}, uj[2];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const bf16x8 kj =
              *reinterpret_cast<const bf16x8*>(p.k + ((first + j0 + c) * p.HK + hk) * kHD + s * 32 + g * 8);
          if (DELTA) kk = mfma(kj, operand(0, I, s), kk);
          qk = mfma(kj, operand(1, I, s), qk);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int64_t row = (first + j0 + g * 4 + r) * p.HV + h;
          const f32x2 x = *reinterpret_cast<const f32x2*>(p.u + row * kHD + dv);
          uj[0][r] = x.x;
          uj[1][r] = x.y;
          const bool in = path >> (g * 4 + r) & 1;
          const float e = in ? fade(sums[I * 16 + c], left[row].sum) : 0.f;
          kk[r] = in ? -strength[I * 16 + c] * e * kk[r] : 0.f;
          qk[r] = in ? e * qk[r] : 0.f;
        }
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          if (DELTA) u[I][f] = times(kk, uj[f], u[I][f]);
          o[I][f] = times(qk, uj[f], o[I][f]);
        }
      }
#pragma unroll
    for (int J = 0; J < I; ++J) {
      const int pair = I * (I - 1) / 2 + J;
      const f32x4 a = mats[7 + pair][lane], pj = mats[13 + pair][lane];
#pragma unroll
      for (int f = 0; f < 2; ++f) {
        if (DELTA) u[I][f] = times(a, u[J][f], u[I][f]);
        o[I][f] = times(pj, u[J][f], o[I][f]);
      }
    }
    if (DELTA && I == 3) {
      lds_barrier();
      if (w == 3) late[lane] = fourth;
      lds_barrier();
    }
    const f32x4 pi = mats[3 + I][lane];
    const f32x4 t = !DELTA ? f32x4{} : I < 3 ? mats[I][lane] : late[lane];
#pragma unroll
    for (int f = 0; f < 2; ++f) {
      if (DELTA) u[I][f] = times(t, u[I][f], f32x4{});
      o[I][f] = times(pi, u[I][f], o[I][f]);
#pragma unroll
      for (int r = 0; r < 4; ++r) odd |= !(fabsf(u[I][f][r]) < INFINITY) || !(fabsf(o[I][f][r]) < INFINITY);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = I * 16 + g * 4 + r;
      const int64_t row = (at + i) * p.HV + h;
      if (i < n) {
        *reinterpret_cast<uint32_t*>(p.o + row * kHD + dv) = cvt_pk2(p.scale * o[I][0][r], p.scale * o[I][1][r]);
        if (LONG) *reinterpret_cast<f32x2*>(p.u + row * kHD + dv) = f32x2{u[I][0][r], u[I][1][r]};
      }
    }
  }
  return odd;
}

// A workgroup per sequence and value head. What bounds it: the states, read once. 64 sequences of 12 rows and 48 heads, 216 MB,
// take 48 us: 4.5 TB/s, where a copy reaches 5.1 and a stream that is only read 5.8. (With states in two pieces 45 us; then two
// workgroups a CU: 50; the rows' loads behind the state's, three workgroups: 57; row by row: 134.) Few sequences of 64 rows are
// bound by their chain, loads, the inverses, K S0, four blocks in turn: 8 of them 25 us (row by row 356), one 15.6; one of 8 rows
// 8.1 us.
template <bool DELTA>
__global__ void __launch_bounds__(256, 3) lintree_k(LinTreeParams p) {
  __shared__ __attribute__((aligned(16))) TreeShared lds;
  float* const red = reinterpret_cast<float*>(lds.mats);  // row by row
  const int64_t b = blockIdx.x / p.HV;
  const int h = blockIdx.x - (int)(b * p.HV), hk = h / (p.HV / p.HK);
  if (b == p.B) {  // rows of no sequence
    int lo, hi;
    seq_span(p.q_ptr, p.B, p.N, lo, hi);
    for (int64_t r = threadIdx.x >> 5; r < p.N; r += 8)
      if (r < lo || r >= hi)
        *reinterpret_cast<uint2*>(p.o + (r * p.HV + h) * kHD + (threadIdx.x & 31) * 4) = make_uint2(0u, 0u);
    return;
  }
  const int64_t slot = p.slot[b];
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = at.n;
  if (n == 0) return;
  if (slot < 0 || slot >= p.slots) {
    const uint32_t x = slot < 0 ? 0u : 0x7fc07fc0u;
    for (int i = threadIdx.x >> 5; i < n; i += 8)
      *reinterpret_cast<uint2*>(p.o + ((int64_t)(at.first + i) * p.HV + h) * kHD + (threadIdx.x & 31) * 4) = make_uint2(x, x);
    return;
  }
  if (n > kTree) return;  // lintree_long_k's
  if (__syncthreads_or(tree_part<DELTA, false>(p, lds, at.first, 0, n, slot, h, hk))) {
    __syncthreads();  // outputs that other waves have stored, before they are stored again
    by_rows<DELTA, true>(p, at, slot, h, hk, red, reinterpret_cast<float4(*)[32]>(lds.rows));
  }
}

// The sequences with more rows than that, part after part; a workgroup for each that there can be, and head. (A kernel of its
// own: in one with the other form, the registers that this one wants cost that one 6 to 110% more time, as it was put; its
// launch costs 2.3 to 4.6 us where no sequence is so long.) One sequence of 65 rows takes 30 us, of 128 rows 55; row by row 313
// and 1098.
template <bool DELTA>
__global__ void __launch_bounds__(256, 2) lintree_long_k(LinTreeParams p) {
  __shared__ __attribute__((aligned(16))) TreeShared lds;
  const int which = blockIdx.x / (uint32_t)p.HV, h = blockIdx.x - which * p.HV, hk = h / (p.HV / p.HK);
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int n) { return (int)(n > kTree); }, [=](int, int upto) { return upto > which; },
                at))
    return;
  const int64_t slot = p.slot[at.seq];
  if (slot < 0 || slot >= p.slots) return;  // lintree_k has seen to these
  bool odd = at.n > kTree * kParts;
  if (!odd)
#pragma unroll 1
    for (int s0 = 0; s0 < at.n; s0 += kTree) {
      odd |= tree_part<DELTA, true>(p, lds, at.first, s0, min(kTree, at.n - s0), slot, h, hk);
      __syncthreads();  // what it leaves is there for the next one, and LDS is free
    }
  if (__syncthreads_or(odd)) by_rows<DELTA, false>(p, at, slot, h, hk, reinterpret_cast<float*>(lds.mats), nullptr);
}

// x summed over the four groups of 16 lanes, in all of them.
__device__ __forceinline__ float add_rows(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The kept tokens of sequence b, rows path[0 .. count - 1] of its own, through its state one after the other. A wave has 32
// value dims of a head's state, lane (g, c) the key dims 32 g .. + 31 of value dims 2 c and 2 c + 1 of those: no wave waits
// for another. Rows of 16 tokens at a time go through LDS, read while the state is on its way.
// What bounds it: the states, read and written once: 64 sequences of 48 heads over up to 6 tokens, 400 MB, take 85 us, 4.7 TB/s
// (90 us with a head a workgroup, its four waves adding their sums in LDS); for one sequence the chain of a state's load, five
// tokens and its store, 6.4 us (9.4).
template <bool DELTA>
__global__ void __launch_bounds__(128) linattn_keep_k(LinTreeParams p) {
  constexpr int kTokens = 16;
  __shared__ __attribute__((aligned(16))) uint16_t all_keys[2][kTokens][kHD];
  __shared__ __attribute__((aligned(16))) uint16_t all_values[2][kTokens][32];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  auto& keys = all_keys[w];
  auto& values = all_values[w];
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const uint32_t wave = blockIdx.x * (blockDim.x >> 6) + w;
  const int64_t b = (wave >> 2) / p.HV;
  const int h = (int)((wave >> 2) - b * p.HV), hk = h / (p.HV / p.HK), dv = (wave & 3) * 32;
  const int64_t slot = p.slot[b];
  const int count = p.count[b];
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = min(at.n, count);
  // A slot belongs to the first sequence that names it: two workgroups that update one state would race.
  bool twice = slot < 0 || slot >= p.slots || n <= 0;
  for (int64_t i = lane; i < b; i += 64) twice |= p.slot[i] == slot;
  if (__any(twice)) return;
  int mine = lane < min(n, kTokens) ? p.path[at.first + lane] : -1;
  float* const st = p.state + (slot * p.HV + h) * (kHD * kHD) + g * 32 * kHD + dv + c * 2;
  f32x2 s[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = *reinterpret_cast<const f32x2*>(st + i * kHD);
  for (int i0 = 0; i0 < n; i0 += kTokens) {
    if (i0 > 0) mine = lane < min(n - i0, kTokens) ? p.path[at.first + i0 + lane] : -1;
    const bool valid = mine >= 0 && mine < at.n;
    const int64_t row = at.first + (valid ? mine : 0);
    unsigned long long todo = __ballot(valid);
    const float gate = p.g[row * p.HV + h], beta = DELTA ? bf2f(p.beta[row * p.HV + h]) : 1.f;
    uint4 piece[4], value;
#pragma unroll
    for (int j = 0; j < 4; ++j)  // tokens 4 j + g, 16 bytes a lane
      piece[j] = *reinterpret_cast<const uint4*>(p.k + ((int64_t)__shfl((int)row, j * 4 + g) * p.HK + hk) * kHD + c * 8);
    value = *reinterpret_cast<const uint4*>(p.v + ((int64_t)__shfl((int)row, lane >> 2) * p.HV + h) * kHD + dv +
                                            (lane & 3) * 8);
#pragma unroll
    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint4*>(&keys[j * 4 + g][c * 8]) = piece[j];
    *reinterpret_cast<uint4*>(&values[lane >> 2][(lane & 3) * 8]) = value;
    const float decay = expf(gate);
    for (; todo != 0; todo &= todo - 1) {
      const int i = __builtin_ctzll(todo);
      const float a = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(decay), i));
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(&values[i][c * 2]);
      f32x2 u = {__uint_as_float(vw << 16), __uint_as_float(vw & 0xffff0000u)};
      float k[32];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint4 x = *reinterpret_cast<const uint4*>(&keys[i][g * 32 + j * 8]);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          k[j * 8 + 2 * m] = __uint_as_float(w[m] << 16);
          k[j * 8 + 2 * m + 1] = __uint_as_float(w[m] & 0xffff0000u);
        }
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        s[j].x *= a;
        s[j].y *= a;
      }
      if (DELTA) {
        float x[2][2] = {};
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          x[j & 1][0] += s[j].x * k[j];
          x[j & 1][1] += s[j].y * k[j];
        }
        const float by = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(beta), i));
        u.x = by * (u.x - add_rows(x[0][0] + x[1][0]));
        u.y = by * (u.y - add_rows(x[0][1] + x[1][1]));
      }
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        s[j].x += k[j] * u.x;
        s[j].y += k[j] * u.y;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 32; ++i) *reinterpret_cast<f32x2*>(st + i * kHD) = s[i];
}

}  // namespace

// Sequences longer than what a workgroup takes at once leave their u in memory.
int64_t lintree_work_bytes(int64_t N, int HV) { return N > kTree ? N * HV * (kHD * 4 + (int64_t)sizeof(TreeLeft)) : 0; }

hipError_t launch_linattn_tree(const LinTreeParams& p, hipStream_t st) {
  hipLaunchKernelGGL(p.beta != nullptr ? lintree_k<true> : lintree_k<false>,
                     dim3((unsigned)((p.B + 1LL) * p.HV)), dim3(256), 0, st, p);
  const int64_t longs = std::min<int64_t>(p.B, p.N / (kTree + 1));  // at most
  if (longs > 0)
    hipLaunchKernelGGL(p.beta != nullptr ? lintree_long_k<true> : lintree_long_k<false>, dim3((unsigned)(longs * p.HV)),
                       dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_linattn_keep(const LinTreeParams& p, hipStream_t st) {
  // Few heads: every wave a workgroup of its own, so that they take all CUs (4 sequences of 48 heads 8.6 us, 9.1 with two waves
  // a workgroup, 9.4 with four); many: two (16 sequences 18.3 us, 21.4 with one, 17.7 with four).
  const int threads = (int64_t)p.B * p.HV <= 384 ? 64 : 128;
  hipLaunchKernelGGL(p.beta != nullptr ? linattn_keep_k<true> : linattn_keep_k<false>, dim3((unsigned)((int64_t)p.B * p.HV * 256 / threads)),
                     dim3(threads), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

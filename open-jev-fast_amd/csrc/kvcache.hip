// Paged key / value cache: tokens written to their slots, in bf16 or quantised to e4m3, and read back as bf16.
//
// A cache is [pages, HKV, page, D]; slot = page index * page + place in the page. A row is one token's D values of one
// head. The e4m3 form keeps one fp32 scale a row, the smallest power of two 2^e (e >= -126) that brings the row's
// largest finite magnitude within e4m3's 448, so that the division before the rounding is exact and the only error is
// the rounding to four significant bits; with a scale that is no power of two the quotient would be rounded twice, and
// e4m3 is a floating format: a larger share of its range used does not make its values more exact.
//
// Both directions move each row once. 16384 tokens of four heads of 256, 101 MB: read back in 17.4 us, 5.8 TB/s, as fast
// as a large copy. Written in 22.5 us, 4.5 TB/s: the scale needs the whole row before the first value can be stored, so a
// wave's chain is a load, the row's maximum over its lanes and a store (24.0 us with the maximum through LDS, 27.3 with the
// values loaded behind the slots and 64-bit divisions for both). In bf16, 134 MB, 26.0 us written and 21.8 read (5.2 and 6.2
// TB/s). A few rows cost the launch: 2.8 us for 64 tokens.
#include "ojx_internal.h"

#include <algorithm>

namespace ojx {

namespace {

// Rows are D / 8 lanes of eight values: 16 bytes of bf16, 8 bytes of e4m3.
template <int D>
constexpr int kRowLanes = D / 8;

__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // e in [-126, 127]

// Where row `slot` of head h lies in the cache, in rows; slots outside the cache give -1.
__device__ __forceinline__ int64_t cache_row(int64_t slot, int h, int HKV, int64_t rows, int page) {
  if (slot < 0 || slot >= rows) return -1;
  const int64_t p = rows >> 32 == 0 ? (int64_t)((uint32_t)slot / (uint32_t)page) : slot / page;
  return (p * HKV + h) * page + (slot - p * page);
}

// The largest value of a row's lanes, in each: rotations within 16 lanes, then a swap of the two halves of 32.
template <int L>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
#define OJX_ROR(n) x = max(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x120 + (n), 0xf, 0xf, true))
  OJX_ROR(8);
  OJX_ROR(4);
  OJX_ROR(2);
  OJX_ROR(1);
#undef OJX_ROR
  if (L == 16) return x;
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  return max(a[0], a[1]);
}

template <int D, bool FP8>
__global__ void __launch_bounds__(256) kv_write_k(const uint16_t* __restrict__ k, const uint16_t* __restrict__ v,
                                                  const int64_t* __restrict__ slots, int64_t N, int HKV, void* kc,
                                                  void* vc, float* ks, float* vs, int64_t rows, int page) {
  constexpr int L = kRowLanes<D>, R = 256 / L;
  const int l = threadIdx.x % L;
  const bool isv = blockIdx.y >= HKV;
  const int h = isv ? blockIdx.y - HKV : blockIdx.y;
  const uint16_t* const from = (isv ? v : k) + (int64_t)h * N * D + l * 8;
  for (int64_t n = (int64_t)blockIdx.x * R + threadIdx.x / L; n < N; n += (int64_t)gridDim.x * R) {
    const uint4 x = *reinterpret_cast<const uint4*>(from + n * D);  // not behind the slot's load
    const int64_t row = cache_row(slots[n], h, HKV, rows, page);
    if (row < 0) continue;  // the whole row's lanes
    if (!FP8) {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(isv ? vc : kc) + row * D + l * 8) = x;
      continue;
    }
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    uint32_t top = 0;  // largest finite magnitude, as bf16 bits
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = w[i] & 0x7fffu, b = (w[i] >> 16) & 0x7fffu;
      top = max(top, max(a < 0x7f80u ? a : 0u, b < 0x7f80u ? b : 0u));
    }
    top = row_max<L>(top);
    // top = 2^(E - 127) (1 + m / 128) and 448 = 2^8 * 1.75: one exponent more where 1 + m / 128 > 1.75
    int e = (int)(top >> 7) - 127 - 8 + ((top & 0x7f) > 96 ? 1 : 0);
    e = top == 0 ? 0 : max(e, -126);
    const float inv = pow2f(-e);
    float f[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[2 * i] = bf2f(w[i] & 0xffffu) * inv;
      f[2 * i + 1] = bf2f(w[i] >> 16) * inv;
      // e4m3 has no infinity
      if ((w[i] & 0x7fffu) >= 0x7f80u) f[2 * i] = __uint_as_float(0x7fc00000u);
      if (((w[i] >> 16) & 0x7fffu) >= 0x7f80u) f[2 * i + 1] = __uint_as_float(0x7fc00000u);
    }
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
    *reinterpret_cast<int2*>(static_cast<uint8_t*>(isv ? vc : kc) + row * D + l * 8) = make_int2(lo, hi);
    if (l == 0) (isv ? vs : ks)[row] = pow2f(e);
  }
}

template <int D, bool FP8>
__global__ void __launch_bounds__(256) kv_read_k(const void* __restrict__ kc, const void* __restrict__ vc,
                                                 const float* __restrict__ ks, const float* __restrict__ vs,
                                                 const int64_t* __restrict__ slots, int64_t N, int HKV,
                                                 uint16_t* __restrict__ k, uint16_t* __restrict__ v, int64_t rows,
                                                 int page) {
  constexpr int L = kRowLanes<D>, R = 256 / L;
  const int l = threadIdx.x % L;
  const bool isv = blockIdx.y >= HKV;
  const int h = isv ? blockIdx.y - HKV : blockIdx.y;
  uint16_t* const to = (isv ? v : k) + (int64_t)h * N * D + l * 8;
  for (int64_t n = (int64_t)blockIdx.x * R + threadIdx.x / L; n < N; n += (int64_t)gridDim.x * R) {
    const int64_t row = cache_row(slots[n], h, HKV, rows, page);
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (row >= 0) {
      if (!FP8) {
        o = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(isv ? vc : kc) + row * D + l * 8);
      } else {
        const int2 x = *reinterpret_cast<const int2*>(static_cast<const uint8_t*>(isv ? vc : kc) + row * D + l * 8);
        const float s = (isv ? vs : ks)[row];
        o = make_uint4(pack2(__builtin_amdgcn_cvt_f32_fp8(x.x, 0) * s, __builtin_amdgcn_cvt_f32_fp8(x.x, 1) * s),
                       pack2(__builtin_amdgcn_cvt_f32_fp8(x.x, 2) * s, __builtin_amdgcn_cvt_f32_fp8(x.x, 3) * s),
                       pack2(__builtin_amdgcn_cvt_f32_fp8(x.y, 0) * s, __builtin_amdgcn_cvt_f32_fp8(x.y, 1) * s),
                       pack2(__builtin_amdgcn_cvt_f32_fp8(x.y, 2) * s, __builtin_amdgcn_cvt_f32_fp8(x.y, 3) * s));
      }
    }
    *reinterpret_cast<uint4*>(to + n * D) = o;
  }
}

// Token blocks, and a kv head's keys or values; at most about 16384 workgroups.
dim3 kv_grid(int64_t N, int HKV, int D) {
  const int64_t per = 256 / (D / 8);
  return dim3((unsigned)std::min<int64_t>((N + per - 1) / per, std::max(1, 8192 / HKV)), (unsigned)(2 * HKV));
}

}  // namespace

hipError_t launch_kv_write(const uint16_t* k, const uint16_t* v, const int64_t* slots, int64_t N, int HKV, int D,
                           bool fp8, void* kc, void* vc, float* ks, float* vs, int64_t rows, int page,
                           hipStream_t st) {
  const auto kernel = D == 256 ? (fp8 ? kv_write_k<256, true> : kv_write_k<256, false>)
                               : (fp8 ? kv_write_k<128, true> : kv_write_k<128, false>);
  hipLaunchKernelGGL(kernel, kv_grid(N, HKV, D), dim3(256), 0, st, k, v, slots, N, HKV, kc, vc, ks, vs, rows,
                     page);
  return hipGetLastError();
}

hipError_t launch_kv_read(const void* kc, const void* vc, const float* ks, const float* vs, const int64_t* slots,
                          int64_t N, int HKV, int D, bool fp8, uint16_t* k, uint16_t* v, int64_t rows, int page,
                          hipStream_t st) {
  const auto kernel = D == 256 ? (fp8 ? kv_read_k<256, true> : kv_read_k<256, false>)
                               : (fp8 ? kv_read_k<128, true> : kv_read_k<128, false>);
  hipLaunchKernelGGL(kernel, kv_grid(N, HKV, D), dim3(256), 0, st, kc, vc, ks, vs, slots, N, HKV, k, v, rows,
                     page);
  return hipGetLastError();
}

}  // namespace ojx

// What becomes of a paged cache around drafted tokens: accepted rows moved together, pages taken, given back, shared and
// copied. A table row names a sequence's pages, refs counts the table entries that name each page; a page with none is free.
//
// All of it is whole numbers and copies. Tables and counts are small: what bounds them is the chain of launches and loads.
#include "ojx_internal.h"

#include <algorithm>

namespace ojx {

namespace {

// ------------------------------------------------------------------------------------------------------- accepted rows
// Sequence b keeps the drafted rows path[0 .. count - 1]: the row at position ctx + path[i] goes to ctx + i. With path[i] >=
// i (any rising path; other entries are left out) a place that is written is none that a later entry reads, so that entries
// may be taken in order, kKeep at a time: read by all, a barrier, written by all.
//
// A workgroup has one sequence's rows of one head of one layer, keys or values; a row is L lanes of 16 bytes, and the rows
// of a batch go to the 256 / L row groups in turn.
template <int ROW>  // bytes of a row
__global__ void __launch_bounds__(256) kv_keep_k(KeepParams p) {
  constexpr int L = ROW / 16, G = 256 / L, E = 4, kKeep = G * E;
  const int64_t b = blockIdx.x;
  const int hz = blockIdx.y, layer = hz / (2 * p.HKV), x = hz - layer * 2 * p.HKV;
  const bool isv = x >= p.HKV;
  const int h = isv ? x - p.HKV : x;
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = min(at.n, p.count[b]), l = threadIdx.x % L, g = threadIdx.x / L;
  const int64_t ctx = max(p.ctx[b], 0);
  uint8_t* const cache = static_cast<uint8_t*>(isv ? p.vc : p.kc) + layer * p.pages * p.HKV * p.page * (int64_t)ROW;
  float* const scales = p.ks == nullptr ? nullptr : (isv ? p.vs : p.ks) + layer * p.pages * p.HKV * p.page;
  const auto place = [&](int64_t pos) -> int64_t {  // in rows of the layer's cache; -1: no page
    const int64_t i = (uint32_t)pos / (uint32_t)p.page;  // below 2^31 + 2^31
    if (i >= p.max_pages) return -1;
    const int64_t t = p.table[b * p.max_pages + i];
    return t < 0 || t >= p.pages ? -1 : (t * p.HKV + h) * p.page + (pos - i * p.page);
  };
  for (int i0 = 0; i0 < n; i0 += kKeep) {
    uint4 row[E];
    float scale[E];
    int64_t to[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int i = i0 + e * G + g;
      to[e] = -1;
      if (i >= n) continue;
      const int from = p.path[at.first + i];
      if (from <= i || from >= at.n) continue;  // lies there already, or is no such row
      const int64_t f = place(ctx + from);
      if (f < 0) continue;
      to[e] = place(ctx + i);
      row[e] = *reinterpret_cast<const uint4*>(cache + f * ROW + l * 16);
      if (scales != nullptr) scale[e] = scales[f];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (to[e] >= 0) {
        *reinterpret_cast<uint4*>(cache + to[e] * ROW + l * 16) = row[e];
        if (scales != nullptr && l == 0) scales[to[e]] = scale[e];
      }
  }
}

// --------------------------------------------------------------------------------------------------- tables and counts
__device__ __forceinline__ bool there(int32_t e, int64_t pages) { return e >= 0 && e < pages; }

// The sum of x over the workgroup's threads before this one, and over all of them. red: 16 ints.
__device__ __forceinline__ int block_before(int x, int* red, int& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int upto = wave_scan_sum(x);
  __syncthreads();
  if (lane == 63) red[wave] = upto;
  __syncthreads();
  int before = 0;
  all = 0;
  for (int w = 0; w < waves; ++w) {
    if (w < wave) before += red[w];
    all += red[w];
  }
  return before + upto - x;
}

// Pages behind what a sequence wants are given back; what it lacks is counted.
__global__ void __launch_bounds__(256) pages_release_k(PagesParams p) {
  __shared__ int red[16];
  const int64_t b = blockIdx.x, tokens = p.tokens[b];
  int lacks = 0;
  if (tokens >= 0) {
    const int64_t want = (tokens + p.page - 1) / p.page;
    int32_t* const row = p.table + b * p.max_pages;
    for (int64_t i = threadIdx.x; i < p.max_pages; i += 256) {
      const int32_t e = row[i];
      if (i < want) {
        lacks += !there(e, p.pages);
      } else {
        if (there(e, p.pages)) atomicSub(p.refs + e, 1);
        row[i] = -1;
      }
    }
  }
  int all;
  block_before(lacks, red, all);
  if (threadIdx.x == 0) p.need[b] = all;
}

// One workgroup: where each sequence's share of the taken pages begins, and the lowest free pages, as many as are wanted
// and there are; each counts once from here on.
__global__ void __launch_bounds__(1024) pages_take_k(PagesParams p) {
  __shared__ int red[16];
  int wanted = 0, all;
  for (int64_t b0 = 0; b0 < p.B; b0 += 1024) {
    const int64_t b = b0 + threadIdx.x;
    const int x = b < p.B ? p.need[b] : 0;
    const int before = block_before(x, red, all);
    if (b < p.B) p.first[b] = wanted + before;
    wanted += all;
  }
  int found = 0;
  for (int64_t t0 = 0; t0 < p.pages && found < wanted; t0 += 4096) {
    const int64_t t = t0 + threadIdx.x * 4;
    int mine = 0;
    int32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = t + i < p.pages ? p.refs[t + i] : 1;
      mine += r[i] <= 0;
    }
    int at = found + block_before(mine, red, all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] <= 0) {
        if (at < wanted) {
          p.taken[at] = (int32_t)(t + i);
          p.refs[t + i] = 1;
        }
        ++at;
      }
    found += all;
  }
  if (threadIdx.x == 0) *p.have = min(found, wanted);
}

// The taken pages into the entries that lack one, in order.
__global__ void __launch_bounds__(256) pages_assign_k(PagesParams p) {
  __shared__ int red[16];
  const int64_t b = blockIdx.x, tokens = p.tokens[b];
  if (tokens < 0) {
    if (threadIdx.x == 0) p.out[b] = 0;
    return;
  }
  const int64_t want = (tokens + p.page - 1) / p.page;
  const int have = *p.have;
  int32_t* const row = p.table + b * p.max_pages;
  int at = p.first[b], all;
  for (int64_t i0 = 0; i0 < min(want, p.max_pages); i0 += 256) {
    const int64_t i = i0 + threadIdx.x;
    const bool lacks = i < min(want, p.max_pages) && !there(row[i], p.pages);
    const int rank = at + block_before(lacks, red, all);
    if (lacks) row[i] = rank < have ? p.taken[rank] : -1;
    at += all;
  }
  // those that the pool, and those that the table had no room for
  if (threadIdx.x == 0)
    p.out[b] = (int32_t)(max(0, at - max(have, p.first[b])) + min(max(want - p.max_pages, (int64_t)0), (int64_t)0x3fffffff));
}

// Slot b goes on as slot src[b]'s sequence: its own pages are given back, the full ones of the other shared; a last page
// that is not full is wanted anew, and the other's is held until it has one (its own slot may be giving it back).
__global__ void __launch_bounds__(256) fork_release_k(PagesParams p) {
  const int64_t b = blockIdx.x, s = p.src[b];
  const bool stays = s == b, some = s >= 0 && s < p.B;
  const int64_t len = some ? max(p.ctx[s], 0) : 0, full = min(len / p.page, p.max_pages);
  const int32_t* const from = p.table + (some ? s : 0) * p.max_pages;
  if (!stays)
    for (int64_t i = threadIdx.x; i < p.max_pages; i += 256) {
      const int32_t old = p.table[b * p.max_pages + i], now = some && i < full ? from[i] : -1;
      if (there(old, p.pages)) atomicSub(p.refs + old, 1);
      if (there(now, p.pages)) atomicAdd(p.refs + now, 1);
      p.rows[b * p.max_pages + i] = there(now, p.pages) ? now : -1;
    }
  if (threadIdx.x == 0) {
    int32_t last = -1;
    if (!stays && len > full * p.page && full < p.max_pages) last = from[full];
    if (!there(last, p.pages)) last = -1;
    if (last >= 0) atomicAdd(p.refs + last, 1);
    p.need[b] = last >= 0;
    p.last[b] = last;
    p.len[b] = (int32_t)len;
  }
}

__global__ void __launch_bounds__(256) fork_assign_k(PagesParams p) {
  const int64_t b = blockIdx.x;
  int32_t last = -1, page = -1;
  if (p.src[b] != b) {
    const int64_t len = p.len[b], full = min(len / p.page, p.max_pages);
    last = p.last[b];
    if (last >= 0 && p.first[b] < *p.have) page = p.taken[p.first[b]];
    for (int64_t i = threadIdx.x; i < p.max_pages; i += 256)
      p.table[b * p.max_pages + i] = page >= 0 && i == full ? page : p.rows[b * p.max_pages + i];
    if (threadIdx.x == 0) {
      p.ctx[b] = (int32_t)(last >= 0 && page < 0 ? full * p.page : len);  // no page left: up to the last full one
      if (last >= 0) atomicSub(p.refs + last, 1);
    }
  }
  if (threadIdx.x == 0) {
    p.out[2 * b] = last;
    p.out[2 * b + 1] = page;
  }
}

// ---------------------------------------------------------------------------------------------------------- page copies
// A workgroup moves 16 KB of one page of one layer, keys or values (then a part of its scales): four loads a lane in flight.
__global__ void __launch_bounds__(256) pages_copy_k(CopyParams p) {
  const int64_t pair = blockIdx.y, from = p.pairs[2 * pair], to = p.pairs[2 * pair + 1];
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages || from == to) return;
  const int layer = blockIdx.z >> 1;
  const bool isv = blockIdx.z & 1;
  uint8_t* const cache = static_cast<uint8_t*>(isv ? p.vc : p.kc) + layer * p.pages * p.bytes;
  const uint4* const src = reinterpret_cast<const uint4*>(cache + from * p.bytes);
  uint4* const dst = reinterpret_cast<uint4*>(cache + to * p.bytes);
  const int64_t many = p.bytes / 16, at = (int64_t)blockIdx.x * 1024 + threadIdx.x;
  uint4 x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 256 < many) x[i] = src[at + i * 256];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i * 256 < many) dst[at + i * 256] = x[i];
  if (p.ks != nullptr) {
    float* const sc = (isv ? p.vs : p.ks) + layer * p.pages * p.scales;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.scales; i += (int64_t)gridDim.x * 256)
      sc[to * p.scales + i] = sc[from * p.scales + i];
  }
}

}  // namespace

hipError_t launch_kv_keep(const KeepParams& p, int layers, int row_bytes, hipStream_t st) {
  const auto kernel = row_bytes == 512 ? kv_keep_k<512> : row_bytes == 256 ? kv_keep_k<256> : kv_keep_k<128>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.B, (unsigned)(2 * p.HKV * layers)), dim3(256), 0, st, p);
  return hipGetLastError();
}

int64_t pages_work_ints(int64_t B, int64_t max_pages, int64_t pages, bool fork) {
  const int64_t taken = std::min(fork ? B : B * max_pages, pages);
  return 4 + (fork ? 4 : 2) * B + taken + (fork ? B * max_pages : 0);
}

hipError_t launch_pages(PagesParams p, bool fork, int32_t* work, hipStream_t st) {
  p.have = work;
  p.need = work + 4;
  p.first = p.need + p.B;
  p.last = p.first + p.B;
  p.len = p.last + p.B;
  p.taken = fork ? p.len + p.B : p.last;
  p.rows = p.taken + std::min(fork ? p.B : p.B * p.max_pages, p.pages);
  hipLaunchKernelGGL(fork ? fork_release_k : pages_release_k, dim3((unsigned)p.B), dim3(256), 0, st, p);
  hipLaunchKernelGGL(pages_take_k, dim3(1), dim3(1024), 0, st, p);
  hipLaunchKernelGGL(fork ? fork_assign_k : pages_assign_k, dim3((unsigned)p.B), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_pages_copy(const CopyParams& p, int64_t n, int layers, hipStream_t st) {
  hipLaunchKernelGGL(pages_copy_k, dim3((unsigned)((p.bytes + 16383) / 16384), (unsigned)n, (unsigned)(2 * layers)),
                     dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

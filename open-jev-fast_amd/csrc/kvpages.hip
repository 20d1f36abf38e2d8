// What becomes of a paged cache around drafted tokens: accepted rows moved together, pages taken, given back, shared and
// copied. A table row names a sequence's pages, refs counts the table entries that name each page; a page with none is free.
//
// All of it is whole numbers and copies. Tables and counts are small: what bounds them is the chain of launches and loads. For 64
// sequences of 16 entries a resize that gives each a page and one that takes it back are 7.7 us, one that changes nothing 3.3, a
// fork of every other sequence 6.6, in one launch each. Where free pages are rare the scan for them counts: 256 sequences of
// 2048 entries get a page each from the 300 free ones of 389000, and give it back, in 155 us.
#include "ojx_internal.h"

#include <algorithm>

namespace ojx {

namespace {

// ------------------------------------------------------------------------------------------------------- accepted rows
// Sequence b keeps the drafted rows path[0 .. count - 1]: the row at position ctx + path[i] goes to ctx + i. With path[i] >=
// i (any rising path; other entries are left out) a place that is written is none that a later entry reads, so that a thread
// may take its 16 bytes of every entry in order, four read and then written, with no barrier between.
//
// A workgroup looks a sequence's places up once, 128 entries at a time, and then moves them for 256 / L heads' keys or values
// of some layer at once, a row being L lanes of 16 bytes. What bounds it: the chain pointers, path, table, rows, 3.1 us for one
// sequence and layer; 64 sequences of up to 6 rows in 16 layers, 9 MB, 6.2 us (27 with a look-up for every head and layer).
template <int ROW>  // bytes of a row
__global__ void __launch_bounds__(256) kv_keep_k(KeepParams p, int parts) {
  constexpr int L = ROW / 16, G = 256 / L, kList = 128;
  __shared__ int64_t from[kList], to[kList];  // places in a head's rows: page * HKV * page size + offset; -1: nothing to move
  const int64_t b = blockIdx.x;
  const int count = p.count[b], l = threadIdx.x % L;
  const int64_t ctx = max(p.ctx[b], 0);
  SeqPlace at;
  if (!seq_find(p.q_ptr, p.B, p.N, [](int, int) { return 0; }, [=](int i, int) { return i == (int)b; }, at)) return;
  const int n = min(at.n, count);
  const auto place = [&](int64_t pos) -> int64_t {
    const int64_t i = (uint32_t)pos / (uint32_t)p.page;  // below 2^31 + 2^31
    if (i >= p.max_pages) return -1;
    const int64_t t = p.table[b * p.max_pages + i];
    return t < 0 || t >= p.pages ? -1 : t * p.HKV * p.page + (pos - i * p.page);
  };
  const int64_t rows = p.pages * p.HKV * p.page;  // of a layer
  for (int i0 = 0; i0 < n; i0 += kList) {
    const int many = min(kList, n - i0);
    if (i0 > 0) __syncthreads();
    if (threadIdx.x < kList) {
      const int i = i0 + threadIdx.x;
      int64_t f = -1, t = -1;
      if (i < n) {
        const int r = p.path[at.first + i];
        if (r > i && r < at.n) {  // else it lies there already, or is no such row
          f = place(ctx + r);
          t = place(ctx + i);
        }
      }
      from[threadIdx.x] = t < 0 ? -1 : f;
      to[threadIdx.x] = t;
    }
    __syncthreads();
    for (int x = blockIdx.y * G + threadIdx.x / L; x < parts; x += gridDim.y * G) {
      const int layer = x / (2 * p.HKV), y = x - layer * 2 * p.HKV;
      const bool isv = y >= p.HKV;
      const int64_t first = layer * rows + (int64_t)(isv ? y - p.HKV : y) * p.page;
      uint8_t* const cache = static_cast<uint8_t*>(isv ? p.vc : p.kc) + first * ROW + l * 16;
      float* const scales = p.ks == nullptr ? nullptr : (isv ? p.vs : p.ks) + first;
      for (int i = 0; i < many; i += 4) {  // kList is a multiple of four, and the list full of -1 behind n
        const int64_t f0 = from[i], f1 = from[i + 1], f2 = from[i + 2], f3 = from[i + 3];
        uint4 r0, r1, r2, r3;
        float s0, s1, s2, s3;
        if (f0 >= 0) r0 = *reinterpret_cast<const uint4*>(cache + f0 * ROW);
        if (f1 >= 0) r1 = *reinterpret_cast<const uint4*>(cache + f1 * ROW);
        if (f2 >= 0) r2 = *reinterpret_cast<const uint4*>(cache + f2 * ROW);
        if (f3 >= 0) r3 = *reinterpret_cast<const uint4*>(cache + f3 * ROW);
        if (scales != nullptr && l == 0) {
          if (f0 >= 0) s0 = scales[f0];
          if (f1 >= 0) s1 = scales[f1];
          if (f2 >= 0) s2 = scales[f2];
          if (f3 >= 0) s3 = scales[f3];
        }
        if (f0 >= 0) *reinterpret_cast<uint4*>(cache + to[i] * ROW) = r0;
        if (f1 >= 0) *reinterpret_cast<uint4*>(cache + to[i + 1] * ROW) = r1;
        if (f2 >= 0) *reinterpret_cast<uint4*>(cache + to[i + 2] * ROW) = r2;
        if (f3 >= 0) *reinterpret_cast<uint4*>(cache + to[i + 3] * ROW) = r3;
        if (scales != nullptr && l == 0) {
          if (f0 >= 0) scales[to[i]] = s0;
          if (f1 >= 0) scales[to[i + 1]] = s1;
          if (f2 >= 0) scales[to[i + 2]] = s2;
          if (f3 >= 0) scales[to[i + 3]] = s3;
        }
      }
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

// A call has three parts: what sequences give back (and what they want), the free pages that are taken, where they go. With
// large tables each is a launch, the first and the last with a workgroup per sequence. A table of up to kSmall entries is one
// workgroup's, an entry a thread at a time, in one launch.
// In one launch and in three, the two resizes above take 7.7 and 17 us for 64 x 16 entries, 15.9 and 17.1 for 64 x 64, 29 and 18
// for 128 x 64; forks 6.6 and 10.2, 11.5 and 10.8, 19.6 and 10.9.
constexpr int kSmall = 4096;

// Pages behind what a sequence wants are given back; what it lacks is counted.
__device__ __forceinline__ void release(const PagesParams& p, int64_t b, int* red) {
  const int64_t tokens = p.tokens[b];
  int lacks = 0;
  if (tokens >= 0) {
    const int64_t want = (tokens + p.page - 1) / p.page;
    int32_t* const row = p.table + b * p.max_pages;
    for (int64_t i = threadIdx.x; i < p.max_pages; i += blockDim.x) {
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

// One workgroup: the lowest free pages, as many as are wanted and there are; each counts once from here on. How many.
__device__ __forceinline__ int take(const PagesParams& p, int wanted, int32_t* taken, int* red) {
  int found = 0, all;
  for (int64_t t0 = 0; t0 < p.pages && found < wanted; t0 += 4 * blockDim.x) {
    const int64_t t = t0 + threadIdx.x * 4;
    int mine = 0;
    int32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      r[i] = t + i < p.pages ? __hip_atomic_load(p.refs + t + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 1;
      mine += r[i] <= 0;
    }
    int at = found + block_before(mine, red, all);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (r[i] <= 0) {
        if (at < wanted) {
          taken[at] = (int32_t)(t + i);
          p.refs[t + i] = 1;
        }
        ++at;
      }
    found += all;
  }
  return min(found, wanted);
}

// The taken pages into the entries that lack one, in order.
__device__ __forceinline__ void assign(const PagesParams& p, int64_t b, int* red) {
  const int64_t tokens = p.tokens[b];
  if (tokens < 0) {
    if (threadIdx.x == 0) p.out[b] = 0;
    return;
  }
  const int64_t want = (tokens + p.page - 1) / p.page;
  const int have = *p.have;
  int32_t* const row = p.table + b * p.max_pages;
  int at = p.first[b], all;
  for (int64_t i0 = 0; i0 < min(want, p.max_pages); i0 += blockDim.x) {
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
__device__ __forceinline__ void fork_release(const PagesParams& p, int64_t b, int*) {
  const int64_t s = p.src[b];
  const bool stays = s == b, some = s >= 0 && s < p.B;
  const int64_t len = some ? max(p.ctx[s], 0) : 0, full = min(len / p.page, p.max_pages);
  const int32_t* const from = p.table + (some ? s : 0) * p.max_pages;
  if (!stays)
    for (int64_t i = threadIdx.x; i < p.max_pages; i += blockDim.x) {
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

__device__ __forceinline__ void fork_assign(const PagesParams& p, int64_t b, int*) {
  int32_t last = -1, page = -1;
  if (p.src[b] != b) {
    const int64_t len = p.len[b], full = min(len / p.page, p.max_pages);
    last = p.last[b];
    if (last >= 0 && p.first[b] < *p.have) page = p.taken[p.first[b]];
    for (int64_t i = threadIdx.x; i < p.max_pages; i += blockDim.x)
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

template <bool FORK>
__global__ void __launch_bounds__(256) pages_release_k(PagesParams p) {
  __shared__ int red[16];
  FORK ? fork_release(p, blockIdx.x, red) : release(p, blockIdx.x, red);
}
// And where each sequence's share of them begins.
__global__ void __launch_bounds__(1024) pages_take_k(PagesParams p) {
  __shared__ int red[16];
  int wanted = 0, all;
  for (int64_t b0 = 0; b0 < p.B; b0 += 1024) {
    const int64_t b = b0 + threadIdx.x;
    const int before = block_before(b < p.B ? p.need[b] : 0, red, all);
    if (b < p.B) p.first[b] = wanted + before;
    wanted += all;
  }
  const int have = take(p, wanted, p.taken, red);
  if (threadIdx.x == 0) *p.have = have;
}
template <bool FORK>
__global__ void __launch_bounds__(256) pages_assign_k(PagesParams p) {
  __shared__ int red[16];
  FORK ? fork_assign(p, blockIdx.x, red) : assign(p, blockIdx.x, red);
}

// B * max_pages at most kSmall (and max_pages at least 1): thread t has the entries t, t + 1024, ..
__global__ void __launch_bounds__(1024) resize_small_k(PagesParams p) {
  __shared__ int red[16], taken[kSmall];
  const int many = (int)(p.B * p.max_pages);
  int rank[kSmall / 1024], wanted = 0, all;
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k) {
    rank[k] = -1;
    if (k * 1024 >= many) continue;  // the same for the whole workgroup
    const int f = k * 1024 + threadIdx.x;
    bool lacks = false;
    if (f < many) {
      const int b = f / (int)p.max_pages, i = f - b * (int)p.max_pages;
      const int64_t tokens = p.tokens[b], want = (tokens + p.page - 1) / p.page;
      const int32_t e = p.table[f];
      const bool some = there(e, p.pages);
      if (tokens >= 0 && i >= want) {
        if (some) atomicSub(p.refs + e, 1);
        p.table[f] = -1;
      }
      lacks = tokens >= 0 && i < want && !some;
    }
    const int before = block_before(lacks, red, all);
    if (lacks) rank[k] = wanted + before;
    wanted += all;
  }
  for (int b = threadIdx.x; b < (int)p.B; b += 1024) {
    const int64_t tokens = p.tokens[b], want = (tokens + p.page - 1) / p.page;
    p.out[b] = tokens < 0 ? 0 : (int32_t)max(want - p.max_pages, (int64_t)0);
  }
  __syncthreads();  // counts (atomic, and read so) and outputs, before other threads go on with them
  const int have = take(p, wanted, taken, red);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k)
    if (rank[k] >= 0) {
      const int f = k * 1024 + threadIdx.x;
      p.table[f] = rank[k] < have ? taken[rank[k]] : -1;
      if (rank[k] >= have) atomicAdd(p.out + f / (int)p.max_pages, 1);
    }
}

__global__ void __launch_bounds__(1024) fork_small_k(PagesParams p) {
  __shared__ int red[16], taken[kSmall];
  const int many = (int)(p.B * p.max_pages), MP = (int)p.max_pages;
  int32_t now[kSmall / 1024], last[kSmall / 1024], len[kSmall / 1024];
  int rank[kSmall / 1024], wanted = 0, all;
  const auto sequence = [&](int b, int64_t& s, int64_t& n, int& full) {  // of which slot, how long, full pages
    s = p.src[b];
    n = s >= 0 && s < p.B ? max(p.ctx[s], 0) : 0;
    full = (int)min(n / p.page, p.max_pages);
    if (s < 0 || s >= p.B) s = -1;
  };
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k) {
    now[k] = -1;
    const int f = k * 1024 + threadIdx.x;
    if (f < many) {
      const int b = f / MP, i = f - b * MP;
      int64_t s, n;
      int full;
      sequence(b, s, n, full);
      if (s != b) {
        const int32_t old = p.table[f];
        if (s >= 0 && i < full) now[k] = p.table[s * MP + i];
        if (!there(now[k], p.pages)) now[k] = -1;
        if (there(old, p.pages)) atomicSub(p.refs + old, 1);
        if (now[k] >= 0) atomicAdd(p.refs + now[k], 1);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k) {
    last[k] = -1, len[k] = 0, rank[k] = 0;
    if (k * 1024 >= p.B) continue;  // the same for the whole workgroup
    const int b = k * 1024 + threadIdx.x;
    if (b < p.B) {
      int64_t s, n;
      int full;
      sequence(b, s, n, full);
      len[k] = (int32_t)n;
      if (s >= 0 && s != b && n > (int64_t)full * p.page && full < MP) last[k] = p.table[s * MP + full];
      if (!there(last[k], p.pages)) last[k] = -1;
      if (last[k] >= 0) atomicAdd(p.refs + last[k], 1);
    }
    const int before = block_before(last[k] >= 0, red, all);
    rank[k] = wanted + before;
    wanted += all;
  }
  __syncthreads();  // counts (atomic, and read so), and reads of the tables before they change
  const int have = take(p, wanted, taken, red);
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k) {
    const int f = k * 1024 + threadIdx.x;
    if (f < many && p.src[f / MP] != f / MP) p.table[f] = now[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kSmall / 1024; ++k) {
    const int b = k * 1024 + threadIdx.x;
    if (b >= p.B) continue;
    int32_t page = -1;
    if (p.src[b] != b) {
      const int full = (int)min((int64_t)len[k] / p.page, p.max_pages);
      if (last[k] >= 0) {
        if (rank[k] < have) page = taken[rank[k]];
        if (page >= 0) p.table[b * MP + full] = page;
        atomicSub(p.refs + last[k], 1);
      }
      p.ctx[b] = last[k] >= 0 && page < 0 ? full * p.page : len[k];
    }
    p.out[2 * b] = last[k];
    p.out[2 * b + 1] = page;
  }
}

// ---------------------------------------------------------------------------------------------------------- page copies
// Past the caches: nothing reads a copy soon, or the copies do not fit (56 pages of 16 layers, 235 MB, in 39 us for 66; 8 MB in
// 3.6 for 4.1; a sum over the copies right after them takes as long either way).
__device__ __forceinline__ void store_past(uint4* p, uint4 x) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  __builtin_nontemporal_store((u32x4{x.x, x.y, x.z, x.w}), reinterpret_cast<u32x4*>(p));
}

// A workgroup moves 16 KB of one page of one layer, keys or values (then a part of its scales): four loads a lane in flight.
// What bounds it: the writes (56 pages of 16 layers from 8, 235 MB: 39 to 43 us, 5.5 to 6 TB/s).
__global__ void __launch_bounds__(256) pages_copy_k(CopyParams p) {
  const int64_t pair = blockIdx.y, from = p.pairs[2 * pair], to = p.pairs[2 * pair + 1];
  if (from < 0 || from >= p.pages || to < 0 || to >= p.pages || from == to) return;
  const int layer = blockIdx.z >> 1;
  const bool isv = blockIdx.z & 1;
  uint8_t* const cache = static_cast<uint8_t*>(isv ? p.vc : p.kc) + layer * p.pages * p.bytes;
  const uint4* const src = reinterpret_cast<const uint4*>(cache + from * p.bytes);
  uint4* const dst = reinterpret_cast<uint4*>(cache + to * p.bytes);
  const int64_t many = p.bytes / 16, at = (int64_t)blockIdx.x * 1024 + threadIdx.x;
  if (at + 768 < many) {
    const uint4 x0 = src[at], x1 = src[at + 256], x2 = src[at + 512], x3 = src[at + 768];
    store_past(dst + at, x0);
    store_past(dst + at + 256, x1);
    store_past(dst + at + 512, x2);
    store_past(dst + at + 768, x3);
  } else {
    for (int64_t i = at; i < min(many, (int64_t)(blockIdx.x + 1) * 1024); i += 256) dst[i] = src[i];
  }
  if (p.ks != nullptr) {
    float* const sc = (isv ? p.vs : p.ks) + layer * p.pages * p.scales;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.scales; i += (int64_t)gridDim.x * 256)
      sc[to * p.scales + i] = sc[from * p.scales + i];
  }
}

}  // namespace

hipError_t launch_kv_keep(const KeepParams& p, int layers, int row_bytes, hipStream_t st) {
  const auto kernel = row_bytes == 512 ? kv_keep_k<512> : row_bytes == 256 ? kv_keep_k<256> : kv_keep_k<128>;
  const int parts = 2 * p.HKV * layers, groups = (parts * (row_bytes / 16) + 255) / 256;
  hipLaunchKernelGGL(kernel, dim3((unsigned)p.B, (unsigned)std::min(groups, std::max(1, 2048 / p.B))), dim3(256), 0, st, p,
                     parts);
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
  if (p.max_pages > 0 && p.B * p.max_pages <= kSmall) {
    hipLaunchKernelGGL(fork ? fork_small_k : resize_small_k, dim3(1), dim3(1024), 0, st, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(fork ? pages_release_k<true> : pages_release_k<false>, dim3((unsigned)p.B), dim3(256), 0, st, p);
  hipLaunchKernelGGL(pages_take_k, dim3(1), dim3(1024), 0, st, p);
  hipLaunchKernelGGL(fork ? pages_assign_k<true> : pages_assign_k<false>, dim3((unsigned)p.B), dim3(256), 0, st, p);
  return hipGetLastError();
}

hipError_t launch_pages_copy(const CopyParams& p, int64_t n, int layers, hipStream_t st) {
  hipLaunchKernelGGL(pages_copy_k, dim3((unsigned)((p.bytes + 16383) / 16384), (unsigned)n, (unsigned)(2 * layers)),
                     dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace ojx

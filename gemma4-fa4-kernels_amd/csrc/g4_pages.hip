// Page tables and reference counts of the paged cache, and the copies of pages.
//
// The tables are small (a few thousand entries) and the pool's counts a few
// bytes a page, so the calls are bound by their launches and by chains of
// dependent loads: each is one or two launches, and what needs an order over the
// whole pool or batch (ranks of free pages, of requests, of moves) is a prefix
// sum by one workgroup.  Ranks, not atomics, decide who gets what, so results
// repeat bitwise; atomics only add to counts.
#include "g4_cache.h"

namespace g4 {

namespace {

__device__ __forceinline__ int pages_of(int len, int page_size) {
  return len > 0 ? (len - 1) / page_size + 1 : 0;
}
__device__ __forceinline__ bool is_page(int id, int num_pages) {
  return (unsigned)id < (unsigned)num_pages;
}

// Inclusive prefix sum of x over the workgroup's threads (kNT, a multiple of 64)
// and the sum of all; every thread calls it.  lds: kNT / 64 ints, free again
// after the next barrier.
template <int kNT>
__device__ __forceinline__ int block_scan(int x, int G4_LDS* lds, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o, 64);
    if (lane >= o) x += y;
  }
  __syncthreads();  // earlier readers of lds are done
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kNT / 64; ++w) {
    const int y = lds[w];
    before += w < wave ? y : 0;
    total += y;
  }
  return x + before;
}

constexpr int kScan = 1024;  // threads of the ordering workgroup

}  // namespace

// ---- fork -------------------------------------------------------------------
// The rows as they will be, from the rows as they are (some of which the call
// replaces too), then written over them by a second launch.
__global__ void __launch_bounds__(256) fork_rows_kernel(PagesParams a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int width = a.tab.width;
  if (x >= (int64_t)a.tab.batch * width) return;
  const int b = (int)(x / width), w = (int)(x % width);
  const int p = a.rows[b];
  if (p == b) return;
  const int old = a.tab.pages[x];
  if (w < pages_of(a.tab.seq_lens[b], a.page_size) && is_page(old, a.num_pages))
    atomicAdd(&a.refs[old], -1);
  int id = -1, len = 0;
  if ((unsigned)p < (unsigned)a.tab.batch) {
    len = a.tab.seq_lens[p];
    if (w < pages_of(len, a.page_size)) {
      id = a.tab.pages[(int64_t)p * width + w];
      if (is_page(id, a.num_pages)) atomicAdd(&a.refs[id], 1);
    }
  }
  a.ws[x] = id;
  if (w == 0) a.ws[(int64_t)a.tab.batch * width + b] = len;
}

__global__ void __launch_bounds__(256) fork_store_kernel(PagesParams a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int width = a.tab.width;
  if (x >= (int64_t)a.tab.batch * width) return;
  const int b = (int)(x / width);
  if (a.rows[b] == b) return;
  a.tab.pages[x] = a.ws[x];
  if (x % width == 0) a.tab.seq_lens[b] = a.ws[(int64_t)a.tab.batch * width + b];
}

// ---- reserve ----------------------------------------------------------------
// Workspace: [free pages in order: num_pages][writers: num_pages][first writer:
// num_pages][per row: first request: batch][requests of all rows that free pages
// were found for: 1].
namespace {
struct ReserveRow {
  int cur, want, have, need, last;  // last: the part-full page to be copied, or -1
  __device__ __forceinline__ void init(const PagesParams& a, int b) {
    cur = max(a.tab.seq_lens[b], 0);
    want = a.rows[b];
    have = pages_of(cur, a.page_size);
    need = pages_of(want, a.page_size);
    last = -1;
    if (grows(a) && cur % a.page_size != 0) {
      const int id = a.tab.pages[(int64_t)b * a.tab.width + cur / a.page_size];
      if (is_page(id, a.num_pages) && a.refs[id] > 1) last = id;
    }
  }
  __device__ __forceinline__ bool grows(const PagesParams& a) const {
    return want > cur && need <= a.tab.width;
  }
};
}  // namespace

__global__ void __launch_bounds__(kScan) reserve_order_kernel(PagesParams a) {
  __shared__ int lds[kScan / 64];
  int G4_LDS* sh = (int G4_LDS*)lds;
  const int tid = threadIdx.x, n = a.num_pages, batch = a.tab.batch;
  int* const free = a.ws;
  int* const writers = free + n;
  int* const first = writers + n;
  int* const begin = first + n;
  // rows that write into the same shared page
  for (int b = tid; b < batch; b += kScan) {
    ReserveRow r;
    r.init(a, b);
    if (r.last >= 0) writers[r.last] = 0, first[r.last] = 0x7fffffff;
  }
  __syncthreads();
  for (int b = tid; b < batch; b += kScan) {
    ReserveRow r;
    r.init(a, b);
    if (r.last >= 0) atomicAdd(&writers[r.last], 1), atomicMin(&first[r.last], b);
  }
  __syncthreads();
  // requests in the order of the rows
  int64_t asked = 0;
  for (int b0 = 0; b0 < batch; b0 += kScan) {
    const int b = b0 + tid;
    int x = 0;
    if (b < batch) {
      ReserveRow r;
      r.init(a, b);
      if (r.grows(a)) x = r.need - r.have;
      if (r.last >= 0) {
        const int held = __hip_atomic_load(&writers[r.last], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
        const int lead = __hip_atomic_load(&first[r.last], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
        const bool copy = held < a.refs[r.last] || lead != b;
        x += copy;
        a.src[b] = copy ? r.last : -1;
      } else {
        a.src[b] = -1;
      }
    }
    int total;
    const int incl = block_scan<kScan>(x, sh, total);
    // (a sum past the pool is as good as one past it by one)
    if (b < batch) begin[b] = (int)min(asked + incl - x, (int64_t)n + 1);
    asked += total;
  }
  // the lowest free pages, as many as were asked for
  const int want = (int)min(asked, (int64_t)n);
  int found = 0;
  for (int p0 = 0; p0 < n && found < want; p0 += 4 * kScan) {
    int ref[4];
    int x = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = p0 + 4 * tid + e;
      ref[e] = p < n ? a.refs[p] : 1;
      x += ref[e] == 0;
    }
    int total;
    int rank = found + block_scan<kScan>(x, sh, total) - x;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (ref[e] == 0) free[rank++] = p0 + 4 * tid + e;
    found += total;
  }
  if (tid == 0) begin[batch] = found;
}

// One wave per row.
__global__ void __launch_bounds__(256) reserve_store_kernel(PagesParams a) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (b >= a.tab.batch) return;
  const int* const free = a.ws;
  const int* const begin = free + 3 * (int64_t)a.num_pages;
  const int width = a.tab.width;
  const int cur = max(a.tab.seq_lens[b], 0), want = a.rows[b];
  const int have = pages_of(cur, a.page_size), need = pages_of(want, a.page_size);
  const int old = a.src[b];
  const int copy = old >= 0, k = begin[b];
  int granted = 1, moved = -1;
  if (want > cur) {
    granted = need <= width && (int64_t)k + copy + need - have <= begin[a.tab.batch];
    if (granted) {
      if (copy) moved = free[k];
      for (int i = lane; i < need - have; i += 64) {
        const int id = free[k + copy + i];
        a.tab.pages[(int64_t)b * width + have + i] = id;
        a.refs[id] = 1;
      }
    }
  }
  if (lane != 0) return;
  if (moved >= 0) {
    a.tab.pages[(int64_t)b * width + cur / a.page_size] = moved;
    a.refs[moved] = 1;
    atomicAdd(&a.refs[old], -1);
  } else {
    a.src[b] = -1;
  }
  a.dst[b] = moved;
  a.granted[b] = granted;
  if (granted && want > cur) a.tab.seq_lens[b] = want;
}

// ---- release ----------------------------------------------------------------
__global__ void __launch_bounds__(64) release_kernel(PagesParams a) {
  const int b = blockIdx.x;
  const int len = max(a.tab.seq_lens[b], 0), keep = min(len, max(a.rows[b], 0));
  const int used = min(pages_of(len, a.page_size), a.tab.width);
  const int kept = pages_of(keep, a.page_size);
  int* const row = a.tab.pages + (int64_t)b * a.tab.width;
  for (int w = threadIdx.x; w < used; w += 64) {
    // (a page past its window: its last token at or before keep - window)
    const int64_t t0 = (int64_t)w * a.page_size;
    const bool passed = a.window > 0 && t0 >= a.sinks &&
                        t0 + a.page_size - 1 <= (int64_t)keep - a.window;
    if (w < kept && !passed) continue;
    const int id = row[w];
    if (is_page(id, a.num_pages)) atomicAdd(&a.refs[id], -1);
    row[w] = -1;
  }
  __syncthreads();
  if (threadIdx.x == 0) a.tab.seq_lens[b] = keep;
}

// ---- compact ----------------------------------------------------------------
// Workspace: [where each page goes: num_pages][pages in use: 1].
__global__ void __launch_bounds__(kScan) compact_order_kernel(PagesParams a) {
  __shared__ int lds[kScan / 64];
  int G4_LDS* sh = (int G4_LDS*)lds;
  const int tid = threadIdx.x, n = a.num_pages, most = max(n / 2, 1);
  int* const to = a.ws;
  int live = 0;
  for (int p = tid; p < n; p += kScan) live += a.refs[p] > 0;
  int count;
  block_scan<kScan>(live, sh, count);
  // moves and holes in order (each at most n / 2, so their ranks share an int's halves
  // only up to 2^16 pages: two scans)
  int moves = 0, holes = 0;
  for (int p0 = 0; p0 < n; p0 += 4 * kScan) {
    bool used[4];
    int m = 0, h = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = p0 + 4 * tid + e;
      used[e] = p < n && a.refs[p] > 0;
      m += used[e] && p >= count;
      h += !used[e] && p < count;
    }
    int mt, ht;
    int mr = moves + block_scan<kScan>(m, sh, mt) - m;
    int hr = holes + block_scan<kScan>(h, sh, ht) - h;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int p = p0 + 4 * tid + e;
      if (p >= n) continue;
      if (p >= count) {
        to[p] = p;
        if (used[e]) a.src[mr++] = p;
      } else if (!used[e]) {
        a.dst[hr++] = p;
      }
    }
    moves += mt;
    holes += ht;
  }
  __syncthreads();
  for (int i = tid; i < most; i += kScan) {
    if (i < moves) {
      const int s = a.src[i], d = a.dst[i];
      to[s] = d;
      a.refs[d] = a.refs[s];
      a.refs[s] = 0;
    } else {
      a.src[i] = a.dst[i] = -1;
    }
  }
  if (tid == 0) to[n] = count;
}

__global__ void __launch_bounds__(256) compact_store_kernel(PagesParams a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= (int64_t)a.tab.batch * a.tab.width) return;
  const int id = a.tab.pages[x];
  if (is_page(id, a.num_pages) && id >= a.ws[a.num_pages]) a.tab.pages[x] = a.ws[id];
}

// ---- copy -------------------------------------------------------------------
// One workgroup per (pair, K or V, 32 KB of the page): a page's heads lie one
// after the other, so that is one run of bytes.
constexpr int kCopyChunk = 32768;

__global__ void __launch_bounds__(256) copy_kernel(CopyParams a) {
  const g4_paged_cache& c = a.c;
  const int pair = blockIdx.x, chunk = blockIdx.y, which = blockIdx.z;
  const int s = a.src[pair], d = a.dst[pair];
  if (!is_page(s, c.num_pages) || !is_page(d, c.num_pages) || s == d) return;
  const int64_t bytes = (int64_t)c.num_kv_heads * c.page_size * c.head_dim;
  uint8_t* const base = (uint8_t*)(which ? c.v : c.k);
  const u32x4* from = (const u32x4*)(base + s * bytes);
  u32x4* to = (u32x4*)(base + d * bytes);
  const int64_t first = (int64_t)chunk * (kCopyChunk / 16) + threadIdx.x;
  const int64_t end = bytes / 16;
  u32x4 x[kCopyChunk / 4096];
#pragma unroll
  for (int i = 0; i < kCopyChunk / 4096; ++i)
    if (first + i * 256 < end) x[i] = from[first + i * 256];
#pragma unroll
  for (int i = 0; i < kCopyChunk / 4096; ++i)
    if (first + i * 256 < end) to[first + i * 256] = x[i];
  if (chunk == 0) {
    const int64_t m = (int64_t)c.num_kv_heads * (c.page_size / kCacheBlock);
    float* const sc = which ? c.v_scale : c.k_scale;
    for (int64_t i = threadIdx.x; i < m; i += 256) sc[d * m + i] = sc[s * m + i];
  }
}

// ---- launches ---------------------------------------------------------------
size_t pages_workspace_bytes(int64_t num_pages, int64_t batch, int64_t width) {
  const int64_t fork = batch * width + batch, reserve = 3 * num_pages + batch + 1;
  return ((size_t)std::max(fork, reserve) * 4 + 255) & ~size_t(255);
}

static unsigned entry_blocks(const PagesParams& a) {
  return (unsigned)(((int64_t)a.tab.batch * a.tab.width + 255) / 256);
}

hipError_t launch_pages_fork(const PagesParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(fork_rows_kernel, dim3(entry_blocks(a)), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fork_store_kernel, dim3(entry_blocks(a)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_reserve(const PagesParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(reserve_order_kernel, dim3(1), dim3(kScan), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(reserve_store_kernel, dim3((unsigned)(a.tab.batch + 3) / 4), dim3(256), 0,
                     stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_release(const PagesParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(release_kernel, dim3((unsigned)a.tab.batch), dim3(64), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PagesParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(compact_order_kernel, dim3(1), dim3(kScan), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(compact_store_kernel, dim3(entry_blocks(a)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_copy(const CopyParams& a, int count, hipStream_t stream) {
  const int64_t bytes = (int64_t)a.c.num_kv_heads * a.c.page_size * a.c.head_dim;
  const dim3 grid((unsigned)count, (unsigned)((bytes + kCopyChunk - 1) / kCopyChunk), 2);
  hipLaunchKernelGGL(copy_kernel, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace g4

// Page tables and reference counts of the paged cache, and the copies of pages.
//
// The tables are small (a few thousand entries) and the pool's counts a few
// bytes a page, so the calls are bound by their launches and by chains of
// dependent loads: each is one or two launches, and what needs an order over the
// whole pool or batch (ranks of free pages, of requests, of moves) is a prefix
// sum by one workgroup.  Ranks, not atomics, decide who gets what, so results
// repeat bitwise; atomics only add to counts.  Kernels: fork of 24 rows of 130 pages
// 7.7 us (two launches 3.7 + 2.8, and 3 us more of host time), reserve for them 7.2
// (5.8 + 3.6), release of 256 rows 4.6, the order of 16000 pages 10.8 and their 16384
// entries 4.6.
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
constexpr int kRun = 16;     // pages of a thread in a step of its scans

// A step of the ordering workgroup over pages p0 .. p0 + kRun kScan - 1 by their
// counts.  A wave takes 1024 pages in a row, 64 an instruction (bit e of a thread's
// masks is its page at(e)), so ballots rank them and only the waves' totals go
// through LDS.
struct PageStep {
  int first;       // the thread's first page
  unsigned there;  // its pages below n
  __device__ __forceinline__ int at(int e) const { return first + 64 * e; }
  // The thread's pages whose count satisfies pred.
  template <class Pred>
  __device__ __forceinline__ unsigned init(int p0, int n, const int* refs, Pred pred) {
    first = p0 + (threadIdx.x >> 6) * (64 * kRun) + (threadIdx.x & 63);
    int ref[kRun];  // (their loads in flight together)
#pragma unroll
    for (int e = 0; e < kRun; ++e) ref[e] = refs[min(at(e), n - 1)];
    unsigned bits = 0;
    there = 0;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      there |= (unsigned)(at(e) < n) << e;
      bits |= (unsigned)(at(e) < n && pred(ref[e])) << e;
    }
    return bits;
  }
  // f(rank, page) for the pages of `bits` in order, ranks from `rank` on (the wave's).
  template <class F>
  __device__ __forceinline__ void each(unsigned bits, int rank, F f) const {
    const unsigned long long below = (1ull << (threadIdx.x & 63)) - 1;
#pragma unroll
    for (int e = 0; e < kRun; ++e) {
      const unsigned long long m = __ballot(bits >> e & 1);
      if (bits >> e & 1) f(rank + __popcll(m & below), at(e));
      rank += __popcll(m);
    }
  }
};

// Set bits of x and of y over the wave, packed (each at most 1024): x + y << 16.
__device__ __forceinline__ int wave_counts(unsigned x, unsigned y) {
  int n = 0;
#pragma unroll
  for (int e = 0; e < kRun; ++e)
    n += __popcll(__ballot(x >> e & 1)) + (__popcll(__ballot(y >> e & 1)) << 16);
  return n;
}
// Sums over the waves before this one, and over all, of a wave's packed counts.
struct WaveSums {
  int before_x, before_y, x, y;
  __device__ __forceinline__ explicit WaveSums(int mine, int G4_LDS* lds) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // earlier readers of lds are done
    if ((threadIdx.x & 63) == 0) lds[wave] = mine;
    __syncthreads();
    before_x = before_y = x = y = 0;
#pragma unroll
    for (int w = 0; w < kScan / 64; ++w) {
      const int v = lds[w];
      before_x += w < wave ? v & 0xffff : 0;
      before_y += w < wave ? v >> 16 : 0;
      x += v & 0xffff;
      y += v >> 16;
    }
  }
};

}  // namespace

// ---- fork -------------------------------------------------------------------
// The rows as they will be, from the rows as they are (some of which the call
// replaces too), then written over them: by a second launch, or for small tables
// behind a barrier of one workgroup.
// Entry w of row b as it will be, counting both pages; false: the row is left alone.
__device__ __forceinline__ bool forked_entry(const PagesParams& a, int b, int w, int& id,
                                             int& len) {
  const int p = a.rows[b];
  if (p == b) return false;
  const int64_t x = (int64_t)b * a.tab.width + w;
  const int old = a.tab.pages[x];
  if (w < pages_of(a.tab.seq_lens[b], a.page_size) && is_page(old, a.num_pages))
    atomicAdd(&a.refs[old], -1);
  id = -1;
  len = 0;
  if ((unsigned)p >= (unsigned)a.tab.batch) return true;
  len = a.tab.seq_lens[p];
  if (w >= pages_of(len, a.page_size)) return true;
  id = a.tab.pages[(int64_t)p * a.tab.width + w];
  if (is_page(id, a.num_pages)) atomicAdd(&a.refs[id], 1);
  return true;
}

__global__ void __launch_bounds__(256) fork_rows_kernel(PagesParams a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= (int64_t)a.tab.batch * a.tab.width) return;
  const int b = (int)(x / a.tab.width), w = (int)(x % a.tab.width);
  int id, len;
  if (!forked_entry(a, b, w, id, len)) return;
  a.ws[x] = id;
  if (w == 0) a.ws[(int64_t)a.tab.batch * a.tab.width + b] = len;
}
__global__ void __launch_bounds__(256) fork_store_kernel(PagesParams a) {
  const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (x >= (int64_t)a.tab.batch * a.tab.width) return;
  const int b = (int)(x / a.tab.width);
  if (a.rows[b] == b) return;
  a.tab.pages[x] = a.ws[x];
  if (x % a.tab.width == 0) a.tab.seq_lens[b] = a.ws[(int64_t)a.tab.batch * a.tab.width + b];
}

// Table entries up to which one workgroup does both, a thread's entries in registers.
constexpr int kForkEach = 8, kForkSmall = kForkEach * kScan;

__global__ void __launch_bounds__(kScan) fork_small_kernel(PagesParams a) {
  const unsigned n = a.tab.batch * a.tab.width, width = a.tab.width;
  int id[kForkEach], len[kForkEach];
  bool changed[kForkEach];
#pragma unroll
  for (int i = 0; i < kForkEach; ++i) {
    const unsigned x = threadIdx.x + i * kScan;
    changed[i] = x < n && forked_entry(a, x / width, x % width, id[i], len[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kForkEach; ++i) {
    const unsigned x = threadIdx.x + i * kScan;
    if (!changed[i]) continue;
    a.tab.pages[x] = id[i];
    if (x % width == 0) a.tab.seq_lens[x / width] = len[i];
  }
}

// ---- reserve ----------------------------------------------------------------
// Workspace: [free pages in order: num_pages][writers: num_pages][first writer:
// num_pages][per row: first request: batch][requests of all rows that free pages
// were found for: 1].
namespace {
struct ReserveRow {
  int cur, want, have, need, last;  // last: the part-full page to be copied, or -1
  __device__ __forceinline__ void none() { cur = want = have = need = 0, last = -1; }
  __device__ __forceinline__ void init(const PagesParams& a, int b, bool shared = true) {
    cur = max(a.tab.seq_lens[b], 0);
    want = a.rows[b];
    have = pages_of(cur, a.page_size);
    need = pages_of(want, a.page_size);
    last = -1;
    if (shared && grows(a) && cur % a.page_size != 0) {
      const int id = a.tab.pages[(int64_t)b * a.tab.width + cur / a.page_size];
      if (is_page(id, a.num_pages) && a.refs[id] > 1) last = id;
    }
  }
  __device__ __forceinline__ bool grows(const PagesParams& a) const {
    return want > cur && need <= a.tab.width;
  }
};
}  // namespace

// Row b's share of the `found` free pages from request k on, of which `copy` is for
// its last page `old`; lanes that share the row (1 or 64).
template <int LANES>
__device__ __forceinline__ void reserve_store_row(const PagesParams& a, int b, const ReserveRow& r,
                                                  int old, int k, int found) {
  const int lane = LANES > 1 ? threadIdx.x & 63 : 0;
  const int* const free = a.ws;
  int* const row = a.tab.pages + (int64_t)b * a.tab.width;
  const int copy = old >= 0;
  int granted = 1, moved = -1;
  if (r.want > r.cur) {
    granted = r.need <= a.tab.width && (int64_t)k + copy + r.need - r.have <= found;
    if (granted) {
      if (copy) moved = free[k];
      for (int i = lane; i < r.need - r.have; i += LANES) {
        const int id = free[k + copy + i];
        row[r.have + i] = id;
        a.refs[id] = 1;
      }
    }
  }
  if (lane != 0) return;
  if (moved >= 0) {
    row[r.cur / a.page_size] = moved;
    a.refs[moved] = 1;
    atomicAdd(&a.refs[old], -1);
  }
  a.src[b] = moved >= 0 ? old : -1;
  a.dst[b] = moved;
  a.granted[b] = granted;
  if (granted && r.want > r.cur) a.tab.seq_lens[b] = r.want;
}

// STORE: up to kScan rows, a thread's kept in registers and stored here too; else the
// rows are read again where they are needed and stored by a launch of their own.
template <bool STORE>
__global__ void __launch_bounds__(kScan) reserve_order_kernel(PagesParams a) {
  __shared__ int lds[kScan / 64];
  int G4_LDS* sh = (int G4_LDS*)lds;
  const int tid = threadIdx.x, n = a.num_pages, batch = a.tab.batch;
  int* const free = a.ws;
  int* const writers = free + n;
  int* const first = writers + n;
  int* const begin = first + n;
  ReserveRow mine;
  if (tid < batch) mine.init(a, tid);
  else mine.none();
  const auto row = [&](int b) {
    if (STORE || b == tid) return mine;
    ReserveRow r;
    r.init(a, b);
    return r;
  };
  // rows that write into the same shared page
  bool any = false;
  for (int b = tid; b < batch; b += kScan) {
    const int last = row(b).last;
    if (last >= 0) writers[last] = 0, first[last] = 0x7fffffff, any = true;
  }
  any = __syncthreads_or(any);
  if (any) {
    for (int b = tid; b < batch; b += kScan) {
      const int last = row(b).last;
      if (last >= 0) atomicAdd(&writers[last], 1), atomicMin(&first[last], b);
    }
    __syncthreads();
  }
  // requests in the order of the rows
  int64_t asked = 0;
  int my_old = -1, my_begin = 0;
  for (int b0 = 0; b0 < batch; b0 += kScan) {
    const int b = b0 + tid;
    int x = 0, old = -1;
    if (b < batch) {
      const ReserveRow r = row(b);
      if (r.grows(a)) x = r.need - r.have;
      if (r.last >= 0) {
        const int held = __hip_atomic_load(&writers[r.last], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
        const int lead = __hip_atomic_load(&first[r.last], __ATOMIC_RELAXED,
                                           __HIP_MEMORY_SCOPE_AGENT);
        if (held < a.refs[r.last] || lead != b) old = r.last, ++x;
      }
    }
    int total;
    const int incl = block_scan<kScan>(x, sh, total);
    // (a sum past the pool is as good as one past it by one)
    my_begin = (int)min(asked + incl - x, (int64_t)n + 1);
    my_old = old;
    if (!STORE && b < batch) a.src[b] = old, begin[b] = my_begin;
    asked += total;
  }
  // the lowest free pages, as many as were asked for
  const int want = (int)min(asked, (int64_t)n);
  int found = 0;
  for (int p0 = 0; p0 < n && found < want; p0 += kRun * kScan) {
    PageStep step;
    const unsigned bits = step.init(p0, n, a.refs, [](int ref) { return ref == 0; });
    const WaveSums sums(wave_counts(bits, 0), sh);
    step.each(bits, found + sums.before_x, [&](int rank, int p) { free[rank] = p; });
    found += sums.x;
  }
  if constexpr (STORE) {
    __syncthreads();
    if (tid < batch) reserve_store_row<1>(a, tid, mine, my_old, my_begin, found);
  } else if (tid == 0) {
    begin[batch] = found;
  }
}

// One wave per row.
__global__ void __launch_bounds__(256) reserve_store_kernel(PagesParams a) {
  const int b = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= a.tab.batch) return;
  const int* const begin = a.ws + 3 * (int64_t)a.num_pages;
  ReserveRow r;
  r.init(a, b, /*shared=*/false);
  reserve_store_row<64>(a, b, r, a.src[b], begin[b], begin[a.tab.batch]);
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
  const auto in_use = [](int ref) { return ref > 0; };
  int count = 0;
  PageStep step;
  unsigned used = 0;  // (a pool of one step is read once)
  for (int p0 = 0; p0 < n; p0 += kRun * kScan) {
    used = step.init(p0, n, a.refs, in_use);
    count += WaveSums(wave_counts(used, 0), sh).x;
  }
  // moves and holes in order
  int moves = 0, holes = 0;
  for (int p0 = 0; p0 < n; p0 += kRun * kScan) {
    if (n > kRun * kScan) used = step.init(p0, n, a.refs, in_use);
    unsigned past = 0;  // pages at or past the count
#pragma unroll
    for (int e = 0; e < kRun; ++e) past |= (unsigned)(step.at(e) >= count) << e;
    const unsigned move = used & past, hole = step.there & ~used & ~past;
    const WaveSums sums(wave_counts(move, hole), sh);
#pragma unroll
    for (int e = 0; e < kRun; ++e)
      if (step.there & past & ~used & (1u << e)) to[step.at(e)] = step.at(e);
    step.each(move, moves + sums.before_x, [&](int rank, int p) { a.src[rank] = p; });
    step.each(hole, holes + sums.before_y, [&](int rank, int p) { a.dst[rank] = p; });
    moves += sums.x;
    holes += sums.y;
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
// One workgroup per (pair, K or V, 16 KB of the page): a page's heads lie one
// after the other, so that is one run of bytes.  Bound by HBM: 3700 pages of 2 x 128 KB
// 374 us, 5.2 TB/s read and written, as a plain copy of as much; with 32 KB a
// workgroup 522, through the caches 390.
constexpr int kCopyChunk = 16384;

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
    if (first + i * 256 < end) x[i] = __builtin_nontemporal_load(from + first + i * 256);
#pragma unroll
  for (int i = 0; i < kCopyChunk / 4096; ++i)
    if (first + i * 256 < end) __builtin_nontemporal_store(x[i], to + first + i * 256);
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
  if ((int64_t)a.tab.batch * a.tab.width <= kForkSmall) {
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kScan), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(fork_rows_kernel, dim3(entry_blocks(a)), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fork_store_kernel, dim3(entry_blocks(a)), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_pages_reserve(const PagesParams& a, hipStream_t stream) {
  if (a.tab.batch <= kScan) {
    hipLaunchKernelGGL(reserve_order_kernel<true>, dim3(1), dim3(kScan), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(reserve_order_kernel<false>, dim3(1), dim3(kScan), 0, stream, a);
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

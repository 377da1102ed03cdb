// The paged cache held in 8 bits: shared device helpers, parameters, launchers.
#pragma once

#include "g4_kernels.h"

namespace g4 {

constexpr int kCacheBlock = G4_CACHE_BLOCK;  // tokens that share a scale
constexpr int kScaleFloor = -64;             // exponent of the smallest scale
constexpr float kE4m3Max = 448.f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// 2^e for -126 <= e <= 127.
__host__ __device__ __forceinline__ float pow2f(int e) {
  return __builtin_bit_cast(float, (e + 127) << 23);
}

// Exponent of the smallest power of two s with amax / s <= 448 = 1.75 x 2^8,
// from amax's bf16 bits (finite, no sign): exact, as it only compares bits.
__device__ __forceinline__ int scale_exponent(int amax) {
  return max((amax >> 7) - 127 - 8 + ((amax & 127) > 96), kScaleFloor);
}

// Two bf16 of the e4m3 pair in the low (HI false) or high half of w, times the
// power of two s: exact, and one instruction per pair.
template <bool HI>
__device__ __forceinline__ uint32_t e4m3_pair(uint32_t w, float s) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, s, HI));
}

// x to [-448, 448], NaN to 0.
__device__ __forceinline__ float e4m3_range(float x) {
  return x == x ? fminf(fmaxf(x, -kE4m3Max), kE4m3Max) : 0.f;
}

// Four e4m3 of four floats, to nearest, ties to even.
__device__ __forceinline__ uint32_t e4m3_quad(float a, float b, float c, float d) {
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(a), e4m3_range(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(e4m3_range(c), e4m3_range(d), w, true);
}

// The sequence that slot x of a launch falls to, where sequence s takes the
// slots from cu[s] / 32 + per_seq s on: the largest s with that <= x.  A wave
// looks at 64 sequences at a time, so 64 need one load and 4096 two (a binary
// search is a chain of 6 and 12).  Uniform; every lane calls it.
__device__ __forceinline__ int find_sequence(const int* cu, int batch, int x, int per_seq) {
  const int lane = __lane_id();
  int lo = 0, n = batch;
  while (n > 1) {
    const int step = (n + 63) / 64;
    const int i = lane * step;
    const bool before = i < n && cu[lo + i] / 32 + per_seq * (lo + i) <= x;
    const int k = max(__popcll(__ballot(before)) - 1, 0);
    lo += k * step;
    n = min(step, n - k * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

// Sequence s's first row, the row past its last, and its length; up to 64 sequences in
// one latency, with find_sequence's loads.  Uniform; every lane calls it.
struct SequenceOf {
  int s, row0, end, len;
  __device__ __forceinline__ SequenceOf(const int* cu, const int* lens, int batch, int x,
                                        int per_seq) {
    if (batch <= 64) {
      const int i = min((int)__lane_id(), batch - 1);
      const int c0 = cu[i], c1 = cu[i + 1], n = lens[i];
      const bool before = (int)__lane_id() < batch && c0 / 32 + per_seq * i <= x;
      s = __builtin_amdgcn_readfirstlane(max(__popcll(__ballot(before)) - 1, 0));
      row0 = __builtin_amdgcn_readlane(c0, s);
      end = __builtin_amdgcn_readlane(c1, s);
      len = __builtin_amdgcn_readlane(n, s);
      return;
    }
    s = find_sequence(cu, batch, x, per_seq);
    row0 = cu[s];
    end = cu[s + 1];
    len = lens[s];
  }
};

// The page that holds token t of sequence s, or -1.
__device__ __forceinline__ int page_of(const g4_page_table& tab, const g4_paged_cache& c, int s,
                                       int t) {
  const int w = t / c.page_size;
  if (t < 0 || w >= tab.width) return -1;
  const int id = tab.pages[(int64_t)s * tab.width + w];
  return (unsigned)id < (unsigned)c.num_pages ? id : -1;
}

struct AppendParams {
  g4_paged_cache c;
  g4_page_table tab;
  const int* cu;
  int64_t total;
  const __bf16* in[2];  // K, V
  g4_layout lay[2];
};
hipError_t launch_cache_append(const AppendParams& a, hipStream_t stream);

struct GatherParams {
  g4_paged_cache c;
  g4_page_table tab;
  const int* cu;
  int64_t total;
  __bf16* out[2];
  g4_layout lay[2];
  // For attention of the queries cu_q (null: every token): of each sequence only what
  // they can see (VisibleRows), and K of a token without a page as NaN.
  const int* cu_q;
  int max_k, window, sinks;
};
hipError_t launch_cache_gather(const GatherParams& a, hipStream_t stream);

// The tokens that nq last queries of a sequence of len tokens can see, closed up:
// rows 0 .. sinks - 1 are the sinks, then row x is token x + shift.  Distances
// between queries and the window's keys stay what they were.
struct VisibleRows {
  int shift, n;
  __device__ __forceinline__ void init(int len, int nq, int window, int sinks) {
    const int lo = window > 0 ? max(len - nq - window + 1, 0) : 0;
    shift = max(lo - sinks, 0);
    n = len - shift;
  }
};

// Cumulative lengths of the closed-up sequences and (from cu_q[0] on) of the queries,
// both within their buffers whatever the lengths on the device are.
struct ExpandParams {
  g4_page_table tab;
  const int* cu_q;
  int64_t total_q;
  int max_q, max_k, window, sinks;
  int most_k;  // rows of a sequence at most
  int *out_q, *out_k;  // (batch + 1) each
};
hipError_t launch_cache_expand_lengths(const ExpandParams& a, hipStream_t stream);

// Attention of new tokens over the cached ones.
struct CacheAttnParams {
  g4_paged_cache c;
  g4_page_table tab;
  const int* cu_q;
  int64_t total_q;
  int num_q_heads, max_q, max_k, window, sinks;
  const __bf16* q;
  __bf16* o;
  float* lse;
  g4_layout ql, ol;
  // Set by the launcher (g4_cache_attn.hip): workgroups at most, groups and queries of
  // a set, tiles that a workgroup takes at once, whether it is the wide kernel's,
  // (sequence, set, KV head) segments at most; the parts' heads, and their sums of the
  // segments that several parts share.
  int parts, set_groups, set_queries, step_tiles, wide;
  int64_t segments;
  struct PartHead* heads;
  float* part;
};
size_t cache_part_bytes(CacheAttnParams a);
hipError_t launch_cache_attn(CacheAttnParams a, void* ws, hipStream_t stream);

// A call on the tables; what a call does not use is null or 0.
struct PagesParams {
  g4_page_table tab;
  int* refs;
  int num_pages, page_size;
  const int* rows;  // parents, new_lens or keep_lens (batch)
  int window, sinks;
  int *src, *dst, *granted;
  int* ws;
};
size_t pages_workspace_bytes(int64_t num_pages, int64_t batch, int64_t width);
hipError_t launch_pages_fork(const PagesParams& a, hipStream_t stream);
hipError_t launch_pages_reserve(const PagesParams& a, hipStream_t stream);
hipError_t launch_pages_release(const PagesParams& a, hipStream_t stream);
hipError_t launch_pages_compact(const PagesParams& a, hipStream_t stream);

struct CopyParams {
  g4_paged_cache c;
  const int *src, *dst;
};
hipError_t launch_pages_copy(const CopyParams& a, int count, hipStream_t stream);

}  // namespace g4

// Storing into, reading back and copying the pages of the 8-bit cache.
#include "g4_cache.h"

namespace g4 {

// ---------------------------------------------------------------------------
// Append.  One workgroup per (32-token block of a sequence that receives new
// tokens, head, K or V): it holds the block's new rows in registers, forms their
// largest finite magnitude, from it and the block's own scale the new scale,
// rounds the block's earlier tokens again if the scale grew, and writes the new
// rows.  Scales are powers of two: an e4m3 value divided by one keeps its bits
// but where it falls below the type's normal range, so a growing scale costs a
// block's earlier tokens next to nothing, and what a block holds does not
// depend on how its tokens were dealt to the calls but there.  Bound by HBM: a
// row is read once (2 bytes an element) and written once (1 byte): 19500 tokens of 16
// heads of 256 in 98 us, 4.9 TB/s (with the heads' rows apart in the grid 109).  One
// token a sequence is a chain of latencies: 64 sequences 5.6 us (6.7 with the table
// read before the rows, and a sequence's length after its number).
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) append_kernel(AppendParams a) {
  constexpr int kLanes = D / 8;              // lanes of a row, 16 bytes each
  constexpr int kRows = 256 / kLanes;        // rows of a pass
  constexpr int kPasses = kCacheBlock / kRows;
  __shared__ int wave_max[4];
  const g4_paged_cache& c = a.c;
  // heads first: neighbouring workgroups read neighbouring runs of the same rows
  const int head = blockIdx.x % c.num_kv_heads, slot = blockIdx.x / c.num_kv_heads;
  const int which = blockIdx.y;
  const SequenceOf seq(a.cu, a.tab.seq_lens, a.tab.batch, slot, 2);
  const int s = seq.s, row0 = seq.row0, n = seq.end - row0, len = seq.len;
  const int first = len - n;  // position of the first new token
  const int begin = max(first, 0);
  const int rel = slot - (row0 / 32 + 2 * s);
  if (n <= 0 || rel < 0 || len <= begin) return;
  const int64_t t0 = (int64_t)(begin / kCacheBlock + rel) * kCacheBlock;
  if (t0 >= len) return;
  const int lo = max(begin - (int)t0, 0), hi = min(len - (int)t0, kCacheBlock);

  const int tid = threadIdx.x, lane = tid & 63, sub = tid / kLanes, col = tid % kLanes;
  const __bf16* in = a.in[which] + (int64_t)head * a.lay[which].head_stride + col * 8;
  u32x4 x[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kRows + sub;
    const int64_t row = row0 + t0 + r - first;
    x[i] = u32x4{};
    if (r >= lo && r < hi && row >= 0 && row < a.total)
      x[i] = *(const u32x4*)(in + row * a.lay[which].token_stride);
  }
  const int page = page_of(a.tab, c, s, (int)t0);  // (after the rows' loads: they overlap)
  if (page < 0) return;
  // largest finite magnitude: bf16 bits without the sign compare as numbers do
  int most = 0;
#pragma unroll
  for (int i = 0; i < kPasses; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int u = x[i][e] & 0x7fff, v = (x[i][e] >> 16) & 0x7fff;
      most = max(most, max(u < 0x7f80 ? u : 0, v < 0x7f80 ? v : 0));
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  if (lane == 0) wave_max[tid >> 6] = most;
  float* const scale_at = (which ? c.v_scale : c.k_scale) +
                          ((int64_t)page * c.num_kv_heads + head) * (c.page_size / kCacheBlock) +
                          t0 % c.page_size / kCacheBlock;
  const float held = lo > 0 ? *scale_at : 0.f;
  __syncthreads();
  most = max(max(wave_max[0], wave_max[1]), max(wave_max[2], wave_max[3]));
  const float scale = fmaxf(pow2f(scale_exponent(most)), held);
  const float inv = 1.f / scale;

  uint8_t* const out = (uint8_t*)(which ? c.v : c.k) +
                       (((int64_t)page * c.num_kv_heads + head) * c.page_size +
                        t0 % c.page_size) * D + col * 8;
  if (lo > 0 && scale > held) {
    const float ratio = held * inv;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int r = i * kRows + sub;
      if (r >= lo) continue;
      u32x2* const p = (u32x2*)(out + r * D);
      u32x2 w = *p;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const f32x2 y = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], false);
        const f32x2 z = __builtin_amdgcn_cvt_pk_f32_fp8(w[e], true);
        w[e] = e4m3_quad(y[0] * ratio, y[1] * ratio, z[0] * ratio, z[1] * ratio);
      }
      *p = w;
    }
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = i * kRows + sub;
    if (r < lo || r >= hi) continue;
    u32x2 w;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const uint32_t p = x[i][2 * e], q = x[i][2 * e + 1];
      w[e] = e4m3_quad(__uint_as_float(p << 16) * inv, __uint_as_float(p & 0xffff0000u) * inv,
                       __uint_as_float(q << 16) * inv, __uint_as_float(q & 0xffff0000u) * inv);
    }
    *(u32x2*)(out + r * D) = w;
  }
  if (tid == 0) *scale_at = scale;
}

hipError_t launch_cache_append(const AppendParams& a, hipStream_t stream) {
  // a sequence's n new tokens touch at most n / 32 + 2 blocks
  const int64_t slots = a.total / kCacheBlock + 2 * (int64_t)a.tab.batch;
  const dim3 grid((unsigned)(slots * a.c.num_kv_heads), 2);
  if (a.c.head_dim == 256)
    hipLaunchKernelGGL(append_kernel<256>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(append_kernel<512>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Gather.  One workgroup per (32 output rows of a sequence, head, K or V).  Bound by
// HBM: 12500 tokens of 4 heads of 512 (51 MB read, 102 written) in 28 us, 5.5 TB/s.
// ---------------------------------------------------------------------------
template <int D>
__global__ void __launch_bounds__(256) gather_kernel(GatherParams a) {
  constexpr int kLanes = D / 8;
  constexpr int kRows = 256 / kLanes;
  const g4_paged_cache& c = a.c;
  const int head = blockIdx.x % c.num_kv_heads, slot = blockIdx.x / c.num_kv_heads;
  const int which = blockIdx.y;
  const SequenceOf seq(a.cu, a.tab.seq_lens, a.tab.batch, slot, 1);
  const int s = seq.s, row0 = seq.row0, n = seq.end - row0;
  const int rel = slot - (row0 / 32 + s);
  if (rel < 0 || rel >= (n + 31) / 32) return;
  int len = seq.len, shift = 0;
  if (a.cu_q != nullptr) {
    VisibleRows v;
    len = min(max(len, 0), a.max_k);
    v.init(len, a.cu_q[s + 1] - a.cu_q[s], a.window, a.sinks);
    shift = v.shift;
  }
  const int tid = threadIdx.x, sub = tid / kLanes, col = tid % kLanes;
  const uint8_t* in = (const uint8_t*)(which ? c.v : c.k) + col * 8;
  const float* scales = which ? c.v_scale : c.k_scale;
  __bf16* out = a.out[which] + (int64_t)head * a.lay[which].head_stride + col * 8;
#pragma unroll
  for (int i = 0; i < kCacheBlock / kRows; ++i) {
    const int x = rel * 32 + i * kRows + sub;
    const int64_t row = (int64_t)row0 + x;
    if (x >= n || row < 0 || row >= a.total) continue;
    const int t = a.cu_q != nullptr && x >= a.sinks ? x + shift : x;
    const int page = t < len ? page_of(a.tab, c, s, t) : -1;
    const uint32_t none = a.cu_q != nullptr && which == 0 ? 0x7fc07fc0u : 0u;  // NaN or 0
    u32x4 y = {none, none, none, none};
    if (page >= 0) {
      const int64_t ph = (int64_t)page * c.num_kv_heads + head;
      const int at = t % c.page_size;
      const u32x2 w = *(const u32x2*)(in + (ph * c.page_size + at) * D);
      const float sc = scales[ph * (c.page_size / kCacheBlock) + at / kCacheBlock];
      y = u32x4{e4m3_pair<false>(w[0], sc), e4m3_pair<true>(w[0], sc),
                e4m3_pair<false>(w[1], sc), e4m3_pair<true>(w[1], sc)};
    }
    *(u32x4*)(out + row * a.lay[which].token_stride) = y;
  }
}

// One workgroup: prefix sums over the sequences.
__global__ void __launch_bounds__(256) expand_lengths_kernel(ExpandParams a) {
  __shared__ int64_t lds[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t first_q = min(max((int64_t)a.cu_q[0], (int64_t)0), a.total_q);
  int64_t base_q = first_q, base_k = 0;
  for (int s0 = 0; s0 < a.tab.batch; s0 += 256) {
    const int s = s0 + tid;
    int64_t q = 0, k = 0;
    if (s < a.tab.batch) {
      const int nq = (int)min(max((int64_t)a.cu_q[s + 1] - a.cu_q[s], (int64_t)0), (int64_t)a.max_q);
      VisibleRows v;
      v.init(min(max(a.tab.seq_lens[s], 0), a.max_k), nq, a.window, a.sinks);
      q = nq;
      k = min(v.n, a.most_k);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t x = __shfl_up(q, o, 64), y = __shfl_up(k, o, 64);
      if (lane >= o) q += x, k += y;
    }
    __syncthreads();
    if (lane == 63) lds[0][wave] = q, lds[1][wave] = k;
    __syncthreads();
    int64_t before_q = base_q, before_k = base_k;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < wave) before_q += lds[0][w], before_k += lds[1][w];
      base_q += lds[0][w];
      base_k += lds[1][w];
    }
    if (s < a.tab.batch) {
      a.out_q[s + 1] = (int)min(before_q + q, a.total_q);
      a.out_k[s + 1] = (int)(before_k + k);
    }
  }
  if (tid == 0) a.out_q[0] = (int)first_q, a.out_k[0] = 0;
}

hipError_t launch_cache_expand_lengths(const ExpandParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(expand_lengths_kernel, dim3(1), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_cache_gather(const GatherParams& a, hipStream_t stream) {
  const int64_t slots = a.total / 32 + a.tab.batch;
  const dim3 grid((unsigned)(slots * a.c.num_kv_heads), 2);
  if (a.c.head_dim == 256)
    hipLaunchKernelGGL(gather_kernel<256>, grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(gather_kernel<512>, grid, dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace g4

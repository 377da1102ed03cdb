// Backward of the sinks: the keys that a sliding window leaves visible at the
// beginning of each sequence.
//
// The window's part of the gradients comes from the text kernels: with the LSE
// and delta of the whole row, P = exp(S - LSE) and dS = P (dP - delta) of a pair
// do not depend on which other pairs the row has.  What is left, for sequences
// longer than the window:
//   dK, dV of the sinks, over every query of the sequence (written anew, so that
//   each is one fp32 sum rounded once), and
//   their dS behind the window, stored as bf16 tiles that the dQ stage adds to the
//   window's as one more key tile (without stored dS that stage recomputes them).
// A workgroup takes a chunk of a sequence's queries and one KV head; its waves
// take 32 rows of one query head at a time: S = Q K^T and dP = dO V^T with keys
// along lanes feed dV^T += dO^T P and dK^T += Q^T dS from registers.  The chunk's
// dK and dV go to the workspace and a second launch adds the chunks in order (no
// atomics).  Q and dO are read once more, 2 x 512 bytes a row, and 64 bytes of dS
// written: bound by HBM, which one tile a wave in flight and one workgroup a CU (128 KB
// of tiles, 256 accumulator registers) keep at 3.5 TB/s (32768 tokens 310 us; the next
// tile held in registers spilled there, 349).  Adding dQ to the stored rows here instead
// cost 4 x 512 bytes a row (558 us) and rounded it twice.
#include <algorithm>

#include "g4_kernels.h"

namespace g4 {

namespace {

constexpr int kSinkKeys = G4_MAX_SINKS;  // one 32-key block
constexpr int D = 256;
constexpr int kNC = D / 16;  // 16-deep steps of S and dP
constexpr int kNB = D / 32;  // 32-wide blocks of the head dim
constexpr int kWaves = 4;
constexpr int kRowsBytes = 32 * D * 2;            // a tile of Q or dO
constexpr int kWaveBytes = 2 * kRowsBytes;        // = 32 fp32 rows of D
constexpr int kLdsStat = kWaves * kWaveBytes;     // [wave][LSE x 32 | delta x 32] fp32
constexpr int kLdsBytes = kLdsStat + kWaves * 256;
static_assert(kLdsBytes <= 160 * 1024, "LDS budget");
static_assert(kWaveBytes == 32 * D * 4, "the sums of a wave fit its tiles");

__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// Chunks of sequence s: none where the window reaches every key.
__device__ __forceinline__ int sink_chunks(const SinkParams& a, int s) {
  const Seq q = resolve_seq(a.b.p, s);
  return q.lk > a.b.p.window && q.lq > 0 ? (q.lq + a.chunk - 1) / a.chunk : 0;
}

// Sequence s of item x where sequence j has count(j) items, x's number c among them and
// the items before them; false past the last.  Every lane of the wave calls it.
template <class Count>
__device__ __forceinline__ bool sink_item(const SinkParams& a, int x, Count count, int& s, int& c) {
  const int lane = __lane_id();
  int base = 0;
  for (int s0 = 0; s0 < a.b.p.num_seqs; s0 += 64) {
    const int n = s0 + lane < a.b.p.num_seqs ? count(s0 + lane) : 0;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    const int total = __builtin_amdgcn_readlane(incl, 63);
    if (x < base + total) {
      const int k = __popcll(__ballot(base + incl <= x));
      s = __builtin_amdgcn_readfirstlane(s0 + k);
      c = __builtin_amdgcn_readfirstlane(x - base - __shfl(incl - n, k, 64));
      return true;
    }
    base += total;
  }
  return false;
}

// Slots (the chunks of all sequences in order) before sequence s.
__device__ __forceinline__ int sink_slots_before(const SinkParams& a, int s) {
  int n = 0;
  for (int j = __lane_id(); j < s; j += 64) n += sink_chunks(a, j);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
  return __builtin_amdgcn_readfirstlane(n);
}

// x += rows . keys^T over the steps CP .. kNC - 1.
template <int CP, class RR>
__device__ __forceinline__ void sink_product(const RR& rrd, const char G4_LDS* rows,
                                             const bf16x8 (&keys)[kNC], f32x16& x) {
  if constexpr (CP < kNC) {
    x = mfma32(rrd.template read<0, 0, CP>(rows), keys[CP], x);
    sink_product<CP + 1>(rrd, rows, keys, x);
  }
}

// Byte of the 16-byte chunk c of fp32 row r in a wave's area (D * 4 bytes a row).
__device__ __forceinline__ int sum_off(int r, int c) { return r * D * 4 + (c ^ r) * 16; }

}  // namespace

__global__ void __launch_bounds__(256, 1) sinks_bwd_kernel(SinkParams sp) {
  extern __shared__ __attribute__((aligned(16))) char smem_raw[];
  char G4_LDS* const smem = (char G4_LDS*)smem_raw;
  const BwdParams& a = sp.b;
  const g4_problem& p = a.p;
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, h32 = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.num_kv_heads, slot = blockIdx.x / p.num_kv_heads;
  int s, chunk;
  if (!sink_item(sp, slot, [&](int j) { return sink_chunks(sp, j); }, s, chunk)) return;
  const Seq sq = resolve_seq(p, s);
  const int off = sq.lk - sq.lq;
  const int grp = p.num_q_heads / p.num_kv_heads;
  const int sinks = min(a.sinks, sq.lk);

  // ---- the sinks' K and V along lanes (rows past them are masked) ---------------
  bf16x8 kf[kNC], vf[kNC];
  {
    const int r = min(l32, sinks - 1);
    const __bf16* krow = a.k + tok_off(sq, s, sq.ktok, r, a.kl) + (int64_t)kvh * a.kl.head_stride;
    const __bf16* vrow = a.v + tok_off(sq, s, sq.ktok, r, a.vl) + (int64_t)kvh * a.vl.head_stride;
#pragma unroll
    for (int c = 0; c < kNC; ++c) {
      kf[c] = ld_global16(krow + 16 * c + 8 * h32);
      vf[c] = ld_global16(vrow + 16 * c + 8 * h32);
    }
  }
  RowReader<32> rrd;
  TrReader<32> trd;
  rrd.init(lane);
  trd.init(lane);

  // ---- the chunk's rows -----------------------------------------------------------
  char G4_LDS* const qt = smem + wave * kWaveBytes;
  char G4_LDS* const dot = qt + kRowsBytes;
  float G4_LDS* const stat = (float G4_LDS*)(smem + kLdsStat + wave * 256);
  TileCopier<32, 32, 1, true> qcp, docp;
  qcp.init(a.ql.token_stride, 0, lane);
  docp.init(a.dol.token_stride, 0, lane);
  f32x16 dk[kNB], dv[kNB];
#pragma unroll
  for (int b = 0; b < kNB; ++b) dk[b] = dv[b] = f32x16{};
  const int i_end = min((chunk + 1) * sp.chunk, sq.lq);
  const int tiles = (i_end - chunk * sp.chunk + 31) / 32;
  for (int t = wave; t < tiles * grp; t += kWaves) {
    const int i0 = chunk * sp.chunk + t / grp * 32, qh = kvh * grp + t % grp;
    const int nrows = min(i_end - i0, 32);
    const __bf16* qrow = a.q + tok_off(sq, s, sq.qtok, i0, a.ql) + (int64_t)qh * a.ql.head_stride;
    const __bf16* dorow =
        a.dout + tok_off(sq, s, sq.qtok, i0, a.dol) + (int64_t)qh * a.dol.head_stride;
    wait_lds();  // the previous tile's reads
    if (nrows == 32) {
      qcp.issue(qrow, qt);
      docp.issue(dorow, dot);
    } else {
      qcp.issue_clamped(qrow, 0, nrows, qt);
      docp.issue_clamped(dorow, 0, nrows, dot);
    }
    {
      // LSE and delta of the rows; a row that sees nothing has no weights
      const int64_t at = lse_off(p, sq, s, qh, i0 + min(l32, nrows - 1));
      const int64_t tok = (int64_t)qh * q_stream_tokens_dev(p) + sq.qtok + i0 + min(l32, nrows - 1);
      const float lse = a.lse[at];
      const float x = h32 ? a.delta[tok] : lse == kNegInf ? -kNegInf : lse * kLog2e;
      stat[lane] = x;
    }
    vm_wait<0>();
    wait_lds();

    const int a0 = i0 + off;
    f32x16 sc = {}, dp = {};
    sink_product<0>(rrd, qt, kf, sc);
    sink_product<0>(rrd, dot, vf, dp);
    bf16x8 pb[2], dsb[2], behind[2];  // P, dS, dS behind the window
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const f32x4 lse = *(const f32x4 G4_LDS*)(stat + 8 * r4 + 4 * h32);
      const f32x4 dl = *(const f32x4 G4_LDS*)(stat + 32 + 8 * r4 + 4 * h32);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * r4 + e, row = 8 * r4 + 4 * h32 + e;
        const bool ok = (l32 < sinks) & (l32 <= a0 + row) & (row < nrows);
        const float pr = ok ? fast_exp2(__builtin_fmaf(sc[r], kLog2e, -lse[e])) : 0.f;
        const float ds = ok ? pr * (dp[r] - dl[e]) : 0.f;
        pb[r / 8][r % 8] = (__bf16)pr;
        dsb[r / 8][r % 8] = (__bf16)ds;
        behind[r / 8][r % 8] = (__bf16)(l32 <= a0 + row - p.window ? ds : 0.f);
      }
    }
    if (a.sink_ds != nullptr && a0 + nrows - 1 >= p.window) {
      // (queries in accumulator order: a lane's 16 are one run)
      const int64_t row = (sq.packed ? sq.qtok / 32 + s : (int64_t)s * ((p.seqlen_q + 31) / 32)) +
                          i0 / 32;
      bf16x8* const out =
          (bf16x8*)(a.sink_ds + ((int64_t)qh * a.ds_rows + row) * 1024 + l32 * 32 + h32 * 16);
      out[0] = behind[0];
      out[1] = behind[1];
    }
    acc_steps<kNB>(trd, dot, pb, dv);
    acc_steps<kNB>(trd, qt, dsb, dk);
  }

  // ---- the waves' sums, key by key --------------------------------------------------
  float* const part = sp.part + ((int64_t)slot * p.num_kv_heads + kvh) * 2 * kSinkKeys * D;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    barrier_lds();
#pragma unroll
    for (int b = 0; b < kNB; ++b)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const f32x16& x = which ? dv[b] : dk[b];
        *(f32x4 G4_LDS*)(qt + sum_off(l32, 8 * b + 2 * r4 + h32)) =
            f32x4{x[4 * r4], x[4 * r4 + 1], x[4 * r4 + 2], x[4 * r4 + 3]};
      }
    barrier_lds();
    for (int r = wave; r < sinks; r += kWaves) {
      f32x4 x = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        x += *(const f32x4 G4_LDS*)(smem + w * kWaveBytes + sum_off(r, lane));
      *(f32x4*)(part + (which * kSinkKeys + r) * D + 4 * lane) = x;
    }
  }
}

// dK and dV of the sinks from the chunks' sums.  One wave per (sequence, KV head,
// K or V, sink).
__global__ void __launch_bounds__(64) sinks_sum_kernel(SinkParams sp) {
  const BwdParams& a = sp.b;
  const g4_problem& p = a.p;
  const int kvh = blockIdx.x % p.num_kv_heads;
  const int r = blockIdx.y % a.sinks, which = blockIdx.y / a.sinks;
  int s, c0;  // of the sequences longer than the window
  if (!sink_item(sp, blockIdx.x / p.num_kv_heads, [&](int j) { return sink_chunks(sp, j) > 0; }, s,
                 c0))
    return;
  const int n = sink_chunks(sp, s);
  const Seq sq = resolve_seq(p, s);
  if (r >= sq.lk) return;
  const int first = sink_slots_before(sp, s);
  const int lane = threadIdx.x;
  const int64_t pitch = (int64_t)p.num_kv_heads * 2 * kSinkKeys * D;
  const float* src = sp.part + (int64_t)first * pitch +
                     ((int64_t)kvh * 2 * kSinkKeys + which * kSinkKeys + r) * D + 4 * lane;
  f32x4 x = {};
#pragma unroll 8
  for (int c = 0; c < n; ++c) x += *(const f32x4*)(src + c * pitch);
  const g4_layout& l = which ? a.dvl : a.dkl;
  *(bf16x4*)((which ? a.dv : a.dk) + tok_off(sq, s, sq.ktok, r, l) + (int64_t)kvh * l.head_stride +
             4 * lane) = bf16x4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
}

// Queries of a chunk: one workgroup per CU for one sequence, about two for several,
// whose last chunks are short (whole training calls, us, 256 / 512 workgroups: 2500
// tokens 399 / 409, 5000 832 / 845, 20 sequences of 30000 tokens 3830 / 3780).
static int sink_chunk(const g4_problem& p) {
  const int64_t rows = q_stream_tokens(p) * p.num_kv_heads;
  const int64_t chunk = (rows / (p.num_seqs == 1 ? 256 : 512) + 31) / 32 * 32;
  return (int)std::max<int64_t>(chunk, 32);
}

// Sequences that the window does not cover at most (they have more keys than it), and
// their chunks.
static int64_t sink_sequences(const g4_problem& p) {
  return std::min<int64_t>(p.num_seqs, k_stream_tokens(p) / ((int64_t)p.window + 1));
}
static int64_t sink_slots(const g4_problem& p) {
  const int64_t longer = sink_sequences(p);
  return longer ? q_stream_tokens(p) / sink_chunk(p) + longer : 0;
}

size_t sinks_part_bytes(const g4_problem& p) {
  return (size_t)sink_slots(p) * p.num_kv_heads * 2 * kSinkKeys * D * 4;
}

// A 2 KB tile per (32-query row, query head), where dS is stored.
size_t sinks_ds_bytes(const g4_problem& p) {
  if (!ds_bytes(p)) return 0;
  int rows, cols;
  ds_geometry(p, &rows, &cols);
  return (size_t)rows * p.num_q_heads * 2048;
}

hipError_t launch_sinks_bwd(const BwdParams& b, float* part, hipStream_t stream) {
  SinkParams a{b, sink_chunk(b.p), part};
  const int64_t blocks = sink_slots(b.p) * b.p.num_kv_heads;
  if (blocks <= 0) return hipSuccess;  // no sequence is longer than the window
  static LdsAttr attr;
  hipError_t e = attr.ensure((const void*)sinks_bwd_kernel, kLdsBytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sinks_bwd_kernel, dim3((unsigned)blocks), dim3(256), kLdsBytes, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(sinks_sum_kernel, dim3((unsigned)(sink_sequences(b.p) * b.p.num_kv_heads),
                                            (unsigned)(2 * b.sinks)),
                     dim3(64), 0, stream, a);
  return hipGetLastError();
}

}  // namespace g4

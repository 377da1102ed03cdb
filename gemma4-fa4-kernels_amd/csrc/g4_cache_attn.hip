// Attention of a few new tokens over the pages of the 8-bit cache.
//
// A KV head's query rows (its query heads x the new tokens) go in groups of 16,
// the columns of a 16 x 16 x 32 matrix instruction; a group's keys are walked in
// tiles of 32, one wave per tile, K and V straight from the pages into registers:
//   S^T (32 keys x 16 rows) = K Q^T, two accumulators over the head dim;
//   O^T (D x 16 rows) += V^T P^T, D / 16 accumulators of one step each.
// A lane's 16-byte loads are 64 bytes of a key's row for four lanes (K) and 256
// bytes for sixteen (V), so the pages are read in whole lines without LDS.  Which
// head-dim element a lane holds is free as long as both operands agree: K takes
// elements 64 c + 16 h + 0..15 of row i in lane (i, h), and Q is loaded likewise; V
// takes 256 g + 16 i + 0..15, so that the 16 bytes are 16 different O^T blocks'
// row i.  e4m3 becomes bf16 exactly (block scales are powers of two, and the
// conversion applies them), Q stays bf16: the only roundings are P's to bf16 and
// the output's.
//
// The tiles of all (sequence, row group, KV head) segments, in that order, are cut
// into equal parts, one workgroup of four waves each, so that the longest sequence
// of a batch does not decide its time.  The waves of a part take every fourth tile
// of a segment and add up through LDS; a segment inside one part is finished there,
// else the parts' sums go to the workspace (slot = part + segment: along the parts
// both only grow, so no two pairs share one) and a second launch merges them.
//
// Bound by HBM for long batches (1 byte an element of K and V), by the chain of
// launch, table, page and merge latencies for short ones.
#include "g4_cache.h"

namespace g4 {

namespace {

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Value of lane l ^ 16: v_permlane16_swap with both operands x gives x with rows
// 1, 3 replaced by rows 0, 2, and x with rows 0, 2 replaced by rows 1, 3.
__device__ __forceinline__ float wave_xor16(float x) {
  const auto r =
      __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((__lane_id() & 16) ? r[0] : r[1]);
}
// Over the four lanes (i, 0..3) that hold a row's scores.
__device__ __forceinline__ float rows_max(float x) {
  x = fmaxf(x, wave_xor16(x));
  return fmaxf(x, wave_xor32(x));
}
__device__ __forceinline__ float rows_sum(float x) {
  x += wave_xor16(x);
  return x + wave_xor32(x);
}

constexpr int kTile = kCacheBlock;  // keys of a tile: one block of a page, one scale
constexpr int kWaves = 4;
constexpr int kGroupRows = 16;
// Tiles a part has at least: one for each of its waves.
constexpr int kPartTiles = kWaves;

// A sequence of the batch as the kernels see it.
struct CacheSeq {
  int q0, lq, len;  // first query row, queries, cached tokens
  __device__ __forceinline__ void init(const CacheAttnParams& a, int s) {
    q0 = a.cu_q[s];
    const int64_t end = min((int64_t)a.cu_q[s + 1], a.total_q);
    lq = q0 < 0 ? 0 : (int)max(min(end - q0, (int64_t)a.max_q), (int64_t)0);
    len = min(max(a.tab.seq_lens[s], 0), a.max_k);
  }
};

// The tiles of the queries [i0, i1] of a sequence: nsink tiles from 0 on, then
// those from tile `first`; n in all, at least one (a row that sees nothing is
// still written).
struct TileRange {
  int nsink, first, n;
  __device__ __forceinline__ void init(const CacheAttnParams& a, const CacheSeq& q, int i0,
                                       int i1) {
    const int off = q.len - q.lq;
    const int lo = a.window > 0 ? max(i0 + off - a.window + 1, 0) : 0;
    first = lo / kTile;
    nsink = min((min(a.sinks, q.len) + kTile - 1) / kTile, first);
    const int end = max(i1 + off + kTile, 0) / kTile;  // past the last query's tile
    n = max(nsink + end - first, 1);
  }
  __device__ __forceinline__ int at(int x) const { return x < nsink ? x : first + x - nsink; }
};

// Tiles of a sequence's row groups together, over all its KV heads.
__device__ __forceinline__ int64_t sequence_tiles(const CacheAttnParams& a, int s) {
  CacheSeq q;
  q.init(a, s);
  int64_t n = 0;
  for (int i = 0; i < q.lq; i += a.group_queries) {
    TileRange t;
    t.init(a, q, i, min(i + a.group_queries, q.lq) - 1);
    n += t.n;
  }
  return n * a.c.num_kv_heads;
}

// Sum of x over the workgroup (256 threads) and the sum before this thread.
__device__ __forceinline__ int64_t block_before(int64_t x, int64_t G4_LDS* lds, int64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t incl = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t y = __shfl_up(incl, o, 64);
    if (lane >= o) incl += y;
  }
  barrier_lds();
  if (lane == 63) lds[wave] = incl;
  barrier_lds();
  int64_t before = incl - x;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int64_t y = lds[w];
    before += w < wave ? y : 0;
    total += y;
  }
  return before;
}

// Tiles of the whole batch; every thread of the workgroup (256) calls it.
__device__ __forceinline__ int64_t batch_tiles(const CacheAttnParams& a, int64_t G4_LDS* lds) {
  int64_t sum = 0;
  for (int s0 = 0; s0 < a.tab.batch; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    int64_t total;
    block_before(s < a.tab.batch ? sequence_tiles(a, s) : 0, lds, total);
    sum += total;
  }
  return sum;
}

// The parts that a batch of `tiles` tiles is cut into, and the part of tile x: part
// w holds the tiles from tiles w / parts on.
__device__ __forceinline__ int64_t part_count(const CacheAttnParams& a, int64_t tiles) {
  return max(min((int64_t)a.parts, tiles / kPartTiles), (int64_t)1);
}
__device__ __forceinline__ int64_t part_of(int64_t x, int64_t parts, int64_t tiles) {
  return ((x + 1) * parts - 1) / tiles;
}

}  // namespace

template <int D>
struct CacheWave {
  static constexpr int kNC = D / 64;   // 16-byte chunks of a lane's K row
  static constexpr int kNG = D / 256;  // 16-byte chunks of a lane's V row
  static constexpr int kNB = D / 16;   // O^T blocks

  u32x4 k[2][kNC];   // keys i and 16 + i of the tile
  u32x4 v[8][kNG];   // keys 16 (j >> 2) + 4 h + (j & 3)
  float ks, vs;      // the tile's scales
  bf16x8 q[2 * kNC];
  f32x4 o[kNB];      // block 16 g + e: element r is head dim 256 g + 64 h + 16 r + e
  float m, l;        // per row, in every lane (i, *): l holds this lane's share

  __device__ __forceinline__ void load_k(const CacheAttnParams& a, int64_t page_head, int blk,
                                         int i, int h) {
    const uint8_t* p = (const uint8_t*)a.c.k +
                       (page_head * a.c.page_size + blk * kTile + i) * D + 16 * h;
    ks = a.c.k_scale[page_head * (a.c.page_size / kTile) + blk];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int c = 0; c < kNC; ++c) k[u][c] = *(const u32x4*)(p + u * 16 * D + c * 64);
  }
  __device__ __forceinline__ void load_v(const CacheAttnParams& a, int64_t page_head, int blk,
                                         int i, int h) {
    const uint8_t* p = (const uint8_t*)a.c.v +
                       (page_head * a.c.page_size + blk * kTile + 4 * h) * D + 16 * i;
    vs = a.c.v_scale[page_head * (a.c.page_size / kTile) + blk];
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int g = 0; g < kNG; ++g)
        v[j][g] = *(const u32x4*)(p + (16 * (j >> 2) + (j & 3)) * D + g * 256);
  }

  __device__ __forceinline__ void scores(f32x4 (&s)[2]) const {
    s[0] = s[1] = f32x4{};
#pragma unroll
    for (int c = 0; c < kNC; ++c)
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const u32x4 w = {e4m3_pair<false>(k[u][c][2 * x], ks), e4m3_pair<true>(k[u][c][2 * x], ks),
                           e4m3_pair<false>(k[u][c][2 * x + 1], ks),
                           e4m3_pair<true>(k[u][c][2 * x + 1], ks)};
          s[u] = mfma16(__builtin_bit_cast(bf16x8, w), q[2 * c + x], s[u]);
        }
  }

  // Masks s (positions j of tile kb0; a_row: this lane's row's position, -1 for
  // none) unless `full`, then the online softmax; P^T in `pb`.
  __device__ __forceinline__ void softmax(const CacheAttnParams& a, f32x4 (&s)[2], int kb0, int h,
                                          int a_row, bool full, bool page, bf16x8& pb) {
    if (!full) {
      const int lo = a.window > 0 ? a_row - a.window : -0x7fffffff;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = kb0 + 16 * u + 4 * h + r;
          const bool ok = (j <= a_row) & ((j > lo) | (j < a.sinks));
          s[u][r] = ok ? (page ? s[u][r] : __builtin_nanf("")) : kNegInf;
        }
    }
    float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                     fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mx = rows_max(mx) * kLog2e;
    // The maximum moves only when exceeded by more than 2^8 (P <= 2^8 meanwhile, exact
    // in fp32 and in bf16 range), so O is rescaled on few tiles.
    const float m_new = mx > m + 8.f ? mx : m;
    const float m_use = m_new == kNegInf ? 0.f : m_new;
    const float alpha = fast_exp2(m - m_use);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float p = fast_exp2(__builtin_fmaf(s[u][r], kLog2e, -m_use));
        sum += p;
        pb[4 * u + r] = (__bf16)p;
      }
    l = l * alpha + sum;
    m = m_new;
    if (__ballot(alpha != 1.f)) {
#pragma unroll
      for (int b = 0; b < kNB; ++b) o[b] *= alpha;
    }
  }

  // O^T += V^T P^T.  Two keys' pairs of neighbouring head-dim elements become two
  // elements' pairs of neighbouring keys by a byte permutation.
  __device__ __forceinline__ void add_values(bf16x8 pb) {
#pragma unroll
    for (int g = 0; g < kNG; ++g)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t lo[8], hi[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lo[j] = e4m3_pair<false>(v[j][g][w], vs);
          hi[j] = e4m3_pair<true>(v[j][g][w], vs);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t* x = e < 2 ? lo : hi;
          const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
          u32x4 f;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            f[j] = __builtin_amdgcn_perm(x[2 * j + 1], x[2 * j], sel);
          f32x4& acc = o[16 * g + 4 * w + e];
          acc = mfma16(__builtin_bit_cast(bf16x8, f), pb, acc);
        }
      }
  }
};

template <int D>
__global__ void __launch_bounds__(256, D == 256 ? 2 : 1) cache_attn_kernel(CacheAttnParams a) {
  using W = CacheWave<D>;
  constexpr int kPitch = D + 4;  // floats of a row in LDS
  __shared__ __attribute__((aligned(16))) float rows[kWaves][kGroupRows][kPitch];
  __shared__ float state[2][kWaves][kGroupRows];
  __shared__ int64_t scan[kWaves];
  __shared__ int64_t found[2];
  int64_t G4_LDS* sh = (int64_t G4_LDS*)scan;
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = a.c.num_kv_heads;

  // ---- this part's tiles [lo, hi) and the sequence of the first --------------
  const int64_t tiles = batch_tiles(a, sh);
  const int64_t parts = part_count(a, tiles);
  const int64_t part = blockIdx.x;
  if (part >= parts || tiles == 0) return;
  int64_t lo = tiles * part / parts;
  const int64_t hi = tiles * (part + 1) / parts;
  int64_t base = 0;
  int s = 0;
  for (int s0 = 0; s0 < a.tab.batch; s0 += 256) {
    const int sx = s0 + tid;
    const int64_t n = sx < a.tab.batch ? sequence_tiles(a, sx) : 0;
    int64_t total;
    const int64_t before = base + block_before(n, sh, total);
    if (before <= lo && lo < before + n) found[0] = sx, found[1] = before;
    base += total;
    if (base > lo) break;
  }
  __syncthreads();
  s = __builtin_amdgcn_readfirstlane((int)found[0]);
  int64_t seg0 = found[1];  // first tile of the segment at hand

  CacheSeq sq;
  sq.init(a, s);
  int group = 0, kvh = 0;
  // the segment of tile lo
  TileRange range;
  for (;; ++group) {
    range.init(a, sq, group * a.group_queries,
               min((group + 1) * a.group_queries, sq.lq) - 1);
    const int64_t n = (int64_t)range.n * hkv;
    if (lo < seg0 + n) break;
    seg0 += n;
  }
  kvh = (int)((lo - seg0) / range.n);
  seg0 += (int64_t)kvh * range.n;

  const int grp = a.num_q_heads / hkv, gsh = __builtin_ctz(grp);
  while (true) {
    // ---- the part's share [x0, x1) of the segment's tiles ---------------------
    const int x0 = (int)(lo - seg0), x1 = (int)min(hi - seg0, (int64_t)range.n);
    const int q_first = group * a.group_queries;
    const int q_last = min(q_first + a.group_queries, sq.lq) - 1;
    const int off = sq.len - sq.lq;
    const int my_q = q_first + (i >> gsh);
    const int head = kvh * grp + (i & (grp - 1));
    const bool valid = my_q <= q_last;
    const int a_row = valid ? my_q + off : -1;
    const int* const pages = a.tab.pages + (int64_t)s * a.tab.width;

    W w;
    {
      const __bf16* qrow = a.q + (int64_t)(sq.q0 + (valid ? my_q : q_first)) * a.ql.token_stride +
                           (int64_t)head * a.ql.head_stride + 16 * h;
#pragma unroll
      for (int c = 0; c < W::kNC; ++c)
#pragma unroll
        for (int x = 0; x < 2; ++x) w.q[2 * c + x] = ld_global16(qrow + 64 * c + 8 * x);
    }
#pragma unroll
    for (int b = 0; b < W::kNB; ++b) w.o[b] = f32x4{};
    w.m = kNegInf;
    w.l = 0.f;

    auto page_head = [&](int t) -> int64_t {  // of tile t; -1: no page
      const int at = t * kTile / a.c.page_size;
      const int id = at < a.tab.width ? __builtin_amdgcn_readfirstlane(pages[at]) : -1;
      return (unsigned)id < (unsigned)a.c.num_pages ? (int64_t)id * hkv + kvh : -1;
    };
    const int blocks = a.c.page_size / kTile;
    int x = x0 + wave;
    int t = 0;
    int64_t ph = -1;
    if (x < x1) {
      t = range.at(x);
      ph = page_head(t);
      if (ph >= 0) {
        w.load_k(a, ph, t % blocks, i, h);
        w.load_v(a, ph, t % blocks, i, h);
      }
    }
    while (x < x1) {
      const int kb0 = t * kTile;
      const bool page = ph >= 0;
      const int xn = x + kWaves;
      int tn = 0;
      int64_t phn = -1;
      if (xn < x1) {
        tn = range.at(xn);
        phn = page_head(tn);
      }
      f32x4 sc[2] = {};
      if (page) w.scores(sc);
      if (phn >= 0) w.load_k(a, phn, tn % blocks, i, h);
      // (rows past the group's last query are never stored: they need no mask)
      const bool full = page && kb0 + kTile - 1 <= q_first + off &&
                        (a.window == 0 || kb0 > q_last + off - a.window || kb0 + kTile <= a.sinks);
      bf16x8 pb;
      w.softmax(a, sc, kb0, h, a_row, full, page, pb);
      if (page) {
        if (kb0 + kTile > sq.len) {
          // rows past the sequence's end hold anything: as zeros
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int g = 0; g < W::kNG; ++g)
              if (kb0 + 16 * (j >> 2) + 4 * h + (j & 3) >= sq.len) w.v[j][g] = u32x4{};
        }
        w.add_values(pb);
      }
      if (phn >= 0) w.load_v(a, phn, tn % blocks, i, h);
      x = xn;
      t = tn;
      ph = phn;
    }

    // ---- the waves' sums ---------------------------------------------------
    const float l = rows_sum(w.l);
    barrier_lds();  // the previous segment's readers are done
    if (h == 0) state[0][wave][i] = w.m, state[1][wave][i] = l;
#pragma unroll
    for (int b = 0; b < W::kNB; b += 4)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *(f32x4*)&rows[wave][i][256 * (b / 16) + 64 * h + 16 * r + b % 16] =
            f32x4{w.o[b][r], w.o[b + 1][r], w.o[b + 2][r], w.o[b + 3][r]};
    barrier_lds();
    const bool whole = x0 == 0 && x1 == range.n;
    const int nrows = (q_last - q_first + 1) << gsh;
    const int64_t segment = ((int64_t)s * a.groups + group) * hkv + kvh;
    float* const part_o = a.part + (part + segment) * kGroupRows * (D + 2);
    constexpr int kCols = D / 4;  // threads of a row, four elements each
    for (int r = tid / kCols; r < nrows; r += 256 / kCols) {
      const int d = tid % kCols * 4;
      float mx = state[0][0][r];
#pragma unroll
      for (int u = 1; u < kWaves; ++u) mx = fmaxf(mx, state[0][u][r]);
      const float m_use = mx == kNegInf ? 0.f : mx;
      float sum = 0.f;
      f32x4 acc = {};
#pragma unroll
      for (int u = 0; u < kWaves; ++u) {
        const float wt = fast_exp2(state[0][u][r] - m_use);
        sum += wt * state[1][u][r];
        acc += wt * *(const f32x4*)&rows[u][r][d];
      }
      if (whole) {
        const int qi = q_first + (r >> gsh), qh = kvh * grp + (r & (grp - 1));
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays)
        *(bf16x4*)(a.o + (int64_t)(sq.q0 + qi) * a.ol.token_stride +
                   (int64_t)qh * a.ol.head_stride + d) =
            bf16x4{(__bf16)(acc[0] * inv), (__bf16)(acc[1] * inv), (__bf16)(acc[2] * inv),
                   (__bf16)(acc[3] * inv)};
        if (d == 0)
          a.lse[(int64_t)qh * a.total_q + sq.q0 + qi] =
              sum == 0.f ? kNegInf : (mx + fast_log2(sum)) * kLn2;
      } else {
        *(f32x4*)(part_o + r * D + d) = acc;
        if (d == 0) {
          part_o[kGroupRows * D + 2 * r] = mx;
          part_o[kGroupRows * D + 2 * r + 1] = sum;
        }
      }
    }

    // ---- the next segment ------------------------------------------------------
    lo = seg0 + range.n;
    if (lo >= hi) break;
    seg0 = lo;
    if (++kvh == hkv) {
      kvh = 0;
      ++group;
      while (group * a.group_queries >= sq.lq) {  // (tiles are left, so sequences are)
        sq.init(a, ++s);
        group = 0;
      }
      range.init(a, sq, group * a.group_queries,
                 min((group + 1) * a.group_queries, sq.lq) - 1);
    }
  }
}

// O and LSE of the segments that more than one part holds.  One workgroup per
// (segment, row, SPLIT-th of the head dim).
template <int D, int SPLIT>
__global__ void __launch_bounds__(256) cache_merge_kernel(CacheAttnParams a) {
  constexpr int kCols = D / SPLIT / 4;  // threads of a row, four elements each
  constexpr int kSubs = 256 / kCols;    // parts added side by side
  __shared__ int64_t scan[kWaves];
  __shared__ float red[2][kWaves];
  __shared__ __attribute__((aligned(16))) float stage[kSubs][D / SPLIT];
  int64_t G4_LDS* sh = (int64_t G4_LDS*)scan;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int hkv = a.c.num_kv_heads;
  const int split = blockIdx.y, row = blockIdx.x % kGroupRows;
  const int64_t segment = blockIdx.x / kGroupRows;
  const int kvh = (int)(segment % hkv), group = (int)(segment / hkv % a.groups);
  const int s = (int)(segment / hkv / a.groups);
  const int grp = a.num_q_heads / hkv, gsh = __builtin_ctz(grp);
  CacheSeq sq;
  sq.init(a, s);
  const int qi = group * a.group_queries + (row >> gsh), qh = kvh * grp + (row & (grp - 1));
  if (row >= a.group_queries << gsh || qi >= sq.lq) return;

  // ---- the parts that hold the segment -----------------------------------------
  int64_t tiles = 0, first = 0;
  for (int s0 = 0; s0 < a.tab.batch; s0 += 256) {
    const int sx = s0 + tid;
    const int64_t n = sx < a.tab.batch ? sequence_tiles(a, sx) : 0;
    int64_t total, mine;
    block_before(n, sh, total);
    tiles += total;
    block_before(sx < s ? n : 0, sh, mine);
    first += mine;
  }
  TileRange range;
  for (int g = 0; g <= group; ++g) {
    range.init(a, sq, g * a.group_queries, min((g + 1) * a.group_queries, sq.lq) - 1);
    first += (int64_t)range.n * (g < group ? hkv : kvh);
  }
  const int64_t parts = part_count(a, tiles);
  const int64_t w0 = part_of(first, parts, tiles);
  const int n = (int)(part_of(first + range.n - 1, parts, tiles) - w0) + 1;
  if (n == 1) return;  // finished by its one part

  // ---- weights 2^(m_c - M), then the rows -----------------------------------------
  constexpr int64_t kSlot = kGroupRows * (D + 2);
  const float* const part = a.part + (w0 + segment) * kSlot;
  const float* const ml = part + kGroupRows * D + 2 * row;
  float mx = kNegInf;
  for (int c = tid; c < n; c += 256) mx = fmaxf(mx, ml[c * kSlot]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
  if (lane == 0) red[0][wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float m_use = mx == kNegInf ? 0.f : mx;
  const int sub = tid / kCols, d = tid % kCols * 4;
  const float* const po = part + row * D + split * (D / SPLIT) + d;
  f32x4 acc = {};
  float sum = 0.f;
#pragma unroll 4
  for (int c = sub; c < n; c += kSubs) {
    const float wt = fast_exp2(ml[c * kSlot] - m_use);
    sum += wt * ml[c * kSlot + 1];
    acc += wt * *(const f32x4*)(po + c * kSlot);
  }
  *(f32x4*)&stage[sub][d] = acc;
  // (each column's thread holds its sub's share of the sum)
  __shared__ float sums[kSubs];
  if (d == 0) sums[sub] = sum;
  __syncthreads();
  if (sub != 0) return;
  acc = f32x4{};
  sum = 0.f;
#pragma unroll
  for (int u = 0; u < kSubs; ++u) {
    acc += *(const f32x4*)&stage[u][d];
    sum += sums[u];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *(bf16x4*)(a.o + (int64_t)(sq.q0 + qi) * a.ol.token_stride + (int64_t)qh * a.ol.head_stride +
             split * (D / SPLIT) + d) = bf16x4{(__bf16)(acc[0] * inv), (__bf16)(acc[1] * inv),
                                               (__bf16)(acc[2] * inv), (__bf16)(acc[3] * inv)};
  if (split == 0 && d == 0)
    a.lse[(int64_t)qh * a.total_q + sq.q0 + qi] =
        sum == 0.f ? kNegInf : (mx + fast_log2(sum)) * kLn2;
}

// ---- launches -------------------------------------------------------------------

// Workgroups that are resident at once.
static int cache_parts(int head_dim) { return head_dim == 256 ? 512 : 256; }

static int64_t cache_segments(const CacheAttnParams& a) {
  return (int64_t)a.tab.batch * a.groups * a.c.num_kv_heads;
}

size_t cache_part_bytes(const CacheAttnParams& a) {
  const int64_t slots = cache_parts(a.c.head_dim) + cache_segments(a);
  return (size_t)slots * kGroupRows * (a.c.head_dim + 2) * 4;
}

template <int D>
static hipError_t launch_cache_attn_d(const CacheAttnParams& a, hipStream_t stream) {
  hipLaunchKernelGGL(cache_attn_kernel<D>, dim3((unsigned)a.parts), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const unsigned rows = (unsigned)(cache_segments(a) * kGroupRows);
  hipLaunchKernelGGL((cache_merge_kernel<D, 4>), dim3(rows, 4), dim3(256), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_cache_attn(CacheAttnParams a, hipStream_t stream) {
  a.parts = cache_parts(a.c.head_dim);
  return a.c.head_dim == 256 ? launch_cache_attn_d<256>(a, stream)
                             : launch_cache_attn_d<512>(a, stream);
}

}  // namespace g4

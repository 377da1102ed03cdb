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
// One, two or four groups (a set) share a workgroup of four waves, which then take
// the set's tiles side by side, so that a tile comes from memory once for up to 64
// rows (head dim 512: more than one group go to cache_wide_kernel).  The tiles of all
// (sequence, set, KV head) segments, in that order, are cut into equal parts, one
// workgroup each, so that the longest sequence of a batch does not decide its time.  A
// group's waves take its tiles in turn and add up through LDS; a segment inside one
// part is finished there, else the parts' sums go to the workspace (two slots a part:
// only the segments it begins and ends in can be cut), and the second launch has
// workgroups for each cut: those of one segment share its rows' elements evenly.
//
// Bound by HBM for long batches (1 byte an element of K and V: 2 x 100000 tokens of 4
// heads of 512 in 145 us, 5.4 TB/s; 16 of 4096 to 8192 tokens 89 + 6 us, of which about
// 8 are the way to the first tile), by the chain of launch, lengths, table, page and
// merge for short ones (one window of 1024 tokens, 16 heads of 256: 9.5 + 5.8 us).
// With one workgroup per (segment, row) the merge took 14 and 23 us (8 sequences of 5
// new tokens) in place of 6 and 4.4.
#include <type_traits>

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

// Tiles of a sequence's sets together, over all its KV heads.
__device__ __forceinline__ int64_t sequence_tiles(const CacheAttnParams& a, const CacheSeq& q) {
  int64_t n = 0;
  for (int i = 0; i < q.lq; i += a.set_queries) {
    TileRange t;
    t.init(a, q, i, min(i + a.set_queries, q.lq) - 1);
    n += t.n;
  }
  return n * a.c.num_kv_heads;
}

__device__ __forceinline__ int64_t sequence_tiles(const CacheAttnParams& a, int s) {
  CacheSeq q;
  q.init(a, s);
  return sequence_tiles(a, q);
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

// Tile x of the batch's `tiles`: the sequence it belongs to and that sequence's first
// tile; every thread of the workgroup (256) calls it.  The part is looked up in the
// same pass: it holds the tiles from tiles part / parts on.  False: no such part.
// (in scalar registers, which the wave's tiles leave free)
__device__ __forceinline__ int64_t uniform(int64_t x) {
  return ((int64_t)__builtin_amdgcn_readfirstlane((int)(x >> 32)) << 32) |
         (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}
struct PartStart {
  int64_t tiles, lo, hi, seq0;
  int parts, s;
  CacheSeq seq;  // sequence s
};
__device__ __forceinline__ int part_count(const CacheAttnParams& a, int64_t tiles) {
  // Few tiles: one each, as segments or a segment's waves that follow one another cost a
  // chain of loads each (4 heads of 512, us with four tiles or segments to a part / so:
  // 4 sequences of 2 tokens 43 / 18, 8 of 100 30 / 19, 3 of 428 28 / 20).  More: as many
  // tiles as a workgroup takes at once, and for one sequence, whose segments are alike, a
  // whole number of parts per segment, so that a part holds one of them (without / so: 4
  // heads of 512, 4000 tokens 29 / 22; a window of 1024, 16 heads of 256 19.8 / 16.0).
  if (tiles <= a.parts) return (int)tiles;
  int64_t n = max(tiles / a.step_tiles, min(tiles, a.segments));
  if (a.tab.batch == 1 && n < a.parts && a.segments <= n) {
    const unsigned seg = (unsigned)a.segments;
    n = ((unsigned)n + seg - 1) / seg * seg;
  }
  return (int)min((int64_t)a.parts, n);
}
__device__ __forceinline__ int part_of(int64_t x, int parts, int64_t tiles) {
  return (int)(((x + 1) * parts - 1) / tiles);
}
__device__ __forceinline__ bool find_part(const CacheAttnParams& a, int part, int64_t G4_LDS* lds,
                                          PartStart& f) {
  if (a.tab.batch <= 64) {
    // one sequence a lane, in every wave by itself: no LDS, no barrier
    const int lane = threadIdx.x & 63;
    CacheSeq q;
    q.init(a, min(lane, a.tab.batch - 1));
    const int64_t n = lane < a.tab.batch ? sequence_tiles(a, q) : 0;
    int64_t incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int64_t y = __shfl_up(incl, o, 64);
      if (lane >= o) incl += y;
    }
    f.tiles = uniform(__shfl(incl, 63, 64));
    f.parts = part_count(a, f.tiles);
    if (part >= f.parts) return false;
    f.lo = f.tiles * part / f.parts;
    f.hi = f.tiles * (part + 1) / f.parts;
    f.s = __builtin_amdgcn_readfirstlane(__popcll(__ballot(incl <= f.lo)));
    f.seq0 = uniform(__shfl(incl - n, f.s, 64));
    f.seq.q0 = __builtin_amdgcn_readlane(q.q0, f.s);
    f.seq.lq = __builtin_amdgcn_readlane(q.lq, f.s);
    f.seq.len = __builtin_amdgcn_readlane(q.len, f.s);
    return true;
  }
  f.tiles = 0;
  for (int s0 = 0; s0 < a.tab.batch; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    int64_t total;
    block_before(s < a.tab.batch ? sequence_tiles(a, s) : 0, lds, total);
    f.tiles = uniform(f.tiles + total);
  }
  f.parts = part_count(a, f.tiles);
  if (part >= f.parts) return false;
  f.lo = f.tiles * part / f.parts;
  f.hi = f.tiles * (part + 1) / f.parts;
  int64_t base = 0;
  for (int s0 = 0; base <= f.lo; s0 += 256) {
    const int s = s0 + (int)threadIdx.x;
    const int64_t n = s < a.tab.batch ? sequence_tiles(a, s) : 0;
    int64_t total;
    const int64_t before = base + block_before(n, lds, total);
    if (before <= f.lo && f.lo < before + n) lds[kWaves] = s, lds[kWaves + 1] = before;
    base += total;
  }
  barrier_lds();
  f.s = __builtin_amdgcn_readfirstlane((int)lds[kWaves]);
  f.seq0 = uniform(lds[kWaves + 1]);
  f.seq.init(a, f.s);
  return true;
}

}  // namespace

// What a part leaves for the merge: the segment it begins in (its first tile, tiles, KV
// head, first query's row and rows) and the batch's tiles and parts.
struct PartHead {
  int64_t tiles, seg0;
  int parts, n, kvh, q_row, rows, pad;
};
static_assert(sizeof(PartHead) == 40, "a part's head");

// Slot of a part's sums for a segment that begins at tile seg0: the first slot for the
// segment that the part begins in, the second for one that begins within it.
__device__ __forceinline__ int64_t part_slot(int part, int64_t part_lo, int64_t seg0) {
  return 2 * (int64_t)part + (seg0 > part_lo);
}

// The segments of a part in order: the one at hand, and the part's share of its tiles.
struct PartWalk {
  int64_t lo, hi, seg0;  // the part's tiles that are left, the segment's first tile
  int s, set, kvh;
  CacheSeq sq;  // sequence s
  TileRange range;
  __device__ __forceinline__ void set_range(const CacheAttnParams& a) {
    range.init(a, sq, set * a.set_queries, min((set + 1) * a.set_queries, sq.lq) - 1);
  }
  __device__ __forceinline__ void init(const CacheAttnParams& a, const PartStart& f) {
    lo = f.lo;
    hi = f.hi;
    seg0 = f.seq0;
    s = f.s;
    sq = f.seq;
    const int hkv = a.c.num_kv_heads;
    for (set = 0;; ++set) {
      set_range(a);
      const int64_t n = (int64_t)range.n * hkv;
      if (lo < seg0 + n) break;
      seg0 += n;
    }
    kvh = (int)((lo - seg0) / range.n);
    seg0 += (int64_t)kvh * range.n;
  }
  __device__ __forceinline__ int x0() const { return (int)(lo - seg0); }
  __device__ __forceinline__ int x1() const { return (int)min(hi - seg0, (int64_t)range.n); }
  __device__ __forceinline__ PartHead head(const CacheAttnParams& a, const PartStart& f) const {
    const int gsh = __builtin_ctz(a.num_q_heads / a.c.num_kv_heads);
    return {f.tiles, seg0, f.parts, range.n, kvh, sq.q0 + set * a.set_queries,
            min(a.set_queries, sq.lq - set * a.set_queries) << gsh, 0};
  }
  // False: the part has no further segment.
  __device__ __forceinline__ bool next(const CacheAttnParams& a) {
    lo = seg0 + range.n;
    if (lo >= hi) return false;
    seg0 = lo;
    if (++kvh == a.c.num_kv_heads) {
      kvh = 0;
      ++set;
      while (set * a.set_queries >= sq.lq) {  // (tiles are left, so sequences are)
        sq.init(a, ++s);
        set = 0;
      }
      set_range(a);
    }
    return true;
  }
};

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
          const uint32_t k0 = k[u][c][2 * x], k1 = k[u][c][2 * x + 1];
          const u32x4 w = {e4m3_pair<false>(k0, ks), e4m3_pair<true>(k0, ks),
                           e4m3_pair<false>(k1, ks), e4m3_pair<true>(k1, ks)};
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
  __shared__ int64_t scan[kWaves + 2];
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hkv = a.c.num_kv_heads;
  const int sets = a.set_groups, turns = kWaves / sets;  // groups of a set, waves of a group
  const int sub = wave % sets, turn = wave / sets;       // this wave's group and turn

  // ---- this part's tiles [lo, hi) and the sequence of the first --------------
  const int part = blockIdx.x;
  PartStart f;
  if (!find_part(a, part, (int64_t G4_LDS*)scan, f)) {
    if (part == 0 && tid == 0) a.heads[0].parts = 0;
    return;
  }
  PartWalk walk;
  walk.init(a, f);
  if (tid == 0) a.heads[part] = walk.head(a, f);
  const int grp = a.num_q_heads / hkv, gsh = __builtin_ctz(grp);
  const int blocks = a.c.page_size / kTile;
  do {
    // ---- the part's share [x0, x1) of the segment's tiles ---------------------
    const CacheSeq& sq = walk.sq;
    const TileRange& range = walk.range;
    const int kvh = walk.kvh, set = walk.set;
    const int x0 = walk.x0(), x1 = walk.x1();
    const int set_first = set * a.set_queries;
    const int set_last = min(set_first + a.set_queries, sq.lq) - 1;
    const int q_first = set_first + sub * (kGroupRows >> gsh);  // of this wave's group
    const int q_last = min(q_first + (kGroupRows >> gsh) - 1, set_last);
    const int off = sq.len - sq.lq;
    const int my_q = q_first + (i >> gsh);
    const int head = kvh * grp + (i & (grp - 1));
    const bool valid = my_q <= q_last;
    const int a_row = valid ? my_q + off : -1;
    const int* const pages = a.tab.pages + (int64_t)walk.s * a.tab.width;

    W w;
    {
      // (rows past the group's queries: the set's first, whose results are dropped)
      const __bf16* qrow = a.q + (int64_t)(sq.q0 + (valid ? my_q : set_first)) * a.ql.token_stride +
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
    const int end = q_first > q_last ? x0 : x1;  // (a group without queries has no tiles)
    int x = x0 + turn;
    int t = 0;
    int64_t ph = -1;
    if (x < end) {
      t = range.at(x);
      ph = page_head(t);
      if (ph >= 0) {
        w.load_k(a, ph, t % blocks, i, h);
        w.load_v(a, ph, t % blocks, i, h);
      }
    }
    while (x < end) {
      const int kb0 = t * kTile;
      const bool page = ph >= 0;
      const int xn = x + turns;
      int tn = 0;
      int64_t phn = -1;
      if (xn < end) {
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
    const int nrows = (set_last - set_first + 1) << gsh;
    float* const part_o =
        a.part + part_slot(part, f.lo, walk.seg0) * (int64_t)(sets * kGroupRows * (D + 2));
    constexpr int kCols = D / 4;  // threads of a row, four elements each
    for (int r = tid / kCols; r < nrows; r += 256 / kCols) {
      const int d = tid % kCols * 4, g = r / kGroupRows, ri = r % kGroupRows;
      float mx = kNegInf;
      for (int u = g; u < kWaves; u += sets) mx = fmaxf(mx, state[0][u][ri]);
      const float m_use = mx == kNegInf ? 0.f : mx;
      float sum = 0.f;
      f32x4 acc = {};
      for (int u = g; u < kWaves; u += sets) {
        const float wt = fast_exp2(state[0][u][ri] - m_use);
        sum += wt * state[1][u][ri];
        acc += wt * *(const f32x4*)&rows[u][ri][d];
      }
      if (whole) {
        const int qi = set_first + (r >> gsh), qh = kvh * grp + (r & (grp - 1));
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
          float* const ml = part_o + sets * kGroupRows * D + 2 * r;
          ml[0] = mx;
          ml[1] = sum;
        }
      }
    }
  } while (walk.next(a));
}

// ---------------------------------------------------------------------------
// More rows of a KV head than 16, head dim 512: a set of 16 G rows in one workgroup,
// which takes 64 keys (two tiles) a step.  A wave scores 16 of the keys against all
// rows (Q from LDS, in the order of the operand), then adds 128 of the columns of V for
// all keys and rows, so that each element of K and V is converted once for the whole
// set.  Between the two P^T goes through LDS: the scores of a lane are 4 of the 8
// elements of the same lane's operand.  All waves keep the rows' maxima; each has its
// keys' share of their sums and whole sums of its columns.
//
// Between HBM (64 KB a step and CU: 3.2 us) and what G costs a step (16 + 16 matrix
// instructions, 64 KB of Q from LDS and a softmax a group: 0.8 us).  Whole calls with
// this kernel / with the one above, a wave a tile and 16 rows: 2 x 100000 tokens, 5 new
// (G = 3) 184 / 351 us, 8 x 8000, 3, 6 and 8 new 56 / 77, 72 / 117 and 85 / 133.  Loads
// are a step ahead, the table's entries two: with the entries one step ahead 212 us for
// the first (each step waits for them and, in order, for the values before them).
// ---------------------------------------------------------------------------
template <int G>
__global__ void __launch_bounds__(256, 1) cache_wide_kernel(CacheAttnParams a) {
  constexpr int D = 512;
  constexpr int kNC = D / 64;               // 16-byte chunks of a lane's K row
  constexpr int kCols = D / kWaves;         // columns of a wave
  constexpr int kNB = kCols / 16;           // its O^T blocks
  constexpr int kRows = G * kGroupRows;
  __shared__ u32x4 qs[G][2 * kNC][64];      // operands of Q
  __shared__ u32x2 ps[2][G][64][2];         // operands of P^T: [tile][group][lane][half]
  __shared__ f32x4 stat[kRows];             // a value of each wave per row
  __shared__ int64_t scan[kWaves + 2];
  const int tid = threadIdx.x, lane = tid & 63, i = lane & 15, h = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int own = wave >> 1, half = wave & 1;  // the tile of the step and its keys to score
  const int hkv = a.c.num_kv_heads;

  const int part = blockIdx.x;
  PartStart f;
  if (!find_part(a, part, (int64_t G4_LDS*)scan, f)) {
    if (part == 0 && tid == 0) a.heads[0].parts = 0;
    return;
  }
  PartWalk w;
  w.init(a, f);
  if (tid == 0) a.heads[part] = w.head(a, f);
  const int grp = a.num_q_heads / hkv, gsh = __builtin_ctz(grp);
  const int blocks = a.c.page_size / kTile;
  do {
    const int x0 = w.x0(), x1 = w.x1();
    const int set_first = w.set * a.set_queries;
    const int set_last = min(set_first + a.set_queries, w.sq.lq) - 1;
    const int off = w.sq.len - w.sq.lq;
    const int nrows = (set_last - set_first + 1) << gsh;
    const int* const pages = a.tab.pages + (int64_t)w.s * a.tab.width;

    // ---- Q (rows past the set's: its first, whose results are dropped) ----------------
    constexpr int kMine = 2 * kNC / kWaves;  // this wave's operands of a group
    u32x4 q[G][kMine];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int row = g * kGroupRows + i, r = row < nrows ? row : 0;
      const __bf16* src = a.q + (int64_t)(w.sq.q0 + set_first + (r >> gsh)) * a.ql.token_stride +
                          (int64_t)(w.kvh * grp + (r & (grp - 1))) * a.ql.head_stride + 16 * h;
#pragma unroll
      for (int n = 0; n < kMine; ++n) {
        const int st = wave * kMine + n;
        q[g][n] = *(const u32x4*)(src + 64 * (st >> 1) + 8 * (st & 1));
      }
    }

    u32x4 k[kNC];     // key i of this wave's half tile
    u32x2 v[2][8];    // keys 16 (j >> 2) + 4 h + (j & 3) of both tiles, columns 8 i + 0..7
    float ks, vs[2];
    int t[2], id[2];  // a step's tiles and their pages, or -1
    int tn[2], entry[2];  // the next step's, whose table entries are on their way
    // (a tile without a page is read from page 0 and masked: no branch around the loads)
    auto fetch = [&](int x) {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        tn[b] = x + b < x1 ? w.range.at(x + b) : -1;
        entry[b] = pages[min(max(tn[b], 0) * kTile / a.c.page_size, a.tab.width - 1)];
      }
    };
    auto resolve = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        t[b] = tn[b];
        const int page = __builtin_amdgcn_readfirstlane(entry[b]);
        id[b] = t[b] >= 0 && t[b] * kTile / a.c.page_size < a.tab.width &&
                        (unsigned)page < (unsigned)a.c.num_pages
                    ? page
                    : -1;
      }
    };
    auto load_k = [&]() {
      const int64_t p = uniform((int64_t)max(own ? id[1] : id[0], 0) * hkv + w.kvh);
      const int blk = max(own ? t[1] : t[0], 0) % blocks;
      const uint8_t* src = (const uint8_t*)a.c.k +
                           (p * a.c.page_size + blk * kTile + 16 * half + i) * D + 16 * h;
      ks = a.c.k_scale[p * blocks + blk];
#pragma unroll
      for (int c = 0; c < kNC; ++c) k[c] = *(const u32x4*)(src + c * 64);
    };
    auto load_v = [&]() {
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        const int64_t p = uniform((int64_t)max(id[b], 0) * hkv + w.kvh);
        const int blk = max(t[b], 0) % blocks;
        const uint8_t* src = (const uint8_t*)a.c.v +
                             (p * a.c.page_size + blk * kTile + 4 * h) * D + wave * kCols + 8 * i;
        vs[b] = a.c.v_scale[p * blocks + blk];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[b][j] = *(const u32x2*)(src + (16 * (j >> 2) + (j & 3)) * D);
      }
    };

    f32x4 o[G][kNB];
    float m[G], l[G];
#pragma unroll
    for (int g = 0; g < G; ++g) {
      m[g] = kNegInf;
      l[g] = 0.f;
#pragma unroll
      for (int b = 0; b < kNB; ++b) o[g][b] = f32x4{};
    }
    fetch(x0);
    resolve();
    // (in the loop's order, which its waits count)
    load_k();
    __builtin_amdgcn_sched_barrier(0);
    fetch(x0 + 2);
    __builtin_amdgcn_sched_barrier(0);
    load_v();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int n = 0; n < kMine; ++n) qs[g][wave * kMine + n][lane] = q[g][n];
    barrier_lds();
    for (int x = x0; x < x1; x += 2) {
      // ---- scores of 16 keys -------------------------------------------------------
      const int now[2] = {t[0], t[1]};
      const bool there[2] = {id[0] >= 0, id[1] >= 0};
      const bool page = own ? there[1] : there[0];
      const int my_t = own ? now[1] : now[0];
      f32x4 s[G];
#pragma unroll
      for (int g = 0; g < G; ++g) s[g] = f32x4{};
      // (Q two steps ahead, K one, in this order: two reads in flight cost 1.2 us a step)
      u32x4 qr[3][G];
      auto read_q = [&](int st) {
#pragma unroll
        for (int g = 0; g < G; ++g) qr[st % 3][g] = qs[g][st][lane];
      };
      auto key = [&](int st) -> bf16x8 {
        const uint32_t k0 = k[st >> 1][2 * (st & 1)], k1 = k[st >> 1][2 * (st & 1) + 1];
        return __builtin_bit_cast(bf16x8, u32x4{e4m3_pair<false>(k0, ks), e4m3_pair<true>(k0, ks),
                                                e4m3_pair<false>(k1, ks), e4m3_pair<true>(k1, ks)});
      };
      read_q(0);
      read_q(1);
      __builtin_amdgcn_sched_barrier(0);
      bf16x8 kf = key(0);
#pragma unroll
      for (int st = 0; st < 2 * kNC; ++st) {
        if (st + 2 < 2 * kNC) read_q(st + 2);
        const bf16x8 kn = key(min(st + 1, 2 * kNC - 1));
#pragma unroll
        for (int g = 0; g < G; ++g)
          s[g] = mfma16(kf, __builtin_bit_cast(bf16x8, qr[st % 3][g]), s[g]);
        kf = kn;
        __builtin_amdgcn_sched_barrier(0);
      }
      resolve();
      load_k();
      __builtin_amdgcn_sched_barrier(0);
      fetch(x + 4);
      __builtin_amdgcn_sched_barrier(0);
      // (a tile past the part's share is masked whole)
      const int kb0 = my_t * kTile + 16 * half;
      if (!page || kb0 + 15 > set_first + off) {
#pragma unroll
        for (int g = 0; g < G; ++g) {
          const int row = g * kGroupRows + i;
          const int a_row =
              my_t >= 0 && row < nrows ? set_first + (row >> gsh) + off : -0x7fffffff;
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[g][r] = kb0 + 4 * h + r <= a_row ? (page ? s[g][r] : __builtin_nanf("")) : kNegInf;
        }
      }
      // ---- the rows' maxima over the waves -----------------------------------------
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float mx = rows_max(fmaxf(fmaxf(s[g][0], s[g][1]), fmaxf(s[g][2], s[g][3])));
        if (h == 0) ((float*)&stat[g * kGroupRows + i])[wave] = mx;
      }
      barrier_lds();
      float alpha[G];
      bool moved = false;
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const f32x4 all = stat[g * kGroupRows + i];
        const float mx = fmaxf(fmaxf(all[0], all[1]), fmaxf(all[2], all[3])) * kLog2e;
        // (moves only when exceeded by more than 2^8, as in CacheWave::softmax)
        const float m_new = mx > m[g] + 8.f ? mx : m[g];
        const float m_use = m_new == kNegInf ? 0.f : m_new;
        alpha[g] = fast_exp2(m[g] - m_use);
        float sum = 0.f;
        bf16x4 pb;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float p = fast_exp2(__builtin_fmaf(s[g][r], kLog2e, -m_use));
          sum += p;
          pb[r] = (__bf16)p;
        }
        l[g] = l[g] * alpha[g] + sum;
        m[g] = m_new;
        moved |= alpha[g] != 1.f;
        ps[own][g][lane][half] = __builtin_bit_cast(u32x2, pb);
      }
      if (__ballot(moved)) {
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int b = 0; b < kNB; ++b) o[g][b] *= alpha[g];
      }
      barrier_lds();
      // ---- O^T += V^T P^T of 128 columns --------------------------------------------
#pragma unroll
      for (int b = 0; b < 2; ++b) {
        if (!there[b]) continue;
        if ((now[b] + 1) * kTile > w.sq.len) {
          // rows past the sequence's end hold anything: as zeros
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (now[b] * kTile + 16 * (j >> 2) + 4 * h + (j & 3) >= w.sq.len) v[b][j] = u32x2{};
        }
        bf16x8 pb[G];
#pragma unroll
        for (int g = 0; g < G; ++g) pb[g] = *(const bf16x8*)&ps[b][g][lane][0];
#pragma unroll
        for (int y2 = 0; y2 < 2; ++y2) {
          uint32_t lo[8], hi[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            lo[j] = e4m3_pair<false>(v[b][j][y2], vs[b]);
            hi[j] = e4m3_pair<true>(v[b][j][y2], vs[b]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t* y = e < 2 ? lo : hi;
            const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
            u32x4 vf;
#pragma unroll
            for (int j = 0; j < 4; ++j) vf[j] = __builtin_amdgcn_perm(y[2 * j + 1], y[2 * j], sel);
#pragma unroll
            for (int g = 0; g < G; ++g)
              o[g][4 * y2 + e] = mfma16(__builtin_bit_cast(bf16x8, vf), pb[g], o[g][4 * y2 + e]);
          }
        }
      }
      load_v();
    }

    // ---- O and LSE, or the part's sums --------------------------------------------------
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float sum = rows_sum(l[g]);
      if (h == 0) ((float*)&stat[g * kGroupRows + i])[wave] = sum;
    }
    barrier_lds();
    const bool whole = x0 == 0 && x1 == w.range.n;
    float* const part_o = a.part + part_slot(part, f.lo, w.seg0) * (int64_t)(kRows * (D + 2));
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const int row = g * kGroupRows + i;
      if (row >= nrows) continue;
      const f32x4 all = stat[row];
      const float sum = (all[0] + all[1]) + (all[2] + all[3]);
      // columns kCols wave + 8 (4 h + r) + 0..7
      const int col = kCols * wave + 32 * h;
      if (whole) {
        const int qi = w.sq.q0 + set_first + (row >> gsh), qh = w.kvh * grp + (row & (grp - 1));
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays)
        __bf16* const out =
            a.o + (int64_t)qi * a.ol.token_stride + (int64_t)qh * a.ol.head_stride + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          bf16x8 y;
#pragma unroll
          for (int b = 0; b < kNB; ++b) y[b] = (__bf16)(o[g][b][r] * inv);
          *(bf16x8*)(out + 8 * r) = y;
        }
        if (wave == 0 && h == 0)
          a.lse[(int64_t)qh * a.total_q + qi] =
              sum == 0.f ? kNegInf : (m[g] + fast_log2(sum)) * kLn2;
      } else {
        float* const out = part_o + row * D + col;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          *(f32x4*)(out + 8 * r) = f32x4{o[g][0][r], o[g][1][r], o[g][2][r], o[g][3][r]};
          *(f32x4*)(out + 8 * r + 4) = f32x4{o[g][4][r], o[g][5][r], o[g][6][r], o[g][7][r]};
        }
        if (wave == 0 && h == 0) {
          float* const ml = part_o + kRows * D + 2 * row;
          ml[0] = m[g];
          ml[1] = sum;
        }
      }
    }
  } while (w.next(a));
}

// O and LSE of the segments that more than one part holds.  The workgroup of part w
// serves the segment that part w begins inside of, as one of the n - 1 workgroups
// whose parts do (gridDim.y for each): each takes an equal run of the rows' elements,
// four a thread, and where those are fewer than the threads, several threads share the
// parts.
template <int D>
__global__ void __launch_bounds__(256) cache_merge_kernel(CacheAttnParams a) {
  __shared__ __attribute__((aligned(16))) float acc_lds[256][4];
  __shared__ float ml_lds[256][2];
  const int w = blockIdx.x + 1, tid = threadIdx.x;
  const PartHead& first = a.heads[0];
  const PartHead hd = a.heads[w];
  const int parts = first.parts;
  if (w >= parts) return;
  const int64_t tiles = first.tiles;
  if (tiles * w / parts == hd.seg0) return;  // begins with the segment
  const int w0 = part_of(hd.seg0, parts, tiles);
  const int n = part_of(hd.seg0 + hd.n - 1, parts, tiles) - w0 + 1;

  const int grp = a.num_q_heads / a.c.num_kv_heads, gsh = __builtin_ctz(grp);
  const int set_rows = a.set_groups * kGroupRows;
  const int64_t slot = (int64_t)set_rows * (D + 2);
  // the segment's parts: its first part's slot, then the first slots of the following
  const float* const part0 = a.part + part_slot(w0, tiles * w0 / parts, hd.seg0) * slot;
  const float* const part1 = a.part + 2 * (int64_t)(w0 + 1) * slot;
  const auto sums = [&](int c) { return c == 0 ? part0 : part1 + 2 * (int64_t)(c - 1) * slot; };

  const int units = hd.rows * (D / 4);  // four elements of a row each
  const int y = gridDim.y * (w - w0 - 1) + blockIdx.y, ny = gridDim.y * (n - 1);
  const int u0 = (int)((int64_t)units * y / ny), u1 = (int)((int64_t)units * (y + 1) / ny);
  const auto store = [&](int u, float mx, float sum, f32x4 acc) {
    const int r = u / (D / 4), d = u % (D / 4) * 4;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    const int qrow = hd.q_row + (r >> gsh), qh = hd.kvh * grp + (r & (grp - 1));
    *(bf16x4*)(a.o + (int64_t)qrow * a.ol.token_stride + (int64_t)qh * a.ol.head_stride +
               d) = bf16x4{(__bf16)(acc[0] * inv), (__bf16)(acc[1] * inv),
                           (__bf16)(acc[2] * inv), (__bf16)(acc[3] * inv)};
    if (d == 0)
      a.lse[(int64_t)qh * a.total_q + qrow] =
          sum == 0.f ? kNegInf : (mx + fast_log2(sum)) * kLn2;
  };
  // U units' sums over the parts c0, c0 + step, ..., C parts at a time, so that the loads
  // of U x C are in flight together.
  const auto add = [&](auto units_at_once, auto parts_at_once, const int* u, int c0, int step,
                       float* mx, float* sum, f32x4* acc) {
    constexpr int U = decltype(units_at_once)::value, C = decltype(parts_at_once)::value;
#pragma unroll
    for (int i = 0; i < U; ++i) mx[i] = kNegInf, sum[i] = 0.f, acc[i] = f32x4{};
    for (; c0 < n; c0 += C * step) {
      f32x2 ml[C][U];
      f32x4 o[C][U];
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const float* const part = sums(min(c0 + c * step, n - 1));
#pragma unroll
        for (int i = 0; i < U; ++i) {
          const int r = u[i] / (D / 4), d = u[i] % (D / 4) * 4;
          ml[c][i] = *(const f32x2*)(part + set_rows * D + 2 * r);
          o[c][i] = *(const f32x4*)(part + r * D + d);
        }
      }
#pragma unroll
      for (int i = 0; i < U; ++i) {
        float m_new = mx[i];
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c0 + c * step < n) m_new = fmaxf(m_new, ml[c][i][0]);
        const float m_use = m_new == kNegInf ? 0.f : m_new;
        const float alpha = fast_exp2(mx[i] - m_use);
        sum[i] *= alpha;
        acc[i] *= alpha;
#pragma unroll
        for (int c = 0; c < C; ++c)
          if (c0 + c * step < n) {
            const float wt = fast_exp2(ml[c][i][0] - m_use);
            sum[i] += wt * ml[c][i][1];
            acc[i] += wt * o[c][i];
          }
        mx[i] = m_new;
      }
    }
  };
  // a thread a unit, up to four of them at a time
  const auto each = [&](auto units_at_once, auto parts_at_once) {
    constexpr int U = decltype(units_at_once)::value;
    for (int ub = u0; ub < u1; ub += U * 256) {
      int u[U];
      float mx[U], sum[U];
      f32x4 acc[U];
#pragma unroll
      for (int i = 0; i < U; ++i) u[i] = min(ub + i * 256 + tid, u1 - 1);
      add(units_at_once, parts_at_once, u, 0, 1, mx, sum, acc);
#pragma unroll
      for (int i = 0; i < U; ++i)
        if (ub + i * 256 + tid < u1) store(u[i], mx[i], sum[i], acc[i]);
    }
  };
  std::integral_constant<int, 1> one;
  std::integral_constant<int, 2> two;
  std::integral_constant<int, 4> four;
  if (u1 - u0 > 512) return each(four, two);
  if (u1 - u0 > 256) return each(two, four);
  if (u1 - u0 > 128) return each(one, four);
  int subs = 2;  // threads of a unit
  while (subs < 16 && subs * 2 * (u1 - u0) <= 256) subs *= 2;
  const int u = u0 + tid / subs, sub = tid % subs;
  float mx, sum;
  f32x4 acc;
  const int at = min(u, max(u1 - 1, 0));
  add(one, four, &at, sub, subs, &mx, &sum, &acc);
  *(f32x4*)acc_lds[tid] = acc;
  ml_lds[tid][0] = mx;
  ml_lds[tid][1] = sum;
  __syncthreads();
  if (sub != 0 || u >= u1) return;
  for (int v = 1; v < subs; ++v) mx = fmaxf(mx, ml_lds[tid + v][0]);
  const float m_use = mx == kNegInf ? 0.f : mx;
  sum = 0.f;
  acc = f32x4{};
  for (int v = 0; v < subs; ++v) {
    const float wt = fast_exp2(ml_lds[tid + v][0] - m_use);
    sum += wt * ml_lds[tid + v][1];
    acc += wt * *(const f32x4*)acc_lds[tid + v];
  }
  store(u, mx, sum, acc);
}

// ---- launches -------------------------------------------------------------------

// Workgroups that are resident at once.
static int cache_parts(int head_dim) { return head_dim == 256 ? 512 : 256; }

// Groups of a set: as many as the batch's longest run of new tokens fills, up to what
// a kernel takes, in sets of about equal rows.
static void cache_sets(CacheAttnParams* a) {
  const int grp = a->num_q_heads / a->c.num_kv_heads;
  const int64_t groups = ((int64_t)a->max_q * grp + kGroupRows - 1) / kGroupRows;
  a->wide = a->c.head_dim == 512 && groups > 1;
  const int64_t sets = (groups + 3) / 4;
  const int n = (int)((groups + sets - 1) / sets);
  a->set_groups = !a->wide && n == 3 ? 4 : n;
  a->set_queries = a->set_groups * kGroupRows / grp;
  a->parts = cache_parts(a->c.head_dim);
  a->step_tiles = a->wide ? 2 : kWaves / a->set_groups;
  a->segments = (int64_t)a->tab.batch * a->c.num_kv_heads *
                ((a->max_q + a->set_queries - 1) / a->set_queries);
}

static size_t heads_bytes(const CacheAttnParams& a) {
  return ((size_t)a.parts * sizeof(PartHead) + 255) & ~size_t(255);
}

size_t cache_part_bytes(CacheAttnParams a) {
  cache_sets(&a);
  return heads_bytes(a) + (size_t)2 * a.parts * a.set_groups * kGroupRows * (a.c.head_dim + 2) * 4;
}

// Workgroups of the merge for a cut: 26 sequences of 12 new tokens (sets of 48 rows) 158
// us in all with one, 147 with three, 142 with six; 5 of 15 20.4, 17.7 and 21.9.
static int merge_blocks(int set_groups) { return set_groups; }

template <int D>
static hipError_t launch_cache_attn_d(const CacheAttnParams& a, hipStream_t stream) {
  void (*kern)(CacheAttnParams) = cache_attn_kernel<D>;
  if constexpr (D == 512)
    if (a.wide)
      kern = a.set_groups == 2   ? cache_wide_kernel<2>
             : a.set_groups == 3 ? cache_wide_kernel<3>
                                 : cache_wide_kernel<4>;
  hipLaunchKernelGGL(kern, dim3((unsigned)a.parts), dim3(256), 0, stream, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(cache_merge_kernel<D>,
                     dim3((unsigned)a.parts - 1, (unsigned)merge_blocks(a.set_groups)), dim3(256),
                     0, stream, a);
  return hipGetLastError();
}

hipError_t launch_cache_attn(CacheAttnParams a, void* ws, hipStream_t stream) {
  cache_sets(&a);
  a.heads = (PartHead*)ws;
  a.part = (float*)((char*)ws + heads_bytes(a));
  return a.c.head_dim == 256 ? launch_cache_attn_d<256>(a, stream)
                             : launch_cache_attn_d<512>(a, stream);
}

}  // namespace g4

// Attention of a chunk of new tokens over a paged KV cache on the matrix cores (bf16 / f16, head size
// 64 or 128): chunked prefill and whole prompts.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * q.k_j,  lse = m + log sum_j p_j
//
// The tile body is the prefill kernel's: a wave holds 32 query rows of one query head; S^T = K.Q^T per
// 64-key tile with v_mfma_f32_32x32x16 (a lane holds one row's scores, so its statistics are scalars),
// O^T += V^T.P^T from the score registers, V transposed on its way out of LDS; K and V go global -> LDS
// directly; exp2 domain, the reference maximum moved only when a row's grows by 2^8.  A workgroup is 4
// waves, 128 rows of one query head (or, for short chunks, of 2 or 4 heads of one KV head), with two
// tiles in LDS, the next one loading: two workgroups fit a compute unit at D = 128, three at D =
// 64, and while one waits at its barrier or for its products another has its softmax to do.  (8 waves, 4
// tiles, one workgroup a compute unit: chunks of 500 tokens over 4000 to 9000 keys, 32/8 heads of 128, 248 us
// against 232; four chunks of 300 over 700 to 4001, 32/4 heads of 64, 63.3 against 51.2; two prompts of
// 2000, 32/4 heads of 64, 58.4 against 53.3, of 128 85.9 and 85.9; 12 tokens of 4 rows of up to 10000 49
// against 31; 128 tokens over 32768 keys 90.4 against 93.4, whose keys cross the L2 twice as often.)
// Bound by the matrix cores (40 % busy over two prompts of 2000), the LDS reads that feed them and the
// softmax's vector instructions, each near half of the time.  What the pages change:
//   * a wave loads 16 rows of a tile, and pages are multiples of 16 slots, so they lie in one page:
//     its address stays scalar; the page indices of 256 tiles at a time wait in LDS (read through the
//     scalar cache, each delayed the next tile's first product);
//   * without positions in the pool slot j is position j, so the tiles that a workgroup visits are
//     a prefix of the row and every mask is one 32-bit comparison with the query row's limit; with
//     them a launch before this one summarises the tiles, writes the positions in 32 bits and
//     what a score starts with, 0 or -inf where no key is, and the workgroup lists the tiles it needs; the
//     products add to that start, so empty slots cost no comparisons (82 us to 61 with the smaller
//     workgroups, four chunks of 300 over 700 to 4001 slots with 2 % of them empty);
//   * lengths are known on the device alone: a launch with few query blocks has room for up to 16 key
//     splits by the table's width, and the device gives every row as many as its tiles are worth, each
//     an equal run of them; a second launch joins the rows that were cut;
//   * hidden keys may hold anything.  Their scores are masked; a value that is not finite shows up as
//     a result that is not, and the workgroup then goes over its tiles once more: such values are taken
//     out of the tiles as they land, and the tiles that had some are visited again to add, per row and
//     feature, the infinity or NaN that the visible ones make.  A chunk without them pays one look at
//     its results.
//   * drafts: the queries are nodes of a tree in the row's last slots.  The slots before them are tiles that
//     every row sees whole; in the last tiles a query row's 64 keys are a window of its mask's words, which wait in
//     LDS, so a tile costs a shift and a test of a bit per score (16 trees of 60 nodes after 500 to 8192 slots of
//     8 bits, 32/8 heads of 128: 124 us, 545 TFLOP/s, 112 of them tiles; 26 nodes after 777, 32/4 heads of 64, 15.5);
//   * pages of 8 bits: a wave's 16 rows of a tile land in LDS as they are, and the wave itself turns them into
//     16-bit rows in the one tile that is computed (v_cvt_scalef32_pk, exact: 4 significant bits and a power of
//     two), a second barrier before the products.  The products are those of the 16-bit form.  128 tokens over
//     32768 keys, 32/8 heads of 128: 97 us, 88 of them tiles and 9 the join, against 92 from 16 bits (83 and 9):
//     the tiles are not bound by memory, the conversion and the products take turns within a workgroup, and each of a
//     KV head's workgroups (four here, two of a tree of 60 nodes) converts every tile for itself.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "cea_lds_dma.hpp"
#include "paged.hpp"

namespace cea {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_ptr;

template <typename T> struct Mfma;
template <> struct Mfma<bf16> {
  typedef bf16x8 frag;
  static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};
template <> struct Mfma<f16> {
  typedef f16x8 frag;
  static __device__ __forceinline__ f32x16 run(frag a, frag b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
// bit patterns of the 16-bit types: exponent all ones (infinity; above it a NaN), and 1
template <typename T> struct Bits16;
template <> struct Bits16<bf16> { static constexpr uint16_t kInf = 0x7f80, kOne = 0x3f80; };
template <> struct Bits16<f16> { static constexpr uint16_t kInf = 0x7c00, kOne = 0x3c00; };

constexpr int NWAVES = 4;
constexpr int NTHREADS = NWAVES * 64;
constexpr int BM = NWAVES * 32;       // query rows per workgroup
constexpr int BN = kTileKeys;         // keys per tile
constexpr int WROWS = BN / NWAVES;    // rows of a tile that a wave loads
constexpr int PASS = 256;             // tiles of a pass: their page indices (and list) are in LDS
static_assert(PASS <= NTHREADS, "a thread looks at one tile of a pass");
constexpr int32_t kHidden32 = INT32_MAX;  // no key; visible positions end below it
constexpr float kRescaleLog2 = 8.0f;

struct ChunkParams {
  PagedParams p;
  const TileInfo* tiles;     // with positions in the pool: [B, ntiles] summaries (pad[0]: some position
  const int32_t* pos32;      // does not fit 31 bits), and [B, ntiles, 2, 64]: positions, kHidden32 where no
                             // key, and what a score starts with: 0, or -inf where no key
  int32_t ntiles;
  int32_t hp;                // query heads of a workgroup: 1, 2, 4
  int32_t splits;            // rows may be cut into key splits: at most so many splits in all (0: no)
  int32_t runs;              // > 0: or the tiles of all rows into so many runs, as their number on the device says
  int32_t kv_units;          // units of query heads that share keys: KV heads (or all heads)
  float* part;               // partial results of the splits: [splits, Sq, Hq, D] and [splits, Hq, Sq]
  float* part_lse;
  int32_t order_units, order_per_kv;  // workgroup columns that an XCD works through together
  int32_t page16;
  uint32_t magic;            // ceil(2^32 / page16), for page16 > 1
  uint8_t kv[kPagedMapHeads];
};

// LDS: two stages of a tile's K, V and positions; with 8-bit pages one tile of 16-bit rows, the positions twice,
// and every wave's rows as they are in the pool (K, V, then their scale bytes).
template <int D, int VIS, bool F8> struct Layout {
  static constexpr int KROW = D * 2;
  static constexpr int NCG = D / 8;
  static constexpr int K_BYTES = BN * KROW;
  static constexpr int V_BYTES = BN * KROW;
  static constexpr int POS_BYTES = VIS == kPosition ? BN * 8 : 0;
  static constexpr int STAGE_BYTES = K_BYTES + V_BYTES + POS_BYTES;
  static constexpr int SRC_ROW = F8 ? D : KROW;  // bytes of a row in the pool
  static constexpr int SRC_NCG = SRC_ROW / 16;
  static constexpr int RAW_TILE = WROWS * D;
  static constexpr int RAW_WAVE = 2 * RAW_TILE + 2 * WROWS;
  static constexpr int RAW = K_BYTES + V_BYTES + 2 * POS_BYTES;
  static constexpr int LDS_BYTES = F8 ? RAW + NWAVES * RAW_WAVE : 2 * STAGE_BYTES;
  static constexpr int KV_LOADS = WROWS * SRC_ROW / 1024;
  static constexpr int ROWS_PER_LOAD = 1024 / SRC_ROW;
  static_assert(KV_LOADS * ROWS_PER_LOAD == WROWS && WROWS == 16, "a wave loads 16 rows, which lie in one page");
  static constexpr int stage(int i) { return F8 ? 0 : i * STAGE_BYTES; }
  static constexpr int pos(int i) { return K_BYTES + V_BYTES + i * (F8 ? POS_BYTES : STAGE_BYTES); }
};

template <int D> __device__ __forceinline__ int k_swz(int key) {
  if constexpr (D / 8 >= 16) return key & 15;
  else return (key >> 1) & 7;
}
template <int D> __device__ __forceinline__ int v_swz(int key) {
  if constexpr (D == 128) return key & 3;
  else return (key >> 1) & 1;
}

template <typename F>
__device__ __forceinline__ F read_tr_frag(const char* a0, const char* a1) {
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)a0);
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)a1);
  F f;
  __builtin_memcpy(&f, &lo, 8);
  __builtin_memcpy((char*)&f + 8, &hi, 8);
  return f;
}
__device__ __forceinline__ float max3f(float a, float b, float c) {
  return __builtin_fmaxf(a, __builtin_fmaxf(b, c));
}
__device__ __forceinline__ float max_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}
__device__ __forceinline__ int wave_min_i32(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = min(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ int wave_max_i32(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = max(v, __shfl_xor(v, off, 64));
  return v;
}
typedef const int64_t __attribute__((address_space(4))) * scalar_i64;  // read through the scalar cache

// A wave-uniform value in scalar registers, whatever the compiler makes of where it came from.
template <typename X> __device__ __forceinline__ X scalar(X v) {
  if constexpr (sizeof(X) == 4) {
    return (X)__builtin_amdgcn_readfirstlane((int)v);
  } else {
    const uint64_t x = (uint64_t)v;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
    const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32));
    return (X)(((uint64_t)hi << 32) | lo);
  }
}

// Key splits: row b's tiles are cut into as many equal runs as they are worth where the tiles of all rows
// make 512 workgroups (at least 4 tiles each: a split costs its start and its part of the join),
// whatever the rows' lengths.  The splits of all rows are one line.  (us, 384 / 512 / 640 / 768 workgroups:
// four chunks of 300 over 700 to 4001 keys, 32/4 heads of 64, 54.6 / 52.4 / 56.7 / 56.2; 6 tokens of 8 rows of 100
// to 4096, 32/8 heads of 128, - / 25.4 / - / 33.8; 128 tokens over 32768 - / 93.5 / - / 94.7)
constexpr int kSplitWgs = 512, kSplitTiles = 4;
// Trees and 8-bit pages are cut from tables of kCutTiles on (18 trees of 59 nodes after up to 457 slots, 8 tiles, 16.9 us
// whole, 26.0 cut; one of 26 nodes after 777, 13 tiles, 18.7 and 15.0), and into runs where these have kRunTiles tiles.
// kCutTiles is compared with the table's width, which the host knows: short rows in a wide table are cut (18 trees of 59
// after up to 457 slots of 8 bits, 32/8 heads of 128: 31 us in a table of 9 tiles, 46 in one of 128).  Both constants lie
// between the few calls that are named here, not on a law.
constexpr int kCutTiles = 12, kRunTiles = 16;
struct Split {
  int b, split, first, count;  // a row, one of its splits, the place of its first one, how many it has
};

__device__ __forceinline__ int scan64(int v) {  // inclusive prefix sum over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int x = __shfl_up(v, off, 64);
    if (lane >= off) v += x;
  }
  return v;
}

// Runs, for trees and 8-bit pages: the tiles of all rows are one line (a row without keys has one, for its result),
// cut into equal runs, whatever the rows' lengths; a run may span several rows.  Part r + b of the partial results
// is what run r has of row b.  Splits of rows one by one are as uneven as the rows, but none starts a second row,
// which counts where they are short.  (us, splits / runs: 16 trees of 60 nodes after 500 to 8192 slots of 8 bits,
// 32/8 heads of 128, 34 tiles a run, 144 / 125; 9 tokens of 5 rows of 13245, 16 tiles, 79 / 60; two trees of 90
// after up to 9715, 14 tiles, 45.0 / 48.3; four of 51 after up to 3566, 4 tiles, 35 / 40.)
struct Line {
  int total, run, more;  // tiles, of a run, runs with one more
  int mine, sums;        // this lane's row of the first 64: its tiles, and their prefix sum
  __device__ __forceinline__ bool by_runs() const { return run >= kRunTiles; }  // (else by splits)
  __device__ __forceinline__ int start(int r) const { return r * run + min(r, more); }
  __device__ __forceinline__ int run_of(int at) const {
    const int big = more * (run + 1);
    return at < big ? at / (run + 1) : more + (at - big) / run;
  }
};
__device__ __forceinline__ int row_tiles(const PagedParams& p, int b) {
  return b < p.B ? ((int)paged_slots(p, b) + BN - 1) / BN : 0;
}
__device__ __forceinline__ int line_tiles(const PagedParams& p, int b) { return b < p.B ? max(1, row_tiles(p, b)) : 0; }
__device__ __forceinline__ Line line_of(const ChunkParams& c_) {
  const int lane = threadIdx.x & 63;
  Line l;
  l.mine = line_tiles(c_.p, lane);
  l.sums = scan64(l.mine);
  l.total = __builtin_amdgcn_readlane(l.sums, 63);
  for (int b0 = 64; b0 < c_.p.B; b0 += 64) l.total += wave_sum_i32(line_tiles(c_.p, b0 + lane));
  l.total = uniform(l.total);
  l.run = c_.runs > 0 ? uniform(l.total / c_.runs) : 0;
  l.more = l.total - l.run * c_.runs;
  return l;
}
// The split at place `at` (count 0 past the line's end), or with at < 0 row `b`'s.  per_row: workgroups of a
// row's split; mine, total: the tiles of this lane's row of the first 64, and of all.
__device__ __forceinline__ Split find_split(const ChunkParams& c, int per_row, int at, int b, int mine, int total) {
  const PagedParams& p = c.p;
  const int lane = threadIdx.x & 63;
  auto tiles_of = [&](int row) { return row_tiles(p, row); };
  int per = (int)max(((int64_t)total * per_row + kSplitWgs - 1) / kSplitWgs, (int64_t)kSplitTiles);
  Split r = {0, 0, 0, 0};
  int before = 0;
  for (int b0 = 0; b0 < p.B; b0 += 64) {
    const int tiles = b0 == 0 ? mine : tiles_of(b0 + lane);
    const int n = b0 + lane < p.B ? max(1, min((tiles + per - 1) / per, kMaxKeySplits)) : 0;
    const int sums = scan64(n);
    const uint64_t found = at >= 0 ? __ballot(before + sums > at) : (b - b0 < 64 ? 1ull << (b - b0) : 0ull);
    if (found != 0) {
      const int l = (int)__builtin_ctzll(found);
      r.b = b0 + l;
      r.count = __builtin_amdgcn_readlane(n, l);
      r.first = before + __builtin_amdgcn_readlane(sums, l) - r.count;
      r.split = at - r.first;
      break;
    }
    before += __builtin_amdgcn_readlane(sums, 63);
  }
  return r;
}

// Summaries and 32-bit positions of a row's tiles, a wave per tile; the row's length, not the table's
// width, decides how many there are.
__global__ __launch_bounds__(256) void paged_tile_info_kernel(const PagedParams p, int ntiles, TileInfo* out,
                                                              int32_t* pos32) {
  const int b = blockIdx.y, lane = threadIdx.x & 63;
  const int n = (int)paged_slots(p, b);
  for (int t = blockIdx.x * 4 + (threadIdx.x >> 6); t * BN < n; t += gridDim.x * 4) {
    const int j = t * BN + lane;
    int64_t pos = -1;
    if (j < n) {
      const int pg = j / p.page, place = j - pg * p.page;
      const int64_t id = p.tables[b * p.ts_b + pg * p.ts_w];
      if (id >= 0 && id < p.P) pos = p.pos[id * p.ps_p + place];
    }
    const bool valid = pos >= 0, wide = pos >= kHidden32;
    const int64_t mn = wave_min_i64(valid ? pos : INT64_MAX);
    const int64_t mx = wave_max_i64(valid ? pos : INT64_MIN);
    const uint64_t some = __ballot(valid), far = __ballot(wide);
    const int64_t at = (int64_t)b * ntiles + t;
    pos32[at * (2 * BN) + lane] = valid && !wide ? (int32_t)pos : kHidden32;
    pos32[at * (2 * BN) + BN + lane] = valid ? 0 : (int32_t)0xff800000u;
    if (lane == 0) {
      TileInfo ti;
      ti.min_valid = mn;
      ti.max_valid = mx;
      ti.n_valid = __builtin_popcountll(some);
      ti.pad[0] = far != 0 ? 1 : 0;
      ti.pad[1] = ti.pad[2] = 0;
      out[at] = ti;
    }
  }
}

constexpr int kTreeWords = CEA_MAX_TREE / 64;

template <int VIS> struct Shared {
  int64_t red_max[NWAVES], red_min[NWAVES];  // what the waves' rows see
  int red_act[NWAVES], wave_cnt[NWAVES];
  int lost[NWAVES];                          // a page of the pass that is not there, by finder
  int odd_result;                            // a result that is not finite; the first pass's alone
  uint32_t marks[PASS / 32];                 // tiles that hold a value that is not finite
  int32_t ids[PASS * BN / 16];               // page indices of the pass, -1 where none
  int2 tile_list[VIS == kPosition ? PASS : 1];  // (tile, 2-bit mode of every wave)
  uint64_t words[VIS == kTree ? BM * kTreeWords : 1];  // the rows' masks
};

__device__ __forceinline__ Split find_split(const ChunkParams& c, int per_row, int at, int b) {
  const int lane = threadIdx.x & 63, mine = row_tiles(c.p, lane);
  int total = wave_sum_i32(mine);
  for (int b0 = 64; b0 < c.p.B; b0 += 64) total += wave_sum_i32(row_tiles(c.p, b0 + lane));
  return find_split(c, per_row, at, b, mine, total);
}

// What a workgroup does at a time: query block qb of head group hg of row b over a split of the row's tiles, or
// over tiles [from, to).  Of a row that is cut the results go to part `place`.
struct Job {
  int qb, b, hg, split, nsplit, from, to, place;
  bool cut;
};
struct Grid {
  int nqb, ngroups;  // query blocks, head groups
};
__device__ __forceinline__ Grid grid_of(const ChunkParams& c_) {
  const int hp_log2 = __builtin_ctz(c_.hp), rows_pb = BM >> hp_log2;
  return {(c_.p.Sq + rows_pb - 1) >> (__builtin_ctz(BM) - hp_log2), c_.p.Hq >> hp_log2};
}

// The job of a workgroup over the 8 XCDs, as the prefill kernel's: KV heads are dealt to the XCDs in turn, an
// XCD takes as many query heads together as its L2 holds the keys of and starts the latest query
// blocks, which see the most, of all of them first; splits are slowest.  (nsplit 0: past the line of splits)
template <bool LINE> __device__ __forceinline__ Job job_of(const ChunkParams& c_, const Line& line) {
  const PagedParams& p = c_.p;
  const Grid x = grid_of(c_);
  const int nqb = x.nqb, ngroups = x.ngroups, units = ngroups * p.B;
  int blk = blockIdx.x, split = 0, nsplit = 1, place = 0, qb, b, hg;
  if (c_.splits > 0) {
    // (split, KV head) in turn over the XCDs, the workgroups that share its keys together
    const int per_kv = ngroups / c_.kv_units, shared = per_kv * nqb;
    const int i = blk >> 3, set = i / shared, in = i - set * shared;
    const int u = uniform(set * 8 + (blk & 7));
    place = u / c_.kv_units;
    Split x;
    if constexpr (LINE) x = find_split(c_, nqb * ngroups, place, 0, line.mine, line.total);
    else x = find_split(c_, nqb * ngroups, place, 0);
    b = x.b, split = x.split, nsplit = x.count;
    qb = nqb - 1 - in / per_kv;
    hg = (u - place * c_.kv_units) * per_kv + in % per_kv;
  } else {
    int unit;
    if (nqb == 1) {
      qb = 0;
      unit = (units & 7) == 0 ? (blk & 7) * (units >> 3) + (blk >> 3) : blk;
    } else if ((units & 7) == 0) {
      const int per_xcd = units >> 3, i = blk >> 3;
      const int set = c_.order_units == per_xcd ? 0 : i / (c_.order_units * nqb);
      const int x = i - set * c_.order_units * nqb;
      const int size = min(c_.order_units, per_xcd - set * c_.order_units);
      qb = x / size;
      const int per_kv = c_.order_per_kv;
      const int turn = per_kv % 4 != 0 && size % 2 == 0 ? qb >> 1 : 0;
      int u = x - qb * size;
      if (turn != 0) u = (u + turn) % size;
      u += set * c_.order_units;
      if (p.group > 0 && ((p.B * p.Hkv) & 7) == 0) {
        const int kv = per_kv == 1 ? u : u / per_kv;
        unit = ((blk & 7) + 8 * kv) * per_kv + (u - kv * per_kv);
      } else {
        unit = (blk & 7) * per_xcd + u;
      }
    } else {
      qb = blk / units;
      unit = blk - qb * units;
    }
    qb = nqb - 1 - qb;
    b = p.B == 1 ? 0 : unit / ngroups;
    hg = unit - b * ngroups;
  }
  Job job;
  job.qb = uniform(qb), job.b = uniform(b), job.hg = uniform(hg), job.split = uniform(split);
  job.nsplit = uniform(nsplit), job.place = uniform(place);
  job.from = job.to = 0;
  job.cut = nsplit > 1;
  return job;
}

// The row that holds tile `at` of the line, or with at < 0 row b: its place, and its tiles.
struct LineRow {
  int b, first, tiles;
};
__device__ __forceinline__ LineRow line_row(const ChunkParams& c_, const Line& l, int at, int b) {
  const int lane = threadIdx.x & 63;
  LineRow r = {0, 0, 1};
  int before = 0;
  for (int b0 = 0; b0 < c_.p.B; b0 += 64) {
    const int sums = b0 == 0 ? l.sums : scan64(line_tiles(c_.p, b0 + lane));
    const uint64_t found = at >= 0 ? __ballot(before + sums > at) : (b - b0 < 64 ? 1ull << (b - b0) : 0ull);
    if (found != 0) {
      const int k = (int)__builtin_ctzll(found);
      const int begin = k > 0 ? __builtin_amdgcn_readlane(sums, k - 1) : 0;
      r = {b0 + k, before + begin, __builtin_amdgcn_readlane(sums, k) - begin};
      break;
    }
    before += __builtin_amdgcn_readlane(sums, 63);
  }
  return r;
}

// PIECES: 16-bit numbers whose sum enters the value product for a probability: one for 16-bit results
// (p rounded once, half a step of the type, as the result's own rounding is), three of bf16 or two of f16
// for f32 results (p to 2^-23 and better; f16's to 2^-32 where p is below 2^-9).  2-norm errors against 64 bits and us, one piece / f32 results: 128 bf16
// tokens over 32768 keys 2.3e-3, 91 / 6.8e-7, 136 (rounded to bf16 1.7e-3); two prompts of 2000 2.1e-3, 83 / 2.3e-7,
// 125; four f16 chunks of 300 with positions 2.9e-4, 58 / 3.2e-7, 80.
// AGAIN: over the tiles a second time, after values that are not finite.  Returns whether that is needed
// (nothing has been written then).
template <typename T, int D, int VIS, int PIECES, bool F8, bool AGAIN>
__device__ __forceinline__ bool chunk_body(const ChunkParams& c_, const Job& job, char* smem, Shared<VIS>& sh) {
  typedef Layout<D, VIS, F8> L;
  constexpr bool POS = VIS == kPosition, TREE = VIS == kTree;
  constexpr int kSize = F8 ? 1 : 2;  // bytes of an element of the pages
  typedef typename Mfma<T>::frag frag;
  const PagedParams& p = c_.p;
  int tid = threadIdx.x;
  // (what follows from the thread's number is computed again for every row of a run: kept across them it took 55
  // registers too many)
  if constexpr (TREE || F8) asm volatile("" : "+v"(tid));
  const int wave = uniform(tid >> 6), lane = tid & 63;
  const int r = lane & 31, g = lane >> 5;

  const int hp_log2 = __builtin_ctz(c_.hp), hp = 1 << hp_log2;
  const int rows_pb = BM >> hp_log2;
  const int qb = job.qb, b = job.b, hg = job.hg;
  const int waves_log2 = __builtin_ctz(NWAVES) - hp_log2;  // waves of one head
  const int h = hg * hp + (wave >> waves_log2);
  const int kvh = p.group > 0 ? hg * hp / p.group : c_.kv[hg * hp];
  const int row = qb * rows_pb + (wave & ((1 << waves_log2) - 1)) * 32 + r;
  const bool row_ok = row < p.Sq;
  // ---- everything that the start reads is under way before any of it is used: positions and queries, the
  // row's length through the scalar cache, then the first pass's page indices, which the length alone decides
  const int64_t qpos = row_ok && !TREE ? p.q_pos[b * p.qps_b + (int64_t)row * p.qps_s] : -1;
  uint4 qraw[D / 16];
  {
    const T* qrow = (const T*)p.q + b * p.qs_b + (int64_t)row * p.qs_s + h * p.qs_h;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
      qraw[ks] = make_uint4(0, 0, 0, 0);
      if (row_ok) qraw[ks] = *(const uint4*)(qrow + ks * 16 + g * 8);
    }
  }
  const int64_t len = ((scalar_i64)(uintptr_t)p.lengths)[b * p.ns_b];
  const int n = scalar((int)max((int64_t)0, min(len, (int64_t)p.W * p.page)));
  const int page16 = scalar(c_.page16);
  const uint32_t magic = scalar(c_.magic);
  auto page_of = [&](int slot) -> int {
    const uint32_t u = (uint32_t)slot >> 4;
    return (int)(page16 == 1 ? u : __umulhi(u, magic));
  };
  // this job's part of the row's tiles (what its queries cannot see is left out below)
  const int tiles_here = (n + BN - 1) / BN;
  int t_first, t_last;
  if (!(TREE || F8) || job.nsplit > 0) {
    const int per_split = job.nsplit > 1 ? (tiles_here + job.nsplit - 1) / job.nsplit : tiles_here;
    t_first = scalar(min(tiles_here, job.split * per_split));
    t_last = scalar(min(tiles_here, t_first + per_split));
  } else {
    t_first = scalar(min(tiles_here, job.from));
    t_last = scalar(min(tiles_here, job.to));
  }

  // the page indices and summaries of a pass, from memory to registers and from there to LDS
  constexpr int kIdsPer = PASS * BN / 16 / NTHREADS;
  struct PassRegs {
    int64_t id[kIdsPer];
    TileInfo ti;
  };
  int pg0 = 0;  // page of the pass's first slot
  auto fetch_pass = [&](int base, int last, PassRegs& x) {
    const int span = min(PASS, last - base);
    pg0 = page_of(base * BN);
    const int npg = span > 0 ? page_of(min((base + span) * BN, n) - 1) - pg0 + 1 : 0;
    const int64_t* tab = p.tables + b * p.ts_b + pg0 * p.ts_w;
#pragma unroll
    for (int i = 0; i < kIdsPer; ++i) {
      x.id[i] = 0;
      if (i * NTHREADS + tid < npg) x.id[i] = tab[(int64_t)(i * NTHREADS + tid) * p.ts_w];
    }
    if constexpr (POS)
      if (tid < span) x.ti = c_.tiles[(int64_t)b * c_.ntiles + base + tid];
  };
  PassRegs regs;
  if constexpr (!POS) fetch_pass(t_first, t_last, regs);

  // ---- what the rows see: slots [0, lim) of this lane's row by their number (POS: positions to qpos)
  // (a tree's: every slot before it, and from there on what the mask says)
  int base = 0;  // slot of the tree's first node
  bool sees;
  int lim;
  if constexpr (TREE) {
    const TreeOf tree = tree_of(p, b);
    base = scalar((int)max(tree.base, -((int64_t)1 << 30)));
    sees = row_ok && row < (int)tree.nodes;
    lim = sees ? max(base, 0) : 0;
    if constexpr (!AGAIN) {
      const int words = (p.Sq + 63) >> 6;
      for (int x = tid; x < rows_pb * words; x += NTHREADS) {
        const int i = x / words, w = x - i * words;
        sh.words[i * kTreeWords + w] = qb * rows_pb + i < p.Sq ? tree_word(p, b, qb * rows_pb + i, w) : 0;
      }
    }
  } else {
    sees = row_ok && (!p.causal || qpos >= 0);
    lim = !sees ? 0 : p.causal && !POS && qpos < n ? (int)qpos + 1 : n;
  }
  int lim_min = 0, lim_max = 0;  // of the wave's rows that see anything
  if constexpr (POS) {
    const int64_t mn = wave_min_i64(sees ? qpos : INT64_MAX), mx = wave_max_i64(sees ? qpos : INT64_MIN);
    const bool act = __ballot(sees) != 0;
    if (lane == 0) sh.red_max[wave] = mx, sh.red_min[wave] = mn, sh.red_act[wave] = act ? 1 : 0;
  } else {
    lim_min = uniform(wave_min_i32(lim > 0 || (TREE && sees) ? lim : INT32_MAX));
    lim_max = uniform(wave_max_i32(TREE ? (sees ? n : 0) : lim));
    if (lane == 0) sh.red_max[wave] = lim_max;
  }
  // (the first time alone: a wave that is late to read what the first pass found shares this word with waves
  // that are in the second already, and no barrier lies between)
  if constexpr (!AGAIN)
    if (tid == 0) sh.odd_result = 0;

  const float scale = (float)p.scale;
  const float c = fabsf(scale) * 1.4426950408889634f;
  const float grow_thr = kRescaleLog2 / c;
  const uint32_t krow = scalar((uint32_t)(p.ks_s * kSize)), vrow = scalar((uint32_t)(p.vs_s * kSize));
  uint32_t k_voff[L::KV_LOADS], v_voff[L::KV_LOADS];
#pragma unroll
  for (int i = 0; i < L::KV_LOADS; ++i) {
    const int local = i * L::ROWS_PER_LOAD + lane / L::SRC_NCG, key = wave * WROWS + local;
    const int pg = lane % L::SRC_NCG;  // physical 16-byte group in the row
    const int lgv = (((pg >> 2) ^ v_swz<D>(key)) << 2) | (pg & 3);
    k_voff[i] = local * krow + ((F8 ? pg : pg ^ k_swz<D>(key)) << 4);
    v_voff[i] = local * vrow + ((F8 ? pg : lgv) << 4);
  }
  // fragment reads: the swizzles are exclusive ors of bits that the features' offsets have to themselves
  const uint32_t k_read0 = r * L::KROW + ((g ^ k_swz<D>(r)) << 4);
  uint32_t v_read0;
  {
    const int src = lane & 15, grp = lane >> 4;
    const int vr = g * 4 + (src >> 2);
    v_read0 = L::K_BYTES + vr * L::KROW + (v_swz<D>(vr) << 6) + (16 * (grp & 1) + 4 * (src & 3)) * 2;
  }
  const uint32_t smem_lds = lds_addr(smem);
  const uint32_t wave_kv = wave * (L::KV_LOADS * 1024);
  const char* kh = scalar((const char*)p.k + (int64_t)kvh * p.ks_h * kSize);
  const char* vh = scalar((const char*)p.v + (int64_t)kvh * p.vs_h * kSize);
  const int64_t ks_p = scalar(p.ks_p * kSize), vs_p = scalar(p.vs_p * kSize);
  char* raw = smem + L::RAW + wave * L::RAW_WAVE;  // this wave's rows of 8-bit pages
  const uint8_t* ksh = F8 ? scalar(p.k_scales + kvh * p.kss_h) : nullptr;
  const uint8_t* vsh = F8 ? scalar(p.v_scales + kvh * p.vss_h) : nullptr;
  const uint32_t kss_p = F8 ? scalar((uint32_t)p.kss_p) : 0, vss_p = F8 ? scalar((uint32_t)p.vss_p) : 0;
  const int32_t* pos32 = POS ? scalar(c_.pos32 + (int64_t)b * c_.ntiles * (2 * BN)) : nullptr;

  // the page index of this wave's rows of a tile (behind the row's end: the last one's)
  auto id_of = [&](int tile) -> int { return sh.ids[page_of(min(tile * BN + wave * WROWS, n - 1)) - pg0]; };
  auto load_tile = [&](int tile, int id, int stage) {
    const int slot = tile * BN + wave * WROWS;
    const int rows = min(n - slot, WROWS);  // rows behind the row's end, and of no page, read 0
    const bool ok = id >= 0 && rows > 0;
    const int at = ok ? id : 0;
    const int place = ok ? slot - page_of(slot) * (page16 * 16) : 0;
    const int64_t at_k = F8 ? (int64_t)((uint64_t)(uint32_t)at * (uint32_t)ks_p) : at * ks_p;
    const int64_t at_v = F8 ? (int64_t)((uint64_t)(uint32_t)at * (uint32_t)vs_p) : at * vs_p;
    const i32x4 krs = make_rsrc(kh + at_k + (int64_t)place * krow, ok ? (uint32_t)(rows - 1) * krow + L::SRC_ROW : 0u);
    const i32x4 vrs = make_rsrc(vh + at_v + (int64_t)place * vrow, ok ? (uint32_t)(rows - 1) * vrow + L::SRC_ROW : 0u);
    const uint32_t stage_lds = smem_lds + L::stage(stage);
    const uint32_t st = F8 ? smem_lds + L::RAW + wave * L::RAW_WAVE : stage_lds;
    const uint32_t k_at = F8 ? 0 : wave_kv;
    constexpr int kVAt = F8 ? L::RAW_TILE : L::K_BYTES;
#pragma unroll
    for (int i = 0; i < L::KV_LOADS; ++i) buffer_load_lds16_m0(krs, st + k_at + i * 1024, k_voff[i]);
#pragma unroll
    for (int i = 0; i < L::KV_LOADS; ++i) buffer_load_lds16_m0(vrs, st + kVAt + k_at + i * 1024, v_voff[i]);
    if constexpr (F8) {  // (the scale bytes of all 16 slots, which their page holds whatever the row's length)
      const uint64_t sk = (uint64_t)ksh + (uint64_t)(uint32_t)at * kss_p + place;
      const uint64_t sv = (uint64_t)vsh + (uint64_t)(uint32_t)at * vss_p + place;
      if (lane < 2) global_load_lds16_m0(lane == 0 ? sk : sv, st + 2 * L::RAW_TILE);
    }
    if constexpr (POS) {
      if (wave == 0) {
        const i32x4 prs = make_rsrc(pos32 + (int64_t)tile * (2 * BN), BN * 8);
        if (lane < BN / 2) buffer_load_lds16_m0(prs, (F8 ? smem_lds + L::pos(stage) : stage_lds + L::pos(0)), lane * 16);
      }
    }
  };
  // 8-bit pages: this wave's rows of the tile that has landed, as 16-bit rows at their place in the tile.  Rows
  // behind the row's end and of no page are 0, whatever their scale bytes.
  auto widen = [&](int tile) {
    const int rows = n - (tile * BN + wave * WROWS);
    const bool ok = scalar(id_of(tile)) >= 0;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv)
#pragma unroll
      for (int i = 0; i < L::KV_LOADS; ++i) {
        const int local = i * L::ROWS_PER_LOAD + lane / L::SRC_NCG, key = wave * WROWS + local;
        const uint4 x = *(const uint4*)(raw + kv * L::RAW_TILE + i * 1024 + lane * 16);
        const uint32_t s = ok && local < rows ? *(const uint8_t*)(raw + 2 * L::RAW_TILE + kv * WROWS + local) : 127u;
        const float scale8 = scale_value(s);
        const uint4 lo = make_uint4(widen2<T, false>(x.x, scale8), widen2<T, true>(x.x, scale8),
                                    widen2<T, false>(x.y, scale8), widen2<T, true>(x.y, scale8));
        const uint4 hi = make_uint4(widen2<T, false>(x.z, scale8), widen2<T, true>(x.z, scale8),
                                    widen2<T, false>(x.w, scale8), widen2<T, true>(x.w, scale8));
        const int cg = 2 * (lane % L::SRC_NCG);  // logical 16-byte groups of the 16-bit row: cg, cg + 1
        char* dst = smem + (kv ? L::K_BYTES : 0) + key * L::KROW;
        auto group = [&](int g16) {
          return kv ? ((((g16 >> 2) ^ v_swz<D>(key)) << 2) | (g16 & 3)) << 4 : (g16 ^ k_swz<D>(key)) << 4;
        };
        *(uint4*)(dst + group(cg)) = lo;
        *(uint4*)(dst + group(cg + 1)) = hi;
      }
  };

  // f16 takes 2^7 p, so small probabilities stay normal numbers: with one piece through the exponent (l
  // holds the factor too), with two as a product, which costs small scores no bits.  bf16 takes 2^-8 p over pages of
  // 8 bits, whose values reach 2^128: p is up to 2^8 before the maximum follows.
  constexpr bool kF16 = std::is_same<T, f16>::value;
  constexpr float kShift = kF16 ? 7.f : F8 ? -kRescaleLog2 : 0.f;
  constexpr float kExpShift = PIECES == 1 ? kShift : 0.f;
  constexpr float kPieceScale = PIECES == 1 ? 1.f : kF16 ? 128.f : F8 ? 1.f / 256 : 1.f;
  frag qf[D / 16];
  f32x16 oacc[D / 32];
  float m_run = -__builtin_inff(), m_use = -kExpShift, l_run = 0.f;

  // the 64 keys from slot0 on that this lane's row sees, by its mask
  auto window = [&](int slot0) -> uint64_t {
    const int off = slot0 - base, words = (p.Sq + 63) >> 6;
    const uint64_t* mine = sh.words + ((wave & ((1 << waves_log2) - 1)) * 32 + r) * kTreeWords;
    uint64_t x;
    if (off < 0) {
      x = off <= -64 ? ~(uint64_t)0 : (((uint64_t)1 << -off) - 1) | (mine[0] << -off);
    } else {
      const int w = off >> 6, sh6 = off & 63;
      x = w < words ? mine[w] >> sh6 : 0;
      if (sh6 != 0 && w + 1 < words) x |= mine[w + 1] << (64 - sh6);
    }
    const int left = n - slot0;
    if (left < 64) x &= ((uint64_t)1 << left) - 1;
    return sees ? x : 0;
  };
  // Which of this lane's keys its row does not see, bit by bit, looked up one by one (rare: the pool's positions
  // are read in place, which waits for every load).
  auto hidden = [&](int slot0) -> uint32_t {
    uint32_t hide = 0;
    uint64_t mask = 0;
    if constexpr (TREE) mask = window(slot0);
#pragma unroll 1
    for (int x = 0; x < 32; ++x) {
      const int slot = slot0 + (x >> 4) * 32 + ((x >> 2) & 3) * 8 + g * 4 + (x & 3);
      bool vis = TREE ? (mask >> (slot - slot0)) & 1 : slot < lim;
      if (vis) {
        const int pg = page_of(slot), id = sh.ids[pg - pg0];
        vis = id >= 0;
        if (POS && vis) {
          const int64_t pos = p.pos[(int64_t)id * p.ps_p + slot - pg * (page16 * 16)];
          vis = pos >= 0 && (!p.causal || pos <= qpos);
        }
      }
      hide |= (vis ? 0u : 1u) << x;
    }
    return hide;
  };
  // The scores of a tile.  mode: 1 every key visible to every row of the wave that sees anything, 2 masked,
  // 3 masked and looked up: a page of the pass that is not there, or (POS) a position beyond 31 bits.  (POS: in
  // mode 1 slots may be empty.  Their scores are -inf plus a product, which is -inf unless the slot holds a value
  // that is not finite; those show up in the results, and the second time over the tiles masks them.)
  const int qlim32 = !sees ? -1 : p.causal ? (int)min(qpos, (int64_t)kHidden32 - 1) : kHidden32 - 1;
  auto scores = [&](int stage, int slot0, int mode, f32x16 (&sacc)[2]) {
    const char* sb = smem + L::stage(stage);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      frag kf[D / 16];
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) kf[ks] = *(const frag*)(sb + kb * 32 * L::KROW + (k_read0 ^ (ks << 5)));
      f32x16 acc = {};
      if constexpr (POS) {  // 0, or -inf where no key
        const char* start = (F8 ? smem + L::pos(stage) : sb + L::pos(0)) + BN * 4 + (kb * 32 + g * 4) * 4;
#pragma unroll
        for (int i4 = 0; i4 < 4; ++i4) {
          const float4 x = *(const float4*)(start + i4 * 32);
          acc[i4 * 4 + 0] = x.x, acc[i4 * 4 + 1] = x.y, acc[i4 * 4 + 2] = x.z, acc[i4 * 4 + 3] = x.w;
        }
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) acc = Mfma<T>::run(kf[ks], qf[ks], acc);
      sacc[kb] = acc;
    }
    __builtin_amdgcn_sched_group_barrier(0x100, D / 16, 0);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, D / 16, 0);

    if (mode == 1) return;
    if (mode == 2) {
      if constexpr (POS) {
        const char* pl = F8 ? smem + L::pos(stage) : sb + L::pos(0);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int i4 = 0; i4 < 4; ++i4) {
            const int4 kp = *(const int4*)(pl + (kb * 32 + i4 * 8 + g * 4) * 4);
            if (kp.x > qlim32) sacc[kb][i4 * 4 + 0] = -__builtin_inff();
            if (kp.y > qlim32) sacc[kb][i4 * 4 + 1] = -__builtin_inff();
            if (kp.z > qlim32) sacc[kb][i4 * 4 + 2] = -__builtin_inff();
            if (kp.w > qlim32) sacc[kb][i4 * 4 + 3] = -__builtin_inff();
          }
      } else if constexpr (TREE) {
        const uint64_t x = window(slot0) >> (g * 4);
        const uint32_t half[2] = {(uint32_t)x, (uint32_t)(x >> 32)};
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (!((half[kb] >> ((e >> 2) * 8 + (e & 3))) & 1u)) sacc[kb][e] = -__builtin_inff();
      } else {
        const int left = lim - slot0 - g * 4;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (kb * 32 + (e >> 2) * 8 + (e & 3) >= left) sacc[kb][e] = -__builtin_inff();
      }
      return;
    }
    const uint32_t hide = hidden(slot0);
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if ((hide >> i) & 1u) sacc[i >> 4][i & 15] = -__builtin_inff();
  };

  auto compute = [&](int stage, int slot0, int mode) {
    const char* sb = smem + L::stage(stage);
    f32x16 sacc[2];
    scores(stage, slot0, mode, sacc);
    float t1[11];
#pragma unroll
    for (int i = 0; i < 10; ++i) {
      const int e = 3 * i;
      t1[i] = max3f(sacc[e >> 4][e & 15], sacc[(e + 1) >> 4][(e + 1) & 15], sacc[(e + 2) >> 4][(e + 2) & 15]);
    }
    t1[10] = __builtin_fmaxf(sacc[1][14], sacc[1][15]);
    const float t2a = max3f(t1[0], t1[1], t1[2]), t2b = max3f(t1[3], t1[4], t1[5]);
    const float t2c = max3f(t1[6], t1[7], t1[8]), t2d = __builtin_fmaxf(t1[9], t1[10]);
    float mx = __builtin_fmaxf(max3f(t2a, t2b, t2c), t2d);
    mx = max_halves(mx);
    const bool grow = mx > m_run + grow_thr;
    if (__ballot(grow) != 0) {
      const float m_new = grow ? mx : m_run;
      const float alpha = grow ? __builtin_amdgcn_exp2f((m_run - m_new) * c) : 1.f;
      m_run = m_new;
      m_use = (m_run == -__builtin_inff() ? 0.f : m_run * c) - kExpShift;
      l_run *= alpha;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) oacc[dt][e] *= alpha;
    }
    frag pf[PIECES][4];
    float pr[32];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        pr[kb * 16 + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sacc[kb][e], c, -m_use));
        float rest = pr[kb * 16 + e] * kPieceScale;
#pragma unroll
        for (int pc = 0; pc < PIECES; ++pc) {
          pf[pc][kb * 2 + (e >> 3)][e & 7] = (T)rest;
          if (pc + 1 < PIECES) rest -= to_f32<T>(pf[pc][kb * 2 + (e >> 3)][e & 7]);
        }
      }
#pragma unroll
    for (int w = 16; w >= 1; w >>= 1)
#pragma unroll
      for (int e = 0; e < w; ++e) pr[e] += pr[e + w];
    l_run += pr[0];
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt) {
      frag vf[4];
#pragma unroll
      for (int s = 0; s < 4; ++s)
        vf[s] = read_tr_frag<frag>(sb + s * 16 * L::KROW + (v_read0 ^ (dt << 6)), sb + (s * 16 + 8) * L::KROW + (v_read0 ^ (dt << 6)));
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int pc = 0; pc < PIECES; ++pc) oacc[dt] = Mfma<T>::run(vf[s], pf[pc][s], oacc[dt]);
    }
    __builtin_amdgcn_sched_group_barrier(0x100, 8, 1);
#pragma unroll
    for (int j = 0; j < D / 32 - 1; ++j) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        __builtin_amdgcn_sched_group_barrier(0x008, PIECES, 1);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x008, 4 * PIECES, 1);
  };

  // ---- the second time over the tiles.  Values that are not finite are taken out of this wave's rows of a
  // tile as they land, and the tile is marked ...
  auto clean_share = [&](int stage, int i) {
    char* v = smem + L::stage(stage) + L::K_BYTES + wave * (WROWS * L::KROW) + lane * 16;
    bool found = false;
#pragma unroll
    for (int l = 0; l < WROWS * L::KROW / 1024; ++l) {
      u16x8 x = *(const u16x8*)(v + l * 1024);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool odd = (x[j] & 0x7fff) >= Bits16<T>::kInf;
        found = found || odd;
        x[j] = odd ? 0 : x[j];
      }
      *(u16x8*)(v + l * 1024) = x;
    }
    if (__ballot(found) != 0 && lane == 0) atomicOr(&sh.marks[i >> 5], 1u << (i & 31));
    wait_lgkmcnt0();  // before the barrier that hands the tile to the other waves
  };
  // ... and a marked tile, V as it is, counts per feature the visible keys with +inf or NaN, then those with
  // -inf or NaN, by products with ones; the sum takes an infinity of that sign (both make a NaN; a
  // visible key of probability 0 counts for both: 0 * inf).
  auto mark = [&](int stage, int slot0) {
    const char* sb = smem + L::stage(stage);
    f32x16 sacc[2];
    scores(stage, slot0, 1, sacc);
    // (a key's score does not say whether it is visible: -inf is a score as well)
    const uint32_t seen = ~hidden(slot0);
    uint32_t none = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = sacc[i >> 4][i & 15];
      none |= (__builtin_amdgcn_exp2f(__builtin_fmaf(x, c, -m_use)) == 0.f ? 1u : 0u) << i;
    }
    none &= seen;
    auto keys = [&](uint32_t bits, int s) {
      u16x8 x;
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = (bits >> (8 * s + j)) & 1 ? Bits16<T>::kOne : 0;
      return __builtin_bit_cast(frag, x);
    };
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int sign = 0; sign < 2; ++sign) {
        __builtin_amdgcn_sched_barrier(0);
        f32x16 count = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const u16x8 x = __builtin_bit_cast(u16x8, read_tr_frag<frag>(sb + s * 16 * L::KROW + (v_read0 ^ (dt << 6)),
                                                                       sb + (s * 16 + 8) * L::KROW + (v_read0 ^ (dt << 6))));
          u16x8 one, any;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint16_t mag = x[j] & 0x7fff;
            any[j] = mag >= Bits16<T>::kInf ? Bits16<T>::kOne : 0;
            one[j] = mag > Bits16<T>::kInf || (x[j] >> 15) == sign ? any[j] : 0;
          }
          count = Mfma<T>::run(__builtin_bit_cast(frag, one), keys(seen, s), count);
          count = Mfma<T>::run(__builtin_bit_cast(frag, any), keys(none, s), count);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          uint32_t add = count[e] > 0.f ? (sign ? 0xff800000u : 0x7f800000u) : 0x80000000u;
          asm volatile("" : "+v"(add));  // the file is compiled as if no NaN occurred
          oacc[dt][e] += __uint_as_float(add);
        }
      }
  };

  // ---- the passes over this run's tiles: the pages' indices (and the list of the tiles needed), then the
  // stream
  int64_t max_wg = 0;
  bool any_wg = !POS;
  auto stream = [&]() {
    for (int base = t_first; base < t_last; base += PASS) {
      if (POS || base != t_first) fetch_pass(base, t_last, regs);
      const int span = min(PASS, t_last - base);
      int nt = span;
      bool lost = false;
#pragma unroll
      for (int i = 0; i < kIdsPer; ++i) {
        const bool ok = (uint64_t)regs.id[i] < (uint64_t)p.P;
        sh.ids[i * NTHREADS + tid] = ok ? (int)regs.id[i] : -1;
        lost = lost || !ok;
      }
      const bool lost_w = __ballot(lost) != 0;
      if (lane == 0) sh.lost[wave] = lost_w ? 1 : 0;
      if (AGAIN && tid < PASS / 32) sh.marks[tid] = 0;
      __syncthreads();
      if (base == t_first) {
        max_wg = sh.red_max[0];
#pragma unroll
        for (int w = 1; w < NWAVES; ++w) max_wg = max(max_wg, sh.red_max[w]);
        if constexpr (POS)
#pragma unroll
          for (int w = 0; w < NWAVES; ++w) any_wg = any_wg || sh.red_act[w] != 0;
        if (!any_wg) t_last = t_first;
        if (!POS) t_last = scalar(min(t_last, ((int)max_wg + BN - 1) / BN));
        if (t_first >= t_last) break;
        nt = min(nt, t_last - base);
      }
      if constexpr (POS) {
        bool need = false;
        int modes = 0;
        if (tid < span) {
          const TileInfo ti = regs.ti;
          need = ti.n_valid > 0 && !(p.causal && max_wg < ti.min_valid);
#pragma unroll
          for (int w = 0; w < NWAVES; ++w) {
            int m;
            if (!sh.red_act[w] || ti.n_valid == 0 || (p.causal && sh.red_max[w] < ti.min_valid)) m = 0;
            else if (!AGAIN && (!p.causal || ti.max_valid <= sh.red_min[w])) m = 1;
            else m = ti.pad[0] ? 3 : 2;
            modes |= m << (2 * w);
          }
        }
        const uint64_t bal = __ballot(need);
        if (lane == 0) sh.wave_cnt[wave] = __builtin_popcountll(bal);
        __syncthreads();
        int off = 0;
        for (int w = 0; w < wave; ++w) off += sh.wave_cnt[w];
        nt = 0;
        for (int w = 0; w < NWAVES; ++w) nt += sh.wave_cnt[w];
        if (need)
          sh.tile_list[off + __builtin_amdgcn_mbcnt_hi((uint32_t)(bal >> 32),
                                                       __builtin_amdgcn_mbcnt_lo((uint32_t)bal, 0))] =
              make_int2(base + tid, modes);
        nt = scalar(nt);
        __syncthreads();
      }
      int lost_any = 0;
      if constexpr (!POS)
#pragma unroll
        for (int w = 0; w < NWAVES; ++w) lost_any |= sh.lost[w];
      const bool bad = !POS && scalar(lost_any) != 0;
      auto tile_of = [&](int i) -> int { return POS ? scalar(sh.tile_list[i].x) : base + i; };
      auto mode_of = [&](int tile, int e) -> int {
        int m;
        if constexpr (POS) m = scalar((e >> (2 * wave)) & 3);
        else m = tile * BN >= lim_max ? 0 : bad ? 3 : (tile + 1) * BN <= lim_min ? 1 : 2;
        return m;
      };
      int issued = 0;
      if (nt > 0) load_tile(tile_of(0), scalar(id_of(tile_of(0))), 0), issued = 1;
      // what the next step needs is read from LDS right after a barrier and used behind that step's work:
      // the tile to load next and its page, the next tile's mode
      int t_load = base, id_load = -1;
      if (issued < nt) t_load = tile_of(issued), id_load = scalar(id_of(t_load));
      int t_cur = base, e_cur = 0;
      if constexpr (POS)
        if (nt > 0) t_cur = tile_of(0), e_cur = sh.tile_list[0].y;
      for (int i = 0; i < nt; ++i) {
        wait_vmcnt<0>();
        if constexpr (F8) {
          wait_lgkmcnt0();
          barrier_no_fence();  // no wave reads tile i-1 any more
          widen(t_cur);
        }
        if constexpr (AGAIN) clean_share(i & 1, i);
        wait_lgkmcnt0();     // tile i-1 is in registers, wherever the compiler puts the products
        barrier_no_fence();  // tile i landed for every wave; the stage of tile i-1 is free
        if (issued < nt) {
          load_tile(t_load, id_load, issued & 1);
          ++issued;
        }
        int2 e_nxt = make_int2(t_cur + 1, 0);
        int l_nxt = t_load, id_nxt = 0;
        if constexpr (POS) {
          e_nxt = sh.tile_list[i + 1 < nt ? i + 1 : i];
          l_nxt = sh.tile_list[issued < nt ? issued : 0].x;
          id_nxt = id_of(scalar(l_nxt));
        } else {
          l_nxt = issued < nt ? base + issued : t_load;
          id_nxt = id_of(l_nxt);
        }
        const int mode = mode_of(t_cur, e_cur);
        if (mode != 0) compute(i & 1, t_cur * BN, mode);
        t_cur = scalar(e_nxt.x);
        e_cur = e_nxt.y;
        t_load = scalar(l_nxt);
        id_load = scalar(id_nxt);
      }
      __syncthreads();  // the next pass rewrites the lists and the stages
      if constexpr (!AGAIN) continue;
      for (int i = 0; i < nt; ++i) {
        if (!((scalar(sh.marks[i >> 5]) >> (i & 31)) & 1)) continue;
        const int tile = tile_of(i);
        load_tile(tile, scalar(id_of(tile)), 0);
        wait_vmcnt<0>();
        if constexpr (F8) widen(tile);
        __syncthreads();
        const int mode = mode_of(tile, POS ? sh.tile_list[i].y : 0);
        if (mode != 0) mark(0, tile * BN);
        __syncthreads();
      }
    }
  };

  if (scale < 0.f) {  // the sign goes into the queries
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
      qraw[ks].x ^= 0x80008000u, qraw[ks].y ^= 0x80008000u, qraw[ks].z ^= 0x80008000u, qraw[ks].w ^= 0x80008000u;
  }
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) __builtin_memcpy(&qf[ks], &qraw[ks], 16);
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) oacc[i][e] = 0.f;
  stream();
  if constexpr (!AGAIN) {
    uint32_t worst = 0;
#pragma unroll
    for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
      for (int e = 0; e < 16; ++e) worst = max(worst, __float_as_uint(oacc[dt][e]) & 0x7fffffffu);
    if (__ballot(sees && worst >= 0x7f800000u) != 0 && lane == 0) sh.odd_result = 1;
    __syncthreads();
    if (sh.odd_result != 0) return true;
  }

  // ---- epilogue.  A row's sum is 0 exactly where it saw no key (a NaN is kept).
  if (!row_ok) return false;
  const float l_tot = sum_halves(l_run);
  uint32_t l_bits = __float_as_uint(l_tot);
  asm volatile("" : "+v"(l_bits));  // (compared as a float, a NaN might be taken for 0 in this file)
  const bool empty = !sees || (l_bits << 1) == 0;
  const float inv = empty ? 0.f : 1.f / (l_tot * kPieceScale);
  if ((p.lse || job.cut) && g == 0) {
    float* lp = job.cut ? c_.part_lse + ((int64_t)job.place * p.Hq + h) * p.Sq + row
                           : (float*)p.lse + b * p.ls_b + h * p.ls_h + (int64_t)row * p.ls_s;
    *lp = empty ? -__builtin_inff() : (m_run * fabsf(scale) + logf(l_tot)) - kExpShift * 0.69314718055994531f;
  }
  const int64_t orow = job.cut ? (((int64_t)job.place * p.Sq + row) * p.Hq + h) * D
                                  : b * p.os_b + (int64_t)row * p.os_s + h * p.os_h;
  float* fout = job.cut ? c_.part : p.out_dtype == CEA_F32 ? (float*)p.out : nullptr;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int i4 = 0; i4 < 4; ++i4) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = empty ? 0.f : oacc[dt][i4 * 4 + j] * inv;
      const int64_t at = orow + dt * 32 + i4 * 8 + g * 4;
      if (fout) {
        *(float4*)(fout + at) = make_float4(x[0], x[1], x[2], x[3]);
      } else {
        const T v4[4] = {(T)x[0], (T)x[1], (T)x[2], (T)x[3]};
        uint2 raw;
        __builtin_memcpy(&raw, v4, 8);
        *(uint2*)((T*)p.out + at) = raw;
      }
    }
  return false;
}

// The second time over the tiles is a function of its own, so its registers are not those of the first.
typedef const void __attribute__((address_space(4))) * kernel_args_ptr;
typedef __attribute__((address_space(3))) char* lds_ptr;
template <typename T, int D, int VIS, int PIECES, bool F8>
__device__ __noinline__ void chunk_again(kernel_args_ptr args, Job job, lds_ptr smem, lds_ptr sh) {
  chunk_body<T, D, VIS, PIECES, F8, true>(*(const ChunkParams*)args, job, (char*)smem, *(Shared<VIS>*)(char*)sh);
}

// Three waves a SIMD at D = 64 and one piece leave 168 registers, of which the form with positions spills 5 (four
// chunks of 300 over 700 to 4001 slots: 60.6 us so, 70.7 with two waves and none), over pages of 8 bits 14; other forms
// spill up to 6 (positions, 8 bits, D = 128) and mostly 0 or 1.  Scalar registers that go to vector ones: none in 16-bit
// sequences, 10 to 13 in their trees; over 8 bits 15 to 27 in trees, 44 to 52 by number, 78 to 82 with positions.
template <typename T, int D, int VIS, int PIECES, bool F8>
__global__ __launch_bounds__(NTHREADS, D == 64 && PIECES == 1 ? 3 : 2) void paged_chunk_kernel(const ChunkParams c_) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ Shared<VIS> sh;
  auto work = [&](const ChunkParams& args, const Job& job) {
    if (chunk_body<T, D, VIS, PIECES, F8, false>(args, job, smem, sh))
      chunk_again<T, D, VIS, PIECES, F8>((kernel_args_ptr)__builtin_amdgcn_kernarg_segment_ptr(), job, (lds_ptr)smem,
                                         (lds_ptr)(char*)&sh);
  };
  if constexpr (VIS != kTree && !F8) {
    const Job job = job_of<false>(c_, Line());
    if (job.nsplit > 0) work(c_, job);
  } else {
    Job job;
    int left = 0, tiles = 0, run = 0;
    Line line = {};
    if (c_.splits > 0) line = line_of(c_);
    const bool by_runs = uniform(line.by_runs() ? 1 : 0) != 0;
    if (by_runs) {
      // (run, KV head) in turn over the XCDs, the workgroups that share its keys together
      const Grid x = grid_of(c_);
      const int per_kv = x.ngroups / c_.kv_units, shared = per_kv * x.nqb;
      const int i = blockIdx.x >> 3, set = i / shared, in = i - set * shared, u = set * 8 + (blockIdx.x & 7);
      run = uniform(u / c_.kv_units);
      if (run >= c_.runs) return;
      const int at = line.start(run);
      const LineRow r = line_row(c_, line, at, 0);
      left = line.run + (run < line.more ? 1 : 0);
      job.qb = uniform(x.nqb - 1 - in / per_kv);
      job.hg = uniform((u - run * c_.kv_units) * per_kv + in % per_kv);
      job.b = uniform(r.b), job.from = uniform(at - r.first), job.split = 0, job.nsplit = 0;
      tiles = uniform(r.tiles), left = uniform(left);
    } else {
      job = job_of<true>(c_, line);
      if (job.nsplit == 0) return;
    }
    while (true) {
      if (by_runs) {
        job.to = min(tiles, job.from + left);
        job.cut = job.from > 0 || job.to < tiles;
        job.place = run + job.b;
      }
      // (the arguments too are read again)
      kernel_args_ptr args = (kernel_args_ptr)__builtin_amdgcn_kernarg_segment_ptr();
      asm volatile("" : "+s"(args));
      work(*(const ChunkParams*)args, job);
      left -= job.to - job.from;
      if (!by_runs || left <= 0 || job.b + 1 >= c_.p.B) return;
      __syncthreads();  // the next row's start writes what this one's end reads
      ++job.b;
      job.from = 0;
      tiles = uniform(line_tiles(c_.p, job.b));
    }
  }
}


// Joins a row's key splits by their log-sum-exp, four features a thread; every read is under way before
// the first weight is known.
// (RUNS: the parts of a row may be many, eight at a time; a row's splits are 16 at most)
template <typename T, int D, bool RUNS>
__global__ __launch_bounds__(256) void paged_chunk_join_kernel(const ChunkParams c, int per_row) {
  constexpr int TURN = RUNS ? 8 : kMaxKeySplits;
  const PagedParams& p = c.p;
  const int b = blockIdx.y;
  int n, part;
  if constexpr (RUNS) {
    const Line line = line_of(c);
    if (line.by_runs()) {
      const LineRow r = line_row(c, line, -1, b);
      const int first = line.run_of(r.first);
      n = uniform(line.run_of(r.first + r.tiles - 1) - first + 1);
      part = uniform(first + b);
    } else {
      const Split cut = find_split(c, per_row, -1, b, line.mine, line.total);
      n = uniform(cut.count);
      part = uniform(cut.first);
    }
  } else {
    const Split cut = find_split(c, per_row, -1, b);
    n = uniform(cut.count);
    part = uniform(cut.first);
  }
  if (n == 1) return;  // written by its workgroups
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)p.Sq * p.Hq * (D / 4)) return;
  const int f = (int)(i % (D / 4)) * 4;
  const int h = (int)(i / (D / 4) % p.Hq), s = (int)(i / ((int64_t)(D / 4) * p.Hq));
  const int64_t o_split = (int64_t)p.Sq * p.Hq * D, l_split = (int64_t)p.Hq * p.Sq;
  const float* o = c.part + part * o_split + ((int64_t)s * p.Hq + h) * D + f;
  const float* l = c.part_lse + part * l_split + (int64_t)h * p.Sq + s;
  float m = -__builtin_inff(), shift = 0.f, sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < n; k0 += TURN) {
    float4 x[TURN];
    float lse[TURN], m_new = m;
#pragma unroll
    for (int k = 0; k < TURN; ++k)
      if (k0 + k < n) lse[k] = l[(k0 + k) * l_split], x[k] = *(const float4*)(o + (k0 + k) * o_split);
#pragma unroll
    for (int k = 0; k < TURN; ++k)
      if (k0 + k < n) m_new = fmaxf(m_new, lse[k]);
    shift = m_new == -__builtin_inff() ? 0.f : m_new;
    if (RUNS && k0 > 0) {
      const float a = expf(m - shift);  // (0 while there was nothing)
      sum *= a, acc.x *= a, acc.y *= a, acc.z *= a, acc.w *= a;
    }
    m = m_new;
#pragma unroll
    for (int k = 0; k < TURN; ++k)
      if (k0 + k < n) {
        const float w = expf(lse[k] - shift);  // 0 for a split that the row sees nothing of, whose output is 0
        sum += w;
        acc.x += x[k].x * w, acc.y += x[k].y * w, acc.z += x[k].z * w, acc.w += x[k].w * w;
      }
    if constexpr (!RUNS) break;
  }
  uint32_t bits = __float_as_uint(sum);
  asm volatile("" : "+v"(bits));  // (the file is compiled as if no NaN occurred)
  const bool empty = bits == 0;
  const float inv = empty ? 0.f : 1.f / sum;
  const float r[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  const int64_t at = b * p.os_b + s * p.os_s + h * p.os_h + f;
  if (p.out_dtype == CEA_F32) {
    *(float4*)((float*)p.out + at) = make_float4(r[0], r[1], r[2], r[3]);
  } else {
    const T v4[4] = {(T)r[0], (T)r[1], (T)r[2], (T)r[3]};
    uint2 raw;
    __builtin_memcpy(&raw, v4, 8);
    *(uint2*)((T*)p.out + at) = raw;
  }
  if (p.lse && f == 0)
    ((float*)p.lse)[b * p.ls_b + h * p.ls_h + s * p.ls_s] = empty ? -__builtin_inff() : shift + logf(sum);
}

template <typename T, int D, int VIS, int PIECES, bool F8>
int launch_form(const ChunkParams& c, hipStream_t st) {
  const PagedParams& p = c.p;
  const int nqb = (p.Sq + BM / c.hp - 1) / (BM / c.hp);
  const int64_t per_row = (int64_t)nqb * (p.Hq / c.hp);
  int64_t total = per_row * p.B;
  const int cuts = std::max(c.splits, c.runs);
  if (cuts > 0) total = ((int64_t)cuts * c.kv_units + 7) / 8 * 8 * (per_row / c.kv_units);
  constexpr int lds = Layout<D, VIS, F8>::LDS_BYTES;
  const hipError_t e = reserve_lds<paged_chunk_kernel<T, D, VIS, PIECES, F8>>(lds);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "paged_attention: cannot reserve %d bytes of LDS: %s", lds,
              hipGetErrorString(e));
  hipLaunchKernelGGL((paged_chunk_kernel<T, D, VIS, PIECES, F8>), dim3((unsigned)total), dim3(NTHREADS), lds, st, c);
  CEA_CHECK_LAUNCH("paged_chunk");
  if (cuts > 0) {
    const int64_t vectors = (int64_t)p.Sq * p.Hq * (D / 4);
    hipLaunchKernelGGL((paged_chunk_join_kernel<T, D, VIS == kTree || F8>), dim3((unsigned)((vectors + 255) / 256), (unsigned)p.B), dim3(256),
                       0, st, c, (int)per_row);
    CEA_CHECK_LAUNCH("paged_chunk_join");
  }
  return CEA_OK;
}

template <typename T, int D, bool F8> int launch_td(const ChunkParams& c, bool f32, hipStream_t st) {
  constexpr int kFull = std::is_same<T, bf16>::value ? 3 : 2;
  if (c.p.masks) return f32 ? launch_form<T, D, kTree, kFull, F8>(c, st) : launch_form<T, D, kTree, 1, F8>(c, st);
  if (c.p.pos) return f32 ? launch_form<T, D, kPosition, kFull, F8>(c, st) : launch_form<T, D, kPosition, 1, F8>(c, st);
  return f32 ? launch_form<T, D, kNumber, kFull, F8>(c, st) : launch_form<T, D, kNumber, 1, F8>(c, st);
}

template <bool F8> int launch_pages(const ChunkParams& c, hipStream_t st) {
  const bool f32 = c.p.out_dtype == CEA_F32;
  if (c.p.in_dtype == CEA_BF16) return c.p.D == 128 ? launch_td<bf16, 128, F8>(c, f32, st) : launch_td<bf16, 64, F8>(c, f32, st);
  return c.p.D == 128 ? launch_td<f16, 128, F8>(c, f32, st) : launch_td<f16, 64, F8>(c, f32, st);
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Query heads of a workgroup: the fewest padded query rows per head, the smallest number on ties.
int heads_per_wg(int64_t Sq, int64_t group) {
  auto padding = [&](int hp) { return (Sq + BM / hp - 1) / (BM / hp) * (BM / hp) - Sq; };
  int best = 1;
  for (int hp = 2; hp <= NWAVES && group > 0 && group % hp == 0; hp *= 2)
    if (padding(hp) < padding(best)) best = hp;
  return best;
}

struct ChunkPlan {
  int hp, splits, runs;
  size_t tiles, pos32, part_out, part_lse;  // bytes: summaries, positions, the splits' partial results
};

ChunkPlan plan_chunk(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots, bool pos, bool runs) {
  ChunkPlan r;
  r.hp = heads_per_wg(Sq, group);
  // Below two workgroups per compute unit the rows may be cut; their splits are at most the workgroups that the
  // tiles are dealt to, over those of a row's split, and one a row more for what does not divide.
  const int64_t per_row = (Sq + BM / r.hp - 1) / (BM / r.hp) * (Hq / r.hp), tiles = (slots + BN - 1) / BN;
  r.splits = r.runs = 0;
  const int64_t most = std::min<int64_t>(B * kMaxKeySplits, kSplitWgs / per_row + 1 + B);
  if (runs) {
    // Runs where a row's query blocks see about the same tiles (of a prompt the last blocks see the most, and would
    // see the most of every row of a run), and up to four rounds of workgroups: rows of uneven length leave the last
    // ones to a few.
    const bool even = Sq <= BM / r.hp || Sq * 8 <= slots;
    if (tiles >= kCutTiles && per_row < kSplitWgs && per_row * B < (even ? 4 : 1) * kSplitWgs) {
      r.splits = (int)most;
      const int64_t runs_at_most = kSplitWgs / per_row;
      r.runs = even && B * tiles >= kRunTiles * runs_at_most ? (int)runs_at_most : 0;
    }
  } else if (per_row * B < kSplitWgs && tiles >= 2 * kSplitTiles) {
    r.splits = (int)most;
  }
  r.tiles = pos ? align256((size_t)B * ((slots + BN - 1) / BN) * sizeof(TileInfo)) : 0;
  r.pos32 = pos ? align256((size_t)B * ((slots + BN - 1) / BN) * 2 * BN * sizeof(int32_t)) : 0;
  const size_t parts = std::max<int64_t>(r.splits, r.runs > 0 ? r.runs + B : 0);
  r.part_out = align256(parts * Sq * Hq * D * sizeof(float));
  r.part_lse = align256(parts * Sq * Hq * sizeof(float));
  return r;
}

}  // namespace

size_t paged_chunk_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots, bool pos,
                                   bool runs) {
  const ChunkPlan r = plan_chunk(B, Sq, Hq, group, D, slots, pos, runs);
  return r.tiles + r.pos32 + r.part_out + r.part_lse;
}

bool paged_chunk_supported(const PagedParams& p, const HeadMap& map) {
  if (map.group <= 0 && (p.Hq > kPagedMapHeads || p.Hkv > 256)) return false;
  for (int64_t s : {p.os_b, p.os_s, p.os_h})
    if (s % 4) return false;
  if ((uintptr_t)p.out % 16 || (p.pos && (uintptr_t)p.pos % 8)) return false;
  // (all rows' tiles, and all workgroups, are counted in 32 bits)
  const int64_t tiles = ((int64_t)p.W * p.page + BN - 1) / BN;
  return p.B < 65536 && p.B * tiles < ((int64_t)1 << 31) &&
         (int64_t)p.B * p.Hq * ((p.Sq + 31) / 32) * kMaxKeySplits < ((int64_t)1 << 31);
}

int launch_paged_chunk(const PagedParams& params, const HeadMap& map, void* ws, hipStream_t st) {
  const int64_t slots = (int64_t)params.W * params.page;
  const PagedParams& o = params;
  const ChunkPlan r = plan_chunk(o.B, o.Sq, o.Hq, map.group, o.D, slots, o.pos != nullptr,
                                 paged_chunk_runs(o));
  ChunkParams c;
  memset(&c, 0, sizeof(c));
  c.p = o;
  c.hp = r.hp, c.splits = r.splits, c.runs = r.runs;
  c.page16 = o.page / 16;
  c.magic = c.page16 > 1 ? (uint32_t)((((uint64_t)1 << 32) + c.page16 - 1) / c.page16) : 0;
  for (int h = 0; h < kPagedMapHeads && h < o.Hq && map.group <= 0; ++h) c.kv[h] = (uint8_t)map.kv[h];
  char* at = (char*)ws;
  if (o.pos) {
    c.tiles = (const TileInfo*)at;
    c.pos32 = (const int32_t*)(at + r.tiles);
    c.ntiles = (int32_t)((slots + BN - 1) / BN);
    hipLaunchKernelGGL(paged_tile_info_kernel, dim3((unsigned)std::min((c.ntiles + 3) / 4, 64), (unsigned)o.B),
                       dim3(256), 0, st, o, c.ntiles, (TileInfo*)at, (int32_t*)(at + r.tiles));
    CEA_CHECK_LAUNCH("paged_tile_info");
    at += r.tiles + r.pos32;
  }
  // query heads that an XCD takes together: whole KV heads, as many as 5 MB of keys and values hold (by
  // the table's width: the lengths are on the device), in sets of even size
  const int64_t kv_bytes = std::max<int64_t>(slots * o.D * 2 * (int64_t)dtype_size(o.kv_dtype), 1);
  const int64_t per_kv = map.group > 0 ? o.Hq / c.hp / o.Hkv : 1;
  c.order_per_kv = (int)per_kv;
  const int64_t heads = std::max<int64_t>(((int64_t)o.B * (o.Hq / c.hp) + 8 * per_kv - 1) / (8 * per_kv), 1);
  const int64_t fit = std::max<int64_t>(((int64_t)5 << 20) / kv_bytes, 1);
  const int64_t sets = (heads + fit - 1) / fit;
  c.order_units = (int)((heads + sets - 1) / sets * per_kv);
  if (o.B == 1 && heads == 1) c.order_units = 1;

  c.kv_units = map.group > 0 ? o.Hkv : o.Hq;
  c.part = (float*)at, c.part_lse = (float*)(at + r.part_out);
  return o.kv_dtype == CEA_F8 ? launch_pages<true>(c, st) : launch_pages<false>(c, st);
}

}  // namespace cea

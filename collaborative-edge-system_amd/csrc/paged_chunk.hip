// The paged chunk kernel over pages of 16 bits, and the launch plan of both forms.
#include "paged_chunk.hpp"

namespace cea {
namespace {

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
      r.runs = even ? (int)(kSplitWgs / per_row) : 0;
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
  return o.kv_dtype == CEA_F8 ? launch_paged_chunk8(c, st) : launch_pages<false>(c, st);
}

}  // namespace cea

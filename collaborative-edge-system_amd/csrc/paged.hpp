// Parameter block and launchers of the paged KV cache: pools of pages of `page` slots, a table of
// page indices per batch row, and the rows' lengths, all read on the device.
//
// Slot j of row b is place j % page of page tables[b, j / page].  It exists while j < lengths[b]
// (clamped to what the table holds); a page index outside the pool holds no keys.  Its position is
// j, or what pos_pages holds there when that is given.  Nothing outside the pools is read or
// written whatever the tables, lengths and offsets hold.
//
// Pages of 8 bits hold e4m3 numbers, and a scale byte s (1 to 254) per slot and head: the values q * 2^(s - 127).
//
// Drafts: with masks the queries are the nodes of a tree in the row's last counts[b] slots.  Node i sees
// every slot before them, and slot lengths[b] - counts[b] + j where bit j of masks[b, i] is set.
#pragma once

#include <type_traits>

#include "cea_kernels.hpp"

namespace cea {

constexpr int kPagedMapHeads = 64;  // query heads of an explicit head map on the matrix-core kernels

struct PagedParams {
  const void* q;
  const void* k;
  const void* v;
  const int64_t* q_pos;
  const int64_t* pos;        // [P, page] or null: position j in slot j
  const int64_t* tables;     // [B, W]
  const int64_t* lengths;    // [B]
  const uint8_t* k_scales;   // [P, H, page], pages of 8 bits alone
  const uint8_t* v_scales;
  const int64_t* masks;      // [B, Sq, words] or null: 64 nodes a word
  const int64_t* counts;     // [B], with masks
  void* out;
  void* lse;                 // may be null
  int64_t P;
  int32_t B, Sq, Hq, Hkv, D, W, page;
  int64_t qs_b, qs_s, qs_h;
  int64_t ks_p, ks_h, ks_s;
  int64_t vs_p, vs_h, vs_s;
  int64_t ps_p, ps_s;
  int64_t ts_b, ts_w, ns_b;  // tables, lengths
  int64_t qps_b, qps_s;
  int64_t os_b, os_s, os_h;
  int64_t ls_b, ls_h, ls_s;
  int64_t kss_p, kss_h, kss_s, vss_p, vss_h, vss_s;  // scales
  int64_t ms_b, ms_s, ms_w, cs_b;                    // masks, counts
  double scale;
  int32_t causal;
  int32_t in_dtype, kv_dtype, out_dtype;
  int32_t group;             // > 0: KV head of query head h is h / group; 0: explicit map
};

// Slots of row b: its length within what its table holds.
__device__ __forceinline__ int64_t paged_slots(const PagedParams& p, int b) {
  const int64_t n = p.lengths[b * p.ns_b], cap = (int64_t)p.W * p.page;
  return n < 0 ? 0 : n < cap ? n : cap;
}

// The tree of row b: its first node's slot (at least -2^40, at most what the row has) and how many nodes
// there are.
struct TreeOf {
  int64_t base, nodes;
};
__device__ __forceinline__ TreeOf tree_of(const PagedParams& p, int b) {
  const int64_t n = p.lengths[b * p.ns_b], c = p.counts[b * p.cs_b];
  const int64_t nodes = c < 0 ? 0 : c, base = (int64_t)((uint64_t)n - (uint64_t)nodes);
  const int64_t top = paged_slots(p, b), low = -((int64_t)1 << 40);
  return {n < low || base < low ? low : base < top ? base : top, nodes < p.Sq ? nodes : p.Sq};
}
// The 64 nodes of word w that node i of row b sees.
__device__ __forceinline__ uint64_t tree_word(const PagedParams& p, int b, int64_t i, int w) {
  const int left = p.Sq - w * 64;
  const uint64_t x = (uint64_t)p.masks[b * p.ms_b + i * p.ms_s + w * p.ms_w];
  return left >= 64 ? x : x & (((uint64_t)1 << left) - 1);
}

// Two e4m3 numbers, the low or the high half of x, times a power of two, as 16-bit numbers: exact in bf16, and in
// f16 but for what is below its normal numbers (rounded) or beyond its largest (infinite).
template <typename T, bool HIGH> __device__ __forceinline__ uint32_t widen2(uint32_t x, float scale) {
  if constexpr (std::is_same<T, bf16>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, scale, HIGH));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, HIGH));
}
// A scale byte (1 to 254) as the power of two that it stands for.
__device__ __forceinline__ float scale_value(uint32_t s) { return __uint_as_float(s << 23); }

// What decides whether a query sees a slot: its number, a position in the pool, or a tree's mask.
enum Vis { kNumber = 0, kPosition = 1, kTree = 2 };

// Layouts that the matrix-core kernels read: 16-bit queries, pages of their type or of 8 bits, head size 64 or
// 128, pages of a multiple of 16 slots, rows of 16-byte vectors, contiguous positions and scales.
bool paged_tiles_supported(const PagedParams& p);

// A few new tokens per row (at most 16 query rows of a unit; an explicit head map within kPagedMapHeads).
bool paged_token_supported(const PagedParams& p, const HeadMap& map);
size_t paged_token_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int group, int64_t D,
                                   int64_t slots, bool f8);
int launch_paged_token(const PagedParams& p, const HeadMap& map, void* ws, hipStream_t s);

// Any number of new tokens per row.  Scratch: tile summaries with positions in the pool, and the partial
// results of key splits.
bool paged_chunk_supported(const PagedParams& p, const HeadMap& map);
// Forms whose rows are cut into runs that cross them, and not one by one.
inline bool paged_chunk_runs(const PagedParams& p) { return p.kv_dtype == CEA_F8 || p.masks != nullptr; }
size_t paged_chunk_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots, bool pos,
                                   bool runs);
int launch_paged_chunk(const PagedParams& p, const HeadMap& map, void* ws, hipStream_t s);

// f32, head size 64 or 128.  Scratch: the partial results of key splits.
bool paged_f32_supported(const PagedParams& p, const HeadMap& map);
size_t paged_f32_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots);
int launch_paged_f32(const PagedParams& p, const HeadMap& map, void* ws, hipStream_t s);

// Merges the f32 partial results of `splits` key splits (the first at part.out / part.lse) into p's.
int merge_paged_splits(const PagedParams& p, const PagedParams& part, int splits, int64_t split_out,
                       int64_t split_lse, hipStream_t s);

int launch_paged_generic(const PagedParams& p, const HeadMap& map, hipStream_t s);

// Appends, one row of k and v per token and head; null tensors are left out.
int launch_paged_append(const cea_tensor* k, const cea_tensor* v, const cea_tensor* pos,
                        const cea_tensor* c, const cea_tensor* sn, const cea_tensor* tables,
                        const cea_tensor* offsets, const cea_tensor* counts, cea_tensor* kp,
                        cea_tensor* vp, cea_tensor* pp, hipStream_t s);

// The same into pages of 8 bits with their scales.
int launch_paged_append8(const cea_tensor* k, const cea_tensor* v, const cea_tensor* pos, const cea_tensor* c,
                         const cea_tensor* sn, const cea_tensor* tables, const cea_tensor* offsets,
                         const cea_tensor* counts, cea_tensor* kp, cea_tensor* vp, cea_tensor* ks, cea_tensor* vs,
                         cea_tensor* pp, hipStream_t s);

// Slots offsets[b] .. of every row into contiguous rows, 0 where there is none; ks / vs null but for pages
// of 8 bits.
int launch_paged_read(const cea_tensor* kp, const cea_tensor* vp, const cea_tensor* ks, const cea_tensor* vs,
                      const cea_tensor* tables, const cea_tensor* offsets, const cea_tensor* counts, cea_tensor* k,
                      cea_tensor* v, hipStream_t s);

// Moves slot offsets[b] + path[b, i] to offsets[b] + i in every pool (kv [N,P,H,page*D], scales [N,P,H,page]
// or null).
int launch_paged_keep(cea_tensor* kv, cea_tensor* scales, int page, const cea_tensor* tables,
                      const cea_tensor* offsets, const cea_tensor* counts, const cea_tensor* path, hipStream_t s);

// Ancestors of every node as bits, and depths.
int launch_tree_masks(const cea_tensor* parents, const cea_tensor* counts, cea_tensor* masks, cea_tensor* depths,
                      hipStream_t s);

// Copies pages src[i] -> dst[i] of every pool (validated by the caller).
int launch_copy_pages(int n, const cea_tensor* pools, const int64_t* src, const int64_t* dst,
                      int64_t m, hipStream_t s);

}  // namespace cea

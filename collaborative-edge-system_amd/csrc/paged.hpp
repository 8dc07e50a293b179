// Parameter block and launchers of the paged KV cache: pools of pages of `page` slots, a table of
// page indices per batch row, and the rows' lengths, all read on the device.
//
// Slot j of row b is place j % page of page tables[b, j / page].  It exists while j < lengths[b]
// (clamped to what the table holds); a page index outside the pool holds no keys.  Its position is
// j, or what pos_pages holds there when that is given.  Nothing outside the pools is read or
// written whatever the tables, lengths and offsets hold.
#pragma once

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
  double scale;
  int32_t causal;
  int32_t in_dtype, out_dtype;
  int32_t group;             // > 0: KV head of query head h is h / group; 0: explicit map
};

// Slots of row b: its length within what its table holds.
__device__ __forceinline__ int64_t paged_slots(const PagedParams& p, int b) {
  const int64_t n = p.lengths[b * p.ns_b], cap = (int64_t)p.W * p.page;
  return n < 0 ? 0 : n < cap ? n : cap;
}

// Layouts that the matrix-core kernels read: 16-bit types, head size 64 or 128, pages of a multiple
// of 16 slots, rows of 16-byte vectors, contiguous positions.
bool paged_tiles_supported(const PagedParams& p);

// A few new tokens per row (at most 16 query rows of a unit; an explicit head map within kPagedMapHeads).
bool paged_token_supported(const PagedParams& p, const HeadMap& map);
size_t paged_token_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int group, int64_t D,
                                   int64_t slots);
int launch_paged_token(const PagedParams& p, const HeadMap& map, void* ws, hipStream_t s);

// Any number of new tokens per row.  Scratch: tile summaries with positions in the pool, and the partial
// results of key splits.
bool paged_chunk_supported(const PagedParams& p, const HeadMap& map);
size_t paged_chunk_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots, bool pos);
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

// Copies pages src[i] -> dst[i] of every pool (validated by the caller).
int launch_copy_pages(int n, const cea_tensor* pools, const int64_t* src, const int64_t* dst,
                      int64_t m, hipStream_t s);

}  // namespace cea

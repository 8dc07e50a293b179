// C ABI of the paged KV cache: argument checks, the choice of kernel and the workspace layout.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <memory>
#include <new>

#include "paged.hpp"

namespace cea {
namespace {

int check_pages(const cea_tensor* kp, const cea_tensor* vp, int dt, int64_t H, int64_t D,
                const char* what) {
  int rc;
  if ((rc = check_tensor(kp, "k_pages", 4, dt, true))) return rc;
  if ((rc = check_tensor(vp, "v_pages", 4, dt, true))) return rc;
  for (const cea_tensor* t : {kp, vp})
    CEA_REQUIRE(t->size[0] == kp->size[0] && t->size[2] == kp->size[2] && t->size[1] == H &&
                    t->size[3] == D,
                CEA_EINVAL, "%s: k_pages and v_pages must be [P, %lld, page, %lld]", what,
                (long long)H, (long long)D);
  return CEA_OK;
}

int check_rows(const cea_tensor* tables, const cea_tensor* per_row, const char* name, int64_t B,
               const char* what) {
  int rc;
  if ((rc = check_tensor(tables, "tables", 2, CEA_I64, false))) return rc;
  CEA_REQUIRE(tables->size[0] == B, CEA_EINVAL, "%s: tables must be [B, W]", what);
  if ((rc = check_tensor(per_row, name, 1, CEA_I64, false))) return rc;
  CEA_REQUIRE(per_row->size[0] == B, CEA_EINVAL, "%s: %s must be [B]", what, name);
  return CEA_OK;
}

int check_pos_pages(const cea_tensor* pp, const cea_tensor* kp, const char* what) {
  int rc;
  if ((rc = check_tensor(pp, "pos_pages", 2, CEA_I64, false))) return rc;
  CEA_REQUIRE(pp->size[0] == kp->size[0] && pp->size[1] == kp->size[2], CEA_EINVAL,
              "%s: pos_pages must be [P, page]", what);
  return CEA_OK;
}

// An attention call: its parameters, the kernel that it takes and the scratch of that kernel.
enum class Form { none, token, chunk, f32, generic };
struct Attention {
  PagedParams p;
  HeadMap map;
  Form form;
  size_t bytes;
};

int prepare_attention(Attention& c, const cea_tensor* q, const cea_tensor* k_pages, const cea_tensor* v_pages,
                      const cea_tensor* pos_pages, const cea_tensor* tables, const cea_tensor* lengths,
                      const cea_tensor* q_pos, int32_t causal, double scale, const int32_t* kv_map,
                      int32_t kv_map_len, const cea_tensor* out, const cea_tensor* lse) {
  memset(&c, 0, sizeof(c));
  const char* what = "paged_attention";
  int rc;
  if ((rc = check_tensor(q, "q", 4, -1, true))) return rc;
  const int dt = q->dtype;
  CEA_REQUIRE(dt != CEA_I64, CEA_EUNSUPPORTED, "%s: unsupported dtype int64", what);
  const int64_t B = q->size[0], Sq = q->size[1], Hq = q->size[2], D = q->size[3];
  CEA_REQUIRE(D >= 1, CEA_EINVAL, "%s: empty head dimension", what);
  CEA_REQUIRE(k_pages != nullptr, CEA_EINVAL, "k_pages: missing tensor");
  const int64_t Hkv = k_pages->ndim == 4 ? k_pages->size[1] : 0;
  if ((rc = check_pages(k_pages, v_pages, dt, Hkv, D, what))) return rc;
  if ((rc = check_rows(tables, lengths, "lengths", B, what))) return rc;
  if (pos_pages && (rc = check_pos_pages(pos_pages, k_pages, what))) return rc;
  if ((rc = check_tensor(q_pos, "q_pos", 2, CEA_I64, false))) return rc;
  CEA_REQUIRE(q_pos->size[0] == B && q_pos->size[1] == Sq, CEA_EINVAL, "%s: q_pos must be [B, Sq]",
              what);
  const int acc = dt == CEA_F64 ? CEA_F64 : CEA_F32;
  if ((rc = check_tensor(out, "out", 4, -1, true))) return rc;
  CEA_REQUIRE(out->size[0] == B && out->size[1] == Sq && out->size[2] == Hq && out->size[3] == D,
              CEA_EINVAL, "%s: out must be [B, Sq, Hq, D]", what);
  CEA_REQUIRE(out->dtype == acc || out->dtype == dt, CEA_EINVAL, "%s: out must be %s or %s", what,
              dtype_name(acc), dtype_name(dt));
  if (lse) {
    if ((rc = check_tensor(lse, "lse", 3, acc, false))) return rc;
    CEA_REQUIRE(lse->size[0] == B && lse->size[1] == Hq && lse->size[2] == Sq, CEA_EINVAL,
                "%s: lse must be [B, Hq, Sq]", what);
  }
  if ((rc = make_head_map(&c.map, Hq, Hkv, kv_map, kv_map_len))) return rc;
  const int64_t page = k_pages->size[2], W = tables->size[1];
  CEA_REQUIRE(W == 0 || page < ((int64_t)1 << 40) / W, CEA_EUNSUPPORTED, "%s: tables too wide", what);

  PagedParams& p = c.p;
  p.q = q->data, p.k = k_pages->data, p.v = v_pages->data;
  p.q_pos = (const int64_t*)q_pos->data;
  p.pos = pos_pages ? (const int64_t*)pos_pages->data : nullptr;
  p.tables = (const int64_t*)tables->data, p.lengths = (const int64_t*)lengths->data;
  p.out = out->data, p.lse = lse ? lse->data : nullptr;
  p.P = k_pages->size[0];
  p.B = (int)B, p.Sq = (int)Sq, p.Hq = (int)Hq, p.Hkv = (int)Hkv, p.D = (int)D;
  p.W = (int)W, p.page = (int)page;
  p.qs_b = q->stride[0], p.qs_s = q->stride[1], p.qs_h = q->stride[2];
  p.ks_p = k_pages->stride[0], p.ks_h = k_pages->stride[1], p.ks_s = k_pages->stride[2];
  p.vs_p = v_pages->stride[0], p.vs_h = v_pages->stride[1], p.vs_s = v_pages->stride[2];
  if (pos_pages) p.ps_p = pos_pages->stride[0], p.ps_s = pos_pages->stride[1];
  p.ts_b = tables->stride[0], p.ts_w = tables->stride[1], p.ns_b = lengths->stride[0];
  p.qps_b = q_pos->stride[0], p.qps_s = q_pos->stride[1];
  p.os_b = out->stride[0], p.os_s = out->stride[1], p.os_h = out->stride[2];
  if (lse) p.ls_b = lse->stride[0], p.ls_h = lse->stride[1], p.ls_s = lse->stride[2];
  p.scale = scale;
  p.causal = causal ? 1 : 0;
  p.in_dtype = dt, p.out_dtype = out->dtype;
  p.group = c.map.group;
  if (B == 0 || Sq == 0 || Hq == 0) return CEA_OK;
  if (page == 0 || p.P == 0) p.W = 0, p.page = 1;  // no slots: every row is empty
  const int group = c.map.group;
  const int64_t slots = (int64_t)p.W * p.page;
  if (paged_tiles_supported(p)) {
    // The token form while one unit holds a KV head's queries, so its keys are read once, and for single
    // tokens of larger groups; two units where all is one launch of small tiles.  us, token / chunk form: 16 query
    // rows of a KV head, D = 64, 16 rows of up to 2500 keys 21.5 / 23.0; 14, 2 rows of up to 8000 15.4 / 18.3; 16,
    // D = 128, 32 rows of up to 8000 157 / 170, but 8 of 100 to 4096 32.1 / 26.4, which the rule does not tell
    // apart; 32 query rows, 4 rows of up to 900, D = 64, 13.1 / 14.9, D = 128, 18.5 / 17.5; 28, 4 of up to 500,
    // D = 64, 11.2 / 14.5; 32, 16 of up to 2500, D = 64, 28.2 / 23.7.
    const int64_t rows = Sq * group;
    const bool few = Sq == 1 || group <= 0 || rows <= 16 || (rows <= 32 && D == 64 && slots <= 1024);
    if (few && paged_token_supported(p, c.map)) {
      c.form = Form::token;
      c.bytes = paged_token_workspace_bytes(B, Sq, Hq, Hkv, group, D, slots);
    } else if (paged_chunk_supported(p, c.map)) {
      c.form = Form::chunk;
      c.bytes = paged_chunk_workspace_bytes(B, Sq, Hq, group, D, slots, p.pos != nullptr);
    }
  }
  if (c.form == Form::none && paged_f32_supported(p, c.map)) {
    c.form = Form::f32;
    c.bytes = paged_f32_workspace_bytes(B, Sq, Hq, group, D, slots);
  }
  if (c.form == Form::none) c.form = Form::generic;
  return CEA_OK;
}

// The pages [N, P] of a pool [N, P, E] are apart: along the dimension of the smaller stride by a page at
// least, along the other one by all that this one spans.  Views of a tensor that holds each element once are.
bool pages_apart(const cea_tensor& t) {
  if (t.size[0] == 0 || t.size[1] == 0) return true;
  int near = t.stride[0] <= t.stride[1] ? 0 : 1;
  if (t.size[near] == 1) near = 1 - near;  // (the stride of a single one says nothing)
  const int far = 1 - near;
  const int64_t span = t.size[near] > 1 ? t.stride[near] * (t.size[near] - 1) + t.size[2] : t.size[2];
  return (t.size[near] <= 1 || t.stride[near] >= t.size[2]) && (t.size[far] <= 1 || t.stride[far] >= span);
}

}  // namespace

bool paged_tiles_supported(const PagedParams& p) {
  if (!(p.in_dtype == CEA_BF16 || p.in_dtype == CEA_F16) || !(p.D == 64 || p.D == 128)) return false;
  if (p.page % 16 != 0 || p.W == 0) return false;
  // slots and places in 32 bits, and page numbers by multiplication (u / m = u * ceil(2^32 / m) >> 32
  // while u * m < 2^32, u the slot's sixteenth, m the page's)
  const int64_t slots = (int64_t)p.W * p.page;
  if (slots >= (int64_t)1 << 30 || slots / 16 * (p.page / 16) >= (int64_t)1 << 32) return false;
  // exponents take |scale| * log2(e) as a factor, which has to be a normal number
  if (!(fabs(p.scale) >= 1e-30 && fabs(p.scale) <= 1e30)) return false;
  const int64_t s8[] = {p.qs_b, p.qs_s, p.qs_h, p.ks_p, p.ks_h, p.ks_s, p.vs_p, p.vs_h, p.vs_s};
  for (int64_t s : s8)
    if (s % 8) return false;
  for (const void* d : {p.q, p.k, p.v})
    if ((uintptr_t)d % 16) return false;
  // a 64-row tile spans less than 2^31 bytes
  for (int64_t s : {p.ks_s, p.vs_s})
    if (s < p.D || s >= (int64_t)1 << 23) return false;
  return p.pos == nullptr || p.ps_s == 1;
}

int merge_paged_splits(const PagedParams& o, const PagedParams& part, int splits, int64_t split_out,
                       int64_t split_lse, hipStream_t st) {
  MergeParams m;
  memset(&m, 0, sizeof(m));
  m.n = splits;
  m.B = o.B, m.Sq = o.Sq, m.H = o.Hq, m.D = o.D;
  m.dtype = CEA_F32, m.out_dtype = o.out_dtype;
  for (int i = 0; i < splits; ++i) {
    m.outs[i] = (const float*)part.out + i * split_out;
    m.lses[i] = (const float*)part.lse + i * split_lse;
    m.os[i][0] = part.os_b, m.os[i][1] = part.os_s, m.os[i][2] = part.os_h;
    m.ls[i][0] = part.ls_b, m.ls[i][1] = part.ls_h, m.ls[i][2] = part.ls_s;
  }
  m.out = o.out, m.lse = o.lse;
  m.dos[0] = o.os_b, m.dos[1] = o.os_s, m.dos[2] = o.os_h;
  m.dls[0] = o.ls_b, m.dls[1] = o.ls_h, m.dls[2] = o.ls_s;
  return launch_merge(m, st);
}

}  // namespace cea

using namespace cea;

extern "C" {

int cea_paged_kv_append(const cea_tensor* k, const cea_tensor* v, const cea_tensor* pos,
                        const cea_tensor* cos, const cea_tensor* sin, const cea_tensor* tables,
                        const cea_tensor* offsets, const cea_tensor* counts, cea_tensor* k_pages,
                        cea_tensor* v_pages, cea_tensor* pos_pages, void* stream) {
  const char* what = "paged_kv_append";
  int rc;
  if ((rc = check_tensor(k, "k", 4, -1, true))) return rc;
  const int dt = k->dtype;
  CEA_REQUIRE(dt != CEA_I64, CEA_EUNSUPPORTED, "%s: unsupported dtype int64", what);
  if ((rc = check_tensor(v, "v", 4, dt, true))) return rc;
  const int64_t B = k->size[0], n = k->size[1], H = k->size[2], D = k->size[3];
  for (int i = 0; i < 4; ++i)
    CEA_REQUIRE(v->size[i] == k->size[i], CEA_EINVAL, "%s: v must match k [B,n,H,D]", what);
  CEA_REQUIRE(D % 2 == 0, CEA_EINVAL, "%s: head size must be even", what);
  if ((rc = check_pages(k_pages, v_pages, dt, H, D, what))) return rc;
  if ((rc = check_rows(tables, offsets, "offsets", B, what))) return rc;
  if (counts) {
    if ((rc = check_tensor(counts, "counts", 1, CEA_I64, false))) return rc;
    CEA_REQUIRE(counts->size[0] == B, CEA_EINVAL, "%s: counts must be [B]", what);
  }
  CEA_REQUIRE((pos == nullptr) == (pos_pages == nullptr), CEA_EINVAL,
              "%s: give both positions and pos_pages or neither", what);
  if (pos) {
    if ((rc = check_tensor(pos, "positions", 2, CEA_I64, false))) return rc;
    CEA_REQUIRE(pos->size[0] == B && pos->size[1] == n, CEA_EINVAL, "%s: positions must be [B, n]",
                what);
    if ((rc = check_pos_pages(pos_pages, k_pages, what))) return rc;
  }
  CEA_REQUIRE((cos == nullptr) == (sin == nullptr), CEA_EINVAL,
              "%s: give both rotary tables or neither", what);
  cea_tensor c, sn;
  if (cos) {
    if ((rc = check_tensor(cos, "cos", 3, dt, true))) return rc;
    if ((rc = check_tensor(sin, "sin", 3, dt, true))) return rc;
    for (const cea_tensor* t : {cos, sin})
      CEA_REQUIRE((t->size[0] == B || t->size[0] == 1) && t->size[1] == n && t->size[2] == D,
                  CEA_EINVAL, "%s: cos/sin must be [B, n, D]", what);
    c = *cos, sn = *sin;
    if (c.size[0] == 1) c.stride[0] = 0;  // broadcast over the batch
    if (sn.size[0] == 1) sn.stride[0] = 0;
  }
  return launch_paged_append(k, v, pos, cos ? &c : nullptr, cos ? &sn : nullptr, tables, offsets,
                             counts, k_pages, v_pages, pos_pages, (hipStream_t)stream);
}

size_t cea_paged_attention_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int64_t D,
                                           int64_t W, int64_t page, int32_t in_dtype) {
  if (!(in_dtype == CEA_BF16 || in_dtype == CEA_F16 || in_dtype == CEA_F32) || !(D == 64 || D == 128)) return 0;
  if (B <= 0 || Sq <= 0 || Hq <= 0 || Hkv <= 0 || W <= 0 || page <= 0 || page % 16) return 0;
  // (an explicit map takes the place of an even grouping, or there is none: room for either)
  const int64_t slots = W * page;
  size_t most = 0;
  for (const int group : {0, Hq % Hkv == 0 ? (int)(Hq / Hkv) : 0})
    if (in_dtype == CEA_F32) most = std::max(most, paged_f32_workspace_bytes(B, Sq, Hq, group, D, slots));
    else most = std::max({most, paged_token_workspace_bytes(B, Sq, Hq, Hkv, group, D, slots),
                     paged_chunk_workspace_bytes(B, Sq, Hq, group, D, slots, true)});
  return most;
}

int cea_paged_attention_workspace(const cea_tensor* q, const cea_tensor* k_pages, const cea_tensor* v_pages,
                                  const cea_tensor* pos_pages, const cea_tensor* tables,
                                  const cea_tensor* lengths, const cea_tensor* q_pos, int32_t causal,
                                  double scale, const int32_t* kv_map, int32_t kv_map_len,
                                  const cea_tensor* out, const cea_tensor* lse, size_t* bytes) {
  CEA_REQUIRE(bytes != nullptr, CEA_EINVAL, "paged_attention: missing arguments");
  Attention c;
  const int rc = prepare_attention(c, q, k_pages, v_pages, pos_pages, tables, lengths, q_pos, causal, scale, kv_map,
                                   kv_map_len, out, lse);
  *bytes = rc ? 0 : c.bytes;
  return rc;
}

int cea_paged_attention(const cea_tensor* q, const cea_tensor* k_pages, const cea_tensor* v_pages,
                        const cea_tensor* pos_pages, const cea_tensor* tables,
                        const cea_tensor* lengths, const cea_tensor* q_pos, int32_t causal,
                        double scale, const int32_t* kv_map, int32_t kv_map_len, cea_tensor* out,
                        cea_tensor* lse, void* workspace, size_t workspace_bytes, void* stream) {
  Attention c;
  const int rc = prepare_attention(c, q, k_pages, v_pages, pos_pages, tables, lengths, q_pos, causal, scale, kv_map,
                                   kv_map_len, out, lse);
  if (rc) return rc;
  CEA_REQUIRE(c.bytes == 0 || (workspace && workspace_bytes >= c.bytes), CEA_ENOSPACE,
              "paged_attention: workspace of %zu bytes needed, %zu given", c.bytes, workspace_bytes);
  hipStream_t st = (hipStream_t)stream;
  switch (c.form) {
    case Form::none: return CEA_OK;  // no query rows
    case Form::token: return launch_paged_token(c.p, c.map, workspace, st);
    case Form::chunk: return launch_paged_chunk(c.p, c.map, workspace, st);
    case Form::f32: return launch_paged_f32(c.p, c.map, workspace, st);
    case Form::generic: break;
  }
  return launch_paged_generic(c.p, c.map, st);
}

int cea_copy_pages(int32_t n, const cea_tensor* pools, const int64_t* src, const int64_t* dst,
                   int64_t moves, void* stream) {
  const char* what = "copy_pages";
  int rc;
  CEA_REQUIRE(n >= 1 && n <= CEA_MAX_PARTS, n < 1 ? CEA_EINVAL : CEA_EUNSUPPORTED,
              "%s: 1 to %d pools, got %d", what, CEA_MAX_PARTS, n);
  CEA_REQUIRE(pools != nullptr && moves >= 0 && (moves == 0 || (src && dst)), CEA_EINVAL,
              "%s: missing arguments", what);
  for (int i = 0; i < n; ++i) {
    if ((rc = check_tensor(&pools[i], "pool", 3, -1, true))) return rc;
    CEA_REQUIRE(pools[i].size[1] == pools[0].size[1], CEA_EINVAL,
                "%s: the pools differ in their number of pages", what);
    CEA_REQUIRE(pages_apart(pools[i]), CEA_EINVAL, "%s: pages overlap", what);
  }
  const int64_t P = pools[0].size[1];
  for (int64_t i = 0; i < moves; ++i)
    CEA_REQUIRE(src[i] >= 0 && src[i] < P && dst[i] >= 0 && dst[i] < P, CEA_EINVAL,
                "%s: move %lld (%lld to %lld) leaves the %lld pages", what, (long long)i, (long long)src[i],
                (long long)dst[i], (long long)P);
  std::unique_ptr<bool[]> written(new (std::nothrow) bool[(size_t)std::max<int64_t>(P, 1)]());
  CEA_REQUIRE(written != nullptr, CEA_ELAUNCH, "%s: out of host memory", what);
  for (int64_t i = 0; i < moves; ++i) {
    CEA_REQUIRE(!written[dst[i]], CEA_EINVAL, "%s: page %lld is written twice", what, (long long)dst[i]);
    written[dst[i]] = true;
  }
  for (int64_t i = 0; i < moves; ++i)
    CEA_REQUIRE(!written[src[i]], CEA_EINVAL, "%s: page %lld is both read and written", what, (long long)src[i]);
  if (moves == 0) return CEA_OK;
  return launch_copy_pages(n, pools, src, dst, moves, (hipStream_t)stream);
}

}  // extern "C"

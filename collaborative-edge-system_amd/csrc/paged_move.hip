// Writing a paged KV cache: the append of new tokens with the rotary of K fused in, and copies of
// whole pages through any number of pools.  Both are HBM-bound: every row is read and written once.
#include <algorithm>

#include "paged.hpp"

namespace cea {
namespace {

template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

struct AppendParams {
  const void *k, *v, *cos, *sin;
  const int64_t *pos, *tables, *offsets, *counts;
  void *kp, *vp;
  int64_t* pp;
  int64_t P;
  int64_t ks_b, ks_s, ks_h, vs_b, vs_s, vs_h, cs_b, cs_s, ss_b, ss_s;
  int64_t ps_b, ps_s, ts_b, ts_w, os_b, ns_b;
  int64_t kps_p, kps_h, kps_s, vps_p, vps_h, vps_s, pps_p, pps_s;
  int32_t B, n, H, D, W, page;
};

// Half-split rotary (the convention of apply_rotary): with h = D / 2,
//   out_i = x_i c_i - x_{i+h} s_i,   out_{i+h} = x_{i+h} c_{i+h} + x_i s_{i+h},
// in f32 (f64 for f64) and rounded once.  apply_rotary rounds both products and their sum, as the
// separate tensor ops that it replaces do; here nothing needs their intermediate values, and one
// rounding leaves 1 / sqrt(2) of that error.
//
// A thread owns VEC features of both halves of one token and head, so the 16-byte accesses of a
// row stay together whatever the page order; its slot comes from offsets and the table, two
// dependent reads that many resident waves hide.
template <typename T, int VEC, bool ROT>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendParams p) {
  typedef typename acc_of<T>::type M;
  typedef Pack<T, VEC> V;
  const int half = p.D / 2, nch = half / VEC;
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= (int64_t)p.B * p.n * p.H * nch) return;
  const int j = (int)(t % nch) * VEC;
  int64_t r = t / nch;
  const int h = (int)(r % p.H);
  r /= p.H;
  const int s = (int)(r % p.n), b = (int)(r / p.n);
  const T* kr = (const T*)p.k + b * p.ks_b + s * p.ks_s + h * p.ks_h + j;
  const T* vr = (const T*)p.v + b * p.vs_b + s * p.vs_s + h * p.vs_h + j;
  // (the rows are read before the slot is known: both trips to memory at once)
  V k1 = *(const V*)kr, k2 = *(const V*)(kr + half);
  const V v1 = *(const V*)vr, v2 = *(const V*)(vr + half);
  const int64_t count = p.counts ? p.counts[b * p.ns_b] : p.n;
  const int64_t slot = p.offsets[b * p.os_b] + s;
  if constexpr (ROT) {
    const T* cr = (const T*)p.cos + b * p.cs_b + s * p.cs_s + j;
    const T* sr = (const T*)p.sin + b * p.ss_b + s * p.ss_s + j;
    const V c1 = *(const V*)cr, c2 = *(const V*)(cr + half);
    const V s1 = *(const V*)sr, s2 = *(const V*)(sr + half);
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const M x = load_acc<T, M>(&k1.v[e]), y = load_acc<T, M>(&k2.v[e]);
      k1.v[e] = store_cast<T, M>(x * load_acc<T, M>(&c1.v[e]) - y * load_acc<T, M>(&s1.v[e]));
      k2.v[e] = store_cast<T, M>(y * load_acc<T, M>(&c2.v[e]) + x * load_acc<T, M>(&s2.v[e]));
    }
  }
  if (s >= count || slot < 0 || slot >= (int64_t)p.W * p.page) return;
  const int64_t pg = slot / p.page, place = slot - pg * p.page;
  const int64_t id = p.tables[b * p.ts_b + pg * p.ts_w];
  if (id < 0 || id >= p.P) return;
  T* ko = (T*)p.kp + id * p.kps_p + h * p.kps_h + place * p.kps_s + j;
  T* vo = (T*)p.vp + id * p.vps_p + h * p.vps_h + place * p.vps_s + j;
  *(V*)ko = k1;
  *(V*)(ko + half) = k2;
  *(V*)vo = v1;
  *(V*)(vo + half) = v2;
  if (p.pp && h == 0 && j == 0) p.pp[id * p.pps_p + place * p.pps_s] = p.pos[b * p.ps_b + s * p.ps_s];
}

bool aligned(const cea_tensor* t, int bytes) {
  if (!t) return true;
  if ((uintptr_t)t->data % bytes) return false;
  for (int i = 0; i + 1 < t->ndim; ++i)
    if (t->size[i] > 1 && t->stride[i] * (int64_t)dtype_size(t->dtype) % bytes) return false;
  return true;
}

template <typename T>
int append_typed(const AppendParams& p, bool vec, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int64_t total = (int64_t)p.B * p.n * p.H * (p.D / 2 / (vec ? V : 1));
  const int64_t blocks = (total + 255) / 256;
  CEA_REQUIRE(blocks < (int64_t)1 << 31, CEA_EUNSUPPORTED, "paged_kv_append: too many tokens");
  const dim3 grid((unsigned)blocks);
  if (vec && p.cos) hipLaunchKernelGGL((paged_append_kernel<T, V, true>), grid, dim3(256), 0, st, p);
  else if (vec) hipLaunchKernelGGL((paged_append_kernel<T, V, false>), grid, dim3(256), 0, st, p);
  else if (p.cos) hipLaunchKernelGGL((paged_append_kernel<T, 1, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_append_kernel<T, 1, false>), grid, dim3(256), 0, st, p);
  CEA_CHECK_LAUNCH("paged_kv_append");
  return CEA_OK;
}

// ---------------------------------------------------------------------------------------
// page copies
// ---------------------------------------------------------------------------------------
// The moves travel as kernel arguments: the page lists live on the host, where the pages are
// handed out, and this way a copy costs neither a transfer nor a wait.
constexpr int kMoves = 256;

struct CopyPool {
  char* base;
  int64_t stride_n, stride_p;  // bytes
  int64_t bytes;               // of one page
  int32_t n;                   // pools in this tensor
  int32_t chunk0;              // first chunk of a move that is this tensor's
  int32_t chunks;              // chunks of one page
};
struct CopyParams {
  int32_t npools, chunks, moves;
  CopyPool pool[CEA_MAX_PARTS];
  int32_t src[kMoves], dst[kMoves];
};

constexpr int kCopyChunk = 16384;  // bytes a workgroup copies: 4 vectors in flight per lane

template <typename V>
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyParams p) {
  const int chunk = blockIdx.x % p.chunks, move = blockIdx.x / p.chunks;
  int i = 0;
  while (i + 1 < p.npools && chunk >= p.pool[i + 1].chunk0) ++i;
  const CopyPool& c = p.pool[i];
  const int r = chunk - c.chunk0, n = r / c.chunks;
  const int64_t at = (int64_t)(r - n * c.chunks) * kCopyChunk;
  const int64_t left = c.bytes - at;
  const char* from = c.base + n * c.stride_n + p.src[move] * c.stride_p + at;
  char* to = c.base + n * c.stride_n + p.dst[move] * c.stride_p + at;
  constexpr int PER = kCopyChunk / 256 / 16;
  constexpr int STEP = 256 * sizeof(V);
  for (int64_t o = threadIdx.x * sizeof(V); o < (left < kCopyChunk ? left : kCopyChunk); o += STEP * PER) {
    V x[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (o + u * STEP < left && o + u * STEP < kCopyChunk) x[u] = *(const V*)(from + o + u * STEP);
#pragma unroll
    for (int u = 0; u < PER; ++u)
      if (o + u * STEP < left && o + u * STEP < kCopyChunk) *(V*)(to + o + u * STEP) = x[u];
  }
}

}  // namespace

int launch_paged_append(const cea_tensor* k, const cea_tensor* v, const cea_tensor* pos,
                        const cea_tensor* c, const cea_tensor* sn, const cea_tensor* tables,
                        const cea_tensor* offsets, const cea_tensor* counts, cea_tensor* kp,
                        cea_tensor* vp, cea_tensor* pp, hipStream_t st) {
  AppendParams p = {};
  p.k = k->data, p.v = v->data, p.kp = kp->data, p.vp = vp->data;
  p.tables = (const int64_t*)tables->data, p.offsets = (const int64_t*)offsets->data;
  p.B = (int)k->size[0], p.n = (int)k->size[1], p.H = (int)k->size[2], p.D = (int)k->size[3];
  p.P = kp->size[0], p.page = (int)kp->size[2], p.W = (int)tables->size[1];
  p.ks_b = k->stride[0], p.ks_s = k->stride[1], p.ks_h = k->stride[2];
  p.vs_b = v->stride[0], p.vs_s = v->stride[1], p.vs_h = v->stride[2];
  p.ts_b = tables->stride[0], p.ts_w = tables->stride[1];
  p.os_b = offsets->stride[0];
  if (counts) p.counts = (const int64_t*)counts->data, p.ns_b = counts->stride[0];
  p.kps_p = kp->stride[0], p.kps_h = kp->stride[1], p.kps_s = kp->stride[2];
  p.vps_p = vp->stride[0], p.vps_h = vp->stride[1], p.vps_s = vp->stride[2];
  if (pp) {
    p.pp = (int64_t*)pp->data, p.pps_p = pp->stride[0], p.pps_s = pp->stride[1];
    p.pos = (const int64_t*)pos->data, p.ps_b = pos->stride[0], p.ps_s = pos->stride[1];
  }
  if (c) {
    p.cos = c->data, p.sin = sn->data;
    p.cs_b = c->stride[0], p.cs_s = c->stride[1], p.ss_b = sn->stride[0], p.ss_s = sn->stride[1];
  }
  if ((int64_t)p.B * p.n * p.H * p.D == 0 || p.P == 0 || p.W == 0 || p.page == 0) return CEA_OK;
  const int V = 16 / (int)dtype_size(k->dtype);
  bool vec = p.D / 2 % V == 0;
  for (const cea_tensor* t : {k, v, c, sn, (const cea_tensor*)kp, (const cea_tensor*)vp})
    vec = vec && aligned(t, 16);
  switch (k->dtype) {
    case CEA_BF16: return append_typed<bf16>(p, vec, st);
    case CEA_F16: return append_typed<f16>(p, vec, st);
    case CEA_F32: return append_typed<float>(p, vec, st);
    case CEA_F64: return append_typed<double>(p, vec, st);
  }
  set_error("paged_kv_append: unsupported dtype %s", dtype_name(k->dtype));
  return CEA_EUNSUPPORTED;
}

int launch_copy_pages(int n, const cea_tensor* pools, const int64_t* src, const int64_t* dst,
                      int64_t m, hipStream_t st) {
  CopyParams p = {};
  bool v16 = true, v4 = true;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    const cea_tensor& t = pools[i];
    const int64_t es = (int64_t)dtype_size(t.dtype);
    CopyPool& c = p.pool[p.npools];
    c.base = (char*)t.data;
    c.stride_n = t.stride[0] * es, c.stride_p = t.stride[1] * es;
    c.bytes = t.size[2] * es;
    c.n = (int32_t)t.size[0];
    if (c.n == 0 || c.bytes == 0) continue;
    c.chunk0 = (int32_t)chunks;
    c.chunks = (int32_t)((c.bytes + kCopyChunk - 1) / kCopyChunk);
    chunks += (int64_t)c.n * c.chunks;
    CEA_REQUIRE(chunks < (int64_t)1 << 22, CEA_EUNSUPPORTED, "copy_pages: pages too large");
    const int64_t a = (int64_t)(uintptr_t)c.base | (c.n > 1 ? c.stride_n : 0) | c.stride_p | c.bytes;
    v16 = v16 && a % 16 == 0, v4 = v4 && a % 4 == 0;
    ++p.npools;
  }
  if (p.npools == 0) return CEA_OK;
  p.chunks = (int32_t)chunks;
  const int64_t per = std::max<int64_t>(1, std::min<int64_t>(kMoves, (((int64_t)1 << 31) - 1) / chunks));
  for (int64_t i = 0; i < m; i += per) {
    p.moves = (int32_t)std::min(per, m - i);
    for (int j = 0; j < p.moves; ++j) p.src[j] = (int32_t)src[i + j], p.dst[j] = (int32_t)dst[i + j];
    const dim3 grid((unsigned)(p.moves * chunks));
    if (v16) hipLaunchKernelGGL(copy_pages_kernel<uint4>, grid, dim3(256), 0, st, p);
    else if (v4) hipLaunchKernelGGL(copy_pages_kernel<uint32_t>, grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL(copy_pages_kernel<uint16_t>, grid, dim3(256), 0, st, p);
    CEA_CHECK_LAUNCH("copy_pages");
  }
  return CEA_OK;
}

}  // namespace cea

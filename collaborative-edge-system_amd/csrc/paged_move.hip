// Writing a paged KV cache: the append of new tokens with the rotary of K fused in, and copies of
// whole pages through any number of pools.  Both are HBM-bound: every row is read and written once.
// Measured: 2 x 4096 tokens of 8 heads of 128 (71 MB, which the Infinity Cache holds) 11.7 us, 6.1 TB/s; 32 single
// tokens 8.6 us a call and 3.5 of it on the GPU; 300 pages of 128 KB through 16 pools (1.26 GB) 254 us, 5.0 TB/s,
// a large copy's rate; 16 pages through 44 pools 8.1 us a call and 3.7 on the GPU.
#include <algorithm>

#include "paged.hpp"

namespace cea {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// VEC elements in registers (an array that is loaded as a struct the compiler kept in LDS)
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T* p, T (&x)[VEC]) {
  if constexpr (VEC * sizeof(T) == 16) {
    const u32x4 raw = *(const u32x4*)p;
    __builtin_memcpy(x, &raw, 16);
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) x[e] = p[e];
  }
}
template <typename T, int VEC> __device__ __forceinline__ void store_vec(T* p, const T (&x)[VEC]) {
  if constexpr (VEC * sizeof(T) == 16) {
    u32x4 raw;
    __builtin_memcpy(&raw, x, 16);
    *(u32x4*)p = raw;
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) p[e] = x[e];
  }
}

struct AppendParams {
  const void *k, *v, *cos, *sin;
  const int64_t *pos, *tables, *offsets, *counts;
  void *kp, *vp;
  int64_t* pp;
  int64_t P;
  int64_t ks_b, ks_s, ks_h, vs_b, vs_s, vs_h, cs_b, cs_s, ss_b, ss_s;
  int64_t ps_b, ps_s, ts_b, ts_w, os_b, ns_b;
  int64_t kps_p, kps_h, kps_s, vps_p, vps_h, vps_s, pps_p, pps_s;
  int32_t B, n, H, D, W, page, total;  // total: threads with work
};

// Half-split rotary (the convention of apply_rotary): with h = D / 2,
//   out_i = x_i c_i - x_{i+h} s_i,   out_{i+h} = x_{i+h} c_{i+h} + x_i s_{i+h},
// in f32 (f64 for f64) and rounded once.  apply_rotary rounds both products and their sum, as the
// separate tensor ops that it replaces do; here nothing needs their intermediate values, and one
// rounding leaves 1 / sqrt(2) of that error.
//
// A thread owns VEC features of both halves of one token and head, so the 16-byte accesses of a
// row stay together whatever the page order; its slot comes from offsets and the table, two
// dependent reads that many resident waves hide.  Indices within a launch fit 32 bits, whose divisions
// are a fraction of 64-bit ones.
template <typename T, int VEC, bool ROT>
__global__ __launch_bounds__(256) void paged_append_kernel(const AppendParams p) {
  typedef typename acc_of<T>::type M;
  const uint32_t half = p.D / 2, nch = half / VEC;
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;  // (the launcher keeps it below 2^31)
  if (t >= (uint32_t)p.total) return;
  uint32_t r = t / nch;
  const uint32_t j = (t - r * nch) * VEC;
  const uint32_t h = r % (uint32_t)p.H;
  r /= (uint32_t)p.H;
  const uint32_t b = r / (uint32_t)p.n, s = r - b * p.n;
  const T* kr = (const T*)p.k + b * p.ks_b + s * p.ks_s + h * p.ks_h + j;
  const T* vr = (const T*)p.v + b * p.vs_b + s * p.vs_s + h * p.vs_h + j;
  // (the rows are read before the slot is known: both trips to memory at once)
  T k1[VEC], k2[VEC], v1[VEC], v2[VEC], c1[VEC], c2[VEC], s1[VEC], s2[VEC];
  load_vec<T, VEC>(kr, k1);
  load_vec<T, VEC>(kr + half, k2);
  load_vec<T, VEC>(vr, v1);
  load_vec<T, VEC>(vr + half, v2);
  if constexpr (ROT) {
    const T* cr = (const T*)p.cos + b * p.cs_b + s * p.cs_s + j;
    const T* sr = (const T*)p.sin + b * p.ss_b + s * p.ss_s + j;
    load_vec<T, VEC>(cr, c1);
    load_vec<T, VEC>(cr + half, c2);
    load_vec<T, VEC>(sr, s1);
    load_vec<T, VEC>(sr + half, s2);
  }
  const int64_t count = p.counts ? p.counts[b * p.ns_b] : p.n;
  const int64_t slot = p.offsets[b * p.os_b] + s;
  if (s >= count || slot < 0 || slot >= (int64_t)p.W * p.page) return;
  // (a table's slots nearly always fit 32 bits)
  const int64_t pg = slot <= INT32_MAX ? (int64_t)((uint32_t)slot / (uint32_t)p.page) : slot / p.page;
  const int64_t place = slot - pg * p.page;
  const int64_t id = p.tables[b * p.ts_b + pg * p.ts_w];
  if (id < 0 || id >= p.P) return;
  if constexpr (ROT) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const M x = load_acc<T, M>(&k1[e]), y = load_acc<T, M>(&k2[e]);
      k1[e] = store_cast<T, M>(x * load_acc<T, M>(&c1[e]) - y * load_acc<T, M>(&s1[e]));
      k2[e] = store_cast<T, M>(y * load_acc<T, M>(&c2[e]) + x * load_acc<T, M>(&s2[e]));
    }
  }
  T* ko = (T*)p.kp + id * p.kps_p + h * p.kps_h + place * p.kps_s + j;
  T* vo = (T*)p.vp + id * p.vps_p + h * p.vps_h + place * p.vps_s + j;
  store_vec<T, VEC>(ko, k1);
  store_vec<T, VEC>(ko + half, k2);
  store_vec<T, VEC>(vo, v1);
  store_vec<T, VEC>(vo + half, v2);
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
int append_typed(AppendParams& p, bool vec, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int64_t total = (int64_t)p.B * p.n * p.H * (p.D / 2 / (vec ? V : 1));
  CEA_REQUIRE(total <= INT32_MAX - 256, CEA_EUNSUPPORTED, "paged_kv_append: too many tokens for one call");
  p.total = (int32_t)total;
  const dim3 grid((unsigned)((total + 255) / 256));
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
constexpr int kMoves = 256;      // of a launch at most
constexpr int kFewMoves = 32;    // a small launch (a fork's): a tenth of the arguments

struct CopyPool {
  char* base;
  int64_t stride_n, stride_p;  // bytes
  int64_t bytes;               // of one page
  int32_t n;                   // pools in this tensor
  int32_t chunk0;              // first chunk of a move that is this tensor's
  int32_t chunks;              // chunks of one page
};
template <int NP, int NM> struct CopyParams {
  static constexpr int kPools = NP;
  int32_t npools, chunks, moves;
  CopyPool pool[NP];
  int32_t src[NM], dst[NM];
};

constexpr int kCopyChunk = 16384;  // bytes a workgroup copies: 4 vectors in flight per lane

template <typename V, int NP, int NM>
__global__ __launch_bounds__(256) void copy_pages_kernel(const CopyParams<NP, NM> p) {
  const int move = blockIdx.x / (uint32_t)p.chunks, chunk = blockIdx.x - move * p.chunks;
  int i = 0;
  if constexpr (NP > 1)
    while (i + 1 < p.npools && chunk >= p.pool[i + 1].chunk0) ++i;
  const CopyPool& c = p.pool[i];
  const int r = chunk - c.chunk0, n = r / (uint32_t)c.chunks;
  const int64_t at = (int64_t)(r - n * c.chunks) * kCopyChunk;
  const char* from = c.base + n * c.stride_n + p.src[move] * c.stride_p + at;
  char* to = c.base + n * c.stride_n + p.dst[move] * c.stride_p + at;
  const int left = (int)min(c.bytes - at, (int64_t)kCopyChunk);
  constexpr int PER = 4, STEP = 256 * sizeof(V);
  for (int o = threadIdx.x * sizeof(V); o < left; o += STEP * PER) {
    V x0{}, x1{}, x2{}, x3{};
    x0 = *(const V*)(from + o);
    if (o + STEP < left) x1 = *(const V*)(from + o + STEP);
    if (o + 2 * STEP < left) x2 = *(const V*)(from + o + 2 * STEP);
    if (o + 3 * STEP < left) x3 = *(const V*)(from + o + 3 * STEP);
    *(V*)(to + o) = x0;
    if (o + STEP < left) *(V*)(to + o + STEP) = x1;
    if (o + 2 * STEP < left) *(V*)(to + o + 2 * STEP) = x2;
    if (o + 3 * STEP < left) *(V*)(to + o + 3 * STEP) = x3;
  }
}

template <int NP, int NM>
int copy_moves(const CopyPool* pools, int npools, int64_t chunks, int vec, const int64_t* src, const int64_t* dst,
               int64_t m, hipStream_t st) {
  CopyParams<NP, NM> p = {};
  p.npools = npools, p.chunks = (int32_t)chunks;
  for (int i = 0; i < npools; ++i) p.pool[i] = pools[i];
  const int64_t per = std::max<int64_t>(1, std::min<int64_t>(NM, (((int64_t)1 << 31) - 1) / chunks));
  for (int64_t i = 0; i < m; i += per) {
    p.moves = (int32_t)std::min(per, m - i);
    for (int j = 0; j < p.moves; ++j) p.src[j] = (int32_t)src[i + j], p.dst[j] = (int32_t)dst[i + j];
    const dim3 grid((unsigned)(p.moves * chunks));
    if (vec == 16) hipLaunchKernelGGL((copy_pages_kernel<u32x4, NP, NM>), grid, dim3(256), 0, st, p);
    else if (vec == 4) hipLaunchKernelGGL((copy_pages_kernel<uint32_t, NP, NM>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((copy_pages_kernel<uint16_t, NP, NM>), grid, dim3(256), 0, st, p);
    CEA_CHECK_LAUNCH("copy_pages");
  }
  return CEA_OK;
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
  if (p.B == 0 || p.n == 0 || p.H == 0 || p.D == 0 || p.P == 0 || p.W == 0 || p.page == 0) return CEA_OK;
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
  CopyPool pool[CEA_MAX_PARTS] = {};
  int npools = 0;
  bool v16 = true, v4 = true;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    const cea_tensor& t = pools[i];
    const int64_t es = (int64_t)dtype_size(t.dtype);
    CopyPool& c = pool[npools];
    c.base = (char*)t.data;
    c.stride_n = t.stride[0] * es, c.stride_p = t.stride[1] * es;
    c.bytes = t.size[2] * es;
    c.n = (int32_t)t.size[0];
    if (c.n == 0 || c.bytes == 0) continue;
    c.chunk0 = (int32_t)chunks;
    const int64_t per_page = (c.bytes + kCopyChunk - 1) / kCopyChunk;
    chunks += c.n * per_page;
    CEA_REQUIRE(per_page < (int64_t)1 << 22 && chunks < (int64_t)1 << 22, CEA_EUNSUPPORTED,
                "copy_pages: pages too large");
    c.chunks = (int32_t)per_page;
    const int64_t a = (int64_t)(uintptr_t)c.base | (c.n > 1 ? c.stride_n : 0) | c.stride_p | c.bytes;
    v16 = v16 && a % 16 == 0, v4 = v4 && a % 4 == 0;
    ++npools;
  }
  if (npools == 0) return CEA_OK;
  const int vec = v16 ? 16 : v4 ? 4 : 2;
  if (npools == 1 && m <= kFewMoves) return copy_moves<1, kFewMoves>(pool, npools, chunks, vec, src, dst, m, st);
  return copy_moves<CEA_MAX_PARTS, kMoves>(pool, npools, chunks, vec, src, dst, m, st);
}

}  // namespace cea

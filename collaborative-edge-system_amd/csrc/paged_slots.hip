// Slots of a paged KV cache: the append into pages of 8 bits, reading rows back, and the bookkeeping of
// drafted trees - the ancestors of their nodes, and the accepted nodes' rows moved into line.  Appends, reads
// and moves are HBM-bound, every row read and written once; masks are bound by latency.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"

namespace cea {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename V, typename T> __device__ __forceinline__ void load_bytes(const void* p, T& x) {
  static_assert(sizeof(T) % sizeof(V) == 0, "whole vectors");
  V raw[sizeof(T) / sizeof(V)];
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / sizeof(V); ++i) raw[i] = ((const V*)p)[i];
  __builtin_memcpy(&x, raw, sizeof(T));
}
template <typename V, typename T> __device__ __forceinline__ void store_bytes(void* p, const T& x) {
  static_assert(sizeof(T) % sizeof(V) == 0, "whole vectors");
  V raw[sizeof(T) / sizeof(V)];
  __builtin_memcpy(raw, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / sizeof(V); ++i) ((V*)p)[i] = raw[i];
}

// Where slot j of row b is: its page, or -1, and its place there.
struct Rows {
  const int64_t *tables, *offsets, *counts;
  int64_t ts_b, ts_w, os_b, ns_b, P;
  int32_t W, page;
};
struct Place {
  int64_t id;
  int32_t at;
};
__device__ __forceinline__ Place place_of(const Rows& r, int b, int64_t slot) {
  if (slot < 0 || slot >= (int64_t)r.W * r.page) return {-1, 0};
  // (a table's slots nearly always fit 32 bits, whose division is a fraction of the 64-bit one)
  const int64_t pg = slot <= INT32_MAX ? (int64_t)((uint32_t)slot / (uint32_t)r.page) : slot / r.page;
  const int64_t id = r.tables[b * r.ts_b + pg * r.ts_w];
  return {id >= 0 && id < r.P ? id : -1, (int32_t)(slot - pg * r.page)};
}
__device__ __forceinline__ int64_t slot_after(int64_t offset, int64_t s) {
  return (int64_t)((uint64_t)offset + (uint64_t)s);  // (offsets may hold anything)
}

Rows rows_of(const cea_tensor* tables, const cea_tensor* offsets, const cea_tensor* counts, int64_t P, int64_t page) {
  Rows r = {};
  r.tables = (const int64_t*)tables->data, r.offsets = (const int64_t*)offsets->data;
  r.ts_b = tables->stride[0], r.ts_w = tables->stride[1], r.os_b = offsets->stride[0];
  if (counts) r.counts = (const int64_t*)counts->data, r.ns_b = counts->stride[0];
  r.P = P, r.W = (int32_t)tables->size[1], r.page = (int32_t)page;
  return r;
}

// A pool [N,] P, H, page, D: base pointer and strides.
struct Pool {
  char* base;
  int64_t s_p, s_h, s_s;
};
Pool pool_of(const cea_tensor* t) { return {(char*)t->data, t->stride[0], t->stride[1], t->stride[2]}; }
__device__ __forceinline__ int64_t at_of(const Pool& x, const Place& l, int h) {
  return l.id * x.s_p + h * x.s_h + l.at * x.s_s;
}

bool aligned_to(const cea_tensor* t, int bytes) {
  if (!t) return true;
  if ((uintptr_t)t->data % bytes) return false;
  for (int i = 0; i + 1 < t->ndim; ++i)
    if (t->size[i] > 1 && t->stride[i] * (int64_t)dtype_size(t->dtype) % bytes) return false;
  return true;
}

// ---------------------------------------------------------------------------------------
// appends into 8 bits
// ---------------------------------------------------------------------------------------
// A row x of D values and its largest finite magnitude m:
//   e = the smallest whole number >= -117 with m <= 448 * 2^e,   q = e4m3(x * 2^-e),   s = e + 127.
// e4m3 is a floating format, so a power of two as scale costs no precision, the product with it is exact,
// and what is read back is a bf16 or f16 number as it is.  The bound -117 keeps every number that is read
// back normal in f32 and bf16.
constexpr int kScaleBias = 127, kScaleMin = 10;

// Of an f32's bits: 448 = 1.75 * 2^8, so e is its exponent less 8, and one more above 1.75 of it.
__device__ __forceinline__ int scale_of(uint32_t top) {
  return max((int)(top >> 23) - 8 + ((top & 0x7fffff) > 0x600000 ? 1 : 0), kScaleMin);
}
// Only the row with the type's largest exponent could round to 256 * 2^e, which the type does not hold.
template <typename T> struct TypeTop { static constexpr int kScale = 247; };  // bf16, f32: below 2^128
template <> struct TypeTop<f16> { static constexpr int kScale = 135; };       // below 2^16

// Magnitude bits, 0 of what is not finite.
__device__ __forceinline__ uint32_t finite_bits(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
  return u < 0x7f800000u ? u : 0u;
}
// (the rotary of f16 rows may leave f16's range, f32's sums do not)
template <typename T> __device__ __forceinline__ float within(float x) {
  if constexpr (std::is_same<T, f16>::value)
    return finite_bits(x) != 0 ? __builtin_fminf(__builtin_fmaxf(x, -65504.f), 65504.f) : x;
  else
    return x;
}
template <typename T> __device__ __forceinline__ uint32_t quantise4(const float* x, int s) {
  float q[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    q[i] = ldexpf(x[i], kScaleBias - s);
    if (s == TypeTop<T>::kScale) q[i] = q[i] > 240.f ? 240.f : q[i] < -240.f ? -240.f : q[i];
    if (!is_finite(x[i])) q[i] = __builtin_nanf("");
  }
  int w = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], w, true);
  return (uint32_t)w;
}

struct Append8Params {
  const void *k, *v, *cos, *sin;
  const int64_t* pos;
  int64_t* pp;
  Rows rows;
  Pool kp, vp, ks, vs;
  int64_t ks_b, ks_s, ks_h, vs_b, vs_s, vs_h, cs_b, cs_s, ss_b, ss_s, ps_b, ps_s, pps_p, pps_s;
  int32_t B, n, H, D, total;
};

// A thread owns 8 features of both halves of a token and head, as in the 16-bit append; the D / 16
// threads of a row are neighbours in a wave and share its maxima.
template <typename T, bool ROT>
__global__ __launch_bounds__(256) void paged_append8_kernel(const Append8Params p) {
  constexpr int VEC = 8;
  const uint32_t half = p.D / 2, nch = half / VEC;  // (a power of two up to 16)
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  const bool live = t < (uint32_t)p.total;  // (whole rows: a row's threads live or end together)
  uint32_t r = live ? t / nch : 0;
  const uint32_t j = live ? (t - r * nch) * VEC : 0;
  const uint32_t h = r % (uint32_t)p.H;
  r /= (uint32_t)p.H;
  const uint32_t b = r / (uint32_t)p.n, s = r - b * p.n;
  const T* kr = (const T*)p.k + b * p.ks_b + s * p.ks_s + h * p.ks_h + j;
  const T* vr = (const T*)p.v + b * p.vs_b + s * p.vs_s + h * p.vs_h + j;
  // (everything is read before the slot is known: all trips to memory at once)
  T raw[4][VEC], c1[VEC], c2[VEC], s1[VEC], s2[VEC];
  load_bytes<u32x4>(kr, raw[0]);
  load_bytes<u32x4>(kr + half, raw[1]);
  load_bytes<u32x4>(vr, raw[2]);
  load_bytes<u32x4>(vr + half, raw[3]);
  if constexpr (ROT) {
    const T* cr = (const T*)p.cos + b * p.cs_b + s * p.cs_s + j;
    const T* sr = (const T*)p.sin + b * p.ss_b + s * p.ss_s + j;
    load_bytes<u32x4>(cr, c1);
    load_bytes<u32x4>(cr + half, c2);
    load_bytes<u32x4>(sr, s1);
    load_bytes<u32x4>(sr + half, s2);
  }
  const int64_t count = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : p.n;
  const Place at = place_of(p.rows, b, slot_after(p.rows.offsets[b * p.rows.os_b], s));
  float x[4][VEC];
  uint32_t top[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i][e] = to_f32<T>(raw[i][e]);
    if constexpr (ROT) {
      // out_i = x_i c_i - x_{i+h} s_i, out_{i+h} = x_{i+h} c_{i+h} + x_i s_{i+h}: products and sum rounded once each
      const float a = x[0][e], z = x[1][e];
      x[0][e] = within<T>(add_rn(mul_rn(a, to_f32<T>(c1[e])), -mul_rn(z, to_f32<T>(s1[e]))));
      x[1][e] = within<T>(add_rn(mul_rn(z, to_f32<T>(c2[e])), mul_rn(a, to_f32<T>(s2[e]))));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i >> 1] = max(top[i >> 1], finite_bits(x[i][e]));
  }
  for (uint32_t off = 1; off < nch; off <<= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], (int)off, 64));
  if (!live || s >= count || at.id < 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int sc = scale_of(top[i]);
    const Pool& pool = i == 0 ? p.kp : p.vp;
    const Pool& scales = i == 0 ? p.ks : p.vs;
    char* o = pool.base + at_of(pool, at, h) + j;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const u32x2 w = {quantise4<T>(x[2 * i + g], sc), quantise4<T>(x[2 * i + g] + 4, sc)};
      *(u32x2*)(o + g * half) = w;
    }
    if (j == 0) scales.base[at_of(scales, at, h)] = (char)sc;
  }
  if (p.pp && h == 0 && j == 0)
    p.pp[at.id * p.pps_p + at.at * p.pps_s] = p.pos[b * p.ps_b + s * p.ps_s];
}

// The same for any head size and alignment: a wave per token and head, one feature a lane at a time, over
// the row twice (its maxima, then the numbers).
template <typename T, bool ROT>
__global__ __launch_bounds__(256) void paged_append8_any_kernel(const Append8Params p) {
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, half = p.D / 2;
  if (row >= p.total) return;
  const int h = (int)(row % p.H);
  const int s = (int)(row / p.H % p.n), b = (int)(row / ((int64_t)p.H * p.n));
  const int64_t count = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : p.n;
  const Place at = place_of(p.rows, b, slot_after(p.rows.offsets[b * p.rows.os_b], s));
  if (s >= count || at.id < 0) return;
  const T* kr = (const T*)p.k + b * p.ks_b + s * p.ks_s + h * p.ks_h;
  const T* vr = (const T*)p.v + b * p.vs_b + s * p.vs_s + h * p.vs_h;
  const T* cr = (const T*)p.cos + b * p.cs_b + s * p.cs_s;
  const T* sr = (const T*)p.sin + b * p.ss_b + s * p.ss_s;
  auto key = [&](int d) -> float {
    const float x = to_f32<T>(kr[d]);
    if constexpr (!ROT) return x;
    const float y = to_f32<T>(kr[d < half ? d + half : d - half]);
    const float z = mul_rn(y, to_f32<T>(sr[d]));
    return within<T>(add_rn(mul_rn(x, to_f32<T>(cr[d])), d < half ? -z : z));
  };
  uint32_t top[2] = {0, 0};
  for (int d = lane; d < p.D; d += 64) {
    top[0] = max(top[0], finite_bits(key(d)));
    top[1] = max(top[1], finite_bits(to_f32<T>(vr[d])));
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    for (int off = 1; off < 64; off <<= 1) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], off, 64));
    const int sc = scale_of(top[i]);
    const Pool& pool = i == 0 ? p.kp : p.vp;
    const Pool& scales = i == 0 ? p.ks : p.vs;
    for (int d = lane; d < p.D; d += 64) {
      const float x[4] = {i == 0 ? key(d) : to_f32<T>(vr[d]), 0.f, 0.f, 0.f};
      pool.base[at_of(pool, at, h) + d] = (char)quantise4<T>(x, sc);
    }
    if (lane == 0) scales.base[at_of(scales, at, h)] = (char)sc;
  }
  if (p.pp && h == 0 && lane == 0) p.pp[at.id * p.pps_p + at.at * p.pps_s] = p.pos[b * p.ps_b + s * p.ps_s];
}

template <typename T> int append8_typed(Append8Params& p, bool vec, hipStream_t st) {
  const int64_t rows = (int64_t)p.B * p.n * p.H, total = vec ? rows * (p.D / 16) : rows;
  CEA_REQUIRE(total <= INT32_MAX - 256, CEA_EUNSUPPORTED, "paged_kv_append: too many tokens for one call");
  p.total = (int32_t)total;
  const dim3 grid((unsigned)(vec ? (total + 255) / 256 : (total + 3) / 4));
  if (vec && p.cos) hipLaunchKernelGGL((paged_append8_kernel<T, true>), grid, dim3(256), 0, st, p);
  else if (vec) hipLaunchKernelGGL((paged_append8_kernel<T, false>), grid, dim3(256), 0, st, p);
  else if (p.cos) hipLaunchKernelGGL((paged_append8_any_kernel<T, true>), grid, dim3(256), 0, st, p);
  else hipLaunchKernelGGL((paged_append8_any_kernel<T, false>), grid, dim3(256), 0, st, p);
  CEA_CHECK_LAUNCH("paged_kv_append");
  return CEA_OK;
}

// ---------------------------------------------------------------------------------------
// reading back
// ---------------------------------------------------------------------------------------
struct ReadParams {
  Rows rows;
  Pool pool[2], scales[2];
  char* out[2];
  int64_t os_b[2], os_s[2], os_h[2];
  int32_t B, n, H, D, total;
};

// VEC e4m3 numbers and their row's scale as values of O.  bf16 holds q * 2^(s - 127) as it is; f16 rounds
// what is below its normal numbers and overflows to infinity.
template <typename O, int VEC> __device__ __forceinline__ void widen(const uint8_t (&q)[VEC], int s, O (&x)[VEC]) {
#pragma unroll
  for (int i = 0; i < VEC; ++i) x[i] = (O)ldexpf(__builtin_amdgcn_cvt_f32_fp8(q[i], 0), s - kScaleBias);
}

// A thread owns VEC features of a slot and head, of the keys or of the values.
template <typename I, typename O, int VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(const ReadParams p) {
  const uint32_t nch = p.D / VEC;
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  if (t >= (uint32_t)p.total) return;
  uint32_t r = t / nch;
  const uint32_t j = (t - r * nch) * VEC;
  const uint32_t h = r % (uint32_t)p.H;
  r /= (uint32_t)p.H;
  const uint32_t b = r / (uint32_t)p.n, s = r - b * p.n;
  const int kv = blockIdx.y;
  const int64_t count = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : p.n;
  const Place at = s < count ? place_of(p.rows, b, slot_after(p.rows.offsets[b * p.rows.os_b], s)) : Place{-1, 0};
  O x[VEC] = {};
  if (at.id >= 0) {
    const I* from = (const I*)p.pool[kv].base + at_of(p.pool[kv], at, h) + j;
    if constexpr (std::is_same<I, uint8_t>::value) {
      uint8_t q[VEC];
      if constexpr (VEC == 1) q[0] = *from;
      else load_bytes<std::conditional_t<VEC % 16 == 0, u32x4, u32x2>>(from, q);
      widen<O, VEC>(q, ((const uint8_t*)p.scales[kv].base)[at_of(p.scales[kv], at, h)], x);
    } else if constexpr (VEC == 1) {
      x[0] = *from;
    } else {
      load_bytes<u32x4>(from, x);
    }
  }
  O* to = (O*)p.out[kv] + b * p.os_b[kv] + s * p.os_s[kv] + h * p.os_h[kv] + j;
  if constexpr (VEC == 1) *to = x[0];
  else store_bytes<u32x4>(to, x);
}

template <typename I, typename O, int VEC> int read_typed(ReadParams& p, hipStream_t st) {
  const int64_t total = (int64_t)p.B * p.n * p.H * (p.D / VEC);
  CEA_REQUIRE(total <= INT32_MAX - 256, CEA_EUNSUPPORTED, "paged_kv_read: too many tokens for one call");
  p.total = (int32_t)total;
  hipLaunchKernelGGL((paged_read_kernel<I, O, VEC>), dim3((unsigned)((total + 255) / 256), 2), dim3(256), 0, st, p);
  CEA_CHECK_LAUNCH("paged_kv_read");
  return CEA_OK;
}

// ---------------------------------------------------------------------------------------
// keeping accepted nodes
// ---------------------------------------------------------------------------------------
struct KeepParams {
  Rows rows;
  const int64_t* path;
  int64_t ps_b, ps_i;
  char *kv, *scales;
  int64_t s_n, s_p, s_h, s_s;      // bytes
  int64_t ss_n, ss_p, ss_h, ss_s;  // bytes
  int32_t B, H, n, nch, all;       // nch: vectors of a row; all: pools * B * H
};

// Slot base + i takes what slot base + path[i] held.  A thread owns a vector of a row, or its scale, in all
// the slots of one sequence, head and pool, so it alone reads and writes there: eight are read, then written.
// Entries with path[i] < i move nothing, so a source is never a slot that an earlier turn has written.
template <typename V>
__global__ __launch_bounds__(256) void paged_keep_kernel(const KeepParams p) {
  constexpr int TURN = 8;
  const int per = p.nch + (p.scales ? 1 : 0);
  const uint32_t t = blockIdx.x * 256 + threadIdx.x;
  uint32_t r = t / (uint32_t)per;
  if (r >= (uint32_t)p.all) return;
  const int c = (int)(t - r * per);
  const int h = (int)(r % (uint32_t)p.H);
  r /= (uint32_t)p.H;
  const int n = (int)(r / (uint32_t)p.B), b = (int)(r - (uint32_t)n * p.B);
  const int64_t base = p.rows.offsets[b * p.rows.os_b];
  const int64_t nodes = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : INT64_MAX;
  const bool scale = c == p.nch;
  char* pool = scale ? p.scales + n * p.ss_n + h * p.ss_h : p.kv + n * p.s_n + h * p.s_h + (int64_t)c * sizeof(V);
  const int64_t s_p = scale ? p.ss_p : p.s_p, s_s = scale ? p.ss_s : p.s_s;
  for (int i0 = 0; i0 < p.n; i0 += TURN) {
    V x[TURN] = {};
    char* to[TURN];
#pragma unroll
    for (int k = 0; k < TURN; ++k) {
      const int i = i0 + k;
      to[k] = nullptr;
      if (i >= p.n) continue;
      const int64_t node = p.path[b * p.ps_b + i * p.ps_i];
      if (node <= i || node >= nodes) continue;  // (node i is in its place)
      const Place from = place_of(p.rows, b, slot_after(base, node)), at = place_of(p.rows, b, slot_after(base, i));
      if (from.id < 0 || at.id < 0) continue;
      to[k] = pool + at.id * s_p + at.at * s_s;
      const char* src = pool + from.id * s_p + from.at * s_s;
      if (scale) {
        const uint8_t y = *(const uint8_t*)src;
        __builtin_memcpy(&x[k], &y, 1);
      } else {
        x[k] = *(const V*)src;
      }
    }
#pragma unroll
    for (int k = 0; k < TURN; ++k) {
      if (to[k] == nullptr) continue;
      if (scale) {
        uint8_t y;
        __builtin_memcpy(&y, &x[k], 1);
        *(uint8_t*)to[k] = y;
      } else {
        *(V*)to[k] = x[k];
      }
    }
  }
}

// ---------------------------------------------------------------------------------------
// masks of trees
// ---------------------------------------------------------------------------------------
struct MaskParams {
  const int64_t *parents, *counts;
  int64_t *masks, *depths;
  int64_t ps_b, ps_t, ns_b, ms_b, ms_t, ms_w, ds_b, ds_t;
  int32_t T, words;
};

// Every node starts with its own bit and a link to its parent, and takes, round by round, the bits of the
// node that it links to and that node's link: after k rounds it holds 2^k nodes of its line.  A workgroup
// per row; the lines are in LDS, what a round reads and what it writes apart.
__global__ __launch_bounds__(512) void tree_masks_kernel(const MaskParams p) {
  extern __shared__ uint64_t bits[];  // [2][T * words], then int16 links [2][T]
  const int b = blockIdx.x, T = p.T, words = p.words, n = T * words;
  int16_t* link = (int16_t*)(bits + 2 * n);
  int64_t count = p.counts ? p.counts[b * p.ns_b] : T;
  count = count < 0 ? 0 : count < T ? count : T;
  for (int i = threadIdx.x; i < T; i += blockDim.x) {
    const int64_t up = i < count ? p.parents[b * p.ps_b + i * p.ps_t] : -1;
    link[i] = (int16_t)(up >= 0 && up < i ? up : -1);
  }
  for (int x = threadIdx.x; x < n; x += blockDim.x) {
    const int i = x / words, w = x - i * words;
    bits[x] = i < count && w == i >> 6 ? (uint64_t)1 << (i & 63) : 0;
  }
  int cur = 0;
  for (int span = 1; span < T; span *= 2) {
    __syncthreads();
    bool more = false;
    const uint64_t* from = bits + cur * n;
    uint64_t* to = bits + (cur ^ 1) * n;
    for (int x = threadIdx.x; x < n; x += blockDim.x) {
      const int i = x / words, w = x - i * words, up = link[cur * T + i];
      to[x] = from[x] | (up >= 0 ? from[up * words + w] : 0);
      if (w == 0) {
        const int16_t next = up >= 0 ? link[cur * T + up] : (int16_t)-1;
        link[(cur ^ 1) * T + i] = next;
        more = more || next >= 0;
      }
    }
    cur ^= 1;
    if (__syncthreads_or(more) == 0) break;
  }
  __syncthreads();
  const uint64_t* done = bits + cur * n;
  for (int x = threadIdx.x; x < n; x += blockDim.x) {
    const int i = x / words, w = x - i * words;
    p.masks[b * p.ms_b + i * p.ms_t + w * p.ms_w] = (int64_t)done[x];
  }
  for (int i = threadIdx.x; i < T; i += blockDim.x) {
    int line = 0;
    for (int w = 0; w < words; ++w) line += __builtin_popcountll(done[i * words + w]);
    p.depths[b * p.ds_b + i * p.ds_t] = line > 0 ? line - 1 : 0;
  }
}

}  // namespace

int launch_paged_append8(const cea_tensor* k, const cea_tensor* v, const cea_tensor* pos, const cea_tensor* c,
                         const cea_tensor* sn, const cea_tensor* tables, const cea_tensor* offsets,
                         const cea_tensor* counts, cea_tensor* kp, cea_tensor* vp, cea_tensor* ks, cea_tensor* vs,
                         cea_tensor* pp, hipStream_t st) {
  Append8Params p = {};
  p.k = k->data, p.v = v->data;
  p.rows = rows_of(tables, offsets, counts, kp->size[0], kp->size[2]);
  p.kp = pool_of(kp), p.vp = pool_of(vp), p.ks = pool_of(ks), p.vs = pool_of(vs);
  p.B = (int)k->size[0], p.n = (int)k->size[1], p.H = (int)k->size[2], p.D = (int)k->size[3];
  p.ks_b = k->stride[0], p.ks_s = k->stride[1], p.ks_h = k->stride[2];
  p.vs_b = v->stride[0], p.vs_s = v->stride[1], p.vs_h = v->stride[2];
  if (pp) {
    p.pp = (int64_t*)pp->data, p.pps_p = pp->stride[0], p.pps_s = pp->stride[1];
    p.pos = (const int64_t*)pos->data, p.ps_b = pos->stride[0], p.ps_s = pos->stride[1];
  }
  if (c) {
    p.cos = c->data, p.sin = sn->data;
    p.cs_b = c->stride[0], p.cs_s = c->stride[1], p.ss_b = sn->stride[0], p.ss_s = sn->stride[1];
  }
  if (p.B == 0 || p.n == 0 || p.H == 0 || p.D == 0 || p.rows.P == 0 || p.rows.W == 0 || p.rows.page == 0) return CEA_OK;
  // a row's threads are D / 16 neighbours of one wave
  bool vec = p.D == 16 || p.D == 32 || p.D == 64 || p.D == 128 || p.D == 256;
  for (const cea_tensor* t : {k, v, c, sn}) vec = vec && aligned_to(t, 16);
  for (const cea_tensor* t : {kp, vp}) vec = vec && aligned_to(t, 8);
  switch (k->dtype) {
    case CEA_BF16: return append8_typed<bf16>(p, vec, st);
    case CEA_F16: return append8_typed<f16>(p, vec, st);
    case CEA_F32: return append8_typed<float>(p, vec, st);
  }
  set_error("paged_kv_append: unsupported dtype %s", dtype_name(k->dtype));
  return CEA_EUNSUPPORTED;
}

int launch_paged_read(const cea_tensor* kp, const cea_tensor* vp, const cea_tensor* ks, const cea_tensor* vs,
                      const cea_tensor* tables, const cea_tensor* offsets, const cea_tensor* counts, cea_tensor* k,
                      cea_tensor* v, hipStream_t st) {
  ReadParams p = {};
  p.rows = rows_of(tables, offsets, counts, kp->size[0], kp->size[2]);
  if (p.rows.P == 0 || p.rows.page == 0) p.rows.W = 0, p.rows.page = 1;  // no slots: everything is 0
  p.B = (int)k->size[0], p.n = (int)k->size[1], p.H = (int)k->size[2], p.D = (int)k->size[3];
  p.pool[0] = pool_of(kp), p.pool[1] = pool_of(vp);
  if (ks) p.scales[0] = pool_of(ks), p.scales[1] = pool_of(vs);
  const cea_tensor* out[2] = {k, v};
  for (int i = 0; i < 2; ++i) {
    p.out[i] = (char*)out[i]->data;
    p.os_b[i] = out[i]->stride[0], p.os_s[i] = out[i]->stride[1], p.os_h[i] = out[i]->stride[2];
  }
  if (p.B == 0 || p.n == 0 || p.H == 0 || p.D == 0) return CEA_OK;
  const bool outs = aligned_to(k, 16) && aligned_to(v, 16);
  if (ks) {
    const bool vec = outs && p.D % 8 == 0 && aligned_to(kp, 8) && aligned_to(vp, 8);
    switch (k->dtype) {
      case CEA_BF16: return vec ? read_typed<uint8_t, bf16, 8>(p, st) : read_typed<uint8_t, bf16, 1>(p, st);
      case CEA_F16: return vec ? read_typed<uint8_t, f16, 8>(p, st) : read_typed<uint8_t, f16, 1>(p, st);
      case CEA_F32: return vec ? read_typed<uint8_t, float, 8>(p, st) : read_typed<uint8_t, float, 1>(p, st);
    }
  } else {
    // (as bytes of the element's size)
    const int size = (int)dtype_size(k->dtype), per = 16 / size;
    const bool vec = outs && p.D % per == 0 && aligned_to(kp, 16) && aligned_to(vp, 16);
    switch (size) {
      case 2: return vec ? read_typed<uint16_t, uint16_t, 8>(p, st) : read_typed<uint16_t, uint16_t, 1>(p, st);
      case 4: return vec ? read_typed<uint32_t, uint32_t, 4>(p, st) : read_typed<uint32_t, uint32_t, 1>(p, st);
      case 8: return vec ? read_typed<uint64_t, uint64_t, 2>(p, st) : read_typed<uint64_t, uint64_t, 1>(p, st);
    }
  }
  set_error("paged_kv_read: unsupported dtype %s", dtype_name(k->dtype));
  return CEA_EUNSUPPORTED;
}

int launch_paged_keep(cea_tensor* kv, cea_tensor* scales, int page, const cea_tensor* tables,
                      const cea_tensor* offsets, const cea_tensor* counts, const cea_tensor* path, hipStream_t st) {
  const int64_t es = (int64_t)dtype_size(kv->dtype), B = path->size[0], N = kv->size[0], H = kv->size[2];
  if (N == 0 || B == 0 || H == 0 || page == 0 || kv->size[1] == 0 || kv->size[3] == 0 || path->size[1] == 0 ||
      tables->size[1] == 0)
    return CEA_OK;
  KeepParams p = {};
  p.rows = rows_of(tables, offsets, counts, kv->size[1], page);
  p.path = (const int64_t*)path->data, p.ps_b = path->stride[0], p.ps_i = path->stride[1];
  p.kv = (char*)kv->data;
  p.s_n = kv->stride[0] * es, p.s_p = kv->stride[1] * es, p.s_h = kv->stride[2] * es;
  p.s_s = kv->size[3] / page * es;
  if (scales) {
    p.scales = (char*)scales->data;
    p.ss_n = scales->stride[0], p.ss_p = scales->stride[1], p.ss_h = scales->stride[2], p.ss_s = scales->stride[3];
  }
  p.B = (int)B, p.H = (int)H, p.n = (int)path->size[1];
  const int64_t bits = (int64_t)(uintptr_t)p.kv | (N > 1 ? p.s_n : 0) | p.s_p | p.s_h | p.s_s;
  const int vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  p.nch = (int)(p.s_s / vec);
  const int64_t all = N * B * H, threads = all * (p.nch + (scales ? 1 : 0));
  CEA_REQUIRE(threads <= INT32_MAX - 256, CEA_EUNSUPPORTED, "paged_kv_keep: too many rows for one call");
  p.all = (int)all;
  const dim3 grid((unsigned)((threads + 255) / 256));
  switch (vec) {
    case 16: hipLaunchKernelGGL((paged_keep_kernel<u32x4>), grid, dim3(256), 0, st, p); break;
    case 4: hipLaunchKernelGGL((paged_keep_kernel<uint32_t>), grid, dim3(256), 0, st, p); break;
    case 2: hipLaunchKernelGGL((paged_keep_kernel<uint16_t>), grid, dim3(256), 0, st, p); break;
    default: hipLaunchKernelGGL((paged_keep_kernel<uint8_t>), grid, dim3(256), 0, st, p); break;
  }
  CEA_CHECK_LAUNCH("paged_kv_keep");
  return CEA_OK;
}

int launch_tree_masks(const cea_tensor* parents, const cea_tensor* counts, cea_tensor* masks, cea_tensor* depths,
                      hipStream_t st) {
  MaskParams p = {};
  p.parents = (const int64_t*)parents->data, p.ps_b = parents->stride[0], p.ps_t = parents->stride[1];
  if (counts) p.counts = (const int64_t*)counts->data, p.ns_b = counts->stride[0];
  p.masks = (int64_t*)masks->data, p.depths = (int64_t*)depths->data;
  p.ms_b = masks->stride[0], p.ms_t = masks->stride[1], p.ms_w = masks->stride[2];
  p.ds_b = depths->stride[0], p.ds_t = depths->stride[1];
  p.T = (int)parents->size[1], p.words = (int)masks->size[2];
  const int64_t B = parents->size[0];
  if (B == 0 || p.T == 0) return CEA_OK;
  const int lds = 2 * p.T * p.words * 8 + 2 * p.T * 2;
  constexpr int most = 2 * CEA_MAX_TREE * (CEA_MAX_TREE / 64) * 8 + 2 * CEA_MAX_TREE * 2;
  const hipError_t e = reserve_lds<tree_masks_kernel>(most);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "tree_masks: cannot reserve %d bytes of LDS: %s", most,
              hipGetErrorString(e));
  const int threads = std::min(512, (p.T * p.words + 63) / 64 * 64);
  hipLaunchKernelGGL(tree_masks_kernel, dim3((unsigned)B), dim3(threads), lds, st, p);
  CEA_CHECK_LAUNCH("tree_masks");
  return CEA_OK;
}

}  // namespace cea

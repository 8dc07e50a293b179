// Slots of a paged KV cache: the append into pages of 8 bits, reading rows back, and the bookkeeping of
// drafted trees - the ancestors of their nodes, and the accepted nodes' rows moved into line.  Appends, reads
// and moves are HBM-bound, every row read and written once; masks are bound by latency.  Measured, us a call in a
// stream of calls on new data (a 1 GB copy moves 5.1 TB/s):
//   * append: 2 x 4096 tokens of 8 heads of 128 from f16 (55 MB) 13.9, 3.9 TB/s; 32 single tokens 9.0, the call's own
//     cost, 3.8 on the GPU;
//   * read: 30000 slots of 8 heads of 128 into bf16 (185 MB) 33, 5.6 TB/s;
//     8 rows of 350 to 700, 4 heads of 64, 11.0, 7.5 on the GPU: a chain of offsets, tables and rows, in waves of which a
//     token's 32 vectors fill half;
//   * moves: up to 9 nodes of 32 rows in 64 pools of 8 heads of 128 (28 MB) 11.1, 2.6 TB/s: three dependent trips to
//     memory (path and offsets, tables, rows), and behind the first 64 vectors' stores a second turn of up to 8, behind
//     that one's the scale bytes; 4 nodes of one row in 44 pools 8.0, 4.3 on the GPU;
//   * masks: 64 trees of 250 nodes 9.4 (5.6 on the GPU), one of 26 9.3 (1.8): the call's own cost.
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
// (past the caches)
template <typename V, typename T> __device__ __forceinline__ void store_bytes(void* p, const T& x) {
  static_assert(sizeof(T) % sizeof(V) == 0, "whole vectors");
  V raw[sizeof(T) / sizeof(V)];
  __builtin_memcpy(raw, &x, sizeof(T));
#pragma unroll
  for (size_t i = 0; i < sizeof(T) / sizeof(V); ++i) __builtin_nontemporal_store(raw[i], (V*)p + i);
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
constexpr uint32_t kInfBits = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t finite_bits(float x) { return magnitude(x) < kInfBits ? magnitude(x) : 0u; }
// (the rotary of f16 rows may leave f16's range, f32's sums do not)
template <typename T> __device__ __forceinline__ float within(float x) {
  if constexpr (std::is_same<T, f16>::value)
    return finite_bits(x) != 0 ? __builtin_fminf(__builtin_fmaxf(x, -65504.f), 65504.f) : x;
  else
    return x;
}
// Four values as numbers of the scale s, whatever they are.
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
// Eight values of a row that is finite and below its type's top scale, which is nearly every row: two an
// instruction, v_cvt_scalef32_pk_fp8, which divides by the scale as it rounds.
typedef short i16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ u32x2 quantise8(const float* x, float scale) {
  u32x2 w;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    i16x2 y = {0, 0};
    y = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(y, x[4 * i], x[4 * i + 1], scale, false);
    y = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(y, x[4 * i + 2], x[4 * i + 3], scale, true);
    w[i] = __builtin_bit_cast(uint32_t, y);
  }
  return w;
}
template <typename T> __device__ __forceinline__ u32x2 quantise8(const T (&x)[8], float scale) {
  if constexpr (sizeof(T) == 4) {
    return quantise8(&x[0], scale);
  } else {
    typedef T pair __attribute__((ext_vector_type(2)));
    u32x2 w;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      i16x2 y = {0, 0};
      const pair a = {x[4 * i], x[4 * i + 1]}, b = {x[4 * i + 2], x[4 * i + 3]};
      if constexpr (std::is_same<T, bf16>::value) {
        y = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(y, a, scale, false);
        y = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(y, b, scale, true);
      } else {
        y = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(y, a, scale, false);
        y = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(y, b, scale, true);
      }
      w[i] = __builtin_bit_cast(uint32_t, y);
    }
    return w;
  }
}
// The largest magnitude of eight values as an f32's bits, infinities and NaN among them.  (16-bit types: two
// an instruction, in their own bits, whose order is that of the magnitudes.)
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
template <typename T> __device__ __forceinline__ uint32_t top8(const T (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, magnitude(x[e]));
    return top;
  } else {
    u32x4 raw;
    __builtin_memcpy(&raw, x, 16);
    u16x2 top = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2, (uint32_t)(raw[i] & 0x7fff7fffu)));
    const uint16_t one = max(top[0], top[1]);
    return magnitude(to_f32<T>(__builtin_bit_cast(T, one)));
  }
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
// threads of a row are neighbours in a wave and share its maxima.  Maxima and numbers two values an instruction
// while the wave's rows are finite and below the type's top scale (value by value 2 x 4096 tokens took 16.4 us, so
// 13.9).
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
  float k[2][VEC];  // the rotated key
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    const float a = to_f32<T>(raw[0][e]), z = to_f32<T>(raw[1][e]);
    k[0][e] = a, k[1][e] = z;
    if constexpr (ROT) {
      // out_i = x_i c_i - x_{i+h} s_i, out_{i+h} = x_{i+h} c_{i+h} + x_i s_{i+h}: products and sum rounded once each
      k[0][e] = add_rn(mul_rn(a, to_f32<T>(c1[e])), -mul_rn(z, to_f32<T>(s1[e])));
      k[1][e] = add_rn(mul_rn(z, to_f32<T>(c2[e])), mul_rn(a, to_f32<T>(s2[e])));
    }
  }
  uint32_t top[2] = {ROT ? max(top8(k[0]), top8(k[1])) : max(top8(raw[0]), top8(raw[1])), max(top8(raw[2]), top8(raw[3]))};
  for (uint32_t off = 1; off < nch; off <<= 1)
#pragma unroll
    for (int i = 0; i < 2; ++i) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], (int)off, 64));
  constexpr uint32_t kPlain = std::is_same<T, f16>::value ? 0x477fe000u : kInfBits - 1;  // the type's largest
  bool plain = true;
  int sc[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    sc[i] = scale_of(top[i]);
    plain = plain && top[i] <= kPlain && sc[i] != TypeTop<T>::kScale;
  }
  u32x2 w[4];
  if (__ballot(!plain) == 0) {
    const float f[2] = {scale_value(sc[0]), scale_value(sc[1])};
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      w[g] = ROT ? quantise8(&k[g][0], f[0]) : quantise8<T>(raw[g], f[0]);
      w[2 + g] = quantise8<T>(raw[2 + g], f[1]);
    }
  } else {
    float x[4][VEC];
    top[0] = top[1] = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        x[i][e] = i < 2 ? within<T>(k[i & 1][e]) : to_f32<T>(raw[i][e]);
        top[i >> 1] = max(top[i >> 1], finite_bits(x[i][e]));
      }
    for (uint32_t off = 1; off < nch; off <<= 1)
#pragma unroll
      for (int i = 0; i < 2; ++i) top[i] = max(top[i], (uint32_t)__shfl_xor((int)top[i], (int)off, 64));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sc[i >> 1] = scale_of(top[i >> 1]);
      w[i] = u32x2{quantise4<T>(x[i], sc[i >> 1]), quantise4<T>(x[i] + 4, sc[i >> 1])};
    }
  }
  if (!live || s >= count || at.id < 0) return;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const Pool& pool = i == 0 ? p.kp : p.vp;
    const Pool& scales = i == 0 ? p.ks : p.vs;
    char* o = pool.base + at_of(pool, at, h) + j;
    *(u32x2*)o = w[2 * i];
    *(u32x2*)(o + half) = w[2 * i + 1];
    if (j == 0) scales.base[at_of(scales, at, h)] = (char)sc[i];
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
  int32_t B, n, H, D, items, turns;  // items: vectors of a token; turns: groups of slots of a row
};

// VEC elements of the pages as values of O, two of 8 bits an instruction.
template <typename I, typename O, int VEC> __device__ __forceinline__ void convert(const I (&q)[VEC], int s, O (&x)[VEC]) {
  if constexpr (!std::is_same<I, uint8_t>::value) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = q[i];
  } else if constexpr (sizeof(O) == 4) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) x[i] = ldexpf(__builtin_amdgcn_cvt_f32_fp8(q[i], 0), s - kScaleBias);
  } else if constexpr (VEC == 8) {
    u32x2 raw;
    __builtin_memcpy(&raw, q, 8);
    const float f = scale_value(s);
    const u32x4 y = {widen2<O, false>(raw[0], f), widen2<O, true>(raw[0], f), widen2<O, false>(raw[1], f),
                     widen2<O, true>(raw[1], f)};
    __builtin_memcpy(x, &y, 16);
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const uint16_t y = (uint16_t)widen2<O, false>(q[i], scale_value(s));
      __builtin_memcpy(&x[i], &y, 2);
    }
  }
}

// A wave owns kReadSlots slots of a row and takes the tokens' vectors 64 at a time: where the slots are is known
// once for all of them, and keys and values of all its slots are under way together.  (A vector a thread, each
// with its own way to its slot: 30000 slots of 8 heads of 128 77 us, so 52; with the rows written past the caches, where
// they pushed the pages out, 33.)
constexpr int kReadSlots = 4;
template <typename I, typename O, int VEC>
__global__ __launch_bounds__(256) void paged_read_kernel(const ReadParams p) {
  const int lane = threadIdx.x & 63;
  const uint32_t group = blockIdx.x * 4 + uniform(threadIdx.x >> 6);
  const uint32_t b = group / (uint32_t)p.turns;
  if (b >= (uint32_t)p.B) return;
  const int s0 = (int)(group - b * p.turns) * kReadSlots;
  const int64_t count = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : p.n;
  const int64_t first = p.rows.offsets[b * p.rows.os_b];
  Place at[kReadSlots];
#pragma unroll
  for (int i = 0; i < kReadSlots; ++i)
    at[i] = s0 + i < count && s0 + i < p.n ? place_of(p.rows, b, slot_after(first, s0 + i)) : Place{-1, 0};
  const uint32_t nch = p.D / VEC;
  for (int item = lane; item < p.items; item += 64) {
    const uint32_t h = (uint32_t)item / nch, j = ((uint32_t)item - h * nch) * VEC;
    I q[2][kReadSlots][VEC] = {};
    int s[2][kReadSlots] = {};
#pragma unroll
    for (int i = 0; i < kReadSlots; ++i)
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        if (at[i].id >= 0) {
          const I* from = (const I*)p.pool[kv].base + at_of(p.pool[kv], at[i], h) + j;
          if constexpr (VEC == 1) q[kv][i][0] = *from;
          else load_bytes<std::conditional_t<sizeof(I) * VEC == 16, u32x4, u32x2>>(from, q[kv][i]);
          if constexpr (std::is_same<I, uint8_t>::value)
            s[kv][i] = ((const uint8_t*)p.scales[kv].base)[at_of(p.scales[kv], at[i], h)];
        }
#pragma unroll
    for (int i = 0; i < kReadSlots; ++i)
#pragma unroll
      for (int kv = 0; kv < 2; ++kv)
        if (s0 + i < p.n) {
          O x[VEC];
          convert<I, O, VEC>(q[kv][i], s[kv][i], x);
          O* to = (O*)p.out[kv] + b * p.os_b[kv] + (s0 + i) * p.os_s[kv] + h * p.os_h[kv] + j;
          if constexpr (VEC == 1) *to = x[0];
          else store_bytes<u32x4>(to, x);
        }
  }
}

template <typename I, typename O, int VEC> int read_typed(ReadParams& p, hipStream_t st) {
  const int64_t items = (int64_t)p.H * (p.D / VEC), turns = ((int64_t)p.n + kReadSlots - 1) / kReadSlots;
  CEA_REQUIRE(items <= INT32_MAX - 64 && turns * p.B <= INT32_MAX - 4, CEA_EUNSUPPORTED,
              "paged_kv_read: too many tokens for one call");
  p.items = (int32_t)items, p.turns = (int32_t)turns;
  hipLaunchKernelGGL((paged_read_kernel<I, O, VEC>), dim3((unsigned)((turns * p.B + 3) / 4)), dim3(256), 0, st, p);
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
  int32_t H, n, nch, pairs;        // nch: vectors of a row; pairs: pools times heads
};

// Slot base + i takes what slot base + path[i] held.  A workgroup serves kKeepPairs (pool, head) pairs of one
// row: a wave finds where up to 64 entries' slots are and lists those that move, then every wave takes four
// pairs and moves their vectors, 64 (entry, vector) at a time, of all four at once.  Entries with path[i] <= i
// move nothing, so a source lies behind every slot that an earlier step of the wave has written, and within a
// step all loads come before the stores.  (A vector of one pool a thread, entry after entry: 20.4 us for 9 nodes of
// 32 rows in 64 pools, so 11.1.)
constexpr int kKeepPairs = 16;
template <typename V>
__global__ __launch_bounds__(256) void paged_keep_kernel(const KeepParams p) {
  constexpr int PER = kKeepPairs / 4;
  __shared__ int64_t src[64], dst[64], src_s[64], dst_s[64];
  __shared__ int moves;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), b = blockIdx.y;
  char *pool[PER], *scales[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int pair = blockIdx.x * kKeepPairs + wave * PER + k, at = min(pair, p.pairs - 1);
    const int n = at / p.H, h = at - n * p.H;
    pool[k] = pair < p.pairs ? p.kv + n * p.s_n + h * p.s_h : nullptr;
    scales[k] = p.scales ? p.scales + n * p.ss_n + h * p.ss_h : nullptr;
  }
  for (int i0 = 0; i0 < p.n; i0 += 64) {
    if (i0 > 0) __syncthreads();  // the last list is used up
    if (wave == 0) {
      const int i = i0 + lane;
      const int64_t base = p.rows.offsets[b * p.rows.os_b];
      const int64_t nodes = p.rows.counts ? p.rows.counts[b * p.rows.ns_b] : INT64_MAX;
      const int64_t node = i < p.n ? p.path[b * p.ps_b + i * p.ps_i] : -1;
      const bool moves_on = node > i && node < nodes;  // (node i is in its place)
      const Place from = moves_on ? place_of(p.rows, b, slot_after(base, node)) : Place{-1, 0};
      const Place to = moves_on ? place_of(p.rows, b, slot_after(base, i)) : Place{-1, 0};
      const bool move = from.id >= 0 && to.id >= 0;
      const uint64_t all = __ballot(move);
      if (move) {
        const int k = __builtin_amdgcn_mbcnt_hi((uint32_t)(all >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)all, 0));
        src[k] = from.id * p.s_p + from.at * p.s_s, dst[k] = to.id * p.s_p + to.at * p.s_s;
        src_s[k] = from.id * p.ss_p + from.at * p.ss_s, dst_s[k] = to.id * p.ss_p + to.at * p.ss_s;
      }
      if (lane == 0) moves = __builtin_popcountll(all);
    }
    __syncthreads();
    const int m = moves;
    for (int x = lane; x < m * p.nch; x += 64) {
      const int e = (uint32_t)x / (uint32_t)p.nch, c = x - e * p.nch;
      const int64_t from = src[e] + (int64_t)c * sizeof(V), to = dst[e] + (int64_t)c * sizeof(V);
      V v[PER] = {};
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (pool[k]) v[k] = *(const V*)(pool[k] + from);
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (pool[k]) *(V*)(pool[k] + to) = v[k];
    }
    if (p.scales && lane < m) {
      uint8_t v[PER] = {};
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (pool[k]) v[k] = *(const uint8_t*)(scales[k] + src_s[lane]);
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (pool[k]) *(uint8_t*)(scales[k] + dst_s[lane]) = v[k];
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

// A wave per row, 64 nodes at a time.  Within them every node starts with its own bit and a link to its parent, and
// takes, round by round, the bits of the node that it links to and that node's link: after k rounds it holds 2^k
// nodes of its line.  Parents come first, so the lowest bit is the line's first node here, and that one's
// parent, in LDS with all its words by now, brings the rest.  (A workgroup per row with a barrier per round: 8.4 us
// on the GPU for 64 trees of 250 nodes, so 5.6; one of 26 nodes 2.9 and 1.8.)
__global__ __launch_bounds__(64) void tree_masks_kernel(const MaskParams p) {
  extern __shared__ uint64_t line[];  // [T][words - 1]: the lines of the nodes before, by their words before the last
  __shared__ int16_t depth[CEA_MAX_TREE];
  const int b = blockIdx.x, lane = threadIdx.x, T = p.T, words = p.words;
  int64_t count = p.counts ? p.counts[b * p.ns_b] : T;
  count = count < 0 ? 0 : count < T ? count : T;
  for (int w = 0; w < words; ++w) {
    const int i = w * 64 + lane;
    const bool real = i < count;
    int64_t up64 = real ? p.parents[b * p.ps_b + i * p.ps_t] : -1;
    const int up = up64 >= 0 && up64 < i ? (int)up64 : -1;
    uint64_t own = real ? (uint64_t)1 << lane : 0;
    int link = up >= w * 64 ? up - w * 64 : -1;
    while (__ballot(link >= 0) != 0) {
      const int from = link >= 0 ? link : lane;
      const uint32_t lo = __shfl((int)(uint32_t)own, from, 64), hi = __shfl((int)(uint32_t)(own >> 32), from, 64);
      const int next = __shfl(link, from, 64);
      own |= ((uint64_t)hi << 32) | lo;
      link = link >= 0 ? next : -1;
    }
    const int first = own != 0 ? (int)__builtin_ctzll(own) : lane;
    const int before = __shfl(up, first, 64);  // the line's last node before these, or none
    int d = __builtin_popcountll(own) - 1;
    if (before >= 0 && real) d += depth[before] + 1;
    if (i < T) {
      int64_t* out = p.masks + b * p.ms_b + i * p.ms_t;
      for (int k = 0; k < words; ++k) {
        uint64_t x = k == w ? own : 0;
        if (k < w && before >= 0 && real) x = line[before * (words - 1) + k];
        out[k * p.ms_w] = (int64_t)x;
        if (k < words - 1) line[i * (words - 1) + k] = x;
      }
      depth[i] = (int16_t)d;
      p.depths[b * p.ds_b + i * p.ds_t] = real ? d : 0;
    }
    __syncthreads();  // (one wave: what it wrote is there)
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
  p.H = (int)H, p.n = (int)path->size[1];
  const int64_t bits = (int64_t)(uintptr_t)p.kv | (N > 1 ? p.s_n : 0) | p.s_p | p.s_h | p.s_s;
  const int vec = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
  p.nch = (int)(p.s_s / vec);
  // (a turn's 64 entries times their vectors are counted in 32 bits, rows by the grid's second dimension)
  CEA_REQUIRE(N * H <= INT32_MAX - kKeepPairs && p.s_s / vec < ((int64_t)1 << 24) && B < 65536, CEA_EUNSUPPORTED,
              "paged_kv_keep: too many rows for one call");
  p.pairs = (int)(N * H);
  const dim3 grid((unsigned)((p.pairs + kKeepPairs - 1) / kKeepPairs), (unsigned)B);
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
  // (up to 28 KB: within what a launch has without asking)
  const int lds = p.T * (p.words - 1) * 8;
  hipLaunchKernelGGL(tree_masks_kernel, dim3((unsigned)B), dim3(64), lds, st, p);
  CEA_CHECK_LAUNCH("tree_masks");
  return CEA_OK;
}

}  // namespace cea

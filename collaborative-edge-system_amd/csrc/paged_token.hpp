// The line of key blocks that the paged token kernels cut into runs, and what ends a unit: the join of its waves
// and, where runs cut it, of its parts.
#pragma once

#include <math.h>

#include <algorithm>

#include "cea_lds_dma.hpp"
#include "cea_mfma16.hpp"
#include "paged.hpp"

namespace cea {

struct TokenParams {
  PagedParams p;
  int32_t G, units;       // query heads of a unit, units of a row
  int32_t page16;         // page / 16
  uint32_t magic;         // ceil(2^32 / page16), for page16 > 1
  int32_t wgs;            // workgroups at most
  float* partial;         // 2 x wgs parts of [rows][D + 2]: o, m, l
  uint8_t kv[kPagedMapHeads];  // explicit head map (p.group == 0)
};

struct TokenPlan {
  int32_t G, units, wgs;
  bool whole;
};

// Over pages of 8 bits, with everything planned.
int launch_paged_token8(const TokenParams& t, bool whole, hipStream_t s);

namespace {

constexpr int ROWS = 16;              // query rows of a unit at most
constexpr float kRescaleLog2 = 8.0f;  // the reference maximum moves when a row's grows by 2^8
constexpr int NW_SPLIT = 4;           // waves of a workgroup that takes a run
constexpr int TK8 = 32;               // keys of a tile of 8-bit pages

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef const int64_t __attribute__((address_space(4))) * scalar_i64;  // read through the scalar cache

// The kernel's arguments behind a pointer that the compiler knows nothing about.
typedef const void __attribute__((address_space(4))) * kernel_args_ptr;
__device__ __forceinline__ kernel_args_ptr opaque(kernel_args_ptr p) {
  asm volatile("" : "+s"(p));
  return p;
}

__device__ __forceinline__ int scan64(int v) {  // inclusive prefix sum over the lanes
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int x = __shfl_up(v, off, 64);
    if (lane >= off) v += x;
  }
  return v;
}

// Slots of row b, a row that the whole wave works on (a scalar read).
__device__ __forceinline__ int slots_of(const PagedParams& p, int b) {
  const int64_t n = ((scalar_i64)(uintptr_t)p.lengths)[b * p.ns_b], cap = (int64_t)p.W * p.page;
  return (int)(n < 0 ? 0 : n < cap ? n : cap);
}

// Key blocks of row b, at least one (which writes the result of a row without keys).
template <int BLK> __device__ __forceinline__ int blocks_of(const PagedParams& p, int b) {
  const int n = (int)paged_slots(p, b);
  return n > 0 ? (n + BLK - 1) / BLK : 1;
}

// The line of blocks: the rows one after the other, each `units` stretches of its blocks.  Every
// workgroup measures it from the lengths for itself, one wave-wide scan per 64 rows.
struct Line {
  int total;  // blocks of the line
  int sums;   // this lane's prefix sum over the first 64 rows' blocks
};
struct LineRow {
  int b, first, blocks;  // a row, the place of its first block, the blocks of each stretch
};

template <int BLK> __device__ __forceinline__ int prefix64(const PagedParams& p, int b0) {
  const int b = b0 + (threadIdx.x & 63);
  return scan64(b < p.B ? blocks_of<BLK>(p, b) : 0);
}

template <int BLK> __device__ __forceinline__ Line line_of(const TokenParams& t) {
  Line line;
  line.sums = prefix64<BLK>(t.p, 0);
  line.total = __builtin_amdgcn_readlane(line.sums, 63);
  for (int b0 = 64; b0 < t.p.B; b0 += 64)
    line.total += __builtin_amdgcn_readlane(prefix64<BLK>(t.p, b0), 63);
  line.total *= t.units;
  return line;
}

// The row that holds block `at` (0 <= at < total), or with at < 0 row `b`.
template <int BLK>
__device__ __forceinline__ LineRow row_of(const TokenParams& t, const Line& line, int at, int b) {
  LineRow r = {0, 0, 1};
  int before = 0;
  for (int b0 = 0; b0 < t.p.B; b0 += 64) {
    const int sums = b0 == 0 ? line.sums : prefix64<BLK>(t.p, b0);
    const uint64_t found =
        at >= 0 ? __ballot((before + sums) * t.units > at) : (b - b0 < 64 ? 1ull << (b - b0) : 0ull);
    if (found != 0) {
      const int l = (int)__builtin_ctzll(found);
      const int begin = l > 0 ? __builtin_amdgcn_readlane(sums, l - 1) : 0;
      r.b = b0 + l;
      r.first = (before + begin) * t.units;
      r.blocks = __builtin_amdgcn_readlane(sums, l) - begin;
      break;
    }
    before += __builtin_amdgcn_readlane(sums, 63);
  }
  return r;
}

// The line cut into runs: the first `more` workgroups take `run + 1` blocks, the others `run`.
struct Runs {
  int run, more;
  __device__ __forceinline__ int start(int wg) const { return wg * run + min(wg, more); }
  __device__ __forceinline__ int wg_of(int at) const {  // the workgroup that takes block `at`
    const int big = more * (run + 1);
    return at < big ? at / (run + 1) : more + (at - big) / run;
  }
};
__device__ __forceinline__ Runs runs_of(const TokenParams& t, int total) {
  const int wgs = max(1, min(t.wgs, total));
  Runs r;
  r.run = total / wgs;
  r.more = total - r.run * wgs;
  return r;
}

// The unit of a run behind the one that `taken` blocks of it were of: false where the run ends.  The run was measured on
// an earlier read of the lengths than blocks_in's, so it ends at the last row too, whatever they hold by now.
template <typename BlocksIn>
__host__ __device__ __forceinline__ bool next_unit(int& b, int& unit, int& lo, int& left, int& blocks, int taken,
                                                   int units, int rows, BlocksIn blocks_in) {
  left -= taken;
  if (left <= 0) return false;
  lo = 0;
  if (++unit == units) {
    unit = 0;
    if (++b >= rows) return false;
    blocks = blocks_in(b);
  }
  return true;
}

template <typename O> __device__ __forceinline__ void write_out(const PagedParams& p, int b, int s, int h, int d,
                                                                float x) {
  ((O*)p.out)[b * p.os_b + s * p.os_s + h * p.os_h + d] = (O)x;
}
template <typename T> __device__ __forceinline__ void write_row(const PagedParams& p, int b, int s, int h, int d,
                                                                float x) {
  if (p.out_dtype == CEA_F32) write_out<float>(p, b, s, h, d, x);
  else write_out<T>(p, b, s, h, d, x);
}

// Joins the waves' sums of a unit in LDS and writes its rows, or (the unit is cut: not from its first block to its
// last) its part.  `wave_bytes`: a wave's own share of `dsmem`, whose tiles are no longer read.  The sums o hold
// 1 / unscale of the products' weights (undone before they are divided), and 2^kHeldLog2 of them beside that, which the
// division undoes: a part of such sums has 2^kHeldLog2 of its weights' sum and a maximum that is as much higher.
template <typename T, int D, int NW, bool WHOLE, int kHeldLog2>
__device__ __forceinline__ void finish_unit(const TokenParams& t, const f32x4 (&o)[D / 16], float m_run, float l_run,
                                            float2 (&red_ml)[ROWS][NW], char* dsmem, int wave_bytes, int b, int unit,
                                            bool first, bool last, float unscale) {
  const PagedParams& p = t.p;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, row = lane & 15, grp = lane >> 4;
  const int nrows = p.Sq * t.G;
  const float scale = (float)p.scale;
  const float c = fabsf(scale) * 1.4426950408889634f;  // exp2 units
  const float held = __builtin_amdgcn_ldexpf(1.f, kHeldLog2);
  // A row's sum is 0 exactly where it saw no key (a NaN is kept).
  const float l_row = sum_halves(sum_rows16(l_run));
  if (grp == 0) red_ml[row][wave] = make_float2(m_run, l_row);
  float* red_o = (float*)(dsmem + wave * wave_bytes);
  if (row < nrows) {
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) *(f32x4*)(red_o + row * D + dt * 16 + grp * 4) = o[dt];
  }
  __syncthreads();
  float* part = t.partial + ((int64_t)blockIdx.x * 2 + (first ? 1 : 0)) * nrows * (D + 2);
  for (int i = tid; i < nrows * D; i += NW * 64) {
    const int r = i / D, d = i % D;
    float2 ml[NW];
    float x[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      ml[w] = red_ml[r][w];
      x[w] = ((const float*)(dsmem + w * wave_bytes))[i];
    }
    float M = -__builtin_inff();  // of the raw scores
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w].x);
    const float shift = M == -__builtin_inff() ? 0.f : M;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      // (a wave that saw nothing has zeros; one whose scores are all NaN keeps its NaN)
      const float wt = ml[w].x == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f((ml[w].x - shift) * c);
      acc = __builtin_fmaf(x[w], wt, acc);
      sum = __builtin_fmaf(ml[w].y, wt, sum);
    }
    acc *= unscale;
    M *= fabsf(scale);
    if (WHOLE || (first && last)) {
      const int s = r / t.G, h = unit * t.G + r - s * t.G;
      write_row<T>(p, b, s, h, d, sum == 0.f ? 0.f : acc / (sum * held));
      if (p.lse && d == 0)
        ((float*)p.lse)[b * p.ls_b + h * p.ls_h + s * p.ls_s] =
            sum == 0.f ? -__builtin_inff() : (M == -__builtin_inff() ? 0.f : M) + logf(sum);
    } else {
      // non-temporal: written back past the caches, they disturb the reads of other workgroups least
      __builtin_nontemporal_store(acc, part + r * (D + 2) + d);
      if (d == 0) {
        __builtin_nontemporal_store(M - kHeldLog2 * 0.69314718055994531f, part + r * (D + 2) + D);
        __builtin_nontemporal_store(sum * held, part + r * (D + 2) + D + 1);
      }
    }
  }
}

// What the tree's mask lets a query row see of the `NK` keys from slot0 on, up to 16 nodes.
struct TreeRow {
  int base;        // slot of the first node
  uint32_t nodes;  // the row's bits
};
template <int NK> __device__ __forceinline__ uint32_t tree_window(const TreeRow& r, int slot0) {
  const int off = slot0 - r.base;
  const uint32_t x = off <= -NK ? ~0u : off < 0 ? (r.nodes << -off) | ((1u << -off) - 1) : off < 32 ? r.nodes >> off : 0;
  return x & ((1u << NK) - 1);
}
// A row's limits for slots by number or tree: it sees all of [0, lim), and nothing from `any` on.
struct Limits {
  int lim, any;
};
template <bool TREE>
__device__ __forceinline__ Limits limits_of(const PagedParams& p, int b, int n, int64_t qpos, int s, TreeRow& tree) {
  if constexpr (TREE) {
    const TreeOf x = tree_of(p, b);
    tree.base = (int)max(x.base, -((int64_t)1 << 30));
    tree.nodes = (uint32_t)tree_word(p, b, s, 0);
    const bool sees = s < (int)x.nodes;
    if (!sees) tree.nodes = 0;
    return {sees ? max(tree.base, 0) : 0, sees ? n : 0};
  } else {
    const int lim = !p.causal || qpos >= n ? n : (int)max((int64_t)0, qpos + 1);
    return {lim, lim};
  }
}

// Joins the parts of the units that the runs cut, one workgroup per (row, token, query head): every
// wave weighs 64 parts at a time, a part a lane, and sums every fourth part's features, whose reads
// are under way by then (one trip to memory for the lengths and one for up to 64 parts).
template <typename T, int D, int BLK>
__global__ __launch_bounds__(256) void paged_token_join_kernel(const TokenParams t) {
  constexpr int FPL = D / 64;  // features per lane
  constexpr int PER = 16;      // parts of a wave among 64
  __shared__ float o_s[4][D];
  const PagedParams& p = t.p;
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int h = blockIdx.x % p.Hq, s = (blockIdx.x / p.Hq) % p.Sq, b = blockIdx.x / (p.Hq * p.Sq);
  const Line line = line_of<BLK>(t);
  const LineRow r = row_of<BLK>(t, line, -1, b);
  const Runs runs = runs_of(t, line.total);
  const int unit = h / t.G, start = r.first + unit * r.blocks;
  const int w0 = runs.wg_of(start), n = runs.wg_of(start + r.blocks - 1) - w0 + 1;
  if (n == 1) return;  // finished by its workgroup
  const int nrows = p.Sq * t.G;
  // the first part is its workgroup's last unit (slot 1), the others' their first (slot 0)
  const int64_t stride = 2 * (int64_t)nrows * (D + 2);
  const float* base = t.partial + w0 * stride + (int64_t)(s * t.G + h - unit * t.G) * (D + 2);
  auto part = [&](int j) { return base + j * stride + (j == 0 ? stride / 2 : 0); };
  float m = -__builtin_inff(), l = 0.f, o[FPL] = {};
  for (int j0 = 0; j0 < n; j0 += 64) {
    float x[PER][FPL];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int j = j0 + wave + 4 * k;
      const float* q = part(j < n ? j : 0) + lane * FPL;
#pragma unroll
      for (int i = 0; i < FPL; ++i) x[k][i] = q[i];
    }
    const float* q = part(j0 + lane < n ? j0 + lane : 0);
    const float pm = j0 + lane < n ? q[D] : -__builtin_inff(), pl = j0 + lane < n ? q[D + 1] : 0.f;
    float m_new = m;
    {
      float v = pm;
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
      m_new = fmaxf(m, max_halves(max_rows16(v)));
    }
    const float shift = m_new == -__builtin_inff() ? 0.f : m_new;
    const float a = m == -__builtin_inff() ? 1.f : expf(m - shift);
    // (parts that saw a key: one whose weight underflows to 0 still counts, as its infinities make a NaN there)
    const uint64_t saw = __ballot(pl != 0.f);
    const float wt = pl == 0.f ? 0.f : pm == -__builtin_inff() ? 1.f : expf(pm - shift);
    float sum = pl * wt;
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) sum += __shfl_xor(sum, off, 64);
    m = m_new;
    l = l * a + sum_halves(sum_rows16(sum));
#pragma unroll
    for (int i = 0; i < FPL; ++i) o[i] *= a;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const float w = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(wt), wave + 4 * k));
#pragma unroll
      for (int i = 0; i < FPL; ++i)
        if ((saw >> (wave + 4 * k)) & 1) o[i] = __builtin_fmaf(x[k][i], w, o[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < FPL; ++i) o_s[wave][lane * FPL + i] = o[i];
  __syncthreads();
  if (tid >= D) return;
  const float acc = (o_s[0][tid] + o_s[1][tid]) + (o_s[2][tid] + o_s[3][tid]);
  write_row<T>(p, b, s, h, tid, l == 0.f ? 0.f : acc / l);
  if (p.lse && tid == 0)
    ((float*)p.lse)[b * p.ls_b + h * p.ls_h + s * p.ls_s] =
        l == 0.f ? -__builtin_inff() : (m == -__builtin_inff() ? 0.f : m) + logf(l);
}

}  // namespace
}  // namespace cea

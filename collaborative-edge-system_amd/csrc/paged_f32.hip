// f32 attention over a paged KV cache on the matrix cores (v_mfma_f32_16x16x4_f32: IEEE f32 products and
// sums), head size 64 or 128, any number of new tokens.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * q.k_j,  lse = m + log sum_j p_j
//
// The tiles are the f32 prefill kernel's: 16 keys by 16 query rows, operands straight from memory in
// registers.  S^T = K.Q^T with the keys placed on the accumulator rows as 4*(r%4) + r/4, so the scores are
// the B operand of O^T += V^T.P^T as they are, and V^T's rows are placed so that a lane ends with runs of
// D/16 features.  What is different:
//   * a tile lies in one page (pages are multiples of 16 slots); its index is a scalar read two tiles
//     ahead, and reads past the row's end return 0;
//   * the 16 query rows are tokens of one head, or for fewer tokens those of several heads of one KV
//     head, whose keys are then read once;
//   * 8 waves take every 8th tile each and are joined in LDS; long tables with few query rows are cut
//     into up to 16 key splits by the table's width (each takes an equal run of the row's own tiles),
//     merged by the list merge.
//   * Bound by latency: a prompt of 512 keys is 4 tiles a wave, 14.2 us for 8 heads of 64.
//   * A tree's nodes see the slots before it as any rows do; in the last tiles a row's bits of the mask are read where
//     they are needed, a few words of L2.
//   * A value that is not finite and hidden from some query would reach it as 0 * inf.  The results show
//     that (they are not finite either), and the workgroup then goes over its tiles again and sums products
//     one by one, over each query's visible keys.
#include <math.h>
#include <string.h>

#include <algorithm>

#include "cea_lds_dma.hpp"
#include "paged.hpp"

namespace cea {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef const int64_t __attribute__((address_space(4))) * scalar_i64;  // read through the scalar cache

constexpr int QB = 16;   // query rows per workgroup
constexpr int KT = 16;   // keys per tile
constexpr int NW = 8;    // waves per workgroup

struct F32Params {
  PagedParams p;
  int32_t G;                     // query heads of a workgroup's rows
  int32_t nqb, splits;
  int64_t split_out, split_lse;  // elements between the splits' partial results
  int32_t page16;
  uint32_t magic;                // ceil(2^32 / page16), for page16 > 1
  uint8_t kv[kPagedMapHeads];
};

__device__ __forceinline__ f32x4 mfma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// 16 bytes at a buffer's base + offset, 0 past its end
__device__ __forceinline__ f32x4 load4(__amdgpu_buffer_rsrc_t rs, uint32_t off) {
  return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, 0, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc(const char* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, bytes, kRsrcFlags);
}

template <int D> struct Tile {
  f32x4 k[D / 16];      // lane (r, g): features 16j + 4g .. of key 4*(r%4) + r/4
  f32x4 v[4][D / 64];   // lane (c, g), k-block i: features c*D/16 .. of key 4i + g
  int64_t pos[4];       // positions of keys 4i + g
};

__device__ __forceinline__ float xor_max(float x) {
  uint32_t u = __float_as_uint(x);
  auto sw = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])));
  sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}
__device__ __forceinline__ float xor_sum(float x) {
  uint32_t u = __float_as_uint(x);
  auto sw = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  u = __float_as_uint(__uint_as_float(sw[0]) + __uint_as_float(sw[1]));
  sw = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

template <int D, int VIS>
__global__ __launch_bounds__(NW * 64) void paged_f32_kernel(const F32Params t) {
  constexpr bool POS = VIS == kPosition, TREE = VIS == kTree;
  constexpr int NB = D / 16;    // output feature blocks, and consecutive features of a lane
  const PagedParams& p = t.p;
  extern __shared__ __attribute__((aligned(16))) float red_o[];  // [NW][QB][D + 4]
  __shared__ float red_m[NW][QB], red_l[NW][QB];
  __shared__ int odd;

  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int c16 = lane & 15, g = lane >> 4;
  const int units = p.Hq / t.G;
  int id = blockIdx.x;
  const int split = id / (t.nqb * units * p.B);
  id -= split * (t.nqb * units * p.B);
  const int qb = t.nqb - 1 - id % t.nqb;  // the latest rows, which see the most, first
  id /= t.nqb;
  const int unit = id % units, b = id / units;
  const int h0 = unit * t.G;
  const int kvh = p.group > 0 ? h0 / p.group : t.kv[h0];
  const int row = qb * QB + c16;
  const bool row_ok = row < p.Sq * t.G;
  const int s = row_ok ? row / t.G : 0, h = h0 + (row_ok ? row - s * t.G : 0);
  const int64_t qpos = TREE ? 0 : p.q_pos[b * p.qps_b + (int64_t)s * p.qps_s];
  const int n = uniform((int)paged_slots(p, b));
  const TreeOf nodes = TREE ? tree_of(p, b) : TreeOf{0, 0};
  const int base = (int)max(nodes.base, -((int64_t)1 << 30));
  // this lane's row sees slots [0, lim) (POS: of those, the positions up to qpos; TREE: those before base, and
  // its nodes)
  const bool sees = row_ok && (TREE ? s < nodes.nodes : !p.causal || qpos >= 0);
  const int lim = !sees ? 0 : !TREE && p.causal && !POS && qpos < n ? (int)qpos + 1 : n;
  int lim_max = lim;
#pragma unroll
  for (int off = 8; off >= 1; off >>= 1) lim_max = max(lim_max, __shfl_xor(lim_max, off, 64));
  lim_max = uniform(lim_max);
  const int ntiles = (lim_max + KT - 1) / KT;
  const int per = (ntiles + t.splits - 1) / t.splits;
  const int t0 = min(ntiles, split * per), t1 = min(ntiles, t0 + per);
  const float scale = (float)p.scale;
  if (tid == 0) odd = 0;

  f32x4 qf[D / 16];
  {
    const float* qrow = (const float*)p.q + b * p.qs_b + s * p.qs_s + h * p.qs_h;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) qf[j] = sees ? *(const f32x4*)(qrow + 16 * j + 4 * g) : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const char* kh = (const char*)((const float*)p.k + (int64_t)kvh * p.ks_h);
  const char* vh = (const char*)((const float*)p.v + (int64_t)kvh * p.vs_h);
  const uint32_t krow = (uint32_t)(p.ks_s * 4), vrow = (uint32_t)(p.vs_s * 4);
  const uint32_t k_off = (4 * (c16 & 3) + (c16 >> 2)) * krow + g * 16;
  const scalar_i64 table = (scalar_i64)(uintptr_t)(p.tables + b * p.ts_b);
  auto page_of = [&](int tile) -> int { return (int)(t.page16 == 1 ? (uint32_t)tile : __umulhi((uint32_t)tile, t.magic)); };
  auto id_of = [&](int tile) -> int64_t { return tile < t1 ? table[(int64_t)page_of(tile) * p.ts_w] : -1; };
  auto load_tile = [&](Tile<D>& x, int tile, int64_t pg) {
    const bool ok = (uint64_t)pg < (uint64_t)p.P;
    const int64_t at = ok ? pg : 0;
    const int place = (tile - page_of(tile) * t.page16) * KT;
    const int rows = min(n - tile * KT, KT);  // (of no page: none)
    const auto krs = rsrc(kh + (at * p.ks_p + place * p.ks_s) * 4, ok ? (rows - 1) * krow + D * 4 : 0u);
    const auto vrs = rsrc(vh + (at * p.vs_p + place * p.vs_s) * 4, ok ? (rows - 1) * vrow + D * 4 : 0u);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) x.k[j] = load4(krs, k_off + j * 64);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = 4 * i + g;
#pragma unroll
      for (int u = 0; u < D / 64; ++u) x.v[i][u] = load4(vrs, key * vrow + c16 * (NB * 4) + u * 16);
      x.pos[i] = -1;
      if (ok && key < rows) x.pos[i] = POS ? p.pos[at * p.ps_p + place + key] : tile * KT + key;
    }
  };

  f32x4 o[NB];
  float m_run, l_run;
  auto stream = [&](auto careful) {
#pragma unroll
    for (int m = 0; m < NB; ++m) o[m] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run = -__builtin_inff(), l_run = 0.f;
    Tile<D> cur, nxt;
    int tile = t0 + wave;
    int64_t id0 = id_of(tile), id1 = id_of(tile + NW);
    if (tile < t1) load_tile(cur, tile, id0);
    for (; tile < t1; tile += NW) {
      const bool more = tile + NW < t1;
      const int64_t id2 = id_of(tile + 2 * NW);
      if (more) load_tile(nxt, tile + NW, id1);
      id1 = id2;
      bool vis[4], any = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // (a position of -1, of a hole or of no page, is past every limit)
        vis[i] = sees && tile * KT + 4 * i + g < lim && cur.pos[i] >= 0 && (!POS || !p.causal || cur.pos[i] <= qpos);
        if constexpr (TREE) {
          const int node = tile * KT + 4 * i + g - base;
          if (vis[i] && node >= 0) vis[i] = node < p.Sq && ((tree_word(p, b, s, node >> 6) >> (node & 63)) & 1);
        }
        any = any || vis[i];
      }
      if (__ballot(any) != 0) {
        f32x4 sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc = mfma4(cur.k[j][e], qf[j][e], sc);
        float mx = -__builtin_inff();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[i] = vis[i] ? sc[i] * scale : -__builtin_inff();
          mx = fmaxf(mx, sc[i]);
        }
        const float m_new = fmaxf(m_run, xor_max(mx));
        const float m_use = m_new == -__builtin_inff() ? 0.f : m_new;
        const float alpha = expf(m_run - m_use);  // 0 while the row has seen nothing
        float pr[4], ls = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pr[i] = vis[i] ? expf(sc[i] - m_use) : 0.f;
          ls += pr[i];
        }
        l_run = l_run * alpha + xor_sum(ls);
        m_run = m_new;
#pragma unroll
        for (int m = 0; m < NB; ++m) o[m] *= alpha;
        if constexpr (!decltype(careful)::value) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int m = 0; m < NB; ++m) o[m] = mfma4(cur.v[i][m / 4][m % 4], pr[i], o[m]);
        } else {
          // key 4i + x: its probability for this lane's query from the lane group x, its features (4g +
          // r) * NB + m from lane 4g + r of that group
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll 1
            for (int x = 0; x < 4; ++x) {
              const float w = __shfl(pr[i], c16 + 16 * x, 64);
              const bool seen = __shfl(vis[i] ? 1 : 0, c16 + 16 * x, 64) != 0;
#pragma unroll
              for (int m = 0; m < NB; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                  const float v = __shfl(cur.v[i][m / 4][m % 4], 4 * g + r + 16 * x, 64);
                  if (seen) o[m][r] = __builtin_fmaf(w, v, o[m][r]);
                }
            }
        }
      }
      if (more) cur = nxt;
    }
  };
  stream(std::false_type());
  __syncthreads();  // odd
  {
    bool bad = false;
#pragma unroll
    for (int m = 0; m < NB; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) bad = bad || !__builtin_isfinite(o[m][r]);
    if (__ballot(sees && bad) != 0 && lane == 0) odd = 1;
    __syncthreads();
    if (odd) stream(std::true_type());
  }

  // ---- join the waves.  A row's sum is 0 exactly where it saw no key (a NaN is kept).
  if (g == 0) red_m[wave][c16] = m_run, red_l[wave][c16] = l_run;
  float* mine = red_o + wave * (QB * (D + 4));
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int m = 0; m < NB; m += 4)
      *(f32x4*)(mine + c16 * (D + 4) + (4 * g + r) * NB + m) = f32x4{o[m][r], o[m + 1][r], o[m + 2][r], o[m + 3][r]};
  __syncthreads();
  for (int i = tid; i < QB * (D / 4); i += NW * 64) {
    const int qq = i / (D / 4), f = i % (D / 4) * 4, orow = qb * QB + qq;
    if (orow >= p.Sq * t.G) break;
    float M = -__builtin_inff();
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, red_m[w][qq]);
    const float shift = M == -__builtin_inff() ? 0.f : M;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = red_m[w][qq], wt = m == -__builtin_inff() ? 1.f : expf(m - shift);
      acc += *(const f32x4*)(red_o + (w * QB + qq) * (D + 4) + f) * wt;
      sum += red_l[w][qq] * wt;
    }
    const bool empty = sum == 0.f;
    const float inv = 1.f / sum;
    const int os = orow / t.G, oh = h0 + orow - os * t.G;
    const f32x4 res = empty ? f32x4{0.f, 0.f, 0.f, 0.f} : acc * inv;
    *(f32x4*)((float*)p.out + split * t.split_out + b * p.os_b + os * p.os_s + oh * p.os_h + f) = res;
    if (p.lse && f == 0)
      ((float*)p.lse)[split * t.split_lse + b * p.ls_b + oh * p.ls_h + os * p.ls_s] =
          empty ? -__builtin_inff() : shift + logf(sum);
  }
}

template <int D, int VIS> int launch_form(const F32Params& t, hipStream_t st) {
  constexpr int lds = NW * QB * (D + 4) * (int)sizeof(float);
  const hipError_t e = reserve_lds<paged_f32_kernel<D, VIS>>(lds);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "paged_attention: cannot reserve %d bytes of LDS: %s", lds,
              hipGetErrorString(e));
  const int64_t grid = (int64_t)t.nqb * (t.p.Hq / t.G) * t.p.B * t.splits;
  hipLaunchKernelGGL((paged_f32_kernel<D, VIS>), dim3((unsigned)grid), dim3(NW * 64), lds, st, t);
  CEA_CHECK_LAUNCH("paged_f32");
  return CEA_OK;
}

size_t align256(size_t x) { return (x + 255) / 256 * 256; }

struct F32Plan {
  int G, nqb, splits;
  size_t part_out, part_lse;
};

F32Plan plan_f32(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots) {
  F32Plan r;
  r.G = 1;
  for (int64_t g = group; g > 1; --g)
    if (group % g == 0 && g * Sq <= QB) {
      r.G = (int)g;
      break;
    }
  r.nqb = (int)((Sq * r.G + QB - 1) / QB);
  // a workgroup per compute unit, at least 2 tiles a wave (us: 24 workgroups of up to 94 tiles 27.6 whole, 16.6
  // in 5 splits; 256 of up to 32 tiles 14.8 whole, 22.6 in 2)
  const int64_t grid = r.nqb * (Hq / r.G) * B, tiles = (slots + KT - 1) / KT;
  r.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)CEA_MAX_PARTS, 256 / std::max<int64_t>(grid, 1),
                                                          tiles / (2 * NW)}));
  r.part_out = align256((size_t)B * Sq * Hq * D * sizeof(float));
  r.part_lse = align256((size_t)B * Sq * Hq * sizeof(float));
  return r;
}

}  // namespace

size_t paged_f32_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int group, int64_t D, int64_t slots) {
  const F32Plan r = plan_f32(B, Sq, Hq, group, D, slots);
  return r.splits > 1 ? r.splits * (r.part_out + r.part_lse) : 0;
}

bool paged_f32_supported(const PagedParams& p, const HeadMap& map) {
  if (p.kv_dtype != CEA_F32 || !(p.D == 64 || p.D == 128) || p.page % KT != 0 || p.W == 0) return false;
  if (map.group <= 0 && (p.Hq > kPagedMapHeads || p.Hkv > 256)) return false;
  if (!std::isfinite(p.scale)) return false;
  // (32-bit slots; u / m = u * ceil(2^32 / m) >> 32 while u * m < 2^32)
  const int64_t slots = (int64_t)p.W * p.page;
  if (slots >= (int64_t)1 << 30 || slots / 16 * (p.page / 16) >= (int64_t)1 << 32) return false;
  for (int64_t s : {p.qs_b, p.qs_s, p.qs_h, p.ks_p, p.ks_h, p.ks_s, p.vs_p, p.vs_h, p.vs_s, p.os_b, p.os_s, p.os_h})
    if (s % 4) return false;
  for (const void* d : {p.q, p.k, p.v, (const void*)p.out})
    if ((uintptr_t)d % 16) return false;
  for (int64_t s : {p.ks_s, p.vs_s})
    if (s < p.D || s >= (int64_t)1 << 24) return false;  // a tile spans less than 2^31 bytes
  return (p.pos == nullptr || p.ps_s == 1) &&
         (int64_t)p.B * p.Hq * ((p.Sq + QB - 1) / QB) * CEA_MAX_PARTS < ((int64_t)1 << 31);
}

int launch_paged_f32(const PagedParams& o, const HeadMap& map, void* ws, hipStream_t st) {
  const F32Plan r = plan_f32(o.B, o.Sq, o.Hq, map.group, o.D, (int64_t)o.W * o.page);
  F32Params t;
  memset(&t, 0, sizeof(t));
  t.p = o;
  t.G = r.G, t.nqb = r.nqb, t.splits = r.splits;
  t.page16 = o.page / 16;
  t.magic = t.page16 > 1 ? (uint32_t)((((uint64_t)1 << 32) + t.page16 - 1) / t.page16) : 0;
  for (int h = 0; h < kPagedMapHeads && h < o.Hq && map.group <= 0; ++h) t.kv[h] = (uint8_t)map.kv[h];
  if (r.splits > 1) {
    char* at = (char*)ws;
    t.p.out = at, t.p.lse = at + r.splits * r.part_out;
    t.p.os_h = o.D, t.p.os_s = (int64_t)o.Hq * o.D, t.p.os_b = t.p.os_s * o.Sq;
    t.p.ls_s = 1, t.p.ls_h = o.Sq, t.p.ls_b = (int64_t)o.Hq * o.Sq;
    t.split_out = (int64_t)(r.part_out / sizeof(float)), t.split_lse = (int64_t)(r.part_lse / sizeof(float));
  }
  int rc;
  if (o.D == 64)
    rc = o.masks ? launch_form<64, kTree>(t, st) : o.pos ? launch_form<64, kPosition>(t, st) : launch_form<64, kNumber>(t, st);
  else
    rc = o.masks ? launch_form<128, kTree>(t, st) : o.pos ? launch_form<128, kPosition>(t, st) : launch_form<128, kNumber>(t, st);
  if (rc || r.splits == 1) return rc;
  return merge_paged_splits(o, t.p, r.splits, t.split_out, t.split_lse, st);
}

}  // namespace cea

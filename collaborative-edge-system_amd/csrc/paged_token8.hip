// Attention of a few new tokens per row over a paged KV cache of 8 bits (bf16 / f16 queries, head size 64 or
// 128): the serving form, HBM-bound at half the bytes of the 16-bit one.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * q.k_j,  lse = m + log sum_j p_j,
//   k_j = kq_j * 2^(ks_j - 127),  v_j = vq_j * 2^(vs_j - 127)
//
// Units, runs, joins and the softmax are the 16-bit form's (paged_token.hip).  What 8 bits change:
//   * a wave's tile is 32 keys, as many bytes as 16 of the 16-bit form: two halves of 16 rows, in one page where
//     pages are multiples of 32 slots, else each with an address of its own, and their 64 scale bytes by one load of
//     four lanes;
//   * S = K.Q^T with v_mfma_f32_16x16x32: a lane reads 16 numbers of a key (the queries' features are in the same
//     order) and turns them into the queries' type with the key's scale, two an instruction, exactly;
//   * O^T += V^T.P^T with v_mfma_f32_16x16x32_bf16: ds_read_b64_tr_b8 gives a lane 8 keys of one feature, which become
//     bf16 as they are (4 significant bits); their scales are the keys', so the probabilities take them, in f32, before
//     they are cut into bf16 pieces (two leave 2^-16 of one, three for f32 results less than 2^-23).  A weight is up to
//     2^8 before the maximum follows, and a scale up to 2^127, so the sums are held at 2^-8 of theirs: no product
//     passes f32 unless the result's own sum does.  At the other end a piece below bf16's normal numbers loses up
//     to 2^-134: 2^-117 of a result's key, where its values are below 2^-92 (scale bytes below 26).  The keys of a
//     lane are those whose scores it holds, the order within a tile being free;
//   * positions and masks are the 16-bit form's;
//   * a number that is not finite can only be NaN.  In a tile that all rows see it makes the NaN that the
//     definition makes.  In others (the last ones of a unit) what no row sees is taken as 0, and a NaN that some rows
//     see sums its tile's products one by one.
//   * Measured: 32 rows of 1024 to 32768 keys, 32/8 heads of 128, bf16: 196 us for 1.12 GB, 5.7 TB/s (the 16-bit form
//     6.2 over twice the bytes), 188 of them the stream and 8 the join.  A byte carries twice the 16-bit form's work:
//     250 vector and 150 scalar instructions a tile (330 and 330, 223 us, with 64-bit addresses for each half and
//     every tile's visibility key by key).
#include <type_traits>

#include "paged_token.hpp"

namespace cea {
namespace {

typedef int i32x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2* lds_i32x2_ptr;

// What the sums hold of the products' weights, as a power of two: the reference maximum's lag.
constexpr int kHeldLog2 = -8;
static_assert(kHeldLog2 == -(int)kRescaleLog2, "the largest weight times the largest scale");

template <int D> struct T8Layout {
  static constexpr int ROW = D;                // bytes
  static constexpr int HALF = 16 * ROW;        // 16 keys, in one page
  static constexpr int TILE_BYTES = TK8 * ROW;
  static constexpr int SCALES = 2 * TILE_BYTES;  // K of both halves, V of both halves
  static constexpr int POS = SCALES + 2 * TK8;
  static constexpr int BUF_BYTES = POS + TK8 * 8;
  static constexpr int WAVE_BYTES = 2 * BUF_BYTES;
  static constexpr int LOADS = HALF / 1024;    // of a half
  static_assert(WAVE_BYTES >= ROWS * D * 4, "a wave's sums take the place of its tiles");
};

// 16-byte groups of a row are placed by an exclusive or with a number of the row: rows that are read together
// (16 keys of one group for K; for V 8 keys, 4 of each half) then lie in different banks.
template <int D> __device__ __forceinline__ int k8_swz(int key) {
  if constexpr (D == 128) return (key & 7) ^ ((key >> 3) & 1);
  else return ((key >> 1) & 3) ^ ((key >> 3) & 1);
}
template <int D> __device__ __forceinline__ int v8_swz(int key) {
  if constexpr (D == 128) return (key & 3) | (key >> 4) << 2;
  else return ((key >> 1) & 1) | (key >> 4) << 1;
}

template <typename T> __device__ __forceinline__ typename Mfma16<T>::frag8 widen8(uint32_t a, uint32_t b, float scale) {
  const u32x4 x = {widen2<T, false>(a, scale), widen2<T, true>(a, scale), widen2<T, false>(b, scale),
                   widen2<T, true>(b, scale)};
  return __builtin_bit_cast(typename Mfma16<T>::frag8, x);
}

// A wave-uniform value that stays in a scalar register (read again from the arguments, it would be waited for where
// it is used, with every LDS read before it).
template <typename X> __device__ __forceinline__ X in_sgpr(X v) {
  asm volatile("" : "+s"(v));
  return v;
}

template <typename T, int D, int VIS, int NW, bool SPLIT, int PC>
__global__ __launch_bounds__(NW * 64, D == 64 ? 4 : 2) void paged_token8_kernel(const TokenParams args) {
  constexpr bool POS = VIS == kPosition, TREE = VIS == kTree;
  typedef T8Layout<D> L;
  typedef typename Mfma16<T>::frag8 frag8;
  constexpr int BLK = NW * TK8;
  extern __shared__ __attribute__((aligned(16))) char dsmem[];
  __shared__ float2 red_ml[ROWS][NW];
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int row = lane & 15, grp = lane >> 4;
  const int nrows = args.p.Sq * args.G;
  const bool row_real = row < nrows;
  const int rs = row_real ? row / args.G : 0, rg = row_real ? row - rs * args.G : 0;
  char* wb = dsmem + wave * L::WAVE_BYTES;
  const uint32_t wave_lds = lds_addr(dsmem) + wave * L::WAVE_BYTES;

  // ---- this workgroup's run of blocks
  int b, unit, lo, left, blocks;
  if constexpr (SPLIT) {
    const Line line = line_of<BLK>(args);
    const Runs runs = runs_of(args, line.total);
    const int at = runs.start(blockIdx.x);
    if (at >= line.total) return;
    const LineRow r = row_of<BLK>(args, line, at, 0);
    b = r.b, blocks = r.blocks;
    unit = (at - r.first) / blocks;
    lo = at - r.first - unit * blocks;
    left = runs.run + (blockIdx.x < runs.more ? 1 : 0);
  } else {
    b = blockIdx.x / args.units;
    unit = blockIdx.x - b * args.units;
    const int n = slots_of(args.p, b);
    blocks = n > 0 ? (n + BLK - 1) / BLK : 1;
    lo = 0;
    left = blocks;
  }

  const int cap = args.p.W * args.p.page;
  const float scale = (float)args.p.scale;
  const float c = fabsf(scale) * 1.4426950408889634f;  // exp2 units
  const float grow_thr = kRescaleLog2 / c;
  const uint32_t flip = scale < 0.f ? 0x80008000u : 0u;
  const uint32_t krow = (uint32_t)args.p.ks_s, vrow = (uint32_t)args.p.vs_s;
  const bool one_page = args.page16 % 2 == 0;  // both halves of a tile lie in the same one
  uint32_t k_voff[2][L::LOADS], v_voff[2][L::LOADS];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < L::LOADS; ++i) {
      const int r = i * (1024 / L::ROW) + lane / (L::ROW / 16), from = one_page ? 16 * h + r : r;
      const int pg = lane % (L::ROW / 16);  // physical 16-byte group
      k_voff[h][i] = from * krow + ((pg ^ k8_swz<D>(r)) << 4);
      v_voff[h][i] = from * vrow + ((pg ^ v8_swz<D>(16 * h + r)) << 4);
    }
  uint32_t k_raddr[D / 64], v_raddr[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 64; ++ks) k_raddr[ks] = row * L::ROW + (((4 * ks + grp) ^ k8_swz<D>(row)) << 4);
  {
    // lane `row` of a group reads 8 bytes of the group's key row / 2: 4 keys of each half
    const int e = row >> 1, key = (e >> 2) * 16 + grp * 4 + (e & 3);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      v_raddr[dt] = L::TILE_BYTES + key * L::ROW + ((dt ^ v8_swz<D>(key)) << 4) + 8 * (row & 1);
  }

  while (true) {
    // ---- one unit of the run, blocks [lo, hi)  (the arguments are read again, as in the 16-bit form)
    const kernel_args_ptr ap = opaque((kernel_args_ptr)__builtin_amdgcn_kernarg_segment_ptr());
    const TokenParams& t = *(const TokenParams*)ap;
    const PagedParams& p = t.p;
    const int hi = min(blocks, lo + left);
    const int kvh = p.group > 0 ? unit * t.G / p.group : t.kv[unit * t.G];
    const int n = slots_of(p, b);
    const scalar_i64 table = (scalar_i64)(uintptr_t)(p.tables + b * p.ts_b);
    const char* kh = (const char*)p.k + (int64_t)kvh * p.ks_h;
    const char* vh = (const char*)p.v + (int64_t)kvh * p.vs_h;
    const uint8_t* ksh = p.k_scales + (int64_t)kvh * p.kss_h;
    const uint8_t* vsh = p.v_scales + (int64_t)kvh * p.vss_h;
    const uint32_t ks_p = in_sgpr((uint32_t)p.ks_p), vs_p = in_sgpr((uint32_t)p.vs_p), pages = in_sgpr((uint32_t)p.P);
    const uint32_t kss_p = in_sgpr((uint32_t)p.kss_p), vss_p = in_sgpr((uint32_t)p.vss_p);
    const uint32_t page16 = in_sgpr((uint32_t)t.page16), magic = in_sgpr(t.magic), ts_w = in_sgpr((uint32_t)p.ts_w);

    // this wave's tiles: slots slot0, slot0 + BLK, ... below end, two halves each; the places in their pages are
    // known as soon as the pages' indices are asked for
    struct Ids {
      int64_t id[2];
      uint32_t place[2];
    };
    auto ids_of = [&](int slot) -> Ids {
      Ids x;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && one_page) {
          x.id[1] = x.id[0], x.place[1] = x.place[0] + 16;
          break;
        }
        const uint32_t u = (uint32_t)(slot + 16 * h) >> 4, pg = page16 == 1 ? u : __umulhi(u, magic);
        x.id[h] = slot + 16 * h < cap ? table[(uint64_t)pg * ts_w] : -1;
        x.place[h] = (u - pg * page16) * 16;
      }
      return x;
    };
    auto there = [&](int64_t id) { return (uint32_t)(id >> 32) == 0 && (uint32_t)id < pages; };
    // Rows `rows` from a place of page `id` on: keys and values of one half or both (to LDS at lds), positions; what is
    // behind the row's end, and of no page, reads 0.  (Strides fit 32 bits, so an address is two multiplications.)
    struct Scales {
      uint64_t k, v;
    };
    auto load_rows = [&](int64_t id, uint32_t place, int rows, uint32_t lds, auto first, auto halves) -> Scales {
      constexpr int H0 = decltype(first)::value, HN = decltype(halves)::value;
      const bool ok = there(id) && rows > 0;
      const uint32_t at = ok ? (uint32_t)id : 0u, last = (uint32_t)(min(rows, 16 * HN) - 1);
      if (!ok) place = 0;
      const i32x4 krs = make_rsrc(kh + (uint64_t)at * ks_p + (uint64_t)place * krow, ok ? last * krow + L::ROW : 0u);
      const i32x4 vrs = make_rsrc(vh + (uint64_t)at * vs_p + (uint64_t)place * vrow, ok ? last * vrow + L::ROW : 0u);
#pragma unroll
      for (int h = H0; h < H0 + HN; ++h)
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i) buffer_load_lds16_nt_m0(krs, lds + h * L::HALF + i * 1024, k_voff[h][i]);
#pragma unroll
      for (int h = H0; h < H0 + HN; ++h)
#pragma unroll
        for (int i = 0; i < L::LOADS; ++i)
          buffer_load_lds16_nt_m0(vrs, lds + L::TILE_BYTES + h * L::HALF + i * 1024, v_voff[h][i]);
      if constexpr (POS) {
        const i32x4 prs = make_rsrc(p.pos + (int64_t)at * p.ps_p + place, ok ? (last + 1) * 8 : 0);
        if (lane < 8 * HN) buffer_load_lds16_m0(prs, lds + L::POS + H0 * 128, lane * 16);
      }
      // (the scale bytes of all slots, which a page holds whatever the row's length; of no page, page 0's)
      return {(uint64_t)ksh + (uint64_t)at * kss_p + place, (uint64_t)vsh + (uint64_t)at * vss_p + place};
    };
    auto load_tile = [&](int slot, const Ids& ids, int buf) {
      const uint32_t lds = wave_lds + buf * L::BUF_BYTES;
      typedef std::integral_constant<int, 0> I0;
      typedef std::integral_constant<int, 1> I1;
      uint64_t from;  // lanes 0, 1: K's scales of the halves, 2, 3: V's
      if (one_page) {
        const Scales x = load_rows(ids.id[0], ids.place[0], n - slot, lds, I0(), std::integral_constant<int, 2>());
        from = (lane & 2 ? x.v : x.k) + 16 * (lane & 1);
      } else {
        const Scales x = load_rows(ids.id[0], ids.place[0], n - slot, lds, I0(), I1());
        const Scales y = load_rows(ids.id[1], ids.place[1], n - slot - 16, lds, I1(), I1());
        const uint64_t k = lane & 1 ? y.k : x.k, v = lane & 1 ? y.v : x.v;
        from = lane & 2 ? v : k;
      }
      if (lane < 4) global_load_lds16_m0(from, lds + L::SCALES);
    };
    // (with positions two of a page's halves come at once, or each by a load of its own)
    constexpr int LPT = 4 * L::LOADS + 1 + (POS ? 1 : 0);

    // (the first two tiles are on their way before the queries' positions are known: they may be read
    // for nothing)
    int end = min(hi * BLK, n);
    int s0 = lo * BLK + wave * TK8;  // the tile being computed; s0 + BLK and s0 + 2 BLK follow
    Ids id0 = ids_of(s0), id1 = ids_of(s0 + BLK), id2 = ids_of(s0 + 2 * BLK);
    if (s0 < end) load_tile(s0, id0, 0);
    if (s0 + BLK < end) load_tile(s0 + BLK, id1, 1);

    const int64_t qpos = TREE ? 0 : p.q_pos[b * p.qps_b + rs * p.qps_s];
    // this lane's query fragments (B operand of S = K.Q^T), the sign of a negative scale folded in: features in
    // the order in which a lane holds a key's
    frag8 qf[D / 32];
    {
      const T* qp = (const T*)p.q + b * p.qs_b + rs * p.qs_s + (int64_t)(unit * t.G + rg) * p.qs_h + grp * 16;
      const uint32_t keep = row_real ? 0xffffffffu : 0u;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        u32x4 raw = *(const u32x4*)(qp + (ks >> 1) * 64 + (ks & 1) * 8);
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[w] = (raw[w] ^ flip) & keep;
        __builtin_memcpy(&qf[ks], &raw, 16);
      }
    }

    // limits: as in the 16-bit form
    int lim = n, lim_all = n, lim_any = n;
    TreeRow tree = {0, 0};
    bool row_sees = true;
    if (POS && p.causal && __ballot(row_real && qpos >= 0) == 0) lim_any = 0;
    if (TREE || (!POS && p.causal)) {
      const Limits x = limits_of<TREE>(p, b, n, qpos, rs, tree);
      lim = x.lim;
      row_sees = x.any > 0;
      lim_all = row_real ? lim : n;
      lim_any = row_real ? x.any : 0;
      if (p.Sq > 1) {
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) {
          lim_all = min(lim_all, __shfl_xor(lim_all, off, 64));
          lim_any = max(lim_any, __shfl_xor(lim_any, off, 64));
        }
      }
      lim_all = uniform(lim_all), lim_any = uniform(lim_any);  // (lane 0 holds a real row)
    }
    end = min(end, lim_any);
    if (s0 >= end) wait_vmcnt<0>();  // no tile to wait for below, but the buffers are free after it

    f32x4 o[D / 16];
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -__builtin_inff(), m_use = 0.f, l_run = 0.f;

    int buf = 0;
    for (; s0 < end; s0 += BLK) {
      if (s0 + BLK >= end) wait_vmcnt<0>();
      else if (POS && !one_page) wait_vmcnt<LPT + 1>();
      else wait_vmcnt<LPT>();  // this tile landed; the next may be in flight
      const char* tb = wb + buf * L::BUF_BYTES;
      u32x4 kr[2][D / 64];
      i32x2 vr[D / 16];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int ks = 0; ks < D / 64; ++ks) kr[h][ks] = *(const u32x4*)(tb + h * L::HALF + k_raddr[ks]);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        vr[dt] = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2_ptr)(tb + v_raddr[dt]));
      // the scales of this lane's key (K's rows) and of the keys whose scores it holds (V's)
      float kscale[2];
      uint32_t vscale[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        kscale[h] = scale_value(*(const uint8_t*)(tb + L::SCALES + 16 * h + row));
        vscale[h] = *(const uint32_t*)(tb + L::SCALES + TK8 + 16 * h + 4 * grp);
      }
      // which of this lane's keys (bits 0-3: 4 grp + i, bits 4-7: 16 + 4 grp + i) its row sees
      uint32_t vis = 0;
      bool whole;
      if constexpr (POS) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int64_t* pl = (const int64_t*)(tb + L::POS) + 16 * h + grp * 4;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t kp = pl[i];
            if (there(id0.id[h]) && s0 + 16 * h + grp * 4 + i < n && kp >= 0 && (!p.causal || kp <= qpos))
              vis |= 1u << (4 * h + i);
          }
        }
        whole = __ballot(row_real && vis != 255u) == 0;
      } else {
        whole = there(id0.id[0]) && there(id0.id[1]) && s0 + TK8 <= lim_all;
        if (!whole) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int slot = s0 + 16 * h + grp * 4;
            if constexpr (TREE) {
              if (there(id0.id[h]) && row_sees) vis |= tree_window<4>(tree, slot) << (4 * h);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (slot + i >= n) vis &= ~(1u << (4 * h + i));
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (there(id0.id[h]) && slot + i < lim) vis |= 1u << (4 * h + i);
            }
          }
        }
      }
      if (!row_real) vis = 0;
      bool odd = false;
      if (!whole) {
        // keys that no row sees hold 0, and is there a NaN among the others?
        uint32_t keep[2] = {0, 0}, nan = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if ((__ballot((vis >> e) & 1u) >> (16 * grp)) & 0xffffu) keep[e >> 2] |= 0xffu << (8 * (e & 3));
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t x = (uint32_t)vr[dt][w] & keep[w];
            vr[dt][w] = (int)x;
            nan |= (x & 0x7f7f7f7fu) + 0x01010101u;  // (bit 7 of a byte: it was 0x7f)
          }
        odd = __ballot(nan & 0x80808080u) != 0;
      }
      const bool more = s0 + 2 * BLK < end;
      if (more && !odd) {
        wait_lgkmcnt0();  // fragments in registers before the buffer is refilled
        load_tile(s0 + 2 * BLK, id2, buf);
      }
      const Ids id3 = ids_of(s0 + 3 * BLK);

      f32x4 s[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < D / 64; ++ks) {
          s[h] = Mfma16<T>::qk(widen8<T>(kr[h][ks][0], kr[h][ks][1], kscale[h]), qf[2 * ks], s[h]);
          s[h] = Mfma16<T>::qk(widen8<T>(kr[h][ks][2], kr[h][ks][3], kscale[h]), qf[2 * ks + 1], s[h]);
        }
      }
      if (!whole) {  // (in whole tiles rows that are none hold scores of 0, which reach no other row)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!((vis >> e) & 1u)) s[e >> 2][e & 3] = -__builtin_inff();
      }
      float mx = __builtin_fmaxf(__builtin_fmaxf(__builtin_fmaxf(s[0][0], s[0][1]), __builtin_fmaxf(s[0][2], s[0][3])),
                                 __builtin_fmaxf(__builtin_fmaxf(s[1][0], s[1][1]), __builtin_fmaxf(s[1][2], s[1][3])));
      mx = max_halves(max_rows16(mx));
      const bool grow = mx > m_run + grow_thr;
      if (__ballot(grow) != 0) {
        const float m_new = grow ? mx : m_run;
        const float alpha = grow ? __builtin_amdgcn_exp2f((m_run - m_new) * c) : 1.f;
        m_run = m_new;
        m_use = m_run == -__builtin_inff() ? 0.f : m_run * c;
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) o[dt] *= alpha;
      }
      float pv[8];  // probabilities, then with V's scales
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[e >> 2][e & 3], c, -m_use));
      l_run += ((pv[0] + pv[1]) + (pv[2] + pv[3])) + ((pv[4] + pv[5]) + (pv[6] + pv[7]));
#pragma unroll
      for (int e = 0; e < 8; ++e)
        pv[e] = __builtin_amdgcn_ldexpf(pv[e], (int)((vscale[e >> 2] >> (8 * (e & 3))) & 255u) - 127 + kHeldLog2);
      if (!odd) {
        bf16x8 pf[PC];
#pragma unroll
        for (int pc = 0; pc < PC; ++pc)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            pf[pc][e] = (bf16)pv[e];
            pv[e] -= to_f32<bf16>(pf[pc][e]);
          }
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
          const bf16x8 vf = widen8<bf16>((uint32_t)vr[dt][0], (uint32_t)vr[dt][1], 1.f);
#pragma unroll
          for (int pc = 0; pc < PC; ++pc) o[dt] = Mfma16<bf16>::qk(vf, pf[pc], o[dt]);
        }
      } else {
        for (int j = 0; j < TK8; ++j) {
          const int from = ((j >> 2) & 3) * 16 + row, at = (j >> 4) * 4 + (j & 3);
          float w = 0.f;
          bool sees = false;
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float x = __shfl(pv[e], from, 64);
            const uint32_t v = __shfl((int)vis, from, 64);
            if (at == e) w = x, sees = (v >> e) & 1u;
          }
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const uint8_t* vj = (const uint8_t*)(tb + L::TILE_BYTES + j * L::ROW + ((dt ^ v8_swz<D>(j)) << 4)) + grp * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (sees) o[dt][i] += w * __builtin_amdgcn_cvt_f32_fp8(vj[i], 0);
          }
        }
        wait_lgkmcnt0();
        if (more) load_tile(s0 + 2 * BLK, id2, buf);
      }
      id0 = id1, id1 = id2, id2 = id3;
      buf ^= 1;
    }

    finish_unit<T, D, NW, !SPLIT, kHeldLog2>(t, o, m_run, l_run, red_ml, dsmem, L::WAVE_BYTES, b, unit, lo == 0, hi == blocks,
                                             1.f);
    if constexpr (!SPLIT) return;
    const auto blocks_in = [&](int row) {
      const int n = slots_of(p, row);
      return n > 0 ? (n + BLK - 1) / BLK : 1;
    };
    if (!next_unit(b, unit, lo, left, blocks, hi - lo, t.units, p.B, blocks_in)) return;
    __syncthreads();  // the next unit's tiles overwrite the waves' sums
  }
}

template <typename T, int D, int VIS, int PC, int NW, bool SPLIT>
int launch_waves(const TokenParams& t, unsigned wgs, hipStream_t st) {
  constexpr int lds = NW * T8Layout<D>::WAVE_BYTES;
  const hipError_t e = reserve_lds<paged_token8_kernel<T, D, VIS, NW, SPLIT, PC>>(lds);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "paged_attention: cannot reserve %d bytes of LDS: %s", lds,
              hipGetErrorString(e));
  hipLaunchKernelGGL((paged_token8_kernel<T, D, VIS, NW, SPLIT, PC>), dim3(wgs), dim3(NW * 64), lds, st, t);
  CEA_CHECK_LAUNCH("paged_token8");
  return CEA_OK;
}

template <typename T, int D, int VIS, int PC> int launch_form(const TokenParams& t, bool whole, hipStream_t st) {
  if (whole) {
    const int64_t pairs = (int64_t)t.p.B * t.units;
    if (D == 64 && pairs <= 256) return launch_waves<T, D, VIS, PC, D == 64 ? 16 : 8, false>(t, (unsigned)pairs, st);
    if (pairs <= (D == 64 ? 512 : 384)) return launch_waves<T, D, VIS, PC, 8, false>(t, (unsigned)pairs, st);
    return launch_waves<T, D, VIS, PC, 4, false>(t, (unsigned)pairs, st);
  }
  const int rc = launch_waves<T, D, VIS, PC, NW_SPLIT, true>(t, (unsigned)t.wgs, st);
  if (rc) return rc;
  hipLaunchKernelGGL((paged_token_join_kernel<T, D, NW_SPLIT * TK8>), dim3((unsigned)(t.p.B * t.p.Sq * t.p.Hq)), dim3(256),
                     0, st, t);
  CEA_CHECK_LAUNCH("paged_token_join");
  return CEA_OK;
}

template <typename T, int D> int launch_td(const TokenParams& t, bool whole, hipStream_t st) {
  const bool f32 = t.p.out_dtype == CEA_F32;
  if (t.p.masks) return f32 ? launch_form<T, D, kTree, 3>(t, whole, st) : launch_form<T, D, kTree, 2>(t, whole, st);
  if (t.p.pos) return f32 ? launch_form<T, D, kPosition, 3>(t, whole, st) : launch_form<T, D, kPosition, 2>(t, whole, st);
  return f32 ? launch_form<T, D, kNumber, 3>(t, whole, st) : launch_form<T, D, kNumber, 2>(t, whole, st);
}

}  // namespace

int launch_paged_token8(const TokenParams& t, bool whole, hipStream_t st) {
  if (t.p.in_dtype == CEA_BF16) return t.p.D == 128 ? launch_td<bf16, 128>(t, whole, st) : launch_td<bf16, 64>(t, whole, st);
  return t.p.D == 128 ? launch_td<f16, 128>(t, whole, st) : launch_td<f16, 64>(t, whole, st);
}

}  // namespace cea

// Attention of a few new tokens per row over a paged KV cache (bf16 / f16, head size 64 or 128):
// the serving form, HBM-bound.
//
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(s_j - m),  s_j = scale * q.k_j,  lse = m + log sum_j p_j
//
// over the keys that a query sees, in one pass with a running maximum and sum (f32) per query row.
//   * A unit is the query heads of one KV head times the row's new tokens, at most 16 query rows:
//     the columns of 16 x 16 matrix-core tiles, so every key and value is read once for all of them.
//     S = K.Q^T with v_mfma_f32_16x16x32 (a lane holds 4 keys of one query row), O^T += V^T.P^T with
//     v_mfma_f32_16x16x16 (P is the score tile as it is).  The products are a tenth of the time that
//     the reads take, so P enters as the sum of two 16-bit pieces, three of bf16 for f32 results
//     (p rounded, then what that left, and so on), and a result is as exact as f32 probabilities.
//   * Every wave streams 16-key tiles of its own, K and V straight into a pair of LDS buffers of its
//     own (buffer_load ... lds, non-temporal, explicit vmcnt waits, no barriers), two tiles in
//     flight.  A tile lies in one page (pages are multiples of 16 slots), so its address is
//     scalar: the page index comes through the scalar cache, requested a tile ahead.
//   * Lengths are known on the device alone.  The keys of all rows and units, in blocks of 64, are one
//     line that the workgroups cut into equal runs, whatever the rows' lengths: a run may
//     span several units (each joined and finished in the workgroup) or be part of one, whose
//     unnormalised (o, m, l) go to the workspace, and a second launch joins the parts of the
//     units that were cut.  Short tables (kTokenWhole) take one workgroup of 4 to 16 waves per
//     unit and one launch.
//   * The nodes of a tree see slots by a window of their mask's word (16 nodes at most, so one) in the tiles that
//     reach into the tree; before it nothing changes.
//   * Measured: 32 rows of 1024 to 32768 keys, 32/8 heads of 128, bf16: 358 us for 2.2 GB, 6.2 TB/s (reads
//     reach 6.3 here, a copy 4.9), 364 with f32 results; 8 rows of 100 to 4096 keys in f16 22.6 us, 18 of them
//     the stream and 4.5 the join; one row of 777 keys, 32/4 heads of 64, 10.7 us, a chain of dependent trips to memory (length,
//     page index, keys) and 4 tiles a wave.
//   * Hidden keys are masked in the scores, and tiles behind the last visible slot are not read.  A
//     value that is not finite would meet the zero probabilities of hidden keys and the zero or
//     negative later pieces of visible ones: a tile that holds one (rare; a look of two instructions
//     per register) sums its products one by one, over each row's visible keys only.
#include "paged_token.hpp"

namespace cea {
namespace {

constexpr int TK = 16;                // keys per tile

template <int D> struct TLayout {
  static constexpr int ROW = D * 2;
  static constexpr int TILE_BYTES = TK * ROW;
  static constexpr int POS_BYTES = TK * 8;
  static constexpr int BUF_BYTES = 2 * TILE_BYTES + POS_BYTES;
  static constexpr int WAVE_BYTES = 2 * BUF_BYTES;
  static constexpr int LOADS = TILE_BYTES / 1024;
};

template <typename T, int D, int VIS, int NW, bool SPLIT, int PC>
__global__ __launch_bounds__(NW * 64, D == 64 ? 4 : 2) void paged_token_kernel(const TokenParams args) {
  constexpr bool POS = VIS == kPosition, TREE = VIS == kTree;
  typedef TLayout<D> L;
  typedef typename Mfma16<T>::frag8 frag8;
  constexpr int BLK = NW * TK;
  constexpr float kPScale = std::is_same<T, f16>::value ? 128.f : 1.f;  // keeps the second piece normal
  extern __shared__ __attribute__((aligned(16))) char dsmem[];
  __shared__ float2 red_ml[ROWS][NW];
  const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const int row = lane & 15, grp = lane >> 4;
  const int nrows = args.p.Sq * args.G;
  const bool row_real = row < nrows;
  const int rs = row_real ? row / args.G : 0, rg = row_real ? row - rs * args.G : 0;
  char* wb = dsmem + wave * L::WAVE_BYTES;

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
  const uint32_t krow = (uint32_t)(args.p.ks_s * sizeof(T)), vrow = (uint32_t)(args.p.vs_s * sizeof(T));
  uint32_t k_voff[L::LOADS], v_voff[L::LOADS];
#pragma unroll
  for (int i = 0; i < L::LOADS; ++i) {
    const int r = i * (1024 / L::ROW) + lane / (L::ROW / 16);
    const int pg = lane % (L::ROW / 16);                                        // physical 16-byte group
    k_voff[i] = r * krow + ((pg ^ (r & (L::ROW / 16 - 1))) << 4);               // K: 16-byte groups ^ row
    const int lgv = ((((pg >> 1) ^ (r & (L::ROW / 32 - 1))) << 1) | (pg & 1));  // V: 32-byte blocks ^ row
    v_voff[i] = r * vrow + (lgv << 4);
  }
  uint32_t k_raddr[D / 32], v_raddr[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 32; ++ks) k_raddr[ks] = row * L::ROW + (((grp + 4 * ks) ^ (row & (L::ROW / 16 - 1))) << 4);
  {
    const int vr = grp * 4 + (row >> 2);
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt)
      v_raddr[dt] = L::TILE_BYTES + vr * L::ROW + ((dt ^ (vr & (L::ROW / 32 - 1))) << 5) + 8 * (row & 3);
  }

  while (true) {
    // ---- one unit of the run, blocks [lo, hi)
    // (the arguments are read again for every unit: kept across units they would fill the scalar
    // registers, whose spills took 24 to 48 vector registers and a wave of the occupancy)
    const kernel_args_ptr ap = opaque((kernel_args_ptr)__builtin_amdgcn_kernarg_segment_ptr());
    const TokenParams& t = *(const TokenParams*)ap;
    const PagedParams& p = t.p;
    const int hi = min(blocks, lo + left);
    const int kvh = p.group > 0 ? unit * t.G / p.group : t.kv[unit * t.G];
    const int n = slots_of(p, b);
    const scalar_i64 table = (scalar_i64)(uintptr_t)(p.tables + b * p.ts_b);
    const char* kh = (const char*)((const T*)p.k + (int64_t)kvh * p.ks_h);
    const char* vh = (const char*)((const T*)p.v + (int64_t)kvh * p.vs_h);

    // this wave's tiles: slots slot0, slot0 + BLK, ... below end
    auto page_of = [&](int slot) -> int {
      const uint32_t u = (uint32_t)slot >> 4;
      return (int)(t.page16 == 1 ? u : __umulhi(u, t.magic));
    };
    // the page index of a slot's tile: a scalar read, which does not wait for lengths or positions
    auto id_of = [&](int slot) -> int64_t {
      return slot < cap ? table[(int64_t)page_of(slot) * p.ts_w] : -1;
    };
    auto load_tile = [&](int slot, int64_t id, int buf) {
      const bool ok = id >= 0 && id < p.P;
      const int64_t at = ok ? id : 0;
      const int place = slot - page_of(slot) * (t.page16 * 16);
      const uint32_t rows = (uint32_t)min(n - slot, TK);  // slots behind the row's end read 0
      const uint32_t kb = ok ? (rows - 1) * krow + L::ROW : 0u, vb = ok ? (rows - 1) * vrow + L::ROW : 0u;
      const i32x4 krs = make_rsrc(kh + (at * p.ks_p + (int64_t)place * p.ks_s) * (int64_t)sizeof(T), kb);
      const i32x4 vrs = make_rsrc(vh + (at * p.vs_p + (int64_t)place * p.vs_s) * (int64_t)sizeof(T), vb);
      char* dst = wb + buf * L::BUF_BYTES;
#pragma unroll
      for (int i = 0; i < L::LOADS; ++i) buffer_load_lds16_nt(krs, dst + i * 1024, k_voff[i]);
#pragma unroll
      for (int i = 0; i < L::LOADS; ++i) buffer_load_lds16_nt(vrs, dst + L::TILE_BYTES + i * 1024, v_voff[i]);
      if constexpr (POS) {
        const i32x4 prs = make_rsrc(p.pos + at * p.ps_p + place, ok ? rows * 8 : 0u);
        if (lane < TK / 2) buffer_load_lds16(prs, dst + 2 * L::TILE_BYTES, lane * 16);
      }
    };
    constexpr int LPT = 2 * L::LOADS + (POS ? 1 : 0);

    // (the first two tiles are on their way before the queries' positions are known: they may be read
    // for nothing)
    int end = min(hi * BLK, n);
    int s0 = lo * BLK + wave * TK;  // the tile being computed; s0 + BLK and s0 + 2 BLK follow
    int64_t id0 = id_of(s0), id1 = id_of(s0 + BLK), id2 = id_of(s0 + 2 * BLK);
    if (s0 < end) load_tile(s0, id0, 0);
    if (s0 + BLK < end) load_tile(s0 + BLK, id1, 1);

    const int64_t qpos = TREE ? 0 : p.q_pos[b * p.qps_b + rs * p.qps_s];
    // this lane's query fragments (B operand of S = K.Q^T), the sign of a negative scale folded in
    frag8 qf[D / 32];
    {
      const T* qp = (const T*)p.q + b * p.qs_b + rs * p.qs_s + (int64_t)(unit * t.G + rg) * p.qs_h + grp * 8;
      const uint32_t keep = row_real ? 0xffffffffu : 0u;
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) {
        u32x4 raw = *(const u32x4*)(qp + ks * 32);
#pragma unroll
        for (int w = 0; w < 4; ++w) raw[w] = (raw[w] ^ flip) & keep;
        __builtin_memcpy(&qf[ks], &raw, 16);
      }
    }

    // this lane's row sees slots [0, lim) by their number, all rows see [0, lim_all), none beyond
    // lim_any (with positions in the pool the slots say nothing but where the row ends)
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
      if (s0 + BLK < end) wait_vmcnt<LPT>();  // this tile landed; the next may be in flight
      else wait_vmcnt<0>();
      const char* tb = wb + buf * L::BUF_BYTES;
      frag8 kf[D / 32];
      s16x4 vf[D / 16];
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) kf[ks] = *(const frag8*)(tb + k_raddr[ks]);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        vf[dt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_ptr)(tb + v_raddr[dt]));
      // which of this lane's keys its row sees
      const bool ok = id0 >= 0 && id0 < p.P;
      uint32_t vis = 0;
      bool whole;
      if constexpr (POS) {
        const int64_t* pl = (const int64_t*)(tb + 2 * L::TILE_BYTES) + grp * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t kp = pl[i];
          if (ok && s0 + grp * 4 + i < n && kp >= 0 && (!p.causal || kp <= qpos)) vis |= 1u << i;
        }
        whole = __ballot(row_real && vis != 15u) == 0;
      } else {
        whole = ok && s0 + TK <= lim_all;
        if constexpr (TREE) {
          if (ok && row_sees) vis = tree_window<4>(tree, s0 + grp * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (s0 + grp * 4 + i >= n) vis &= ~(1u << i);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (ok && s0 + grp * 4 + i < lim) vis |= 1u << i;
        }
      }
      if (!row_real) vis = 0;
      // a value that is not finite (products with zero or negative pieces would spoil it)
      u16x2 top = {0, 0};
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const u16x2 mag = {(uint16_t)(vf[dt][i] & 0x7fff), (uint16_t)(vf[dt][i + 1] & 0x7fff)};
          top = __builtin_elementwise_max(top, mag);
        }
      constexpr uint16_t kInf = std::is_same<T, bf16>::value ? 0x7f80 : 0x7c00;
      const bool odd = __ballot(top[0] >= kInf || top[1] >= kInf) != 0;
      const bool more = s0 + 2 * BLK < end;
      if (more && !odd) {
        wait_lgkmcnt0();  // fragments in registers before the buffer is refilled
        load_tile(s0 + 2 * BLK, id2, buf);
      }
      const int64_t id3 = id_of(s0 + 3 * BLK);

      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < D / 32; ++ks) s = Mfma16<T>::qk(kf[ks], qf[ks], s);
      if (!whole || nrows < ROWS) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (!((vis >> i) & 1u)) s[i] = -__builtin_inff();
      }
      float mx = __builtin_fmaxf(__builtin_fmaxf(s[0], s[1]), __builtin_fmaxf(s[2], s[3]));
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
      float pv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) pv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -m_use));
      l_run += (pv[0] + pv[1]) + (pv[2] + pv[3]);
      if (!odd) {
        float rest[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) rest[i] = pv[i] * kPScale;
#pragma unroll
        for (int pc = 0; pc < PC; ++pc) {
          const s16x4 pf = Mfma16<T>::pack(rest[0], rest[1], rest[2], rest[3]);
#pragma unroll
          for (int i = 0; i < 4; ++i) rest[i] -= to_f32<T>(__builtin_bit_cast(T, (short)pf[i]));
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) o[dt] = Mfma16<T>::pv(vf[dt], pf, o[dt]);
        }
      } else {
        for (int j = 0; j < TK; ++j) {
          const int from = (j >> 2) * 16 + row;
          float w = 0.f;
          bool sees = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = __shfl(pv[i], from, 64);
            const uint32_t v = __shfl((int)vis, from, 64);
            if ((j & 3) == i) w = x * kPScale, sees = (v >> i) & 1u;
          }
#pragma unroll
          for (int dt = 0; dt < D / 16; ++dt) {
            const T* vr = (const T*)(tb + L::TILE_BYTES + j * L::ROW + ((dt ^ (j & (L::ROW / 32 - 1))) << 5));
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (sees) o[dt][i] += w * to_f32<T>(vr[grp * 4 + i]);
          }
        }
        wait_lgkmcnt0();
        if (more) load_tile(s0 + 2 * BLK, id2, buf);
      }
      id0 = id1, id1 = id2, id2 = id3;
      buf ^= 1;
    }

    finish_unit<T, D, NW, !SPLIT, 0>(t, o, m_run, l_run, red_ml, dsmem, L::WAVE_BYTES, b, unit, lo == 0, hi == blocks,
                                  1.f / kPScale);
    if constexpr (!SPLIT) return;
    const auto blocks_in = [&](int row) {
      const int n = slots_of(p, row);
      return n > 0 ? (n + BLK - 1) / BLK : 1;
    };
    if (!next_unit(b, unit, lo, left, blocks, hi - lo, t.units, p.B, blocks_in)) return;
    __syncthreads();  // the next unit's tiles overwrite the waves' sums
  }
}

template <typename T, int D, int VIS, int PC, int NW>
int launch_whole(const TokenParams& t, hipStream_t st) {
  constexpr int lds = NW * TLayout<D>::WAVE_BYTES;
  const hipError_t e = reserve_lds<paged_token_kernel<T, D, VIS, NW, false, PC>>(lds);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "paged_attention: cannot reserve %d bytes of LDS: %s", lds,
              hipGetErrorString(e));
  hipLaunchKernelGGL((paged_token_kernel<T, D, VIS, NW, false, PC>), dim3((unsigned)(t.p.B * t.units)), dim3(NW * 64),
                     lds, st, t);
  CEA_CHECK_LAUNCH("paged_token");
  return CEA_OK;
}

template <typename T, int D, int VIS, int PC>
int launch_form(const TokenParams& t, bool whole, hipStream_t st) {
  typedef TLayout<D> L;
  if (whole) {
    // as many waves as keep all units resident at once (us, 4 / 8 / 16 waves: 4 units of 777 keys, D =
    // 64, 14.9 / 10.3 / 9.8; 256 units of up to 1000, D = 64, 18.6 / 13.9 / 13.6; D = 128: 64 units
    // of up to 1000 keys 21.4 / 16.4 / -, 320 26.3 / 24.5 / -, 512 of up to 700 26.6 / 28.1 / -)
    const int64_t pairs = (int64_t)t.p.B * t.units;
    if (D == 64 && pairs <= 256) return launch_whole<T, D, VIS, PC, D == 64 ? 16 : 8>(t, st);
    if (pairs <= (D == 64 ? 512 : 384)) return launch_whole<T, D, VIS, PC, 8>(t, st);
    return launch_whole<T, D, VIS, PC, 4>(t, st);
  }
  constexpr int lds = NW_SPLIT * L::WAVE_BYTES;
  const hipError_t e = reserve_lds<paged_token_kernel<T, D, VIS, NW_SPLIT, true, PC>>(lds);
  CEA_REQUIRE(e == hipSuccess, CEA_ELAUNCH, "paged_attention: cannot reserve %d bytes of LDS: %s", lds,
              hipGetErrorString(e));
  hipLaunchKernelGGL((paged_token_kernel<T, D, VIS, NW_SPLIT, true, PC>), dim3((unsigned)t.wgs), dim3(NW_SPLIT * 64),
                     lds, st, t);
  CEA_CHECK_LAUNCH("paged_token");
  hipLaunchKernelGGL((paged_token_join_kernel<T, D, NW_SPLIT * TK>), dim3((unsigned)(t.p.B * t.p.Sq * t.p.Hq)), dim3(256),
                     0, st, t);
  CEA_CHECK_LAUNCH("paged_token_join");
  return CEA_OK;
}

template <typename T, int D> int launch_td(const TokenParams& t, bool whole, hipStream_t st) {
  constexpr int kFull = std::is_same<T, bf16>::value ? 3 : 2;  // pieces that hold an f32 probability
  const bool f32 = t.p.out_dtype == CEA_F32;
  if (t.p.masks)
    return f32 ? launch_form<T, D, kTree, kFull>(t, whole, st) : launch_form<T, D, kTree, 2>(t, whole, st);
  if (t.p.pos)
    return f32 ? launch_form<T, D, kPosition, kFull>(t, whole, st) : launch_form<T, D, kPosition, 2>(t, whole, st);
  return f32 ? launch_form<T, D, kNumber, kFull>(t, whole, st) : launch_form<T, D, kNumber, 2>(t, whole, st);
}

// Query heads of a unit: a KV head's whole group, or the largest part of it whose rows fit.
int unit_heads(int64_t Sq, int64_t Hq, int64_t Hkv, int group) {
  if (group <= 0) return Sq <= ROWS ? 1 : 0;
  for (int64_t g = group; g >= 1; --g)
    if (group % g == 0 && g * Sq <= ROWS) return (int)g;
  return 0;
}

// Slots of a table up to which a unit is one workgroup's.  The second launch of a split costs the host 3 us,
// and more on the GPU than it saves from a few hundred units on; a captured call of few units at D = 128 would
// gain by it.  us, whole / split, in a stream of calls (in a graph): 4 units of 300 keys, D = 64, 11.7 / 14.9 (6.9 /
// 9.7), 4 of 777 11.7 / 14.8 (9.8 / 9.9), 4 of 1500 - (14.1 / 9.9), 256 of up to 1000 13.7 / 26.4; D = 128: 8 of 777
// 13.1 / 15.0 (12.4 / 10.8), 64 of up to 1000 16.7 / 15.8 (16.3 / 14.9), 320 24.5 / 32.9, 512 of up to 700 26.1 / 42.2.
constexpr int64_t kTokenWhole = 1024;

TokenPlan plan_token(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int group, int64_t slots, bool f8) {
  TokenPlan r;
  r.G = unit_heads(Sq, Hq, Hkv, group);
  r.units = r.G > 0 ? (int32_t)(Hq / r.G) : 0;
  r.whole = slots <= kTokenWhole;
  const int64_t block = NW_SPLIT * (f8 ? TK8 : TK), blocks = std::max<int64_t>(1, (slots + block - 1) / block);
  const int cus = device_cus() > 0 ? device_cus() : 256;
  // two workgroups per compute unit, as many as are resident at D = 128 (us, 512 / 1024: 8 rows of
  // 100 to 4096 keys, 32/8 heads of 128, 22.7 / 27.7; one row of 30000 31.4 / 37.1; 32 rows of 1024 to
  // 32768 346 / 348; 64 rows of 2500 to 7500, 32/4 heads of 64, 69.4 / 72.1; 16 of 500 to 2500 18.3 / 17.3)
  r.wgs = (int32_t)std::min<int64_t>(B * r.units * blocks, 2 * cus);
  return r;
}

}  // namespace

size_t paged_token_workspace_bytes(int64_t B, int64_t Sq, int64_t Hq, int64_t Hkv, int group, int64_t D,
                                   int64_t slots, bool f8) {
  const TokenPlan r = plan_token(B, Sq, Hq, Hkv, group, slots, f8);
  if (r.G == 0 || r.whole) return 0;
  return (size_t)r.wgs * 2 * Sq * r.G * (D + 2) * sizeof(float);
}

bool paged_token_supported(const PagedParams& p, const HeadMap& map) {
  if (map.group <= 0 && (p.Hq > kPagedMapHeads || p.Hkv > 256)) return false;
  const int g = unit_heads(p.Sq, p.Hq, p.Hkv, map.group);
  if (g == 0) return false;
  const int64_t units = p.Hq / g, blocks = ((int64_t)p.W * p.page + 63) / 64 + 1;
  return blocks < ((int64_t)1 << 25) && p.B * units * blocks < ((int64_t)1 << 30) &&
         (int64_t)p.B * p.Sq * p.Hq < ((int64_t)1 << 31);
}

int launch_paged_token(const PagedParams& p, const HeadMap& map, void* ws, hipStream_t st) {
  const TokenPlan r = plan_token(p.B, p.Sq, p.Hq, p.Hkv, map.group, (int64_t)p.W * p.page,
                                 p.kv_dtype == CEA_F8);
  TokenParams t;
  t.p = p;
  t.G = r.G, t.units = r.units, t.wgs = r.wgs;
  t.page16 = p.page / 16;
  t.magic = t.page16 > 1 ? (uint32_t)((((uint64_t)1 << 32) + t.page16 - 1) / t.page16) : 0;
  t.partial = (float*)ws;
  for (int h = 0; h < kPagedMapHeads; ++h) t.kv[h] = map.group <= 0 && h < p.Hq ? (uint8_t)map.kv[h] : 0;
  if (p.kv_dtype == CEA_F8) return launch_paged_token8(t, r.whole, st);
  if (p.in_dtype == CEA_BF16)
    return p.D == 128 ? launch_td<bf16, 128>(t, r.whole, st) : launch_td<bf16, 64>(t, r.whole, st);
  return p.D == 128 ? launch_td<f16, 128>(t, r.whole, st) : launch_td<f16, 64>(t, r.whole, st);
}

}  // namespace cea

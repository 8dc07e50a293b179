// Attention over a paged KV cache for any element type, head size up to 256, page size and
// strides: the form behind f64, head sizes and layouts that the matrix-core kernels do not tile.
//
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale * q.k_j,  m = max_j s_j,
//   lse = m + log sum_j exp(s_j - m), over the keys j that the query sees; none: (0, -inf).
//
// One workgroup per (token, query head); its four waves take 64-key blocks in turn.  A lane owns
// one key for the scores and one feature in 64 for the values, so hidden keys are never read and
// cannot reach a sum, whatever they hold.  Bound by latency and by the L2 reads of K and V, which
// every query row repeats: one row of 777 keys, 32/4 heads of 64 in bf16, takes 52 us (the token kernel 11),
// 128 tokens over 32768 keys 20 ms (the chunk kernel 0.09).
#include "paged.hpp"

namespace cea {
namespace {

constexpr int GWAVES = 4;
constexpr int DMAX = 256;

__device__ __forceinline__ float wave_max_of(float v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmaxf(v, __shfl_xor(v, off, 64));
  return v;
}
__device__ __forceinline__ double wave_max_of(double v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v = fmax(v, __shfl_xor(v, off, 64));
  return v;
}

template <typename T, typename A, typename O>
__global__ __launch_bounds__(GWAVES * 64) void paged_generic_kernel(const PagedParams p,
                                                                    const HeadMap map) {
  __shared__ A q_s[DMAX];
  __shared__ A o_s[GWAVES][DMAX];
  __shared__ A m_s[GWAVES], l_s[GWAVES];
  const int64_t id = blockIdx.x;
  const int h = (int)(id % p.Hq);
  const int s = (int)((id / p.Hq) % p.Sq);
  const int b = (int)(id / ((int64_t)p.Hq * p.Sq));
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int D = p.D, kvh = map.kv_of(h);
  const A scale = (A)p.scale;
  const T* qp = (const T*)p.q + b * p.qs_b + s * p.qs_s + h * p.qs_h;
  for (int d = tid; d < D; d += GWAVES * 64) q_s[d] = load_acc<T, A>(qp + d);
  __syncthreads();

  const int64_t n = paged_slots(p, b);
  const int64_t qpos = p.q_pos[b * p.qps_b + s * p.qps_s];
  const T* kbase = (const T*)p.k + kvh * p.ks_h;
  const T* vbase = (const T*)p.v + kvh * p.vs_h;
  A m = neg_inf<A>(), l = 0, o[DMAX / 64];
#pragma unroll
  for (int i = 0; i < DMAX / 64; ++i) o[i] = 0;

  for (int64_t k0 = wave * 64; k0 < n; k0 += GWAVES * 64) {
    const int64_t j = k0 + lane;
    bool vis = false;
    int64_t koff = 0, voff = 0;
    if (j < n) {
      const int64_t pg = j / p.page, place = j - pg * p.page;
      const int64_t id = p.tables[b * p.ts_b + pg * p.ts_w];
      if (id >= 0 && id < p.P) {
        const int64_t pos = p.pos ? p.pos[id * p.ps_p + place * p.ps_s] : j;
        vis = pos >= 0 && (!p.causal || pos <= qpos);
        koff = id * p.ks_p + place * p.ks_s;
        voff = id * p.vs_p + place * p.vs_s;
      }
    }
    uint64_t left = __ballot(vis);
    if (left == 0) continue;
    A x = neg_inf<A>();
    if (vis) {
      const T* kr = kbase + koff;
      A dot = 0;
      for (int d = 0; d < D; ++d) dot += q_s[d] * load_acc<T, A>(kr + d);
      x = dot * scale;
    }
    const A mx = wave_max_of(x);
    const A m_new = mx > m ? mx : m;
    const A shift = m_new == neg_inf<A>() ? (A)0 : m_new;
    const A alpha = m == neg_inf<A>() ? (A)0 : exp_acc(m - shift);
    const A pr = vis ? exp_acc(x - shift) : (A)0;
    m = m_new;
    l = l * alpha + wave_sum(pr);
#pragma unroll
    for (int i = 0; i < DMAX / 64; ++i) o[i] *= alpha;
    while (left != 0) {
      const int key = (int)__builtin_ctzll(left);
      left &= left - 1;
      const A w = __shfl(pr, key, 64);
      const T* vr = vbase + __shfl(voff, key, 64);
#pragma unroll
      for (int i = 0; i < DMAX / 64; ++i)
        if (i * 64 + lane < D) o[i] += w * load_acc<T, A>(vr + i * 64 + lane);
    }
  }

  // join the waves; a row's sum is 0 exactly where it saw no key (a NaN is kept)
  if (lane == 0) m_s[wave] = m, l_s[wave] = l;
#pragma unroll
  for (int i = 0; i < DMAX / 64; ++i)
    if (i * 64 + lane < D) o_s[wave][i * 64 + lane] = o[i];
  __syncthreads();
  A top = neg_inf<A>(), total = 0;
  for (int w = 0; w < GWAVES; ++w) top = m_s[w] > top ? m_s[w] : top;
  const A shift = top == neg_inf<A>() ? (A)0 : top;
  A wt[GWAVES];
  for (int w = 0; w < GWAVES; ++w) {
    wt[w] = l_s[w] == 0 ? (A)0 : m_s[w] == neg_inf<A>() ? (A)1 : exp_acc(m_s[w] - shift);
    total += l_s[w] * wt[w];
  }
  O* orow = (O*)p.out + b * p.os_b + s * p.os_s + h * p.os_h;
  for (int d = tid; d < D; d += GWAVES * 64) {
    A acc = 0;
    for (int w = 0; w < GWAVES; ++w)
      if (l_s[w] != 0) acc += o_s[w][d] * wt[w];
    orow[d] = store_cast<O, A>(total == 0 ? (A)0 : acc / total);
  }
  if (p.lse && tid == 0) {
    A* lp = (A*)p.lse + b * p.ls_b + h * p.ls_h + s * p.ls_s;
    *lp = total == 0 ? neg_inf<A>() : shift + log_acc(total);
  }
}

template <typename T, typename A, typename O>
int launch_rows(const PagedParams& p, const HeadMap& map, hipStream_t st) {
  const int64_t rows = (int64_t)p.B * p.Sq * p.Hq;
  CEA_REQUIRE(rows < (int64_t)1 << 31, CEA_EUNSUPPORTED, "paged_attention: too many query rows");
  hipLaunchKernelGGL((paged_generic_kernel<T, A, O>), dim3((unsigned)rows), dim3(GWAVES * 64), 0, st,
                     p, map);
  CEA_CHECK_LAUNCH("paged_attention");
  return CEA_OK;
}

}  // namespace

int launch_paged_generic(const PagedParams& p, const HeadMap& map, hipStream_t st) {
  CEA_REQUIRE(p.D <= DMAX, CEA_EUNSUPPORTED, "paged_attention: head size %d exceeds %d", p.D, DMAX);
  const bool acc = p.out_dtype == CEA_F32;
  switch (p.in_dtype) {
    case CEA_F64: return launch_rows<double, double, double>(p, map, st);
    case CEA_F32: return launch_rows<float, float, float>(p, map, st);
    case CEA_BF16:
      return acc ? launch_rows<bf16, float, float>(p, map, st) : launch_rows<bf16, float, bf16>(p, map, st);
    case CEA_F16:
      return acc ? launch_rows<f16, float, float>(p, map, st) : launch_rows<f16, float, f16>(p, map, st);
  }
  set_error("paged_attention: unsupported dtype %s", dtype_name(p.in_dtype));
  return CEA_EUNSUPPORTED;
}

}  // namespace cea

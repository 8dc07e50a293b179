// PyTorch operators of the collab_edge library: the thin PyTorch-ROCm layer between the
// package's Python functions and the C ABI of include/collab_edge_attn.h.
//
// Each operator checks that its tensors live on one ROCm device, allocates its outputs (and
// the kernels' workspace) through PyTorch's caching allocator on that device, makes the
// device current, and calls the C ABI on PyTorch's current stream of that device.  C ABI
// status codes become the exceptions the reference raises for the same conditions:
// CEA_EINVAL -> ValueError, CEA_EUNSUPPORTED -> NotImplementedError, others -> RuntimeError.
// Host (CPU) tensors are refused with RuntimeError: there is no host path.
#include <ATen/ATen.h>
#include <c10/core/Allocator.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/library.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

#include "collab_edge_attn.h"

namespace {

using at::Tensor;

int32_t code_of(c10::ScalarType t) {
  switch (t) {
    case at::kFloat: return CEA_F32;
    case at::kBFloat16: return CEA_BF16;
    case at::kHalf: return CEA_F16;
    case at::kDouble: return CEA_F64;
    case at::kLong: return CEA_I64;
    default: return -1;
  }
}

// The same with the types of 8-bit pages, which the paged cache's operators alone take.
int32_t page_code_of(c10::ScalarType t) {
  return t == at::kFloat8_e4m3fn ? CEA_F8 : t == at::kByte ? CEA_U8 : code_of(t);
}

cea_tensor arg(const Tensor& t, bool pages = false) {
  cea_tensor a;
  const int32_t code = pages ? page_code_of(t.scalar_type()) : code_of(t.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(code >= 0, "dtype ", t.scalar_type(), " is not supported by the kernels");
  TORCH_CHECK_VALUE(t.dim() <= CEA_MAX_DIMS, "at most ", CEA_MAX_DIMS, " dimensions supported, got ",
                    t.dim());
  a.data = t.numel() > 0 ? t.data_ptr() : nullptr;
  a.dtype = code;
  a.ndim = (int32_t)t.dim();
  for (int i = 0; i < CEA_MAX_DIMS; ++i) {
    a.size[i] = i < t.dim() ? t.size(i) : 0;
    a.stride[i] = i < t.dim() ? t.stride(i) : 0;
  }
  return a;
}

std::vector<cea_tensor> args(at::TensorList ts) {
  std::vector<cea_tensor> v;
  v.reserve(ts.size());
  for (const Tensor& t : ts) v.push_back(arg(t));
  return v;
}

void check_rc(int rc, const char* what) {
  if (rc == CEA_OK) return;
  const std::string msg = std::string(what) + ": " + cea_last_error();
  TORCH_CHECK_VALUE(rc != CEA_EINVAL, msg);
  TORCH_CHECK_NOT_IMPLEMENTED(rc != CEA_EUNSUPPORTED, msg);
  TORCH_CHECK(false, msg);
}

// The device all tensors share (every defined tensor must be on one ROCm device).
at::Device device_of(std::initializer_list<const Tensor*> ts, at::TensorList more = {}) {
  c10::optional<at::Device> dev;
  auto visit = [&](const Tensor& t) {
    if (!t.defined()) return;
    TORCH_CHECK(t.is_cuda(), "collaborative-edge-system_amd runs its kernels on a ROCm GPU; got a tensor on ",
                t.device());
    if (!dev) dev = t.device();
    TORCH_CHECK(t.device() == *dev, "tensors on different devices: ", *dev, " and ", t.device());
  };
  for (const Tensor* t : ts) visit(*t);
  for (const Tensor& t : more) visit(t);
  TORCH_CHECK(dev.has_value(), "no tensor given");
  return *dev;
}

// Every tensor of a further list on the device `dev` found for the call's other tensors.
void on_device(const at::Device& dev, at::TensorList more) {
  if (more.empty()) return;
  const at::Device d = device_of({}, more);
  TORCH_CHECK(d == dev, "tensors on different devices: ", dev, " and ", d);
}

void* stream_of(const at::Device& d) {
  return (void*)c10::hip::getCurrentHIPStream(d.index()).stream();
}

// The scratch of one call, on the current stream.  Each call takes its own from PyTorch's caching
// allocator, which hands freed memory out again in stream order only and serves a capture from
// the graph's own pool.  Scratch kept per stream would be shared: a call of several launches
// (tile summaries or partial sums, then the kernel that reads them) does not hold its stream, so
// another thread's call on it may come in between, and graphs captured on one stream may be
// replayed on several.
struct Scratch {
  c10::DataPtr mem;
  size_t size = 0;
  void* data() const { return mem.get(); }
};

// (the device is the current one: every operator holds a DeviceGuard when it asks)
Scratch workspace(size_t bytes) {
  static c10::Allocator* const device_memory = c10::GetAllocator(c10::DeviceType::CUDA);
  Scratch s;
  s.size = std::max<size_t>((bytes + 4095) & ~(size_t)4095, 4096);
  s.mem = device_memory->allocate(s.size);
  return s;
}

// q / k / v style operands need a unit innermost stride
Tensor inner(const Tensor& t) {
  return (t.dim() == 0 || t.size(-1) <= 1 || t.stride(-1) == 1) ? t : t.contiguous();
}

Tensor as_i64(const Tensor& t) { return t.scalar_type() == at::kLong ? t : t.to(at::kLong); }

at::ScalarType acc_of(at::ScalarType t) { return t == at::kDouble ? at::kDouble : at::kFloat; }

std::vector<int32_t> map_of(const c10::optional<at::IntArrayRef>& kv_map) {
  std::vector<int32_t> m;
  if (kv_map) for (int64_t x : *kv_map) m.push_back((int32_t)x);
  return m;
}

// ---------------------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------------------
std::vector<Tensor> attention(const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                              const Tensor& q_pos_in, const Tensor& k_pos_in, bool causal, double scale,
                              c10::optional<at::IntArrayRef> kv_map, bool with_lse) {
  const at::Device dev = device_of({&q_in, &k_in, &v_in, &q_pos_in, &k_pos_in});
  const Tensor q = inner(q_in), k = inner(k_in), v = inner(v_in);
  const Tensor qp = as_i64(q_pos_in), kp = as_i64(k_pos_in);
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "q and k must be [B, S, H, D]");
  const int64_t B = q.size(0), Sq = q.size(1), Hq = q.size(2), D = q.size(3);
  const int64_t Sk = k.size(1), Hkv = k.size(2);
  const at::ScalarType acc = acc_of(q.scalar_type());
  const auto o_opts = at::TensorOptions().device(dev).dtype(with_lse ? acc : q.scalar_type());
  Tensor out = at::empty({B, Sq, Hq, D}, o_opts);
  Tensor lse = with_lse ? at::empty({B, Hq, Sq}, o_opts.dtype(acc)) : Tensor();
  c10::DeviceGuard guard(dev);
  const std::vector<int32_t> m = map_of(kv_map);
  const Scratch ws = workspace(cea_attention_workspace_bytes(B, Sq, Hq, Sk, Hkv, D, code_of(q.scalar_type())));
  cea_tensor a[5] = {arg(q), arg(k), arg(v), arg(qp), arg(kp)};
  cea_tensor o = arg(out), l = with_lse ? arg(lse) : cea_tensor{};
  check_rc(cea_attention_with_lse(&a[0], &a[1], &a[2], &a[3], &a[4], causal ? 1 : 0, scale,
                                  m.empty() ? nullptr : m.data(), (int32_t)m.size(), &o,
                                  with_lse ? &l : nullptr, 0, ws.data(), ws.size,
                                  stream_of(dev)),
           "attention_with_lse");
  if (with_lse) return {out, lse};
  return {out};
}

void attention_into(Tensor out, Tensor lse, const Tensor& q_in, const Tensor& k_in, const Tensor& v_in,
                    const Tensor& q_pos_in, const Tensor& k_pos_in, bool causal, double scale,
                    c10::optional<at::IntArrayRef> kv_map, bool accumulate,
                    c10::optional<Tensor> final_out) {
  const Tensor fin = final_out ? *final_out : Tensor();
  const at::Device dev = device_of({&out, &lse, &q_in, &k_in, &v_in, &q_pos_in, &k_pos_in, &fin});
  const Tensor q = inner(q_in), k = inner(k_in), v = inner(v_in);
  const Tensor qp = as_i64(q_pos_in), kp = as_i64(k_pos_in);
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4, "q and k must be [B, S, H, D]");
  c10::DeviceGuard guard(dev);
  const std::vector<int32_t> m = map_of(kv_map);
  const Scratch ws = workspace(cea_attention_workspace_bytes(q.size(0), q.size(1), q.size(2), k.size(1),
                                                             k.size(2), q.size(3), code_of(q.scalar_type())));
  cea_tensor a[5] = {arg(q), arg(k), arg(v), arg(qp), arg(kp)};
  cea_tensor o = arg(out), l = arg(lse);
  if (fin.defined()) {
    cea_tensor f = arg(fin);
    check_rc(cea_attention_merge_final(&a[0], &a[1], &a[2], &a[3], &a[4], causal ? 1 : 0, scale,
                                       m.empty() ? nullptr : m.data(), (int32_t)m.size(), &o, &l, &f,
                                       ws.data(), ws.size, stream_of(dev)),
             "attention_merge_final");
    return;
  }
  check_rc(cea_attention_with_lse(&a[0], &a[1], &a[2], &a[3], &a[4], causal ? 1 : 0, scale,
                                  m.empty() ? nullptr : m.data(), (int32_t)m.size(), &o, &l,
                                  accumulate ? 1 : 0, ws.data(), ws.size, stream_of(dev)),
           "attention_with_lse");
}

std::vector<Tensor> merge(at::TensorList outs_in, at::TensorList lses, bool pairwise,
                          c10::optional<at::ScalarType> out_dtype) {
  TORCH_CHECK_VALUE(!outs_in.empty() && outs_in.size() == lses.size(),
                    "need the same positive number of outputs and lses");
  const at::Device dev = device_of({}, outs_in);
  on_device(dev, lses);
  std::vector<Tensor> outs;
  for (const Tensor& o : outs_in) outs.push_back(inner(o));
  const Tensor& o0 = outs[0];
  Tensor out = at::empty(o0.sizes(), o0.options().dtype(out_dtype ? *out_dtype : o0.scalar_type()));
  Tensor lse = at::empty(lses[0].sizes(), lses[0].options());
  c10::DeviceGuard guard(dev);
  std::vector<cea_tensor> oa = args(outs), la = args(lses);
  cea_tensor o = arg(out), l = arg(lse);
  if (pairwise && outs.size() == 2)
    check_rc(cea_merge_attention(&oa[0], &la[0], &oa[1], &la[1], &o, &l, stream_of(dev)), "merge_attention");
  else
    check_rc(cea_merge_attention_list((int32_t)outs.size(), oa.data(), la.data(), &o, &l, stream_of(dev)),
             "merge_attention_list");
  return {out, lse};
}

std::vector<Tensor> partitioned(const Tensor& q_in, const Tensor& q_pos_in, at::TensorList ks_in,
                                at::TensorList vs_in, at::TensorList ps_in, bool causal, double scale,
                                c10::optional<at::IntArrayRef> kv_map, at::ScalarType out_dtype,
                                bool with_lse, bool with_parts) {
  const int64_t n = (int64_t)ks_in.size();
  TORCH_CHECK_VALUE(n >= 1 && (int64_t)vs_in.size() == n && (int64_t)ps_in.size() == n,
                    "need one k, v and position tensor per partition");
  const at::Device dev = device_of({&q_in, &q_pos_in}, ks_in);
  on_device(dev, vs_in);
  on_device(dev, ps_in);
  const Tensor q = inner(q_in), qp = as_i64(q_pos_in);
  std::vector<Tensor> ks, vs, ps;
  for (int64_t i = 0; i < n; ++i) {
    ks.push_back(inner(ks_in[i]));
    vs.push_back(inner(vs_in[i]));
    ps.push_back(as_i64(ps_in[i]));
  }
  const int64_t B = q.size(0), Sq = q.size(1), Hq = q.size(2), D = q.size(3);
  const at::ScalarType acc = acc_of(q.scalar_type());
  const auto opts = q.options();
  Tensor out = at::empty({B, Sq, Hq, D}, opts.dtype(out_dtype));
  Tensor lse = with_lse ? at::empty({B, Hq, Sq}, opts.dtype(acc)) : Tensor();
  std::vector<Tensor> pouts, plses;
  if (with_parts)
    for (int64_t i = 0; i < n; ++i) {
      pouts.push_back(at::empty({B, Sq, Hq, D}, opts.dtype(acc)));
      plses.push_back(at::empty({B, Hq, Sq}, opts.dtype(acc)));
    }
  c10::DeviceGuard guard(dev);
  std::vector<int64_t> sks;
  for (const Tensor& k : ks) sks.push_back(k.size(1));
  const size_t ws_bytes = cea_partitioned_attention_workspace_bytes(
      (int32_t)n, sks.data(), B, Sq, Hq, ks[0].size(2), D, code_of(q.scalar_type()));
  const Scratch ws = workspace(ws_bytes);
  const std::vector<int32_t> m = map_of(kv_map);
  cea_tensor qa = arg(q), qpa = arg(qp), o = arg(out);
  cea_tensor l = with_lse ? arg(lse) : cea_tensor{};
  std::vector<cea_tensor> ka = args(ks), va = args(vs), pa = args(ps);
  std::vector<cea_tensor> poa = args(pouts), pla = args(plses);
  check_rc(cea_partitioned_attention(&qa, (int32_t)n, ka.data(), va.data(), &qpa, pa.data(), causal ? 1 : 0,
                                     scale, m.empty() ? nullptr : m.data(), (int32_t)m.size(),
                                     with_parts ? poa.data() : nullptr, with_parts ? pla.data() : nullptr, &o,
                                     with_lse ? &l : nullptr, ws.data(), ws.size, stream_of(dev)),
           "partitioned_attention");
  std::vector<Tensor> res{out};
  if (with_lse) res.push_back(lse);
  for (int64_t i = 0; i < (int64_t)pouts.size(); ++i) {
    res.push_back(pouts[i]);
    res.push_back(plses[i]);
  }
  return res;
}

// One rank's share of ring attention over KV blocks in ring order (cea_ring_attention).
std::vector<Tensor> ring(const Tensor& q_in, const Tensor& q_pos_in, at::TensorList ks_in,
                         at::TensorList vs_in, at::TensorList ps_in, bool causal, double scale,
                         c10::optional<at::IntArrayRef> kv_map, bool with_lse) {
  const int64_t n = (int64_t)ks_in.size();
  TORCH_CHECK_VALUE(n >= 1 && (int64_t)vs_in.size() == n && (int64_t)ps_in.size() == n,
                    "need one k, v and position tensor per KV block");
  const at::Device dev = device_of({&q_in, &q_pos_in}, ks_in);
  on_device(dev, vs_in);
  on_device(dev, ps_in);
  const Tensor q = inner(q_in), qp = as_i64(q_pos_in);
  TORCH_CHECK_VALUE(q.dim() == 4, "q must be [B, S, H, D]");
  std::vector<Tensor> ks, vs, ps;
  for (int64_t i = 0; i < n; ++i) {
    ks.push_back(inner(ks_in[i]));
    vs.push_back(inner(vs_in[i]));
    ps.push_back(as_i64(ps_in[i]));
  }
  const int64_t B = q.size(0), Sq = q.size(1), Hq = q.size(2), D = q.size(3);
  const at::ScalarType acc = acc_of(q.scalar_type());
  const auto opts = q.options();
  Tensor out = at::empty({B, Sq, Hq, D}, opts.dtype(with_lse ? acc : q.scalar_type()));
  Tensor lse = with_lse ? at::empty({B, Hq, Sq}, opts.dtype(acc)) : Tensor();
  c10::DeviceGuard guard(dev);
  const std::vector<int32_t> m = map_of(kv_map);
  cea_tensor qa = arg(q), qpa = arg(qp), o = arg(out);
  cea_tensor l = with_lse ? arg(lse) : cea_tensor{};
  std::vector<cea_tensor> ka = args(ks), va = args(vs), pa = args(ps);
  const size_t ws_bytes = cea_ring_attention_workspace_bytes(
      &qa, (int32_t)n, ka.data(), va.data(), &qpa, pa.data(), causal ? 1 : 0,
      m.empty() ? nullptr : m.data(), (int32_t)m.size(), &o, with_lse ? &l : nullptr);
  const Scratch ws = workspace(ws_bytes);
  check_rc(cea_ring_attention(&qa, (int32_t)n, ka.data(), va.data(), &qpa, pa.data(), causal ? 1 : 0, scale,
                              m.empty() ? nullptr : m.data(), (int32_t)m.size(), &o,
                              with_lse ? &l : nullptr, ws.data(), ws.size, stream_of(dev)),
           "ring_attention");
  if (with_lse) return {out, lse};
  return {out};
}

// ---------------------------------------------------------------------------------------
// wire formats
// ---------------------------------------------------------------------------------------
void pack_partial(const Tensor& out_in, const Tensor& lse, Tensor packed) {
  const at::Device dev = device_of({&out_in, &lse, &packed});
  const Tensor out = inner(out_in);
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(out), l = arg(lse), p = arg(packed);
  check_rc(cea_pack_partial(&a, &l, &p, stream_of(dev)), "pack_partial");
}

std::vector<Tensor> merge_packed(at::TensorList parts_in, at::ScalarType out_dtype, bool with_lse) {
  TORCH_CHECK_VALUE(!parts_in.empty(), "need at least one packed partial");
  const at::Device dev = device_of({}, parts_in);
  std::vector<Tensor> parts;
  for (const Tensor& p : parts_in) parts.push_back(inner(p));
  const Tensor& p0 = parts[0];
  TORCH_CHECK_VALUE(p0.dim() == 4, "packed partials must be [B, Sq, H, D+1]");
  const int64_t B = p0.size(0), Sq = p0.size(1), H = p0.size(2), D1 = p0.size(3);
  Tensor out = at::empty({B, Sq, H, D1 - 1}, p0.options().dtype(out_dtype));
  Tensor lse = with_lse ? at::empty({B, H, Sq}, p0.options()) : Tensor();
  c10::DeviceGuard guard(dev);
  std::vector<cea_tensor> pa = args(parts);
  cea_tensor o = arg(out), l = with_lse ? arg(lse) : cea_tensor{};
  check_rc(cea_merge_packed((int32_t)parts.size(), pa.data(), &o, with_lse ? &l : nullptr, stream_of(dev)),
           "merge_packed");
  if (with_lse) return {out, lse};
  return {out};
}

std::vector<Tensor> ulysses_scatter(at::TensorList qs, at::TensorList ks, at::TensorList vs,
                                    at::TensorList ps, int64_t q_start, int64_t q_count, int64_t kv_start,
                                    int64_t kv_count) {
  const int64_t n = (int64_t)qs.size();
  TORCH_CHECK_VALUE(n >= 1 && (int64_t)ks.size() == n && (int64_t)vs.size() == n && (int64_t)ps.size() == n,
                    "need one q, k, v and position shard per rank");
  const at::Device dev = device_of({}, qs);
  on_device(dev, ks);
  on_device(dev, vs);
  on_device(dev, ps);
  std::vector<Tensor> pl;
  for (const Tensor& p : ps) pl.push_back(as_i64(p));
  int64_t S = 0;
  for (const Tensor& q : qs) S += q.size(1);
  const Tensor& q0 = qs[0];
  Tensor full = at::empty({q0.size(0), S, q_count + 2 * kv_count, q0.size(3)}, q0.options());
  Tensor pos_f = at::empty({q0.size(0), S}, q0.options().dtype(at::kLong));
  c10::DeviceGuard guard(dev);
  std::vector<cea_tensor> qa = args(qs), ka = args(ks), va = args(vs), pa = args(pl);
  cea_tensor f = arg(full), pf = arg(pos_f);
  check_rc(cea_ulysses_scatter((int32_t)n, qa.data(), ka.data(), va.data(), pa.data(), (int32_t)q_start,
                               (int32_t)q_count, (int32_t)kv_start, (int32_t)kv_count, &f, &pf, stream_of(dev)),
           "ulysses_scatter");
  return {full, pos_f};
}

Tensor ulysses_gather(at::TensorList outs, int64_t start, int64_t length) {
  TORCH_CHECK_VALUE(!outs.empty(), "need one head output per rank");
  const at::Device dev = device_of({}, outs);
  const Tensor& o0 = outs[0];
  int64_t H = 0;
  for (const Tensor& o : outs) H += o.size(2);
  Tensor res = at::empty({o0.size(0), length, H, o0.size(3)}, o0.options());
  c10::DeviceGuard guard(dev);
  std::vector<cea_tensor> oa = args(outs);
  cea_tensor r = arg(res);
  check_rc(cea_ulysses_gather((int32_t)outs.size(), oa.data(), start, &r, stream_of(dev)), "ulysses_gather");
  return res;
}

// ---------------------------------------------------------------------------------------
// layer ops
// ---------------------------------------------------------------------------------------
Tensor rmsnorm(const Tensor& x, const Tensor& weight_in, double eps) {
  const at::Device dev = device_of({&x, &weight_in});
  const Tensor w = inner(weight_in);
  Tensor y = at::empty(x.sizes(), x.options().dtype(at::promote_types(w.scalar_type(), x.scalar_type())));
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(x), b = arg(w), c = arg(y);
  check_rc(cea_rmsnorm(&a, &b, eps, &c, stream_of(dev)), "rmsnorm");
  return y;
}

// rmsnorm over the last dimension of x [..., C]: rows as a view (a copy only when the leading
// dimensions do not collapse), the result in x's shape.
Tensor rmsnorm_nd(const Tensor& x, const Tensor& weight, double eps) {
  TORCH_CHECK_INDEX(x.dim() >= 1, "rmsnorm: x must have at least one dimension");
  const Tensor rows = inner(x);
  return rmsnorm(rows.reshape({-1, rows.size(-1)}), weight, eps).view(x.sizes());
}

std::vector<Tensor> rope_tables(const Tensor& pos_in, const Tensor& inv, at::ScalarType dtype) {
  const at::Device dev = device_of({&pos_in, &inv});
  const Tensor pos = as_i64(pos_in);
  TORCH_CHECK_VALUE(pos.dim() == 2 && inv.dim() == 1, "positions must be [B, S] and inv_freq [D/2]");
  const auto opts = inv.options().dtype(dtype);
  Tensor cos = at::empty({pos.size(0), pos.size(1), 2 * inv.size(0)}, opts);
  Tensor sin = at::empty({pos.size(0), pos.size(1), 2 * inv.size(0)}, opts);
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(pos), b = arg(inv), c = arg(cos), d = arg(sin);
  check_rc(cea_rope_tables(&a, &b, &c, &d, stream_of(dev)), "rope_tables");
  return {cos, sin};
}

Tensor apply_rotary(const Tensor& x_in, const Tensor& cos_in, const Tensor& sin_in) {
  const at::Device dev = device_of({&x_in, &cos_in, &sin_in});
  const Tensor x = inner(x_in), cos = inner(cos_in), sin = inner(sin_in);
  Tensor out = at::empty(x.sizes(), x.options());
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(x), b = arg(cos), c = arg(sin), d = arg(out);
  check_rc(cea_apply_rotary(&a, &b, &c, &d, stream_of(dev)), "apply_rotary");
  return out;
}

Tensor rmsnorm_rope(const Tensor& x, const Tensor& weight, double eps, const Tensor& pos_in, const Tensor& inv,
                    int64_t num_heads) {
  const at::Device dev = device_of({&x, &weight, &pos_in, &inv});
  const Tensor pos = as_i64(pos_in);
  Tensor out = at::empty(x.sizes(), x.options());
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(x), b = arg(weight), c = arg(pos), d = arg(inv), e = arg(out);
  check_rc(cea_rmsnorm_rope(&a, &b, eps, &c, &d, (int32_t)num_heads, &e, stream_of(dev)), "rmsnorm_rope");
  return out;
}

Tensor gated_mul(const Tensor& gate, const Tensor& up, int64_t act) {
  const at::Device dev = device_of({&gate, &up});
  Tensor out = at::empty(gate.sizes(), gate.options());
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(gate), b = arg(up), c = arg(out);
  check_rc(cea_gated_mul(&a, &b, &c, (int32_t)act, stream_of(dev)), "gated_mul");
  return out;
}

// x [..., K] as a 2-D [M, K] view (a copy only when the leading dimensions do not collapse)
Tensor rows_of(const Tensor& x) {
  TORCH_CHECK_VALUE(x.dim() >= 1, "x must have at least one dimension");
  int64_t rows = 1;
  for (int64_t i = 0; i + 1 < x.dim(); ++i) rows *= x.size(i);
  return inner(x.reshape({rows, x.size(-1)}));
}

std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = n;
  return s;
}

// The scratch of a projection to n columns (null when it needs none).
Scratch linear_workspace(const Tensor& x2, int64_t n, int gated) {
  const size_t bytes =
      cea_linear_workspace_bytes(x2.size(0), n, x2.size(1), code_of(x2.scalar_type()), gated);
  return bytes ? workspace(bytes) : Scratch();
}

void linear_call(const Tensor& x2, const Tensor& weight, const c10::optional<Tensor>& bias,
                 const Tensor& y2, const at::Device& dev) {
  const Tensor w = inner(weight);
  const Tensor b = bias ? inner(*bias) : Tensor();
  c10::DeviceGuard guard(dev);
  const Scratch ws = linear_workspace(x2, w.size(0), 0);
  cea_tensor a = arg(x2), c = arg(w), d, e = arg(y2);
  if (b.defined()) d = arg(b);
  check_rc(cea_linear_ws(&a, &c, b.defined() ? &d : nullptr, &e, ws.data(), ws.size, stream_of(dev)),
           "linear");
}

Tensor linear(const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias) {
  const Tensor bd = bias ? *bias : Tensor();
  const at::Device dev = device_of({&x, &weight, &bd});
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [out_features, in_features]");
  const Tensor x2 = rows_of(x);
  Tensor y = at::empty(out_shape(x, weight.size(0)), x.options());
  linear_call(x2, weight, bias, y.view({x2.size(0), weight.size(0)}), dev);
  return y;
}

// y: a preallocated [M, N] buffer (any row stride, innermost stride 1)
void linear_into(Tensor y, const Tensor& x, const Tensor& weight, const c10::optional<Tensor>& bias) {
  const Tensor bd = bias ? *bias : Tensor();
  const at::Device dev = device_of({&y, &x, &weight, &bd});
  TORCH_CHECK_VALUE(weight.dim() == 2, "weight must be [out_features, in_features]");
  TORCH_CHECK_VALUE(y.dim() == 2, "out must be 2-D [rows, out_features]");
  TORCH_CHECK_VALUE(y.size(-1) <= 1 || y.stride(-1) == 1, "out must have innermost stride 1");
  linear_call(rows_of(x), weight, bias, y, dev);
}

Tensor linear_gated(const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                    const c10::optional<Tensor>& b_gate, const c10::optional<Tensor>& b_up, int64_t act) {
  const Tensor bg = b_gate ? inner(*b_gate) : Tensor(), bu = b_up ? inner(*b_up) : Tensor();
  const at::Device dev = device_of({&x, &w_gate, &w_up, &bg, &bu});
  TORCH_CHECK_VALUE(w_gate.dim() == 2 && w_up.dim() == 2, "weights must be [units, in_features]");
  const Tensor x2 = rows_of(x);
  Tensor wg = inner(w_gate), wu = inner(w_up);
  if (wg.size(0) > 1 && wu.stride(0) != wg.stride(0)) {
    wg = wg.contiguous();
    wu = wu.contiguous();
  }
  Tensor y = at::empty(out_shape(x, w_gate.size(0)), x.options());
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(x2), c = arg(wg), d = arg(wu), e = arg(y.view({x2.size(0), w_gate.size(0)}));
  cea_tensor f, g;
  if (bg.defined()) f = arg(bg);
  if (bu.defined()) g = arg(bu);
  const Scratch ws = linear_workspace(x2, w_gate.size(0), 1);
  check_rc(cea_linear_gated_ws(&a, &c, &d, bg.defined() ? &f : nullptr, bu.defined() ? &g : nullptr, &e,
                               (int32_t)act, ws.data(), ws.size,
                               stream_of(dev)),
           "linear_gated");
  return y;
}

void kv_append(Tensor cache_k, Tensor cache_v, Tensor cache_pos, int64_t offset, const Tensor& k_in,
               const Tensor& v_in, const Tensor& pos_in, c10::optional<Tensor> cos_in,
               c10::optional<Tensor> sin_in) {
  TORCH_CHECK_VALUE(cos_in.has_value() == sin_in.has_value(), "give both rotary tables or neither");
  const Tensor cosd = cos_in ? *cos_in : Tensor(), sind = sin_in ? *sin_in : Tensor();
  const at::Device dev = device_of({&cache_k, &cache_v, &cache_pos, &k_in, &v_in, &pos_in, &cosd, &sind});
  const Tensor k = inner(k_in), v = inner(v_in), pos = as_i64(pos_in);
  c10::DeviceGuard guard(dev);
  cea_tensor a = arg(k), b = arg(v), c = arg(pos), ck = arg(cache_k), cv = arg(cache_v), cp = arg(cache_pos);
  if (cosd.defined()) {
    const Tensor cs = inner(cosd.to(k.scalar_type())), sn = inner(sind.to(k.scalar_type()));
    cea_tensor tc = arg(cs), ts = arg(sn);
    check_rc(cea_kv_append(&a, &b, &c, &tc, &ts, &ck, &cv, &cp, offset, stream_of(dev)), "kv_append");
  } else {
    check_rc(cea_kv_append(&a, &b, &c, nullptr, nullptr, &ck, &cv, &cp, offset, stream_of(dev)), "kv_append");
  }
}

// ---------------------------------------------------------------------------------------
// paged KV cache
// ---------------------------------------------------------------------------------------
Tensor given(const c10::optional<Tensor>& t) { return t ? *t : Tensor(); }

// Caches are written and read in place, so their layout is the caller's: no copies are made.
void check_pools(const Tensor& k_pages, const Tensor& v_pages) {
  TORCH_CHECK_VALUE(k_pages.dim() == 4 && v_pages.dim() == 4, "k_pages and v_pages must be [P, H, page, D]");
}

// Pages of 8 bits come with both scales, others with neither.
bool bytes8(const Tensor& k_pages, const Tensor& v_pages, const Tensor& ks, const Tensor& vs) {
  const bool f8 = k_pages.scalar_type() == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(f8 == (v_pages.scalar_type() == at::kFloat8_e4m3fn), "k_pages and v_pages must share one dtype");
  TORCH_CHECK_VALUE(ks.defined() == f8 && vs.defined() == f8,
                    "k_scales and v_scales go with float8_e4m3fn pages, both of them");
  return f8;
}

// Arguments of a C call: a tensor that is not given is a null pointer.
template <size_t N> struct Args {
  cea_tensor a[N];
  cea_tensor* p[N];
  explicit Args(const Tensor* const (&t)[N]) {
    for (size_t i = 0; i < N; ++i) {
      p[i] = nullptr;
      if (t[i]->defined()) a[i] = arg(*t[i], true), p[i] = &a[i];
    }
  }
  cea_tensor* operator[](size_t i) const { return p[i]; }
};

void paged_kv_append(Tensor k_pages, Tensor v_pages, const c10::optional<Tensor>& pos_pages_in,
                     const Tensor& tables_in, const Tensor& offsets_in, const c10::optional<Tensor>& counts_in,
                     const Tensor& k_in, const Tensor& v_in, const c10::optional<Tensor>& pos_in,
                     const c10::optional<Tensor>& cos_in, const c10::optional<Tensor>& sin_in,
                     const c10::optional<Tensor>& k_scales_in, const c10::optional<Tensor>& v_scales_in) {
  const Tensor pp = given(pos_pages_in), counts0 = given(counts_in), pos0 = given(pos_in);
  const Tensor cos0 = given(cos_in), sin0 = given(sin_in), ks = given(k_scales_in), vs = given(v_scales_in);
  const at::Device dev = device_of({&k_pages, &v_pages, &ks, &vs, &pp, &tables_in, &offsets_in, &counts0, &k_in, &v_in,
                                    &pos0, &cos0, &sin0});
  check_pools(k_pages, v_pages);
  const bool f8 = bytes8(k_pages, v_pages, ks, vs);
  TORCH_CHECK_VALUE(cos0.defined() == sin0.defined(), "give both rotary tables or neither");
  c10::DeviceGuard guard(dev);
  const Tensor k = inner(k_in), v = inner(v_in), tables = as_i64(tables_in), offsets = as_i64(offsets_in);
  const Tensor counts = counts0.defined() ? as_i64(counts0) : counts0, pos = pos0.defined() ? as_i64(pos0) : pos0;
  const Tensor cos = cos0.defined() ? inner(cos0.to(k.scalar_type())) : cos0;
  const Tensor sin = sin0.defined() ? inner(sin0.to(k.scalar_type())) : sin0;
  const Args<13> p({&k, &v, &pos, &cos, &sin, &tables, &offsets, &counts, &k_pages, &v_pages, &ks, &vs, &pp});
  check_rc(f8 ? cea_paged_kv_append8(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[10], p[11], p[12],
                                     stream_of(dev))
              : cea_paged_kv_append(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[12], stream_of(dev)),
           "paged_kv_append");
}

std::vector<Tensor> paged_kv_read(const Tensor& k_pages, const Tensor& v_pages, const c10::optional<Tensor>& k_scales_in,
                                  const c10::optional<Tensor>& v_scales_in, const Tensor& tables_in,
                                  const Tensor& offsets_in, const c10::optional<Tensor>& counts_in, int64_t n,
                                  at::ScalarType dtype) {
  const Tensor ks = given(k_scales_in), vs = given(v_scales_in), counts0 = given(counts_in);
  const at::Device dev = device_of({&k_pages, &v_pages, &ks, &vs, &tables_in, &offsets_in, &counts0});
  check_pools(k_pages, v_pages);
  const bool f8 = bytes8(k_pages, v_pages, ks, vs);
  TORCH_CHECK_VALUE(n >= 0, "n must not be negative");
  TORCH_CHECK_VALUE(tables_in.dim() == 2, "tables must be [B, W]");
  TORCH_CHECK_VALUE(f8 || dtype == k_pages.scalar_type(), "pages of ", k_pages.scalar_type(),
                    " are read in their own dtype");
  c10::DeviceGuard guard(dev);
  const Tensor tables = as_i64(tables_in), offsets = as_i64(offsets_in);
  const Tensor counts = counts0.defined() ? as_i64(counts0) : counts0;
  const auto opts = at::TensorOptions().device(dev).dtype(dtype);
  Tensor k = at::empty({tables.size(0), n, k_pages.size(1), k_pages.size(3)}, opts), v = at::empty_like(k);
  const Args<9> p({&k_pages, &v_pages, &ks, &vs, &tables, &offsets, &counts, &k, &v});
  check_rc(cea_paged_kv_read(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], stream_of(dev)), "paged_kv_read");
  return {k, v};
}

// Outputs of an attention call, and the call with the scratch it asks for.
template <typename Sizes, typename Call>
std::vector<Tensor> attend(const Tensor& q, bool with_lse, const at::Device& dev, const char* what, Sizes sizes,
                           Call call) {
  const at::ScalarType acc = acc_of(q.scalar_type());
  const auto o_opts = at::TensorOptions().device(dev).dtype(with_lse ? acc : q.scalar_type());
  Tensor out = at::empty(q.sizes(), o_opts);
  Tensor lse = with_lse ? at::empty({q.size(0), q.size(2), q.size(1)}, o_opts.dtype(acc)) : Tensor();
  cea_tensor o = arg(out), l;
  if (with_lse) l = arg(lse);
  cea_tensor* lp = with_lse ? &l : nullptr;
  size_t bytes = 0;
  check_rc(sizes(&o, lp, &bytes), what);
  const Scratch ws = bytes ? workspace(bytes) : Scratch();
  check_rc(call(&o, lp, ws.data(), ws.size), what);
  if (with_lse) return {out, lse};
  return {out};
}

std::vector<Tensor> paged_attention(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages,
                                    const c10::optional<Tensor>& pos_pages_in, const Tensor& tables_in,
                                    const Tensor& lengths_in, const Tensor& q_pos_in, bool causal, double scale,
                                    c10::optional<at::IntArrayRef> kv_map, bool with_lse,
                                    const c10::optional<Tensor>& k_scales_in,
                                    const c10::optional<Tensor>& v_scales_in) {
  const Tensor pp = given(pos_pages_in), ks = given(k_scales_in), vs = given(v_scales_in);
  const at::Device dev = device_of({&q_in, &k_pages, &v_pages, &ks, &vs, &pp, &tables_in, &lengths_in, &q_pos_in});
  check_pools(k_pages, v_pages);
  const bool f8 = bytes8(k_pages, v_pages, ks, vs);
  TORCH_CHECK_VALUE(q_in.dim() == 4, "q must be [B, S, H, D]");
  TORCH_CHECK_VALUE(tables_in.dim() == 2, "tables must be [B, W]");
  c10::DeviceGuard guard(dev);
  const Tensor q = inner(q_in), tables = as_i64(tables_in), lengths = as_i64(lengths_in), qp = as_i64(q_pos_in);
  const std::vector<int32_t> m = map_of(kv_map);
  const int32_t* map = m.empty() ? nullptr : m.data();
  const int32_t len = (int32_t)m.size(), c = causal ? 1 : 0;
  const Args<9> p({&q, &k_pages, &v_pages, &pp, &tables, &lengths, &qp, &ks, &vs});
  return attend(
      q, with_lse, dev, "paged_attention",
      [&](cea_tensor* o, cea_tensor* l, size_t* bytes) {
        return f8 ? cea_paged_attention8_workspace(p[0], p[1], p[2], p[7], p[8], p[3], p[4], p[5], p[6], c, scale, map,
                                                   len, o, l, bytes)
                  : cea_paged_attention_workspace(p[0], p[1], p[2], p[3], p[4], p[5], p[6], c, scale, map, len, o, l,
                                                  bytes);
      },
      [&](cea_tensor* o, cea_tensor* l, void* ws, size_t size) {
        return f8 ? cea_paged_attention8(p[0], p[1], p[2], p[7], p[8], p[3], p[4], p[5], p[6], c, scale, map, len, o, l,
                                         ws, size, stream_of(dev))
                  : cea_paged_attention(p[0], p[1], p[2], p[3], p[4], p[5], p[6], c, scale, map, len, o, l, ws, size,
                                        stream_of(dev));
      });
}

std::vector<Tensor> paged_tree_attention(const Tensor& q_in, const Tensor& k_pages, const Tensor& v_pages,
                                         const c10::optional<Tensor>& k_scales_in,
                                         const c10::optional<Tensor>& v_scales_in, const Tensor& tables_in,
                                         const Tensor& lengths_in, const Tensor& counts_in, const Tensor& masks_in,
                                         double scale, c10::optional<at::IntArrayRef> kv_map, bool with_lse) {
  const Tensor ks = given(k_scales_in), vs = given(v_scales_in);
  const at::Device dev =
      device_of({&q_in, &k_pages, &v_pages, &ks, &vs, &tables_in, &lengths_in, &counts_in, &masks_in});
  check_pools(k_pages, v_pages);
  bytes8(k_pages, v_pages, ks, vs);
  TORCH_CHECK_VALUE(q_in.dim() == 4, "q must be [B, T, H, D]");
  TORCH_CHECK_VALUE(masks_in.scalar_type() == at::kLong, "masks must be int64 words");
  c10::DeviceGuard guard(dev);
  const Tensor q = inner(q_in), tables = as_i64(tables_in), lengths = as_i64(lengths_in), counts = as_i64(counts_in);
  const std::vector<int32_t> m = map_of(kv_map);
  const int32_t* map = m.empty() ? nullptr : m.data();
  const int32_t len = (int32_t)m.size();
  const Args<9> p({&q, &k_pages, &v_pages, &ks, &vs, &tables, &lengths, &counts, &masks_in});
  return attend(
      q, with_lse, dev, "paged_tree_attention",
      [&](cea_tensor* o, cea_tensor* l, size_t* bytes) {
        return cea_paged_tree_attention_workspace(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], scale, map, len,
                                                  o, l, bytes);
      },
      [&](cea_tensor* o, cea_tensor* l, void* ws, size_t size) {
        return cea_paged_tree_attention(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], scale, map, len, o, l, ws,
                                        size, stream_of(dev));
      });
}

std::vector<Tensor> tree_masks(const Tensor& parents_in, const c10::optional<Tensor>& counts_in) {
  const Tensor counts0 = given(counts_in);
  const at::Device dev = device_of({&parents_in, &counts0});
  TORCH_CHECK_VALUE(parents_in.dim() == 2, "parents must be [B, T]");
  c10::DeviceGuard guard(dev);
  const Tensor parents = as_i64(parents_in), counts = counts0.defined() ? as_i64(counts0) : counts0;
  const int64_t B = parents.size(0), T = parents.size(1);
  const auto opts = at::TensorOptions().device(dev).dtype(at::kLong);
  Tensor masks = at::empty({B, T, (T + 63) / 64}, opts), depths = at::empty({B, T}, opts);
  const Args<4> p({&parents, &counts, &masks, &depths});
  check_rc(cea_tree_masks(p[0], p[1], p[2], p[3], stream_of(dev)), "tree_masks");
  return {masks, depths};
}

// The pools of all layers as [N, P, H, page * D] (scales: [N, P, H, page]): the dimensions before the pages
// have to collapse into one.
cea_tensor pools_arg(const Tensor& t, int64_t rest, const char* what) {
  cea_tensor a;
  a.dtype = page_code_of(t.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(a.dtype >= 0, "dtype ", t.scalar_type(), " is not supported by the kernels");
  const int64_t lead = t.dim() - rest;
  int64_t n = 1, stride = 0;
  for (int64_t i = lead - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    TORCH_CHECK_VALUE(n == 1 || t.stride(i) == stride * n || t.numel() == 0,
                      "paged_kv_keep: the dimensions of ", what, " before the pages must collapse");
    if (n == 1) stride = t.stride(i);
    n *= t.size(i);
  }
  a.data = t.numel() > 0 ? t.data_ptr() : nullptr;
  a.ndim = 4;
  a.size[0] = n, a.stride[0] = stride;
  for (int i = 0; i < 3; ++i) a.size[1 + i] = t.size(lead + i), a.stride[1 + i] = t.stride(lead + i);
  return a;
}

void paged_kv_keep(Tensor kv, const c10::optional<Tensor>& scales_in, const Tensor& tables_in, const Tensor& offsets_in,
                   const c10::optional<Tensor>& counts_in, const Tensor& path_in) {
  const Tensor scales = given(scales_in), counts0 = given(counts_in);
  const at::Device dev = device_of({&kv, &scales, &tables_in, &offsets_in, &counts0, &path_in});
  TORCH_CHECK_VALUE(kv.dim() >= 4, "kv must be [..., P, H, page, D]");
  TORCH_CHECK_VALUE(!scales.defined() || scales.dim() == kv.dim() - 1, "scales must be [..., P, H, page]");
  TORCH_CHECK_VALUE(scales.defined() == (kv.scalar_type() == at::kFloat8_e4m3fn),
                    "scales go with float8_e4m3fn pages");
  const int64_t page = kv.size(-2), D = kv.size(-1);
  TORCH_CHECK_VALUE(kv.numel() == 0 || ((D == 1 || kv.stride(-1) == 1) && (page == 1 || kv.stride(-2) == D)),
                    "paged_kv_keep: a head's slots of a page must be contiguous");
  c10::DeviceGuard guard(dev);
  const Tensor tables = as_i64(tables_in), offsets = as_i64(offsets_in), path = as_i64(path_in);
  const Tensor counts = counts0.defined() ? as_i64(counts0) : counts0;
  cea_tensor a = pools_arg(kv, 4, "kv"), sc;
  a.size[3] = page * D, a.stride[3] = 1;
  if (scales.defined()) sc = pools_arg(scales, 3, "scales");
  const Args<4> p({&tables, &offsets, &counts, &path});
  check_rc(cea_paged_kv_keep(&a, scales.defined() ? &sc : nullptr, (int32_t)page, p[0], p[1], p[2], p[3], stream_of(dev)),
           "paged_kv_keep");
}

// A pool tensor with its page dimension `dim` as [N, P, E]: the dimensions before it have to
// collapse into one, those after it to be contiguous (they are copied as bytes).
cea_tensor pool_arg(const Tensor& t, int64_t dim) {
  cea_tensor a;
  a.dtype = page_code_of(t.scalar_type());
  TORCH_CHECK_NOT_IMPLEMENTED(a.dtype >= 0, "dtype ", t.scalar_type(), " is not supported by the kernels");
  TORCH_CHECK_VALUE(dim >= 0 && dim < t.dim(), "copy_pages: a pool of ", t.dim(), " dimensions has no dimension ",
                    dim);
  int64_t e = 1, n = 1, stride = 0;
  for (int64_t i = t.dim() - 1; i > dim; --i) {
    TORCH_CHECK_VALUE(t.size(i) == 1 || t.stride(i) == e || t.numel() == 0, "copy_pages: a page must be contiguous");
    e *= t.size(i);
  }
  for (int64_t i = dim - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    TORCH_CHECK_VALUE(n == 1 || t.stride(i) == stride * n || t.numel() == 0,
                      "copy_pages: the dimensions before the pages must collapse");
    if (n == 1) stride = t.stride(i);
    n *= t.size(i);
  }
  a.data = t.numel() > 0 ? t.data_ptr() : nullptr;
  a.ndim = 3;
  for (int i = 0; i < CEA_MAX_DIMS; ++i) a.size[i] = a.stride[i] = 0;
  a.size[0] = n, a.size[1] = t.size(dim), a.size[2] = e;
  a.stride[0] = stride, a.stride[1] = t.stride(dim), a.stride[2] = 1;
  return a;
}

void copy_pages(at::TensorList pools, int64_t dim, const Tensor& src_in, const Tensor& dst_in) {
  TORCH_CHECK_VALUE(!pools.empty(), "copy_pages: need at least one pool");
  TORCH_CHECK_VALUE(src_in.device().is_cpu() && dst_in.device().is_cpu() && src_in.dim() == 1 && dst_in.dim() == 1 &&
                        src_in.size(0) == dst_in.size(0),
                    "copy_pages: src and dst must be host lists of the same length");
  TORCH_CHECK_VALUE(at::isIntegralType(src_in.scalar_type(), false) && at::isIntegralType(dst_in.scalar_type(), false),
                    "copy_pages: page indices must be whole numbers");
  const at::Device dev = device_of({}, pools);
  const Tensor src = as_i64(src_in).contiguous(), dst = as_i64(dst_in).contiguous();
  std::vector<cea_tensor> a;
  a.reserve(pools.size());
  for (const Tensor& t : pools) a.push_back(pool_arg(t, dim));
  c10::DeviceGuard guard(dev);
  check_rc(cea_copy_pages((int32_t)a.size(), a.data(), src.data_ptr<int64_t>(), dst.data_ptr<int64_t>(), src.numel(),
                          stream_of(dev)),
           "copy_pages");
}

}  // namespace

TORCH_LIBRARY(collab_edge, m) {
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor q_pos, Tensor k_pos, bool causal, float scale, "
        "int[]? kv_map, bool with_lse) -> Tensor[]");
  m.def("attention_into(Tensor(a!) out, Tensor(b!) lse, Tensor q, Tensor k, Tensor v, Tensor q_pos, "
        "Tensor k_pos, bool causal, float scale, int[]? kv_map, bool accumulate, Tensor(c!)? final) -> ()");
  m.def("merge(Tensor[] outs, Tensor[] lses, bool pairwise, ScalarType? out_dtype) -> Tensor[]");
  m.def("partitioned(Tensor q, Tensor q_pos, Tensor[] ks, Tensor[] vs, Tensor[] ps, bool causal, "
        "float scale, int[]? kv_map, ScalarType out_dtype, bool with_lse, bool with_parts) -> Tensor[]");
  m.def("ring(Tensor q, Tensor q_pos, Tensor[] ks, Tensor[] vs, Tensor[] ps, bool causal, float scale, "
        "int[]? kv_map, bool with_lse) -> Tensor[]");
  m.def("pack_partial(Tensor out, Tensor lse, Tensor(a!) packed) -> ()");
  m.def("merge_packed(Tensor[] parts, ScalarType out_dtype, bool with_lse) -> Tensor[]");
  m.def("ulysses_scatter(Tensor[] qs, Tensor[] ks, Tensor[] vs, Tensor[] ps, int q_start, int q_count, "
        "int kv_start, int kv_count) -> Tensor[]");
  m.def("ulysses_gather(Tensor[] outs, int start, int length) -> Tensor");
  m.def("rmsnorm(Tensor x, Tensor weight, float eps) -> Tensor");
  m.def("rmsnorm_nd(Tensor x, Tensor weight, float eps) -> Tensor");
  m.def("rope_tables(Tensor positions, Tensor inv_freq, ScalarType dtype) -> Tensor[]");
  m.def("apply_rotary(Tensor x, Tensor cos, Tensor sin) -> Tensor");
  m.def("rmsnorm_rope(Tensor x, Tensor weight, float eps, Tensor positions, Tensor inv_freq, int num_heads) "
        "-> Tensor");
  m.def("gated_mul(Tensor gate, Tensor up, int act) -> Tensor");
  m.def("linear(Tensor x, Tensor weight, Tensor? bias) -> Tensor");
  m.def("linear_into(Tensor(a!) out, Tensor x, Tensor weight, Tensor? bias) -> ()");
  m.def("linear_gated(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, int act) -> Tensor");
  m.def("kv_append(Tensor(a!) cache_k, Tensor(b!) cache_v, Tensor(c!) cache_pos, int offset, Tensor k, "
        "Tensor v, Tensor pos, Tensor? cos, Tensor? sin) -> ()");
  m.def("paged_kv_append(Tensor(a!) k_pages, Tensor(b!) v_pages, Tensor(c!)? pos_pages, Tensor tables, "
        "Tensor offsets, Tensor? counts, Tensor k, Tensor v, Tensor? pos, Tensor? cos, Tensor? sin, "
        "Tensor(d!)? k_scales=None, Tensor(e!)? v_scales=None) -> ()");
  m.def("paged_kv_read(Tensor k_pages, Tensor v_pages, Tensor? k_scales, Tensor? v_scales, Tensor tables, "
        "Tensor offsets, Tensor? counts, int n, ScalarType dtype) -> Tensor[]");
  m.def("paged_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? pos_pages, Tensor tables, "
        "Tensor lengths, Tensor q_pos, bool causal, float scale, int[]? kv_map, bool with_lse, "
        "Tensor? k_scales=None, Tensor? v_scales=None) -> Tensor[]");
  m.def("paged_tree_attention(Tensor q, Tensor k_pages, Tensor v_pages, Tensor? k_scales, Tensor? v_scales, "
        "Tensor tables, Tensor lengths, Tensor counts, Tensor masks, float scale, int[]? kv_map, bool with_lse) "
        "-> Tensor[]");
  m.def("tree_masks(Tensor parents, Tensor? counts) -> Tensor[]");
  m.def("paged_kv_keep(Tensor(a!) kv, Tensor(b!)? scales, Tensor tables, Tensor offsets, Tensor? counts, Tensor path) "
        "-> ()");
  m.def("copy_pages(Tensor(a!)[] pools, int dim, Tensor src, Tensor dst) -> ()");
}

TORCH_LIBRARY_IMPL(collab_edge, CompositeExplicitAutograd, m) {
  m.impl("attention", attention);
  m.impl("attention_into", attention_into);
  m.impl("merge", merge);
  m.impl("partitioned", partitioned);
  m.impl("ring", ring);
  m.impl("pack_partial", pack_partial);
  m.impl("merge_packed", merge_packed);
  m.impl("ulysses_scatter", ulysses_scatter);
  m.impl("ulysses_gather", ulysses_gather);
  m.impl("rmsnorm", rmsnorm);
  m.impl("rmsnorm_nd", rmsnorm_nd);
  m.impl("rope_tables", rope_tables);
  m.impl("apply_rotary", apply_rotary);
  m.impl("rmsnorm_rope", rmsnorm_rope);
  m.impl("gated_mul", gated_mul);
  m.impl("linear", linear);
  m.impl("linear_into", linear_into);
  m.impl("linear_gated", linear_gated);
  m.impl("kv_append", kv_append);
  m.impl("paged_kv_append", paged_kv_append);
  m.impl("paged_kv_read", paged_kv_read);
  m.impl("paged_attention", paged_attention);
  m.impl("paged_tree_attention", paged_tree_attention);
  m.impl("tree_masks", tree_masks);
  m.impl("paged_kv_keep", paged_kv_keep);
  m.impl("copy_pages", copy_pages);
}

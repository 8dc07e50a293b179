"""Seeded inputs of the paged KV cache's tests, their results in 64 bits, and error bounds.

Bounds, from the formula out = sum_j p_j v_j / sum_j p_j with p_j = exp(s_j - m) over the n keys that
a query sees, u = 2^-24 (half a step of f32) and t = half a step of the tensor's type:

* a score of D products summed in f32, scaled, moved by the maximum and put through exp, is off by
  at most d_j = u ((D + 4) |scale| sum |q_i k_ji| + 4 |s_j| + 8), which is p_j's relative error;
* sums of n terms in f32 add n u; a second or third 16-bit piece of p_j leaves less than 2^-16 of it
  (two bf16 pieces; three, or two of f16, leave less than u), one piece leaves t;
* so |out - exact| <= t' |exact| + (2 max d_j + 2 (n + 16) u + e_p) A,  A = sum p_j |v_j| / sum p_j,
  with t' half a step of the output's type, and e_p what the pieces leave;
* |lse - exact| <= max d_j + (n + 16) u + 4 u |exact|.

f64 uses u = 2^-53.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

U = {torch.float64: 2.0 ** -53}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(B=2, n=1, Hq=8, Hkv=2, D=128, page=16, lengths=(40, 5), dtype=torch.bfloat16, explicit=False,
         causal=True, scale=None, kv_map=None, seed=0, layout="hnd", spare=3, width=None, q_scale=1.0,
         stale=None, pad_rows=()):
    """A case on the CPU: pools whose unused slots hold `stale` values (random ones without it)."""
    g = torch.Generator().manual_seed(seed)
    lengths = list(lengths)
    W = width if width is not None else max([-(-x // page) for x in lengths] + [1])
    P = sum(-(-x // page) for x in lengths) + spare
    c = SimpleNamespace(B=B, n=n, Hq=Hq, Hkv=Hkv, D=D, page=page, dtype=dtype, causal=causal, P=P, W=W,
                        scale=1.0 / math.sqrt(D) if scale is None else scale, kv_map=kv_map)
    shape = (P, Hkv, page, D) if layout == "hnd" else (P, page, Hkv, D)
    c.k_pages = torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)
    c.v_pages = torch.randn(shape, generator=g, dtype=torch.float64).to(dtype)
    if layout != "hnd":
        c.k_pages, c.v_pages = c.k_pages.transpose(1, 2), c.v_pages.transpose(1, 2)
    c.q = (q_scale * torch.randn(B, n, Hq, D, generator=g, dtype=torch.float64)).to(dtype)
    order = torch.randperm(P, generator=g)
    c.tables = torch.full((B, W), -1, dtype=torch.int64)
    c.lengths = torch.tensor(lengths)
    used = torch.zeros(P, page, dtype=torch.bool)
    at = 0
    for b, x in enumerate(lengths):
        k = -(-x // page)
        c.tables[b, :k] = order[at:at + k]
        at += k
        for j in range(x):
            used[c.tables[b, j // page], j % page] = True
    c.q_pos = c.lengths.view(B, 1) - n + torch.arange(n)
    c.pos_pages = None
    if explicit:
        c.pos_pages = torch.randint(0, 50, (P, page), generator=g)  # stale ones look valid
        for b, x in enumerate(lengths):
            for j in range(x):
                p = 2 * j if torch.rand((), generator=g) > 0.1 else -1
                c.pos_pages[c.tables[b, j // page], j % page] = p
        c.q_pos = 2 * c.q_pos
    c.q_pos = c.q_pos.clamp(min=-1)
    for b, i in pad_rows:
        c.q_pos[b, i] = -1
    if stale is not None:
        c.k_pages.transpose(1, 2)[~used] = stale
        c.v_pages.transpose(1, 2)[~used] = stale
    return c


def to(c, dev):
    d = SimpleNamespace(**vars(c))
    for name in ("k_pages", "v_pages", "q", "tables", "lengths", "q_pos", "pos_pages"):
        t = getattr(c, name)
        if t is not None:
            setattr(d, name, t.to(dev))  # (keeps the strides of a transposed layout)
    return d


def call(cea, d, with_lse=False):
    fn = cea.paged_attention_with_lse if with_lse else cea.paged_attention
    return fn(d.q, d.k_pages, d.v_pages, d.tables, d.lengths, d.q_pos, pos_pages=d.pos_pages,
              causal=d.causal, scale=d.scale, kv_map=d.kv_map)


def keys_of(c, b):
    """(page, place, position) of row b's slots that exist."""
    got = []
    for j in range(max(0, min(int(c.lengths[b]), c.W * c.page))):
        p = int(c.tables[b, j // c.page])
        if 0 <= p < c.P:
            pos = j if c.pos_pages is None else int(c.pos_pages[p, j % c.page])
            if pos >= 0:
                got.append((p, j % c.page, pos))
    return got


def reference(c):
    """(out, lse, allowed error of out but for its own rounding and P's pieces, A, of lse) in f64."""
    u = U.get(c.dtype, 2.0 ** -24)
    out = torch.zeros(c.B, c.n, c.Hq, c.D, dtype=torch.float64)
    lse = torch.full((c.B, c.Hq, c.n), -math.inf, dtype=torch.float64)
    tol, mass, tol_lse = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(c.B):
        keys = keys_of(c, b)
        if not keys:
            continue
        pg, pl, pos = (torch.tensor(x) for x in zip(*keys))
        for h in range(c.Hq):
            kv = c.kv_map[h] if c.kv_map is not None else h // (c.Hq // c.Hkv)
            K, V = c.k_pages[pg, kv, pl].double(), c.v_pages[pg, kv, pl].double()
            for i in range(c.n):
                seen = pos <= int(c.q_pos[b, i]) if c.causal else torch.ones_like(pos, dtype=torch.bool)
                if not bool(seen.any()):
                    continue
                qv, k, v = c.q[b, i, h].double(), K[seen], V[seen]
                s = c.scale * (k @ qv)
                m = s.max()
                p = torch.exp(s - m)
                l = p.sum()
                out[b, i, h] = (p[:, None] * v).sum(0) / l
                lse[b, h, i] = m + torch.log(l)
                d = u * ((c.D + 4) * abs(c.scale) * (k.abs() @ qv.abs()) + 4 * s.abs() + 8).max()
                n = s.numel()
                mass[b, i, h] = (p[:, None] * v.abs()).sum(0) / l
                tol[b, i, h] = (2 * d + 2 * (n + 16) * u) * mass[b, i, h]
                tol_lse[b, h, i] = d + (n + 16) * u + 4 * u * abs(lse[b, h, i])
    return SimpleNamespace(out=out, lse=lse, tol=tol, mass=mass, tol_lse=tol_lse)


def check(c, ref, out, lse=None, pieces_left=None):
    """`pieces_left`: what the 16-bit pieces of p may leave of it (default: one piece of the type)."""
    out = out.detach().cpu()
    half = 0.0 if c.dtype in (torch.float32, torch.float64) else half_step(c.dtype)
    left = half if pieces_left is None else pieces_left
    bound = ref.tol + left * ref.mass + half_step(out.dtype) * ref.out.abs() + 1e-30
    if out.dtype == torch.float16:
        bound = bound + 2.0 ** -25  # subnormal steps
    err = (out.double() - ref.out).abs()
    assert not bool(torch.isnan(out).any()), "NaN"
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"out is {worst:.2f} of its bound off"
    empty = torch.isinf(ref.lse)
    assert bool((out.transpose(1, 2)[empty] == 0).all()), "empty rows must be 0"
    if lse is not None:
        lse = lse.detach().cpu().double()
        assert torch.equal(torch.isinf(lse) & (lse < 0), empty), "empty rows must have lse -inf"
        e = ((lse - ref.lse).abs() / ref.tol_lse)[~empty]
        assert e.numel() == 0 or e.max().item() <= 1.0, f"lse is {e.max().item():.2f} of its bound off"

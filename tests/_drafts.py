"""Seeded inputs of the tests of 8-bit pages and drafted trees, and their results in 64 bits.

Attention is held to the bounds of tests/_paged.py: the values that 8-bit pages stand for have 4 significant
bits and enter the products as they are, their scales are powers of two, so nothing but what those bounds count
is rounded.  Appends, reads, masks and moves are compared bit by bit: the rotary's products and sum are rounded to
f32 once each, as torch's, and what follows has one right answer.
"""

from __future__ import annotations

import math
from types import SimpleNamespace

import torch

import _paged as P

F8 = torch.float8_e4m3fn


# ---- 8 bits ------------------------------------------------------------------------------
def _codes():
    """The values of e4m3's codes 0..126 (all that are finite and not negative), in order."""
    v = []
    for c in range(127):
        e, m = c >> 3, c & 7
        v.append(math.ldexp(1 + m / 8, e - 7) if e else math.ldexp(m / 8, -6))
    return torch.tensor(v, dtype=torch.float64)


CODES = _codes()


def quantise(x, dtype):
    """Rows of f32 values [..., D] of a tensor of `dtype` as (codes uint8, scale bytes uint8), by the definition."""
    assert x.dtype == torch.float32
    x = x.double()
    ok = torch.isfinite(x)
    if dtype == torch.float16:
        x = torch.where(ok, x.clamp(-65504.0, 65504.0), x)
    m = torch.where(ok, x, torch.zeros_like(x)).abs().amax(-1)
    e = torch.full(m.shape, -117, dtype=torch.int64)
    for _ in range(250):
        e = torch.where(m > 448.0 * 2.0 ** e.double(), e + 1, e)
    y = torch.where(ok, x * 2.0 ** -e.double().unsqueeze(-1), torch.zeros_like(x))
    top = 135 if dtype == torch.float16 else 247
    y = torch.where((e + 127 == top).unsqueeze(-1), y.clamp(-240.0, 240.0), y)
    mag = y.abs()
    hi = torch.searchsorted(CODES, mag.contiguous()).clamp(max=126)  # the first code not below
    lo = (hi - 1).clamp(min=0)
    up, down = CODES[hi] - mag, mag - CODES[lo]
    c = torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))
    c = torch.where(mag == CODES[hi], hi, c)
    c = c + 128 * torch.signbit(y)
    c = torch.where(ok, c, torch.full_like(c, 0x7f))
    return c.to(torch.uint8), (e + 127).to(torch.uint8)


def values(codes, scales):
    """What 8-bit rows stand for, in f64."""
    c = codes.long()
    v = torch.cat([CODES, torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    v = torch.where(c >= 128, -v, v)
    return v * 2.0 ** (scales.double().unsqueeze(-1) - 127)


def rotate(x, cos, sin):
    """[B, n, H, D] rotated in f32, products and sum rounded once each."""
    x, c, s = x.float(), cos.float().unsqueeze(2), sin.float().unsqueeze(2)
    h = x.shape[-1] // 2
    return x * c + torch.cat([-x[..., h:], x[..., :h]], -1) * s


def pool8(c, seed):
    """The case's pools in 8 bits (c.codes, c.scales_), and c.k_pages / c.v_pages what they stand for."""
    g = torch.Generator().manual_seed(seed)
    for which in "kv":
        x = getattr(c, which + "_pages")
        q, s = quantise(x.float().contiguous(), torch.float32)
        s = (s.int() + torch.randint(-2, 3, s.shape, generator=g)).to(torch.uint8)
        setattr(c, which + "_codes", q)
        setattr(c, which + "_scales", s)
        setattr(c, which + "_pages", values(q, s))
    return c


# ---- trees -------------------------------------------------------------------------------
def parents(B, T, seed, back=6, root=0.15):
    g = torch.Generator().manual_seed(seed)
    i = torch.arange(T)
    p = i - torch.randint(1, back + 1, (B, T), generator=g)
    return torch.where(torch.rand(B, T, generator=g) < root, torch.full_like(p, -1), p.clamp(min=-1))


def ancestors(parents, counts=None):
    """Booleans [B, T, T]: node i's row holds itself and its ancestors."""
    B, T = parents.shape
    seen = torch.zeros(B, T, T, dtype=torch.bool)
    for b in range(B):
        for i in range(T if counts is None else max(0, min(T, int(counts[b])))):
            p = int(parents[b, i])
            if 0 <= p < i:
                seen[b, i] = seen[b, p]
            seen[b, i, i] = True
    return seen


def words(seen):
    """The booleans as int64 words, by Python's integers."""
    B, T, _ = seen.shape
    n = -(-T // 64)
    out = torch.zeros(B, T, n, dtype=torch.int64)
    for b in range(B):
        for i in range(T):
            x = sum(1 << j for j in range(T) if seen[b, i, j])
            for w in range(n):
                y = x >> 64 * w & (1 << 64) - 1
                out[b, i, w] = y - (1 << 64) if y >> 63 else y
    return out


def make_tree(T, lengths, counts=None, bits=16, seen=None, seed=0, **kw):
    """A case of tests/_paged.py whose queries are the nodes of trees in the rows' last slots."""
    c = P.make(B=len(lengths), n=T, lengths=lengths, seed=seed, **kw)
    c.counts = torch.tensor([T] * len(lengths) if counts is None else counts)
    c.seen = ancestors(parents(c.B, T, seed + 1)) if seen is None else seen
    c.masks = words(c.seen)
    if bits == 8:
        pool8(c, seed)
    return c


def sees(c, b, i, slot):
    """Whether query i of row b sees a slot that exists."""
    if not hasattr(c, "seen"):
        return slot <= int(c.q_pos[b, i]) if c.causal else True
    if i >= int(c.counts[b]):
        return False
    node = slot - (int(c.lengths[b]) - int(c.counts[b]))
    return node < 0 or (node < c.n and bool(c.seen[b, i, node]))


def reference(c):
    """As tests/_paged.py's, over the slots that `sees` names."""
    u = P.U.get(c.dtype, 2.0 ** -24)
    out = torch.zeros(c.B, c.n, c.Hq, c.D, dtype=torch.float64)
    lse = torch.full((c.B, c.Hq, c.n), -math.inf, dtype=torch.float64)
    tol, mass, tol_lse = torch.zeros_like(out), torch.zeros_like(out), torch.zeros_like(lse)
    for b in range(c.B):
        slots = [j for j in range(max(0, min(int(c.lengths[b]), c.W * c.page)))
                 if 0 <= int(c.tables[b, j // c.page]) < c.P]
        if c.pos_pages is not None:
            slots = [j for j in slots if int(c.pos_pages[int(c.tables[b, j // c.page]), j % c.page]) >= 0]
        if not slots:
            continue
        pg = torch.tensor([int(c.tables[b, j // c.page]) for j in slots])
        pl = torch.tensor([j % c.page for j in slots])
        pos = slots if c.pos_pages is None else c.pos_pages[pg, pl].tolist()
        seen = [torch.tensor([sees(c, b, i, x) for x in pos]) for i in range(c.n)]
        for h in range(c.Hq):
            kv = c.kv_map[h] if c.kv_map is not None else h // (c.Hq // c.Hkv)
            K, V = c.k_pages[pg, kv, pl].double(), c.v_pages[pg, kv, pl].double()
            for i in range(c.n):
                if not bool(seen[i].any()):
                    continue
                qv, k, v = c.q[b, i, h].double(), K[seen[i]], V[seen[i]]
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


def call(cea, c, dev, with_lse=False):
    """The case's call on the device: over trees or sequences, 8-bit or other pages."""
    kw = {"scale": c.scale, "kv_map": c.kv_map}
    pages = [c.k_pages.to(dev), c.v_pages.to(dev)]
    if hasattr(c, "k_codes"):
        pages = [c.k_codes.to(dev).view(F8), c.v_codes.to(dev).view(F8)]
        kw.update(k_scales=c.k_scales.to(dev), v_scales=c.v_scales.to(dev))
    args = [c.q.to(dev), *pages, c.tables.to(dev), c.lengths.to(dev)]
    name = "paged_tree_attention" if hasattr(c, "seen") else "paged_attention"
    if hasattr(c, "seen"):
        args += [c.counts.to(dev), c.masks.to(dev)]
    else:
        args.append(c.q_pos.to(dev))
        kw.update(causal=c.causal, pos_pages=None if c.pos_pages is None else c.pos_pages.to(dev))
    return getattr(cea, name + ("_with_lse" if with_lse else ""))(*args, **kw)


def check(cea, dev, c):
    """Both entry points: the plain one in q's type, the other in f32 (f64), whose probabilities keep f32's bits."""
    ref = reference(c)
    P.check(c, ref, call(cea, c, dev))
    out, lse = call(cea, c, dev, with_lse=True)
    acc = torch.float64 if c.dtype == torch.float64 else torch.float32
    assert out.dtype == acc and lse.dtype == acc
    P.check(c, ref, out, lse, pieces_left=0.0 if c.dtype in (torch.float32, torch.float64) else 2.0 ** -23)
    return ref

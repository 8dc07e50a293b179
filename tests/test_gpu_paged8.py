"""GPU tests of 8-bit pages: appends, reads and attention against their definitions (tests/_drafts.py)."""

from __future__ import annotations

import math

import pytest
import torch

import _drafts as D
import _paged as P

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
F8 = torch.float8_e4m3fn


def _same(got, want):
    """Codes bit by bit, but for NaN, which has two."""
    got, want = got.cpu(), want.cpu()
    nan = (got & 127) == 127
    assert torch.equal(nan, (want & 127) == 127), "NaN"
    assert torch.equal(got[~nan], want[~nan])


def _pools(P_, H, page, D_, seed, layout="hnd"):
    g = torch.Generator().manual_seed(seed)
    shape = (P_, H, page, D_) if layout == "hnd" else (P_, page, H, D_)
    out = []
    for _ in "kv":
        q = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
        s = torch.randint(1, 255, shape[:3], generator=g, dtype=torch.uint8)
        if layout != "hnd":
            q, s = q.transpose(1, 2), s.transpose(1, 2)
        out += [q, s]
    return out


def _append(cea, dev, x, y, page, dtype, rotary=True, counts=None, offsets=None, tables=None, pos=False, layout="hnd",
            P_=None, seed=0):
    """An append of rows x, y [B, n, H, D], compared with the definition; every other place stays as it was."""
    B, n, H, d = x.shape
    W = -(-(n + 37) // page)
    P_ = P_ or B * W + 2
    kq, ks, vq, vs = _pools(P_, H, page, d, seed, layout)
    g = torch.Generator().manual_seed(seed + 1)
    if tables is None:
        tables = torch.randperm(P_, generator=g)[:B * W].view(B, W)
    if offsets is None:
        offsets = torch.randint(0, 37, (B,), generator=g)
    ang = torch.rand(B, n, d // 2, generator=g, dtype=F64) * 6.3
    ang = torch.cat([ang, ang], -1)
    cos, sin = ang.cos().to(dtype), ang.sin().to(dtype)
    dk, dv, dks, dvs = (t.to(dev) for t in (kq, vq, ks, vs))
    kw = {}
    if rotary:
        kw.update(cos=cos.to(dev), sin=sin.to(dev))
    if counts is not None:
        kw["counts"] = counts.to(dev)
    if pos:
        pp, ps = torch.randint(0, 9, (P_, page), generator=g), torch.randint(0, 999, (B, n), generator=g)
        dpp = pp.to(dev)
        kw.update(pos_pages=dpp, pos=ps.to(dev))
    cea.paged_kv_append(dk.view(F8), dv.view(F8), tables.to(dev), offsets.to(dev), x.to(dev), y.to(dev),
                        k_scales=dks, v_scales=dvs, **kw)
    xr = D.rotate(x, cos, sin) if rotary else x.float()
    want_k, want_ks = D.quantise(xr.contiguous(), dtype)
    want_v, want_vs = D.quantise(y.float().contiguous(), dtype)
    for b in range(B):
        for i in range(n if counts is None else max(0, min(n, int(counts[b])))):
            j = int(offsets[b]) + i
            if not 0 <= j < tables.shape[1] * page:
                continue
            p = int(tables[b, j // page])
            if not 0 <= p < P_:
                continue
            kq[p, :, j % page], vq[p, :, j % page] = want_k[b, i], want_v[b, i]
            ks[p, :, j % page], vs[p, :, j % page] = want_ks[b, i], want_vs[b, i]
            if pos:
                pp[p, j % page] = ps[b, i]
    _same(dk, kq)
    _same(dv, vq)
    assert torch.equal(dks.cpu(), ks) and torch.equal(dvs.cpu(), vs)
    if pos:
        assert torch.equal(dpp.cpu(), pp)


def _rows(B, n, H, d, dtype, seed, spread=1):
    """Rows of every magnitude: a power of two of their own each."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, n, H, d, generator=g, dtype=F64)
    top = 14 if dtype == F16 else 40
    e = torch.randint(-top * spread, top * spread + 1, (B, n, H, 1), generator=g).double()
    return (x * 2.0 ** e).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("B,n,H,d,page", [(1, 1, 1, 128, 16), (3, 1, 8, 128, 64), (2, 70, 4, 64, 16), (2, 9, 3, 80, 48),
                                          (1, 33, 2, 16, 7), (2, 5, 2, 256, 32), (4, 3, 1, 2, 5), (1, 300, 8, 128, 64)])
def test_append(cea, dev, dtype, B, n, H, d, page):
    x, y = _rows(B, n, H, d, dtype, n), _rows(B, n, H, d, dtype, n + 1)
    _append(cea, dev, x, y, page, dtype, seed=d)
    _append(cea, dev, x, y, page, dtype, rotary=False, pos=True, seed=d)


@pytest.mark.parametrize("layout", ["hnd", "nhd"])
def test_append_counts_offsets_and_missing_pages(cea, dev, layout):
    x, y = _rows(4, 20, 2, 64, BF16, 1), _rows(4, 20, 2, 64, BF16, 2)
    tables = torch.tensor([[3, 7, 1, -1], [0, 99, 4, 5], [8, 9, 10, 11], [12, 13, 2, 6]])
    _append(cea, dev, x, y, 16, BF16, counts=torch.tensor([20, 20, -3, 50]), tables=tables,
            offsets=torch.tensor([40, 10, 0, -7]), P_=14, layout=layout)
    _append(cea, dev, x, y, 16, BF16, counts=torch.tensor([0, 1, 19, 2]), tables=tables,
            offsets=torch.tensor([0, 1 << 40, -(1 << 62), (1 << 63) - 5]), P_=14, layout=layout, pos=True)


def test_append_of_strided_rows(cea, dev):
    """Columns of a fused projection (unaligned ones too), and head-major rows."""
    g = torch.Generator().manual_seed(3)
    fused = torch.randn(2, 11, 7 * 64 + 3, generator=g).to(BF16)
    for lead in (0, 3):
        x = fused[..., lead:lead + 192].view(2, 11, 3, 64)
        y = fused[..., lead + 192:lead + 384].view(2, 11, 3, 64)
        _append(cea, dev, x, y, 16, BF16)
    x = torch.randn(2, 3, 11, 128, generator=g).to(F16).transpose(1, 2)
    _append(cea, dev, x, x * 0.5, 32, F16)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_append_of_extreme_rows(cea, dev, dtype):
    """Zeros, one value alone, the type's largest and smallest, infinities and NaN, ties of the rounding."""
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    for d in (64, 24):
        x = torch.zeros(1, 14, 1, d, dtype=F64)
        x[0, 1, 0, 3] = 1.0
        x[0, 2, 0, 5] = -448.0
        x[0, 3, 0, 5], x[0, 3, 0, 6] = 448.5, -0.01
        x[0, 4] = big
        x[0, 5, 0, 0] = small * 2.0 ** -3
        x[0, 6, 0, :3] = torch.tensor([math.inf, 2.0, -3.0])
        x[0, 7, 0, :3] = torch.tensor([math.nan, -math.inf, 0.125])
        x[0, 8] = math.nan
        x[0, 9] = torch.linspace(-448, 448, d)
        x[0, 10, 0, :8] = torch.tensor([256.0, 8.5, 17.0, 19.0, 0.0146484375, 0.001953125, 0.0009765625, 0.0029296875])
        x[0, 11, 0, 0], x[0, 11, 0, 1] = big, -big * 0.97
        x[0, 12] = -0.0
        x[0, 13, 0, :4] = torch.tensor([256.0, 224.0, 225.0, 1.75])
        x = x.to(dtype)
        _append(cea, dev, x, x, 16, dtype, rotary=False)
        _append(cea, dev, x, x, 16, dtype, rotary=True)  # (f16: beyond the type's range on the way)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("H,d,page,layout", [(2, 128, 16, "hnd"), (3, 64, 48, "hnd"), (2, 80, 7, "hnd"), (1, 6, 5, "nhd"),
                                             (4, 64, 32, "nhd")])
def test_read(cea, dev, dtype, H, d, page, layout):
    g = torch.Generator().manual_seed(d)
    kq, ks, vq, vs = _pools(9, H, page, d, d, layout)
    lo, hi = (110, 130) if dtype == F16 else (10, 240)  # (f16: into its subnormal numbers and beyond its largest)
    ks, vs = (torch.randint(lo, hi, s.shape, generator=g, dtype=torch.uint8) for s in (ks, vs))
    tables = torch.tensor([[2, 5, -1], [1, 9, 0], [8, 7, 6]])
    offsets, counts = torch.tensor([0, page - 1, -2]), torch.tensor([3 * page, 2 * page, 5])
    n = 2 * page + 3
    k, v = cea.paged_kv_read(kq.to(dev).view(F8), vq.to(dev).view(F8), tables.to(dev), offsets.to(dev), n,
                             counts=counts.to(dev), dtype=dtype, k_scales=ks.to(dev), v_scales=vs.to(dev))
    for got, q, s in ((k, kq, ks), (v, vq, vs)):
        assert got.shape == (3, n, H, d) and got.dtype == dtype
        val = D.values(q, s)
        want = torch.zeros(3, n, H, d, dtype=F64)
        for b in range(3):
            for i in range(min(n, int(counts[b]))):
                j = int(offsets[b]) + i
                p = int(tables[b, j // page]) if 0 <= j < 3 * page else -1
                if 0 <= p < 9:
                    want[b, i] = val[p, :, j % page]
        want = want.to(dtype)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu().float(), 0.0), torch.nan_to_num(want.float(), 0.0))


@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("d,page", [(64, 16), (10, 3)])
def test_read_of_pages_in_their_own_type(cea, dev, dtype, d, page):
    c = P.make(B=3, lengths=(2 * page, 5, 0), Hkv=2, D=d, page=page, dtype=dtype)
    n = 2 * page + 1
    k, v = cea.paged_kv_read(c.k_pages.to(dev), c.v_pages.to(dev), c.tables.to(dev), torch.zeros(3, dtype=torch.int64,
                             device=dev), n, counts=c.lengths.to(dev))
    for got, pages in ((k, c.k_pages), (v, c.v_pages)):
        want = torch.zeros(3, n, 2, d, dtype=dtype)
        for b in range(3):
            for j in range(min(n, int(c.lengths[b]))):
                want[b, j] = pages[c.tables[b, j // page], :, j % page]
        assert torch.equal(got.cpu(), want)


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
def _case(seed=0, **kw):
    return D.pool8(P.make(seed=seed, **kw), seed)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("Hq,Hkv,d,page", [(8, 2, 128, 16), (8, 1, 64, 32), (14, 2, 64, 64), (4, 4, 128, 128),
                                           (6, 2, 80, 16), (8, 2, 64, 48), (4, 2, 128, 24), (32, 1, 64, 16)])
def test_token(cea, dev, dtype, explicit, Hq, Hkv, d, page):
    D.check(cea, dev, _case(B=4, Hq=Hq, Hkv=Hkv, D=d, page=page, lengths=(301, 1, 64, 0), dtype=dtype, explicit=explicit,
                            seed=Hq + page))


@pytest.mark.parametrize("lengths", [(0,), (1,), (15,), (16,), (17,), (31,), (32,), (33,), (63,), (64,), (65,), (127,),
                                     (129,), (0, 0, 0), (1, 0, 2000), (4097,), (700, 1, 650, 33, 0, 129, 900)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 48])
def test_token_lengths(cea, dev, lengths, d, page):
    D.check(cea, dev, _case(B=len(lengths), Hq=8, Hkv=2, D=d, page=page, lengths=lengths, seed=len(lengths)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,Hq,Hkv", [(2, 8, 1), (2, 8, 2), (3, 8, 2), (5, 4, 4), (16, 2, 2), (7, 14, 2), (17, 4, 1)])
def test_few_tokens(cea, dev, dtype, n, Hq, Hkv):
    for explicit in (False, True):
        D.check(cea, dev, _case(B=3, n=n, Hq=Hq, Hkv=Hkv, D=64, page=16, lengths=(200, n, 1), dtype=dtype,
                                explicit=explicit, seed=n, pad_rows=[(0, n - 1), (2, 0)]))


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("n,lengths,Hq,Hkv,d,page", [
    (40, (100, 40, 333), 4, 2, 128, 16), (130, (130, 600), 4, 1, 64, 32), (257, (300, 259), 2, 2, 64, 16),
    (64, (64,), 8, 2, 128, 64), (33, (1025, 33), 14, 2, 64, 128), (300, (301,), 8, 1, 128, 48)])
def test_chunk(cea, dev, dtype, explicit, n, lengths, Hq, Hkv, d, page):
    D.check(cea, dev, _case(B=len(lengths), n=n, Hq=Hq, Hkv=Hkv, D=d, page=page, lengths=lengths, dtype=dtype,
                            explicit=explicit, seed=n))


def test_long_rows(cea, dev):
    """Keys split over workgroups, in every form."""
    D.check(cea, dev, _case(B=2, n=1, Hq=4, Hkv=1, D=128, page=64, lengths=(9000, 700), seed=1))
    D.check(cea, dev, _case(B=1, n=3, Hq=4, Hkv=1, D=64, page=16, lengths=(7777,), seed=2, dtype=F16))
    D.check(cea, dev, _case(B=2, n=20, Hq=4, Hkv=1, D=128, page=64, lengths=(5000, 700), seed=3))
    D.check(cea, dev, _case(B=1, n=18, Hq=2, Hkv=1, D=64, page=16, lengths=(3333,), seed=4, explicit=True))


@pytest.mark.parametrize("n", [1, 5, 40])
def test_options(cea, dev, n):
    """No causal rule, negative and large scales, an explicit head map, missing pages, clamped lengths."""
    kw = dict(B=2, n=n, Hq=6, Hkv=3, D=64, page=16, lengths=(150, 70))
    D.check(cea, dev, _case(causal=False, **kw))
    D.check(cea, dev, _case(scale=-0.3, **kw))
    D.check(cea, dev, _case(scale=2.0, q_scale=3.0, **kw))
    D.check(cea, dev, _case(kv_map=[2, 0, 1, 1, 0, 2], **kw))
    c = _case(**kw)
    c.tables[0, 3], c.tables[1, 0] = 10 ** 12, -5
    c.lengths = torch.tensor([1 << 40, 70])
    c.q_pos = torch.full_like(c.q_pos, 1 << 50)
    D.check(cea, dev, c)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n", [1, 4, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_hidden_nan_and_visible_nan(cea, dev, dtype, n, d):
    """NaN in slots that no query sees, or some queries, and in a value that all see."""
    for explicit in (False, True):
        c = P.make(B=2, n=n, Hq=4, Hkv=2, D=d, page=16, lengths=(200, 77), dtype=dtype, explicit=explicit, stale=math.nan)
        D.pool8(c, 1)
        want = D.reference(c)
        D.check(cea, dev, c)
        # the last token's own value: the queries before it do not see it
        p, at = int(c.tables[0, 199 // 16]), 199 % 16
        if explicit:
            c.pos_pages[p, at] = 398
        c.v_codes[p, 0, at, 5] = 0x7f
        out = D.call(cea, c, dev).cpu()
        bad = torch.isnan(out)
        expect = torch.zeros_like(bad)
        expect[0, n - 1, :2, 5] = True
        assert torch.equal(bad, expect)
        clean = ~expect
        err = (out.double() - want.out).abs()[clean] if not explicit else torch.zeros(1)
        bound = (want.tol + 2 * P.half_step(dtype) * (want.mass + want.out.abs()))[clean] if not explicit else torch.ones(1)
        assert bool((err <= bound + 2.0 ** -25).all())


def test_values_of_every_magnitude(cea, dev):
    """Scale bytes from one end to the other: rows of tiny and of large values in one softmax."""
    for n in (1, 30):
        c = P.make(B=1, n=n, Hq=2, Hkv=1, D=64, page=16, lengths=(100,), dtype=BF16)
        D.pool8(c, 5)
        g = torch.Generator().manual_seed(6)
        c.v_scales = torch.randint(87, 167, c.v_scales.shape, generator=g, dtype=torch.uint8)
        c.v_pages = D.values(c.v_codes, c.v_scales)
        D.check(cea, dev, c)


@pytest.mark.parametrize("n", [1, 24])
def test_repeats_itself(cea, dev, n):
    c = _case(B=3, n=n, Hq=8, Hkv=2, D=128, page=16, lengths=(3000, 40, 777))
    first = D.call(cea, c, dev, with_lse=True)
    for _ in range(5):
        again = D.call(cea, c, dev, with_lse=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def _any_bytes_where_unused(c, seed):
    """Numbers and scale bytes of every value in the slots that no row has, as in memory that nothing was written to."""
    g = torch.Generator().manual_seed(seed)
    used = torch.zeros(c.P, c.page, dtype=torch.bool)
    for b in range(c.B):
        for j in range(int(c.lengths[b])):
            used[c.tables[b, j // c.page], j % c.page] = True
    for which in "kv":
        q, s = getattr(c, which + "_codes"), getattr(c, which + "_scales")
        rq = torch.randint(0, 256, q.shape, generator=g, dtype=torch.uint8)
        rs = torch.randint(0, 256, s.shape, generator=g, dtype=torch.uint8)
        keep = used[:, None, :].expand(s.shape)
        setattr(c, which + "_codes", torch.where(keep.unsqueeze(-1), q, rq))
        setattr(c, which + "_scales", torch.where(keep, s, rs))
    return c


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 64), (128, 48), (80, 16)])
def test_unused_slots_hold_anything(cea, dev, dtype, d, page):
    for n in (1, 4, 40):
        for explicit in (False, True):
            c = _case(B=3, n=n, Hq=4, Hkv=2, D=d, page=page, lengths=(203, n, 81), dtype=dtype, explicit=explicit, seed=n)
            D.check(cea, dev, _any_bytes_where_unused(c, n))
    for T in (5, 50):
        c = D.make_tree(T, (203, T, 81), counts=(T, T, 3), bits=8, Hq=4, Hkv=2, D=d, page=page, dtype=dtype, seed=T)
        D.check(cea, dev, _any_bytes_where_unused(c, T))


def test_two_streams_at_once(cea, dev):
    """Calls with scratch of their own, overlapping on two streams."""
    cases = [_case(B=2, n=n, Hq=8, Hkv=2, D=128, page=64, lengths=(6000, 3000), seed=n) for n in (1, 40)]
    cases += [D.make_tree(30, (5000, 2000), bits=8, Hq=8, Hkv=2, D=64, seed=3)]
    want = [D.call(cea, c, dev) for c in cases]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for turn in range(6):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([D.call(cea, c, dev) for c in cases])
    torch.cuda.synchronize()
    for x in got:
        assert all(torch.equal(a, b) for a, b in zip(x, want))

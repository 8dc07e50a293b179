"""GPU tests of attention over 8-bit pages at the ends of the scale bytes' range, against 64 bits (tests/_drafts.py).

Weights reach 2^8 before a row's reference maximum follows them (half of a tile's scores may be above it), so
the values here stand where such a weight and a value would pass f32's largest number, and at the other end
where a weight's later pieces would be below its smallest.  Bounds beside those of tests/_paged.py: sums are held
at 2^-8 of theirs, and a piece of a weight in bf16, or a product in f32, loses at most 2^-134 below the normal
numbers, which is 2^-126 of a sum's own scale for each code of at most 448: n keys, whose weights' sum l is 1 at
least, are within n 2^-117 / l.
"""

from __future__ import annotations

import math

import pytest
import torch

import _drafts as D
import _paged as P

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def _compare(c, out, pieces, scale=None):
    """`out` against the case's definition; every value finite."""
    ref = D.reference(c)
    out = out.cpu()
    assert bool(torch.isfinite(out).all()), "not finite"
    keys = int(c.lengths.max())
    bound = ref.tol + pieces * ref.mass + P.half_step(out.dtype) * ref.out.abs() + keys * 2.0 ** -117 + 2.0 ** -134
    err = (out.double() - ref.out).abs()
    assert bool((err <= bound).all()), f"{(err / bound).max().item():.2f} of its bound off"


def _peak(n, B, H, d, page, lengths, far, byte, code, dtype=BF16, score=5.5, tree=False):
    """Scores of 0 but for slot `far`, whose score is within the lag of the maximum (exp(5.5) = 2^7.93), and its
    value 2^(byte - 127) times a code in feature 5 and 0 in all others; the other values are near 1."""
    if tree:
        c = D.make_tree(n, lengths, bits=16, Hq=H, Hkv=H, D=d, page=page, scale=1.0)
    else:
        c = P.make(B=B, n=n, Hq=H, Hkv=H, D=d, page=page, lengths=lengths, dtype=dtype, scale=1.0)
    D.pool8(c, 1)
    c.q.zero_()
    c.q[..., 0] = 1
    c.k_codes.zero_()
    c.k_scales.fill_(127)
    for b in range(B):
        p, at = int(c.tables[b, far // page]), far % page
        c.k_codes[p, :, at, 0] = int((D.CODES == score).nonzero())
        c.v_codes[p, :, at] = 0
        c.v_codes[p, :, at, 5] = int((D.CODES == code).nonzero())
        c.v_scales[p, :, at] = byte
    c.k_pages, c.v_pages = D.values(c.k_codes, c.k_scales), D.values(c.v_codes, c.v_scales)
    return c


# bytes and codes: the largest values of bf16's range with the largest byte that an append leaves, and with the
# largest that a page may hold
TOPS = [(247, 240.0), (254, 1.75), (250, 1.0), (240, 448.0)]


@pytest.mark.parametrize("byte,code", TOPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 4])
def test_weights_of_the_largest_values_in_one_launch(cea, dev, byte, code, d, n):
    c = _peak(n, 1, 2, d, 16, (600,), 512, byte, code)
    _compare(c, D.call(cea, c, dev), 2.0 ** -16)
    out, lse = D.call(cea, c, dev, with_lse=True)
    _compare(c, out, 2.0 ** -23)
    ref = D.reference(c)
    assert bool(((lse.cpu().double() - ref.lse).abs() <= ref.tol_lse).all())


@pytest.mark.parametrize("byte,code", TOPS)
@pytest.mark.parametrize("d", [64, 128])
def test_weights_of_the_largest_values_in_runs(cea, dev, byte, code, d):
    """Rows cut into runs of several blocks, and joined."""
    c = _peak(1, 2, 64, d, 64, (2100, 1900), 1100, byte, code)
    _compare(c, D.call(cea, c, dev), 2.0 ** -16)
    out, lse = D.call(cea, c, dev, with_lse=True)
    _compare(c, out, 2.0 ** -23)
    ref = D.reference(c)
    assert bool(((lse.cpu().double() - ref.lse).abs() <= ref.tol_lse).all())


@pytest.mark.parametrize("byte,code", TOPS)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
def test_weights_of_the_largest_values_in_chunks(cea, dev, byte, code, d, tree):
    c = _peak(40, 1, 2, d, 16, (600,), 512, byte, code, tree=tree)
    _compare(c, D.call(cea, c, dev), P.half_step(BF16))
    out, lse = D.call(cea, c, dev, with_lse=True)
    _compare(c, out, 2.0 ** -23)
    ref = D.reference(c)
    assert bool(((lse.cpu().double() - ref.lse).abs() <= ref.tol_lse).all())


@pytest.mark.parametrize("byte,code", TOPS)
def test_weights_of_the_largest_values_elsewhere(cea, dev, byte, code):
    """f32 queries, and a head size of the generic kernel."""
    c = _peak(3, 1, 2, 80, 16, (600,), 512, byte, code)
    _compare(c, D.call(cea, c, dev), 2.0 ** -23)
    c = _peak(3, 1, 2, 64, 16, (600,), 512, byte, code, dtype=F32)
    _compare(c, D.call(cea, c, dev), 0.0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n", [1, 4, 40])
def test_the_smallest_values(cea, dev, n, d):
    """All values at the append's smallest scale bytes."""
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=d, page=16, lengths=(300, 77), dtype=BF16)
    D.pool8(c, 2)
    g = torch.Generator().manual_seed(3)
    for lo, hi in ((10, 11), (10, 30), (30, 60)):
        c.v_scales = torch.randint(lo, hi, c.v_scales.shape, generator=g, dtype=torch.uint8)
        c.v_pages = D.values(c.v_codes, c.v_scales)
        _compare(c, D.call(cea, c, dev), 2.0 ** -16 if n < 40 else P.half_step(BF16))
        _compare(c, D.call(cea, c, dev, with_lse=True)[0], 2.0 ** -23)


def test_appended_rows_at_the_ends_of_bf16(cea, dev):
    """What an append makes of rows near bf16's largest and smallest numbers, attended by single tokens."""
    c = P.make(B=2, n=1, Hq=2, Hkv=2, D=64, page=16, lengths=(600, 40), dtype=BF16, scale=1.0)
    x = torch.zeros(c.P, c.Hkv, c.page, c.D)
    x[..., 0] = -1.0
    y = torch.zeros_like(x)
    y[..., 7] = torch.finfo(BF16).smallest_normal
    for b, j in ((0, 512), (1, 3)):
        p, at = int(c.tables[b, j // 16]), j % 16
        x[p, :, at, 0] = 4.5
        y[p, :, at, 5] = torch.finfo(BF16).max
    for which, t in (("k", x), ("v", y)):
        codes, scales = D.quantise(t, BF16)
        setattr(c, which + "_codes", codes)
        setattr(c, which + "_scales", scales)
        setattr(c, which + "_pages", D.values(codes, scales))
    c.q.zero_()
    c.q[..., 0] = 1
    assert int(c.v_scales.max()) == 247 and int(c.v_scales.min()) == 10
    _compare(c, D.call(cea, c, dev), 2.0 ** -16)
    _compare(c, D.call(cea, c, dev, with_lse=True)[0], 2.0 ** -23)

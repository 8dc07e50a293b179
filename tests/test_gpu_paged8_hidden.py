"""GPU tests of 8-bit pages with NaN in values that some queries see and others do not: what is not NaN is right too,
with slots by number and with positions in the pool, against 64 bits (tests/_drafts.py)."""

from __future__ import annotations

import math

import pytest
import torch

import _drafts as D
import _paged as P

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("n,Hq,Hkv,d,page", [(1, 4, 2, 128, 16), (4, 4, 2, 64, 16), (4, 4, 2, 128, 48), (16, 2, 2, 64, 32),
                                             (40, 4, 2, 128, 16), (150, 4, 1, 64, 16), (3, 4, 2, 80, 16)])
def test_what_is_not_nan_is_right(cea, dev, n, Hq, Hkv, d, page, explicit, dtype):
    """NaN in the newest value, which the last query alone sees, and in one in the middle of the new tokens, which the
    queries from it on see; stale NaN behind the rows' ends."""
    c = P.make(B=2, n=n, Hq=Hq, Hkv=Hkv, D=d, page=page, lengths=(200, 173), dtype=dtype, explicit=explicit, stale=math.nan,
               seed=n)
    D.pool8(c, n)
    marks = [(0, 199, 5, n - 1)]
    if n > 2:
        marks.append((1, 172 - n // 2, 7, n - 1 - n // 2))
    if explicit:  # (those slots hold a token, whatever the case left there)
        for b, j, _, _ in marks:
            c.pos_pages[c.tables[b, j // page], j % page] = 2 * j
    want = D.reference(c)
    bad = torch.zeros_like(want.out, dtype=torch.bool)
    for b, j, f, first in marks:
        c.v_codes[c.tables[b, j // page], 0, j % page, f] = 0x7f
        bad[b, first:, :Hq // Hkv, f] = True
    # (two or three bf16 pieces of a probability in the forms of few tokens, one of the type in chunks)
    for with_lse, left in ((False, P.half_step(dtype)), (True, 2.0 ** -23)):
        got = D.call(cea, c, dev, with_lse=with_lse)
        out = (got[0] if with_lse else got).cpu()
        assert torch.equal(torch.isnan(out), bad)
        bound = want.tol + left * want.mass + P.half_step(out.dtype) * want.out.abs() + 2.0 ** -25
        err = (out.double() - want.out).abs()
        assert bool((err <= bound)[~bad].all()), f"{(err / bound)[~bad].max().item():.2f} of its bound off"
    lse = got[1].cpu().double()
    assert bool(((lse - want.lse).abs() <= want.tol_lse).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [5, 16, 40])
def test_what_is_not_nan_is_right_in_trees(cea, dev, T, dtype):
    """NaN in a value of one node: its descendants have it, the others' results are right."""
    p = D.parents(2, T, 3)
    seen = D.ancestors(p)
    c = D.make_tree(T, (150, T + 3), bits=8, seen=seen, Hq=4, Hkv=2, D=64, page=16, dtype=dtype)
    want = D.reference(c)
    bad = torch.zeros_like(want.out, dtype=torch.bool)
    for b in range(2):
        j = int(c.lengths[b]) - T + T // 3
        c.v_codes[c.tables[b, j // 16], 1, j % 16, 9] = 0x7f
        bad[b, :, 2:, 9] = seen[b, :, T // 3].view(-1, 1)
    for with_lse, left in ((False, P.half_step(dtype)), (True, 2.0 ** -23)):
        got = D.call(cea, c, dev, with_lse=with_lse)
        out = (got[0] if with_lse else got).cpu()
        assert torch.equal(torch.isnan(out), bad)
        bound = want.tol + left * want.mass + P.half_step(out.dtype) * want.out.abs() + 2.0 ** -25
        assert bool(((out.double() - want.out).abs() <= bound)[~bad].all())

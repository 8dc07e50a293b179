"""GPU tests of the paged KV cache against its formulas in 64 bits (bounds: tests/_paged.py)."""

from __future__ import annotations

import math
import random

import pytest
import torch

import _paged as P
from oracle import cache_ref as C
from oracle import layers_ref as L

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64


def _check(cea, dev, c, lse=True):
    """Both entry points on the case: the plain one in q's type, the other in f32 (f64)."""
    ref = P.reference(c)
    d = P.to(c, dev)
    P.check(c, ref, P.call(cea, d))
    if lse:
        out, l = P.call(cea, d, with_lse=True)
        assert out.dtype == (F64 if c.dtype == F64 else F32)
        # f32 results carry their probabilities to 2^-24 and better
        P.check(c, ref, out, l, pieces_left=0.0 if c.dtype in (F32, F64) else 2.0 ** -23)
    return ref


# ---------------------------------------------------------------------------------------
# single tokens
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (8, 1, 64, 32), (14, 2, 64, 64), (4, 4, 128, 128),
                                           (6, 2, 80, 16), (8, 2, 64, 48), (4, 2, 128, 24), (32, 1, 64, 16)])
def test_token(cea, dev, dtype, explicit, Hq, Hkv, D, page):
    _check(cea, dev, P.make(B=4, Hq=Hq, Hkv=Hkv, D=D, page=page, lengths=(301, 1, 64, 0), dtype=dtype,
                            explicit=explicit, seed=Hq + page))


@pytest.mark.parametrize("lengths", [(0,), (1,), (15,), (16,), (17,), (63,), (64,), (65,), (0, 0, 0), (1, 0, 2000),
                                     (4097,), (700, 1, 650, 33, 0, 129, 900)])
@pytest.mark.parametrize("D", [64, 128])
def test_token_lengths(cea, dev, lengths, D):
    _check(cea, dev, P.make(B=len(lengths), Hq=8, Hkv=2, D=D, page=16, lengths=lengths, seed=len(lengths)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("n,Hq,Hkv", [(2, 8, 1), (2, 8, 2), (3, 8, 2), (4, 8, 2), (5, 4, 4), (16, 2, 2), (7, 14, 2),
                                      (12, 8, 8), (17, 4, 1)])
def test_few_tokens(cea, dev, dtype, n, Hq, Hkv):
    """A verification step: a few new tokens a row, causal among themselves, and padded rows."""
    for explicit in (False, True):
        _check(cea, dev, P.make(B=3, n=n, Hq=Hq, Hkv=Hkv, D=64, page=16, lengths=(200, n, 1), dtype=dtype,
                                explicit=explicit, seed=n, pad_rows=[(0, n - 1), (2, 0)]))


# ---------------------------------------------------------------------------------------
# chunks
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("n,lengths,Hq,Hkv,D,page", [
    (40, (100, 40, 333), 4, 2, 128, 16), (130, (130, 600), 4, 1, 64, 32), (257, (300, 259), 2, 2, 64, 16),
    (64, (64,), 8, 2, 128, 64), (33, (1025, 33), 14, 2, 64, 128), (300, (301,), 8, 1, 128, 48)])
def test_chunk(cea, dev, dtype, explicit, n, lengths, Hq, Hkv, D, page):
    _check(cea, dev, P.make(B=len(lengths), n=n, Hq=Hq, Hkv=Hkv, D=D, page=page, lengths=lengths, dtype=dtype,
                            explicit=explicit, seed=n))


def test_chunk_over_many_keys(cea, dev):
    """Few query rows against a long row: the keys are split over workgroups."""
    _check(cea, dev, P.make(B=2, n=20, Hq=4, Hkv=1, D=128, page=64, lengths=(5000, 700), seed=1))
    _check(cea, dev, P.make(B=1, n=18, Hq=2, Hkv=1, D=64, page=16, lengths=(3333,), seed=2, explicit=True))


@pytest.mark.parametrize("n", [1, 5, 70])
def test_padded_and_empty_rows(cea, dev, n):
    """Queries of position -1 and rows without slots give (0, -inf); their values are not read into
    any other row."""
    c = P.make(B=4, n=n, Hq=8, Hkv=2, D=64, page=16, lengths=(0, n, 90, 77), seed=n,
               pad_rows=[(3, i) for i in range(n // 2, n)] + [(2, 0)])
    _check(cea, dev, c)


@pytest.mark.parametrize("n", [1, 3, 50])
def test_not_causal(cea, dev, n):
    for explicit in (False, True):
        _check(cea, dev, P.make(B=2, n=n, Hq=4, Hkv=2, D=128, page=16, lengths=(99, 50), causal=False,
                                explicit=explicit, seed=n, pad_rows=[(0, 0)]))


@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1e-35, 2.0])
def test_scales(cea, dev, n, scale):
    _check(cea, dev, P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(130, 60), scale=scale, seed=3))


@pytest.mark.parametrize("n", [1, 2, 60])
@pytest.mark.parametrize("kv_map", [(0, 0, 1, 1, 2), (2, 1, 0, 0, 0), (1, 1, 1, 1, 1)])
def test_head_maps(cea, dev, n, kv_map):
    _check(cea, dev, P.make(B=2, n=n, Hq=5, Hkv=3, D=64, page=16, lengths=(200, 64), kv_map=kv_map, seed=4))


@pytest.mark.parametrize("n", [1, 4, 90])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_token_major_pages(cea, dev, n, dtype):
    """Pools laid out [P, page, H, D], handed over as a transposed view, read in place."""
    _check(cea, dev, P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(150, 95), layout="nhd", dtype=dtype,
                            explicit=True, seed=5))


@pytest.mark.parametrize("n", [1, 3, 80])
def test_strided_queries_tables_and_positions(cea, dev, n):
    """Column slices of a fused projection, every second table column, int32 tables, and positions
    with another stride or type."""
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(150, 95), explicit=True, seed=6)
    ref = P.reference(c)
    d = P.to(c, dev)
    fused = torch.randn(2, n, 4 * 64 + 40, device=dev).to(BF16)
    fused[:, :, 24:24 + 256] = d.q.view(2, n, 256)
    d.q = fused[:, :, 24:24 + 256].view(2, n, 4, 64)
    wide = torch.full((2, 2 * c.W), 10 ** 12, dtype=torch.int64, device=dev)
    wide[:, ::2] = d.tables
    d.tables = wide[:, ::2]
    both = torch.zeros(2, n, 2, dtype=torch.int64, device=dev)
    both[:, :, 1] = d.q_pos
    d.q_pos = both[:, :, 1]
    P.check(c, ref, P.call(cea, d))
    pos = torch.zeros(c.P, 16, 2, dtype=torch.int64, device=dev)
    pos[:, :, 0] = d.pos_pages
    d.pos_pages = pos[:, :, 0]
    P.check(c, ref, P.call(cea, d))
    d = P.to(c, dev)
    d.tables, d.lengths, d.q_pos = d.tables.int(), d.lengths.int(), d.q_pos.int()
    P.check(c, ref, P.call(cea, d))


def test_unaligned_queries(cea, dev):
    """A query view that starts off the 16-byte grid."""
    for n in (1, 40):
        c = P.make(B=1, n=n, Hq=2, Hkv=2, D=64, page=16, lengths=(70,), seed=7)
        d = P.to(c, dev)
        buf = torch.zeros(n * 128 + 1, dtype=BF16, device=dev)
        buf[1:] = d.q.view(-1)
        d.q = buf[1:].view(1, n, 2, 64)
        P.check(c, P.reference(c), P.call(cea, d))


# ---------------------------------------------------------------------------------------
# what must not be seen
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n", [1, 3, 100])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_stale_slots_hold_anything(cea, dev, bad, n, dtype):
    """Slots behind a row's length, of pages that end inside a tile and of other pages."""
    for explicit in (False, True):
        _check(cea, dev, P.make(B=2, n=n, Hq=8, Hkv=2, D=64, page=64, lengths=(n + 67, n), dtype=dtype,
                                explicit=explicit, stale=bad, seed=8))


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n", [1, 4, 100])
@pytest.mark.parametrize("D", [64, 128])
def test_hidden_keys_hold_anything(cea, dev, bad, n, D):
    """Keys inside a row's length that nobody sees (position -1), and keys that only later queries
    see: an infinity or NaN in their values reaches exactly the rows that see it."""
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=D, page=16, lengths=(n + 50, n + 9), explicit=True, seed=9)
    for b in range(2):
        for j in range(int(c.lengths[b])):
            p, i = int(c.tables[b, j // 16]), j % 16
            if c.pos_pages[p, i] < 0:
                c.k_pages[p, :, i], c.v_pages[p, :, i] = bad, bad
    ref = _check(cea, dev, c)
    # now the last key of row 0 in one value: only queries at or behind it see it
    j = int(c.lengths[0]) - 1 - n // 2
    p, i = int(c.tables[0, j // 16]), j % 16
    c.pos_pages[p, i] = 2 * j
    ref = P.reference(c)
    c.v_pages[p, 0, i, 5] = bad
    sees = c.q_pos[0] >= 2 * j
    for with_lse in (False, True):
        got = P.call(cea, P.to(c, dev), with_lse)
        out = (got[0] if with_lse else got).cpu()
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[0, sees, :2, 5] = True
        assert bool(hit.any())
        assert bool((out[hit].isnan() if math.isnan(bad) else out[hit] == bad).all())
        P.check(c, ref, torch.where(hit, ref.out.to(out.dtype), out), got[1] if with_lse else None)


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("n,D", [(1, 64), (3, 128), (20, 64), (20, 128)])
def test_hidden_keys_of_long_rows_hold_anything(cea, dev, bad, n, D):
    """The same where a row is cut into parts and splits: only the parts that hold such a value differ."""
    c = P.make(B=2, n=n, Hq=4, Hkv=1, D=D, page=64, lengths=(5003, 1100), explicit=True, stale=bad, seed=22)
    for b, js in ((0, (7, 2500, 5001)), (1, (64,))):
        for j in js:
            p, i = int(c.tables[b, j // 64]), j % 64
            c.pos_pages[p, i] = -1
            c.k_pages[p, :, i], c.v_pages[p, :, i] = bad, bad
    _check(cea, dev, c)
    c = P.make(B=2, n=n, Hq=4, Hkv=1, D=D, page=64, lengths=(5003, 1100), stale=bad, seed=23)
    p, i = int(c.tables[0, 5002 // 64]), 5002 % 64  # the last token, which only the last query sees
    ref = P.reference(c)
    c.v_pages[p, 0, i, 9] = bad
    out, lse = P.call(cea, P.to(c, dev), True)
    out = out.cpu()
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[0, n - 1, :, 9] = True
    assert bool((out[hit].isnan() if math.isnan(bad) else out[hit] == bad).all())
    P.check(c, ref, torch.where(hit, ref.out.float(), out), lse, pieces_left=2.0 ** -23)


def test_values_of_probability_zero(cea, dev):
    """A visible key whose probability underflows to 0 still meets its infinite value: 0 * inf."""
    for n in (1, 40):
        c = P.make(B=1, n=n, Hq=2, Hkv=2, D=64, page=16, lengths=(n + 20,), seed=10)
        c.k_pages[int(c.tables[0, 0]), :, 3] = 0
        for i in range(n):
            for h in range(2):
                c.k_pages[int(c.tables[0, 0]), h, 0] = 200.0
        c.q[:] = 4.0
        c.v_pages[int(c.tables[0, 0]), 0, 3, 7] = math.inf
        out = P.call(cea, P.to(c, dev)).cpu()
        assert bool(out[:, :, 0, 7].isnan().all() | (out[:, :, 0, 7] == math.inf).all())
        assert bool(torch.isfinite(out[:, :, 1]).all())


@pytest.mark.parametrize("D,explicit", [(64, False), (64, True), (128, True)])
def test_every_workgroup_looks_at_its_tiles_again(cea, dev, D, explicit):
    """Hidden values that are not finite under every query block of many equal rows: each goes over its
    tiles twice, and every time every row is the same and right."""
    n, copies = 130, 48
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=D, page=16, lengths=(n + 150, n + 33), explicit=explicit, seed=26)
    ref = P.reference(c)
    for b in range(2):  # a slot that nobody sees, or (by its number) the last query alone
        j = 20 if explicit else int(c.lengths[b]) - 1
        p, i = int(c.tables[b, j // 16]), j % 16
        if explicit:
            c.pos_pages[p, i] = -1
        c.v_pages[p, :, i] = math.nan
    if explicit:
        ref = P.reference(c)
    d = P.to(c, dev)
    for name in ("q", "tables", "lengths", "q_pos"):
        t = getattr(d, name)
        setattr(d, name, t.repeat(copies, *[1] * (t.dim() - 1)))
    first = None
    for _ in range(20):
        out = P.call(cea, d).view(copies, 2, n, 4, D)
        first = out[0].clone() if first is None else first
        assert torch.equal(out.nan_to_num(7.0), first.nan_to_num(7.0).expand_as(out))
    got = first.cpu()
    if not explicit:
        assert bool(got[:, n - 1].isnan().all())
        got[:, n - 1] = ref.out[:, n - 1].to(got.dtype)
    P.check(c, ref, got)


def _zero_probability_case(n, length, dtype, explicit, top, bad):
    """One key of slot `top` takes every query's whole sum (scores of 6400 against a few), so slot 3, which
    every query sees as well, has probability 0 in any precision; its value is `bad` in KV head 0's feature 7."""
    c = P.make(B=1, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(length,), dtype=dtype, explicit=explicit, seed=27)
    c.q[:] = 4.0
    for j in (3, top):
        p, i = int(c.tables[0, j // 16]), j % 16
        c.k_pages[p, :, i] = 200.0 if j == top else 0.0
        if explicit:
            c.pos_pages[p, i] = 2 * j
    ref = P.reference(c)
    c.v_pages[int(c.tables[0, 0]), 0, 3, 7] = bad
    hit = torch.zeros(1, n, 4, 64, dtype=torch.bool)
    hit[:, :, :2, 7] = True  # 0 * inf and 0 * NaN
    return c, ref, hit


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("n,length", [(1, 70), (1, 1500), (1, 9000), (4, 2100), (40, 90), (40, 1900)])
def test_a_visible_value_of_probability_zero_is_still_met(cea, dev, n, length, dtype, explicit, bad):
    """0 * inf is NaN wherever rows are cut: the key that takes the sum lies in the first tile, or far behind."""
    for top in (0, length - n - 1):
        c, ref, hit = _zero_probability_case(n, length, dtype, explicit, top, bad)
        d = P.to(c, dev)
        for with_lse in (False, True):
            got = P.call(cea, d, with_lse)
            out = (got[0] if with_lse else got).cpu()
            assert bool(out[hit].isnan().all()), (top, with_lse)
            P.check(c, ref, torch.where(hit, ref.out.to(out.dtype), out), got[1] if with_lse else None)


@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("n,length", [(1, 70), (1, 1500), (40, 90), (40, 1900)])
def test_a_visible_score_of_minus_infinity(cea, dev, n, length, dtype, explicit):
    """Its probability is 0 as any other's that underflows, and the key is visible all the same: an infinite
    value there makes a NaN, a finite one nothing."""
    c = P.make(B=1, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(length,), dtype=dtype, explicit=explicit, seed=29)
    c.q = c.q.abs() + 1  # of one sign: a feature of -inf makes a score of -inf
    page = int(c.tables[0, 0])
    c.k_pages[page, :, 3] = -200.0
    if explicit:
        c.pos_pages[page, 3] = 0
    ref = P.reference(c)
    c.k_pages[page, :, 3, 11] = -math.inf
    P.check(c, ref, P.call(cea, P.to(c, dev)))
    c.v_pages[page, 0, 3, 7] = math.inf
    hit = torch.zeros(1, n, 4, 64, dtype=torch.bool)
    hit[:, :, :2, 7] = True
    out = P.call(cea, P.to(c, dev)).cpu()
    assert bool(out[hit].isnan().all())
    P.check(c, ref, torch.where(hit, ref.out.to(out.dtype), out))


@pytest.mark.parametrize("n", [1, 30])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_not_a_number_in_a_visible_place(cea, dev, n, dtype):
    """A NaN that a query sees is its result, in q, K or V."""
    c = P.make(B=1, n=n, Hq=2, Hkv=2, D=64, page=16, lengths=(n + 20,), dtype=dtype, seed=11)
    ref = P.reference(c)
    for where in ("q", "k"):
        d = P.to(c, dev)
        if where == "q":
            d.q = d.q.clone()
            d.q[0, n - 1, 0, 3] = math.nan
        else:
            d.k_pages = d.k_pages.clone()
            j = n + 19
            d.k_pages[int(c.tables[0, j // 16]), 0, j % 16, 3] = math.nan
        out = P.call(cea, d).cpu()
        assert bool(out[0, n - 1, 0].isnan().all())
        out[0, n - 1, 0] = ref.out[0, n - 1, 0].to(dtype)
        P.check(c, ref, out)


@pytest.mark.parametrize("n", [1, 50])
def test_pages_that_do_not_exist(cea, dev, n):
    """Page indices outside the pool hold no keys, lengths count only what the table holds."""
    for explicit in (False, True):
        c = P.make(B=3, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(n + 100, n + 40, n + 30), explicit=explicit, seed=12)
        c.tables[0, 1], c.tables[0, 3], c.tables[1, 0] = c.P, -5, 2 ** 40
        c.tables[2, -1] = 2 ** 62
        c.lengths[2] = 10 ** 15
        c.q_pos[:] = 10 ** 9
        _check(cea, dev, c)
    c.lengths[:] = torch.tensor([-3, 0, -(2 ** 60)])
    _check(cea, dev, c)


def test_empty_calls(cea, dev):
    i64 = dict(dtype=torch.int64, device=dev)
    kp = torch.randn(3, 2, 16, 64, device=dev).to(BF16)
    for B, n in ((0, 1), (2, 0)):
        out = cea.paged_attention(torch.zeros(B, n, 4, 64, dtype=BF16, device=dev), kp, kp, torch.zeros(B, 1, **i64),
                                  torch.ones(B, **i64), torch.zeros(B, n, **i64))
        assert out.shape == (B, n, 4, 64)
    q = torch.randn(2, 3, 4, 64, device=dev).to(BF16)
    for pool, W in ((kp, 0), (kp[:0], 2), (kp[:, :, :0], 2)):
        out, lse = cea.paged_attention_with_lse(q, pool, pool, torch.zeros(2, W, **i64), torch.full((2,), 5, **i64),
                                                torch.full((2, 3), 9, **i64))
        assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_offsets_past_32_bits(cea, dev):
    """Pages whose elements lie beyond 2^32 elements of the pool's start."""
    page, D, H = 16, 64, 2
    pages = (2 ** 32 + 2 ** 20) // (H * page * D)
    pool = torch.empty(pages, H, page, D, dtype=BF16, device=dev)
    for n, explicit in ((1, False), (3, True), (60, False), (60, True)):
        c = P.make(B=2, n=n, Hq=4, Hkv=H, D=D, page=page, lengths=(n + 100, n + 7), explicit=explicit, seed=13)
        d = P.to(c, dev)
        far = pages - c.P
        pool[far:] = d.k_pages
        d.k_pages = pool
        d.v_pages = pool  # values are the keys
        cv = P.to(c, "cpu")
        cv.v_pages = c.k_pages
        ref = P.reference(cv)
        d.tables = torch.where(d.tables >= 0, d.tables + far, d.tables)
        if explicit:
            pos = torch.full((pages, page), -1, dtype=torch.int64, device=dev)
            pos[far:] = d.pos_pages
            d.pos_pages = pos
        P.check(c, ref, P.call(cea, d))


def test_a_row_of_a_wide_table(cea, dev):
    """A table much wider than its rows are long, pages in any order, the same page twice."""
    c = P.make(B=3, n=1, Hq=8, Hkv=2, D=64, page=16, lengths=(100, 3, 40), width=4000, seed=14)
    c.tables[0, 2] = c.tables[0, 1]
    _check(cea, dev, c)


def test_many_rows(cea, dev):
    c = P.make(B=150, n=1, Hq=4, Hkv=2, D=64, page=16, lengths=[(7 * b) % 90 for b in range(150)], seed=15)
    _check(cea, dev, c)


@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(4, 1, 64, 16), (2, 2, 128, 48)])
def test_long_rows(cea, dev, explicit, Hq, Hkv, D, page):
    """Tens of thousands of keys: a unit cut into hundreds of parts, a chunk in several passes."""
    for n in (1, 3, 35):
        _check(cea, dev, P.make(B=1, n=n, Hq=Hq, Hkv=Hkv, D=D, page=page, lengths=(41003,), explicit=explicit, seed=n))


def test_long_rows_f32(cea, dev):
    for n in (1, 20):
        for explicit in (False, True):
            _check(cea, dev, P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(9001, 300), dtype=F32,
                                    explicit=explicit, seed=n))


@pytest.mark.parametrize("n", [1, 2, 20])
@pytest.mark.parametrize("explicit", [False, True])
def test_more_rows_than_lanes(cea, dev, n, explicit):
    """More than 64 rows, of lengths from none to long, behind a wide table: runs over many rows, rows cut
    between workgroups and rows that are not."""
    lengths = [0 if b % 7 == 3 else n + (37 * b) % 61 + (1500 if b % 50 == 9 else 0) for b in range(135)]
    _check(cea, dev, P.make(B=135, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=lengths, width=130, explicit=explicit,
                            seed=18))


@pytest.mark.parametrize("n", [1, 3, 40])
def test_positions_beyond_31_bits(cea, dev, n):
    """Positions of any size, on both sides of 2^31 and far above, in one row and one tile."""
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(n + 300, n + 40), explicit=True, seed=19)
    base = 2 ** 31 - 200
    c.pos_pages = torch.where(c.pos_pages >= 0, c.pos_pages + base, c.pos_pages)
    c.q_pos += base
    for b in range(2):
        for j in (5, 60, 61):
            p, i = int(c.tables[b, j // 16 if j < int(c.lengths[b]) else 0]), j % 16
            c.pos_pages[p, i] = 2 ** 31 - 1 if j == 5 else 2 ** 62 + j
    c.q_pos[0, -1] = 2 ** 62 + 60
    _check(cea, dev, c)
    c.causal = False
    _check(cea, dev, c)


@pytest.mark.parametrize("dtype", [BF16, F32, F64])
@pytest.mark.parametrize("explicit", [False, True])
@pytest.mark.parametrize("n", [1, 3, 40])
def test_the_largest_query_position(cea, dev, dtype, explicit, n):
    """A query at the largest 64-bit position sees every key under the causal rule."""
    c = P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(n + 300, n + 5), dtype=dtype, explicit=explicit, seed=24)
    c.q_pos[0, 0] = c.q_pos[1, -1] = torch.iinfo(torch.int64).max
    if explicit:
        c.pos_pages[int(c.tables[0, 3]), 5] = torch.iinfo(torch.int64).max
    _check(cea, dev, c)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("n", [1, 60])
def test_large_scores(cea, dev, dtype, n):
    """Scores of hundreds: one key takes nearly everything, and the running maximum moves often."""
    _check(cea, dev, P.make(B=2, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(n + 400, n + 30), dtype=dtype,
                            q_scale=30.0, seed=20))


def test_same_page_in_two_rows(cea, dev):
    """Rows that share a prefix name the same pages."""
    for n in (1, 50):
        c = P.make(B=3, n=n, Hq=4, Hkv=2, D=64, page=16, lengths=(n + 200, n + 180, n + 64), seed=21)
        c.tables[1, :4], c.tables[2, :4] = c.tables[0, :4], c.tables[0, :4]
        _check(cea, dev, c)


def test_merges_with_another_share(cea, dev):
    """Two ranks' shares of the rows' keys, each in its own pool with positions, merged by their
    log-sum-exp, are the whole."""
    c = P.make(B=2, n=3, Hq=4, Hkv=2, D=64, page=16, lengths=(90, 41), seed=16)
    ref = P.reference(c)
    parts = []
    for r in (0, 1):
        s = P.to(c, dev)
        pos = torch.full((c.P, 16), -1, dtype=torch.int64)
        for b in range(2):
            for j in range(int(c.lengths[b])):
                if j // 8 % 2 == r:
                    pos[c.tables[b, j // 16], j % 16] = j
        s.pos_pages = pos.to(dev)
        parts.append(P.call(cea, s, with_lse=True))
    out, lse = cea.merge_attention_list([p[0] for p in parts], [p[1] for p in parts])
    # (each share's error is within its own bound, which the whole's covers twice over)
    ref.tol, ref.tol_lse = 3 * ref.tol, 3 * ref.tol_lse
    P.check(c, ref, out, lse, pieces_left=2.0 ** -22)


@pytest.mark.parametrize("n", [1, 30])
def test_wide_tables_without_positions_take_no_scratch_for_them(cea, dev, n):
    """64 rows of tables of 131072 slots (71 MB of positions and summaries, if there were any)."""
    c = P.make(B=64, n=n, Hq=4, Hkv=1, D=64, page=64, lengths=[n + 3 * b for b in range(64)], width=2048, seed=28)
    d = P.to(c, dev)
    P.call(cea, d)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = P.call(cea, d)
    parts = 64 * 16 * n * 4 * 65 * 4 if n > 1 else 512 * 2 * 4 * 66 * 4  # of all key splits, or of all runs
    assert torch.cuda.max_memory_allocated() - before <= out.numel() * 2 + parts + (1 << 20)
    P.check(c, P.reference(c), out)


# ---------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------
def _append_case(B, n, H, D, page, offsets, dtype, seed, counts=None, rot=True):
    g = torch.Generator().manual_seed(seed)
    k = torch.randn(B, n, H, D, generator=g, dtype=F64).to(dtype)
    v = torch.randn(B, n, H, D, generator=g, dtype=F64).to(dtype)
    W = max(1, -(-(max(offsets) + n) // page))
    pages = B * W + 2
    tables = torch.randperm(pages, generator=g)[:B * W].view(B, W)
    pos = 3 * torch.arange(n).expand(B, n) + torch.tensor(offsets).view(B, 1)
    wide = F64 if dtype == F64 else F32
    cos, sin = L.rope_tables(pos, L.inv_freq(D, 1e4, dtype=wide), dtype) if rot else (None, None)
    kp = torch.randn(pages, H, page, D, generator=g, dtype=F64).to(dtype)
    vp = torch.randn(pages, H, page, D, generator=g, dtype=F64).to(dtype)
    pp = torch.randint(-1, 99, (pages, page), generator=g)
    return k, v, pos, cos, sin, tables, torch.tensor(offsets), kp, vp, pp


def _append_ref(k, v, pos, cos, sin, tables, offsets, kp, vp, pp, counts=None):
    """The pools after the append, K in f64, and the error it may have."""
    B, n, H, D = k.shape
    page = kp.shape[2]
    kd, vp, pp, tol = kp.double(), vp.clone(), pp.clone(), torch.zeros(kp.shape, dtype=F64)
    x = k.double()
    exact, mag = x, x.abs() * 0
    if cos is not None:
        c, s = cos.double().unsqueeze(2), sin.double().unsqueeze(2)
        turned = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
        exact, mag = x * c + turned * s, (x * c).abs() + (turned * s).abs()
    u = 2.0 ** -53 if k.dtype == F64 else 2.0 ** -24
    err = P.half_step(k.dtype) * exact.abs() * (1 + u) + 3 * u * mag
    if k.dtype == F16:
        err = err + 2.0 ** -25
    if cos is None:
        err = torch.zeros_like(err)
    for b in range(B):
        for i in range(n if counts is None else min(n, int(counts[b]))):
            slot = int(offsets[b]) + i
            if not 0 <= slot < tables.shape[1] * page:
                continue
            p = int(tables[b, slot // page])
            if not 0 <= p < kp.shape[0]:
                continue
            kd[p, :, slot % page], tol[p, :, slot % page] = exact[b, i], err[b, i]
            vp[p, :, slot % page] = v[b, i]
            pp[p, slot % page] = pos[b, i]
    return kd, tol, vp, pp


def _append_check(cea, dev, case, counts=None, with_pos=True):
    want_k, tol, want_v, want_p = _append_ref(*case, counts=counts)
    k, v, pos, cos, sin, tables, offsets, kp, vp, pp = (None if t is None else t.to(dev) for t in case)
    cea.paged_kv_append(kp, vp, tables, offsets, k, v, cos=cos, sin=sin,
                        counts=None if counts is None else torch.as_tensor(counts).to(dev),
                        pos_pages=pp if with_pos else None, pos=pos if with_pos else None)
    assert bool(((kp.cpu().double() - want_k).abs() <= tol).all())
    assert torch.equal(vp.cpu(), want_v)
    assert torch.equal(pp.cpu(), want_p if with_pos else case[-1])


@pytest.mark.parametrize("dtype", [BF16, F16, F32, F64])
@pytest.mark.parametrize("rot", [True, False])
@pytest.mark.parametrize("B,n,H,D,page,offsets", [(3, 1, 8, 128, 64, (0, 63, 64)), (2, 37, 2, 64, 16, (5, 200)),
                                                  (1, 130, 4, 80, 24, (9,)), (2, 3, 1, 6, 1, (0, 4))])
def test_append(cea, dev, dtype, rot, B, n, H, D, page, offsets):
    for with_pos in (True, False):
        _append_check(cea, dev, _append_case(B, n, H, D, page, offsets, dtype, n, rot=rot), with_pos=with_pos)


def test_append_drops_what_has_no_place(cea, dev):
    """Counts, slots outside the table and pages outside the pool: nothing else is touched."""
    case = list(_append_case(5, 9, 2, 64, 16, (0, 20, 30, 3, 7), BF16, 1))
    case[5] = case[5].clone()
    case[5][3, 0] = -1
    case[5][4, 0], case[5][4, 1] = 10 ** 10, case[7].shape[0]
    case[6] = torch.tensor([-4, 20, 10 ** 14, 3, 7])
    _append_check(cea, dev, case)
    _append_check(cea, dev, _append_case(4, 6, 2, 64, 16, (0, 20, 30, 3), BF16, 2), counts=[0, 6, 3, -1])
    _append_check(cea, dev, _append_case(2, 6, 2, 64, 16, (0, 20), BF16, 2), counts=[99, 1])


def test_append_strides(cea, dev):
    """Column slices of a fused projection, tables of one row for all, token-major pages."""
    case = _append_case(2, 11, 2, 64, 16, (3, 40), BF16, 3)
    k, v, pos, cos, sin, tables, offsets, kp, vp, pp = case
    case = (k, v, pos, cos[:1].expand(2, -1, -1), sin[:1].expand(2, -1, -1), tables, offsets, kp, vp, pp)
    want_k, tol, want_v, _ = _append_ref(*case)
    fused = torch.cat([torch.zeros(2, 11, 256, dtype=BF16), k.flatten(2), v.flatten(2)], -1).to(dev)
    kd, vd = fused[..., 256:384].view(2, 11, 2, 64), fused[..., 384:].view(2, 11, 2, 64)
    kpd = kp.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    vpd = vp.transpose(1, 2).contiguous().to(dev).transpose(1, 2)
    cea.paged_kv_append(kpd, vpd, tables.to(dev), offsets.to(dev), kd, vd, cos=cos[:1].to(dev), sin=sin[:1].to(dev))
    assert bool(((kpd.cpu().double() - want_k).abs() <= tol).all()) and torch.equal(vpd.cpu(), want_v)


def test_append_is_the_contiguous_append_but_for_roundings(cea, dev):
    """Against apply_rotary and a plain copy: values and positions the same, keys within the three
    roundings of the one and the one of the other."""
    case = _append_case(2, 40, 4, 128, 16, (0, 0), BF16, 4)
    k, v, pos, cos, sin, tables, offsets, kp, vp, pp = (t.to(dev) for t in case)
    cea.paged_kv_append(kp, vp, tables, offsets, k, v, cos=cos, sin=sin)
    cache = cea.LayerKVCache()
    cache.append_rotary(k, v, pos, cos, sin)
    kc, vc, _ = cache.view()
    kg = kp[tables].transpose(2, 3).flatten(1, 2)[:, :40]
    vg = vp[tables].transpose(2, 3).flatten(1, 2)[:, :40]
    assert torch.equal(vg, vc)
    a, b = k.float() * cos.float().unsqueeze(2), k.float().roll(64, -1) * sin.float().unsqueeze(2)
    assert bool(((kg.float() - kc.float()).abs() <= 2.0 ** -8 * (a.abs() + b.abs() + 2 * kg.float().abs())).all())


def test_append_empty(cea, dev):
    z = torch.zeros(0, dtype=torch.int64, device=dev)
    kp = torch.randn(2, 2, 16, 64, device=dev)
    before = kp.clone()
    cea.paged_kv_append(kp, kp, z.view(0, 3), z, torch.zeros(0, 4, 2, 64, device=dev), torch.zeros(0, 4, 2, 64, device=dev))
    k = torch.ones(1, 0, 2, 64, device=dev)
    one = torch.zeros(1, 1, dtype=torch.int64, device=dev)
    cea.paged_kv_append(kp, kp, one, one[0], k, k)
    k = torch.ones(1, 2, 2, 64, device=dev)
    cea.paged_kv_append(kp, kp, one[:, :0], one[0], k, k)
    assert torch.equal(kp, before)


# ---------------------------------------------------------------------------------------
# page copies
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32, F64, torch.int64])
@pytest.mark.parametrize("shape,dim", [((6, 2, 16, 64), 0), ((3, 2, 7, 2, 16, 8), 2), ((5, 1), 0), ((2, 6, 3), 1),
                                       ((2, 40, 70001), 1)])
def test_copy_pages(cea, dev, dtype, shape, dim):
    pool = torch.randint(-99, 99, shape, device=dev).to(dtype)
    src, dst = [0, 3, 0], [4, 1, 2]
    want = pool.clone()
    want.index_copy_(dim, torch.tensor(dst, device=dev), pool.index_select(dim, torch.tensor(src, device=dev)))
    cea.copy_pages(pool, src, dst, dim=dim)
    assert torch.equal(pool, want)
    cea.copy_pages(pool, [], [], dim=dim)
    assert torch.equal(pool, want)


def test_copy_many_pages_through_several_pools(cea, dev):
    """More moves than one launch takes, pools of different types, pages at odd places."""
    n = 1500
    order = torch.randperm(2 * n + 5)
    src, dst = order[:n], order[n:2 * n]
    a = torch.randint(-99, 99, (2, 2 * n + 5, 3, 16), device=dev).to(BF16)
    b = torch.randint(-99, 99, (2 * n + 5, 8), device=dev).unsqueeze(0)
    c = torch.randint(-99, 99, (2 * n + 5, 48 + 1), device=dev).to(BF16)[:, 1:].unsqueeze(0)  # 2-byte aligned rows
    want = [t.clone() for t in (a, b, c)]
    for t, w in zip((a, b, c), want):
        w[:, dst.to(dev)] = t[:, src.to(dev)]
    cea.copy_pages([a, b, c], src, dst, dim=1)
    for t, w in zip((a, b, c), want):
        assert torch.equal(t, w)


def test_copy_pages_of_a_pool_with_pages_first(cea, dev):
    """[P, layers, 2, page, D], handed over as a view with the pages behind the layers."""
    pool = torch.randint(-99, 99, (7, 3, 2, 16, 8), device=dev).to(BF16)
    want = pool.clone()
    want[torch.tensor([4, 1], device=dev)] = pool[torch.tensor([0, 3], device=dev)]
    cea.copy_pages(pool.permute(1, 2, 0, 3, 4), [0, 3], [4, 1], dim=2)
    assert torch.equal(pool, want)
    with pytest.raises(ValueError, match="overlap"):
        cea.copy_pages(pool.view(-1).as_strided((2, 6, 32), (32, 32, 1)), [0], [1], dim=1)


def test_copy_pages_refusals(cea, dev):
    pool = torch.zeros(2, 6, 4, 8, device=dev)
    for src, dst in (([0], [6]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [1, 2])):
        with pytest.raises(ValueError):
            cea.copy_pages(pool, src, dst, dim=1)
    with pytest.raises(ValueError):  # pages that are not contiguous
        cea.copy_pages(pool.transpose(2, 3), [0], [1], dim=1)
    with pytest.raises(ValueError):
        cea.copy_pages(pool, [0], [1], dim=4)
    with pytest.raises(ValueError):  # lists on the device
        cea.copy_pages(pool, torch.tensor([0], device=dev), torch.tensor([1], device=dev), dim=1)
    with pytest.raises(ValueError):
        cea.copy_pages(pool, torch.tensor([0.0]), torch.tensor([1.0]), dim=1)


# ---------------------------------------------------------------------------------------
# streams, graphs, and a run of them together
# ---------------------------------------------------------------------------------------
def test_another_stream_than_the_default(cea, dev):
    for n in (1, 70):
        c = P.make(B=3, n=n, Hq=8, Hkv=2, D=64, page=16, lengths=(n + 700, n, n + 40), seed=17)
        ref = P.reference(c)
        d = P.to(c, dev)
        torch.cuda.synchronize()
        s, other = torch.cuda.Stream(), torch.cuda.Stream()
        outs = []
        for st in (s, other) * 3:
            with torch.cuda.stream(st):
                outs.append(P.call(cea, d))
        torch.cuda.synchronize()
        for o in outs:
            P.check(c, ref, o)
            assert torch.equal(o, outs[0])


@pytest.mark.parametrize("n,W,explicit", [(1, 40, False), (4, 40, True), (1, 140, False), (3, 140, True), (40, 140, False),
                                         (40, 140, True)])
def test_captured_calls_follow_their_tensors(cea, dev, n, W, explicit):
    """An append and an attention in one graph, replayed as the row grows: every replay equals the
    eager calls on the same contents, bit for bit; two graphs replayed in turn do not disturb each
    other."""
    H, D, page = 2, 64, 16
    pages = 3 * W
    g = torch.Generator().manual_seed(n)
    kp = torch.randn(pages, H, page, D, generator=g).to(BF16).to(dev)
    vp = torch.randn(pages, H, page, D, generator=g).to(BF16).to(dev)
    tables = torch.randperm(pages, generator=g)[:3 * W].view(3, W).to(dev)
    lengths = torch.tensor([300, 0, 77], device=dev)
    k, v = (torch.zeros(3, n, H, D, dtype=BF16, device=dev) for _ in range(2))
    q = torch.zeros(3, n, 8, D, dtype=BF16, device=dev)
    after = torch.zeros(3, dtype=torch.int64, device=dev)
    q_pos = torch.zeros(3, n, dtype=torch.int64, device=dev)
    steps = torch.arange(n, device=dev)
    pp = torch.arange(page, device=dev).expand(pages, page).contiguous() if explicit else None

    def step():
        after.copy_(lengths + n)
        q_pos.copy_(lengths.view(3, 1) + steps)
        cea.paged_kv_append(kp, vp, tables, lengths, k, v, pos_pages=pp, pos=q_pos if explicit else None)
        return cea.paged_attention(q, kp, vp, tables, after, q_pos, pos_pages=pp)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for i in range(6):
        for t in (k, v, q):
            t.copy_(torch.randn(t.shape, generator=g).to(BF16))
        want = step().clone()
        kept = kp.clone()
        graph, out = graphs[i % 2]
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(kp, kept)
        lengths += n
        torch.randn(1 << 16, device=dev).sum().item()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 40])
def test_two_graphs_replayed_at_once(cea, dev, dtype, n):
    """Calls that cut their rows, captured twice and replayed on two streams together, share no scratch."""
    cases = [P.to(P.make(B=2, n=n, Hq=4, Hkv=1, D=64, page=16, lengths=(2500, 1800), dtype=dtype, seed=25 + i), dev)
             for i in range(2)]
    want = [P.call(cea, c, True) for c in cases]
    torch.cuda.synchronize()
    streams, graphs, got = [torch.cuda.Stream() for _ in cases], [], []
    for c, s in zip(cases, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs = [P.call(cea, c, True) for _ in range(8)]
        graphs.append(g)
        got.append(outs)
    for _ in range(4):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for outs, ref in zip(got, want):
            for o in outs:
                assert torch.equal(o[0], ref[0]) and torch.equal(o[1], ref[1])


def test_pages_are_not_handed_out_in_a_capture(cea, dev):
    cache = cea.PagedKVCache(1, 6, 16, 2, 64, device=dev)
    a = cache.new()
    step = cache.extend([a], 5)
    q = torch.randn(1, 1, 2, 64, device=dev, dtype=BF16)
    pos = torch.tensor([[4]], device=dev)
    kv = torch.randn(1, 5, 2, 64, device=dev, dtype=BF16)
    cache.append(0, step, kv, kv)
    want = cache.attention(0, step, q, pos)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="capture"):
            cache.extend([a], 1)
        with pytest.raises(RuntimeError, match="capture"):
            cache.compact()
        out = cache.attention(0, step, q, pos)
    assert cache.length(a) == 5 and cache.free_pages == 5
    for _ in range(3):
        graph.replay()
        assert torch.equal(out, want)


@pytest.mark.parametrize("positions", [False, True])
def test_a_life_of_the_cache(cea, dev, positions):
    """Prompts, decode steps, forks, a sequence that leaves, drafts that are rejected and a
    compaction, in every layer, against contiguous caches of each sequence (test oracle)."""
    layers, H, Hq, D, page = 2, 2, 4, 64, 16
    cache = cea.PagedKVCache(layers, 64, page, H, D, device=dev, positions=positions)
    refs, g = {}, torch.Generator().manual_seed(5)
    inv = L.inv_freq(D, 1e4)

    def step(seqs, counts):
        n = max(counts)
        st = cache.extend(seqs, counts)
        B = len(seqs)
        start = [refs[s][0][0].shape[0] if refs[s] else 0 for s in seqs]
        pos = torch.tensor(start).view(B, 1) + torch.arange(n)
        pos = torch.where(torch.arange(n) < torch.tensor(counts).view(B, 1), pos, torch.full_like(pos, -1))
        cos, sin = L.rope_tables(pos.clamp(min=0), inv, BF16)
        for layer in range(layers):
            q, k, v = (torch.randn(B, n, h, D, generator=g).to(BF16) for h in (Hq, H, H))
            cache.append(layer, st, k.to(dev), v.to(dev), cos=cos.to(dev), sin=sin.to(dev),
                         pos=pos.to(dev) if positions else None)
            out = cache.attention(layer, st, q.to(dev), pos.to(dev))
            o32, lse = cache.attention_with_lse(layer, st, q.to(dev), pos.to(dev))
            torch.cuda.synchronize()
            for b, s in enumerate(seqs):
                x = k[b].float()
                c, z = cos[b].float().unsqueeze(1), sin[b].float().unsqueeze(1)
                kr = (x * c + torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1) * z).to(BF16)
                m = counts[b]
                old = refs[s][layer] if len(refs[s]) > layer else None
                kk = kr[:m] if old is None else torch.cat([old[0], kr[:m]])
                vv = v[b, :m] if old is None else torch.cat([old[1], v[b, :m]])
                if old is None:
                    refs[s].append((kk, vv))
                else:
                    refs[s][layer] = (kk, vv)
                total = kk.shape[0]
                # what the pages hold: the values, and the keys within a step (f32 products that are
                # fused or not round to one bf16 or its neighbour)
                t = torch.tensor(cache.book.table(s), dtype=torch.int64)
                kg, vg = (x[t.to(dev)].transpose(1, 2).flatten(0, 1)[:total].cpu() for x in cache.pages(layer))
                assert torch.equal(vg, vv)
                assert bool(((kg.float() - kk.float()).abs() <= 2.0 ** -7 * kk.float().abs() + 1e-6).all())
                # the same keys in one page of a pool of their own
                one = P.make(B=1, n=n, Hq=Hq, Hkv=H, D=D, page=max(total, 1), lengths=(total,), seed=0)
                if total:
                    own = int(one.tables[0, 0])
                    one.k_pages[own], one.v_pages[own] = kg.transpose(0, 1), vg.transpose(0, 1)
                one.q, one.q_pos = q[b:b + 1], pos[b:b + 1]
                ref = P.reference(one)
                P.check(one, ref, out[b:b + 1])
                P.check(one, ref, o32[b:b + 1], lse[b:b + 1], pieces_left=2.0 ** -23)

    def new():
        s = cache.new()
        refs[s] = []
        return s

    def fork(s):
        c = cache.fork(s)
        refs[c] = [tuple(t.clone() for t in kv) for kv in refs[s]]
        return c

    def cut(s, n):
        cache.truncate(s, n)
        refs[s] = [tuple(t[:n] for t in kv) for kv in refs[s]]

    a, b, c = new(), new(), new()
    step([a, b, c], [37, 5, 20])
    step([a, b, c], [1, 1, 1])
    d, e = fork(a), fork(a)
    step([a, d, e, b], [1, 1, 1, 1])
    step([d, a], [4, 4])
    cut(d, 40)
    step([d, e, a], [2, 0, 1])
    cache.free(b)
    cache.free(c)
    moved = cache.compact()
    assert moved > 0 and cache.free_pages == 64 - len({p for s in (a, d, e) for p in cache.book.table(s)})
    step([a, d, e], [1, 30, 2])


@pytest.mark.parametrize("seed", range(40))
def test_random_calls(cea, dev, seed):
    """Types, heads, page sizes, lengths, masks, layouts and bad pages drawn together."""
    rng = random.Random(1000 + seed)
    dtype = rng.choice([BF16, BF16, F16, F16, F32, F64])
    D = rng.choice([64, 64, 128, 128, 40])
    page = rng.choice([16, 32, 48, 64, 128, 20])
    Hkv, g = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 4, 8])
    Hq = Hkv * g
    n = rng.choice([1, 1, 2, 3, 5, 9, 17, 33, 65, 130, 200])
    B = rng.choice([1, 2, 3, 5])
    while B > 1 and B * n * Hq > 1600:
        B -= 1
    lengths = [rng.choice([0, n, n + rng.randint(0, 70), n + rng.randint(0, 700), rng.randint(0, 1500)]) for _ in range(B)]
    kv_map = [rng.randrange(Hkv) for _ in range(Hq)] if rng.random() < 0.2 else None
    c = P.make(B=B, n=n, Hq=Hq, Hkv=Hkv, D=D, page=page, lengths=lengths, dtype=dtype, explicit=rng.random() < 0.5,
               causal=rng.random() < 0.8, scale=rng.choice([None, None, 0.5, -0.2]), kv_map=kv_map, seed=seed,
               layout=rng.choice(["hnd", "nhd"]), stale=rng.choice([None, math.nan, math.inf]),
               width=max([-(-x // page) for x in lengths] + [1]) + rng.choice([0, 0, 1, 30]),
               pad_rows=[(rng.randrange(B), rng.randrange(n)) for _ in range(rng.choice([0, 0, 2]))])
    if rng.random() < 0.3:
        c.tables[rng.randrange(B), rng.randrange(c.W)] = rng.choice([-1, c.P, 2 ** 40])
    _check(cea, dev, c)

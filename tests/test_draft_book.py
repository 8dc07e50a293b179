"""The host side of 8-bit pages and drafted trees: the book through drafts, and the argument checks of the entry
points (no kernel runs here); the tests' own definitions against torch's e4m3."""

import ctypes
import math

import pytest
import torch

import _drafts as D
from test_abi import _t

F8 = torch.float8_e4m3fn
BF16, F16, F32, F64, I64, E4M3, U8 = 1, 2, 0, 3, 4, 5, 6


def test_the_tests_codes_are_e4m3():
    c = torch.arange(256, dtype=torch.uint8)
    want = c.view(F8).double()
    got = D.values(c, torch.full((), 127, dtype=torch.uint8))
    ok = ~torch.isnan(want)
    assert torch.equal(torch.isnan(got), ~ok) and torch.equal(got[ok], want[ok])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_the_tests_rounding_is_e4m3s(dtype):
    """Rows in their own scale, rounded by the tests' definition and by torch's conversion."""
    g = torch.Generator().manual_seed(0)
    x = (torch.randn(300, 64, generator=g) * 2.0 ** torch.randint(-12, 10, (300, 1), generator=g)).to(dtype).float()
    q, s = D.quantise(x, dtype)
    e = s.double().unsqueeze(-1) - 127
    top = x.double().abs().amax(-1, keepdim=True)
    assert bool((top <= 448 * 2.0 ** e).all()) and bool((top > 448 * 2.0 ** (e - 1)).all())
    assert torch.equal(q, (x.double() * 2.0 ** -e).float().to(F8).view(torch.uint8))
    err = (D.values(q, s) - x.double()).abs()
    assert bool((err <= torch.maximum(x.double().abs() * 2.0 ** -4, 2.0 ** (e - 10))).all())


def test_words_and_ancestors():
    p = torch.tensor([[-1, 0, 0, 2, 7, 1]])
    seen = D.ancestors(p)
    assert seen[0].long().tolist() == [[1, 0, 0, 0, 0, 0], [1, 1, 0, 0, 0, 0], [1, 0, 1, 0, 0, 0], [1, 0, 1, 1, 0, 0],
                                       [0, 0, 0, 0, 1, 0], [1, 1, 0, 0, 0, 1]]
    assert D.words(seen)[0, :, 0].tolist() == [1, 3, 5, 13, 16, 35]
    wide = torch.zeros(1, 65, 65, dtype=torch.bool)
    wide[0, 0, 63], wide[0, 0, 64] = True, True
    assert D.words(wide)[0, 0].tolist() == [-(1 << 63), 1]


def _cache(cea, **kw):
    return cea.PagedKVCache(2, 10, 4, 1, 8, device="cpu", **kw)


def test_keep_is_checked_before_anything_moves(cea):
    c = _cache(cea)
    a, b = c.new(), c.new()
    step = c.extend([a, b], [6, 3])
    path = torch.zeros(2, 4, dtype=torch.int64)
    for kept in ([1], [7, 0], [5, 0], [0, 4], [-1, 0]):
        with pytest.raises(ValueError):
            c.keep(step, path, kept)
    for bad in (path[:1], path[0]):
        with pytest.raises(ValueError):
            c.keep(step, bad, [1, 1])
    with pytest.raises(TypeError):
        c.keep(step, path, [1.5, 1])
    with pytest.raises(RuntimeError):  # (host pools: nothing moves, and nothing is dropped)
        c.keep(step, path, [1, 1])
    assert c.length(a) == 6 and c.length(b) == 3
    later = c.extend([b], 1)
    with pytest.raises(RuntimeError, match="extended"):
        c.keep(step, path, [1, 1])
    c.fork(a)
    for s in (step, later):
        with pytest.raises(RuntimeError, match="older"):
            c.keep(s, path, [1, 1])
    with pytest.raises(RuntimeError, match="not this cache"):
        _cache(cea).keep(step, path, [1, 1])


def test_trees_need_a_cache_without_positions_and_all_nodes(cea):
    c = _cache(cea, positions=True)
    step = c.extend([c.new()], 3)
    q, m = torch.zeros(1, 3, 1, 8, dtype=torch.bfloat16), torch.zeros(1, 3, 1, dtype=torch.int64)
    with pytest.raises(NotImplementedError):
        c.tree_attention(0, step, q, m)
    with pytest.raises(NotImplementedError):
        c.keep(step, m[..., 0], [1])
    c = _cache(cea)
    step = c.extend([c.new()], 3)
    with pytest.raises(ValueError, match="up to 3"):
        c.tree_attention(0, step, q[:, :2], m[:, :2])


def test_scales_belong_to_8_bit_caches(cea):
    c = _cache(cea, dtype=F8)
    assert c.scales.shape == (2, 2, 10, 1, 4) and c.scales.dtype == torch.uint8
    assert _cache(cea).scales is None
    q = torch.zeros(1, 1, 1, 8, dtype=torch.bfloat16)
    kp, sc = torch.zeros(3, 1, 4, 8, dtype=F8), torch.zeros(3, 1, 4, dtype=torch.uint8)
    t, n, p = torch.zeros(1, 1, dtype=torch.int64), torch.ones(1, dtype=torch.int64), torch.zeros(1, 1, dtype=torch.int64)
    for kw in ({}, {"k_scales": sc}, {"v_scales": sc}):
        with pytest.raises(ValueError):
            cea.paged_attention(q, kp, kp, t, n, p, **kw)
        with pytest.raises(ValueError):
            cea.paged_kv_append(kp, kp, t, n, q, q, **kw)
        with pytest.raises(ValueError):
            cea.paged_kv_read(kp, kp, t, n, 1, **kw)
        with pytest.raises(ValueError):
            cea.paged_tree_attention(q, kp, kp, t, n, n, p.unsqueeze(-1), **kw)
    half = kp.to(torch.bfloat16)
    with pytest.raises(ValueError):
        cea.paged_attention(q, half, half, t, n, p, k_scales=sc, v_scales=sc)
    with pytest.raises(ValueError):
        cea.paged_kv_read(half, half, t, n, 1, dtype=torch.float16)
    with pytest.raises(TypeError):
        cea.paged_kv_read(half, half, t, n, 1.5)


def test_host_tensors_are_refused(cea):
    q = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16)
    kp, sc = torch.zeros(3, 1, 4, 8, dtype=F8), torch.zeros(3, 1, 4, dtype=torch.uint8)
    t, n = torch.zeros(1, 1, dtype=torch.int64), torch.ones(1, dtype=torch.int64)
    m = torch.zeros(1, 2, 1, dtype=torch.int64)
    s = {"k_scales": sc, "v_scales": sc}
    for call in (lambda: cea.paged_kv_append(kp, kp, t, n, q, q, **s),
                 lambda: cea.paged_kv_read(kp, kp, t, n, 2, **s),
                 lambda: cea.paged_attention(q, kp, kp, t, n, m[..., 0], **s),
                 lambda: cea.paged_tree_attention(q, kp, kp, t, n, n, m, **s),
                 lambda: cea.paged_tree_attention_with_lse(q, kp, kp, t, n, n, m, **s),
                 lambda: cea.tree_masks(m[..., 0]),
                 lambda: cea.paged_kv_keep(kp, t, n, t, scales=sc)):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()


# ---------------------------------------------------------------------------------------
# the C ABI: bad arguments, before anything is launched
# ---------------------------------------------------------------------------------------
def _refused(cea, name, code, *args):
    lib = cea._native.load_library()
    rc = getattr(lib, name)(*[ctypes.byref(a) if isinstance(a, cea._native.CeaTensor) else a for a in args])
    assert rc == code, (name, rc, cea._native.last_error())
    assert cea._native.last_error()


EINVAL, EUNSUPPORTED, ENOSPACE = -1, -2, -4


def _args(T=3, dt=BF16, B=2, W=4, P=9, H=2, page=16, D=64, Hq=4):
    a = dict(q=_t((B, T, Hq, D), dt), kp=_t((P, H, page, D), E4M3), vp=_t((P, H, page, D), E4M3), ks=_t((P, H, page), U8),
             vs=_t((P, H, page), U8), tables=_t((B, W), I64), lengths=_t((B,), I64), counts=_t((B,), I64),
             q_pos=_t((B, T), I64), masks=_t((B, T, (T + 63) // 64), I64), out=_t((B, T, Hq, D), dt), k=_t((B, T, H, D), dt),
             cos=_t((B, T, D), dt), path=_t((B, 5), I64), parents=_t((B, T), I64), depths=_t((B, T), I64),
             kv=_t((6, P, H, page * D), E4M3), sc=_t((6, P, H, page), U8))
    return a


def _attend8(cea, code, **over):
    a = {**_args(), **over}
    _refused(cea, "cea_paged_attention8", code, a["q"], a["kp"], a["vp"], a["ks"], a["vs"], None, a["tables"], a["lengths"],
             a["q_pos"], 1, 0.1, None, 0, a["out"], None, None, 0, None)


def test_attention8_refusals(cea):
    _attend8(cea, EINVAL, ks=None)
    _attend8(cea, EINVAL, ks=_t((9, 2, 15), U8))
    _attend8(cea, EINVAL, vs=_t((9, 2, 16), I64))
    _attend8(cea, EINVAL, kp=_t((9, 2, 16, 64), BF16))
    _attend8(cea, EINVAL, vp=_t((9, 2, 16, 64), U8))
    _attend8(cea, EINVAL, kp=_t((9, 3, 16, 64), E4M3))
    _attend8(cea, EINVAL, lengths=_t((3,), I64))
    _attend8(cea, EUNSUPPORTED, q=_t((2, 3, 4, 64), F64), out=_t((2, 3, 4, 64), F64))
    _attend8(cea, EUNSUPPORTED, q=_t((2, 3, 4, 64), E4M3))
    big = _args(T=40, W=4096)  # (a form with scratch, and none given)
    _attend8(cea, ENOSPACE, **{k: big[k] for k in ("q", "out", "q_pos", "tables")})


def _tree(cea, code, **over):
    a = {**_args(), **over}
    _refused(cea, "cea_paged_tree_attention", code, a["q"], a["kp"], a["vp"], a["ks"], a["vs"], a["tables"], a["lengths"],
             a["counts"], a["masks"], 0.1, None, 0, a["out"], None, None, 0, None)


def test_tree_refusals(cea):
    _tree(cea, EINVAL, masks=None)
    _tree(cea, EINVAL, counts=None)
    _tree(cea, EINVAL, masks=_t((2, 3, 2), I64))
    _tree(cea, EINVAL, masks=_t((1, 3, 1), I64))
    _tree(cea, EINVAL, masks=_t((2, 3, 1), U8))
    _tree(cea, EINVAL, counts=_t((1,), I64))
    _tree(cea, EINVAL, vs=None)
    _tree(cea, EINVAL, ks=None, vs=None)  # (8-bit pages without scales)
    many = _args(T=513)
    _tree(cea, EUNSUPPORTED, **{k: many[k] for k in ("q", "out", "masks")})


def test_append8_refusals(cea):
    def go(code, **over):
        a = {**_args(), "v": None, **over}
        v = a["v"] or a["k"]
        _refused(cea, "cea_paged_kv_append8", code, a["k"], v, None, a["cos"], a["cos"], a["tables"], a["lengths"], None,
                 a["kp"], a["vp"], a["ks"], a["vs"], None, None)

    go(EINVAL, ks=None)
    go(EINVAL, vs=_t((9, 2, 17), U8))
    go(EINVAL, kp=_t((9, 2, 16, 64), BF16))
    go(EINVAL, v=_t((2, 3, 2, 32), BF16))
    go(EINVAL, cos=_t((2, 3, 64), F32))
    go(EUNSUPPORTED, k=_t((2, 3, 2, 64), F64), cos=_t((2, 3, 64), F64))
    odd = _args(D=63)
    go(EINVAL, **{k: odd[k] for k in ("k", "kp", "vp", "cos")})


def test_read_refusals(cea):
    def go(code, **over):
        a = {**_args(), **over}
        _refused(cea, "cea_paged_kv_read", code, a["kp"], a["vp"], a["ks"], a["vs"], a["tables"], a["lengths"], a["counts"],
                 a["k"], a.get("v2") or a["k"], None)

    go(EINVAL, ks=None)
    go(EINVAL, ks=None, vs=None)
    go(EINVAL, k=_t((3, 3, 2, 64), BF16))
    go(EINVAL, k=_t((2, 3, 3, 64), BF16))
    go(EINVAL, v2=_t((2, 3, 2, 64), F16))
    go(EINVAL, counts=_t((3,), I64))
    go(EUNSUPPORTED, k=_t((2, 3, 2, 64), F64))


def test_masks_refusals(cea):
    def go(code, **over):
        a = {**_args(), **over}
        _refused(cea, "cea_tree_masks", code, a["parents"], a["counts"], a["masks"], a["depths"], None)

    go(EINVAL, masks=_t((2, 3, 2), I64))
    go(EINVAL, depths=_t((2, 4), I64))
    go(EINVAL, parents=_t((2, 3), F32))
    go(EINVAL, counts=_t((4,), I64))
    many = _args(T=513)
    go(EUNSUPPORTED, **{k: many[k] for k in ("parents", "masks", "depths")})


def test_keep_refusals(cea):
    def go(code, page=16, **over):
        a = {**_args(), **over}
        _refused(cea, "cea_paged_kv_keep", code, a["kv"], a["sc"], page, a["tables"], a["lengths"], a["counts"], a["path"], None)

    go(EINVAL, page=15)
    go(EINVAL, page=-1)
    go(EINVAL, sc=None)
    go(EINVAL, sc=_t((6, 9, 2, 15), U8))
    go(EINVAL, kv=_t((6, 9, 2, 1024), BF16))
    go(EINVAL, path=_t((3, 5), I64))
    go(EINVAL, counts=_t((3,), I64))
    twice = _t((6, 9, 2, 1024), E4M3)
    twice.stride[0] = 0
    go(EINVAL, kv=twice)
    near = _t((6, 9, 2, 16), U8)
    near.stride[1] = 16
    go(EINVAL, sc=near)


def test_other_entry_points_still_refuse_8_bit_tensors(cea):
    lib, nat = cea._native.load_library(), cea._native
    x = _t((4, 64), E4M3)
    assert lib.cea_rmsnorm(ctypes.byref(x), ctypes.byref(_t((64,), E4M3)), 1e-6, ctypes.byref(x), None) < 0
    a = _args()
    assert lib.cea_paged_attention(*[ctypes.byref(a[k]) for k in ("q", "kp", "vp")], None,
                                   *[ctypes.byref(a[k]) for k in ("tables", "lengths", "q_pos")], 1, 0.1, None, 0,
                                   ctypes.byref(a["out"]), None, None, 0, None) == EINVAL

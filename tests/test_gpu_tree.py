"""GPU tests of drafted trees: masks, attention, and the accepted nodes moved into line (tests/_drafts.py)."""

from __future__ import annotations

import importlib
import math

import pytest
import torch

import _drafts as D
import _paged as P

pytestmark = pytest.mark.gpu

BF16, F16, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
F8 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------
# masks
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,T", [(1, 1), (3, 2), (2, 26), (5, 63), (2, 64), (1, 65), (4, 128), (2, 250), (1, 512)])
def test_masks(cea, dev, B, T):
    for p in (D.parents(B, T, T), torch.arange(T).expand(B, T) - 1, torch.full((B, T), -1), D.parents(B, T, 1, T, 0.0)):
        masks, depths = cea.tree_masks(p.to(dev))
        seen = D.ancestors(p)
        assert torch.equal(masks.cpu(), D.words(seen))
        assert torch.equal(depths.cpu(), seen.sum(-1) - 1)


def test_masks_of_padded_rows_and_strange_parents(cea, dev):
    p = D.parents(4, 70, 3)
    p[0, 5], p[0, 6], p[1, 0], p[2, 69] = 5, 60, 1 << 40, -(1 << 62)  # itself, a later node, none at all
    counts = torch.tensor([70, 0, -4, 33])
    for n in (counts, torch.tensor([1 << 50, 1, 64, 65])):
        masks, depths = cea.tree_masks(p.to(dev), n.to(dev))
        seen = D.ancestors(p, n)
        assert torch.equal(masks.cpu(), D.words(seen))
        assert torch.equal(depths.cpu(), (seen.sum(-1) - 1).clamp(min=0))
    masks, _ = cea.tree_masks(p.to(dev).t().contiguous().t())
    assert torch.equal(masks.cpu(), D.words(D.ancestors(p)))


# ---------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("T,lengths,Hq,Hkv,d,page", [
    (1, (300, 1, 64), 8, 2, 128, 16), (3, (50, 3, 200), 8, 2, 64, 32), (5, (90, 5), 4, 4, 128, 16), (16, (33, 500), 2, 2, 64, 16),
    (26, (777, 26), 8, 1, 64, 16), (60, (200, 60, 333), 8, 2, 128, 64), (64, (64, 129), 4, 2, 64, 48), (65, (300,), 2, 1, 128, 16),
    (130, (131, 400), 4, 1, 64, 16), (200, (1000,), 2, 2, 128, 128), (26, (100, 30), 6, 2, 80, 16), (26, (100, 30), 4, 2, 64, 20)])
def test_tree(cea, dev, bits, dtype, T, lengths, Hq, Hkv, d, page):
    D.check(cea, dev, D.make_tree(T, lengths, bits=bits, Hq=Hq, Hkv=Hkv, D=d, page=page, dtype=dtype, seed=T))


def test_tree_f64(cea, dev):
    D.check(cea, dev, D.make_tree(20, (50, 20), Hq=4, Hkv=2, D=64, dtype=F64))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [4, 40, 100])
def test_padded_rows(cea, dev, bits, dtype, T):
    """Rows with fewer nodes than the call holds, none, negative counts, a tree that is all there is."""
    D.check(cea, dev, D.make_tree(T, (300, 80, 7, 40, 2), counts=(T, T // 2, 0, -3, 2), bits=bits, Hq=8, Hkv=2, D=128, dtype=dtype))


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T", [6, 70])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_any_mask(cea, dev, bits, T, dtype):
    """Bits of no tree: none at all (a node over the sequence alone, or over nothing), all of them, later nodes'."""
    g = torch.Generator().manual_seed(T)
    seen = torch.rand(3, T, T, generator=g) < 0.3
    seen[:, 0], seen[:, 1], seen[:, 2] = False, True, torch.arange(T) > 2
    for lengths in ((200, T, 150), (T, T + 1, 64 + T)):
        c = D.make_tree(T, lengths, seen=seen, bits=bits, Hq=4, Hkv=2, D=64, dtype=dtype)
        D.check(cea, dev, c)
        # bits beyond the nodes, and counts beyond the call's nodes
        if T % 64:
            c.masks[..., -1] |= -1 << (T % 64)
            D.check(cea, dev, c)
        c.counts = c.counts + 3
        c.lengths = torch.maximum(c.lengths, c.counts)
        c.lengths = torch.minimum(c.lengths, torch.full_like(c.lengths, c.W * c.page))
        D.check(cea, dev, c)


def test_every_node_sees_the_base_and_nothing_else(cea, dev):
    """With empty masks a tree's result is plain attention over what precedes it, bit for bit in f32 results' bounds."""
    T = 30
    c = D.make_tree(T, (130, 90), seen=torch.zeros(2, T, T, dtype=torch.bool), Hq=8, Hkv=2, D=128)
    out, lse = D.call(cea, c, dev, with_lse=True)
    ref = D.reference(c)
    P.check(c, ref, out, lse, pieces_left=2.0 ** -23)
    c2 = D.make_tree(T, (T, T), seen=torch.zeros(2, T, T, dtype=torch.bool), Hq=8, Hkv=2, D=128)
    out, lse = D.call(cea, c2, dev, with_lse=True)
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("bits", [16, 8])
def test_a_chain_is_causal_attention(cea, dev, bits):
    for T in (7, 40):
        c = D.make_tree(T, (150, 77), seen=torch.ones(2, T, T).tril().bool(), bits=bits, Hq=8, Hkv=2, D=64, seed=T)
        tree = D.call(cea, c, dev, with_lse=True)
        del c.seen
        plain = D.call(cea, c, dev, with_lse=True)
        for a, b in zip(tree, plain):
            assert (a - b).abs().max().item() <= 1e-5 * b.abs().max().item()


@pytest.mark.parametrize("T", [5, 50])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_hidden_values_that_are_not_finite(cea, dev, T, dtype):
    """Infinities and NaN in the slots behind the row, and in nodes that others do not see."""
    for bad in (math.nan, math.inf, -math.inf):
        seen = torch.ones(2, T, T).tril().bool()
        seen[:, :, 2] = False
        seen[0, 2, 2] = True
        c = D.make_tree(T, (100, T), seen=seen, Hq=4, Hkv=2, D=64, dtype=dtype, stale=bad)
        for b, at in ((0, 100 - T + 2), (1, 2)):
            p = int(c.tables[b, at // 16])
            c.v_pages[p, :, at % 16] = bad
        out = D.call(cea, c, dev).cpu()
        ok = torch.ones(2, T, dtype=torch.bool)
        ok[0, 2] = False
        assert bool(torch.isfinite(out[ok]).all())
        assert bool((~torch.isfinite(out[0, 2])).all())
        c.v_pages = torch.where(torch.isfinite(c.v_pages.float()), c.v_pages, torch.zeros_like(c.v_pages))
        c.k_pages = torch.where(torch.isfinite(c.k_pages.float()), c.k_pages, torch.zeros_like(c.k_pages))
        ref = D.reference(c)
        half = 0.0 if dtype == F32 else P.half_step(dtype)
        bound = ref.tol + half * ref.mass + P.half_step(out.dtype) * ref.out.abs() + 2.0 ** -25
        assert bool(((out.double() - ref.out).abs() <= bound)[ok].all())


def test_long_context(cea, dev):
    D.check(cea, dev, D.make_tree(20, (6000, 900), Hq=4, Hkv=1, D=128, page=64))
    D.check(cea, dev, D.make_tree(3, (5000,), Hq=4, Hkv=1, D=64, bits=8))
    D.check(cea, dev, D.make_tree(20, (4444,), Hq=4, Hkv=1, D=64, bits=8, dtype=F16))
    D.check(cea, dev, D.make_tree(18, (2500, 30), Hq=2, Hkv=1, D=64, dtype=F32))


@pytest.mark.parametrize("bits", [16, 8])
def test_strides_maps_scales(cea, dev, bits):
    """Masks of other strides and one for all rows, an explicit head map, a negative scale, missing pages."""
    for T in (6, 40):
        c = D.make_tree(T, (90, 140), bits=bits, Hq=6, Hkv=3, D=64, kv_map=[2, 0, 1, 1, 0, 2], scale=-0.2)
        c.tables[0, 1] = -1
        D.check(cea, dev, c)
        c.seen[1] = c.seen[0]
        one = D.words(c.seen)[:1]
        c.masks = one
        D.check(cea, dev, c)
        wide = torch.zeros(2, T, 3, dtype=torch.int64)
        wide[:, :, 1:2] = one
        c.masks = wide[:, :, 1:2]
        D.check(cea, dev, c)


# ---------------------------------------------------------------------------------------
# keeping nodes
# ---------------------------------------------------------------------------------------
def _keep(cea, dev, lead, P_, H, page, d, dtype, path, offsets, tables, counts=None):
    g = torch.Generator().manual_seed(7)
    if dtype == F8:
        kv = torch.randint(0, 256, (*lead, P_, H, page, d), generator=g, dtype=torch.uint8)
        scales = torch.randint(0, 256, (*lead, P_, H, page), generator=g, dtype=torch.uint8)
    else:
        kv, scales = torch.randn(*lead, P_, H, page, d, generator=g, dtype=F64).to(dtype), None
    dkv, dsc = kv.to(dev), None if scales is None else scales.to(dev)
    cea.paged_kv_keep(dkv.view(F8) if dtype == F8 else dkv, tables.to(dev), offsets.to(dev), path.to(dev), scales=dsc,
                      counts=None if counts is None else counts.to(dev))
    want = [kv.clone(), None if scales is None else scales.clone()]
    for b in range(path.shape[0]):
        for i, node in enumerate(path[b].tolist()):
            if node < i or (counts is not None and node >= int(counts[b])):
                continue
            at = []
            for j in (int(offsets[b]) + node, int(offsets[b]) + i):
                p = int(tables[b, j // page]) if 0 <= j < tables.shape[1] * page else -1
                at.append((p, j % page) if 0 <= p < P_ else None)
            if None in at:
                continue
            (p, x), (q, y) = at
            want[0][..., q, :, y, :] = kv[..., p, :, x, :]
            if scales is not None:
                want[1][..., q, :, y] = scales[..., p, :, x]
    assert torch.equal(dkv.cpu(), want[0])
    if scales is not None:
        assert torch.equal(dsc.cpu(), want[1])


@pytest.mark.parametrize("dtype,d", [(BF16, 64), (F16, 128), (F32, 20), (F64, 6), (F8, 64), (F8, 80), (F8, 6), (BF16, 3)])
@pytest.mark.parametrize("lead", [(), (3,), (2, 2)])
def test_keep(cea, dev, dtype, d, lead):
    path = torch.tensor([[0, 1, 4, 9, -1], [3, 5, 6, 7, 20], [-1, -1, -1, -1, -1], [0, 1, 2, 3, 4], [1, 30, -1, 5, -1]])
    tables = torch.randperm(23, generator=torch.Generator().manual_seed(1))[:20].view(5, 4)
    offsets = torch.tensor([0, 13, 20, 3, 15])
    _keep(cea, dev, lead, 23, 2, 16, d, dtype, path, offsets, tables)
    _keep(cea, dev, lead, 23, 2, 16, d, dtype, path, offsets, tables, counts=torch.tensor([9, 6, 0, 100, 31]))


def test_keep_of_long_paths_and_strange_places(cea, dev):
    """More entries than a thread's turn, the same node twice, any order above the line, slots without pages."""
    path = torch.stack([torch.arange(40) * 2, torch.arange(40) + 1, 79 - torch.arange(40), torch.full((40,), 60)])
    path[3, 20:] = 1 << 40
    tables = torch.arange(24).view(4, 6)
    tables[1, 2], tables[2, 5] = -1, 1 << 33
    for offsets in ((0, 5, 16, 17), (-5, 1 << 62, -(1 << 63), 90)):
        _keep(cea, dev, (2,), 24, 3, 16, 64, BF16, path, torch.tensor(offsets), tables)
        _keep(cea, dev, (2,), 24, 3, 16, 64, F8, path, torch.tensor(offsets), tables)


# ---------------------------------------------------------------------------------------
# as they are used together
# ---------------------------------------------------------------------------------------
def _tables_of(pos, d, dtype):
    inv = 1.0 / 1e4 ** (torch.arange(0, d, 2, device=pos.device, dtype=F64) / d)
    a = torch.cat([pos.double().unsqueeze(-1) * inv] * 2, -1)
    return a.cos().to(dtype), a.sin().to(dtype)


@pytest.mark.parametrize("bits", [16, 8])
def test_draft_verify_keep(cea, dev, bits):
    """A prompt, a tree of drafts, the accepted line kept: what the cache then holds and attends is what appending the
    accepted tokens one by one would have left, bit by bit."""
    L, H, Hq, d, page, T = 3, 2, 8, 64, 16, 20
    g = torch.Generator().manual_seed(bits)
    kv_dtype = F8 if bits == 8 else BF16
    lens = [37, 16, 5]
    caches = [cea.PagedKVCache(L, 40, page, H, d, dtype=kv_dtype, device=dev) for _ in range(2)]
    seqs = [[c.new() for _ in lens] for c in caches]
    rand = lambda *s: torch.randn(*s, generator=g).to(dev, BF16)
    prompt = [[rand(len(lens), max(lens), H, d) for _ in "kv"] for _ in range(L)]
    pos = torch.arange(max(lens), device=dev).expand(len(lens), -1)
    cos, sin = _tables_of(pos, d, BF16)
    for c, s in zip(caches, seqs):
        step = c.extend(s, lens)
        for layer in range(L):
            c.append(layer, step, *prompt[layer], cos=cos, sin=sin)
    parents = D.parents(len(lens), T, 4).to(dev)
    nodes = [T, 13, T]
    masks, depths = cea.tree_masks(parents, torch.tensor(nodes, device=dev))
    drafts = [[rand(len(lens), T, H, d) for _ in "kv"] for _ in range(L)]
    cos, sin = _tables_of(torch.tensor(lens, device=dev).view(-1, 1) + depths, d, BF16)
    a, sa = caches[0], seqs[0]
    step = a.extend(sa, nodes)
    q = rand(len(lens), T, Hq, d)
    outs = []
    for layer in range(L):
        a.append(layer, step, *drafts[layer], cos=cos, sin=sin)
        outs.append(a.tree_attention(layer, step, q, masks))
    # the deepest node's line is accepted, in the second row nothing
    seen = D.ancestors(parents.cpu(), nodes)
    path = torch.full((len(lens), T), -1, dtype=torch.int64)
    kept = []
    for b in range(len(lens)):
        line = [] if b == 1 else torch.nonzero(seen[b, int(depths[b].argmax())]).flatten().tolist()
        path[b, :len(line)] = torch.tensor(line, dtype=torch.int64)
        kept.append(len(line))
    path = path[:, :max(kept)]
    a.keep(step, path.to(dev), kept)
    assert [a.length(s) for s in sa] == [n + k for n, k in zip(lens, kept)]
    with pytest.raises(RuntimeError):
        a.attention(0, step, q, pos[:, :T])
    # the other cache appends the line's tokens as tokens
    b_, sb = caches[1], seqs[1]
    step_b = b_.extend(sb, kept)
    at = path.clamp(min=0).to(dev)
    rows = torch.arange(len(lens), device=dev).view(-1, 1)
    posb = torch.tensor(lens, device=dev).view(-1, 1) + torch.arange(path.shape[1], device=dev)
    cosb, sinb = _tables_of(posb, d, BF16)
    for layer in range(L):
        b_.append(layer, step_b, *(x[rows, at] for x in drafts[layer]), cos=cosb, sin=sinb)
    n = max(lens) + T
    sa_step, sb_step = a.extend(sa, 0), b_.extend(sb, 0)
    for layer in range(L):
        for x, y in zip(a.read(layer, sa_step, n), b_.read(layer, sb_step, n)):
            assert torch.equal(x, y)
        # and a node of the line saw, as a tree's node, what it sees now as a token
        now = b_.attention(layer, b_.extend(sb, 0), q[rows, at], torch.where(path.to(dev) >= 0, posb, -1))
        for r in (0, 2):
            was = outs[layer][r, path[r, :kept[r]].to(dev)]
            assert (was.float() - now[r, :kept[r]].float()).abs().max().item() <= 2.0 ** -6 * now.float().abs().max().item()


def test_keep_refuses(cea, dev):
    c = cea.PagedKVCache(1, 8, 16, 1, 64, device=dev)
    s = [c.new(), c.new()]
    step = c.extend(s, [5, 3])
    path = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    for bad in ([1], [6, 0], [5, 0], [0, 4], [-1, 0]):
        with pytest.raises(ValueError):
            c.keep(step, path, bad)
    assert [c.length(x) for x in s] == [5, 3]
    other = c.extend(s, 1)
    with pytest.raises(RuntimeError):
        c.keep(step, path, [1, 1])
    with pytest.raises(RuntimeError):  # (this step adds one token behind the first's)
        cea.PagedKVCache(1, 8, 16, 1, 64, device=dev).keep(other, path, [1, 1])
    c.keep(other, path, [1, 0])
    assert [c.length(x) for x in s] == [6, 3]
    p = cea.PagedKVCache(1, 8, 16, 1, 64, device=dev, positions=True)
    step = p.extend([p.new()], 3)
    with pytest.raises(NotImplementedError):
        p.keep(step, path[:1], [1])


def test_forks_and_compaction_carry_scales(cea, dev):
    c = cea.PagedKVCache(2, 12, 16, 3, 64, dtype=F8, device=dev)
    g = torch.Generator().manual_seed(0)
    a, b = c.new(), c.new()
    step = c.extend([a, b], [20, 40])
    for layer in range(2):
        c.append(layer, step, *(torch.randn(2, 40, 3, 64, generator=g).to(dev, F16) for _ in "kv"))
    read = lambda seq: [t.clone() for l in range(2) for t in c.read(l, c.extend([seq], 0), 40)]
    was = read(b)
    child = c.fork(b)
    step = c.extend([child], 1)  # (the shared last page is copied)
    for layer in range(2):
        c.append(layer, step, *(torch.randn(1, 1, 3, 64, generator=g).to(dev, F16) for _ in "kv"))
    c.free(a)
    c.compact()
    for x, y, z in zip(was, read(b), read(child)):
        assert torch.equal(x, y) and torch.equal(x, z)


@pytest.mark.parametrize("bits", [16, 8])
def test_captured_step(cea, dev, bits):
    """Masks, append, tree attention and the move in one graph, replayed with other trees, lengths and paths."""
    H, Hq, d, page, T, B = 2, 8, 64, 16, 12, 2
    g = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=g).to(dev, BF16)
    if bits == 8:
        kv0 = torch.randint(0, 100, (2, 20, H, page, d), generator=g, dtype=torch.uint8).to(dev).view(F8)
        sc0 = torch.randint(118, 124, (2, 20, H, page), generator=g, dtype=torch.uint8).to(dev)
    else:
        kv0, sc0 = rand(2, 20, H, page, d), None
    tables = torch.randperm(20, generator=g)[:14].view(B, 7).to(dev)
    parents, path = torch.empty(B, T, dtype=torch.int64, device=dev), torch.empty(B, 4, dtype=torch.int64, device=dev)
    offsets, counts, lengths = (torch.empty(B, dtype=torch.int64, device=dev) for _ in range(3))
    k, v, q = (torch.empty(B, T, n, d, dtype=BF16, device=dev) for n in (H, H, Hq))
    kv, sc = kv0.clone(), None if sc0 is None else sc0.clone()
    kw = {} if sc is None else {"k_scales": sc[0], "v_scales": sc[1]}

    def fill(i):
        parents.copy_(D.parents(B, T, i))
        path.copy_(torch.tensor([[0, 2, 5, 7], [1, 3, -1, -1]]) + (i % 2))
        offsets.copy_(torch.tensor([30 + i, 3 * i]))
        counts.copy_(torch.tensor([T, T - i]))
        lengths.copy_(offsets + counts)
        for t in (k, v, q):
            t.copy_(rand(*t.shape))
        kv.view(torch.uint8).copy_(kv0.view(torch.uint8)) if sc is not None else kv.copy_(kv0)
        if sc is not None:
            sc.copy_(sc0)

    def step():
        masks, _ = cea.tree_masks(parents, counts)
        cea.paged_kv_append(kv[0], kv[1], tables, offsets, k, v, counts=counts, **kw)
        out = cea.paged_tree_attention(q, kv[0], kv[1], tables, lengths, counts, masks, **kw)
        cea.paged_kv_keep(kv, tables, offsets, path, counts=counts, scales=sc)
        return out, *cea.paged_kv_read(kv[0], kv[1], tables, torch.zeros_like(offsets), 60, counts=lengths, **kw)

    fill(0)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(5):
        fill(i)
        want = [t.clone() for t in step()]
        fill_state = (kv, sc)
        kv.view(torch.uint8).copy_(kv0.view(torch.uint8)) if sc is not None else kv.copy_(kv0)
        if sc is not None:
            sc.copy_(sc0)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), i


def test_other_stream(cea, dev):
    c = D.make_tree(30, (400, 90), bits=8, Hq=8, Hkv=2, D=128)
    want = D.call(cea, c, dev)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = D.call(cea, c, dev)
    s.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------------------
# rows cut into runs that cross them, and many rows
# ---------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits,dtype", [(16, BF16), (8, BF16), (8, F16)])
def test_runs_across_rows(cea, dev, bits, dtype):
    """Long uneven rows of many heads: a workgroup's run of tiles ends one row and starts the next."""
    T = 18
    c = D.make_tree(T, (4000, 0, 300, 5003, 18), counts=(T, 0, 7, T, T), bits=bits, Hq=64, Hkv=64, D=64, page=16, dtype=dtype)
    D.check(cea, dev, c)


@pytest.mark.parametrize("explicit", [False, True])
def test_runs_of_8_bit_chunks(cea, dev, explicit):
    c = D.pool8(P.make(B=4, n=18, Hq=64, Hkv=64, D=64, page=32, lengths=(5000, 40, 0, 4100), explicit=explicit,
                       pad_rows=[(0, 17), (1, 0)]), 3)
    D.check(cea, dev, c)


def test_runs_with_values_that_are_not_finite(cea, dev):
    """The second time over a row's tiles, between the rows of a run."""
    T = 18
    seen = torch.ones(3, T, T).tril().bool()
    c = D.make_tree(T, (4000, 300, 5003), seen=seen, Hq=64, Hkv=64, D=64, page=16)
    want = D.call(cea, c, dev).cpu()
    for b, at in ((0, 4000 - 1), (1, 299), (2, 5002)):
        c.v_pages[c.tables[b, at // 16], 5, at % 16, 3] = math.inf
    out = D.call(cea, c, dev).cpu()
    last = torch.zeros_like(out, dtype=torch.bool)
    last[:, T - 1, 5, 3] = True
    assert bool((out[last] == math.inf).all())
    half = P.half_step(BF16)
    assert bool(((out - want).abs()[~last].double() <= 4 * half * want.abs()[~last].double() + 1e-6).all())


@pytest.mark.parametrize("bits", [16, 8])
def test_many_rows(cea, dev, bits):
    """More rows than a wave has lanes, in runs, in splits and in the token form's."""
    lengths = [900 if i % 3 == 0 else 17 + i % 40 for i in range(70)]
    D.check(cea, dev, D.make_tree(17, lengths, bits=bits, Hq=4, Hkv=4, D=64))
    D.check(cea, dev, D.make_tree(17, [x * 2 for x in lengths[:66]], bits=bits, Hq=16, Hkv=16, D=64))
    D.check(cea, dev, D.make_tree(2, [x + 300 * (i == 9) for i, x in enumerate(lengths)], bits=bits, Hq=4, Hkv=1, D=64))


@pytest.mark.parametrize("seed", range(24))
def test_sweep(cea, dev, seed):
    """Random calls of the documented ranges."""
    import random

    r = random.Random(seed)
    T = r.choice([1, 2, r.randint(3, 16), r.randint(17, 70), r.randint(17, 70), r.randint(71, 140)])
    bits, dtype = r.choice([(8, BF16), (8, F16), (16, BF16), (16, F16), (32, F32), (8, F32)])
    Hkv = r.choice([1, 2, 3])
    Hq = Hkv * r.choice([1, 2, 4, 5, 7])
    B = r.randint(1, 4)
    lengths = [r.randint(0, r.choice([40, 300, 1200])) + T for _ in range(B)]
    counts = [r.choice([T, r.randint(0, T)]) for _ in range(B)]
    kw = dict(Hq=Hq, Hkv=Hkv, D=r.choice([64, 64, 128, 128, 96]), page=r.choice([16, 16, 32, 48, 64, 10]), dtype=dtype)
    D.check(cea, dev, D.make_tree(T, lengths, counts=counts, bits=bits, seed=seed, **kw))
    n = r.choice([1, 1, r.randint(2, 12), r.randint(17, 90)])
    c = P.make(B=B, n=n, lengths=[max(x, n) for x in lengths], seed=seed, explicit=r.random() < 0.4, causal=r.random() < 0.8,
               **{**kw, "dtype": r.choice([BF16, F16])})
    D.check(cea, dev, D.pool8(c, seed))


def test_pools_beyond_4_gib(cea, dev):
    """Pages whose offsets pass 32 bits, in every operator on 8-bit pools."""
    P_, H, page, d, n = 72000, 8, 64, 128, 40  # 4.7 GB each
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of device memory")
    kv = torch.empty(2, P_, H, page, d, dtype=torch.uint8, device=dev)
    sc = torch.empty(2, P_, H, page, dtype=torch.uint8, device=dev)
    g = torch.Generator().manual_seed(2)
    tables = torch.tensor([[P_ - 1, 3, P_ - 7], [P_ - 2, 70001, 65600]])
    lengths, counts = torch.tensor([150, 130]), torch.tensor([n, n])
    small = torch.arange(6).view(2, 3)
    for t in (tables, small):  # the same contents in far pages, and in the first pages of a small pool
        pools = (kv, sc) if t is tables else (torch.empty(2, 6, H, page, d, dtype=torch.uint8, device=dev),
                                              torch.empty(2, 6, H, page, dtype=torch.uint8, device=dev))
        a, s = pools
        gg = torch.Generator().manual_seed(5)
        rand = lambda *x: torch.randn(*x, generator=gg).to(dev, BF16)
        k, v, q = rand(2, 150, H, d), rand(2, 150, H, d), rand(2, n, 32, d)
        td, z = t.to(dev), torch.zeros(2, dtype=torch.int64, device=dev)
        kw = {"k_scales": s[0], "v_scales": s[1]}
        cea.paged_kv_append(a[0].view(F8), a[1].view(F8), td, z, k, v, counts=lengths.to(dev), **kw)
        masks, _ = cea.tree_masks(D.parents(2, n, 3).to(dev))
        got = [cea.paged_tree_attention(q, a[0].view(F8), a[1].view(F8), td, lengths.to(dev), counts.to(dev), masks, **kw),
               cea.paged_attention(q[:, :1], a[0].view(F8), a[1].view(F8), td, lengths.to(dev), lengths.view(2, 1).to(dev) - 1, **kw)]
        path = torch.tensor([[1, 5, 39], [0, 2, 3]], device=dev)
        cea.paged_kv_keep(a.view(F8), td, (lengths - n).to(dev), path, scales=s)
        got += cea.paged_kv_read(a[0].view(F8), a[1].view(F8), td, z, 150, counts=lengths.to(dev), **kw)
        if t is tables:
            want = got
    for x, y in zip(want, got):
        assert torch.equal(x, y)

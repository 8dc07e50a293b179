"""The paged KV cache in 8 bits, and trees of drafted tokens over a paged cache.

A pool holds pages of ``page`` slots, ``k_pages`` / ``v_pages`` ``[P, H, page, D]``; row ``b`` of a
batch has its slots in the pages ``tables[b, slot // page]``.  In an 8-bit pool a slot and head is a
row of ``D`` e4m3 numbers ``q`` and a byte ``s`` of ``[P, H, page]``, the values ``q * 2^(s - 127)``.
Every case is a dict of plain values with a ``kind``:

* ``append`` - rotary on the new keys, then keys and values into 8-bit pages: ``s - 127`` is the
               smallest whole number ``e >= -117`` with ``max |x| <= 448 * 2^e``
* ``read``   - the slots of each row as contiguous keys and values again, in 16 bits
* ``attend`` - causal attention of ``chunk`` new tokens a row (one: a decode step) over 8-bit pages
* ``tree``   - attention of a tree of drafted tokens, a row's last slots: a node sees the slots
               before the tree, its ancestors and itself; pages of 8, 16 or 32 bits
* ``masks``  - the ancestors of a tree's nodes as bits of 64-bit words, and the nodes' depths
* ``keep``   - the rows of the accepted nodes move into line behind the slots before the tree, in
               the pools of all layers

``listed()`` names the measured ones, ``draw`` gives more of the same ranges.  ``run`` computes the
plain form, or calls the package's operators where ``own`` is true.
"""

import importlib
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
F8 = torch.float8_e4m3fn

# (query heads, KV heads, head size) of a model: 8B-shaped, tinyllama-1.1b, qwen2-0.5b, and the
# eight equal heads of the f32 mode
SHAPES = {
    "8b": (32, 8, 128),
    "1b": (32, 4, 64),
    "half": (14, 2, 64),
    "eight": (8, 8, 64),
}


def _case(kind, name=None, **kw):
    c = {"kind": kind, **kw}
    if name is not None:
        c["name"] = name
    return c


def listed():
    return [
        # the append of a decode step, once a layer: the call itself is what counts
        _case("append", "append_b32_token", shape="8b", page=64, batch=32, chunk=1, past=2000,
              dtype="bf16"),
        # the append of two prompts' chunks
        _case("append", "append_b2_4096", shape="8b", page=64, batch=2, chunk=4096, past=333,
              dtype="f16"),
        # short rows of several users handed to a program with a contiguous cache
        _case("read", "read_b8_700", shape="1b", page=16, batch=8, chunk=700, dtype="f16", bits=8),
        # a long sequence leaves for another device
        _case("read", "read_b1_30000", shape="8b", page=64, batch=1, chunk=30000, dtype="bf16",
              bits=8),
        # a full batch with long contexts: the cache is read once, nothing else counts
        _case("attend", "token_b32_32k", shape="8b", page=64, batch=32, chunk=1, min_len=1024,
              max_len=32768, dtype="bf16"),
        # a chunk of a chunked prefill late in a long prompt
        _case("attend", "chunk_128_of_32k", shape="8b", page=64, batch=1, chunk=128, min_len=32768,
              max_len=32768, dtype="bf16"),
        # one chat user's drafts: a small tree after a short context
        _case("tree", "tree_b1_26_of_777", shape="1b", page=16, batch=1, nodes=26, min_len=777,
              max_len=777, dtype="bf16", bits=16),
        # a server's verification step: trees of 60 nodes after contexts of every length up to 8192,
        # the cache in 8 bits
        _case("tree", "tree_b16_60_of_8k", shape="8b", page=64, batch=16, nodes=60, min_len=500,
              max_len=8192, dtype="bf16", bits=8),
        # the masks of one user's tree, once a step
        _case("masks", "masks_b1_26", batch=1, nodes=26),
        # large trees of a full batch
        _case("masks", "masks_b64_250", batch=64, nodes=250),
        # four drafted tokens of one user accepted, in the pools of 22 layers
        _case("keep", "keep_b1_4", shape="1b", page=16, layers=22, batch=1, nodes=26, kept=4,
              past=777, bits=16, dtype="bf16"),
        # up to nine accepted in each row of a full batch, in the 8-bit pools of 32 layers
        _case("keep", "keep_b32_9", shape="8b", page=64, layers=32, batch=32, nodes=60, kept=9,
              past=500, bits=8, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "append", "read", "attend", "attend", "attend", "tree", "tree",
                       "tree", "masks", "keep"])
    shape = rng.choice(["8b", "8b", "1b", "half"])
    page = rng.choice([16, 16, 32, 64, 64, 128])
    half = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        chunk = rng.choice([1, _log(rng, 2, 6000)])
        return _case(kind, shape=shape, page=page, batch=min(_log(rng, 1, 64), max(1, 8192 // chunk)),
                     chunk=chunk, past=_log(rng, 1, 3000), dtype=half)
    if kind == "read":
        chunk = _log(rng, 1, 30000)
        return _case(kind, shape=shape, page=page, batch=min(_log(rng, 1, 64), max(1, 30000 // chunk)),
                     chunk=chunk, dtype=half, bits=rng.choice([8, 8, 16]))
    if kind == "attend":
        form = rng.choice(["token", "token", "few", "chunk", "chunk", "prompt"])
        if form in ("token", "few"):
            chunk = 1 if form == "token" else rng.randint(2, 12)
            top = _log(rng, 60, 30000)
            batch = min(_log(rng, 1, 64), max(1, 480000 // top))
            return _case(kind, shape=shape, page=page, batch=batch, chunk=chunk,
                         min_len=max(chunk, top // rng.choice([1, 3, 16])), max_len=max(chunk, top),
                         dtype=half)
        if form == "chunk":
            chunk = _log(rng, 17, 512)
            top = max(chunk, _log(rng, 400, 30000))
            batch = rng.choice([1, 1, 2, 4]) if top < 9000 else 1
        else:
            chunk = top = _log(rng, 40, 3000)
            batch = min(rng.choice([1, 2, 3, 8]), max(1, 6000 // chunk))
        return _case(kind, shape=shape, page=page, batch=batch, chunk=chunk,
                     min_len=max(chunk, top // 2), max_len=top, dtype=half)
    if kind == "tree":
        nodes = rng.choice([rng.randint(2, 16), rng.randint(17, 64), rng.randint(17, 64),
                            _log(rng, 65, 200)])
        top = max(nodes, _log(rng, 60, 16000))
        bits = rng.choice([8, 8, 16, 16, 32])
        if bits == 32:
            shape, half, top = "eight", "f32", min(top, 1500)
        batch = min(_log(rng, 1, 32), max(1, 131072 // top), max(1, 4 * 131072 // (top * nodes)) + 2)
        return _case(kind, shape=shape, page=page, batch=batch, nodes=nodes,
                     min_len=max(nodes, top // rng.choice([1, 3, 16])), max_len=top, dtype=half,
                     bits=bits)
    nodes = rng.choice([rng.randint(2, 64), _log(rng, 65, 250)])
    if kind == "masks":
        return _case(kind, batch=_log(rng, 1, 64), nodes=nodes)
    return _case(kind, shape=shape, page=page, layers=rng.randint(1, 24), batch=_log(rng, 1, 32),
                 nodes=nodes, kept=rng.randint(1, min(12, nodes)), past=_log(rng, 1, 600),
                 bits=rng.choice([8, 16]), dtype=half)


# --------------------------------------------------------------------------------------
# inputs, made from the seed alone
# --------------------------------------------------------------------------------------
def _randn(g, *shape, dtype):
    x = torch.empty(*shape, device="cuda", dtype=dtype)
    flat = x.view(-1)
    step = 1 << 28  # the f32 values of a large pool a gigabyte at a time
    for i in range(0, flat.numel(), step):
        part = flat[i:i + step]
        part.copy_(torch.randn(part.numel(), generator=g, device="cuda"))
    return x


def _pool8(g, *shape):
    """Rows of an 8-bit pool: numbers whose largest is near the top of e4m3's range, and scale bytes
    of values around 1."""
    q = _randn(g, *shape, dtype=torch.bfloat16)
    q = q.mul_(100.0).clamp_(-448.0, 448.0).to(F8)
    s = torch.randint(119, 122, shape[:-1], generator=g, device="cuda", dtype=torch.uint8)
    return q, s


def _lengths(case):
    """The rows' lengths, spread evenly from min_len to max_len."""
    n, lo, hi = case["batch"], case["min_len"], case["max_len"]
    return [hi - (hi - lo) * i // max(1, n - 1) for i in range(n)]


def _tables(g, lengths, page, width, pages):
    """Every row's pages, drawn without order from the pool; -1 where a row has none."""
    order = torch.randperm(pages, generator=g, device="cuda")
    tables = torch.full((len(lengths), width), -1, dtype=torch.int64, device="cuda")
    at = 0
    for b, n in enumerate(lengths):
        k = -(-n // page)
        tables[b, :k] = order[at:at + k]
        at += k
    return tables


def _parents(g, batch, nodes):
    """Trees of drafts, parents first: most nodes continue one of the last few, some start anew."""
    i = torch.arange(nodes, device="cuda")
    back = torch.randint(1, 9, (batch, nodes), generator=g, device="cuda")
    root = torch.rand(batch, nodes, generator=g, device="cuda") < 0.1
    return torch.where(root, torch.full_like(back, -1), (i - back).clamp(min=-1))


def _words(seen):
    """Booleans [B, T, T] as bits of 64-bit words [B, T, ceil(T / 64)]."""
    B, T, _ = seen.shape
    n = -(-T // 64)
    bits = torch.zeros(B, T, 64 * n, dtype=torch.int64, device=seen.device)
    bits[:, :, :T] = seen
    return (bits.view(B, T, n, 64) << torch.arange(64, device=seen.device)).sum(-1)


def _ancestors(parents):
    """Node i's row: itself and the row of its parent."""
    B, T = parents.shape
    seen = torch.zeros(B, T + 1, T, dtype=torch.bool, device=parents.device)  # the last row: no parent
    rows = torch.arange(B, device=parents.device)
    for i in range(T):
        seen[:, i] = seen[rows, parents[:, i]]  # (-1: the last row)
        seen[:, i, i] = True
    return seen[:, :T]


def prepare(case, seed):
    """The cache's pools, the rows' tables and lengths, and the call's own tokens."""
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, B = case["kind"], case["batch"]
    s = {"case": case}
    if kind in ("masks", "tree"):
        s["parents"] = _parents(g, B, case["nodes"])
        if kind == "masks":
            return s
        s["masks"] = _words(_ancestors(s["parents"]))
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = SHAPES[case["shape"]]
    page, n = case["page"], case.get("chunk", case.get("nodes"))
    if kind in ("attend", "tree"):
        lengths = _lengths(case)
    elif kind == "read":
        lengths = [n - i * (n // 2) // B for i in range(B)]
    else:
        lengths = [case["past"] + n] * B
    width = -(-max(lengths) // page)
    pages = sum(-(-x // page) for x in lengths) + 3
    s["tables"] = _tables(g, lengths, page, width, pages)
    s["lengths"] = torch.tensor(lengths, device="cuda")
    s["k_scales"] = s["v_scales"] = s["scales"] = None
    bits = case.get("bits", 8)
    if kind == "keep":
        shape = (2 * case["layers"], pages, hkv, page, d)
        if bits == 8:
            s["kv"], s["scales"] = _pool8(g, *shape)
        else:
            s["kv"] = _randn(g, *shape, dtype=dt)
        # the accepted nodes of each row, in order, some rows with fewer
        pick = torch.rand(B, n, generator=g, device="cuda").argsort(-1)[:, :case["kept"]].sort(-1).values
        drop = torch.randint(0, 2 * case["kept"], (B, 1), generator=g, device="cuda")
        i = torch.arange(case["kept"], device="cuda")
        s["path"] = torch.where(i < torch.where(drop > 0, drop, case["kept"]), pick, torch.full_like(pick, -1))
        s["offsets"] = s["lengths"] - n
        return s
    if bits == 8:
        s["k_pages"], s["k_scales"] = _pool8(g, pages, hkv, page, d)
        s["v_pages"], s["v_scales"] = _pool8(g, pages, hkv, page, d)
    else:
        s["k_pages"] = _randn(g, pages, hkv, page, d, dtype=dt)
        s["v_pages"] = _randn(g, pages, hkv, page, d, dtype=dt)
    if kind == "read":
        s["offsets"] = torch.zeros(B, dtype=torch.int64, device="cuda")
        return s
    if kind == "append":
        past = torch.randint(max(1, case["past"] // 2), case["past"] + 1, (B,), generator=g,
                             device="cuda")
        s["offsets"] = past
        s["k"] = _randn(g, B, n, hkv, d, dtype=dt)
        s["v"] = _randn(g, B, n, hkv, d, dtype=dt)
        pos = past.view(B, 1) + torch.arange(n, device="cuda")
        inv = 1.0 / 1e4 ** (torch.arange(0, d, 2, device="cuda").double() / d)
        ang = pos.double().unsqueeze(-1) * inv
        ang = torch.cat([ang, ang], -1)
        s["cos"], s["sin"] = ang.cos().to(dt), ang.sin().to(dt)
        return s
    s["q"] = _randn(g, B, n, hq, d, dtype=dt)
    # the new tokens are the row's last ones
    s["q_pos"] = s["lengths"].view(B, 1) - n + torch.arange(n, device="cuda")
    s["counts"] = torch.full((B,), n, device="cuda")
    return s


# --------------------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------------------
def _values(pages, scales, at):
    """The pages `at` [B, W] in f32, [B, W, H, page, D]."""
    if scales is None:
        return pages[at].float()
    q = pages.view(torch.uint8)[at].view(F8).float()
    return torch.ldexp(q, scales[at].int().unsqueeze(-1) - 127)


def _gather(s, which):
    """A row's pages one after the other, [B, H, slots, D] in f32 (its missing pages: page 0)."""
    x = _values(s[which + "_pages"], s[which + "_scales"], s["tables"].clamp(min=0))
    B, W, H, n, D = x.shape
    return x.transpose(1, 2).reshape(B, H, W * n, D)


def _attend(s, seen):
    """Softmax over the slots that `seen` [B, n, slots] names."""
    q = s["q"]
    B, n, hq, d = q.shape
    k, v = _gather(s, "k"), _gather(s, "v")
    hkv, S = k.shape[1], k.shape[2]
    x = q.float().view(B, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, d)
    score = torch.matmul(x, k.transpose(2, 3).contiguous()).view(B, hq, n, S) * d ** -0.5
    score = score.masked_fill_(~seen[:, None], float("-inf"))
    top = score.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(B, hkv, -1, S), v).view(B, hq, n, d)
    out = out / total.clamp(min=1e-30)
    return out.transpose(1, 2).to(q.dtype)


def _causal(s):
    slots = torch.arange(s["tables"].shape[1] * s["case"]["page"], device="cuda")
    return (slots <= s["q_pos"].unsqueeze(-1)) & (slots < s["lengths"].view(-1, 1, 1))


def _tree(s):
    """Which slots each node sees: those before the tree, and its bits of the tree's own."""
    masks, base = s["masks"], (s["lengths"] - s["counts"]).view(-1, 1, 1)
    slots = torch.arange(s["tables"].shape[1] * s["case"]["page"], device="cuda")
    B, T, n = masks.shape
    node = (slots - base).expand(B, T, -1)
    word = masks.gather(2, node.div(64, rounding_mode="floor").clamp(0, n - 1))
    bit = (word >> node.remainder(64)) & 1
    return (node < 0) | ((node < s["counts"].view(-1, 1, 1)) & (bit == 1))


def _quantise(x):
    """Rows of f32 values as e4m3 numbers and scale bytes."""
    top = x.abs().amax(-1)
    m, e = torch.frexp(top)  # top = m 2^e, 1/2 <= m < 1; 448 = 0.875 * 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-117)
    e = torch.where(top == 0, torch.full_like(e, -117), e)
    return torch.ldexp(x, -e.unsqueeze(-1)).to(F8), (e + 127).to(torch.uint8)


def _append(s):
    k, v, cos, sin = s["k"], s["v"], s["cos"].float().unsqueeze(2), s["sin"].float().unsqueeze(2)
    B, n, _, d = k.shape
    x = k.float()
    turned = torch.cat([-x[..., d // 2:], x[..., :d // 2]], -1)
    page = s["k_pages"].shape[2]
    slot = s["offsets"].view(B, 1) + torch.arange(n, device=k.device)
    at = s["tables"].gather(1, slot // page)
    for which, new in (("k", x * cos + turned * sin), ("v", v.float())):
        q, e = _quantise(new)
        s[which + "_pages"].view(torch.uint8)[at, :, slot % page] = q.view(torch.uint8)
        s[which + "_scales"][at, :, slot % page] = e
    return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]


def _read(s):
    n, dt = s["case"]["chunk"], DTYPES[s["case"]["dtype"]]
    live = torch.arange(n, device="cuda") < s["lengths"].view(-1, 1)
    got = []
    for which in ("k", "v"):
        x = _gather(s, which).transpose(1, 2)[:, :n]
        got.append(torch.where(live[:, :, None, None], x, torch.zeros_like(x)).to(dt))
    return got


def _masks(s):
    seen = _ancestors(s["parents"])
    return _words(seen), seen.sum(-1) - 1


def _keep(s):
    path, page = s["path"], s["case"]["page"]
    i = torch.arange(path.shape[1], device="cuda").expand_as(path)
    use = path >= i
    rows = torch.arange(path.shape[0], device="cuda").unsqueeze(1).expand_as(path)[use]
    src, dst = s["offsets"][rows] + path[use], s["offsets"][rows] + i[use]
    src_at, dst_at = s["tables"][rows, src // page], s["tables"][rows, dst // page]
    kv = s["kv"].view(torch.uint8) if s["scales"] is not None else s["kv"]
    for pool in (kv, s["scales"]):
        if pool is not None:
            pool[:, dst_at, :, dst % page] = pool[:, src_at, :, src % page]
    return (s["kv"],) if s["scales"] is None else (s["kv"], s["scales"])


def run(s):
    kind = s["case"]["kind"]
    if not own:
        if kind == "attend":
            return _attend(s, _causal(s))
        if kind == "tree":
            return _attend(s, _tree(s))
        return {"append": _append, "read": _read, "masks": _masks, "keep": _keep}[kind](s)
    cea = importlib.import_module("collaborative-edge-system_amd")
    if kind == "append":
        cea.paged_kv_append(s["k_pages"], s["v_pages"], s["tables"], s["offsets"], s["k"], s["v"],
                            cos=s["cos"], sin=s["sin"], k_scales=s["k_scales"], v_scales=s["v_scales"])
        return s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]
    if kind == "read":
        return cea.paged_kv_read(s["k_pages"], s["v_pages"], s["tables"], s["offsets"], s["case"]["chunk"],
                                 counts=s["lengths"], dtype=DTYPES[s["case"]["dtype"]],
                                 k_scales=s["k_scales"], v_scales=s["v_scales"])
    if kind == "attend":
        return cea.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"],
                                   s["q_pos"], k_scales=s["k_scales"], v_scales=s["v_scales"])
    if kind == "tree":
        return cea.paged_tree_attention(s["q"], s["k_pages"], s["v_pages"], s["tables"], s["lengths"],
                                        s["counts"], s["masks"], k_scales=s["k_scales"],
                                        v_scales=s["v_scales"])
    if kind == "masks":
        return cea.tree_masks(s["parents"])
    cea.paged_kv_keep(s["kv"], s["tables"], s["offsets"], s["path"], scales=s["scales"])
    return (s["kv"],) if s["scales"] is None else (s["kv"], s["scales"])


# --------------------------------------------------------------------------------------
# what a pass cannot do without
# --------------------------------------------------------------------------------------
def work(case):
    B, kind = case["batch"], case["kind"]
    if kind == "masks":
        T = case["nodes"]
        return {"bytes": 8 * B * T * (2 + -(-T // 64)), "flops": 0}
    hq, hkv, d = SHAPES[case["shape"]]
    bits = case.get("bits", 8)
    row = d + 1 if bits == 8 else d * bits // 8  # bytes of a slot and head
    size = 4 if case["dtype"] == "f32" else 2
    if kind == "append":
        rows = B * case["chunk"] * hkv
        return {"bytes": 2 * rows * (d * size + row) + 2 * B * case["chunk"] * d * size,
                "flops": 7 * rows * d}
    if kind == "read":
        n = case["chunk"]
        held = sum(n - i * (n // 2) // B for i in range(B))
        return {"bytes": 2 * hkv * (held * row + B * n * d * size), "flops": 2 * held * hkv * d}
    if kind == "keep":  # (rows keep three quarters of `kept` on average)
        moved = B * case["kept"] * 3 // 4 or 1
        return {"bytes": 2 * 2 * case["layers"] * hkv * moved * row, "flops": 0}
    lengths = _lengths(case)
    n = case["chunk"] if kind == "attend" else case["nodes"]
    # a row's new token sees the slots before the new ones, and itself; a token of a chunk also
    # those before it, a node its ancestors, a few
    own_pairs = n * (n + 1) // 2 if kind == "attend" else n
    pairs = sum(n * (x - n) + own_pairs for x in lengths)
    return {"bytes": sum(lengths) * 2 * hkv * row + 2 * B * n * hq * d * size,
            "flops": 4 * d * hq * pairs}


# --------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------
def _slots64(s, which, b, head, ids, L):
    """The first L slots of the pages `ids` of one KV head, in 64 bits."""
    x = s[which + "_pages"]
    if s[which + "_scales"] is None:
        return x[ids, head].reshape(-1, x.shape[3])[:L].double()
    q = x.view(torch.uint8)[ids, head].view(F8).double().reshape(-1, x.shape[3])[:L]
    e = s[which + "_scales"][ids, head].double().reshape(-1, 1)[:L]
    return q * 2.0 ** (e - 127.0)


def _hidden64(s, b, L):
    """Which of row b's first L slots each query does not see."""
    j = torch.arange(L, device="cuda")
    if s["case"]["kind"] == "attend":
        return j[None, :] > s["q_pos"][b][:, None]
    T = s["case"]["nodes"]
    up = s["parents"][b].tolist()
    see = torch.zeros(T, T, dtype=torch.bool)
    for i in range(T):
        at = i
        while at >= 0:
            see[i, at] = True
            at = up[at]
    return torch.cat([torch.zeros(T, L - T, dtype=torch.bool), ~see], 1).to("cuda")


def exact(case, seed):
    s = prepare(case, seed)
    kind, B = case["kind"], case["batch"]
    if kind == "masks":
        masks, depths = [], []
        for up in s["parents"].tolist():
            rows = []
            for i, p in enumerate(up):
                rows.append((rows[p] if p >= 0 else 0) | 1 << i)
            words = [[r >> 64 * w & (1 << 64) - 1 for w in range(-(-len(up) // 64))] for r in rows]
            masks.append([[x - (1 << 64) if x >> 63 else x for x in w] for w in words])
            depths.append([bin(r).count("1") - 1 for r in rows])
        return torch.tensor(masks), torch.tensor(depths)
    page = case["page"]
    if kind == "keep":
        pools = [s["kv"]] if s["scales"] is None else [s["kv"].view(torch.uint8), s["scales"]]
        want = [x.clone() for x in pools]
        table, path, base = s["tables"].tolist(), s["path"].tolist(), s["offsets"].tolist()
        for b in range(B):
            for i, node in enumerate(path[b]):
                if node >= 0:
                    a, z = base[b] + node, base[b] + i
                    for x, y in zip(pools, want):
                        y[:, table[b][z // page], :, z % page] = x[:, table[b][a // page], :, a % page]
        return (want[0],) if s["scales"] is None else (want[0].view(F8), want[1])
    if kind in ("attend", "tree"):
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        hq, hkv, d = SHAPES[case["shape"]]
        for b in range(B):
            L = int(s["lengths"][b])
            ids = s["tables"][b, :-(-L // page)]
            hidden = _hidden64(s, b, L)
            for j in range(hkv):
                k, v = (_slots64(s, x, b, j, ids, L) for x in "kv")
                for h in range(j * (hq // hkv), (j + 1) * (hq // hkv)):
                    z = s["q"][b, :, h].double() @ k.T / math.sqrt(d)
                    out[b, :, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v
        return out
    if kind == "read":
        n, hkv = case["chunk"], s["k_pages"].shape[1]
        got = [torch.zeros(B, n, hkv, s["k_pages"].shape[3], dtype=torch.float64, device="cuda") for _ in "kv"]
        for b in range(B):
            L = int(s["lengths"][b])
            ids = s["tables"][b, :-(-L // page)]
            for j in range(hkv):
                for x, which in zip(got, "kv"):
                    x[b, :L, j] = _slots64(s, which, b, j, ids, L)
        return got
    # append: the numbers before their rounding to e4m3, in their rows' scale
    half = s["k"].shape[3] // 2
    lo, hi = s["k"].double().split(half, -1)
    c, z = s["cos"].double()[:, :, None], s["sin"].double()[:, :, None]
    rotated = torch.cat([lo * c[..., :half] - hi * z[..., :half], hi * c[..., half:] + lo * z[..., half:]], -1)
    pools = []
    for which, new in (("k", rotated), ("v", s["v"].double())):
        pool = s[which + "_pages"].double()
        e = torch.ceil(torch.log2(new.abs().amax(-1, keepdim=True) / 448.0)).clamp(min=-117.0)
        new = new / 2.0 ** e
        for b in range(B):
            slot = int(s["offsets"][b]) + torch.arange(case["chunk"], device="cuda")
            ids, rest = s["tables"][b][slot // page], slot % page
            for j in range(pool.shape[1]):
                pool[ids, j, rest] = new[b, :, j]
        pools.append(pool)
    return pools[0], pools[1], None, None

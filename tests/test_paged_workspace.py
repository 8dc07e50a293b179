"""The scratch of attention over 8-bit pages and of trees, on the host (no kernel runs here)."""

from __future__ import annotations

import ctypes
import random
import re
from pathlib import Path

from test_abi import _t

BF16, F32, I64, E4M3, U8 = 1, 0, 4, 5, 6
HEADER = Path(__file__).resolve().parents[1] / "include" / "collab_edge_attn.h"


def _refs(*ts):
    return [ctypes.byref(t) if t is not None else None for t in ts]


def _needed(nat, tree, f8, B, n, Hq, Hkv, D, W, page, out=None):
    """What the call's own function gives; the call itself wants as much."""
    lib = nat.load_library()
    q, o = _t((B, n, Hq, D), BF16), _t((B, n, Hq, D), BF16 if out is None else out)
    kp, vp = (_t((8, Hkv, page, D), E4M3 if f8 else BF16) for _ in "kv")
    ks, vs = (_t((8, Hkv, page), U8) if f8 else None for _ in "kv")
    tab, ln = _t((B, W), I64), _t((B,), I64)
    got = ctypes.c_size_t(7)
    if tree:
        counts, masks = _t((B,), I64), _t((B, n, -(-n // 64)), I64)
        args = _refs(q, kp, vp, ks, vs, tab, ln, counts, masks) + [0.125, None, 0]
        size, call = lib.cea_paged_tree_attention_workspace, lib.cea_paged_tree_attention
    else:
        args = _refs(q, kp, vp, ks, vs, None, tab, ln, _t((B, n), I64)) + [1, 0.125, None, 0]
        size, call = lib.cea_paged_attention8_workspace, lib.cea_paged_attention8
    assert size(*args, *_refs(o, None), ctypes.byref(got)) == 0, nat.last_error()
    if got.value:
        assert call(*args, *_refs(o, None), 1 << 20, got.value - 1, None) == nat.ENOSPACE
        assert f"{got.value} bytes" in nat.last_error()
    return got.value


def test_trees_and_8_bit_pages_say_their_own_scratch(cea):
    nat = cea._native
    bound = nat.load_library().cea_paged_attention_workspace_bytes
    more = 0
    rng = random.Random(5)
    shapes = [(40, 60, 32, 8, 128, 200, 64), (16, 60, 32, 8, 128, 128, 64), (1, 26, 32, 4, 64, 49, 16)]
    shapes += [(rng.choice([1, 3, 20, 70]), rng.choice([1, 9, 40, 200]), 8 * rng.choice([1, 4]), 8, rng.choice([64, 128]),
                rng.choice([1, 20, 300]), rng.choice([16, 64])) for _ in range(60)]
    for s in shapes:
        for tree, f8 in ((True, False), (True, True), (False, True)):
            more += _needed(nat, tree, f8, *s, out=rng.choice([None, F32])) > bound(*s, BF16)
    assert more  # the other call's bound does not cover these


def test_the_header_names_the_functions_that_give_it():
    """A caller who reads the contract is not sent to the bound of cea_paged_attention."""
    text = HEADER.read_text()
    comments = {m.group(2): " ".join(re.sub(r"^ \*", " ", m.group(1), flags=re.M).split())
                for m in re.finditer(r"/\*((?:(?!\*/).)*)\*/\s*\w+\s+(\w+)\(", text, re.S)}
    tree = comments["cea_paged_tree_attention_workspace"]
    assert "the size that cea_paged_tree_attention_workspace() gives" in tree
    assert "the workspace as cea_paged_attention" not in tree
    assert "the size that cea_paged_attention8_workspace() gives" in comments["cea_paged_kv_append8"]
    assert "not for those over 8-bit pages or of trees" in comments["cea_paged_attention_workspace_bytes"]

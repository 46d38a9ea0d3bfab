"""Where the 27B-shaped pass records the cache and the attention over it, when it is asked to, and what a launch planner makes of them; without a device."""
import ctypes as C

import pytest

from test_decode_pass_steps import record


def test_behind_the_heads_and_in_front_of_the_output_projection():
    caches = ["c0", "c1"]
    steps = record(n_layers=8, heads=dict(positions="p"), cache=dict(caches=caches, table="t", lengths="l", begin="b"))
    at = [i for i, s in enumerate(steps) if s[0] == "attention"]
    assert len(at) == 2
    for i, cache, il in zip(at, caches, (3, 7)):
        heads, append, attention, quantize, out = steps[i - 2:i + 3]
        assert [s[0] for s in (heads, append, attention, quantize, out)] == ["qk_norm_rope", "cache_append", "attention", "quantize", "gemv"]
        assert append[1][0] == attention[1][0] == cache and append[1][3:] == attention[1][3:] == ("t", "l", "b")
        k, v = append[1][1:3]
        assert k["buf"] == v["buf"] == heads[1][1]["buf"] and v["off"] == 4 * 256
        q, mixed = attention[1][1:3]
        assert q == heads[1][0] and quantize[1][:3] == (mixed["buf"], 0, q["n_heads"] * 256) and out[1][0] == f"l{il}.o"


def test_without_them_nothing_changes():
    cache = dict(caches=["c"], table="t", lengths="l", begin="b")
    plain, more = record(n_layers=4), record(n_layers=4, cache=cache)
    assert [s[0] for s in plain] == [s[0] for s in more if s[0] not in ("cache_append", "attention")]


@pytest.mark.parametrize("kind", [8, 9])
def test_a_matvec_does_not_step_over_them(kind):
    from qwengine_b200 import build, load_library
    build.build()
    lib = load_library()
    steps = [(1, 4, 0), (kind, 0, 0), (1, 4, 512)]
    flat = (C.c_int * (3 * len(steps)))(*[v for s in steps for v in s])
    out = (C.c_int * len(steps))()
    assert lib.q38b_debug_merge_plan(1, 1, len(steps), flat, out) == 0 and list(out) == [0, 1, 2]
    own = (C.c_int * 3)()
    steps = [(1, 4, 0), (4, 0, 0), (kind, 0, 0)]
    flat = (C.c_int * 9)(*[v for s in steps for v in s])
    assert lib.q38b_debug_barriers(2, 1, 3, flat, own) == 0 and list(own) == [-1, 1, -1]

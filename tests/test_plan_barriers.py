"""Steps behind a cross-GPU barrier on several ranks, without a device: where the barrier runs (q38b_plan.cu: barrier_joins_launch), and where the 27B-shaped
pass records it.  Only a merged matvec launch of one column and the SwiGLU kernel can begin with a barrier; in front of heads, logit rules and the top-k, which read what
the peers have stored, it has to run by itself."""
import ctypes as C

import numpy as np
import pytest

from qwengine_b200 import decode_pass

from test_decode_pass_steps import Recorder

Q, MV, SW, GA, BA, HD, LG, TK = range(8)   # step kinds of the test hook


def record(**kw):
    ps = Recorder()
    decode_pass.build(ps, lambda spec, rows, replicated=False: spec.name, **kw)
    return [s for s in ps.steps if s[0] != "set_peer_store"]


@pytest.fixture(scope="module")
def barriers():
    from qwengine_b200 import build, load_library
    build.build()
    fn = load_library().q38b_debug_barriers
    i32p = np.ctypeslib.ndpointer(np.int32, flags="C_CONTIGUOUS")
    fn.argtypes = [C.c_int, C.c_int, C.c_int, i32p, i32p]

    def run(nb, steps, n_ranks=2):
        s = np.array(steps, np.int32).reshape(-1, 3)
        out = np.zeros(len(s), np.int32)
        assert fn(n_ranks, nb, len(s), s, out) == 0
        return out.tolist()
    return run


@pytest.mark.parametrize("nb", [1, 4])
@pytest.mark.parametrize("step", [HD, LG, TK])
def test_in_front_of_a_step_without_a_prologue_it_runs_by_itself(barriers, nb, step):
    assert barriers(nb, [(MV, 4, 0), (BA, 0, 0), (step, 0, 0), (Q, 5, 0), (MV, 5, 2048)]) == [-1, 1, -1, -1, -1]
    # ... also where a launch that could begin with it follows the step, and behind another barrier
    assert barriers(nb, [(Q, 4, 0), (MV, 4, 0), (MV, 4, 512), (BA, 0, 0), (BA, 0, 0), (step, 0, 0), (SW, 5, 0)]) == [-1, -1, -1, 1, 1, -1, -1]


def test_launches_that_begin_with_it(barriers):
    assert barriers(1, [(MV, 4, 0), (BA, 0, 0), (Q, 5, 0), (MV, 5, 2048)])[1] == 0
    assert barriers(4, [(MV, 4, 0), (BA, 0, 0), (Q, 5, 0), (MV, 5, 2048)])[1] == 1      # several columns
    assert barriers(1, [(MV, 4, 0), (BA, 0, 0), (SW, 5, 0)])[1] == 0
    assert barriers(1, [(MV, 4, 0), (BA, 0, 0), (GA, 0, 0), (SW, 5, 0)])[1] == 1        # a gather in between
    assert barriers(1, [(MV, 4, 0), (BA, 0, 0)])[1] == 1


@pytest.mark.parametrize("world", [2, 4, 8])
@pytest.mark.parametrize("replicate_small", [True, False])
def test_the_27b_shaped_pass_on_several_ranks(world, replicate_small):
    """Every row that heads or rules read is there: computed whole by this rank, or followed by a barrier before the step; their own consumer comes right
    behind them, with nothing of another rank in between."""
    steps = record(n_layers=8, heads=dict(positions="p"), rules=dict(penalties="r"), world=world, rank=world - 1, gather="peer", replicate_small=replicate_small)
    names = [s[0] for s in steps]
    assert names.count("qk_norm_rope") == 2 and names.count("adjust_logits") == 1
    for i, (name, a, kw) in enumerate(steps):
        if name == "qk_norm_rope":
            made = steps[i - 3:i] if replicate_small else steps[i - 4:i - 1]
            assert [s[0] for s in made] == ["gemv"] * 3 and all(bool(s[2].get("local")) == replicate_small for s in made)
            assert replicate_small or names[i - 1] == "barrier"
            assert {made[0][1][2]} == {a[0]["buf"]} and {s[1][2] for s in made[1:]} == {a[1]["buf"]}
            assert names[i + 1] == "quantize" and steps[i + 1][1][0] == a[0]["buf"]
        elif name == "adjust_logits":
            assert names[i - 2:i] == ["gemv", "barrier"] and steps[i - 2][1][2] == a[0]
            assert names[i + 1] == "topk" and steps[i + 1][1][0] == a[0]


def test_with_gathers_the_rules_come_behind_the_heads_gather():
    steps = record(n_layers=4, heads=dict(positions="p"), rules=dict(penalties="r"), world=2, rank=0, gather="nccl", replicate_small=False)
    names = [s[0] for s in steps]
    i, j = names.index("qk_norm_rope"), names.index("adjust_logits")
    assert names[i - 6:i] == ["gemv", "allgather"] * 3 and names[j - 2:j] == ["gemv", "allgather"]

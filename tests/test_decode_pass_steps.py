"""Where the 27B-shaped pass records the steps between its products, when it is asked to."""
from qwengine_b200 import decode_pass


class Recorder:
    def __init__(self):
        self.steps, self.n = [], 0

    def buffer_f32(self, n):
        self.n += 1
        return self.n - 1

    buffer_q8k = buffer_f32

    def __getattr__(self, name):
        return lambda *a, **kw: self.steps.append((name, a, kw))


def record(**kw):
    ps = Recorder()
    decode_pass.build(ps, lambda spec, rows: spec.name, **kw)
    return [s for s in ps.steps if s[0] != "set_peer_store"]


def test_without_them_nothing_changes():
    names = [s[0] for s in record()]
    assert "qk_norm_rope" not in names and "adjust_logits" not in names
    assert names == [s[0] for s in record(heads=dict(a=1), rules=dict(b=2)) if s[0] not in ("qk_norm_rope", "adjust_logits")]


def test_heads_behind_the_projections_and_rules_before_the_top_k():
    steps = record(n_layers=8, heads=dict(positions="p"), rules=dict(penalties="r"))
    at = [i for i, s in enumerate(steps) if s[0] == "qk_norm_rope"]
    assert len(at) == 2
    for i, il in zip(at, (3, 7)):
        assert [s[1][0] for s in steps[i - 3:i]] == [f"l{il}.q_gate", f"l{il}.k", f"l{il}.v"] and steps[i + 1][0] == "quantize"
        q, k, D = steps[i][1]
        assert q["n_heads"] * q["head"] == 12288 and k["n_heads"] * D == 1024 and D == 256 and steps[i][2] == dict(positions="p")
    assert [s[0] for s in steps[-2:]] == ["adjust_logits", "topk"] and steps[-3][1][0] == "lm_head"
    assert steps[-2][1][0] == steps[-1][1][0] and steps[-2][2] == dict(penalties="r")

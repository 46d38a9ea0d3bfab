"""What Pass refuses of its arguments before it comes to the library."""
import types

import pytest
import torch

import qwengine_b200 as q


def test_frequencies_without_positions():
    ps = q.Pass.__new__(q.Pass)
    ps.ctx, ps.lib, ps.max_nb, ps.h = types.SimpleNamespace(device=torch.device("cpu")), None, 2, None
    with pytest.raises(ValueError, match="positions"):
        ps.qk_norm_rope(dict(buf=0, n_heads=1), None, 64, None, torch.ones(8, dtype=torch.float64))

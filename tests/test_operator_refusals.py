"""fmidx.head and fmidx.constraint refuse arguments that are no tensors with a
TypeError that names them (no GPU needed)."""
import pytest
import torch


@pytest.mark.parametrize("name", ["bias", "residual", "out"])
def test_head_scores_wants_tensors(name):
    from fmidx.head import head_scores

    h, w = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match=name):
        head_scores(h, w, **{name: [0.0] * 5})


def test_prefix_constraint_wants_tensors():
    from fmidx.constraint import prefix_constraint

    t = torch.zeros((2, 3), dtype=torch.int64)
    lo = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(TypeError, match="tokens"):
        prefix_constraint(None, t.tolist(), 8)
    with pytest.raises(TypeError, match="lo"):
        prefix_constraint(None, t, 8, lo=[0, 0], hi=lo)
    with pytest.raises(TypeError, match="hi"):
        prefix_constraint(None, t, 8, lo=lo, hi=3)

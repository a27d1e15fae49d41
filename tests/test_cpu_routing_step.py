"""
The routing options of the training step without a GPU: what RasterStep refuses when it is built (with a capacity given, building launches
nothing), and sizes that the operators refuse.
"""
import pytest
import torch

from common import make_case
from igs_b200 import ops, pipeline


def build(**options):
    _, d = make_case(24, 40, 20, seed=3)
    return pipeline.RasterStep(d["means"], d["scales"], d["rotations"], d["features"], d["target"], capacity=1024, **options)


@pytest.mark.parametrize("state", [
    torch.arange(4)[::2],              # every second word
    torch.arange(6).view(2, 3)[:, 1],  # a column of a table
    torch.arange(1).expand(2),         # one word twice: the second would be read past its storage
], ids=["strided", "column", "expanded"])
def test_step_refuses_a_state_that_is_not_two_words_side_by_side(state):
    assert state.dtype == torch.int64 and state.numel() == 2
    with pytest.raises(ValueError, match="rng_state"):
        build(gate_dropout=dict(p=0.5, rng_state=state))


@pytest.mark.parametrize("shape", [(2,), (1, 2), (2, 1)])
def test_step_moves_the_offset_whatever_the_shape(shape):
    states = torch.arange(6).view(3, 2)  # the second of three rows, and nothing beside it
    step = build(gate_dropout=dict(p=0.5, rng_state=states[1].view(shape)))
    for _ in range(2):
        step._next_mask()
    assert states.tolist() == [[0, 1], [2, 5], [4, 5]]


@pytest.mark.parametrize("h,w,n", [(4, 6, (1 << 32) + 3), (0, (1 << 32) + 5, 7), ((1 << 32) + 4, 0, 7), (4, 6, 1 << 31)])
def test_sizes_past_the_entry_points_integers_are_refused(h, w, n, monkeypatch):
    """An entry point takes 32-bit sizes and would see the low 32 bits of these: 3 Gaussians, 5 columns. (Tensors without storage.)"""
    monkeypatch.setattr(ops, "_check_input", lambda t, name, dtype=None: None)  # which wants CUDA tensors
    xys, conics = torch.empty(n, 2, device="meta"), torch.empty(n, 3, device="meta")
    topk = torch.empty(h, w, 10, dtype=torch.int32, device="meta")
    with pytest.raises(RuntimeError, match="2\\^26 Gaussians"):
        ops._check_lists(h, w, xys, conics, topk)
    assert ops._check_lists(4, 6, xys[:7], conics[:7], torch.empty(4, 6, 10, device="meta"))[:3] == (4, 6, 7)

"""Positions that a RotaryEmbedding on several axes takes, without a GPU: which
axis and which sequence each row is, and what is refused."""

import pytest
import torch

from polarquant_kv import rotary


@pytest.fixture
def handed_over(monkeypatch):
    """embedding(query, None, positions) -> the positions that the rotation gets."""
    monkeypatch.setattr(rotary, "apply_rotary", lambda q, k, positions, f, **kw: positions)
    return lambda e, B, positions: e(torch.zeros(B, 2, positions.shape[-1], 64), None, positions)


@pytest.mark.parametrize("B,T", [(8, 1), (1, 5), (2, 3), (4, 7)])
def test_a_row_per_sequence_is_on_every_axis(handed_over, B, T):
    e = rotary.RotaryEmbedding(64, sections=(12, 10, 10))
    text = torch.randint(0, 1000, (B, T))
    got = handed_over(e, B, text)
    assert got.shape == (3, B, T) and all(torch.equal(axis, text) for axis in got)


def test_axes_in_front_stay(handed_over):
    e = rotary.RotaryEmbedding(64, sections=(12, 10, 10))
    for B, shape in ((8, (3, 8, 4)), (3, (3, 3, 4)), (8, (3, 4)), (1, (3, 4)), (2, (3, 2, 4))):
        positions = torch.randint(0, 1000, shape)
        assert torch.equal(handed_over(e, B, positions), positions)
    assert handed_over(e, 3, torch.arange(4)).shape == (3, 4)
    one = rotary.RotaryEmbedding(64, sections=(32,))
    for B, shape in ((1, (1, 4)), (5, (1, 4)), (5, (5, 4)), (5, (1, 5, 4))):
        positions = torch.randint(0, 1000, shape)
        assert torch.equal(handed_over(one, B, positions).expand(1, B, 4), positions.expand(1, B, 4))
    flat = rotary.RotaryEmbedding(64)
    assert handed_over(flat, 3, torch.zeros(3, 4)).shape == (3, 4)


def test_rows_that_could_be_either_or_neither_are_refused(handed_over):
    e = rotary.RotaryEmbedding(64, sections=(12, 10, 10))
    with pytest.raises(ValueError, match="could be of 3 sequences or on 3 axes"):
        handed_over(e, 3, torch.zeros(3, 4, dtype=torch.int64))
    for B, shape in ((2, (5, 4)), (2, (4, 2, 4)), (8, (2, 8, 4)), (2, (1, 4))):
        with pytest.raises(ValueError, match="positions must be"):
            handed_over(e, B, torch.zeros(shape, dtype=torch.int64))


def test_positions_of_other_ranks_are_the_rotation_s_to_refuse():
    e = rotary.RotaryEmbedding(64, sections=(12, 10, 10))
    for positions in (torch.tensor(3), torch.zeros(3, 2, 4, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="positions must be"):
            rotary.check_axes(e.axes, e.positions_by_axis(positions, 2), 32, 2, 4)

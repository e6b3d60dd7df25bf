"""Beam selection over rows of any alignment: which beam wins a tie, and every bit of the scores, go by the rows' values alone (gpu)."""

from __future__ import annotations

import pytest
import torch

from lastkv_amd import ops
from test_gpu_search import DEV, check, logits_of, scores_of

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [9, 1023, 2050, 32001, 50257])
def test_equal_beams_of_an_odd_vocabulary(V, dtype):
    """Rows that follow each other without padding begin at every alignment; equal ones tie in every bit, lowest beam first."""

    for seed in range(6):
        rows = logits_of(100 * seed + V, 2, 1, V, dtype).expand(2, 9, V).contiguous()
        check(rows, torch.full((2, 9), -1.25, device=DEV), 13)  # (13 of 9 beams: the cut lies inside a tie)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride", [32001, 32008, 32003, 40000])
@pytest.mark.parametrize("lead", [0, 1, 5, 6])
def test_a_rows_place_in_memory_changes_no_bit(stride, lead, dtype):
    V, B, K = 31987, 2, 5
    x, s = logits_of(3, B, K, V, dtype), scores_of(4, B, K)
    room = torch.zeros(lead + B * K * stride, dtype=dtype, device=DEV)
    view = room[lead:].view(B, K, stride)[:, :, :V]
    view.copy_(x)
    for a, b in zip(ops.beam_select(x, s, 40), ops.beam_select(view, s, 40)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 4, 5, 7, 8, 9, 15, 17, 2047, 2048, 2049, 8191, 8192, 8193, 8199])
def test_every_value_of_rows_around_a_piece_counts(V, dtype):
    """The best value at the row's ends and beside the borders of pieces and slices, what surrounds the rows being larger."""

    K = 3
    for lead in (0, 1, 3):
        room = torch.full((lead + K * (V + 5) + 8,), 50.0, dtype=dtype, device=DEV)
        view = room[lead:lead + K * (V + 5)].view(1, K, V + 5)[:, :, 2:2 + V]
        view.copy_(logits_of(V, 1, K, V, dtype))
        for at in sorted({0, 1, V // 2, V - 2, V - 1, min(V - 1, 2047), min(V - 1, 2048)} & set(range(V))):
            kept = view[0, 1, at].clone()
            view[0, 1, at] = 20
            got = check(view, torch.zeros(1, K, device=DEV), 4)
            assert (int(got[1][0, 0]), int(got[2][0, 0])) == (1, at) or V <= 2
            view[0, 1, at] = kept

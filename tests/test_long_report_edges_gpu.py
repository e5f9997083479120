"""Rotary positions and windowed attention on the device where a call can go wrong: one long sequence among many short ones."""
import pytest
import torch

from tests.test_long_reports_gpu import run_case

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("lengths,first,H,Hk,D,window,sinks", [
    ([3] * 40 + [700] + [9] * 50 + [400, 1, 23, 0, 22], 0, 2, 1, 64, (20, 10), 40),       # a step of the smallest sequences: two blocks in 44 rows
    ([30] * 60 + [900] + [30] * 30, 5, 2, 2, 32, (100, 0), 4),                            # one block
    ([64] * 70 + [500, 66, 65, 98], 0, 4, 2, 128, (63, 20), 90),                          # just too short, and just long enough
    ([5] * 20 + [1500], 0, 1, 1, 64, (600, -1), 3),                                       # ... with the rows of a key tile split over workgroups
])
def test_sinks_of_packed_sequences_most_of_which_are_short(lengths, first, H, Hk, D, window, sinks, dtype):
    run_case(dtype, None, None, None, H, Hk, D, window, sinks, lengths=lengths, first=first, tail=2, seed=len(lengths))

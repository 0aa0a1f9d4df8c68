"""QuantAttention's host side without a GPU: the step's indexes and the refusals."""
import pytest
import torch
from torch import nn

from dscquant_amd.core.attention import QuantAttention, step
from dscquant_amd.core.linear import QuantLinear


class _Config:
    weight_bits = activation_bits = 4


def test_step_of_mixed_sequences():
    tables = torch.tensor([[4, 1, 9], [7, 3, 0], [2, 5, 8]], dtype=torch.int32)
    cos = torch.zeros(64, 8)
    s = step(tables, [0, 15, 20], [18, 1, 0], 16, cos, cos)
    assert s.lengths.tolist() == [18, 16, 20] and s.starts.tolist() == [0, 18, 19, 19]
    assert s.max_q == 18 and s.max_length == 20
    assert s.slots.tolist() == [4 * 16 + i for i in range(16)] + [16, 17] + [7 * 16 + 15]
    assert s.positions.tolist() == [*range(18), 15]
    assert s.slots.dtype == s.positions.dtype == torch.int64
    assert s.lengths.dtype == s.starts.dtype == torch.int32


def test_step_of_single_tokens_and_none():
    tables = torch.tensor([[4], [7]], dtype=torch.int32)
    s = step(tables, [0, 9], [1, 1], 16)
    assert s.starts is None and s.positions is None and s.max_q == 1 and s.max_length == 10
    assert s.slots.tolist() == [64, 7 * 16 + 9]
    s = step(tables, [3, 0], [0, 0], 16)
    assert s.slots.numel() == 0 and s.starts.tolist() == [0, 0, 0] and s.lengths.tolist() == [3, 0]


def test_step_refusals():
    tables = torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="2 sequences have tables, 1 and 2 counts"):
        step(tables, [0], [1, 1], 16)
    with pytest.raises(RuntimeError, match="17 tokens do not fit 1 pages of 16"):
        step(tables, [16, 0], [1, 1], 16)
    with pytest.raises(RuntimeError, match="negative"):
        step(tables, [0, -1], [1, 1], 16)


def test_module_refuses_projections_of_other_sizes():
    lin = lambda n, k: QuantLinear(nn.Linear(k, n, bias=False), _Config())  # noqa: E731
    QuantAttention(lin(256, 96), lin(128, 96), lin(128, 96), lin(96, 256), 4, 2, 64)
    with pytest.raises(RuntimeError, match="need projections of other sizes"):
        QuantAttention(lin(256, 96), lin(64, 96), lin(128, 96), lin(96, 256), 4, 2, 64)
    with pytest.raises(RuntimeError, match="o projection takes 128 of 256"):
        QuantAttention(lin(256, 96), lin(128, 96), lin(128, 96), lin(96, 128), 4, 2, 64)

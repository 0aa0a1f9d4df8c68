"""QuantAttention (dscquant_amd/core/attention.py): the projections, the 4-bit cache and the
attention over it run together, prompts and single tokens."""
import pytest
import torch
from torch import nn

from dscquant_amd import kv4
from dscquant_amd.core.attention import QuantAttention, step
from dscquant_amd.core.linear import QuantLinear

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}


class _Config:
    weight_bits = activation_bits = 4


def block(gpu, dtype, heads, kv_heads, D, hidden, seed=0, plain_o=False, **options):
    torch.manual_seed(seed)

    def linear(rows, cols):
        base = nn.Linear(cols, rows, bias=False)
        base.weight.data.normal_(0, cols ** -0.5)
        layer = QuantLinear(base.to(DT[dtype]).to(gpu), _Config())
        layer.enabled = True
        return layer

    o = linear(hidden, heads * D)
    if plain_o:  # hands the attention's result through as it is
        assert hidden == heads * D
        o.base.weight.data.copy_(torch.eye(hidden))
        o.enabled = False
    return QuantAttention(linear(heads * D, hidden), linear(kv_heads * D, hidden),
                          linear(kv_heads * D, hidden), o, heads, kv_heads, D, **options)


def angles(rows, R, gpu):
    a = torch.arange(rows)[:, None] * 10000.0 ** (-torch.arange(0, R, 2) / R)
    return a.cos().float().to(gpu), a.sin().float().to(gpu)


@pytest.mark.parametrize("dtype,heads,kv_heads,D,rotate", [
    ("fp16", 4, 2, 64, True), ("bf16", 4, 1, 128, True), ("fp16", 2, 2, 128, False)])
@torch.no_grad()
def test_block_is_its_parts(gpu, dtype, heads, kv_heads, D, rotate):
    hidden = 256
    attn = block(gpu, dtype, heads, kv_heads, D, hidden, rotate=rotate, window=30)
    cos, sin = angles(64, D, gpu)
    tables = torch.tensor([[3, 0, 5], [1, 4, 2]], dtype=torch.int32, device=gpu)
    x = torch.randn(42, hidden, device=gpu).to(DT[dtype])
    s = step(tables, [0, 0], [37, 5], 16, cos, sin)
    cache, other = attn.new_cache(6, 16), attn.new_cache(6, 16)
    got = attn(x, cache, s)
    q, k, v = (m(x).reshape(42, -1, D) for m in (attn.q, attn.k, attn.v))
    q = kv4.append(other, q, k, v, s.slots, s.positions, cos, sin, rotate=rotate)
    y = kv4.attention(other, q, tables, s.lengths, s.starts, 37, 37, window=30)
    assert torch.equal(cache, other)
    assert torch.equal(got, attn.o(y.reshape(42, heads * D)))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@torch.no_grad()
def test_token_by_token_is_the_prompt(gpu, dtype):
    """A token's keys and values do not depend on what it comes with, so the cache is the same
    byte for byte; the results differ by the roundings of the two kernels alone: each within
    2^-11 (bf16: 2^-8) of the result and 2^-10 of sum p |v|, which is less than eight times
    the result over these few tokens."""
    heads, kv_heads, D = 4, 2, 64
    attn = block(gpu, dtype, heads, kv_heads, D, heads * D, plain_o=True)
    cos, sin = angles(64, D, gpu)
    tables = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=gpu)
    x = torch.randn(40, heads * D, device=gpu).to(DT[dtype])
    whole, alone = attn.new_cache(3, 16), attn.new_cache(3, 16)
    a = attn(x, whole, step(tables, [0], [40], 16, cos, sin))
    b = torch.cat([attn(x[i:i + 1], alone, step(tables, [i], [1], 16, cos, sin))
                   for i in range(40)])
    assert torch.equal(whole, alone)
    unit = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
    assert (a.float() - b.float()).norm() <= 2 * (unit + 8 * 2.0 ** -10) * a.float().norm()


@torch.no_grad()
def test_empty_step(gpu):
    attn = block(gpu, "fp16", 4, 2, 64, 256)
    cache = attn.new_cache(2, 16)
    tables = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    x = torch.empty(0, 256, dtype=torch.float16, device=gpu)
    assert attn(x, cache, step(tables, [3], [0], 16)).shape == (0, 256)

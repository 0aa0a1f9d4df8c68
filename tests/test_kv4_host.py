"""The 4-bit key/value cache without a GPU: the oracle's own rules, and the checks of the
C entry points (include/dscq.h, dscq_kv_*) and of the Python layer that need no device."""
import numpy as np
import pytest
import torch

from dscquant_amd import _lib, kv4
from oracle import kv4 as oracle

B16 = 16  # stands for a 16-byte aligned device pointer: every call here returns before a launch


def _einval(name, *args):
    L = _lib.lib()
    assert getattr(L, name)(*args) == -1
    return L.dscq_last_error().decode()


def _append(q=B16, dtype=0, T=1, Hq=4, H=2, D=128, positions=None, cos=None, sin=None, rows=0,
            rotary=0, slots=B16, cache=B16, pages=3, P=16, k=B16, q_out=B16):
    return ("dscq_kv_append", q, Hq * D, D, k, H * D, D, B16, H * D, D, dtype, T, Hq, H, D,
            positions, cos, sin, rows, rotary, 0, 0, slots, cache, pages, P, q_out, None)


@pytest.mark.parametrize("change,message", [
    (dict(dtype=1), "kv cache: only FP16 and BF16 rows are supported"),
    (dict(D=96), "kv cache: head_dim must be 64 or 128 (got 96)"),
    (dict(P=24), "kv cache: page size must be a multiple of 16 up to 4096 (got 24)"),
    (dict(P=0), "kv cache: page size must be a multiple of 16 up to 4096 (got 0)"),
    (dict(pages=0), "kv cache: invalid dimensions"),
    (dict(H=0), "kv cache: invalid dimensions"),
    (dict(cache=8), "kv cache: needs a 16-byte aligned buffer"),
    (dict(T=-1), "kv append: invalid dimensions"),
    (dict(k=None), "kv append: null buffer"),
    (dict(slots=None), "kv append: null buffer"),
    (dict(q_out=None), "kv append: null buffer"),
    (dict(cos=B16), "kv append: cos, sin and positions go together"),
    (dict(cos=B16, sin=B16, rows=4, rotary=64), "kv append: cos, sin and positions go together"),
    (dict(cos=B16, sin=B16, positions=B16, rows=4, rotary=24),
     "kv append: the turned part of a head must be a multiple of 16 up to head_dim (got 24)"),
    (dict(cos=B16, sin=B16, positions=B16, rows=4, rotary=144),
     "kv append: the turned part of a head must be a multiple of 16 up to head_dim (got 144)"),
])
def test_c_append_argument_checks(change, message):
    assert _einval(*_append(**change)) == message


def test_c_empty_calls_launch_nothing():
    L = _lib.lib()
    name, *args = _append(T=0)
    assert getattr(L, name)(*args) == 0
    assert L.dscq_kv_read(B16, 3, 16, 2, 128, B16, 0, 0, 0, B16, B16, None) == 0
    name, *args = _attention(T=0)
    assert getattr(L, name)(*args) == 0


def test_c_read_argument_checks():
    assert _einval("dscq_kv_read", B16, 3, 16, 2, 128, None, 1, 0, 0, B16, B16, None) == \
        "kv read: null buffer"
    assert _einval("dscq_kv_read", B16, 3, 16, 2, 32, B16, 1, 0, 0, B16, B16, None) == \
        "kv cache: head_dim must be 64 or 128 (got 32)"
    assert _einval("dscq_kv_read", B16, 3, 16, 2, 128, B16, -1, 0, 0, B16, B16, None) == \
        "kv read: invalid dimensions"


def _attention(T=1, Hq=4, H=2, D=128, dtype=0, tables=B16, width=4, starts=None, B=1, max_q=1,
               max_length=64, scale=0.1, window=0, q=B16):
    return ("dscq_kv_attention", q, Hq * D, D, dtype, T, Hq, B16, 3, 16, H, D, tables, width, B16,
            starts, B, max_q, max_length, scale, window, B16, None, None, 0, None)


@pytest.mark.parametrize("change,message", [
    (dict(Hq=5), "kv attention: query heads must be a multiple of the cache's heads"),
    (dict(Hq=0), "kv attention: query heads must be a multiple of the cache's heads"),
    (dict(B=65536, T=65536), "kv attention: invalid dimensions"),
    (dict(window=-1), "kv attention: invalid dimensions"),
    (dict(max_length=-1), "kv attention: invalid dimensions"),
    (dict(width=1 << 40), "kv attention: invalid dimensions"),
    (dict(scale=0.0), "kv attention: scale must be positive"),
    (dict(scale=float("nan")), "kv attention: scale must be positive"),
    (dict(scale=float("inf")), "kv attention: scale must be positive"),
    (dict(q=None), "kv attention: null buffer"),
    (dict(tables=None), "kv attention: null buffer"),
    (dict(max_q=2), "kv attention: without starts every sequence has one query"),
    (dict(T=2), "kv attention: without starts there are B queries"),
    (dict(dtype=1), "kv cache: only FP16 and BF16 rows are supported"),
])
def test_c_attention_argument_checks(change, message):
    assert _einval(*_attention(**change)) == message


def test_c_workspace_query():
    L = _lib.lib()
    assert L.dscq_kv_attention_workspace_bytes(0, 4, 2, 128, 1, 64, 0) == 0
    assert L.dscq_kv_attention_workspace_bytes(1, 4, 2, 128, 0, 64, 0) == 0
    assert L.dscq_kv_attention_workspace_bytes(1, 4, 2, 128, 1, 0, 0) >= 0
    assert L.dscq_kv_attention_workspace_bytes(1, 5, 2, 128, 1, 64, 0) == -1
    # Windows that no sequence fills, up to the largest number, plan as none does.
    for max_q in (1, 100):
        plain = L.dscq_kv_attention_workspace_bytes(2, 8, 2, 128, max_q, 100000, 0)
        assert plain > 0
        for window in ((1 << 28) + 1, (1 << 63) - 1):
            assert L.dscq_kv_attention_workspace_bytes(2, 8, 2, 128, max_q, 100000, window) == plain


def test_python_refuses_cpu_tensors_and_layouts():
    cache = kv4.new_cache(2, 16, 2, 64, device="cpu")
    assert cache.shape == (2, 2, 16, 72) and cache.dtype == torch.uint8
    x = torch.zeros(1, 2, 64, dtype=torch.float16)
    where = torch.zeros(1, dtype=torch.int64)
    for call in (lambda: kv4.append(cache, x, x, x, where), lambda: kv4.read(cache, where),
                 lambda: kv4.attention(cache, x, where.int().reshape(1, 1), where.int())):
        with pytest.raises(RuntimeError, match="Expected contiguous CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match="head_dim must be 64 or 128"):
        kv4.new_cache(2, 16, 2, 96, device="cpu")
    with pytest.raises(RuntimeError, match="page size must be a multiple of 16"):
        kv4.new_cache(2, 20, 2, 64, device="cpu")
    with pytest.raises(RuntimeError, match="key/value heads"):
        kv4.new_cache(2, 16, 0, 64, device="cpu")
    with pytest.raises(RuntimeError, match="at least one page"):
        kv4.new_cache(0, 16, 2, 64, device="cpu")


def test_slots_of_places():
    tables = torch.tensor([[5, 2], [0, 7]], dtype=torch.int32)
    got = kv4.slots(tables, torch.tensor([0, 0, 1, 1]), torch.tensor([3, 17, 0, 31]), 16)
    assert got.tolist() == [5 * 16 + 3, 2 * 16 + 1, 0, 7 * 16 + 15]


# ---------------------------------------------------------------- the oracle's own rules

@pytest.mark.parametrize("D", [64, 128])
def test_oracle_hadamard_is_sylvester(D):
    i = np.arange(D)
    parity = np.array([[bin(a & b).count("1") & 1 for b in i] for a in i])
    assert np.array_equal(oracle.hadamard(np.eye(D)), 1.0 - 2.0 * parity)


@pytest.mark.parametrize("P,D", [(16, 64), (48, 128)])
def test_oracle_places_fill_a_block_once(P, D):
    taken = np.zeros((P * D, 2), int)
    for byte, shift in oracle.places(P, D):
        np.add.at(taken, (byte, shift // 4), 1)
    assert (taken == 1).all()


def test_oracle_rows_stand_for_themselves_to_half_a_step():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((64, 128)) * np.exp(rng.uniform(-8, 8, (64, 1)))).astype(np.float32)
    x[3] = np.abs(x[3])
    x[4] = -np.abs(x[4])
    x[5] = 0
    codes, words = oracle.quantize(x)
    scale, zero = words.view(np.float32), (words & 15).astype(np.float64)
    got = (codes - zero[:, None]) * scale[:, None].astype(np.float64)
    # Half a step, and at the ends half a step more: the zero-point is rounded too.
    assert (np.abs(got - x) <= scale[:, None] * (1.0 + 2 ** -18)).all()
    assert np.mean(np.abs(got - x) <= scale[:, None] * (0.5 + 2 ** -18)) > 0.95
    assert (got[5] == 0).all()
    want = np.maximum((np.maximum(x.max(1), 0) - np.minimum(x.min(1), 0)) / 15, 1e-8)
    assert (scale >= want).all() and (scale <= want * (1 + 2 ** -18)).all()


def test_oracle_cache_round_trip_and_rows_that_are_not_finite():
    rng = np.random.default_rng(1)
    cache = rng.integers(0, 256, (3, 2, 32, 72)).astype(np.uint8)
    before = cache.copy()
    k, v = (rng.standard_normal((5, 2, 64)).astype(np.float32) for _ in range(2))
    k[2, 1, 7] = np.inf
    slots = [33, 95, 0, -1, 96]
    oracle.put(cache, slots, k, v)
    got_k, got_v = (x.reshape(-1, 2, 64) for x in oracle.values(cache))
    for i in (0, 1, 2):
        for h in range(2):
            codes, words = oracle.quantize(v[i, h])
            want = (codes.astype(np.float32) - np.float32(words & 15)) * words.view(np.float32)
            assert np.array_equal(got_v[slots[i], h], want)
    assert np.isnan(got_k[0, 1]).all() and np.isfinite(got_k[0, 0]).all()
    changed = (cache != before).reshape(3, 2, -1).sum()
    assert 0 < changed <= 3 * 2 * (64 + 8)


def test_c_attention_of_more_rows_than_a_launch_holds():
    """A grid of 2^32 threads wraps: refused.  A large max_q alone is a bound and no row."""
    message = "kv attention: invalid dimensions"
    rows = dict(Hq=2, starts=B16, max_q=(1 << 30) - 1, max_length=64)
    assert _einval(*_attention(T=1 << 30, **rows)) == message
    assert _einval(*_attention(T=(1 << 30) - (1 << 19) + 1, **rows)) == message
    name, *args = _attention(T=0, **rows)
    assert getattr(_lib.lib(), name)(*args) == 0

"""The 4-bit paged key/value cache on the GPU (dscquant_amd/kv4.py) against oracle/kv4.py.

append and read are compared bit for bit: every step of the row rule is one fp32
operation.  attention is compared element by element with the 64-bit result on the numbers
the cache holds, within a bound from the formula: with weights p_j that carry a relative
error of at most d, the output is off by at most 2 d sum p_j |v_j|.  Here d counts the
fp32 scores (products of an 11-bit and a 5-bit number are exact; at most 128 additions of
2^-24 relative to sum |q k| scale, under 32 for these inputs: 2^-12), and the rounding of
the weights to 11 bits for the matrix cores counts once (2^-11); then the output's own
rounding.
"""
import numpy as np
import pytest
import torch

from dscquant_amd import kv4
from oracle import kv4 as oracle

pytestmark = pytest.mark.gpu

DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
UNIT = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def f32(t):
    return t.detach().float().cpu().numpy()


def random_cache(rng, pages, H, P, D, key_scale=0.2, value_scale=0.2):
    """A cache of random codes and words, as numpy bytes."""
    cache = rng.integers(0, 256, (pages, H, P, D + 8)).astype(np.uint8)
    flat = cache.reshape(pages, H, -1)
    for which, scale in enumerate((key_scale, value_scale)):
        s = (scale * np.exp(rng.uniform(-1, 1, (pages, H, P)))).astype(np.float32)
        words = (s.view(np.uint32) & ~np.uint32(15)) | rng.integers(3, 13, s.shape).astype(np.uint32)
        at = P * D + which * P * 4
        flat[:, :, at:at + 4 * P] = words.view(np.uint8).reshape(pages, H, 4 * P)
    return cache


# ------------------------------------------------------------------- append and read

APPENDS = [
    # T, Hq, H, D, P, rotary (0: none), interleaved, rotate, dtype
    (1, 4, 2, 128, 16, 128, False, False, "fp16"),
    (1, 3, 3, 64, 64, 64, False, True, "bf16"),
    (17, 6, 2, 128, 32, 64, True, True, "fp16"),
    (33, 2, 1, 64, 16, 32, False, False, "fp16"),
    (16, 4, 4, 128, 48, 0, False, True, "bf16"),
    (5, 5, 1, 64, 128, 16, True, False, "bf16"),
]


@pytest.mark.parametrize("T,Hq,H,D,P,R,interleaved,rotate,dtype", APPENDS)
@pytest.mark.parametrize("fused", [False, True])
def test_append_and_read_are_bit_exact(gpu, T, Hq, H, D, P, R, interleaved, rotate, dtype, fused):
    g = torch.Generator().manual_seed(T * 1000 + D + Hq)
    dt = DT[dtype]
    q, k, v = (torch.randn(T, h, D, generator=g) for h in (Hq, H, H))
    k[..., 5] *= 30
    v[0] = 0
    v[T // 2, :, :] = v[T // 2].abs()
    if fused:  # parts of one product's rows, at an odd element offset
        rows = torch.zeros(T, (Hq + 2 * H) * D + 3, dtype=dt)
        x = rows[:, 1:-2].view(T, Hq + 2 * H, D)
        x.copy_(torch.cat((q, k, v), 1))
        rows = rows.to(gpu)
        x = rows[:, 1:-2].view(T, Hq + 2 * H, D)
        q, k, v = x[:, :Hq], x[:, Hq:Hq + H], x[:, Hq + H:]
    else:
        q, k, v = (x.to(dt).to(gpu) for x in (q, k, v))
    pages = T // P + 3
    rng = np.random.default_rng(T)
    slots = rng.permutation(pages * P)[:T]
    if T > 4:
        slots[1], slots[3] = -1, pages * P
    cos = sin = pos = None
    table = 70
    if R:
        angle = torch.rand(table, R // 2, generator=g) * 6
        cos, sin = angle.cos(), angle.sin()
        pos = torch.randint(0, table, (T,), generator=g)
        if T > 6:
            pos[5] = table
            pos[6] = -1
    cache = torch.full((pages, H, P, D + 8), 0xA5, dtype=torch.uint8, device=gpu)
    at = torch.from_numpy(slots).to(gpu)
    on = lambda t: None if t is None else t.to(gpu)  # noqa: E731
    got = kv4.append(cache, q, k, v, at, positions=on(pos), cos=on(cos), sin=on(sin),
                     interleaved=interleaved, rotate=rotate)
    qn, kn, vn = f32(q), f32(k), f32(v)
    known = np.ones(T, bool)
    if R:
        known = ((pos >= 0) & (pos < table)).numpy()
        row = np.where(known, pos.numpy(), 0)
        c, s = cos.numpy()[row], sin.numpy()[row]
        qn, kn = (oracle.turn(x, c, s, interleaved) for x in (qn, kn))
    if rotate:
        qn, kn = oracle.hadamard(qn) * np.float32(1 / D), oracle.hadamard(kn)
    want = np.full((pages, H, P, D + 8), 0xA5, np.uint8)
    oracle.put(want, np.where(known, slots, -1), kn, vn)
    qn[~known] = np.nan
    assert np.array_equal(f32(got), f32(torch.from_numpy(qn).to(dt)), equal_nan=True)
    assert np.array_equal(cache.cpu().numpy(), want)

    rk, rv = kv4.read(cache, at, dt, rotate=rotate)
    kept = known & (slots >= 0) & (slots < pages * P)
    ok, ov = (x.reshape(pages * P, H, D)[np.where(kept, slots, 0)] for x in oracle.values(want))
    if rotate:
        ok = oracle.hadamard(ok) * np.float32(1 / D)
    inside = (slots >= 0) & (slots < pages * P)
    for have, expect in ((rk, ok), (rv, ov)):
        expect = f32(torch.from_numpy(np.where(inside[:, None, None], expect, 0)).to(dt))
        assert np.array_equal(f32(have)[kept | ~inside], expect[kept | ~inside])


def test_append_without_queries_and_empty_steps(gpu):
    cache = kv4.new_cache(2, 16, 2, 64, gpu)
    x = torch.randn(3, 2, 64, device=gpu).half()
    at = torch.tensor([0, 9, 31], device=gpu)
    assert kv4.append(cache, None, x, x, at) is None
    with_q = kv4.new_cache(2, 16, 2, 64, gpu)
    kv4.append(with_q, x, x, x, at)
    assert torch.equal(cache, with_q)
    none = torch.empty(0, 2, 64, dtype=torch.float16, device=gpu)
    assert kv4.append(cache, none, none, none, at[:0]).shape == (0, 2, 64)
    assert kv4.read(cache, at[:0])[0].shape == (0, 2, 64)
    table = torch.zeros(0, 1, dtype=torch.int32, device=gpu)
    assert kv4.attention(cache, none, table, table[:, 0]).shape == (0, 2, 64)


def test_rows_that_are_not_finite_are_nan_to_those_that_see_them(gpu):
    cache = kv4.new_cache(3, 16, 1, 128, gpu)
    k, v = (torch.randn(40, 1, 128, device=gpu).half() for _ in range(2))
    k[20, 0, 3] = float("inf")
    v[30, 0, 9] = float("nan")
    kv4.append(cache, None, k, v, torch.arange(40, device=gpu))
    q = torch.randn(40, 2, 128, device=gpu).half()
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=gpu)
    starts = torch.tensor([0, 40], dtype=torch.int32, device=gpu)
    out = kv4.attention(cache, q, table, starts[1:], starts, max_q=40)
    bad = torch.isnan(out).all(-1).all(-1).cpu()
    assert bad.tolist() == [i >= 20 for i in range(40)]
    assert torch.isfinite(out[:20]).all()
    # A window that has passed the first of them sees the second alone.
    out = kv4.attention(cache, q, table, starts[1:], starts, max_q=40, window=5)
    bad = torch.isnan(out).all(-1).all(-1).cpu()
    assert bad.tolist() == [20 <= i < 25 or 30 <= i < 35 for i in range(40)]


# ------------------------------------------------------------------- attention

def check_attention(gpu, lengths, queries, Hq, H, D, P, dtype, window=0, seed=0, max_length=None,
                    given_starts=True, hide=False, key_scale=0.2, value_scale=0.2, extra_width=1,
                    strided=False, scale=None, pages=None):
    rng = np.random.default_rng(seed)
    per = [-(-n // P) for n in lengths]
    B, width = len(lengths), max([1, *per]) + extra_width
    total = sum(per) + 2
    if pages is None:
        pages = total
    raw = random_cache(rng, pages, H, P, D, key_scale, value_scale)
    perm = rng.permutation(pages)[:total]
    tables = np.full((B, width), 0x7FFFFFF0, np.int32)  # what a table holds past its pages
    used = np.zeros((pages, P), bool)
    at = 0
    for b, n in enumerate(per):
        tables[b, :n] = perm[at:at + n]
        for i in range(n):
            used[perm[at + i], :min(P, lengths[b] - i * P)] = True
        at += n
    # Words of tokens past a sequence's end are NaN; so are those of pages nobody has.
    flat = raw.reshape(pages, H, -1)
    for which in range(2):
        words = flat[:, :, P * D + which * 4 * P:P * D + (which + 1) * 4 * P].reshape(pages, H, P, 4)
        words[~used[:, None].repeat(H, 1)] = 0xFF
        flat[:, :, P * D + which * 4 * P:P * D + (which + 1) * 4 * P] = words.reshape(pages, H, -1)
    hidden = [np.zeros(n, bool) for n in lengths]
    if hide:  # a page outside the cache in the middle
        for b, n in enumerate(lengths):
            if per[b] > 2:
                tables[b, 1] = -1 if b % 2 else pages
                hidden[b][P:2 * P] = True
    starts = np.concatenate(([0], np.cumsum(queries))).astype(np.int32)
    T = int(starts[-1])
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(T, Hq, D, generator=g).to(DT[dtype])
    cache = torch.from_numpy(raw).to(gpu)
    tq = q.to(gpu)
    if strided:
        wide = torch.zeros(T, Hq + 3, D + 5, dtype=q.dtype, device=gpu)
        wide[:, 2:Hq + 2, 1:D + 1] = tq
        tq = wide[:, 2:Hq + 2, 1:D + 1]
    as_gpu = lambda a: torch.from_numpy(np.asarray(a, np.int32)).to(gpu)  # noqa: E731
    call = lambda: kv4.attention(  # noqa: E731
        cache, tq, as_gpu(tables), as_gpu(lengths), as_gpu(starts) if given_starts else None,
        max_q=max(queries), max_length=max(lengths) if max_length is None else max_length,
        window=window, scale=scale, return_lse=True)
    out, lse = call()
    again, lse2 = call()
    assert torch.equal(out.view(torch.int16), again.view(torch.int16)) and torch.equal(lse, lse2)
    keys, values = oracle.values(raw)
    worst = 0.0
    for b, L in enumerate(lengths):
        n = queries[b]
        page = tables[b, :per[b]]
        page = np.where((page >= 0) & (page < pages), page, 0)
        k, v = (x[page].reshape(-1, H, D)[:L] for x in (keys, values))
        qn = f32(q[starts[b]:starts[b + 1]])
        want, sums, spread = oracle.attention(qn, np.where(hidden[b][:, None, None], 0, k),
                                              np.where(hidden[b][:, None, None], 0, v),
                                              np.arange(L - n, L), D ** -0.5 if scale is None else scale,
                                              window, hidden[b])
        have, have_lse = f32(out[starts[b]:starts[b + 1]]), f32(lse[starts[b]:starts[b + 1]])
        top = np.abs(v[~hidden[b]]).max() if (~hidden[b]).any() else 0
        bound = (UNIT[dtype] * np.abs(want) + spread * (2 ** -11 + 2 * 2 ** -12) + 2.0 ** -24
                 + L * 2.0 ** -30 * top)
        # A result past the type's range is an infinity of its sign.
        most = float(torch.finfo(DT[dtype]).max)
        inside = np.abs(want) - bound <= most
        assert np.array_equal(have[~inside], np.sign(want[~inside]) * np.inf)
        at_edge = inside & (np.abs(want) + bound >= most)
        assert np.isfinite(have[inside & ~at_edge]).all()
        err = np.where(inside & ~at_edge, np.abs(np.where(np.isfinite(have), have, 0) - want), 0)
        assert (err <= bound).all(), (b, L, n, float((err / bound).max()))
        worst = max(worst, float((err / bound).max())) if err.size else worst
        seen = np.isfinite(sums)
        assert np.array_equal(np.isfinite(have_lse), seen) and (have_lse[~seen] == -np.inf).all()
        assert (np.abs(have_lse[seen] - sums[seen]) <= 2 ** -12 + np.abs(sums[seen]) * 2 ** -22).all()
        assert (have[~seen] == 0).all()
    return worst


@pytest.mark.parametrize("L", [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 500, 1023])
@pytest.mark.parametrize("D,dtype", [(128, "fp16"), (64, "bf16")])
def test_one_query_at_every_kind_of_length(gpu, L, D, dtype):
    check_attention(gpu, [L], [1], 8, 2, D, 16 if L % 2 else 64, dtype, seed=L)


@pytest.mark.parametrize("Hq,H", [(1, 1), (4, 4), (6, 2), (16, 1), (8, 1), (40, 1), (14, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_head_groups(gpu, Hq, H, D):
    check_attention(gpu, [200, 3, 77], [1, 1, 1], Hq, H, D, 32, "fp16", seed=Hq)
    check_attention(gpu, [150, 40], [40, 33], Hq, H, D, 32, "bf16", seed=Hq)


@pytest.mark.parametrize("given", [False, True])
def test_a_decode_batch_of_ragged_lengths(gpu, given):
    lengths = [1, 700, 16, 0, 333, 64, 2048, 5] if given else [1, 700, 16, 2, 333, 64, 2048, 5]
    queries = [1 if n else 0 for n in lengths]
    check_attention(gpu, lengths, queries, 8, 2, 128, 64, "bf16", given_starts=given)


@pytest.mark.parametrize("Hq,H,D,window", [(32, 16, 64, 0), (16, 16, 128, 0), (32, 16, 64, 1100)])
def test_many_long_sequences_in_equal_shares(gpu, Hq, H, D, window):
    """More long sequences than workgroups for four parts of each: shares that begin and end
    inside sequences, span short and empty ones, and are many or few."""
    lengths = [1, 1500, 0, 40, 1100, 0, 2000, 3, 64, 1025, 17, 1030]
    check_attention(gpu, lengths, [1 if n else 0 for n in lengths], Hq, H, D, 64, "fp16",
                    window=window)
    check_attention(gpu, lengths, [min(n, 1 + i % 8) for i, n in enumerate(lengths)], H, H, D, 16,
                    "bf16", window=window)


@pytest.mark.parametrize("window", [1, 7, 16, 100, 4096])
def test_windows(gpu, window):
    check_attention(gpu, [1, 90, 400], [1, 1, 1], 4, 2, 128, 16, "fp16", window=window)
    check_attention(gpu, [90, 400, 300], [5, 3, 1], 4, 2, 64, 64, "bf16", window=window)
    check_attention(gpu, [90, 400, 300], [70, 130, 300], 4, 2, 128, 64, "fp16", window=window)


@pytest.mark.parametrize("D,dtype", [(128, "fp16"), (128, "bf16"), (64, "fp16")])
@pytest.mark.parametrize("lengths,queries", [
    ([40], [2]), ([40], [40]), ([300, 17], [5, 16]), ([513], [513]), ([257, 0, 1, 64], [129, 0, 1, 64]),
    ([1000, 90], [33, 90]), ([700], [96]),
])
def test_prompts_and_few_queries(gpu, lengths, queries, D, dtype):
    check_attention(gpu, lengths, queries, 8, 2, D, 16, dtype, seed=sum(lengths))
    check_attention(gpu, lengths, queries, 4, 4, D, 64, dtype, seed=sum(lengths) + 1)


def test_pages_outside_the_cache_are_not_seen(gpu):
    check_attention(gpu, [200, 300], [1, 1], 8, 2, 128, 64, "fp16", hide=True)
    check_attention(gpu, [200, 300], [60, 200], 8, 2, 128, 16, "fp16", hide=True)
    # The only page a query could see is one of them.
    check_attention(gpu, [48, 48], [1, 1], 4, 2, 64, 16, "bf16", hide=True, window=1)


def test_more_queries_than_tokens_see_nothing_first(gpu):
    """A sequence whose queries outnumber its cached tokens: the first see none."""
    check_attention(gpu, [3, 0], [5, 4], 4, 2, 128, 16, "fp16", max_length=16)
    check_attention(gpu, [20, 0], [150, 140], 4, 2, 64, 16, "bf16", max_length=32)


def test_strides_and_bounds(gpu):
    check_attention(gpu, [120, 64], [1, 1], 6, 3, 128, 32, "fp16", strided=True)
    check_attention(gpu, [120, 64], [100, 2], 6, 3, 64, 32, "bf16", strided=True)
    # The host's bound on the length: far over, and under (a longer context is still whole).
    check_attention(gpu, [120, 1500], [1, 1], 8, 2, 128, 16, "fp16", max_length=100000)
    check_attention(gpu, [120, 1500], [1, 1], 8, 2, 128, 16, "fp16", max_length=1)
    check_attention(gpu, [120, 1500], [70, 80], 8, 2, 128, 16, "fp16", max_length=1)


@pytest.mark.parametrize("key_scale,value_scale,scale", [(1e-8, 1e-8, None), (4.0, 3000.0, 0.002),
                                                         (0.2, 1e-6, None), (2e-5, 0.2, 900.0)])
def test_scales_of_keys_and_values(gpu, key_scale, value_scale, scale):
    """fp16's range bounds neither: bf16 holds small values, scores go with scale * key."""
    for dtype in ("bf16", "fp16") if value_scale > 1e-3 else ("bf16",):
        check_attention(gpu, [300, 40], [1, 1], 4, 2, 128, 16, dtype, key_scale=key_scale,
                        value_scale=value_scale, scale=scale)
        check_attention(gpu, [300, 140], [90, 140], 4, 2, 128, 16, dtype, key_scale=key_scale,
                        value_scale=value_scale, scale=scale)


def test_values_whose_scales_differ_by_a_lot(gpu):
    """Tokens of large values that carry no weight leave the others' sums as they are."""
    D, L, P = 128, 200, 16
    rng = np.random.default_rng(3)
    for late in (10, 150):
        raw = random_cache(rng, 13, 1, P, D)
        flat = raw.reshape(13, 1, -1)
        words = np.ascontiguousarray(flat[:, 0, P * D:]).view("<u4").reshape(13, 2, P).copy()
        f = words.view("<f4")
        f[late // P, 1, late % P] = 2.0 ** 20    # a value of 1e6 ...
        f[late // P, 0, late % P] = 1e-30
        flat[:, 0, P * D:] = words.view(np.uint8).reshape(13, -1)
        keys, values = (x.reshape(-1, 1, D) for x in oracle.values(raw))
        q = np.abs(rng.standard_normal((1, 1, D))).astype(np.float16)
        # ... that scores -40 below the others: its weight is e^-40 or so.
        scale = 0.1
        want, _, spread = oracle.attention(q, keys[:L], values[:L], [L - 1], scale)
        t = lambda x: torch.from_numpy(np.asarray(x)).to(gpu)  # noqa: E731
        out = kv4.attention(t(raw), t(q), t(np.arange(13, dtype=np.int32)[None]),
                            t(np.array([L], np.int32)), scale=scale)
        bound = (2 ** -11 * np.abs(want) + spread * 2 ** -10 + 2.0 ** -24
                 + L * 2.0 ** -30 * np.abs(values[:L]).max())
        assert (np.abs(f32(out) - want) <= bound).all()


def test_offsets_past_32_bits(gpu):
    """Pages beyond 4 GiB of the cache."""
    D, P, H = 128, 64, 8
    pages = (5 << 30) // (P * H * (D + 8))
    cache = torch.zeros((pages, H, P, D + 8), dtype=torch.uint8, device=gpu)
    k, v, q = (torch.randn(200, h, D, device=gpu).half() for h in (H, H, 16))
    far = torch.tensor([[pages - 1, 0, pages - 2, pages - 3]], dtype=torch.int32, device=gpu)
    near = torch.arange(4, dtype=torch.int32, device=gpu)[None]
    small = kv4.new_cache(4, P, H, D, gpu)
    n = torch.arange(200, device=gpu)
    got = []
    for c, table in ((cache, far), (small, near)):
        at = kv4.slots(table, torch.zeros_like(n), n, P)
        kv4.append(c, None, k, v, at)
        starts = torch.tensor([0, 200], dtype=torch.int32, device=gpu)
        got.append((*kv4.read(c, at), kv4.attention(c, q, table, starts[1:], starts, max_q=200),
                    kv4.attention(c, q[:1], table, starts[1:])))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_a_long_context_in_parts(gpu):
    """Parts of a context joined by their log sums are the whole context."""
    L, D, P = 30000, 128, 64
    cache = kv4.new_cache(-(-L // P), P, 2, D, gpu)
    k, v = (torch.randn(L, 2, D, device=gpu).half() for _ in range(2))
    kv4.append(cache, None, k, v, torch.arange(L, device=gpu))
    q = torch.randn(1, 8, D, device=gpu).half()
    table = torch.arange(-(-L // P), dtype=torch.int32, device=gpu)[None]
    n = lambda x: torch.tensor([x], dtype=torch.int32, device=gpu)  # noqa: E731
    whole, lse = kv4.attention(cache, q, table, n(L), return_lse=True)
    cut = 20032
    a, la = kv4.attention(cache, q, table, n(cut), return_lse=True)
    b, lb = kv4.attention(cache, q, table[:, cut // P:].contiguous(), n(L - cut), return_lse=True)
    both = torch.logaddexp(la, lb)
    join = a.float() * (la - both).exp()[..., None] + b.float() * (lb - both).exp()[..., None]
    assert (both - lse).abs().max() < 1e-4
    # Three roundings to fp16 (2^-11) and two of the weights.
    assert (join - whole.float()).norm() <= 4 * 2 ** -11 * whole.float().norm()


def test_graph_replays_and_side_streams(gpu):
    """A step captured once and replayed on new contents, and one on a stream of its own."""
    D, P, H, Hq, B = 128, 64, 2, 8, 3
    table = torch.arange(B * 16, dtype=torch.int32, device=gpu).reshape(B, 16)
    lengths = torch.tensor([5, 700, 1000], dtype=torch.int32, device=gpu)
    cache = kv4.new_cache(B * 16, P, H, D, gpu)
    x = [torch.randn(B, h, D, device=gpu).half() for h in (Hq, H, H)]
    b = torch.arange(B, device=gpu)
    at = torch.zeros(B, dtype=torch.int64, device=gpu)

    def step():
        q = kv4.append(cache, *x, at)
        return kv4.attention(cache, q, table, lengths, max_length=1024)

    def fill():
        for t in x:
            t.normal_()
        lengths.add_(1)
        at.copy_(kv4.slots(table, b, lengths.long() - 1, P))

    fill()
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(on_side, step())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        fill()
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, step())


def test_python_refusals(gpu):
    cache = kv4.new_cache(2, 16, 2, 64, gpu)
    x = torch.zeros(3, 2, 64, dtype=torch.float16, device=gpu)
    at = torch.zeros(3, dtype=torch.int64, device=gpu)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    cos = torch.zeros(4, 16, device=gpu)

    def refuses(message, f, *args, **kw):
        with pytest.raises(RuntimeError, match=message):
            f(*args, **kw)

    refuses("u8 ", kv4.read, cache.float(), at)
    refuses("Expected contiguous CUDA tensor", kv4.read, cache[..., :40], at)
    refuses("slots must be contiguous int64", kv4.read, cache, at.int())
    refuses("Only FP16 and BF16", kv4.read, cache, at, torch.float32)
    refuses("Only FP16 and BF16", kv4.append, cache, x.float(), x.float(), x.float(), at)
    refuses("same dtype", kv4.append, cache, x.bfloat16(), x, x, at)
    refuses(r"v must be \[3, 2, 64\]", kv4.append, cache, x, x, x[:, :1], at)
    refuses("slots must be", kv4.append, cache, x, x, x, at[:2])
    refuses("same device", kv4.append, cache, x, x, x, at.cpu())
    refuses("elements of a head", kv4.append, cache, None, x.transpose(1, 2).contiguous().transpose(1, 2),
            x, at)
    refuses("go together", kv4.append, cache, x, x, x, at, cos=cos)
    refuses("multiple of 16", kv4.append, cache, x, x, x, at, at, cos[:, :5].contiguous(),
            cos[:, :5].contiguous())
    refuses("sin must be", kv4.append, cache, x, x, x, at, at, cos, cos[:2])
    refuses("positions must be", kv4.append, cache, x, x, x, at, at.int(), cos, cos)
    refuses("inference-only", kv4.append, cache, x.clone().requires_grad_(), x, x, at)
    refuses("inference-only", kv4.attention, cache, x.clone().requires_grad_(), i32(3, 1), i32(3))
    refuses("multiple of the cache's heads", kv4.attention, cache, x[:, :1], i32(3, 1), i32(3))
    refuses("tables must be", kv4.attention, cache, x, i32(3, 1).long(), i32(3))
    refuses("lengths must be", kv4.attention, cache, x, i32(3, 1), i32(2))
    refuses("one query", kv4.attention, cache, x, i32(2, 1), i32(2))
    refuses("one query", kv4.attention, cache, x, i32(3, 1), i32(3), max_q=2)
    refuses("starts must be", kv4.attention, cache, x, i32(2, 1), i32(2), i32(2))
    refuses("must not be negative", kv4.attention, cache, x, i32(3, 1), i32(3), window=-1)
    refuses("scale must be positive", kv4.attention, cache, x, i32(3, 1), i32(3), scale=0)

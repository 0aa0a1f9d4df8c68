"""What attention over the 4-bit cache does at its edges, in each of its forms, against
oracle/kv4.py in 64 bits.

The bound.  With weights that carry a relative error of at most d an output is off by at most
2 d sum p |v|.  d counts the rounding of a weight to the 11 bits of fp16 (once, 2^-11 in all,
since the sum is of unrounded weights) and the fp32 scores (2^-12 for sum |q k| scale < 32, as
these inputs have).  fp16's smallest numbers are 2^-24 apart and a part's largest weight times
scale is held at 2^7 or above, so that each token may add half of 2^-24 2^-7 of that weight
times scale for each of the up to 15 steps its value is from zero: L 15 2^-32.  Then the
output's own rounding (fp16: half of 2^-24 at least).  Tokens without weight enter nowhere.
"""
import numpy as np
import pytest
import torch

from dscquant_amd import kv4
from oracle import kv4 as oracle
from test_gpu_kv4 import DT, UNIT, f32, random_cache

pytestmark = pytest.mark.gpu

# Hq, H, sequences, queries of each, the host's bound on the length: what chooses the form.
FORMS = {
    "whole": (4, 2, 2, 3, 1000),
    "parts": (4, 2, 2, 3, 5000),
    "shares": (32, 32, 6, 3, 5000),
    "prompt, 4 waves": (8, 2, 2, 20, 1000),
    "prompt, 8 waves": (8, 2, 2, 40, 1000),
}
every_form = pytest.mark.parametrize("form", FORMS)


class Batch:
    """Sequences of random codes on pages of their own; ``k_words``, ``v_words`` [pages, H, P]
    are the words of the cache's rows, changed before the first use."""

    def __init__(self, form, dtype, D=128, P=16, L=300, seed=0):
        self.Hq, self.H, self.B, n, self.max_length = FORMS[form]
        self.dtype, self.D, self.P, self.counts = dtype, D, P, [n] * self.B
        self.rng = np.random.default_rng(seed)
        self.lengths = [L - 61 * (b % 3) for b in range(self.B)]
        self.per = -(-L // P)
        self.raw = random_cache(self.rng, self.B * self.per, self.H, P, D, 0.1)
        at = P * D
        flat = self.raw.reshape(self.B * self.per, self.H, -1)
        self.k_words = flat[..., at:at + 4 * P].view("<u4")
        self.v_words = flat[..., at + 4 * P:].view("<u4")
        self.tables = np.arange(self.B * self.per, dtype=np.int32).reshape(self.B, -1)
        T = sum(self.counts)
        g = torch.Generator().manual_seed(seed)
        self.q = torch.randn(T, self.Hq, D, generator=g).to(DT[dtype])

    def words(self, which, b, j):
        """The words [H] of sequence b's token j, as a view."""
        return (self.k_words, self.v_words)[which][b * self.per + j // self.P, :, j % self.P]

    def run(self, gpu, **options):
        i32 = lambda a: torch.tensor(np.asarray(a, np.int32), device=gpu)  # noqa: E731
        starts = np.concatenate(([0], np.cumsum(self.counts)))
        options = {"max_q": max(self.counts), "max_length": self.max_length, **options}
        out, lse = kv4.attention(torch.from_numpy(self.raw).to(gpu), self.q.to(gpu),
                                 i32(self.tables), i32(self.lengths), i32(starts),
                                 return_lse=True, **options)
        return f32(out), f32(lse)

    def expect(self, b, scale=None, window=0):
        """(out, lse, bound) of sequence b's queries."""
        k, v = (x[self.tables[b]].reshape(-1, self.H, self.D)[:self.lengths[b]].astype(np.float64)
                for x in oracle.values(self.raw))
        first, n, L = sum(self.counts[:b]), self.counts[b], self.lengths[b]
        q = f32(self.q[first:first + n]).astype(np.float64)
        scale = self.D ** -0.5 if scale is None else scale
        out, lse, spread = oracle.attention(q, k, v, np.arange(L - n, L), scale, window)
        f = self.v_words.view("<f4").astype(np.float64)[self.tables[b]].transpose(0, 2, 1)
        f = f.reshape(-1, self.H)[:L]
        G = self.Hq // self.H
        most = np.zeros((n, self.Hq, 1))
        for i in range(n):
            for h in range(self.Hq):
                end = L - n + i + 1
                seen = slice(max(end - window, 0) if window else 0, end)
                w = np.exp(scale * (k[seen, h // G] @ q[i, h]) - lse[i, h])
                most[i, h] = np.max(w * f[seen, h // G])
        bound = (UNIT[self.dtype] * np.abs(out) + spread * 2.0 ** -10 + L * 15 * 2.0 ** -32 * most
                 + (2.0 ** -25 if self.dtype == "fp16" else 0))
        return out, lse, bound

    def check(self, gpu, scale=None, **options):
        have, have_lse = self.run(gpu, scale=scale, **options)
        for b in range(self.B):
            first = sum(self.counts[:b])
            rows = slice(first, first + self.counts[b])
            out, lse, bound = self.expect(b, scale)
            # All zeros would not pass.
            assert (np.abs(out) > 2 * bound)[np.isfinite(out)].mean() > 0.5
            close(have[rows], out, bound)
            close(have_lse[rows], lse, 2.0 ** -12 + np.abs(lse) * 2.0 ** -22)


def close(have, want, bound):
    """Elements that are not finite are the same; the others within the bound."""
    finite = np.isfinite(want)
    assert np.array_equal(have[~finite], want[~finite], equal_nan=True)
    off = np.abs(have - want)[finite] - bound[finite]
    assert (off <= 0).all(), float(off.max())


# ------------------------------------------------------------------- tokens of scale 0

@every_form
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("what", ["key", "value", "both"])
def test_a_scale_of_zero_is_a_row_of_zeros(gpu, form, D, what):
    """Whatever the codes: a key of zeros scores 0, a value of zeros keeps its weight.  Words
    of less than fp32's smallest normal number are as good as 0."""
    x = Batch(form, "fp16", D)
    for b in range(x.B):
        for j, word in ((0, 0), (17, 0), (18, 0), (100, 5), (x.lengths[b] - 5, 0)):
            if what != "value":
                x.words(0, b, j)[:] = word
            if what != "key":
                x.words(1, b, j)[:] = word
    x.check(gpu)


@every_form
def test_all_values_zero(gpu, form):
    """The results are 0 and the log sums are the scores'."""
    x = Batch(form, "bf16")
    x.v_words[:] = 0
    out, lse = x.run(gpu)
    assert (out == 0).all()
    for b in range(x.B):
        first = sum(x.counts[:b])
        want = x.expect(b)[1]
        close(lse[first:first + x.counts[b]], want, 2.0 ** -12 + np.abs(want) * 2.0 ** -22)


@pytest.mark.parametrize("n", [1, 3, 12, 40])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_tokens_left_out_of_a_new_cache(gpu, n, dtype):
    """A token whose slot is outside the cache stays a place of zeros that its sequence counts."""
    L, D, P, Hq = 60, 64, 16, 4
    g = torch.Generator().manual_seed(n)
    q, k, v = (torch.randn(L, h, D, generator=g).to(DT[dtype]).to(gpu) for h in (Hq, 1, 1))
    cache = kv4.new_cache(4, P, 1, D, gpu)
    slots = torch.arange(L, device=gpu)
    for j in (7, 33, L - 2):
        slots[j] = -1
    kv4.append(cache, None, k, v, slots)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=gpu)  # noqa: E731
    out, lse = kv4.attention(cache, q[L - n:], i32([[0, 1, 2, 3]]), i32([L]), i32([0, n]), max_q=n,
                             max_length=L, return_lse=True)
    kk, vv = (x.reshape(-1, 1, D)[:L] for x in oracle.values(cache.cpu().numpy()))
    assert (kk[7] == 0).all() and (vv[33] == 0).all()
    want, sums, spread = oracle.attention(f32(q[L - n:]), kk, vv, np.arange(L - n, L), D ** -0.5)
    close(f32(out), want, UNIT[dtype] * np.abs(want) + spread * 2.0 ** -10 + 2.0 ** -25)
    close(f32(lse), sums, 2.0 ** -12 + np.abs(sums) * 2.0 ** -22)


# ------------------------------------------------------------------- rows that are not finite

@every_form
@pytest.mark.parametrize("which", ["key", "value"])
def test_a_row_that_is_not_finite_and_the_log_sum(gpu, form, which):
    """Who sees a NaN value has a NaN result and the log sum of its scores; who sees a NaN key
    has neither; who sees neither is not touched."""
    x = Batch(form, "fp16", 64)
    n = x.counts[0]
    for b in range(x.B):
        # One for the last query alone, in one head; in the second sequence for half of them.
        j = x.lengths[b] - (1 if b != 1 else n // 2 + 1)
        x.words(which == "value", b, j)[:1] = 0x7FC00000
    have, have_lse = x.run(gpu)
    for b in range(x.B):
        first = sum(x.counts[:b])
        out, lse, bound = x.expect(b)
        sees = np.isnan(out).all(-1)
        rows = 1 if b != 1 else n // 2 + 1
        assert sees.sum() == rows * x.Hq // x.H and np.isnan(out).any(-1).sum() == sees.sum()
        assert np.array_equal(np.isnan(lse), sees if which == "key" else np.zeros_like(sees))
        close(have[first:first + n], out, np.where(np.isnan(out), 0, bound))
        close(have_lse[first:first + n], lse, 2.0 ** -12 + np.abs(lse) * 2.0 ** -22)


@every_form
def test_a_value_that_is_not_finite_far_below_the_rest(gpu, form):
    """... is NaN to whoever sees it however small its weight, also as a part of its own."""
    x = Batch(form, "bf16", 64, L=420)
    x.q = x.q.abs()
    for b in range(x.B):
        for j in range(0, 260, x.P):  # whole pages of keys of -15 scale: scores some 200 below
            page = b * x.per + j // x.P
            x.raw.reshape(x.B * x.per, x.H, -1)[page, :, :x.P * x.D // 2] = 0
            x.k_words[page] |= 15
        x.words(1, b, 0)[:1] = 0x7FC00000
    have, have_lse = x.run(gpu, scale=2.0)
    for b in range(x.B):
        rows = slice(sum(x.counts[:b]), sum(x.counts[:b + 1]))
        out, lse, _ = x.expect(b, scale=2.0)
        assert np.isnan(out).any() and np.array_equal(np.isnan(have[rows]), np.isnan(out))
        assert (np.abs(have_lse[rows] - lse) <= 2.0 ** -6 + np.abs(lse) * 2.0 ** -22).all()


# ------------------------------------------------------------------- bounds and rows

@every_form
@pytest.mark.parametrize("window", [0, 40])
def test_queries_past_max_q_leave_the_others_in_their_places(gpu, form, window):
    x = Batch(form, "fp16", 64)
    n = x.counts[0]
    x.counts[1] = 1  # one that is not cut off
    x.q = x.q[:sum(x.counts)]
    for max_q in (n - 1, n - n // 8 - 1):
        have, have_lse = x.run(gpu, max_q=max_q, window=window)
        for b in range(x.B):
            first, m = sum(x.counts[:b]), min(x.counts[b], max_q)
            out, lse, bound = x.expect(b, window=window)
            close(have[first:first + m], out[:m], bound[:m])
            close(have_lse[first:first + m], lse[:m], 2.0 ** -12 + np.abs(lse[:m]) * 2.0 ** -22)


# ------------------------------------------------------------------- scales of values

@every_form
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("places", [16, 20, 24, 28, 40])
def test_a_large_value_without_weight_changes_nothing(gpu, form, dtype, places):
    """Values 2^places times the others' whose scores lie some 100 below (weights of 2^-140):
    the first tokens, ones in the middle, and one that the last query alone sees."""
    x = Batch(form, dtype, 64)
    x.q = x.q.abs()
    byte = oracle.places(x.P, x.D)[0][0]
    flat = x.raw.reshape(x.B * x.per, x.H, -1)
    for b in range(x.B):
        for j in (0, 1, 130, x.lengths[b] - 1):
            flat[b * x.per + j // x.P][:, byte[j % x.P]] = 0  # a key of -15
            x.words(0, b, j)[:] = np.float32(1).view(np.uint32) | 15
            x.words(1, b, j)[:] += np.uint32(places << 23)
    x.check(gpu)


@every_form
@pytest.mark.parametrize("D", [64, 128])
def test_values_of_all_sizes(gpu, form, D):
    """Scales from 2^-26 to 2^40, weights as they come."""
    x = Batch(form, "bf16", D)
    x.v_words += (x.rng.integers(-24, 42, x.v_words.shape) << 23).astype(np.uint32)
    x.check(gpu)


# ------------------------------------------------------------------- queries of all sizes

@every_form
@pytest.mark.parametrize("dtype,size", [("fp16", 1.0), ("bf16", 1.0), ("bf16", 2.0 ** 20)])
@pytest.mark.parametrize("factor", [2.0 ** 12, 2.0 ** 34, 2.0 ** 100, 2.0 ** -40, float("inf"),
                                    float("nan")])
def test_a_query_does_not_depend_on_the_others(gpu, form, dtype, size, factor):
    """One head of one query far larger or smaller than the rest, infinite or NaN: the other
    rows are what they are without it, bit for bit."""
    x = Batch(form, dtype, 64)
    x.q *= size
    scale = 0.125 / size
    plain, plain_lse = x.run(gpu, scale=scale)
    assert np.isfinite(plain).all()
    others = np.ones((x.q.shape[0], x.Hq), bool)
    n = x.counts[0]
    for row, head in ((0, x.Hq - 1), (n + n // 2, 0)):
        x.q[row, head] *= factor
        others[row, head] = False
    have, have_lse = x.run(gpu, scale=scale)
    assert np.array_equal(have[others], plain[others])
    assert np.array_equal(have_lse[others], plain_lse[others])
    if np.isnan(factor):
        assert np.isnan(have[~others]).all() and np.isnan(have_lse[~others]).all()
    if factor == 2.0 ** -40:  # scores of 0: the mean of what it sees
        for b, head in ((0, x.Hq - 1), (1, 0)):
            out, lse, bound = x.expect(b, scale)
            i = b * (n // 2)
            close(have[b * n + i, head], out[i, head], bound[i, head])
            close(have_lse[b * n + i, head], lse[i, head], np.array(2.0 ** -12 + 8 * 2.0 ** -22))


@every_form
@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -30, 2.0 ** 30, 2.0 ** 60])
def test_queries_of_one_size_and_a_scale_that_undoes_it(gpu, form, size):
    """bf16 queries of any size: each element counts with its eight bits."""
    x = Batch(form, "bf16", 128)
    x.q *= size
    x.check(gpu, scale=128 ** -0.5 / size)


@every_form
def test_elements_of_a_query_far_apart(gpu, form):
    """Elements 2^25 times the others that meet keys of zeros there: what is left counts in full."""
    x = Batch(form, "bf16", 64)
    byte, shift = oracle.places(x.P, x.D)[0]
    flat = x.raw.reshape(x.B * x.per, x.H, -1)
    d = 5
    for t in range(x.P):  # the code of element d is its zero-point
        zero = (x.k_words[..., t] & 15).astype(np.uint8)
        at, s = byte[t, d], int(shift[t, d])
        flat[..., at] = (flat[..., at] & np.uint8(255 ^ 15 << s)) | zero << np.uint8(s)
    x.q[..., d] *= 2.0 ** 25
    x.check(gpu)


# ------------------------------------------------------------------- rows of no sequence

@pytest.fixture
def dirty(monkeypatch):
    """Results are allocated with NaN in them."""
    empty = torch.Tensor.new_empty
    monkeypatch.setattr(torch.Tensor, "new_empty",
                        lambda *a, **k: empty(*a, **k).fill_(float("nan")))


@every_form
@pytest.mark.parametrize("before,after,cut", [(0, 3, 0), (2, 0, 0), (5, 700, 0), (0, 0, 1),
                                              (1, 2, 2)])
def test_rows_of_no_sequence_see_nothing(gpu, dirty, form, before, after, cut):
    """Rows before the first sequence's, after the last one's and past max_q: 0 and -inf."""
    x = Batch(form, "fp16", 64, L=140)
    n, T = x.counts[0], sum(x.counts)
    starts = before + np.arange(x.B + 1) * n
    i32 = lambda a: torch.tensor(np.asarray(a, np.int32), device=gpu)  # noqa: E731
    q = torch.cat((torch.full((before, x.Hq, 64), 7.0), x.q.float(),
                   torch.full((after, x.Hq, 64), float("nan")))).to(x.q.dtype)
    args = (torch.from_numpy(x.raw).to(gpu), q.to(gpu), i32(x.tables), i32(x.lengths), i32(starts))
    kw = dict(max_q=n - cut, max_length=x.max_length)
    out, lse = (f32(t) for t in kv4.attention(*args, return_lse=True, **kw))
    assert np.array_equal(f32(kv4.attention(*args, **kw)), out)
    row = np.arange(before + T + after) - before
    none = (row < 0) | (row >= T) | (row % n >= n - cut)
    assert (out[none] == 0).all() and (lse[none] == -np.inf).all()
    for b in range(x.B):
        want, sums, bound = x.expect(b)
        m = n - cut
        close(out[starts[b]:starts[b] + m], want[:m], bound[:m])
        close(lse[starts[b]:starts[b] + m], sums[:m], 2.0 ** -12 + np.abs(sums[:m]) * 2.0 ** -22)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_rows_without_sequences_or_queries(gpu, dirty, dtype):
    cache = kv4.new_cache(2, 16, 2, 64, gpu)
    q = torch.full((300, 6, 64), float("nan"), device=gpu).to(DT[dtype])
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
    for B, max_q in ((0, 5), (2, 0), (0, 0), (2, 5), (2, 70)):
        out, lse = kv4.attention(cache, q, i32(B, 1), i32(B), i32(B + 1), max_q=max_q,
                                 return_lse=True)
        assert (out == 0).all() and (lse == -float("inf")).all(), (B, max_q)
        assert (kv4.attention(cache, q, i32(B, 1), i32(B), i32(B + 1), max_q=max_q) == 0).all()


def test_rows_of_no_sequence_in_many_short_ones(gpu, dirty):
    """A padded batch in equal shares: sequences of no tokens, of no queries, of more than max_q."""
    H, D, P = 64, 64, 16
    cache = torch.from_numpy(random_cache(np.random.default_rng(0), 8, H, P, D)).to(gpu)
    counts = [0, 2, 0, 5, 1, 0, 3, 0]
    lengths = [0, 3, 9, 16, 0, 0, 2, 16]
    starts = np.concatenate(([4], 4 + np.cumsum(counts)))
    T = int(starts[-1]) + 9
    i32 = lambda a: torch.tensor(np.asarray(a, np.int32), device=gpu)  # noqa: E731
    q = torch.randn(T, H, D, generator=torch.Generator().manual_seed(0)).half().to(gpu)
    out, lse = kv4.attention(cache, q, i32(np.arange(8)[:, None]), i32(lengths), i32(starts),
                             max_q=2, max_length=5000, return_lse=True)
    assert torch.isfinite(out).all()
    seen = np.zeros(T, bool)
    for b, n in enumerate(counts):
        for i in range(min(n, 2)):
            seen[starts[b] + i] = lengths[b] - n + i >= 0
    assert np.array_equal(np.isfinite(f32(lse)).all(-1), seen)
    assert (f32(out)[~seen] == 0).all() and (f32(lse)[~seen] == -np.inf).all()


# ------------------------------------------------------------------- more tokens than a launch

def test_append_of_more_tokens_than_a_launch_holds(gpu):
    """2^28 tokens of 128 elements and a few more (all of them one row in memory), of which those
    at the ends of launches are kept."""
    D, T = 128, (1 << 28) + 5
    x = torch.randn(3, 1, D, device=gpu).half()
    q, k, v = (x[i:i + 1].expand(T, 1, D) for i in range(3))
    kept = [0, 1, (1 << 27) - 1, 1 << 27, (1 << 28) - 16, (1 << 28) - 1, 1 << 28, T - 1]
    slots = torch.full((T,), -1, dtype=torch.int64, device=gpu)
    slots[torch.tensor(kept, device=gpu)] = torch.arange(len(kept), device=gpu) + 5
    cache, want = (kv4.new_cache(1, 16, 1, D, gpu) for _ in range(2))
    kv4.append(cache, None, k, v, slots)
    n = len(kept)
    kv4.append(want, None, k[:n], v[:n], torch.arange(n, device=gpu) + 5)
    assert torch.equal(cache, want) and want.any()


def test_read_of_more_tokens_than_a_launch_holds(gpu):
    D, T = 128, (1 << 28) + 5
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 160 << 30:
        pytest.skip("needs 160 GB of free device memory")
    cache = kv4.new_cache(1, 16, 1, D, gpu)
    x = torch.randn(16, 1, D, device=gpu).half()
    kv4.append(cache, None, x, x + 1, torch.arange(16, device=gpu))
    slots = (torch.arange(T, device=gpu) * 7) % 16
    want = kv4.read(cache, torch.arange(16, device=gpu))
    got = kv4.read(cache, slots)
    for a, b in zip(got, want):
        for first in (0, (1 << 27) - 50, (1 << 28) - 50, T - 50):
            assert torch.equal(a[first:first + 50], b[slots[first:first + 50]])
    del got, a
    torch.cuda.empty_cache()


@pytest.mark.parametrize("form", ["prompt, 4 waves", "prompt, 8 waves"])
def test_a_bound_on_the_queries_far_above_them(gpu, form):
    x = Batch(form, "fp16", 64, L=140)
    x.check(gpu, max_q=((1 << 31) - 1) // x.Hq)


@pytest.mark.parametrize("T,Hq,H,D,P,R,interleaved,rotate,dtype", [
    (9000, 7, 3, 128, 64, 128, False, True, "bf16"),   # groups of 4 heads
    (20000, 5, 5, 64, 16, 32, True, False, "fp16"),    # of 4, and of 2 read back
    (20000, 0, 6, 64, 16, 64, False, True, "fp16"),    # no queries: of 3, and of 2
    (33001, 2, 2, 128, 128, 0, False, True, "fp16"),   # all heads one after another
])
def test_append_and_read_of_prompts_are_bit_exact(gpu, T, Hq, H, D, P, R, interleaved, rotate,
                                                  dtype):
    """Enough tokens that a workgroup takes several heads one after another, from q to k to v."""
    g = torch.Generator().manual_seed(T + Hq)
    rows = torch.randn(T, Hq + 2 * H, D, generator=g)
    rows[..., 5] *= 30
    rows = rows.to(DT[dtype])
    q, k, v = rows[:, :Hq], rows[:, Hq:Hq + H], rows[:, Hq + H:]
    on = rows.to(gpu)
    pages = -(-T // P) + 1
    slots = np.random.default_rng(T).permutation(pages * P)[:T]
    slots[T // 3] = -1
    at = torch.from_numpy(slots).to(gpu)
    turned, options = lambda x: f32(x), {}  # noqa: E731
    if R:
        angle = torch.rand(500, R // 2, generator=g) * 6
        pos = torch.randint(0, 500, (T,), generator=g)
        c, s = angle.cos(), angle.sin()
        cn, sn = c[pos].numpy(), s[pos].numpy()
        turned = lambda x: oracle.turn(f32(x), cn, sn, interleaved)  # noqa: E731
        options = dict(positions=pos.to(gpu), cos=c.to(gpu), sin=s.to(gpu), interleaved=interleaved)
    cache = torch.full((pages, H, P, D + 8), 0xA5, dtype=torch.uint8, device=gpu)
    got = kv4.append(cache, on[:, :Hq] if Hq else None, on[:, Hq:Hq + H], on[:, Hq + H:], at,
                     rotate=rotate, **options)
    qn, kn, vn = turned(q), turned(k), f32(v)
    if rotate:
        qn, kn = oracle.hadamard(qn) * np.float32(1 / D), oracle.hadamard(kn)
    if Hq:
        assert np.array_equal(f32(got), f32(torch.from_numpy(qn).to(DT[dtype])))
    empty = np.full((pages, H, P, D + 8), 0xA5, np.uint8)
    kept = slots >= 0
    have = oracle.values(cache.cpu().numpy())
    back = kv4.read(cache, at, DT[dtype], rotate=rotate)
    for which, x in enumerate((kn, vn)):
        codes, words = oracle.quantize(x)
        stored = (codes.astype(np.float32) - (words & 15).astype(np.float32)[..., None]) \
            * words.view(np.float32)[..., None]
        want = oracle.values(empty)[which].reshape(pages * P, H, D)
        want[slots[kept]] = stored[kept]
        assert np.array_equal(have[which].reshape(pages * P, H, D), want)
        if rotate and which == 0:
            stored = oracle.hadamard(stored) * np.float32(1 / D)
        stored[~kept] = 0
        assert np.array_equal(f32(back[which]), f32(torch.from_numpy(stored).to(DT[dtype])))


@every_form
@pytest.mark.parametrize("D", [64, 128])
def test_the_least_scales(gpu, form, D):
    """Keys and values about the rule's least scale, 1e-8: results of 1e-7, which bf16 holds as
    it holds others."""
    x = Batch(form, "bf16", D)
    x.v_words -= np.uint32(24 << 23)
    x.k_words -= np.uint32(23 << 23)
    assert x.v_words.view("<f4").min() < 1e-8 and x.k_words.view("<f4").min() < 1e-8
    x.check(gpu, scale=2.0 ** 23 * D ** -0.5)
    x.check(gpu)  # scores of 0 or so


@every_form
@pytest.mark.parametrize("size", [2.0 ** -90, 2.0 ** 122])
def test_queries_at_the_ends_of_their_range(gpu, form, size):
    """A power of two that the scale undoes changes nothing, also beside a page that is not there."""
    x = Batch(form, "bf16", 128)
    x.tables = np.concatenate((x.tables[:, :1], np.full_like(x.tables[:, :1], -1), x.tables[:, 1:]), 1)
    x.lengths = [n + x.P for n in x.lengths]
    plain = x.run(gpu, scale=128 ** -0.5)
    x.q *= size
    have = x.run(gpu, scale=128 ** -0.5 / size)
    for a, b in zip(have, plain):
        assert np.isfinite(b).all() and np.array_equal(a, b)

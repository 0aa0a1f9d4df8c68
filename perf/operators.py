"""Timing cases of the 4-bit key/value cache: appending to it, reading it back, attending over it.

A case is a dict of plain values; ``kind`` names the operator:

  append   ``kv4.append``: the step's keys and values, rotated by position, quantized to
           4 bits and written into their pages, the queries rotated on the way; the
           tokens' stored values are read back with ``kv4.read``, so the updated cache
           is among the outputs;
  read     ``kv4.read``: cached tokens as 16-bit keys and values;
  attend   ``kv4.attention``: the queries of a ragged batch over their pages.

The cache is a byte tensor [pages, heads, P, D + 8] of pages of P tokens.  The P (D + 8)
bytes of one (page, head), one after another:

  keys     [P / 16][4][16][D / 32] 32-bit words: token 16 a + r, elements g D / 4 + 8 w to
           + 7 are word [a][g][r][w], the eight of them in its nibbles 0, 4, 1, 5, 2, 6, 3, 7
           (from the lowest);
  values   [P / 4][16][2][D / 64] words: token 4 a + 2 b + h, element d = c D / 16 + 4 m + j
           is nibble 4 h + j of word [a][c][b][m];
  words    [P] of the keys, then [P] of the values: a row's scale as an fp32 number whose
           last four bits are the row's zero-point.

A row x (D numbers in 32 bits) is stored as

  lo = min(x, 0), hi = max(x, 0), base = max((hi - lo) / 15, 1e-8) rounded up to a multiple
  of 16 last places, zero = round(-lo / base) in [0, 15], scale = base + zero last places,
  code = round(x / scale + zero) in [0, 15], and stands for (code - zero) * scale.

With ``rotate`` the keys are multiplied with the Sylvester Hadamard matrix H_D before they
are quantized (unnormalised, as the activations' rotation is), and the queries with H_D / D,
so that the scores are the same; reading back undoes it.
"""
import functools
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
PAGE = 64


# ------------------------------------------------------------------ the cases

def _append(T, Hq, Hkv, D, dtype, rotate=False, rotary=None, interleaved=False, skip=False,
            page=PAGE):
    return {"kind": "append", "T": T, "Hq": Hq, "Hkv": Hkv, "D": D, "dtype": dtype,
            "rotate": rotate, "rotary": D if rotary is None else rotary,
            "interleaved": interleaved, "skip": skip, "page": page}


def _read(T, Hkv, D, dtype, rotate=False, page=PAGE):
    return {"kind": "read", "T": T, "Hkv": Hkv, "D": D, "dtype": dtype, "rotate": rotate,
            "page": page}


def _attend(B, lo, hi, queries, Hq, Hkv, D, dtype, window=0, lse=False, page=PAGE, spread=False):
    """``lo`` to ``hi`` cached tokens a sequence, ``queries`` of them new (with ``spread``: up
    to that many)."""
    return {"kind": "attend", "B": B, "lo": lo, "hi": hi, "queries": queries, "Hq": Hq, "Hkv": Hkv,
            "D": D, "dtype": dtype, "window": window, "lse": lse, "page": page, "spread": spread}


def listed():
    return [
        # One generated token of a 7B-shaped layer: the smallest call.
        dict(_append(1, 32, 32, 128, "fp16"), name="append_token"),
        # A prompt of 8192 tokens of a 70B-shaped layer, its keys rotated for 4 bits.
        dict(_append(8192, 64, 8, 128, "bf16", rotate=True), name="append_prompt"),
        # A ragged step of short heads: part of each head rotated by position in
        # neighbouring pairs, some tokens kept out of the cache.
        dict(_append(1777, 12, 4, 64, "fp16", rotary=32, interleaved=True, skip=True, page=16),
             name="append_ragged"),
        # A short shared prefix taken out of the cache.
        dict(_read(331, 32, 128, "fp16"), name="read_prefix"),
        # A long context taken out whole, for export or for another attention.
        dict(_read(16384, 8, 128, "bf16", rotate=True), name="read_context"),
        # One token of one sequence, a few hundred cached: latency.
        dict(_attend(1, 777, 777, 1, 32, 32, 128, "fp16"), name="decode_short"),
        # The decode step of 64 sequences of all lengths, 70B-shaped.
        dict(_attend(64, 1, 4096, 1, 64, 8, 128, "bf16"), name="decode_batch"),
        # One token of one long context.
        dict(_attend(1, 131072, 131072, 1, 64, 8, 128, "fp16", lse=True), name="decode_long"),
        # Five drafted tokens of each of eight sequences, verified at once.
        dict(_attend(8, 1000, 3000, 5, 64, 8, 128, "bf16"), name="verify_drafts"),
        # A prompt of 2048 tokens of a 7B-shaped layer.
        dict(_attend(1, 2048, 2048, 2048, 32, 32, 128, "fp16"), name="prompt"),
        # Prompts of odd lengths (an empty one among them) under a sliding window,
        # short heads, pages of 16 tokens.
        dict(_attend(7, 0, 1500, 1500, 12, 4, 64, "fp16", window=512, lse=True, page=16,
                     spread=True), name="prompts_ragged"),
        # The largest: 4096 new tokens after 12288 cached ones, 70B-shaped.
        dict(_attend(1, 16384, 16384, 4096, 64, 8, 128, "bf16"), name="prompt_chunk"),
    ]


def _size(rng, lo, hi):
    """A size spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "read", "attend", "attend", "attend"])
    Hq, Hkv = rng.choice([(32, 32), (64, 8), (32, 8), (12, 4), (14, 2), (8, 1), (5, 5)])
    D, dtype = rng.choice([128, 128, 64]), rng.choice(["fp16", "bf16"])
    page, rotate = rng.choice([16, 32, 64, 64, 128]), rng.random() < 0.5
    if kind == "append":
        return _append(_size(rng, 1, 8192), Hq, Hkv, D, dtype, rotate,
                       rotary=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.3,
                       skip=rng.random() < 0.3, page=page)
    if kind == "read":
        return _read(_size(rng, 1, 16384), Hkv, D, dtype, rotate, page)
    window, lse = rng.choice([0, 0, 0, 700]), rng.random() < 0.5
    form = rng.choice(["decode", "decode", "few", "prompt", "prompt"])
    if form == "decode":
        B = _size(rng, 1, 128)
        hi = _size(rng, 16, min(131072, 400000 // B))
        return _attend(B, rng.choice([1, hi]), hi, 1, Hq, Hkv, D, dtype, window, lse, page)
    if form == "few":
        B, n = _size(rng, 1, 32), rng.randint(2, 16)
        return _attend(B, n, _size(rng, n, 8192), n, Hq, Hkv, D, dtype, window, lse, page)
    B, n = rng.choice([1, 1, 2, 5]), _size(rng, 17, 2048)
    old = rng.choice([0, 0, _size(rng, 1, 4096)])
    return _attend(B, old if B > 1 else n + old, n + old, n, Hq, Hkv, D, dtype, window, lse, page,
                   spread=B > 1)


# ------------------------------------------------------------------ inputs

def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _gen(seed, n):
    return torch.Generator(device=_device()).manual_seed(1000 * seed + n)


def _heads(rows, heads, D, seed, n, outliers):
    """[rows, heads, D] numbers as a projection gives them; a few channels of the keys are
    far larger than the rest."""
    g = _gen(seed, n)
    x = torch.randn(rows, heads, D, generator=g, device=_device())
    top = torch.randperm(D, generator=g, device=_device())[:outliers]
    x[..., top] *= 8
    return x


def _angles(rows, rotary):
    """cos and sin [rows, rotary / 2] of the positions 0, 1, ..."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=_device()) / rotary)
    a = torch.arange(rows, dtype=torch.float64, device=_device())[:, None] * freq
    return a.cos().float(), a.sin().float()


def _queries(case):
    """The new tokens of each sequence; a batch's shape goes by the case alone."""
    B, n = case["B"], case["queries"]
    if not case["spread"]:
        return [n] * B
    some = torch.randint(0, n + 1, (B,), generator=torch.Generator().manual_seed(n)).tolist()
    return [0, *some[2:], n] if B > 1 else [n]


def _lengths(case, seed):
    """The cached tokens of each sequence, the new ones among them."""
    g = torch.Generator().manual_seed(1000 * seed + 7)
    queries, hi = _queries(case), case["hi"]
    some = torch.randint(case["lo"], hi + 1, (case["B"],), generator=g).tolist()
    return [max(n, L) for n, L in zip(queries, [case["lo"], *some[1:]][:case["B"] - 1] + [hi])]


def prepare(case, seed):
    dev, D, P, dtype = _device(), case["D"], case["page"], DTYPES[case["dtype"]]
    if case["kind"] == "attend":
        lengths, queries = _lengths(case, seed), _queries(case)
        per = [-(-n // P) for n in lengths]
        width, pages = max(1, *per), sum(per) + 3
        perm = torch.randperm(pages, generator=_gen(seed, 3), device=dev).to(torch.int32)
        tables = torch.zeros((case["B"], width), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(per):
            tables[b, :n] = perm[at:at + n]
            at += n
        cache = torch.empty((pages, case["Hkv"], P, D + 8), dtype=torch.uint8, device=dev)
        for first in range(0, pages, 512):  # in parts, so that their fp32 forms stay small
            part = cache[first:first + 512]
            rows = part.size(0) * P
            split = lambda x: x.reshape(-1, P, case["Hkv"], D).transpose(1, 2)  # noqa: E731
            part.copy_(_blocks(split(_heads(rows, case["Hkv"], D, seed + first, 4, D // 64)),
                               split(_heads(rows, case["Hkv"], D, seed + first, 5, 0))))
        starts = [0]
        for n in queries:
            starts.append(starts[-1] + n)
        q = _heads(starts[-1], case["Hq"], D, seed, 6, 0).to(dtype)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
        return {"case": case, "cache": cache, "q": q, "tables": tables, "lengths": i32(lengths),
                "starts": i32(starts), "max_q": max(queries), "max_length": max(lengths)}
    T, Hkv = case["T"], case["Hkv"]
    pages = -(-T // P) + 3
    cache = torch.zeros((pages, Hkv, P, D + 8), dtype=torch.uint8, device=dev)
    perm = torch.randperm(pages, generator=_gen(seed, 3), device=dev)
    where = torch.arange(T, device=dev)
    slots = perm[where // P] * P + where % P
    k = _heads(T, Hkv, D, seed, 4, D // 64)
    v = _heads(T, Hkv, D, seed, 5, 0)
    state = {"case": case, "cache": cache, "slots": slots, "dtype": dtype}
    if case["kind"] == "read":
        full = torch.zeros((2, pages * P, Hkv, D), device=dev)
        full[0, slots], full[1, slots] = k, v
        split = lambda x: x.reshape(pages, P, Hkv, D).transpose(1, 2)  # noqa: E731
        cache.copy_(_blocks(_hadamard(split(full[0])) if case["rotate"] else split(full[0]),
                            split(full[1])))
        return state
    if case["skip"]:
        slots[torch.rand(T, generator=_gen(seed, 8), device=dev) < 0.1] = -1
    # The three parts of one projection's rows, as a fused q|k|v product leaves them.
    q = _heads(T, case["Hq"], D, seed, 6, 0)
    rows = torch.cat([q, k, v], dim=1).to(dtype)
    cos, sin = _angles(T + 100, case["rotary"])
    return state | {"q": rows[:, :case["Hq"]], "k": rows[:, case["Hq"]:case["Hq"] + Hkv],
                    "v": rows[:, case["Hq"] + Hkv:], "cos": cos, "sin": sin,
                    "positions": where + 37}


# ------------------------------------------------------------------ the plain form

def _stage(x, h):
    """One butterfly stage of H_D: elements h apart become their sum and difference."""
    y = x.unflatten(-1, (-1, 2, h))
    a, b = y[..., 0, :], y[..., 1, :]
    return torch.stack((a + b, a - b), dim=-2).flatten(-3)


def _hadamard(x):
    return functools.reduce(_stage, [1 << i for i in range(x.shape[-1].bit_length() - 1)], x)


def _quantize(x):
    """(codes, words) of rows x [..., D]."""
    lo, hi = x.amin(-1).clamp(max=0), x.amax(-1).clamp(min=0)
    fifteen = torch.full_like(lo, 15.0)
    base = ((hi - lo) / fifteen).clamp(min=1e-8)
    bits = (base.view(torch.int32) + 15) & ~15
    zero = (-lo / bits.view(torch.float32)).round().clamp(0, 15)
    words = bits | zero.int()
    t = x / words.view(torch.float32)[..., None] + zero[..., None]
    return t.round().clamp(0, 15).int(), words


def _key_order(D, device):
    """The element at each nibble of a key row."""
    n = torch.arange(D, device=device)
    e = n % 8
    return n // 8 * 8 + torch.where(e < 4, 2 * e, 2 * e - 7)


def _join(nibbles):
    return (nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)).to(torch.uint8)


def _split(data):
    return torch.stack((data & 15, data >> 4), dim=-1).flatten(-2)


def _blocks(k, v):
    """Pages of the cache [N, H, P, D + 8] from keys and values [N, H, P, D]."""
    N, H, P, D = k.shape
    kc, kw = _quantize(k.contiguous())
    vc, vw = _quantize(v.contiguous())
    kb = _join(kc[..., _key_order(D, k.device)]).reshape(N, H, P // 16, 16, 4, D // 8)
    kb = kb.transpose(3, 4).reshape(N, H, -1)
    # [a][b][h][c][m][j] -> [a][c][b][m][h][j]
    vb = vc.reshape(N, H, P // 4, 2, 2, 16, D // 64, 4).permute(0, 1, 2, 5, 3, 6, 4, 7)
    vb = _join(vb.reshape(N, H, -1, 8)).reshape(N, H, -1)
    words = torch.cat((kw, vw), dim=-1).view(torch.uint8)
    return torch.cat((kb, vb, words), dim=-1).reshape(N, H, P, D + 8)


def _unblock(pages):
    """Keys and values [N, H, P, D] in 32 bits of the cache's pages [N, H, P, D + 8]."""
    N, H, P, D = pages.shape
    D = D - 8
    flat = pages.reshape(N, H, -1)
    kn = _split(flat[..., :P * D // 2]).reshape(N, H, P // 16, 4, 16, D // 4)
    kn = kn.transpose(3, 4).reshape(N, H, P, D)
    k = torch.empty_like(kn)
    k[..., _key_order(D, pages.device)] = kn
    vn = _split(flat[..., P * D // 2:P * D]).reshape(N, H, P // 4, 16, 2, D // 64, 2, 4)
    v = vn.permute(0, 1, 2, 4, 6, 3, 5, 7).reshape(N, H, P, D)
    words = flat[..., P * D:].contiguous().view(torch.int32).reshape(N, H, 2, P, 1)
    zero, scale = (words & 15).float(), words.view(torch.float32)
    return (k.float() - zero[:, :, 0]) * scale[:, :, 0], (v.float() - zero[:, :, 1]) * scale[:, :, 1]


def _turn(x, cos, sin, interleaved):
    """x [T, H, D] with its first 2 cos.shape[-1] elements turned by position."""
    half = cos.shape[-1]
    c, s = cos[:, None], sin[:, None]
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else \
        (x[..., :half], x[..., half:2 * half])
    y = (a * c - b * s, b * c + a * s)
    y = torch.stack(y, dim=-1).flatten(-2) if interleaved else torch.cat(y, dim=-1)
    return torch.cat((y, x[..., 2 * half:]), dim=-1)


def _plain_read(s):
    cache, slots, P = s["cache"], s["slots"], s["cache"].shape[2]
    k, v = _unblock(cache)
    at = slots.clamp(min=0)
    k, v = k[at // P, :, at % P], v[at // P, :, at % P]
    if s["case"]["rotate"]:
        k = _hadamard(k) * (1.0 / k.shape[-1])
    gone = (slots < 0)[:, None, None]
    return k.masked_fill(gone, 0).to(s["dtype"]), v.masked_fill(gone, 0).to(s["dtype"])


def _plain_append(s):
    case, cache, slots = s["case"], s["cache"], s["slots"]
    cos, sin = s["cos"][s["positions"]], s["sin"][s["positions"]]
    q = _turn(s["q"].float(), cos, sin, case["interleaved"])
    k = _turn(s["k"].float(), cos, sin, case["interleaved"])
    v = s["v"].float()
    if case["rotate"]:
        q, k = _hadamard(q) * (1.0 / q.shape[-1]), _hadamard(k)
    pages, H, P, D = cache.shape
    D = D - 8
    at = torch.nonzero(slots >= 0).flatten()
    # The tokens in a staging area of whole pages, and the bytes that are theirs in it.
    stage = torch.zeros((3, pages * P, H, D), device=k.device)
    stage[0, slots[at]], stage[1, slots[at]], stage[2, slots[at]] = k[at], v[at], 1.0
    split = stage.reshape(3, pages, P, H, D).transpose(2, 3)
    fresh = _blocks(split[0], split[1])
    mine = _blocks_mask(split[2])
    cache.copy_((fresh & mine) | (cache & ~mine))
    return q.to(s["dtype"]), *_plain_read(s)


def _blocks_mask(m):
    """The bytes of the pages that belong to the tokens whose m is not 0."""
    N, H, P, D = m.shape
    on = (m[..., 0] != 0).to(torch.uint8) * 255
    kb = on.reshape(N, H, P // 16, 1, 16, 1).expand(N, H, P // 16, 4, 16, D // 8)
    vb = on.reshape(N, H, P // 4, 1, 2, 1, 2, 1).expand(N, H, P // 4, 16, 2, D // 64, 2, 2)
    words = on[..., None].expand(N, H, P, 4).reshape(N, H, -1)
    parts = (kb.reshape(N, H, -1), vb.reshape(N, H, -1), words, words)
    return torch.cat(parts, dim=-1).reshape(N, H, P, D + 8)


def _plain_attend(s):
    case, q, starts, lengths = s["case"], s["q"], s["starts"], s["lengths"]
    B, Hq, Hkv, D, n, L = case["B"], case["Hq"], case["Hkv"], case["D"], s["max_q"], s["max_length"]
    G, dev = Hq // Hkv, q.device
    k, v = _unblock(s["cache"])
    P = k.shape[2]
    at = torch.arange(L, device=dev)
    page = s["tables"].long()[:, at // P]
    k, v = (x[page, :, at % P].transpose(1, 2) for x in (k, v))  # [B, Hkv, L, D]
    count = (starts[1:] - starts[:-1]).long()
    i = torch.arange(n, device=dev)
    row = (starts[:-1, None].long() + i).clamp(max=max(q.shape[0] - 1, 0))
    x = q.float()[row].reshape(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    t = torch.matmul(x, k.transpose(-1, -2).contiguous()).reshape(B, Hkv, G, n, L)
    place = (lengths.long() - count)[:, None] + i  # a query's place in its sequence
    seen = (at <= place[..., None]) & (at < lengths[:, None, None])
    if case["window"]:
        seen = seen & (at > place[..., None] - case["window"])
    seen = seen[:, None, None]
    t = (t * (1.0 / math.sqrt(D))).masked_fill_(~seen, -math.inf)
    top = t.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    t = (t - top).exp_()
    total = t.sum(-1, keepdim=True)
    out = torch.matmul(t.reshape(B, Hkv, G * n, L), v.contiguous()).reshape(B, Hkv, G, n, D)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log()).squeeze(-1)
    b, j = torch.nonzero(i < count[:, None], as_tuple=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D)[b, j].to(q.dtype)
    return [out, lse.permute(0, 3, 1, 2).reshape(B, n, Hq)[b, j]] if case["lse"] else [out]


# ------------------------------------------------------------------ one pass

def run(state):
    case = state["case"]
    if own:
        from dscquant_amd import kv4
        if case["kind"] == "attend":
            got = kv4.attention(state["cache"], state["q"], state["tables"], state["lengths"],
                                starts=None if case["queries"] == 1 and case["lo"] > 0
                                else state["starts"],
                                max_q=state["max_q"], max_length=state["max_length"],
                                window=case["window"], return_lse=case["lse"])
            return list(got) if case["lse"] else [got]
        if case["kind"] == "read":
            return list(kv4.read(state["cache"], state["slots"], state["dtype"],
                                 rotate=case["rotate"]))
        q = kv4.append(state["cache"], state["q"], state["k"], state["v"], state["slots"],
                       positions=state["positions"], cos=state["cos"], sin=state["sin"],
                       interleaved=case["interleaved"], rotate=case["rotate"])
        return [q, *kv4.read(state["cache"], state["slots"], state["dtype"],
                             rotate=case["rotate"])]
    if case["kind"] == "attend":
        return _plain_attend(state)
    return list(_plain_read(state) if case["kind"] == "read" else _plain_append(state))


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    D, Hkv = case["D"], case["Hkv"]
    if case["kind"] == "read":
        # Codes and words in, two 16-bit rows out; H_D is D log2(D) additions a row.
        T = case["T"]
        return {"bytes": T * (8 + Hkv * ((D + 8) + 4 * D)),
                "flops": T * Hkv * D * (4 + case["rotate"] * math.log2(D))}
    if case["kind"] == "append":
        # Rows of q, k and v in, q out, codes and words out, and what read takes and gives.
        T, Hq = case["T"], case["Hq"]
        rows = T * (Hq + Hkv)
        return {"bytes": T * (16 + 4 * case["rotary"]) + 4 * T * D * (Hq + Hkv)
                + T * Hkv * (2 * (D + 8) + 4 * D),
                "flops": rows * D * (3 + case["rotate"] * math.log2(D)) + 12 * T * Hkv * D}
    # The lengths are drawn; the figures are those of the middle one of each sequence.
    Hq, window = case["Hq"], case["window"] or math.inf
    pairs = kept = 0
    for n in _queries(case):
        length = max(n, (case["lo"] + case["hi"]) / 2)
        first = length - n  # a query sees min(window, its place + 1) tokens
        free = min(max(window - first, 0), n)  # the queries that see all before them
        pairs += free * first + free * (free + 1) / 2 + ((n - free) * window if free < n else 0)
        kept += min(length, window + n - 1) if n else 0
    rows = sum(_queries(case)) * Hq
    return {"bytes": Hkv * kept * (D + 8) + rows * (4 * D + 4 * case["lse"]),
            "flops": 4 * D * Hq * pairs}


# ------------------------------------------------------------------ in 64 bits

def _exact_values(cache):
    """Keys and values [pages, P, H, D] in 64 bits, a byte's two nibbles at a time."""
    N, H, P, E = cache.shape
    D, dev = E - 8, cache.device
    flat = cache.reshape(N, H, P * E)
    words = flat[..., P * D:].contiguous().view(torch.float32).double().reshape(N, H, 2, P)
    zeros = (flat[..., P * D::4] & 15).double().reshape(N, H, 2, P)
    k = torch.empty((N, P, H, D), dtype=torch.float64, device=dev)
    v = torch.empty_like(k)
    for d in range(D):
        t = torch.arange(P, device=dev)
        place = [0, 4, 1, 5, 2, 6, 3, 7][d % 8]
        word = ((t // 16 * 4 + d // (D // 4)) * 16 + t % 16) * (D // 32) + d % (D // 4) // 8
        at = word * 4 + place // 2
        code = (flat[..., at] >> (4 * (place % 2))) & 15
        k[..., d] = ((code - zeros[:, :, 0]) * words[:, :, 0]).transpose(1, 2)
        c, m, j = d // (D // 16), d % (D // 16) // 4, d % 4
        word = ((t // 4 * 16 + c) * 2 + t % 4 // 2) * (D // 64) + m
        nibble = t % 2 * 4 + j
        code = (flat[..., P * D // 2 + word * 4 + nibble // 2] >> (4 * (j % 2))) & 15
        v[..., d] = ((code - zeros[:, :, 1]) * words[:, :, 1]).transpose(1, 2)
    return k, v


def _exact_matrix(D, device):
    """H_D: the sign is the parity of the common bits."""
    i = torch.arange(D, device=device)
    both = i[:, None] & i
    odd = sum((both >> b) & 1 for b in range(7)) % 2
    return 1.0 - 2.0 * odd.double()


def _exact_stored(x):
    """What a row x stands for once it is stored, from the rule at the top in 64 bits."""
    lo, hi = x.min(-1).values.clamp(max=0), x.max(-1).values.clamp(min=0)
    base = ((hi - lo) / 15).clamp(min=1e-8)
    ulp = 2.0 ** (torch.floor(torch.log2(base)) - 23)
    base = torch.ceil(base / (16 * ulp)) * (16 * ulp)
    zero = torch.round(-lo / base).clamp(0, 15)
    scale = (base + zero * ulp)[..., None]
    return (torch.round(x / scale + zero[..., None]).clamp(0, 15) - zero[..., None]) * scale


def _exact_turn(x, positions, cos, sin, interleaved):
    half = cos.shape[1]
    a = torch.arange(half, device=x.device) * (2 if interleaved else 1)
    b = a + (1 if interleaved else half)
    c, s = cos.double()[positions][:, None], sin.double()[positions][:, None]
    y = x.clone()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., a] * s + x[..., b] * c
    return y


def exact(case, seed):
    s = prepare(case, seed)
    D, P, dev = case["D"], case["page"], s["cache"].device
    if case["kind"] == "append":
        H = _exact_matrix(D, dev)
        q, k = (_exact_turn(s[n].double(), s["positions"], s["cos"], s["sin"], case["interleaved"])
                for n in ("q", "k"))
        if case["rotate"]:
            q, k = q @ H / D, _exact_stored(k @ H) @ H / D
        else:
            k = _exact_stored(k)
        v = _exact_stored(s["v"].double())
        k[s["slots"] < 0] = 0
        v[s["slots"] < 0] = 0
        return [q, k, v]
    k, v = _exact_values(s["cache"])
    if case["kind"] == "read":
        k, v = (x.reshape(-1, *x.shape[2:])[s["slots"]] for x in (k, v))
        return [k @ _exact_matrix(D, dev) / D if case["rotate"] else k, v]
    Hq, Hkv = case["Hq"], case["Hkv"]
    outs, sums = [], []
    lengths, starts = s["lengths"].tolist(), s["starts"].tolist()
    for b in range(case["B"]):
        n, L = starts[b + 1] - starts[b], lengths[b]
        x = s["q"][starts[b]:starts[b + 1]].double()
        pages = s["tables"][b, :-(-L // P)].long()
        y = torch.zeros((n, Hq, D), dtype=torch.float64, device=dev)
        z = torch.full((n, Hq), -math.inf, dtype=torch.float64, device=dev)
        for h in range(Hq if n and L else 0):
            g = h // (Hq // Hkv)
            kh, vh = (a[pages, :, g].reshape(-1, D)[:L] for a in (k, v))
            place = torch.arange(L - n, L, device=dev)[:, None]
            j = torch.arange(L, device=dev)
            hidden = j > place
            if case["window"]:
                hidden = hidden | (j <= place - case["window"])
            t = (x[:, h] @ kh.T / math.sqrt(D)).masked_fill(hidden, -math.inf)
            z[:, h] = torch.logsumexp(t, dim=1)
            y[:, h] = torch.softmax(t, dim=1) @ vh
        outs.append(y)
        sums.append(z)
    return [torch.cat(outs), torch.cat(sums)] if case["lse"] else [torch.cat(outs)]

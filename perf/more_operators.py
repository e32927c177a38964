"""Attention over packed prompts and over a cache held in 4 bits, with their inputs, their least work and their plain forms.

A program that serves the language model takes prompts of different lengths behind one another in one batch (`swa_packed`), keeps their
keys and values in a ring of 4-bit codes (`KV4Cache.write`, `KV4Cache.read` gives them back) and from then on has one query a sequence,
each sequence at a position of its own, over that ring (`KV4Cache.attend`).  Query heads may share key heads; scores take the model's
window, ALiBi and soft-cap or do without.  `listed()` has each of them at the heads of the repository's configurations (12 of 64, 16 of
128, windows 512 and 1024), with grouped heads and long contexts, and at ragged sizes; `draw()` anywhere in between.

The cache's format: 32 values of a head's row share a scale 2^e, e the smallest whole number from -120 to 125 with amax <= 7 * 2^e; a
value is the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives times that, ties to the even code.  Position j of a sequence lives
in slot j % capacity."""
import functools
import math
import os
import random
import sys

import torch

own = False

BLOCK = 32                                         # values that share a scale
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)    # what the codes 0..7 stand for
DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # three short questions in one batch: latency
        dict(name="packed_short_3x12x64", kind="packed", rows=58, seqs=3, spread=1, heads=12, kv_heads=12, width=64, window=512, alibi=True, softcap=50.0,
             dtype="bf16"),
        # eight prompts of different lengths on the 768-wide model, its window and soft-cap
        dict(name="packed_prompts_8x12x64", kind="packed", rows=4096, seqs=8, spread=2, heads=12, kv_heads=12, width=64, window=512, alibi=True, softcap=50.0,
             dtype="bf16"),
        # long prompts on the 2048-wide model, its window and soft-cap, an odd number of rows
        dict(name="packed_prompts_4x16x128", kind="packed", rows=16383, seqs=4, spread=3, heads=16, kv_heads=16, width=128, window=1024, alibi=True,
             softcap=50.0, dtype="bf16"),
        # two long documents, the whole context, four query heads to a key head: the matrix products
        dict(name="packed_documents_2x16x128", kind="packed", rows=16384, seqs=2, spread=4, heads=16, kv_heads=4, width=128, window=None, alibi=False,
             softcap=0.0, dtype="bf16"),
        # the fp32 model, ragged, an odd window, two query heads to a key head
        dict(name="packed_ragged_fp32", kind="packed", rows=777, seqs=5, spread=5, heads=4, kv_heads=2, width=64, window=129, alibi=True, softcap=50.0,
             dtype="fp32"),
        # one interactive request on the 768-wide model: latency
        dict(name="attend_1x12x64", kind="attend", seqs=1, idle=0, spread=1, heads=12, kv_heads=12, width=64, capacity=513, longest=700, window=512, alibi=True,
             softcap=50.0, dtype="bf16"),
        # a full batch on the 2048-wide model, rings wrapped
        dict(name="attend_32x16x128", kind="attend", seqs=32, idle=0, spread=2, heads=16, kv_heads=16, width=128, capacity=1025, longest=4096, window=1024,
             alibi=True, softcap=50.0, dtype="bf16"),
        # long contexts with four query heads to a key head: the cache's bytes
        dict(name="attend_long_16x32x128", kind="attend", seqs=16, idle=0, spread=3, heads=32, kv_heads=8, width=128, capacity=32768, longest=32768, window=None,
             alibi=False, softcap=0.0, dtype="bf16"),
        # fp32 queries, no size a multiple of anything, a row of the batch that is not in use
        dict(name="attend_ragged_fp32", kind="attend", seqs=5, idle=1, spread=4, heads=6, kv_heads=2, width=64, capacity=1001, longest=3000, window=777, alibi=True,
             softcap=50.0, dtype="fp32"),
        # a decode step's new keys and values: latency
        dict(name="keep_step_8x12x64", kind="keep", rows=8, seqs=8, spread=1, kv_heads=12, width=64, capacity=513, dtype="bf16"),
        # the keys and values of long prompts on the 2048-wide model
        dict(name="keep_prompts_16384x16x128", kind="keep", rows=16384, seqs=6, spread=2, kv_heads=16, width=128, capacity=8192, dtype="bf16"),
        # fp32, prompts longer than the ring, which keeps their ends
        dict(name="keep_ragged_fp32", kind="keep", rows=2777, seqs=7, spread=3, kv_heads=3, width=64, capacity=333, dtype="fp32"),
    ]


def _between(rng, lo, hi):
    """A whole number of lo..hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    """One more case of the same kinds: one token to long documents, few and many heads, any window or none."""
    kind = rng.choice(["packed", "packed", "attend", "attend", "keep"])
    width = rng.choice([32, 64, 64, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    spread = rng.randrange(1 << 20)
    scores = dict(alibi=rng.choice([True, False]), softcap=rng.choice([0.0, 30.0, 50.0]))
    if kind == "packed":
        case = dict(kind=kind, rows=_between(rng, 1, 16384 if dtype == "bf16" else 4096), seqs=_between(rng, 1, 64), spread=spread, heads=kv_heads * group,
                    kv_heads=kv_heads, width=width, window=rng.choice([None, _between(rng, 16, 4096)]), dtype=dtype, **scores)
        most = work(listed()[3])["flops"] / (16 if dtype == "fp32" else 1)
        while work(case)["flops"] > most:
            case["rows"] = case["rows"] * 2 // 3
        return case
    seqs = _between(rng, 1, 64)
    capacity = _between(rng, 1, 65536)
    most = 16 * 8 * 32768 * 128
    capacity = max(1, min(capacity, most // (seqs * kv_heads * width)))
    if kind == "attend":
        window = rng.choice([None, _between(rng, 1, capacity) - 1])
        return dict(kind=kind, seqs=seqs, idle=rng.choice([0, 0, seqs // 4]), spread=spread, heads=kv_heads * group, kv_heads=kv_heads, width=width,
                    capacity=capacity, longest=_between(rng, 1, 2 * capacity), window=window, dtype=dtype, **scores)
    if rng.choice([True, False]):
        rows = seqs
    else:
        rows = min(_between(rng, 1, 16384), 16384 * 2048 // (kv_heads * width))
    return dict(kind=kind, rows=rows, seqs=seqs, spread=spread, kv_heads=kv_heads, width=width, capacity=capacity, dtype=dtype)


# ---------------------------------------------------------------- lengths and positions, by the case alone
@functools.lru_cache(maxsize=None)
def _lengths(rows, seqs, spread):
    """`rows` tokens dealt to sequences: some short, some long, a token each where there are as many tokens as sequences."""
    if rows == seqs:
        return (1,) * seqs
    rng = random.Random(spread * 1000003 + rows * 101 + seqs)
    share = [math.exp(rng.gauss(0.0, 0.6)) for _ in range(seqs)]
    ends = [round(rows * sum(share[:i + 1]) / sum(share)) for i in range(seqs)]
    ends[-1] = rows
    return tuple(b - a for a, b in zip([0] + ends[:-1], ends))


@functools.lru_cache(maxsize=None)
def _positions(seqs, idle, longest, spread):
    """The position of each sequence's query: half the longest and more, one of them the longest, the idle ones at -1."""
    rng = random.Random(spread * 1000003 + seqs)
    at = [longest - 1] + [rng.randrange(longest // 2, longest) for _ in range(seqs - 1)]
    rng.shuffle(at)
    for i in rng.sample(range(seqs), idle):
        at[i] = -1
    return tuple(at)


def _starts(case):
    """Where the sequences of a kept batch begin: anywhere in the ring's first rounds."""
    rng = random.Random(case["spread"] * 7 + case["seqs"])
    return tuple(rng.randrange(2 * case["capacity"]) for _ in range(case["seqs"]))


def _slopes(heads):
    """ALiBi's slopes as the model has them."""
    def powers(n):
        first = 2.0 ** (-(2.0 ** -(math.log2(n) - 3)))
        return [first ** (i + 1) for i in range(n)]
    near = 2 ** int(math.log2(heads))
    s = powers(near) + powers(2 * near)[0::2][:heads - near]
    return torch.tensor(s, dtype=torch.float32) * 0.25


# ---------------------------------------------------------------- the plain forms
def _codes(v):
    """Codes, two to a byte, and scales' bytes of v (..., width) fp32, 32 values to a scale."""
    b = v.unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(b.abs().amax(-1))
    e = torch.where(m <= 0.875, e - 3, e - 2).clamp(-120, 125)
    a = b * ((127 - e) << 23).view(torch.float32)[..., None]
    size = a.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp_max(6.0)
    code = torch.bucketize(size, torch.tensor(GRID, device=v.device)).to(torch.uint8) + 8 * torch.signbit(a).to(torch.uint8)
    code = code.flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], (e + 127).to(torch.uint8)


def _values(codes, scales):
    """What codes and scales stand for, in fp32."""
    table = torch.tensor(GRID + tuple(-g for g in GRID), device=codes.device)
    v = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).flatten(-2)
    s = (scales.int() << 23).view(torch.float32)
    return (v.unflatten(-1, (-1, BLOCK)) * s[..., None]).flatten(-2)


def _weights(s, far, visible, slopes, softcap):
    """softmax over the last axis of scores s (..., heads of a key head, queries, keys); rows that see nothing are zero."""
    if softcap:
        s = softcap * torch.tanh(s / softcap)
    if slopes is not None:
        s = s - slopes * far
    s = torch.where(visible, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(top), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, 1.0)


def _plain_packed(state):
    case = state["case"]
    heads, kv, width, window = case["heads"], case["kv_heads"], case["width"], case["window"]
    group, out = heads // kv, state["out"]
    slopes = None if state["slopes"] is None else state["slopes"].view(kv, group, 1, 1)
    start = 0
    for n in state["lengths"]:
        if n == 0:
            continue
        k = state["k"][start:start + n].float().transpose(0, 1)            # (kv, n, width)
        v = state["v"][start:start + n].float().transpose(0, 1)
        for a in range(0, n, 1024):
            b = min(n, a + 1024)
            first = 0 if window is None else max(0, a - window)
            q = state["q"][start + a:start + b].float().view(b - a, kv, group, width).permute(1, 2, 0, 3)
            s = (q.reshape(kv, -1, width) @ k[:, first:b].transpose(1, 2)).view(kv, group, b - a, b - first) * width ** -0.5
            far = torch.arange(a, b, device=q.device)[:, None] - torch.arange(first, b, device=q.device)
            seen = (far >= 0) if window is None else (far >= 0) & (far <= window)
            p = _weights(s, far, seen, slopes, case["softcap"])
            o = (p.view(kv, -1, b - first) @ v[:, first:b]).view(kv, group, b - a, width)
            out[start + a:start + b] = o.permute(2, 0, 1, 3).reshape(b - a, heads, width).to(out.dtype)
        start += n
    return dict(o=out)


def _plain_attend(state):
    case = state["case"]
    seqs, heads, kv, width, capacity = case["seqs"], case["heads"], case["kv_heads"], case["width"], case["capacity"]
    pos = state["pos"].long()
    slot = torch.arange(capacity, device=pos.device)
    far = (pos[:, None] - slot) % capacity                                 # how far behind the query a slot's position is
    window = capacity - 1 if case["window"] is None else case["window"]
    seen = (far <= window) & (far <= pos[:, None])
    q = state["q"].float().view(seqs, kv, heads // kv, width)
    slopes = None if state["slopes"] is None else state["slopes"].view(kv, -1, 1)
    s = (q @ _values(*state["k"]).transpose(2, 3)) * width ** -0.5
    p = _weights(s, far[:, None, None], seen[:, None, None], slopes, case["softcap"])
    o = p @ _values(*state["v"])
    return dict(o=o.view(seqs, heads, width).to(DTYPES[case["dtype"]]))


def _plain_keep(state):
    seq, slot = state["at"]
    kept, back = state["kept"], {}
    for name in ("k", "v"):
        codes, scales = _codes(state[name][kept].float())
        ring_codes, ring_scales = state["ring"][name]
        ring_codes[seq, slot], ring_scales[seq, slot] = codes, scales
        back[name] = _values(ring_codes[seq, slot], ring_scales[seq, slot]).to(state[name].dtype)
    return back


# ---------------------------------------------------------------- the framework's
@functools.lru_cache(maxsize=None)
def _package():
    sys.path.insert(0, os.path.join(os.getcwd(), "flash-stu-2_amd"))
    import flash_stu
    return flash_stu


def _own_packed(state):
    case = state["case"]
    return dict(o=_package().swa_packed(state["q"], state["k"], state["v"], state["cu"], slopes=state["slopes"], window=case["window"],
                                        softcap=case["softcap"], out=state["out"]))


def _own_attend(state):
    case = state["case"]
    return dict(o=state["cache"].attend(state["q"], state["pos"], slopes=state["slopes"], window=case["window"], softcap=case["softcap"]))


def _own_keep(state):
    cache = state["cache"]
    cache.write(state["k"], state["v"], state["pos"], state["cu"])
    k, v = cache.read(state["kept_pos"], state["kept_cu"], rows=state["kept_rows"], dtype=state["k"].dtype)
    return dict(k=k, v=v)


# ---------------------------------------------------------------- what a program has in hand before the call
def _rows(gen, rows, heads, width, dtype):
    """Projected rows: a few channels of each head stand out."""
    x = torch.randn(rows, heads, width, generator=gen, device="cuda")
    x *= torch.exp(0.5 * torch.randn(1, heads, width, generator=gen, device="cuda"))
    return x.to(dtype)


def _bounds(lengths):
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _cache_values(case, gen):
    """Keys and values by slot, (seqs, capacity, kv_heads, width); slots that no query sees hold something too."""
    n = case["seqs"] * case["capacity"]
    return [_rows(gen, n, case["kv_heads"], case["width"], DTYPES[case["dtype"]]).view(case["seqs"], case["capacity"], case["kv_heads"], case["width"])
            for _ in range(2)]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    kind, t, seqs, kv, width = case["kind"], DTYPES[case["dtype"]], case["seqs"], case["kv_heads"], case["width"]
    state = dict(case=case)
    if kind != "keep":
        state["slopes"] = _slopes(case["heads"]).cuda() if case["alibi"] else None
    if kind == "packed":
        # one fused projection, as the layer makes it: queries, keys and values are parts of its rows
        rows, heads = case["rows"], case["heads"]
        fused = _rows(gen, rows, heads + 2 * kv, width, t)
        state["q"], state["k"], state["v"] = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
        state["lengths"] = _lengths(rows, seqs, case["spread"])
        state["cu"] = _bounds(state["lengths"])
        state["out"] = torch.zeros(rows, heads, width, dtype=t, device="cuda")
        return state
    capacity = case["capacity"]
    if kind == "attend":
        state["q"] = _rows(gen, seqs, case["heads"], width, t)
        state["pos"] = torch.tensor(_positions(seqs, case["idle"], case["longest"], case["spread"]), dtype=torch.int32, device="cuda")
        k, v = _cache_values(case, gen)
        if own:
            state["cache"] = _package().KV4Cache(seqs, kv, width, capacity, device="cuda")
            full = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * capacity
            state["cache"].write(k.flatten(0, 1), v.flatten(0, 1), torch.zeros(seqs, dtype=torch.int32, device="cuda"), full)
        else:
            for name, x in (("k", k), ("v", v)):
                codes, scales = zip(*(_codes(x[i].transpose(0, 1).float()) for i in range(seqs)))
                state[name] = torch.stack(codes), torch.stack(scales)
        return state
    state["k"], state["v"] = (_rows(gen, case["rows"], kv, width, t) for _ in range(2))
    lengths, starts = _lengths(case["rows"], seqs, case["spread"]), _starts(case)
    state["pos"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    single = case["rows"] == seqs
    state["cu"] = None if single else _bounds(lengths)
    held = [min(n, capacity) for n in lengths]
    state["kept_pos"] = torch.tensor([s + n - h for s, n, h in zip(starts, lengths, held)], dtype=torch.int32, device="cuda")
    state["kept_cu"], state["kept_rows"] = None if single else _bounds(held), sum(held)
    if own:
        state["cache"] = _package().KV4Cache(seqs, kv, width, capacity, device="cuda")
        return state
    row, seq, slot, first = [], [], [], 0
    for i, (s, n, h) in enumerate(zip(starts, lengths, held)):
        row += range(first + n - h, first + n)
        seq += [i] * h
        slot += [j % capacity for j in range(s + n - h, s + n)]
        first += n
    state["kept"] = torch.tensor(row, device="cuda")
    state["at"] = torch.tensor(seq, device="cuda"), torch.tensor(slot, device="cuda")
    state["ring"] = {name: (torch.zeros(seqs, capacity, kv, width // 2, dtype=torch.uint8, device="cuda"),
                            torch.zeros(seqs, capacity, kv, width // BLOCK, dtype=torch.uint8, device="cuda")) for name in ("k", "v")}
    return state


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"packed": _own_packed, "attend": _own_attend, "keep": _own_keep}[kind](state)
    return {"packed": _plain_packed, "attend": _plain_attend, "keep": _plain_keep}[kind](state)


# ---------------------------------------------------------------- the definition in 64 bits
def _exact_kept(x):
    """What the cache holds of x (..., width), in 64 bits."""
    v = x.double()
    shape = v.shape
    v = v.reshape(*shape[:-1], shape[-1] // BLOCK, BLOCK)
    most = v.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(most.clamp_min(2.0 ** -200) / 7.0))
    e = torch.where(7.0 * torch.exp2(e - 1.0) >= most, e - 1.0, e)
    e = torch.where(7.0 * torch.exp2(e) < most, e + 1.0, e).clamp(-120.0, 125.0)
    a = v / torch.exp2(e)
    size, held = a.abs(), torch.zeros_like(a)
    for below, above in zip(GRID[:-1], GRID[1:]):        # past the middle to the next one; on it where that one's code is even
        mid = (below + above) / 2
        held = torch.where((size >= mid) if GRID.index(above) % 2 == 0 else (size > mid), above, held)
    return (torch.sign(a) * held * torch.exp2(e)).reshape(shape)


def _exact_scores(s, far, slopes, softcap):
    if softcap:
        s = torch.tanh(s / softcap) * softcap
    return s if slopes is None else s - slopes.double() * far.double()


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "keep":
        lengths, x, first, rows = _lengths(case["rows"], case["seqs"], case["spread"]), {}, 0, []
        for n in lengths:
            rows.append(torch.arange(first + max(0, n - case["capacity"]), first + n))
            first += n
        rows = torch.cat(rows).cuda()
        return {name: _exact_kept(state[name][rows]) for name in ("k", "v")}
    heads, kv, width = case["heads"], case["kv_heads"], case["width"]
    group, root = heads // kv, math.sqrt(width)
    if kind == "attend":
        gen = torch.Generator(device="cuda").manual_seed(int(seed))
        _rows(gen, case["seqs"], heads, width, DTYPES[case["dtype"]])        # the queries come first
        keys, values = _cache_values(case, gen)
        window = case["capacity"] - 1 if case["window"] is None else case["window"]
        y = torch.zeros(case["seqs"], heads, width, dtype=torch.float64, device="cuda")
        for i, at in enumerate(_positions(case["seqs"], case["idle"], case["longest"], case["spread"])):
            if at < 0:
                continue
            j = torch.arange(max(0, at - window), at + 1, device="cuda")
            k, v = _exact_kept(keys[i][j % case["capacity"]]), _exact_kept(values[i][j % case["capacity"]])
            for h in range(heads):
                s = _exact_scores(k[:, h // group] @ state["q"][i, h].double() / root, at - j, None if state["slopes"] is None else state["slopes"][h],
                                  case["softcap"])
                y[i, h] = torch.softmax(s, 0) @ v[:, h // group]
        return dict(o=y)
    y = torch.zeros(case["rows"], heads, width, dtype=torch.float64, device="cuda")
    first = 0
    for n in _lengths(case["rows"], case["seqs"], case["spread"]):
        at = torch.arange(n, device="cuda")
        for h in range(heads):
            k, v = (state[x][first:first + n, h // group].double() for x in ("k", "v"))
            for i in at.split(2048) if n else ():
                lo = 0 if case["window"] is None else max(0, int(i[0]) - case["window"])
                j = at[lo:int(i[-1]) + 1]
                far = i[:, None] - j[None]
                s = _exact_scores(torch.mm(state["q"][first:first + n, h][i].double(), k[j].t()) / root, far,
                                  None if state["slopes"] is None else state["slopes"][h], case["softcap"])
                hidden = (far < 0) if case["window"] is None else (far < 0) | (far > case["window"])
                y[first + i, h] = torch.mm(torch.softmax(s.masked_fill(hidden, -math.inf), 1), v[j])
        first += n
    return dict(o=y)


# ---------------------------------------------------------------- the least it takes
def _pairs(n, window):
    """Keys that the queries 0..n-1 see, all together."""
    if window is None or window >= n:
        return n * (n + 1) // 2
    return (window + 1) * n - window * (window + 1) // 2


def work(case):
    kind, kv, width, t = case["kind"], case["kv_heads"], case["width"], 4 if case["dtype"] == "fp32" else 2
    held = width // 2 + width // BLOCK                     # bytes of a head's row in the cache
    if kind == "keep":
        lengths = _lengths(case["rows"], case["seqs"], case["spread"])
        kept = sum(min(n, case["capacity"]) for n in lengths)
        # the ring's rows written and read again, their values read and written
        return {"bytes": 2 * kept * kv * 2 * (width * t + held), "flops": 2.0 * kept * kv * width * 4}
    heads = case["heads"]
    if kind == "attend":
        window = case["capacity"] - 1 if case["window"] is None else case["window"]
        seen = sum(min(window, at) + 1 for at in _positions(case["seqs"], case["idle"], case["longest"], case["spread"]))
        return {"bytes": seen * kv * 2 * held + 2 * case["seqs"] * heads * width * t, "flops": 4.0 * seen * heads * width}
    pairs = sum(_pairs(n, case["window"]) for n in _lengths(case["rows"], case["seqs"], case["spread"]))
    return {"bytes": case["rows"] * width * t * 2 * (heads + kv), "flops": 4.0 * pairs * heads * width}

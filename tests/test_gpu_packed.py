"""Attention over packed prompts against its definition in 64 bits.  In bf16 the probabilities go into the second product as bf16 values (p_step 2^-8, half
a step); in fp32 they are not cut."""
import math

import pytest
import torch

from attention_reference import Ring, check, held, packed

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
P_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -23}


@pytest.fixture(scope="module")
def fs():
    import flash_stu
    from flash_stu import _hip
    _hip.load()
    return flash_stu


def rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(1, *shape[1:], generator=g))
    return x.to(dtype)


def bounds(lengths, begin=0):
    total = [begin]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def slopes_of(heads):
    return 0.25 * 2.0 ** (-8.0 * (torch.arange(heads) + 1) / heads)


def fused(seed, rows, heads, kvh, hd, dtype):
    x = rand(seed, rows, heads + 2 * kvh, hd, dtype=dtype)
    return [(t[:, :heads], t[:, heads:heads + kvh], t[:, heads + kvh:]) for t in (x, x.cuda())]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,hd,lengths,window,softcap,alibi", [
    (12, 12, 64, [17, 1, 40], 512, 50.0, True),
    (2, 2, 64, [1], None, 0.0, False),
    (1, 1, 128, [0, 2, 0, 0, 3, 0], None, 0.0, True),
    (4, 2, 64, [129, 63, 64, 65, 128], 31, 50.0, True),
    (4, 1, 128, [300, 33, 127], None, 0.0, False),
    (6, 2, 32, [100, 257, 5], 0, 0.0, True),
    (3, 1, 32, [200, 31], None, 30.0, False),
    (2, 1, 256, [150, 70, 1], 100, 0.0, True),
    (5, 5, 256, [33, 64], None, 50.0, False),
    (8, 8, 128, [1] * 40 + [90], 16, 0.0, True),
    (2, 2, 128, [515, 260], 200, 50.0, True),
    (16, 2, 64, [190, 191, 192], None, 0.0, True),
])
def test_packed(fs, heads, kvh, hd, lengths, window, softcap, alibi, dtype):
    rows = sum(lengths)
    (q, k, v), dev = fused(7, rows, heads, kvh, hd, dtype)
    slopes = slopes_of(heads) if alibi else None
    y = fs.swa_packed(*dev, bounds(lengths), slopes=None if slopes is None else slopes.cuda(), window=window, softcap=softcap)
    assert y.shape == q.shape and y.dtype is dtype and y.is_contiguous()
    check(y, *packed(q, k, v, lengths, slopes, window, softcap, P_STEP[dtype]), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,hd,lengths,window,softcap,alibi", [
    (32, 1, 64, [1, 4200, 0, 130, 64, 17], 70, 0.0, True),
    (32, 4, 32, [33, 2] * 35 + [80], 50, 50.0, True),
    (32, 2, 128, [700, 1500, 90], None, 50.0, True),
    (32, 32, 128, [0, 900, 1100, 0], None, 0.0, False),
    (64, 8, 256, [520, 300, 1], 200, 0.0, True),
    (64, 64, 64, [65] * 64, None, 0.0, True),
    (128, 16, 32, [33, 2] * 35 + [80], 50, 50.0, True),
    (128, 16, 32, [700, 130], None, 0.0, False),
    (48, 3, 128, [700, 1500, 90], None, 50.0, True),
    (64, 64, 128, [0, 900, 1100, 0], 333, 0.0, True),
    (64, 8, 128, [1300, 33], None, 0.0, False),
    (64, 8, 64, [1700, 33], 1000, 30.0, False),
])
def test_more_workgroups_than_the_card_holds(fs, heads, kvh, hd, lengths, window, softcap, alibi, dtype):
    (q, k, v), dev = fused(17, sum(lengths), heads, kvh, hd, dtype)
    slopes = slopes_of(heads) * 4
    y = fs.swa_packed(*dev, bounds(lengths), slopes=slopes.cuda() if alibi else None, window=window, softcap=softcap)
    h = torch.tensor([0, 1, heads // 2 + 3, heads - 1])
    kv = h // (heads // kvh)
    check(y.cpu()[:, h], *packed(q[:, h], k[:, kv], v[:, kv], lengths, slopes[h] if alibi else None, window, softcap, P_STEP[dtype]), dtype)
    assert bool(torch.isfinite(y).all())


@pytest.mark.parametrize("lengths,window,softcap,alibi", [
    ([4500], None, 0.0, False),
    ([4500], None, 50.0, False),
    ([4131], 4100, 0.0, True),
    ([8190, 33], 4096, 50.0, True),
])
def test_documents_of_many_thousands(fs, lengths, window, softcap, alibi):
    (q, k, v), dev = fused(23, sum(lengths), 2, 1, 128, torch.bfloat16)
    y = fs.swa_packed(*dev, bounds(lengths), slopes=slopes_of(2).cuda() if alibi else None, window=window, softcap=softcap)
    one = slice(1, 2)
    check(y[:, one], *packed(q[:, one], k, v, lengths, slopes_of(2)[one] if alibi else None, window, softcap, P_STEP[torch.bfloat16]), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_one_long_document(fs, hd, dtype):
    (q, k, v), dev = fused(3, 2100, 2, 1, hd, dtype)
    y = fs.swa_packed(*dev, bounds([2100]))
    check(y, *packed(q, k, v, [2100], None, None, 0.0, P_STEP[dtype]), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [None, 20])
def test_what_a_row_does_not_see_may_be_anything(fs, hd, window, dtype):
    """NaN and infinities in keys and values of other sequences, of later rows and of rows beyond the window leave a row as it is."""
    lengths, heads = [70, 90, 45], 2
    rows = sum(lengths)
    q, k, v = (rand(i, rows, heads, hd, dtype=dtype) for i in range(3))
    bad = [5, 69, 70 + 30, 70 + 31, 70 + 89]
    dirty_k, dirty_v = k.clone(), v.clone()
    for n, r in enumerate(bad):
        dirty_k[r, n % 2], dirty_v[r, 1 - n % 2, n::7] = math.nan, (math.inf, -math.inf, math.nan)[n % 3]
    y = fs.swa_packed(q.cuda(), dirty_k.cuda(), dirty_v.cuda(), bounds(lengths), window=window).cpu()
    o, bound = packed(q, k, v, lengths, None, window, 0.0, P_STEP[dtype])
    start = [0] * 70 + [70] * 90 + [160] * 45
    clean = torch.tensor([not any(start[r] <= b <= r and (window is None or r - b <= window) for b in bad) for r in range(rows)])
    check(y[clean], o[clean], bound[clean], dtype)
    for n, r in enumerate(bad):                                          # the row itself sees it
        assert bool(torch.isnan(y[r, n % 2]).any()) and not bool(torch.isfinite(y[r, 1 - n % 2, n::7]).any())


@pytest.mark.parametrize("hd,heads,lengths,window,softcap,alibi", [
    (32, 128, [400, 500, 130], None, 0.0, True),
    (64, 128, [400, 500, 130], 90, 50.0, True),
    (64, 128, [400, 500, 130], None, 0.0, False),
    (128, 128, [400, 500, 130], 90, 0.0, True),
    (128, 128, [400, 500, 130], None, 50.0, False),
    (256, 32, [400, 500, 130], 90, 50.0, True),
    (128, 2, [4200], None, 0.0, True),
])
def test_what_a_row_does_not_see_may_be_anything_in_large_calls(fs, hd, heads, lengths, window, softcap, alibi):
    rows, dtype, slopes = sum(lengths), torch.bfloat16, slopes_of(heads)
    q, k, v = rand(0, rows, heads, hd, dtype=dtype), rand(1, rows, 2, hd, dtype=dtype), rand(2, rows, 2, hd, dtype=dtype)
    start = [sum(lengths[:i]) for i, n in enumerate(lengths) for _ in range(n)]
    bad = [r for r in (rows - 7, 300, 399, 520, 521, 899) if window or r > rows - 10 or start[r] + 350 < r]
    k[bad[0], 0], v[bad[0], 1, 3::5] = math.nan, math.inf
    for n, r in enumerate(bad):
        k[r, n % 2], v[r, 1 - n % 2, n::7] = math.nan, (math.inf, -math.inf, math.nan)[n % 3]
    h = torch.tensor([0, heads - 1])
    y = fs.swa_packed(q.cuda(), k.cuda(), v.cuda(), bounds(lengths), slopes=slopes.cuda() if alibi else None, window=window, softcap=softcap).cpu()[:, h]
    o, bound = packed(q[:, h], k.nan_to_num(0.0, 0.0, 0.0), v.nan_to_num(0.0, 0.0, 0.0), lengths, slopes[h] if alibi else None, window, softcap, P_STEP[dtype])
    clean = torch.tensor([not any(start[r] <= b <= r and (window is None or r - b <= window) for b in bad) for r in range(rows)])
    assert int(clean.sum()) >= 300
    check(y[clean], o[clean], bound[clean], dtype)
    for n, r in enumerate(bad):
        assert bool(torch.isnan(y[r, n % 2]).all()) and not bool(torch.isfinite(y[r, 1 - n % 2, n::7]).any())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [2.0 ** -40, 0.01, 1.0, 511.0, 513.0, 1e5, 2.0 ** 40])
def test_under_any_soft_cap(fs, softcap, dtype):
    for size in (1.0, 40.0):
        (q, k, v), dev = fused(4, 150, 2, 1, 64, dtype)
        q = (q.float() * size).to(dtype)
        y = fs.swa_packed(q.cuda(), dev[1], dev[2], bounds([70, 80]), softcap=softcap, slopes=slopes_of(2).cuda())
        check(y, *packed(q, k, v, [70, 80], slopes_of(2), None, softcap, P_STEP[dtype]), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_no_sequence_are_left(fs, dtype):
    (q, k, v), dev = fused(5, 200, 3, 3, 64, dtype)
    out = torch.full((200, 3, 64), 7.0, dtype=dtype, device="cuda")
    got = fs.swa_packed(*dev, bounds([40, 0, 77], begin=10), out=out)
    assert got is out
    assert bool((out[:10] == 7).all()) and bool((out[127:] == 7).all())
    o, bound = packed(q[10:], k[10:], v[10:], [40, 0, 77], None, None, 0.0, P_STEP[dtype])
    check(out[10:127], o[:117], bound[:117], dtype)
    out.fill_(7.0)
    fs.swa_packed(*dev, bounds([0, 0]), out=out)
    fs.swa_packed(*dev, bounds([]), out=out)
    assert bool((out == 7).all())
    assert fs.swa_packed(*(t[:0] for t in dev), bounds([0])).shape == (0, 3, 64)


def test_bounds_beyond_the_rows_touch_nothing_else(fs):
    """Bounds that name rows which are not there: those that are come out, nothing beyond them is read or written."""
    (q, k, v), dev = fused(6, 50, 2, 2, 64, torch.bfloat16)
    whole = torch.full((60, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    fs.swa_packed(*dev, torch.tensor([0, 20, 1000], dtype=torch.int32, device="cuda"), out=whole[:50])
    o, bound = packed(q, k, v, [20, 30], None, None, 0.0, 2.0 ** -8)
    check(whole[:50], o, bound, torch.bfloat16)
    assert bool((whole[50:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,hd", [(96, 64), (80, 256)])
def test_rows_and_bounds_of_large_calls(fs, heads, hd, dtype):
    """As the two tests before, where long tiles come first: rows of no sequence, then bounds beyond the rows."""
    (q, k, v), dev = fused(31, 1300, heads, 2, hd, dtype)
    h = torch.tensor([1, heads - 1])
    out = torch.full((1310, heads, hd), 7.0, dtype=dtype, device="cuda")
    fs.swa_packed(*dev, bounds([500, 0, 3, 700], begin=10), window=200, out=out[:1300])
    assert bool((out[:10] == 7).all()) and bool((out[1213:] == 7).all())
    o, bound = packed(q[10:, h], k[10:], v[10:], [500, 0, 3, 700], None, 200, 0.0, P_STEP[dtype])
    check(out[10:1213].cpu()[:, h], o[:1203], bound[:1203], dtype)
    fs.swa_packed(*dev, torch.tensor([-4, 700, 9000, 9000], dtype=torch.int32, device="cuda"), window=200, out=out[:1300])
    check(out[:1300].cpu()[:, h], *packed(q[:, h], k, v, [700, 600], None, 200, 0.0, P_STEP[dtype]), dtype)
    assert bool((out[1300:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_and_heads_far_apart_and_in_other_orders(fs, dtype):
    lengths, heads, kvh, hd = [65, 30], 4, 2, 64
    q, k, v = rand(1, 95, heads, hd, dtype=dtype), rand(2, 95, kvh, hd, dtype=dtype), rand(3, 95, kvh, hd, dtype=dtype)
    o, bound = packed(q, k, v, lengths, None, 50, 0.0, P_STEP[dtype])
    dq = q.cuda().transpose(0, 1).contiguous().transpose(0, 1)            # heads outside of rows
    wide = torch.full((95, 3, kvh, hd + 8), math.nan, dtype=dtype, device="cuda")
    dk, dv = wide[:, 0, :, :hd], wide[:, 2, :, :hd]
    dk.copy_(k)
    dv.copy_(v)
    check(fs.swa_packed(dq, dk, dv, bounds(lengths), window=50), o, bound, dtype)
    one = k[:, :1].cuda().expand(95, 2, hd)                               # one head for all, by a stride of zero
    o, bound = packed(q, k[:, :1].expand(95, 2, hd), v, lengths, None, 50, 0.0, P_STEP[dtype])
    check(fs.swa_packed(dq, one, dv, bounds(lengths), window=50), o, bound, dtype)


def test_in_a_captured_graph_and_on_a_stream(fs):
    rows = 300
    (q, k, v), dev = fused(8, rows, 4, 2, 64, torch.bfloat16)
    x = [t.clone() for t in dev]
    cu = bounds([100, 150, 20])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out = torch.zeros(rows, 4, 64, dtype=torch.bfloat16, device="cuda")
    with torch.cuda.stream(side):
        fs.swa_packed(*x, cu, window=64, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fs.swa_packed(*x, cu, window=64, out=out)
    for n, lengths in enumerate([[100, 150, 20], [300, 0, 0], [1, 1, 290]]):
        for a, b in zip(x, dev):
            a.copy_(b.roll(n, 0))
        cu.copy_(bounds(lengths))
        out.zero_()
        graph.replay()
        want = torch.zeros_like(out)
        fs.swa_packed(*x, cu, window=64, out=want)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        check(out[:sum(lengths)], *(t[:sum(lengths)] for t in packed(*(t.roll(n, 0) for t in (q, k, v)), lengths, None, 64, 0.0, 2.0 ** -8)), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_equal_prompts_as_the_layer_runs_them(fs, dtype):
    """Three prompts of one length: what swa_prefill gives for the batch, to both sides' bounds."""
    from flash_stu import _hip
    heads, hd, T, window = 4, 64, 75, 32
    (q, k, v), dev = fused(9, 3 * T, heads, heads, hd, dtype)
    slopes = slopes_of(heads)
    o, bound = packed(q, k, v, [T] * 3, slopes, window, 50.0, P_STEP[dtype])
    whole = torch.cat(dev, 1).reshape(3, T, 3 * heads * hd).contiguous()
    a = _hip.swa_prefill(whole, slopes.cuda(), heads, window, 50.0).view(3 * T, heads, hd)
    check(a, o, bound, dtype)
    check(fs.swa_packed(*dev, bounds([T] * 3), slopes=slopes.cuda(), window=window, softcap=50.0), o, bound, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_then_steps(fs, dtype):
    """As a program serves: prompts of different lengths, their keys and values into the ring, then a query a sequence, step by step."""
    heads, kvh, hd, window, cap = 4, 2, 64, 30, 37
    lengths = [50, 3, 0, 29]
    rows, slopes = sum(lengths), slopes_of(heads)
    (q, k, v), dev = fused(1, rows, heads, kvh, hd, dtype)
    cu, pos = bounds(lengths), torch.zeros(4, dtype=torch.int32, device="cuda")
    cache, ring = fs.KV4Cache(4, kvh, hd, cap), Ring(4, kvh, hd, cap)
    y = fs.swa_packed(*dev, cu, slopes=slopes.cuda(), window=window, softcap=50.0)
    cache.write(dev[1], dev[2], pos, cu)
    check(y, *packed(q, k, v, lengths, slopes, window, 50.0, P_STEP[dtype]), dtype)
    ring.write(k, v, [0] * 4, lengths)
    at = list(lengths)
    pos += cu.diff()
    for step in range(12):
        (q, k, v), dev = fused(20 + step, 4, heads, kvh, hd, dtype)
        y = cache.attend(dev[0], pos, dev[1], dev[2], slopes=slopes.cuda(), window=window, softcap=50.0)
        ring.write(k, v, at)
        check(y, *ring.attend(q, at, slopes, window, 50.0, 2.0 ** -16), dtype)
        pos += 1
        at = [p + 1 for p in at]
    gk, _ = cache.read(pos - 1, dtype=torch.float32)
    assert torch.equal(gk.cpu().double(), held(k))


def test_refusals(fs):
    from flash_stu._hip import FlashSTUHipError
    q, k, cu = torch.zeros(8, 4, 64, device="cuda"), torch.zeros(8, 2, 64, device="cuda"), bounds([5, 3])
    bad = [lambda: fs.swa_packed(q, k, k.bfloat16(), cu), lambda: fs.swa_packed(q.half(), k.half(), k.half(), cu), lambda: fs.swa_packed(q, k[:7], k[:7], cu),
           lambda: fs.swa_packed(q[:, :3], k, k, cu), lambda: fs.swa_packed(q, k[:, :, :32], k[:, :, :32], cu), lambda: fs.swa_packed(q, k, k[:, :1], cu),
           lambda: fs.swa_packed(q[..., :48], k[..., :48], k[..., :48], cu), lambda: fs.swa_packed(q, k, k, cu.long()), lambda: fs.swa_packed(q, k, k, cu.cpu()),
           lambda: fs.swa_packed(q, k, k, cu[:0]), lambda: fs.swa_packed(q, k, k, cu, window=-1), lambda: fs.swa_packed(q, k, k, cu, softcap=-1.0),
           lambda: fs.swa_packed(q, k, k, cu, softcap=math.nan), lambda: fs.swa_packed(q, k, k, cu, slopes=torch.zeros(2, device="cuda")),
           lambda: fs.swa_packed(q, k, k, cu, out=q), lambda: fs.swa_packed(q, k, k, cu, out=q.bfloat16()), lambda: fs.swa_packed(q, k, k, cu, out=torch.zeros(8, 4, 64)),
           lambda: fs.swa_packed(q, k, k, cu, out=torch.zeros(8, 64, 4, device="cuda").transpose(1, 2)), lambda: fs.swa_packed(q.cpu(), k, k, cu),
           lambda: fs.swa_packed(q, k.cpu(), k, cu), lambda: fs.swa_packed(q[:, :, ::2], k[:, :, ::2], k[:, :, ::2], cu),
           lambda: fs.swa_packed(torch.zeros(8 * 4 * 64 + 1, device="cuda")[1:].view(8, 4, 64), k, k, cu), lambda: fs.swa_packed(q, k[:, :0], k[:, :0], cu)]
    for call in bad:
        with pytest.raises(FlashSTUHipError):
            call()
    with pytest.raises(NotImplementedError, match="forward only"):
        fs.swa_packed(q.requires_grad_(), k, k, cu)
    with torch.no_grad():
        fs.swa_packed(q, k, k, cu)


@pytest.mark.parametrize("hd,heads,rows,window,softcap,alibi", [
    (32, 2, 320, 100, 50.0, True),
    (64, 2, 320, None, 0.0, False),
    (64, 2, 320, None, 600.0, False),
    (64, 96, 1024, 300, 50.0, True),
    (128, 2, 320, 100, 0.0, True),
    (128, 96, 1024, None, 0.0, False),
    (128, 2, 8192, 5000, 0.0, True),
    (256, 2, 320, None, 50.0, False),
])
@pytest.mark.parametrize("tail", [1, 2, 40])
def test_a_tile_ends_with_its_sequence(fs, tail, hd, heads, rows, window, softcap, alibi):
    """A tile holds zeros behind its sequence's last row: a NaN from there would send rows to the form that goes key by key, whose roundings differ."""
    n, after = rows + tail, 90
    (q, k, v), dev = fused(37, n + after, heads, 2, hd, torch.bfloat16)
    args = dict(slopes=slopes_of(heads).cuda() if alibi else None, window=window, softcap=softcap)
    want = fs.swa_packed(*dev, bounds([n, after]), **args)[:n]
    assert bool(torch.isfinite(want).all())
    dirty = [t.clone() for t in dev]
    dirty[1][n:], dirty[2][n:] = math.nan, math.nan
    assert torch.equal(fs.swa_packed(*dirty, bounds([n, after]), **args)[:n], want)
    assert torch.equal(fs.swa_packed(*dirty, bounds([n]), **args)[:n], want)
    if tail > 2:                                                         # that it would show: a NaN inside of the tile does
        dirty[2][n - 1] = math.nan
        assert not torch.equal(fs.swa_packed(*dirty, bounds([n, after]), **args)[:n - 1], want[:n - 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("window", [None, 20])
@pytest.mark.parametrize("size", [-math.inf, -3.3e38])
def test_a_score_of_minus_infinity_beside_an_infinity_that_is_not_seen(fs, size, window, hd, dtype):
    """A key whose score is -infinity (an infinite key, or a product past fp32's range) has no weight, whether or not its row is formed key by key."""
    from attention_reference import attention
    n, heads = 75, 2
    q, k, v = (rand(50 + i, n, heads, hd, dtype=dtype) for i in range(3))
    q[:, :, 0] = q[:, :, 0].abs() + 2
    gone = [0, 30, 31]
    k[gone], v[70, :, ::9] = 0, 0
    far = torch.arange(n)[:, None] - torch.arange(n)
    far = torch.where((far >= 0) & (far <= (n if window is None else window)), far, -1)
    far[:, gone] = -1
    dk, dv = k.clone(), v.clone()
    dk[gone, :, 0], dv[70, :, ::9] = size, math.inf
    y = fs.swa_packed(q.cuda(), dk.cuda(), dv.cuda(), bounds([n]), window=window).cpu()
    clean = torch.arange(1, 70)                                          # row 0 sees nothing else, row 70 and those behind it the infinity
    for h in range(heads):
        o, bound = attention(q[:, h].double(), k[:, h].double(), v[:, h].double(), far.double(), 0.0, 0.0, P_STEP[dtype])
        check(y[clean, h], o[clean], bound[clean], dtype)
    assert bool(torch.isnan(y[0]).all()) and not bool(torch.isfinite(y[70, :, ::9]).any())


@pytest.mark.parametrize("heads,kvh,hd,lengths,window,softcap,alibi", [
    (12, 12, 64, [17, 1, 40], 512, 50.0, True),
    (1, 1, 128, [0, 2, 0, 0, 3, 0], None, 0.0, True),
    (4, 2, 64, [129, 63, 64, 65, 128], 31, 600.0, True),
    (4, 1, 128, [300, 33, 127], None, 0.0, False),
    (6, 2, 32, [100, 257, 5], 0, 0.0, True),
    (2, 1, 256, [150, 70, 1], 100, 0.0, True),
    (5, 5, 256, [33, 64], None, 50.0, False),
    (64, 1, 64, [1, 1700, 0, 130, 64, 17], 70, 50.0, True),
    (128, 16, 32, [700, 130], None, 50.0, False),
    (64, 32, 128, [0, 900, 500, 0], 333, 50.0, True),
    (2, 1, 128, [4500], None, 0.0, True),
])
def test_probabilities_in_two_parts(fs, heads, kvh, hd, lengths, window, softcap, alibi):
    """fine: as a bf16 value and what its rounding left, 2^-16 of them; in fp32 the same bits as without."""
    rows = sum(lengths)
    (q, k, v), dev = fused(7, rows, heads, kvh, hd, torch.bfloat16)
    slopes, h = slopes_of(heads), torch.tensor([0, heads - 1])
    args = dict(slopes=slopes.cuda() if alibi else None, window=window, softcap=softcap)
    y = fs.swa_packed(*dev, bounds(lengths), fine=True, **args)
    kv = h // (heads // kvh)
    check(y.cpu()[:, h], *packed(q[:, h], k[:, kv], v[:, kv], lengths, slopes[h] if alibi else None, window, softcap, 2.0 ** -16), torch.bfloat16)
    assert bool(torch.isfinite(y).all())
    wide = [t.float() for t in dev]
    assert torch.equal(fs.swa_packed(*wide, bounds(lengths), fine=True, **args), fs.swa_packed(*wide, bounds(lengths), **args))


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("heads,window,softcap,alibi", [(2, 20, 50.0, True), (96, None, 0.0, False)])
def test_what_a_row_does_not_see_leaves_its_two_parts_alone(fs, heads, window, softcap, alibi, hd):
    lengths, bad = [300, 330], [250, 299, 620]
    (q, k, v), dev = fused(41, sum(lengths), heads, 2, hd, torch.bfloat16)
    args = dict(slopes=slopes_of(heads).cuda() if alibi else None, window=window, softcap=softcap, fine=True)
    dirty = [t.clone() for t in dev]
    dirty[1][bad, 0], dirty[2][bad, 1, ::5] = math.nan, math.inf
    y = fs.swa_packed(*dirty, bounds(lengths), **args)
    start = [0] * 300 + [300] * 330
    clean = [r for r in range(630) if not any(start[r] <= b <= r and (window is None or r - b <= window) for b in bad)]
    h = torch.tensor([0, heads - 1])
    kv = h // (heads // 2)
    o, bound = packed(q[:, h], k[:, kv], v[:, kv], lengths, slopes_of(heads)[h] if alibi else None, window, softcap, 2.0 ** -16)
    check(y.cpu()[clean][:, h], o[clean], bound[clean], torch.bfloat16)
    assert bool(torch.isnan(y[bad, 0]).all()) and not bool(torch.isfinite(y[bad, heads - 1, ::5]).any())


def test_two_parts_in_a_captured_graph(fs):
    (_, _, _), dev = fused(8, 300, 4, 2, 64, torch.bfloat16)
    x, cu = [t.clone() for t in dev], bounds([100, 150, 20])
    fs.swa_packed(*x, cu, window=64, fine=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = fs.swa_packed(*x, cu, window=64, fine=True)
    for n in range(3):
        for a, b in zip(x, dev):
            a.copy_(b.roll(n, 0))
        graph.replay()
        want = fs.swa_packed(*x, cu, window=64, fine=True)
        torch.cuda.synchronize()
        assert torch.equal(y[:270], want[:270])

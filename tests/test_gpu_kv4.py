"""The 4-bit ring cache against its definition in 64 bits: what it holds (exactly, in any type), and the attention of one query a sequence over it.
Where a bound's p_step is 2^-16 the probabilities go into the product as two bf16 parts, 8 bits each."""
import math

import pytest
import torch

from attention_reference import Ring, check, held

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]
P_STEP = 2.0 ** -16


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


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bounds(lengths, begin=0):
    total = [begin]
    for n in lengths:
        total.append(total[-1] + n)
    return ints(total)


def same(a, b):
    """Equal values, NaN where NaN, zeros of one sign."""
    a, b = a.detach().cpu().double(), b.detach().cpu().double()
    nan = torch.isnan(a) & torch.isnan(b)
    return bool(((a == b) & (torch.signbit(a) == torch.signbit(b)) | nan).all())


# ---------------------------------------------------------------- what is held
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,kvh,cap,lengths,pos", [
    (64, 12, 513, [5, 1, 0, 9], [0, 511, 7, 1000]),
    (128, 2, 33, [70, 33, 32, 34, 1], [0, 5, 40, 31, 32]),
    (32, 3, 1, [1, 4, 0], [0, 7, 9]),
    (256, 1, 40, [41, 3, 80], [100, 39, 2 ** 31 - 100]),
    (64, 1, 8, [0, 0, 1], [3, -1, 8]),
    (128, 4, 100, [301], [17]),
])
def test_what_is_written_is_read_back(fs, hd, kvh, cap, lengths, pos, dtype):
    rows = sum(lengths)
    k, v = rand(1, rows, kvh, hd, dtype=dtype), rand(2, rows, kvh, hd, dtype=dtype)
    cache = fs.KV4Cache(len(lengths), kvh, hd, cap)
    ring = Ring(len(lengths), kvh, hd, cap)
    cache.write(k.cuda(), v.cuda(), ints(pos), bounds(lengths))
    ring.write(k, v, pos, lengths)
    full = bounds([cap] * len(lengths))                                   # every slot of the ring, those never written zero
    for t in DTYPES:
        gk, gv = cache.read(ints([0] * len(lengths)), full, rows=cap * len(lengths), dtype=t)
        assert gk.dtype is t and same(gk, ring.k.flatten(0, 1)) and same(gv, ring.v.flatten(0, 1))
    last = [min(n, cap) for n in lengths]
    gk, gv = cache.read(ints([p + n - m if p >= 0 else p for p, n, m in zip(pos, lengths, last)]), bounds(last), rows=sum(last), dtype=torch.float32)
    keep = torch.cat([torch.arange(sum(lengths[:i + 1]) - m, sum(lengths[:i + 1])) for i, m in enumerate(last)])
    assert same(gk, held(k)[keep]) and same(gv, held(v)[keep])


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_row_to_each_sequence_from_a_fused_projection(fs, dtype):
    kvh, hd, cap = 3, 64, 50
    cache, ring = fs.KV4Cache(6, kvh, hd, cap), Ring(6, kvh, hd, cap)
    for step in range(3):
        fused = rand(step, 6, 5 * kvh, hd, dtype=dtype)
        k, v = fused[:, 2 * kvh:3 * kvh], fused[:, 4 * kvh:]
        pos = [0 + step, 49 + step, -1, 99 + step, 7 + step, 2 ** 31 - 4 + step]
        cache.write(fused.cuda()[:, 2 * kvh:3 * kvh], fused.cuda()[:, 4 * kvh:], ints(pos))
        ring.write(k, v, pos)
        gk, gv = cache.read(ints(pos), dtype=dtype)
        used = [i for i in range(6) if pos[i] >= 0]
        assert same(gk[used], held(k)[used]) and same(gv[used], held(v)[used])
        assert not gk[2].any() and not gv[2].any()
    gk, gv = cache.read(ints([0] * 6), bounds([cap] * 6), rows=6 * cap)
    assert same(gk, ring.k.flatten(0, 1)) and same(gv, ring.v.flatten(0, 1))


def test_every_code_to_the_nearest(fs):
    """The codes' values, the middles between them (to the even code) and what lies beside those, both signs, under scales of all sizes."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
    mid = (grid[1:] + grid[:-1]) / 2
    even = torch.where(torch.arange(7) % 2 == 0, grid[:-1], grid[1:])
    x = torch.cat([grid, mid, mid * (1 + 2.0 ** -20), mid * (1 - 2.0 ** -20), torch.tensor([6.5, 6.99, 5.001, 0.01, 2.25])])
    want = torch.cat([grid, even, grid[1:], grid[:-1], torch.tensor([6.0, 6.0, 6.0, 0.0, 2.0])]).double()
    x, want = torch.cat([x, -x]), torch.cat([want, -want])
    n = -(-len(x) // 31) * 31
    x, want = (torch.cat([t, t.new_zeros(n - len(t))]).view(-1, 31) for t in (x, want))
    x, want = (torch.cat([torch.full((len(t), 1), w, dtype=torch.float64), t], 1) for t, w in ((x, 7.0), (want, 6.0)))
    cache = fs.KV4Cache(1, 1, 32, 64)
    for e in (-118, -60, -3, 0, 2, 40, 124):
        scaled = (x * 2.0 ** e).float()[:, None].cuda()
        cache.write(scaled, scaled, ints([0]), bounds([len(x)]))
        for got in cache.read(ints([0]), bounds([len(x)]), rows=len(x), dtype=torch.float32):
            assert same(got[:, 0], want * 2.0 ** e)


@pytest.mark.parametrize("dtype", DTYPES)
def test_zeros_extremes_and_values_that_are_not_finite(fs, dtype):
    x = torch.zeros(12, 1, 64, dtype=dtype)
    x[1] = -0.0
    x[2] = 2.0 ** -126
    x[3, 0, 5], x[3, 0, 40] = math.inf, 1.0
    x[4, 0, 63] = math.nan
    x[5, 0, 0] = -math.inf
    x[6, 0, 7] = torch.finfo(dtype).max
    x[7, 0, :32] = torch.finfo(dtype).min
    x[8, 0, ::2] = 1.75 * 2.0 ** 127
    x[9] = 7 * 2.0 ** -120
    x[10] = 2.0 ** -121
    x[11] = 1.25 * 2.0 ** -121
    cache = fs.KV4Cache(1, 1, 64, 12)
    cache.write(x.cuda(), x.flip(0).cuda(), ints([0]), bounds([12]))
    for t in DTYPES:
        gk, gv = cache.read(ints([0]), bounds([12]), rows=12, dtype=t)
        assert same(gk, held(x)) and same(gv, held(x.flip(0)))
        assert bool(torch.isfinite(gk[[0, 1, 2, 6, 7, 8, 9, 10, 11]]).all())
        assert bool(torch.isnan(gk[3, 0, :32]).all()) and float(gk[3, 0, 40]) == 1.0


def test_rows_of_no_sequence(fs):
    k, v = rand(3, 20, 2, 32), rand(4, 20, 2, 32)
    cache, ring = fs.KV4Cache(2, 2, 32, 16), Ring(2, 2, 32, 16)
    cu = ints([3, 8, 12])                                                # rows in front of the first and behind the last
    cache.write(k.cuda(), v.cuda(), ints([14, 0]), cu)
    ring.write(k[3:], v[3:], [14, 0], [5, 4])
    gk, gv = cache.read(ints([0, 0]), bounds([16, 16]), rows=32, dtype=torch.float32)
    assert same(gk, ring.k.flatten(0, 1)) and same(gv, ring.v.flatten(0, 1))
    gk, gv = cache.read(ints([14, 0]), cu, rows=20, dtype=torch.float32)
    assert same(gk[3:12], held(k)[3:12]) and not gk[:3].any() and not gk[12:].any() and not gv[12:].any()


# ---------------------------------------------------------------- one query a sequence
def filled(fs, batch, kvh, hd, cap, seed, dtype=torch.bfloat16):
    """A ring with something in every slot, and its definition."""
    k, v = rand(seed, batch * cap, kvh, hd, dtype=dtype), rand(seed + 1, batch * cap, kvh, hd, dtype=dtype)
    cache, ring = fs.KV4Cache(batch, kvh, hd, cap), Ring(batch, kvh, hd, cap)
    cache.write(k.cuda(), v.cuda(), ints([0] * batch), bounds([cap] * batch))
    ring.k, ring.v = held(k).view(batch, cap, kvh, hd), held(v).view(batch, cap, kvh, hd)
    return cache, ring


def slopes_of(heads):
    return 0.25 * 2.0 ** (-8.0 * (torch.arange(heads) + 1) / heads)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,hd,cap,window,pos,softcap,alibi", [
    (12, 12, 64, 513, 512, [0, 1, 511, 512, 513, 700, -1], 50.0, True),
    (16, 16, 128, 300, 255, [299, 300, 31, 32, 1000], 50.0, True),
    (4, 4, 64, 1, 0, [0, 5], 0.0, False),
    (4, 2, 32, 70, 0, [0, 69, 70, 33], 0.0, True),
    (8, 2, 256, 100, None, [99, 50, 100, 163], 0.0, False),
    (3, 1, 128, 1000, 777, [776, 777, 999, 5000], 30.0, True),
    (5, 1, 64, 257, None, [256, 511, 3], 0.0, True),
    (16, 2, 128, 4100, None, [4099, 2 ** 31 - 2], 0.0, False),
    (16, 1, 64, 64, 63, [63, 64, 65, 127, 95, 96], 0.0, True),
    (34, 2, 64, 129, None, [128, 77], 50.0, True),
    (24, 1, 128, 33, 32, [31, 32, 33, 65], 0.0, False),
    (64, 2, 32, 40, 7, [6, 7, 8, 39, 40, 41], 0.0, False),
    (2, 2, 32, 9000, None, [8999], 0.0, False),
    (1, 1, 256, 2500, 2400, [7000], 50.0, True),
])
def test_attend(fs, heads, kvh, hd, cap, window, pos, softcap, alibi, dtype):
    batch = len(pos)
    cache, ring = filled(fs, batch, kvh, hd, cap, 10)
    q, slopes = rand(5, batch, heads, hd, dtype=dtype), slopes_of(heads) if alibi else None
    y = cache.attend(q.cuda(), ints(pos), slopes=None if slopes is None else slopes.cuda(), window=window, softcap=softcap)
    o, bound = ring.attend(q, pos, slopes, window, softcap, P_STEP)
    assert y.shape == q.shape and y.dtype is dtype
    check(y, o, bound, dtype)
    for s, p in enumerate(pos):
        assert p >= 0 or not y[s].any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [2.0 ** -40, 0.01, 1.0, 511.0, 513.0, 1e5, 2.0 ** 40])
def test_attend_under_any_soft_cap(fs, softcap, dtype):
    cache, ring = filled(fs, 2, 2, 64, 100, 60)
    for size in (1.0, 40.0):
        q = (rand(8, 2, 4, 64) * size).to(dtype)
        y = cache.attend(q.cuda(), ints([99, 130]), softcap=softcap)
        check(y, *ring.attend(q, [99, 130], None, None, softcap, P_STEP), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,heads,kvh,hd,cap,window,softcap", [
    (3, 4, 4, 32, 20, None, 0.0),
    (2, 22, 2, 64, 513, 512, 50.0),              # 11 query heads to a key head: two workgroups to a head
    (1, 12, 12, 64, 2500, None, 0.0),            # in parts
    (1, 34, 2, 128, 1700, None, 50.0),           # both
    (5, 16, 8, 128, 100, 70, 0.0),
    (2, 3, 1, 256, 33, 32, 0.0),
    (2, 8, 8, 256, 1400, 1200, 0.0),
    (64, 32, 32, 32, 6200, None, 0.0),           # dealt evenly
    (40, 20, 10, 64, 64, None, 0.0),             # more workgroups than compute units
])
def test_a_step_is_its_write_and_its_attend(fs, batch, heads, kvh, hd, cap, window, softcap, dtype):
    one, two = fs.KV4Cache(batch, kvh, hd, cap), fs.KV4Cache(batch, kvh, hd, cap)
    n = min(cap, 300)
    prompt = rand(1, n * batch, 2 * kvh, hd).to(dtype).cuda()
    cu = ints(range(0, n * batch + 1, n))
    at = ints([(0, cap - n // 2, 3 * cap + 7)[b % 3] for b in range(batch)])
    for c in (one, two):
        c.write(prompt[:, :kvh], prompt[:, kvh:], at, cu)
    pos = at + n
    pos[batch // 2 if batch > 1 else 1:][:1] = -1
    slopes = slopes_of(heads).cuda()
    for step in range(3):
        qkv = rand(2 + step, batch, heads + 2 * kvh, hd).to(dtype).cuda()
        q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
        y = one.attend(q, pos, k, v, slopes=slopes, window=window, softcap=softcap)
        two.write(k, v, pos)
        assert torch.equal(y, two.attend(q, pos, slopes=slopes, window=window, softcap=softcap)) and torch.equal(one.data, two.data)
        pos = torch.where(pos < 0, pos, pos + (1 if step == 0 else cap // 2 + 1))
    k = rand(9, batch, kvh, hd).to(torch.bfloat16 if dtype is torch.float32 else torch.float32).cuda()       # of another type than q
    y = one.attend(q, pos, k, k, slopes=slopes, window=window, softcap=softcap)
    two.write(k, k, pos)
    assert torch.equal(y, two.attend(q, pos, slopes=slopes, window=window, softcap=softcap)) and torch.equal(one.data, two.data)


def test_a_refused_call_writes_nothing(fs):
    from flash_stu._hip import FlashSTUHipError
    cache = fs.KV4Cache(2, 2, 64, 40)
    k, q, pos = torch.ones(2, 2, 64, device="cuda"), torch.ones(2, 4, 64, device="cuda"), ints([0, 0])
    for call in (lambda: cache.attend(q[:, :3], pos, k, k), lambda: cache.attend(q, pos, k, k, window=40), lambda: cache.attend(q, pos, k, k, softcap=-1.0),
                 lambda: cache.attend(q, pos, k), lambda: cache.attend(q, pos, k, k, slopes=torch.ones(3, device="cuda")), lambda: cache.attend(q, pos, k, k, out=q[:1]),
                 lambda: cache.attend(q, pos, k, k, out=q), lambda: cache.attend(q, pos, k[:1], k[:1]), lambda: cache.attend(q, pos, k, k[..., :32]),
                 lambda: cache.attend(q[:, :2], pos, k, k, out=k)):
        with pytest.raises(FlashSTUHipError):
            call()
    assert not cache.data.any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("splits", [1, 2, 7, 64, 65, 100, 300])
@pytest.mark.parametrize("heads,kvh,hd,cap,window,pos", [(4, 2, 64, 700, None, [699, 20, -1, 1500]), (9, 1, 128, 300, 250, [299, 0, 310]), (2, 2, 256, 90, 63, [-1, 500]),
                                                        (3, 3, 32, 64, None, [-1, -1])])
def test_attend_in_any_number_of_parts(fs, monkeypatch, heads, kvh, hd, cap, window, pos, splits, dtype):
    """Every way to cut the keys, more parts than tiles among them."""
    from flash_stu import _hip
    monkeypatch.setattr(_hip, "_kv4_splits", lambda *a: (splits, _hip.load().fstu_kv4_attend_ws(*a[:4], splits)))
    cache, ring = filled(fs, len(pos), kvh, hd, cap, 40)
    q, slopes = rand(5, len(pos), heads, hd, dtype=dtype), slopes_of(heads)
    y = cache.attend(q.cuda(), ints(pos), slopes=slopes.cuda(), window=window, softcap=50.0)
    check(y, *ring.attend(q, pos, slopes, window, 50.0, P_STEP), dtype)


def test_attend_dealt_evenly_over_many_sequences(fs, monkeypatch):
    """More sequences than a wave has lanes, many of them not in use."""
    from flash_stu import _hip
    batch, cap = 150, 200
    pos = [-1 if i % 3 == 1 or 60 <= i < 130 else (i * 37) % 450 for i in range(batch)]
    cache, ring = filled(fs, batch, 1, 32, cap, 50)
    q = rand(6, batch, 2, 32, dtype=torch.bfloat16)
    o, bound = ring.attend(q, pos, None, None, 0.0, P_STEP)
    for splits in (65, 256, 1):
        monkeypatch.setattr(_hip, "_kv4_splits", lambda *a: (splits, _hip.load().fstu_kv4_attend_ws(*a[:4], splits)))
        check(cache.attend(q.cuda(), ints(pos)), o, bound, torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_what_the_window_leaves_out_may_be_anything(fs, hd, dtype):
    """NaN in every slot that the query does not see, at every offset of the window's ends in a tile."""
    batch, kvh, cap, window = 70, 1, 150, 41
    pos = list(range(batch))[:-3] + [149, 150, 400]
    k, v = rand(1, batch * cap, kvh, hd).view(batch, cap, kvh, hd), rand(2, batch * cap, kvh, hd).view(batch, cap, kvh, hd)
    for s, p in enumerate(pos):
        unseen = torch.ones(cap, dtype=torch.bool)
        unseen[torch.arange(max(0, p - window), p + 1) % cap] = False
        k[s, unseen], v[s, unseen] = math.nan, math.inf
    cache, ring = fs.KV4Cache(batch, kvh, hd, cap), Ring(batch, kvh, hd, cap)
    cache.write(k.flatten(0, 1).cuda(), v.flatten(0, 1).cuda(), ints([0] * batch), bounds([cap] * batch))
    ring.k, ring.v = held(k), held(v)
    q = rand(3, batch, 2, hd, dtype=dtype)
    y = cache.attend(q.cuda(), ints(pos), window=window)
    check(y, *ring.attend(q, pos, None, window, 0.0, P_STEP), dtype)


def test_a_key_that_is_not_finite_spoils_its_own_head_alone(fs):
    cache, ring = filled(fs, 2, 2, 64, 40, 3)
    k, v = torch.zeros(2, 2, 64), torch.zeros(2, 2, 64)
    v[0, 1, 33] = math.inf                                               # one block of one head's value
    q = rand(4, 2, 4, 64)
    y = cache.attend(q.cuda(), ints([45, 45]), k.cuda(), v.cuda())
    ring.write(k, v, [45, 45])
    o, bound = ring.attend(q, [45, 45], None, None, 0.0, P_STEP)
    assert bool(torch.isnan(y[0, 2:, 32:]).all())
    fine = torch.isfinite(o)
    assert bool(torch.isfinite(y.cpu()[fine]).all()) and int(fine.sum()) == 2 * 4 * 64 - 2 * 32
    check(torch.where(fine.cuda(), y, 0.0), torch.where(fine, o, 0.0), torch.where(fine, bound, 0.0), torch.float32)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kvh,hd,cap,pos", [(12, 12, 64, 513, [0, 512, 600, -1, 31]), (8, 2, 128, 2100, [2099, 0, 4000]), (3, 3, 32, 1, [4, 0]), (6, 1, 256, 65, [64, 65])])
def test_the_new_position_with_its_query(fs, heads, kvh, hd, cap, pos, dtype):
    """attend with k and v is write and attend, to the bit, in the result and in the cache."""
    a, _ = filled(fs, len(pos), kvh, hd, cap, 20)
    b = fs.KV4Cache(len(pos), kvh, hd, cap)
    b.data.copy_(a.data)
    fused = rand(9, len(pos), heads + 2 * kvh, hd, dtype=dtype).cuda()
    q, k, v = fused[:, :heads], fused[:, heads:heads + kvh], fused[:, heads + kvh:]
    slopes = slopes_of(heads).cuda()
    a.write(k, v, ints(pos))
    want = a.attend(q, ints(pos), slopes=slopes, softcap=50.0)
    out = torch.full_like(want, 7.0)
    got = b.attend(q, ints(pos), k, v, slopes=slopes, softcap=50.0, out=out)
    assert got is out and torch.equal(got, want) and torch.equal(a.data, b.data)


def test_long_ring_beyond_32_bits(fs):
    """Two sequences of a ring whose codes take more than 4 GiB: the offsets of the second."""
    kvh, hd, cap = 16, 256, 1 << 20
    cache = fs.KV4Cache(2, kvh, hd, cap)
    assert cache.data.numel() > 2 * 2 ** 32
    k, v = rand(1, 80, kvh, hd, dtype=torch.bfloat16), rand(2, 80, kvh, hd, dtype=torch.bfloat16)
    start = cap - 40
    cache.write(k.cuda(), v.cuda(), ints([start, start]), bounds([0, 80]))
    gk, gv = cache.read(ints([start, start]), bounds([0, 80]), rows=80, dtype=torch.float32)
    assert same(gk, held(k)) and same(gv, held(v))
    q = rand(3, 2, 16, hd, dtype=torch.bfloat16)
    pos = [-1, start + 79]
    y = cache.attend(q.cuda(), ints(pos), window=79)
    ring = Ring(2, kvh, hd, 80)
    ring.k[1], ring.v[1] = held(k), held(v)
    check(y, *ring.attend(q, [-1, 79], None, 79, 0.0, P_STEP), torch.bfloat16)


def test_steps_in_a_captured_graph(fs):
    """A step (position counted on the device) captured once and replayed gives what eager steps give, eager work in between."""
    heads, kvh, hd, cap, steps = 6, 2, 64, 40, 50
    cache, other = fs.KV4Cache(3, kvh, hd, cap), fs.KV4Cache(3, kvh, hd, cap)
    slopes = slopes_of(heads).cuda()
    rows = rand(1, steps, 3, heads + 2 * kvh, hd, dtype=torch.bfloat16).cuda()
    first = ints([0, 30, -100])
    x, pos = rows[0].clone(), first.clone()

    def step(c, x, pos):
        return c.attend(x[:, :heads], pos, x[:, heads:heads + kvh], x[:, heads + kvh:], slopes=slopes, window=33, softcap=50.0)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, x, pos)
    torch.cuda.current_stream().wait_stream(side)
    cache.data.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = step(cache, x, pos)
        pos += 1
    pos.copy_(first)
    eager_pos = first.clone()
    for t in range(steps):
        x.copy_(rows[t])
        graph.replay()
        want = step(other, rows[t], eager_pos)
        eager_pos += 1
        torch.cuda.synchronize()
        assert torch.equal(y, want), t
    assert torch.equal(cache.data, other.data) and torch.equal(pos, eager_pos)


def test_two_streams_share_nothing(fs):
    """Calls on two streams at once over the same cache, many splits each."""
    cache, ring = filled(fs, 1, 2, 64, 6000, 30)
    qs = [rand(i, 1, 4, 64, dtype=torch.bfloat16) for i in range(2)]
    dq = [q.cuda() for q in qs]
    pos = [ints([5999]), ints([3000])]
    torch.cuda.synchronize()
    streams, ys = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                ys[i].append(cache.attend(dq[i], pos[i]))
    torch.cuda.synchronize()
    for i, p in enumerate((5999, 3000)):
        check(ys[i][0], *ring.attend(qs[i], [p], None, None, 0.0, P_STEP), torch.bfloat16)
        assert all(torch.equal(y, ys[i][0]) for y in ys[i])


# ---------------------------------------------------------------- refusals
def test_refusals(fs):
    from flash_stu._hip import FlashSTUHipError
    cache = fs.KV4Cache(2, 2, 64, 40)
    k, q, pos = torch.zeros(2, 2, 64, device="cuda"), torch.zeros(2, 4, 64, device="cuda"), ints([0, 0])
    for args in ((0, 1, 64, 8), (1, 0, 64, 8), (1, 1, 48, 8), (1, 1, 64, 0), (1, 1, 64, 2 ** 30 + 1)):
        with pytest.raises(FlashSTUHipError):
            fs.KV4Cache(*args)
    with pytest.raises(FlashSTUHipError, match="CPU"):
        fs.KV4Cache(1, 1, 64, 8, device="cpu")
    bad = [lambda: cache.write(k, k.bfloat16(), pos), lambda: cache.write(k.half(), k.half(), pos), lambda: cache.write(k[:, :1], k[:, :1], pos),
           lambda: cache.write(k[:1], k[:1], pos), lambda: cache.write(k, k, pos.long()), lambda: cache.write(k, k, pos[:1]), lambda: cache.write(k, k, pos.cpu()),
           lambda: cache.write(k.cpu(), k, pos), lambda: cache.write(k, k, pos, ints([0, 2])), lambda: cache.write(k.transpose(1, 2), k.transpose(1, 2), pos),
           lambda: cache.read(pos, ints([0, 1, 2])), lambda: cache.read(pos, rows=3), lambda: cache.read(pos, dtype=torch.float16),
           lambda: cache.read(pos, ints([0, 1, 2]), rows=-1),
           lambda: cache.attend(q[:, :3], pos), lambda: cache.attend(q[:1], pos), lambda: cache.attend(q, pos, window=40), lambda: cache.attend(q, pos, window=-1),
           lambda: cache.attend(q, pos, k), lambda: cache.attend(q, pos, softcap=-1.0), lambda: cache.attend(q, pos, softcap=math.inf),
           lambda: cache.attend(q, pos, softcap=math.nan), lambda: cache.attend(q, pos, slopes=torch.zeros(3, device="cuda")),
           lambda: cache.attend(q, pos, slopes=torch.zeros(4, device="cuda").double()), lambda: cache.attend(q, pos, out=torch.zeros(2, 4, 64)),
           lambda: cache.attend(q, pos, out=torch.zeros(2, 4, 64, device="cuda").bfloat16()), lambda: cache.attend(q, pos, out=q),
           lambda: cache.attend(torch.zeros(2 * 4 * 64 + 1, device="cuda")[1:].view(2, 4, 64), pos)]
    for i, call in enumerate(bad):
        with pytest.raises(FlashSTUHipError):
            call()
            print("not refused:", i)
    for call in (lambda: cache.write(k.requires_grad_(), k, pos), lambda: cache.attend(q.requires_grad_(), pos)):
        with pytest.raises(NotImplementedError, match="forward only"):
            call()
    with torch.no_grad():
        cache.write(k, k, pos)
    assert not cache.data[:64].any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_refused_call_of_another_type_writes_nothing(fs, dtype):
    from flash_stu._hip import FlashSTUHipError
    cache = fs.KV4Cache(2, 2, 64, 40)
    other = torch.bfloat16 if dtype is torch.float32 else torch.float32
    k, q, pos = torch.ones(2, 2, 64, dtype=other, device="cuda"), torch.ones(2, 4, 64, dtype=dtype, device="cuda"), ints([0, 0])
    wide, ends = torch.ones(2 * 4 * 64 + 1, dtype=dtype, device="cuda"), torch.ones(2, 2, 72, dtype=other, device="cuda")
    for call in (lambda: cache.attend(q, pos, k, k, out=q), lambda: cache.attend(wide[1:].view(2, 4, 64), pos, k, k), lambda: cache.attend(q, pos, k, k[:1]),
                 lambda: cache.attend(q, pos, k, k.to(dtype)), lambda: cache.attend(q, pos, k.half(), k.half()), lambda: cache.attend(q, pos, k, k.transpose(0, 1)[..., :32]),
                 lambda: cache.attend(q, pos, ends[..., 1:65], k), lambda: cache.attend(q, pos, k.cpu(), k), lambda: cache.attend(q, pos, None, k),
                 lambda: cache.attend(q, pos, k, k, out=q.to(other))):
        with pytest.raises(FlashSTUHipError):
            call()
    assert not cache.data.any()
    assert bool(torch.isfinite(cache.attend(q, pos, k, k)).all()) and bool(cache.data.any())


def test_two_threads_on_one_stream(fs):
    """Calls in parts from two threads, whose workspaces come from the same stream's memory."""
    import threading
    caches = [filled(fs, 1, 2, 64, 6000, 30 + i)[0] for i in range(2)]
    qs = [rand(i, 1, 4, 64, dtype=torch.bfloat16).cuda() for i in range(2)]
    pos = [ints([5999]), ints([3000])]
    want = [caches[i].attend(qs[i], pos[i]) for i in range(2)]
    got, errors = [[], []], []

    def calls(i):
        try:
            for _ in range(300):
                got[i].append(caches[i].attend(qs[i], pos[i]))
        except Exception as e:
            errors.append(e)

    threads = [threading.Thread(target=calls, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not errors and all(len(g) == 300 for g in got)
    for i in range(2):
        assert all(torch.equal(y, want[i]) for y in got[i])

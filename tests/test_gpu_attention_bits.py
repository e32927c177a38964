"""How many bits the packed attention and the attention over the 4-bit cache keep, against their definitions in 64 bits: in fp32 element by element, the third
bf16 part of a value and the soft-cap's own accuracy included, in bf16 by the 2-norm, which tells one rounding of the probabilities from none and from a cut.

A value of 8 significant bits whose mantissa m is spread evenly over its logarithm is off by 2^-8 / sqrt(3) / m in the mean, evenly to both sides, and the mean of
1 / m^2 over 1 .. 2 is 3 / (8 ln 2): SIGMA of itself.  Roundings are independent, so the squares of what they change add up: SIGMA^2 o^2 for an output's own and
SIGMA^2 p_j^2 v_j^2 for each probability that goes into the second product as one bf16 value.  Over tens of thousands of outputs the 2-norm leaves its mean by a
percent; the margin is 15.  Probabilities cut off instead of rounded would be off by twice that in the mean and to one side, which is 1.5 times the norm."""
import math

import pytest
import torch

from attention_reference import Ring

pytestmark = pytest.mark.gpu
SIGMA = 2.0 ** -8 / math.sqrt(3) * math.sqrt(3 / (8 * math.log(2)))
MARGIN = 1.15


@pytest.fixture(scope="module")
def fs():
    import flash_stu
    from flash_stu import _hip
    _hip.load()
    return flash_stu


def rand(seed, *shape, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * torch.exp(0.5 * torch.randn(1, *shape[1:], generator=g))).to(dtype)


def ints(x):
    return torch.tensor(list(x), dtype=torch.int32, device="cuda")


def slopes_of(heads):
    return 0.25 * 2.0 ** (-8.0 * (torch.arange(heads) + 1) / heads)


def head(q, k, v, far, slope, softcap):
    """One query head in 64 bits: (o, sum of p_j^2 v_j^2, how far fp32 arithmetic may be from o, the mean square of how far it is).  far: how far behind a query
    a key is, negative where unseen.

    A score in fp32 is off by (hd + 16) * 2^-23 of its products' sizes (each product and each sum 2^-24 of a partial sum, and as much again for what is left of
    a value in three bf16 parts), by 2^-22 of itself and of ALiBi's term (scale, argument, product, difference), and by 2^-21 of itself from tanh (a quotient of
    polynomials or 1 - 2 / (exp(2x) + 1) where that is over a half: six roundings and a reciprocal of one bit); a probability by that, by 2^-22 * (1 + |s - max|)
    for its exp, and by 2^-23 where it goes in three bf16 parts (8 bits each, the last one rounded).

    In the mean these add up as squares, a rounding being 2^-48 / 3 of its operand's: hd + 16 of them to a score, of partial sums whose square is that of the
    products together; 8 of the score, 4 of 1 + |s - max| and 4 of ALiBi's term; one for each 8 keys and 16 more of the output, whose partial sums are as large as
    itself or the root of its terms' squares."""
    hd = q.shape[1]
    raw, size = q @ k.t() * hd ** -0.5, q.abs() @ k.abs().t() * hd ** -0.5
    s = softcap * torch.tanh(raw / softcap) if softcap else raw
    off = (hd + 16) * 2.0 ** -23 * size + 2.0 ** -22 * (raw.abs() + slope * far.abs()) + (2.0 ** -21 * s.abs() if softcap else 0.0)
    s = (s - slope * far).masked_fill(far < 0, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True)
    off = torch.where(far < 0, 0.0, off + 2.0 ** -22 * (1 + (s - top).abs()) + 2.0 ** -23)
    o = p @ v
    sums = (2 * k.shape[0] + 16) * 2.0 ** -24
    bound = 1.01 * ((p * off) @ v.abs() + (p * off).sum(-1, keepdim=True) * o.abs()) + sums * (p @ v.abs() + o.abs())
    e = (hd + 16) * (q.square() @ k.square().t()) / hd + 8 * raw.square() + 4 * (1 + (s - top).abs()).square() + 4 * (slope * far).square()
    e = p.square() * torch.where(far < 0, 0.0, e)
    squares = p.square() @ v.square()
    mean = 2.0 ** -48 / 3 * (e @ v.square() + e.sum(-1, keepdim=True) * o.square() + (k.shape[0] / 8 + 16) * (o.square() + squares))
    return o, squares, bound, mean


def packed(q, k, v, lengths, slopes, window, softcap, heads):
    """The same of packed prompts for these query heads."""
    group, got = q.shape[1] // k.shape[1], []
    for h in heads:
        a = 0
        for n in lengths:
            far = torch.arange(n)[:, None] - torch.arange(n)
            far = torch.where((far >= 0) & (far <= (n if window is None else window)), far, -1).double()
            rows = slice(a, a + n)
            got.append(head(q[rows, h].double(), k[rows, h // group].double(), v[rows, h // group].double(), far, 0.0 if slopes is None else float(slopes[h]), softcap))
            a += n
    return [torch.cat(x).view(len(heads), sum(lengths), -1).transpose(0, 1) for x in zip(*got)]


def off_in_norm(y, o, squares):
    """The error's 2-norm over what the roundings make of it."""
    return float((y.cpu().double() - o).norm() / (SIGMA * (o.square() + squares).sum().sqrt()))


def keeps_fp32(y, o, squares, bound, mean):
    """Each output to within its bound, all of them together to what roundings make in the mean (queries in two bf16 parts: 1.6 to 3 times that)."""
    off = y.cpu().double() - o
    worst = (off.abs() - 2.0 ** -24 * (o.abs() + bound)) / bound
    assert float(worst.max()) <= 1, float(worst.max())
    assert float(off.norm()) <= MARGIN * float(mean.sum().sqrt()), float(off.norm() / mean.sum().sqrt())


FORMS = [
    (12, 12, 64, [700, 513, 90], 512, 50.0, True),          # partners for half of the keys
    (64, 8, 64, [1700, 33], 1000, 30.0, False),             # four waves
    (16, 4, 128, [1300, 400], None, 0.0, False),
    (64, 8, 128, [1300, 33], 300, 50.0, True),
    (2, 1, 128, [4500], None, 0.0, False),                  # eight waves
    (8, 2, 256, [900, 300], None, 50.0, True),
    (12, 4, 32, [800, 601], 256, 0.0, True),
]


@pytest.mark.parametrize("fine", [False, True])
@pytest.mark.parametrize("heads,kvh,hd,lengths,window,softcap,alibi", FORMS)
def test_packed_prompts_round_each_probability_once_or_not_at_all(fs, heads, kvh, hd, lengths, window, softcap, alibi, fine):
    x = rand(1, sum(lengths), heads + 2 * kvh, hd, dtype=torch.bfloat16)
    q, k, v = x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:]
    slopes, d, some = slopes_of(heads) if alibi else None, x.cuda(), [0, heads - 1]
    cu = ints([0] + list(torch.tensor(lengths).cumsum(0)))
    y = fs.swa_packed(d[:, :heads], d[:, heads:heads + kvh], d[:, heads + kvh:], cu, slopes=None if slopes is None else slopes.cuda(), window=window, softcap=softcap,
                      fine=fine)
    o, squares, _, _ = packed(q, k, v, lengths, slopes, window, softcap, some)
    assert off_in_norm(y[:, some], o, 0 * squares if fine else squares) <= MARGIN


def test_prompts_of_one_length_keep_more_in_the_layers_own_attention(fs):
    """swa_prefill holds a probability in two bf16 parts: of its error only the output's own rounding is left.  swa_packed does that where it is asked to."""
    from flash_stu import _hip
    heads, hd, T, window = 4, 64, 512, 300
    x, slopes = rand(2, 2 * T, 3 * heads, hd, dtype=torch.bfloat16), slopes_of(heads)
    q, k, v = x[:, :heads], x[:, heads:2 * heads], x[:, 2 * heads:]
    o, squares, _, _ = packed(q, k, v, [T, T], slopes, window, 50.0, range(heads))
    d = x.cuda()
    layer = _hip.swa_prefill(d.reshape(2, T, 3 * heads * hd), slopes.cuda(), heads, window, 50.0).view(2 * T, heads, hd)
    once, fine = (fs.swa_packed(d[:, :heads], d[:, heads:2 * heads], d[:, 2 * heads:], ints([0, T, 2 * T]), slopes=slopes.cuda(), window=window, softcap=50.0, fine=f)
                  for f in (False, True))
    none = torch.zeros(1)
    assert off_in_norm(layer, o, none) <= MARGIN and off_in_norm(fine, o, none) <= MARGIN
    assert off_in_norm(once, o, squares) <= MARGIN and off_in_norm(fine, o, none) < off_in_norm(once, o, none)
    # what is left between the two is outputs next to the middle of two bf16 values
    assert float((layer.double() - fine.double()).norm()) < 0.5 * float((layer.double() - once.double()).norm())


ATTENDS = [
    (24, 8, 2, 64, 513, None, 50.0),
    (40, 12, 12, 64, 300, 255, 0.0),
    (4, 32, 4, 128, 2500, None, 50.0),           # in parts
    (16, 16, 4, 128, 700, 600, 50.0),
    (3, 18, 2, 256, 1000, None, 0.0),
    (30, 8, 8, 32, 400, None, 50.0),
]


def attended(fs, batch, heads, kvh, hd, cap, window, softcap, dtype, size=1.0, alibi=True):
    n = min(cap, 2500)
    k, v = rand(3, batch * n, kvh, hd), rand(4, batch * n, kvh, hd)
    cache, ring = fs.KV4Cache(batch, kvh, hd, cap), Ring(batch, kvh, hd, cap)
    start, lengths = [cap - n + 7 * s for s in range(batch)], [n] * batch
    cache.write(k.cuda(), v.cuda(), ints(start), ints(range(0, batch * n + 1, n)))
    ring.write(k, v, start, lengths)
    q, slopes = rand(5, batch, heads, hd, dtype=dtype) * size, slopes_of(heads) * alibi
    pos = [a + n - 1 for a in start]
    y = cache.attend(q.cuda(), ints(pos), slopes=slopes.cuda(), window=window, softcap=softcap)
    parts = []
    for s, p in enumerate(pos):
        j = torch.arange(max(0, p - (cap - 1 if window is None else window)), p + 1)
        for h in range(heads):
            kj, vj = (x[s, j % cap, h // (heads // kvh)] for x in (ring.k, ring.v))
            parts.append(head(q[s, h].double()[None], kj, vj, (p - j)[None].double(), float(slopes[h]), softcap))
    return y, *(torch.cat(x).view(batch, heads, hd) for x in zip(*parts))


@pytest.mark.parametrize("splits", [None, 7, 100])
@pytest.mark.parametrize("batch,heads,kvh,hd,cap,window,softcap", ATTENDS)
def test_attend_in_fp32_keeps_fp32(fs, monkeypatch, batch, heads, kvh, hd, cap, window, softcap, splits):
    from flash_stu import _hip
    if splits:
        monkeypatch.setattr(_hip, "_kv4_splits", lambda *a: (splits, _hip.load().fstu_kv4_attend_ws(*a[:4], splits)))
    keeps_fp32(*attended(fs, batch, heads, kvh, hd, cap, window, softcap, torch.float32))


@pytest.mark.parametrize("batch,heads,kvh,hd,cap,window,softcap", ATTENDS)
def test_attend_in_fp32_keeps_its_probabilities(fs, batch, heads, kvh, hd, cap, window, softcap):
    """Scores near zero, so that little but the probabilities' own error is left: in two bf16 parts instead of three they would be off by 2 to 5 times the mean."""
    keeps_fp32(*attended(fs, batch, heads, kvh, hd, cap, window, softcap, torch.float32, size=2.0 ** -6, alibi=False))


@pytest.mark.parametrize("batch,heads,kvh,hd,cap,window,softcap", ATTENDS)
def test_attend_in_bf16_rounds_its_output_alone(fs, batch, heads, kvh, hd, cap, window, softcap):
    y, o, _, _, _ = attended(fs, batch, heads, kvh, hd, cap, window, softcap, torch.bfloat16)
    assert off_in_norm(y, o, torch.zeros(1)) <= MARGIN


@pytest.mark.parametrize("heads,kvh,hd,lengths,window,softcap,alibi", FORMS)
def test_packed_prompts_in_fp32_keep_fp32(fs, heads, kvh, hd, lengths, window, softcap, alibi):
    x = rand(6, sum(lengths), heads + 2 * kvh, hd)
    slopes, d, some = slopes_of(heads) if alibi else None, x.cuda(), [0, heads - 1]
    cu = ints([0] + list(torch.tensor(lengths).cumsum(0)))
    y = fs.swa_packed(d[:, :heads], d[:, heads:heads + kvh], d[:, heads + kvh:], cu, slopes=None if slopes is None else slopes.cuda(), window=window, softcap=softcap)
    keeps_fp32(y[:, some], *packed(x[:, :heads], x[:, heads:heads + kvh], x[:, heads + kvh:], lengths, slopes, window, softcap, some))


@pytest.mark.parametrize("kind", ["packed", "attend"])
def test_small_scores_under_a_soft_cap_in_fp32(fs, kind):
    """A score of 0.13 under a soft-cap of 50: tanh's error counts against the score and not against the cap, 2^-20 of which is ten times as much as is allowed."""
    hd, n, softcap = 64, 16, 50.0
    # the last of 16 keys has that score and the others zero; its value is 1 and theirs 0, so that the output is its weight
    k, v, q = torch.zeros(n, 1, hd), torch.zeros(n, 1, hd), torch.zeros(n, 1, hd)
    q[:, 0, 0], k[n - 1, 0, 0], v[n - 1, 0] = 1.0, 1.0, 1.0
    q[n - 1, 0, 0] = 0.375 * 8 ** 0.5
    if kind == "packed":
        y = fs.swa_packed(q.cuda(), k.cuda(), v.cuda(), ints([0, n]), softcap=softcap)[-1, 0]
    else:
        cache = fs.KV4Cache(1, 1, hd, n)
        cache.write(k.cuda(), v.cuda(), ints([0]), ints([0, n]))
        y = cache.attend(q[-1:].cuda(), ints([n - 1]), softcap=softcap)[0, 0]
    s = softcap * math.tanh(float(q[n - 1, 0, 0]) * hd ** -0.5 / softcap)
    w = math.exp(s) / (math.exp(s) + n - 1)
    # a score is off by 2^-21 of itself and less, a weight's exp by 2^-22 (1 + s), in numerator and sum; 16 weights are added up
    off = 2.0 ** -20 * (1 + s) + (2 * n + 16) * 2.0 ** -24
    assert float((y.cpu().double() - w).abs().max()) <= w * off

"""The definitions of the packed attention and of the 4-bit ring cache in 64 bits on the CPU, and how far fp32 arithmetic may be from them."""
import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def held(x):
    """What the cache holds of x (..., head_dim), in 64 bits: 32 values share 2^e, the smallest with amax <= 7 * 2^e, -120 <= e <= 125."""
    v = x.detach().cpu().double().unflatten(-1, (-1, 32))
    most = v.abs().amax(-1, keepdim=True)
    e = torch.full_like(most, -120.0)
    for _ in range(245):
        e = torch.where((most > 7.0 * torch.exp2(e)) & (e < 125), e + 1, e)
    a = (v / torch.exp2(e)).nan_to_num(0.0, 0.0, 0.0)
    size = a.abs().clamp_max(6.0)
    below = (torch.searchsorted(GRID, size, right=True) - 1).clamp(0, 6)
    lo, hi = GRID[below], GRID[below + 1]
    up = (size - lo > hi - size) | ((size - lo == hi - size) & (below % 2 == 1))
    y = torch.copysign(torch.where(up, hi, lo), a) * torch.exp2(e)
    y = torch.where(torch.isfinite(v).all(-1, keepdim=True), y, math.nan)
    return y.flatten(-2)


def attention(q, k, v, far, slope, softcap, p_step):
    """(o, bound) of one query head: q (n, hd), k, v (m, hd) in 64 bits, far (n, m) how far behind its query a key is, negative where it is not seen.

    In fp32 a score is off by (hd + 16) * 2^-23 of the sum of its products' sizes (each product and addition 2^-24 at most of a partial sum, twice
    that where a value goes in three bf16 parts), 2^-22 of itself (the scale, the soft-cap's argument, ALiBi's product and its difference), and, capped, by
    2^-20 * softcap (1 - 2 / (exp(2x) + 1) on the hardware's exp and reciprocal: the reciprocal's, the exp's and the difference's last bit, 2^-22 each), from soft-caps
    of 512 on by 2^-18 of itself instead (a series where x < 0.25, and 2^-20 of softcap is 2^-18 of what is larger); a probability by that, by 2^-22 * (1 + |s - max|) for its
    exp, and by p_step where it is cut to bf16 parts.  A probability's error e_j changes the output by p_j e_j (|v_j| + |o|) at most.  Sums over m keys and
    their rescaling: (2 m + 16) * 2^-24 of the sum of sizes, for numerator and denominator."""
    hd = q.shape[1]
    raw = q @ k.t() * hd ** -0.5
    size = q.abs() @ k.abs().t() * hd ** -0.5
    s = softcap * torch.tanh(raw / softcap) if softcap else raw
    off = (hd + 16) * 2.0 ** -23 * size + 2.0 ** -22 * (raw.abs() + slope * far.abs()) + (2.0 ** -20 * softcap if 0 < softcap <= 512 else 2.0 ** -18 * s.abs() if softcap else 0.0)
    s = (s - slope * far).masked_fill(far < 0, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    p = p / p.sum(-1, keepdim=True)
    p = torch.where(far < 0, 0.0, p)
    off = torch.where(far < 0, 0.0, off + 2.0 ** -22 * (1 + (s - top).abs()) + p_step)
    o = p @ v
    sums = (2 * k.shape[0] + 16) * 2.0 ** -24
    bound = 1.01 * ((p * off) @ v.abs() + (p * off).sum(-1, keepdim=True) * o.abs()) + sums * (p @ v.abs() + o.abs())
    return o, bound


def check(y, o, bound, dtype, p_step=0.0):
    """y is o to within bound and one rounding to its type, and in bf16 all of it together to twice the roundings' 2-norm."""
    off = (y.detach().cpu().double() - o).abs()
    assert bool(torch.isfinite(y).all())
    worst = off - bound - torch.finfo(dtype).eps / 2 * (o.abs() + bound) - 1e-40
    assert bool((worst <= 0).all()), (float(worst.max()), float(off.max()))


def packed(q, k, v, lengths, slopes, window, softcap, p_step):
    """(o, bound) of packed prompts, rows of no sequence zero."""
    q, k, v = (x.detach().cpu().double() for x in (q, k, v))
    rows, heads, hd = q.shape
    group = heads // k.shape[1]
    o, bound, a = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64), 0
    for n in lengths:
        if n:
            i = torch.arange(n)
            far = i[:, None] - i
            far = torch.where((far >= 0) & (far <= (n if window is None else window)), far, -1).double()
            for h in range(heads):
                kv = [x[a:a + n, h // group] for x in (k, v)]
                o[a:a + n, h], bound[a:a + n, h] = attention(q[a:a + n, h], *kv, far, 0.0 if slopes is None else float(slopes[h]), softcap, p_step)
        a += n
    return o, bound


class Ring:
    """The cache's definition: a dict of positions' values by slot."""

    def __init__(self, batch, kv_heads, head_dim, capacity):
        self.k = torch.zeros(batch, capacity, kv_heads, head_dim, dtype=torch.float64)
        self.v = torch.zeros_like(self.k)
        self.capacity = capacity

    def write(self, k, v, pos, lengths=None):
        k, v, row = held(k), held(v), 0
        for s, n in enumerate([1] * len(pos) if lengths is None else lengths):
            for t in range(n):
                if pos[s] >= 0:
                    self.k[s, (pos[s] + t) % self.capacity] = k[row + t]
                    self.v[s, (pos[s] + t) % self.capacity] = v[row + t]
            row += n

    def attend(self, q, pos, slopes, window, softcap, p_step):
        q = q.detach().cpu().double()
        batch, heads, hd = q.shape
        group = heads // self.k.shape[2]
        o, bound = torch.zeros(q.shape, dtype=torch.float64), torch.zeros(q.shape, dtype=torch.float64)
        for s in range(batch):
            if pos[s] < 0:
                continue
            j = torch.arange(max(0, pos[s] - (self.capacity - 1 if window is None else window)), pos[s] + 1)
            far = (pos[s] - j)[None].double()
            for h in range(heads):
                k, v = (x[s, j % self.capacity, h // group] for x in (self.k, self.v))
                a, b = attention(q[s, h][None], k, v, far, 0.0 if slopes is None else float(slopes[h]), softcap, p_step)
                o[s, h], bound[s, h] = a[0], b[0]
        return o, bound

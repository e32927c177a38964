"""What the packed attention and the 4-bit cache refuse, without a GPU: at the C entry points before any launch, and in the Python calls."""
import ctypes
import math

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flash_stu import _hip
    return _hip.load()


@pytest.fixture(scope="module")
def mem():
    buf = (ctypes.c_char * (1 << 16))()
    return (ctypes.addressof(buf) + 63) // 64 * 64, buf


def why(lib):
    return lib.fstu_last_error().decode()


def test_bytes(lib):
    assert lib.fstu_kv4_bytes(1, 1, 32, 1) == 32 * 34 and lib.fstu_kv4_bytes(3, 2, 128, 33) == 3 * 2 * 64 * (128 + 8)
    assert lib.fstu_kv4_bytes(64, 16, 256, 1 << 20) == 64 * 16 * 272 << 20


def test_cache_entry_points_refuse(lib, mem):
    p = mem[0]

    def write(k=p, kr=128, kh=64, v=p, c=p, pos=p, cu=p, rows=2, seqs=2, kvh=2, hd=64, cap=8, dt=1):
        return lib.fstu_kv4_write(k, kr, kh, v, 128, 64, c, pos, cu, rows, seqs, kvh, hd, cap, dt, None)

    def read(c=p, k=p, v=p, pos=p, cu=p, rows=2, seqs=2, kvh=2, hd=64, cap=8, dt=1):
        return lib.fstu_kv4_read(c, k, v, pos, cu, rows, seqs, kvh, hd, cap, dt, None)

    for f in (write, read):
        assert f(k=None) == -1 and f(v=None) == -1 and f(c=None) == -1 and f(pos=None) == -1 and "null" in why(lib)
        assert f(hd=48) == -3 and f(hd=0) == -3 and f(seqs=0) == -3 and f(kvh=0) == -3 and f(cap=0) == -3 and f(cap=(1 << 30) + 1) == -3
        assert f(rows=1 << 29, kvh=64, hd=256) == -3 and "launch" in why(lib)
        assert f(rows=-1) == -5 and f(cu=None, rows=3) == -5 and "rows" in why(lib)
        assert f(c=p + 8) == -4 and f(k=p + 2) == -4 and f(v=p + 8) == -4
        assert f(dt=7) == -2
        assert f(rows=0) == 0
    assert write(kr=100) == -4 and write(kh=33) == -4 and write(kr=-128) == -4

    def attend(q=p, qr=256, qh=64, c=p + 8192, out=p + 4096, pos=p, slopes=None, seqs=2, heads=4, kvh=2, hd=64, cap=8, window=7, softcap=0.0, dt=1, splits=1,
               ws=None):
        return lib.fstu_kv4_attend(q, qr, qh, c, out, ws, splits, pos, slopes, seqs, heads, kvh, hd, cap, window, softcap, dt, None)

    assert attend(q=None) == -1 and attend(c=None) == -1 and attend(out=None) == -1 and attend(pos=None) == -1
    assert attend(hd=96) == -3 and attend(heads=3) == -3 and attend(heads=0) == -3 and attend(seqs=65536) == -3 and attend(cap=0) == -3
    assert attend(window=8) == -5 and attend(window=-1) == -5 and "window" in why(lib)
    assert attend(softcap=-1.0) == -5 and attend(softcap=math.nan) == -5 and attend(softcap=math.inf) == -5 and attend(softcap=1e-13) == -5 and attend(softcap=2e12) == -5
    assert attend(seqs=60000, heads=256, out=p + (1 << 40), splits=1) == -3 and attend(seqs=4096, splits=64, ws=p, kvh=32, heads=32, out=p + (1 << 40)) == -3 and "launch" in why(lib)
    assert attend(q=p + 8) == -4 and attend(qr=100) == -4 and attend(qh=-64) == -4 and attend(out=p + 4096 + 4) == -4 and attend(c=p + 8200) == -4
    assert attend(out=p) == -5 and "overlaps" in why(lib)
    assert attend(out=p + 8192) == -5 and attend(out=p + 8192 + 2 * 2 * 32 * 68 - 16) == -5
    assert attend(dt=2) == -2
    assert attend(splits=0) == -5 and attend(splits=2) == -5 and attend(splits=70000, ws=p) == -5 and attend(splits=2, ws=p + 2) == -4
    assert lib.fstu_kv4_attend_splits(64, 8, 8, 64, 100, 99) == 1 and lib.fstu_kv4_attend_ws(64, 8, 8, 64, 1) == 0
    assert lib.fstu_kv4_attend_splits(1, 8, 8, 64, 1 << 20, (1 << 20) - 1) > 64 and lib.fstu_kv4_attend_ws(1, 9, 1, 64, 256) == (2 + 256) * 8 * 66


def test_step_entry_point_refuses(lib, mem):
    p = mem[0]

    def step(q=p, k=p + 2048, kr=128, kh=64, v=p + 2048, c=p + 8192, out=p + 4096, splits=1, ws=None, window=7, cap=40, dt=1):
        return lib.fstu_kv4_step(q, 256, 64, k, kr, kh, v, 128, 64, c, out, ws, splits, p, None, 2, 4, 2, 64, cap, window, 0.0, dt, None)

    assert step(k=None) == -1 and step(v=None) == -1 and step(q=None) == -1 and step(c=None) == -1
    assert step(window=40) == -5 and step(splits=2) == -5 and "fstu_kv4_step" in why(lib)
    assert step(k=p + 2056) == -4 and step(v=p + 2050) == -4 and step(kr=100) == -4 and step(kh=-64) == -4 and "of k and v" in why(lib)
    assert step(k=p + 4096) == -5 and step(v=p + 4096 + 512) == -5 and step(k=p + 8192) == -5 and "overlaps k or v" in why(lib)
    assert step(out=p) == -5 and "overlaps q" in why(lib)
    assert step(dt=2) == -2


def test_packed_entry_point_refuses(lib, mem):
    p = mem[0]

    def f(q=p, qr=256, qh=64, k=p, kr=128, kh=64, v=p, out=p + 8192, cu=p, rows=8, seqs=2, heads=4, kvh=2, hd=64, window=7, softcap=0.0, dt=1):
        return lib.fstu_swa_packed(q, qr, qh, k, kr, kh, v, 128, 64, out, cu, None, rows, seqs, heads, kvh, hd, window, softcap, dt, None)

    assert f(q=None) == -1 and f(k=None) == -1 and f(v=None) == -1 and f(out=None) == -1 and f(cu=None) == -1
    assert f(hd=80) == -3 and f(heads=5) == -3 and f(kvh=0) == -3 and f(rows=-1) == -3 and f(seqs=-1) == -3 and f(heads=0) == -3
    assert f(rows=(1 << 30) + 1) == -3 and f(rows=1 << 28, heads=8) == -3 and "launch" in why(lib) and f(kr=1 << 23) == -3
    assert f(window=-1) == -5 and f(softcap=-0.5) == -5 and f(softcap=math.nan) == -5 and f(softcap=math.inf) == -5
    assert f(q=p + 4) == -4 and f(k=p + 2) == -4 and f(v=p + 8) == -4 and f(out=p + 8196) == -4 and f(qr=257) == -4 and f(kh=60) == -4 and f(kr=-8) == -4
    assert f(out=p) == -5 and f(out=p + 256 * 7 * 2) == -5 and "overlaps" in why(lib)
    assert f(dt=3) == -2
    assert f(rows=0) == 0 and f(seqs=0) == 0


def test_the_calls_refuse_tensors_of_the_cpu():
    from flash_stu import KV4Cache, _hip, swa_packed
    q, k, cu = torch.zeros(4, 2, 64), torch.zeros(4, 1, 64), torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(_hip.FlashSTUHipError, match="no CPU fallback"):
        swa_packed(q, k, k, cu)
    with pytest.raises(_hip.FlashSTUHipError, match="no CPU fallback"):
        KV4Cache(1, 1, 64, 8, device="cpu")
    with pytest.raises(NotImplementedError, match="forward only"):
        swa_packed(q.requires_grad_(), k, k, cu)
    for bad in ((0, 1, 64, 8), (1, 1, 65, 8), (1, 1, 64, 0)):
        with pytest.raises(_hip.FlashSTUHipError, match="no cache"):
            KV4Cache(*bad)


def test_the_reference_of_the_tests():
    """The cache's definition by hand, and the attention's against torch's softmax."""
    from attention_reference import attention, held
    x = torch.zeros(4, 32)
    x[0, :4] = torch.tensor([7.0, 5.0, 0.25, -0.75])
    x[1, :4] = torch.tensor([7.1, 5.0, 0.5, -2.6])
    x[2, 0] = 2.0 ** -126
    x[3, 5] = math.inf
    y = held(x)
    assert y[0, :4].tolist() == [6.0, 4.0, 0.0, -1.0] and y[1, :4].tolist() == [8.0, 4.0, 0.0, -3.0] and not y[2].any() and bool(torch.isnan(y[3]).all())
    q, k, v = (torch.randn(5, 8, dtype=torch.float64) for _ in range(3))
    far = (torch.arange(5)[:, None] - torch.arange(5)).double().clamp_min(-1)
    o, bound = attention(q, k, v, far, 0.0, 0.0, 0.0)
    want = torch.nn.functional.scaled_dot_product_attention(q[None], k[None], v[None], is_causal=True)[0]
    assert torch.allclose(o, want) and bool((bound < 1e-4).all())


class OnGpu(torch.Tensor):
    """A tensor of the CPU that says it is on device 0."""

    def get_device(self):
        return 0


class Recorded:
    """A library whose attention entry points note the calls and answer what is asked of them; all else is the real one's."""

    def __init__(self, lib, seen, rc=0):
        self.lib, self.seen, self.rc = lib, seen, rc

    def __getattr__(self, name):
        if name.startswith(("fstu_kv4_attend", "fstu_kv4_step", "fstu_kv4_write")) and name not in ("fstu_kv4_attend_ws", "fstu_kv4_attend_splits"):
            return lambda *args: self.seen(name, args) or self.rc
        return getattr(self.lib, name)


def stand_in(monkeypatch, lib, seen, rc=0):
    """Calls of a cache without a GPU: (cache of 2 sequences, 1 key head of 64 and long rings, a maker of tensors)."""
    from flash_stu import KV4Cache, _hip
    monkeypatch.setattr(_hip, "load", lambda: Recorded(lib, seen, rc))
    monkeypatch.setattr(_hip, "_device_now", lambda: 0)
    monkeypatch.setattr(_hip, "raw_stream", lambda dev: 0)

    def on_gpu(*shape, dtype=torch.bfloat16):
        return torch.zeros(*shape, dtype=dtype).as_subclass(OnGpu)

    cache = object.__new__(KV4Cache)
    cache.batch, cache.kv_heads, cache.head_dim, cache.capacity = 2, 1, 64, 20000
    cache.data = on_gpu(lib.fstu_kv4_bytes(2, 1, 64, 20000), dtype=torch.uint8)
    return cache, on_gpu


@pytest.mark.parametrize("step", [False, True])
def test_the_parts_stay_this_calls_until_it_has_returned(lib, monkeypatch, step):
    """The library is called without the interpreter's lock: memory of the parts that the allocator had back by then could become another thread's."""
    import weakref

    from flash_stu import _hip
    given, held = [], []
    empty = _hip._empty

    def recorded(*args, **kw):
        x = empty(*args, **kw)
        if kw.get("dtype") is torch.float32:
            given.append((weakref.ref(x), x.data_ptr()))
        return x

    monkeypatch.setattr(_hip, "_empty", recorded)
    cache, on_gpu = stand_in(monkeypatch, lib, lambda name, args: held.append([name, [ref() is not None and at in args for ref, at in given]]))
    k = on_gpu(2, 1, 64)
    cache.attend(on_gpu(2, 4, 64), on_gpu(2, dtype=torch.int32), *((k, k) if step else ()))
    assert len(held) == 1 and held[0][0].startswith("fstu_kv4_step" if step else "fstu_kv4_attend") and held[0][1] == [True]


def test_tiles_past_31_bits_are_not_dealt(lib, mem):
    """The even deal counts all tiles of 32 slots of a call's key heads (and chunks of 8 query heads) in an int."""
    p, ring = mem[0], 1 << 30
    assert 1 <= lib.fstu_kv4_attend_splits(1, 512, 1, 32, ring, ring - 1) <= 64          # 64 chunks of 2^25 tiles
    assert lib.fstu_kv4_attend_splits(1, 504, 1, 32, ring, ring - 1) == 256              # 63
    assert 1 <= lib.fstu_kv4_attend_splits(64, 8, 1, 32, ring, ring - 1) <= 64

    def attend(heads, splits, window=ring - 1):
        return lib.fstu_kv4_attend(p, 32 * heads, 32, p + 8192, p + (1 << 40), p, splits, p, None, 1, heads, 1, 32, ring, window, 0.0, 1, None)

    assert attend(512, 256) == -3 and "launch" in why(lib)
    assert attend(512, 65535) == -3 and attend(8192, 65, window=(1 << 26) - 1) == -3


def test_a_refused_step_of_another_type_writes_nothing(lib, mem, monkeypatch):
    """k and v of another type than q go to the cache in a launch of their own: after everything that the attention refuses."""
    from flash_stu import _hip
    names = []
    cache, on_gpu = stand_in(monkeypatch, lib, lambda name, args: names.append(name), rc=-5)
    k = on_gpu(2, 1, 64, dtype=torch.float32)
    with pytest.raises(_hip.FlashSTUHipError):
        cache.attend(on_gpu(2, 4, 64), on_gpu(2, dtype=torch.int32), k, k)
    assert names == ["fstu_kv4_step_of"]

    p = mem[0]

    def step(q=p, dt=1, k=p + 2048, kr=128, kh=64, v=p + 2048, kv_dt=0, c=p + 16384, out=p + 4096, splits=1, ws=None, window=7, heads=4):
        return lib.fstu_kv4_step_of(q, 64 * heads, 64, dt, k, kr, kh, v, 128, 64, kv_dt, c, out, ws, splits, p, None, 2, heads, 2, 64, 40, window, 0.0, None)

    for other in (dict(dt=1, kv_dt=0), dict(dt=0, kv_dt=1)):
        assert step(k=None, **other) == -1 and step(window=40, **other) == -5 and step(splits=2, **other) == -5 and step(heads=3, **other) == -3
        assert step(out=p, **other) == -5 and "overlaps q" in why(lib)
        assert step(out=p + 16384, **other) == -5 and step(k=p + 4096, **other) == -5 and step(v=p + 16384, **other) == -5
        assert step(out=p + 4100, **other) == -4 and step(q=p + 2, **other) == -4 and step(k=p + 2056, **other) == -4
    assert step(dt=1, kv_dt=1, kr=68) == -4 and step(kv_dt=7) == -2 and step(dt=7) == -2 and step(kv_dt=7, splits=65, ws=p) == -2
    assert step(k=p + 4096 - 1008) == -5                                 # its end, by its own type's size: 1024 bytes


def test_a_batch_that_no_launch_attends_over_is_no_cache(lib, mem):
    from flash_stu import KV4Cache, _hip
    p = mem[0]
    for batch, kv_heads in ((65536, 1), (1 << 40, 1), (1, 65536), (65535, 129), (1 << 12, 1 << 11)):
        with pytest.raises(_hip.FlashSTUHipError, match="up to 65535"):
            KV4Cache(batch, kv_heads, 32, 4)
    for splits in (1, 64, 65):
        assert lib.fstu_kv4_attend(p, 64, 32, p + 8192, p + 4096, p, splits, p, None, 65536, 2, 1, 32, 4, 3, 0.0, 1, None) == -3
    assert lib.fstu_kv4_attend(p, 0, 32, p + 8192, p + 4096, p, 1, p, None, 1, 65536, 1, 32, 4, 3, 0.0, 1, None) == -3


def test_only_kernels_that_a_call_reaches_are_built(lib):
    """Of the packed prompts' bf16 kernels <head dim, waves of queries, waves to their keys, soft-cap, ALiBi, two parts of a probability>: four waves of queries (heads of 256: two) for all
    calls, eight for long documents of heads of 128, two with partners for few workgroups of heads up to 128, these two under ordinary soft-caps."""
    import re
    from flash_stu import _hip
    with open(_hip.LIB_PATH, "rb") as f:
        built = set(re.findall(rb"swa_packed_mfma_kernelILi(\d+)ELi(\d+)ELi(\d+)ELi(\d+)ELb([01])ELb([01])E", f.read()))
    forms = [(hd, 2 if hd == 256 else 4, 1, cap) for hd in (32, 64, 128, 256) for cap in (0, 1, 2)]
    forms += [(128, 8, 1, cap) for cap in (0, 1)] + [(hd, 2, 2, cap) for hd in (32, 64, 128) for cap in (0, 1)]
    assert built == {tuple(b"%d" % x for x in f + (bias, fine)) for f in forms for bias in (0, 1) for fine in (0, 1)}

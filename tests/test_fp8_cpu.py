"""What the 8-bit operators refuse, without a GPU: at the C entry points before any launch, and in the Python calls."""
import ctypes
import os
import subprocess
import sys

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from flash_stu import _hip
    return _hip.load()


@pytest.fixture(scope="module")
def mem():
    buf = (ctypes.c_char * 4096)()
    return (ctypes.addressof(buf) + 63) // 64 * 64, buf


def why(lib):
    return lib.fstu_last_error().decode()


def test_quantize_entry_points_refuse(lib, mem):
    p = mem[0]
    q = lambda x=p, ldx=128, c=p, ldc=128, s=p, rows=2, d=128, dt=1: lib.fstu_fp8_quantize_rows(x, ldx, c, ldc, s, 1, rows, rows, d, dt, None)
    assert q(x=None) == -1 and q(c=None) == -1 and q(s=None) == -1 and "null" in why(lib)
    assert q(rows=0) == -3 and q(d=0) == -3 and q(ldx=127) == -3
    assert q(c=p + 8) == -4 and q(ldc=136) == -4 and q(ldc=112) == -4 and "16" in why(lib)
    assert q(dt=7) == -2
    w = lambda x=p, ldx=128, c=p, ldc=128, s=p, n=2, k=128, dt=1: lib.fstu_fp8_quantize_weight(x, ldx, c, ldc, s, 1, 1, n, k, dt, None)
    assert w(x=None) == -1 and w(n=0) == -3 and w(k=0) == -3 and w(ldx=100) == -3 and w(c=p + 1) == -4 and w(ldc=120) == -4 and w(dt=2) == -2
    assert w(n=65535 * 128 + 1) == -3


def test_norm_entry_point_refuses(lib, mem):
    p = mem[0]
    f = lambda x=p, ldx=64, de=None, ldd=64, xo=None, ldo=64, w=p, c=p, ldc=64, s=p, rows=2, d=64, dt=1: lib.fstu_fp8_rmsnorm(
        x, ldx, de, ldd, xo, ldo, w, 1e-6, c, ldc, s, 1, rows, rows, d, dt, None)
    assert f(x=None) == -1 and f(w=None) == -1 and f(c=None) == -1 and f(s=None) == -1
    assert f(de=p) == -5 and f(xo=p) == -5 and "together" in why(lib)
    assert f(rows=0) == -3 and f(d=0) == -3 and f(d=32769, ldx=40000, ldc=40000) == -3 and f(ldx=63) == -3
    assert f(de=p, xo=p, ldd=63) == -3 and f(de=p, xo=p, ldo=63) == -3
    assert f(c=p + 4) == -4 and f(ldc=72) == -4 and f(dt=3) == -2


def test_product_entry_points_refuse(lib, mem):
    p = mem[0]

    def lin(x=p, ldx=128, xs=p, w=p, ldw=128, ws=p, b=None, r=None, ldr=8, y=p, ldy=8, M=2, N=8, K=128, dt=1, part=None, slices=1):
        return lib.fstu_fp8_linear(x, ldx, xs, 1, 2, w, ldw, ws, 1, 1, b, r, ldr, y, ldy, M, N, K, dt, part, slices, None)
    assert lin(x=None) == -1 and lin(xs=None) == -1 and lin(w=None) == -1 and lin(ws=None) == -1 and lin(y=None) == -1
    assert lin(M=0) == -3 and lin(N=0) == -3 and lin(K=0) == -3 and lin(ldy=7) == -3 and lin(r=p, ldr=7) == -3
    assert lin(x=p + 8) == -4 and lin(w=p + 4) == -4 and lin(ldx=136) == -4 and lin(ldw=112) == -4 and lin(ldx=112) == -4
    assert "16-byte" in why(lib) and lin(dt=9) == -2
    assert lin(slices=0) == -5 and lin(slices=2, part=p + 4, K=256, ldx=256, ldw=256) == -5 and lin(slices=2, K=256, ldx=256, ldw=256) == -5 and lin(slices=2, part=p) == -5 and "slices=2" in why(lib)

    def glu(x=p, ldx=128, xs=p, g=p, ldg=128, gs=p, u=p, ldu=128, us=p, y=p, ldy=16, s=None, M=2, N=16, K=128, dt=1):
        return lib.fstu_fp8_glu(x, ldx, xs, 1, 2, g, ldg, gs, 1, 1, u, ldu, us, 1, 1, y, ldy, s, 1, 2, M, N, K, dt, None)
    assert glu(x=None) == -1 and glu(g=None) == -1 and glu(us=None) == -1 and glu(y=None) == -1
    assert glu(M=0) == -3 and glu(N=0) == -3 and glu(K=0) == -3 and glu(ldy=15) == -3
    assert glu(u=p + 1) == -4 and glu(ldg=120) == -4 and glu(s=p, y=p + 8) == -4 and glu(s=p, ldy=24) == -4
    assert glu(s=p, dt=0) == -2 and glu(dt=5) == -2


def test_python_calls_refuse_what_is_not_on_the_gpu():
    import flash_stu as fs
    from flash_stu._hip import FlashSTUHipError
    x, w = torch.zeros(2, 128), torch.zeros(16, 128)
    c, s = torch.zeros(2, 128).to(torch.float8_e4m3fn), torch.zeros(2, 1)
    for call in (lambda: fs.quantize_fp8(x), lambda: fs.quantize_weight_fp8(w), lambda: fs.rms_norm_fp8(x, torch.ones(128), 1e-6),
                 lambda: fs.linear_fp8(c, s, c, s), lambda: fs.glu_fp8(c, s, c, s, c, s)):
        with pytest.raises(FlashSTUHipError, match="not on the GPU"):
            call()


def test_what_overlaps_otherwise_than_as_a_whole_is_refused(lib, mem):
    """Refusals only: a call that passes the check would be launched."""
    p = mem[0]
    f = lambda xo, ldo=64, de=p + 2048, rows=2, dt=1: lib.fstu_fp8_rmsnorm(p, 64, de, 64, xo, ldo, p, 1e-6, p, 64, p, 1, 2, rows, 64, dt, None)
    assert f(p + 2) == -5 and f(p + 128) == -5 and f(p + 2050) == -5 and "overlaps" in why(lib)
    assert f(p, ldo=65) == -5 and f(p + 2, rows=1) == -5 and f(p + 256, dt=0) == -5
    g = lambda r, ldr, y=p, ldy=20, M=2, N=8: lib.fstu_fp8_linear(p, 128, p, 1, 2, p, 128, p, 1, 1, None, r, ldr, y, ldy, M, N, 128, 1, None, 1, None)
    assert g(p, 21) == -5 and g(p + 2, 20) == -5 and g(p + 14, 20) == -5 and g(p + 40, 20) == -5 and g(p + 26, 20) == -5 and g(p + 14, 20, M=1) == -5
    assert "overlaps" in why(lib)


def test_sizes_beyond_a_launch_are_refused(lib, mem):
    p = mem[0]
    assert lib.fstu_fp8_quantize_rows(p, 1 << 20, p, 1 << 20, p, 1, 1, 1 << 18, 1 << 20, 1, None) == -3
    assert lib.fstu_fp8_rmsnorm(p, 32768, None, 0, None, 0, p, 1e-6, p, 32768, p, 1, 1, 1 << 22, 32768, 1, None) == -3
    for M, N, K in ((65535 * 64 + 1, 8, 128), (1, (1 << 26) + 1, 128), (1 << 20, 1 << 20, 128), (1, 8, (1 << 30) + 1)):
        ld = (K + 15) & -16
        assert lib.fstu_fp8_linear(p, ld, p, 1, 1, p, ld, p, 1, 1, None, None, 0, p, N, M, N, K, 1, None, 1, None) == -3
        assert lib.fstu_fp8_glu(p, ld, p, 1, 1, p, ld, p, 1, 1, p, ld, p, 1, 1, p, N, None, 1, 1, M, N, K, 1, None) == -3
    assert lib.fstu_fp8_linear(p, 256, p, 1, 1, p, 256, p, 1, 1, None, None, 0, p, 1 << 16, 1 << 15, 1 << 16, 256, 1, p, 2, None) == -5


@pytest.mark.gpu
def test_python_calls_refuse_what_does_not_go_together():
    import flash_stu as fs
    from flash_stu._hip import FlashSTUHipError
    g = dict(device="cuda")
    f8 = lambda *n: torch.zeros(*n, **g).to(torch.float8_e4m3fn)
    x, c, s, w, ws = torch.zeros(4, 256, **g), f8(4, 256), torch.ones(4, 2, **g), f8(130, 256), torch.ones(2, 2, **g)

    def refused(call, what):
        with pytest.raises(FlashSTUHipError, match=what):
            call()
    refused(lambda: fs.quantize_fp8(x.half()), "unsupported dtype")
    refused(lambda: fs.quantize_fp8(x.t()), "dense rows")
    refused(lambda: fs.quantize_fp8(x[0]), "2-D")
    refused(lambda: fs.quantize_fp8(x[:1].expand(4, 256)), "ldx=0")
    refused(lambda: fs.quantize_fp8(torch.zeros(4, 0, **g)), "dense rows")
    refused(lambda: fs.quantize_weight_fp8(torch.zeros(0, 4, **g)), "must have rows")
    refused(lambda: fs.rms_norm_fp8(x, torch.ones(255, **g), 1e-6), "weight must be")
    refused(lambda: fs.rms_norm_fp8(x, torch.ones(256, **g).bfloat16(), 1e-6), "weight must be")
    refused(lambda: fs.rms_norm_fp8(x, torch.ones(256, **g), 1e-6, delta=torch.zeros(4, 255, **g)), "delta must be")
    refused(lambda: fs.rms_norm_fp8(x, torch.ones(256, **g), 1e-6, x_out=x), "needs delta")
    refused(lambda: fs.rms_norm_fp8(x, torch.ones(256, **g), 1e-6, delta=x, x_out=x.bfloat16()), "x_out must be")
    refused(lambda: fs.rms_norm_fp8(torch.zeros(2, 32769, **g), torch.ones(32769, **g), 1e-6), "32768")
    refused(lambda: fs.linear_fp8(c.view(torch.uint8), s, w, ws), "float8_e4m3fn")
    refused(lambda: fs.linear_fp8(c, s.double(), w, ws), "float32")
    refused(lambda: fs.linear_fp8(c, s[:3], w, ws), "scales must be")
    refused(lambda: fs.linear_fp8(c, s, w, ws[:1]), "scales must be")
    refused(lambda: fs.linear_fp8(c, s, w[:, :128], ws[:, :1]), "do not go together")
    refused(lambda: fs.linear_fp8(c[:, 8:136], s[:, :1], w[:, :128], ws[:, :1]), "16-byte")
    refused(lambda: fs.linear_fp8(c, s, w, ws, bias=torch.zeros(129, **g)), "bias must be")
    refused(lambda: fs.linear_fp8(c, s, w, ws, residual=torch.zeros(4, 129, **g)), "residual must be")
    refused(lambda: fs.linear_fp8(c, s, w, ws, residual=torch.zeros(4, 130, **g), dtype=torch.bfloat16), "residual must be")
    refused(lambda: fs.linear_fp8(c, s, w, ws, out=torch.zeros(130, 4, **g).t()), "out must be")
    refused(lambda: fs.linear_fp8(c, s, w, ws, out=torch.zeros(1, 130, **g).expand(4, 130)), "ldy=0")
    refused(lambda: fs.linear_fp8(c, s, w, ws, dtype=torch.float16), "unsupported dtype")
    refused(lambda: fs.glu_fp8(c, s, w, ws, w[:129], ws), "do not go together")
    refused(lambda: fs.glu_fp8(c, s, w, ws, w, ws, dtype=torch.float32, quantize=True), "unsupported dtype")
    refused(lambda: fs.glu_fp8(c, s, w, ws.cpu(), w, ws), "not on the GPU")


def test_a_torch_without_gpu_bindings_imports_the_package():
    """And is told by each call that its tensors are not on the GPU."""
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import flash_stu as fs
x = torch.zeros(2, 128)
c, s = x.to(torch.float8_e4m3fn), torch.zeros(2, 1)
for call in (lambda: fs.quantize_fp8(x), lambda: fs.quantize_weight_fp8(x), lambda: fs.rms_norm_fp8(x, torch.ones(128), 1e-6),
             lambda: fs.linear_fp8(c, s, c, s[:1]), lambda: fs.glu_fp8(c, s, c, s[:1], c, s[:1])):
    try:
        call()
        raise SystemExit("not refused")
    except RuntimeError as e:
        assert "not on the GPU" in str(e), e
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    found = subprocess.run([sys.executable, "-c", code], env=dict(os.environ, PYTHONPATH=os.path.join(root, "flash-stu-2_amd")), capture_output=True, text=True)
    assert found.returncode == 0, found.stderr + found.stdout


def parts_without_a_gpu(monkeypatch, d=72, scale=3):
    """An FP8MLP on the CPU: codes and scales from the definition, where the module asks the kernels for them."""
    import flash_stu as fs
    from flash_stu import _hip
    from flash_stu.config import FlashSTUConfig
    from flash_stu.modules import MLP, RMSNorm

    def codes(w):
        n, k = w.shape
        held = torch.zeros(n, (k + 15) & -16, dtype=torch.uint8).view(torch.float8_e4m3fn)[:, :k]
        held.copy_((w.float() * 50).to(torch.float8_e4m3fn))
        return held, torch.rand((n + 127) // 128, (k + 127) // 128) / 3
    monkeypatch.setattr(_hip, "quantize_weight_fp8", codes)
    cfg = FlashSTUConfig(n_embd=d, n_heads=1, mlp_scale=scale, torch_dtype=torch.bfloat16)
    return fs.FP8MLP(RMSNorm(d, 1e-6, dtype=torch.bfloat16), MLP(cfg, dtype=torch.bfloat16))


@pytest.mark.parametrize("change", [lambda m: m.to(torch.bfloat16), lambda m: m.float(), lambda m: m.half(), lambda m: m.double(), lambda m: m.to("cpu", torch.float32),
                                    lambda m: m.type(torch.float32), lambda m: m.cpu()])
@pytest.mark.parametrize("inside", [False, True])
def test_the_8_bit_mlp_keeps_its_weights_through_a_change_of_type(monkeypatch, change, inside):
    m = parts_without_a_gpu(monkeypatch)
    before = {k: v.clone() for k, v in m.state_dict().items()}
    change(torch.nn.Sequential(m) if inside else m)
    after = m.state_dict()
    assert list(after) == list(before)
    for k, v in before.items():
        if not k.startswith("norm."):
            assert after[k].dtype is v.dtype and after[k].stride() == v.stride()
            assert torch.equal(after[k].view(torch.uint8), v.view(torch.uint8))
    want = change(torch.nn.Linear(2, 2, dtype=torch.bfloat16)).weight.dtype
    assert after["norm.weight"].dtype is want


def test_the_8_bit_mlp_moves_to_another_device(monkeypatch):
    m = parts_without_a_gpu(monkeypatch)
    kinds = {k: v.dtype for k, v in m.state_dict().items()}
    m.to("meta")
    assert all(v.device.type == "meta" and v.dtype is kinds[k] for k, v in m.state_dict().items())
    m.to_empty(device="cpu")
    assert all(v.device.type == "cpu" and v.dtype is kinds[k] for k, v in m.state_dict().items())


def calls_with(grad_of):
    """Each operator with one of its tensors asking for a gradient: (name, call)."""
    import flash_stu as fs
    g = lambda name, t: t.requires_grad_() if name == grad_of else t
    x, d, w = g("x", torch.zeros(2, 128)), g("delta", torch.zeros(2, 128)), g("weight", torch.ones(128))
    c, s = torch.zeros(2, 128).to(torch.float8_e4m3fn), g("scales", torch.zeros(2, 1))
    wc, ws = torch.zeros(16, 128).to(torch.float8_e4m3fn), g("w_scales", torch.zeros(1, 1))
    bias, res, out = g("bias", torch.zeros(16)), g("residual", torch.zeros(2, 16)), g("out", torch.zeros(2, 16))
    return {"quantize_fp8": (("x",), lambda: fs.quantize_fp8(x)), "quantize_weight_fp8": ((), lambda: fs.quantize_weight_fp8(x)),
            "rms_norm_fp8": (("x", "delta", "weight", "out"), lambda: fs.rms_norm_fp8(x, w, 1e-6, delta=d, x_out=out)),
            "linear_fp8": (("scales", "w_scales", "bias", "residual", "out"), lambda: fs.linear_fp8(c, s, wc, ws, bias=bias, residual=res, out=out)),
            "glu_fp8": (("scales", "w_scales"), lambda: fs.glu_fp8(c, s, wc, ws, wc, ws))}


@pytest.mark.parametrize("grad_of", ["x", "delta", "weight", "scales", "w_scales", "bias", "residual", "out"])
def test_a_gradient_that_would_be_lost_is_refused(grad_of):
    """Results have no graph: a tensor that requires a gradient is refused where gradients are on, and taken where they are off.  A weight
    is taken as it is: its codes are made when a model is loaded, from its parameters."""
    from flash_stu._hip import FlashSTUHipError
    for name, (takes, call) in calls_with(grad_of).items():
        if grad_of in takes:
            with pytest.raises(NotImplementedError, match=name + " is forward only"):
                call()
        with torch.no_grad(), pytest.raises(FlashSTUHipError, match="not on the GPU"):
            call()

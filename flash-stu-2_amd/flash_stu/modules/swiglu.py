"""Gated MLP of Flash STU: down(gelu_tanh(gate(x)) * up(x))
(reference: flash_stu/modules/swiglu.py:4-29; the gate is tanh-GELU despite the
file name)."""
import torch
import torch.nn as nn

from .. import _hip


class MLP(nn.Module):
    def __init__(self, config, dtype=None):
        super().__init__()
        dtype = dtype if dtype is not None else config.torch_dtype
        self.hidden_size = config.n_embd
        self.intermediate_size = config.n_embd * config.mlp_scale
        self.gate_proj = nn.Linear(self.hidden_size, self.intermediate_size, bias=config.bias, dtype=dtype)
        self.up_proj = nn.Linear(self.hidden_size, self.intermediate_size, bias=config.bias, dtype=dtype)
        self.down_proj = nn.Linear(self.intermediate_size, self.hidden_size, bias=config.bias, dtype=dtype)

    @_hip.inference
    def forward(self, x: torch.Tensor, residual: torch.Tensor = None):
        """x (..., d).  Up to 16 rows take the skinny MFMA kernels with the gate fused; more rows in bf16 take the
        matrix-core GEMM kernel with the gate as the epilogue of the gate/up pair.  With `residual` (same shape as x,
        contiguous rows) the sum residual + mlp(x) is written into `residual` where the down projection can carry the add
        as its epilogue, and None is returned; otherwise the MLP output is returned and the caller adds it."""
        shape = x.shape
        x2 = x.reshape(-1, shape[-1])
        rows = x2.shape[0]
        if self.gate_proj.bias is not None:
            g = _hip.linear(x2, self.gate_proj.weight, self.gate_proj.bias)
            u = _hip.linear(x2, self.up_proj.weight, self.up_proj.bias)
            act = _hip.gelu_mul(g.contiguous(), u.contiguous(), out=g)
            out = _hip.linear(act, self.down_proj.weight, self.down_proj.bias)
        elif rows <= _hip.MAX_DECODE_ROWS:
            act = _hip.glu_decode(x2, self.gate_proj.weight, self.up_proj.weight)
            out = _hip.linear_decode(act, self.down_proj.weight)
        elif (_hip.gemm_supported(x2, self.gate_proj.weight) and self.up_proj.weight.is_contiguous()
              and self.intermediate_size % 32 == 0 and self.down_proj.weight.is_contiguous()
              and self.down_proj.weight.data_ptr() % 16 == 0):
            act = _hip.gemm(x2, self.gate_proj.weight, up_weight=self.up_proj.weight)
            if residual is not None and residual.is_contiguous():
                r2 = residual.view(-1, shape[-1])
                _hip.gemm(act, self.down_proj.weight, residual=r2, out=r2)
                return None
            out = _hip.gemm(act, self.down_proj.weight)
        else:
            # fp32 (the parity configuration) and shapes the bf16 matrix-core kernel does not take: the general kernel
            g = _hip.gemm_any(x2, self.gate_proj.weight)
            u = _hip.gemm_any(x2, self.up_proj.weight)
            act = _hip.gelu_mul(g, u, out=g)
            out = _hip.gemm_any(act, self.down_proj.weight)
        return out.reshape(shape)


class FP8MLP(nn.Module):
    """The norm and the MLP of a layer with the weights as 8-bit codes: x + delta, then x + down(gelu_tanh(gate(n)) * up(n)) with n = norm(x),
    as the layers form them from RMSNorm and MLP, in three launches (fp32: four).  The codes are laid out here, from the weights as
    they are now, one scale for each 128 x 128; the activations are cut to codes on their way, one scale for each 128 values of a row.  The
    norm's weight stays the norm's own.  Inference only, as RMSNorm and MLP are: nothing here has a gradient."""

    def __init__(self, norm: nn.Module, mlp: MLP):
        super().__init__()
        if mlp.gate_proj.bias is not None:
            raise NotImplementedError("FP8MLP covers bias-free MLPs")
        self.norm = norm
        self.hidden_size, self.intermediate_size = mlp.hidden_size, mlp.intermediate_size
        for name in ("gate", "up", "down"):
            codes, scales = _hip.quantize_weight_fp8(getattr(mlp, name + "_proj").weight.detach())
            # whole rows of 16 bytes, so that a copy of the buffer has them too
            self.register_buffer(name + "_codes", codes.as_strided((codes.shape[0], codes.stride(0)), codes.stride()))
            self.register_buffer(name + "_scales", scales)

    def _apply(self, fn, recurse: bool = True):
        """Moves codes and scales as the bits they are: both count as floating point, and .to(dtype) or .float() of a model would round them.  The
        norm's weight takes the type, as the layers' own do."""
        def move(t):
            if not any(t is b for b in self._buffers.values()):
                return fn(t)
            bits = t.view(torch.uint8 if t.dtype is torch.float8_e4m3fn else torch.int32)
            moved = fn(bits)
            return (moved if moved.dtype is bits.dtype else bits.to(moved.device)).view(t.dtype)
        return super()._apply(move, recurse)

    def _weight(self, name: str, width: int):
        codes = getattr(self, name + "_codes")
        return (codes if codes.shape[1] == width else codes[:, :width]), getattr(self, name + "_scales")

    @_hip.inference
    def forward(self, x: torch.Tensor, delta: torch.Tensor = None) -> torch.Tensor:
        """x (..., d) contiguous, updated in place; delta (same shape) is added first where it is given.  Returns x."""
        d = self.hidden_size
        if x.shape[-1] != d or not x.is_contiguous():
            raise _hip.FlashSTUHipError(f"x must be (..., {d}) and contiguous, got {tuple(x.shape)} stride {x.stride()}")
        if delta is not None and delta.shape != x.shape:
            raise _hip.FlashSTUHipError(f"delta must be {tuple(x.shape)}, got {tuple(delta.shape)}")
        x2 = x.view(-1, d)
        codes, scales = _hip.rms_norm_fp8(x2, self.norm.weight, self.norm.eps, delta=None if delta is None else delta.reshape(-1, d))
        if x.dtype is torch.bfloat16:
            act = _hip.glu_fp8(codes, scales, *self._weight("gate", d), *self._weight("up", d), quantize=True)
        else:
            act = _hip.quantize_fp8(_hip.glu_fp8(codes, scales, *self._weight("gate", d), *self._weight("up", d), dtype=x.dtype))
        _hip.linear_fp8(*act, *self._weight("down", self.intermediate_size), residual=x2, out=x2)
        return x

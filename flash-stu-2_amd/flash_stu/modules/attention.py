"""Sliding-window attention with ALiBi and tanh soft-capping
(reference: flash_stu/modules/attention.py:16-105, whose only backend is the
flash-attn CUDA wheel).  K/V are cached in a ring of window+1 positions laid
out (B,H,cap,hd); a reference-style growing cache (k,v) of shape (B,t,H,hd) is
accepted and converted."""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import _hip
from ..utils.numerics import nearest_power_of_two


def alibi_slopes(n_heads: int, interpolation_factor: float = 0.25) -> torch.Tensor:
    """fp32 slopes (attention.py:38-57)."""
    def gen(n):
        start = 2 ** (-(2 ** -(math.log2(n) - 3)))
        return [start * (start ** i) for i in range(n)]
    if math.log2(n_heads).is_integer():
        s = gen(n_heads)
    else:
        n = nearest_power_of_two(n_heads, round_up=False)
        s = gen(n) + gen(2 * n)[0::2][: n_heads - n]
    return torch.tensor(s, dtype=torch.float32) * interpolation_factor


class Attention(nn.Module):
    def __init__(self, config):
        super().__init__()
        assert config.n_embd % config.n_heads == 0
        self.n_heads = config.n_heads
        self.head_dim = config.n_embd // config.n_heads
        self.c_attn = nn.Linear(config.n_embd, 3 * config.n_embd, bias=config.bias, dtype=config.torch_dtype)
        self.c_proj = nn.Linear(config.n_embd, config.n_embd, bias=config.bias, dtype=config.torch_dtype)
        self.c_proj.SCALE_INIT = 1
        self.register_buffer("alibi_slopes", alibi_slopes(self.n_heads), persistent=False)
        w = config.window_size
        if isinstance(w, (tuple, list)):
            if len(w) != 2 or int(w[1]) != 0:
                raise NotImplementedError("only causal windows (left, 0) are supported")
            w = w[0]
        self.window_size = int(w)
        self.softcap = float(config.softcap or 0.0)

    def _ring_from_reference_cache(self, k: torch.Tensor, v: torch.Tensor):
        B, t, H, hd = k.shape
        cap = self.window_size + 1
        kr = k.new_zeros(B, H, cap, hd)
        vr = v.new_zeros(B, H, cap, hd)
        keep = min(t, cap)
        pos = torch.arange(t - keep, t, device=k.device)
        kr[:, :, pos % cap] = k[:, t - keep:].transpose(1, 2)
        vr[:, :, pos % cap] = v[:, t - keep:].transpose(1, 2)
        return kr, vr, torch.full((B,), t, dtype=torch.int64)

    @_hip.inference
    def forward(self, x: torch.Tensor, past_key_value=None, use_cache: bool = True):
        x = x.contiguous()
        B, T, d = x.shape
        H, hd, W = self.n_heads, self.head_dim, self.window_size
        slopes = self.alibi_slopes
        if past_key_value is None:
            qkv = _hip.linear(x, self.c_attn.weight, self.c_attn.bias).contiguous()
            o = _hip.swa_prefill(qkv, slopes, H, W, self.softcap)
            y = _hip.linear(o, self.c_proj.weight, self.c_proj.bias)
            if not use_cache:
                return y
            cap = W + 1
            # slots the prompt does not fill are written by the decode step that reaches their position before any
            # step reads them (a step reads positions below its own only): no zero fill
            kr = x.new_empty(B, H, cap, hd)
            vr = x.new_empty(B, H, cap, hd)
            _hip.kv_fill(qkv, kr, vr, 0)
            return y, (kr, vr, torch.full((B,), T, dtype=torch.int64))
        if T != 1:
            raise ValueError("a decode call with past_key_value takes exactly one new position")
        if len(past_key_value) == 2:
            past_key_value = self._ring_from_reference_cache(*past_key_value)
        kr, vr, pos_t = past_key_value
        pos = int(pos_t[0])
        qkv = _hip.linear(x.reshape(B, d), self.c_attn.weight, self.c_attn.bias)
        o = _hip.swa_decode(qkv, kr, vr, slopes, pos, W, self.softcap, append=True)
        y = _hip.linear(o, self.c_proj.weight, self.c_proj.bias).reshape(B, 1, d)
        return (y, (kr, vr, pos_t + 1)) if use_cache else y


class KV4Cache:
    """A ring cache of keys and values in 4 bits for a batch of sequences, each at a position of its own.

    Position j of a sequence lives in slot j % capacity.  Values are e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives); 32 values of a head's
    row share a power of two 2^e, e the smallest whole number from -120 to 125 with amax <= 7 * 2^e (125 where none is; values beyond 7 * 2^125 become
    6 * 2^125); a value's code is the nearest, ties to the even one.  32 values with an infinity or a NaN among them stand for NaN.  A key and its value take 17/16 of a byte for each dim, bf16 ones 4.

    `pos` is (batch,) int32 on the GPU and counted by the caller, so that a captured step runs for every position; a sequence at a negative position
    is not in use.  The capacity may exceed a window by any number and is 2^30 at most; head_dim is 32, 64, 128 or 256.  One launch attends over all of it:
    batch and heads are 65535 at most, batch * heads less than 2^23.  Forward only."""

    def __init__(self, batch: int, kv_heads: int, head_dim: int, capacity: int, device=None):
        if (not 1 <= batch <= 65535 or not 1 <= kv_heads <= 65535 or batch * kv_heads >= 1 << 23 or not 1 <= capacity <= 1 << 30
                or head_dim not in (32, 64, 128, 256) or batch * kv_heads * capacity > 1 << 40):
            raise _hip.FlashSTUHipError(f"KV4Cache: batch {batch}, {kv_heads} key heads (each up to 65535, less than 2^23 together), capacity {capacity} (up to 2^30) and head_dim {head_dim} "
                                        "(32, 64, 128 or 256) are no cache")
        device = torch.device("cuda" if device is None else device)
        if device.type != "cuda":
            raise _hip.FlashSTUHipError("KV4Cache lives on the GPU: the HIP path has no CPU fallback")
        self.batch, self.kv_heads, self.head_dim, self.capacity = batch, kv_heads, head_dim, capacity
        self.data = torch.zeros(_hip.kv4_bytes(batch, kv_heads, head_dim, capacity), dtype=torch.uint8, device=device)

    def write(self, k: torch.Tensor, v: torch.Tensor, pos: torch.Tensor, cu_seqlens: torch.Tensor = None) -> None:
        """Rows of k and v (rows, kv_heads, head_dim) float32 or bfloat16 become positions pos[s], pos[s] + 1, ... of sequence s: rows cu_seqlens[s] ..
        cu_seqlens[s + 1] - 1 (of more than `capacity` the last ones), or row s alone without cu_seqlens."""
        _hip.kv4_write(self, k, v, pos, cu_seqlens)

    def read(self, pos: torch.Tensor, cu_seqlens: torch.Tensor = None, rows: int = None, dtype: torch.dtype = torch.bfloat16):
        """What write's rows are held as: (k, v), each (rows, kv_heads, head_dim) of dtype (exact in both); zero for rows of no sequence.  A position that
        the ring no longer holds reads as the one that took its slot."""
        return _hip.kv4_read(self, pos, cu_seqlens, rows, dtype)

    def attend(self, q: torch.Tensor, pos: torch.Tensor, k: torch.Tensor = None, v: torch.Tensor = None, slopes: torch.Tensor = None, window: int = None,
               softcap: float = 0.0, out: torch.Tensor = None) -> torch.Tensor:
        """One query a sequence, q (batch, heads, head_dim), at position pos[s], over the positions max(0, pos[s] - window) .. pos[s] as the cache holds
        them (window None: capacity - 1); heads a multiple of kv_heads, scores as swa_packed's.  k, v (batch, kv_heads, head_dim): those of position
        pos[s], written first (in the same launch but for very long calls, where they are of q's type).  Returns out (batch, heads, head_dim), zero for a
        sequence not in use; out must not overlap q, k, v or the cache."""
        return _hip.kv4_attend(self, q, pos, k, v, slopes, window, softcap, out)

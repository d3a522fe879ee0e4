"""Activation checkpoints in 8 bits, and their use in the backward pass.

A bf16 activation [T, H] is held as int8 with one fp32 scale per 128 columns of
a row (1.03 bytes per value): scale = amax * (1/127), q = round(x * ((1/amax) * 127)),
so a value is off by at most amax / 254 of its block. Blocks whose largest
magnitude is below 1e-30 are held as zeros; a block with an inf or a NaN reads
back as NaN. The kernels that write a checkpoint also do the forward op that
reads the same tensor, and those that read it also do the backward-pass op
that needs it, so a checkpoint costs its own bytes and no pass of its own.

CUDA tensors run the native kernels; CPU tensors run the PyTorch definitions
below. H is a multiple of 8; rows may be strided (16-byte aligned)."""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F

from ._lib import native

BLOCK = 128
_TINY = 1e-30


@dataclass
class Act8:
    """An activation in 8 bits: q int8 [T, H], s fp32 [T, ceil(H / 128)]."""
    q: torch.Tensor
    s: torch.Tensor

    @property
    def shape(self):
        return self.q.shape

    def nbytes(self) -> int:
        return self.q.numel() + 4 * self.s.numel()


def empty(T: int, H: int, device) -> Act8:
    if H <= 0 or H % 8:
        raise ValueError(f"act8: H must be a positive multiple of 8, got {H}")
    return Act8(torch.empty(T, H, dtype=torch.int8, device=device),
                torch.empty(T, -(-H // BLOCK), dtype=torch.float32, device=device))


def _quantise(x: torch.Tensor, a: Act8) -> None:
    T, H = x.shape
    nb = a.s.shape[1]
    b = F.pad(x.float(), (0, nb * BLOCK - H)).view(T, nb, BLOCK)
    amax = b.abs().amax(-1)
    fine = torch.isfinite(b).all(-1)
    live = fine & (amax >= _TINY)
    inv = torch.where(live, amax.reciprocal() * 127.0, torch.zeros_like(amax))
    q = torch.round(torch.where(live.unsqueeze(-1), b, torch.zeros_like(b)) * inv.unsqueeze(-1))
    a.q.copy_(q.view(T, nb * BLOCK)[:, :H])
    s = torch.where(live, amax * (1.0 / 127.0), torch.zeros_like(amax))
    a.s.copy_(torch.where(fine, s, torch.full_like(s, float("nan"))))


def _values(a: Act8) -> torch.Tensor:
    T, H = a.shape
    return a.q.float() * a.s.repeat_interleave(BLOCK, 1)[:, :H]


def save(x: torch.Tensor, out: Optional[Act8] = None) -> Act8:
    """The 8-bit copy of x [T, H]."""
    if x.is_cuda:
        q, s = native().act8_save(x, None if out is None else out.q, None if out is None else out.s)
        return Act8(q, s)
    a = out if out is not None else empty(x.shape[0], x.shape[1], x.device)
    _quantise(x, a)
    return a


def load(a: Act8, out: Optional[torch.Tensor] = None, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that ``a`` stands for, rounded to ``dtype`` (CUDA: bf16)."""
    if a.q.is_cuda:
        if dtype != torch.bfloat16:
            raise ValueError("act8: CUDA checkpoints load as bf16")
        return native().act8_load(a.q, a.s, out)
    if out is None:
        out = torch.empty(a.shape, dtype=dtype)
    return out.copy_(_values(a))


def rmsnorm_save(x: torch.Tensor, w: torch.Tensor, eps: float):
    """Forward: (hn = rmsnorm(x) * w, rstd [T] fp32, x in 8 bits), one read of x."""
    if x.is_cuda:
        hn, rstd, q, s = native().act8_rmsnorm_save(x, w, float(eps))
        return hn, rstd, Act8(q, s)
    T, H = x.shape
    hn, rstd, a = torch.empty_like(x), torch.empty(T), empty(T, H, x.device)
    xf = x.float()
    r = torch.rsqrt(xf.pow(2).mean(-1) + eps)
    rstd.copy_(r)
    hn.copy_(xf * r.unsqueeze(1) * w.float())
    _quantise(x, a)
    return hn, rstd, a


def rmsnorm_load(a: Act8, w: torch.Tensor, eps: float):
    """Backward: (x, hn, rstd) again from the 8-bit copy. hn and rstd are those
    of the held values before x's rounding to the weight's type."""
    if a.q.is_cuda:
        return native().act8_rmsnorm_load(a.q, a.s, w, float(eps))
    x = torch.empty(a.shape, dtype=w.dtype)
    hn, rstd = torch.empty_like(x), torch.empty(x.shape[0])
    v = _values(a)
    r = torch.rsqrt(v.pow(2).mean(-1) + eps)
    rstd.copy_(r)
    x.copy_(v)
    hn.copy_(v * r.unsqueeze(1) * w.float())
    return x, hn, rstd


def swiglu_save(gu: torch.Tensor):
    """Forward: (silu(gate) * up of gu = [gate | up] [T, 2 F], gu in 8 bits)."""
    T, f2 = gu.shape
    if f2 % 16:
        raise ValueError(f"act8: [gate | up] needs a width that is a multiple of 16, got {f2}")
    if gu.is_cuda:
        a, q, s = native().act8_swiglu_save(gu)
        return a, Act8(q, s)
    a, held = torch.empty(T, f2 // 2, dtype=gu.dtype), empty(T, f2, gu.device)
    g, u = gu.float().chunk(2, -1)
    a.copy_(F.silu(g) * u)
    _quantise(gu, held)
    return a, held


def swiglu_bwd(dout: torch.Tensor, held: Act8):
    """Backward from the 8-bit [gate | up]: (d[gate | up] [T, 2 F], the
    activation silu(gate) * up again [T, F], for the down projection's weight
    gradient)."""
    if dout.is_cuda:
        return native().act8_swiglu_bwd(dout, held.q, held.s)
    T, f2 = held.shape
    dgu, a = torch.empty(T, f2, dtype=dout.dtype), torch.empty(T, f2 // 2, dtype=dout.dtype)
    g, u = _values(held).chunk(2, -1)
    d = dout.float()
    sg = torch.sigmoid(g)
    act = g * sg
    dgu.copy_(torch.cat([d * u * (sg + act * (1 - sg)), d * act], -1))
    a.copy_(act * u)
    return dgu, a

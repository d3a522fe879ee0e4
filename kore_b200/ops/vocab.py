"""The two ends of the model that are as wide as the vocabulary: the head's
loss in pieces of the vocabulary, without keeping logits, and the embedding
with its gradient by sorted tokens.

CUDA tensors run the native kernels; CPU tensors run the PyTorch definitions
below (any floating type, for CPU tests and gloo runs)."""
from __future__ import annotations

from typing import Optional

import torch

from ._lib import native


def _inv_temp(temperature: float) -> float:
    if not temperature > 0:
        raise ValueError("temperature must be positive")
    return 1.0 / float(temperature)


def head_fwd(x: torch.Tensor, w: torch.Tensor, targets: Optional[torch.Tensor] = None, temperature: float = 1.0,
             *, want_entropy: bool = False):
    """Statistics of softmax(x @ w.T / temperature) per row of x [T, H], w [V, H].

    Returns (logp [T] of ``targets`` or None, entropy [T] or None, lse [T]), all
    fp32. The logits are never stored: they go from the fp32 accumulator into
    the rows' running maxima and sums. ``logp`` is 0 where the target is
    outside [0, V) (no label). ``lse`` is what :func:`head_bwd` needs."""
    inv = _inv_temp(temperature)
    if x.is_cuda:
        return native().head_fwd(x, w, targets, inv, want_entropy)
    T, dev = x.shape[0], x.device
    lse = torch.empty(T, dtype=torch.float32, device=dev)
    logp = torch.empty(T, dtype=torch.float32, device=dev) if targets is not None else None
    ent = torch.empty(T, dtype=torch.float32, device=dev) if want_entropy else None
    z = (x.float() @ w.float().t()) * inv
    l = torch.logsumexp(z, -1)
    lse.copy_(l)
    if logp is not None:
        ok = (targets >= 0) & (targets < w.shape[0])
        zt = z.gather(1, torch.where(ok, targets, torch.zeros_like(targets)).unsqueeze(1))[:, 0]
        logp.copy_(torch.where(ok, zt - l, torch.zeros_like(l)))
    if ent is not None:
        lp = z - l.unsqueeze(1)
        ent.copy_(-torch.xlogy(lp.exp(), lp.exp()).sum(-1))
    return logp, ent, lse


def head_bwd(x: torch.Tensor, w: torch.Tensor, targets: Optional[torch.Tensor], lse: torch.Tensor,
             coef: torch.Tensor, temperature: float = 1.0, *, dx: Optional[torch.Tensor] = None,
             dw: Optional[torch.Tensor] = None, accumulate: bool = False, piece: int = 0):
    """Gradient of L = sum_t coef_t logp_t of :func:`head_fwd`; returns (dx, dw).

    dx [T, H] is overwritten; dw [V, H] (bf16 or fp32) is overwritten, or added
    to with ``accumulate``. The logits are computed again for ``piece``
    vocabulary entries at a time (0: the size whose dz, [T, piece] bf16, takes
    about 256 MB, and 4,096 at least), so no [T, V] tensor exists. Rows with coefficient 0
    contribute nothing, even if x holds inf or NaN there. A row whose target is
    outside [0, V) has no label: its gradient is that of -coef_t * lse_t."""
    inv = _inv_temp(temperature)
    if accumulate and dw is None:
        raise ValueError("accumulate needs dw")
    if dw is None:
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
    if x.is_cuda:
        return native().head_bwd(x, w, targets, lse, coef, inv, dx, dw, bool(accumulate), int(piece)), dw
    if dx is None:
        dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    V = w.shape[0]
    live = (coef != 0).unsqueeze(1)
    xm = torch.where(live, x.float(), torch.zeros((), dtype=torch.float32))
    acc = torch.zeros(x.shape, dtype=torch.float32)
    ct = (coef.float() * inv).unsqueeze(1)
    step = piece or V
    for v0 in range(0, V, step):
        wp = w[v0:v0 + step].float()
        dz = -ct * torch.exp((xm @ wp.t()) * inv - lse.unsqueeze(1))
        if targets is not None:
            hit = targets.unsqueeze(1) == torch.arange(v0, v0 + wp.shape[0])
            dz = dz + torch.where(hit, ct, torch.zeros_like(ct))
        dz = torch.where(live, dz, torch.zeros_like(dz))
        acc += dz @ wp
        g = dz.t() @ xm
        out = dw[v0:v0 + step]
        out.copy_(g + out.float() if accumulate else g)
    dx.copy_(acc)
    return dx, dw


def embed(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0, out: Optional[torch.Tensor] = None):
    """out[t] = scale * table[ids[t]] (rounded once); ids outside the table give zero rows."""
    flat = ids.reshape(-1)
    if table.is_cuda:
        return native().embed_scaled(flat, table, out, float(scale))
    if out is None:
        out = torch.empty(flat.numel(), table.shape[1], dtype=table.dtype, device=table.device)
    ok = (flat >= 0) & (flat < table.shape[0])
    rows = table[torch.where(ok, flat, torch.zeros_like(flat))].float() * scale
    out.copy_(torch.where(ok.unsqueeze(1), rows, torch.zeros_like(rows)))
    return out


def embed_grad(ids: torch.Tensor, dy: torch.Tensor, dtable: torch.Tensor, scale: float = 1.0, *,
               accumulate: bool = True):
    """dtable[v] (+)= scale * sum of the rows dy[t] with ids[t] == v.

    Each row's sum runs over its tokens in ascending order in fp32 and is
    rounded once, so equal calls give equal bits. ``accumulate=False``
    overwrites the whole table (rows without a token become zero). ids outside
    the table are ignored. dtable: contiguous bf16 or fp32 [V, H]."""
    flat = ids.reshape(-1)
    if dy.is_cuda:
        native().embed_grad_sorted(flat, dy, dtable, float(scale), bool(accumulate))
        return dtable
    ok = (flat >= 0) & (flat < dtable.shape[0])
    g = torch.zeros(dtable.shape, dtype=torch.float32)
    g.index_add_(0, flat[ok], dy[ok].float())
    g *= scale
    if not accumulate:
        dtable.copy_(g)
        return dtable
    used = torch.unique(flat[ok])
    dtable[used] = (dtable[used].float() + g[used]).to(dtable.dtype)
    return dtable

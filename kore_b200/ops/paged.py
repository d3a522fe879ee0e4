"""The paged KV cache: a step's plan and attention for batches with shared prefixes.

CUDA tensors run the native kernels; CPU tensors run the PyTorch definitions
below (any floating type and head size, for CPU tests).

A cache is two tensors [slots, Hkv, 128]; page p holds slots p * page_size up to
(p + 1) * page_size, and row b of a block table lists the pages of sequence b."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional, Tuple

import torch

from ._lib import native

MAX_SEQUENCES = 512                    # of one prefix_attention call on CUDA


@dataclass
class Plan:
    """Where a step's rows go (int32 tensors; ``ok`` is bool)."""
    q_start: torch.Tensor              # [B + 1] first row of each sequence
    lens: torch.Tensor                 # [B] tokens in the cache after the step
    pos: torch.Tensor                  # [rows] position in its sequence
    slots: torch.Tensor                # [rows] cache slot, -1: not written
    ok: torch.Tensor                   # [B] False: no room, the sequence keeps its old length
    held: torch.Tensor                 # [B] pages in the table after the step
    free_count: Optional[torch.Tensor]  # [1] pages left on the stack (None without a pool)


def plan(ctx: torch.Tensor, new: torch.Tensor, table: torch.Tensor, page_size: int, rows: int, *,
         held: Optional[torch.Tensor] = None, free: Optional[torch.Tensor] = None,
         free_count: Optional[torch.Tensor] = None) -> Plan:
    """Plan of a step that appends ``new[b]`` tokens to sequence b of ``ctx[b]``
    cached ones (int32 [B]; negative counts as 0), packed in order into ``rows`` rows.

    ``table`` (int32 [B, pages]) holds ``held[b]`` pages a sequence (default: those
    that ``ctx`` fills). With a pool (``free``: a stack of page ids of which the
    first ``free_count`` are free), the pages that a sequence lacks are taken from
    the top of the stack, in the order of the sequences, and written into the
    table in place (its rows must not overlap); the stack itself is only read, and ``Plan.free_count`` says how
    many are left. A sequence whose tokens do not fit its table row, or whose
    pages together with those that the sequences before it asked for are more than
    the pool has, is not ``ok``: it gets no page, its rows have slot -1 and its
    length stays. Rows behind the last sequence have position 0 and slot -1;
    tokens behind row ``rows`` are not planned.

    Every result is a new tensor, so a step can be planned again; the host is not waited for."""
    page_size, rows = int(page_size), int(rows)
    if ctx.is_cuda:
        return Plan(*native().paged_plan(ctx, new, table, page_size, rows, held, free, free_count))
    if (free is None) != (free_count is None):
        raise ValueError("paged: give free and free_count, or neither")
    if page_size <= 0 or rows < 0:
        raise ValueError("paged: page_size must be positive and rows not negative")
    B, M = table.shape
    if ctx.numel() != B or new.numel() != B or (held is not None and held.numel() != B):
        raise ValueError("paged: ctx, new and held need one entry for each row of the table")
    if free is not None and B > 1 and table.stride(0) < M:
        raise ValueError("paged: rows of a table that pages are written to must not overlap")
    count = min(max(int(free_count), 0), free.numel()) if free is not None else 0
    asked = granted = at = 0
    q_start, lens, ok, held_out = [0], [], [], []
    pos, slots = torch.zeros(rows, dtype=torch.int32), torch.full((rows,), -1, dtype=torch.int32)
    for b in range(B):
        c, n = max(int(ctx[b]), 0), min(max(int(new[b]), 0), rows - at)
        need = -(-(c + n) // page_size)
        h = -(-c // page_size) if held is None else min(max(int(held[b]), 0), M)
        take = max(0, need - h) if free is not None and need <= M else 0
        asked += take
        fine = need <= M and (free is None or asked <= count)
        if fine:
            for j in range(take):
                table[b, h + j] = free[count - 1 - (asked - take) - j]
            granted += take
        p = torch.arange(c, c + n)
        pos[at:at + n] = p.int()
        if fine:
            page = table[b].long()[p // page_size]
            slots[at:at + n] = torch.where(page < 0, torch.full_like(p, -1), page * page_size + p % page_size).int()
        at += n
        q_start.append(at)
        lens.append(c + n if fine else c)
        ok.append(fine)
        held_out.append(h + take if fine else h)
    i32 = dict(dtype=torch.int32)
    return Plan(torch.tensor(q_start, **i32), torch.tensor(lens, **i32), pos, slots, torch.tensor(ok, dtype=torch.bool),
                torch.tensor(held_out, **i32), None if free is None else torch.tensor([count - granted], **i32))


def prefix_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                     lens: torch.Tensor, q_start: torch.Tensor, page_size: int, *, max_q: int = 1,
                     scale: Optional[float] = None, group_start: Optional[torch.Tensor] = None,
                     prefix_len: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                     want_lse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Causal attention of each sequence's newest tokens over its paged history.

    Rows q_start[b] .. q_start[b + 1] of q [T, Hq, D] are the last tokens of
    sequence b, whose ``lens[b]`` tokens (these included) are in the cache. Returns
    (out [T, Hq, D], lse [T, Hq] fp32 or None). A row without keys gives zeros and
    lse -inf; rows before the first sequence (q_start[0] need not be 0) and behind the
    last one are left as they were in ``out`` (their lse is not defined).

    Sequences group_start[g] .. group_start[g + 1] share their first
    ``prefix_len[g]`` tokens (int32 [groups + 1] and [groups]; any length, also one
    that ends inside a page). Those keys are read through the table of the group's
    first sequence, once for all rows of the group, so the other sequences' tables
    are not read there. Without groups each sequence reads its own history. On CUDA
    groups pay from a few thousand shared tokens of eight or more sequences on; below
    that, and for chunks of many tokens a sequence, the extra parts cost more than the
    reads they save. A call with groups takes 1 KB of workspace for each row and head.

    ``max_q`` is the largest number of rows of a sequence as far as the host knows
    (it chooses the split, not the result). Neither q_start nor group_start may
    decrease: on CUDA the rows of such a call get zeros and ``check_device_error``
    reports 3, on the CPU it raises. CUDA: bf16, D = 128, page_size a
    multiple of 8, at most 512 sequences, scale a positive normal fp32 number. What the cache holds behind a
    sequence's last token does not matter, NaN included; among the tokens of a
    call, a row's value that is not finite reaches the sequence's earlier rows too."""
    scale = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device) if want_lse else None
    if q.is_cuda:
        native().paged_prefix_attention(q, k_cache, v_cache, table, lens, q_start, int(page_size), int(max_q), float(scale),
                                        group_start, prefix_len, out, lse)
        return out, lse
    if (group_start is None) != (prefix_len is None):
        raise ValueError("prefix_attention: give group_start and prefix_len, or neither")
    hq, hkv = q.shape[1], k_cache.shape[1]
    if hkv == 0 or hq % hkv:
        raise ValueError("prefix_attention: Hq must be a multiple of Hkv")
    if any((t is not None and (t[1:] < t[:-1]).any()) for t in (q_start, group_start)):
        raise ValueError("prefix_attention: q_start and group_start must not decrease")
    lead, shared = list(range(lens.numel())), [0] * lens.numel()
    if prefix_len is not None:
        for g, n in enumerate(prefix_len.tolist()):
            for b in range(int(group_start[g]), int(group_start[g + 1])):
                lead[b], shared[b] = int(group_start[g]), n
    starts = q_start.tolist()
    for b, n in enumerate(lens.tolist()):
        first, m = starts[b], starts[b + 1] - starts[b]
        at = torch.arange(n)
        page = torch.where(at < shared[b], table[lead[b]].long()[at // page_size], table[b].long()[at // page_size])
        slots = page * page_size + at % page_size
        k, v = (c[slots].float().repeat_interleave(hq // hkv, 1) for c in (k_cache, v_cache))
        s = torch.einsum("mhd,nhd->mhn", q[first:first + m].float(), k) * scale
        s = s.masked_fill((at[None] > torch.arange(n - m, n)[:, None])[:, None], -math.inf)
        z = torch.logsumexp(s, -1)
        w = torch.where(z.isneginf()[..., None], torch.zeros_like(s), torch.exp(s - z[..., None]))
        out[first:first + m] = torch.einsum("mhn,nhd->mhd", w, v).to(q.dtype)
        if lse is not None:
            lse[first:first + m] = z
    return out, lse

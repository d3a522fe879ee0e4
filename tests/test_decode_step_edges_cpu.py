"""Edges of the step plan, shared-prefix attention and draft verification on CPU tensors."""
import math

import pytest
import torch
from paged_oracle import attention_oracle, build_cache

from test_paged_cpu import check_verify, verify_case

from kore_b200.ops import paged


def _i(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("lead", [1, 5])
def test_rows_before_the_first_sequence(lead):
    a = build_cache([(5, [(9, 1), (30, 3)]), (0, [(7, 2)])], 8, 6, 2, dtype=torch.float32, D=16)
    want = attention_oracle(a)[0]
    q = torch.cat([torch.full((lead, 6, 16), math.nan), a["q"]])
    out = torch.full_like(q, 7.0)
    paged.prefix_attention(**{**a, "q": q, "q_start": a["q_start"] + lead}, max_q=3, out=out)
    assert (out[:lead] == 7).all() and torch.allclose(out[lead:].double(), want, atol=1e-5)


@pytest.mark.parametrize("tau", [0.8, 0.0])
def test_verify_rows_before_the_first_sequence(tau):
    z, tokens, qs, u, _ = verify_case(7, 100, [3, 4, 2])
    v = check_verify((z, tokens, qs[1:].contiguous(), u, None), tau)
    assert (v.logp[:3] == 0).all()

"""Packed attention on offsets that name tokens twice or over and over: what is named is computed, and nothing else is touched."""
import math

import numpy as np
import pytest
import torch

import serving_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def S(lib):
    from vesper_b200 import serving_capi
    return serving_capi


def int32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


def case(S, total, Hq, Hkv, D, guard=300):
    """q, k, v with NaN tokens, and o and lse with threes, behind the `total` tokens; what one sequence of them all gives."""
    g = torch.Generator(device=DEV).manual_seed(total + Hq)
    q, k, v = (torch.randn(total + guard, h, D, generator=g, device=DEV).bfloat16() for h in (Hq, Hkv, Hkv))
    for x in (q, k, v):
        x[total:] = math.nan
    return q, k, v, torch.full_like(q, 3.0), torch.full((Hq, total + guard), 3.0, device=DEV)


def one(S, q, k, v, a, b, causal=True):
    o, lse = torch.empty_like(q[a:b]), torch.empty(q.shape[1], b - a, device=DEV)
    S.prefill_packed(q[a:b].contiguous(), k[a:b].contiguous(), v[a:b].contiguous(), o, lse, scale=0.125, cu_seqlens_q=int32([0, b - a]), causal=causal)
    want, want_lse, weighted, size = R.attention(q[a:b], k[a:b], v[a:b], scale=0.125, causal=causal)
    R.check(o, want, R.attention_bound(want, weighted, size, dtype=q.dtype, weights=q.dtype, D=q.shape[2], v=v[a:b]), "o")
    R.check(lse, want_lse, R.lse_bound(want_lse, size, q.shape[2]), "lse")
    return o, lse


@pytest.mark.parametrize("Hq, Hkv, D", [(4, 2, 64), (64, 64, 64), (16, 4, 128)])
def test_two_sequences_that_share_tokens(S, Hq, Hkv, D):
    """[0, 30) and [20, 60) with a sequence between them whose offsets descend, and one behind that passes the tokens given: 0-19 are the first one's, 30-59 the
    second's, each of 20-29 one or the other's, and the rest stays."""
    q, k, v, o, _ = case(S, 100, Hq, Hkv, D)
    lse = torch.full((Hq, 100), 3.0, device=DEV)
    S.prefill_packed(q[:100], k[:100], v[:100], o[:100], lse, scale=0.125, cu_seqlens_q=int32([0, 30, 20, 60, 101]))
    (a, a_lse), (b, b_lse) = one(S, q, k, v, 0, 30), one(S, q, k, v, 20, 60)
    assert torch.equal(o[:20], a[:20]) and torch.equal(o[30:60], b[10:]) and torch.equal(lse[:, :20], a_lse[:, :20]) and torch.equal(lse[:, 30:60], b_lse[:, 10:])
    assert bool(((o[20:30] == a[20:]) | (o[20:30] == b[:10])).all()) and bool(((lse[:, 20:30] == a_lse[:, 20:]) | (lse[:, 20:30] == b_lse[:, :10])).all())
    assert bool((o[60:] == 3.0).all()) and bool((lse[:, 60:] == 3.0).all())


@pytest.mark.parametrize("Hq, Hkv, D, total", [(160, 80, 64, 100), (16, 4, 128, 100), (16, 4, 128, 300), (80, 80, 64, 40)])
@pytest.mark.parametrize("times", [2, 300])
def test_the_same_tokens_over_and_over(S, Hq, Hkv, D, total, times):
    """Offsets that go back to 0 again and again.  The list has room for a sequence's first items at the least: they are there, whatever else is; the first tokens of
    every head are written, every token written has its value, and those behind are as they were."""
    q, k, v, o, lse = case(S, total, Hq, Hkv, D)
    S.prefill_packed(q, k, v, o, lse, scale=0.125, cu_seqlens_q=int32([0, total] * times))
    want, want_lse = one(S, q, k, v, 0, total)
    assert torch.equal(o[:total], want) and torch.equal(lse[:, :total], want_lse)
    assert bool((o[total:] == 3.0).all()) and bool((lse[:, total:] == 3.0).all())

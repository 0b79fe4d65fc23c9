"""Packed attention on values that are not finite, in every column of a block of scores; 4-bit decode on queries of nothing."""
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


def randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def int32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


def packed(S, q, k, v, nq, nk, n, causal):
    o, lse = torch.full_like(q, 9.0), torch.full((q.shape[1], q.shape[0]), 9.0, device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=q.shape[2] ** -0.5, cu_seqlens_q=int32(np.arange(n + 1) * nq), cu_seqlens_k=int32(np.arange(n + 1) * nk), causal=causal)
    return o.view(n, nq, *o.shape[1:]), lse.view(lse.shape[0], n, nq)


# A block holds 80 keys with head_dim 128 and 112 with 64; 240 keys are two whole blocks, which no mask touches, and a part of one.
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(4, 2, 128, torch.bfloat16), (2, 2, 64, torch.float16), (16, 2, 64, torch.bfloat16), (4, 4, 128, torch.float16)])
def test_one_nan_key_anywhere(S, Hq, Hkv, D, dtype, causal):
    """Sequence i has one NaN, in key i of key head 0: the outputs and the lse of that head's queries are NaN; the other head's are the bits that they were."""
    nq, nk, n, rep = 2, 240, 239, Hq // Hkv
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = randn(g, n * nq, Hq, D, dtype=dtype), randn(g, n * nk, Hkv, D, dtype=dtype), randn(g, n * nk, Hkv, D, dtype=dtype)
    clean, clean_lse = packed(S, q, k, v, nq, nk, n, causal)
    k.view(n, nk, Hkv, D)[torch.arange(n), torch.arange(n), 0, 5] = math.nan
    o, lse = packed(S, q, k, v, nq, nk, n, causal)                 # (key 239 is left out: the first of two causal queries does not see it)
    assert bool(torch.isnan(lse[:rep]).all()), sorted(set((~torch.isnan(lse[:rep])).nonzero()[:, 1].tolist()))
    assert bool(torch.isnan(o[:, :, :rep]).all())
    assert torch.equal(o[:, :, rep:], clean[:, :, rep:]) and torch.equal(lse[rep:], clean_lse[rep:])


@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(4, 2, 128, torch.bfloat16), (2, 2, 64, torch.float16), (2, 2, 64, torch.bfloat16)])
def test_one_score_of_minus_infinity_anywhere(S, Hq, Hkv, D, dtype):
    """Key i of sequence i scores -infinity: it weighs nothing, and the rest is attention without it."""
    nq, nk, n = 1, 240, 240
    g = torch.Generator(device=DEV).manual_seed(D + 1)
    q, k, v = randn(g, n * nq, Hq, D, dtype=dtype), randn(g, n * nk, Hkv, D, dtype=dtype), randn(g, n * nk, Hkv, D, dtype=dtype)
    q[:, :, 0] = 1.0
    k.view(n, nk, Hkv, D)[torch.arange(n), torch.arange(n), :, 0] = -math.inf
    o, lse = packed(S, q, k, v, nq, nk, n, False)
    for i in range(n):
        rest = [x.view(n, nk, Hkv, D)[i, torch.arange(nk, device=DEV) != i] for x in (k, v)]
        want, want_lse, weighted, size = R.attention(q[i:i + 1], *rest, scale=D ** -0.5, causal=False)
        R.check(o[i], want, R.attention_bound(want, weighted, size, dtype=dtype, weights=dtype, D=D, v=rest[1]), f"o without key {i}")
        R.check(lse[:, i], want_lse, R.lse_bound(want_lse, size, D), f"lse without key {i}")


@pytest.mark.parametrize("nk", [1, 14, 15, 80, 112, 240])
@pytest.mark.parametrize("D, dtype", [(128, torch.bfloat16), (64, torch.float16), (64, torch.bfloat16)])
def test_every_score_minus_infinity(S, D, dtype, nk):
    """Keys are seen and every score is -infinity: the sum of the weights is zero, so the outputs are 0 / 0 and the lse is ln 0; a query that sees no key has
    zeros, and another head's results are its own."""
    g = torch.Generator(device=DEV).manual_seed(nk)
    q, k, v = randn(g, 3, 4, D, dtype=dtype), randn(g, nk, 2, D, dtype=dtype), randn(g, nk, 2, D, dtype=dtype)
    q[:, :, 0] = 1.0
    clean, clean_lse = packed(S, q, k, v, 3, nk, 1, False)
    k[:, 0, 0] = -math.inf
    o, lse = packed(S, q, k, v, 3, nk, 1, False)
    assert bool(torch.isnan(o[0, :, :2]).all()) and bool((lse[:2] == -math.inf).all())
    assert torch.equal(o[0, :, 2:], clean[0, :, 2:]) and torch.equal(lse[2:], clean_lse[2:])
    if nk == 1:                                                     # causal: of three queries the last alone sees the key
        o, lse = packed(S, q, k, v, 3, 1, 1, True)
        assert not o[0, :2].any() and bool((lse[:, 0, :2] == -math.inf).all())
        assert bool(torch.isnan(o[0, 2, :2]).all()) and bool((lse[:2, 0, 2] == -math.inf).all()) and torch.equal(o[0, 2, 2:], clean[0, 2, 2:])


@pytest.mark.parametrize("size", [0.0, 2.0 ** -100])
@pytest.mark.parametrize("exponent, scale", [(-64, 0.1), (-30, 0.1), (-25, 128 ** -0.5), (0, 1e-30), (64, 1e-38)])
@pytest.mark.parametrize("Hq, Hkv, D", [(8, 2, 128), (2, 2, 64), (16, 1, 64)])
def test_decode_kv4_queries_of_nothing(S, Hq, Hkv, D, exponent, scale, size):
    """Queries of zero (a padded row of the batch), or nearly: the mean of the values and ln n, whatever the scale and the cache's exponents."""
    lens = [1, 50, 64, 90, 300, 1000]
    g = torch.Generator(device=DEV).manual_seed(D + exponent)
    B, cap = len(lens), 1000
    k, v = randn(g, B, Hkv, cap, D, scale=2.0 ** exponent), randn(g, B, Hkv, cap, D)
    cache = S.Kv4Cache(B, Hkv, cap, D, device=DEV, k_exponent=exponent)
    cache.append(k, v)
    q = randn(g, B, Hq, 1, D, scale=size)
    held_k, held_v = R.quantise(k, exponent), R.quantise(v)
    for splits in (0, 1, 3):
        o, lse = torch.full_like(q, 9.0), torch.full((B, Hq), 9.0, device=DEV)
        S.decode_kv4(q, o, cache, scale=scale, lse=lse, seq_lens=int32(lens), num_splits=splits)
        for b, n in enumerate(lens):
            vv = held_v[b, :, :n].transpose(0, 1)
            want, want_lse, weighted, score = R.attention(q[b].transpose(0, 1), held_k[b, :, :n].transpose(0, 1), vv, scale=scale, causal=False)
            R.check(o[b].transpose(0, 1), want, R.attention_bound(want, weighted, score, dtype=q.dtype, weights=torch.float16, D=D, v=vv), f"o of {n} rows")
            R.check(lse[b][:, None], want_lse, R.lse_bound(want_lse, score, D), f"lse of {n} rows")

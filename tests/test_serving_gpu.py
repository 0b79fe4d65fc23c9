"""The serving operators on the GPU against their formulas in 64 bits (tests/serving_reference.py).  The bounds there count the roundings of each path."""
import math

import numpy as np
import pytest
import torch

import serving_reference as R

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
THETA = 10000.0


@pytest.fixture(scope="module")
def S(lib):
    from vesper_b200 import serving_capi
    return serving_capi


@pytest.fixture(autouse=True)
def status_is_clean():
    from vesper_b200 import capi
    yield
    torch.cuda.synchronize()
    capi.check_kernel_status(0)


def rng(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.bfloat16, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device=DEV)).to(dtype)


def int32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


def expect_full(seq):
    """The status word reports a place out of the cache, and is cleared."""
    from vesper_b200 import capi
    torch.cuda.synchronize()
    with pytest.raises(capi.Vb200Error) as e:
        capi.check_kernel_status(0)
    assert e.value.status == -8 and (seq is None or f"sequence {seq} " in str(e.value))


# ---- norms of queries and keys with the rotation ---------------------------------------------------
def norm_bound(want, dtype):
    """Rounded once to `dtype`; before that fp32: the sum of squares (D roundings, half of it in the root), root, two products, then a product, a product and a sum
    with cos and sin, each within 2^-22 of a pair's size: well within 2^-18 of it."""
    pair = want.unflatten(-1, (-1, 2)).norm(dim=-1, keepdim=True).expand(want.shape[:-1] + (want.shape[-1] // 2, 2)).flatten(-2)
    return R.unit(dtype) * want.abs() + 2.0 ** -18 * pair + 1e-30


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B, T, Hq, Hkv, D", [(1, 1, 4, 1, 128), (3, 7, 6, 2, 64), (1, 1, 1, 1, 8), (2, 129, 5, 5, 72), (1, 700, 16, 4, 128), (33, 1, 16, 4, 128), (2, 19, 3, 1, 40),
                                              (1, 2400, 8, 8, 16)])
def test_norm_rope(S, dtype, B, T, Hq, Hkv, D):
    from vesper_b200 import capi
    g = rng(B * 1000 + T + D)
    qkv = randn(g, B, T, Hq + 2 * Hkv, D, dtype=dtype, scale=3.0)
    q, k, v = (x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], dim=2))
    qw, kw = 1 + 0.3 * randn(g, D, dtype=torch.float32), 1 + 0.3 * randn(g, D, dtype=torch.float32)
    pos = torch.randint(0, 131072, (B, T), generator=g, device=DEV, dtype=torch.int32)
    f = list(capi.inv_freq(THETA, D))
    q_out, k_out, v_out = (torch.empty_like(x, memory_format=torch.contiguous_format) for x in (q, k, v))
    S.qk_norm_rope(q, k, v, eps=1e-6, q_weight=qw, k_weight=kw, theta=THETA, positions=pos, q_out=q_out, k_out=k_out, v_out=v_out)
    for got, x, w in ((q_out, q, qw), (k_out, k, kw)):
        want = R.norm_rope(x, eps=1e-6, weight=w, positions=pos, inv_freq=f)
        R.check(got, want, norm_bound(want, dtype), "norm and rotation")
    assert torch.equal(v_out, v)
    # in place, on the views of the projection: the same bits
    before = v.clone()
    S.qk_norm_rope(q, k, eps=1e-6, q_weight=qw, k_weight=kw, theta=THETA, positions=pos)
    assert torch.equal(q, q_out) and torch.equal(k, k_out) and torch.equal(v, before)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norm_rope_parts(S, dtype):
    """The norm alone, the rotation alone, without weights, one tensor alone, a start position."""
    from vesper_b200 import capi
    g = rng(5)
    B, T, H, D = 2, 37, 6, 128
    q, k = randn(g, B, H, T, D, dtype=dtype), randn(g, B, 2, T, D, dtype=dtype)
    pos = torch.arange(16000, 16000 + T, device=DEV).expand(B, T)
    f = list(capi.inv_freq(THETA, D))
    q_out, _, _ = S.qk_norm_rope(q, None, eps=1e-5, q_out=torch.empty_like(q))
    want = R.norm_rope(q, eps=1e-5)
    R.check(q_out, want, norm_bound(want, dtype), "norm")
    q_out, k_out, _ = S.qk_norm_rope(q, k, theta=THETA, start_pos=16000, q_out=torch.empty_like(q), k_out=torch.empty_like(k))
    for got, x in ((q_out, q), (k_out, k)):
        want = R.norm_rope(x, positions=pos, inv_freq=f)
        R.check(got, want, norm_bound(want, dtype), "rotation")
    _, k_out, _ = S.qk_norm_rope(None, k, eps=0.0, theta=THETA, start_pos=16000, k_out=torch.empty_like(k))
    want = R.norm_rope(k, eps=0.0, positions=pos, inv_freq=f)
    R.check(k_out, want, norm_bound(want, dtype), "keys alone")
    zero = torch.zeros_like(q)
    S.qk_norm_rope(zero, None, eps=1e-6, theta=THETA)
    assert not zero.any()


def test_norm_rope_far_positions(S):
    """Angles of positions up to 2^30: the product with the frequency is not rounded to fp32."""
    from vesper_b200 import capi
    g = rng(6)
    pos = int32([0, 1, 16384, 131071, 1048576, 2 ** 24 + 1, 2 ** 30, 2 ** 31 - 1]).view(1, -1)
    q = randn(g, 1, 2, 8, 128, dtype=torch.float32)
    got, _, _ = S.qk_norm_rope(q, None, theta=THETA, positions=pos, q_out=torch.empty_like(q))
    want = R.norm_rope(q, positions=pos, inv_freq=list(capi.inv_freq(THETA, 128)))
    R.check(got, want, norm_bound(want, torch.float32), "far positions")


def test_norm_rope_into_a_cache(S):
    """Keys and values to the rows that the call names; a negative row is left out, one past the cache too, with the status word set; nothing else is touched."""
    from vesper_b200 import capi
    g = rng(7)
    Hq, Hkv, D, cap, lens = 4, 2, 64, 40, [3, 0, 17, 1]
    T = sum(lens) + 3                                                    # three tokens of padding
    q, k, v = randn(g, 1, Hq, T, D), randn(g, 1, Hkv, T, D), randn(g, 1, Hkv, T, D)
    rows = np.concatenate([np.arange(n) + 5 * i for i, n in enumerate(lens)] + [[-1, -1, -7]])
    seqs = np.concatenate([np.full(n, i) for i, n in enumerate(lens)] + [[0, 99, -5]])
    k_cache, v_cache = (torch.full((4, Hkv, cap, D), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    f = list(capi.inv_freq(THETA, D))
    q_out = torch.empty_like(q)
    pos = int32(np.maximum(rows, 0)).view(1, T)
    S.qk_norm_rope(q, k, v, eps=1e-6, inv_freq=f, positions=pos, q_out=q_out, k_out=k_cache, v_out=v_cache, rows=int32(rows).view(1, T), seqs=int32(seqs).view(1, T))
    want_q = R.norm_rope(q, eps=1e-6, positions=pos, inv_freq=f)
    R.check(q_out, want_q, norm_bound(want_q, q.dtype), "queries")
    want_k, named = R.norm_rope(k, eps=1e-6, positions=pos, inv_freq=f), torch.zeros(4, cap, dtype=torch.bool, device=DEV)
    for i in range(T - 3):
        b, r = int(seqs[i]), int(rows[i])
        named[b, r] = True
        R.check(k_cache[b, :, r], want_k[0, :, i], norm_bound(want_k[0, :, i], k.dtype), "keys")
        assert torch.equal(v_cache[b, :, r], v[0, :, i])
    for cache in (k_cache, v_cache):
        assert bool((cache.transpose(1, 2)[~named] == 7.0).all())
    kept = k_cache.clone()
    bad = rows.copy()
    bad[0] = cap                                                           # does not fit
    bad[1:] = -1
    S.qk_norm_rope(None, k, eps=1e-6, inv_freq=f, positions=pos, k_out=k_cache, rows=int32(bad).view(1, T), seqs=int32(seqs).view(1, T))
    expect_full(0)
    assert torch.equal(kept, k_cache)
    bad[0], seqs[0] = 3, 4                                                 # no such sequence
    S.qk_norm_rope(None, k, eps=1e-6, inv_freq=f, positions=pos, k_out=k_cache, rows=int32(bad).view(1, T), seqs=int32(seqs).view(1, T))
    expect_full(4)
    assert torch.equal(kept, k_cache)


# ---- attention over packed prompts -------------------------------------------------------------------
def packed_case(g, lens_q, lens_k, Hq, Hkv, D, dtype, tail=0, scale=1.0):
    tq, tk = sum(lens_q) + tail, sum(lens_k) + tail
    qkv = [randn(g, max(1, n), H, D, dtype=dtype, scale=scale) for n, H in ((tq, Hq), (tk, Hkv), (tk, Hkv))]
    return qkv, int32(np.cumsum([0] + list(lens_q))), int32(np.cumsum([0] + list(lens_k)))


def check_packed(q, k, v, o, lse, lens_q, lens_k, scale, causal):
    a = x = 0
    for nq, nk in zip(lens_q, lens_k):
        if nq:
            want, want_lse, weighted, size = R.attention(q[a:a + nq], k[x:x + nk], v[x:x + nk], scale=scale, causal=causal)
            D = q.shape[2]
            R.check(o[a:a + nq], want, R.attention_bound(want, weighted, size, dtype=q.dtype, weights=q.dtype, D=D, v=v[x:x + nk]), f"o of {nq} on {nk}")
            R.check(lse[:, a:a + nq], want_lse, R.lse_bound(want_lse, size, D), f"lse of {nq} on {nk}")
        a += nq
        x += nk


LENGTHS = [[1], [128], [79, 80, 81], [111, 112, 113, 15], [159, 160, 161, 223, 224, 225], [5, 0, 130, 1], [129, 127, 300, 64, 65], [31, 32, 33, 16, 17, 8, 9], [700, 3, 513], [0, 2, 0], list(range(1, 41))]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", LENGTHS)
@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(8, 2, 128, torch.bfloat16), (4, 4, 64, torch.float16), (6, 2, 128, torch.float16), (8, 1, 64, torch.bfloat16), (3, 3, 128, torch.bfloat16), (80, 80, 64, torch.bfloat16),
                                               (320, 80, 128, torch.float16)])
def test_packed(S, lens, causal, Hq, Hkv, D, dtype):
    g = rng(len(lens) * 7 + Hq)
    (q, k, v), cu, _ = packed_case(g, lens, lens, Hq, Hkv, D, dtype)
    o, lse = torch.empty_like(q), torch.empty(Hq, q.shape[0], device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=D ** -0.5, cu_seqlens_q=cu, causal=causal)
    check_packed(q, k, v, o, lse, lens, lens, D ** -0.5, causal)


@pytest.mark.parametrize("rep", [1, 2, 3, 4, 5, 6, 7, 8, 12, 16, 32])
def test_packed_groups(S, rep):
    """Every number of query heads per key head."""
    g = rng(rep)
    lens = [40, 1, 200, 129]
    (q, k, v), cu, _ = packed_case(g, lens, lens, 2 * rep, 2, 64, torch.bfloat16)
    o, lse = torch.empty_like(q), torch.empty(2 * rep, q.shape[0], device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=0.125, cu_seqlens_q=cu)
    check_packed(q, k, v, o, lse, lens, lens, 0.125, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens_q, lens_k", [([1, 5, 64], [300, 5, 1000]), ([33, 0, 7, 260], [33, 50, 1029, 515]), ([10, 200, 3], [4, 130, 0]), ([1] * 9, [1, 127, 128, 129, 255, 256, 257, 2, 0]),
                                            ([300], [1]), ([0, 0], [5, 0])])
@pytest.mark.parametrize("Hq, Hkv, D", [(8, 2, 128), (2, 2, 64)])
def test_packed_portions(S, lens_q, lens_k, causal, Hq, Hkv, D):
    """More keys than queries (a prompt's next portion), fewer (rows that see no key: zeros and -infinity), and none."""
    g = rng(sum(lens_q) + Hq)
    (q, k, v), cu_q, cu_k = packed_case(g, lens_q, lens_k, Hq, Hkv, D, torch.bfloat16)
    o, lse = torch.full_like(q, 9.0), torch.full((Hq, q.shape[0]), 9.0, device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=D ** -0.5, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, causal=causal)
    check_packed(q, k, v, o, lse, lens_q, lens_k, D ** -0.5, causal)
    if sum(lens_q) == 0:
        assert bool((o == 9.0).all()) and bool((lse == 9.0).all())


@pytest.mark.parametrize("Hq, Hkv, D", [(8, 2, 64), (40, 40, 64)])
def test_packed_many_sequences(S, Hq, Hkv, D):
    """More sequences than the planning block keeps at hand, most of them of a few tokens, some empty."""
    r = np.random.RandomState(Hq)
    lens = [int(x) for x in r.randint(0, 7, 1500)]
    lens[700], lens[1499] = 400, 90
    g = rng(Hq)
    (q, k, v), cu, _ = packed_case(g, lens, lens, Hq, Hkv, D, torch.bfloat16)
    o, lse = torch.empty_like(q), torch.empty(Hq, q.shape[0], device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=0.125, cu_seqlens_q=cu)
    check_packed(q, k, v, o, lse, lens, lens, 0.125, True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(16, 16, 64, torch.float16), (16, 16, 128, torch.bfloat16), (32, 8, 128, torch.bfloat16), (12, 4, 64, torch.bfloat16), (64, 2, 128, torch.float16),
                                               (15, 15, 64, torch.bfloat16)])
def test_packed_short_sequences(S, Hq, Hkv, D, dtype, many, causal):
    """Sequences of less than a tile, most of them, of which two blocks of heads are computed together (an odd number of blocks: not); prefixes, fewer keys than
    tokens, none, and NaN behind the last."""
    rep = Hq // Hkv
    fold = 16 if rep == 32 else 4 if rep == 4 else 1
    tile = 128 // fold
    n = 150 * fold // Hq + 2 if not many else 700 * fold // Hq + 3
    r = np.random.RandomState(Hq + D)
    lens_q = [int(x) for x in r.randint(0, tile + 1, n)]
    lens_q[0], lens_q[1] = 2 * tile + 3, 1
    lens_k = [a + int(r.choice([0, 0, 3, 117, 400])) if i % 7 else a // 2 for i, a in enumerate(lens_q)]
    lens_k[-1] = 0 if lens_q[-1] else 5
    g = rng(Hq)
    (q, k, v), cu_q, cu_k = packed_case(g, lens_q, lens_k, Hq, Hkv, D, dtype)
    k, v = (torch.cat([x, torch.full_like(x[:40], math.nan)]) for x in (k, v))
    o, lse = torch.full_like(q, 9.0), torch.full((Hq, q.shape[0]), 9.0, device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=D ** -0.5, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, causal=causal)
    check_packed(q, k, v, o, lse, lens_q, lens_k, D ** -0.5, causal)
    again = torch.zeros_like(o)
    S.prefill_packed(q, k, v, again, scale=D ** -0.5, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k, causal=causal)
    assert torch.equal(o, again)


def test_packed_workspace_of_the_largest_call(S):
    """A workspace made for a batch's most tokens serves every smaller number."""
    Hq, Hkv, D, n = 16, 16, 64, 40
    q, k = torch.empty(n * 300, Hq, D, dtype=torch.bfloat16, device=DEV), torch.empty(n * 300, Hkv, D, dtype=torch.bfloat16, device=DEV)
    workspace = S.prefill_packed_workspace(q, k, batch=n)
    for each in (300, 161, 160, 159, 128, 20, 1):
        g = rng(each)
        (q, k, v), cu, _ = packed_case(g, [each] * n, [each] * n, Hq, Hkv, D, torch.bfloat16)
        o, lse = torch.empty_like(q), torch.empty(Hq, q.shape[0], device=DEV)
        S.prefill_packed(q, k, v, o, lse, scale=0.125, cu_seqlens_q=cu, workspace=workspace)
        check_packed(q, k, v, o, lse, [each] * n, [each] * n, 0.125, True)


def test_packed_two_calls_at_once(S):
    """Two streams, a workspace each, and a graph replayed: the CTAs' counter of one call is not another's."""
    lens = [300, 7, 0, 900, 64, 513] * 5
    g = rng(21)
    (q, k, v), cu, _ = packed_case(g, lens, lens, 16, 4, 128, torch.bfloat16)
    o, lse = torch.empty_like(q), torch.empty(16, q.shape[0], device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=0.09, cu_seqlens_q=cu)
    check_packed(q, k, v, o, lse, lens, lens, 0.09, True)
    streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(q) for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for s, x in zip(streams, outs):
            S.prefill_packed(q, k, v, x, scale=0.09, cu_seqlens_q=cu, stream=s)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], o) and torch.equal(outs[1], o)
    x, workspace, graph = torch.zeros_like(q), S.prefill_packed_workspace(q, k, batch=len(lens)), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        S.prefill_packed(q, k, v, x, scale=0.09, cu_seqlens_q=cu, workspace=workspace)
        S.prefill_packed(q, k, v, x, scale=0.09, cu_seqlens_q=cu, workspace=workspace)
    for _ in range(2):
        x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(x, o)


def test_packed_no_keys_at_all(S):
    g = rng(1)
    q = randn(g, 5, 4, 64)
    k = torch.empty(0, 2, 64, dtype=torch.bfloat16, device=DEV)
    o, lse = torch.full_like(q, 9.0), torch.full((4, 5), 9.0, device=DEV)
    S.prefill_packed(q, k, k, o, lse, scale=0.1, cu_seqlens_q=int32([0, 5]), cu_seqlens_k=int32([0, 0]))
    assert not o.any() and bool((lse == -math.inf).all())


@pytest.mark.parametrize("D", [64, 128])
def test_packed_strides_and_tails(S, D):
    """q, k, v as views of one projection; NaN in every token behind the last sequence, o and lse there as they were; no lse asked for."""
    g = rng(D)
    lens, Hq, Hkv, tail = [70, 131, 1], 8, 2, 150
    total = sum(lens)
    qkv = randn(g, total + tail, Hq + 2 * Hkv, D)
    qkv[total:] = math.nan
    q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
    wide = torch.full((total + tail, Hq + 3, D), 5.0, dtype=torch.bfloat16, device=DEV)
    o, lse = wide[:, 1:1 + Hq], torch.full((Hq, total + tail), 5.0, device=DEV)
    cu = int32(np.cumsum([0] + lens))
    S.prefill_packed(q, k, v, o, lse, scale=D ** -0.5, cu_seqlens_q=cu)
    check_packed(q[:total], k[:total], v[:total], o[:total], lse[:, :total], lens, lens, D ** -0.5, True)
    assert bool((wide[:, 0] == 5.0).all()) and bool((wide[:, 1 + Hq:] == 5.0).all()) and bool((wide[total:] == 5.0).all()) and bool((lse[:, total:] == 5.0).all())
    again = torch.zeros_like(q, memory_format=torch.contiguous_format)
    S.prefill_packed(q, k, v, again, scale=D ** -0.5, cu_seqlens_q=cu)
    assert torch.equal(again[:total], o[:total])


def test_packed_sequences_do_not_reach_each_other(S):
    """A sequence whose keys and values are NaN and infinite leaves its neighbours' bits alone."""
    g = rng(3)
    lens = [60, 77, 190]
    (q, k, v), cu, _ = packed_case(g, lens, lens, 8, 2, 128, torch.bfloat16)
    clean = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu)
    k2, v2 = k.clone(), v.clone()
    k2[60:137], v2[60:137] = math.nan, math.inf
    v2[60:80] = math.nan
    got = S.prefill_packed(q, k2, v2, scale=0.09, cu_seqlens_q=cu)
    assert torch.equal(got[:60], clean[:60]) and torch.equal(got[137:], clean[137:]) and not torch.isfinite(got[60:137].float()).all()


def test_packed_short_sequences_do_not_reach_each_other(S):
    """The same where two blocks of heads are computed together; and a key head full of NaN and infinities leaves the other heads' bits alone."""
    g = rng(5)
    lens = [37, 80, 5] * 14
    (q, k, v), cu, _ = packed_case(g, lens, lens, 16, 16, 64, torch.bfloat16)
    clean = S.prefill_packed(q, k, v, scale=0.125, cu_seqlens_q=cu)
    a, b = sum(lens[:4]), sum(lens[:5])
    k2, v2 = k.clone(), v.clone()
    k2[a:b], v2[a:b] = math.nan, math.inf
    got = S.prefill_packed(q, k2, v2, scale=0.125, cu_seqlens_q=cu)
    assert torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:]) and not torch.isfinite(got[a:b].float()).any()
    k2, v2 = k.clone(), v.clone()
    k2[:, 6], v2[:, 6] = math.nan, math.inf
    got = S.prefill_packed(q, k2, v2, scale=0.125, cu_seqlens_q=cu)
    assert torch.equal(got[:, :6], clean[:, :6]) and torch.equal(got[:, 7:], clean[:, 7:]) and not torch.isfinite(got[:, 6].float()).any()


def test_packed_refuses_offsets_on_the_device(S):
    """Sequences whose offsets descend or pass the tokens given are left out; the others are computed."""
    g = rng(4)
    (q, k, v), _, _ = packed_case(g, [100], [100], 4, 2, 64, torch.bfloat16)
    for cu, whole in (([0, 30, 20, 60, 101], [(0, 30), (20, 60)]), ([-5, 10, 40, 1 << 30, 100], [(10, 40)])):
        o = torch.full_like(q, 3.0)
        S.prefill_packed(q, k, v, o, scale=0.125, cu_seqlens_q=int32(cu))
        touched = torch.zeros(100, dtype=torch.bool, device=DEV)
        for a, b in whole:
            want = S.prefill_packed(q[a:b], k[a:b], v[a:b], scale=0.125, cu_seqlens_q=int32([0, b - a]))
            touched[a:b] = True
            if (a, b) != (0, 30):                                          # (0, 30) and (20, 60) share tokens here: whichever came last stands
                assert torch.equal(o[max(a, 30):b], want[max(a, 30) - a:])
        assert bool((o[~touched] == 3.0).all())
    # the same tokens named over and over: more items than the tokens make, and nothing outside them
    q2, k2, v2 = (x.repeat(1, 40, 1).contiguous() for x in (q, k, v))
    o = torch.full_like(q2, 3.0)
    S.prefill_packed(q2, k2, v2, o, scale=0.125, cu_seqlens_q=int32([0, 100] * 300))
    want = S.prefill_packed(q2, k2, v2, scale=0.125, cu_seqlens_q=int32([0, 100]))
    assert bool(((o == want) | (o == 3.0)).all())


def test_packed_large_scores(S):
    """Scores of hundreds, of both signs, and negative scale."""
    g = rng(8)
    lens = [257, 90]
    (q, k, v), cu, _ = packed_case(g, lens, lens, 4, 2, 128, torch.bfloat16, scale=4.0)
    for scale in (1.0, -0.5, 0.0):
        o, lse = torch.empty_like(q), torch.empty(4, sum(lens), device=DEV)
        S.prefill_packed(q, k, v, o, lse, scale=scale, cu_seqlens_q=cu)
        check_packed(q, k, v, o, lse, lens, lens, scale, True)


def test_packed_long(S):
    g = rng(9)
    lens_q, lens_k = [130, 1, 2000], [9000, 20001, 2000]
    (q, k, v), cu_q, cu_k = packed_case(g, lens_q, lens_k, 8, 2, 128, torch.bfloat16)
    o, lse = torch.empty_like(q), torch.empty(8, q.shape[0], device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=128 ** -0.5, cu_seqlens_q=cu_q, cu_seqlens_k=cu_k)
    check_packed(q, k, v, o, lse, lens_q, lens_k, 128 ** -0.5, True)


# ---- the 4-bit cache -----------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B, H, T", [(1, 1, 1), (3, 2, 37), (2, 8, 200)])
def test_kv4_append_and_read(S, dtype, D, B, H, T):
    """What comes back is the formula's value, bit for bit: the scales and codes are whole numbers of both types."""
    g = rng(D + T)
    k = randn(g, B, T, H, D, dtype=dtype).transpose(1, 2)
    v = randn(g, B, T, H, D, dtype=dtype, scale=20.0).transpose(1, 2)
    v[:, :, ::3] *= 0.01
    v[:, :, ::5] = 0
    cache = S.Kv4Cache(B, H, T + 11, D, device=DEV)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.fill_(0x5A)
    cache.append(k, v, start_row=3)
    k_back, v_back = torch.empty(B, H, T, D, dtype=dtype, device=DEV), torch.empty(B, H, T, D, dtype=dtype, device=DEV)
    cache.read(k_back, v_back, start_row=3)
    assert torch.equal(k_back.double(), R.quantise(k) + 0.0) and torch.equal(v_back.double(), R.quantise(v) + 0.0)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        assert bool((t[:, :, :3] == 0x5A).all()) and bool((t[:, :, 3 + T:] == 0x5A).all())
    only = torch.empty_like(v_back)
    cache.read(None, only, start_row=3)
    assert torch.equal(only, v_back)


def test_kv4_borders(S):
    """Maxima on and next to the borders between scales, elements on and next to the borders between codes, zeros, the ends of the range, what is not finite."""
    halves = torch.tensor([1.0, 2.0 ** -6, 2.0 ** -9, 300.0], device=DEV)
    rows = []
    for s in halves:
        for m in range(8, 17):                                              # maxima 7 * (m + 1/2 +- a step) / 8 * s
            for step in (-1, 0, 1):
                top = (7 * (m + 0.5) / 8 * s).to(torch.bfloat16).float() * (1 + step * 2.0 ** -8)
                x = torch.zeros(32, device=DEV)
                x[0] = top
                x[1:16] = (torch.arange(1, 16, device=DEV) / 2) * (top / 7)
                x[16:31] = -x[1:16]
                rows.append(x)
    for value in (0.0, 1e-30, 2.0 ** -10 * 7 * 0.99, 2.0 ** -10 * 7, 3136.0, 5000.0, 1e30):
        x = torch.zeros(32, device=DEV)
        x[5], x[6] = value, -value / 2
        rows.append(x)
    for value in (math.inf, -math.inf, math.nan):
        x = torch.ones(32, device=DEV)
        x[31] = value
        rows.append(x)
    while len(rows) % 4:
        rows.append(torch.zeros(32, device=DEV))
    x = torch.stack(rows).view(1, 1, -1, 128)
    for dtype in (torch.bfloat16, torch.float16):
        y = x.to(dtype)
        cache = S.Kv4Cache(1, 1, y.shape[2], 128, device=DEV)
        cache.append(y, y)
        back = torch.empty_like(y)
        cache.read(back, None)
        want = R.quantise(y)
        assert torch.equal(torch.isnan(back), torch.isnan(want)) and torch.equal(torch.nan_to_num(back.double()), torch.nan_to_num(want) + 0.0)


def test_kv4_exponents(S):
    g = rng(12)
    k, v = randn(g, 1, 2, 9, 64, scale=1e5), randn(g, 1, 2, 9, 64, scale=1e-5)
    cache = S.Kv4Cache(1, 2, 16, 64, device=DEV, k_exponent=16, v_exponent=-16)
    cache.append(k, v)
    kb, vb = torch.empty_like(k), torch.empty_like(v)
    cache.read(kb, vb)
    assert torch.equal(kb.double(), R.quantise(k, 16) + 0.0) and torch.equal(vb.double(), R.quantise(v, -16) + 0.0)
    assert float((kb - k).abs().max() / k.abs().max()) < 0.08 and float((vb - v).abs().max() / v.abs().max()) < 0.08      # half a code step of 1/7, and the scale's rounding


def test_kv4_places(S):
    """Packed tokens into rows of their sequences: padding and places out of the cache are left out."""
    g = rng(13)
    H, D, T = 2, 128, 9
    k, v = randn(g, 1, H, T, D), randn(g, 1, H, T, D)
    cache = S.Kv4Cache(3, H, 16, D, device=DEV)
    rows, seqs = int32([0, 15, -1, 3, 4, -9, 5, 6, 7]).view(1, T), int32([2, 0, 0, 1, 1, 50, 1, 1, 1]).view(1, T)
    cache.append(k, v, rows=rows, seqs=seqs)
    back, vback = torch.full_like(k, 3.0), torch.full_like(v, 3.0)
    cache.read(back, vback, rows=rows, seqs=seqs)
    live = (rows[0] >= 0)
    assert torch.equal(back[:, :, live].double(), R.quantise(k)[:, :, live] + 0.0) and torch.equal(vback[:, :, live].double(), R.quantise(v)[:, :, live] + 0.0)
    assert bool((back[:, :, ~live] == 3.0).all())
    named = torch.zeros(3, 16, dtype=torch.bool, device=DEV)
    named[seqs[0][live].long(), rows[0][live].long()] = True
    assert not cache.k_codes.transpose(1, 2)[~named].any() and not cache.v_scales.transpose(1, 2)[~named].any()
    kept = cache.k_codes.clone()
    cache.append(k, v, rows=int32([16] + [-1] * 8).view(1, T), seqs=seqs)
    expect_full(2)
    cache.append(k, v, rows=int32([1] + [-1] * 8).view(1, T), seqs=int32([3] * 9).view(1, T))
    expect_full(3)
    cache.read(back, None, rows=int32([-1] * 8 + [1 << 30]).view(1, T), seqs=seqs)
    expect_full(1)
    assert torch.equal(kept, cache.k_codes)


# ---- decode over the 4-bit cache -------------------------------------------------------------------------
def filled_cache(S, g, B, Hkv, cap, D, dtype, lens, exponents=(0, 0), junk=True):
    """A cache whose rows hold random tokens up to lens and, behind them, codes at random with NaN scales."""
    k, v = randn(g, B, Hkv, cap, D, dtype=dtype, scale=2.0 ** exponents[0]), randn(g, B, Hkv, cap, D, dtype=dtype, scale=2.0 ** exponents[1])
    cache = S.Kv4Cache(B, Hkv, cap, D, device=DEV, k_exponent=exponents[0], v_exponent=exponents[1])
    cap = cache.cap
    rows = torch.arange(k.shape[2], device=DEV, dtype=torch.int32).expand(B, -1).contiguous()
    cache.append(k, v, rows=rows)
    if junk:
        behind = torch.arange(cap, device=DEV)[None] >= int32(lens)[:, None]
        for t in (cache.k_scales, cache.v_scales):
            t.transpose(1, 2)[behind] = 0x7F
        for t in (cache.k_codes, cache.v_codes):
            t.transpose(1, 2)[behind] = 0xF3
    return cache, R.quantise(k, exponents[0]), R.quantise(v, exponents[1])


def check_decode(q, o, lse, k, v, lens, scale, k_new=None, v_new=None, exponents=(0, 0)):
    D = q.shape[3]
    for b, n in enumerate(lens):
        kk, vv = k[b, :, :n].transpose(0, 1), v[b, :, :n].transpose(0, 1)
        if k_new is not None:
            kk = torch.cat([kk, R.quantise(k_new[b, :, 0], exponents[0])[None]])
            vv = torch.cat([vv, R.quantise(v_new[b, :, 0], exponents[1])[None]])
        want, want_lse, weighted, size = R.attention(q[b].transpose(0, 1), kk, vv, scale=scale, causal=False)
        R.check(o[b].transpose(0, 1), want, R.attention_bound(want, weighted, size, dtype=q.dtype, weights=torch.float16, D=D, v=vv), f"o of sequence {b} with {n} rows")
        R.check(lse[b][:, None], want_lse, R.lse_bound(want_lse, size, D), f"lse of sequence {b}")


def run_decode(S, g, B, Hq, Hkv, D, dtype, lens, *, append=False, cap=None, exponents=(0, 0), num_splits=0, max_len=0, q_scale=1.0, advance=False):
    cap = cap or max(lens) + 9
    cache, k, v = filled_cache(S, g, B, Hkv, cap, D, dtype, lens, exponents)
    q = randn(g, B, Hq, 1, D, dtype=dtype, scale=q_scale)
    new = [randn(g, B, Hkv, 1, D, dtype=dtype, scale=2.0 ** e) for e in exponents] if append else [None, None]
    o, lse, seq = torch.full_like(q, 9.0), torch.full((B, Hq), 9.0, device=DEV), int32(lens)
    scale = D ** -0.5 * 2.0 ** -exponents[0]
    S.decode_kv4(q, o, cache, scale=scale, k_new=new[0], v_new=new[1], lse=lse, seq_lens=seq, num_splits=num_splits, max_len=max_len, advance_lens=advance)
    check_decode(q, o, lse, k, v, lens, scale, *new, exponents=exponents)
    if append:
        kb, vb = (torch.empty_like(x) for x in new)
        cache.read(kb, vb, rows=int32(lens).view(B, 1))
        assert torch.equal(kb.double(), R.quantise(new[0], exponents[0]) + 0.0) and torch.equal(vb.double(), R.quantise(new[1], exponents[1]) + 0.0)
    assert seq.tolist() == [n + int(advance and append) for n in lens]
    return q, o, lse, cache


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("append", [False, True])
@pytest.mark.parametrize("Hq, Hkv, D, dtype", [(16, 4, 128, torch.bfloat16), (8, 8, 64, torch.float16), (8, 1, 128, torch.float16), (6, 2, 64, torch.bfloat16), (2, 1, 128, torch.bfloat16)])
def test_decode_kv4_lengths(S, append, Hq, Hkv, D, dtype):
    run_decode(S, rng(Hq + D), len(EDGES), Hq, Hkv, D, dtype, EDGES, append=append, advance=append)


@pytest.mark.parametrize("num_splits", [1, 2, 3, 7, 16, 33, 1000])
@pytest.mark.parametrize("D", [64, 128])
def test_decode_kv4_splits(S, num_splits, D):
    run_decode(S, rng(num_splits), 3, 8, 2, D, torch.bfloat16, [900, 0, 333], append=True, num_splits=num_splits)


@pytest.mark.parametrize("rep", [1, 2, 3, 4, 5, 7, 8, 9, 12, 16, 17, 32])
def test_decode_kv4_groups(S, rep):
    run_decode(S, rng(rep), 2, 2 * rep, 2, 128 if rep % 2 else 64, torch.bfloat16, [200, 77], append=True)


@pytest.mark.parametrize("lens", [[5000, 70, 12345], [40000]])
def test_decode_kv4_long(S, lens):
    run_decode(S, rng(1), len(lens), 16, 2, 128, torch.bfloat16, lens, append=True, max_len=max(lens) + 1)


@pytest.mark.parametrize("B, Hkv, most", [(1, 8, 9000), (37, 4, 1500), (1300, 1, 700), (3, 2, 40000)])
def test_decode_kv4_ragged(S, B, Hkv, most):
    """Lengths of every size in one batch, empty sequences among them, the work shared out over the device."""
    r = np.random.RandomState(B)
    lens = [int(x) for x in np.exp(r.uniform(0, math.log(most), B))]
    for i in range(0, B, 7):
        lens[i] = 0 if B > 1 else most
    lens[-1] = most
    run_decode(S, rng(B), B, 4 * Hkv, Hkv, 64, torch.bfloat16, lens, append=True, advance=True)
    run_decode(S, rng(B), B, 4 * Hkv, Hkv, 128, torch.bfloat16, lens)


def test_decode_kv4_exponents_and_large_queries(S):
    run_decode(S, rng(2), 2, 8, 2, 128, torch.bfloat16, [150, 31], append=True, exponents=(5, -7))
    run_decode(S, rng(3), 2, 8, 2, 128, torch.bfloat16, [150, 31], q_scale=30.0)
    run_decode(S, rng(4), 2, 8, 2, 64, torch.bfloat16, [150, 31], exponents=(-30, 10), append=True)


def test_decode_kv4_query_range(S):
    """Queries far beyond and below fp16's range: the scores are those of fp32."""
    g = rng(5)
    cache, k, v = filled_cache(S, g, 1, 2, 100, 128, torch.bfloat16, [90])
    base = randn(g, 1, 8, 1, 128)
    for size in (2.0 ** 40, 2.0 ** -40):
        q = base * size
        o, lse = torch.empty_like(q), torch.empty(1, 8, device=DEV)
        S.decode_kv4(q, o, cache, scale=0.1 / size, lse=lse, uniform_len=90)
        check_decode(q, o, lse, k, v, [90], 0.1 / size)
    zero = torch.zeros_like(base)
    o, lse = torch.empty_like(zero), torch.empty(1, 8, device=DEV)
    S.decode_kv4(zero, o, cache, scale=0.1, lse=lse, uniform_len=90)
    check_decode(zero, o, lse, k, v, [90], 0.1)
    bad = base.clone()
    bad[0, 3, 0, 7] = math.nan
    S.decode_kv4(bad, o, cache, scale=0.1, lse=lse, uniform_len=90)
    assert torch.isnan(o[0, 3]).all() and torch.isfinite(o[0, [0, 1, 2, 4, 5, 6, 7]].float()).all()


def test_decode_kv4_nan_rows(S):
    """A live row that holds NaN makes its sequence's key head NaN and nothing else."""
    g = rng(6)
    cache, _, _ = filled_cache(S, g, 2, 2, 128, 128, torch.bfloat16, [100, 100])
    cache.v_scales[1, 0, 50, :] = 0x7F
    q = randn(g, 2, 8, 1, 128)
    o = torch.empty_like(q)
    S.decode_kv4(q, o, cache, scale=0.1, seq_lens=int32([100, 100]))
    assert torch.isnan(o[1, :4]).all() and torch.isfinite(o[0].float()).all() and torch.isfinite(o[1, 4:].float()).all()


def test_decode_kv4_full_sequences(S):
    """A token that does not fit is not written and its length stays; the sequence attends to what it has."""
    g = rng(7)
    lens = [64, 63, 10]
    cache, k, v = filled_cache(S, g, 3, 2, 64, 128, torch.bfloat16, lens)
    q, kn, vn = randn(g, 3, 8, 1, 128), randn(g, 3, 2, 1, 128), randn(g, 3, 2, 1, 128)
    o, lse, seq = torch.empty_like(q), torch.empty(3, 8, device=DEV), int32(lens)
    before = cache.k_codes[0].clone()
    S.decode_kv4(q, o, cache, scale=0.1, k_new=kn, v_new=vn, lse=lse, seq_lens=seq, advance_lens=True)
    expect_full(0)
    assert seq.tolist() == [64, 64, 11] and torch.equal(before, cache.k_codes[0])
    check_decode(q[:1], o[:1], lse[:1], k[:1], v[:1], [64], 0.1)
    check_decode(q[1:], o[1:], lse[1:], k[1:], v[1:], [63, 10], 0.1, kn[1:], vn[1:])
    for bad in (-3, 2 ** 31 - 1):
        seq = int32([5, bad, 6])
        S.decode_kv4(q, o, cache, scale=0.1, k_new=kn, v_new=vn, seq_lens=seq, advance_lens=True)
        expect_full(1)
        assert seq.tolist() == [6, bad, 7]


def test_decode_kv4_strides(S):
    """A cache whose heads stand apart, more sequences in it than the call has, queries and new rows as views of one projection."""
    g = rng(8)
    B, Hq, Hkv, D, cap = 3, 8, 2, 128, 80
    lens = [70, 1, 33]
    whole, k, v = filled_cache(S, g, 5, 3, cap, D, torch.bfloat16, lens + [0, 0])
    part = S.Kv4Cache(k_codes=whole.k_codes[:, 1:], v_codes=whole.v_codes[:, 1:], k_scales=whole.k_scales[:, 1:], v_scales=whole.v_scales[:, 1:])
    qkv = randn(g, B, 1, Hq + 2 * Hkv, D)
    q, kn, vn = (x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], dim=2))
    o, lse = torch.empty(B, 1, Hq, D, dtype=q.dtype, device=DEV).transpose(1, 2), torch.empty(B, Hq, device=DEV)
    S.decode_kv4(q, o, part, scale=0.1, k_new=kn, v_new=vn, lse=lse, seq_lens=int32(lens))
    check_decode(q, o, lse, k[:, 1:], v[:, 1:], lens, 0.1, kn, vn)


# ---- streams, graphs, workspaces ---------------------------------------------------------------------------
def test_operators_on_another_stream(S):
    g = rng(20)
    lens = [200, 50]
    (q, k, v), cu, _ = packed_case(g, lens, lens, 8, 2, 128, torch.bfloat16)
    want = S.prefill_packed(q, k, v, scale=0.1, cu_seqlens_q=cu)
    cache, _, _ = filled_cache(S, g, 2, 2, 256, 128, torch.bfloat16, lens)
    qd = randn(g, 2, 8, 1, 128)
    want_d = S.decode_kv4(qd, torch.empty_like(qd), cache, scale=0.1, seq_lens=int32(lens))
    seq = int32(lens)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got, got_d = torch.empty_like(q), torch.empty_like(qd)
    S.prefill_packed(q, k, v, got, scale=0.1, cu_seqlens_q=cu, stream=side)
    S.decode_kv4(qd, got_d, cache, scale=0.1, seq_lens=seq, stream=side)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(got_d, want_d)


def test_operators_in_a_graph(S):
    """A captured step replays on what its buffers hold: lengths advance, prompts of other lengths come through the same offsets."""
    g = rng(21)
    B, Hq, Hkv, D, cap = 2, 8, 2, 128, 128
    lens = [60, 3]
    cache, k, v = filled_cache(S, g, B, Hkv, cap, D, torch.bfloat16, lens)
    qkv = randn(g, B, 1, Hq + 2 * Hkv, D)
    q, kn, vn = (x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], dim=2))
    qo, ko = torch.empty(B, Hq, 1, D, dtype=q.dtype, device=DEV), torch.empty(B, Hkv, 1, D, dtype=q.dtype, device=DEV)
    o, seq = torch.empty_like(qo), int32(lens)
    ws = S.decode_kv4_workspace(qo, cache)

    def step():
        S.qk_norm_rope(q, kn, eps=1e-6, theta=THETA, positions=seq.view(B, 1), q_out=qo, k_out=ko)
        S.decode_kv4(qo, o, cache, scale=0.1, k_new=ko, v_new=vn, seq_lens=seq, advance_lens=True, workspace=ws)

    total, pq = 300, randn(g, 300, Hq, D)
    pk, pv = randn(g, total, Hkv, D), randn(g, total, Hkv, D)
    po, cu = torch.zeros_like(pq), int32([0, 100, 300])
    pws = S.prefill_packed_workspace(pq, pk, batch=2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        step()
        S.prefill_packed(pq, pk, pv, po, scale=0.1, cu_seqlens_q=cu, workspace=pws)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step()
        S.prefill_packed(pq, pk, pv, po, scale=0.1, cu_seqlens_q=cu, workspace=pws)
    seq.copy_(int32(lens))
    outs = []
    for i in range(3):
        qkv.copy_(randn(g, *qkv.shape))
        cu[1] = 100 - 40 * i
        ws.fill_(0xFF)
        pws.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        outs.append((qkv.clone(), o.clone(), po.clone()))
    assert seq.tolist() == [63, 6]
    eager, _, _ = filled_cache(S, rng(21), B, Hkv, cap, D, torch.bfloat16, lens)
    seq.copy_(int32(lens))
    for i, (x, want, packed) in enumerate(outs):
        qkv.copy_(x)
        S.qk_norm_rope(q, kn, eps=1e-6, theta=THETA, positions=seq.view(B, 1), q_out=qo, k_out=ko)
        S.decode_kv4(qo, o, eager, scale=0.1, k_new=ko, v_new=vn, seq_lens=seq, advance_lens=True)
        assert torch.equal(o, want)
        n = 100 - 40 * i
        assert torch.equal(packed, S.prefill_packed(pq, pk, pv, scale=0.1, cu_seqlens_q=int32([0, n, 300])))


def test_results_repeat(S):
    """The same call gives the same bits: nothing depends on the order in which blocks finish."""
    g = rng(22)
    lens = [900, 1, 333, 40]
    (q, k, v), cu, _ = packed_case(g, lens, lens, 16, 4, 128, torch.bfloat16)
    first = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu)
    cache, _, _ = filled_cache(S, g, 4, 4, 904, 128, torch.bfloat16, lens)
    qd = randn(g, 4, 16, 1, 128)
    first_d = S.decode_kv4(qd, torch.empty_like(qd), cache, scale=0.09, seq_lens=int32(lens))
    for _ in range(5):
        assert torch.equal(first, S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu))
        assert torch.equal(first_d, S.decode_kv4(qd, torch.empty_like(qd), cache, scale=0.09, seq_lens=int32(lens)))


# ---- as they are used together -------------------------------------------------------------------------------
def test_prompts_then_tokens(S):
    """Packed prompts through norm, rotation, attention and the 4-bit cache, then three decode steps: every output against 64 bits computed from what the
    operators before it handed on."""
    from vesper_b200 import capi
    g = rng(30)
    lens, Hq, Hkv, D, cap = [40, 0, 131, 7], 8, 2, 128, 160
    total, B, scale = sum(lens), 4, 128 ** -0.5
    f = list(capi.inv_freq(THETA, D))
    qw, kw = 1 + 0.2 * randn(g, D, dtype=torch.float32), 1 + 0.2 * randn(g, D, dtype=torch.float32)
    qkv = randn(g, total, Hq + 2 * Hkv, D)
    q, k, v = qkv.split([Hq, Hkv, Hkv], dim=1)
    pos = int32(np.concatenate([np.arange(n) for n in lens])).view(1, total)
    seqs = int32(np.repeat(np.arange(B), lens)).view(1, total)
    four = lambda x: x.transpose(0, 1).unsqueeze(0)  # noqa: E731
    raw_q, raw_k = four(q).clone(), four(k).clone()
    S.qk_norm_rope(four(q), four(k), eps=1e-6, q_weight=qw, k_weight=kw, theta=THETA, positions=pos)
    for got, x, w in ((four(q), raw_q, qw), (four(k), raw_k, kw)):
        want = R.norm_rope(x, eps=1e-6, weight=w, positions=pos, inv_freq=f)
        R.check(got, want, norm_bound(want, q.dtype), "prompt norm")
    o, lse = torch.empty(total, Hq, D, dtype=q.dtype, device=DEV), torch.empty(Hq, total, device=DEV)
    S.prefill_packed(q, k, v, o, lse, scale=scale, cu_seqlens_q=int32(np.cumsum([0] + lens)))
    check_packed(q, k, v, o, lse, lens, lens, scale, True)
    cache = S.Kv4Cache(B, Hkv, cap, D, device=DEV)
    cache.append(four(k), four(v), rows=pos, seqs=seqs)
    held_k, held_v = torch.zeros(B, Hkv, cap, D, dtype=torch.float64, device=DEV), torch.zeros(B, Hkv, cap, D, dtype=torch.float64, device=DEV)
    at = 0
    for b, n in enumerate(lens):
        held_k[b, :, :n], held_v[b, :, :n] = R.quantise(k[at:at + n].transpose(0, 1)), R.quantise(v[at:at + n].transpose(0, 1))
        at += n
    seq, now = int32(lens), list(lens)
    for _ in range(3):
        step = randn(g, B, 1, Hq + 2 * Hkv, D)
        sq, sk, sv = (x.transpose(1, 2) for x in step.split([Hq, Hkv, Hkv], dim=2))
        S.qk_norm_rope(sq, sk, eps=1e-6, q_weight=qw, k_weight=kw, theta=THETA, positions=seq.view(B, 1))
        so, sl = torch.empty(B, Hq, 1, D, dtype=q.dtype, device=DEV), torch.empty(B, Hq, device=DEV)
        S.decode_kv4(sq, so, cache, scale=scale, k_new=sk, v_new=sv, lse=sl, seq_lens=seq, advance_lens=True, max_len=max(now) + 1)
        check_decode(sq, so, sl, held_k, held_v, now, scale, sk, sv)
        for b in range(B):
            held_k[b, :, now[b]], held_v[b, :, now[b]] = R.quantise(sk[b, :, 0]), R.quantise(sv[b, :, 0])
        now = [n + 1 for n in now]
        assert seq.tolist() == now

"""Operators of a serving batch: norms of queries and keys with the position rotation, attention over packed prompts, and a key / value
cache held in 4 bits with the attention that reads it.

listed() names cases, draw() takes another one of the same ranges, prepare() holds what a program has in hand before the call, run() makes one
pass (the framework's operators where `own` is true, else their plain form in 32-bit torch), and exact() states the same results in 64 bits."""
import math
import random

import numpy as np
import torch

own = False

GROUP = 32                      # elements of a cached row that share a scale
EPS, THETA = 1e-6, 10000.0
CODE_MAX, SCALE_MAX = 7.0, 448.0


def listed():
    return [
        # one decode step of a batch of eight: heads of the 24-layer decoder, latency alone
        _norm("norm_step", "bfloat16", 8, 1, 16, 4, 128, 2048, True),
        # an odd number of packed prompt tokens, queries and keys to plain tensors for the attention behind them
        _norm("norm_packed", "bfloat16", 1, 8191, 32, 8, 128, 0, False),
        # a batch of prompts behind 1000 tokens, keys and values into the cache, heads of 64
        _norm("norm_cache", "float16", 4, 2048, 32, 8, 64, 1000, True),
        # eight short requests in one call
        _packed("packed_short", "bfloat16", 8, 5, 96, 0, 0, 16, 4, 128, True),
        # a serving batch's prompts, from a word to a long document
        _packed("packed_mixed", "bfloat16", 24, 16, 4096, 0, 0, 32, 8, 128, True),
        # long prompts in portions: new tokens behind what the sequences hold already
        _packed("packed_portions", "bfloat16", 4, 1024, 4096, 2048, 16384, 32, 8, 128, True),
        # bidirectional rows of an embedding model, one key head per query head
        _packed("packed_both_ways", "float16", 40, 20, 512, 0, 0, 16, 16, 64, False),
        # prompts into the 4-bit cache, and the rows read back
        _append("kv4_prompts", "bfloat16", 12, 64, 4096, 8, 128),
        # a step's new tokens into the 4-bit cache, and the rows read back
        _append("kv4_token", "bfloat16", 32, 1, 1, 8, 128),
        # one user's next token behind a short prompt, appended and attended to
        _decode("kv4_step", "bfloat16", 1, 300, 300, 16, 4, 128, True),
        # a serving batch with contexts of every length
        _decode("kv4_ragged", "bfloat16", 32, 1024, 8192, 32, 8, 128, False),
        # one sequence with a very long context
        _decode("kv4_long", "bfloat16", 1, 131072, 131072, 64, 8, 128, False),
    ]


def draw(rng):
    """One more case: sizes log-uniform over their ranges, so that most are odd."""
    log = lambda lo, hi: int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))  # noqa: E731
    kind = rng.choice(["norm", "packed", "packed", "append", "decode", "decode"])
    most = {c["kind"]: 0 for c in listed()}
    for c in listed():
        most[c["kind"]] = max(most[c["kind"]], _cost(c))
    while True:
        dtype, D, hkv = rng.choice(["bfloat16", "bfloat16", "float16"]), rng.choice([64, 128, 128]), rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 3, 4, 8])
        if kind == "norm":
            c = _norm("", rng.choice([dtype, dtype, "float32"]), log(1, 32), log(1, 8192), hq, hkv, D, log(1, 100000), rng.random() < 0.5)
            fits = c["start"] + c["T"] <= 120000 and c["B"] * (c["start"] + c["T"]) * hkv * D <= 2 ** 29
        elif kind == "packed":
            lo = log(1, 2048)
            prefix = log(1, 16384) if rng.random() < 0.4 else 0
            c = _packed("", dtype, log(1, 64), lo, min(16384, lo * log(1, 64)), prefix // 4, prefix, hq, hkv, D, rng.random() < 0.75)
            fits = sum(_lens(c)[1]) <= 131072
        elif kind == "append":
            lo = log(1, 2048)
            c = _append("", dtype, log(1, 64), lo, min(16384, lo * log(1, 16)), hkv, D)
            fits = c["B"] * c["hi"] <= 131072
        else:
            lo = log(1, 65536)
            c = _decode("", dtype, log(1, 64), lo, min(131072, lo * log(1, 16)), hq, hkv, D, rng.random() < 0.5)
            fits = c["B"] * c["hi"] * hkv <= 2 ** 21 + 2 ** 18
        if fits and _cost(c) <= most[kind]:
            del c["name"]
            c["lens_seed"] = rng.randrange(10 ** 6)
            if _cost(c) <= most[kind]:
                return c


def prepare(case, seed):
    return {"norm": _prepare_norm, "packed": _prepare_packed, "append": _prepare_append, "decode": _prepare_decode}[case["kind"]](case, seed)


def run(state):
    return state["own" if own else "plain"](state)


def exact(case, seed):
    state = prepare(case, seed)
    return {"norm": _exact_norm, "packed": _exact_packed, "append": _exact_append, "decode": _exact_decode}[case["kind"]](case, state)


def work(case):
    """Bytes and operations a pass cannot do without: inputs read once, outputs written once, products of visible pairs."""
    c = case
    size = 4 if c["dtype"] == "float32" else 2
    if c["kind"] == "norm":
        rows = c["B"] * c["T"]
        heads = c["heads"] + c["kv_heads"] * (2 if c["scatter"] else 1)
        return {"bytes": 2 * rows * heads * c["D"] * size + 4 * rows, "flops": 8 * rows * (c["heads"] + c["kv_heads"]) * c["D"]}
    if c["kind"] == "packed":
        lq, lk = _lens(c)
        pairs = sum(q * k - (q * (q - 1) // 2 if c["causal"] else 0) for q, k in zip(lq, lk))
        moved = 2 * c["D"] * (2 * sum(lq) * c["heads"] + 2 * sum(lk) * c["kv_heads"]) + 4 * sum(lq) * c["heads"]
        return {"bytes": moved, "flops": 4 * c["D"] * c["heads"] * pairs}
    row = c["D"] // 2 + c["D"] // GROUP
    if c["kind"] == "append":
        rows = sum(_lens(c)[0]) * c["kv_heads"] * 2
        return {"bytes": rows * (4 * c["D"] + 2 * row), "flops": 6 * rows * c["D"]}
    keys = sum(_lens(c)[0])
    moved = 2 * keys * c["kv_heads"] * row + 4 * c["B"] * c["heads"] * c["D"]
    if c["append"]:
        moved += 4 * c["B"] * c["kv_heads"] * (2 * c["D"] + row)
    return {"bytes": moved, "flops": 4 * c["D"] * c["heads"] * keys}


def _cost(c):
    w = work(c)
    return w["flops"] / 2e15 + w["bytes"] / 7e12


def _norm(name, dtype, B, T, heads, kv_heads, D, start, scatter):
    return dict(name=name, kind="norm", dtype=dtype, B=B, T=T, heads=heads, kv_heads=kv_heads, D=D, start=start, scatter=scatter, lens_seed=0)


def _packed(name, dtype, B, lo, hi, prefix_lo, prefix_hi, heads, kv_heads, D, causal):
    return dict(name=name, kind="packed", dtype=dtype, B=B, lo=lo, hi=hi, prefix_lo=prefix_lo, prefix_hi=prefix_hi, heads=heads, kv_heads=kv_heads, D=D,
                causal=causal, lens_seed=0)


def _append(name, dtype, B, lo, hi, kv_heads, D):
    return dict(name=name, kind="append", dtype=dtype, B=B, lo=lo, hi=hi, kv_heads=kv_heads, D=D, lens_seed=0)


def _decode(name, dtype, B, lo, hi, heads, kv_heads, D, append):
    return dict(name=name, kind="decode", dtype=dtype, B=B, lo=lo, hi=hi, heads=heads, kv_heads=kv_heads, D=D, append=append, lens_seed=0)


def _lens(c):
    """Lengths of the case's sequences: (new tokens, keys); prompts log-uniform, contexts of a decode step uniform.  One empty sequence per dozen prompts."""
    r = random.Random(1000003 * c["lens_seed"] + c["B"])
    if c["kind"] == "decode":
        got = [r.randint(c["lo"], c["hi"]) for _ in range(c["B"])]
        return got, got
    new = [min(c["hi"], max(c["lo"], int(round(math.exp(r.uniform(math.log(c["lo"]), math.log(c["hi"]))))))) for _ in range(c["B"])]
    for i in range(11, c["B"], 12):
        if c["kind"] == "packed":
            new[i] = 0
    prefix = [r.randint(c["prefix_lo"], c["prefix_hi"]) if c.get("prefix_hi") else 0 for _ in range(c["B"])]
    return new, [a + b if a else 0 for a, b in zip(new, prefix)]


def _rng(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def _dtype(case):
    return getattr(torch, case["dtype"])


def _int32(values):
    return torch.tensor(np.asarray(values, dtype=np.int32), device="cuda")


# ---- norms of queries and keys with the rotation --------------------------------------------------
def _prepare_norm(c, seed):
    g, t = _rng(seed), _dtype(c)
    B, T, D, hq, hkv = c["B"], c["T"], c["D"], c["heads"], c["kv_heads"]
    qkv = _randn(g, (B, T, hq + 2 * hkv, D), t)                         # what the projection wrote
    q, k, v = (x.transpose(1, 2) for x in qkv.split([hq, hkv, hkv], dim=2))
    s = dict(q=q, k=k, v=v, qw=1 + 0.2 * torch.randn(D, generator=g, device="cuda"), kw=1 + 0.2 * torch.randn(D, generator=g, device="cuda"))
    s["inv_freq"] = (THETA ** (-2.0 * np.arange(D // 2) / D)).astype(np.float32)
    first = torch.randint(0, c["start"] + 1, (B, 1), generator=g, device="cuda", dtype=torch.int64)
    s["positions"] = (first + torch.arange(T, device="cuda")).to(torch.int32)
    s["q_out"] = torch.empty(B, T, hq, D, dtype=t, device="cuda").transpose(1, 2)
    if c["scatter"]:
        cap = c["start"] + T
        s["k_out"], s["v_out"] = (torch.zeros(B, hkv, cap, D, dtype=t, device="cuda") for _ in range(2))
    else:
        s["k_out"], s["v_out"] = torch.empty(B, T, hkv, D, dtype=t, device="cuda").transpose(1, 2), None
    s["own"], s["plain"] = _own_norm, _plain_norm
    return s


def _own_norm(s):
    from vesper_b200 import serving_capi as serving
    scatter = s["v_out"] is not None
    serving.qk_norm_rope(s["q"], s["k"], s["v"] if scatter else None, q_weight=s["qw"], k_weight=s["kw"], eps=EPS, inv_freq=s["inv_freq"],
                         positions=s["positions"], q_out=s["q_out"], k_out=s["k_out"], v_out=s["v_out"], rows=s["positions"] if scatter else None)
    return [s["q_out"], s["k_out"]] + ([s["v_out"]] if scatter else [])


def _plain_norm(s):
    angle = s["positions"].double()[:, None, :, None] * torch.from_numpy(s["inv_freq"]).to("cuda").double()
    cos, sin = angle.cos().float(), angle.sin().float()

    def one(x, w):
        y = x.float()
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * w
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2).to(x.dtype)

    s["q_out"].copy_(one(s["q"], s["qw"]))
    k = one(s["k"], s["kw"])
    if s["v_out"] is None:
        s["k_out"].copy_(k)
        return [s["q_out"], s["k_out"]]
    at = s["positions"].long()[:, None, :, None].expand(k.shape)
    s["k_out"].scatter_(2, at, k)
    s["v_out"].scatter_(2, at, s["v"])
    return [s["q_out"], s["k_out"], s["v_out"]]


def _exact_norm(c, s):
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                       s["positions"].double().unsqueeze(-1) * torch.tensor(s["inv_freq"], dtype=torch.float64, device="cuda")).unsqueeze(1)

    def one(x, w):
        y = x.double()
        y = y / torch.sqrt(y.square().sum(-1, keepdim=True) / y.shape[-1] + EPS) * w.double()
        return torch.view_as_real(torch.view_as_complex(y.reshape(y.shape[:-1] + (-1, 2)).contiguous()) * turn).reshape(y.shape)

    q, k = one(s["q"], s["qw"]), one(s["k"], s["kw"])
    if not c["scatter"]:
        return [q, k]
    kc, vc = s["k_out"].double(), s["v_out"].double()
    for b in range(c["B"]):
        p = int(s["positions"][b, 0])
        kc[b, :, p:p + c["T"]] = k[b]
        vc[b, :, p:p + c["T"]] = s["v"][b].double()
    return [q, kc, vc]


# ---- attention over packed prompts -----------------------------------------------------------------
def _prepare_packed(c, seed):
    g, t = _rng(seed), _dtype(c)
    lq, lk = _lens(c)
    s = dict(q=_randn(g, (sum(lq), c["heads"], c["D"]), t), k=_randn(g, (sum(lk), c["kv_heads"], c["D"]), t), v=_randn(g, (sum(lk), c["kv_heads"], c["D"]), t))
    s["lens"], s["causal"], s["scale"] = (lq, lk), c["causal"], c["D"] ** -0.5
    s["cu_q"], s["cu_k"] = _int32(np.cumsum([0] + lq)), _int32(np.cumsum([0] + lk))
    s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty(c["heads"], sum(lq), device="cuda")
    if own:
        from vesper_b200 import serving_capi as serving
        s["workspace"] = serving.prefill_packed_workspace(s["q"], s["k"], batch=c["B"])
    s["own"], s["plain"] = _own_packed, _plain_packed
    return s


def _own_packed(s):
    from vesper_b200 import serving_capi as serving
    serving.prefill_packed(s["q"], s["k"], s["v"], s["o"], s["lse"], scale=s["scale"], cu_seqlens_q=s["cu_q"], cu_seqlens_k=s["cu_k"], causal=s["causal"],
                           workspace=s["workspace"])
    return [s["o"], s["lse"]]


def _plain_packed(s):
    q, k, v, o, lse = s["q"], s["k"], s["v"], s["o"], s["lse"]
    hkv, rep = k.shape[1], q.shape[1] // k.shape[1]
    at_q = at_k = 0
    for nq, nk in zip(*s["lens"]):
        kk, vv = (x[at_k:at_k + nk].float().transpose(0, 1) for x in (k, v))                            # [Hkv, nk, D]
        most = max(1, min(nq, 2 ** 28 // max(1, q.shape[1] * nk)))
        for r0 in range(0, nq, most):
            r1 = min(nq, r0 + most)
            qq = q[at_q + r0:at_q + r1].float().reshape(r1 - r0, hkv, rep, -1).permute(1, 2, 0, 3).flatten(1, 2)      # [Hkv, rep * rows, D]
            p = (qq @ kk.transpose(1, 2)) * s["scale"]
            if s["causal"]:
                last = torch.arange(r0, r1, device="cuda") + (nk - nq)
                p.view(hkv, rep, r1 - r0, nk).masked_fill_(torch.arange(nk, device="cuda") > last[:, None], -math.inf)
            m = p.amax(-1, keepdim=True)
            p = torch.exp(p - m)
            l = p.sum(-1, keepdim=True)
            got = ((p @ vv) / l).view(hkv, rep, r1 - r0, -1).permute(2, 0, 1, 3).flatten(1, 2)
            o[at_q + r0:at_q + r1] = got.to(o.dtype)
            lse[:, at_q + r0:at_q + r1] = (m + torch.log(l)).view(hkv * rep, r1 - r0)
        at_q += nq
        at_k += nk
    return [o, lse]


def _exact_packed(c, s):
    q, k, v = (s[n].double() for n in "qkv")
    o, lse = torch.zeros_like(q), torch.zeros(q.shape[1], q.shape[0], dtype=torch.float64, device="cuda")
    ends_q, ends_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for h in range(c["heads"]):
        g = h * c["kv_heads"] // c["heads"]
        for a, b, x, y in zip(ends_q, ends_q[1:], ends_k, ends_k[1:]):
            for i in range(a, b, 4096):
                j = min(b, i + 4096)
                score = torch.einsum("id,jd->ij", q[i:j, h], k[x:y, g]) * s["scale"]
                if c["causal"]:
                    seen = torch.ones_like(score, dtype=torch.bool).tril(diagonal=(y - x) - (b - a) + (i - a))
                    score = torch.where(seen, score, torch.full_like(score, -math.inf))
                lse[h, i:j] = torch.logsumexp(score, 1)
                o[i:j, h] = torch.softmax(score, 1) @ v[x:y, g]
    return [o, lse]


# ---- the 4-bit cache ---------------------------------------------------------------------------------
# A row of D elements: groups of 32 with scale s = e4m3(max|x| / 7) and codes c = sign(x) * min(7, floor(|x| / s + 1/2)); byte j holds the codes of
# elements 2j (low half) and 2j + 1 (high half), each plus 8; then D / 32 bytes of scales in an array of their own.
def _quantise(x):
    """codes (whole numbers in 32-bit floats) and scales of [..., D] rows."""
    y = x.float().unflatten(-1, (-1, GROUP))
    s = (y.abs().amax(-1).double() / CODE_MAX).clamp(max=SCALE_MAX).float().to(torch.float8_e4m3fn).float()      # 64 bits: many maxima lie on a border
    c = torch.where(s[..., None] > 0, torch.floor(y.abs() / s[..., None] + 0.5).clamp(max=CODE_MAX), torch.zeros_like(y))
    return (torch.sign(y) * c).flatten(-2), s


def _pack(codes, scales):
    n = (codes + 8).to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4), scales.to(torch.float8_e4m3fn).view(torch.uint8)


def _unpack(codes, scales):
    n = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2).float() - 8
    return (n.unflatten(-1, (-1, GROUP)) * scales.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _empty_cache(B, hkv, cap, D):
    make = lambda n: torch.zeros(B, hkv, cap, n, dtype=torch.uint8, device="cuda")  # noqa: E731
    return dict(k_codes=make(D // 2), v_codes=make(D // 2), k_scales=make(D // GROUP), v_scales=make(D // GROUP))


def _handle(s):
    if own:
        from vesper_b200 import serving_capi as serving
        s["handle"] = serving.Kv4Cache(**s["cache"])


def _prepare_append(c, seed):
    g, t = _rng(seed), _dtype(c)
    lens, D, hkv = _lens(c)[0], c["D"], c["kv_heads"]
    total, cap = sum(lens), (c["hi"] + 500 + 7) // 8 * 8
    wide = torch.exp(0.5 * torch.randn(hkv, 1, D, generator=g, device="cuda"))                  # some channels of keys are wider than others
    s = dict(k=(torch.randn(1, hkv, total, D, generator=g, device="cuda") * wide).to(t), v=_randn(g, (1, hkv, total, D), t))
    start = [int(x) for x in torch.randint(0, 501, (c["B"],), generator=g, device="cuda")]
    s["rows"] = _int32(np.concatenate([np.arange(n) + a for n, a in zip(lens, start)])[None])
    s["seqs"] = _int32(np.repeat(np.arange(c["B"]), lens)[None])
    s["cache"] = _empty_cache(c["B"], hkv, cap, D)
    s["k_back"], s["v_back"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    _handle(s)
    s["own"], s["plain"] = _own_append, _plain_append
    return s


def _own_append(s):
    s["handle"].append(s["k"], s["v"], rows=s["rows"], seqs=s["seqs"])
    s["handle"].read(s["k_back"], s["v_back"], rows=s["rows"], seqs=s["seqs"])
    return [s["k_back"], s["v_back"]]


def _plain_append(s):
    at = (s["seqs"][0].long(), slice(None), s["rows"][0].long())
    for n in "kv":
        codes, scales = _pack(*_quantise(s[n][0].transpose(0, 1)))
        s["cache"][n + "_codes"][at], s["cache"][n + "_scales"][at] = codes, scales
        s[n + "_back"][0] = _unpack(s["cache"][n + "_codes"][at], s["cache"][n + "_scales"][at]).transpose(0, 1).to(s[n].dtype)
    return [s["k_back"], s["v_back"]]


def _nearest_scale(x):
    """The nearest number of 4 significant bits, 2^-9 its smallest step, ties to even: e4m3 in 64 bits."""
    step = torch.exp2(torch.floor(torch.log2(x.clamp(min=2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(max=448.0)


def _exact_rows(x):
    y = x.double().reshape(x.shape[:-1] + (-1, GROUP))
    s = _nearest_scale(y.abs().max(-1, keepdim=True).values / 7)
    near = torch.where(s > 0, y.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(y))
    return (torch.copysign((near + 0.5).floor().clamp(max=7), y) * s).reshape(x.shape)


def _exact_append(c, s):
    return [_exact_rows(s["k"]), _exact_rows(s["v"])]


def _prepare_decode(c, seed):
    g, t = _rng(seed), _dtype(c)
    lens, D, hkv, B = _lens(c)[0], c["D"], c["kv_heads"], c["B"]
    cap = (max(lens) + 1 + 7) // 8 * 8
    s = dict(cache=_empty_cache(B, hkv, cap, D), lens=lens, scale=D ** -0.5)
    wide = torch.exp(0.5 * torch.randn(hkv, 1, D, generator=g, device="cuda"))
    for b in range(B):
        for n in "kv":
            x = torch.randn(hkv, lens[b], D, generator=g, device="cuda")
            s["cache"][n + "_codes"][b, :, :lens[b]], s["cache"][n + "_scales"][b, :, :lens[b]] = _pack(*_quantise(x * wide if n == "k" else x))
    s["q"] = _randn(g, (B, c["heads"], 1, D), t)
    s["k_new"], s["v_new"] = (_randn(g, (B, hkv, 1, D), t) for _ in range(2)) if c["append"] else (None, None)
    s["seq_lens"] = _int32(lens)
    s["rows"] = _int32(lens).view(B, 1)
    s["max_len"] = max(lens) + int(c["append"])
    s["o"], s["lse"] = torch.empty_like(s["q"]), torch.empty(B, c["heads"], device="cuda")
    s["k_back"], s["v_back"] = (torch.empty(B, hkv, 1, D, dtype=t, device="cuda") for _ in range(2))
    _handle(s)
    if own:
        from vesper_b200 import serving_capi as serving
        s["workspace"] = serving.decode_kv4_workspace(s["q"], s["handle"], max_len=s["max_len"])
    s["own"], s["plain"] = _own_decode, _plain_decode
    return s


def _own_decode(s):
    from vesper_b200 import serving_capi as serving
    serving.decode_kv4(s["q"], s["o"], s["handle"], scale=s["scale"], k_new=s["k_new"], v_new=s["v_new"], lse=s["lse"], seq_lens=s["seq_lens"],
                       max_len=s["max_len"], workspace=s["workspace"])
    if s["k_new"] is None:
        return [s["o"], s["lse"]]
    s["handle"].read(s["k_back"], s["v_back"], rows=s["rows"])
    return [s["o"], s["lse"], s["k_back"], s["v_back"]]


def _plain_decode(s):
    q, o, lse, cache = s["q"], s["o"], s["lse"], s["cache"]
    hkv = cache["k_codes"].shape[1]
    for b, n in enumerate(s["lens"]):
        if s["k_new"] is not None:
            for x in "kv":
                codes, scales = _pack(*_quantise(s[x + "_new"][b, :, 0]))
                cache[x + "_codes"][b, :, n], cache[x + "_scales"][b, :, n] = codes, scales
                s[x + "_back"][b, :, 0] = _unpack(codes, scales).to(q.dtype)
            n += 1
        k, v = (_unpack(cache[x + "_codes"][b, :, :n], cache[x + "_scales"][b, :, :n]) for x in "kv")
        p = (q[b].float().view(hkv, -1, q.shape[-1]) @ k.transpose(1, 2)) * s["scale"]                 # [Hkv, rep, n]
        m = p.amax(-1, keepdim=True)
        p = torch.exp(p - m)
        l = p.sum(-1, keepdim=True)
        o[b, :, 0] = ((p @ v) / l).flatten(0, 1).to(o.dtype)
        lse[b] = (m + torch.log(l)).flatten()
    return [o, lse] + ([s["k_back"], s["v_back"]] if s["k_new"] is not None else [])


def _exact_decode(c, s):
    out, sums = [], []
    if c["append"]:
        new = {x: _exact_rows(s[x + "_new"]) for x in "kv"}
    for b, n in enumerate(s["seq_lens"].tolist()):
        rows = {}
        for x in "kv":
            byte = s["cache"][x + "_codes"][b, :, :n].to(torch.int64)
            code = torch.empty(byte.shape[:-1] + (2 * byte.shape[-1],), dtype=torch.float64, device="cuda")
            code[..., 0::2], code[..., 1::2] = byte % 16 - 8, byte // 16 - 8
            rows[x] = code * s["cache"][x + "_scales"][b, :, :n].view(torch.float8_e4m3fn).double().repeat_interleave(GROUP, dim=-1)
            if c["append"]:
                rows[x] = torch.cat([rows[x], new[x][b]], dim=1)
        rep = c["heads"] // c["kv_heads"]
        score = torch.einsum("grd,gnd->grn", s["q"][b, :, 0].double().reshape(c["kv_heads"], rep, -1), rows["k"]) * s["scale"]
        out.append(torch.einsum("grn,gnd->grd", torch.softmax(score, -1), rows["v"]).reshape(c["heads"], 1, -1))
        sums.append(torch.logsumexp(score, -1).reshape(-1))
    got = [torch.stack(out), torch.stack(sums)]
    return got + ([new["k"], new["v"]] if c["append"] else [])

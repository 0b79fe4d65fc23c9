"""The serving operators called from several host threads and streams at once."""
import threading

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def S(lib):
    from vesper_b200 import serving_capi
    return serving_capi


def randn(g, *shape, dtype=torch.bfloat16):
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def int32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


def together(works):
    """Runs each in a thread of its own; raises what any of them raised."""
    wrong = []

    def run(work):
        try:
            torch.cuda.set_device(DEV)
            work()
        except BaseException as e:                                       # noqa: BLE001
            wrong.append(e)
    threads = [threading.Thread(target=run, args=(w,)) for w in works]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if wrong:
        raise wrong[0]


def test_threads_on_one_stream_without_workspaces(S):
    """Two threads share the default stream: each call's plan is read by its own attention kernel."""
    batches = [[300, 7, 0, 900, 64, 513] * 3, [20, 40, 1500, 3] * 5, [2000]]
    works, outs = [], []
    for i, lens in enumerate(batches):
        g = torch.Generator(device=DEV).manual_seed(i)
        q, k, v = randn(g, sum(lens), 16, 128), randn(g, sum(lens), 4, 128), randn(g, sum(lens), 4, 128)
        cu = int32(np.cumsum([0] + lens))
        cache = S.Kv4Cache(len(lens), 4, 2008, 128, device=DEV)
        k4 = randn(g, len(lens), 4, 2000, 128)
        cache.append(k4, k4)
        qd, seq = randn(g, len(lens), 16, 1, 128), int32(lens)
        want, want_d = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu), S.decode_kv4(qd, torch.empty_like(qd), cache, scale=0.09, seq_lens=seq)
        got = [(torch.zeros_like(q), torch.zeros_like(qd)) for _ in range(20)]
        outs.append((want, want_d, got))

        def work(q=q, k=k, v=v, cu=cu, cache=cache, qd=qd, seq=seq, got=got):
            for o, od in got:
                S.prefill_packed(q, k, v, o, scale=0.09, cu_seqlens_q=cu)
                S.decode_kv4(qd, od, cache, scale=0.09, seq_lens=seq)
        works.append(work)
    torch.cuda.synchronize()
    together(works)
    torch.cuda.synchronize()
    for want, want_d, got in outs:
        for o, od in got:
            assert torch.equal(o, want) and torch.equal(od, want_d)


def test_an_output_on_another_stream_while_the_current_one_is_busy(S):
    """Memory that the current stream has let go of, and still writes to, is not the output of a call on another stream."""
    g = torch.Generator(device=DEV).manual_seed(3)
    lens = [700, 324]
    q, q2, k, v = randn(g, 1024, 16, 128), randn(g, 1024, 16, 128), randn(g, 1024, 4, 128), randn(g, 1024, 4, 128)
    cu = int32(np.cumsum([0] + lens))
    want, want2 = (S.prefill_packed(x, k, v, scale=0.09, cu_seqlens_q=cu) for x in (q, q2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        old = torch.empty_like(q)
        torch.cuda._sleep(20_000_000)                        # some 10 ms: the fill below comes after the attention
        old.fill_(7.0)
        del old
        o = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(o, want)
        torch.cuda._sleep(20_000_000)
        used = o + 0                                         # the current stream reads it, and lets go of it before that is done
        del o
        again = S.prefill_packed(q2, k, v, scale=0.09, cu_seqlens_q=cu, stream=side)
        torch.cuda.synchronize()
        assert torch.equal(used, want) and torch.equal(again, want2)


def test_gradients_on_another_stream_while_the_current_one_is_busy(S):
    """The same for the outputs of the fp32 attention's backward pass."""
    from vesper_b200 import capi
    g = torch.Generator(device=DEV).manual_seed(4)
    q, k, v, do = (randn(g, 1, 8, 700, 64, dtype=torch.float32) for _ in range(4))
    o, lse = torch.empty_like(q), torch.empty(1, 8, 700, device=DEV)
    capi.prefill(q, k, v, o, lse, scale=0.125)
    want = capi.attention_bwd(do, q, k, v, o, lse, scale=0.125)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        old = [torch.empty_like(q) for _ in range(3)]
        torch.cuda._sleep(20_000_000)
        for t in old:
            t.fill_(7.0)
        del old, t
        got = capi.attention_bwd(do, q, k, v, o, lse, scale=0.125, stream=side)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        del got


def test_a_stream_of_another_library(S):
    """An object with a `cuda_stream` alone: what the call allocates is that stream's, while the current one writes over what it has let go of."""
    g = torch.Generator(device=DEV).manual_seed(5)
    lens = [700, 324]
    q, k, v = randn(g, 1024, 16, 128), randn(g, 1024, 4, 128), randn(g, 1024, 4, 128)
    cu = int32(np.cumsum([0] + lens))
    want = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu)
    side = torch.cuda.Stream()
    theirs = type("Theirs", (), {"cuda_stream": side.cuda_stream})()
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        got = S.prefill_packed(q, k, v, scale=0.09, cu_seqlens_q=cu, stream=theirs)
        for nbytes in (1 << 10, 1 << 14, 1 << 18, 1 << 20, 4 << 20):
            torch.empty(nbytes, dtype=torch.uint8, device=DEV).fill_(255)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
        del got

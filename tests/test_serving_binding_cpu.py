"""The Python binding of the serving operators without a GPU: what it allocates, where and for how long, and what it refuses.  Tensors of the CPU say that they
are on device 0, and the library's entry points are functions that look at what they are given."""
import weakref

import pytest
import torch


class OnDevice(torch.Tensor):
    """A CPU tensor that calls itself one of device 0, and that knows which streams it was recorded on."""

    def get_device(self):
        return 0

    def record_stream(self, stream):
        self.recorded = getattr(self, "recorded", []) + [stream]


def zeros(*shape, dtype=torch.bfloat16, kind=OnDevice):
    return torch.zeros(*shape, dtype=dtype).as_subclass(kind)


class Library:
    """Answers every entry point: sizes are 512 bytes, calls go to `seen` and succeed."""

    def __init__(self):
        self.seen, self.during = [], lambda: None

    def __getattr__(self, name):
        def entry(args):
            if "_bytes" in name:
                return 512
            self.seen.append(name)
            self.during()
            return 0
        return entry


@pytest.fixture
def serving(monkeypatch):
    from vesper_b200 import serving_capi
    library = Library()
    monkeypatch.setattr(serving_capi, "load", lambda: library)
    monkeypatch.setattr(serving_capi, "_stream", lambda device, stream: 0)
    serving_capi.library = library
    yield serving_capi
    del serving_capi.library


def packed_call(serving, kind=OnDevice, **kw):
    q, k = zeros(6, 4, 64, kind=kind), zeros(6, 2, 64, kind=kind)
    kw = {"cu_seqlens_q": zeros(3, dtype=torch.int32, kind=kind), **kw}
    return serving.prefill_packed(q, k, k, scale=0.1, **kw)


def a_cache(serving, kind=OnDevice):
    u = lambda n: zeros(2, 2, 16, n, dtype=torch.uint8, kind=kind)  # noqa: E731
    return serving.Kv4Cache(k_codes=u(32), v_codes=u(32), k_scales=u(2), v_scales=u(2))


def decode_call(serving, kind=OnDevice, **kw):
    q = zeros(2, 4, 1, 64, kind=kind)
    return serving.decode_kv4(q, torch.empty_like(q), a_cache(serving, kind), scale=0.1, **{"uniform_len": 3, **kw})


def norm_call(serving, kind=OnDevice, **kw):
    return serving.qk_norm_rope(zeros(2, 4, 3, 64, kind=kind), zeros(2, 2, 3, 64, kind=kind), **{"eps": 1e-6, "theta": 1e4, **kw})


def append_call(serving, kind=OnDevice, **kw):
    k = zeros(2, 2, 3, 64, kind=kind)
    a_cache(serving, kind).append(k, k, **kw)


def read_call(serving, kind=OnDevice, **kw):
    k = zeros(2, 2, 3, 64, kind=kind)
    a_cache(serving, kind).read(k, k, **kw)


CALLS = [norm_call, packed_call, append_call, read_call, decode_call]


@pytest.mark.parametrize("call", [packed_call, decode_call])
def test_the_workspace_lives_through_the_call(serving, monkeypatch, call):
    """The one that the binding allocates is not another thread's, and not unmapped, before the kernels are launched; and it is let go of afterwards."""
    made, alive = [], []
    allocate = serving.capi._workspace

    def workspace(*args, **kw):
        t = allocate(*args, **kw)
        made.append(weakref.ref(t))
        return t
    monkeypatch.setattr(serving.capi, "_workspace", workspace)
    serving.library.during = lambda: alive.append([r() is not None for r in made])
    call(serving)
    assert alive == [[True]]
    assert made[0]() is None


class Streams:
    """torch.cuda's streams, in so far as allocations ask for them: each notes the stream that is current."""

    def __init__(self, monkeypatch):
        class Stream:
            device, cuda_stream = torch.device("cpu"), 0

        class Within:
            def __init__(self, stream):
                self.stream = stream

            def __enter__(within):
                within.before, self.now = self.now, within.stream

            def __exit__(within, *error):
                self.now = within.before
        self.main, self.side = Stream(), Stream()
        self.now, self.made = self.main, []
        monkeypatch.setattr(torch.cuda, "Stream", Stream)
        monkeypatch.setattr(torch.cuda, "stream", Within)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.now)
        for name in ("empty", "empty_like"):
            def allocate(*args, _whole=getattr(torch, name), **kw):
                t = _whole(*args, **kw)
                self.made.append((t, self.now))
                return t
            monkeypatch.setattr(torch, name, allocate)


def test_an_output_on_another_stream_is_that_streams_memory(serving, monkeypatch):
    """Pending work of the current stream may still use what it has let go of: an output that another stream writes at once comes from that stream's memory, and
    what the current stream does with it later is waited for before it is given out again."""
    streams = Streams(monkeypatch)
    o = packed_call(serving, stream=streams.side)
    assert streams.made and all(s is streams.side for _, s in streams.made) and any(t is o for t, _ in streams.made)
    assert o.recorded == [streams.main] and streams.now is streams.main
    streams.made.clear()
    o = packed_call(serving)
    assert all(s is streams.main for _, s in streams.made) and not hasattr(o, "recorded")


def test_gradients_on_another_stream_are_that_streams_memory(monkeypatch):
    """The same for the outputs of the fp32 attention's backward pass."""
    from vesper_b200 import capi
    library = Library()
    monkeypatch.setattr(capi, "load", lambda: library)
    streams = Streams(monkeypatch)
    x, lse = zeros(1, 2, 5, 64, dtype=torch.float32), zeros(1, 2, 5, dtype=torch.float32)
    got = capi.attention_bwd(x, x, x, x, x, lse, scale=0.1, stream=streams.side)
    assert library.seen == ["vb200_attention_bwd"] and len(streams.made) == 4 and all(s is streams.side for _, s in streams.made)
    assert all(g.recorded == [streams.main] and g.shape == x.shape and g.is_contiguous() for g in got)
    streams.made.clear()
    assert not any(hasattr(g, "recorded") for g in capi.attention_bwd(x, x, x, x, x, lse, scale=0.1)) and all(s is streams.main for _, s in streams.made)


@pytest.mark.parametrize("call", CALLS)
def test_tensors_of_the_cpu_are_refused(serving, monkeypatch, call):
    """Their addresses would go to a kernel: get_device() is -1 for all of them, which the library takes for the current device."""
    monkeypatch.setattr(serving.capi, "inv_freq", lambda theta, D: [1.0] * (D // 2))
    call(serving)
    assert len(serving.library.seen) == 1
    with pytest.raises(ValueError, match="CUDA"):
        call(serving, kind=torch.Tensor)
    assert len(serving.library.seen) == 1


def test_workspaces_of_the_cpu_are_refused(serving):
    with pytest.raises(ValueError, match="CUDA"):
        serving.prefill_packed_workspace(torch.zeros(6, 4, 64, dtype=torch.bfloat16), torch.zeros(6, 2, 64, dtype=torch.bfloat16), batch=2)
    with pytest.raises(ValueError, match="CUDA"):
        serving.decode_kv4_workspace(torch.zeros(2, 4, 1, 64, dtype=torch.bfloat16), a_cache(serving, torch.Tensor))


def test_arrays_have_to_have_their_shape(serving, monkeypatch):
    """[T, B] for [B, T] would be read in the wrong order.  One dimension for all is the documented order, and dimensions of one change nothing."""
    monkeypatch.setattr(serving.capi, "inv_freq", lambda theta, D: [1.0] * (D // 2))
    i, f = lambda *s: zeros(*s, dtype=torch.int32), lambda *s: zeros(*s, dtype=torch.float32)  # noqa: E731
    k_cache = zeros(2, 2, 16, 64)
    to_cache = dict(k_out=k_cache, q_out=zeros(2, 4, 3, 64))
    right = [(norm_call, dict(positions=i(2, 3))), (norm_call, dict(positions=i(6))), (norm_call, dict(positions=i(2, 3, 1))), (norm_call, dict(q_weight=f(64), k_weight=f(1, 64))),
             (norm_call, dict(rows=i(2, 3), seqs=i(2, 3), **to_cache)), (packed_call, dict(lse=f(4, 6))), (packed_call, dict(lse=f(24))), (packed_call, dict(cu_seqlens_k=i(3))),
             (append_call, dict(rows=i(2, 3), seqs=i(2, 3))), (read_call, dict(rows=i(2, 3))), (decode_call, dict(lse=f(2, 4))), (decode_call, dict(lse=f(2, 4, 1))),
             (decode_call, dict(seq_lens=i(2, 1)))]
    wrong = [(norm_call, dict(positions=i(3, 2))), (norm_call, dict(positions=i(2, 4))), (norm_call, dict(q_weight=f(8, 8))), (norm_call, dict(rows=i(3, 2), **to_cache)),
             (norm_call, dict(rows=i(2, 3), seqs=i(3, 2), **to_cache)), (packed_call, dict(lse=f(6, 4))), (packed_call, dict(lse=f(2, 12))), (packed_call, dict(cu_seqlens_k=i(4))),
             (append_call, dict(rows=i(3, 2))), (append_call, dict(rows=i(2, 3), seqs=i(3, 2))), (read_call, dict(rows=i(3, 2))), (decode_call, dict(lse=f(4, 2))),
             (decode_call, dict(seq_lens=i(3)))]
    for call, kw in right:
        call(serving, **kw)
    assert len(serving.library.seen) == len(right)
    for call, kw in wrong:
        with pytest.raises(ValueError, match="shape"):
            call(serving, **kw)
    assert len(serving.library.seen) == len(right)


@pytest.mark.parametrize("which", ["q_weight", "k_weight"])
def test_weights_without_a_norm_are_refused(serving, monkeypatch, which):
    """They would be left out without a word."""
    monkeypatch.setattr(serving.capi, "inv_freq", lambda theta, D: [1.0] * (D // 2))
    with pytest.raises(ValueError, match="eps"):
        norm_call(serving, eps=None, **{which: zeros(64, dtype=torch.float32)})
    assert not serving.library.seen
    norm_call(serving, eps=None)
    norm_call(serving, eps=0.0, **{which: zeros(64, dtype=torch.float32)})
    assert len(serving.library.seen) == 2


def test_what_is_allocated_for_a_stream_of_another_library_is_that_streams(serving, monkeypatch):
    """Any object with a `cuda_stream` names a stream; the memory of a call on it is not the current stream's."""
    streams = Streams(monkeypatch)
    theirs, default = type("Theirs", (), {"cuda_stream": 0x50})(), type("Theirs", (), {"cuda_stream": 0})()

    class External(type(streams.side)):
        def __init__(self, handle, device=None):
            assert handle                                    # (torch makes a new stream of a handle of zero)
            self.cuda_stream = handle
    monkeypatch.setattr(torch.cuda, "ExternalStream", External)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device=None: streams.main)
    for call in (packed_call, decode_call):
        streams.made.clear()
        call(serving, stream=theirs)
        mine = [s for t, s in streams.made if t.dtype is torch.uint8 or call is packed_call]
        assert mine and all(s.cuda_stream == 0x50 for s in mine)
        streams.made.clear()
        call(serving, stream=default)
        assert all(s is streams.main for _, s in streams.made)

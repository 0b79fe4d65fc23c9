"""The serving operators' entry points without a GPU: symbols, structs, plans and refusals (which come before any device is touched)."""
import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000                      # stands for a device pointer that no refused call looks at


@pytest.fixture(scope="module")
def serving(lib):
    from vesper_b200 import serving_capi
    serving_capi.load()
    return serving_capi


def test_header_symbols_are_exported(lib, serving):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "vesper_b200_serving.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(vb200_[a-z0-9_]+)\s*\(", text)))
    assert names == sorted(serving.SERVING_EXPORTS)
    for n in names:
        assert hasattr(lib, n), n


def test_structs_match_the_header(serving, tmp_path):
    pairs = [("vb200_rows", serving.Rows), ("vb200_qk_norm_rope_args", serving.QkNormRopeArgs), ("vb200_prefill_packed_args", serving.PackedArgs),
             ("vb200_kv4_cache", serving.Kv4CacheView), ("vb200_kv4_rows_args", serving.Kv4RowsArgs), ("vb200_decode_kv4_args", serving.DecodeKv4Args)]
    lines = []
    for name, cls in pairs:
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f[0]}));' for f in cls._fields_]
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "vesper_b200_serving.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "sizes")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for _, cls in pairs:
        want += [C.sizeof(cls)] + [getattr(cls, f[0]).offset for f in cls._fields_]
    assert got == want
    # the binding's packings are these structs
    for packing, cls in ((serving._NORM, serving.QkNormRopeArgs), (serving._PACKED, serving.PackedArgs), (serving._KV4_ROWS, serving.Kv4RowsArgs), (serving._DECODE, serving.DecodeKv4Args)):
        n = len(packing.unpack(bytes(packing.size)))
        a = cls.from_buffer_copy(packing.pack(*range(1, n + 1)))
        flat = []

        def walk(x):
            for f in x._fields_:
                y = getattr(x, f[0])
                walk(y) if isinstance(y, C.Structure) else flat.append(C.cast(y, C.c_void_p).value if isinstance(y, C._Pointer) else y)
        walk(a)
        assert packing.size == C.sizeof(cls) and flat == list(range(1, n + 1)), cls


def view(capi, H, S, D, ptr=P):
    return capi.Tensor4(ptr, H * S * D, S * D, D)


def norm_args(serving, **kw):
    from vesper_b200 import capi
    B, Hq, Hkv, T, D = 2, 8, 2, 5, 128
    a = serving.QkNormRopeArgs(struct_size=C.sizeof(serving.QkNormRopeArgs), device=0, dtype=capi.BF16, B=B, Hq=Hq, Hkv=Hkv, T=T, D=D, q=view(capi, Hq, T, D),
                               k=view(capi, Hkv, T, D), v=view(capi, Hkv, T, D), q_out=view(capi, Hq, T, D), k_out=view(capi, Hkv, T, D), v_out=view(capi, Hkv, T, D),
                               norm=1, eps=1e-6)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("status, change", [
    (-1, dict(struct_size=8)), (-2, dict(dtype=7)), (-1, dict(B=0)), (-1, dict(T=-1)), (-1, dict(Hq=0)), (-1, dict(Hkv=0)), (-2, dict(D=12)), (-2, dict(D=136)),
    (-1, dict(eps=-1.0)), (-1, dict(eps=float("nan"))), (-1, dict(start_pos=-1)), (-1, dict(start_pos=2 ** 31 - 3)), (-3, dict(q_weight=P + 4)), (-3, dict(k_weight=P + 8)),
    (-1, dict(B=2 ** 20, T=2 ** 12))])
def test_norm_refuses(serving, status, change):
    assert serving.load().vb200_qk_norm_rope(C.byref(norm_args(serving, **change))) == status


def test_norm_refuses_views(serving):
    from vesper_b200 import capi
    call = lambda **kw: serving.load().vb200_qk_norm_rope(C.byref(norm_args(serving, **kw)))  # noqa: E731
    none = capi.Tensor4(None, 0, 0, 0)
    assert serving.load().vb200_qk_norm_rope(None) == -1
    assert call(q=none) == -1 and call(q_out=none) == -1 and call(k=none) == -1 and call(v_out=none) == -1
    assert call(q=none, q_out=none, k=none, k_out=none, v=none, v_out=none) == -1
    assert call(q=view(capi, 8, 5, 128, P + 2)) == -3 and call(v_out=view(capi, 2, 5, 128, P + 8)) == -3
    assert call(k=capi.Tensor4(P, 2 * 5 * 128, 5 * 128 + 4, 128)) == -3
    assert call(rope=capi.Rope(1, None)) == -1
    assert call(rope=capi.Rope(1, (C.c_float * 64)(*[1.0] * 63, float("inf")))) == -1
    assert call(q=capi.Tensor4(P, 8 * 5 * 128, -5 * 128, 128)) == -3
    assert call(dst=serving.Rows(None, P, 0, 0)) == -1 and call(dst=serving.Rows(P, None, 0, 8)) == -1 and call(dst=serving.Rows(P, None, 2, 0)) == -1


def test_outputs_may_not_be_broadcast(serving):
    """An element that several results would be written to (or, in place, that several would read): refused; a dimension of one may have any stride."""
    from vesper_b200 import capi
    L = serving.load()
    norm = lambda **kw: L.vb200_qk_norm_rope(C.byref(norm_args(serving, **kw)))  # noqa: E731
    H, T = 8 * 5 * 128, 5 * 128
    for strides in ((0, T, 128), (H, 0, 128), (H, T, 0)):
        assert norm(q_out=capi.Tensor4(P, *strides)) == -2 and norm(k_out=capi.Tensor4(P, *strides)) == -2 and norm(v_out=capi.Tensor4(P, *strides)) == -2
        cache = serving.Rows(P, None, 4, 64)
        assert norm(dst=cache, k_out=capi.Tensor4(P, *strides)) == -2
        read = rows_args(serving, k=capi.Tensor4(P, *strides))
        assert L.vb200_kv4_read(C.byref(read)) == -2
        read = rows_args(serving, v=capi.Tensor4(P, *strides))
        assert L.vb200_kv4_read(C.byref(read)) == -2
    assert norm(dst=serving.Rows(P, None, 4, 64), T=1, k_out=capi.Tensor4(P, H, T, 0)) == -2                 # the cache has more rows than the call has tokens
    assert norm(T=1, q_out=capi.Tensor4(P, H, T, 0), q=capi.Tensor4(P + 2, H, T, 0)) == -3                  # (not refused for its stride)
    for strides in ((0, 128, 128), (1024, 0, 128)):
        assert L.vb200_decode_kv4_fwd(C.byref(decode_args(serving, o=capi.Tensor4(P, *strides)))) == -2


def packed_args(serving, **kw):
    from vesper_b200 import capi
    t = lambda H: capi.Tensor4(P, 0, 128, H * 128)  # noqa: E731
    a = serving.PackedArgs(struct_size=C.sizeof(serving.PackedArgs), device=0, dtype=capi.BF16, batch=3, Hq=8, Hkv=2, D=128, total_q=100, total_k=100, causal=1, scale=0.1,
                           q=t(8), o=t(8), k=t(2), v=t(2), cu_seqlens_q=P, workspace=P, workspace_bytes=1 << 30)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("status, change", [
    (-1, dict(struct_size=8)), (-2, dict(dtype=0)), (-2, dict(D=96)), (-2, dict(D=256)), (-1, dict(batch=0)), (-1, dict(batch=70000)), (-1, dict(Hkv=3)), (-1, dict(Hkv=0)),
    (-1, dict(total_q=0)), (-1, dict(total_k=-1)), (-1, dict(cu_seqlens_q=None)), (-4, dict(workspace=None)), (-4, dict(workspace_bytes=16)), (-3, dict(workspace=P + 16)),
    (-1, dict(total_q=2 ** 30)), (-1, dict(batch=65536, Hq=65536, Hkv=65536))])
def test_packed_refuses(serving, status, change):
    assert serving.load().vb200_prefill_packed_fwd(C.byref(packed_args(serving, **change))) == status


def test_packed_refuses_views(serving):
    from vesper_b200 import capi
    call = lambda **kw: serving.load().vb200_prefill_packed_fwd(C.byref(packed_args(serving, **kw)))  # noqa: E731
    for name in "qokv":
        assert call(**{name: capi.Tensor4(None, 0, 128, 1024)}) == -1
        assert call(**{name: capi.Tensor4(P + 8, 0, 128, 1024)}) == -3
        assert call(**{name: capi.Tensor4(P, 0, 128, 1028)}) == -3
        assert call(**{name: capi.Tensor4(P, 0, 0, 1024)}) == -2 and call(**{name: capi.Tensor4(P, 0, 128, 0)}) == -2
    assert serving.load().vb200_prefill_packed_workspace_bytes(C.byref(packed_args(serving, Hkv=3))) == 0
    assert serving.load().vb200_prefill_packed_workspace_bytes(C.byref(packed_args(serving))) > 0


def cache_view(serving, D=128, cap=64, **kw):
    c = serving.Kv4CacheView(P, P, P, P, 2 * cap, cap, 4, cap, 0, 0)
    for name, x in kw.items():
        setattr(c, name, x)
    return c


BAD_CACHES = [(-1, dict(k_codes=None)), (-1, dict(v_scales=None)), (-1, dict(seqs=0)), (-1, dict(cap=0)), (-3, dict(cap=60, stride_b=120, stride_h=60)), (-1, dict(k_exponent=65)),
              (-1, dict(v_exponent=-65)), (-1, dict(stride_h=56)), (-1, dict(stride_b=8)), (-3, dict(k_scales=P + 4)), (-3, dict(v_codes=P + 8)), (-3, dict(stride_h=68))]


def rows_args(serving, **kw):
    from vesper_b200 import capi
    a = serving.Kv4RowsArgs(struct_size=C.sizeof(serving.Kv4RowsArgs), device=0, dtype=capi.BF16, B=4, Hkv=2, T=5, D=128, k=view(capi, 2, 5, 128), v=view(capi, 2, 5, 128),
                            cache=cache_view(serving))
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("entry", ["vb200_kv4_append", "vb200_kv4_read"])
@pytest.mark.parametrize("status, change", [
    (-1, dict(struct_size=8)), (-2, dict(dtype=0)), (-2, dict(D=32)), (-2, dict(D=96)), (-1, dict(B=0)), (-1, dict(T=0)), (-1, dict(Hkv=0)), (-1, dict(start_row=-1)),
    (-1, dict(start_row=60)), (-1, dict(B=5)), (-1, dict(T=2 ** 29))])
def test_kv4_rows_refuse(serving, entry, status, change):
    assert getattr(serving.load(), entry)(C.byref(rows_args(serving, **change))) == status


@pytest.mark.parametrize("entry", ["vb200_kv4_append", "vb200_kv4_read"])
def test_kv4_rows_refuse_views(serving, entry):
    from vesper_b200 import capi
    call = lambda **kw: getattr(serving.load(), entry)(C.byref(rows_args(serving, **kw)))  # noqa: E731
    for status, change in BAD_CACHES:
        assert call(cache=cache_view(serving, **change)) == status, change
    none = capi.Tensor4(None, 0, 0, 0)
    assert call(k=none, v=none) == -1
    if entry == "vb200_kv4_append":
        assert call(k=none) == -1 and call(v=none) == -1
    assert call(k=view(capi, 2, 5, 128, P + 4)) == -3
    assert call(at=serving.Rows(None, P, 0, 0)) == -1


def decode_args(serving, **kw):
    from vesper_b200 import capi
    row = lambda H: capi.Tensor4(P, H * 128, 128, 128)  # noqa: E731
    a = serving.DecodeKv4Args(struct_size=C.sizeof(serving.DecodeKv4Args), device=0, dtype=capi.BF16, B=4, Hq=8, Hkv=2, D=128, scale=0.1, q=row(8), k_new=row(2), v_new=row(2),
                              o=row(8), cache=cache_view(serving), seq_lens=P, workspace=P, workspace_bytes=1 << 30)
    for name, x in kw.items():
        setattr(a, name, x)
    return a


@pytest.mark.parametrize("status, change", [
    (-1, dict(struct_size=8)), (-2, dict(dtype=0)), (-2, dict(D=96)), (-1, dict(B=0)), (-1, dict(Hkv=3)), (-1, dict(Hq=0)), (-1, dict(max_len=-1)), (-1, dict(num_splits=-1)),
    (-1, dict(B=5)), (-1, dict(seq_lens=None, uniform_len=64)), (-1, dict(seq_lens=None, uniform_len=-1)), (-1, dict(seq_lens=None, uniform_len=10, max_len=10)),
    (-1, dict(seq_lens=None, advance_lens=1)), (-4, dict(workspace=None)), (-4, dict(workspace_bytes=64)), (-3, dict(workspace=P + 128))])
def test_decode_refuses(serving, status, change):
    assert serving.load().vb200_decode_kv4_fwd(C.byref(decode_args(serving, **change))) == status


def test_decode_refuses_views(serving):
    from vesper_b200 import capi
    call = lambda **kw: serving.load().vb200_decode_kv4_fwd(C.byref(decode_args(serving, **kw)))  # noqa: E731
    for status, change in BAD_CACHES:
        assert call(cache=cache_view(serving, **change)) == status, change
    none = capi.Tensor4(None, 0, 0, 0)
    assert call(q=none) == -1 and call(o=none) == -1 and call(k_new=none) == -1 and call(v_new=none) == -1
    assert call(q=capi.Tensor4(P, 1024, 132, 128)) == -3 and call(o=capi.Tensor4(P + 8, 1024, 128, 128)) == -3 and call(k_new=capi.Tensor4(P, 257, 128, 128)) == -3


def test_workspace_of_a_generation_covers_every_step(serving):
    L = serving.load()
    for B, Hq, Hkv, cap in ((1, 16, 4, 512), (32, 32, 8, 1024), (3, 8, 8, 776)):
        a = decode_args(serving, B=B, Hq=Hq, Hkv=Hkv, cache=cache_view(serving, cap=cap, seqs=B, stride_b=Hkv * cap, stride_h=cap))
        most = L.vb200_decode_kv4_workspace_bytes_max(C.byref(a))
        for n in range(1, cap + 1, 5):
            a.max_len = n
            for lens in (None, P):
                a.seq_lens = lens
                assert 0 < L.vb200_decode_kv4_workspace_bytes(C.byref(a)) <= most
    assert L.vb200_decode_kv4_workspace_bytes(C.byref(decode_args(serving, struct_size=3))) == 0
    assert L.vb200_decode_kv4_workspace_bytes_max(C.byref(decode_args(serving, Hkv=3))) == 0


def test_wrapper_refuses(serving):
    """The Python binding looks at types, shapes and strides before it hands out pointers."""
    import torch
    x = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(ValueError):
        serving.qk_norm_rope(None, None)
    with pytest.raises(ValueError):
        serving.Kv4Cache(k_codes=torch.zeros(1, 1, 8, 64), v_codes=torch.zeros(1, 1, 8, 64), k_scales=torch.zeros(1, 1, 8, 4), v_scales=torch.zeros(1, 1, 8, 4))
    with pytest.raises(ValueError):
        u = lambda n: torch.zeros(1, 1, 8, n, dtype=torch.uint8)  # noqa: E731
        serving.Kv4Cache(k_codes=u(64), v_codes=u(64), k_scales=u(4), v_scales=u(8))
    with pytest.raises(ValueError):
        serving._view("k", x(1, 1, 2, 8), x(1, 1, 2, 8), (1, 1, 3, 8))
    with pytest.raises(ValueError):
        serving._view("k", x(1, 1, 2, 8).float(), x(1, 1, 2, 8), (1, 1, 2, 8))
    with pytest.raises(ValueError):
        serving._view("k", x(1, 1, 8, 2).transpose(2, 3), x(1, 1, 2, 8), (1, 1, 2, 8))
    with pytest.raises(ValueError):
        serving._view3("k", x(2, 1, 8), x(2, 1, 8), (2, 2, 8))
    with pytest.raises(ValueError):
        serving._whole("rows", torch.zeros(4, 2, dtype=torch.int32).t(), torch.int32, -1, 8)
    with pytest.raises(ValueError):
        serving._whole("rows", torch.zeros(8, dtype=torch.int64), torch.int32, -1, 8)
    c = serving.Kv4Cache(2, 3, 60, 128, device="cpu")
    assert c.cap == 64 and c.view.stride_h == 64 and c.view.stride_b == 192
    with pytest.raises(ValueError):
        serving._workspace(torch.zeros(64, 2, dtype=torch.uint8)[:, 0], 0, x(1), None)
    with pytest.raises(ValueError):
        serving._code(torch.zeros(1, dtype=torch.float64))

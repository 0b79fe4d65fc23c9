"""ctypes binding of include/vesper_b200_serving.h on torch tensors: norms of queries and keys with the rotation, attention over packed prompts, and the
4-bit key / value cache with the decode step that reads it."""
from __future__ import annotations

import ctypes as C

from . import capi

SERVING_EXPORTS = ["vb200_qk_norm_rope", "vb200_prefill_packed_workspace_bytes", "vb200_prefill_packed_fwd", "vb200_kv4_append", "vb200_kv4_read",
                   "vb200_decode_kv4_workspace_bytes", "vb200_decode_kv4_workspace_bytes_max", "vb200_decode_kv4_fwd"]

_i32, _i64, _p, _f = C.c_int32, C.c_int64, C.c_void_p, C.c_float
GROUP = 32                       # elements of a row that share a scale


class Rows(C.Structure):
    _fields_ = [("rows", _p), ("seq_ids", _p), ("seqs", _i32), ("cap", _i32)]


class QkNormRopeArgs(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("device", _i32), ("stream", _p), ("dtype", _i32), ("B", _i32), ("Hq", _i32), ("Hkv", _i32), ("T", _i32), ("D", _i32),
                ("q", capi.Tensor4), ("k", capi.Tensor4), ("v", capi.Tensor4), ("q_out", capi.Tensor4), ("k_out", capi.Tensor4), ("v_out", capi.Tensor4),
                ("norm", _i32), ("eps", _f), ("q_weight", _p), ("k_weight", _p), ("rope", capi.Rope), ("start_pos", _i32), ("positions", _p), ("dst", Rows)]


class PackedArgs(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("device", _i32), ("stream", _p), ("dtype", _i32), ("batch", _i32), ("Hq", _i32), ("Hkv", _i32), ("D", _i32),
                ("total_q", _i32), ("total_k", _i32), ("causal", _i32), ("scale", _f), ("q", capi.Tensor4), ("o", capi.Tensor4), ("k", capi.Tensor4), ("v", capi.Tensor4),
                ("lse", _p), ("cu_seqlens_q", _p), ("cu_seqlens_k", _p), ("workspace", _p), ("workspace_bytes", C.c_size_t)]


class Kv4CacheView(C.Structure):
    _fields_ = [("k_codes", _p), ("v_codes", _p), ("k_scales", _p), ("v_scales", _p), ("stride_b", _i64), ("stride_h", _i64), ("seqs", _i32), ("cap", _i32),
                ("k_exponent", _i32), ("v_exponent", _i32)]


class Kv4RowsArgs(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("device", _i32), ("stream", _p), ("dtype", _i32), ("B", _i32), ("Hkv", _i32), ("T", _i32), ("D", _i32),
                ("k", capi.Tensor4), ("v", capi.Tensor4), ("cache", Kv4CacheView), ("start_row", _i32), ("at", Rows)]


class DecodeKv4Args(C.Structure):
    _fields_ = [("struct_size", C.c_size_t), ("device", _i32), ("stream", _p), ("dtype", _i32), ("B", _i32), ("Hq", _i32), ("Hkv", _i32), ("D", _i32), ("scale", _f),
                ("q", capi.Tensor4), ("k_new", capi.Tensor4), ("v_new", capi.Tensor4), ("o", capi.Tensor4), ("lse", _p), ("cache", Kv4CacheView), ("seq_lens", _p),
                ("uniform_len", _i32), ("advance_lens", _i32), ("max_len", _i32), ("num_splits", _i32), ("workspace", _p), ("workspace_bytes", C.c_size_t)]


_lib = None


def load():
    global _lib
    if _lib is None:
        L = capi.load()
        L.vb200_qk_norm_rope.argtypes = [C.POINTER(QkNormRopeArgs)]
        L.vb200_prefill_packed_fwd.argtypes = L.vb200_prefill_packed_workspace_bytes.argtypes = [C.POINTER(PackedArgs)]
        L.vb200_kv4_append.argtypes = L.vb200_kv4_read.argtypes = [C.POINTER(Kv4RowsArgs)]
        for name in ("vb200_decode_kv4_fwd", "vb200_decode_kv4_workspace_bytes", "vb200_decode_kv4_workspace_bytes_max"):
            getattr(L, name).argtypes = [C.POINTER(DecodeKv4Args)]
        for name in ("vb200_prefill_packed_workspace_bytes", "vb200_decode_kv4_workspace_bytes", "vb200_decode_kv4_workspace_bytes_max"):
            getattr(L, name).restype = C.c_size_t
        _lib = L
    return _lib


def _stream(t, stream):
    import torch
    return (stream if stream is not None else torch.cuda.current_stream(t.device)).cuda_stream


def _ptr(t):
    return None if t is None else t.data_ptr()


def _like(name, t, model, shape):
    """`t` has to be of the model's type and device and of this shape."""
    if t is not None and (t.dtype != model.dtype or t.device != model.device or tuple(t.shape) != tuple(shape)):
        raise ValueError(f"{name}: expected {tuple(shape)} {model.dtype} on {model.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if t is not None and t.stride(-1) != 1:
        raise ValueError(f"{name}: the last dimension must be contiguous")


def _whole(name, t, dtype, device, numel):
    """An array of the device that the kernels read as it lies."""
    if t is not None and (t.dtype != dtype or t.device != device or t.numel() != numel or not t.is_contiguous()):
        raise ValueError(f"{name}: expected {numel} contiguous {dtype} on {device}, got {tuple(t.shape)} {t.dtype} on {t.device}")


def _view3(t):
    """[tokens, H, D] -> the view the packed operators take."""
    return capi.Tensor4(t.data_ptr(), 0, t.stride(1), t.stride(0))


def _rows(rows, seqs, device, tokens, n_seqs, cap):
    import torch
    _whole("rows", rows, torch.int32, device, tokens)
    _whole("seqs", seqs, torch.int32, device, tokens)
    return Rows(_ptr(rows), _ptr(seqs), n_seqs, cap)


def _workspace(workspace, need, t, stream):
    if workspace is None:
        workspace = capi._workspace(need, t.device, stream)
    return workspace, workspace.data_ptr(), workspace.numel() * workspace.element_size()


def qk_norm_rope(q, k, v=None, *, eps=None, q_weight=None, k_weight=None, theta=None, inv_freq=None, start_pos=0, positions=None, q_out=None, k_out=None, v_out=None,
                 rows=None, seqs=None, stream=None):
    """vb200_qk_norm_rope on [B, H, T, D] views: norms with eps (None: no norm), the rotation by theta or by inv_freq (D / 2 floats of the host; neither: no
    rotation).  q_out, k_out None: in place.  rows (and seqs) [B, T] int32: k_out and v_out are caches [sequences, H, cap, D] and these name the places.
    Returns (q_out, k_out, v_out)."""
    import torch
    some = q if q is not None else k if k is not None else v
    if some is None:
        raise ValueError("qk_norm_rope: one of q, k, v must be given")
    B, _, T, D = some.shape
    kv = k if k is not None else v
    a = QkNormRopeArgs(struct_size=C.sizeof(QkNormRopeArgs), device=some.device.index, stream=_stream(some, stream), dtype=capi.dtype_code(some), B=B,
                       Hq=q.shape[1] if q is not None else 0, Hkv=kv.shape[1] if kv is not None else 0, T=T, D=D, start_pos=start_pos)
    scatter = rows is not None
    if not scatter and v is not None and v_out is None:
        raise ValueError("qk_norm_rope: v needs v_out")
    q_out = q if q_out is None else q_out
    k_out = k if k_out is None and not scatter else k_out
    for name, t, to, H in (("q", q, q_out, a.Hq), ("k", k, k_out, a.Hkv), ("v", v, v_out, a.Hkv)):
        _like(name, t, some, (B, H, T, D))
        cached = scatter and name != "q" and to is not None
        _like(name + "_out", to, some, (to.shape[0], H, to.shape[2], D) if cached else (B, H, T, D))
        setattr(a, name, capi.view4(t))
        setattr(a, name + "_out", capi.view4(to))
    if scatter:
        cache = k_out if k_out is not None else v_out
        if cache is None:
            raise ValueError("qk_norm_rope: rows need k_out or v_out")
        if k_out is not None and v_out is not None and (k_out.shape[0], k_out.shape[2]) != (v_out.shape[0], v_out.shape[2]):
            raise ValueError("qk_norm_rope: k_out and v_out must have the same sequences and rows")
        a.dst = _rows(rows, seqs, some.device, B * T, cache.shape[0], cache.shape[2])
    _whole("positions", positions, torch.int32, some.device, B * T)
    a.positions = _ptr(positions)
    if eps is not None:
        _whole("q_weight", q_weight, torch.float32, some.device, D)
        _whole("k_weight", k_weight, torch.float32, some.device, D)
        a.norm, a.eps, a.q_weight, a.k_weight = 1, eps, _ptr(q_weight), _ptr(k_weight)
    if inv_freq is None and theta is not None:
        inv_freq = capi.inv_freq(theta, D)
    if inv_freq is not None:
        if len(inv_freq) != D // 2:
            raise ValueError(f"qk_norm_rope: expected {D // 2} frequencies, got {len(inv_freq)}")
        if not isinstance(inv_freq, C.Array):
            import numpy as np
            inv_freq = (C.c_float * (D // 2)).from_buffer_copy(np.ascontiguousarray(inv_freq, dtype=np.float32))
        a.rope = capi.Rope(1, inv_freq)
    capi.check(load().vb200_qk_norm_rope(C.byref(a)))
    return q_out, k_out, v_out


def _packed_args(q, k, batch):
    return PackedArgs(struct_size=C.sizeof(PackedArgs), device=q.device.index, dtype=capi.dtype_code(q), batch=batch, Hq=q.shape[1], Hkv=k.shape[1], D=q.shape[2],
                      total_q=q.shape[0], total_k=k.shape[0])


def prefill_packed_workspace(q, k, *, batch):
    """A workspace for vb200_prefill_packed_fwd on tensors of these shapes and `batch` sequences."""
    return capi._workspace(load().vb200_prefill_packed_workspace_bytes(C.byref(_packed_args(q, k, batch))), q.device, None)


def prefill_packed(q, k, v, o=None, lse=None, *, scale, cu_seqlens_q, cu_seqlens_k=None, causal=True, workspace=None, stream=None):
    """vb200_prefill_packed_fwd: q [total_q, Hq, D], k, v [total_k, Hkv, D], cu_seqlens int32 [batch + 1] on the device, lse [Hq, total_q] fp32.  Returns o."""
    import torch
    o = torch.empty_like(q) if o is None else o
    batch = cu_seqlens_q.numel() - 1
    _like("q", q, q, q.shape)
    _like("k", k, q, (k.shape[0], k.shape[1], q.shape[2]))
    _like("v", v, q, k.shape)
    _like("o", o, q, q.shape)
    _whole("lse", lse, torch.float32, q.device, q.shape[0] * q.shape[1])
    _whole("cu_seqlens_q", cu_seqlens_q, torch.int32, q.device, batch + 1)
    _whole("cu_seqlens_k", cu_seqlens_k, torch.int32, q.device, batch + 1)
    if cu_seqlens_k is None and k.shape[0] < q.shape[0]:
        raise ValueError("prefill_packed: fewer keys than queries need cu_seqlens_k")
    a = _packed_args(q, k, batch)
    a.stream, a.causal, a.scale = _stream(q, stream), int(causal), scale
    a.q, a.o, a.k, a.v, a.lse = _view3(q), _view3(o), _view3(k), _view3(v), _ptr(lse)
    a.cu_seqlens_q, a.cu_seqlens_k = _ptr(cu_seqlens_q), _ptr(cu_seqlens_k)
    L = load()
    need = L.vb200_prefill_packed_workspace_bytes(C.byref(a)) if workspace is None else 0
    workspace, a.workspace, a.workspace_bytes = _workspace(workspace, need, q, stream)
    capi.check(L.vb200_prefill_packed_fwd(C.byref(a)))
    return o


class Kv4Cache:
    """Keys and values of `seqs` sequences in 4 bits: four uint8 tensors, codes [seqs, Hkv, cap, D / 2] and scales [seqs, Hkv, cap, D / 32], cap a multiple
    of 8.  Made empty from the sizes, or around tensors that are there."""

    def __init__(self, seqs=None, Hkv=None, cap=None, D=None, *, device=None, k_exponent=0, v_exponent=0, k_codes=None, v_codes=None, k_scales=None, v_scales=None):
        import torch
        if k_codes is None:
            cap = (cap + 7) // 8 * 8
            k_codes, v_codes = (torch.zeros(seqs, Hkv, cap, D // 2, dtype=torch.uint8, device=device) for _ in range(2))
            k_scales, v_scales = (torch.zeros(seqs, Hkv, cap, D // GROUP, dtype=torch.uint8, device=device) for _ in range(2))
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = k_codes, v_codes, k_scales, v_scales
        self.seqs, self.Hkv, self.cap, self.D = k_codes.shape[0], k_codes.shape[1], k_codes.shape[2], 2 * k_codes.shape[3]
        row = k_codes.stride(2)
        for name, t, n in (("k_codes", k_codes, self.D // 2), ("v_codes", v_codes, self.D // 2), ("k_scales", k_scales, self.D // GROUP), ("v_scales", v_scales, self.D // GROUP)):
            if t.dtype != torch.uint8 or t.device != k_codes.device or tuple(t.shape) != (self.seqs, self.Hkv, self.cap, n) or t.stride(3) != 1 or t.stride(2) != n:
                raise ValueError(f"Kv4Cache: {name} must be uint8 [{self.seqs}, {self.Hkv}, {self.cap}, {n}] with contiguous rows")
            if any(t.shape[d] > 1 and t.stride(d) * row != k_codes.stride(d) * n for d in (0, 1)):
                raise ValueError("Kv4Cache: codes and scales must have the same strides, in rows")
        self.view = Kv4CacheView(_ptr(k_codes), _ptr(v_codes), _ptr(k_scales), _ptr(v_scales), k_codes.stride(0) // row, k_codes.stride(1) // row, self.seqs, self.cap,
                                 k_exponent, v_exponent)

    def _call(self, entry, k, v, start_row, rows, seqs, stream):
        some = k if k is not None else v
        if some is None:
            raise ValueError("Kv4Cache: k and v are both missing")
        B, _, T, _ = some.shape
        for name, t in (("k", k), ("v", v)):
            _like(name, t, some, (B, self.Hkv, T, self.D))
        if some.device != self.k_codes.device:
            raise ValueError(f"Kv4Cache: rows on {some.device}, cache on {self.k_codes.device}")
        a = Kv4RowsArgs(struct_size=C.sizeof(Kv4RowsArgs), device=some.device.index, stream=_stream(some, stream), dtype=capi.dtype_code(some), B=B, Hkv=self.Hkv, T=T, D=self.D,
                        k=capi.view4(k), v=capi.view4(v), cache=self.view, start_row=start_row, at=_rows(rows, seqs, some.device, B * T, self.seqs, self.cap))
        capi.check(entry(C.byref(a)))

    def append(self, k, v, *, start_row=0, rows=None, seqs=None, stream=None):
        """vb200_kv4_append: [B, Hkv, T, D] keys and values into rows start_row + t of sequence b, or where rows (and seqs) [B, T] int32 say."""
        self._call(load().vb200_kv4_append, k, v, start_row, rows, seqs, stream)

    def read(self, k, v, *, start_row=0, rows=None, seqs=None, stream=None):
        """vb200_kv4_read: the values of those rows into k and v (either may be None)."""
        self._call(load().vb200_kv4_read, k, v, start_row, rows, seqs, stream)


def _decode_args(q, cache, max_len, num_splits):
    return DecodeKv4Args(struct_size=C.sizeof(DecodeKv4Args), device=q.device.index, dtype=capi.dtype_code(q), B=q.shape[0], Hq=q.shape[1], Hkv=cache.Hkv, D=q.shape[3],
                         cache=cache.view, max_len=max_len, num_splits=num_splits)


def decode_kv4_workspace(q, cache, *, max_len=0, num_splits=0, whole_generation=False):
    """A workspace for vb200_decode_kv4_fwd: for steps planned with this max_len, or for every step of a generation over this cache."""
    L = load()
    entry = L.vb200_decode_kv4_workspace_bytes_max if whole_generation else L.vb200_decode_kv4_workspace_bytes
    return capi._workspace(entry(C.byref(_decode_args(q, cache, max_len, num_splits))), q.device, None)


def decode_kv4(q, o, cache, *, scale, k_new=None, v_new=None, lse=None, seq_lens=None, uniform_len=0, advance_lens=False, max_len=0, num_splits=0, workspace=None, stream=None):
    """vb200_decode_kv4_fwd: one token per sequence, q and o [B, Hq, 1, D], k_new and v_new [B, Hkv, 1, D] appended first, seq_lens int32 [B] on the device."""
    import torch
    B = q.shape[0]
    _like("q", q, q, (B, q.shape[1], 1, cache.D))
    _like("o", o, q, q.shape)
    _like("k_new", k_new, q, (B, cache.Hkv, 1, cache.D))
    _like("v_new", v_new, q, (B, cache.Hkv, 1, cache.D))
    _whole("lse", lse, torch.float32, q.device, B * q.shape[1])
    _whole("seq_lens", seq_lens, torch.int32, q.device, B)
    if q.device != cache.k_codes.device:
        raise ValueError(f"decode_kv4: q on {q.device}, cache on {cache.k_codes.device}")
    a = _decode_args(q, cache, max_len, num_splits)
    a.stream, a.scale = _stream(q, stream), scale
    a.q, a.o, a.lse, a.k_new, a.v_new = capi.view4(q), capi.view4(o), _ptr(lse), capi.view4(k_new), capi.view4(v_new)
    a.seq_lens, a.uniform_len, a.advance_lens = _ptr(seq_lens), uniform_len, int(advance_lens)
    L = load()
    need = L.vb200_decode_kv4_workspace_bytes(C.byref(a)) if workspace is None else 0
    workspace, a.workspace, a.workspace_bytes = _workspace(workspace, need, q, stream)
    capi.check(L.vb200_decode_kv4_fwd(C.byref(a)))
    return o

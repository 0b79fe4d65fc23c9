"""ctypes binding of include/vesper_b200_serving.h on torch tensors: norms of queries and keys with the rotation, attention over packed prompts, and the
4-bit key / value cache with the decode step that reads it."""
from __future__ import annotations

import ctypes as C
import math
import struct

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
        for name in SERVING_EXPORTS:                              # an args struct by reference, or its bytes
            getattr(L, name).argtypes = [_p]
        for name in ("vb200_prefill_packed_workspace_bytes", "vb200_decode_kv4_workspace_bytes", "vb200_decode_kv4_workspace_bytes_max"):
            getattr(L, name).restype = C.c_size_t
        _lib = L
    return _lib


# The args structs as one packing each: filling ctypes structures field by field takes most of a small call's time.
_VIEW = "P3q"                                                 # vb200_tensor4
_CACHE = "4P2q4i"                                             # vb200_kv4_cache
_ROWS = "2P2i"                                                # vb200_rows
_NORM = struct.Struct("@NiP6i" + 6 * _VIEW + "if2PiPiP" + _ROWS + "0q")
_PACKED = struct.Struct("@NiP8if" + 4 * _VIEW + "4PN0q")
_KV4_ROWS = struct.Struct("@NiP5i" + 2 * _VIEW + _CACHE + "i" + "0q" + _ROWS + "0q")
_DECODE = struct.Struct("@NiP5if" + 4 * _VIEW + "P" + _CACHE + "P4iPN0q")
_NONE4 = (0, 0, 0, 0)
_TYPES = {}


def _code(t):
    """vb200_dtype of a tensor's type."""
    if not _TYPES:
        import torch
        _TYPES.update({torch.float32: capi.F32, torch.bfloat16: capi.BF16, torch.float16: capi.F16})
    if t.dtype not in _TYPES:
        raise ValueError(f"expected float32, bfloat16 or float16, got {t.dtype}")
    return _TYPES[t.dtype]


def _device(name, t):
    """The device that a call runs on: its first tensor's, which the others are compared with.  (-1, as all tensors of the CPU have it, would be the current device
    to the library.)"""
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name}: expected a tensor of a CUDA device, got one on {t.device}")
    return device


def _stream(device, stream):
    """The raw handle of `stream`, or of the device's current one."""
    if stream is not None:
        return stream.cuda_stream
    import torch
    return torch._C._cuda_getCurrentRawStream(device)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _wrong(name, t, shape, model):
    raise ValueError(f"{name}: expected {tuple(shape)} {model.dtype} on {model.device}, the last dimension contiguous, got {tuple(t.shape)} {t.dtype} on {t.device}, "
                     f"strides {t.stride()}")


def _view(name, t, model, shape):
    """The view of a 4-D tensor, which has to be of the model's type and device and of this shape."""
    s = t.stride()
    if t.shape != shape or t.dtype is not model.dtype or t.get_device() != model.get_device() or s[3] != 1:
        _wrong(name, t, shape, model)
    return t.data_ptr(), s[0], s[1], s[2]


def _view3(name, t, model, shape):
    """[tokens, H, D] -> the view the packed operators take."""
    s = t.stride()
    if t.shape != shape or t.dtype is not model.dtype or t.get_device() != model.get_device() or s[2] != 1:
        _wrong(name, t, shape, model)
    return t.data_ptr(), 0, s[1], s[0]


def _same_order(got, shape):
    """Whether an array of shape `got` lies as one of `shape` does: but for dimensions of one, or in one dimension for all."""
    long = lambda s: [n for n in s if n != 1]  # noqa: E731
    return long(got) == long(shape) or (len(got) == 1 and got[0] == math.prod(shape))


def _whole(name, t, dtype, device, shape):
    """The address of an array that the kernels read as it lies (0: none)."""
    if t is None:
        return 0
    if t.dtype is not dtype or t.get_device() != device or not t.is_contiguous() or (t.shape != shape and not _same_order(t.shape, shape)):
        raise ValueError(f"{name}: expected contiguous {dtype} of shape {shape} on device {device}, got {tuple(t.shape)} {t.dtype} on {t.device}, strides {t.stride()}")
    return t.data_ptr()


def _rows(rows, seqs, device, shape, n_seqs, cap):
    import torch
    return _whole("rows", rows, torch.int32, device, shape), _whole("seqs", seqs, torch.int32, device, shape), n_seqs, cap


def _workspace(workspace, need, t, stream):
    """(memory, address, bytes) of the caller's workspace or of a new one.  The caller holds on to the memory until its call has launched: before that, another
    thread on the same stream could be given the same."""
    if workspace is None:
        workspace = capi._workspace(need, t.device, stream)
    elif workspace.get_device() != t.get_device() or not workspace.is_contiguous():
        raise ValueError(f"workspace: expected contiguous memory on {t.device}, got one on {workspace.device}, strides {workspace.stride()}")
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
    device, scatter = _device("qk_norm_rope", some), rows is not None
    kv = k if k is not None else v
    Hq, Hkv = q.shape[1] if q is not None else 0, kv.shape[1] if kv is not None else 0
    q_out = q if q_out is None else q_out
    k_out = k if k_out is None and not scatter else k_out
    if not scatter and v is not None and v_out is None:
        raise ValueError("qk_norm_rope: v needs v_out")
    dst, kv_out_shape = _NONE4, (B, Hkv, T, D)
    if scatter:
        cache = k_out if k_out is not None else v_out
        if cache is None:
            raise ValueError("qk_norm_rope: rows need k_out or v_out")
        kv_out_shape = (cache.shape[0], Hkv, cache.shape[2], D)
        dst = _rows(rows, seqs, device, (B, T), cache.shape[0], cache.shape[2])
    elif seqs is not None:
        raise ValueError("qk_norm_rope: seqs need rows")
    shape_q, shape_kv = (B, Hq, T, D), (B, Hkv, T, D)
    qw = kw = turned = table = 0
    if eps is None and (q_weight is not None or k_weight is not None):
        raise ValueError("qk_norm_rope: weights need eps, without which there is no norm")
    if eps is not None:
        qw, kw = _whole("q_weight", q_weight, torch.float32, device, (D,)), _whole("k_weight", k_weight, torch.float32, device, (D,))
    if inv_freq is None and theta is not None:
        inv_freq = capi.inv_freq(theta, D)
    if inv_freq is not None:
        if len(inv_freq) != D // 2:
            raise ValueError(f"qk_norm_rope: expected {D // 2} frequencies, got {len(inv_freq)}")
        numpy = getattr(inv_freq, "__array_interface__", None)
        if numpy is not None and numpy["typestr"] == "<f4" and numpy["strides"] is None:
            turned, table = 1, numpy["data"][0]
        else:
            if not (isinstance(inv_freq, C.Array) and inv_freq._type_ is C.c_float):
                inv_freq = (C.c_float * (D // 2))(*[float(x) for x in inv_freq])
            turned, table = 1, C.addressof(inv_freq)
    a = _NORM.pack(_NORM.size, device, _stream(device, stream), _code(some), B, Hq, Hkv, T, D,
                   *(_NONE4 if q is None else _view("q", q, some, shape_q)), *(_NONE4 if k is None else _view("k", k, some, shape_kv)),
                   *(_NONE4 if v is None else _view("v", v, some, shape_kv)), *(_NONE4 if q_out is None else _view("q_out", q_out, some, shape_q)),
                   *(_NONE4 if k_out is None else _view("k_out", k_out, some, kv_out_shape)), *(_NONE4 if v_out is None else _view("v_out", v_out, some, kv_out_shape)),
                   int(eps is not None), eps or 0.0, qw, kw, turned, table, start_pos, _whole("positions", positions, torch.int32, device, (B, T)), *dst)
    rc = load().vb200_qk_norm_rope(a)
    if rc:
        capi.check(rc)
    return q_out, k_out, v_out


def _packed_args(q, k, batch):
    return PackedArgs(struct_size=C.sizeof(PackedArgs), device=_device("q", q), dtype=_code(q), batch=batch, Hq=q.shape[1], Hkv=k.shape[1], D=q.shape[2],
                      total_q=q.shape[0], total_k=k.shape[0])


def prefill_packed_workspace(q, k, *, batch):
    """A workspace for vb200_prefill_packed_fwd on tensors of these shapes and `batch` sequences."""
    return capi._workspace(load().vb200_prefill_packed_workspace_bytes(C.byref(_packed_args(q, k, batch))), q.device, None)


def prefill_packed(q, k, v, o=None, lse=None, *, scale, cu_seqlens_q, cu_seqlens_k=None, causal=True, workspace=None, stream=None):
    """vb200_prefill_packed_fwd: q [total_q, Hq, D], k, v [total_k, Hkv, D], cu_seqlens int32 [batch + 1] on the device, lse [Hq, total_q] fp32.  Returns o."""
    import torch
    device, batch = _device("q", q), cu_seqlens_q.numel() - 1
    if o is None:
        o = capi._output_like(q, stream)
    (tq, Hq, D), (tk, Hkv, _) = q.shape, k.shape
    if cu_seqlens_k is None and tk < tq:
        raise ValueError("prefill_packed: fewer keys than queries need cu_seqlens_k")
    L = load()
    workspace, address, size = _workspace(workspace, 0 if workspace is not None else L.vb200_prefill_packed_workspace_bytes(C.byref(_packed_args(q, k, batch))), q, stream)
    rc = L.vb200_prefill_packed_fwd(_PACKED.pack(
        _PACKED.size, device, _stream(device, stream), _code(q), batch, Hq, Hkv, D, tq, tk, int(causal), scale, *_view3("q", q, q, (tq, Hq, D)), *_view3("o", o, q, (tq, Hq, D)),
        *_view3("k", k, q, (tk, Hkv, D)), *_view3("v", v, q, (tk, Hkv, D)), _whole("lse", lse, torch.float32, device, (Hq, tq)),
        _whole("cu_seqlens_q", cu_seqlens_q, torch.int32, device, (batch + 1,)), _whole("cu_seqlens_k", cu_seqlens_k, torch.int32, device, (batch + 1,)), address, size))
    if rc:
        capi.check(rc)
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
        self.device = k_codes.get_device()
        fields = (_ptr(k_codes), _ptr(v_codes), _ptr(k_scales), _ptr(v_scales), k_codes.stride(0) // row, k_codes.stride(1) // row, self.seqs, self.cap,
                  k_exponent, v_exponent)
        self.view, self._fields = Kv4CacheView(*fields), fields

    def _call(self, entry, k, v, start_row, rows, seqs, stream):
        some = k if k is not None else v
        if some is None:
            raise ValueError("Kv4Cache: k and v are both missing")
        B, _, T, _ = some.shape
        shape, device = (B, self.Hkv, T, self.D), _device("k and v", some)
        if device != self.device:
            raise ValueError(f"Kv4Cache: rows on {some.device}, cache on {self.k_codes.device}")
        if seqs is not None and rows is None:
            raise ValueError("Kv4Cache: seqs need rows")
        rc = entry(_KV4_ROWS.pack(
            _KV4_ROWS.size, device, _stream(device, stream), _code(some), B, self.Hkv, T, self.D, *(_NONE4 if k is None else _view("k", k, some, shape)),
            *(_NONE4 if v is None else _view("v", v, some, shape)), *self._fields, start_row, *_rows(rows, seqs, device, (B, T), self.seqs, self.cap)))
        if rc:
            capi.check(rc)

    def append(self, k, v, *, start_row=0, rows=None, seqs=None, stream=None):
        """vb200_kv4_append: [B, Hkv, T, D] keys and values into rows start_row + t of sequence b, or where rows (and seqs) [B, T] int32 say."""
        self._call(load().vb200_kv4_append, k, v, start_row, rows, seqs, stream)

    def read(self, k, v, *, start_row=0, rows=None, seqs=None, stream=None):
        """vb200_kv4_read: the values of those rows into k and v (either may be None)."""
        self._call(load().vb200_kv4_read, k, v, start_row, rows, seqs, stream)


def _decode_args(q, cache, max_len, num_splits):
    return DecodeKv4Args(struct_size=C.sizeof(DecodeKv4Args), device=_device("q", q), dtype=_code(q), B=q.shape[0], Hq=q.shape[1], Hkv=cache.Hkv, D=q.shape[3],
                         cache=cache.view, max_len=max_len, num_splits=num_splits)


def decode_kv4_workspace(q, cache, *, max_len=0, num_splits=0, whole_generation=False):
    """A workspace for vb200_decode_kv4_fwd: for steps planned with this max_len, or for every step of a generation over this cache."""
    L = load()
    entry = L.vb200_decode_kv4_workspace_bytes_max if whole_generation else L.vb200_decode_kv4_workspace_bytes
    return capi._workspace(entry(C.byref(_decode_args(q, cache, max_len, num_splits))), q.device, None)


def decode_kv4(q, o, cache, *, scale, k_new=None, v_new=None, lse=None, seq_lens=None, uniform_len=0, advance_lens=False, max_len=0, num_splits=0, workspace=None, stream=None):
    """vb200_decode_kv4_fwd: one token per sequence, q and o [B, Hq, 1, D], k_new and v_new [B, Hkv, 1, D] appended first, seq_lens int32 [B] on the device."""
    import torch
    B, Hq = q.shape[0], q.shape[1]
    device, shape, new = _device("q", q), (B, Hq, 1, cache.D), (B, cache.Hkv, 1, cache.D)
    if device != cache.device:
        raise ValueError(f"decode_kv4: q on {q.device}, cache on {cache.k_codes.device}")
    L = load()
    workspace, address, size = _workspace(workspace, 0 if workspace is not None else L.vb200_decode_kv4_workspace_bytes(C.byref(_decode_args(q, cache, max_len, num_splits))), q, stream)
    rc = L.vb200_decode_kv4_fwd(_DECODE.pack(
        _DECODE.size, device, _stream(device, stream), _code(q), B, Hq, cache.Hkv, cache.D, scale, *_view("q", q, q, shape),
        *(_NONE4 if k_new is None else _view("k_new", k_new, q, new)), *(_NONE4 if v_new is None else _view("v_new", v_new, q, new)), *_view("o", o, q, shape),
        _whole("lse", lse, torch.float32, device, (B, Hq)), *cache._fields, _whole("seq_lens", seq_lens, torch.int32, device, (B,)), uniform_len, int(advance_lens), max_len, num_splits,
        address, size))
    if rc:
        capi.check(rc)
    return o

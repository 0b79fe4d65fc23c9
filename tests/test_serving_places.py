"""What the status word says of a token whose place is not in the cache."""
import ctypes as C

import numpy as np
import pytest


def message(lib, word):
    assert lib.vb200_kernel_status_of(C.c_int32(word)) == -8
    return lib.vb200_last_error_detail().decode()


def test_a_place_and_a_full_sequence_read_differently(lib):
    full = message(lib, 2 << 24 | 7)
    assert "sequence 7 is full" in full
    for seq in (0, 7, -1, -5, 2 ** 22 - 1, -2 ** 22):
        place = message(lib, 2 << 24 | 0x800000 | (seq & 0x7FFFFF))
        assert f"sequence {seq} " in place and "full" not in place and "decode" not in place and "left out" in place


@pytest.mark.gpu
def test_places_out_of_the_cache_are_named(lib):
    """Each entry point that takes places: a row past the end, a sequence past the end, one below zero, and one beyond what the word can hold."""
    import torch
    from vesper_b200 import capi, serving_capi as S
    dev = "cuda:0"
    k = torch.randn(1, 2, 1, 64, device=dev).bfloat16()
    k_cache, cache = torch.zeros(3, 2, 16, 64, dtype=torch.bfloat16, device=dev), S.Kv4Cache(3, 2, 16, 64, device=dev)
    int32 = lambda x: torch.tensor(np.asarray(x, dtype=np.int32), device=dev).view(1, 1)  # noqa: E731
    calls = [lambda r, s: S.qk_norm_rope(None, k, eps=1e-6, k_out=k_cache, rows=int32(r), seqs=int32(s)), lambda r, s: cache.append(k, k, rows=int32(r), seqs=int32(s)),
             lambda r, s: cache.read(k, None, rows=int32(r), seqs=int32(s))]
    for call in calls:
        for row, seq, named in ((16, 2, 2), (2 ** 31 - 1, 0, 0), (3, 3, 3), (3, -5, -5), (3, 2 ** 31 - 1, 2 ** 22 - 1), (3, -2 ** 31, -2 ** 22)):
            call(row, seq)
            with pytest.raises(capi.Vb200Error) as e:
                capi.check_kernel_status(0)
            assert e.value.status == -8 and f"sequence {named} " in str(e.value) and "full" not in str(e.value)
        call(15, 2)
        call(-1, 77)                                         # no place: left out, no error
        capi.check_kernel_status(0)

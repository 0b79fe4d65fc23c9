"""The largest calls of the serving operators' entry points, which no device is needed to refuse."""
import ctypes as C


def test_more_tiles_than_a_decode_step_can_deal_out_are_refused(lib):
    """The tiles of all units stand in one row, dealt out to the CTAs in 32 bits: the number of both together has to fit them, or a share would be one tile."""
    from vesper_b200 import capi, serving_capi as S
    P = 0x10000                                                  # stands for a device pointer that no refused call looks at
    row = lambda H: capi.Tensor4(P, H * 64, 64, 64)  # noqa: E731

    def status(B, shares, tiles, splits=0):
        cap, Hq = 256 * tiles, 8 * shares
        a = S.DecodeKv4Args(struct_size=C.sizeof(S.DecodeKv4Args), device=0, dtype=capi.BF16, B=B, Hq=Hq, Hkv=1, D=64, scale=0.1, q=row(Hq), o=row(Hq),
                            cache=S.Kv4CacheView(P, P, P, P, cap, cap, B, cap, 0, 0), seq_lens=P, num_splits=splits, workspace=P, workspace_bytes=0)
        return lib.vb200_decode_kv4_fwd(C.byref(a))
    counted = -4                                                 # (refused for its workspace)
    assert status(64, 8191, 4096) == counted                     # 2^31 - 2^18 tiles
    assert status(120, 4859, 3683) == -1                         # 2^31 - 8
    assert status(120, 4859, 3683, splits=2) == counted          # (pieces of a given size)
    assert status(65, 8191, 4096) == -1                          # above 2^31

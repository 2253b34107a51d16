"""CPU: how the token mixers' C entries cut a call, and the sizes they refuse before anything is launched."""
import ctypes as C

import pytest

BUF = 1 << 20        # an address that is never touched


@pytest.mark.parametrize("pairs,splits", [(1, 8), (40, 6), (72, 3), (96, 2), (128, 2), (132, 3), (160, 3), (170, 3), (192, 1), (252, 1), (256, 1),
                                          (264, 3), (340, 3), (352, 2), (384, 2), (416, 1), (512, 1), (640, 1)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_splits_of_a_frame(pairs, splits, dtype):
    """Into as many parts as were fastest for that many (item, key head) pairs over 4016 slots; never ranges below 512 slots."""
    from dtt_amd._lib import DttWattnStep, lib
    for slots, most in ((4016, 8), (1024, 2), (512, 1), (20, 1)):
        g = DttWattnStep(q=BUF, k=BUF, v=BUF, kc=BUF, vc=BUF, out=BUF, positions=BUF, B=pairs, Hq=4, Hk=1, DH=64, S=16, W=slots - 16, scale=1.0,
                         dtype=dtype, q_sb=256, q_sh=64, k_sb=64, k_sh=64, v_sb=64, v_sh=64, kc_sb=slots * 64, kc_st=64, vc_sb=slots * 64, vc_st=64)
        part = pairs * 32 * (64 + 2) * 4
        got = max(1, lib().dtt_wattn_step_ws_bytes(C.byref(g)) // part)
        assert got <= most
        if slots == 4016:
            assert got == splits
        if slots == 1024 and dtype == 0 and 128 < pairs <= 256:
            assert got == 1

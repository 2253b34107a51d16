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


def test_sizes_beyond_a_launch():
    """2^32 threads and more, or a rotary workgroup of 2^31 items, are refused by name."""
    from dtt_amd._lib import DttRecurrence, DttRotary, DttWattn, DttWattnStep, lib
    L = lib()

    def refused(rc, part):
        assert rc == -1 and part in L.dtt_last_error().decode(), (rc, L.dtt_last_error())

    a = DttWattn(q=BUF, k=BUF, v=BUF, out=BUF, rest=BUF, lse=BUF, dout=BUF, dq=BUF, dk=BUF, dv=BUF, dd=BUF, B=1 << 20, Tq=1, Tk=1, Hq=16, Hk=16, DH=32,
                 left=3, scale=1.0, dtype=1, q_sb=512, q_sh=32, k_sb=512, k_sh=32, v_sb=512, v_sh=32, g_sb=512, g_sh=32)
    refused(L.dtt_wattn_fwd(C.byref(a), None), "too many rows")
    refused(L.dtt_wattn_bwd(C.byref(a), None), "too many rows")
    s = DttWattnStep(q=BUF, k=BUF, v=BUF, kc=BUF, vc=BUF, out=BUF, positions=BUF, B=1 << 20, Hq=16, Hk=16, DH=32, S=0, W=1, scale=1.0, dtype=1,
                     q_sb=512, q_sh=32, k_sb=512, k_sh=32, v_sb=512, v_sh=32, kc_sb=512, kc_st=512, kc_sh=32, vc_sb=512, vc_st=512, vc_sh=32)
    refused(L.dtt_wattn_step(C.byref(s), None), "too many rows")
    s.B, s.W = 1, 1 << 26
    refused(L.dtt_wattn_cache_fill(C.byref(s), None, 5, None), "too many rows")
    r = DttRecurrence(x=BUF, f=BUF, y=BUF, x_so=1 << 16, f_so=1 << 16, N=1 << 17, NI=1, L=1, D=1 << 16)
    refused(L.dtt_recurrence_fwd(C.byref(r), None), "too many columns")
    refused(L.dtt_recurrence_step(BUF, BUF, BUF, BUF, 1 << 18, 1 << 16, 1 << 16, 1 << 16, 1, None), "too many columns")
    t = DttRotary(q=BUF, qo=BUF, positions=BUF, freq=BUF, B=1, T=1, Hq=1 << 26, dh=66, r=2, q_sh=66, amplitude=1.0, dtype=1)
    refused(L.dtt_rotary(C.byref(t), None), "too many heads")
    t = DttRotary(q=BUF, qo=BUF, positions=BUF, freq=BUF, B=1 << 16, T=1 << 16, Hq=1 << 12, dh=32, r=32, q_sb=32, q_st=32, q_sh=32, amplitude=1.0)
    refused(L.dtt_rotary(C.byref(t), None), "too many tokens")

"""CPU: the C entries of the long-recording token mixers refuse bad arguments before they launch anything, their structs match
the header, and the Python entries refuse CPU tensors."""
import ctypes as C
import os
import subprocess

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BUF = 1 << 20        # an address that the refused calls never touch


def _fails(rc, part):
    from dtt_amd._lib import lib
    assert rc < 0 and part in lib().dtt_last_error().decode(), (rc, lib().dtt_last_error())


def test_structs_match_the_header(tmp_path):
    from dtt_amd import _lib
    names = {n: getattr(_lib, n) for n in ("DttRecurrence", "DttRotary", "DttWattn", "DttWattnStep")}
    body = "".join(f'printf("%zu\\n", sizeof({n}));' + "".join(f'printf("%zu\\n", offsetof({n}, {f}));' for f, _ in t._fields_)
                   for n, t in names.items())
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "dtt_hip.h"\nint main(){' + body + "return 0;}")
    subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(tmp_path / "s")])
    got = [int(v) for v in subprocess.check_output([str(tmp_path / "s")]).split()]
    want = [v for t in names.values() for v in [C.sizeof(t)] + [getattr(t, f).offset for f, _ in t._fields_]]
    assert got == want


def test_recurrence_refusals():
    from dtt_amd._lib import lib, DttRecurrence
    L = lib()

    def g(**kw):
        d = dict(x=BUF, f=BUF, y=BUF, dy=BUF, dx=BUF, df=BUF, states=BUF, x_so=64, x_sl=8, f_so=64, f_sl=8, g_so=64, g_sl=8,
                 N=2, NI=1, L=8, D=8)
        return DttRecurrence(**{**d, **kw})

    for kw, part in ((dict(N=0), "sizes"), (dict(L=0), "sizes"), (dict(D=0), "sizes"), (dict(NI=3), "sizes"), (dict(NI=0), "sizes"),
                     (dict(dtype=2), "dtype"), (dict(x=None), "null"), (dict(L=(1 << 30) + 1), "2^30"),
                     (dict(L=1 << 16, D=8), "workspace")):
        _fails(L.dtt_recurrence_fwd(C.byref(g(**kw)), None), part)
        _fails(L.dtt_recurrence_bwd(C.byref(g(**kw)), None), part)
    _fails(L.dtt_recurrence_fwd(C.byref(g(y=None)), None), "null")
    _fails(L.dtt_recurrence_bwd(C.byref(g(dy=None)), None), "null")
    _fails(L.dtt_recurrence_bwd(C.byref(g(states=None, L=65)), None), "null")
    _fails(L.dtt_recurrence_fwd(None, None), "null")
    need = L.dtt_recurrence_ws_bytes(C.byref(g(L=1 << 16)))
    assert need > 0 and L.dtt_recurrence_ws_bytes(C.byref(g())) == 0 and L.dtt_recurrence_ws_bytes(None) == 0
    _fails(L.dtt_recurrence_fwd(C.byref(g(L=1 << 16, ws=BUF, ws_bytes=need - 1)), None), "workspace")
    # the backward call cuts its tiles as the forward call did, whatever the strides of dy are
    assert L.dtt_recurrence_states(C.byref(g(L=1000))) == L.dtt_recurrence_states(C.byref(g(L=1000, g_sl=9, dy=BUF + 2)))
    p = C.c_void_p(BUF)
    _fails(L.dtt_recurrence_step(None, p, p, p, 1, 1, C.c_int64(1), C.c_int64(1), 0, None), "null")
    _fails(L.dtt_recurrence_step(p, p, p, p, 0, 1, C.c_int64(1), C.c_int64(1), 0, None), "bad arguments")
    _fails(L.dtt_recurrence_step(p, p, p, p, 1, 1, C.c_int64(1), C.c_int64(1), 3, None), "bad arguments")


def test_attention_refusals():
    from dtt_amd._lib import lib, DttWattn, DttWattnStep
    L = lib()

    def g(**kw):
        d = dict(q=BUF, k=BUF, v=BUF, out=BUF, lse=BUF, dout=BUF, dq=BUF, dk=BUF, dv=BUF, dd=BUF, B=1, Tq=4, Tk=4, Hq=2, Hk=1,
                 DH=32, left=3, scale=1.0, q_sb=256, q_st=64, q_sh=32, k_sb=128, k_st=32, k_sh=32, v_sb=128, v_st=32, v_sh=32,
                 g_sb=256, g_st=64, g_sh=32)
        return DttWattn(**{**d, **kw})

    for kw, part in ((dict(B=0), "sizes"), (dict(Tq=0), "sizes"), (dict(Tk=0), "sizes"), (dict(Hq=3, Hk=2), "sizes"), (dict(DH=48), "head width"),
                     (dict(left=-1), "window"), (dict(right=-1), "window"), (dict(offset=-1), "window"), (dict(sinks=129), "sinks"),
                     (dict(sinks=-1), "sinks"), (dict(q=None), "null"), (dict(q_st=33), "16 bytes"), (dict(q_st=24), "row strides"),
                     (dict(k_st=(1 << 22) + 8), "row strides"), (dict(v_st=0), "row strides"), (dict(k=BUF + 4), "16 bytes"),
                     (dict(dtype=7), "dtype"), (dict(scale=0.0), "scale"), (dict(scale=-1.0), "scale"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale")):
        _fails(L.dtt_wattn_fwd(C.byref(g(**kw)), None), part)
        _fails(L.dtt_wattn_bwd(C.byref(g(**kw)), None), part)
    _fails(L.dtt_wattn_fwd(C.byref(g(out=None)), None), "output")
    _fails(L.dtt_wattn_bwd(C.byref(g(lse=None)), None), "null")
    _fails(L.dtt_wattn_bwd(C.byref(g(g_st=33)), None), "16 bytes")
    far = dict(Tq=5000, Tk=5000, sinks=2)
    need = L.dtt_wattn_bwd_ws_bytes(C.byref(g(**far)))
    assert need > 0 and L.dtt_wattn_bwd_ws_bytes(C.byref(g())) == 0 and L.dtt_wattn_bwd_ws_bytes(None) == 0
    _fails(L.dtt_wattn_bwd(C.byref(g(ws=BUF, ws_bytes=need - 1, **far)), None), "workspace")

    def s(**kw):
        d = dict(q=BUF, k=BUF, v=BUF, kc=BUF, vc=BUF, out=BUF, positions=BUF, B=1, Hq=2, Hk=1, DH=64, S=2, W=30, scale=1.0, q_sh=64,
                 kc_st=64, vc_st=64)
        return DttWattnStep(**{**d, **kw})

    for kw, part in ((dict(B=0), "sizes"), (dict(W=0), "sizes"), (dict(S=-1), "sizes"), (dict(Hq=3, Hk=2), "sizes"), (dict(DH=33), "head width"),
                     (dict(kc=None), "null"), (dict(kc_st=62), "16 bytes"), (dict(W=1 << 30), "sizes"), (dict(dtype=-1), "dtype"),
                     (dict(scale=-1.0), "scale")):
        _fails(L.dtt_wattn_step(C.byref(s(**kw)), None), part)
        _fails(L.dtt_wattn_cache_fill(C.byref(s(**kw)), None, 5, None), part)
    _fails(L.dtt_wattn_step(C.byref(s(positions=None)), None), "null")
    _fails(L.dtt_wattn_step(C.byref(s(W=8000)), None), "workspace")
    _fails(L.dtt_wattn_cache_fill(C.byref(s()), None, 0, None), "T=0")


def test_rotary_refusals():
    from dtt_amd._lib import lib, DttRotary

    def g(**kw):
        d = dict(q=BUF, k=BUF, qo=BUF, ko=BUF, positions=BUF, freq=BUF, B=1, T=2, Hq=1, Hk=1, dh=8, r=8, q_st=8, k_st=8, amplitude=1.0)
        return DttRotary(**{**d, **kw})

    for kw, part in ((dict(T=0), "sizes"), (dict(r=7), "sizes"), (dict(r=10), "sizes"), (dict(Hk=-1), "sizes"), (dict(k=None), "null"),
                     (dict(freq=None), "null"), (dict(dtype=4), "dtype"), (dict(dh=9000, r=8000), "4096")):
        _fails(lib().dtt_rotary(C.byref(g(**kw)), None), part)


def test_cpu_tensors_are_refused():
    import dtt_amd as a
    x, q, kc = torch.zeros(2, 4, 8), torch.zeros(2, 4, 2, 32), torch.zeros(2, 6, 2, 32)
    pos = torch.zeros(2, dtype=torch.int64)
    for f in (lambda: a.gated_recurrence(x, x), lambda: a.gated_recurrence_step(x[:, 0], x[:, 0], torch.zeros(2, 8)),
              lambda: a.window_attention(q, q, q, 3), lambda: a.window_attention_step(q[:, 0], q[:, 0], q[:, 0], kc, kc, pos),
              lambda: a.window_cache_fill(q, q, kc, kc), lambda: a.rotary(q, q, torch.arange(4), a.rotary_frequencies(32))):
        with pytest.raises(a.DttError, match="CUDA"):
            f()

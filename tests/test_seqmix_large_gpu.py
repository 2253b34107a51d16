"""The token mixers' kernels for large calls, against the same float64 references and bounds as the small ones: attention over
more row and key tiles than the forms that split them take, rotary workgroups of several tokens, the recurrence with one
time lane over an odd number of channels.  Many short items keep the references small; what ran is read from a trace, so
that a changed rule cannot empty the tests."""
import re

import pytest
import torch
from test_seqmix_gpu import A, BF, DEV, F32, attn_check, attn_ref, rec_check, rec_ref, R, rnd, rot_ref, seen, within

pytestmark = pytest.mark.gpu
NAME = {BF: "bf16", F32: "float"}


def kernels(call):
    """The kernels that `call` launches, with their template arguments, and what it returns."""
    from torch.profiler import ProfilerActivity, profile
    call()
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA], acc_events=True) as p:
        out = call()
        torch.cuda.synchronize()
    names = (re.search(r"(\w+_kernel)<([^>]*)>", e.name) for e in p.events())
    return {(m.group(1), m.group(2).replace(" ", "")) for m in names if m}, out


LARGE = [  # B, Tq, Tk, Hq, Hk, left, right, sinks, offset, ragged
    (32, 260, 260, 8, 4, 20, 9, 33, None, True),        # first tokens on both sides of a 32-key border, rows beyond their chunks' edge
    (64, 140, 140, 4, 4, 200, 0, 0, None, True),        # everything before is seen
    (64, 129, 300, 4, 2, 60, 3, 4, 171, False),         # the last rows of longer sequences
    (32, 150, 150, 10, 5, 31, 0, 1, None, False),
]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hk,left,right,sinks,offset,ragged", LARGE)
def test_attention_of_many_rows(dt, dh, B, Tq, Tk, Hq, Hk, left, right, sinks, offset, ragged):
    q, k, v = rnd(1, B, Tq, Hq, dh, dt=dt, grad=True), rnd(2, B, Tk, Hk, dh, dt=dt, grad=True), rnd(3, B, Tk, Hk, dh, dt=dt, grad=True)
    do = rnd(4, B, Tq, Hq, dh, dt=dt)
    ln = None
    if ragged:
        ln = torch.randint(0, Tk + 1, (B,), generator=torch.Generator().manual_seed(5), dtype=torch.int32)
        ln[:3] = torch.tensor([Tk, 0, 1])
        ln = ln.to(DEV)

    def call():
        o = A().window_attention(q, k, v, left, right, sinks, lengths=ln, offset=offset)
        return (o,) + torch.autograd.grad(o, (q, k, v), do)

    ran, outs = kernels(call)
    t = NAME[dt]
    for want in (("wattn_fwd_kernel", f"{t},{dh},4,1"), ("wattn_dq_kernel", f"{t},{dh},4,1"),
                 ("wattn_dkv_kernel", f"{t},{dh},4,{2 if dt == BF else 1}")):
        assert want in ran, ran
    assert (("wattn_sink_sum_kernel", t) in ran) == (sinks > 0 and Tq > 128 + left - (offset or 0)), ran
    see = seen(Tq, Tk, left, right, sinks, Tk - Tq if offset is None else offset, ln, B)
    refs = attn_ref(q, k, v, see, dh ** -0.5, dt, do)
    attn_check(outs, refs)
    dead = ~see.any(-1)
    assert not outs[0][dead].any() and not outs[1][dead].any()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("D,reverse", [(255, False), (255, True), (257, False)])
def test_recurrence_of_many_odd_rows(dt, D, reverse):
    N, L = 1042, 19
    x, f = rnd(1, N, L, D, dt=dt, grad=True), rnd(2, N, L, D, dt=dt, mean=2.0, std=1.5, grad=True)
    h0, dy, dl = rnd(3, N, D, grad=True), rnd(4, N, L, D, dt=dt), rnd(5, N, D)
    lens = torch.randint(0, L + 1, (N,), generator=torch.Generator().manual_seed(1)).to(DEV)

    def call():
        out = A().gated_recurrence(x, f, h0, reverse=reverse, lengths=lens)
        return out + torch.autograd.grad(out, (x, f, h0), (dy, dl))

    ran, outs = kernels(call)
    for name in ("rec_fwd_kernel", "rec_bwd_kernel"):
        assert (name, f"{NAME[dt]},1,1") in ran, ran
    rec_check(outs, rec_ref(x.detach(), f.detach(), h0.detach(), reverse, lens, dy, dl), dt)


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,dh,r", [(1, 5003, 2, 1, 32, 32), (3, 1667, 3, 1, 64, 48), (2, 4099, 1, 1, 128, 96)])
def test_rotary_of_many_tokens(dt, inter, B, T, Hq, Hk, dh, r):
    """Several tokens a workgroup (n / 1024 of them; none of these counts is a multiple of that)."""
    assert B * T // 1024 > 1 and B * T % (B * T // 1024)
    q, k = rnd(1, B, T, Hq, dh, dt=dt, grad=True), rnd(2, B, T, Hk, dh, dt=dt, grad=True)
    dq, dk = rnd(3, B, T, Hq, dh, dt=dt), rnd(4, B, T, Hk, dh, dt=dt)
    freq, pos = A().rotary_frequencies(r, device=DEV), torch.arange(T, device=DEV)[None] + 1000 * torch.arange(B, device=DEV)[:, None]
    qo, ko = A().rotary(q, k, pos, freq, interleaved=inter)
    g = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
    for got, src, sign in ((qo, q, 1), (ko, k, 1), (g[0], dq, -1), (g[1], dk, -1)):
        ref, err = rot_ref(src, pos, freq, inter, 1.0, sign)
        within(got, ref, err * 1.01 + R(dt) * (ref.abs() + err))
    assert torch.equal(qo[..., r:], q[..., r:])

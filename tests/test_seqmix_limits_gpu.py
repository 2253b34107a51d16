"""Attention calls at the ends of what the documentation allows."""
import pytest
import torch
from test_seqmix_gpu import A, BF, DEV, F32, attn_check, attn_ref, rnd, seen, within

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("left", [1 << 30, 1 << 40, (1 << 28) - 1, (1 << 28) + 1])
def test_windows_beyond_the_last_position(dt, left):
    """Rows at positions 2^28 - 1, 2^28, 2^28 + 1 over ten keys: a window that reaches back to key 0 sees it."""
    Tq, Tk, offset = 3, 10, (1 << 28) - 1
    q, k, v = rnd(1, 1, Tq, 2, 32, dt=dt, grad=True), rnd(2, 1, Tk, 2, 32, dt=dt, grad=True), rnd(3, 1, Tk, 2, 32, dt=dt, grad=True)
    do = rnd(4, 1, Tq, 2, 32, dt=dt)
    o = A().window_attention(q, k, v, left, offset=offset)
    g = torch.autograd.grad(o, (q, k, v), do)
    see = seen(Tq, Tk, left, 0, 0, offset, None, 1)
    assert bool(see.all()) == (left > 1 << 28)
    attn_check((o,) + g, attn_ref(q, k, v, see, 32 ** -0.5, dt, do))


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,Hq,Hk,M", [(40, 8, 4, 1700), (33, 4, 4, 1100), (66, 20, 4, 1600), (90, 4, 4, 1030)])
def test_frames_of_many_streams_in_parts(dt, B, Hq, Hk, M):
    """More (item, key head) pairs than half the CUs, cut into two or three parts, some items too young to have slots in all."""
    q, k, v = rnd(1, B, Hq, 64, dt=dt), rnd(2, B, Hk, 64, dt=dt), rnd(3, B, Hk, 64, dt=dt)
    kc, vc = rnd(4, B, M, Hk, 64, dt=dt), rnd(5, B, M, Hk, 64, dt=dt)
    pos = torch.randint(-1, 2 * M, (B,), generator=torch.Generator().manual_seed(3))
    pos[:4] = torch.tensor([-1, 0, 511, 5 * M])
    pos = pos.to(DEV)
    out = A().window_attention_step(q, k, v, kc, vc, pos, 3)
    see = (torch.arange(M, device=DEV)[None] <= pos[:, None])[:, None]
    (ref, err), = attn_ref(q[:, None], kc, vc, see, 0.125, dt)
    within(out, ref[:, 0], err[:, 0] * 1.01 + 1e-30)
    assert not out[pos < 0].any()

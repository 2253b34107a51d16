"""Attention calls at the ends of what the documentation allows."""
import pytest
import torch
from test_seqmix_gpu import A, BF, DEV, F32, attn_check, attn_ref, rnd, seen

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

"""How the token mixers' calls that replace tensors in place, and arguments that could want a gradient, meet autograd."""
import pytest
import torch
from test_seqmix_gpu import A, BF, DEV, F32, rnd

pytestmark = pytest.mark.gpu


def test_a_state_that_was_stepped_on_is_not_read_by_a_backward_pass():
    """The recurrence saves its h0 for the backward pass; a step replaces the same tensor: an error, as behind state.copy_()."""
    x, f = rnd(1, 2, 9, 8, grad=True), rnd(2, 2, 9, 8, grad=True)
    state = rnd(3, 2, 8)
    y, _ = A().gated_recurrence(x, f, state)
    with torch.no_grad():
        A().gated_recurrence_step(x[:, 0], f[:, 0], state)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, _ = A().gated_recurrence(x, f, state.clone())                          # of a copy: as ever
    want = torch.autograd.grad(y.sum(), f, retain_graph=True)[0]
    with torch.no_grad():
        A().gated_recurrence_step(x[:, 0], f[:, 0], state)
    assert torch.equal(torch.autograd.grad(y.sum(), f)[0], want)


@pytest.mark.parametrize("how", ["step", "fill"])
@pytest.mark.parametrize("dt", [F32, BF])
def test_caches_that_were_written_are_not_read_by_a_backward_pass(dt, how):
    q, kc, vc = rnd(1, 2, 5, 2, 32, dt=dt, grad=True), rnd(2, 2, 20, 2, 32, dt=dt), rnd(3, 2, 20, 2, 32, dt=dt)
    k, v = rnd(4, 2, 2, 32, dt=dt), rnd(5, 2, 2, 32, dt=dt)
    for keys, values in ((kc[:, 3:17], vc.clone()[:, 3:17]), (kc.clone()[:, 3:17], vc[:, 3:17])):      # views of either cache
        o = A().window_attention(q, keys, values, 4)
        with torch.no_grad():
            if how == "step":
                A().window_attention_step(q[:, 0], k, v, kc, vc, torch.tensor([4, 5], device=DEV))
            else:
                A().window_cache_fill(k[:, None], v[:, None], kc, vc)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            o.sum().backward()


def test_caches_in_a_graph_are_refused():
    """Their gradient would miss what is written: refused while gradients are recorded, taken under no_grad."""
    q, k = rnd(1, 1, 2, 32), rnd(2, 1, 2, 32)
    kc, vc, pos = rnd(3, 1, 6, 2, 32, grad=True), rnd(4, 1, 6, 2, 32), torch.zeros(1, dtype=torch.int64, device=DEV)
    for a, b in ((kc, vc), (vc, kc), (kc * 1, vc)):
        for call in (lambda: A().window_attention_step(q, k, k, a, b, pos), lambda: A().window_cache_fill(k[:, None], k[:, None], a, b)):
            with pytest.raises(A().DttError, match="no gradient"):
                call()
            with torch.no_grad():
                call()


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("N,L,D", [(4, 20, 6), (4, 4000, 16), (1040, 12, 256)])
def test_padding_has_no_gradient_when_the_state_is_not_finite(N, L, D, dt, reverse):
    """One time lane, tiles of eight lanes, segments: gradients behind an item's length are 0 whatever passes there, and items and
    channels whose state is finite get the gradients that they get alone."""
    x, f = rnd(1, N, L, D, dt=dt, grad=True), rnd(2, N, L, D, dt=dt, mean=2.0, grad=True)
    h0, dy, dl = rnd(3, N, D), rnd(4, N, L, D, dt=dt), rnd(5, N, D)
    lens = torch.randint(0, L + 1, (N,), generator=torch.Generator().manual_seed(1))
    lens[:4] = torch.tensor([0, L, L // 2, 1])
    lens = lens.to(DEV)
    clean = torch.autograd.grad(A().gated_recurrence(x, f, h0, reverse, lens), (x, f), (dy, dl))
    bad, badl = h0.clone(), dl.clone()
    bad[0, 0], bad[2, 1], bad[3, 2] = float("inf"), float("nan"), float("-inf")
    badl[0, 3], badl[2, 4], badl[3, 5] = float("nan"), float("inf"), float("nan")
    dirty = torch.zeros(N, D, dtype=torch.bool, device=DEV)
    dirty[[0, 0, 2, 2, 3, 3], [0, 3, 1, 4, 2, 5]] = True
    got = torch.autograd.grad(A().gated_recurrence(x, f, bad, reverse, lens), (x, f), (dy, badl))
    pad = (torch.arange(L, device=DEV)[None] >= lens[:, None])[..., None].expand(N, L, D)
    for g, c in zip(got, clean):
        assert not g[pad].any()
        fine = ~dirty[:, None].expand(N, L, D)
        assert torch.equal(g[fine], c[fine])


def test_frequencies_that_want_a_gradient_are_refused():
    freq, pos = A().rotary_frequencies(32, device=DEV).requires_grad_(), torch.arange(4, device=DEV)
    q = rnd(1, 1, 4, 2, 32)
    for t in (q, rnd(1, 1, 4, 2, 32, grad=True)):
        with pytest.raises(A().DttError, match="gradient of freq"):
            A().rotary(t, t, pos, freq)
    with torch.no_grad():
        a = A().rotary(q, q, pos, freq)
    assert all(torch.equal(x, y) for x, y in zip(a, A().rotary(q, q, pos, freq.detach())))

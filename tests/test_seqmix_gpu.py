"""Token mixers for long recordings against plain implementations in float64: the gated linear recurrence, windowed
attention with first tokens that stay visible (whole sequences and one frame at a time) and rotary positions.

Tolerances are bounds, element by element, computed in float64 beside the reference: U = 2^-24 is half a step of float32,
R(dtype) half a step of the output's type (bfloat16 2^-8, float32 2^-24), and every bound counts roundings of the sums of
magnitudes that the kernel adds up."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
U = 2.0 ** -24
BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64


def R(dt):
    return torch.finfo(dt).eps / 2


def A():
    import dtt_amd
    return dtt_amd


def rnd(seed, *shape, dt=F32, std=1.0, mean=0.0, grad=False):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * std + mean).to(dt).requires_grad_(grad)


def within(got, ref, bound, what=""):
    """|got - ref| <= bound everywhere (float64)."""
    got = got.detach().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert torch.isfinite(got).all(), what
    over = (got - ref).abs() - bound
    assert float(over.max() if over.numel() else 0.0) <= 0.0, (what, float(over.max()), float((got - ref).abs().max()))


# --------------------------------------------------------------------------- #
# gated linear recurrence
# --------------------------------------------------------------------------- #
def rec_ref(x, f, h0, reverse, lens, dy=None, dlast=None):
    """[N, L, D] float64 loops; values and bounds.  A step's error: the gates carry at most 6 U, the product and sum 2 U, and
    the tree over time lanes adds two more per combination: C = 16 U of the magnitudes, passed on by a."""
    C = 16 * U
    N, L, D = x.shape
    x, f = x.double(), f.double()
    h = torch.zeros(N, D, dtype=F64, device=x.device) if h0 is None else h0.double().clone()
    a, i = torch.sigmoid(f), torch.sigmoid(-f)
    m, e = h.abs(), torch.zeros_like(h)
    y, ey = torch.zeros_like(x), torch.zeros_like(x)
    hb, mb, eb = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    order = range(L - 1, -1, -1) if reverse else range(L)
    lens = torch.full((N,), L, device=x.device) if lens is None else lens
    for t in order:
        on = (t < lens)[:, None]
        hb[:, t], mb[:, t], eb[:, t] = h, m, e
        xt = torch.where(on, x[:, t], 0.0)
        m = torch.where(on, a[:, t] * m + i[:, t] * xt.abs(), m)
        h = torch.where(on, a[:, t] * h + i[:, t] * xt, h)
        e = torch.where(on, a[:, t] * e + C * m, e)
        y[:, t], ey[:, t] = torch.where(on, h, 0.0), torch.where(on, e, 0.0)
    out = [(y, ey), (h, e)]
    if dy is None:
        return out
    dy = dy.double()
    s = torch.zeros(N, D, dtype=F64, device=x.device) if dlast is None else dlast.double().clone()
    ms, es = s.abs(), torch.zeros_like(s)
    dx, edx, df, edf = (torch.zeros_like(x) for _ in range(4))
    for t in reversed(order):
        on = (t < lens)[:, None]
        at, it, d = a[:, t], i[:, t], torch.where(on, dy[:, t], 0.0)
        xt = torch.where(on, x[:, t], 0.0)
        g, mg, eg = d + s, d.abs() + ms, es + C * (d.abs() + ms)
        dx[:, t], edx[:, t] = torch.where(on, it * g, 0.0), torch.where(on, it * (eg + C * mg), 0.0)
        diff, mdiff = hb[:, t] - xt, mb[:, t] + xt.abs()
        df[:, t] = torch.where(on, at * it * g * diff, 0.0)
        edf[:, t] = torch.where(on, at * it * (eg * mdiff + mg * eb[:, t] + C * mg * mdiff), 0.0)
        s, ms, es = torch.where(on, at * g, s), torch.where(on, at * mg, ms), torch.where(on, at * (eg + C * mg), es)
    return out + [(dx, edx), (df, edf), (s, es)]


# The floor of the recurrence's bounds: the gates' exponentials and products below 2^-126 may be flushed to zero, and what is
# flushed is then multiplied by at most |g| |h - x|, below 64 for the inputs here: 2^-126 x 64 = 2^-120.
FLUSH = 2.0 ** -120


def rec_check(outs, refs, dt):
    for got, (ref, err), name, o in zip(outs, refs, ("y", "last", "dx", "df", "dh0"), (dt, F32, dt, dt, F32)):
        within(got.reshape(ref.shape), ref, err * (1 + 2.0 ** -7) + R(o) * ref.abs() + FLUSH, name)


REC = [  # N, L, D, reverse, lens, h0
    (1, 1, 1, False, None, False), (3, 2, 5, True, None, True), (2, 63, 8, False, None, True), (2, 64, 12, True, None, False),
    (2, 65, 64, False, None, True), (3, 130, 33, True, (130, 0, 1), True), (4, 47, 100, False, (47, 1, 0, 31), True),
    (1, 1500, 16, False, None, True), (2, 4100, 24, True, (4099, 700), True), (1, 9001, 4, False, None, False),
    (2100, 5, 252, False, None, True), (2048, 17, 256, True, "r", True), (70, 9, 7500, False, None, False),
]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N,L,D,reverse,lens,h0", REC)
def test_recurrence_forward_and_gradients(dt, N, L, D, reverse, lens, h0):
    x, f = rnd(1, N, L, D, dt=dt, grad=True), rnd(2, N, L, D, dt=dt, mean=2.0, std=1.5, grad=True)
    h = rnd(3, N, D, grad=True) if h0 else None
    dy, dl = rnd(4, N, L, D, dt=dt), rnd(5, N, D)
    if lens == "r":
        lens = torch.randint(0, L + 1, (N,), generator=torch.Generator().manual_seed(1))
    lens = None if lens is None else torch.as_tensor(lens, device=DEV, dtype=torch.int32)
    y, last = A().gated_recurrence(x, f, h, reverse=reverse, lengths=lens)
    assert y.dtype == dt and last.dtype == F32
    with torch.no_grad():
        y2, last2 = A().gated_recurrence(x, f, h, reverse=reverse, lengths=lens)
    assert torch.equal(y, y2) and torch.equal(last, last2)
    ins = (x, f) + ((h,) if h0 else ())
    g1 = torch.autograd.grad((y, last), ins, (dy, dl), retain_graph=True)
    g2 = torch.autograd.grad((y, last), ins, (dy, dl))
    assert all(torch.equal(a, b) for a, b in zip(g1, g2))
    rec_check((y, last) + g1, rec_ref(x.detach(), f.detach(), h.detach() if h0 else None, reverse, lens, dy, dl), dt)


@pytest.mark.parametrize("dt", [F32, BF])
def test_recurrence_extreme_gates(dt):
    f = torch.tensor([0.0, -0.0, 1e-6, 20.0, -20.0, 88.0, -88.0, 200.0, -200.0, math.inf, -math.inf, 8.0], device=DEV)
    f = f[None, None].repeat(2, 70, 1).to(dt).requires_grad_()
    x, dy = rnd(1, 2, 70, 12, dt=dt, grad=True), rnd(2, 2, 70, 12, dt=dt)
    y, last = A().gated_recurrence(x, f)
    g = torch.autograd.grad(y, (x, f), dy)
    rec_check((y, last) + g, rec_ref(x.detach(), f.detach(), None, False, None, dy), dt)


def test_recurrence_padding_is_never_read():
    lens = torch.tensor([40, 0, 1, 100], dtype=torch.int32, device=DEV)
    dead = (torch.arange(100, device=DEV)[None] >= lens[:, None])[..., None]
    for dt in (F32, BF):
        for rev in (False, True):
            x, f, dy = (rnd(s, 4, 100, 32, dt=dt) for s in (1, 2, 3))
            clean = A().gated_recurrence(x, f, None, rev, lens)
            xn, fn, dn = (torch.where(dead, v, t).to(dt) for t, v in ((x, math.nan), (f, math.inf), (dy, math.nan)))
            xn, fn = xn.requires_grad_(), fn.requires_grad_()
            y, last = A().gated_recurrence(xn, fn, None, rev, lens)
            assert torch.equal(y, clean[0]) and torch.equal(last, clean[1])
            assert not torch.where(dead, y, 0).any()
            for g in torch.autograd.grad(y, (xn, fn), dn):
                assert torch.isfinite(g).all() and not torch.where(dead, g, 0).any()


def test_recurrence_nan_gate_is_seen():
    x, f = rnd(1, 1, 40, 8), rnd(2, 1, 40, 8)
    f[0, 20, 3] = math.nan
    y, last = A().gated_recurrence(x, f)
    assert torch.isnan(y[0, 20:, 3]).all() and torch.isnan(last[0, 3])
    assert torch.isfinite(y[0, :20]).all() and torch.isfinite(y[0, :, 4:]).all()


@pytest.mark.parametrize("dt", [F32, BF])
def test_recurrence_strided_views(dt):
    """Slices of a fused projection, the frequency-axis view of [B, T, F, C] rows (two batch axes), odd offsets."""
    xf = rnd(1, 3, 50, 2 * 36, dt=dt, grad=True)
    x, f = xf[..., :36], xf[..., 36:]
    dy = rnd(2, 3, 50, 36, dt=dt)
    y, _ = A().gated_recurrence(x, f)
    g, = torch.autograd.grad(y, xf, dy)
    ref = rec_ref(x.detach(), f.detach(), None, False, None, dy)
    rec_check((y,), ref[:1], dt)
    within(g[..., :36], ref[2][0], ref[2][1] * 1.01 + R(dt) * ref[2][0].abs(), "dx")
    within(g[..., 36:], ref[3][0], ref[3][1] * 1.01 + R(dt) * ref[3][0].abs(), "df")
    z = rnd(3, 2, 21, 6, 40, dt=dt)                                          # [B, F, T, C] -> items (B, T), steps F
    zt, ft = z.permute(0, 2, 1, 3), z.flip(1).permute(0, 2, 1, 3)
    lens = torch.arange(12, device=DEV).view(2, 6) * 2
    h0 = rnd(4, 2, 6, 40)
    y, last = A().gated_recurrence(zt, ft, h0, True, lens)
    ref = rec_ref(zt.reshape(12, 21, 40), ft.reshape(12, 21, 40), h0.view(12, 40), True, lens.view(-1))
    rec_check((y, last), ref, dt)
    w = rnd(5, 2 * 30 * 17 + 1, dt=dt)[1:].view(2, 30, 17)                   # rows on odd elements
    y, last = A().gated_recurrence(w[:, :, 1:], w[:, :, :-1])
    rec_check((y, last), rec_ref(w[:, :, 1:], w[:, :, :-1], None, False, None), dt)
    wt = rnd(6, 2, 24, 30, dt=dt).transpose(1, 2)                            # innermost axis strided: copied
    rec_check(A().gated_recurrence(wt, wt), rec_ref(wt, wt, None, False, None), dt)
    one = rnd(7, 1, 30, 24, dt=dt).expand(3, 30, 24)                         # broadcast input
    rec_check(A().gated_recurrence(one, one), rec_ref(one, one, None, False, None), dt)


@pytest.mark.parametrize("which", ["last", "y", "expanded"])
def test_recurrence_partial_and_expanded_gradients(which):
    x, f, h0 = rnd(1, 2, 90, 20, grad=True), rnd(2, 2, 90, 20, grad=True), rnd(3, 2, 20, grad=True)
    y, last = A().gated_recurrence(x, f, h0)
    loss = {"last": last.sum(), "y": y[:, 3].sum(), "expanded": y.sum()}[which]
    g = torch.autograd.grad(loss, (x, f, h0))
    dy, dl = torch.zeros(2, 90, 20, device=DEV), torch.zeros(2, 20, device=DEV)
    if which == "last":
        dl += 1
    elif which == "y":
        dy[:, 3] = 1
    else:
        dy += 1
    rec_check((y, last) + g, rec_ref(x.detach(), f.detach(), h0.detach(), False, None, dy, dl), F32)


def test_recurrence_gradient_against_differences():
    """Central differences of the float64 formula along random directions: truncation O(eps^2) = 1e-8 relative to the third
    derivatives (gates' are below 1), kernel error below 1e-5 of the gradient's norm."""
    x, f, h0 = rnd(1, 2, 40, 8, grad=True), rnd(2, 2, 40, 8, grad=True), rnd(3, 2, 8, grad=True)
    dy, dl = rnd(4, 2, 40, 8), rnd(5, 2, 8)
    g = torch.autograd.grad(A().gated_recurrence(x, f, h0), (x, f, h0), (dy, dl))

    def loss(*a):
        (y, _), (last, _) = rec_ref(*a, False, None)
        return float((y * dy.double()).sum() + (last * dl.double()).sum())

    base = [t.detach().double() for t in (x, f, h0)]
    for k in range(3):
        d = rnd(10 + k, *base[k].shape).double()
        eps = 1e-4
        up, dn = ([b + s * eps * d if i == k else b for i, b in enumerate(base)] for s in (1, -1))
        num = (loss(*up) - loss(*dn)) / (2 * eps)
        assert abs(num - float((g[k].double() * d).sum())) <= 1e-5 * float(g[k].double().norm() * d.norm()) + 1e-6


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("N,D", [(1, 1), (3, 7), (64, 1024), (5, 40)])
def test_recurrence_steps_follow_the_sequence(dt, N, D):
    x, f, state = rnd(1, N, 6, D, dt=dt), rnd(2, N, 6, D, dt=dt, mean=2.0), rnd(3, N, D)
    y, last = A().gated_recurrence(x, f, state)
    ref = rec_ref(x, f, state, False, None)
    st = state.clone()
    for t in range(6):
        yt = A().gated_recurrence_step(x[:, t], f[:, t], st)                 # strided rows
        within(yt, ref[0][0][:, t], ref[0][1][:, t] + R(dt) * ref[0][0][:, t].abs() * 1.01 + FLUSH, f"step {t}")
    within(st, ref[1][0], ref[1][1] * 1.01 + R(F32) * ref[1][0].abs(), "state")


def test_recurrence_empty():
    x = torch.zeros(2, 0, 8, device=DEV)
    h0 = rnd(1, 2, 8)
    y, last = A().gated_recurrence(x, x, h0)
    assert y.shape == (2, 0, 8) and torch.equal(last, h0)
    y, last = A().gated_recurrence(torch.zeros(0, 5, 8, device=DEV), torch.zeros(0, 5, 8, device=DEV))
    assert y.shape == (0, 5, 8) and last.shape == (0, 8)


# --------------------------------------------------------------------------- #
# windowed attention
# --------------------------------------------------------------------------- #
def seen(Tq, Tk, left, right, sinks, offset, lens, B):
    p, j = (offset + torch.arange(Tq, device=DEV))[:, None], torch.arange(Tk, device=DEV)[None]
    s = ((j <= p + right) & ((j >= p - left) | (j < sinks)))[None].expand(B, Tq, Tk)
    if lens is not None:
        n = lens.to(DEV)[:, None, None]
        s = s & (j[None] < n) & (p[None] < n)
    return s


def attn_ref(q, k, v, see, scale, dt, do=None):
    """Float64 values and bounds, [B, T, H, dh].  A score's error is that of a sum of dh products in float32, (dh + 4) U of
    its magnitudes; it and a few U of the exponential move a weight by a relative `w`; bfloat16 rounds the weights (and dS)
    once more, R(bf16) each; sums over n keys add n U of their magnitudes."""
    B, Tq, Hq, dh = q.shape
    Tk, Hk = k.shape[1:3]
    G = Hq // Hk
    qd, kd, vd = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    qd = qd.reshape(B, Hk, G, Tq, dh)
    kd, vd = kd[:, :, None], vd[:, :, None]
    sm = see[:, None, None]
    alive = sm.transpose(-1, -2).any(-1)                                      # keys that anyone sees
    kd, vd = (torch.where(alive[..., None], t, 0.0) for t in (kd, vd))
    rows = sm.any(-1)[..., None]
    qd = torch.where(rows, qd, 0.0)
    s = torch.where(sm, qd @ kd.transpose(-1, -2) * scale, -math.inf)
    P = torch.softmax(s, -1).nan_to_num(0.0)
    es = torch.where(sm, (dh + 8) * U * abs(scale) * (qd.abs() @ kd.abs().transpose(-1, -2)), 0.0)
    rp = R(BF) if dt == BF else 2 * U
    n = Tk
    w = 2 * es.amax(-1, keepdim=True) + 16 * U + n * U                      # relative error of a normalised weight
    o = P @ vd
    eo = (w + rp) * (P @ vd.abs()) + n * U * (P @ vd.abs())
    back = lambda t, H, T: t.reshape(B, H, T, dh).transpose(1, 2)  # noqa: E731
    out = [(back(o, Hq, Tq), back(eo + R(dt) * o.abs(), Hq, Tq))]
    if do is None:
        return out
    dd = do.detach().double().transpose(1, 2).reshape(B, Hk, G, Tq, dh)
    dd = torch.where(rows, dd, 0.0)
    dP, mP = dd @ vd.transpose(-1, -2), dd.abs() @ vd.abs().transpose(-1, -2)
    D = (dd * o).sum(-1, keepdim=True)
    rest = 2.0 ** -16 if dt == BF else U                                    # (bfloat16: O and what its rounding left off)
    eD = (dd.abs() * (eo + rest * o.abs())).sum(-1, keepdim=True) + (dh + 4) * U * (dd.abs() * o.abs()).sum(-1, keepdim=True)
    dS = P * (dP - D)
    mS = P * (dP - D).abs()
    eS = P * ((dh + 4) * U * mP + eD) + (w + 8 * U) * mS + rp * mS
    big = abs(scale)
    dq, edq = dS @ kd * scale, (eS + n * U * mS) @ kd.abs() * big
    nq = Tq * G
    dk, edk = (dS.transpose(-1, -2) @ qd).sum(2) * scale, ((eS + nq * U * mS).transpose(-1, -2) @ qd.abs()).sum(2) * big
    dv, edv = (P.transpose(-1, -2) @ dd).sum(2), ((P * (w + rp + nq * U)).transpose(-1, -2) @ dd.abs()).sum(2)
    fin = lambda t, e, H, T: (back(t, H, T), back(e * 1.02 + R(dt) * (t.abs() + e), H, T))  # noqa: E731
    return out + [fin(dq, edq, Hq, Tq), fin(dk, edk, Hk, Tk), fin(dv, edv, Hk, Tk)]


def attn_check(outs, refs):
    for got, (ref, err), name in zip(outs, refs, ("o", "dq", "dk", "dv")):
        within(got, ref, err * 1.01 + 1e-30, name)


ATT = [  # B, Tq, Tk, Hq, Hk, dh, left, right, sinks, offset, lens
    (1, 1, 1, 1, 1, 32, 0, 0, 0, None, None),
    (2, 5, 5, 2, 1, 64, 0, 0, 0, None, None),
    (1, 33, 33, 4, 4, 128, 7, 0, 2, None, None),
    (2, 130, 130, 4, 2, 96, 31, 9, 0, None, (130, 77)),
    (1, 200, 200, 3, 3, 32, 1000, 0, 0, None, None),
    (1, 300, 300, 2, 2, 64, 20, 0, 70, None, None),
    (3, 257, 257, 6, 2, 128, 64, 64, 5, None, (257, 0, 1)),
    (1, 1500, 1500, 2, 1, 64, 100, 0, 33, None, None),
    (2, 1030, 1030, 4, 2, 32, 63, 3, 128, None, (1030, 600)),
    (1, 17, 400, 2, 2, 64, 64, 0, 4, None, None),
    (1, 100, 40, 2, 1, 32, 10, 2, 3, 0, None),
    (2, 64, 300, 5, 1, 128, 50, 10, 1, 200, (290, 230)),
    (1, 129, 129, 1, 1, 96, 0, 40, 0, None, None),
    (1, 40, 40, 40, 1, 32, 12, 0, 1, None, None),
    (1, 700, 60, 2, 2, 32, 5, 0, 10, 0, None),          # late rows see first tokens alone
    (1, 70, 50, 2, 2, 64, 5, 0, 0, 30, None),           # late rows see nothing
]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hk,dh,left,right,sinks,offset,lens", ATT)
def test_attention_forward_and_gradients(dt, B, Tq, Tk, Hq, Hk, dh, left, right, sinks, offset, lens):
    q, k, v = rnd(1, B, Tq, Hq, dh, dt=dt, grad=True), rnd(2, B, Tk, Hk, dh, dt=dt, grad=True), rnd(3, B, Tk, Hk, dh, dt=dt, grad=True)
    do = rnd(4, B, Tq, Hq, dh, dt=dt)
    ln = None if lens is None else torch.tensor(lens, device=DEV, dtype=torch.int32)
    o = A().window_attention(q, k, v, left, right, sinks, lengths=ln, offset=offset)
    with torch.no_grad():
        assert torch.equal(o, A().window_attention(q, k, v, left, right, sinks, lengths=ln, offset=offset))
    g = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(g, torch.autograd.grad(o, (q, k, v), do)))
    see = seen(Tq, Tk, left, right, sinks, Tk - Tq if offset is None else offset, ln, B)
    attn_check((o,) + g, attn_ref(q, k, v, see, dh ** -0.5, dt, do))
    dead = ~see.any(-1)
    assert not o[dead].any() and not g[0][dead].any()


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_padding_is_never_read(dt):
    B, T, H, dh = 3, 150, 2, 64
    ln = torch.tensor([150, 37, 0], device=DEV, dtype=torch.int32)
    dead = (torch.arange(T, device=DEV)[None] >= ln[:, None])[..., None, None]
    q, k, v, do = (rnd(s, B, T, H, dh, dt=dt) for s in (1, 2, 3, 4))

    def run(*ts):
        q, k, v = (t.clone().requires_grad_() for t in ts[:3])
        o = A().window_attention(q, k, v, 40, 10, 3, lengths=ln)
        return (o,) + torch.autograd.grad(o, (q, k, v), ts[3])

    clean = run(q, k, v, do)
    for bad in (math.nan, math.inf, torch.finfo(dt).min):
        for a, b in zip(clean, run(*(torch.where(dead, bad, t).to(dt) for t in (q, k, v, do)))):
            assert torch.equal(a, b)
            assert not torch.where(dead, b, 0).any()


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_large_and_equal_scores(dt):
    """Scores of +-1e4 (one key takes all) and rows of equal scores."""
    B, T, H, dh = 1, 90, 2, 32
    q, k, v = rnd(1, B, T, H, dh, dt=dt, std=60.0), rnd(2, B, T, H, dh, dt=dt, std=60.0), rnd(3, B, T, H, dh, dt=dt)
    see = seen(T, T, 40, 0, 2, 0, None, B)
    o = A().window_attention(q, k, v, 40, 0, 2)
    attn_check((o,), attn_ref(q, k, v, see, dh ** -0.5, dt))
    q = torch.zeros_like(q)
    attn_check((A().window_attention(q, k, v, 40, 0, 2),), attn_ref(q, k, v, see, dh ** -0.5, dt))


@pytest.mark.parametrize("dt", [F32, BF])
def test_attention_strided_views(dt):
    B, T, H, dh = 2, 75, 2, 32
    qkv = rnd(1, B, T, 3 * H * dh, dt=dt, grad=True)
    q, k, v = qkv.view(B, T, 3, H, dh).unbind(2)
    do = rnd(2, B, H, T, dh, dt=dt).transpose(1, 2)
    o = A().window_attention(q, k, v, 20, 0, 1)
    g, = torch.autograd.grad(o, qkv, do)
    see = seen(T, T, 20, 0, 1, 0, None, B)
    ref = attn_ref(q, k, v, see, dh ** -0.5, dt, do)
    attn_check((o,) + g.view(B, T, 3, H, dh).unbind(2), ref)
    flat = rnd(1, B * T * 3 * H * dh + 1, dt=dt)[1:]                          # rows off 16 bytes: copied
    q, k, v = flat.view(B, T, 3, H, dh).unbind(2)
    attn_check((A().window_attention(q, k, v, 20, 0, 1),), attn_ref(q, k, v, see, dh ** -0.5, dt))
    q, k, v = (rnd(s, B, H, dh, T, dt=dt).permute(0, 3, 1, 2) for s in (4, 5, 6))    # innermost axis strided: copied
    with pytest.raises(A().DttError):                                         # (the running maximum is taken before the scale)
        A().window_attention(q, k, v, 20, 0, 1, scale=-0.3)
    attn_check((A().window_attention(q, k, v, 20, 0, 1, scale=0.3),), attn_ref(q, k, v, see, 0.3, dt))
    k1, v1 = (rnd(s, 1, T, 1, dh, dt=dt).expand(B, T, H, dh) for s in (7, 8))        # broadcast keys
    attn_check((A().window_attention(q, k1, v1, 20, 0, 1),), attn_ref(q, k1, v1, see, dh ** -0.5, dt))


def test_attention_gradient_against_differences():
    """Central differences of the float64 formula: truncation below 1e-7, kernel error below 1e-5 of the norms."""
    q, k, v = (rnd(s, 1, 50, 2, 32, grad=True) for s in (1, 2, 3))
    do = rnd(4, 1, 50, 2, 32)
    g = torch.autograd.grad(A().window_attention(q, k, v, 9, 2, 3), (q, k, v), do)
    see = seen(50, 50, 9, 2, 3, 0, None, 1)
    base = [t.detach().double() for t in (q, k, v)]
    for i in range(3):
        d = rnd(10 + i, *base[i].shape).double()
        up, dn = ([b + s * 1e-4 * d if m == i else b for m, b in enumerate(base)] for s in (1, -1))
        f = lambda a: float((attn_ref(*a, see, 32 ** -0.5, F32)[0][0] * do.double()).sum())  # noqa: E731
        num = (f(up) - f(dn)) / 2e-4
        assert abs(num - float((g[i].double() * d).sum())) <= 1e-5 * float(g[i].double().norm() * d.norm()) + 1e-6


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("T,left,dh", [(1, 5, 64), (1, 0, 128), (300, 0, 32), (90, 0, 96), (2000, 0, 128)])
def test_attention_rows_of_one_key_have_no_gradient_through_their_weights(dt, T, left, dh):
    """A softmax over one key is 1 whatever its score is: dq = dk = 0 exactly (o and dv, in float32, to the rounding of a
    weight: an exponential of a score less its own log, 4 U and the 2 U |score| of the products, |score| below 32)."""
    q, k, v = (rnd(s, 2, T, 2, dh, dt=dt, grad=True) for s in (1, 2, 3))
    do = rnd(4, 2, T, 2, dh, dt=dt)
    o = A().window_attention(q, k, v, left)
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    assert not dq.any() and not dk.any()
    for got, want in ((o, v.detach().double()), (dv, do.double())):
        within(got, want, (70 * U + R(dt)) * want.abs())


def test_attention_gradients_of_broadcast_keys():
    q, do = rnd(1, 2, 70, 4, 32, grad=True), rnd(4, 2, 70, 4, 32)
    k, v = rnd(2, 1, 70, 1, 32, grad=True), rnd(3, 1, 70, 1, 32, grad=True)
    ke, ve = k.expand(2, 70, 4, 32), v.expand(2, 70, 4, 32)
    g = torch.autograd.grad(A().window_attention(q, ke, ve, 9, 0, 1), (q, k, v), do)
    ref = attn_ref(q, ke, ve, seen(70, 70, 9, 0, 1, 0, None, 2), 32 ** -0.5, F32, do)
    within(g[0], *[t * 1.0 for t in (ref[1][0], ref[1][1] * 1.01 + 1e-30)])
    for got, (r, e) in zip(g[1:], ref[2:]):
        # (autograd adds the 2 x 4 copies in float32: 8 U of their magnitudes)
        within(got, r.sum((0, 2), keepdim=True), (e * 1.01 + 8 * U * r.abs()).sum((0, 2), keepdim=True) + 1e-30)


def test_attention_empty():
    q = torch.zeros(2, 0, 2, 32, device=DEV)
    k = rnd(1, 2, 7, 2, 32)
    assert A().window_attention(q, k, k, 3).shape == (2, 0, 2, 32)
    assert not A().window_attention(rnd(1, 2, 3, 2, 32), k[:, :0], k[:, :0], 3, offset=0).any()


# --------------------------------------------------------------------------- #
# one frame at a time
# --------------------------------------------------------------------------- #
STEP = [(1, 1, 1, 32, 1, 0), (2, 2, 1, 64, 5, 2), (3, 6, 2, 128, 130, 4), (2, 40, 1, 32, 33, 0), (1, 8, 8, 96, 700, 16),
        (2, 35, 1, 64, 1500, 3), (5, 4, 4, 128, 1024, 0), (1, 2, 2, 64, 3000, 1),
        (2, 9, 3, 128, 61, 2), (1, 4, 2, 32, 70, 0), (2, 8, 2, 96, 90, 1), (1, 5, 1, 64, 200, 0)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("B,Hq,Hk,dh,window,sinks", STEP)
def test_step_matches_the_window(dt, B, Hq, Hk, dh, window, sinks):
    """Caches filled from a prefix, then steps, against the whole sequence's last rows; unused slots hold NaN."""
    M = sinks + window
    for n0 in {0, 1, max(0, M - 1), M, M + 3, 2 * M + window // 2 + 1}:
        T = n0 + 3
        q, k, v = rnd(1, B, T, Hq, dh, dt=dt), rnd(2, B, T, Hk, dh, dt=dt), rnd(3, B, T, Hk, dh, dt=dt)
        kc, vc = (torch.full((B, M, Hk, dh), math.nan, dtype=dt, device=DEV) for _ in range(2))
        A().window_cache_fill(k[:, :n0], v[:, :n0], kc, vc, sinks)
        see = seen(3, T, window - 1, 0, sinks, n0, None, B)
        (ref, err), = attn_ref(q[:, n0:], k, v, see, dh ** -0.5, dt)
        pos = torch.full((B,), n0, dtype=torch.int64, device=DEV)
        for i in range(3):
            o = A().window_attention_step(q[:, n0 + i], k[:, n0 + i], v[:, n0 + i], kc, vc, pos, sinks)
            within(o, ref[:, i], err[:, i] * 1.01 + 1e-30, f"{n0} + {i}")
            pos += 1
        kf, vf = (torch.full((B, M, Hk, dh), math.nan, dtype=dt, device=DEV) for _ in range(2))
        A().window_cache_fill(k, v, kf, vf, sinks)
        assert torch.equal(kf.nan_to_num(7.0), kc.nan_to_num(7.0)) and torch.equal(vf.nan_to_num(7.0), vc.nan_to_num(7.0))


@pytest.mark.parametrize("dt", [F32, BF])
def test_step_mixed_ages_idle_items_and_cache_views(dt):
    B, Hq, Hk, dh, window, sinks = 6, 4, 2, 64, 300, 3
    M = sinks + window
    pos = torch.tensor([0, -1, 2, M - 1, M + 5, 10 ** 12 + 17], dtype=torch.int64, device=DEV)
    both = rnd(1, B, M, 2, Hk, dh, dt=dt)                                     # keys and values in one buffer
    kc, vc = both[:, :, 0], both[:, :, 1]
    before = both.clone()
    q, k, v = rnd(2, B, Hq, dh, dt=dt), rnd(3, B, Hk, dh, dt=dt), rnd(4, B, Hk, dh, dt=dt)
    o = A().window_attention_step(q, k, v, kc, vc, pos, sinks)
    want = before.clone()
    for b, p in enumerate(pos.tolist()):
        if p >= 0:
            s = p if p < sinks else sinks + (p - sinks) % window
            want[b, s, 0], want[b, s, 1] = k[b], v[b]
    assert torch.equal(both, want)
    n = (pos + 1).clamp(0, M)
    see = (torch.arange(M, device=DEV)[None] < n[:, None])[:, None]
    (ref, err), = attn_ref(q[:, None], want[:, :, 0], want[:, :, 1], see, dh ** -0.5, dt)
    within(o, ref[:, 0], err[:, 0] * 1.01 + 1e-30)
    assert not o[1].any()


@pytest.mark.parametrize("dt", [F32, BF])
def test_cache_fill_lengths(dt):
    lens = torch.tensor([0, 1, 9, 40], device=DEV)
    k, v = rnd(1, 4, 40, 2, 32, dt=dt), rnd(2, 4, 40, 2, 32, dt=dt)
    kc, vc = rnd(3, 4, 10, 2, 32, dt=dt), rnd(4, 4, 10, 2, 32, dt=dt)
    wk, wv = kc.clone(), vc.clone()
    for b, n in enumerate(lens.tolist()):
        for p in range(n):
            s = p if p < 3 else 3 + (p - 3) % 7
            wk[b, s], wv[b, s] = k[b, p], v[b, p]
    A().window_cache_fill(k, v, kc, vc, 3, lengths=lens)
    assert torch.equal(kc, wk) and torch.equal(vc, wv)


# --------------------------------------------------------------------------- #
# rotary positions
# --------------------------------------------------------------------------- #
def rot_ref(x, pos, freq, inter, amp, sign=1.0):
    """Values and bounds: the fraction of a turn is rounded to float32 (2^-25 turns = 3.2 U rad), sine and cosine to 2 U, times
    the amplitude, two products and a sum: 12 U of (|u| + |v|) amp, plus the float64 angle's own 2^-50 of its size."""
    x = x.detach().double()
    h = freq.numel()
    ang = (pos.double() if pos.dim() == 2 else pos.double()[None])[..., None] * freq
    c, s = torch.cos(ang)[:, :, None] * amp, torch.sin(ang)[:, :, None] * amp * sign
    u, v = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if inter else (x[..., :h], x[..., h:2 * h])
    a, b = u * c - v * s, u * s + v * c
    e = (12 * U + ang.abs()[:, :, None] * 2.0 ** -50) * (u.abs() + v.abs()) * abs(amp)
    val, err = x.clone(), torch.zeros_like(x)
    for t, p, r in ((val, a, b), (err, e, e)):
        if inter:
            t[..., 0:2 * h:2], t[..., 1:2 * h:2] = p, r
        else:
            t[..., :h], t[..., h:2 * h] = p, r
    return val, err


ROT = [(1, 1, 1, 1, 32, 32, 0), (2, 5, 4, 2, 64, 64, 100), (3, 7, 3, 3, 96, 48, 10 ** 7), (2, 600, 8, 2, 128, 128, 0),
       (2, 9, 2, 1, 32, 24, 5), (64, 1, 16, 4, 128, 96, 9999), (1, 11, 2, 2, 20, 6, 3), (2, 3, 5, 1, 17, 10, 2 ** 31)]


@pytest.mark.parametrize("dt", [F32, BF])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,T,Hq,Hk,dh,r,start", ROT)
def test_rotary_forward_and_gradients(dt, inter, B, T, Hq, Hk, dh, r, start):
    q, k = rnd(1, B, T, Hq, dh, dt=dt, grad=True), rnd(2, B, T, Hk, dh, dt=dt, grad=True)
    dq, dk = rnd(3, B, T, Hq, dh, dt=dt), rnd(4, B, T, Hk, dh, dt=dt)
    freq = A().rotary_frequencies(r, device=DEV)
    pos = start + torch.arange(T, device=DEV)[None] + 3 * torch.arange(B, device=DEV)[:, None]
    for p in (pos, pos[0].contiguous(), pos[0].to(torch.int32) if start < 2 ** 30 else pos.t().contiguous().t()):
        qo, ko = A().rotary(q, k, p, freq, interleaved=inter, amplitude=1.25)
        g = torch.autograd.grad((qo, ko), (q, k), (dq, dk))
        for got, src, sign in ((qo, q, 1), (ko, k, 1), (g[0], dq, -1), (g[1], dk, -1)):
            ref, err = rot_ref(src, p, freq, inter, 1.25, sign)
            within(got, ref, err * 1.01 + R(dt) * (ref.abs() + err))
        assert torch.equal(qo[..., r:], q[..., r:])


@pytest.mark.parametrize("dt", [F32, BF])
def test_rotary_views_single_tensor_and_partial_gradients(dt):
    freq = A().rotary_frequencies(32, device=DEV)
    pos = torch.arange(40, device=DEV)
    qkv = rnd(1, 2, 40, 3, 2, 32, dt=dt, grad=True)
    q, k, _ = qkv.unbind(2)
    for inter in (False, True):
        qo, ko = A().rotary(q, k, pos, freq, inter)
        for got, src in ((qo, q), (ko, k)):
            ref, err = rot_ref(src, pos, freq, inter, 1.0)
            within(got, ref, err * 1.01 + R(dt) * (ref.abs() + err))
        g, = torch.autograd.grad(ko.sum(), qkv)                              # q's gradient missing, k's expanded
        ref, err = rot_ref(torch.ones_like(k), pos, freq, inter, 1.0, -1.0)
        within(g[:, :, 1], ref, err * 1.01 + R(dt) * (ref.abs() + err))
        assert not g[:, :, 0].any() and not g[:, :, 2].any()
        alone = A().rotary(q, None, pos, freq, inter)
        assert torch.equal(alone, qo)
        odd = rnd(2, 2 * 40 * 2 * 33 + 1, dt=dt)[1:].view(2, 40, 2, 33)       # rows on odd elements
        ref, err = rot_ref(odd, pos, freq, inter, 1.0)
        within(A().rotary(odd, None, pos, freq, inter), ref, err * 1.01 + R(dt) * (ref.abs() + err))
        neg = pos - 20
        ref, err = rot_ref(q, neg, freq, inter, 1.0)
        within(A().rotary(q, None, neg, freq, inter), ref, err * 1.01 + R(dt) * (ref.abs() + err))


def test_rotary_frequencies():
    import dtt_amd
    f = dtt_amd.rotary_frequencies(8, base=100.0)
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 100 ** -0.5, 100 ** -0.75], dtype=F64), rtol=1e-14)
    assert torch.equal(dtt_amd.rotary_frequencies(8, base=100.0, stretch=4.0), f / 4)
    trained = 200.0
    turns = trained * f / (2 * math.pi)                                       # 31.8, 10.07, 3.18, 1.007
    g = dtt_amd.rotary_frequencies(8, base=100.0, stretch=4.0, trained=trained, blend=(2.0, 12.0))
    keep = ((turns - 2) / 10).clamp(0, 1)
    assert torch.allclose(g, f * (keep + (1 - keep) / 4), rtol=1e-14) and g[0] == f[0] and g[3] == f[3] / 4


# --------------------------------------------------------------------------- #
# together, as they are used
# --------------------------------------------------------------------------- #
class Block:
    """q, k, v from one projection -> rotary -> windowed attention -> recurrence gated by a second projection."""

    def __init__(self, dt, H=4, Hk=2, dh=32, seed=0, grad=False):
        self.H, self.Hk, self.dh, self.C = H, Hk, dh, H * dh
        self.w = rnd(seed, self.C, (H + 2 * Hk) * dh, dt=dt, std=self.C ** -0.5, grad=grad)
        self.wg = rnd(seed + 1, self.C, 2 * self.C, dt=dt, std=self.C ** -0.5, grad=grad)
        self.freq = A().rotary_frequencies(dh, device=DEV)

    def split(self, x):
        h = (x @ self.w).unflatten(-1, (self.H + 2 * self.Hk, self.dh))
        return h[..., :self.H, :], h[..., self.H:self.H + self.Hk, :], h[..., self.H + self.Hk:, :]

    def full(self, x, left, sinks, lengths=None):
        q, k, v = self.split(x)
        q, k = A().rotary(q, k, torch.arange(x.shape[1], device=DEV), self.freq)
        o = A().window_attention(q, k, v, left, 0, sinks, lengths=lengths).flatten(2)
        z, f = (o @ self.wg).chunk(2, -1)
        return A().gated_recurrence(z, f, lengths=lengths)

    def frame(self, x, kc, vc, pos, sinks, state):
        q, k, v = self.split(x)
        q, k = A().rotary(q[:, None], k[:, None], pos[:, None], self.freq)
        o = A().window_attention_step(q[:, 0], k[:, 0], v, kc, vc, pos, sinks).flatten(1)
        z, f = (o @ self.wg).chunk(2, -1)
        return A().gated_recurrence_step(z, f, state)


def test_together_frames_follow_the_sequence():
    """fp32: attention outputs of both paths within their bounds of one another: 1e-5 of the largest value leaves a factor of
    ten over (dh + window) U through two projections."""
    b = Block(F32)
    B, T, window, sinks = 3, 60, 17, 2
    x = rnd(9, B, T, b.C)
    with torch.no_grad():
        y, last = b.full(x, window - 1, sinks)
        kc, vc = (torch.full((B, sinks + window, b.Hk, b.dh), math.nan, device=DEV) for _ in range(2))
        state, pos = torch.zeros(B, b.C, device=DEV), torch.zeros(B, dtype=torch.int64, device=DEV)
        for t in range(T):
            yt = b.frame(x[:, t], kc, vc, pos, sinks, state)
            assert float((yt - y[:, t]).abs().max()) <= 1e-5 * float(y.abs().max())
            pos += 1
        assert float((state - last).abs().max()) <= 1e-5 * float(last.abs().max())


def test_together_training_gradients():
    """The chain's gradients (fp32) against autograd through the same chain of plain float64 operations, 2-norms to 2e-5:
    each stage's bound is below 1e-6 of its norms here."""
    b = Block(F32, grad=True)
    B, T, left, sinks = 2, 70, 11, 3
    lens = torch.tensor([70, 41], device=DEV, dtype=torch.int32)
    x = rnd(9, B, T, b.C, grad=True)
    dy = rnd(10, B, T, b.C)
    y, _ = b.full(x, left, sinks, lens)
    got = torch.autograd.grad(y, (x, b.w, b.wg), dy)

    xd, wd, gd = (t.detach().double().requires_grad_() for t in (x, b.w, b.wg))
    h = (xd @ wd).unflatten(-1, (b.H + 2 * b.Hk, b.dh))
    q, k, v = h[..., :b.H, :], h[..., b.H:b.H + b.Hk, :], h[..., b.H + b.Hk:, :]
    ang = torch.arange(T, device=DEV).double()[:, None, None] * b.freq
    turn = lambda t: torch.cat([t[..., :16] * ang.cos() - t[..., 16:] * ang.sin(), t[..., :16] * ang.sin() + t[..., 16:] * ang.cos()], -1)  # noqa: E731
    q, k = turn(q).transpose(1, 2), turn(k).repeat_interleave(2, 2).transpose(1, 2)
    v = v.repeat_interleave(2, 2).transpose(1, 2)
    see = seen(T, T, left, 0, sinks, 0, lens, B)[:, None]
    s = (q @ k.transpose(-1, -2)) * b.dh ** -0.5
    P = torch.softmax(torch.where(see, s, -1e300), -1) * see
    o = (P @ v).transpose(1, 2).flatten(2)
    z, f = (o @ gd).chunk(2, -1)
    st, ys = torch.zeros(B, b.C, dtype=F64, device=DEV), []
    for t in range(T):
        a = torch.sigmoid(f[:, t])
        st = a * st + (1 - a) * z[:, t]
        ys.append(torch.where((t < lens)[:, None], st, 0.0))
    want = torch.autograd.grad(torch.stack(ys, 1), (xd, wd, gd), dy.double())
    for a, c in zip(got, want):
        assert float((a.double() - c).norm()) <= 2e-5 * float(c.norm())


def test_captured_frames_replay():
    """One captured frame replayed as the stream goes on, against eager frames: equal bits at every replay, with eager work
    and synchronisations between."""
    b = Block(BF)
    B, window, sinks = 4, 600, 4                                              # (two launches: splits are joined)
    kc, vc = (torch.zeros(B, sinks + window, b.Hk, b.dh, dtype=BF, device=DEV) for _ in range(2))
    state, pos = torch.zeros(B, b.C, device=DEV), torch.zeros(B, dtype=torch.int64, device=DEV)
    x = rnd(5, 12, B, b.C, dt=BF)
    xin = x[0].clone()
    with torch.no_grad():
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            b.frame(xin, kc, vc, pos, sinks, state)
        torch.cuda.current_stream().wait_stream(s)
        for t in (kc, vc, state):
            t.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = b.frame(xin, kc, vc, pos, sinks, state)
        ek, ev, es = kc.clone().zero_(), vc.clone().zero_(), torch.zeros_like(state)
        for t in (kc, vc, state):
            t.zero_()
        for t in range(12):
            xin.copy_(x[t])
            pos.fill_(t * 150)
            graph.replay()
            want = b.frame(x[t], ek, ev, pos, sinks, es)
            if t % 3 == 0:
                torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(kc, ek) and torch.equal(state, es)


def test_captured_training_step_replays():
    """Forward and backward of the three in one captured graph (workspaces and saved states from its pool), replayed on new
    inputs, against the eager result: equal bits."""
    T, C, H = 700, 64, 2
    q0 = rnd(1, 1, T, H, 32, dt=BF)
    freq, pos = A().rotary_frequencies(32, device=DEV), torch.arange(T, device=DEV)
    dy = rnd(2, 1, T, C, dt=BF)

    def step(x):
        x = x.detach().requires_grad_()
        q, k = A().rotary(x, x, pos, freq)
        o = A().window_attention(q, k, x, 64, 0, 3).flatten(2)
        y, _ = A().gated_recurrence(o, o)
        return (y,) + torch.autograd.grad(y, x, dy)

    xin = q0.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(xin)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(xin)
    for t in range(4):
        x = rnd(20 + t, 1, T, H, 32, dt=BF)
        xin.copy_(x)
        graph.replay()
        got = [o.clone() for o in outs]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step(x)))


def test_side_streams():
    """Calls on two streams at once, each with its own buffers, agree with the default stream's results."""
    args = [[rnd(10 * i + s, 2, 700, 2, 64, dt=BF) for s in (1, 2, 3)] for i in range(2)]
    want = [A().window_attention(*a, 100, 0, 4) for a in args]
    wr = [A().gated_recurrence(a[0].flatten(2), a[1].flatten(2))[0] for a in args]
    torch.cuda.synchronize()
    streams, got, gr = [torch.cuda.Stream() for _ in range(2)], [], []
    for st, a in zip(streams, args):
        with torch.cuda.stream(st):
            got.append(A().window_attention(*a, 100, 0, 4))
            gr.append(A().gated_recurrence(a[0].flatten(2), a[1].flatten(2))[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want + wr, got + gr))


def test_beyond_32_bit_offsets():
    """Tensors of more than 2^31 elements (4.6 GB each): the far end agrees with the same call on a slice of it.  The state
    halves with every step (f = 0), so 64 steps ahead of the slice's last 64 leave 2^-64 of it; bfloat16 rounds both sides:
    one step, 2 R, of the value, where they straddle a border."""
    L, D = 2_200_000, 1024
    x = torch.empty(1, L, D, dtype=BF, device=DEV)
    x.view(-1, 1 << 10)[:] = rnd(1, 1 << 10, dt=BF)
    x[0, -128:] = rnd(2, 128, D, dt=BF)
    f = torch.zeros(1, 1, D, dtype=BF, device=DEV).expand(1, L, D)
    y, _ = A().gated_recurrence(x, f)
    want, _ = A().gated_recurrence(x[:, -128:], f[:, -128:])
    a, b = y[:, -64:].double(), want[:, -64:].double()
    assert float(((a - b).abs() - 2 * R(BF) * b.abs()).max()) <= 2.0 ** -60
    q = x.view(1, L // 2, 16, 128)
    k = q[:, :, :1]
    o = A().window_attention(q, k, k, 20, 0)
    # (against the formula on the slice: tiles cut the two calls' keys at different places, so bits may differ)
    attn_check((o[:, -64:],), attn_ref(q[:, -64:], k[:, -128:], k[:, -128:], seen(64, 128, 20, 0, 0, 64, None, 1), 128 ** -0.5, BF))
    del y, o, want
    kc, vc = x.view(2, L // 2, 8, 128), torch.zeros(2, L // 2, 8, 128, dtype=BF, device=DEV)
    vc[1, L // 2 - 5] = 3.0                                                   # one slot of 1.1 million, equal weights: 3 / M
    out = A().window_attention_step(torch.zeros(2, 8, 128, dtype=BF, device=DEV), kc[:, 0].clone(), vc[:, 0].clone(), kc, vc,
                                    torch.tensor([L, L], device=DEV), 1)
    assert not out[0].any()
    assert float((out[1].double() * (L // 2) - 3.0).abs().max()) <= 3.0 * 2 * R(BF)


@pytest.mark.parametrize("how", ["checkpoint", "offload"])
def test_hooks_on_saved_tensors(how):
    """Recomputed (checkpoint) and moved (offload) saved tensors give the gradients of kept ones, bit by bit."""
    from torch.utils.checkpoint import checkpoint
    w = rnd(1, 64, 3 * 64, std=0.2, grad=True)
    x = rnd(2, 2, 150, 64, grad=True)
    freq, pos = A().rotary_frequencies(32, device=DEV), torch.arange(150, device=DEV)
    lens = torch.tensor([150, 90], device=DEV, dtype=torch.int32)

    def block(x):
        q, k, v = (t.unflatten(-1, (2, 32)) for t in (x @ w).chunk(3, -1))
        q, k = A().rotary(q, k, pos, freq)
        o = A().window_attention(q, k, v, 20, 0, 2, lengths=lens).flatten(2)
        return A().gated_recurrence(o, o * 2, lengths=lens)[0]

    want = torch.autograd.grad(block(x).square().sum(), (x, w))
    if how == "checkpoint":
        got = torch.autograd.grad(checkpoint(block, x, use_reentrant=False).square().sum(), (x, w))
    else:
        with torch.autograd.graph.save_on_cpu():
            y = block(x).square().sum()
        junk = [torch.full((2, 150, 192), math.nan, device=DEV) for _ in range(20)]      # (what a stale address would read)
        got = torch.autograd.grad(y, (x, w))
        del junk
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_second_derivatives_are_refused():
    """A gradient taken with create_graph is right; differentiating it again raises instead of giving zeros."""
    q, x, f = rnd(1, 1, 20, 2, 32, grad=True), rnd(2, 1, 20, 8, grad=True), rnd(3, 1, 20, 8, grad=True)
    freq, pos = A().rotary_frequencies(32, device=DEV), torch.arange(20, device=DEV)
    for fn, leaf in ((lambda: A().window_attention(q, q, q, 5), q), (lambda: A().gated_recurrence(x, f)[0], x),
                     (lambda: A().rotary(q, q, pos, freq)[0], q)):
        g, = torch.autograd.grad(fn().square().sum(), leaf, create_graph=True)
        assert torch.equal(g, torch.autograd.grad(fn().square().sum(), leaf)[0])
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), leaf)


# --------------------------------------------------------------------------- #
# refusals
# --------------------------------------------------------------------------- #
def test_refusals():
    from dtt_amd import DttError
    a = A()
    x = torch.zeros(2, 4, 8, device=DEV)
    q, k = torch.zeros(2, 4, 4, 32, device=DEV), torch.zeros(2, 4, 2, 32, device=DEV)
    kc = torch.zeros(2, 6, 2, 32, device=DEV)
    pos = torch.zeros(2, dtype=torch.int64, device=DEV)
    freq, tp = a.rotary_frequencies(32, device=DEV), torch.arange(4, device=DEV)
    bad = [
        lambda: a.gated_recurrence(x, x[:, :3]), lambda: a.gated_recurrence(x, x.bfloat16()),
        lambda: a.gated_recurrence(x.half(), x.half()), lambda: a.gated_recurrence(x[0], x[0]),
        lambda: a.gated_recurrence(x, x, torch.zeros(2, 7, device=DEV)),
        lambda: a.gated_recurrence(x, x, torch.zeros(2, 8, device=DEV, dtype=BF)),
        lambda: a.gated_recurrence(x, x, lengths=torch.zeros(3, dtype=torch.int32, device=DEV)),
        lambda: a.gated_recurrence(x, x, lengths=torch.zeros(2, dtype=torch.int32)),
        lambda: a.gated_recurrence(x.cpu(), x.cpu()), lambda: a.gated_recurrence(x, x.cpu()),
        lambda: a.gated_recurrence_step(x[:, 0], x[:, 0], x[:, 0]),
        lambda: a.gated_recurrence_step(x[:, 0], x[:, 0], torch.zeros(2, 8, device=DEV, dtype=BF)),
        lambda: a.gated_recurrence_step(x[:, 0].requires_grad_(), x[:, 0], torch.zeros(2, 8, device=DEV)),
        lambda: a.window_attention(q, k, k[:, :3], 3), lambda: a.window_attention(q, k.bfloat16(), k, 3),
        lambda: a.window_attention(q[:, :, :3], k, k, 3), lambda: a.window_attention(q, k, k, -1),
        lambda: a.window_attention(q, k, k, 3, -1), lambda: a.window_attention(q, k, k, 3, 0, 129),
        lambda: a.window_attention(q, k, k, 3, offset=-1), lambda: a.window_attention(q, k[:, :2], k[:, :2], 3),
        lambda: a.window_attention(q[..., :16], k[..., :16], k[..., :16], 3),
        lambda: a.window_attention(q.double(), k.double(), k.double(), 3),
        lambda: a.window_attention(q, k.cpu(), k, 3),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc[:, :5], pos),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc.clone(), pos, 6),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc.clone(), pos.int()),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc.clone(), pos.cpu()),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc.bfloat16(), kc.bfloat16(), pos),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc.transpose(2, 3).contiguous().transpose(2, 3), kc.clone(), pos),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc, pos),
        lambda: a.window_attention_step(q[:, 0], k[:, 0], k[:, 0], kc, kc[:1].clone().expand(2, 6, 2, 32), pos),
        lambda: a.window_attention_step(q[:, 0].clone().requires_grad_(), k[:, 0], k[:, 0], kc, kc.clone(), pos),
        lambda: a.window_cache_fill(k, k, kc, kc.clone(), 6), lambda: a.window_cache_fill(k, k[:, :2], kc, kc.clone()),
        lambda: a.rotary(q, k, tp.float(), freq), lambda: a.rotary(q, k, tp[:3], freq), lambda: a.rotary(q, k, tp, freq.float()),
        lambda: a.rotary(q, k[..., :16], tp, freq), lambda: a.rotary(q, k, tp, torch.ones(17, dtype=F64, device=DEV)),
        lambda: a.rotary(q, k, tp, freq.cpu()), lambda: a.rotary(q, k.bfloat16(), tp, freq),
        lambda: a.rotary_frequencies(7), lambda: a.rotary_frequencies(8, stretch=0.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(DttError):
            f()
            pytest.fail(f"call {i} was not refused")


def test_sizes_beyond_32_bits():
    """Refused before anything is allocated (such a size would be cut to its low 32 bits on its way to C)."""
    n = (1 << 32) + 1
    x, t = torch.zeros(1, 1, 1, device=DEV).expand(n, 1, 1), torch.zeros(1, 1, 1, 32, device=DEV).expand(n, 1, 1, 32)
    freq = A().rotary_frequencies(32, device=DEV)
    for call in (lambda: A().gated_recurrence(x, x),
                 lambda: A().gated_recurrence(x.view(1, n, 1, 1), x.view(1, n, 1, 1)),
                 lambda: A().window_attention(t, t, t, 1),
                 lambda: A().rotary(t, None, torch.zeros(1, dtype=torch.int64, device=DEV), freq),
                 lambda: A().rotary(t[:1], t[:1].expand(1, 1, n, 32), torch.zeros(1, dtype=torch.int64, device=DEV), freq)):
        with pytest.raises(A().DttError):
            call()


@pytest.mark.parametrize("tq,tk", [(3, 0), (0, 3)])
def test_attention_without_rows_or_keys(tq, tk):
    """No key: rows of zeros whatever q holds; zero gradients both ways."""
    q = torch.full((2, tq, 2, 32), float("nan"), device=DEV, requires_grad=True)
    k, v = (torch.full((2, tk, 1, 32), float("nan"), device=DEV, requires_grad=True) for _ in range(2))
    out = A().window_attention(q, k, v, 4, sinks=1, offset=0)
    assert out.shape == q.shape and bool((out == 0).all())
    out.sum().backward()
    for t in (q, k, v):
        assert t.grad.shape == t.shape and bool((t.grad == 0).all())

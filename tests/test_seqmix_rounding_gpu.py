"""The token mixers' bfloat16 results are the exact ones rounded once, up to what 32-bit sums and weights of 16 bits leave: every
element within half a step of its own binade and a bound far below that, counted in float64 beside the reference.

U = 2^-24.  A score is a sum of dh products in float32, (dh + 8) U of their magnitudes; a weight is an exponential of
a score less the log of the row's sum, both below 16 here: 48 U in all for the roundings of the two, of the exponential and of the
sum, n U for the sum over n keys.  A weight (and dS) enters its product in two bfloat16 pieces, 2^-16 of it."""
import math

import pytest
import torch
from test_seqmix_gpu import A, BF, DEV, F64, rnd, seen

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
PIECES = 2.0 ** -16


def rounded_once(got, ref, err, what):
    """got is a bfloat16 neighbour of a value within err of ref: off by err and half a step of the binade it lies in."""
    top = (ref.abs() + err).clamp(min=2.0 ** -120)
    half = torch.exp2(torch.floor(torch.log2(top)) - 8)
    over = (got.detach().double() - ref).abs() - half - err
    assert got.dtype == BF and torch.isfinite(got).all() and float(over.max()) <= 0.0, (what, float(over.max()))


def bounds(q, k, v, see, scale, do):
    """o, dq, dk, dv [B, T, H, dh] in float64 with the errors their kernels may have ahead of the final rounding.  D is the sum of
    dO O with O in two pieces, or of P dP: what moves O or a weight moves either by as much, its products' sums add (dh + 4) U."""
    B, Tq, Hq, dh = q.shape
    n, Hk = k.shape[1:3]
    G = Hq // Hk
    qd, kd, vd, dd = (t.detach().double().transpose(1, 2) for t in (q, k, v, do))
    qd, dd = qd.reshape(B, Hk, G, Tq, dh), dd.reshape(B, Hk, G, Tq, dh)
    kd, vd, sm = kd[:, :, None], vd[:, :, None], see[:, None, None]
    s = qd @ kd.transpose(-1, -2) * scale
    assert float(s[sm.expand_as(s)].abs().max()) * math.log2(math.e) + math.log2(n) < 16
    P = torch.softmax(torch.where(sm, s, -math.inf), -1).nan_to_num(0.0)
    es = torch.where(sm, (dh + 8) * U * scale * (qd.abs() @ kd.abs().transpose(-1, -2)), 0.0)
    w = 2 * es.amax(-1, keepdim=True) + 48 * U + n * U
    back = lambda t, H, T: t.reshape(B, H, T, dh).transpose(1, 2)  # noqa: E731
    o, eo = P @ vd, (w + PIECES + n * U) * (P @ vd.abs())
    dv, edv = (P.transpose(-1, -2) @ dd).sum(2), ((P * (w + PIECES + Tq * G * U)).transpose(-1, -2) @ dd.abs()).sum(2)
    dP, mP = dd @ vd.transpose(-1, -2), dd.abs() @ vd.abs().transpose(-1, -2)
    D = (dd * o).sum(-1, keepdim=True)
    eD = (dd.abs() * (eo + PIECES * o.abs())).sum(-1, keepdim=True) + 2 * (dh + 4) * U * (P * mP).sum(-1, keepdim=True)
    dS, mS = P * (dP - D), P * (dP - D).abs()
    eS = P * ((dh + 4) * U * mP + eD) + (w + 8 * U + PIECES) * mS
    dq, edq = dS @ kd * scale, (eS + n * U * mS) @ kd.abs() * scale
    dk, edk = (dS.transpose(-1, -2) @ qd).sum(2) * scale, ((eS + Tq * G * U * mS).transpose(-1, -2) @ qd.abs()).sum(2) * scale
    return {"o": (back(o, Hq, Tq), back(eo, Hq, Tq)), "dq": (back(dq, Hq, Tq), back(edq, Hq, Tq)),
            "dk": (back(dk, Hk, n), back(edk, Hk, n)), "dv": (back(dv, Hk, n), back(edv, Hk, n))}


def case(B, T, Hq, Hk, dh, std=0.5):
    """Scores below a standard deviation: their own errors stay far below a weight's rounding to bfloat16."""
    q, k = (rnd(s, B, T, h, dh, dt=BF, std=std, grad=True) for s, h in ((1, Hq), (2, Hk)))
    return q, k, rnd(3, B, T, Hk, dh, dt=BF, grad=True), rnd(4, B, T, Hq, dh, dt=BF)


CASES = [  # B, T, Hq, Hk, left, right, sinks: few row tiles and many
    (2, 200, 2, 1, 20, 0, 0), (2, 200, 4, 2, 150, 4, 3), (64, 140, 4, 4, 20, 12, 0), (32, 180, 8, 4, 33, 0, 4),
]


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("B,T,Hq,Hk,left,right,sinks", CASES)
def test_attention_and_values_gradient_are_rounded_once(dh, B, T, Hq, Hk, left, right, sinks):
    q, k, v, do = case(B, T, Hq, Hk, dh)
    o = A().window_attention(q, k, v, left, right, sinks)
    dv, = torch.autograd.grad(o, v, do)
    want = bounds(q, k, v, seen(T, T, left, right, sinks, 0, None, B), dh ** -0.5, do)
    rounded_once(o, *want["o"], "o")
    rounded_once(dv, *want["dv"], "dv")


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("B,T,Hq,Hk,left,right,sinks", CASES)
def test_attention_score_gradients_are_rounded_once(dh, B, T, Hq, Hk, left, right, sinks):
    q, k, v, do = case(B, T, Hq, Hk, dh, 0.25)
    dq, dk = torch.autograd.grad(A().window_attention(q, k, v, left, right, sinks), (q, k), do)
    want = bounds(q, k, v, seen(T, T, left, right, sinks, 0, None, B), dh ** -0.5, do)
    rounded_once(dq, *want["dq"], "dq")
    rounded_once(dk, *want["dk"], "dk")


@pytest.mark.parametrize("dh", [32, 64, 96, 128])
@pytest.mark.parametrize("B,Hq,Hk,window,sinks", [(40, 8, 2, 60, 2), (3, 4, 4, 900, 0)])
def test_a_frame_is_rounded_once(dh, B, Hq, Hk, window, sinks):
    M = window + sinks
    q, k, v = rnd(1, B, Hq, dh, dt=BF, std=0.5), rnd(2, B, Hk, dh, dt=BF, std=0.5), rnd(3, B, Hk, dh, dt=BF)
    kc, vc = rnd(4, B, M, Hk, dh, dt=BF, std=0.5), rnd(5, B, M, Hk, dh, dt=BF)
    pos = torch.randint(0, 2 * M, (B,), generator=torch.Generator().manual_seed(7)).to(DEV)
    out = A().window_attention_step(q, k, v, kc, vc, pos, sinks)
    see = (torch.arange(M, device=DEV)[None] <= pos[:, None])[:, None]
    ref, err = bounds(q[:, None], kc, vc, see, dh ** -0.5, torch.zeros_like(q)[:, None])["o"]
    rounded_once(out, ref[:, 0], err[:, 0], "frame")


def plain_score_gradients(q, k, v, do, see, scale, dt):
    """dq, dk [B, T, H, dh] of every item's own head (Hq = Hk) by plain operations in `dt`, on the CPU (its products are float32)."""
    q, k, v, do = (t.detach().cpu().to(dt).transpose(1, 2).contiguous() for t in (q, k, v, do))
    s = torch.where(see.cpu(), (q @ k.transpose(-1, -2)) * scale, -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    dw = do @ v.transpose(-1, -2)
    dw = w * (dw - (w * dw).sum(-1, keepdim=True)) * scale
    return tuple(t.transpose(1, 2).double() for t in (dw @ k, dw.transpose(-1, -2).contiguous() @ q))


@pytest.mark.parametrize("B,T,H,dh", [(16, 100, 8, 128), (16, 100, 8, 64), (64, 140, 4, 128), (64, 140, 4, 32)])
def test_float32_rows_of_few_keys_in_a_wide_window(B, T, H, dh):
    """The first rows of a causal sequence see one, two, three keys, whatever the window.  D = sum(P dP) cancels against dP as in
    plain float32; the kernel rounds at most twice as often, by steps of the same size, so that in 2-norm (hundreds of rows) it is
    off by no more than sqrt(2) of plain float32's error: 1.5.  (D = sum(dO O) is off by 1.7 to 2.2 of it.)"""
    q, k, v = (rnd(s, B, T, H, dh, std=std, grad=True) for s, std in ((1, 2.0), (2, 1.0), (3, 1.0)))
    do = rnd(4, B, T, H, dh)
    do[:, 4:] = 0                                                            # (so that dk comes from these rows alone)
    got = torch.autograd.grad(A().window_attention(q, k, v, 200, 0, 2), (q, k), do)
    see = seen(T, T, 200, 0, 2, 0, None, 1)
    exact, plain = (plain_score_gradients(q, k, v, do, see, dh ** -0.5, dt) for dt in (F64, torch.float32))
    for g, p, e, name in zip(got, plain, exact, ("dq", "dk")):
        mine, theirs = float((g.cpu().double() - e)[:, :4].norm()), float((p - e)[:, :4].norm())
        assert mine <= 1.5 * theirs, (name, mine, theirs, mine / theirs)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("start", [0, 20_000_000])
def test_float32_rotary_with_whole_angles(inter, start):
    """In 2-norm over half a million elements no further off than plain float32 with sines and cosines rounded from float64: the
    kernel's own may be an ulp off, a rounding more beside the three of the products and their sum: sqrt(4 / 3), 1.16.  (A
    fraction of a turn rounded to float32 first: 1.3.)"""
    q = rnd(1, 2, 2003, 2, 64)
    freq, pos = A().rotary_frequencies(64, device=DEV), start + torch.arange(2003, device=DEV)
    got = A().rotary(q, None, pos, freq, interleaved=inter)
    ang = (pos.double()[:, None] * freq)[:, None]
    c, s = torch.cos(ang), torch.sin(ang)

    def turned(x, c, s):
        u, v = (x[..., 0::2], x[..., 1::2]) if inter else (x[..., :32], x[..., 32:])
        pair = u * c - v * s, u * s + v * c
        return torch.stack(pair, -1).flatten(-2) if inter else torch.cat(pair, -1)

    exact, plain = turned(q.double(), c, s), turned(q, c.float(), s.float())
    assert float((got - exact).norm()) <= 1.16 * float((plain - exact).norm())


@pytest.mark.parametrize("B,T,H,dh", [(16, 100, 8, 64), (64, 140, 4, 128)])
@pytest.mark.parametrize("left,rows", [(1, 100), (7, 100), (200, 20)])
@pytest.mark.parametrize("spread", [3.0, 8.0])
def test_rows_with_nearly_all_weight_on_one_key(B, T, H, dh, left, rows, spread):
    """Their gradients are small differences: dP - D, where D has to be the sum of P dP with the very weights that dS is formed
    from, and those have to sum to 1 as closely as float32 lets them.  Errors row by row, relative to the row, rounded to bfloat16 at
    the end: 99 of 100 rows no worse than 1.5 times what plain float32 gives for 99 of 100 (the same float32 roundings, at most
    twice as many).  Of the rows whose gradient float32 resolves: it is 1 - P of the one key's dP - D, which carries a few U of dP in any
    float32 arithmetic, so a row counts where 1 - P is at least 2^-12.  (Below 2^-24 plain float32 rounds P to 1 and the gradient
    to 0, off by exactly 1 of it, and any rounding elsewhere, however small, by more.)"""
    q, k, v = (rnd(s, B, T, H, dh, dt=BF, std=std, grad=True) for s, std in ((1, spread), (2, 1.0), (3, 1.0)))
    do = rnd(4, B, T, H, dh, dt=BF)
    got, = torch.autograd.grad(A().window_attention(q, k, v, left), q, do)
    see = seen(T, T, left, 0, 0, 0, None, 1)
    exact, plain = (plain_score_gradients(q, k, v, do, see, dh ** -0.5, dt)[0][:, 1:rows] for dt in (F64, torch.float32))
    s = torch.einsum("bthd,bshd->bths", q.detach().double(), k.detach().double()) * dh ** -0.5
    top = torch.softmax(torch.where(see[:, :, None], s, -math.inf), -1).topk(2, -1).values
    counts = (top[..., 1] >= 2.0 ** -12)[:, 1:rows].cpu()
    assert int(counts.sum()) > 1000

    def worst(t):
        e = (t.to(BF).double() - exact).norm(dim=-1) / exact.norm(dim=-1)
        return float(torch.quantile(e[counts], 0.99))

    assert worst(got.cpu()[:, 1:rows]) <= 1.5 * worst(plain), (worst(got.cpu()[:, 1:rows]), worst(plain))

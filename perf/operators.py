"""Measured cases of the long-recording token mixers: the gated linear recurrence, windowed attention with first tokens
that stay visible (training, whole-sequence and single-token form over a rolling cache), and rotary positions.

`own` false: the operators in their plain form, elementary torch operations in 32 bits (rotary angles in 64).
`own` true: the calls that a user makes of dtt_amd."""
import math
import os
import sys

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_DEV = "cuda"


# --------------------------------------------------------------------------- #
# the cases
# --------------------------------------------------------------------------- #
def listed():
    return [
        # the latent rows of the 6 s audio-visual model: 16 items x 65 bands, 47 frames, 1024 channels, one training pass
        dict(name="recurrence latent train", op="recurrence", type="bf16", train=True, n=1040, l=47, d=1024, reverse=False,
             ragged=False),
        # two recordings of four minutes (frames of 16 ms), one training pass over the whole of them
        dict(name="recurrence long train", op="recurrence", type="bf16", train=True, n=2, l=15001, d=1024, reverse=False,
             ragged=True),
        # the backward direction over one recording of ten minutes, in fp32, inference
        dict(name="recurrence 10 min fp32", op="recurrence", type="fp32", train=False, n=1, l=37501, d=512, reverse=True,
             ragged=False),
        # one frame of 64 live streams
        dict(name="recurrence frame", op="recurrence_step", type="bf16", n=64, d=1024),
        # training on minute-long clips, four query heads to a key head
        dict(name="attention train", op="attention", type="bf16", train=True, b=2, t=4096, hq=16, hk=4, dh=128, left=511,
             right=0, sinks=4, ragged=False),
        # 6 s clips of unequal lengths, window to both sides, fp32 as the token networks train
        dict(name="attention ragged fp32", op="attention", type="fp32", train=True, b=16, t=376, hq=2, hk=2, dh=128,
             left=64, right=64, sinks=0, ragged=True),
        # a recording of four minutes read in before streaming goes on
        dict(name="attention read-in", op="attention", type="bf16", train=False, b=1, t=15001, hq=8, hk=2, dh=64, left=1023,
             right=0, sinks=16, ragged=False),
        # one frame of 64 live streams, a minute of context
        dict(name="attention frame 64", op="attention_step", type="bf16", b=64, window=4000, sinks=16, hq=16, hk=4, dh=128),
        # one frame of one stream, a short window: latency
        dict(name="attention frame 1", op="attention_step", type="fp32", b=1, window=251, sinks=5, hq=2, hk=2, dh=128),
        # queries and keys of minute-long clips, forward and backward
        dict(name="rotary train", op="rotary", type="bf16", train=True, b=4, t=4096, hq=16, hk=4, dh=128, r=128,
             interleaved=False, start=0),
        # adjacent pairs, part of the head, positions far into a stream that has run for days
        dict(name="rotary far fp32", op="rotary", type="fp32", train=False, b=3, t=5001, hq=8, hk=8, dh=64, r=48,
             interleaved=True, start=20_000_000),
        # one frame of 64 live streams
        dict(name="rotary frame", op="rotary", type="bf16", train=False, b=64, t=1, hq=16, hk=4, dh=128, r=128,
             interleaved=False, start=5000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        if c["op"] == "attention" and c["b"] * c["hq"] * c["t"] ** 2 > 1.8e9:
            continue
        w, top = work(c), {"recurrence": 9e8, "recurrence_step": 1e6, "attention": 9e7 if c["type"] == "bf16" else 1.2e7,
                           "attention_step": 5.5e8, "rotary": 1.6e8}[c["op"]]
        if w["bytes"] > top or w["flops"] > (6e10 if c["type"] == "bf16" else 1.2e10):
            continue
        return c


def _draw(rng):
    op = rng.choice(["recurrence", "recurrence_step", "attention", "attention", "attention_step", "rotary"])
    typ = rng.choice(["bf16", "bf16", "fp32"])
    if op == "recurrence":
        d = _log(rng, 32, 1100)
        d = d if rng.random() < 0.25 else max(8, d // 8 * 8)
        return dict(op=op, type=typ, train=rng.random() < 0.6, n=_log(rng, 1, 2000), l=_log(rng, 1, 37501), d=d,
                    reverse=rng.random() < 0.5, ragged=rng.random() < 0.5)
    if op == "recurrence_step":
        return dict(op=op, type=typ, n=_log(rng, 1, 128), d=_log(rng, 32, 1024))
    hk, group, dh = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 1, 2, 4, 5]), rng.choice([32, 64, 96, 128])
    if op == "attention":
        return dict(op=op, type=typ, train=rng.random() < 0.6, b=_log(rng, 1, 16), t=_log(rng, 1, 15001), hq=hk * group, hk=hk,
                    dh=dh, left=_log(rng, 1, 1200) - 1, right=rng.choice([0, 0, _log(rng, 1, 200)]),
                    sinks=rng.choice([0, 1, 4, 16, 33]), ragged=rng.random() < 0.4)
    if op == "attention_step":
        return dict(op=op, type=typ, b=_log(rng, 1, 64), window=_log(rng, 1, 4200), sinks=rng.choice([0, 1, 4, 16]), hq=hk * group,
                    hk=hk, dh=dh)
    return dict(op=op, type=typ, train=rng.random() < 0.5, b=_log(rng, 1, 64), t=_log(rng, 1, 15001), hq=hk * group, hk=hk, dh=dh,
                r=rng.choice([dh, dh // 2, dh // 4 * 3]), interleaved=rng.random() < 0.5, start=_log(rng, 1, 20_000_000))


# --------------------------------------------------------------------------- #
# inputs
# --------------------------------------------------------------------------- #
def prepare(case, seed):
    c, dt = case, _DT[case["type"]]
    g = torch.Generator(device=_DEV).manual_seed(seed)

    def normal(*shape, mean=0.0, std=1.0, grad=False, t=dt):
        x = torch.randn(shape, generator=g, device=_DEV).mul_(std).add_(mean).to(t)
        return x.requires_grad_(grad)

    def lengths(n, t):
        if not c["ragged"]:
            return None
        x = torch.randint(max(1, t // 2), t + 1, (n,), generator=g, device=_DEV, dtype=torch.int32)
        x[0] = t
        return x

    s = {"case": c}
    train = c.get("train", False)
    if c["op"] == "recurrence":
        n, l, d = c["n"], c["l"], c["d"]
        s.update(x=normal(n, l, d, grad=train), f=normal(n, l, d, mean=2.0, std=1.5, grad=train),
                 h0=normal(n, d, t=torch.float32, grad=train), lengths=lengths(n, l))
        if train:
            s.update(dy=normal(n, l, d), dlast=normal(n, d, t=torch.float32))
    elif c["op"] == "recurrence_step":
        n, d = c["n"], c["d"]
        s.update(x=normal(n, d), f=normal(n, d, mean=2.0, std=1.5), state=normal(n, d, t=torch.float32))
    elif c["op"] == "attention":
        b, t, dh = c["b"], c["t"], c["dh"]
        s.update(q=normal(b, t, c["hq"], dh, grad=train), k=normal(b, t, c["hk"], dh, grad=train),
                 v=normal(b, t, c["hk"], dh, grad=train), lengths=lengths(b, t))
        if train:
            s.update(do=normal(b, t, c["hq"], dh))
    elif c["op"] == "attention_step":
        b, m, dh = c["b"], c["sinks"] + c["window"], c["dh"]
        # streams of every age: some have not filled their window yet, some have run round it many times
        pos = torch.randint(0, 4 * m, (b,), generator=g, device=_DEV, dtype=torch.int64)
        pos[b // 2] = m + 7
        s.update(q=normal(b, c["hq"], dh), k=normal(b, c["hk"], dh), v=normal(b, c["hk"], dh),
                 k_cache=normal(b, m, c["hk"], dh), v_cache=normal(b, m, c["hk"], dh), positions=pos)
    else:
        b, t, dh = c["b"], c["t"], c["dh"]
        first = torch.randint(0, c["start"] + 1, (b, 1), generator=g, device=_DEV, dtype=torch.int64)
        i = torch.arange(c["r"] // 2, device=_DEV, dtype=torch.float64)
        s.update(q=normal(b, t, c["hq"], dh, grad=train), k=normal(b, t, c["hk"], dh, grad=train),
                 positions=first + torch.arange(t, device=_DEV), freq=torch.pow(10000.0, -2.0 * i / c["r"]))
        if train:
            s.update(dq=normal(b, t, c["hq"], dh), dk=normal(b, t, c["hk"], dh))
    return s


# --------------------------------------------------------------------------- #
# one pass
# --------------------------------------------------------------------------- #
def run(s):
    c = s["case"]
    if own:
        return _RUN_OWN[c["op"]](_package(), c, s)
    with torch.no_grad():
        return _RUN_PLAIN[c["op"]](c, s)


def _package():
    p = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "speech-separation_amd")
    if p not in sys.path:
        sys.path.insert(0, p)
    import dtt_amd
    return dtt_amd


def _own_recurrence(A, c, s):
    y, last = A.gated_recurrence(s["x"], s["f"], s["h0"], reverse=c["reverse"], lengths=s["lengths"])
    if not c["train"]:
        return y, last
    return (y, last) + torch.autograd.grad((y, last), (s["x"], s["f"], s["h0"]), (s["dy"], s["dlast"]))


def _own_recurrence_step(A, c, s):
    return A.gated_recurrence_step(s["x"], s["f"], s["state"]), s["state"]


def _own_attention(A, c, s):
    o = A.window_attention(s["q"], s["k"], s["v"], c["left"], c["right"], c["sinks"], lengths=s["lengths"])
    if not c["train"]:
        return o
    return (o,) + torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])


def _own_attention_step(A, c, s):
    o = A.window_attention_step(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], c["sinks"])
    return o, s["k_cache"], s["v_cache"]


def _own_rotary(A, c, s):
    q, k = A.rotary(s["q"], s["k"], s["positions"], s["freq"], interleaved=c["interleaved"])
    if not c["train"]:
        return q, k
    return (q, k) + torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))


_RUN_OWN = dict(recurrence=_own_recurrence, recurrence_step=_own_recurrence_step, attention=_own_attention,
                attention_step=_own_attention_step, rotary=_own_rotary)


# the gated linear recurrence: h_t = a_t h_{t-1} + (1 - a_t) x_t, a = sigmoid(f), by doubling
def _scan(a, b):
    """All h_t = a_t h_{t-1} + b_t from h_{-1} = 0, along dim 1."""
    step = 1
    while step < a.shape[1]:
        b = torch.cat([b[:, :step], b[:, step:] + a[:, step:] * b[:, :-step]], 1)
        a = torch.cat([a[:, :step], a[:, step:] * a[:, :-step]], 1)
        step *= 2
    return b


def _turn(t, on):
    return t.flip(1) if on else t


def _plain_recurrence(c, s):
    x, f, rev = _turn(s["x"], c["reverse"]).float(), _turn(s["f"], c["reverse"]).float(), c["reverse"]
    n, l, d = x.shape
    live = torch.ones(1, l, 1, dtype=torch.bool, device=x.device)
    if s["lengths"] is not None:
        live = _turn((torch.arange(l, device=x.device)[None, :] < s["lengths"][:, None])[:, :, None], rev)
    a = torch.where(live, torch.sigmoid(f), 1.0)               # padding: the state stays
    i = torch.where(live, torch.sigmoid(-f), 0.0)              # 1 - a without its cancellation
    b = torch.where(live, i * x, 0.0)
    h = _scan(a, torch.cat([b[:, :1] + a[:, :1] * s["h0"][:, None], b[:, 1:]], 1))
    out = (_turn(torch.where(live, h, 0.0), rev).to(s["x"].dtype), h[:, -1])
    if not c["train"]:
        return out
    dy = torch.where(live, _turn(s["dy"], rev).float(), 0.0)
    dy = torch.cat([dy[:, :-1], dy[:, -1:] + s["dlast"][:, None]], 1)
    late = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = _scan(late.flip(1), dy.flip(1)).flip(1)                # g_t = dy_t + a_{t+1} g_{t+1}
    before = torch.cat([s["h0"][:, None], h[:, :-1]], 1)
    dx, df = g * i, torch.where(live, g * a * i * (before - x), 0.0)
    return out + (_turn(dx, rev).to(s["x"].dtype), _turn(df, rev).to(s["f"].dtype), a[:, 0] * g[:, 0])


def _plain_recurrence_step(c, s):
    f = s["f"].float()
    s["state"].copy_(torch.sigmoid(f) * s["state"] + torch.sigmoid(-f) * s["x"].float())
    return s["state"].to(s["x"].dtype), s["state"]


# windowed attention: key j is visible to the query at p where j <= p + right and (j >= p - left or j < sinks)
def _plain_attention(c, s):
    b, t, hq, dh = s["q"].shape
    hk = c["hk"]
    q, k, v = (s[n].float().transpose(1, 2) for n in ("q", "k", "v"))                  # [b, heads, t, dh]
    q = q.reshape(b, hk, hq // hk, t, dh)
    k, v = k[:, :, None], v[:, :, None]
    p = torch.arange(t, device=q.device)
    i, j = p[:, None], p[None, :]
    see = ((j <= i + c["right"]) & ((j >= i - c["left"]) | (j < c["sinks"])))[None]
    if s["lengths"] is not None:
        n = s["lengths"][:, None, None]
        see = see & (j[None] < n) & (i[None] < n)
        k, v = (torch.where((p < n)[:, :, None, :, None], x, 0.0) for x in (k, v))
    see = see[:, None, None]
    scale = 1.0 / math.sqrt(dh)
    w = torch.where(see, (q @ k.transpose(-1, -2)) * scale, -math.inf)
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(top > -math.inf, top, 0.0))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, 1.0)
    o = w @ v
    back = lambda x, h, like: x.reshape(b, h, t, dh).transpose(1, 2).to(like.dtype).contiguous()  # noqa: E731
    if not c["train"]:
        return back(o, hq, s["q"])
    do = s["do"].float().transpose(1, 2).reshape(b, hk, hq // hk, t, dh)
    dv = (w.transpose(-1, -2) @ do).sum(2)
    dw = do @ v.transpose(-1, -2)
    dw = w * (dw - (w * dw).sum(-1, keepdim=True)) * scale
    return (back(o, hq, s["q"]), back(dw @ k, hq, s["q"]), back((dw.transpose(-1, -2) @ q).sum(2), hk, s["k"]),
            back(dv, hk, s["v"]))


def _plain_attention_step(c, s):
    b, hq, dh = s["q"].shape
    hk, sinks, window = c["hk"], c["sinks"], c["window"]
    pos, rows = s["positions"], torch.arange(b, device=s["q"].device)
    at = torch.where(pos < sinks, pos, sinks + (pos - sinks) % window)
    s["k_cache"][rows, at] = s["k"]
    s["v_cache"][rows, at] = s["v"]
    k, v = s["k_cache"].float().transpose(1, 2), s["v_cache"].float().transpose(1, 2)  # [b, hk, m, dh]
    q = s["q"].float().reshape(b, hk, hq // hk, dh)
    see = (torch.arange(sinks + window, device=q.device)[None, :] <= pos[:, None])[:, None, None]
    w = torch.where(see, (q @ k.transpose(-1, -2)) / math.sqrt(dh), -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    o = w @ torch.where(see[:, :, 0, :, None], v, 0.0)
    return o.reshape(b, hq, dh).to(s["q"].dtype), s["k_cache"], s["v_cache"]


# rotary positions: the pair (u, v) turned by position x freq
def _turned(x, cos, sin, r, interleaved):
    x32 = x.float()
    head, rest = x32[..., :r], x32[..., r:]
    if interleaved:
        u, v = head[..., 0::2], head[..., 1::2]
        head = torch.stack([u * cos - v * sin, u * sin + v * cos], -1).flatten(-2)
    else:
        u, v = head[..., :r // 2], head[..., r // 2:]
        head = torch.cat([u * cos - v * sin, u * sin + v * cos], -1)
    return torch.cat([head, rest], -1).to(x.dtype)


def _plain_rotary(c, s):
    angle = s["positions"].double()[:, :, None, None] * s["freq"]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    out = tuple(_turned(s[n], cos, sin, c["r"], c["interleaved"]) for n in ("q", "k"))
    if not c["train"]:
        return out
    return out + tuple(_turned(s[n], cos, -sin, c["r"], c["interleaved"]) for n in ("dq", "dk"))


_RUN_PLAIN = dict(recurrence=_plain_recurrence, recurrence_step=_plain_recurrence_step, attention=_plain_attention,
                  attention_step=_plain_attention_step, rotary=_plain_rotary)


# --------------------------------------------------------------------------- #
# what a pass cannot do without
# --------------------------------------------------------------------------- #
def _pairs(t, left, right, sinks):
    """Visible (query, key) pairs of one head over t positions."""
    inside = sum(min(t - 1, p + right) - max(0, p - left) + 1 for p in range(t))
    return inside + sum(max(0, min(sinks, p - left, t)) for p in range(t))


def work(case):
    c, e = case, 2 if case["type"] == "bf16" else 4
    train, live = c.get("train", False), 0.75 if c.get("ragged") else 1.0       # ragged: lengths from t / 2 to t
    if c["op"] == "recurrence":
        m, st = c["n"] * c["l"] * c["d"], c["n"] * c["d"] * 4
        # forward: x, f in, y out; backward: x, f, dy in, dx, df out
        return {"bytes": ((5 * live + 3) if train else (2 * live + 1)) * m * e + (4 if train else 2) * st,
                "flops": (14 if train else 5) * m * live}
    if c["op"] == "recurrence_step":
        m = c["n"] * c["d"]
        return {"bytes": m * (3 * e + 8), "flops": 5 * m}
    if c["op"] == "attention":
        nq, nk = c["b"] * c["t"] * c["hq"] * c["dh"], c["b"] * c["t"] * c["hk"] * c["dh"]
        pairs = _pairs(c["t"], c["left"], c["right"], c["sinks"]) * c["b"] * c["hq"]
        # forward: q, k, v in, o out; backward: q, k, v, o, do in, dq, dk, dv out
        return {"bytes": e * (((4 * nq + 4 * nk) * live + 2 * nq + 2 * nk) if train else ((nq + 2 * nk) * live + nq)),
                "flops": (14 if train else 4) * c["dh"] * pairs * live}
    if c["op"] == "attention_step":
        m = c["b"] * (c["sinks"] + c["window"]) * c["hk"] * c["dh"]
        return {"bytes": e * (2 * m + 2 * c["b"] * c["hq"] * c["dh"] + 4 * c["b"] * c["hk"] * c["dh"]),
                "flops": 4 * m * (c["hq"] // c["hk"])}
    m = c["b"] * c["t"] * (c["hq"] + c["hk"]) * c["dh"]
    return {"bytes": (4 if train else 2) * m * e + c["b"] * c["t"] * 8, "flops": (2 if train else 1) * 3 * m}


# --------------------------------------------------------------------------- #
# the definitions in 64 bits
# --------------------------------------------------------------------------- #
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        s = {n: x.double() if torch.is_tensor(x) and x.is_floating_point() else x for n, x in s.items()}
        return getattr(_Exact, case["op"])(case, s)


class _Exact:
    @staticmethod
    def recurrence(c, s):
        x, n, l = s["x"], c["n"], c["l"]
        a = 1 / (1 + torch.exp(-s["f"]))
        i = 1 / (1 + torch.exp(s["f"]))
        end = torch.full((n,), l, device=x.device) if s["lengths"] is None else s["lengths"]
        order = range(l - 1, -1, -1) if c["reverse"] else range(l)
        h, y, before = s["h0"].clone(), torch.zeros_like(x), torch.zeros_like(x)
        for t in order:
            on = (t < end)[:, None]
            before[:, t] = h
            h = torch.where(on, a[:, t] * h + i[:, t] * x[:, t], h)
            y[:, t] = torch.where(on, h, 0)
        if not c["train"]:
            return y, h
        g, dx, df = s["dlast"].clone(), torch.zeros_like(x), torch.zeros_like(x)
        for t in reversed(order):
            on = (t < end)[:, None]
            mine = g + s["dy"][:, t]
            dx[:, t] = torch.where(on, mine * i[:, t], 0)
            df[:, t] = torch.where(on, mine * a[:, t] * i[:, t] * (before[:, t] - x[:, t]), 0)
            g = torch.where(on, mine * a[:, t], g)
        return y, h, dx, df, g

    @staticmethod
    def recurrence_step(c, s):
        a = 1 / (1 + torch.exp(-s["f"]))
        h = s["state"] + (1 - a) * (s["x"] - s["state"])
        return h, h

    @staticmethod
    def attention(c, s):
        outs = [[] for _ in range(4 if c["train"] else 1)]
        group = c["hq"] // c["hk"]
        for b in range(c["b"]):                                    # item by item, key head by key head, over its own length
            n = c["t"] if s["lengths"] is None else int(s["lengths"][b])
            p = torch.arange(n, device=s["q"].device)
            gap = p[None, :] - p[:, None]
            hidden = (gap > c["right"]) | ((gap < -c["left"]) & (p[None, :] >= c["sinks"]))
            o, dq = torch.zeros_like(s["q"][b]), torch.zeros_like(s["q"][b])
            dk, dv = torch.zeros_like(s["k"][b]), torch.zeros_like(s["v"][b])
            for h in range(c["hq"]):
                q, k, v = s["q"][b, :n, h], s["k"][b, :n, h // group], s["v"][b, :n, h // group]
                w = torch.softmax((q @ k.t() * c["dh"] ** -0.5).masked_fill(hidden, -math.inf), -1)
                o[:n, h] = w @ v
                if c["train"]:
                    do = s["do"][b, :n, h]
                    dw = w * (do @ v.t() - (do * o[:n, h]).sum(-1, keepdim=True)) * c["dh"] ** -0.5
                    dv[:n, h // group] += w.t() @ do
                    dk[:n, h // group] += dw.t() @ q
                    dq[:n, h] = dw @ k
            for got, x in zip(outs, (o, dq, dk, dv)):
                got.append(x)
        outs = tuple(torch.stack(x) for x in outs)
        return outs if c["train"] else outs[0]

    @staticmethod
    def attention_step(c, s):
        o = torch.zeros_like(s["q"])
        for b, p in enumerate(s["positions"].tolist()):
            slot = p if p < c["sinks"] else c["sinks"] + (p - c["sinks"]) % c["window"]
            s["k_cache"][b, slot], s["v_cache"][b, slot] = s["k"][b], s["v"][b]
            n = min(p + 1, c["sinks"] + c["window"])
            for h in range(c["hq"]):
                kv = h // (c["hq"] // c["hk"])
                w = torch.softmax(s["k_cache"][b, :n, kv] @ s["q"][b, h] * c["dh"] ** -0.5, 0)
                o[b, h] = w @ s["v_cache"][b, :n, kv]
        return o, s["k_cache"], s["v_cache"]

    @staticmethod
    def rotary(c, s):
        half = c["r"] // 2
        angle = (s["positions"].double()[..., None] * s["freq"])[:, :, None]
        turn = torch.complex(torch.cos(angle), torch.sin(angle))

        def rotated(x, by):
            u = torch.arange(half, device=x.device) * (2 if c["interleaved"] else 1)
            v = u + (1 if c["interleaved"] else half)
            z, out = torch.complex(x[..., u], x[..., v]) * by, x.clone()
            out[..., u], out[..., v] = z.real, z.imag
            return out

        out = rotated(s["q"], turn), rotated(s["k"], turn)
        return out + (rotated(s["dq"], turn.conj()), rotated(s["dk"], turn.conj())) if c["train"] else out

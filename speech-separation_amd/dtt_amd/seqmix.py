"""Token mixers for long recordings: a gated linear recurrence (beside the BiLSTM of the dual-path modules), windowed
attention with first tokens that stay visible (beside the dense token attention of the fusion block) and rotary positions
(beside its additive sinusoids).  They train over whole recordings in memory linear in their length, and run one frame at
a time with a state of fixed size: ``gated_recurrence_step`` and ``window_attention_step``.

All of them take float32 or bfloat16 tensors on one GPU and launch on its current stream; nothing synchronises, and no
result depends on the order of atomics.  Wrong arguments raise DttError.  Inputs may be views (slices of a fused
projection, permuted axes) as long as their innermost axis is contiguous; others are copied first.  The single-frame forms
can be captured into HIP graphs: positions and lengths are read from device memory.

The reference has none of these; latent.py:87-96 and cross_attention_positional.py:6-12,66-69 are what they stand beside.
"""
from __future__ import annotations

import ctypes as C
import math

import torch
from torch.autograd.function import once_differentiable

from ._lib import lib, check, stream_ptr, dtype_code, DttError, DttRecurrence, DttRotary, DttWattn, DttWattnStep

F32 = torch.float32


# --------------------------------------------------------------------------- #
# arguments
# --------------------------------------------------------------------------- #
class _on:
    """Launches inside go to `dev`, whatever the current device is."""

    def __init__(self, dev):
        self.ctx = None if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)
        return False


def _need(ok, what):
    if not ok:
        raise DttError(what)


def _same(name, first, *others):
    """`others` ((name, tensor) pairs, None allowed) on first's device; first on a GPU."""
    if not first.is_cuda:
        raise DttError("dtt_amd ops need CUDA(HIP) tensors; there is no CPU path")
    for n, t in others:
        if t is not None and t.device != first.device:
            raise DttError(f"{name}: {n} is on {t.device}, the other tensors on {first.device}")


def _p(t):
    return None if t is None else t.data_ptr()


def _rows(t, bytes_=1):
    """`t` with a contiguous innermost axis and, where asked, every row on `bytes_` bytes; a copy if it has not."""
    e = t.element_size()
    if (t.stride(-1) == 1 or t.shape[-1] == 1) and (bytes_ <= e or (
            t.data_ptr() % bytes_ == 0 and all(s * e % bytes_ == 0 or n == 1 for s, n in zip(t.stride()[:-1], t.shape)))):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    """Strides of all axes but the innermost; 0 for axes of one element."""
    return [s if n > 1 else 0 for s, n in zip(t.stride()[:-1], t.shape)]


def _lengths(name, lengths, batch, first):
    if lengths is None:
        return None
    _need(torch.is_tensor(lengths) and lengths.dtype in (torch.int32, torch.int64) and tuple(lengths.shape) == tuple(batch),
          f"{name}: lengths must be an int32 or int64 tensor of shape {tuple(batch)}")
    _same(name, first, ("lengths", lengths))
    return lengths.to(torch.int32).contiguous()


def _wants_grad(*ts):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def _workspace(n, dev):
    return torch.empty(n, dtype=torch.uint8, device=dev) if n > 0 else None


# --------------------------------------------------------------------------- #
# gated linear recurrence
# --------------------------------------------------------------------------- #
def _rec_args(x, f, reverse, lengths, h0):
    """The struct's common part; x, f [(outer,) inner, L, D] as rows."""
    L, D = x.shape[-2:]
    n = x.numel() // (L * D)
    ni = x.shape[1] if x.dim() == 4 else 1
    g = DttRecurrence(N=n, NI=ni, L=L, D=D, reverse=1 if reverse else 0, dtype=dtype_code(x.dtype))
    g.x, g.f, g.lengths, g.h0 = x.data_ptr(), f.data_ptr(), _p(lengths), _p(h0)
    g.x_so, g.x_si, g.x_sl = _rec_strides(x)
    g.f_so, g.f_si, g.f_sl = _rec_strides(f)
    return g


def _rec_strides(t):
    s = _strides(t)
    return s if len(s) == 3 else (s[0], 0, s[1])


def _rec_forward(x, f, h0, reverse, lengths, keep):
    dev = x.device
    with _on(dev):
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        last = torch.empty(x.shape[:-2] + x.shape[-1:], dtype=F32, device=dev)
        g = _rec_args(x, f, reverse, lengths, h0)
        g.y, g.last = y.data_ptr(), last.data_ptr()
        L = lib()
        states = None
        if keep:
            states = torch.empty(L.dtt_recurrence_states(C.byref(g)), dtype=F32, device=dev)
            g.states = states.data_ptr()
        ws = _workspace(L.dtt_recurrence_ws_bytes(C.byref(g)), dev)
        if ws is not None:
            g.ws, g.ws_bytes = ws.data_ptr(), ws.numel()
        check(L.dtt_recurrence_fwd(C.byref(g), stream_ptr()), "dtt_recurrence_fwd")
    return y, last, states


class GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, h0, reverse, lengths):
        y, last, states = _rec_forward(x, f, h0, reverse, lengths, True)
        ctx.save_for_backward(x, f, h0, lengths, states)
        ctx.reverse = reverse
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, f, h0, lengths, states = ctx.saved_tensors
        dev = x.device
        with _on(dev):
            dy = torch.zeros(x.shape[-1], dtype=x.dtype, device=dev).expand(x.shape) if dy is None else _rows(dy)
            dlast = dlast.contiguous() if dlast is not None else None
            dx, df = (torch.empty(x.shape, dtype=x.dtype, device=dev) for _ in range(2))
            dh0 = torch.empty(h0.shape, dtype=F32, device=dev) if h0 is not None and ctx.needs_input_grad[2] else None
            g = _rec_args(x, f, ctx.reverse, lengths, h0)
            g.dy, g.dx, g.df, g.dlast, g.dh0, g.states = (dy.data_ptr(), dx.data_ptr(), df.data_ptr(), _p(dlast), _p(dh0),
                                                         states.data_ptr())
            g.g_so, g.g_si, g.g_sl = _rec_strides(dy)
            L = lib()
            ws = _workspace(L.dtt_recurrence_ws_bytes(C.byref(g)), dev)
            if ws is not None:
                g.ws, g.ws_bytes = ws.data_ptr(), ws.numel()
            check(L.dtt_recurrence_bwd(C.byref(g), stream_ptr()), "dtt_recurrence_bwd")
        return dx, df, dh0, None, None


def gated_recurrence(x, f, h0=None, reverse=False, lengths=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t per channel, a = sigmoid(f); returns (y, last): y_t = h_t in x's dtype and the state
    behind the last step in float32.

    x, f [B, L, D] or [B, N, L, D] (two batch axes, e.g. the frequency-axis view of [B, T, F, C] rows) of one dtype; h0
    float32 [B(, N), D] or None (zero).  ``reverse``: from an item's last step to its first.  ``lengths`` [B(, N)]: steps
    from lengths on are padding: never read, y and the gradients are 0 there, and ``last`` is the state of the item's own
    last step.  Differentiable in x, f and h0; states are float32 throughout."""
    name = "gated_recurrence"
    _need(torch.is_tensor(x) and torch.is_tensor(f) and x.dim() in (3, 4) and x.shape == f.shape,
          f"{name}: x and f must have one shape, [B, L, D] or [B, N, L, D]")
    _same(name, x, ("f", f), ("h0", h0))
    _need(x.dtype == f.dtype, f"{name}: x is {x.dtype}, f is {f.dtype}")
    dtype_code(x.dtype)
    batch, D = x.shape[:-2], x.shape[-1]
    if h0 is not None:
        _need(h0.dtype == F32 and tuple(h0.shape) == tuple(batch) + (D,), f"{name}: h0 must be float32 {tuple(batch) + (D,)}")
    lengths = _lengths(name, lengths, batch, x)
    if x.numel() == 0:
        return x * f, (h0.clone() if h0 is not None else torch.zeros(tuple(batch) + (D,), dtype=F32, device=x.device))
    x, f, h0 = _rows(x), _rows(f), h0.contiguous() if h0 is not None else None
    if _wants_grad(x, f, h0):
        return GatedRecurrence.apply(x, f, h0, bool(reverse), lengths)
    return _rec_forward(x, f, h0, reverse, lengths, False)[:2]


def gated_recurrence_step(x, f, state):
    """One step of gated_recurrence for every item: x, f [N, D], state float32 [N, D] (contiguous), replaced by the new
    state; returns it in x's dtype.  No gradients."""
    name = "gated_recurrence_step"
    _need(x.dim() == 2 and x.shape == f.shape and x.shape == state.shape, f"{name}: x, f and state must have one shape [N, D]")
    _same(name, x, ("f", f), ("state", state))
    _need(x.dtype == f.dtype and state.dtype == F32 and state.is_contiguous(),
          f"{name}: x and f of one dtype, state float32 and contiguous")
    _need(not _wants_grad(x, f, state), f"{name} has no gradient: call it under torch.no_grad()")
    d = dtype_code(x.dtype)
    N, D = x.shape
    x, f = _rows(x), _rows(f)
    y = torch.empty((N, D), dtype=x.dtype, device=x.device)
    if y.numel():
        with _on(x.device):
            check(lib().dtt_recurrence_step(C.c_void_p(x.data_ptr()), C.c_void_p(f.data_ptr()), C.c_void_p(state.data_ptr()),
                                            C.c_void_p(y.data_ptr()), N, D, C.c_int64(x.stride(0) if N > 1 else 0),
                                            C.c_int64(f.stride(0) if N > 1 else 0), d, stream_ptr()), "dtt_recurrence_step")
    return y


# --------------------------------------------------------------------------- #
# windowed attention
# --------------------------------------------------------------------------- #
def _attn_args(q, k, v, lengths, cfg):
    left, right, sinks, offset, scale = cfg
    B, Tq, Hq, dh = q.shape
    g = DttWattn(B=B, Tq=Tq, Tk=k.shape[1], Hq=Hq, Hk=k.shape[2], DH=dh, left=left, right=right, sinks=sinks, offset=offset,
                 dtype=dtype_code(q.dtype), scale=scale)
    g.q, g.k, g.v, g.lengths = q.data_ptr(), k.data_ptr(), v.data_ptr(), _p(lengths)
    g.q_sb, g.q_st, g.q_sh = _strides(q)
    g.k_sb, g.k_st, g.k_sh = _strides(k)
    g.v_sb, g.v_st, g.v_sh = _strides(v)
    return g


def _attn_forward(q, k, v, lengths, cfg, keep):
    with _on(q.device):
        B, Tq, Hq, dh = q.shape
        out = torch.empty((B, Tq, Hq, dh), dtype=q.dtype, device=q.device)
        lse = torch.empty((B, Hq, Tq), dtype=F32, device=q.device) if keep else None
        g = _attn_args(q, k, v, lengths, cfg)
        g.out, g.lse = out.data_ptr(), _p(lse)
        check(lib().dtt_wattn_fwd(C.byref(g), stream_ptr()), "dtt_wattn_fwd")
    return out, lse


class WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, cfg):
        out, lse = _attn_forward(q, k, v, lengths, cfg, True)
        ctx.save_for_backward(q, k, v, lengths, out, lse)
        ctx.cfg = cfg
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, lengths, out, lse = ctx.saved_tensors
        dev = q.device
        with _on(dev):
            do = _rows(do, 16)
            dq = torch.empty(q.shape, dtype=q.dtype, device=dev)
            dk, dv = (torch.empty(k.shape, dtype=q.dtype, device=dev) for _ in range(2))
            dd = torch.empty_like(lse)
            g = _attn_args(q, k, v, lengths, ctx.cfg)
            g.out, g.lse, g.dout, g.dq, g.dk, g.dv, g.dd = (out.data_ptr(), lse.data_ptr(), do.data_ptr(), dq.data_ptr(),
                                                           dk.data_ptr(), dv.data_ptr(), dd.data_ptr())
            g.g_sb, g.g_st, g.g_sh = _strides(do)
            L = lib()
            ws = _workspace(L.dtt_wattn_bwd_ws_bytes(C.byref(g)), dev)
            if ws is not None:
                g.ws, g.ws_bytes = ws.data_ptr(), ws.numel()
            check(L.dtt_wattn_bwd(C.byref(g), stream_ptr()), "dtt_wattn_bwd")
        return dq, dk, dv, None, None


def _heads_check(name, q, k, v, dims):
    _need(all(torch.is_tensor(t) and t.dim() == dims for t in (q, k, v)), f"{name}: q, k and v must have {dims} axes")
    _same(name, q, ("k", k), ("v", v))
    _need(q.dtype == k.dtype == v.dtype, f"{name}: q, k and v must have one dtype")
    dtype_code(q.dtype)
    _need(k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[-1] == q.shape[-1],
          f"{name}: shapes {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)} do not fit")
    _need(k.shape[-2] > 0 and q.shape[-2] > 0 and q.shape[-2] % k.shape[-2] == 0,
          f"{name}: {q.shape[-2]} query heads over {k.shape[-2]} key heads")
    _need(q.shape[-1] in (32, 64, 96, 128), f"{name}: head width {q.shape[-1]} (32, 64, 96 or 128)")


_BIG = 1 << 28


def window_attention(q, k, v, left, right=0, sinks=0, lengths=None, offset=None, scale=None):
    """softmax(scale q k^T) v over a window: the query at position p = offset + i sees key j where j <= p + right and
    (j >= p - left or j < sinks); a row that sees no key is zero.

    q [B, Tq, Hq, dh], k, v [B, Tk, Hk, dh] of one dtype, Hq a multiple of Hk (query head h reads key head
    h // (Hq // Hk)), dh 32, 64, 96 or 128; ``sinks`` <= 128.  ``offset`` defaults to Tk - Tq (the queries are the last
    Tq positions), ``scale`` (positive) to dh ** -0.5.  ``lengths`` [B]: positions from lengths on are padding -- keys there are never
    read, rows there are zero and take no part in any gradient.  A non-finite key or value inside lengths may reach rows
    of the same 32 positions that do not see it.  Differentiable in q, k and v."""
    name = "window_attention"
    _heads_check(name, q, k, v, 4)
    B, Tq, Hq, dh = q.shape
    Tk = k.shape[1]
    offset = Tk - Tq if offset is None else int(offset)
    left, right, sinks = int(left), int(right), int(sinks)
    _need(left >= 0 and right >= 0 and 0 <= sinks <= 128, f"{name}: left={left}, right={right} and sinks={sinks} (0 to 128)")
    _need(0 <= offset < _BIG and Tq < _BIG and Tk < _BIG, f"{name}: offset={offset}, Tq={Tq}, Tk={Tk} must be in [0, 2^28)")
    lengths = _lengths(name, lengths, (B,), q)
    if q.numel() == 0 or Tk == 0:
        return q * 0.0 + k.sum() * 0.0 + v.sum() * 0.0 if _wants_grad(q, k, v) else torch.zeros_like(q)
    cfg = (min(left, _BIG), min(right, _BIG), sinks, offset, dh ** -0.5 if scale is None else float(scale))
    q, k, v = _rows(q, 16), _rows(k, 16), _rows(v, 16)
    if _wants_grad(q, k, v):
        return WindowAttention.apply(q, k, v, lengths, cfg)
    return _attn_forward(q, k, v, lengths, cfg, False)[0]


def _cache_check(name, k, k_cache, v_cache, sinks):
    _need(k_cache.dim() == 4 and k_cache.shape == v_cache.shape and k_cache.shape[0] == k.shape[0] and
          k_cache.shape[2:] == k.shape[-2:], f"{name}: caches must be [B, sinks + window, Hk, dh], got {tuple(k_cache.shape)}")
    _need(k_cache.dtype == k.dtype and v_cache.dtype == k.dtype, f"{name}: caches must have the dtype of k")
    _same(name, k, ("k_cache", k_cache), ("v_cache", v_cache))
    _need(0 <= sinks < k_cache.shape[1], f"{name}: sinks={sinks} of {k_cache.shape[1]} slots (at least one for the window)")
    for c in (k_cache, v_cache):
        e = c.element_size()
        _need(c.stride(-1) == 1 and c.data_ptr() % 16 == 0 and all(s * e % 16 == 0 for s in c.stride()[:-1]),
              f"{name}: cache rows must be contiguous and start on 16 bytes")


def _step_args(k, v, k_cache, v_cache, sinks, scale):
    B, M, Hk, dh = k_cache.shape
    g = DttWattnStep(B=B, Hq=Hk, Hk=Hk, DH=dh, S=sinks, W=M - sinks, dtype=dtype_code(k.dtype), scale=scale)
    g.k, g.v, g.kc, g.vc = k.data_ptr(), v.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr()
    g.kc_sb, g.kc_st, g.kc_sh = _strides(k_cache)
    g.vc_sb, g.vc_st, g.vc_sh = _strides(v_cache)
    return g


def window_attention_step(q, k, v, k_cache, v_cache, positions, sinks=0, scale=None):
    """One frame per item against its rolling cache.  The caches [B, sinks + window, Hk, dh] hold the first ``sinks``
    positions and the last ``window``: position p lives in slot p, once the window is full in sinks + (p - sinks) % window.
    Writes k, v [B, Hk, dh] of position ``positions[b]`` (int64 [B], on the device) into their slot, then attends
    q [B, Hq, dh] to every slot filled so far: what window_attention(left=window - 1, sinks=sinks) gives for that row.
    An item with a negative position is idle: its cache stays as it is and its row is zero.  No gradients."""
    name = "window_attention_step"
    _heads_check(name, q, k, v, 3)
    sinks = int(sinks)
    _cache_check(name, k, k_cache, v_cache, sinks)
    _need(positions.dtype == torch.int64 and positions.dim() == 1 and positions.shape[0] == q.shape[0] and positions.is_contiguous(),
          f"{name}: positions must be a contiguous int64 tensor [B]")
    _same(name, q, ("positions", positions), ("k_cache", k_cache))
    _need(not _wants_grad(q, k, v), f"{name} has no gradient: call it under torch.no_grad()")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.numel() == 0:
        return out
    q, k, v = _rows(q, 16), _rows(k, 16), _rows(v, 16)
    with _on(q.device):
        g = _step_args(k, v, k_cache, v_cache, sinks, q.shape[-1] ** -0.5 if scale is None else float(scale))
        g.Hq = q.shape[1]
        g.q, g.out, g.positions = q.data_ptr(), out.data_ptr(), positions.data_ptr()
        g.q_sb, g.q_sh = _strides(q)
        g.k_sb, g.k_sh = _strides(k)
        g.v_sb, g.v_sh = _strides(v)
        L = lib()
        ws = _workspace(L.dtt_wattn_step_ws_bytes(C.byref(g)), q.device)
        if ws is not None:
            g.ws, g.ws_bytes = ws.data_ptr(), ws.numel()
        check(L.dtt_wattn_step(C.byref(g), stream_ptr()), "dtt_wattn_step")
    return out


def window_cache_fill(k, v, k_cache, v_cache, sinks=0, lengths=None):
    """Fills rolling caches (see window_attention_step) from whole sequences k, v [B, T, Hk, dh] that start at position 0, as
    T (or lengths[b]) single steps would: the next position of item b is then T (or lengths[b]).  Slots that hold none of
    those positions stay as they are."""
    name = "window_cache_fill"
    _heads_check(name, k, k, v, 4)
    sinks = int(sinks)
    _cache_check(name, k, k_cache, v_cache, sinks)
    _need(k.shape[1] < _BIG, f"{name}: T={k.shape[1]}")
    lengths = _lengths(name, lengths, k.shape[:1], k)
    if k.numel() == 0:
        return
    k, v = _rows(k.detach(), 16), _rows(v.detach(), 16)
    with _on(k.device):
        g = _step_args(k, v, k_cache, v_cache, sinks, 1.0)
        g.k_sb, g.k_st, g.k_sh = _strides(k)
        g.v_sb, g.v_st, g.v_sh = _strides(v)
        check(lib().dtt_wattn_cache_fill(C.byref(g), C.c_void_p(_p(lengths)), k.shape[1], stream_ptr()), "dtt_wattn_cache_fill")


# --------------------------------------------------------------------------- #
# rotary positions
# --------------------------------------------------------------------------- #
def rotary_frequencies(dim, base=10000.0, stretch=1.0, trained=None, blend=(1.0, 32.0), device=None):
    """Angles per position of the dim / 2 pairs, float64: base ** (-2 i / dim), divided by ``stretch`` for contexts that many
    times longer than the trained one.  With ``trained`` (that context's length) only slow pairs are stretched: a pair that
    turns ``blend[1]`` times or more over it keeps its frequency, one that turns ``blend[0]`` times or fewer is divided by
    stretch, those between are blended linearly in their number of turns."""
    _need(dim > 0 and dim % 2 == 0 and base > 0 and stretch > 0, f"rotary_frequencies: dim={dim}, base={base}, stretch={stretch}")
    i = torch.arange(dim // 2, dtype=torch.float64, device=device)
    freq = torch.exp(i * (-2.0 * math.log(base) / dim))
    if trained is None:
        return freq / stretch
    lo, hi = blend
    _need(trained > 0 and hi > lo >= 0, f"rotary_frequencies: trained={trained}, blend={blend}")
    keep = ((trained * freq / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
    return freq * (keep + (1.0 - keep) / stretch)


def _rotate(q, k, positions, freq, interleaved, amplitude, back):
    """q (k: or None) [B, T, H, dh] -> turned copies."""
    B, T, Hq, dh = q.shape
    with _on(q.device):
        qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        ko = torch.empty(k.shape, dtype=k.dtype, device=k.device) if k is not None else None
        g = DttRotary(B=B, T=T, Hq=Hq, Hk=k.shape[2] if k is not None else 0, dh=dh, r=2 * freq.shape[0],
                      interleaved=1 if interleaved else 0, back=1 if back else 0, pos64=1 if positions.dtype == torch.int64 else 0,
                      dtype=dtype_code(q.dtype), amplitude=amplitude)
        g.q, g.k, g.qo, g.ko, g.positions, g.freq = q.data_ptr(), _p(k), qo.data_ptr(), _p(ko), positions.data_ptr(), freq.data_ptr()
        g.q_sb, g.q_st, g.q_sh = _strides(q)
        if k is not None:
            g.k_sb, g.k_st, g.k_sh = _strides(k)
        if positions.dim() == 2:
            g.p_sb, g.p_st = positions.stride()
        else:
            g.p_st = positions.stride(0)
        check(lib().dtt_rotary(C.byref(g), stream_ptr()), "dtt_rotary")
    return qo, ko


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freq, interleaved, amplitude):
        qo, ko = _rotate(q, k, positions, freq, interleaved, amplitude, False)
        ctx.save_for_backward(positions, freq)
        ctx.cfg = (interleaved, amplitude)
        ctx.set_materialize_grads(False)
        return qo, ko

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        positions, freq = ctx.saved_tensors
        have = [_rows(t) for t in (dq, dk) if t is not None]
        got = _rotate(have[0], have[1] if len(have) > 1 else None, positions, freq, *ctx.cfg, True) if have else (None, None)
        if dq is None:
            got = (None, got[0])
        return got + (None, None, None, None)


def rotary(q, k, positions, freq, interleaved=False, amplitude=1.0):
    """Turns the pairs of the first 2 len(freq) channels of every head by position * freq (and scales them by ``amplitude``);
    the other channels are copied.  Pairs are (i, i + len(freq)), or (2 i, 2 i + 1) when ``interleaved``.

    q [B, T, Hq, dh] and k [B, T, Hk, dh] (or None) of one dtype; positions int64 or int32 [T] or [B, T]; freq float64
    (rotary_frequencies).  Angles are formed in float64, so positions far into a stream keep their precision.  Returns the
    turned q and k (or q alone where k is None); differentiable in both."""
    name = "rotary"
    _need(torch.is_tensor(q) and q.dim() == 4 and (k is None or (k.dim() == 4 and k.shape[:2] == q.shape[:2] and
                                                                k.shape[3] == q.shape[3] and k.dtype == q.dtype)),
          f"{name}: q and k must be [B, T, H, dh] of one dtype, with one B, T and dh")
    _same(name, q, ("k", k), ("positions", positions), ("freq", freq))
    dtype_code(q.dtype)
    B, T, _, dh = q.shape
    _need(positions.dtype in (torch.int32, torch.int64) and tuple(positions.shape) in ((T,), (B, T)),
          f"{name}: positions must be int32 or int64 [T] or [B, T], got {positions.dtype} {tuple(positions.shape)}")
    _need(freq.dtype == torch.float64 and freq.dim() == 1 and freq.is_contiguous() and 0 < 2 * freq.shape[0] <= min(dh, 4096),
          f"{name}: freq must be a contiguous float64 vector of 1 to dh / 2 elements")
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        _need(q.numel() == 0 and (k is None or k.numel() == 0), f"{name}: q and k must both have heads")
        return q.clone() if k is None else (q.clone(), k.clone())
    q, k = _rows(q), _rows(k) if k is not None else None
    args = (positions, freq, bool(interleaved), float(amplitude))
    out = Rotary.apply(q, k, *args) if _wants_grad(q, k) else _rotate(q, k, *args, False)
    return out[0] if k is None else out

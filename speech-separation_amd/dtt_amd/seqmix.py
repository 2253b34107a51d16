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

from ._lib import lib, check, dtype_code, DttError, DttRecurrence, DttRotary, DttWattn, DttWattnStep

# The single-frame forms and short training steps are bound by what the host spends on a call: arguments are checked with
# plain comparisons (messages are formatted on failure alone), structs are filled once and kept for the backward call.

F32, BF16, F64, I32, I64 = torch.float32, torch.bfloat16, torch.float64, torch.int32, torch.int64
_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)
# tells autograd that tensors were overwritten (through their addresses, which it cannot see): a backward pass that saved one of
# them, or a view of it, then raises as it does behind any in-place operation
_overwritten = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)
_ROWS = torch.contiguous_format
_addr = C.addressof
if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _stream = torch._C._cuda_getCurrentRawStream
else:
    def _stream(device):
        return torch.cuda.current_stream(device).cuda_stream


# --------------------------------------------------------------------------- #
# arguments
# --------------------------------------------------------------------------- #
def _fail(name, what):
    raise DttError(f"{name}: {what}")


def _on_gpu(name, t):
    """The index of t's GPU; refuses other devices and types."""
    if not t.is_cuda:
        _fail(name, "dtt_amd ops need CUDA(HIP) tensors; there is no CPU path")
    if t.dtype is not F32 and t.dtype is not BF16:
        dtype_code(t.dtype)
    return t.get_device()


def _beside(name, t, what, other):
    if other.device != t.device:
        _fail(name, f"{what} is on {other.device}, the other tensors on {t.device}")


def _sizes(name, t):
    """Refuses axes (and, of the axes before the last two, products) that 32 bits do not hold; t is known to be large."""
    if max(t.shape) >> 31 or math.prod(t.shape[:-2]) >> 31:
        _fail(name, f"shape {tuple(t.shape)}: sizes must be below 2^31")


def _inner(t):
    """`t` with a contiguous innermost axis, a copy if it has not."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.clone(memory_format=torch.contiguous_format)


def _rows16(t):
    """`t` with a contiguous innermost axis and every row on 16 bytes, a copy if it has not."""
    st, e = t.stride(), t.element_size()
    if st[-1] == 1 and t.data_ptr() % 16 == 0:
        bits = 0
        for s in st[:-1]:
            bits |= s
        if bits * e % 16 == 0 or all(s * e % 16 == 0 or n == 1 for s, n in zip(st[:-1], t.shape)):
            return t
    return t.clone(memory_format=torch.contiguous_format)


def _rows_attn(t):
    """What the whole-sequence attention reads: _rows16 with the rows of a head 1 row to 2^22 elements apart."""
    return _rows16(t) if t.shape[-1] <= t.stride(1) <= 1 << 22 or t.shape[1] == 1 else t.clone(memory_format=torch.contiguous_format)


def _lengths(name, lengths, batch, first):
    if lengths is None:
        return None
    if not torch.is_tensor(lengths) or lengths.dtype not in (I32, I64) or lengths.shape != batch:
        _fail(name, f"lengths must be an int32 or int64 tensor of shape {tuple(batch)}")
    _beside(name, first, "lengths", lengths)
    # (int64 lengths are clamped into int32 rather than wrapped: C treats all beyond the sequence alike)
    return (lengths if lengths.dtype is I32 else lengths.clamp(-1, (1 << 31) - 1).to(I32)).contiguous()


def _first_order(backward):
    """backward() without a derivative of its own: once_differentiable where a graph of the backward pass is recorded (which
    then refuses second derivatives), the bare function where none is."""
    refuses = once_differentiable(backward)

    def run(ctx, *grads):
        return refuses(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return staticmethod(run)


def _workspace(g, need, dev):
    """Scratch for one call; the caller keeps the tensor until the call is enqueued (the caching allocator orders reuse)."""
    if need <= 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    g.ws, g.ws_bytes = ws.data_ptr(), need
    return ws


def _again(g):
    """A copy of a forward call's struct (backward calls of one graph may run at the same time), for its sizes: the addresses
    are those of the forward call, and hooks on saved tensors (checkpoints, offloading) hand back others."""
    return type(g).from_buffer_copy(g)


# --------------------------------------------------------------------------- #
# gated linear recurrence
# --------------------------------------------------------------------------- #
def _rec_strides(t):
    s = t.stride()
    return s[:3] if len(s) == 4 else (s[0], 0, s[1])


def _rec_inputs(g, x, f, h0, lengths):
    g.x, g.f = x.data_ptr(), f.data_ptr()
    g.x_so, g.x_si, g.x_sl = _rec_strides(x)
    g.f_so, g.f_si, g.f_sl = _rec_strides(f)
    g.lengths = None if lengths is None else lengths.data_ptr()
    g.h0 = None if h0 is None else h0.data_ptr()


def _rec_forward(x, f, h0, reverse, lengths, keep):
    shape = x.shape
    L, D = shape[-2:]
    N = math.prod(shape[:-2])
    g = DttRecurrence(N=N, NI=shape[1] if len(shape) == 4 else 1, L=L, D=D, reverse=1 if reverse else 0,
                      dtype=1 if x.dtype is BF16 else 0)
    _rec_inputs(g, x, f, h0, lengths)
    y = torch.empty_like(x, memory_format=_ROWS)
    last = torch.empty(shape[:-2] + shape[-1:], dtype=F32, device=x.device)
    g.y, g.last = y.data_ptr(), last.data_ptr()
    lib_, ref, states = lib(), _addr(g), None
    if keep:
        states = torch.empty(lib_.dtt_recurrence_states(ref), dtype=F32, device=x.device)
        g.states = states.data_ptr()
    ws = _workspace(g, lib_.dtt_recurrence_ws_bytes(ref), x.device)  # noqa: F841 (alive until the call returns)
    check(lib_.dtt_recurrence_fwd(ref, _stream(x.get_device())), "dtt_recurrence_fwd")
    return y, last, states, g


class GatedRecurrence(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, h0, reverse, lengths):
        y, last, states, ctx.call = _rec_forward(x, f, h0, reverse, lengths, True)
        ctx.save_for_backward(x, f, h0, lengths, states)
        ctx.set_materialize_grads(False)
        return y, last

    @_first_order
    def backward(ctx, dy, dlast):
        x, f, h0, lengths, states = ctx.saved_tensors
        g, x, f = _again(ctx.call), _inner(x), _inner(f)
        _rec_inputs(g, x, f, h0, lengths)
        g.states = states.data_ptr()
        dy = x.new_zeros(x.shape[-1]).expand(x.shape) if dy is None else _inner(dy)
        if dlast is not None:
            dlast = dlast.contiguous()
            g.dlast = dlast.data_ptr()
        dx, df, dh0 = torch.empty_like(x, memory_format=_ROWS), torch.empty_like(x, memory_format=_ROWS), None
        if h0 is not None and ctx.needs_input_grad[2]:
            dh0 = torch.empty_like(h0)
            g.dh0 = dh0.data_ptr()
        g.dy, g.dx, g.df = dy.data_ptr(), dx.data_ptr(), df.data_ptr()
        g.g_so, g.g_si, g.g_sl = _rec_strides(dy)
        lib_, ref = lib(), _addr(g)
        ws = _workspace(g, lib_.dtt_recurrence_ws_bytes(ref), x.device)  # noqa: F841
        check(lib_.dtt_recurrence_bwd(ref, _stream(x.get_device())), "dtt_recurrence_bwd")
        return dx, df, dh0, None, None


def gated_recurrence(x, f, h0=None, reverse=False, lengths=None):
    """h_t = a_t h_{t-1} + (1 - a_t) x_t per channel, a = sigmoid(f); returns (y, last): y_t = h_t in x's dtype and the state
    behind the last step in float32.

    x, f [B, L, D] or [B, N, L, D] (two batch axes, e.g. the frequency-axis view of [B, T, F, C] rows) of one dtype; h0
    float32 [B(, N), D] or None (zero).  ``reverse``: from an item's last step to its first.  ``lengths`` [B(, N)]: steps
    from lengths on are padding: never read, y and the gradients are 0 there, and ``last`` is the state of the item's own
    last step.  Differentiable in x, f and h0; states are float32 throughout."""
    name = "gated_recurrence"
    if not torch.is_tensor(x) or not torch.is_tensor(f) or x.dim() not in (3, 4) or x.shape != f.shape:
        _fail(name, "x and f must have one shape, [B, L, D] or [B, N, L, D]")
    dev = _on_gpu(name, x)
    if x.dtype is not f.dtype:
        _fail(name, f"x is {x.dtype}, f is {f.dtype}")
    if f.get_device() != dev:
        _beside(name, x, "f", f)
    batch = x.shape[:-2]
    if h0 is not None:
        if h0.dtype is not F32 or h0.shape != batch + x.shape[-1:]:
            _fail(name, f"h0 must be float32 {tuple(batch + x.shape[-1:])}")
        _beside(name, x, "h0", h0)
    if lengths is not None:
        lengths = _lengths(name, lengths, batch, x)
    if x.numel() == 0:
        return x * f, (h0.clone() if h0 is not None else torch.zeros(batch + x.shape[-1:], dtype=F32, device=x.device))
    if dev != _device():
        with torch.cuda.device(dev):
            return gated_recurrence(x, f, h0, reverse, lengths)
    if x.numel() >> 31:
        _sizes(name, x)
    x, f = _inner(x), _inner(f)
    if h0 is not None:
        h0 = h0.contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or f.requires_grad or (h0 is not None and h0.requires_grad)):
        return GatedRecurrence.apply(x, f, h0, reverse, lengths)
    return _rec_forward(x, f, h0, reverse, lengths, False)[:2]


def gated_recurrence_step(x, f, state):
    """One step of gated_recurrence for every item: x, f [N, D], state float32 [N, D] (contiguous), replaced by the new
    state; returns it in x's dtype.  No gradients."""
    name = "gated_recurrence_step"
    shape = x.shape
    if len(shape) != 2 or f.shape != shape or state.shape != shape:
        _fail(name, "x, f and state must have one shape [N, D]")
    dev, dt = _on_gpu(name, x), x.dtype
    if f.dtype is not dt or state.dtype is not F32 or not state.is_contiguous():
        _fail(name, "x and f must have one dtype, state must be float32 and contiguous")
    if f.get_device() != dev or state.get_device() != dev:
        _fail(name, "x, f and state must be on one device")
    if torch.is_grad_enabled() and (x.requires_grad or f.requires_grad or state.requires_grad):
        _fail(name, "no gradient: call it under torch.no_grad()")
    if dev != _device():
        with torch.cuda.device(dev):
            return gated_recurrence_step(x, f, state)
    N, D = shape
    if N * D >> 31:
        _sizes(name, x)
    (xs, xe), (fs, fe) = x.stride(), f.stride()
    if xe != 1 or fe != 1:
        x, f = _inner(x), _inner(f)
        xs, fs = x.stride(0), f.stride(0)
    y = torch.empty_like(x, memory_format=_ROWS)
    if N * D:
        rc = lib().dtt_recurrence_step(x.data_ptr(), f.data_ptr(), state.data_ptr(), y.data_ptr(), N, D, xs, fs,
                                       1 if dt is BF16 else 0, _stream(dev))
        if rc:
            check(rc, "dtt_recurrence_step")
        _overwritten((state,))
    return y


# --------------------------------------------------------------------------- #
# windowed attention
# --------------------------------------------------------------------------- #
def _attn_inputs(g, q, k, v, lengths):
    g.q, g.k, g.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    g.q_sb, g.q_st, g.q_sh, _ = q.stride()
    g.k_sb, g.k_st, g.k_sh, _ = k.stride()
    g.v_sb, g.v_st, g.v_sh, _ = v.stride()
    g.lengths = None if lengths is None else lengths.data_ptr()


def _attn_forward(q, k, v, lengths, cfg, keep):
    B, Tq, Hq, dh = q.shape
    g = DttWattn(B=B, Tq=Tq, Tk=k.shape[1], Hq=Hq, Hk=k.shape[2], DH=dh, left=cfg[0], right=cfg[1], sinks=cfg[2], offset=cfg[3],
                 dtype=1 if q.dtype is BF16 else 0, scale=cfg[4])
    _attn_inputs(g, q, k, v, lengths)
    out, rest, lse = torch.empty_like(q, memory_format=_ROWS), None, None
    g.out = out.data_ptr()
    if keep:
        if q.dtype is BF16:                                 # what rounding leaves off `out`: the gradients take it whole
            rest = torch.empty_like(out)
            g.rest = rest.data_ptr()
        lse = torch.empty((2, B, Hq, Tq), dtype=F32, device=q.device)
        g.lse = lse.data_ptr()
    check(lib().dtt_wattn_fwd(_addr(g), _stream(q.get_device())), "dtt_wattn_fwd")
    return out, rest, lse, g


class WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, cfg):
        out, rest, lse, ctx.call = _attn_forward(q, k, v, lengths, cfg, True)
        ctx.save_for_backward(q, k, v, lengths, out, rest, lse)
        return out

    @_first_order
    def backward(ctx, do):
        q, k, v, lengths, out, rest, lse = ctx.saved_tensors
        q, k, v, do, g = _rows_attn(q), _rows_attn(k), _rows_attn(v), _rows_attn(do), _again(ctx.call)
        _attn_inputs(g, q, k, v, lengths)
        g.out, g.rest, g.lse = out.data_ptr(), None if rest is None else rest.data_ptr(), lse.data_ptr()
        dq, dk, dv = (torch.empty_like(t, memory_format=_ROWS) for t in (q, k, v))
        dd = torch.empty_like(lse[0])
        g.dout, g.dq, g.dk, g.dv, g.dd = do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dd.data_ptr()
        g.g_sb, g.g_st, g.g_sh, _ = do.stride()
        lib_, ref = lib(), _addr(g)
        ws = _workspace(g, lib_.dtt_wattn_bwd_ws_bytes(ref), q.device)  # noqa: F841 (alive until the call returns)
        check(lib_.dtt_wattn_bwd(ref, _stream(q.get_device())), "dtt_wattn_bwd")
        return dq, dk, dv, None, None


def _heads_check(name, q, k, v, dims):
    """The index of the tensors' GPU."""
    if not (torch.is_tensor(q) and torch.is_tensor(k) and torch.is_tensor(v)):
        _fail(name, "q, k and v must be tensors")
    qs, ks = q.shape, k.shape
    if len(qs) != dims or len(ks) != dims:
        _fail(name, f"q, k and v must have {dims} axes")
    dev, dt = _on_gpu(name, q), q.dtype
    if ks != v.shape or ks[0] != qs[0] or ks[-1] != qs[-1]:
        _fail(name, f"shapes {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)} do not fit")
    if k.dtype is not dt or v.dtype is not dt:
        _fail(name, "q, k and v must have one dtype")
    if k.get_device() != dev or v.get_device() != dev:
        _fail(name, f"q, k and v are on {q.device}, {k.device} and {v.device}")
    hq, hk = qs[-2], ks[-2]
    if hq == 0 or hk == 0 or hq % hk:
        _fail(name, f"{hq} query heads over {hk} key heads")
    if qs[-1] not in (32, 64, 96, 128):
        _fail(name, f"head width {qs[-1]} (32, 64, 96 or 128)")
    if q.numel() >> 31:
        _sizes(name, q)
    return dev


_BIG = 1 << 28


def window_attention(q, k, v, left, right=0, sinks=0, lengths=None, offset=None, scale=None):
    """softmax(scale q k^T) v over a window: the query at position p = offset + i sees key j where j <= p + right and
    (j >= p - left or j < sinks); a row that sees no key is zero.

    q [B, Tq, Hq, dh], k, v [B, Tk, Hk, dh] of one dtype, Hq a multiple of Hk (query head h reads key head
    h // (Hq // Hk)), dh 32, 64, 96 or 128; ``sinks`` <= 128.  ``offset`` defaults to Tk - Tq (the queries are the last
    Tq positions), ``scale`` (positive) to dh ** -0.5.  ``lengths`` [B]: positions from lengths on are padding -- keys there
    are never read, rows there are zero and take no part in any gradient.  A non-finite key or value inside lengths gives
    NaN, also in rows of the same 32 positions that do not see it.  bfloat16: weights enter their products with 16 bits,
    sums are float32, results are rounded once.  Differentiable in q, k and v."""
    name = "window_attention"
    dev = _heads_check(name, q, k, v, 4)
    Tq, Tk = q.shape[1], k.shape[1]
    offset = Tk - Tq if offset is None else int(offset)
    left, right, sinks = int(left), int(right), int(sinks)
    if left < 0 or right < 0 or not 0 <= sinks <= 128:
        _fail(name, f"left={left}, right={right} and sinks={sinks} (0 to 128)")
    if not 0 <= offset < _BIG or Tq >= _BIG or Tk >= _BIG:
        _fail(name, f"offset={offset}, Tq={Tq}, Tk={Tk} must be in [0, 2^28)")
    if lengths is not None:
        lengths = _lengths(name, lengths, q.shape[:1], q)
    grad = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if q.numel() == 0 or Tk == 0:
        return torch.zeros_like(q) + sum(t[..., :0].sum() for t in (q, k, v)) if grad else torch.zeros_like(q)
    if dev != _device():
        with torch.cuda.device(dev):
            return window_attention(q, k, v, left, right, sinks, lengths, offset, scale)
    # (positions reach offset + Tq < 2^29: a window cut to less than that would hide keys)
    cfg = (min(left, 2 * _BIG - 1), min(right, _BIG), sinks, offset, q.shape[-1] ** -0.5 if scale is None else float(scale))
    q, k, v = _rows_attn(q), _rows_attn(k), _rows_attn(v)
    return WindowAttention.apply(q, k, v, lengths, cfg) if grad else _attn_forward(q, k, v, lengths, cfg, False)[0]


def _step_args(name, k, v, k_cache, v_cache, sinks, scale):
    """Checks the caches of k, v and fills what the step and the fill share."""
    cs = k_cache.shape
    if len(cs) != 4 or cs != v_cache.shape or cs[0] != k.shape[0] or cs[2:] != k.shape[-2:]:
        _fail(name, f"caches must be [B, sinks + window, Hk, dh], got {tuple(cs)} and {tuple(v_cache.shape)}")
    if k_cache.dtype is not k.dtype or v_cache.dtype is not k.dtype:
        _fail(name, "caches must have the dtype of k")
    if k_cache.get_device() != k.get_device() or v_cache.get_device() != k.get_device():
        _fail(name, "caches must be on the device of k")
    if torch.is_grad_enabled() and (k_cache.requires_grad or v_cache.requires_grad):
        _fail(name, "no gradient through caches: call it under torch.no_grad()")
    if not 0 <= sinks < cs[1] or cs[1] >> 30:
        _fail(name, f"sinks={sinks} of {cs[1]} slots (at least one for the window, less than 2^30)")
    g = DttWattnStep(B=cs[0], Hq=cs[2], Hk=cs[2], DH=cs[3], S=sinks, W=cs[1] - sinks, dtype=1 if k.dtype is BF16 else 0, scale=scale)
    g.kc_sb, g.kc_st, g.kc_sh, ke = k_cache.stride()
    g.vc_sb, g.vc_st, g.vc_sh, ve = v_cache.stride()
    g.kc, g.vc = k_cache.data_ptr(), v_cache.data_ptr()
    if ke != 1 or ve != 1 or (g.kc | g.vc) % 16 or (g.kc_sb | g.kc_st | g.kc_sh | g.vc_sb | g.vc_st | g.vc_sh) * k.element_size() % 16:
        _fail(name, "cache rows must be contiguous and start on 16 bytes")
    if g.kc == g.vc or (cs[0] > 1 and not (g.kc_sb and g.vc_sb)) or (cs[1] > 1 and not (g.kc_st and g.vc_st)) or (
            cs[2] > 1 and not (g.kc_sh and g.vc_sh)):
        _fail(name, "every slot of every cache must have memory of its own (no broadcast caches)")
    return g


def window_attention_step(q, k, v, k_cache, v_cache, positions, sinks=0, scale=None):
    """One frame per item against its rolling cache.  The caches [B, sinks + window, Hk, dh] hold the first ``sinks``
    positions and the last ``window``: position p lives in slot p, once the window is full in sinks + (p - sinks) % window.
    Writes k, v [B, Hk, dh] of position ``positions[b]`` (int64 [B], on the device) into their slot, then attends
    q [B, Hq, dh] to every slot filled so far: what window_attention(left=window - 1, sinks=sinks) gives for that row.
    An item with a negative position is idle: its cache stays as it is and its row is zero.  No gradients."""
    name = "window_attention_step"
    dev = _heads_check(name, q, k, v, 3)
    if positions.dtype is not I64 or positions.dim() != 1 or positions.shape[0] != q.shape[0] or not positions.is_contiguous():
        _fail(name, "positions must be a contiguous int64 tensor [B]")
    if positions.get_device() != dev:
        _beside(name, q, "positions", positions)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        _fail(name, "no gradient: call it under torch.no_grad()")
    if dev != _device():
        with torch.cuda.device(dev):
            return window_attention_step(q, k, v, k_cache, v_cache, positions, sinks, scale)
    out = torch.empty_like(q, memory_format=_ROWS)
    if q.shape[0] == 0:
        return out
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    g = _step_args(name, k, v, k_cache, v_cache, int(sinks), q.shape[-1] ** -0.5 if scale is None else float(scale))
    g.Hq = q.shape[1]
    g.q, g.k, g.v, g.out, g.positions = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), positions.data_ptr()
    g.q_sb, g.q_sh, _ = q.stride()
    g.k_sb, g.k_sh, _ = k.stride()
    g.v_sb, g.v_sh, _ = v.stride()
    lib_, ref = lib(), _addr(g)
    ws = _workspace(g, lib_.dtt_wattn_step_ws_bytes(ref), q.device)  # noqa: F841 (alive until the call returns)
    check(lib_.dtt_wattn_step(ref, _stream(dev)), "dtt_wattn_step")
    _overwritten((k_cache, v_cache))
    return out


def window_cache_fill(k, v, k_cache, v_cache, sinks=0, lengths=None):
    """Fills rolling caches (see window_attention_step) from whole sequences k, v [B, T, Hk, dh] that start at position 0, as
    T (or lengths[b]) single steps would: the next position of item b is then T (or lengths[b]).  Slots that hold none of
    those positions stay as they are."""
    name = "window_cache_fill"
    _heads_check(name, k, k, v, 4)
    if k.shape[1] >= _BIG:
        _fail(name, f"T={k.shape[1]} must be below 2^28")
    lengths = _lengths(name, lengths, k.shape[:1], k)
    if k.get_device() != _device():
        with torch.cuda.device(k.device):
            return window_cache_fill(k, v, k_cache, v_cache, sinks, lengths)
    k, v = _rows16(k.detach()), _rows16(v.detach())
    g = _step_args(name, k, v, k_cache, v_cache, int(sinks), 1.0)
    if k.numel() == 0:
        return
    g.k, g.v = k.data_ptr(), v.data_ptr()
    g.k_sb, g.k_st, g.k_sh, _ = k.stride()
    g.v_sb, g.v_st, g.v_sh, _ = v.stride()
    check(lib().dtt_wattn_cache_fill(_addr(g), None if lengths is None else lengths.data_ptr(), k.shape[1],
                                     _stream(k.get_device())), "dtt_wattn_cache_fill")
    _overwritten((k_cache, v_cache))


# --------------------------------------------------------------------------- #
# rotary positions
# --------------------------------------------------------------------------- #
def rotary_frequencies(dim, base=10000.0, stretch=1.0, trained=None, blend=(1.0, 32.0), device=None):
    """Angles per position of the dim / 2 pairs, float64: base ** (-2 i / dim), divided by ``stretch`` for contexts that many
    times longer than the trained one.  With ``trained`` (that context's length) only slow pairs are stretched: a pair that
    turns ``blend[1]`` times or more over it keeps its frequency, one that turns ``blend[0]`` times or fewer is divided by
    stretch, those between are blended linearly in their number of turns."""
    name = "rotary_frequencies"
    if not (dim > 0 and dim % 2 == 0 and base > 0 and stretch > 0):
        _fail(name, f"dim={dim} (even), base={base}, stretch={stretch}")
    i = torch.arange(dim // 2, dtype=F64, device=device)
    freq = torch.exp(i * (-2.0 * math.log(base) / dim))
    if trained is None:
        return freq / stretch
    lo, hi = blend
    if not (trained > 0 and hi > lo >= 0):
        _fail(name, f"trained={trained}, blend={blend}")
    keep = ((trained * freq / (2 * math.pi) - lo) / (hi - lo)).clamp(0.0, 1.0)
    return freq * (keep + (1.0 - keep) / stretch)


def _rotate(q, k, g):
    """q and k (or None) [B, T, H, dh] -> turned copies, by the positions, frequencies and layout that `g` holds."""
    qo, ko = torch.empty_like(q, memory_format=_ROWS), None
    g.q, g.qo, g.Hq = q.data_ptr(), qo.data_ptr(), q.shape[2]
    g.q_sb, g.q_st, g.q_sh, _ = q.stride()
    if k is not None:
        ko = torch.empty_like(k, memory_format=_ROWS)
        g.k, g.ko, g.Hk = k.data_ptr(), ko.data_ptr(), k.shape[2]
        g.k_sb, g.k_st, g.k_sh, _ = k.stride()
    else:
        g.Hk = 0
    check(lib().dtt_rotary(_addr(g), _stream(q.get_device())), "dtt_rotary")
    return qo, ko


def _rot_inputs(g, positions, freq):
    g.positions, g.freq, g.p_st = positions.data_ptr(), freq.data_ptr(), positions.stride(-1)
    if positions.dim() == 2:
        g.p_sb = positions.stride(0)


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freq, g):
        ctx.save_for_backward(positions, freq)
        ctx.call = g
        ctx.set_materialize_grads(False)
        return _rotate(q, k, _again(g))

    @_first_order
    def backward(ctx, dq, dk):
        positions, freq = ctx.saved_tensors
        g = _again(ctx.call)
        g.back = 1
        _rot_inputs(g, positions, freq)
        if dq is None:
            return (None, None if dk is None else _rotate(_inner(dk), None, g)[0], None, None, None)
        return _rotate(_inner(dq), None if dk is None else _inner(dk), g) + (None, None, None)


def rotary(q, k, positions, freq, interleaved=False, amplitude=1.0):
    """Turns the pairs of the first 2 len(freq) channels of every head by position * freq (and scales them by ``amplitude``);
    the other channels are copied.  Pairs are (i, i + len(freq)), or (2 i, 2 i + 1) when ``interleaved``.

    q [B, T, Hq, dh] and k [B, T, Hk, dh] (or None) of one dtype; positions int64 or int32 [T] or [B, T]; freq float64
    (rotary_frequencies).  Angles are formed in float64, so positions far into a stream keep their precision.  Returns the
    turned q and k (or q alone where k is None); differentiable in both, not in freq."""
    name = "rotary"
    if not torch.is_tensor(q) or q.dim() != 4:
        _fail(name, "q must be [B, T, H, dh]")
    dev = _on_gpu(name, q)
    B, T, _, dh = q.shape
    if k is not None:
        ks = k.shape
        if len(ks) != 4 or ks[0] != B or ks[1] != T or ks[3] != dh or k.dtype is not q.dtype:
            _fail(name, f"q {tuple(q.shape)} {q.dtype} and k {tuple(ks)} {k.dtype} must agree in all but heads")
        if k.get_device() != dev:
            _beside(name, q, "k", k)
    pd = positions.dim()
    if positions.dtype not in (I64, I32) or positions.shape != ((T,) if pd == 1 else (B, T)):
        _fail(name, f"positions must be int32 or int64 [T] or [B, T], got {positions.dtype} {tuple(positions.shape)}")
    if freq.dtype is not F64 or freq.dim() != 1 or not freq.is_contiguous() or not 0 < 2 * freq.shape[0] <= min(dh, 4096):
        _fail(name, "freq must be a contiguous float64 vector of 1 to dh / 2 elements (2048 at most)")
    if freq.requires_grad and torch.is_grad_enabled():
        _fail(name, "no gradient of freq: detach it")
    if positions.get_device() != dev or freq.get_device() != dev:
        _fail(name, f"positions and freq must be on {q.device}")
    if q.numel() == 0 or (k is not None and k.numel() == 0):
        if q.numel() or (k is not None and k.numel()):
            _fail(name, "q and k must both have heads")
        return q.clone() if k is None else (q.clone(), k.clone())
    if q.numel() >> 31:
        _sizes(name, q)
    if k is not None and k.numel() >> 31:
        _sizes(name, k)
    if dev != _device():
        with torch.cuda.device(dev):
            return rotary(q, k, positions, freq, interleaved, amplitude)
    g = DttRotary(B=B, T=T, dh=dh, r=2 * freq.shape[0], interleaved=1 if interleaved else 0, pos64=1 if positions.dtype is I64 else 0,
                  dtype=1 if q.dtype is BF16 else 0, amplitude=amplitude)
    _rot_inputs(g, positions, freq)
    q = _inner(q)
    if k is None:
        return Rotary.apply(q, None, positions, freq, g)[0] if torch.is_grad_enabled() and q.requires_grad else _rotate(q, None, g)[0]
    k = _inner(k)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad):
        return Rotary.apply(q, k, positions, freq, g)
    return _rotate(q, k, g)

"""Sequence-layer operators of the public `ops` module: root-mean-square norm (csrc/rms_norm.hip), dropout from a counter-based generator
(csrc/dropout.hip) and linear attention with a decay for each head (csrc/linear_attention.hip).  They stand beside the layer factories of
the reference's code/ops.py:45-88 and have no counterpart there.

Each operator takes device tensors (fp32, bf16 or fp16), enqueues its HIP kernels on the current stream of the tensors' device and
allocates its outputs and workspaces like any torch operation; nothing synchronises.  Where an input requires a gradient the result
carries one (first order, reverse mode; dual tensors of forward mode are refused).  The explicit forms - `stats=True` and the `*_backward`
functions - are what a captured step uses: autograd itself is not captured (a backward pass recorded while an eager graph of the same leaves
lives ends the process), so inside a capture a call that would build an autograd graph raises; use torch.no_grad() there, or the explicit
forms on detached tensors."""
import struct

import torch

from . import _lib as L
from .kernels import tg_dtype

__all__ = ["rms_norm", "rms_norm_backward", "rms_norm_e4m3", "dropout", "dropout_backward", "dropout_rng", "linear_attention",
           "linear_attention_backward", "linear_attention_step"]

MAX_HEAD = 128   # largest Dk / Dv of linear_attention
MOST = 1 << 30   # channels of a normalised row, sequences and tokens


def _fail(text):
    raise L.TecoganHipError(text)


# Host time counts where a call is a few microseconds of GPU time: the device and the stream are asked for as plain integers (a Stream
# object is 3 us), entry points are looked up once
_device, _stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_entry = {}


def _call(dev, name, *args):
    """one entry point of the library on the current stream of `dev`"""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(L.load(), name)
    index = dev.index
    if index == _device():
        rc = fn(*args, _stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(index))
    if rc:
        L.check(rc, name)


_DTYPES = {torch.bfloat16: L.TG_BF16, torch.float16: L.TG_F16, torch.float32: L.TG_F32}


def _floats_of(name, *args):
    """a workspace's size"""
    fn = _entry.get(name)
    if fn is None:
        fn = _entry[name] = getattr(L.load(), name)
    return fn(*args)


def _floats(x, what):
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _fail(f"{what} must be a device tensor (no CPU fallback)")
    dt = _DTYPES.get(x.dtype)
    return tg_dtype(x.dtype) if dt is None else dt   # (raises for other element types)


def _like(x, t, what, shape=None):
    shape = x.shape if shape is None else shape
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.dtype != x.dtype or t.shape != shape:
        _fail(f"{what} must be a {x.dtype} tensor of shape {tuple(shape)} on {x.device} (nothing is broadcast)")
    return t


def _f32(x, t, what, shape):
    if not isinstance(t, torch.Tensor) or t.device != x.device or t.dtype != torch.float32 or t.shape != shape:
        _fail(f"{what} must be a float32 tensor of shape {tuple(shape)} on {x.device}")
    return t if t.is_contiguous() else t.contiguous()


_forward_ad = torch.autograd.forward_ad


def _no_tangents(*tensors):
    """refuses dual tensors: they do not require a gradient, so their tangents would be dropped without a word"""
    if _forward_ad._current_level >= 0 and any(isinstance(t, torch.Tensor) and _forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        _fail("no forward-mode derivatives: the operators have gradients (reverse mode) only")


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors)


def _capturing(dev):
    """whether the current stream of `dev` records a graph (torch asks the current device's)"""
    if dev.index == _device():
        return torch.cuda.is_current_stream_capturing()
    with torch.cuda.device(dev):
        return torch.cuda.is_current_stream_capturing()


def _grad(x, *others):
    """whether autograd has to record this call on x's device"""
    if not _wants_grad(x, *others) or not isinstance(x, torch.Tensor) or not x.is_cuda:   # (an x that is none is refused by the call itself)
        return False
    if _capturing(x.device):
        _fail("autograd is not captured into graphs: use torch.no_grad(), or the explicit backward functions on detached tensors")
    return True


# ------------------------------------------------------------------------------------------------------------ RMS norm
def _rows(x, channels):
    """(tensor, row stride) of x as rows of contiguous channels; a copy only where the leading dimensions do not collapse"""
    if x.is_contiguous():
        return x, channels
    if channels == 1 or x.stride(-1) == 1:
        try:
            r = x.view(-1, channels)
            return r, r.stride(0)
        except RuntimeError:
            pass
    return x.contiguous(), channels


def _rowmajor(x):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _norm_args(x, weight, residual, eps):
    dt = _floats(x, "x")
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MOST:
        _fail("rms_norm normalises the last dimension: it must have 1 .. 2^30 channels")
    if not eps >= 0:
        _fail("eps must not be negative")
    channels = x.shape[-1]
    if weight is not None:
        weight = _f32(x, weight, "weight", (channels,))
    if residual is not None:
        _like(x, residual, "residual")
    return dt, channels, weight


def _ptr(t):
    return None if t is None else t.data_ptr()


def _norm_fwd(x, weight, residual, eps, stats):
    dt, channels, weight = _norm_args(x, weight, residual, eps)
    xr, xs = _rows(x, channels)
    rr, rs = (None, 0) if residual is None else _rows(residual, channels)
    y = _rowmajor(x)
    s = None if residual is None else _rowmajor(x)
    rstd = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device) if stats else None
    _call(x.device, "tg_rms_norm", dt, xr.data_ptr(), xs, _ptr(rr), rs, _ptr(weight), y.data_ptr(), _ptr(s), _ptr(rstd),
          x.numel() // channels, channels, eps)
    return y, s, rstd


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, s, rstd = _norm_fwd(x, weight, residual, eps, True)
        ctx.save_for_backward(x, residual, rstd, weight)
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(rstd)
        return (y, rstd) if s is None else (y, s, rstd)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, *rest):
        x, residual, rstd, weight = ctx.saved_tensors
        ds = rest[0] if len(rest) == 2 else None
        if dy is None:   # only the sum was used
            return ds, None, ds, None
        dx, dw = rms_norm_backward(dy, x, rstd, weight, residual=residual, ds=ds, dweight=ctx.needs_input_grad[1])
        return dx if ctx.needs_input_grad[0] else None, dw, dx if ctx.needs_input_grad[2] else None, None


def rms_norm(x, weight=None, residual=None, eps=1e-6, stats=False):
    """y = s / sqrt(mean(s^2) + eps) * weight over the last dimension, s = x (+ residual).  weight: float32 (channels,) or None (ones);
    residual: like x.  Returns y, or (y, s) with a residual (s, the residual stream, in x's type; y comes from the unrounded sum), and at the
    end the rows' 1 / sqrt(...) (float32) with `stats` - what rms_norm_backward takes."""
    _no_tangents(x, weight, residual)
    if _grad(x, weight, residual):
        out = _RMSNorm.apply(x, weight, residual, eps)
        out = out if stats else out[:-1]
    else:
        y, s, rstd = _norm_fwd(x, weight, residual, eps, stats)
        out = (y,) + (() if s is None else (s,)) + ((rstd,) if stats else ())
    return out[0] if len(out) == 1 else out


def rms_norm_backward(dy, x, rstd, weight=None, residual=None, ds=None, dweight=True):
    """(dx, dweight) of rms_norm from dy, its inputs and its `stats`; ds: the gradient that reaches s on other ways (the residual stream's).
    dx is the gradient of x and of the residual alike; dweight is float32, None if not wanted.  Rows are added in a fixed order: the same
    call gives the same bits."""
    _no_tangents(dy, x, rstd, weight, residual, ds)
    dt, channels, weight = _norm_args(x, weight, residual, 0.0)
    _like(x, dy, "dy")
    rows = x.numel() // channels
    rstd = _f32(x, rstd, "rstd", x.shape[:-1])
    if ds is not None:
        _like(x, ds, "ds")
    gr, gs = _rows(dy, channels)
    xr, xs = _rows(x, channels)
    rr, rs = (None, 0) if residual is None else _rows(residual, channels)
    er, es = (None, 0) if ds is None else _rows(ds, channels)
    dx = _rowmajor(x)
    dw = scratch = None
    if dweight:
        dw = torch.empty(channels, dtype=torch.float32, device=x.device)
        scratch = torch.empty(_floats_of("tg_rms_norm_bwd_scratch_floats", rows, channels), dtype=torch.float32, device=x.device)
    _call(x.device, "tg_rms_norm_bwd", dt, gr.data_ptr(), gs, xr.data_ptr(), xs, _ptr(rr), rs, rstd.data_ptr(), _ptr(weight), _ptr(er), es,
          dx.data_ptr(), _ptr(dw), _ptr(scratch), rows, channels)
    return dx, dw


def rms_norm_e4m3(x, weight=None, residual=None, eps=1e-6):
    """rms_norm with an 8-bit output: (q, scale), or (q, scale, s) with a residual; q float8_e4m3fn like x, scale float32 per row =
    max(max|y|, 2^-100) / 448, y ~ q * scale.  A serving form: it has no gradient."""
    _no_tangents(x, weight, residual)
    if _wants_grad(x, weight, residual):
        _fail("rms_norm_e4m3 has no gradient: call it under torch.no_grad()")
    dt, channels, weight = _norm_args(x, weight, residual, eps)
    xr, xs = _rows(x, channels)
    rr, rs = (None, 0) if residual is None else _rows(residual, channels)
    q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    s = None if residual is None else _rowmajor(x)
    _call(x.device, "tg_rms_norm_e4m3", dt, xr.data_ptr(), xs, _ptr(rr), rs, _ptr(weight), q.data_ptr(), scale.data_ptr(), _ptr(s),
          x.numel() // channels, channels, eps)
    return (q, scale) if s is None else (q, scale, s)


# ------------------------------------------------------------------------------------------------------------- dropout
def dropout_rng(seed, device, step=0):
    """The generator's state, (seed, step) as an int64 device tensor.  One serves a whole model: give every dropout its own `layer`, and move
    `rng[1] += 1` between training steps (in a captured step: as its last operation, behind the backward passes)."""
    return torch.tensor([int(seed), int(step)], dtype=torch.int64, device=device)


def _drop(x, p, rng, layer, residual):
    dt = _floats(x, "x")
    if not 0.0 <= p < 1.0:
        _fail("dropout needs 0 <= p < 1")
    if not isinstance(rng, torch.Tensor) or rng.dtype != torch.int64 or rng.shape != (2,) or rng.device != x.device:
        _fail(f"rng must be an int64 tensor (seed, step) on {x.device} (dropout_rng)")
    if not 0 <= layer < 1 << 31:
        _fail("layer must be in 0 .. 2^31 - 1")
    if residual is not None:
        _like(x, residual, "residual")
        residual = residual.contiguous()
    x, rng = x.contiguous(), rng.contiguous()
    y = torch.empty_like(x)
    _call(x.device, "tg_dropout", dt, x.data_ptr(), _ptr(residual), y.data_ptr(), x.numel(), p, rng.data_ptr(), layer)
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, layer, residual):
        ctx.save_for_backward(rng)   # (moved in place before the backward pass: autograd says so instead of drawing another mask)
        ctx.p, ctx.layer = p, layer
        return _drop(x, p, rng, layer, residual)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        dx = dropout_backward(dy, ctx.p, ctx.saved_tensors[0], ctx.layer) if ctx.needs_input_grad[0] else None
        return dx, None, None, None, dy if ctx.needs_input_grad[4] else None


def dropout(x, p, rng, layer=0, residual=None):
    """(residual +) keep * x / (1 - p).  Element i of x (in row-major order, whatever x's strides) is dropped with probability p (to 2^-32) by
    the counter-based generator at (rng seed, rng step, layer, i); the mask is not stored, and is the same for every element type."""
    _no_tangents(x, residual)
    if _grad(x, residual):
        return _Dropout.apply(x, p, rng, layer, residual)
    return _drop(x, p, rng, layer, residual)


def dropout_backward(dy, p, rng, layer=0):
    """The gradient of x from y's: the same mask again, from the same (seed, step) and layer.  (The residual's gradient is dy.)"""
    _no_tangents(dy)
    return _drop(dy, p, rng, layer, None)


# ---------------------------------------------------------------------------------------------------- linear attention
_DESC = struct.Struct("6i9qf4x")   # tg_la_desc
_STRIDES = struct.Struct("3q")


def _channels_last(t):
    """t with contiguous channels (and a token stride that the kernels' 32-bit integers hold)"""
    return t if (t.stride(-1) == 1 or t.shape[-1] == 1) and t.stride(1) < 1 << 31 else t.contiguous()


def _desc(q, k, v, log_decay, scale, step, recorded=True):
    """(dtype, descriptor, (B, T, H, Dk, Dv), tensors) after the checks that the sequence and the single-token form share"""
    dt = _floats(q, "q")
    dims = 3 if step else 4
    for t, what in ((k, "k"), (v, "v")):
        if not isinstance(t, torch.Tensor) or t.device != q.device or t.dtype != q.dtype or t.dim() != dims:
            _fail(f"{what} must be a {q.dtype} tensor of {dims} dimensions on {q.device}")
    sq, sk, sv = q.shape, k.shape, v.shape
    if len(sq) != dims or sk[:-2] != sq[:-2] or sv[:-1] != sk[:-1] or sk[-1] != sq[-1]:
        form = "(B, heads, channels)" if step else "(B, T, heads, channels)"
        _fail(f"q, k, v must be {form} with q and k of the same channels, k and v of the same heads")
    B, H, HK, DK, DV = sq[0], sq[-2], sk[-2], sq[-1], sv[-1]
    T = 1 if step else sq[1]
    if H < 1 or HK < 1 or H % HK:
        _fail(f"{H} query heads do not divide over {HK} key / value heads")
    if not (1 <= DK <= MAX_HEAD and 1 <= DV <= MAX_HEAD):
        _fail(f"head sizes must be 1 .. {MAX_HEAD}: got {DK} and {DV}")
    if B > MOST or T > MOST:
        _fail("at most 2^30 sequences and tokens")
    log_decay = _f32(q, log_decay, "log_decay", (H,))
    if recorded and log_decay.requires_grad and torch.is_grad_enabled():
        _fail("log_decay is a constant of the heads: it has no gradient")
    q, k, v = _channels_last(q), _channels_last(k), _channels_last(v)
    scale = DK ** -0.5 if scale is None else float(scale)
    tq, tk, tv = q.stride(), k.stride(), v.stride()
    if step:
        d = _DESC.pack(B, T, H, HK, DK, DV, tq[0], 0, tq[1], tk[0], 0, tk[1], tv[0], 0, tv[1], scale)
    else:
        d = _DESC.pack(B, T, H, HK, DK, DV, *tq[:3], *tk[:3], *tv[:3], scale)
    return dt, d, (B, T, H, DK, DV), q, k, v, log_decay


def _lengths(q, lengths):
    if lengths is None:
        return None
    if not isinstance(lengths, torch.Tensor) or lengths.dtype != torch.int32 or lengths.device != q.device or lengths.shape != (q.shape[0],):
        _fail(f"lengths must be an int32 tensor of shape ({q.shape[0]},) on {q.device}")
    return lengths.contiguous()


def _attention_fwd(q, k, v, log_decay, scale, state, lengths):
    dt, d, (B, T, H, DK, DV), q, k, v, log_decay = _desc(q, k, v, log_decay, scale, False)
    dev = q.device
    state = None if state is None else _f32(q, state, "state", (B, H, DK, DV))
    lengths = _lengths(q, lengths)
    o = torch.empty((B, T, H, DV), dtype=q.dtype, device=dev)
    last = torch.empty((B, H, DK, DV), dtype=torch.float32, device=dev)
    n = _floats_of("tg_linear_attention_scratch_floats", dt, d)
    scratch = torch.empty(n, dtype=torch.float32, device=dev) if n else None
    _call(dev, "tg_linear_attention", dt, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), _ptr(lengths), _ptr(state), o.data_ptr(),
          last.data_ptr(), _ptr(scratch))
    return o, last


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, scale, state, lengths):
        ctx.save_for_backward(q, k, v, log_decay, state, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _attention_fwd(q, k, v, log_decay, scale, state, lengths)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do, dlast):
        q, k, v, log_decay, state, lengths = ctx.saved_tensors
        if do is None:   # only the state was used
            do = torch.zeros((*q.shape[:3], v.shape[3]), dtype=q.dtype, device=q.device)
        dq, dk, dv, dstate = linear_attention_backward(do, q, k, v, log_decay, ctx.scale, state, lengths, dlast)
        need = ctx.needs_input_grad
        return dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, None, None, dstate if need[5] else None, None


def linear_attention(q, k, v, log_decay, scale=None, state=None, lengths=None):
    """S_t = exp(log_decay) S_{t-1} + k_t v_t^T, o_t = scale q_t S_t for every sequence and head -> (o, last S).

    q (B, T, H, Dk), k (B, T, Hk, Dk), v (B, T, Hk, Dv) with channels contiguous (other strides as they are; H a multiple of Hk, head h reads
    k / v head h // (H / Hk)); log_decay float32 (H,), <= 0 for a memory that fades, a constant; scale: Dk^-0.5 if None; state: the first S,
    float32 (B, H, Dk, Dv), zeros if None; lengths: int32 (B,), tokens at and behind it are not read, their rows of o are zero and the last S is
    the one at the length.  o (B, T, H, Dv) in q's type, S in float32.  Gradients reach q, k, v and state.  An infinity or NaN in one token
    reaches that token and later ones only."""
    _no_tangents(q, k, v, log_decay, state)
    if _grad(q, k, v, state):
        _desc(q, k, v, log_decay, scale, False)   # (its refusals, before anything is recorded)
        return _LinearAttention.apply(q, k, v, log_decay, scale, state, lengths)
    return _attention_fwd(q, k, v, log_decay, scale, state, lengths)


def linear_attention_backward(do, q, k, v, log_decay, scale=None, state=None, lengths=None, dstate=None):
    """(dq, dk, dv, gradient of the first state) of linear_attention from the gradients of o and, if given, of the last state; the gradient of
    the first state is None where `state` is.  The gradients of shared key / value heads are summed in 32 bits."""
    _no_tangents(do, q, k, v, log_decay, state, dstate)
    dt, d, (B, T, H, DK, DV), q, k, v, log_decay = _desc(q, k, v, log_decay, scale, False, recorded=False)
    dev, shape = q.device, (B, H, DK, DV)
    do = _channels_last(_like(q, do, "do", (B, T, H, DV)))
    state = None if state is None else _f32(q, state, "state", shape)
    dstate = None if dstate is None else _f32(q, dstate, "dstate", shape)
    lengths = _lengths(q, lengths)
    dq, dk, dv = _rowmajor(q), _rowmajor(k), _rowmajor(v)
    first = None if state is None else torch.empty(shape, dtype=torch.float32, device=dev)
    n = _floats_of("tg_linear_attention_bwd_scratch_floats", dt, d)
    scratch = torch.empty(n, dtype=torch.float32, device=dev) if n else None
    _call(dev, "tg_linear_attention_bwd", dt, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), do.data_ptr(), _STRIDES.pack(*do.stride()[:3]),
          log_decay.data_ptr(), _ptr(lengths), _ptr(state), _ptr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(first), _ptr(scratch))
    return dq, dk, dv, first


def linear_attention_step(q, k, v, log_decay, state, scale=None):
    """The next token of every sequence: q (B, H, Dk), k (B, Hk, Dk), v (B, Hk, Dv) -> o (B, H, Dv); `state`, float32 (B, H, Dk, Dv) and
    contiguous, is updated in place (and counts as modified for autograd).  The single-token form of linear_attention (as generator.recurrent_step is
    of generator.recurrent); it has no gradient."""
    _no_tangents(q, k, v, log_decay, state)
    if _wants_grad(q, k, v, state):
        _fail("linear_attention_step has no gradient: call it under torch.no_grad(), or linear_attention with one token")
    dt, d, (B, _, H, DK, DV), q, k, v, log_decay = _desc(q, k, v, log_decay, scale, True)
    _f32(q, state, "state", (B, H, DK, DV))
    if not state.is_contiguous():
        _fail("state is updated in place: it must be contiguous")
    o = torch.empty((B, H, DV), dtype=q.dtype, device=q.device)
    _call(q.device, "tg_linear_attention_step", dt, d, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), o.data_ptr(), state.data_ptr())
    torch.autograd.graph.increment_version(state)   # (written through its address: a backward pass that saved the old values is to notice)
    return o

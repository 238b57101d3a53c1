"""The sequence-layer operators (ops.rms_norm, ops.dropout, ops.linear_attention and their explicit and single-token forms) against plain
64-bit statements of the same formulas on the same inputs.

Tolerances, from the arithmetic: a stored result is off by half a step of its type (HALF, relative to the value; fp16 also by half its
smallest step, 2^-25).  Sums in fp32 are off by at most (number of additions one after the other) x 2^-24 of the sum of the terms'
magnitudes; the operators add at most ADDS in a row before they join partial sums in a tree.  The bounds of linear_attention's random cases leave
room for scores and states of two bf16 halves beside 16-bit inputs: 2^-16 of the magnitudes for each split on the way of a term (at most 4: weight,
state, fp16's own two halves); the cases of whole numbers and of single terms hold them to fp32's 24 bits."""
import ctypes as C
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
import pytorch_tecogan_amd  # noqa: E402,F401
from pytorch_tecogan_amd import _lib as L  # noqa: E402
from pytorch_tecogan_amd import ops  # noqa: E402

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
HALF = {t: torch.finfo(t).eps / 2 for t in (F32, BF16, F16)}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -25}
U = 2.0 ** -24
DEV = "cuda"


def close(got, want, dt, magnitude, units, what=""):
    """|got - want| <= half a step of dt + units * 2^-24 * magnitude, everywhere; non-finite values in the same places"""
    got, want = got.double().cpu(), want.double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), f"{what}: non-finite values in other places"
    bound = HALF[dt] * (1 + 2.0 ** -7) * want.abs() + TINY[dt] + units * U * magnitude.double().cpu().expand_as(want)
    over = ((got - want).abs() - bound)[fine]
    assert not over.numel() or float(over.max()) <= 0, f"{what}: over the bound by {float(over.max()):.3e} ({dt})"


def randn(*shape, dt=F32, seed=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(dt).to(DEV)


# ------------------------------------------------------------------------------------------------------------ RMS norm
ADDS = 80   # additions in a row: up to 64 in a lane's registers, 6 + 2 across lanes and waves, and the roundings of the formula itself
NORM_SHAPES = [(1, 1), (1, 64), (3, 64), (5, 17), (257, 64), (130, 96), (33, 128), (9, 255), (4, 1000), (7, 1001), (3, 2048), (2, 4097), (2, 8192),
               (2, 8200), (2, 8201), (1025, 64)]


def norm_oracle(s, weight, eps):
    s = s.double()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + eps)
    return s * rstd * (1 if weight is None else weight.double()), rstd[..., 0]


def check_norm(x, res, wt, dy, ds, eps=1e-5):
    """forward, statistics and gradients of one call, on the tensors as they are (views included)"""
    dt = x.dtype
    out = ops.rms_norm(x, wt, residual=res, eps=eps, stats=True)
    total = x.double() if res is None else x.double() + res.double()
    y64, rstd64 = norm_oracle(total, wt, eps)
    close(out[0], y64, dt, y64.abs(), ADDS, "y")
    close(out[-1], rstd64, F32, rstd64, ADDS, "rstd")
    if res is not None:
        close(out[1], total, dt, x.double().abs() + res.double().abs(), 1, "s")
    rstd = out[-1].double()[..., None]
    dx, dw = ops.rms_norm_backward(dy, x, out[-1], wt, residual=res, ds=ds)
    xh = total * rstd
    g = dy.double() * (1 if wt is None else wt.double())
    dx64 = rstd * (g - xh * (g * xh).mean(-1, keepdim=True))
    mag = rstd * (g.abs() + xh.abs() * (g * xh).abs().mean(-1, keepdim=True))
    if ds is not None:
        dx64, mag = dx64 + ds.double(), mag + ds.double().abs()
    close(dx, dx64, dt, mag, ADDS, "dx")
    terms = (dy.double() * xh).reshape(-1, x.shape[-1])
    close(dw, terms.sum(0), F32, terms.abs().sum(0), ADDS, "dweight")
    assert ops.rms_norm_backward(dy, x, out[-1], wt, dweight=False)[1] is None


def check_e4m3(x, res, w, eps=1e-6):
    out = ops.rms_norm_e4m3(x, w, residual=res, eps=eps)
    total = x.double() if res is None else x.double() + res.double()
    y64, _ = norm_oracle(total, w, eps)
    scale = y64.abs().amax(-1) / 448
    close(out[1], scale, F32, scale, ADDS, "scale")
    got = out[0].float().double() * out[1].double()[..., None]
    # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale below the normal range
    bound = y64.abs() * (2.0 ** -4 + 2 * ADDS * U) + scale[..., None] * 2.0 ** -10 * (1 + ADDS * U)
    assert bool(((got - y64).abs() <= bound).all())
    assert bool((out[0].float().abs().amax(-1) == 448.0).all())   # the row's largest value takes the whole range
    if res is not None:
        close(out[2], total, x.dtype, x.double().abs() + res.double().abs(), 1, "s")


@pytest.mark.parametrize("rows,channels", NORM_SHAPES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_rms_norm_and_gradient(rows, channels, dt):
    x, r = randn(rows, channels, dt=dt, seed=1), randn(rows, channels, dt=dt, seed=2)
    w = 1 + 0.3 * randn(channels, seed=3)
    dy, ds = randn(rows, channels, dt=dt, seed=4), randn(rows, channels, dt=dt, seed=5)
    for res, wt in ((None, w), (r, w), (r, None)):
        for d in (None, ds):
            check_norm(x, res, wt, dy, d)


@pytest.mark.parametrize("rows,channels", NORM_SHAPES)
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_rms_norm_e4m3(rows, channels, dt):
    x, r, w = randn(rows, channels, dt=dt, seed=11), randn(rows, channels, dt=dt, seed=12), 1 + 0.3 * randn(channels, seed=13)
    for res in (None, r):
        check_e4m3(x, res, w)


def test_rms_norm_gradient_against_differences():
    x, r, w, dy, ds = (randn(3, 24, seed=i).double().cpu() for i in range(20, 25))
    w = w[0]
    gpu = [t.float().to(DEV) for t in (x, r, w, dy, ds)]
    out = ops.rms_norm(gpu[0], gpu[2], residual=gpu[1], eps=1e-3, stats=True)
    dx, dw = ops.rms_norm_backward(gpu[3], gpu[0], out[2], gpu[2], residual=gpu[1], ds=gpu[4])
    x, r, w, dy, ds = (t.float().double() for t in (x, r, w, dy, ds))

    def loss(x, w):
        s = x + r
        return float((norm_oracle(s, w, 1e-3)[0] * dy).sum() + (s * ds).sum())

    h = 1e-5
    for got, t, f in ((dx, x, lambda t: loss(t, w)), (dw, w, lambda t: loss(x, t))):
        for i in range(0, t.numel(), 5):
            a, b = t.clone(), t.clone()
            a.view(-1)[i] += h
            b.view(-1)[i] -= h
            # central differences in 64 bits: h^2 of the third derivative (<= 1e2 here), 2^-53 / h of the value; the kernel: fp32
            assert abs(float(got.reshape(-1)[i]) - (f(a) - f(b)) / (2 * h)) < 2e-5


def test_rms_norm_autograd_matches_the_explicit_form():
    for dt in (F32, BF16):
        x, r, w = randn(4, 5, 64, dt=dt, seed=31), randn(4, 5, 64, dt=dt, seed=32), 1 + 0.1 * randn(64, seed=33)
        dy, ds = randn(4, 5, 64, dt=dt, seed=34), randn(4, 5, 64, dt=dt, seed=35)
        y0, s0, rstd = ops.rms_norm(x, w, residual=r, stats=True)
        dx0, dw0 = ops.rms_norm_backward(dy, x, rstd, w, residual=r, ds=ds)
        xl, rl, wl = (t.clone().requires_grad_() for t in (x, r, w))
        y, s = ops.rms_norm(xl, wl, residual=rl)
        assert torch.equal(y, y0) and torch.equal(s, s0)
        gx, gr, gw = torch.autograd.grad([y, s], [xl, rl, wl], [dy, ds])
        assert torch.equal(gx, dx0) and torch.equal(gr, dx0) and torch.equal(gw, dw0)
        y, s = ops.rms_norm(xl, wl, residual=rl)           # the sum alone
        gx, = torch.autograd.grad([s], [xl], [ds])
        assert torch.equal(gx, ds)
        y = ops.rms_norm(xl, None)                         # no residual, no weight; an expanded gradient
        y.sum().backward()
        want, _ = ops.rms_norm_backward(torch.ones_like(x), x, ops.rms_norm(x, stats=True)[1])
        assert torch.equal(xl.grad, want)


def test_rms_norm_strides_and_alignment():
    base = randn(6, 10, 96, dt=BF16, seed=41)
    w = 1 + 0.1 * randn(96, seed=42)
    for view in (lambda t: t[..., :51], lambda t: t[..., 1:52], lambda t: t[..., 8:72], lambda t: t[:, 3], lambda t: t.transpose(0, 1),
                 lambda t: t[:, ::2, 3:67], lambda t: t[:1].expand(4, 10, 96), lambda t: t.transpose(1, 2)[..., :10]):
        x = view(base)
        c = x.shape[-1]
        check_norm(x, None, w[:c], x, None)
        check_norm(x, x.flip(0), w[:c], x.flip(-1), x)
        check_norm(x.contiguous(), x, w[1:c + 1] if c < 96 else w, x, x.flip(0))   # one unaligned operand among aligned ones
        check_e4m3(x, x.flip(0), w[:c])
    # a storage that starts off 16 bytes
    flat = randn(64 * 9 + 3, dt=F16, seed=43)
    check_norm(flat[3:].view(9, 64), flat[1:-2].view(9, 64), None, flat[:-3].view(9, 64), flat[3:].view(9, 64))


def test_rms_norm_rows_of_zeros_infinities_and_nan():
    x = randn(8, 64, dt=BF16, seed=51)
    x[1] = 0
    x[2, 5] = math.inf
    x[3, 7] = math.nan
    x[4] = 1e-30
    x[5] = torch.finfo(BF16).max
    y, rstd = ops.rms_norm(x, eps=1e-6, stats=True)
    clean = ops.rms_norm(torch.where(torch.isfinite(x), x, torch.zeros_like(x)), eps=1e-6)
    for row in (0, 1, 4, 6, 7):
        assert torch.equal(y[row], clean[row])
    assert not y[1].any()
    assert bool(torch.isnan(y[2, 5])) and not y[2, :5].any() and bool(torch.isnan(y[3]).all())
    q, scale = ops.rms_norm_e4m3(x, eps=1e-6)
    assert not q[1].float().any() and float(scale[1]) == float(np.float32(2.0 ** -100 / 448))
    assert bool(torch.isnan(scale[3])) and bool(torch.isnan(scale[2])) and bool(torch.isfinite(scale[[0, 1, 4, 6, 7]]).all())
    assert float(q[4].float().abs().min()) == 448.0
    # the gradient of the zero row: rstd = eps^-1/2, xhat = 0
    dy = randn(8, 64, dt=BF16, seed=52)
    dx, _ = ops.rms_norm_backward(dy, x, rstd, dweight=False)
    close(dx[1], dy[1].double() * rstd[1].double(), BF16, dy[1].double().abs() * 1e3, 2, "zero row")


def test_rms_norm_nothing_and_determinism():
    w = randn(64)
    assert ops.rms_norm(torch.empty(0, 64, device=DEV), w).shape == (0, 64)
    q, scale, s = ops.rms_norm_e4m3(torch.empty(0, 64, device=DEV, dtype=BF16), residual=torch.empty(0, 64, device=DEV, dtype=BF16))
    assert q.shape == s.shape == (0, 64) and scale.shape == (0,)
    dx, dw = ops.rms_norm_backward(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV), torch.empty(0, device=DEV), w)
    assert dx.shape == (0, 64) and dw.shape == (64,) and not dw.any()
    x, dy = randn(5000, 64, dt=BF16, seed=61), randn(5000, 64, dt=BF16, seed=62)
    _, rstd = ops.rms_norm(x, stats=True)
    first = ops.rms_norm_backward(dy, x, rstd, w)
    for _ in range(3):
        again = ops.rms_norm_backward(dy, x, rstd, w)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


# ------------------------------------------------------------------------------------------------------------- dropout
def philox_words(n, seed, step, layer):
    """the generator in numpy's 64-bit integers"""
    low = np.uint64(0xffffffff)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [block & low, block >> np.uint64(32), np.full_like(block, layer), np.full_like(block, step & 0xffffffff)]
    seed &= 0xffffffffffffffff
    k0, k1 = seed & 0xffffffff, seed >> 32
    for r in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        x0, x1 = np.uint64((k0 + r * 0x9E3779B9) & 0xffffffff), np.uint64((k1 + r * 0xBB67AE85) & 0xffffffff)
        c = [(b >> np.uint64(32)) ^ c[1] ^ x0, b & low, (a >> np.uint64(32)) ^ c[3] ^ x1, a & low]
    return np.stack(c, axis=1).reshape(-1)[:n]


def keep_mask(shape, p, seed, step, layer):
    n = int(np.prod(shape))
    return torch.from_numpy(philox_words(n, seed, step, layer) >= np.uint64(math.floor(p * 2.0 ** 32 + 0.5))).view(*shape)


def test_generator_known_answers():
    """the generator's published test vectors (Random123's known-answer file: counter and key all zeros; all ones)"""
    assert [int(w) for w in philox_words(4, 0, 0, 0)] == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]


@pytest.mark.parametrize("n", [1, 3, 4, 7, 8, 9, 255, 2048, 2049, 100003])
@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_dropout_mask_and_values(n, dt):
    for p, seed, step, layer, with_res in ((0.1, 1234567890123, 5, 0, True), (0.5, -7, 2 ** 32 + 9, 3, False), (0.0, 1, 0, 0, True),
                                           (0.999, 2 ** 62 + 1, 2 ** 31, 2 ** 31 - 1, False)):
        x, res, dy = randn(n, dt=dt, seed=1) + 8, randn(n, dt=dt, seed=2), randn(n, dt=dt, seed=3) + 8   # (x away from zero: a zero is a dropped one)
        rng = ops.dropout_rng(seed, DEV, step)
        keep = keep_mask((n,), p, seed, step, layer).to(DEV)
        y = ops.dropout(x, p, rng, layer=layer, residual=res if with_res else None)
        want = torch.where(keep, x.double() / (1 - p), torch.zeros((), device=DEV, dtype=torch.float64))
        mag = want.abs()
        if with_res:
            want, mag = want + res.double(), mag + res.double().abs()
        else:
            assert torch.equal(y != 0, keep)
        close(y, want, dt, mag, 4, "y")
        dx = ops.dropout_backward(dy, p, rng, layer=layer)
        assert torch.equal(dx != 0, keep)
        close(dx, torch.where(keep, dy.double() / (1 - p), 0.0), dt, dy.double().abs() / (1 - p), 4, "dx")
        assert rng.tolist() == [seed, step]


def test_dropout_dropped_infinities_and_nan_are_gone():
    x = torch.full((4096,), math.inf, device=DEV, dtype=BF16)
    x[1::2] = math.nan
    keep = keep_mask((4096,), 0.5, 9, 0, 1).to(DEV)
    y = ops.dropout(x, 0.5, ops.dropout_rng(9, DEV), layer=1)
    assert not y[~keep].any() and not torch.isfinite(y[keep]).any()


def test_dropout_strides_types_and_independence():
    x = randn(40, 96, seed=5)
    rng = ops.dropout_rng(77, DEV)
    for view in (x.t(), x[:, 1:52], x[::3], x[:1].expand(6, 96), x.reshape(-1)[3:]):
        assert torch.equal(ops.dropout(view, 0.3, rng), ops.dropout(view.contiguous(), 0.3, rng))
        assert torch.equal(ops.dropout(view, 0.3, rng, residual=view), ops.dropout(view.contiguous(), 0.3, rng, residual=view.contiguous()))
    one = torch.ones(1 << 20, device=DEV)
    masks = [ops.dropout(one.to(t), 0.25, rng).float() != 0 for t in (F32, BF16, F16)]
    assert torch.equal(masks[0], masks[1]) and torch.equal(masks[0], masks[2])
    # other layers, steps and seeds: other masks, each with its share of drops (6 standard deviations of a binomial) and unrelated to the first
    for other in (ops.dropout(one, 0.25, rng, layer=1), ops.dropout(one, 0.25, ops.dropout_rng(77, DEV, 1)), ops.dropout(one, 0.25, ops.dropout_rng(78, DEV))):
        m = other != 0
        n = one.numel()
        assert abs(float(m.float().mean()) - 0.75) < 6 * math.sqrt(0.75 * 0.25 / n)
        both = float((m & masks[0]).float().mean())
        assert abs(both - 0.5625) < 6 * math.sqrt(0.5625 * 0.4375 / n)


def test_dropout_autograd():
    x, r = randn(33, 7, seed=1).requires_grad_(), randn(33, 7, seed=2).requires_grad_()
    rng = ops.dropout_rng(5, DEV)
    dy = randn(33, 7, seed=3)
    y = ops.dropout(x, 0.4, rng, layer=2, residual=r)
    gx, gr = torch.autograd.grad(y, [x, r], dy)
    assert torch.equal(gx, ops.dropout_backward(dy, 0.4, rng, layer=2)) and torch.equal(gr, dy)
    y = ops.dropout(x, 0.4, rng)
    rng[1] += 1   # the state moved before the backward pass: refused, not another mask
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_dropout_past_32_bit_indices():
    """4 elements behind index 2^32 (8.6 GB of bf16): the counter's high word counts"""
    n = (1 << 32) + 4
    x = torch.ones(n, device=DEV, dtype=BF16)
    y = ops.dropout(x, 0.5, ops.dropout_rng(3, DEV))
    del x
    # words of block 2^30: counter (2^30, 0, ..): 32-bit element arithmetic would have wrapped to block 0
    tail = y[-4:].float().cpu() != 0
    first = y[:4].float().cpu() != 0
    c = philox_block(1 << 30, 3)
    assert torch.equal(tail, torch.tensor([w >= 1 << 31 for w in c])), (tail, c)
    assert torch.equal(first, torch.tensor([int(w) >= 1 << 31 for w in philox_words(4, 3, 0, 0)]))


def philox_block(block, seed, step=0, layer=0):
    c, k = [block & 0xffffffff, block >> 32, layer, step], [seed & 0xffffffff, seed >> 32]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(b >> 32) ^ c[1] ^ k[0], b & 0xffffffff, (a >> 32) ^ c[3] ^ k[1], a & 0xffffffff]
        k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
    return c


# ---------------------------------------------------------------------------------------------------- linear attention
def attention_oracle(q, k, v, log_decay, scale, state, lengths, do=None, dstate=None):
    """the sums over pairs of tokens in 64 bits on the CPU -> ({name: value}, {name: sum of the terms' magnitudes})"""
    q, k, v, a = (t.double().cpu() for t in (q, k, v, log_decay))
    B, T, H, DK = q.shape
    HK, DV = k.shape[2], v.shape[3]
    G = H // HK
    live = torch.ones(B, T, dtype=torch.bool) if lengths is None else torch.arange(T)[None] < lengths.cpu().long().clamp(0, T)[:, None]
    n = live.sum(1)
    t = torch.arange(T).double()
    gap = t[:, None] - t[None]
    power = lambda e: torch.where(e == 0, 1.0, torch.exp(a.view(-1, *([1] * e.dim())) * e))   # noqa: E731  (0 * -inf)
    w = torch.where(gap >= 0, power(gap.clamp_min(0)), 0.0)[None] * scale                       # (1, H, T, T)
    since = torch.stack([power((t + 1))] * B)[..., None] if T else torch.zeros(B, H, 0, 1, dtype=torch.float64)
    left = torch.stack([power((int(m) - 1 - t).clamp_min(0)) for m in n])[..., None]
    last = torch.stack([power(torch.tensor(float(m))) for m in n])[..., None, None].double()
    cut = lambda x: torch.where(live[..., None, None], x, 0.0).permute(0, 2, 1, 3)              # noqa: E731
    S0 = torch.zeros(B, H, DK, DV, dtype=torch.float64) if state is None else state.double().cpu()
    res = []
    for f in (lambda x: x, torch.abs):
        qq, kk, vv, ss = f(cut(q)), f(cut(k)).repeat_interleave(G, 1), f(cut(v)).repeat_interleave(G, 1), f(S0)
        lv = live[:, None, :, None].double()
        score = (qq @ kk.transpose(2, 3)) * w
        o = (score @ vv + scale * (qq * since) @ ss) * lv
        out = {"o": o.permute(0, 2, 1, 3), "state": (kk * left * lv).transpose(2, 3) @ vv + last * ss}
        if do is not None:
            dd = f(cut(do.double().cpu()))
            dS = f(torch.zeros_like(S0) if dstate is None else dstate.double().cpu())
            ds = (dd @ vv.transpose(2, 3)) * w
            dq = (ds @ kk + scale * since * (dd @ ss.transpose(2, 3))) * lv
            dk = ds.transpose(2, 3) @ qq + left * lv * (vv @ dS.transpose(2, 3))
            dv = score.transpose(2, 3) @ dd + left * lv * (kk @ dS)
            share = lambda x: x.view(B, HK, G, T, x.shape[3]).sum(2).permute(0, 2, 1, 3)        # noqa: E731
            out.update(dq=dq.permute(0, 2, 1, 3), dk=share(dk), dv=share(dv),
                       dstate=last * dS + scale * (qq * since * lv).transpose(2, 3) @ dd)
        res.append(out)
    return res


def attention_units(dt, T, D):
    """fp32 additions one after the other (tokens and channels), and four splits of 2^-16 = 256 x 2^-24 beside 16-bit inputs"""
    return T + D + 64 + (0 if dt == F32 else 4 * 256)


def attention_inputs(B, T, H, HK, DK, DV, dt, seed=0):
    q, k, v, do = (randn(*s, dt=dt, seed=seed + i) for i, s in enumerate(((B, T, H, DK), (B, T, HK, DK), (B, T, HK, DV), (B, T, H, DV))))
    state, dstate = randn(B, H, DK, DV, seed=seed + 5), randn(B, H, DK, DV, seed=seed + 6)
    decay = -torch.tensor([0.0, 0.7, 0.05, 2.0 ** -7, 3.0, 2.0 ** -12, 0.3, 0.011][:H], device=DEV)
    return q, k, v, do, state, dstate, decay


def attention_case(B, T, H, HK, DK, DV, dt, lengths=None, with_state=True, scale=None, seed=0):
    q, k, v, do, state, dstate, decay = attention_inputs(B, T, H, HK, DK, DV, dt, seed)
    if not with_state:
        state = dstate = None
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device=DEV)
    sc = DK ** -0.5 if scale is None else scale
    o, last = ops.linear_attention(q, k, v, decay, scale=scale, state=state, lengths=ln)
    dq, dk, dv, first = ops.linear_attention_backward(do, q, k, v, decay, scale=scale, state=state, lengths=ln, dstate=dstate)
    want, mag = attention_oracle(q, k, v, decay, sc, state, ln, do, dstate)
    units = attention_units(dt, T, max(DK, DV)) * (H // HK)
    for name, got, t in (("o", o, dt), ("state", last, F32), ("dq", dq, dt), ("dk", dk, dt), ("dv", dv, dt), ("dstate", first, F32)):
        if got is not None:
            close(got, want[name], t, mag[name], units, name)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T", [1, 2, 10, 15, 16, 17, 31, 33, 63, 64, 65, 100, 127, 129, 200, 257])
def test_attention_lengths(T, dt):
    attention_case(2, T, 3, 3, 16, 16, dt)
    attention_case(1, T, 2, 1, 64, 64, dt, with_state=T % 2 == 0)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("DK,DV", [(1, 1), (3, 5), (8, 16), (16, 8), (17, 31), (32, 32), (32, 64), (40, 56), (64, 32), (65, 64), (64, 96), (96, 128),
                                   (127, 1), (128, 128)])
def test_attention_head_sizes(DK, DV, dt):
    attention_case(2, 37, 2, 2, DK, DV, dt, lengths=[37, 20])
    attention_case(1, 90, 2, 1, DK, DV, dt, seed=9)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("H,HK", [(1, 1), (4, 4), (4, 2), (6, 2), (3, 1), (8, 1)])
def test_attention_shared_heads(H, HK, dt):
    attention_case(2, 50, H, HK, 32, 16, dt, lengths=[50, 33])


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_attention_ragged_batches(dt):
    attention_case(6, 70, 2, 2, 32, 32, dt, lengths=[0, 1, 16, 64, 69, 70])
    attention_case(4, 130, 4, 2, 64, 48, dt, lengths=[0, 65, 129, 130], with_state=False)
    attention_case(3, 20, 2, 1, 16, 16, dt, lengths=[-3, 20, 1000])   # clamped to 0 .. T


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,H,D", [(1, 1500, 2, 64), (1, 4097, 1, 32), (3, 1030, 2, 128)])
def test_attention_long(B, T, H, D, dt):
    attention_case(B, T, H, H, D, D, dt)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("DK,DV", [(16, 16), (24, 40), (17, 31), (64, 128)])
def test_attention_segments_of_ragged_batches(DK, DV, dt):
    """lengths that end in the first segment, in a later one, at its border, at none"""
    attention_case(4, 777, 4, 2, DK, DV, dt, lengths=[777, 300, 64, 0])
    attention_case(1, 1029, 1, 1, DK, DV, dt, with_state=False)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
def test_attention_nonfinite_tokens_across_segments(dt):
    """the segments in front of an infinity give the same bits as without it; what follows is not finite"""
    q, k, v, _, state, _, decay = attention_inputs(2, 640, 2, 2, 32, 32, dt)
    o, last = ops.linear_attention(q, k, v, decay, state=state)
    k[0, 333, 0, 5] = math.inf
    o1, last1 = ops.linear_attention(q, k, v, decay, state=state)
    assert torch.equal(o1[0, :333], o[0, :333]) and torch.equal(o1[1], o[1]) and torch.equal(o1[0, :, 1], o[0, :, 1])
    assert torch.equal(last1[1], last[1]) and torch.equal(last1[0, 1], last[0, 1])
    assert not o1[0, 333:, 0].isfinite().all(-1).any() and not last1[0, 0, 5].isfinite().any()


def test_attention_many_short_sequences():
    attention_case(700, 10, 4, 4, 16, 16, BF16)
    attention_case(300, 3, 4, 2, 16, 24, F32, lengths=[i % 4 for i in range(300)])


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("DK,DV", [(64, 64), (32, 64), (40, 24), (48, 16)])
def test_attention_many_wide_heads(DK, DV, dt):
    """enough sequences for slices of 32 columns, whole and in segments"""
    B = 600
    attention_case(B, 70, 2, 1, DK, DV, dt, lengths=[(17 * i) % 71 for i in range(B)])
    attention_case(150, 40, 4, 4, DK, DV, dt)
    attention_case(66, 1100, 4, 4, DK, DV, dt, lengths=[1100 - (37 * i) % 1101 for i in range(66)])


def test_attention_scale_and_extreme_decays():
    attention_case(2, 40, 3, 3, 24, 24, BF16, scale=1.0)
    q, k, v, do, state, dstate, _ = attention_inputs(2, 40, 3, 3, 24, 24, F32)
    decay = torch.tensor([-math.inf, -200.0, 0.0], device=DEV)   # no memory at all; underflowing powers; a memory that does not fade
    o, last = ops.linear_attention(q, k, v, decay, state=state)
    got = ops.linear_attention_backward(do, q, k, v, decay, state=state, dstate=dstate)
    want, mag = attention_oracle(q, k, v, decay, 24 ** -0.5, state, None, do, dstate)
    for name, g in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, last, *got)):
        close(g, want[name], F32, mag[name], attention_units(F32, 40, 24), name)


def test_attention_values_past_the_range_of_fp16():
    """scores and states beyond 65504 with fp16 inputs, and a result that fits again through the scale"""
    q, k, v = (randn(1, 80, 2, 64, dt=F16, seed=i) * 100 for i in range(3))
    decay = torch.tensor([0.0, -0.1], device=DEV)
    o, last = ops.linear_attention(q, k, v, decay, scale=1e-6)
    want, mag = attention_oracle(q, k, v, decay, 1e-6, None, None)
    assert float(want["state"].abs().max()) > 65504
    close(o, want["o"], F16, mag["o"], attention_units(F16, 80, 64), "o")
    close(last, want["state"], F32, mag["state"], attention_units(F16, 80, 64), "state")


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("which", ["q", "k", "v"])
def test_attention_nonfinite_tokens_reach_no_earlier_one(which, value, dt):
    for T, at, D in ((40, 21, 16), (150, 77, 64)):
        q, k, v, do, state, dstate, decay = attention_inputs(1, T, 2, 2, D, D, dt, seed=3)
        o, _ = ops.linear_attention(q, k, v, decay, state=state)
        bad = {"q": q, "k": k, "v": v}
        bad[which] = bad[which].clone()
        bad[which][0, at, 1, 5] = value
        p, _ = ops.linear_attention(bad["q"], bad["k"], bad["v"], decay, state=state)
        assert torch.equal(p[:, :at], o[:, :at]) and torch.equal(p[:, :, 0], o[:, :, 0])
        assert not bool(torch.isfinite(p[0, at, 1]).all())
        if which == "q":
            assert torch.equal(p[:, at + 1:], o[:, at + 1:])


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("which", ["q", "k", "v", "do"])
def test_attention_nonfinite_tokens_in_the_gradients(which, value, dt):
    """dq_i takes from do_i and from k, v up to i; dk_j from v_j and from q, do at j and behind it; dv_j from k_j and from q, do there"""
    for T, at, D in ((10, 6, 16), (16, 3, 20), (40, 21, 17), (150, 77, 64)):
        q, k, v, do, state, dstate, decay = attention_inputs(1, T, 2, 2, D, D, dt, seed=3)
        decay = torch.tensor([-0.05, -0.2], device=DEV)
        good = ops.linear_attention_backward(do, q, k, v, decay, state=state, dstate=dstate)
        bad = dict(q=q, k=k, v=v, do=do)
        bad[which] = bad[which].clone()
        bad[which][0, at, 1, 5] = value
        got = ops.linear_attention_backward(bad["do"], bad["q"], bad["k"], bad["v"], decay, state=state, dstate=dstate)
        clean = {"q": (range(T), range(at + 1, T), range(at + 1, T)), "do": ([i for i in range(T) if i != at], range(at + 1, T), range(at + 1, T)),
                 "k": (range(at), range(T), [j for j in range(T) if j != at]), "v": (range(at), [j for j in range(T) if j != at], range(T))}[which]
        for name, a, b, rows in zip(("dq", "dk", "dv"), got, good, clean):
            rows = list(rows)
            assert torch.equal(a[:, rows], b[:, rows]), (which, name, T)
            assert torch.equal(a[:, :, 0], b[:, :, 0]), (which, name, T)
        touched = {"q": (1, 2), "do": (0, 1, 2), "k": (0, 2), "v": (0, 1)}[which]
        for i in touched:
            assert not bool(torch.isfinite(got[i][0, at, 1]).all())


def test_attention_does_not_read_behind_the_lengths():
    for dt in (F32, BF16, F16):
        q, k, v, do, state, dstate, decay = attention_inputs(3, 90, 2, 2, 32, 32, dt, seed=4)
        ln = torch.tensor([0, 17, 64], dtype=torch.int32, device=DEV)
        base = ops.linear_attention(q, k, v, decay, state=state, lengths=ln) + ops.linear_attention_backward(
            do, q, k, v, decay, state=state, lengths=ln, dstate=dstate)
        for i, m in enumerate(ln.tolist()):
            for t in (q, k, v, do):
                t[i, m:] = math.nan
        bad = ops.linear_attention(q, k, v, decay, state=state, lengths=ln) + ops.linear_attention_backward(
            do, q, k, v, decay, state=state, lengths=ln, dstate=dstate)
        for a, b in zip(base, bad):
            assert torch.equal(a, b)
        for i, m in enumerate(ln.tolist()):
            for t in (bad[0], *bad[2:5]):
                assert not t[i, m:].any()


def test_attention_nothing():
    decay = torch.zeros(2, device=DEV)
    e = lambda *s: torch.empty(*s, device=DEV, dtype=BF16)   # noqa: E731
    state = randn(3, 2, 16, 8)
    o, last = ops.linear_attention(e(3, 0, 2, 16), e(3, 0, 2, 16), e(3, 0, 2, 8), decay, state=state)
    assert o.shape == (3, 0, 2, 8) and torch.equal(last, state)
    o, last = ops.linear_attention(e(3, 0, 2, 16), e(3, 0, 1, 16), e(3, 0, 1, 8), decay)
    assert not last.any()
    g = ops.linear_attention_backward(e(3, 0, 2, 8), e(3, 0, 2, 16), e(3, 0, 1, 16), e(3, 0, 1, 8), decay, state=state, dstate=2 * state)
    assert g[0].shape == (3, 0, 2, 16) and torch.equal(g[3], 2 * state)
    assert ops.linear_attention_backward(e(3, 0, 2, 8), e(3, 0, 2, 16), e(3, 0, 1, 16), e(3, 0, 1, 8), decay)[3] is None
    o, last = ops.linear_attention(e(0, 5, 2, 16), e(0, 5, 2, 16), e(0, 5, 2, 8), decay)
    assert o.shape == (0, 5, 2, 8) and last.shape == (0, 2, 16, 8)
    assert ops.linear_attention_step(e(0, 2, 16), e(0, 2, 16), e(0, 2, 8), decay, torch.empty(0, 2, 16, 8, device=DEV)).shape == (0, 2, 8)


def test_attention_strides():
    """q, k, v as slices of one packed tensor, token-major and head-major, odd offsets; expanded gradients"""
    B, T, H, D = 2, 45, 3, 24
    decay = -torch.tensor([0.1, 0.5, 0.02], device=DEV)
    for dt in (F32, BF16):
        packed = randn(B, T, H, 3 * D + 2, dt=dt, seed=1)
        packed2 = randn(B, H, T, 3 * D, dt=dt, seed=2)
        do = randn(B, T, H, D, dt=dt, seed=3)
        for q, k, v in ((packed[..., :D], packed[..., D:2 * D], packed[..., 2 * D:3 * D]), (packed[..., 1:D + 1], packed[..., D + 1:2 * D + 1], packed[..., 2 * D + 2:]),
                        tuple(packed2.transpose(1, 2)[..., i * D:(i + 1) * D] for i in range(3)),
                        (packed[..., :D], packed[:1, :, :, :D].expand(B, T, H, D), packed.transpose(0, 1)[:2, :2].repeat(1, 23, 1, 1)[:, :T, :, :D])):
            c = [t.contiguous() for t in (q, k, v)]
            for a, b in zip(ops.linear_attention(q, k, v, decay), ops.linear_attention(*c, decay)):
                assert torch.equal(a, b)
            for d in (do, do.transpose(1, 2).contiguous().transpose(1, 2), do[:, :1].expand(B, T, H, D), do[..., :1].expand(B, T, H, D)):
                got, want = ops.linear_attention_backward(d, q, k, v, decay), ops.linear_attention_backward(d.contiguous(), *c, decay)
                assert got[3] is None and all(torch.equal(a, b) for a, b in zip(got[:3], want[:3]))


def test_attention_autograd():
    B, T, H, HK, D = 2, 33, 4, 2, 16
    q, k, v, do, state, dstate, decay = attention_inputs(B, T, H, HK, D, D, BF16)
    want = ops.linear_attention_backward(do, q, k, v, decay, state=state, dstate=dstate)
    leaf = [t.clone().requires_grad_() for t in (q, k, v, state)]
    o, last = ops.linear_attention(*leaf[:3], decay, state=leaf[3])
    got = torch.autograd.grad([o, last], leaf, [do, dstate])
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    o, last = ops.linear_attention(*leaf[:3], decay, state=leaf[3])   # the state alone
    got = torch.autograd.grad([last], leaf, [dstate])
    for a, b in zip(got, ops.linear_attention_backward(torch.zeros_like(do), q, k, v, decay, state=state, dstate=dstate)):
        assert torch.equal(a, b)


def test_attention_gradient_against_differences():
    B, T, H, HK, DK, DV = 1, 19, 2, 1, 5, 4
    q, k, v, do, state, dstate, decay = attention_inputs(B, T, H, HK, DK, DV, F32, seed=7)
    g = ops.linear_attention_backward(do, q, k, v, decay, state=state, dstate=dstate)
    leaf = [t.double().cpu() for t in (q, k, v, state)]

    def loss(q, k, v, s):
        out, _ = attention_oracle(q, k, v, decay, DK ** -0.5, s, None)
        return float((out["o"] * do.double().cpu()).sum() + (out["state"] * dstate.double().cpu()).sum())

    h = 1e-4   # the loss is of third degree: differences are exact up to h^2 times its third derivative in one variable, which is zero
    for i, (t, got) in enumerate(zip(leaf, g)):
        for at in range(0, t.numel(), 7):
            a, b = [x.clone() for x in leaf], [x.clone() for x in leaf]
            a[i].view(-1)[at] += h
            b[i].view(-1)[at] -= h
            assert abs(float(got.reshape(-1)[at]) - (loss(*a) - loss(*b)) / (2 * h)) < 1e-4


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("B,H,HK,DK,DV", [(1, 1, 1, 1, 1), (2, 4, 2, 16, 16), (5, 3, 1, 17, 31), (3, 4, 4, 64, 64), (2, 2, 2, 128, 128), (1, 2, 1, 7, 100),
                                          (3, 2, 2, 33, 127), (70, 4, 4, 16, 16), (1, 2, 2, 128, 4), (1100, 4, 2, 16, 16), (1367, 3, 3, 15, 12),
                                          (600, 2, 1, 32, 64), (600, 2, 2, 5, 128), (9000, 2, 2, 8, 4)])
def test_attention_step(B, H, HK, DK, DV, dt):
    q, k, v, state = randn(B, H, DK, dt=dt, seed=1), randn(B, HK, DK, dt=dt, seed=2), randn(B, HK, DV, dt=dt, seed=3), randn(B, H, DK, DV, seed=4)
    decay = -torch.rand(H, generator=torch.Generator().manual_seed(5)).to(DEV)
    kk, vv = (t.double().repeat_interleave(H // HK, 1) for t in (k, v))
    old = state.double()
    want = old * decay.double().exp()[:, None, None] + kk[..., None] * vv[..., None, :]
    mag = old.abs() + (kk[..., None] * vv[..., None, :]).abs()
    o64 = DK ** -0.5 * (q.double()[..., None, :] @ want)[..., 0, :]
    omag = DK ** -0.5 * (q.double().abs()[..., None, :] @ mag)[..., 0, :]
    o = ops.linear_attention_step(q, k, v, decay, state)
    close(state, want, F32, mag, 4, "state")
    close(o, o64, dt, omag, DK + 16, "o")


def test_attention_step_strides_and_sequence_form():
    """steps over a packed tensor's tokens give what the whole sequence gives"""
    B, T, H, HK, D = 3, 21, 4, 2, 32
    packed = randn(B, T, 8 * D, dt=BF16, seed=1)
    q, k, v = packed[..., :4 * D].view(B, T, H, D), packed[..., 4 * D:6 * D].view(B, T, HK, D), packed[..., 6 * D:].view(B, T, HK, D)
    decay = -torch.tensor([0.5, 0.1, 0.02, 0.0], device=DEV)
    first = randn(B, H, D, D, seed=2)
    state = first.clone()
    o = torch.stack([ops.linear_attention_step(q[:, t], k[:, t], v[:, t], decay, state) for t in range(T)], dim=1)
    want, mag = attention_oracle(q, k, v, decay, D ** -0.5, first, None)
    close(o, want["o"], BF16, mag["o"], attention_units(F32, T, D), "steps")
    whole, last = ops.linear_attention(q, k, v, decay, state=first)
    close(whole, want["o"], BF16, mag["o"], attention_units(BF16, T, D), "whole")
    close(last, want["state"], F32, mag["state"], attention_units(F32, T, D), "last state")
    close(state, want["state"], F32, mag["state"], attention_units(F32, T, D), "state after the steps")


def test_attention_in_pieces():
    """a long sequence in pieces, the state carried and its gradient handed back"""
    q, k, v, do, state, dstate, decay = attention_inputs(1, 150, 2, 2, 32, 32, F32, seed=8)
    cut = [0, 40, 41, 104, 150]
    s, pieces, states = state, [], []
    for a, b in zip(cut, cut[1:]):
        states.append(s)
        o, s = ops.linear_attention(q[:, a:b], k[:, a:b], v[:, a:b], decay, state=s)
        pieces.append(o)
    want, mag = attention_oracle(q, k, v, decay, 32 ** -0.5, state, None, do, dstate)
    units = attention_units(F32, 150, 32)
    close(torch.cat(pieces, 1), want["o"], F32, mag["o"], units, "o")
    close(s, want["state"], F32, mag["state"], units, "state")
    d, grads = dstate, []
    for (a, b), s in reversed(list(zip(zip(cut, cut[1:]), states))):
        *g, d = ops.linear_attention_backward(do[:, a:b], q[:, a:b], k[:, a:b], v[:, a:b], decay, state=s, dstate=d)
        grads.insert(0, g)
    for i, name in enumerate(("dq", "dk", "dv")):
        close(torch.cat([g[i] for g in grads], 1), want[name], F32, mag[name], units, name)
    close(d, want["dstate"], F32, mag["dstate"], units, "dstate")


# ------------------------------------------------------------------------- scores, states and decays at fp32's own precision
# what each result sums, sum_j (a_i . b_j) c_j and a_i S: the names of a, b, c and of the state
ROLES = {"o": ("q", "k", "v", "state"), "dq": ("do", "v", "k", "state"), "dk": ("v", "do", "q", "dstate"), "dv": ("k", "q", "do", "dstate")}
EXACT_SHAPES = [(2, 16, 16), (9, 16, 24), (16, 32, 16), (16, 64, 64), (12, 128, 128), (14, 17, 9), (33, 16, 16), (40, 32, 32), (70, 64, 64), (50, 40, 24),
                (48, 128, 128), (61, 19, 33), (30, 65, 97), (1040, 64, 64), (1100, 21, 16)]


def exact_run(name, x, scale):
    """result `name` of the operands x, memory that does not fade"""
    decay = torch.zeros(x["q"].shape[2], device=DEV)
    x = {n: None if t is None else t.to(DEV) for n, t in x.items()}
    if name == "o":
        got = ops.linear_attention(x["q"], x["k"], x["v"], decay, scale=scale, state=x["state"])[0]
    else:
        got = ops.linear_attention_backward(x["do"], x["q"], x["k"], x["v"], decay, scale=scale, state=x["state"], dstate=x["dstate"])[("dq", "dk", "dv").index(name)]
    want, mag = attention_oracle(x["q"], x["k"], x["v"], decay, scale, x["state"], None, x["do"], x["dstate"])
    # the premise: whole numbers of units of `scale` that fp32 adds in any order
    assert float(mag[name].max()) < 2.0 ** 24 * scale and float(want[name].abs().max()) < 60000
    want = want[name].to(got.dtype).double()
    off = got.double().cpu() != want
    assert not off.any(), (name, int(off.sum()), float((got.double().cpu() - want).abs().max()))


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,DK,DV", EXACT_SHAPES)
def test_attention_scores_that_cancel(T, DK, DV, dt):
    """Neighbouring tokens b, b' that differ in the last places, with c' = -c: the scores are whole numbers below 2^20, their sums exact in fp32 in any
    order, and the results (small whole numbers, times a power of two) carry no rounding but their own.  Scores held to 16 bits are off by up
    to 8, more than most results."""
    for name, (a, b, c, _) in ROLES.items():
        g = torch.Generator().manual_seed(T)
        pick = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).to(F32)   # noqa: E731
        x = {n: torch.zeros(1, T, 2, DK if n in ("q", "k") else DV) for n in ("q", "k", "v", "do")}
        wide = x[a].shape[-1]
        for m, w in ((wide - 1, 2.0 ** 4), (wide // 2, 2.0 ** 2), (0, 1.0)):   # a b = 2^14 r + 2^7 r' + r''
            x[a][..., m] = w
        x[a] *= 2 * pick(0, 1, 1, T, 2, 1) - 1
        for at in sorted({0, T // 4 * 2, (T - 2) // 2 * 2}):
            for m, w in ((wide - 1, 2.0 ** 10), (wide // 2, 2.0 ** 5), (0, 1.0)):
                x[b][0, at, :, m] = x[b][0, at + 1, :, m] = w * pick(1, 31, 2)
            x[b][0, at + 1, :, 0] += pick(1, 3, 2)
            x[c][0, at] = pick(1, 2, *x[c].shape[2:])
            x[c][0, at + 1] = -x[c][0, at]
        y = {n: t.to(dt) for n, t in x.items()}
        assert all(torch.equal(y[n].float(), x[n]) for n in x)
        exact_run(name, dict(y, state=None, dstate=None), 2.0 ** -6)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,DK,DV", EXACT_SHAPES)
def test_attention_states_that_cancel(T, DK, DV, dt):
    """differences of neighbouring rows of a state of whole numbers below 2^22: small whole numbers, exact in fp32"""
    for name, (a, _, _, s) in ROLES.items():
        g = torch.Generator().manual_seed(T + 1)
        pick = lambda lo, hi, *s: torch.randint(lo, hi + 1, s, generator=g).to(F32)   # noqa: E731
        x = {n: torch.zeros(1, T, 2, DK if n in ("q", "k") else DV, dtype=dt) for n in ("q", "k", "v", "do")}
        x[a][..., 0], x[a][..., x[a].shape[-1] - 1] = 1, -1
        x[a] *= (2 * pick(0, 1, 1, T, 2, 1) - 1).to(dt)
        state = pick(1 << 20, 1 << 22, 1, 2, DK, DV)
        if x[a].shape[-1] == DK and a in ("q", "k"):
            state[:, :, -1] = state[:, :, 0] + pick(-3, 3, 1, 2, DV)
        else:
            state[..., -1] = state[..., 0] + pick(-3, 3, 1, 2, DK)
        exact_run(name, dict(x, state=state if s == "state" else torch.zeros_like(state), dstate=state if s == "dstate" else torch.zeros_like(state)), 1.0)


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("value", [math.inf, math.nan])
@pytest.mark.parametrize("T,D,off", [(10, 16, 0), (10, 17, 0), (40, 17, 0), (40, 32, 1), (150, 64, 0), (150, 63, 0), (40, 127, 0), (1100, 33, 0)])
def test_attention_nonfinite_channels_reach_no_other_channel(T, D, off, value, dt):
    """One channel of one token is not finite: an infinite v makes one column of o, of the state; an infinite k one row of the state and one
    channel of dq; q and do likewise in dk, dv and the state's gradient.  All others keep their bits - whatever the alignment and the head size."""
    x = dict(zip(("q", "k", "v", "do", "state", "dstate", "decay"), attention_inputs(1, T, 2, 2, D, D, dt, seed=3)))
    x["decay"] = torch.tensor([-0.05, -0.2], device=DEV)
    if off:   # (addresses off 16 bytes)
        for n in ("q", "k", "v", "do"):
            flat = torch.empty(x[n].numel() + off, dtype=dt, device=DEV)
            x[n] = flat[off:].view(x[n].shape).copy_(x[n])
    names = ("o", "state", "dq", "dk", "dv", "dstate")

    def run(x):
        o = ops.linear_attention(x["q"], x["k"], x["v"], x["decay"], state=x["state"])
        return dict(zip(names, (*o, *ops.linear_attention_backward(x["do"], x["q"], x["k"], x["v"], x["decay"], state=x["state"], dstate=x["dstate"]))))

    good = run(x)
    at, m = T // 2, 5
    # the results that have the non-finite channel as a channel of their own, and the dimension of it
    alone = {"q": (("dk", 3), ("dstate", 2)), "k": (("state", 2), ("dq", 3)), "v": (("o", 3), ("state", 3)), "do": (("dv", 3), ("dstate", 3))}
    for which in ("q", "k", "v", "do"):
        y = dict(x)
        y[which] = x[which].clone() if not off else torch.empty(x[which].numel() + off, dtype=dt, device=DEV)[off:].view(x[which].shape).copy_(x[which])
        y[which][0, at, 1, m] = value
        bad = run(y)
        others = [i for i in range(D) if i != m]
        for name, dim in alone[which]:
            keep = lambda t: t.index_select(dim, torch.tensor(others, device=DEV))   # noqa: E731
            assert torch.equal(keep(bad[name]), keep(good[name])), (which, name)
            one = bad[name].select(dim, m)
            assert not torch.isfinite(one[0, 1] if name in ("state", "dstate") else one[0, at, 1]).any(), (which, name)


def test_attention_step_moves_the_states_version():
    """a state that a recorded call saved, stepped before its backward pass: refused by autograd, not differentiated with the new values"""
    B, T, H, D = 2, 5, 2, 16
    q, k, v, do, state, _, decay = attention_inputs(B, T, H, H, D, D, F32)
    leaf = q.clone().requires_grad_()
    o, _ = ops.linear_attention(leaf, k, v, decay, state=state)
    before = state._version
    with torch.no_grad():
        ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.backward(do)
    # a view's step counts for its base; inference tensors keep no version
    both = randn(2, B, H, D, D)
    before = both._version
    ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, both[1])
    assert both._version > before
    with torch.inference_mode():
        ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, torch.zeros(B, H, D, D, device=DEV))


@pytest.mark.parametrize("B,DK,DV", [(40, 16, 16), (3, 64, 64), (300, 40, 24), (5, 33, 15), (600, 64, 128)])
def test_attention_step_keeps_slow_decays(B, DK, DV):
    """One step of a state with k = 0: exp(log_decay) S rounded once.  A factor rounded to fp32 before the product would be off by up to 2^-25, a rate of
    -1e-6 by 3 %.  fp32's expm1 (decays slower than -0.5) and exp are off by at most 2 units in the last place, of exp(a) - 1 and exp(a)."""
    decays = (-1e-6, -1e-5, -1e-4, -3e-3, -0.11, -0.4, -0.6, -2.5, 0.0, 1e-5, 0.3)
    decay = torch.tensor(decays, device=DEV)
    H = len(decays)
    state = randn(B, H, DK, DV, seed=1)
    old = state.double()
    q, k, v = randn(B, H, DK, seed=2), torch.zeros(B, H, DK, device=DEV), randn(B, H, DV, seed=3)
    ops.linear_attention_step(q, k, v, decay, state)
    a = decay.double()[:, None, None]
    off = 4 * U * torch.where(a.abs() < 0.5, torch.expm1(a).abs(), torch.exp(a)) * old.abs()
    want = old * torch.exp(a)
    bound = HALF[F32] * (1 + 2.0 ** -7) * want.abs() + off + TINY[F32]
    assert bool(((state.double() - want).abs() <= bound).all()), float((((state.double() - want).abs() - bound) / want.abs()).max()) / U


def test_attention_step_keeps_infinite_states():
    """a state that has left fp32's range stays there, whatever the decay"""
    decay = torch.tensor([0.0, -1e-5, -0.3, -3.0], device=DEV)
    for DK, DV in ((16, 16), (64, 64), (5, 7)):
        q, k, v, state = randn(2, 4, DK, seed=1), randn(2, 4, DK, seed=2), randn(2, 4, DV, seed=3), randn(2, 4, DK, DV, seed=4)
        state[:, :, 1, 2], state[:, :, 3, 0] = math.inf, -math.inf
        ops.linear_attention_step(q, k, v, decay, state)
        assert bool((state[:, :, 1, 2] == math.inf).all()) and bool((state[:, :, 3, 0] == -math.inf).all())
        assert int(torch.isfinite(state).logical_not().sum()) == 16


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,D", [(10, 16), (16, 20), (33, 16), (64, 64), (64, 17), (40, 128), (1100, 32), (1100, 19)])
def test_attention_fading_states_keep_their_digits(T, D, dt):
    """Tokens with k = 0 (q, do = 0 for the gradient) leave exp(log_decay T) S however small it is: one power and one product for each 16 (10) tokens or
    more, each off by at most 4 units in the last place (the power: 3, fp32's exponent included)."""
    decays = (-0.2, -0.5, -0.9, -0.05)
    decay = torch.tensor(decays if T < 100 else [d / 16 for d in decays], device=DEV)
    q, k, v, do, state, dstate, _ = attention_inputs(2, T, 4, 4, D, D, dt)
    last = ops.linear_attention(q, torch.zeros_like(k), v, decay, state=state)[1]
    first = ops.linear_attention_backward(torch.zeros_like(do), q, k, v, decay, state=state, dstate=dstate)[3]
    g = torch.exp(decay.double() * T)[:, None, None]
    units = 5 * (T // 16 + 1)
    for got, s in ((last, state), (first, dstate)):
        want = s.double() * g
        assert bool(((got.double() - want).abs() <= units * U * want.abs() + TINY[F32]).all()), float(((got.double() - want) / want).abs().max()) / U


@pytest.mark.parametrize("rate", [-1.1e-6, -2.3e-6, -1.7e-5])
def test_attention_slow_decays_across_segments(rate):
    """One sequence of 16384 tokens with k = 0: what is left of the state.  Its elements are rounded at every joint (256 at most) by errors that do not depend on each
    other, so their mean over 4096 elements is off by less than 6 sqrt(256 / 4096 / 3) 2^-24; a joint's factor that is itself rounded is off the same
    way for all of them, up to 256 times 2^-25."""
    T, D = 16384, 64
    decay = torch.full((1,), rate, device=DEV)
    state = 1 + torch.rand(1, 1, D, D, generator=torch.Generator().manual_seed(1)).to(DEV)
    q, k, v = (randn(1, T, 1, D, dt=BF16, seed=i) for i in range(3))
    zero = torch.zeros_like(k)
    want = state.double() * torch.exp(decay.double() * T)
    for got in (ops.linear_attention(q, zero, v, decay, state=state)[1], ops.linear_attention_backward(zero, q, k, v, decay, state=state, dstate=state)[3]):
        e = (got.double() - want) / want
        assert abs(float(e.mean())) < 6 * math.sqrt(256 / (3 * D * D)) * U, float(e.mean()) / U
        assert float(e.abs().max()) < 257 * U


@pytest.mark.parametrize("dt", [BF16, F16, F32])
def test_attention_output_off_16_bytes(dt):
    """the C entry takes any output that is aligned to its elements: o one element, 8 or 12 bytes past a multiple of 16, beside aligned operands"""
    lib, size, code = L.load(), torch.finfo(dt).bits // 8, {F32: L.TG_F32, BF16: L.TG_BF16, F16: L.TG_F16}[dt]
    for B, T, H, DK, DV in ((3, 10, 2, 16, 16), (2, 40, 2, 32, 64), (1, 900, 1, 64, 64), (700, 20, 2, 64, 64)):
        q, k, v, _, state, _, decay = attention_inputs(B, T, H, H, DK, DV, dt)
        want, mag = attention_oracle(q, k, v, decay, DK ** -0.5, state, None)
        st = lambda d: (T * H * d, H * d, d)   # noqa: E731
        desc = L.LaDesc(B, T, H, H, DK, DV, st(DK), st(DK), st(DV), DK ** -0.5)
        need = lib.tg_linear_attention_scratch_floats(code, C.byref(desc))
        for off in (size, 8, 12):
            room = torch.full((B * T * H * DV + 32 // size,), 7.0, dtype=dt, device=DEV)
            last, scratch = torch.empty_like(state), torch.empty(max(need, 1), device=DEV)
            assert room.data_ptr() % 16 == 0
            rc = lib.tg_linear_attention(code, C.byref(desc), q.data_ptr(), k.data_ptr(), v.data_ptr(),
                                         decay.data_ptr(), None, state.data_ptr(), room.data_ptr() + off, last.data_ptr(), scratch.data_ptr(),
                                         torch.cuda.current_stream().cuda_stream)
            assert rc == 0
            o = room[off // size:off // size + B * T * H * DV].view(B, T, H, DV)
            close(o, want["o"], dt, mag["o"], attention_units(dt, T, max(DK, DV)), "o")
            assert bool((room[:off // size] == 7).all()) and bool((room[off // size + B * T * H * DV:] == 7).all())


@pytest.mark.parametrize("dt", [F32, BF16, F16])
@pytest.mark.parametrize("T,D,units", [(1, 16, 16), (2, 16, 24), (1, 17, 16), (2, 17, 24), (40, 16, 40), (40, 64, 40), (40, 33, 40), (40, 128, 40)])
def test_attention_states_are_fp32(T, D, units, dt):
    """One term (two for T = 2) in each element of the last state and of the first one's gradient, with weights that no 16 bits hold: off by the power
    (4 units of 2^-24), up to three more factors of it (5 each), the products and the parts' sums (8), the decay of the state (5) - not by the 64 units of
    an operand in two bf16 parts."""
    q, k, v, do, state, dstate, _ = attention_inputs(6, T, 4, 4, D, D, dt)
    decay = -torch.tensor([0.3, 0.011, 0.17, 0.05], device=DEV)
    if T > 2:
        for t in (k, q):
            one = t[:, T // 2].clone()
            t.zero_()
            t[:, T // 2] = one
    for s, ds in ((state, dstate), (None, None)):
        last = ops.linear_attention(q, k, v, decay, scale=0.25, state=s)[1]
        first = ops.linear_attention_backward(do, q, k, v, decay, scale=0.25, state=torch.zeros_like(state) if s is None else s, dstate=ds)[3]
        want, mag = attention_oracle(q, k, v, decay, 0.25, s, None, do, ds)
        close(last, want["state"], F32, mag["state"], units, "state")
        close(first, want["dstate"], F32, mag["dstate"], units, "dstate")


def test_generator_published_vectors():
    """Random123's known answers for ten rounds: the oracle at all zeros, all ones and the digits of pi; the kernel at all zeros, word by word - kept at
    p = word / 2^32 and dropped at (word + 1) / 2^32"""
    zeros = [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert philox_block(0, 0) == zeros
    assert philox_block((1 << 64) - 1, (1 << 64) - 1, 0xffffffff, 0xffffffff) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert philox_block(0x85a308d3243f6a88, 0x299f31d0a4093822, 0x03707344, 0x13198a2e) == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]
    x, rng = torch.ones(4, device=DEV), ops.dropout_rng(0, DEV)
    for i, word in enumerate(zeros):
        assert float(ops.dropout(x, word / 2.0 ** 32, rng)[i]) != 0 and float(ops.dropout(x, (word + 1) / 2.0 ** 32, rng)[i]) == 0


def test_the_same_tensor_twice():
    """one tensor in several places of a call: its gradient is the sum over them"""
    x, w, dy, ds = randn(5, 64, seed=1), randn(64, seed=2), randn(5, 64, seed=3), randn(5, 64, seed=4)
    leaf = x.clone().requires_grad_()
    y, s = ops.rms_norm(leaf, w, residual=leaf)
    got, = torch.autograd.grad([y, s], [leaf], [dy, ds])
    dx, _ = ops.rms_norm_backward(dy, x, ops.rms_norm(x, w, residual=x, stats=True)[2], w, residual=x, ds=ds)
    assert torch.equal(got, 2 * dx)
    rng = ops.dropout_rng(3, DEV)
    got, = torch.autograd.grad(ops.dropout(leaf, 0.4, rng, residual=leaf), [leaf], dy)
    assert torch.equal(got, ops.dropout_backward(dy, 0.4, rng) + dy)
    q, _, _, do, _, _, decay = attention_inputs(2, 21, 3, 3, 16, 16, F32)
    leaf = q.clone().requires_grad_()
    got, = torch.autograd.grad(ops.linear_attention(leaf, leaf, leaf, decay)[0], [leaf], do)
    dq, dk, dv, _ = ops.linear_attention_backward(do, q, q, q, decay)
    close(got, dq.double() + dk.double() + dv.double(), F32, dq.double().abs() + dk.double().abs() + dv.double().abs(), 2, "dq + dk + dv")


@pytest.mark.parametrize("dt", [F32, BF16])
def test_attention_growing_memories(dt):
    """log_decay above zero: powers that grow, in one chunk, in several and across segments"""
    for T, D in ((9, 16), (40, 32), (70, 33), (900, 64)):
        q, k, v, do, state, dstate, _ = attention_inputs(1, T, 3, 3, D, D, dt, seed=T)
        decay = torch.tensor([0.3, 0.02, 1e-4], device=DEV) * min(1.0, 40 / T)
        o, last = ops.linear_attention(q, k, v, decay, state=state)
        got = ops.linear_attention_backward(do, q, k, v, decay, state=state, dstate=dstate)
        want, mag = attention_oracle(q, k, v, decay, D ** -0.5, state, None, do, dstate)
        for name, g, t in zip(("o", "state", "dq", "dk", "dv", "dstate"), (o, last, *got), (dt, F32, dt, dt, dt, F32)):
            close(g, want[name], t, mag[name], attention_units(dt, T, D), name)


@pytest.mark.parametrize("D", [64, 63])
def test_attention_past_32_bit_offsets(D):
    """4194344 tokens of 8 heads: 4.3 GB an operand.  The memory is gone after 400 tokens (e^-80), so the first and the last 200 are those of windows of 600"""
    T, H = (1 << 22) + 40, 8
    g = torch.Generator(device=DEV).manual_seed(1)
    q, k, v, do = (torch.randn(1, T, h, D, dtype=BF16, device=DEV, generator=g) for h in (H, 1, 1, H))
    decay = torch.linspace(-0.2, -0.6, H, device=DEV)
    o, last = ops.linear_attention(q, k, v, decay)
    dq, dk, dv, _ = ops.linear_attention_backward(do, q, k, v, decay)
    for lo, rows in ((0, slice(0, 200)), (T - 600, slice(400, 600))):
        cut = lambda t: t[:, lo:lo + 600]   # noqa: E731
        want, mag = attention_oracle(cut(q), cut(k), cut(v), decay, D ** -0.5, None, None, cut(do))
        for name, t in (("o", o), ("dq", dq), ("dk", dk), ("dv", dv)):
            close(cut(t)[:, rows], want[name][:, rows], BF16, mag[name][:, rows], attention_units(BF16, 600, D) * H, name)
        if lo:
            close(last, want["state"], F32, mag["state"], attention_units(BF16, 600, D), "state")


def test_rms_norm_past_32_bit_offsets():
    """33554435 rows of 64 and 65537 of 32772 (4.3 GB each): the last rows have the bits that they have alone"""
    for rows, channels in (((1 << 25) + 3, 64), ((1 << 16) + 1, (1 << 15) + 4)):
        x = torch.randn(rows, channels, dtype=BF16, device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
        y, rstd = ops.rms_norm(x, stats=True)
        dx, _ = ops.rms_norm_backward(x, x, rstd, dweight=False)
        q, scale = ops.rms_norm_e4m3(x)
        end = x[-5:].clone()
        y1, r1 = ops.rms_norm(end, stats=True)
        q1, s1 = ops.rms_norm_e4m3(end)
        assert torch.equal(y[-5:], y1) and torch.equal(rstd[-5:], r1) and torch.equal(q[-5:].float(), q1.float()) and torch.equal(scale[-5:], s1)
        assert torch.equal(dx[-5:], ops.rms_norm_backward(end, end, r1, dweight=False)[0])
        del x, y, dx, q


# ------------------------------------------------------------------------------------- streams, graphs, refusals, together
def all_operators(x, w, rng, q, k, v, decay, state, out):
    """every operator once into the dict `out` (explicit forms, as a captured step calls them)"""
    out["y"], out["s"], rstd = ops.rms_norm(x, w, residual=x, stats=True)
    out["dx"], out["dw"] = ops.rms_norm_backward(x, x, rstd, w, residual=x, ds=x)
    out["q8"], out["scale"], _ = ops.rms_norm_e4m3(x, w, residual=x)
    out["drop"] = ops.dropout(x, 0.3, rng, layer=1, residual=x)
    out["ddrop"] = ops.dropout_backward(x, 0.3, rng, layer=1)
    out["o"], out["last"] = ops.linear_attention(q, k, v, decay, state=state)
    for name, t in zip(("dq", "dk", "dv", "dstate"), ops.linear_attention_backward(q, q, k, v, decay, state=state, dstate=state)):
        out[name] = t
    live = state.clone()
    out["step"] = ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, live)
    out["live"] = live


def graph_inputs(seed, T=700):
    x, w = randn(300, 64, dt=BF16, seed=seed), randn(64, seed=seed + 1)
    q, k, v = randn(2, T, 4, 32, dt=BF16, seed=seed + 2), randn(2, T, 2, 32, dt=BF16, seed=seed + 3), randn(2, T, 2, 32, dt=BF16, seed=seed + 4)
    return [x, w, ops.dropout_rng(seed, DEV), q, k, v, -torch.tensor([0.5, 0.1, 0.02, 0.003], device=DEV), randn(2, 4, 32, 32, seed=seed + 5)]


def test_operators_in_graphs():
    """captured and replayed with new inputs and a moved generator, two graphs in turn, eager work between: every replay equals the eager result"""
    graphs = []
    for seed in (1, 100):
        static = graph_inputs(seed)
        out = {}
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            all_operators(*static, {})
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            all_operators(*static, out)
            static[2][1] += 1
        graphs.append((g, static, out))
    for turn in range(4):
        for g, static, out in graphs:
            fresh = graph_inputs(1000 + 10 * turn)
            for a, b in zip(static, fresh):
                a.copy_(b)
            want = {}
            all_operators(*fresh, want)
            g.replay()
            torch.cuda.synchronize()
            for name in want:
                assert torch.equal(out[name].float(), want[name].float()), (turn, name)
            assert static[2].tolist()[1] == 1


def test_operators_on_another_stream():
    args = graph_inputs(7)
    want, got = {}, {}
    all_operators(*args, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_operators(*args, got)
    side.synchronize()
    for name in want:
        assert torch.equal(got[name].float(), want[name].float()), name


def test_two_calls_at_once():
    """the same calls on two streams, nothing waiting between them: workspaces are each call's own"""
    a, b = graph_inputs(3, T=5000), graph_inputs(4, T=5000)
    want = [{}, {}]
    all_operators(*a, want[0])
    all_operators(*b, want[1])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = [{}, {}]
        for s, args, out in zip(streams, (a, b), got):
            with torch.cuda.stream(s):
                all_operators(*args, out)
        torch.cuda.synchronize()
        for w, o in zip(want, got):
            for name in w:
                assert torch.equal(o[name].float(), w[name].float()), name


def test_autograd_is_refused_inside_a_capture():
    x = randn(8, 64).requires_grad_()
    rng, decay = ops.dropout_rng(1, DEV), torch.zeros(2, device=DEV)
    q = randn(1, 4, 2, 16).requires_grad_()
    ops.rms_norm(x).sum().backward()
    torch.cuda.synchronize()
    seen = []
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        for call in (lambda: ops.rms_norm(x), lambda: ops.dropout(x, 0.1, rng), lambda: ops.linear_attention(q, q, q, decay)):
            try:
                call()
            except L.TecoganHipError as e:
                seen.append(str(e))
        with torch.no_grad():
            y = ops.rms_norm(x)
    assert len(seen) == 3 and all("not captured" in s for s in seen)
    assert y.shape == x.shape


def test_forward_mode_is_refused():
    """no operator hands a tangent on: a dual tensor is refused instead of losing its own"""
    x, w, r = randn(4, 64), randn(64), randn(4, 64)
    q, state, decay, rng = randn(2, 3, 2, 16), randn(2, 2, 16, 16), torch.zeros(2, device=DEV), ops.dropout_rng(1, DEV)
    fw = torch.autograd.forward_ad
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: ops.rms_norm(d(x), w), lambda: ops.rms_norm(x, d(w)), lambda: ops.rms_norm(x, w, residual=d(r)), lambda: ops.rms_norm_e4m3(d(x), w),
                     lambda: ops.rms_norm_backward(d(x), x, randn(4), w), lambda: ops.rms_norm_backward(x, x, randn(4), w, ds=d(x)), lambda: ops.dropout(d(x), 0.1, rng),
                     lambda: ops.dropout(x, 0.1, rng, residual=d(r)), lambda: ops.dropout_backward(d(x), 0.1, rng), lambda: ops.linear_attention(d(q), q, q, decay),
                     lambda: ops.linear_attention(q, q, d(q), decay), lambda: ops.linear_attention(q, q, q, d(decay)), lambda: ops.linear_attention(q, q, q, decay, state=d(state)),
                     lambda: ops.linear_attention_backward(d(q), q, q, q, decay), lambda: ops.linear_attention_backward(q, q, q, q, decay, state=state, dstate=d(state)),
                     lambda: ops.linear_attention_step(d(q[:, 0]), q[:, 0], q[:, 0], decay, state[:2])):
            with pytest.raises(L.TecoganHipError, match="forward-mode"):
                call()
        assert torch.equal(ops.rms_norm(x, w), ops.rms_norm(x.clone(), w))   # (plain tensors inside a level are served)


FIRST_CALL = """
import torch
import pytorch_tecogan_amd
from pytorch_tecogan_amd import ops
torch.manual_seed(5)
x, w = torch.randn(70, 200, device="cuda"), torch.randn(200, device="cuda")
q, k, v, do = (torch.randn(2, 300, 2, 64, device="cuda").bfloat16() for _ in range(4))
decay, state = torch.tensor([-0.1, -0.5], device="cuda"), torch.randn(2, 2, 64, 64, device="cuda")
rng = torch.tensor([1, 2], device="cuda")
def run():
    one = state.clone()
    return (ops.rms_norm(x, w), ops.rms_norm_e4m3(x, w)[1], ops.dropout(x, 0.3, rng), *ops.linear_attention(q, k, v, decay, state=state),
            *ops.linear_attention_backward(do, q, k, v, decay, state=state), ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, one), one)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
for i in range(3):
    x.normal_(), q.normal_()
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, run()):
        assert torch.equal(a, b), i
print("replays equal")
"""


def test_the_first_call_of_a_process_inside_a_capture():
    """kernels are loaded and their attributes set by the captured call itself"""
    r = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=ROOT, env={**os.environ, "PYTHONPATH": ROOT}, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and "replays equal" in r.stdout, r.stderr[-2000:]


def test_refusals():
    x, w = randn(4, 64), randn(64)
    rng, decay = ops.dropout_rng(1, DEV), torch.zeros(2, device=DEV)
    q, k, v = randn(2, 5, 2, 16), randn(2, 5, 2, 16), randn(2, 5, 2, 8)
    state = randn(2, 2, 16, 8)
    ln = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    bad = [
        lambda: ops.rms_norm(x.cpu()), lambda: ops.rms_norm(x.double()), lambda: ops.rms_norm(x.long()), lambda: ops.rms_norm(randn(1)[0]),
        lambda: ops.rms_norm(torch.empty(4, 0, device=DEV)), lambda: ops.rms_norm(x, w[:63]), lambda: ops.rms_norm(x, w.bfloat16()),
        lambda: ops.rms_norm(x, w.cpu()), lambda: ops.rms_norm(x, w, residual=x[:1]), lambda: ops.rms_norm(x, w, residual=x.bfloat16()),
        lambda: ops.rms_norm(x, w, eps=-1.0), lambda: ops.rms_norm(x, w, eps=math.nan),
        lambda: ops.rms_norm_backward(x, x, w), lambda: ops.rms_norm_backward(x[:2], x, randn(4), w), lambda: ops.rms_norm_backward(x, x, randn(4), w, ds=x[:1]),
        lambda: ops.rms_norm_backward(x, x, randn(4), w, residual=x[:1]),
        lambda: ops.rms_norm_e4m3(x.clone().requires_grad_()),
        lambda: ops.dropout(x, 1.0, rng), lambda: ops.dropout(x, -0.1, rng), lambda: ops.dropout(x, math.nan, rng), lambda: ops.dropout(x, 0.1, rng.int()),
        lambda: ops.dropout(x, 0.1, rng.cpu()), lambda: ops.dropout(x, 0.1, rng, layer=-1), lambda: ops.dropout(x, 0.1, rng, layer=1 << 31),
        lambda: ops.dropout(x, 0.1, rng, residual=x[0]), lambda: ops.dropout(x, 0.1, 1234),
        lambda: ops.linear_attention(q, k, v, decay[:1]), lambda: ops.linear_attention(q, k, v, decay.double()), lambda: ops.linear_attention(q, k, v.half(), decay),
        lambda: ops.linear_attention(q, k[:, :4], v, decay), lambda: ops.linear_attention(q, k, v[:, :4], decay), lambda: ops.linear_attention(q, k[..., :8], v, decay),
        lambda: ops.linear_attention(q[0], k[0], v[0], decay), lambda: ops.linear_attention(randn(2, 5, 3, 16), k, v, torch.zeros(3, device=DEV)),
        lambda: ops.linear_attention(randn(2, 5, 2, 129), randn(2, 5, 2, 129), v, decay), lambda: ops.linear_attention(q, k, v, decay, state=state[:1]),
        lambda: ops.linear_attention(q, k, v, decay, state=state.half()), lambda: ops.linear_attention(q, k, v, decay, lengths=ln.long()),
        lambda: ops.linear_attention(q, k, v, decay, lengths=ln[:1]), lambda: ops.linear_attention(q, k, v, decay.clone().requires_grad_()),
        lambda: ops.linear_attention_backward(q, q, k, v, decay), lambda: ops.linear_attention_step(q, k, v, decay, state),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, state.transpose(2, 3)),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, randn(2, 2, 8, 16).transpose(2, 3)),
        lambda: ops.linear_attention_step(q[:, 0].clone().requires_grad_(), k[:, 0], v[:, 0], decay, state),
        # no tensors
        lambda: ops.rms_norm([1.0]), lambda: ops.rms_norm(x, 2.0), lambda: ops.rms_norm(x, w, residual=1.0), lambda: ops.rms_norm_e4m3(x, 2.0),
        lambda: ops.dropout(None, 0.1, rng), lambda: ops.dropout(x, 0.1, rng, residual=0.0), lambda: ops.linear_attention(None, k, v, decay),
        lambda: ops.linear_attention(q, [1.0], v, decay), lambda: ops.linear_attention(q, k, v, -0.1), lambda: ops.linear_attention(q, k, v, decay, state=0.0),
        lambda: ops.linear_attention(q, k, v, decay, lengths=[1, 2]), lambda: ops.linear_attention_step(q[:, 0], None, v[:, 0], decay, state),
        lambda: ops.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], decay, None),
        # 2^30 + 1 sequences (strides of zero: nothing is allocated before the refusal)
        lambda: ops.linear_attention_step(*(t[:1, 0].expand((1 << 30) + 1, -1, -1) for t in (q, k, v)), decay, state),
        lambda: ops.linear_attention(*(t[:1, :1].expand(-1, (1 << 30) + 1, -1, -1) for t in (q, k, v)), decay),
        lambda: ops.rms_norm(x[:1, :1].expand(1, (1 << 30) + 1)),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(L.TecoganHipError):
            call()
            pytest.fail(f"call {i} was not refused")


def temporal_block(x, norm_w, proj, out_proj, decay, rng, layer, state=None, heads=4):
    """norm -> q, k, v -> attention over the tokens -> projection -> dropout with the skip: x (B, T, C) -> (x', state)"""
    B, T, C_ = x.shape
    q, k, v = (ops.rms_norm(x, norm_w) @ proj).view(B, T, 3, heads, C_ // heads).unbind(2)
    o, state = ops.linear_attention(q, k, v, decay, state=state)
    return ops.dropout(o.reshape(B, T, C_) @ out_proj, 0.1, rng, layer=layer, residual=x), state


def test_the_operators_together():
    """two blocks over a clip, forward and gradients, against the same composition in 64 bits; and the clip frame by frame"""
    B, T, C_, H = 6, 20, 64, 4
    D = C_ // H
    decay = -torch.tensor([0.5, 0.2, 0.05, 0.01], device=DEV)
    rng = ops.dropout_rng(99, DEV, 4)
    x0 = randn(B, T, C_, seed=1)
    params = [[1 + 0.1 * randn(C_, seed=10 * l + 2), randn(C_, 3 * C_, seed=10 * l + 3) / 8, randn(C_, C_, seed=10 * l + 4) / 8] for l in range(2)]
    dy = randn(B, T, C_, seed=5)
    leaf = [x0.clone().requires_grad_()] + [p.clone().requires_grad_() for ps in params for p in ps]
    x = leaf[0]
    for l in range(2):
        x, _ = temporal_block(x, *leaf[1 + 3 * l:4 + 3 * l], decay, rng, l)
    got = torch.autograd.grad(x, leaf, dy)

    ref = [t.detach().double().cpu().requires_grad_() for t in leaf]
    a = decay.double().cpu()
    gap = (torch.arange(T)[:, None] - torch.arange(T)[None]).double()
    w = torch.where(gap >= 0, torch.exp(a[:, None, None] * gap.clamp_min(0)), 0.0) * D ** -0.5
    z = ref[0]
    for l in range(2):
        nw, pr, op = ref[1 + 3 * l:4 + 3 * l]
        y, _ = norm_oracle(z, None, 1e-6)
        q, k, v = ((y * nw) @ pr).view(B, T, 3, H, D).permute(2, 0, 3, 1, 4)
        o = (((q @ k.transpose(2, 3)) * w) @ v).permute(0, 2, 1, 3).reshape(B, T, C_)
        keep = keep_mask((B, T, C_), 0.1, 99, 4, l)
        z = z + torch.where(keep, (o @ op) / 0.9, 0.0)
    want = torch.autograd.grad(z, ref, dy.double().cpu())
    # fp32 throughout: two blocks of five sums of 64 .. 120 products each, every one off by at most (its additions) 2^-24 of its magnitudes;
    # ten of them in a row, whole-tensor: 10 * 120 * 2^-24 = 7e-5
    for g, r, name in zip((x, *got), (z, *want), ("out", "dx", "w0", "p0", "o0", "w1", "p1", "o1")):
        e = float((g.detach().double().cpu() - r.detach()).norm() / r.detach().norm())
        assert e < 7e-5, (name, e)

    with torch.no_grad():   # frame by frame without dropout, as a live stream runs
        seq = x0
        for ps in params:
            q, k, v = (ops.rms_norm(seq, ps[0]) @ ps[1]).view(B, T, 3, H, D).unbind(2)
            seq = seq + ops.linear_attention(q, k, v, decay)[0].reshape(B, T, C_) @ ps[2]
        states = [torch.zeros(B, H, D, D, device=DEV) for _ in params]
        for t in range(T):
            cur = x0[:, t]
            for ps, s in zip(params, states):
                q, k, v = (ops.rms_norm(cur, ps[0]) @ ps[1]).view(B, 3, H, D).unbind(1)
                cur = cur + ops.linear_attention_step(q, k, v, decay, s).reshape(B, C_) @ ps[2]
            e = float((cur - seq[:, t]).norm() / seq[:, t].norm())
            assert e < 7e-5, (t, e)

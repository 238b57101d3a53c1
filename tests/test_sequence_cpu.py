"""The sequence-layer operators without a GPU: the C entry points check their arguments before any launch (status codes below), the Python
forms refuse host tensors, and the names are where a user of `from ops import *` finds them."""
import ctypes as C
import os
import sys

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)
import pytorch_tecogan_amd  # noqa: E402,F401
from pytorch_tecogan_amd import _lib as L  # noqa: E402
from pytorch_tecogan_amd import ops  # noqa: E402

BADARG, UNSUPPORTED, ALIGN = -1, -2, -3
P = 0x10000   # never dereferenced: every call below is refused before a launch


def desc(B=2, T=5, H=2, HK=2, DK=16, DV=8):
    st = lambda h, d: (T * h * d, h * d, d)   # noqa: E731
    return L.LaDesc(B, T, H, HK, DK, DV, st(H, DK), st(HK, DK), st(HK, DV), 0.25)


def test_rms_norm_arguments():
    f = L.load().tg_rms_norm
    good = [L.TG_BF16, P, 64, None, 0, P, P, None, None, 4, 64, 1e-6, None]
    for at, value, want in ((0, 7, BADARG), (1, None, BADARG), (6, None, BADARG), (9, -1, BADARG), (10, 0, BADARG), (2, -64, BADARG), (11, -1.0, BADARG),
                            (11, float("nan"), BADARG), (1, P + 1, ALIGN), (3, P + 1, ALIGN), (6, P + 1, ALIGN), (5, P + 2, ALIGN), (8, P + 2, ALIGN),
                            (10, (1 << 30) + 1, UNSUPPORTED)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == want, (at, value)
    assert f(*(good[:9] + [0] + good[10:])) == 0   # no rows: nothing to launch
    f = L.load().tg_rms_norm_e4m3
    good = [L.TG_F32, P, 64, None, 0, P, P, P, None, 4, 64, 1e-6, None]
    for at, value, want in ((7, None, BADARG), (6, None, BADARG), (7, P + 2, ALIGN), (1, P + 2, ALIGN)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == want, (at, value)
    f = L.load().tg_rms_norm_bwd
    good = [L.TG_F16, P, 64, P, 64, None, 0, P, P, None, 0, P, P, P, 4, 64, None]
    for at, value, want in ((1, None, BADARG), (3, None, BADARG), (7, None, BADARG), (11, None, BADARG), (13, None, BADARG), (14, -1, BADARG), (15, 0, BADARG),
                            (1, P + 1, ALIGN), (9, P + 1, ALIGN), (12, P + 2, ALIGN), (13, P + 2, ALIGN), (15, (1 << 30) + 1, UNSUPPORTED)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == want, (at, value)
    n = L.load().tg_rms_norm_bwd_scratch_floats
    assert n(0, 64) == 0 and n(3, 0) == 0 and n(1, 64) >= 64 and n(1 << 40, 128) >= 128


def test_dropout_arguments():
    f = L.load().tg_dropout
    good = [L.TG_BF16, P, None, P, 100, 0.5, P, 0, None]
    for at, value, want in ((0, 3, BADARG), (1, None, BADARG), (3, None, BADARG), (4, -1, BADARG), (5, 1.0, BADARG), (5, -0.1, BADARG), (5, float("nan"), BADARG),
                            (6, None, BADARG), (1, P + 1, ALIGN), (2, P + 1, ALIGN), (3, P + 1, ALIGN), (6, P + 4, ALIGN)):
        bad = list(good)
        bad[at] = value
        assert f(*bad) == want, (at, value)
    assert f(*(good[:4] + [0] + good[5:])) == 0


def test_linear_attention_arguments():
    lib = L.load()
    ref = C.byref
    for d, want in ((desc(B=-1), BADARG), (desc(T=-1), BADARG), (desc(H=0), BADARG), (desc(HK=0), BADARG), (desc(DK=0), BADARG), (desc(DV=0), BADARG),
                    (desc(H=3), UNSUPPORTED), (desc(DK=129), UNSUPPORTED), (desc(DV=129), UNSUPPORTED), (desc(B=(1 << 30) + 1), UNSUPPORTED), (desc(T=(1 << 30) + 1), UNSUPPORTED)):
        assert lib.tg_linear_attention(L.TG_F32, ref(d), P, P, P, P, None, None, P, P, None, None) == want
        assert lib.tg_linear_attention_scratch_floats(L.TG_BF16, ref(d)) == 0
        assert lib.tg_linear_attention_step(L.TG_F32, ref(d), P, P, P, P, P, P, None) == want
        assert lib.tg_linear_attention_bwd(L.TG_F32, ref(d), P, P, P, P, (C.c_int64 * 3)(80, 16, 8), P, None, None, None, P, P, P, None, P, None) == want
        assert lib.tg_linear_attention_bwd_scratch_floats(L.TG_BF16, ref(d)) == 0
    d = desc()
    good = [L.TG_BF16, ref(d), P, P, P, P, None, None, P, P, None, None]
    for at, value, want in ((0, 9, BADARG), (1, None, BADARG), (2, None, BADARG), (3, None, BADARG), (4, None, BADARG), (5, None, BADARG), (8, None, BADARG),
                            (9, None, BADARG), (2, P + 1, ALIGN), (4, P + 1, ALIGN), (8, P + 1, ALIGN), (9, P + 2, ALIGN), (5, P + 2, ALIGN), (7, P + 2, ALIGN),
                            (6, P + 2, ALIGN), (10, P + 2, ALIGN)):
        bad = list(good)
        bad[at] = value
        assert lib.tg_linear_attention(*bad) == want, (at, value)
    good = [L.TG_BF16, ref(d), P, P, P, P, P, P, None]
    for at, value, want in ((2, None, BADARG), (3, None, BADARG), (4, None, BADARG), (5, None, BADARG), (6, None, BADARG), (7, None, BADARG), (2, P + 1, ALIGN),
                            (7, P + 2, ALIGN), (5, P + 2, ALIGN)):
        bad = list(good)
        bad[at] = value
        assert lib.tg_linear_attention_step(*bad) == want, (at, value)
    shared = desc(H=10, HK=2)   # (more shared heads than a workgroup sums: through scratch)
    good = [L.TG_BF16, ref(shared), P, P, P, P, (C.c_int64 * 3)(400, 80, 8), P, None, None, None, P, P, P, None, P, None]
    for at, value, want in ((2, None, BADARG), (5, None, BADARG), (6, None, BADARG), (7, None, BADARG), (11, None, BADARG), (13, None, BADARG), (15, None, BADARG),
                            (12, P + 1, ALIGN), (15, P + 2, ALIGN), (14, P + 2, ALIGN), (9, P + 2, ALIGN), (10, P + 2, ALIGN)):
        bad = list(good)
        bad[at] = value
        assert lib.tg_linear_attention_bwd(*bad) == want, (at, value)
    # one long sequence is cut into segments: their states need scratch
    long = desc(B=1, T=4096, H=1, HK=1)
    need = lib.tg_linear_attention_scratch_floats(L.TG_BF16, ref(long))
    assert need >= 2 * 16 * 8 and lib.tg_linear_attention_bwd_scratch_floats(L.TG_BF16, ref(long)) >= 4 * 16 * 8
    assert lib.tg_linear_attention(L.TG_BF16, ref(long), P, P, P, P, None, None, P, P, None, None) == BADARG
    wild = desc()
    wild.k_stride[1] = 1 << 31
    assert lib.tg_linear_attention(L.TG_BF16, ref(wild), P, P, P, P, None, None, P, P, None, None) == UNSUPPORTED
    wild.k_stride[1] = -16
    assert lib.tg_linear_attention(L.TG_BF16, ref(wild), P, P, P, P, None, None, P, P, None, None) == BADARG
    # an empty batch: nothing to launch
    assert lib.tg_linear_attention(L.TG_F32, ref(desc(B=0)), None, None, None, None, None, None, None, None, None, None) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(4, 64)
    q = torch.zeros(2, 3, 2, 16)
    rng, decay = torch.zeros(2, dtype=torch.int64), torch.zeros(2)
    for call in (lambda: ops.rms_norm(x), lambda: ops.rms_norm_e4m3(x), lambda: ops.rms_norm_backward(x, x, torch.zeros(4)), lambda: ops.dropout(x, 0.1, rng),
                 lambda: ops.dropout_backward(x, 0.1, rng), lambda: ops.linear_attention(q, q, q, decay),
                 lambda: ops.linear_attention_backward(q, q, q, q, decay), lambda: ops.linear_attention_step(q[0], q[0], q[0], decay, torch.zeros(3, 2, 16, 16))):
        with pytest.raises(L.TecoganHipError):
            call()


def test_forward_mode_is_refused():
    """a dual tensor does not require a gradient: without a check its tangent would be dropped"""
    fw = torch.autograd.forward_ad
    x, q = torch.zeros(4, 64), torch.zeros(2, 3, 2, 16)
    rng, decay, state = torch.zeros(2, dtype=torch.int64), torch.zeros(2), torch.zeros(2, 2, 16, 16)
    with fw.dual_level():
        d = lambda t: fw.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: ops.rms_norm(d(x)), lambda: ops.rms_norm(x, residual=d(x)), lambda: ops.rms_norm_e4m3(d(x)), lambda: ops.rms_norm_backward(d(x), x, x[:, 0]),
                     lambda: ops.dropout(d(x), 0.1, rng), lambda: ops.dropout(x, 0.1, rng, residual=d(x)), lambda: ops.dropout_backward(d(x), 0.1, rng),
                     lambda: ops.linear_attention(q, d(q), q, decay), lambda: ops.linear_attention(q, q, q, decay, state=d(state)),
                     lambda: ops.linear_attention_backward(q, q, q, q, decay, state=state, dstate=d(state)), lambda: ops.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], decay, d(state))):
            with pytest.raises(L.TecoganHipError, match="forward-mode"):
                call()
        with pytest.raises(L.TecoganHipError, match="device tensor"):
            ops.rms_norm(x)   # (a plain tensor inside a level is looked at as ever)


class OnDevice(torch.Tensor):
    """a host tensor that says it is on a device"""
    index = 0
    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", self.index))


@pytest.mark.parametrize("current,of_tensor,capturing,refused", [(0, 0, 0, True), (0, 1, 1, True), (0, 1, 0, False), (1, 0, 1, False), (1, 0, 0, True), (0, 0, 1, False)])
def test_a_capture_is_looked_for_on_the_tensors_device(monkeypatch, current, of_tensor, capturing, refused):
    """the stream that a call enqueues on is its tensors' device's, whichever device is the current one"""
    from pytorch_tecogan_amd import sequence
    now = [current]

    class Device:
        def __init__(self, dev):
            self.index = dev.index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *a):
            now[0] = self.before

    monkeypatch.setattr(sequence, "_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == capturing)
    x = torch.zeros(4, 64).as_subclass(OnDevice).requires_grad_()
    x.index = of_tensor
    if refused:
        with pytest.raises(L.TecoganHipError, match="not captured"):
            sequence._grad(x)
    else:
        assert sequence._grad(x)
    assert now == [current]


def test_the_packed_descriptor_is_the_structure():
    """sequence.py packs tg_la_desc as bytes; _lib.LaDesc says its layout field by field"""
    from pytorch_tecogan_amd import sequence
    d = L.LaDesc(3, 5, 8, 2, 24, 40, (1, 2, 3), (4, 5, 6), (7, 8, 1 << 40), 0.3)
    assert sequence._DESC.pack(3, 5, 8, 2, 24, 40, 1, 2, 3, 4, 5, 6, 7, 8, 1 << 40, 0.3) == bytes(d)


def test_names_are_public():
    """`from ops import *` (code/ops.py) re-exports every public name of the package's ops module"""
    from pytorch_tecogan_amd import sequence
    for name in sequence.__all__:
        assert getattr(ops, name) is getattr(sequence, name)
        assert getattr(ops, name).__doc__

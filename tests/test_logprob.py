"""rl_hip_token_logprob and its gradient without a GPU: the ctypes mirror and every refusal (the arguments are checked
before the device)."""
import ctypes as C

import pytest

import helpers

P = 1 << 20  # an aligned address that is never read


def test_mirror(rl):
    probe = helpers.load_shared("tests/c/logprob_probe.c", link_runtime=False)
    probe.logprob_probe.restype = C.c_size_t
    a, g = rl.TokenLogprobArgs, rl.TokenLogprobGradArgs
    want = [C.sizeof(a), a.scale.offset, a.workspace_bytes.offset, C.sizeof(g), g.lse.offset, g.dw_stride.offset,
            g.workspace_bytes.offset]
    assert [probe.logprob_probe(i) for i in range(7)] == want


def forward_args(rl, **kw):
    a = dict(x=P, w=P, targets=P, rows=10, vocab=1000, hidden=128, x_stride=128, w_stride=128, scale=0.0, logprob=P, lse=P,
             workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return rl.TokenLogprobArgs(**a)


def grad_args(rl, **kw):
    a = dict(x=P, w=P, targets=P, rows=10, vocab=1000, hidden=128, x_stride=128, w_stride=128, scale=0.0, lse=P,
             grad_logprob=P, dx=P, dw=P, dx_stride=128, dw_stride=128, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return rl.TokenLogprobGradArgs(**a)


BOTH = [(dict(x=None), "NULL"), (dict(w=None), "NULL"), (dict(targets=None), "NULL"), (dict(lse=None), "NULL"),
        (dict(rows=0), "rows"), (dict(rows=(1 << 20) + 1), "rows"), (dict(vocab=0), "vocab"),
        (dict(vocab=(1 << 24) + 1), "vocab"), (dict(hidden=0), "hidden"), (dict(hidden=100), "hidden"),
        (dict(hidden=(1 << 16) + 64, x_stride=1 << 17, w_stride=1 << 17, dx_stride=1 << 17, dw_stride=1 << 17), "hidden"),
        (dict(rows=1 << 20, vocab=1 << 20), "2^23"), (dict(x_stride=120), "strides"), (dict(w_stride=132), "strides"),
        (dict(x_stride=(1 << 22) + 8), "strides"), (dict(w_stride=(1 << 22) + 8), "strides"), (dict(scale=-1.0), "scale"),
        (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(x=P + 8), "aligned"),
        (dict(w=P + 2), "aligned")]


@pytest.mark.parametrize("kw, words", BOTH + [(dict(logprob=None), "NULL")])
def test_forward_refusals(rl, kw, words):
    kw = {k: v for k, v in kw.items() if k not in ("dx_stride", "dw_stride")}
    for call, ret in ((rl.lib().rl_hip_token_logprob, -1), (rl.lib().rl_hip_token_logprob_workspace, 0)):
        assert call(C.byref(forward_args(rl, **kw))) == ret
        assert words in rl.lib().rl_hip_last_error().decode()


@pytest.mark.parametrize("kw, words", BOTH + [
    (dict(grad_logprob=None), "NULL"), (dict(dx=None, dw=None), "NULL"), (dict(dx_stride=120), "strides"),
    (dict(dw_stride=132), "strides"), (dict(dx=P + 8), "aligned"), (dict(dw=P + 4), "aligned")])
def test_grad_refusals(rl, kw, words):
    for call, ret in ((rl.lib().rl_hip_token_logprob_grad, -1), (rl.lib().rl_hip_token_logprob_grad_workspace, 0)):
        assert call(C.byref(grad_args(rl, **kw))) == ret
        assert words in rl.lib().rl_hip_last_error().decode()


@pytest.mark.parametrize("kw", [dict(dx=None, dx_stride=0), dict(dw=None, dw_stride=0), dict(rows=1 << 20), dict(vocab=1)])
def test_what_is_allowed(rl, kw):
    """Up to the device, which is not open."""
    if rl.lib().rl_hip_is_open():
        pytest.skip("a device is open")
    assert rl.lib().rl_hip_token_logprob_grad(C.byref(grad_args(rl, **kw))) == -1
    assert "no device open" in rl.lib().rl_hip_last_error().decode()


def test_null(rl):
    L = rl.lib()
    assert L.rl_hip_token_logprob(None) == -1 and L.rl_hip_token_logprob_grad(None) == -1
    assert L.rl_hip_token_logprob_workspace(None) == 0 and L.rl_hip_token_logprob_grad_workspace(None) == 0

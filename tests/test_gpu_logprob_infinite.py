"""rl_hip_token_logprob where a logit is infinite: lse = log sum exp z is infinity with one that is +infinity, and one that
is -infinity has no part."""
import numpy as np
import pytest

import kv8_helpers as k8
from test_gpu_logprob import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, vocab", [(9, 40), (20, 9000), (100, 16000), (130, 700), (300, 8000), (200, 31990), (500, 32001)])
@pytest.mark.parametrize("at", [0, -1])
def test_infinite_logits(rl, gpu, rows, vocab, at):
    c = Case(rows + vocab, rows, vocab, 128, none=0)
    x, w = k8.floats(c.x, "bf16"), k8.floats(c.w, "bf16")
    entry = vocab + at if at < 0 else vocab // 3
    c.target[:3] = entry
    x[:, 5] = np.where(np.arange(rows) % 2 == 0, 2.0, -2.0)
    c.x = k8.bits(x, "bf16")
    clean = c.run(rl, dx=False, dw=False)
    w[entry, 5] = np.inf
    c.w = k8.bits(w, "bf16")
    lp, lse, _, _ = c.run(rl, dx=False, dw=False)
    up = np.arange(rows) % 2 == 0                  # rows with a logit of +infinity; the others' is -infinity
    own = c.target == entry
    assert np.isposinf(lse[up]).all() and np.isneginf(lp[up & ~own]).all() and np.isnan(lp[up & own]).all()
    assert np.isneginf(lp[~up & own]).all()
    # without that entry: log(exp(lse) - exp(z)), which is lower; its bound is the one of the sums before
    z = np.where(up[:, None], 0.0, x @ np.where(np.isinf(w), 0.0, w).T)
    z[:, entry] = -np.inf
    top = z.max(1)
    ref = top + np.log(np.exp(z - top[:, None]).sum(1))
    off = 2.0 ** -24 * 130 * (np.abs(x) @ np.abs(np.where(np.isinf(w), 0.0, w)).T).max(1)
    off += 2.0 ** -20 + 1200 * 2.0 ** -24 + 2.0 ** -22 * (1 + np.abs(ref))
    assert (np.abs(lse - ref) <= off)[~up].all()
    assert np.isfinite(clean[1]).all()


def test_all_of_them(rl, gpu):
    """Every logit +infinity, every one -infinity, and one NaN among the first."""
    c = Case(2, 40, 300, 64, none=0, lean=0.0)
    x, w = np.zeros((40, 64)), np.zeros((300, 64))
    w[:, 0], x[:, 0] = np.inf, np.where(np.arange(40) < 20, 1.0, -1.0)
    c.x, c.w = k8.bits(x, "bf16"), k8.bits(w, "bf16")
    # (the other products are zeros)
    lp, lse, _, _ = c.run(rl, dx=False, dw=False)
    assert np.isposinf(lse[:20]).all() and np.isneginf(lse[20:]).all() and np.isnan(lp).all()
    w[7, 1] = np.nan
    c.w = k8.bits(w, "bf16")
    lp, lse, _, _ = c.run(rl, dx=False, dw=False)
    assert np.isnan(lse).all()


def test_gradient_of_rows_beside(rl, gpu):
    """dw where every row has a logit of -infinity: that entry's is zero, the others' are numbers."""
    c = Case(6, 40, 500, 128, none=0)
    x, w = k8.floats(c.x, "bf16"), k8.floats(c.w, "bf16")
    x[:, 5] = -2.0
    c.target[c.target == 77] = 78
    c.x = k8.bits(x, "bf16")
    w[77, 5] = np.inf
    c.w = k8.bits(w, "bf16")
    lp, lse, dx, dw = c.run(rl)
    assert np.isfinite(lp).all() and np.isfinite(lse).all()
    f = k8.floats(dw, "bf16")
    assert np.isfinite(np.delete(f, 77, 0)).all() and (f[77] == 0).all()

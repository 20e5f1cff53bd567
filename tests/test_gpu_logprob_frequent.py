"""Frequent tokens: what rounding takes from the gradient at the targets is put back for every row of an entry."""
import numpy as np
import pytest

import kv8_helpers as k8
from logprob_rules import Rules
from test_gpu_logprob import E, U, Case

pytestmark = pytest.mark.gpu


def skewed(seed, rows, vocab, hidden, **kw):
    """Targets as tokens are: entry i in proportion to 1 / (i + 1), at places that are mixed."""
    c = Case(seed, rows, vocab, hidden, **kw)
    p = 1.0 / np.arange(1, vocab + 1)
    where = c.rng.permutation(vocab)
    none = c.target >= vocab
    c.target[:] = where[c.rng.choice(vocab, rows, p=p / p.sum())]
    c.target[none] = 0xFFFFFFFF
    return c


def check_dw(c, out):
    """dw alone, to the bounds of Case.check, where every row's element of D at its target is as exact as fp32 products and
    sums leave it (2 E of it): what its rounding takes has at most 16 bits and is put back whole."""
    lse, got = out[1], k8.floats(out[3][:, :c.hidden], "bf16")
    x, w = k8.floats(c.x, "bf16"), k8.floats(c.w, "bf16")
    has = c.target < c.vocab
    t = np.where(has, c.target, 0)
    g = np.where(has, c.grad.astype(np.float64), 0.0) * c.scale
    ref, mag, err = (np.zeros((c.vocab, c.hidden)) for _ in range(3))
    step = max(1, (1 << 25) // c.vocab)
    for r0 in range(0, c.rows, step):
        r = slice(r0, min(c.rows, r0 + step))
        i = np.arange(r.stop - r.start)
        z = x[r] @ w.T * c.scale
        z_off = (c.hidden + 2) * E * c.scale * (np.abs(x[r]) @ np.abs(w).T).max(1)
        top = z.max(1)
        exact = top + np.log(np.exp(z - top[:, None]).sum(1))
        lse_off = z_off + 2.0 ** -20 + 1200 * E + 2.0 ** -22 * (1 + np.abs(exact))
        assert (np.abs(lse[r] - exact) <= lse_off).all()
        p = np.exp(z - exact[:, None])
        d = -p
        d[i, t[r]] += 1.0
        d *= g[r, None]
        e = np.abs(g[r, None]) * p * (z_off + lse_off + 2.0 ** -15)[:, None] + U * 1.01 * np.abs(d)
        e[i, t[r]] -= (U * 1.01 - 2 * E) * np.abs(d[i, t[r]])
        xs = np.where(has[r, None], x[r], 0.0)
        ref += d.T @ xs
        mag += np.abs(d).T @ np.abs(xs)
        err += e.T @ np.abs(xs)
    tol = err + (c.rows + 80) * E * mag + U * 1.01 * np.abs(ref) + 1e-38
    far = np.abs(got - ref)
    assert (far <= tol).all(), (float((far / tol).max()), np.argwhere(~(far <= tol))[:4].tolist())
    return float(np.linalg.norm(got - ref) / np.linalg.norm(ref))


@pytest.mark.parametrize("rows, vocab, hidden, lean", [(129, 40, 64, 5.0), (300, 5000, 192, 5.0), (700, 3000, 320, 0.0),
                                                       (2049, 9000, 128, 5.0), (4500, 700, 64, 2.0)])
def test_frequent_tokens(rl, gpu, rows, vocab, hidden, lean):
    c = skewed(rows + vocab, rows, vocab, hidden, none=0.05, lean=lean)
    out = c.run(rl)
    check_dw(c, out)
    for a, b in zip(out, c.run(rl, graph=2)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("rows", [131, 200])
def test_frequent_tokens_on_the_largest_tiles(rl, gpu, rows):
    c = skewed(rows, rows, 33001, 192, none=0.05)
    assert Rules(gpu.cu_count).dw_kind(192, 33001) == "Dw256"
    check_dw(c, c.run(rl))


@pytest.mark.parametrize("rows", [140, 2048, 2049, 4103])
def test_one_token_alone(rl, gpu, rows):
    """Every row has the same target (the last entry), but for a few without any: as many as are looked at together, one
    more, and several times that."""
    c = Case(rows, rows, 515, 64, none=0.0, lean=0.0)
    c.target[:] = 514
    c.target[[0, 77, rows - 1]] = 0xFFFFFFFF
    check_dw(c, c.run(rl))


def test_how_far_skewed_targets_are_off(rl, gpu):
    """As far from 64 bits as the exact value rounded once, beside what rounding D to bf16 away from the targets leaves. The
    two are independent, so their squares add up; 5% for what fp32 logits (2^-18 of a probability) move."""
    c = skewed(5, 2000, 8000, 128, none=0.0, lean=0.0)
    off = check_dw(c, c.run(rl))
    x, w = k8.floats(c.x, "bf16"), k8.floats(c.w, "bf16")
    z, i = x @ w.T, np.arange(c.rows)
    d = -np.exp(z - np.log(np.exp(z).sum(1))[:, None])
    d[i, c.target] += 1.0
    d *= c.grad.astype(np.float64)[:, None]
    near = k8.floats(k8.bits(d, "bf16"), "bf16")
    near[i, c.target] = d[i, c.target]
    ref = d.T @ x
    once = np.linalg.norm(k8.floats(k8.bits(ref, "bf16"), "bf16") - ref)
    rest = np.linalg.norm(near.T @ x - ref)
    assert off <= 1.05 * np.hypot(once, rest) / np.linalg.norm(ref), (off, once, rest, np.linalg.norm(ref))

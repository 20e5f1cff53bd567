"""rl_hip_token_logprob and its gradient against the formulas in 64 bits."""
import numpy as np
import pytest

import kv8_helpers as k8

pytestmark = pytest.mark.gpu

U = k8.HALF_STEP["bf16"]
E = 2.0 ** -24  # half a step of fp32


class Case:
    def __init__(self, seed, rows, vocab, hidden, scale=1.0, none=0.1, lean=4.0, pad=(0, 0, 0, 0)):
        self.rng = rng = np.random.default_rng(seed)
        self.rows, self.vocab, self.hidden, self.scale, self.pad = rows, vocab, hidden, scale, pad
        self.target = rng.integers(0, vocab, rows).astype(np.uint32)
        w = rng.standard_normal((vocab, hidden), dtype=np.float32) * np.float32(1.28 / hidden ** 0.5)
        x = rng.standard_normal((rows, hidden), dtype=np.float32)
        x += rng.random((rows, 1), dtype=np.float32) * np.float32(lean) * w[self.target]
        if none:
            self.target[rng.random(rows) < none] = 0xFFFFFFFF
            self.target[rng.random(rows) < none / 4] = vocab
        self.x, self.w = k8.bits(x, "bf16"), k8.bits(w, "bf16")
        self.grad = (rng.standard_normal(rows) / rows).astype(np.float32)

    def run(self, rl, lse=None, forward=True, dx=True, dw=True, graph=0):
        up = rl.DeviceBuffer.from_array

        def wide(a, p):
            return np.concatenate([a, np.full((len(a), p), 0x7FC0, np.uint16)], 1) if p else a

        h, p = self.hidden, self.pad
        dev = dict(x=up(wide(self.x, p[0])), w=up(wide(self.w, p[1])), t=up(self.target), g=up(self.grad),
                   lp=up(np.full(self.rows, 77, np.float32)),
                   lse=up(np.full(self.rows, 77, np.float32) if lse is None else lse.astype(np.float32)),
                   dx=up(np.full((self.rows, h + p[2]), 0x1234, np.uint16)),
                   dw=up(np.full((self.vocab, h + p[3]), 0x1234, np.uint16)))
        same = dict(x=dev["x"].ptr, w=dev["w"].ptr, targets=dev["t"].ptr, rows=self.rows, vocab=self.vocab, hidden=h,
                    x_stride=h + p[0], w_stride=h + p[1], scale=self.scale)
        a = rl.TokenLogprobArgs(logprob=dev["lp"].ptr, lse=dev["lse"].ptr, **same)
        g = rl.TokenLogprobGradArgs(lse=dev["lse"].ptr, grad_logprob=dev["g"].ptr, dx=dev["dx"].ptr if dx else None,
                                    dw=dev["dw"].ptr if dw else None, dx_stride=h + p[2], dw_stride=h + p[3], **same)
        dev["wa"] = rl.token_logprob_workspace(a)
        if dx or dw:
            dev["wg"] = rl.token_logprob_grad_workspace(g)
        spaces = [k for k in ("wa", "wg") if k in dev]
        for k in spaces:  # what a workspace holds does not count
            rl.check(rl.lib().rl_hip_memset_d(dev[k].ptr, 0xFF, dev[k].nbytes), "memset")

        def step():
            if forward:
                rl.token_logprob(a)
            if dx or dw:
                rl.token_logprob_grad(g)

        if graph:
            gr = rl.Graph(step)
            for _ in range(graph):
                for k in spaces:
                    rl.check(rl.lib().rl_hip_memset_d(dev[k].ptr, 0xFF, dev[k].nbytes), "memset")
                gr.launch()
                rl.sync()
            gr.close()
        else:
            step()
            rl.sync()
        out = (dev["lp"].download(np.float32, self.rows), dev["lse"].download(np.float32, self.rows),
               dev["dx"].download(np.uint16, (self.rows, h + p[2])), dev["dw"].download(np.uint16, (self.vocab, h + p[3])))
        for b in dev.values():
            b.close()
        return out

    def check(self, out, dx=True, dw=True, targets_whole=False):
        """Bounds. A logit is an fp32 sum of hidden exact products: off by at most z_off = (hidden + 2) E scale sum |x w|.
        Its exponential's argument (rounded twice, at most 88 where the result counts) and the exponential add 2^-16 of
        it at the most where it is smallest, and less than 2^-20 of the sum; sums of up to 128 in a lane, of two lanes
        and of all tiles' add fewer than 1,200 roundings; the logarithm and the last sum 2^-22 (1 + |lse|). So
        lse_off = z_off + 2^-20 + 1200 E + 2^-22 (1 + |lse|), and a logprob z_off + lse_off + 2 E |logprob|. An element of
        D is off by p (z_off + lse_off + 2^-15) |scale g|, then rounded to bf16: U |D|; the products add fp32 sums of
        vocab (or rows) terms and one rounding. targets_whole: but in dx what rounding takes from D at the target is put
        back (its product and sum are off by 2 E of it), in dw too for the first four rows of an entry; with at most 128
        rows dw's D is rounded to 16 bits in two
        parts, U^2 |D| (or 2^-133, below the smallest bf16)."""
        x, w = k8.floats(self.x, "bf16"), k8.floats(self.w, "bf16")
        lp, lse, got_dx, got_dw = out
        has = self.target < self.vocab
        t = np.where(has, self.target, 0)
        g_all = np.where(has, self.grad.astype(np.float64), 0.0) * self.scale
        ref_dw, mag_dw, err_dw = (np.zeros((self.vocab, self.hidden)) for _ in range(3))
        step = max(1, (1 << 25) // self.vocab)
        for r0 in range(0, self.rows, step):
            r = slice(r0, min(self.rows, r0 + step))
            i = np.arange(r.stop - r.start)
            z = x[r] @ w.T * self.scale
            z_off = (self.hidden + 2) * E * self.scale * (np.abs(x[r]) @ np.abs(w).T).max(1)
            top = z.max(1)
            ref = top + np.log(np.exp(z - top[:, None]).sum(1))
            lse_off = z_off + 2.0 ** -20 + 1200 * E + 2.0 ** -22 * (1 + np.abs(ref))
            assert (np.abs(lse[r] - ref) <= lse_off).all(), float((np.abs(lse[r] - ref) / lse_off).max())
            ref_lp = np.where(has[r], z[i, t[r]] - ref, 0.0)
            off = np.where(has[r], z_off + lse_off + 2 * E * np.abs(ref_lp), 0.0)
            assert (np.abs(lp[r] - ref_lp) <= off).all(), float((np.abs(lp[r] - ref_lp) / (off + 1e-30)).max())
            if not (dx or dw):
                continue
            p = np.exp(z - ref[:, None])
            d = -p
            d[i, t[r]] += 1.0
            d *= g_all[r, None]
            e = np.abs(g_all[r, None]) * p * (z_off + lse_off + 2.0 ** -15)[:, None] + U * 1.01 * np.abs(d)
            if dx:
                want, mag = d @ w, np.abs(d) @ np.abs(w)
                e_dx = e.copy()
                if targets_whole:
                    e_dx[i, t[r]] -= (U * 1.01 - 2 * E) * np.abs(d[i, t[r]])
                tol = e_dx @ np.abs(w) + (self.vocab + 16) * E * mag + U * 1.01 * np.abs(want) + 1e-38
                far = np.abs(k8.floats(got_dx[r, :self.hidden], "bf16") - want)
                tol[~has[r]] = 0
                assert (far <= tol).all(), (r0, float((far / (tol + 1e-300)).max()), np.argwhere(~(far <= tol))[:4].tolist())
            if dw:
                xs = np.where(has[r, None], x[r], 0.0)
                if targets_whole and self.rows <= 128:
                    e = e - U * 1.01 * np.abs(d) + 1.01 * U * U * np.abs(d) + 2.0 ** -133
                elif targets_whole:
                    first = np.array([(self.target[:r0 + k] == self.target[r0 + k]).sum() < 4 for k in i])
                    e[i, t[r]] -= np.where(has[r] & first, (U * 1.01 - 2 * E) * np.abs(d[i, t[r]]), 0.0)
                ref_dw += d.T @ xs
                mag_dw += np.abs(d).T @ np.abs(xs)
                err_dw += e.T @ np.abs(xs)
        if dw:
            tol = err_dw + (self.rows + 80) * E * mag_dw + U * 1.01 * np.abs(ref_dw) + 1e-38
            far = np.abs(k8.floats(got_dw[:, :self.hidden], "bf16") - ref_dw)
            assert (far <= tol).all(), (float((far / (tol + 1e-300)).max()), np.argwhere(~(far <= tol))[:4].tolist())


@pytest.mark.parametrize("rows", [1, 7, 31, 32, 33, 64, 65, 100, 128, 129, 200, 256, 257, 500])
@pytest.mark.parametrize("vocab, hidden", [(1000, 128), (513, 320)])
def test_sizes(rl, gpu, rows, vocab, hidden):
    c = Case(rows + vocab, rows, vocab, hidden)
    c.check(c.run(rl))


@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 255, 256, 257, 4099])
@pytest.mark.parametrize("rows", [5, 300])
def test_vocabularies(rl, gpu, vocab, rows):
    c = Case(vocab, rows, vocab, 64, scale=0.7)
    c.check(c.run(rl))


@pytest.mark.parametrize("hidden", [64, 192, 448, 1024, 2112])
@pytest.mark.parametrize("rows", [20, 40, 90, 150, 290])
def test_hidden(rl, gpu, hidden, rows):
    c = Case(hidden, rows, 700, hidden, scale=1.25)
    c.check(c.run(rl))


@pytest.mark.parametrize("rows, vocab", [(1, 700), (2, 9000), (20, 3000), (33, 500), (60, 30000), (64, 2000), (100, 700),
                                         (128, 20000), (129, 900), (300, 500), (1000, 300)])
@pytest.mark.parametrize("lean", [0.0, 5.0])
def test_what_rounding_takes_at_the_targets(rl, gpu, rows, vocab, lean):
    """A gradient that is mostly one element of D times a row is not off by that element's rounding to bf16."""
    c = Case(rows + vocab, rows, vocab, 192, none=0.05 if rows > 2 else 0, lean=lean)
    c.check(c.run(rl), targets_whole=True)


@pytest.mark.parametrize("rows, vocab, hidden", [(129, 5000, 192), (200, 300, 64), (700, 2000, 320), (1500, 9, 128)])
def test_what_rounding_takes_from_many_rows(rl, gpu, rows, vocab, hidden):
    """The same with more rows than have D in two parts, entries with up to hundreds of rows, and rows that repeat."""
    c = Case(rows, rows, vocab, hidden, none=0.05, lean=5.0)
    c.target[rows // 2:rows // 2 + 7] = c.target[0] = 3
    out = c.run(rl)
    c.check(out, targets_whole=True)
    for a, b in zip(out, c.run(rl, graph=2)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("rows, vocab", [(500, 32001), (300, 40000), (200, 31990), (490, 16001), (1000, 4500), (120, 30001),
                                         (300, 8000), (61, 30003), (100, 15000), (70, 2000), (33, 300), (161, 1030)])
def test_tiles(rl, gpu, rows, vocab):
    """Every kind of tiles, with several along the rows and the last ones partly filled."""
    c = Case(rows, rows, vocab, 128, none=0.05)
    c.check(c.run(rl))


@pytest.mark.parametrize("rows, vocab, hidden", [(24, 9000, 512), (130, 9000, 256), (1100, 3000, 512)])
def test_shares_of_the_vocabulary(rl, gpu, rows, vocab, hidden):
    """dx in shares that are joined; the same bits at every replay."""
    c = Case(rows, rows, vocab, hidden)
    out = c.run(rl)
    c.check(out)
    for a, b in zip(out, c.run(rl, graph=3)):
        assert np.array_equal(a, b)


def test_pieces_of_the_vocabulary(rl, gpu):
    """So many rows that the vocabulary is taken in two pieces, the second of another size."""
    c = Case(9, 65600, 2000, 64, none=0.02)
    c.check(c.run(rl))


def test_no_target_at_all(rl, gpu):
    c = Case(10, 70, 300, 128)
    c.target[:] = 0xFFFFFFFF
    out = c.run(rl)
    c.check(out)
    assert not out[0].any() and not out[2].any() and not (out[3] & 0x7FFF).any()


@pytest.mark.parametrize("rows", [20, 40, 100, 200, 400])
def test_rows_without_target_hold_anything(rl, gpu, rows):
    """NaN and infinities in rows without a target change nothing else, whether they come first, between or last."""
    c = Case(rows, rows, 600, 192, none=0.3)
    c.target[[0, rows - 1]] = 0xFFFFFFFF
    clean = c.run(rl)
    c.check(clean)
    none = c.target >= c.vocab
    c.x[none] = np.where(c.rng.random((int(none.sum()), 192)) < 0.5, 0x7FC0, 0x7F80)
    c.grad[none] = np.nan
    lp, lse, dx, dw = c.run(rl)
    assert np.array_equal(lp, clean[0]) and np.array_equal(lse[~none], clean[1][~none])
    assert np.array_equal(dx, clean[2]) and np.array_equal(dw, clean[3])


@pytest.mark.parametrize("rows", [9, 300])
def test_values_that_are_no_numbers(rl, gpu, rows):
    """A NaN in a row with a target is that row's alone, but for dw; one in w is everyone's."""
    c = Case(3, rows, 500, 128, none=0)
    clean = c.run(rl)
    c.x[4, 17] = 0x7FC0
    lp, lse, dx, dw = c.run(rl)
    rest = np.arange(rows) != 4
    assert np.isnan(lp[4]) and np.isnan(lse[4]) and np.isnan(k8.floats(dx[4], "bf16")).all()
    assert np.array_equal(lp[rest], clean[0][rest]) and np.array_equal(dx[rest], clean[2][rest])
    assert np.isnan(k8.floats(dw, "bf16")).all()
    c.x[4, 17] = 0
    c.w[499, 5] = 0x7FC0
    lp, lse, dx, dw = c.run(rl)
    assert np.isnan(lp).all() and np.isnan(k8.floats(dx, "bf16")).all()


def test_steep_logits(rl, gpu):
    """Rows all but sure of their token, and rows that all but rule it out."""
    c = Case(11, 90, 2000, 256, none=0, lean=40.0)
    c.x[::2] = k8.bits(-k8.floats(c.x[::2], "bf16"), "bf16")
    out = c.run(rl)
    c.check(out)
    assert out[0].max() > -1e-3 and out[0].min() < -30


@pytest.mark.parametrize("rows,vocab", [(1, 4000), (24, 4000), (50, 8000), (100, 16000), (200, 32000)])
def test_small_products_beside_a_large_one(rl, gpu, rows, vocab):
    """Every logit is one product of 2^12 and 4,095 of 2^-17. The matrix instruction adds sixteen of these, 2^-13, at a
    time: to 2^12 in 32 bits they are lost, all 256 of them if the large one comes first. Sums of 512 products are exact
    unless the large one is among them (512 x 2^-17 lost at most), and each of the eight is added to within half a step
    of 2^12, 2^-12; so is the logarithm of the entries' number, off by less than 2^-18 with the exponentials' sum."""
    c = Case(21, rows, vocab, 4096, none=0.0)
    w = np.full((1, 4096), 2.0 ** -17, np.float32)
    x = np.ones((rows, 4096), np.float32)
    w[0, 0] = x[:, 0] = 64.0
    c.w, c.x = np.ascontiguousarray(np.repeat(k8.bits(w, "bf16"), vocab, 0)), k8.bits(x, "bf16")
    lp, lse, _, _ = c.run(rl, dx=False, dw=False)
    ref = 4096 + 4095 * 2.0 ** -17 + np.log(vocab)
    off = 512 * 2.0 ** -17 + 8 * 2.0 ** -12 + 2.0 ** -12 + 2.0 ** -18
    assert (np.abs(lse - ref) <= off).all(), float(np.abs(lse - ref).max() / off)


def test_strides(rl, gpu):
    c = Case(12, 150, 400, 192)
    plain = c.run(rl)
    for pad in ((8, 16, 24, 32), (64, 0, 8, 0)):
        c.pad = pad
        out = c.run(rl)
        assert np.array_equal(out[0], plain[0]) and np.array_equal(out[1], plain[1])
        assert np.array_equal(out[2][:, :192], plain[2]) and (out[2][:, 192:] == 0x1234).all()
        assert np.array_equal(out[3][:, :192], plain[3]) and (out[3][:, 192:] == 0x1234).all()


@pytest.mark.parametrize("rows", [30, 300])
def test_one_gradient(rl, gpu, rows):
    c = Case(13, rows, 900, 128)
    lp, lse, dx, dw = c.run(rl)
    only = c.run(rl, dw=False)
    assert np.array_equal(only[2], dx) and (only[3] == 0x1234).all()
    only = c.run(rl, dx=False, lse=lse, forward=False)
    assert np.array_equal(only[3], dw) and (only[2] == 0x1234).all() and (only[0] == 77).all()
    only = c.run(rl, dx=False, dw=False)
    assert np.array_equal(only[0], lp) and (only[3] == 0x1234).all()


def test_differences(rl, gpu):
    """The gradient of sum g logprob against differences of the formula in 64 bits."""
    c = Case(14, 6, 80, 64, scale=1.25)
    _, _, dx, dw = c.run(rl)
    x, w = k8.floats(c.x, "bf16"), k8.floats(c.w, "bf16")
    has = c.target < c.vocab

    def loss(x, w):
        z = x @ w.T * c.scale
        lse = np.log(np.exp(z).sum(1))
        return (c.grad * np.where(has, z[np.arange(6), np.where(has, c.target, 0)] - lse, 0)).sum()

    for got, a, at in ((dx, x, [(i, j) for i in range(6) for j in (0, 13, 63)]),
                       (dw, w, [(int(c.target[i]) if has[i] else 3, j) for i in range(6) for j in (2, 40)])):
        f = k8.floats(got, "bf16")
        for i, j in at:
            step = np.zeros_like(a)
            step[i, j] = 1e-4
            up = loss(x + step, w) if a is x else loss(x, w + step)
            down = loss(x - step, w) if a is x else loss(x, w - step)
            # a central difference is off by the third derivative times 1e-8; D and the result are rounded to bf16
            assert abs(f[i, j] - (up - down) / 2e-4) <= 3 * U * np.abs(f).max() + 1e-7


def test_against_projection_and_sampler(rl, gpu):
    """The logprob of a sampled token: rl_hip_logits_proj and rl_hip_sample's, at the same temperature."""
    rows, vocab, hidden, temp = 50, 3000, 512, 0.8
    c = Case(15, rows, vocab, hidden, scale=1 / temp, none=0)
    up = rl.DeviceBuffer.from_array
    x, w = up(c.x), up(c.w)
    lg, tok, lp = (rl.DeviceBuffer(n) for n in (rows * vocab * 4, rows * 4, rows * 4))
    rl.logits_proj(x, w, lg, rows, vocab, hidden)
    s = rl.sample_args(lg, rows, vocab, vocab, tok, lp, temperature=temp, seed=5, step=1)
    ws = rl.sample_workspace(s)
    rl.sample(s)
    rl.sync()
    c.target = tok.download(np.uint32, rows)
    want = lp.download(np.float32, rows)
    got = c.run(rl, dx=False, dw=False)[0]
    # the sampler's logprobs are within 1e-4 of 64 bits, these within the bound of `check`
    c.check((got, c.run(rl, dx=False, dw=False)[1], None, None), dx=False, dw=False)
    assert np.abs(got - want).max() <= 2e-4
    for b in (x, w, lg, tok, lp, ws):
        b.close()


def test_workspaces(rl, gpu):
    """The workspace of the largest call serves smaller ones; a smaller one is refused."""
    P = 4096

    def grad(rows, vocab, hidden, **kw):
        return rl.TokenLogprobGradArgs(x=P, w=P, targets=P, rows=rows, vocab=vocab, hidden=hidden, x_stride=hidden,
                                       w_stride=hidden, lse=P, grad_logprob=P, dx=P, dw=P, dx_stride=hidden,
                                       dw_stride=hidden, **kw)

    def forward(rows, vocab, hidden, **kw):
        return rl.TokenLogprobArgs(x=P, w=P, targets=P, rows=rows, vocab=vocab, hidden=hidden, x_stride=hidden,
                                   w_stride=hidden, logprob=P, lse=P, **kw)

    for make, need in ((grad, rl.token_logprob_grad_workspace_bytes), (forward, rl.token_logprob_workspace_bytes)):
        for big in ((4096, 128256, 4096), (300, 32000, 2048), (100, 5000, 512)):
            most = need(make(*big))
            for r in (1, 32, 33, 64, 128, 129, 200, 256, 257, 300, 1000, 4096):
                for v in (1, 100, 5000, 32000, 128256):
                    for h in (64, 512, 2048, 4096):
                        if r <= big[0] and v <= big[1] and h <= big[2]:
                            assert need(make(r, v, h)) <= most, (big, r, v, h)
    with pytest.raises(rl.RlrtError, match="workspace"):
        rl.token_logprob(forward(10, 100, 64, workspace=P, workspace_bytes=16))
    with pytest.raises(rl.RlrtError, match="workspace"):
        rl.token_logprob_grad(grad(10, 100, 64, workspace=P, workspace_bytes=16))
    with pytest.raises(rl.RlrtError, match="workspace"):
        rl.token_logprob_grad(grad(10, 100, 64, workspace=None, workspace_bytes=1 << 30))


def test_offsets_past_4_gib(rl, gpu):
    """A row of the projection behind 4 GiB."""
    rows, vocab, hidden, stride = 3, 1300, 64, 1 << 21
    c = Case(16, rows, vocab, hidden, none=0)
    c.target[:] = [1299, 0, 1100]
    want = c.run(rl)
    up = rl.DeviceBuffer.from_array
    w = rl.DeviceBuffer(vocab * stride * 2)
    for v in range(vocab):
        w.upload(c.w[v], v * stride * 2)
    dev = [up(c.x), up(c.target), up(c.grad), rl.DeviceBuffer(rows * 4), rl.DeviceBuffer(rows * 4),
           rl.DeviceBuffer(rows * hidden * 2), rl.DeviceBuffer(vocab * hidden * 2)]
    same = dict(x=dev[0].ptr, w=w.ptr, targets=dev[1].ptr, rows=rows, vocab=vocab, hidden=hidden, x_stride=hidden,
                w_stride=stride, scale=1.0)
    a = rl.TokenLogprobArgs(logprob=dev[3].ptr, lse=dev[4].ptr, **same)
    g = rl.TokenLogprobGradArgs(lse=dev[4].ptr, grad_logprob=dev[2].ptr, dx=dev[5].ptr, dw=dev[6].ptr, dx_stride=hidden,
                                dw_stride=hidden, **same)
    ws = [rl.token_logprob_workspace(a), rl.token_logprob_grad_workspace(g)]
    rl.token_logprob(a)
    rl.token_logprob_grad(g)
    rl.sync()
    assert np.array_equal(dev[3].download(np.float32, rows), want[0])
    assert np.array_equal(dev[5].download(np.uint16, (rows, hidden)), want[2])
    assert np.array_equal(dev[6].download(np.uint16, (vocab, hidden)), want[3])
    for b in dev + ws + [w]:
        b.close()

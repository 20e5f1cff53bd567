"""rl_hip_attn_prompt against attention in 64 bits, and a prompt taken through
the whole path: prompt attention, the 8-bit cache, decode steps."""
import ctypes as C

import numpy as np
import pytest

import kv8_helpers as k8

pytestmark = pytest.mark.gpu


def tolerance(dtype, ref, mag, q, k, scale, n):
    """What rounding may do to an output o = sum w_j v_j / sum w_j of n keys. The weights are rounded to 16 bits (half a
    step u each; fp16 weights below 2^-14 by at most 2^-25, relative to a largest weight of 1 or more) and the output
    once more (u |o|): u (mag + |o|), mag = sum w_j |v_j| / sum w_j. A score is a sum of head_dim fp32 products, off by
    at most (head_dim + 2) 2^-24 scale sum |q k|, which moves a weight and the sum of weights by that much relatively
    (2 x mag); exp2, the fp32 sums over n keys and the division add less than (n + 16) 2^-24 mag."""
    u = k8.HALF_STEP[dtype]
    d = q.shape[-1]
    score = (d + 2) * 2.0 ** -24 * scale * np.abs(q).sum(-1).max() * np.abs(k).max()
    small = n * 2.0 ** -25 if dtype == "fp16" else 0.0
    return u * (mag + np.abs(ref)) * 1.01 + (2 * score + (n + 16) * 2.0 ** -24) * mag + small * mag.max(initial=0) + 1e-30


def compare(got, q, k, v, q_starts, kv_starts, kvh, dtype, scale=None, rows=None):
    """got, q [tokens][heads][d], k, v [tokens][kv heads][d] as 16-bit arrays."""
    f = [k8.floats(x, dtype) for x in (got, q, k, v)]
    group, d = q.shape[1] // kvh, q.shape[2]
    scale = scale or d ** -0.5
    for s in range(len(q_starts) - 1):
        a, b, c, e = q_starts[s], q_starts[s + 1], kv_starts[s], kv_starts[s + 1]
        seen = [i + 1 + (e - c) - (b - a) for i in range(b - a)]
        for h in range(q.shape[1]):
            kk, vv = f[2][c:e, h // group], f[3][c:e, h // group]
            ref, mag = k8.attend(f[1][a:b, h], kk, vv, scale, seen)
            if b > a:
                tol = tolerance(dtype, ref, mag, f[1][a:b, h], kk if e > c else np.zeros((1, d)), scale, e - c)
                off = np.abs(f[0][a:b, h] - ref)
                assert (off <= tol).all(), (s, h, float(np.nanmax(off / tol)), np.argwhere(~(off <= tol))[:4].tolist())


def inputs(rng, nq, nk, qh, kvh, d, dtype, q_size=1.0):
    return (k8.bits(rng.standard_normal((nq, qh, d)) * q_size, dtype), k8.bits(rng.standard_normal((nk, kvh, d)), dtype),
            k8.bits(rng.standard_normal((nk, kvh, d)), dtype))


def starts_of(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(int).tolist()


def run(rl, q, k, v, qs, kvh, dtype, **kw):
    n, qh, d = q.shape
    out = k8.run_prompt(rl, q.reshape(n, -1), k.reshape(len(k), -1), v.reshape(len(v), -1), qs, qh, kvh, d, dtype, **kw)
    return out


@pytest.mark.parametrize("d, qh, kvh, dtype", [(128, 8, 2, "bf16"), (64, 4, 4, "fp16"), (128, 8, 1, "fp16"),
                                               (64, 6, 2, "bf16"), (128, 2, 2, "bf16")])
@pytest.mark.parametrize("lens", [[1], [0, 1, 2, 0], [63, 64, 65], [127, 0, 128, 129], [300, 5]])
def test_packed(rl, gpu, d, qh, kvh, dtype, lens):
    rng = np.random.default_rng(sum(lens) + d)
    qs = starts_of(lens)
    q, k, v = inputs(rng, qs[-1], qs[-1], qh, kvh, d, dtype)
    out = run(rl, q, k, v, qs, kvh, dtype)
    compare(out.reshape(q.shape), q, k, v, qs, qs, kvh, dtype)


@pytest.mark.parametrize("d, qh, kvh, dtype", [(128, 16, 2, "bf16"), (64, 4, 4, "fp16")])
def test_pieces(rl, gpu, d, qh, kvh, dtype):
    """Queries that are the last tokens of longer sequences; a sequence with fewer keys than queries (its first queries
    see none and yield zeros), and one without keys."""
    rng = np.random.default_rng(7)
    nq, nk = [1, 17, 40, 5, 3, 64], [200, 17, 333, 2, 0, 1000]
    qs, ks = starts_of(nq), starts_of(nk)
    q, k, v = inputs(rng, qs[-1], ks[-1], qh, kvh, d, dtype)
    out = run(rl, q, k, v, qs, kvh, dtype, kv_starts=ks).reshape(q.shape)
    compare(out, q, k, v, qs, ks, kvh, dtype)
    assert not out[qs[3]:qs[3] + 3].any() and not out[qs[4]:qs[5]].any()


@pytest.mark.parametrize("d, kvh, dtype", [(128, 1, "bf16"), (64, 3, "fp16")])
def test_tile_counts(rl, gpu, d, kvh, dtype):
    """Sequences of two to eight tiles, whole and not, and equal ones: every order of the kinds of steps."""
    rng = np.random.default_rng(d)
    lens = [128, 192, 193, 256, 319, 320, 385, 448, 192, 512]
    qs = starts_of(lens)
    q, k, v = inputs(rng, qs[-1], qs[-1], 2 * kvh, kvh, d, dtype)
    out = run(rl, q, k, v, qs, kvh, dtype)
    compare(out.reshape(q.shape), q, k, v, qs, qs, kvh, dtype)
    assert np.array_equal(run(rl, q, k, v, qs, kvh, dtype, graph=3), out)


def test_many_sequences(rl, gpu):
    """More sequences than are put in order, most of one or two tokens, and a key group that no XCD count divides."""
    rng = np.random.default_rng(70)
    lens = rng.integers(0, 4, 90).tolist()
    lens[33], lens[88] = 140, 77
    qs = starts_of(lens)
    q, k, v = inputs(rng, qs[-1], qs[-1], 9, 3, 64, "bf16")
    out = run(rl, q, k, v, qs, 3, "bf16")
    compare(out.reshape(q.shape), q, k, v, qs, qs, 3, "bf16")


@pytest.mark.parametrize("seqs", [2, 63, 64])
def test_sequences_in_order(rl, gpu, seqs):
    """As many sequences as are put in order, by lengths that are equal, nearly equal, none and far apart."""
    rng = np.random.default_rng(seqs)
    lens = rng.choice([0, 1, 2, 30, 31, 64, 130], seqs)
    lens[seqs - 1] = 700
    qs = starts_of(lens.tolist())
    q, k, v = inputs(rng, qs[-1], qs[-1], 4, 2, 64, "bf16")
    out = run(rl, q, k, v, qs, 2, "bf16")
    compare(out.reshape(q.shape), q, k, v, qs, qs, 2, "bf16")


@pytest.mark.parametrize("max_q", [1024, 1025])
def test_sequences_in_batch_order(rl, gpu, max_q):
    """At most 64 sequences, with as many row blocks as they are put in order by length for, and more."""
    rng = np.random.default_rng(max_q)
    lens = rng.choice([0, 1, 17, 64, 129], 64)
    lens[[7, 63]] = 300, 0
    qs = starts_of(lens.tolist())
    q, k, v = inputs(rng, qs[-1], qs[-1], 8, 8, 64, "fp16")
    out = run(rl, q, k, v, qs, 8, "fp16", max_q=max_q)
    compare(out.reshape(q.shape), q, k, v, qs, qs, 8, "fp16")


@pytest.mark.parametrize("seqs, longest", [(130, 9300), (200, 6200), (20, 9300)])
def test_one_long_among_short(rl, gpu, seqs, longest):
    """More row blocks than half the compute units share the keys of the one long sequence, one or two workgroups each."""
    rng = np.random.default_rng(seqs)
    lq, lk = rng.integers(1, 4, seqs), rng.integers(3, 40, seqs)
    lk[seqs // 3] = longest
    qs, ks = starts_of(lq.tolist()), starts_of(lk.tolist())
    q, k, v = inputs(rng, qs[-1], ks[-1], 2, 1, 64, "fp16")
    out = run(rl, q, k, v, qs, 1, "fp16", kv_starts=ks)
    compare(out.reshape(q.shape), q, k, v, qs, ks, 1, "fp16")
    assert np.array_equal(run(rl, q, k, v, qs, 1, "fp16", kv_starts=ks, graph=2), out)


@pytest.mark.parametrize("n, kvh", [(1500, 2), (2100, 1)])
def test_long(rl, gpu, n, kvh):
    rng = np.random.default_rng(n)
    q, k, v = inputs(rng, n, n, 2, kvh, 128, "bf16")
    out = run(rl, q, k, v, [0, n], kvh, "bf16").reshape(q.shape)
    compare(out, q, k, v, [0, n], [0, n], kvh, "bf16")


def test_few_queries_long_context(rl, gpu):
    """One and three queries behind thousands of keys; the same bits at every replay."""
    rng = np.random.default_rng(12)
    nq, nk = [1, 3], [7001, 5000]
    qs, ks = starts_of(nq), starts_of(nk)
    q, k, v = inputs(rng, 4, ks[-1], 4, 1, 128, "bf16")
    out = run(rl, q, k, v, qs, 1, "bf16", kv_starts=ks)
    compare(out.reshape(q.shape), q, k, v, qs, ks, 1, "bf16")
    assert np.array_equal(run(rl, q, k, v, qs, 1, "bf16", kv_starts=ks, graph=3), out)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_steep_scores(rl, gpu, dtype):
    """Scores that climb along the keys (the reference maximum rises tile by tile), and large ones where a key takes all."""
    rng = np.random.default_rng(3)
    n, d = 400, 128
    q, k, v = inputs(rng, n, n, 2, 1, d, dtype)
    fk = k8.floats(k, dtype) * np.linspace(0.05, 6, n)[:, None, None]
    fk[:, 0, 0] = np.linspace(0, 40, n)
    fq = k8.floats(q, dtype)
    fq[:, 0, 0] = 4.0
    q, k = k8.bits(fq, dtype), k8.bits(fk, dtype)
    out = run(rl, q, k, v, [0, n], 1, dtype).reshape(q.shape)
    compare(out, q, k, v, [0, n], [0, n], 1, dtype)


@pytest.mark.parametrize("d", [128, 64])
def test_what_is_not_seen_has_no_part(rl, gpu, d):
    """NaN and infinities in keys and values: rows that do not see them are as without them, rows that do are not numbers
    where the values are not. Also in the next sequence and behind the last one."""
    rng = np.random.default_rng(8)
    lens, dtype = [100, 150], "bf16"
    qs = starts_of(lens)
    q, k, v = inputs(rng, 300, 300, 4, 2, d, dtype)
    clean = run(rl, q, k, v, qs, 2, dtype).reshape(q.shape)
    bad_k, bad_v = k8.floats(k, dtype), k8.floats(v, dtype)
    bad_v[70, 0, 3] = np.nan       # sequence 0, key 70, KV head 0, dim 3
    bad_v[90, 1, 5] = np.inf
    bad_k[180, 1, 2] = np.nan      # sequence 1, key 80
    bad_v[250:], bad_k[250:] = np.nan, np.inf
    bad_k[100 + 149] = np.nan      # the last key of the last sequence
    out = run(rl, q, k8.bits(bad_k, dtype), k8.bits(bad_v, dtype), qs, 2, dtype).reshape(q.shape)
    f, c = k8.floats(out, dtype), k8.floats(clean, dtype)
    tol = 3 * k8.HALF_STEP[dtype] * np.abs(c) + 2 * k8.HALF_STEP[dtype]  # (rows computed again round their weights otherwise)
    same = np.abs(f - c) <= tol
    assert same[:70].all() and same[100:180].all() and same[180:249, :2].all()
    assert np.isnan(f[70:100, :2, 3]).all() and same[70:100, :2][..., np.arange(d) != 3].all()
    assert np.isposinf(f[90:100, 2:, 5]).all() and same[90:100, 2:][..., np.arange(d) != 5].all() and same[70:90, 2:].all()
    assert np.isnan(f[180:249, 2:]).all() and np.isnan(f[249]).all()


def test_shares_and_what_is_not_seen(rl, gpu):
    """The same where workgroups share a row's keys: the last queries of a long sequence, a value that is no number among
    the keys that only the last one sees, and one that all see."""
    rng = np.random.default_rng(18)
    nq, nk = 5, 3000
    q, k, v = inputs(rng, nq, nk, 4, 1, 128, "bf16")
    clean = k8.floats(run(rl, q, k, v, [0, nq], 1, "bf16", kv_starts=[0, nk]).reshape(q.shape), "bf16")
    bad = k8.floats(v, "bf16")
    bad[nk - 1, 0, 7] = np.nan
    bad[nk - 2, 0, 8] = -np.inf
    bad[1000, 0, 9] = np.inf
    f = k8.floats(run(rl, q, k, k8.bits(bad, "bf16"), [0, nq], 1, "bf16", kv_starts=[0, nk]).reshape(q.shape), "bf16")
    tol = 3 * k8.HALF_STEP["bf16"] * np.abs(clean) + 2 * k8.HALF_STEP["bf16"]
    same = np.abs(f - clean) <= tol
    assert np.isposinf(f[:, :, 9]).all() and np.isnan(f[4, :, 7]).all() and np.isneginf(f[3:, :, 8]).all()
    seen = np.ones(f.shape, bool)
    seen[:, :, 9] = seen[4, :, 7] = seen[3:, :, 8] = False
    assert same[seen].all()


@pytest.mark.parametrize("dtype, d", [("bf16", 128), ("fp16", 128), ("fp16", 64), ("bf16", 64)])
def test_values_that_are_no_numbers_early(rl, gpu, dtype, d):
    """A NaN in a value that every row sees, one that only the later ones see, infinities beside them and in every value of
    a dim: each in its own dims, all the others as without them."""
    rng = np.random.default_rng(17)
    n, qh, qs = 1300, 4, [0, 1300]
    q, k, v = inputs(rng, n, n, qh, 1, d, dtype)
    clean = run(rl, q, k, v, qs, 1, dtype).reshape(q.shape)
    bad = k8.floats(v, dtype)
    bad[0, 0, 3], bad[700, 0, 9], bad[700, 0, 11], bad[:, 0, 20] = np.nan, np.nan, -np.inf, np.inf
    out = run(rl, q, k, k8.bits(bad, dtype), qs, 1, dtype).reshape(q.shape)
    f = k8.floats(out, dtype)
    assert np.isnan(f[:, :, 3]).all() and np.isnan(f[700:, :, 9]).all() and np.isneginf(f[700:, :, 11]).all()
    assert np.isposinf(f[:, :, 20]).all()
    out[:, :, [3, 20]], out[700:, :, [9, 11]] = clean[:, :, [3, 20]], clean[700:, :, [9, 11]]
    compare(clean, q, k, v, qs, qs, 1, dtype)
    compare(out, q, k, v, qs, qs, 1, dtype)
    # where no row's last tiles hold one, the others keep their bits (in fp16 such rows are computed again)
    bad = k8.floats(v, dtype)
    bad[0, 0, 3] = np.nan
    out = run(rl, q, k, k8.bits(bad, dtype), qs, 1, dtype).reshape(q.shape)
    assert dtype == "fp16" or np.array_equal(np.delete(out, 3, 2), np.delete(clean, 3, 2))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("nq, nk", [(1, 710), (3, 710), (70, 70), (2, 64), (1, 1), (5, 2501)])
def test_infinity_in_the_last_value(rl, gpu, dtype, nq, nk):
    """The last key, which a tile may hold more than once, has infinite values: so has the only row that sees it."""
    q, k, v = inputs(np.random.default_rng(nk), nq, nk, 4, 2, 128, dtype)
    clean = run(rl, q, k, v, [0, nq], 2, dtype, kv_starts=[0, nk]).reshape(q.shape)
    bad = k8.floats(v, dtype)
    bad[-1, 0, 33], bad[-1, 1, 4] = np.inf, -np.inf
    out = run(rl, q, k, k8.bits(bad, dtype), [0, nq], 2, dtype, kv_starts=[0, nk]).reshape(q.shape)
    f = k8.floats(out, dtype)
    assert np.isposinf(f[-1, :2, 33]).all() and np.isneginf(f[-1, 2:, 4]).all()
    out[-1, :2, 33], out[-1, 2:, 4] = clean[-1, :2, 33], clean[-1, 2:, 4]
    compare(out, q, k, v, [0, nq], [0, nk], 2, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_infinity_of_little_weight(rl, gpu, dtype):
    """A seen infinity whose weight, 2^-40 of the largest, fp16 does not hold: the outputs are infinite, not NaN. Whole
    prompts, and the last queries behind keys that workgroups share."""
    rng = np.random.default_rng(19)
    n, d = 900, 64
    q, k, v = inputs(rng, n, n, 2, 1, d, dtype)
    fq, fk, fv = (k8.floats(x, dtype) for x in (q, k, v))
    fq[:] = fk[:] = 0.0
    fq[:, :, 0], fk[1:, 0, 0] = 8.0, 28.0  # scores 0 for key 0 and 28 (2^40.4) for the others
    fv[0, 0, 6], fv[0, 0, 7] = np.inf, -np.inf
    q, k, v = (k8.bits(x, dtype) for x in (fq, fk, fv))
    f = k8.floats(run(rl, q, k, v, [0, n], 1, dtype).reshape(q.shape), dtype)
    assert np.isposinf(f[:, :, 6]).all() and np.isneginf(f[:, :, 7]).all() and np.isfinite(np.delete(f, [6, 7], 2)).all()
    f = k8.floats(run(rl, q[-3:], k, v, [0, 3], 1, dtype, kv_starts=[0, n]).reshape(3, 2, d), dtype)
    assert np.isposinf(f[:, :, 6]).all() and np.isneginf(f[:, :, 7]).all() and np.isfinite(np.delete(f, [6, 7], 2)).all()


@pytest.mark.parametrize("nq, nk", [(3000, 3000), (16, 6000)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_values_that_are_no_numbers_cost_little(rl, gpu, dtype, nq, nk):
    """A NaN in the first value, and infinities in a dim of all: the call takes a few times as long as without them, not
    hundreds of times (each of its rows again, key by key)."""
    d, qh, kvh = 128, 8, 2
    q, k, v = inputs(np.random.default_rng(23), nq, nk, qh, kvh, d, dtype)
    up = rl.DeviceBuffer.from_array
    dev = [up(q), up(k), up(v), up(np.zeros_like(q)), up(np.array([0, nq], np.uint32)), up(np.array([0, nk], np.uint32))]
    args = rl.AttnPromptArgs(q=dev[0].ptr, k=dev[1].ptr, v=dev[2].ptr, out=dev[3].ptr, q_starts=dev[4].ptr,
                             kv_starts=dev[5].ptr, seqs=1, q_tokens=nq, kv_tokens=nk, max_q=nq, max_kv=nk, q_heads=qh,
                             kv_heads=kvh, head_dim=d, dtype=k8.dtype_id(rl, dtype))
    ws = rl.attn_prompt_workspace(args)
    timer = rl.Timer()

    def least():
        times = []
        for _ in range(6):
            timer.begin()
            rl.attn_prompt(args)
            times.append(timer.end())
        return min(times)

    clean = least()
    for rows, what in ((0, np.nan), (slice(None), np.inf)):
        bad = k8.floats(v, dtype)
        bad[rows, :, 5] = what
        dev[2].upload(k8.bits(bad, dtype))
        assert least() < 12 * clean + 0.1
    for b in dev + [ws]:
        b.close()


def test_strides_and_bounds(rl, gpu):
    """q, k and v as slices of one row, a wider output whose gaps stay, rows of no sequence left alone, starts past the
    arrays cut off, a sequence longer than max_q."""
    rng = np.random.default_rng(10)
    d, qh, kvh, n = 64, 4, 2, 150
    wide = (qh + 2 * kvh) * d
    x = k8.bits(rng.standard_normal((n, wide)), "fp16")
    q, k, v = (x[:, a * d:b * d].reshape(n, -1, d) for a, b in ((0, qh), (qh, qh + kvh), (qh + kvh, qh + 2 * kvh)))
    qs = [10, 75, 75, 140]
    out = k8.run_prompt(rl, x, x, x, qs, qh, kvh, d, "fp16", strides=(wide, wide, wide, qh * d + 8),
                        offsets=(0, qh * d, (qh + kvh) * d))
    compare(np.ascontiguousarray(out[:, :qh * d]).reshape(n, qh, d), q, k, v, qs, qs, kvh, "fp16")
    assert (out[:, qh * d:] == 0x1234).all() and (out[:10] == 0x1234).all() and (out[140:] == 0x1234).all()
    cut = k8.run_prompt(rl, x, x, x, [10, 75, 75, 4000], qh, kvh, d, "fp16", strides=(wide, wide, wide, qh * d + 8),
                        offsets=(0, qh * d, (qh + kvh) * d), q_tokens=140, kv_tokens=140, max_q=65)
    assert np.array_equal(cut, out)
    # rows past max_q of a sequence may be left out, the others are the same
    few = k8.run_prompt(rl, x, x, x, qs, qh, kvh, d, "fp16", strides=(wide, wide, wide, qh * d + 8),
                        offsets=(0, qh * d, (qh + kvh) * d), max_q=33)
    assert np.array_equal(few[10:43], out[10:43]) and np.array_equal(few[75:108], out[75:108])


@pytest.mark.parametrize("max_q", [1, 33, 64])
def test_queries_past_max_q(rl, gpu, max_q):
    """A sequence's queries from max_q on get no output; the others are those without them."""
    rng = np.random.default_rng(11)
    lens, kvh = [100, 20, 65], 2
    qs = starts_of(lens)
    q, k, v = inputs(rng, qs[-1], qs[-1], 6, kvh, 128, "bf16")
    cut = run(rl, q, k, v, qs, kvh, "bf16", max_q=max_q)
    for a, n in zip(qs, lens):
        m = min(n, max_q)
        compare(cut[a:a + m].reshape(m, 6, 128), q[a:a + m], k[a:a + m], v[a:a + m], [0, m], [0, m], kvh, "bf16")
        assert (cut[a + m:a + n] == 0x1234).all()


def test_scores_without_weight(rl, gpu):
    """A key whose score is minus infinity beside a value that is no number and that the row does not see, with the
    keys shared by several workgroups: the row's other shares give its output."""
    rng = np.random.default_rng(12)
    nq, nk, finite = 2, 1500, 768  # the later shares have no score above minus infinity
    q, k, v = inputs(rng, nq, nk, 1, 1, 64, "fp16")
    fq, fk, fv = (k8.floats(x, "fp16") for x in (q, k, v))
    fq[:, :, 0], fk[:finite, 0, 0], fk[finite:, 0, 0], fv[nk - 1, 0, 5] = 1.0, 0.0, -np.inf, np.nan
    out = run(rl, *(k8.bits(x, "fp16") for x in (fq, fk, fv)), [0, nq], 1, "fp16", kv_starts=[0, nk])
    out = k8.floats(out.reshape(q.shape), "fp16")
    ref, mag = k8.attend(fq[:, 0], fk[:finite, 0], fv[:finite, 0], 1 / 8.0, [finite, finite])
    tol = tolerance("fp16", ref, mag, fq[:, 0], fk[:finite, 0], 1 / 8.0, finite)
    ok = np.abs(out[:, 0] - ref) <= tol
    assert np.isnan(out[1, 0, 5]) and ok[0].all() and np.delete(ok[1], 5).all()


def test_far_tokens(rl, gpu):
    """The widest strides: tokens of q, k, v and out behind 4 GiB."""
    rng = np.random.default_rng(33)
    d, qh, kvh, stride = 128, 4, 1, 1 << 24
    qs = starts_of([70, 65])
    n = qs[-1]
    assert 2 * stride * (n - 1) > 1 << 32
    q, k, v = inputs(rng, n, n, qh, kvh, d, "bf16")
    bufs = [rl.DeviceBuffer(2 * stride * (n - 1) + 2 * qh * d) for _ in range(4)]
    for buf, x in zip(bufs, (q, k, v)):
        for i in range(n):
            buf.upload(x[i], 2 * stride * i)
    sb = rl.DeviceBuffer.from_array(np.array(qs, np.uint32))
    args = rl.AttnPromptArgs(q=bufs[0].ptr, k=bufs[1].ptr, v=bufs[2].ptr, out=bufs[3].ptr, q_stride=stride, k_stride=stride,
                             v_stride=stride, out_stride=stride, q_starts=sb.ptr, seqs=2, q_tokens=n, kv_tokens=n, max_q=70,
                             max_kv=70, q_heads=qh, kv_heads=kvh, head_dim=d, dtype=rl.DTYPE_BF16)
    ws = rl.attn_prompt_workspace(args)
    rl.attn_prompt(args)
    rl.sync()
    out = np.stack([bufs[3].download(np.uint16, (qh, d), 2 * stride * i) for i in range(n)])
    compare(out, q, k, v, qs, qs, kvh, "bf16")
    for b in bufs + [sb, ws]:
        b.close()


def test_graphs_share_a_workspace(rl, gpu):
    """Two captured calls that share keys among workgroups on one workspace, in turn: each as it is alone."""
    d, qh, kvh, nq, nk = 128, 8, 2, 3, 2100
    up, calls, want = rl.DeviceBuffer.from_array, [], []
    for i in range(2):
        q, k, v = inputs(np.random.default_rng(70 + i), nq, nk, qh, kvh, d, "bf16")
        want.append(run(rl, q, k, v, [0, nq], kvh, "bf16", kv_starts=[0, nk]))
        dev = [up(q), up(k), up(v), up(np.zeros((nq, qh * d), np.uint16)), up(np.array([0, nq], np.uint32)),
               up(np.array([0, nk], np.uint32))]
        calls.append((dev, rl.AttnPromptArgs(q=dev[0].ptr, k=dev[1].ptr, v=dev[2].ptr, out=dev[3].ptr, q_starts=dev[4].ptr,
                                             kv_starts=dev[5].ptr, seqs=1, q_tokens=nq, kv_tokens=nk, max_q=nq, max_kv=nk,
                                             q_heads=qh, kv_heads=kvh, head_dim=d, dtype=rl.DTYPE_BF16)))
    ws = rl.attn_prompt_workspace(calls[0][1])
    assert ws.nbytes > 4096  # (the keys are shared)
    for _, args in calls:
        args.workspace, args.workspace_bytes = ws.ptr, ws.nbytes
    graphs = [rl.Graph(lambda a=args: rl.attn_prompt(a)) for _, args in calls]
    for _ in range(3):
        for g in graphs:
            g.launch()
        rl.sync()
        for (dev, _), ref in zip(calls, want):
            assert np.array_equal(dev[3].download(np.uint16, ref.shape), ref)
            rl.check(rl.lib().rl_hip_memset_d(dev[3].ptr, 0, dev[3].nbytes), "memset")
    for g in graphs:
        g.close()
    for dev, _ in calls:
        for b in dev:
            b.close()
    ws.close()


@pytest.mark.parametrize("short", [0, 1])
def test_workspace_refusal(rl, gpu, short):
    a = rl.AttnPromptArgs(q=1 << 20, k=1 << 20, v=1 << 20, out=1 << 20, q_starts=1 << 20, seqs=1, q_tokens=4, kv_tokens=4,
                          max_q=4, max_kv=4000, q_heads=8, kv_heads=2, head_dim=64, dtype=0)
    need = rl.attn_prompt_workspace_bytes(a)
    a.workspace, a.workspace_bytes = (1 << 20, need - 1) if short else (None, need)
    with pytest.raises(rl.RlrtError, match="workspace"):
        rl.attn_prompt(a)


@pytest.mark.parametrize("qh, kvh, d", [(32, 8, 128), (3, 1, 64)])
def test_workspace_of_smaller_calls(rl, gpu, qh, kvh, d):
    """A workspace of the largest call is enough for fewer sequences, queries and keys."""
    def need(seqs, max_q, max_kv):
        return rl.attn_prompt_workspace_bytes(rl.AttnPromptArgs(
            q=1 << 20, k=1 << 20, v=1 << 20, out=1 << 20, q_starts=1 << 20, seqs=seqs, q_tokens=4, kv_tokens=4, max_q=max_q,
            max_kv=max_kv, q_heads=qh, kv_heads=kvh, head_dim=d, dtype=0))

    seqs, qs = [1, 2, 3, 5, 8, 16, 31, 32, 33, 64, 200], [0, 1, 16, 33, 64, 100, 517, 1024, 8192]
    ks = [0, 64, 383, 384, 700, 768, 769, 3100, 6000, 6144, 12300, 50000, 200000]
    all_ = np.array([[[need(s, q, k) for k in ks] for q in qs] for s in seqs])
    assert all((np.diff(all_, axis=i) >= 0).all() for i in range(3)) and all_[0, 0, 0] > 0


def test_pieces_on_the_workspace_of_a_prompt(rl, gpu):
    """A long prompt, then its last queries behind its keys, on the workspace of the first call."""
    rng = np.random.default_rng(41)
    n, qh, kvh, d, dtype = 1700, 8, 2, 64, "fp16"
    q, k, v = inputs(rng, n, n, qh, kvh, d, dtype)
    up = rl.DeviceBuffer.from_array
    ws = None
    for m in (n, 33, 1):
        dev = [up(q[n - m:]), up(k), up(v), up(np.zeros((m, qh, d), np.uint16)), up(np.array([0, m], np.uint32)),
               up(np.array([0, n], np.uint32))]
        args = rl.AttnPromptArgs(q=dev[0].ptr, k=dev[1].ptr, v=dev[2].ptr, out=dev[3].ptr, q_starts=dev[4].ptr,
                                 kv_starts=dev[5].ptr, seqs=1, q_tokens=m, kv_tokens=n, max_q=m, max_kv=n, q_heads=qh,
                                 kv_heads=kvh, head_dim=d, dtype=rl.DTYPE_FP16)
        ws = ws or rl.attn_prompt_workspace(args)
        args.workspace, args.workspace_bytes = ws.ptr, ws.nbytes
        rl.attn_prompt(args)
        rl.sync()
        compare(dev[3].download(np.uint16, (m, qh, d)), q[n - m:], k, v, [0, m], [0, n], kvh, dtype)
        for b in dev:
            b.close()
    ws.close()


def test_nothing_to_do(rl, gpu):
    a = rl.AttnPromptArgs(q=1 << 20, k=1 << 20, v=1 << 20, out=1 << 20, q_starts=1 << 20, seqs=1, q_tokens=0, kv_tokens=0,
                          max_q=0, max_kv=0, q_heads=8, kv_heads=2, head_dim=64, dtype=0, workspace=1 << 20,
                          workspace_bytes=1 << 30)
    assert rl.lib().rl_hip_attn_prompt(C.byref(a)) == 0
    rl.sync()


def test_prompt_to_tokens(rl, gpu):
    """The operators together, as a rollout uses them: the prompts' attention, their K/V into the 8-bit arena, then
    decode steps, each attending what is cached and appending its token; every step against the model's arena."""
    rng = np.random.default_rng(21)
    lens, steps, qh, kvh, d, t, dtype = [37, 5, 80], 20, 8, 2, 128, 16, "bf16"
    batch, qs = len(lens), starts_of(lens)
    q, k, v = inputs(rng, qs[-1], qs[-1], qh, kvh, d, dtype)
    out = run(rl, q, k, v, qs, kvh, dtype).reshape(q.shape)
    compare(out, q, k, v, qs, qs, kvh, dtype)

    need = [-(-(n + steps) // t) for n in lens]
    stride, blocks = max(need), sum(need) * kvh
    perm = rng.permutation(blocks).astype(np.uint32)
    table, at = np.zeros((batch, kvh, stride), np.uint32), 0
    for b in range(batch):
        for g in range(kvh):
            table[b, g, :need[b]] = perm[at:at + need[b]]
            at += need[b]
    model = k8.Arena8(blocks, t, d, fill=False)
    layout, up = rl.KvLayoutDesc.paged8(t, d), rl.DeviceBuffer.from_array
    arena = rl.Arena(blocks * layout.block_bytes, layout.block_bytes)
    assert np.array_equal(arena.acquire_n(blocks), np.arange(blocks))
    tb, kb, vb, sb = up(table), up(k), up(v), up(np.array(qs, np.uint32))
    pos = up(np.zeros(batch, np.uint32))
    fill = rl.Kv8AppendArgs(arena_base=arena.ptr, arena_bytes=arena.nbytes, layout=layout, block_table=tb.ptr,
                            table_stride=stride, batch=batch, kv_heads=kvh, dtype=rl.DTYPE_BF16, positions=pos.ptr,
                            starts=sb.ptr, tokens=qs[-1], max_new=max(lens), k_new=kb.ptr, v_new=vb.ptr)
    rl.kv8_append(fill)
    rl.sync()
    f = [k8.floats(x, dtype) for x in (k, v)]
    for b in range(batch):
        for g in range(kvh):
            s = slice(qs[b], qs[b + 1])
            model.append(table[b, g], 0, np.stack((f[0][s, g], f[1][s, g])))
    assert np.array_equal(arena.download(np.uint8, model.bytes.shape), model.bytes)

    q1, k1, v1 = (rl.DeviceBuffer(batch * h * d * 2) for h in (qh, kvh, kvh))
    o16, o32 = rl.DeviceBuffer(batch * qh * d * 2), rl.DeviceBuffer(batch * qh * d * 4)
    attn = rl.attn_args(arena, layout, tb, stride, batch, qh, kvh, rl.DTYPE_BF16, pos, max(lens) + steps, q1, o16, o32)
    ws = rl.attn_kv8_workspace(attn)
    step_args = rl.Kv8AppendArgs(arena_base=arena.ptr, arena_bytes=arena.nbytes, layout=layout, block_table=tb.ptr,
                                 table_stride=stride, batch=batch, kv_heads=kvh, dtype=rl.DTYPE_BF16, positions=pos.ptr,
                                 tokens=batch, max_new=1, k_new=k1.ptr, v_new=v1.ptr)

    def step():
        rl.attn_decode_kv8(attn)
        rl.kv8_append(step_args)

    graph = rl.Graph(step)
    for i in range(steps):
        ctx = np.array(lens, np.uint32) + i
        hq, hk, hv = inputs(rng, batch, batch, qh, kvh, d, dtype)
        for dev, host in ((pos, ctx), (q1, hq), (k1, hk), (v1, hv)):
            dev.upload(host)
        if i % 2:
            graph.launch()
        else:
            step()
        rl.sync()
        got = o32.download(np.float32, (batch, qh, d)).astype(float)
        for b in range(batch):
            for g in range(kvh):
                kv = model.tokens(table[b, g], int(ctx[b]))
                hs = slice(g * 4, g * 4 + 4)
                ref, _ = k8.attend(k8.floats(hq, dtype)[b, hs], kv[0], kv[1], d ** -0.5, [int(ctx[b])] * 4)
                assert (np.abs(got[b, hs] - ref).max(-1) <= 1e-4 * np.abs(ref).max(-1)).all(), (i, b, g)
                model.append(table[b, g], int(ctx[b]), np.stack((k8.floats(hk, dtype)[b:b + 1, g],
                                                                k8.floats(hv, dtype)[b:b + 1, g])))
        assert np.array_equal(arena.download(np.uint8, model.bytes.shape), model.bytes), i
    graph.close()
    arena.close()

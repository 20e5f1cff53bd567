"""rl_hip_kv8_append and rl_hip_attn_decode_kv8 against the 64-bit model: the
arena byte for byte, the attention within its bounds."""
import ctypes as C

import numpy as np
import pytest

import kv8_helpers as k8
import synth

pytestmark = pytest.mark.gpu


def make_table(rng, need, kv_heads, stride, spare=0):
    """Random distinct blocks for `need` blocks per row; entries past them name no block of the arena."""
    n = int(np.sum(need)) * kv_heads
    perm = rng.permutation(n + spare)
    table = np.full((len(need), kv_heads, stride), 0xFFFFFFFF, np.uint32)
    at = 0
    for b, m in enumerate(need):
        for g in range(kv_heads):
            table[b, g, :m] = perm[at:at + m]
            at += m
    return table, n + spare


def rows(rng, n, kv_heads, d, dtype, spread=1.0):
    x = rng.standard_normal((n, kv_heads, d)) * np.exp(spread * rng.standard_normal((n, kv_heads, 1)))
    return k8.bits(x, dtype)


# ---------------------------------------------------------------- append
@pytest.mark.parametrize("t, d, dtype", [(16, 128, "bf16"), (32, 128, "fp16"), (16, 64, "fp16"), (32, 64, "bf16")])
def test_append_ragged(rl, gpu, t, d, dtype):
    """No token, one, a block's end, several blocks; rows that start anywhere in a block: the whole arena's bytes."""
    rng = np.random.default_rng(t + d)
    kvh, new = 3, [0, 1, t - 1, t + 1, 3 * t + 5, 1, t, 2]
    pos = [5, 0, t - 1, 3, 2 * t + 7, 2 * t - 1, t, t - 1]
    need = [-(-(p + n) // t) for p, n in zip(pos, new)]
    table, blocks = make_table(rng, need, kvh, max(need) + 1, spare=2)
    arena = k8.Arena8(blocks, t, d, seed=1)
    starts = np.concatenate([[0], np.cumsum(new)])
    k, v = rows(rng, starts[-1], kvh, d, dtype), rows(rng, starts[-1], kvh, d, dtype)
    got = k8.run_append(rl, arena, table, pos, k, v, dtype, starts=starts, max_new=max(new))
    fk, fv = k8.floats(k, dtype), k8.floats(v, dtype)
    for b in range(len(new)):
        for g in range(kvh):
            s = slice(starts[b], starts[b + 1])
            arena.append(table[b, g], pos[b], np.stack((fk[s, g], fv[s, g])))
    assert np.array_equal(got, arena.bytes)


def test_append_tokens_growing(rl, gpu):
    """Token by token with growing, shrinking and again growing magnitudes: each growth rescales the block's earlier tokens."""
    rng = np.random.default_rng(5)
    t, d, kvh = 16, 128, 2
    table, blocks = make_table(rng, [3, 3], kvh, 3)
    arena = k8.Arena8(blocks, t, d, fill=False)
    for i in range(2 * t + 3):
        size = 2.0 ** ((i * 7) % 23 - 11)
        k, v = rows(rng, 2, kvh, d, "bf16", 0.5), rows(rng, 2, kvh, d, "bf16", 0.5)
        k = k8.bits(k8.floats(k, "bf16") * size, "bf16")
        pos = [i, i + 1 if i else 0]
        got = k8.run_append(rl, arena, table, pos, k, v, "bf16")
        for b in range(2):
            for g in range(kvh):
                arena.append(table[b, g], pos[b], np.stack((k8.floats(k, "bf16")[b:b + 1, g], k8.floats(v, "bf16")[b:b + 1, g])))
        assert np.array_equal(got, arena.bytes), i


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_append_special_values(rl, gpu, dtype):
    """Zeros, subnormals, the type's extremes, infinities and NaN, magnitudes at the scale's borders, ties."""
    t, d = 16, 64
    big, tiny = (3.3895e38, 1e-40) if dtype == "bf16" else (65504.0, 6e-8)
    cases = [[0.0], [-0.0, 0.0], [tiny, -tiny], [big, 1.0, -big], [np.inf, 3.0], [-np.inf, np.nan], [np.nan, 1e-3, np.inf],
             [1.75, 1.0], [1.7578125 if dtype == "bf16" else 1.7509765625, 1.0], [448.0, 0.9375, 17.0, 19.0, -25.0],
             [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11], [3.5, 0.0078125 * 3]]
    kvh = len(cases)
    x = np.zeros((t, kvh, d))
    for g, c in enumerate(cases):
        x[:, g, :len(c)] = c
        x[1:, g, len(c):2 * len(c)] = c
    table = np.arange(kvh, dtype=np.uint32).reshape(1, kvh, 1)
    arena = k8.Arena8(kvh, t, d, seed=2)
    with np.errstate(over="ignore"):
        k = k8.bits(x, dtype)
    got = k8.run_append(rl, arena, table, [0], k, k[::-1].copy(), dtype, starts=[0, t], max_new=t)
    for g in range(kvh):
        f = k8.floats(k, dtype)[:, g]
        arena.append(table[0, g], 0, np.stack((f, f[::-1])))
    nan = (arena.bytes[:, :arena.n] & 127) == 127
    assert np.array_equal((got[:, :arena.n] & 127) == 127, nan) and nan.any()
    assert np.array_equal(np.where(nan, 0, got[:, :arena.n]), np.where(nan, 0, arena.bytes[:, :arena.n]))
    assert np.array_equal(got[:, arena.n:], arena.bytes[:, arena.n:])


def test_append_copy_on_write(rl, gpu):
    """The shared block's slots arrive in the row's own block, at the larger scale; the shared block stays."""
    rng = np.random.default_rng(9)
    t, d, kvh = 16, 128, 2
    table, blocks = make_table(rng, [2, 2, 2], kvh, 2, spare=2)
    shared = [b for b in range(blocks) if b not in set(table.reshape(-1).tolist())]
    for size in (0.01, 30.0):  # below the shared block's scale, above it
        arena = k8.Arena8(blocks, t, d, seed=3)
        k, v = rows(rng, 3, kvh, d, "bf16", 0.3), rows(rng, 3, kvh, d, "bf16", 0.3)
        k = k8.bits(k8.floats(k, "bf16") * size, "bf16")
        pos, cow = [t + 5, 3, 4], [[shared[0], shared[1]], [-1, shared[0]], [blocks + 7, -1]]
        got = k8.run_append(rl, arena, table, pos, k, v, "bf16", cow=cow)
        for b in range(3):
            for g in range(kvh):
                c = cow[b][g] if cow[b][g] < blocks else -1
                arena.append(table[b, g], pos[b], np.stack((k8.floats(k, "bf16")[b:b + 1, g], k8.floats(v, "bf16")[b:b + 1, g])),
                             cow=c)
        assert np.array_equal(got, arena.bytes)


def test_append_bounds_and_strides(rl, gpu):
    """Idle rows (position UINT32_MAX), rows past the table, blocks past the arena and token rows past `tokens` write
    nothing; K and V as slices of wider rows; a captured append replayed."""
    rng = np.random.default_rng(11)
    t, d, kvh, wide = 16, 64, 2, 2 * 64 * 4
    table, blocks = make_table(rng, [2, 2, 2, 2], kvh, 2)
    qkv = k8.bits(rng.standard_normal((12, wide)), "fp16")
    k, v = qkv.reshape(12, 8, d)[:, 2:4], qkv.reshape(12, 8, d)[:, 6:8]
    starts, pos = [0, 3, 6, 9, 14], [0xFFFFFFFF, 2 * t - 1, 4, t - 2]
    arena = k8.Arena8(blocks, t, d, seed=4)
    table[2, 0, 0] = blocks - 1 if table[2, 0, 0] != blocks - 1 else table[2, 0, 0]
    table[2, 1, 0] = 0xFFFF0000
    table[2, 0, 0] = blocks  # one past the arena
    up = rl.DeviceBuffer.from_array
    dev = up(qkv)
    a, tb, pb, sb = up(arena.bytes), up(table), up(np.array(pos, np.uint32)), up(np.array(starts, np.uint32))
    args = rl.Kv8AppendArgs(arena_base=a.ptr, arena_bytes=a.nbytes, layout=rl.KvLayoutDesc.paged8(t, d), block_table=tb.ptr,
                            table_stride=2, batch=4, kv_heads=kvh, dtype=rl.DTYPE_FP16, positions=pb.ptr, starts=sb.ptr,
                            tokens=12, max_new=5, cow_src=None, k_new=dev.ptr + 2 * 2 * d, v_new=dev.ptr + 2 * 6 * d,
                            k_stride=wide, v_stride=wide)
    gr = rl.Graph(lambda: rl.kv8_append(args))
    fk, fv = k8.floats(k, "fp16"), k8.floats(v, "fp16")
    for b, n in ((1, 3), (3, 3)):  # row 3 has 5 tokens, 3 of them exist
        for g in range(kvh):
            s = slice(starts[b], starts[b] + n)
            arena.append(table[b, g], pos[b], np.stack((fk[s, g], fv[s, g])))
    for _ in range(3):  # every replay leaves the same bytes
        gr.launch()
        rl.sync()
        assert np.array_equal(a.download(np.uint8, arena.bytes.shape), arena.bytes)
    gr.close()


# ---------------------------------------------------------------- decode
def check(arena, table, ctx, q, out16, out32, dtype, scale=None):
    """fp32 sums: within 1e-4 of the row's largest output, and the 16-bit output the fp32 one's rounding."""
    b_, qh, d = q.shape
    kvh = table.shape[1]
    f = k8.floats(q, dtype)
    for b in range(b_):
        for g in range(kvh):
            kv = arena.tokens(table[b, g][:-(-int(ctx[b]) // arena.t)], int(ctx[b]))
            hs = slice(g * qh // kvh, (g + 1) * qh // kvh)
            ref, _ = k8.attend(f[b, hs], kv[0], kv[1], scale or d ** -0.5, [int(ctx[b])] * (qh // kvh))
            got = out32[b, hs].astype(float)
            assert np.isfinite(got).all(), (b, g)
            err = np.abs(got - ref).max(-1) / np.maximum(np.abs(ref).max(-1), 1e-30)
            assert err.max() < 1e-4, (b, g, err.max())
    assert np.array_equal(out16, synth.to_scalar16(out32, dtype))


def decode_case(rng, ctx, kvh, group, t, d, dtype, stride=None, seed=3):
    need = [-(-c // t) for c in ctx]
    table, blocks = make_table(rng, need, kvh, stride or max(max(need), 1), spare=1)
    arena = k8.Arena8(blocks, t, d, seed=seed)
    # what lies behind a row's last token is NaN
    for b, c in enumerate(ctx):
        if c % t:
            for g in range(kvh):
                arena.planes(table[b, g, c // t])[:, c % t:] = 0x7F
    return arena, table, k8.bits(rng.standard_normal((len(ctx), kvh * group, d)), dtype)


@pytest.mark.parametrize("t, d, group, dtype", [(16, 128, 4, "bf16"), (32, 128, 8, "fp16"), (16, 64, 1, "fp16"),
                                                (32, 64, 2, "bf16"), (16, 128, 16, "bf16"), (16, 64, 3, "bf16")])
def test_decode_ragged(rl, gpu, t, d, group, dtype):
    """Contexts around tile, block and unit ends, none at all, and long ones; NaN behind every last token."""
    rng = np.random.default_rng(group)
    ctx = [0, 1, 15, 16, 17, 31, 32, 33, 48, 63, 64, 65, 700, 257]
    arena, table, q = decode_case(rng, ctx, 2, group, t, d, dtype)
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, dtype, max(ctx))
    assert not out32[0].any()
    check(arena, table, ctx, q, out16, out32, dtype)


@pytest.mark.parametrize("batch, max_ctx, lens", [(1, 517, [517]), (1, 40000, [40000]), (1, 40000, [3]), (2, 9000, [8999, 31]),
                                                  (70, 300, None), (3, 1 << 20, [100, 0, 5000])])
def test_decode_splits(rl, gpu, batch, max_ctx, lens):
    """Rows shared by many workgroups, rows much shorter than max_ctx, many rows; replays give the same bits."""
    rng = np.random.default_rng(batch)
    ctx = lens or rng.integers(0, max_ctx + 1, batch).tolist()
    arena, table, q = decode_case(rng, ctx, 2, 4, 16, 128, "bf16", stride=-(-max_ctx // 16))
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, "bf16", max_ctx, scale=0.11)
    check(arena, table, ctx, q, out16, out32, "bf16", scale=0.11)
    again = k8.run_decode(rl, arena, table, ctx, q, "bf16", max_ctx, scale=0.11, graph=3)
    assert np.array_equal(again[1].view(np.uint32), out32.view(np.uint32))


@pytest.mark.parametrize("batch, kvh, group, t, d, dtype, max_ctx, lens", [
    (100, 2, 16, 16, 128, "bf16", 900, (1, 260)),   # one row per compute unit, eight waves, sixteen heads
    (160, 1, 1, 32, 64, "fp16", 800, (0, 800)),     # the same, small heads
    (64, 2, 4, 16, 128, "bf16", 4096, (0, 200)),    # even shares, most rows short
    (130, 1, 8, 32, 128, "fp16", 4100, (0, 90)),    # even shares, three groups of 64 rollouts
    (7, 3, 2, 16, 64, "bf16", 200000, (3000, 9000)),  # even shares, rows in many pieces
])
def test_decode_kernels(rl, gpu, batch, kvh, group, t, d, dtype, max_ctx, lens):
    """Every way the rows are shared out, with empty rows first, last and between."""
    rng = np.random.default_rng(batch)
    ctx = rng.integers(lens[0], lens[1] + 1, batch)
    ctx[rng.random(batch) < 0.15] = 0
    ctx[[0, -1]] = 0, 0 if batch % 2 else lens[1]
    ctx = ctx.tolist()
    arena, table, q = decode_case(rng, ctx, kvh, group, t, d, dtype, stride=-(-max_ctx // t))
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, dtype, max_ctx)
    for b in range(batch):
        assert ctx[b] or not out32[b].any()
    check(arena, table, ctx, q, out16, out32, dtype)
    again = k8.run_decode(rl, arena, table, ctx, q, dtype, max_ctx, graph=2)
    assert np.array_equal(again[1].view(np.uint32), out32.view(np.uint32))
    # no tokens at all
    out16, out32 = k8.run_decode(rl, arena, table, [0] * batch, q, dtype, max_ctx)
    assert not out32.any() and not out16.any()


@pytest.mark.parametrize("kvh", [1, 2])
@pytest.mark.parametrize("ctx", [[1, 0, 0], [0, 0, 40], [30, 700, 0], [300, 31, 900], [0, 3, 2500]])
def test_decode_far_below_max_ctx(rl, gpu, ctx, kvh):
    """Contexts far below max_ctx: fewer runs than XCDs, none on some, and a few more than XCDs."""
    rng = np.random.default_rng(sum(ctx))
    for max_ctx in (1 << 20, 20000):  # even shares, and workgroups that own their rows
        arena, table, q = decode_case(rng, ctx, kvh, 4, 16, 128, "bf16", stride=-(-max_ctx // 16))
        out16, out32 = k8.run_decode(rl, arena, table, ctx, q, "bf16", max_ctx)
        check(arena, table, ctx, q, out16, out32, "bf16")
        again = k8.run_decode(rl, arena, table, ctx, q, "bf16", max_ctx, graph=2)
        assert np.array_equal(again[1].view(np.uint32), out32.view(np.uint32))


def test_decode_bad_rows(rl, gpu):
    """A context past max_ctx and a block past the arena give NaN rows; the others keep their bits. NaN among a row's own
    tokens reaches only the outputs that see it."""
    rng = np.random.default_rng(1)
    ctx = [100, 130, 90, 77]
    arena, table, q = decode_case(rng, ctx, 2, 4, 16, 128, "bf16", stride=9)
    good16, good = k8.run_decode(rl, arena, table, ctx, q, "bf16", 130)
    check(arena, table, ctx, q, good16, good, "bf16")
    bad = table.copy()
    bad[2, 1, 3] = len(arena.bytes)
    _, out = k8.run_decode(rl, arena, bad, [100, 131, 90, 77], q, "bf16", 130)
    assert np.isnan(out[1]).all() and np.isnan(out[2, 4:]).all()
    assert np.array_equal(out[0], good[0]) and np.array_equal(out[3], good[3]) and np.array_equal(out[2, :4], good[2, :4])
    arena.planes(table[3, 0, 2])[1, 5, 9] = 0x7F  # V of one token, dim 9
    _, out = k8.run_decode(rl, arena, table, ctx, q, "bf16", 130)
    nan = np.isnan(out)
    assert nan[3, :4, 9].all() and nan.sum() == 4
    arena.planes(table[3, 0, 2])[0, 5, 9] = 0x7F  # K of one token: every output of the head's group
    _, out = k8.run_decode(rl, arena, table, ctx, q, "bf16", 130)
    assert np.isnan(out[3, :4]).all() and np.isnan(out).sum() == 4 * 128


def test_decode_far_apart_scores(rl, gpu):
    """Scores that grow along the context (each unit rescales), one token that takes all, scales far apart."""
    rng = np.random.default_rng(2)
    ctx = [400, 400]
    arena, table, q = decode_case(rng, ctx, 1, 4, 16, 128, "fp16")
    for j in range(25):
        arena.scales()[table[0, 0, j]] = [2.0 ** (j // 2 - 9), 2.0 ** (3 - j)]
        arena.scales()[table[1, 0, j]] = [2.0 ** (-(j // 3) - 2), 2.0 ** (j - 12)]
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, "fp16", 400)
    check(arena, table, ctx, q, out16, out32, "fp16")


def test_decode_row_alone(rl, gpu):
    """A row's bits do not depend on what the other rows hold."""
    rng = np.random.default_rng(4)
    ctx = [300, 20, 1000, 64]
    arena, table, q = decode_case(rng, ctx, 2, 4, 16, 128, "bf16")
    _, a = k8.run_decode(rl, arena, table, ctx, q, "bf16", 1000)
    q2, c2 = q.copy(), [300, 1000, 0, 999]
    q2[1:] = q[[0, 1, 2]]
    t2 = table.copy()
    t2[1], t2[3] = table[2], table[2]
    _, b = k8.run_decode(rl, arena, t2, c2, q2, "bf16", 1000)
    assert np.array_equal(a[0], b[0])


def test_decode_workspace_refused(rl, gpu):
    a = rl.AttnArgs(arena_base=1 << 20, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged8(16, 128), block_table=1 << 20,
                    table_stride=1000, batch=1, q_heads=8, kv_heads=2, dtype=0, ctx_lens=1 << 20, max_ctx=16000, q=1 << 20,
                    out=1 << 20)
    need = rl.attn_kv8_workspace_bytes(a)
    for a.workspace, a.workspace_bytes in ((None, 1 << 30), (1 << 20, need - 1)):
        assert rl.lib().rl_hip_attn_decode_kv8(C.byref(a)) == -1
        assert "workspace" in rl.lib().rl_hip_last_error().decode()


@pytest.mark.parametrize("kvh, group, d", [(8, 4, 128), (1, 16, 64), (2, 1, 128)])
def test_decode_workspace_of_smaller_calls(rl, gpu, kvh, group, d):
    """A workspace of the largest call is enough for every smaller batch and max_ctx."""
    def args(batch, max_ctx, **kw):
        return rl.AttnArgs(arena_base=1 << 20, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged8(16, d), block_table=1 << 20,
                           table_stride=1 << 16, batch=batch, q_heads=kvh * group, kv_heads=kvh, dtype=0, ctx_lens=1 << 20,
                           max_ctx=max_ctx, q=1 << 20, out=1 << 20, **kw)

    batches = [1, 2, 3, 8, 15, 16, 17, 24, 31, 32, 33, 64, 100, 128, 256, 257, 300, 512, 1024]
    ctxs = [1, 500, 736, 737, 800, 2048, 3168, 3169, 4096, 16000, 33000, 500000]
    need = np.array([[rl.attn_kv8_workspace_bytes(args(b, c)) for c in ctxs] for b in batches])
    assert (np.diff(need, axis=0) >= 0).all() and (np.diff(need, axis=1) >= 0).all() and need[0, 0] > 0


def test_decode_batch_shrinks_on_one_workspace(rl, gpu):
    """A rollout whose members end one after the other, on the workspace of its first step."""
    rng = np.random.default_rng(40)
    t, d, kvh, group, dtype, max_ctx, batch = 16, 64, 4, 2, "bf16", 1100, 96
    ctx = rng.integers(1, max_ctx + 1, batch).tolist()
    arena, table, q = decode_case(rng, ctx, kvh, group, t, d, dtype, stride=-(-max_ctx // t))
    up = rl.DeviceBuffer.from_array
    a, tb, cb, qb = up(arena.bytes), up(table), up(np.asarray(ctx, np.uint32)), up(q)
    out, out32 = rl.DeviceBuffer(q.size * 2), rl.DeviceBuffer(q.size * 4)
    ws = None
    for n in (96, 64, 63, 33, 17, 8, 3, 1):
        args = rl.attn_args(a, rl.KvLayoutDesc.paged8(t, d), tb, table.shape[2], n, kvh * group, kvh, rl.DTYPE_BF16, cb, max_ctx,
                            qb, out, out32)
        ws = ws or rl.attn_kv8_workspace(args)
        args.workspace, args.workspace_bytes = ws.ptr, ws.nbytes
        rl.attn_decode_kv8(args)
        rl.sync()
        got16, got32 = out.download(np.uint16, q.shape)[:n], out32.download(np.float32, q.shape)[:n]
        check(arena, table[:n], ctx[:n], q[:n], got16, got32, dtype)
    for b in (a, tb, cb, qb, out, out32, ws):
        b.close()


def test_far_blocks(rl, gpu):
    """Blocks behind 4 GiB of arena: tokens appended to them and read back by the decode."""
    rng = np.random.default_rng(32)
    t, d, kvh, group, n, dtype = 16, 128, 2, 4, 40, "bf16"
    near = k8.Arena8(6, t, d, fill=False)
    near_table = rng.permutation(6).astype(np.uint32).reshape(1, kvh, 3)
    block, ids = near.bytes.shape[1], np.array([3, 1_020_000, 1_020_001, 7, 1_039_998, 1_039_999], np.uint32)
    assert int(ids[1]) * block > 1 << 32
    k, v = rows(rng, n, kvh, d, dtype), rows(rng, n, kvh, d, dtype)
    q = k8.bits(rng.standard_normal((1, kvh * group, d)), dtype)
    up = rl.DeviceBuffer.from_array
    arena = rl.DeviceBuffer(1_040_000 * block)
    table, zero, starts = up(ids[near_table]), up(np.zeros(1, np.uint32)), up(np.array([0, n], np.uint32))
    kb, vb, qb, ctx = up(k), up(v), up(q), up(np.array([n], np.uint32))
    out, out32 = rl.DeviceBuffer(q.size * 2), rl.DeviceBuffer(q.size * 4)
    layout = rl.KvLayoutDesc.paged8(t, d)
    rl.kv8_append(rl.Kv8AppendArgs(arena_base=arena.ptr, arena_bytes=arena.nbytes, layout=layout, block_table=table.ptr,
                                   table_stride=3, batch=1, kv_heads=kvh, dtype=rl.DTYPE_BF16, positions=zero.ptr,
                                   starts=starts.ptr, tokens=n, max_new=n, k_new=kb.ptr, v_new=vb.ptr))
    args = rl.attn_args(arena, layout, table, 3, 1, kvh * group, kvh, rl.DTYPE_BF16, ctx, 48, qb, out, out32)
    ws = rl.attn_kv8_workspace(args)
    rl.attn_decode_kv8(args)
    rl.sync()
    fk, fv = k8.floats(k, dtype), k8.floats(v, dtype)
    for g in range(kvh):
        near.append(near_table[0, g], 0, np.stack((fk[:, g], fv[:, g])))
        for j, blk in enumerate(near_table[0, g]):
            m = min(t, n - j * t)
            got = arena.download(np.uint8, (block,), int(ids[blk]) * block)
            assert np.array_equal(got[:near.n].reshape(2, t, d)[:, :m], near.planes(blk)[:, :m])
            assert np.array_equal(got[near.n:near.n + 8], near.bytes[blk, near.n:near.n + 8])
    check(near, near_table, [n], q, out.download(np.uint16, q.shape), out32.download(np.float32, q.shape), dtype)
    for b in (arena, table, zero, starts, kb, vb, qb, ctx, out, out32, ws):
        b.close()


@pytest.mark.parametrize("max_ctx, batch", [(9000, 3), (3300, 80)])
def test_decode_graphs_share_a_workspace(rl, gpu, max_ctx, batch):
    """Two captured calls on one workspace, replayed in turn with an eager one between: each as it is alone."""
    t, d, kvh, group, dtype = 16, 128, 2, 4, "bf16"
    up, calls, want = rl.DeviceBuffer.from_array, [], []
    for i in range(3):
        rng = np.random.default_rng(50 + i)
        ctx = rng.integers(0, min(max_ctx, 900) + 1, batch).tolist()
        ctx[0] = max_ctx
        arena, table, q = decode_case(rng, ctx, kvh, group, t, d, dtype, stride=-(-max_ctx // t), seed=60 + i)
        want.append(k8.run_decode(rl, arena, table, ctx, q, dtype, max_ctx)[1])
        dev = [up(arena.bytes), up(table), up(np.asarray(ctx, np.uint32)), up(q), rl.DeviceBuffer(q.size * 2),
               rl.DeviceBuffer(q.size * 4, zero=True)]
        calls.append((dev, rl.attn_args(dev[0], rl.KvLayoutDesc.paged8(t, d), dev[1], table.shape[2], batch, kvh * group, kvh,
                                        rl.DTYPE_BF16, dev[2], max_ctx, dev[3], dev[4], dev[5]), q.shape))
    ws = rl.attn_kv8_workspace(calls[0][1])
    for _, args, _ in calls:
        args.workspace, args.workspace_bytes = ws.ptr, ws.nbytes
    graphs = [rl.Graph(lambda a=args: rl.attn_decode_kv8(a)) for _, args, _ in calls[:2]]
    for _ in range(3):
        graphs[0].launch()
        rl.attn_decode_kv8(calls[2][1])
        graphs[1].launch()
        rl.sync()
        for (dev, _, shape), ref in zip(calls, want):
            assert np.array_equal(dev[5].download(np.float32, shape).view(np.uint32), ref.view(np.uint32))
            rl.check(rl.lib().rl_hip_memset_d(dev[5].ptr, 0, dev[5].nbytes), "memset")
    for g in graphs:
        g.close()
    for dev, _, _ in calls:
        for b in dev:
            b.close()
    ws.close()


@pytest.mark.parametrize("t, d, kvh, n, dtype", [(16, 128, 8, 7800, "bf16"), (32, 64, 16, 7900, "fp16")])
def test_decode_more_than_the_caches_keep(rl, gpu, t, d, kvh, n, dtype):
    """More than 256 MiB of cache, a part of it prompts that neighbours share: alone, first, last and between."""
    rng = np.random.default_rng(d)
    ctx = (n + rng.integers(0, 1000, 18)).tolist()
    ctx[5] = 0
    arena, table, q = decode_case(rng, ctx, kvh, 2, t, d, dtype)
    assert 2 * d * kvh * sum(ctx) > 256 << 20
    shared = n // t // 2
    for b in (1, 9, 10, 17):  # with the one before
        table[b, :, :shared] = table[b - 1, :, :shared]
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, dtype, max(ctx))
    rows = [0, 1, 4, 6, 9, 10, 11, 16, 17]
    check(arena, table[rows], np.array(ctx)[rows], q[rows], out16[rows], out32[rows], dtype)
    assert not out32[5].any()


@pytest.mark.parametrize("t, d, kvh, n, dtype", [(16, 128, 8, 8000, "bf16")])
def test_decode_shared_prompts_apart(rl, gpu, t, d, kvh, n, dtype):
    """More than 256 MiB of cache whose rollouts share prompts with others that are not their neighbours, and one with the
    whole of its blocks."""
    rng = np.random.default_rng(n)
    ctx = (n + rng.integers(0, 700, 17)).tolist()
    ctx[8] = ctx[2] = n  # the same blocks and length, other queries
    arena, table, q = decode_case(rng, ctx, kvh, 2, t, d, dtype)
    assert 2 * d * kvh * sum(ctx) > 256 << 20
    shared = n // t // 2
    for b, other in ((3, 0), (6, 0), (9, 5), (16, 1)):
        table[b, :, :shared] = table[other, :, :shared]
    table[8] = table[2]
    out16, out32 = k8.run_decode(rl, arena, table, ctx, q, dtype, max(ctx))
    rows = [0, 1, 2, 3, 5, 6, 8, 9, 16]
    check(arena, table[rows], np.array(ctx)[rows], q[rows], out16[rows], out32[rows], dtype)

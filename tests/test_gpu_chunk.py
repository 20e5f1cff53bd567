"""rl_hip_attn_chunk against attention in 64 bits over what the arena holds."""
import numpy as np
import pytest

import kv8_helpers as k8
from test_gpu_prompt import compare, starts_of

pytestmark = pytest.mark.gpu


class Case:
    """lens[b] new queries of row b, whose cache has ctx[b] tokens (the queries' own among them). What no token of any row
    holds is NaN."""

    def __init__(self, seed, lens, ctx, qh, kvh, d, tpb, dtype, spare=5, stride=None, share=0):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.ctx = np.asarray(lens), np.asarray(ctx, np.int64)
        self.qh, self.kvh, self.d, self.tpb, self.dtype = qh, kvh, d, tpb, dtype
        b = len(lens)
        need = -(-self.ctx // tpb)
        self.stride = stride or max(1, int(need.max()))
        n = int(need.sum()) * kvh
        self.blocks = n + spare
        ids = rng.permutation(self.blocks)[:n]
        self.table = np.full((b, kvh, self.stride), 0xFFFFFFF0, np.uint32)  # entries past a row's tokens are never read
        at = 0
        for i in range(b):
            for g in range(kvh):
                self.table[i, g, :need[i]] = ids[at:at + need[i]]
                at += need[i]
            if share and i:
                self.table[i, :, :share] = self.table[0, :, :share]
        self.arena = np.full((self.blocks, 2, tpb, d), 0x7FFF, np.uint16)  # NaN in both types
        self.fill()
        self.q = k8.bits(rng.standard_normal((int(self.lens.sum()), qh, d)), dtype)
        self.q_starts = starts_of(self.lens.tolist())

    def fill(self):
        for i, c in enumerate(self.ctx):
            for g in range(self.kvh):
                for j in range(-(-int(c) // self.tpb)):
                    m = min(self.tpb, int(c) - j * self.tpb)
                    x = self.rng.standard_normal((2, m, self.d))
                    self.arena[self.table[i, g, j], :, :m] = k8.bits(x, self.dtype)

    def rows(self):
        """K and V of all rows' tokens one behind the other, [tokens][kv heads][d], and their starts."""
        ks = starts_of(self.ctx.tolist())
        kv = np.zeros((2, ks[-1], self.kvh, self.d), np.uint16)
        for i, c in enumerate(self.ctx):
            if c:
                t = np.arange(c)
                kv[:, ks[i]:ks[i + 1]] = self.arena[self.table[i][:, t // self.tpb].T, :, (t % self.tpb)[:, None]].transpose(
                    2, 0, 1, 3)
        return kv[0], kv[1], ks

    def run(self, rl, max_q=None, max_ctx=None, pad=(0, 0), scale=0.0, q_starts=None, q_tokens=None, arena_blocks=None,
            ctx=None, graph=0, ws_size=None):
        up = rl.DeviceBuffer.from_array
        n, w = len(self.q), self.qh * self.d
        q = np.concatenate([self.q.reshape(n, w), np.full((n, pad[0]), 0x5A5A, np.uint16)], 1)
        blocks = self.blocks if arena_blocks is None else arena_blocks
        ctx = self.ctx if ctx is None else ctx
        dev = dict(a=up(self.arena), t=up(self.table), c=up(np.asarray(ctx, np.uint32)), q=up(q),
                   s=up(np.asarray(self.q_starts if q_starts is None else q_starts, np.uint32)),
                   o=up(np.full((n, w + pad[1]), 0x1234, np.uint16)))
        args = rl.AttnChunkArgs(
            arena_base=dev["a"].ptr, arena_bytes=blocks * 4 * self.tpb * self.d,
            layout=rl.KvLayoutDesc.paged(self.tpb, self.d), block_table=dev["t"].ptr, table_stride=self.stride,
            batch=len(self.lens), q_heads=self.qh, kv_heads=self.kvh, dtype=k8.dtype_id(rl, self.dtype),
            ctx_lens=dev["c"].ptr, max_ctx=int(self.ctx.max()) if max_ctx is None else max_ctx, q_starts=dev["s"].ptr,
            q_tokens=n if q_tokens is None else q_tokens, max_q=int(self.lens.max()) if max_q is None else max_q,
            q=dev["q"].ptr, out=dev["o"].ptr, q_stride=w + pad[0] if pad[0] else 0,
            out_stride=w + pad[1] if pad[1] else 0, scale=scale)
        dev["w"] = rl.attn_chunk_workspace(args)
        if graph:
            g = rl.Graph(lambda: rl.attn_chunk(args))
            for _ in range(graph):
                rl.check(rl.lib().rl_hip_memset_d(dev["w"].ptr, 0xFF, dev["w"].nbytes), "memset")
                g.launch()
                rl.sync()
            g.close()
        else:
            rl.attn_chunk(args)
            rl.sync()
        out = dev["o"].download(np.uint16, (n, w + pad[1]))
        for b in dev.values():
            b.close()
        return out

    def check(self, out, scale=None):
        k, v, ks = self.rows()
        compare(out[:, :self.qh * self.d].reshape(self.q.shape), self.q, k, v, self.q_starts, ks, self.kvh, self.dtype,
                scale=scale)


SHAPES = [(128, 16, 8, 2, "bf16"), (64, 32, 4, 4, "fp16"), (128, 32, 8, 1, "fp16"), (64, 16, 6, 2, "bf16"),
          (128, 16, 2, 2, "bf16"), (64, 16, 16, 1, "fp16")]


@pytest.mark.parametrize("d, tpb, qh, kvh, dtype", SHAPES)
@pytest.mark.parametrize("lens, old", [([1], [0]), ([1, 0, 3, 0, 1], [0, 5, 15, 0, 16]), ([63, 64, 65], [1, 0, 63]),
                                       ([127, 5, 128, 129], [300, 0, 17, 200]), ([4] * 9, [0, 1, 31, 32, 33, 63, 64, 65, 640]),
                                       ([300, 5], [13, 900])])
def test_chunks(rl, gpu, d, tpb, qh, kvh, dtype, lens, old):
    c = Case(sum(lens) + d, lens, np.add(lens, old), qh, kvh, d, tpb, dtype)
    c.check(c.run(rl))


@pytest.mark.parametrize("d, tpb, kvh, dtype", [(128, 16, 1, "bf16"), (64, 32, 3, "fp16"), (128, 32, 2, "fp16")])
def test_tile_counts(rl, gpu, d, tpb, kvh, dtype):
    """Contexts of one to eight tiles, whole and not: every order of the kinds of steps."""
    ctx = [64, 65, 128, 192, 193, 256, 319, 320, 385, 448, 449, 512]
    c = Case(d, [min(x, 130) for x in ctx], ctx, 2 * kvh, kvh, d, tpb, dtype)
    out = c.run(rl)
    c.check(out)
    assert np.array_equal(c.run(rl, graph=3), out)


@pytest.mark.parametrize("d, tpb, dtype", [(128, 16, "bf16"), (64, 32, "fp16"), (64, 16, "bf16")])
@pytest.mark.parametrize("lens, old", [([1, 3], [7000, 5000]), ([16], [9001]), ([2, 1, 0, 40], [4200, 12, 3, 8300])])
def test_few_queries_long_context(rl, gpu, d, tpb, dtype, lens, old):
    """More than 64 tiles in one workgroup's share, and keys shared among workgroups; the same bits at every replay."""
    c = Case(d, lens, np.add(lens, old), 4, 1, d, tpb, dtype)
    out = c.run(rl)
    c.check(out)
    assert np.array_equal(c.run(rl, graph=3), out)


def test_many_tiles_in_one_workgroup(rl, gpu):
    """So many rows that no keys are shared, and two contexts of more than 64 and 128 tiles."""
    lens = [3] * 300
    ctx = [3 + i % 40 for i in range(300)]
    ctx[7], ctx[250] = 4500, 8500
    c = Case(3, lens, ctx, 2, 1, 64, 16, "bf16")
    c.check(c.run(rl))


def test_shared_prefix(rl, gpu):
    """The members of a group read the same blocks."""
    c = Case(17, [5, 60, 1, 130], [101, 156, 97, 226], 8, 2, 128, 16, "bf16", share=6)
    c.check(c.run(rl))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_fewer_keys_than_queries(rl, gpu, dtype):
    """Queries that see no key yield zeros; so do rows without any."""
    c = Case(4, [5, 3, 70], [2, 0, 66], 4, 2, 128, 16, dtype)
    out = c.run(rl)
    c.check(out)
    assert not out[:3].any() and not out[5:8].any() and not out[8:12].any() and out[12:].any(1).all()


def test_strides_bounds_and_rows_of_nobody(rl, gpu):
    c = Case(8, [9, 33, 2], [40, 133, 500], 6, 2, 64, 16, "bf16")
    plain = c.run(rl)
    c.check(plain)
    out = c.run(rl, pad=(8, 24))
    assert np.array_equal(out[:, :6 * 64], plain) and (out[:, 6 * 64:] == 0x1234).all()
    # queries past max_q, and rows past q_tokens, get no output
    out = c.run(rl, max_q=8)
    assert np.array_equal(out[:8], plain[:8]) and (out[8] == 0x1234).all() and (out[17:42] == 0x1234).all()
    assert np.array_equal(out[42:], plain[42:])
    starts = [1, 10, 30, 30]
    c.lens, c.q_starts = np.array([9, 20, 0]), starts
    out = c.run(rl)
    assert (out[0] == 0x1234).all() and (out[30:] == 0x1234).all() and not (out[1:30] == 0x1234).all(1).any()
    assert (c.run(rl, max_q=0) == 0x1234).all()


def test_scale_and_steep_scores(rl, gpu):
    c = Case(12, [40, 7], [300, 70], 4, 2, 128, 16, "bf16")
    c.check(c.run(rl, scale=0.5), scale=0.5)


def test_lost_blocks(rl, gpu):
    """Rows that see a block past the arena are no numbers, the others stand; so with contexts past max_ctx."""
    c = Case(13, [40, 20, 60], [200, 120, 60], 4, 2, 64, 16, "bf16")
    want = c.run(rl)
    c.check(want)
    c.table[1, 1, 6] = 0xFFFFFFFF                    # tokens 96 .. 111 of row 1, KV head 1
    out = c.run(rl)
    f = k8.floats(out, "bf16").reshape(-1, 4, 64)
    w = want.reshape(f.shape)
    bad = np.zeros(f.shape[:2], bool)
    bad[40:60, 2:] = True                            # its queries are the tokens 100 .. 119
    c.table[2, 0, 2] = c.blocks                      # tokens 32 .. 47 of row 2, KV head 0
    out = c.run(rl)
    f = k8.floats(out, "bf16").reshape(-1, 4, 64)
    bad[60 + 32:, :2] = True
    assert np.isnan(f[bad]).all() and np.array_equal(out.reshape(w.shape)[~bad], w[~bad])
    c = Case(14, [40, 20, 60], [200, 120, 60], 4, 2, 64, 16, "bf16")
    want = c.run(rl)
    out = c.run(rl, ctx=[200, 201, 60], max_ctx=200)
    assert np.isnan(k8.floats(out[40:60], "bf16")).all()
    assert np.array_equal(out[:40], want[:40]) and np.array_equal(out[60:], want[60:])
    out = c.run(rl, ctx=[0xFFFFFFFF, 120, 60])
    assert np.isnan(k8.floats(out[:40], "bf16")).all() and np.array_equal(out[40:], want[40:])


def test_lost_blocks_of_shared_keys(rl, gpu):
    """The same where workgroups share a row's keys."""
    c = Case(15, [3], [6000], 4, 1, 128, 16, "fp16")
    c.table[0, 0, 100] = 0xFFFFFFFF
    assert np.isnan(k8.floats(c.run(rl), "fp16")).all()
    c = Case(15, [3], [6000], 4, 1, 128, 16, "fp16", stride=400)
    assert np.isnan(k8.floats(c.run(rl, ctx=[6001], max_ctx=6000), "fp16")).all()


@pytest.mark.parametrize("d, tpb, dtype", [(128, 16, "bf16"), (64, 32, "bf16"), (128, 32, "fp16")])
def test_what_is_not_seen_has_no_part(rl, gpu, d, tpb, dtype):
    """NaN and infinities in keys and values that a query does not see leave its output as it is; seen ones do not."""
    c = Case(16, [100, 150], [100, 190], 4, 2, d, tpb, dtype)
    clean = k8.floats(c.run(rl).reshape(c.q.shape), dtype)

    def put(row, head, token, plane, dim, value):
        c.arena[c.table[row, head, token // tpb], plane, token % tpb, dim] = k8.bits(np.array([value]), dtype)[0]

    put(0, 0, 70, 1, 3, np.nan)
    put(0, 1, 90, 1, 5, np.inf)
    put(1, 1, 120, 0, 2, np.nan)           # query 80 of row 1
    f = k8.floats(c.run(rl).reshape(c.q.shape), dtype)
    # (rows computed again round their weights otherwise: each within the weights' rounding and its own of the exact one)
    tol = 3 * k8.HALF_STEP[dtype] * np.abs(clean) + 4 * k8.HALF_STEP[dtype]
    same = np.abs(f - clean) <= tol
    other = np.arange(d)
    assert same[:70].all() and np.isnan(f[70:100, :2, 3]).all() and same[70:100, :2][..., other != 3].all()
    assert same[70:90, 2:].all() and np.isposinf(f[90:100, 2:, 5]).all() and same[90:100, 2:][..., other != 5].all()
    assert same[100:, :2].all() and same[100:180, 2:].all() and np.isnan(f[180:, 2:]).all()


@pytest.mark.parametrize("d, tpb, qh, kvh, dtype", SHAPES)
@pytest.mark.parametrize("new", [1, 3, 21])
def test_few_rows(rl, gpu, d, tpb, qh, kvh, dtype, new):
    """Few rows, whose keys a workgroup's waves share in runs of 32: every number of runs, whole and not."""
    ctx = [1, 15, 31, 32, 33, 63, 64, 65, 96, 97, 127, 128, 129, 160, 255, 256, 257, 300, 511, 900]
    for part in (ctx[:10], ctx[10:]):
        c = Case(new + d, [min(new, x) for x in part], part, qh, kvh, d, tpb, dtype)
        out = c.run(rl)
        c.check(out)
        assert np.array_equal(c.run(rl, graph=3), out)


@pytest.mark.parametrize("d, tpb, dtype", [(128, 16, "bf16"), (64, 32, "bf16"), (128, 32, "fp16"), (64, 16, "fp16")])
def test_few_rows_what_is_not_seen(rl, gpu, d, tpb, dtype):
    """As above with few rows; in fp16 also an infinity whose weight 16 bits round to 0."""
    c = Case(26, [20, 30, 5], [20, 190, 100], 4, 2, d, tpb, dtype)
    clean = k8.floats(c.run(rl).reshape(c.q.shape), dtype)

    def put(row, head, token, plane, dim, value):
        c.arena[c.table[row, head, token // tpb], plane, token % tpb, dim] = k8.bits(np.array([value]), dtype)[0]

    put(0, 0, 7, 1, 3, np.nan)
    put(0, 1, 18, 1, 5, np.inf)
    put(1, 1, 175, 0, 2, np.nan)           # query 15 of row 1
    put(1, 0, 40, 1, 9, -np.inf)           # seen by all of row 1
    f = k8.floats(c.run(rl).reshape(c.q.shape), dtype)
    tol = 3 * k8.HALF_STEP[dtype] * np.abs(clean) + 4 * k8.HALF_STEP[dtype]
    same, other = np.abs(f - clean) <= tol, np.arange(d)
    assert same[:7].all() and np.isnan(f[7:20, :2, 3]).all() and same[7:20, :2][..., other != 3].all()
    assert same[7:18, 2:].all() and np.isposinf(f[18:20, 2:, 5]).all() and same[18:20, 2:][..., other != 5].all()
    assert np.isneginf(f[20:50, :2, 9]).all() and same[20:50, :2][..., other != 9].all()
    assert same[20:35, 2:].all() and np.isnan(f[35:50, 2:]).all() and same[50:].all()
    # a key of row 2 that all queries weigh with about 2^-40 of the others
    q = k8.floats(c.q, dtype)
    q[50:] = np.abs(q[50:])
    c.q = k8.bits(q, dtype)
    low = -28.0 * d ** 0.5 / np.abs(q[50:]).sum(-1).min() * np.ones(d)
    for g in range(2):
        c.arena[c.table[2, g, 48 // tpb], 0, 48 % tpb] = k8.bits(low, dtype)
        put(2, g, 48, 1, 11, np.inf)
    assert np.isposinf(k8.floats(c.run(rl).reshape(c.q.shape), dtype)[50:, :, 11]).all()


def test_few_rows_or_many(rl, gpu):
    """The sizes between which the calls change hands: 256 rows, a workgroup per compute unit, and the keys' times."""
    for lens, ctx, qh, kvh in (([64, 3], [300, 90], 8, 2), ([65, 3], [300, 90], 8, 2), ([1] * 64, [70] * 64, 4, 4),
                               ([1] * 65, [70] * 65, 4, 4), ([5], [1200], 8, 2), ([5], [1900], 8, 2)):
        c = Case(len(lens), lens, ctx, qh, kvh, 64, 16, "bf16")
        c.check(c.run(rl))


def test_equals_a_prompt(rl, gpu):
    """The same tokens as packed rows: rl_hip_attn_prompt's bits."""
    lens, ctx = [70, 12, 200], [70, 300, 333]
    c = Case(18, lens, ctx, 8, 2, 128, 16, "bf16")
    k, v, ks = c.rows()
    out = k8.run_prompt(rl, c.q.reshape(len(c.q), -1), k.reshape(len(k), -1), v.reshape(len(v), -1), c.q_starts, 8, 2, 128,
                        "bf16", kv_starts=ks)
    assert np.array_equal(c.run(rl), out)


def test_one_token_is_a_decode_step(rl, gpu):
    """One query per row: rl_hip_attn_decode's outputs up to the weights' rounding."""
    ctx = [1, 17, 700, 64]
    c = Case(19, [1] * 4, ctx, 8, 2, 128, 16, "bf16")
    up = rl.DeviceBuffer.from_array
    table = np.where(c.table < c.blocks, c.table, 0)
    dev = [up(x) for x in (c.arena, table, np.asarray(ctx, np.uint32), c.q)]
    out = rl.DeviceBuffer(c.q.nbytes)
    a = rl.attn_args(dev[0], rl.KvLayoutDesc.paged(16, 128), dev[1], c.stride, 4, 8, 2, rl.DTYPE_BF16, dev[2], 700, dev[3],
                     out)
    ws = rl.attn_workspace(a)
    rl.attn_decode(a)
    rl.sync()
    want = k8.floats(out.download(np.uint16, c.q.shape), "bf16")
    got = k8.floats(c.run(rl).reshape(c.q.shape), "bf16")
    # both are within (u (mag + |o|)) of the exact output, mag <= 5 here (values of a normal distribution)
    assert np.abs(got - want).max() <= 2 * 2.0 ** -8 * (5 + np.abs(want).max())
    for b in dev + [out, ws]:
        b.close()


def test_workspaces(rl, gpu):
    """The workspace of the largest call serves smaller ones; a smaller one is refused."""
    def need(**kw):
        a = dict(arena_base=4096, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged(16, 128), block_table=4096,
                 table_stride=4096, batch=8, q_heads=32, kv_heads=8, dtype=rl.DTYPE_BF16, ctx_lens=4096, max_ctx=65536,
                 q_starts=4096, q_tokens=4096, max_q=512, q=4096, out=4096)
        a.update(kw)
        return rl.attn_chunk_workspace_bytes(rl.AttnChunkArgs(**a))

    most = need()
    for b in (1, 2, 5, 8):
        for mq in (1, 4, 37, 200, 512):
            for mc in (1, 500, 6000, 30000, 65536):
                assert need(batch=b, max_q=mq, max_ctx=mc) <= most
    a = rl.AttnChunkArgs(arena_base=4096, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged(16, 128), block_table=4096,
                         table_stride=4096, batch=1, q_heads=32, kv_heads=8, dtype=rl.DTYPE_BF16, ctx_lens=4096,
                         max_ctx=65536, q_starts=4096, q_tokens=1, max_q=1, q=4096, out=4096, workspace=4096,
                         workspace_bytes=100)
    with pytest.raises(rl.RlrtError, match="workspace"):
        rl.attn_chunk(a)


def test_offsets_past_4_gib(rl, gpu):
    """Blocks behind 4 GiB of arena."""
    c = Case(20, [5], [50], 2, 1, 128, 16, "bf16")
    blocks = (5 << 30) // (4 * 16 * 128)
    big = rl.DeviceBuffer(blocks * 4 * 16 * 128, zero=True)
    want = c.run(rl)
    table = c.table.copy()
    for j in range(4):
        table[0, 0, j] = blocks - 1 - 3 * j
        big.upload(c.arena[c.table[0, 0, j]], int(table[0, 0, j]) * 4 * 16 * 128)
    up = rl.DeviceBuffer.from_array
    dev = [up(x) for x in (table, np.array([50], np.uint32), c.q, np.array([0, 5], np.uint32))]
    out = rl.DeviceBuffer(c.q.nbytes)
    args = rl.AttnChunkArgs(arena_base=big.ptr, arena_bytes=big.nbytes, layout=rl.KvLayoutDesc.paged(16, 128),
                            block_table=dev[0].ptr, table_stride=c.stride, batch=1, q_heads=2, kv_heads=1,
                            dtype=rl.DTYPE_BF16, ctx_lens=dev[1].ptr, max_ctx=50, q_starts=dev[3].ptr, q_tokens=5, max_q=5,
                            q=dev[2].ptr, out=out.ptr)
    ws = rl.attn_chunk_workspace(args)
    rl.attn_chunk(args)
    rl.sync()
    assert np.array_equal(out.download(np.uint16, (5, 256)), want)
    for x in dev + [big, out, ws]:
        x.close()

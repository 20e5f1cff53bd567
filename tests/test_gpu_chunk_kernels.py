"""rl_hip_attn_chunk: what its few-rows kernel and its tiled one have to do alike, on both, unsplit."""
import numpy as np
import pytest

import kv8_helpers as k8
from chunk_rules import kernel
from test_gpu_chunk import Case

pytestmark = pytest.mark.gpu

SHAPES = [(128, 16, "bf16"), (64, 32, "fp16"), (64, 16, "bf16"), (128, 32, "fp16")]


def takes(gpu, c, what, max_ctx=None):
    assert kernel(gpu.cu_count, c.lens.tolist(), int(c.ctx.max()) if max_ctx is None else max_ctx, c.qh, c.kvh) == what


@pytest.mark.parametrize("d, tpb, dtype", SHAPES)
@pytest.mark.parametrize("what, last", [("few", 70), ("tiled", 140)])
def test_fewer_keys_than_queries(rl, gpu, d, tpb, dtype, what, last):
    """Queries that see no key yield zeros; so do rows without any."""
    c = Case(4, [5, 3, last], [2, 0, last - 4], 4, 2, d, tpb, dtype)
    takes(gpu, c, what)
    out = c.run(rl)
    c.check(out)
    assert not out[:3].any() and not out[5:8].any() and not out[8:12].any() and out[12:].any(1).all()


@pytest.mark.parametrize("d, tpb, dtype", SHAPES)
@pytest.mark.parametrize("what, mid, ctx", [("few", 33, [40, 133, 350]), ("tiled", 133, [40, 233, 350])])
def test_strides_bounds_and_rows_of_nobody(rl, gpu, d, tpb, dtype, what, mid, ctx):
    c = Case(8, [9, mid, 2], ctx, 6, 2, d, tpb, dtype)
    takes(gpu, c, what)
    w = 6 * d
    plain = c.run(rl)
    c.check(plain)
    out = c.run(rl, pad=(8, 24))
    assert np.array_equal(out[:, :w], plain) and (out[:, w:] == 0x1234).all()
    # queries past max_q, and rows past q_tokens, get no output
    cut = mid - 5
    assert kernel(gpu.cu_count, c.lens.tolist(), max(ctx), 6, 2, max_q=cut) == what
    out = c.run(rl, max_q=cut)
    assert np.array_equal(out[:9 + cut], plain[:9 + cut]) and (out[9 + cut:9 + mid] == 0x1234).all()
    assert np.array_equal(out[9 + mid:], plain[9 + mid:])
    out = c.run(rl, q_tokens=9 + mid)
    assert np.array_equal(out[:9 + mid], plain[:9 + mid]) and (out[9 + mid:] == 0x1234).all()
    # the first query and the last ones belong to no row
    starts = [1, 10, 7 + mid, 7 + mid]
    c.lens, c.q_starts = np.array([9, mid - 3, 0]), starts
    takes(gpu, c, what)
    out = c.run(rl)
    assert (out[0] == 0x1234).all() and (out[7 + mid:] == 0x1234).all() and not (out[1:7 + mid] == 0x1234).all(1).any()
    c.q = c.q[1:7 + mid]
    c.q_starts = [0, 9, 6 + mid, 6 + mid]
    c.check(out[1:7 + mid])


@pytest.mark.parametrize("d, tpb, dtype", SHAPES)
@pytest.mark.parametrize("what, first", [("few", 40), ("tiled", 200)])
def test_scale_and_steep_scores(rl, gpu, d, tpb, dtype, what, first):
    c = Case(12, [first, 7], [300, 70], 4, 2, d, tpb, dtype)
    takes(gpu, c, what)
    c.check(c.run(rl, scale=0.5), scale=0.5)


@pytest.mark.parametrize("d, tpb, dtype", SHAPES)
@pytest.mark.parametrize("what, lens, ctx", [("few", [40, 20, 60], [200, 120, 60]),
                                             ("tiled", [140, 20, 160], [300, 120, 160])])
def test_lost_blocks(rl, gpu, d, tpb, dtype, what, lens, ctx):
    """Rows that see a block past the arena are no numbers, the others stand; so with contexts past max_ctx."""
    def case():
        c = Case(13, lens, ctx, 4, 2, d, tpb, dtype)
        takes(gpu, c, what)
        return c

    c, (a, b, n) = case(), lens
    want = c.run(rl)
    c.check(want)
    want = want.reshape(-1, 4, d)
    bad = np.zeros(want.shape[:2], bool)
    c.table[1, 1, 96 // tpb] = 0xFFFFFFFF            # row 1, KV head 1: its queries are the tokens 100 .. 119
    bad[a:a + b, 2:] = True
    c.table[2, 0, 32 // tpb] = c.blocks              # row 2, KV head 0: the queries from token 32 on
    bad[a + b + 32:, :2] = True
    out = c.run(rl).reshape(want.shape)
    assert np.isnan(k8.floats(out, dtype)[bad]).all() and np.array_equal(out[~bad], want[~bad])
    c = case()
    want = c.run(rl)
    out = c.run(rl, ctx=[ctx[0], ctx[0] + 1, ctx[2]], max_ctx=ctx[0])
    assert np.isnan(k8.floats(out[a:a + b], dtype)).all()
    assert np.array_equal(out[:a], want[:a]) and np.array_equal(out[a + b:], want[a + b:])
    out = c.run(rl, ctx=[0xFFFFFFFF, *ctx[1:]])
    assert np.isnan(k8.floats(out[:a], dtype)).all() and np.array_equal(out[a:], want[a:])


@pytest.mark.parametrize("d, tpb, qh, dtype", [(128, 16, 4, "bf16"), (64, 32, 1, "fp16"), (64, 16, 2, "bf16")])
def test_few_rows_long_contexts(rl, gpu, d, tpb, qh, dtype):
    """So many rollouts that no keys are shared among workgroups, with contexts of more keys than a wave of the few-rows
    kernel knows block ids for (4,096), and more than twice as many; and blocks that are lost there."""
    n = gpu.cu_count // 2 + 2
    lens, ctx = [1 + i % 2 for i in range(n)], [2 + 7 * i % 90 for i in range(n)]
    ctx[3], ctx[60], ctx[n - 1] = 4097, 9000, 8200
    c = Case(d + tpb, lens, ctx, qh, 1, d, tpb, dtype)
    takes(gpu, c, "few")
    out = c.run(rl)
    c.check(out)
    assert np.array_equal(c.run(rl, graph=2), out)
    at = int(c.q_starts[60])
    c.table[60, 0, 8500 // tpb] = 0xFFFFFFFF
    f = c.run(rl)
    assert np.isnan(k8.floats(f[at:at + lens[60]], dtype)).all()
    assert np.array_equal(f[:at], out[:at]) and np.array_equal(f[at + lens[60]:], out[at + lens[60]:])


@pytest.mark.parametrize("what, new, ctx", [("few", 5, 200), ("tiled", 300, 350)])
def test_offsets_past_4_gib(rl, gpu, what, new, ctx):
    """Blocks behind 4 GiB of arena."""
    c = Case(20, [new], [ctx], 2, 1, 128, 16, "bf16")
    takes(gpu, c, what)
    size = 4 * 16 * 128
    blocks, held = (5 << 30) // size, -(-ctx // 16)
    big = rl.DeviceBuffer(blocks * size, zero=True)
    want = c.run(rl)
    c.check(want)
    table = c.table.copy()
    for j in range(held):
        table[0, 0, j] = blocks - 1 - 3 * j
        big.upload(c.arena[c.table[0, 0, j]], int(table[0, 0, j]) * size)
    up = rl.DeviceBuffer.from_array
    dev = [up(x) for x in (table, np.array([ctx], np.uint32), c.q, np.array([0, new], np.uint32))]
    out = rl.DeviceBuffer(c.q.nbytes)
    args = rl.AttnChunkArgs(arena_base=big.ptr, arena_bytes=big.nbytes, layout=rl.KvLayoutDesc.paged(16, 128),
                            block_table=dev[0].ptr, table_stride=c.stride, batch=1, q_heads=2, kv_heads=1,
                            dtype=rl.DTYPE_BF16, ctx_lens=dev[1].ptr, max_ctx=ctx, q_starts=dev[3].ptr, q_tokens=new,
                            max_q=new, q=dev[2].ptr, out=out.ptr)
    ws = rl.attn_chunk_workspace(args)
    rl.attn_chunk(args)
    rl.sync()
    assert np.array_equal(out.download(np.uint16, (new, 256)), want)
    for x in dev + [big, out, ws]:
        x.close()

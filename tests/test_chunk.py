"""rl_hip_attn_chunk without a GPU: the ctypes mirror and every refusal (the arguments are checked before the device)."""
import ctypes as C

import pytest

import helpers

P = 1 << 20  # an aligned address that is never read


def test_mirror(rl):
    probe = helpers.load_shared("tests/c/chunk_probe.c", link_runtime=False)
    probe.chunk_probe.restype = C.c_size_t
    a = rl.AttnChunkArgs
    want = [C.sizeof(a), a.max_ctx.offset, a.q_tokens.offset, a.scale.offset, a.workspace_bytes.offset]
    assert [probe.chunk_probe(i) for i in range(5)] == want


def chunk_args(rl, **kw):
    a = dict(arena_base=P, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged(16, 128), block_table=P, table_stride=8,
             batch=2, q_heads=32, kv_heads=8, dtype=rl.DTYPE_BF16, ctx_lens=P, max_ctx=128, q_starts=P, q_tokens=10,
             max_q=8, q=P, out=P, scale=0.0, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return rl.AttnChunkArgs(**a)


@pytest.mark.parametrize("kw, words", [
    (dict(arena_base=None), "NULL"), (dict(block_table=None), "NULL"), (dict(ctx_lens=None), "NULL"),
    (dict(q_starts=None), "NULL"), (dict(q=None), "NULL"), (dict(out=None), "NULL"),
    (dict(layout=lambda rl: rl.KvLayoutDesc.paged8(16, 128)), "layout"),
    (dict(layout=lambda rl: rl.KvLayoutDesc.paged(8, 128)), "layout"), (dict(dtype=2), "dtype"),
    (dict(q_heads=12), "kv_heads"), (dict(kv_heads=0), "kv_heads"), (dict(q_heads=0), "kv_heads"),
    (dict(q_heads=65536), "kv_heads"), (dict(batch=0), "batch"), (dict(batch=65536), "batch"),
    (dict(arena_bytes=100), "no block"), (dict(max_ctx=129), "table_stride"),
    (dict(max_ctx=1 << 31, table_stride=1 << 28), "max_ctx"), (dict(max_q=1 << 29), "max_q"),
    (dict(q_tokens=1 << 31), "q_tokens"), (dict(batch=65535, max_q=1 << 11), "2^24"), (dict(scale=-1.0), "scale"),
    (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(q_stride=4088), "stride"),
    (dict(q_stride=4100), "stride"), (dict(out_stride=(1 << 24) + 8), "stride"),
    (dict(q_heads=65528, kv_heads=8, layout=lambda rl: rl.KvLayoutDesc.paged(16, 128), max_q=1), None),
    (dict(arena_base=P + 8), "aligned"), (dict(q=P + 2), "aligned"), (dict(out=P + 4), "aligned")])
def test_refusals(rl, kw, words):
    kw = {k: v(rl) if callable(v) else v for k, v in kw.items()}
    for call in (rl.lib().rl_hip_attn_chunk, rl.lib().rl_hip_attn_chunk_workspace):
        if words is None:  # the most heads are allowed, up to the device
            if rl.lib().rl_hip_is_open():
                continue
            words_ = "no device open"
        else:
            words_ = words
        assert call(C.byref(chunk_args(rl, **kw))) == (0 if call is rl.lib().rl_hip_attn_chunk_workspace else -1)
        assert words_ in rl.lib().rl_hip_last_error().decode()


def test_null(rl):
    assert rl.lib().rl_hip_attn_chunk(None) == -1
    assert rl.lib().rl_hip_attn_chunk_workspace(None) == 0

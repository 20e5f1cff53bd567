"""The 8-bit KV cache and the prompt attention without a GPU: layouts, the
ctypes mirror, and every refusal (the arguments are checked before the device)."""
import ctypes as C
from collections import Counter

import numpy as np
import pytest

import helpers
import kv8_helpers as k8

P = 1 << 20  # an aligned address that is never read


def test_layout_and_mirror(rl):
    probe = helpers.load_shared("tests/c/kv8_probe.c", link_runtime=False)
    probe.kv8_probe.restype = C.c_size_t
    a, p = rl.Kv8AppendArgs, rl.AttnPromptArgs
    want = [C.sizeof(a), a.tokens.offset, a.v_stride.offset, C.sizeof(p), p.q_starts.offset, p.scale.offset,
            p.workspace_bytes.offset]
    assert [probe.kv8_probe(i) for i in range(7)] == want
    for t in (16, 32):
        for d in (64, 128):
            got = rl.KvLayoutDesc()
            assert probe.kv8_layout(t, d, C.byref(got)) == 0
            assert bytes(got) == bytes(rl.KvLayoutDesc.paged8(t, d))
            assert got.block_bytes == 2 * t * d + 128
    assert probe.kv8_layout(24, 128, C.byref(rl.KvLayoutDesc())) == -1
    assert probe.kv8_layout(16, 96, C.byref(rl.KvLayoutDesc())) == -1


def test_e4m3_model():
    """The numpy model rounds as the definition says: midpoints to the even byte, the rest to the nearer."""
    pos = k8.E4M3[:127]
    assert pos[-1] == 448 and pos[1] == 2.0 ** -9 and np.all(np.diff(pos) > 0)
    mid = (pos[:-1] + pos[1:]) / 2
    assert np.array_equal(k8.to_e4m3(mid), np.arange(126) + np.arange(126) % 2)
    assert np.array_equal(k8.to_e4m3(-mid * (1 - 2.0 ** -40)), np.arange(126) | 128)
    assert np.array_equal(k8.to_e4m3(mid * (1 + 2.0 ** -40)), np.arange(1, 127))
    assert k8.scale_of(np.array([448.0])) == 1 and k8.scale_of(np.array([448.01])) == 2
    assert k8.scale_of(np.array([0.0, np.inf, np.nan])) == k8.LEAST


@pytest.mark.parametrize("grid", [512, 64, 16, 510])
def test_runs_over_the_xcds(grid):
    """However few of a grid's workgroups have work (workgroup b runs on XCD b % 8): each run once, on all XCDs alike,
    neighbours on one XCD."""
    probe = helpers.load_shared("tests/c/kv8_runs_probe.c", link_runtime=False)
    probe.kv8_probe_run.restype = C.c_uint32
    for n in [1, 2, 7, 8, 9, grid // 3, grid - 1, grid]:
        runs = {b: probe.kv8_probe_run(b, grid, n) for b in range(grid)}
        has = {r: b % 8 for b, r in runs.items() if r != 0xFFFFFFFF}
        assert sorted(has) == list(range(n)) and sum(r != 0xFFFFFFFF for r in runs.values()) == n
        per_xcd = [Counter(has.values())[x] for x in range(8)]
        assert max(per_xcd) - min(per_xcd) <= 1, (n, per_xcd)
        if grid % 8 == 0:
            assert [has[r] for r in range(n)] == sorted(has.values())


@pytest.mark.parametrize("rows, tokens, d, past", [(64 * 8, 1800, 128, False), (512 * 8, 200, 128, False), (64 * 8, 2048, 128, False),
                                                   (64 * 8, 2080, 128, True), (512 * 8, 260, 128, True), (8 * 8, 32768, 64, False),
                                                   (8 * 8, 32800, 64, True), (0, 0, 128, False)])
def test_bytes_that_are_read(rows, tokens, d, past):
    """What is read past the caches is decided by the bytes of the rows, not by what turning to them costs as well."""
    probe = helpers.load_shared("tests/c/kv8_runs_probe.c", link_runtime=False)
    probe.kv8_probe_bytes.restype = C.c_uint64
    units = -(-tokens // 32)
    got = probe.kv8_probe_bytes(C.c_uint64(rows * (units + 8)), rows, d)
    assert got == rows * units * 32 * 2 * d and (got > 256 << 20) == past


def append_args(rl, **kw):
    a = dict(arena_base=P, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged8(16, 128), block_table=P, table_stride=4,
             batch=2, kv_heads=8, dtype=rl.DTYPE_BF16, positions=P, starts=None, tokens=2, max_new=1, cow_src=None,
             k_new=P, v_new=P, k_stride=0, v_stride=0)
    a.update(kw)
    return rl.Kv8AppendArgs(**a)


def attn_args(rl, **kw):
    a = dict(arena_base=P, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged8(16, 128), block_table=P, table_stride=4,
             batch=2, q_heads=32, kv_heads=8, dtype=rl.DTYPE_BF16, ctx_lens=P, max_ctx=64, grid_waves=0, scale=0.0, q=P,
             out=P, out_f32=None, workspace=P, workspace_bytes=1 << 30)
    a.update(kw)
    return rl.AttnArgs(**a)


def prompt_args(rl, **kw):
    a = dict(q=P, k=P, v=P, out=P, q_starts=P, kv_starts=None, seqs=2, q_tokens=100, kv_tokens=100, max_q=60, max_kv=60,
             q_heads=32, kv_heads=8, head_dim=128, dtype=rl.DTYPE_BF16, scale=0.0, workspace=P,
             workspace_bytes=1 << 30)
    a.update(kw)
    return rl.AttnPromptArgs(**a)


L16 = ("layout", lambda rl: rl.KvLayoutDesc.paged(16, 128))


@pytest.mark.parametrize("kw, words", [
    (dict(arena_base=None), "NULL"), (dict(block_table=None), "NULL"), (dict(positions=None), "NULL"),
    (dict(k_new=None), "NULL"), (dict(v_new=None), "NULL"), (dict([L16]), "layout"), (dict(dtype=2), "dtype"),
    (dict(batch=0), "batch"), (dict(kv_heads=0), "kv_heads"), (dict(batch=65536, tokens=65536), "batch"),
    (dict(max_new=0), "max_new"), (dict(max_new=2), "max_new"), (dict(tokens=3), "tokens"),
    (dict(batch=65535, starts=P, max_new=1 << 20, table_stride=1 << 16), "2^25"),
    (dict(arena_bytes=4223), "no block"), (dict(k_stride=1016), "stride"), (dict(v_stride=1028), "stride"),
    (dict(arena_base=P + 8), "aligned"), (dict(k_new=P + 2), "aligned"), (dict(v_new=P + 4), "aligned")])
def test_append_refusals(rl, kw, words):
    kw = {k: v(rl) if callable(v) else v for k, v in kw.items()}
    assert rl.lib().rl_hip_kv8_append(C.byref(append_args(rl, **kw))) == -1
    assert words in rl.lib().rl_hip_last_error().decode()


@pytest.mark.parametrize("kw, words", [
    (dict(arena_base=None), "NULL"), (dict(block_table=None), "NULL"), (dict(ctx_lens=None), "NULL"),
    (dict(q=None), "NULL"), (dict(out=None), "NULL"), (dict([L16]), "layout"), (dict(dtype=7), "dtype"),
    (dict(q_heads=12), "kv_heads"), (dict(q_heads=136), "kv_heads"), (dict(kv_heads=0), "kv_heads"),
    (dict(q_heads=0), "kv_heads"), (dict(batch=0), "batch"), (dict(batch=65536), "batch"),
    (dict(arena_bytes=100), "no block"), (dict(grid_waves=8), "grid_waves"), (dict(max_ctx=65), "table_stride"),
    (dict(batch=65535, kv_heads=256, q_heads=256, max_ctx=8000, table_stride=500), "units"),
    (dict(batch=65535, kv_heads=257, q_heads=257), "batch"),
    (dict(batch=65535, kv_heads=33, q_heads=528), "batch"),
    (dict(arena_base=P + 64 + 8), "aligned"), (dict(q=P + 2), "aligned")])
def test_decode_refusals(rl, kw, words):
    kw = {k: v(rl) if callable(v) else v for k, v in kw.items()}
    a = attn_args(rl, **kw)
    assert rl.lib().rl_hip_attn_decode_kv8(C.byref(a)) == -1
    assert words in rl.lib().rl_hip_last_error().decode()
    assert rl.lib().rl_hip_attn_decode_kv8_workspace(C.byref(a)) == 0
    assert words in rl.lib().rl_hip_last_error().decode()


@pytest.mark.parametrize("kw, words", [
    (dict(q=None), "NULL"), (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(out=None), "NULL"),
    (dict(q_starts=None), "NULL"), (dict(head_dim=96), "head_dim"), (dict(q_heads=12), "kv_heads"),
    (dict(kv_heads=0), "kv_heads"), (dict(q_heads=0), "kv_heads"), (dict(dtype=2), "dtype"), (dict(seqs=0), "sequences"),
    (dict(seqs=65536), "sequences"), (dict(max_q=1 << 29), "max_q"), (dict(max_kv=1 << 31), "max_kv"),
    (dict(q_tokens=1 << 31), "q_tokens"), (dict(kv_tokens=1 << 31), "kv_tokens"),
    (dict(seqs=65535, max_q=8192), "2^24"), (dict(seqs=65535, kv_heads=256, q_heads=256, max_q=129), "2^24"),
    (dict(scale=-1.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(q_stride=4088), "stride"), (dict(k_stride=1028), "stride"), (dict(v_stride=(1 << 24) + 8), "stride"),
    (dict(out_stride=100), "stride"), (dict(q=P + 8), "aligned"), (dict(k=P + 2), "aligned"), (dict(out=P + 4), "aligned")])
def test_prompt_refusals(rl, kw, words):
    a = prompt_args(rl, **kw)
    assert rl.lib().rl_hip_attn_prompt(C.byref(a)) == -1
    assert words in rl.lib().rl_hip_last_error().decode()
    assert rl.lib().rl_hip_attn_prompt_workspace(C.byref(a)) == 0
    assert words in rl.lib().rl_hip_last_error().decode()


def test_null_and_closed(rl):
    """NULL arguments, and right ones without a device."""
    lib = rl.lib()
    for f in (lib.rl_hip_kv8_append, lib.rl_hip_attn_decode_kv8, lib.rl_hip_attn_prompt):
        assert f(None) == -1
        assert "NULL" in lib.rl_hip_last_error().decode()
    if lib.rl_hip_is_open():
        pytest.skip("a device is open in this process")
    assert lib.rl_hip_kv8_append(C.byref(append_args(rl))) == -1
    assert "no device open" in lib.rl_hip_last_error().decode()
    assert lib.rl_hip_attn_decode_kv8(C.byref(attn_args(rl))) == -1
    assert "no device open" in lib.rl_hip_last_error().decode()
    assert lib.rl_hip_attn_prompt(C.byref(prompt_args(rl))) == -1
    assert "no device open" in lib.rl_hip_last_error().decode()

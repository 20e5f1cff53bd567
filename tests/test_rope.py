"""rl_hip_rope_append without a GPU: the ctypes mirror, the frequencies, and every refusal (the arguments are checked
before the device)."""
import ctypes as C

import numpy as np
import pytest

import helpers

P = 1 << 20  # an aligned address that is never read


def test_mirror(rl):
    probe = helpers.load_shared("tests/c/rope_probe.c", link_runtime=False)
    probe.rope_probe.restype = C.c_size_t
    a = rl.RopeAppendArgs
    want = [C.sizeof(a), a.tokens.offset, a.rot_dim.offset, a.k_out.offset, a.k_out_stride.offset]
    assert [probe.rope_probe(i) for i in range(5)] == want


def test_freqs(rl):
    f = rl.rope_freqs(128, 500000.0)
    want = 500000.0 ** (-np.arange(64) / 64)
    assert np.allclose(f, want, rtol=1e-14) and f[0] == 1
    assert len(rl.rope_freqs(0)) == 0
    assert rl.lib().rl_rope_freqs(None, 64, 1e4) == -1
    out = np.zeros(64)
    for rot, theta in ((63, 1e4), (64, 0.0), (64, -1.0), (64, float("nan"))):
        assert rl.lib().rl_rope_freqs(out.ctypes.data, rot, theta) == -1


def rope_args(rl, **kw):
    a = dict(arena_base=P, arena_bytes=1 << 20, layout=rl.KvLayoutDesc.paged(16, 128), block_table=P, table_stride=4,
             batch=2, q_heads=32, kv_heads=8, dtype=rl.DTYPE_BF16, positions=P, starts=None, tokens=2, cow_src=None,
             freqs=P, rot_dim=128, pairing=rl.ROPE_HALVES, q=P, q_out=P, k_new=P, v_new=P, k_out=None)
    a.update(kw)
    return rl.RopeAppendArgs(**a)


@pytest.mark.parametrize("kw, words", [
    (dict(positions=None), "NULL"), (dict(q=None), "NULL"), (dict(q_out=None), "NULL"), (dict(k_new=None), "NULL"),
    (dict(v_new=None), "NULL"), (dict(block_table=None), "NULL"), (dict(freqs=None), "NULL"),
    (dict(arena_base=None, q=None, q_out=None), "NULL"), (dict(arena_base=None, k_out=P, k_new=None), "NULL"),
    (dict(layout=lambda rl: rl.KvLayoutDesc.paged8(16, 128)), "layout"),
    (dict(layout=lambda rl: rl.KvLayoutDesc.paged(16, 96)), "layout"), (dict(dtype=2), "dtype"),
    (dict(rot_dim=24), "rot_dim"), (dict(rot_dim=144), "rot_dim"), (dict(pairing=2), "pairing"), (dict(batch=0), "batch"),
    (dict(batch=65536, tokens=65536), "batch"), (dict(q_heads=0), "q_heads"), (dict(q_heads=65536), "q_heads"),
    (dict(kv_heads=0), "kv_heads"), (dict(kv_heads=65536), "kv_heads"), (dict(tokens=3), "tokens"),
    (dict(starts=P, tokens=1 << 31), "tokens"), (dict(arena_base=None, cow_src=P), "cow_src"),
    (dict(arena_bytes=8191), "no block"), (dict(q_stride=4088), "stride"), (dict(q_out_stride=4100), "stride"),
    (dict(q_stride=4096, q_out_stride=4104), "another stride"), (dict(k_stride=1016), "stride"),
    (dict(v_stride=1028), "stride"), (dict(k_out=P, k_out_stride=8), "stride"),
    (dict(arena_base=P + 8), "aligned"), (dict(q=P + 2), "aligned"), (dict(q_out=P + 8), "aligned"),
    (dict(k_new=P + 4), "aligned"), (dict(v_new=P + 2), "aligned"), (dict(k_out=P + 2), "aligned"),
    (dict(freqs=P + 4), "aligned")])
def test_refusals(rl, kw, words):
    kw = {k: v(rl) if callable(v) else v for k, v in kw.items()}
    assert rl.lib().rl_hip_rope_append(C.byref(rope_args(rl, **kw))) == -1
    assert words in rl.lib().rl_hip_last_error().decode()


def test_null(rl):
    assert rl.lib().rl_hip_rope_append(None) == -1


@pytest.mark.parametrize("kw", [dict(), dict(q=None, q_out=None, q_heads=0), dict(rot_dim=0, freqs=None),
                                dict(arena_base=None, block_table=None, v_new=None, k_out=P),
                                dict(arena_base=None, block_table=None, v_new=None, k_new=None, kv_heads=0),
                                dict(starts=P, tokens=0), dict(q_stride=8192, k_stride=2048, q_out=2 * P)])
def test_what_is_allowed(rl, kw):
    """Up to the device, which is not open."""
    if rl.lib().rl_hip_is_open():
        pytest.skip("a device is open")
    assert rl.lib().rl_hip_rope_append(C.byref(rope_args(rl, **kw))) == -1
    assert "no device open" in rl.lib().rl_hip_last_error().decode()

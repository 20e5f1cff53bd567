"""The rotating append, chunk attention, token logprobs and their gradients one after the other, as a rollout and its
training step use them: prompts in pieces behind a shared prefix, tokens one by one, then the tokens' scores. Each stage
is checked against its formula on what the stage before it left on the device."""
import numpy as np
import pytest

import kv8_helpers as k8
import test_gpu_logprob as lpt
from test_gpu_prompt import compare, starts_of
from test_gpu_rope import close, turned

pytestmark = pytest.mark.gpu

QH, KVH, D, TPB, VOCAB = 4, 2, 128, 16, 900


def test_pieces_tokens_and_scores(rl, gpu):
    rng = np.random.default_rng(5)
    up = rl.DeviceBuffer.from_array
    dtype, hidden = "bf16", QH * D
    prefix, own, steps, b = 40, [30, 3, 77], 6, 3       # 40 shared tokens end inside a block
    total = [prefix + n + steps for n in own]
    stride = max(-(-t // TPB) for t in total)
    shared = -(-prefix // TPB)
    # blocks: the prefix's per head, then each row's own from the prefix's last, partly filled block on
    prefix_blocks = np.arange(KVH * shared).reshape(KVH, shared)
    table = np.zeros((b, KVH, stride), np.uint32)
    n = KVH * shared
    for i in range(b):
        for g in range(KVH):
            table[i, g, :shared - 1] = prefix_blocks[g, :-1]
            k = stride - (shared - 1)
            table[i, g, shared - 1:] = n + np.arange(k)
            n += k
    perm = rng.permutation(n)
    table, prefix_blocks = perm[table].astype(np.uint32), perm[prefix_blocks].astype(np.uint32)
    arena = up(np.full((n, 2, TPB, D), 0x7FFF, np.uint16))
    layout = rl.KvLayoutDesc.paged(TPB, D)
    freqs = rl.rope_freqs(D, 500000.0)
    dev_f, dev_t, dev_pt = up(freqs), up(table), up(prefix_blocks[None])
    held = {}  # what each row's cache should hold: (row, position) -> K, V as the device wrote them

    def piece(tab, tab_host, lens, positions, cow=None):
        """Append and attend; returns the attention's rows [tokens][hidden]."""
        m, rows = int(sum(lens)), len(lens)
        q, k, v = (k8.bits(rng.standard_normal((m, h, D)), dtype) for h in (QH, KVH, KVH))
        st, ctx = starts_of(list(lens)), [p + x for p, x in zip(positions, lens)]
        one = all(x == 1 for x in lens)
        dev = dict(q=up(q), k=up(k), v=up(v), p=up(np.asarray(positions, np.uint32)), s=up(np.asarray(st, np.uint32)),
                   c=up(np.asarray(ctx, np.uint32)), o=rl.DeviceBuffer(q.nbytes))
        if cow is not None:
            dev["w"] = up(np.asarray(cow, np.int32))
        rl.rope_append(rl.RopeAppendArgs(
            arena_base=arena.ptr, arena_bytes=arena.nbytes, layout=layout, block_table=tab.ptr,
            table_stride=tab_host.shape[2], batch=rows, q_heads=QH, kv_heads=KVH, dtype=rl.DTYPE_BF16,
            positions=dev["p"].ptr, starts=None if one else dev["s"].ptr, tokens=m,
            cow_src=dev["w"].ptr if cow is not None else None, freqs=dev_f.ptr, rot_dim=D, pairing=rl.ROPE_HALVES,
            q=dev["q"].ptr, q_out=dev["q"].ptr, k_new=dev["k"].ptr, v_new=dev["v"].ptr))
        a = rl.AttnChunkArgs(arena_base=arena.ptr, arena_bytes=arena.nbytes, layout=layout, block_table=tab.ptr,
                             table_stride=tab_host.shape[2], batch=rows, q_heads=QH, kv_heads=KVH, dtype=rl.DTYPE_BF16,
                             ctx_lens=dev["c"].ptr, max_ctx=max(ctx), q_starts=dev["s"].ptr, q_tokens=m, max_q=max(lens),
                             q=dev["q"].ptr, out=dev["o"].ptr)
        ws = rl.attn_chunk_workspace(a)
        rl.attn_chunk(a)
        rl.sync()
        out, qt = dev["o"].download(np.uint16, q.shape), dev["q"].download(np.uint16, q.shape)
        blocks = arena.download(np.uint16, (n, 2, TPB, D))
        at = np.concatenate([np.arange(p, p + x) for p, x in zip(positions, lens)])
        row = np.repeat(np.arange(rows), lens)
        ref, mag = turned(k8.floats(q, dtype), at, freqs, D, True)
        close(qt, ref, mag, dtype)
        ref, mag = turned(k8.floats(k, dtype), at, freqs, D, True)
        kk, vv = [], []
        for i in range(rows):
            t = np.arange(ctx[i])
            rows_kv = blocks[tab_host[i][:, t // TPB].T, :, (t % TPB)[:, None]]   # [tokens][heads][plane][d]
            kk.append(rows_kv[:, :, 0])
            vv.append(rows_kv[:, :, 1])
            new = slice(positions[i], ctx[i])
            close(kk[i][new], ref[row == i], mag[row == i], dtype)
            assert np.array_equal(vv[i][new], v[row == i])
            key = ("prefix", 0) if tab is dev_pt else ("row", i)
            before = held.get(key, held.get(("prefix", 0)))
            if positions[i]:  # nothing that was cached before has changed
                assert np.array_equal(kk[i][:positions[i]], before[0]) and np.array_equal(vv[i][:positions[i]], before[1])
            held[key] = kk[i], vv[i]
        compare(out, qt, np.concatenate(kk), np.concatenate(vv), st, starts_of(ctx), KVH, dtype)
        for x in list(dev.values()) + [ws]:
            x.close()
        return out.reshape(m, hidden)

    # the shared prefix in two pieces, then each row's own prompt, whose first token copies the prefix's last block
    piece(dev_pt, prefix_blocks[None], [23], [0])
    piece(dev_pt, prefix_blocks[None], [17], [23])
    cow = np.repeat(prefix_blocks[None, :, -1], b, 0)
    piece(dev_t, table, own, [prefix] * b, cow=cow)
    x = [piece(dev_t, table, [1] * b, [prefix + m + s for m in own]) for s in range(steps)]
    # the generated tokens' hidden states, [row][step], scored; the last row ended two tokens early
    c = lpt.Case(6, b * steps, VOCAB, hidden, none=0)
    c.x = np.ascontiguousarray(np.stack(x, 1).reshape(b * steps, hidden))
    c.target[-2:] = 0xFFFFFFFF
    out = c.run(rl)
    c.check(out)
    # the same as graph, three times over
    for got, want in zip(c.run(rl, graph=3), out):
        assert np.array_equal(got, want)
    for d in (arena, dev_f, dev_t, dev_pt):
        d.close()


def test_a_step_down_the_gradient(rl, gpu):
    """A policy gradient step, -advantage logprob: the rewarded tokens' logprobs rise and the others' fall, by what the
    gradient says (to first order)."""
    rows, vocab, hidden = 40, 500, 256
    c = lpt.Case(7, rows, vocab, hidden, none=0)
    advantage = np.where(np.arange(rows) % 2, 1.0, -1.0)
    c.grad = (-advantage / rows).astype(np.float32)
    lp, _, dx, _ = c.run(rl)
    rate = 0.5
    was = k8.floats(c.x, "bf16")
    step = -rate * k8.floats(dx, "bf16")
    c.x = k8.bits(was + step, "bf16")
    moved = k8.floats(c.x, "bf16") - was          # the step that bf16 rows took
    now = c.run(rl, dx=False, dw=False)[0]
    # d logprob = (dloss/dx / grad) . step; the second-order term is at most half of |step|^2 times the largest variance of
    # w . direction, which is below max |w|^2
    first = (k8.floats(dx, "bf16") / c.grad[:, None] * moved).sum(1)
    w2 = (k8.floats(c.w, "bf16") ** 2).sum(1).max()
    second = (moved ** 2).sum(1) * w2
    rounding = 2 * 2.0 ** -8 * np.abs(k8.floats(dx, "bf16") / c.grad[:, None] * moved).sum(1)
    assert (np.abs(now - lp - first) <= second + rounding + 2e-5).all()

"""rl_hip_rope_append against the rotation in 64 bits and the arena's rule."""
import numpy as np
import pytest

import kv8_helpers as k8

pytestmark = pytest.mark.gpu


def turned(x, pos, freqs, rot, halves):
    """x [tokens][heads][d] in 64 bits and, of each element, the magnitudes that were added up."""
    t = pos[:, None].astype(np.float64) * freqs
    c, s = np.cos(t)[:, None], np.sin(t)[:, None]
    y, mag = x.copy(), np.zeros_like(x)
    i = (slice(0, rot // 2), slice(rot // 2, rot)) if halves else (slice(0, rot, 2), slice(1, rot, 2))
    a, b = x[..., i[0]], x[..., i[1]]
    y[..., i[0]], y[..., i[1]] = a * c - b * s, a * s + b * c
    mag[..., i[0]] = mag[..., i[1]] = np.abs(a) + np.abs(b)
    return y, mag


def close(got, ref, mag, dtype):
    """Sine and cosine in 32 bits: the reduced angle (at most 1) is rounded (2^-25), the series cut off (2^-24) and its
    terms rounded (2^-23 in all), so each is within 2^-22; the two products and their sum add 3 x 2^-24. Together less than
    2^-21 of the magnitudes. Then one rounding to 16 bits (fp16 below 2^-14: half of 2^-24)."""
    tol = k8.HALF_STEP[dtype] * np.abs(ref) * 1.01 + 2.0 ** -21 * mag + (2.0 ** -25 if dtype == "fp16" else 0.0)
    off = np.abs(k8.floats(got, dtype) - ref)
    assert (off <= np.where(mag > 0, tol, 0)).all(), (float((off / (tol + 1e-300)).max()), np.argwhere(~(off <= tol))[:4])


class Case:
    def __init__(self, seed, lens, pos, qh, kvh, d, tpb, dtype, spare=4, stride=None):
        self.rng = rng = np.random.default_rng(seed)
        self.lens, self.pos, self.d, self.tpb, self.dtype = np.asarray(lens), np.asarray(pos, np.uint32), d, tpb, dtype
        self.qh, self.kvh = qh, kvh
        n = int(self.lens.sum())
        need = -(-(self.pos.astype(np.int64) + self.lens) // tpb)
        self.stride = stride or max(1, int(need.max()))
        b = len(lens)
        self.table = rng.permutation(b * kvh * self.stride).astype(np.uint32).reshape(b, kvh, self.stride)
        self.blocks = b * kvh * self.stride + spare
        self.arena = rng.integers(0, 1 << 16, (self.blocks, 2, tpb, d), dtype=np.uint16)
        self.q, self.k, self.v = (k8.bits(rng.standard_normal((n, h, d)), dtype) for h in (qh, kvh, kvh))
        self.starts = np.concatenate([[0], np.cumsum(self.lens)]).astype(np.uint32)
        self.row = np.repeat(np.arange(b), self.lens)
        self.at = self.pos[self.row].astype(np.int64) + np.arange(n) - self.starts[self.row]

    def run(self, rl, rot=None, halves=True, theta=10000.0, freqs=None, starts=True, cow=None, arena=True, k_out=False,
            q=True, inplace=False, pad=(0, 0, 0, 0, 0), tokens=None, arena_blocks=None, graph=0, rows=None):
        rot = self.d if rot is None else rot
        self.freqs = rl.rope_freqs(rot, theta) if freqs is None else freqs
        up = rl.DeviceBuffer.from_array

        def wide(x, p):
            return np.concatenate([x.reshape(len(x), -1), np.full((len(x), p), 0x5A5A, np.uint16)], 1)

        n = len(self.q) if rows is None else rows
        qw, kw = self.qh * self.d, self.kvh * self.d
        dev = dict(a=up(self.arena), t=up(self.table), p=up(self.pos), f=up(self.freqs), q=up(wide(self.q, pad[0])),
                   k=up(wide(self.k, pad[2])), v=up(wide(self.v, pad[3])), s=up(self.starts),
                   ko=up(np.full((n, kw + pad[4]), 0x1234, np.uint16)))
        dev["qo"] = dev["q"] if inplace else up(np.full((n, qw + pad[1]), 0x1234, np.uint16))
        if cow is not None:
            dev["c"] = up(np.asarray(cow, np.int32))
        stride = [w + p if p else 0 for w, p in zip((qw, qw, kw, kw, kw), pad)]
        if inplace:
            stride[1] = stride[0]
        blocks = self.blocks if arena_blocks is None else arena_blocks
        args = rl.RopeAppendArgs(
            arena_base=dev["a"].ptr if arena else None, arena_bytes=blocks * 4 * self.tpb * self.d,
            layout=rl.KvLayoutDesc.paged(self.tpb, self.d), block_table=dev["t"].ptr, table_stride=self.stride,
            batch=len(self.lens), q_heads=self.qh, kv_heads=self.kvh, dtype=k8.dtype_id(rl, self.dtype),
            positions=dev["p"].ptr, starts=dev["s"].ptr if starts else None,
            tokens=len(self.q) if tokens is None else tokens, cow_src=dev["c"].ptr if cow is not None else None,
            freqs=dev["f"].ptr, rot_dim=rot, pairing=rl.ROPE_HALVES if halves else rl.ROPE_NEIGHBOURS,
            q=dev["q"].ptr if q else None, q_out=dev["qo"].ptr if q else None, k_new=dev["k"].ptr, v_new=dev["v"].ptr,
            k_out=dev["ko"].ptr if k_out else None, q_stride=stride[0], q_out_stride=stride[1], k_stride=stride[2],
            v_stride=stride[3], k_out_stride=stride[4])
        if graph:
            g = rl.Graph(lambda: rl.rope_append(args))
            for _ in range(graph):
                dev["a"].upload(self.arena)
                g.launch()
                rl.sync()
            g.close()
        else:
            rl.rope_append(args)
            rl.sync()
        qo = dev["qo"].download(np.uint16, (n, qw + (pad[0] if inplace else pad[1])))
        ko, a = dev["ko"].download(np.uint16, (n, kw + pad[4])), dev["a"].download(np.uint16, self.arena.shape)
        for b in set(dev.values()):
            b.close()
        return qo, ko, a

    def check(self, qo, ko, a, rot, halves, skip=(), k_out=False, q=True, base=None):
        """base: the arena as it would be with nothing appended; skip: tokens whose place is past the table or arena."""
        n = len(self.q)
        if q:
            ref, mag = turned(k8.floats(self.q, self.dtype), self.at, self.freqs, rot, halves)
            got = qo[:n, :self.qh * self.d].reshape(self.q.shape)
            close(got, ref, mag, self.dtype)
            same = np.broadcast_to(mag == 0, got.shape) & (np.arange(self.d) >= rot)
            assert np.array_equal(got[same], self.q[same])
        ref, mag = turned(k8.floats(self.k, self.dtype), self.at, self.freqs, rot, halves)
        if k_out:
            close(ko[:n, :self.kvh * self.d].reshape(self.k.shape), ref, mag, self.dtype)
        want = (self.arena if base is None else base).copy()
        for t in range(n):
            if t in skip:
                continue
            blk = self.table[self.row[t], :, self.at[t] // self.tpb]
            slot = self.at[t] % self.tpb
            got = a[blk, 0, slot]
            close(got, ref[t], mag[t], self.dtype)
            assert np.array_equal(got[:, rot:], self.k[t, :, rot:])
            want[blk, 0, slot], want[blk, 1, slot] = got, self.v[t]
        assert np.array_equal(a, want)


@pytest.mark.parametrize("d, tpb, qh, kvh, dtype", [(128, 16, 8, 2, "bf16"), (64, 32, 4, 4, "fp16"), (128, 32, 5, 5, "fp16"),
                                                    (64, 16, 7, 1, "bf16")])
@pytest.mark.parametrize("halves", [True, False])
@pytest.mark.parametrize("part", [1, 2, 4])
def test_one_token_each(rl, gpu, d, tpb, qh, kvh, dtype, halves, part):
    rng = np.random.default_rng(d + part)
    b = 37
    c = Case(d + qh, [1] * b, rng.integers(0, 300, b), qh, kvh, d, tpb, dtype)
    rot = d // part
    c.check(*c.run(rl, rot=rot, halves=halves, starts=False), rot, halves)


@pytest.mark.parametrize("d, tpb, qh, kvh, dtype, halves", [(128, 16, 8, 2, "bf16", True), (64, 32, 4, 4, "fp16", False),
                                                            (64, 16, 3, 1, "fp16", True)])
@pytest.mark.parametrize("lens", [[1], [0, 0, 5, 0], [17, 1, 0, 64, 33], [300], [7] * 70])
def test_pieces(rl, gpu, d, tpb, qh, kvh, dtype, halves, lens):
    rng = np.random.default_rng(sum(lens))
    c = Case(len(lens), lens, rng.integers(0, 100, len(lens)), qh, kvh, d, tpb, dtype)
    c.check(*c.run(rl, halves=halves, k_out=True), d, halves, k_out=True)


@pytest.mark.parametrize("batch", [63, 64, 65, 400, 4500])
def test_many_rows(rl, gpu, batch):
    """Most rows without a new token, more of them between two that have one than are looked at together."""
    rng = np.random.default_rng(batch)
    lens = np.zeros(batch, int)
    lens[rng.integers(0, batch, 12)] = rng.integers(1, 20, 12)
    lens[batch - 1] = 3
    c = Case(batch, lens, rng.integers(0, 20, batch), 2, 1, 64, 16, "bf16")
    c.check(*c.run(rl), 64, True)
    lens[:] = 0
    lens[batch // 2] = 9
    c = Case(batch, lens, rng.integers(0, 20, batch), 2, 1, 64, 16, "bf16")
    c.check(*c.run(rl), 64, True)


@pytest.mark.parametrize("tokens", [1500, 12000])
def test_heads_per_wave(rl, gpu, tokens):
    """As many tokens as each wave takes two, and four, heads for; head counts that do not divide."""
    c = Case(tokens, [tokens // 3, tokens - tokens // 3], [3, 40], 13, 3, 128, 16, "bf16")
    c.check(*c.run(rl), 128, True)
    c = Case(tokens, [tokens // 3, tokens - tokens // 3], [0, 7], 32, 1, 64, 32, "fp16")
    c.check(*c.run(rl, halves=False), 64, False)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_far_positions(rl, gpu, dtype):
    """Angles of millions of radians, and at every octant's border."""
    c = Case(5, [40], [0], 4, 1, 128, 16, dtype)
    c.pos[:] = 3_000_000_000
    c.at = c.pos[0].astype(np.int64) + np.arange(40)
    c.stride = 3
    got = c.run(rl, theta=500000.0)
    ref, mag = turned(k8.floats(c.q, dtype), c.at, c.freqs, 128, True)
    # the product in 64 bits is off by up to 2^-53 of 3e9 radians, here and in the model alike
    tol = k8.HALF_STEP[dtype] * np.abs(ref) * 1.01 + (2.0 ** -21 + 3e9 * 2.0 ** -51) * mag + 2.0 ** -25
    assert (np.abs(k8.floats(got[0].reshape(c.q.shape), dtype) - ref) <= tol).all()
    assert np.array_equal(got[2], c.arena)  # (past the table)
    c = Case(6, [64], [0], 4, 1, 128, 16, dtype)
    got = c.run(rl, freqs=np.arange(64) * (np.pi / 4))
    c.check(*got, 128, True)


def test_strides_in_place_and_rows_of_nobody(rl, gpu):
    rng = np.random.default_rng(2)
    c = Case(3, [3, 20, 9], rng.integers(0, 50, 3), 6, 2, 64, 16, "bf16")
    qo, ko, a = c.run(rl, pad=(8, 16, 24, 40, 64), k_out=True)
    c.check(qo, ko, a, 64, True, k_out=True)
    assert (qo[:, 6 * 64:] == 0x1234).all() and (ko[:, 2 * 64:] == 0x1234).all()
    plain = qo[:, :6 * 64]
    got = c.run(rl, pad=(8, 0, 0, 0, 0), inplace=True)[0]
    assert np.array_equal(got[:, :6 * 64], plain) and (got[:, 6 * 64:] == 0x5A5A).all()
    # the first token and the last two belong to no row
    starts = c.starts.copy()
    c.starts = starts + 1
    c.starts[-1] = len(c.q) - 2
    c.at = c.pos[c.row].astype(np.int64) + np.arange(len(c.q)) - starts[c.row]
    qo, _, _ = c.run(rl)
    assert (qo[0] == 0x1234).all() and (qo[-2:] == 0x1234).all() and not (qo[1:-2] == 0x1234).all(1).any()


def test_without_arena_or_queries(rl, gpu):
    c = Case(9, [5, 30], [4, 70], 4, 2, 128, 16, "fp16")
    full = c.run(rl, k_out=True)
    qo, ko, a = c.run(rl, arena=False, k_out=True)
    assert np.array_equal(qo, full[0]) and np.array_equal(ko, full[1]) and np.array_equal(a, c.arena)
    qo, ko, a = c.run(rl, q=False, k_out=True)
    assert (qo == 0x1234).all() and np.array_equal(ko, full[1]) and np.array_equal(a, full[2])
    qo, ko, a = c.run(rl, arena=False)
    assert np.array_equal(qo, full[0]) and (ko == 0x1234).all() and np.array_equal(a, c.arena)
    # nothing turned: the rows' bits, whatever they are
    c.k[:], c.q[:] = c.rng.integers(0, 1 << 16, c.k.shape), c.rng.integers(0, 1 << 16, c.q.shape)
    qo, ko, _ = c.run(rl, rot=0, k_out=True)
    assert np.array_equal(qo.reshape(c.q.shape), c.q) and np.array_equal(ko.reshape(c.k.shape), c.k)


@pytest.mark.parametrize("starts", [True, False])
@pytest.mark.parametrize("d, tpb", [(128, 16), (64, 32)])
def test_copy_on_write(rl, gpu, d, tpb, starts):
    rng = np.random.default_rng(tpb)
    b, kvh = 12, 3
    lens = rng.integers(1, 40, b) if starts else [1] * b
    if starts:
        lens[4] = 0
    c = Case(b, lens, rng.integers(0, 60, b), 2, kvh, d, tpb, "bf16", spare=20)
    cow = np.full((b, kvh), -1)
    shared = c.blocks - 20 + rng.integers(0, 20, (b, kvh))
    cow[::2] = shared[::2]
    cow[1, 0] = c.blocks + 5              # past the arena: nothing is copied
    base = c.arena.copy()
    for i in range(0, b, 2):
        for g in range(kvh):
            slot = c.pos[i] % tpb
            if c.lens[i]:
                base[c.table[i, g, c.pos[i] // tpb], :, :slot] = c.arena[cow[i, g], :, :slot]
    got = c.run(rl, starts=starts, cow=cow)
    c.check(*got, d, True, base=base)


def test_past_table_and_arena(rl, gpu):
    """Positions past the table, idle rows and blocks past the arena write nothing; the queries are turned all the same."""
    c = Case(11, [1] * 6, [5, 47, 48, 0xFFFFFFFF, 20, 33], 2, 2, 64, 16, "bf16", stride=3)
    lost = [2, 3]
    c.check(*c.run(rl, starts=False), 64, True, skip=lost)
    c = Case(12, [1] * 6, [5, 47, 12, 30, 20, 33], 2, 2, 64, 16, "bf16", stride=3)
    c.table[4, :, 1] = 0xFFFFFFFF
    c.check(*c.run(rl, starts=False), 64, True, skip=[4])
    c = Case(13, [30, 25], [5, 0], 2, 1, 64, 16, "bf16", stride=3)
    keep = int(c.table[1, 0, 1])
    got = c.run(rl, arena_blocks=keep)
    lost = [t for t in range(55) if c.table[c.row[t], 0, c.at[t] // 16] >= keep]
    assert lost
    c.check(*got, 64, True, skip=lost)


def test_graph(rl, gpu):
    c = Case(21, [12, 0, 50], [3, 9, 60], 8, 2, 128, 16, "bf16")
    one = c.run(rl, k_out=True)
    for a, b in zip(one, c.run(rl, k_out=True, graph=3)):
        assert np.array_equal(a, b)


def test_equals_the_plain_append(rl, gpu):
    """Nothing turned, one token each: the arena of rl_hip_kv_append byte for byte, copies on write included."""
    rng = np.random.default_rng(1)
    b, kvh = 9, 2
    c = Case(31, [1] * b, rng.integers(0, 48, b), 1, kvh, 128, 16, "fp16", spare=6)
    cow = np.where(rng.random((b, kvh)) < 0.5, c.blocks - 6 + rng.integers(0, 6, (b, kvh)), -1).astype(np.int32)
    got = c.run(rl, rot=0, starts=False, cow=cow, q=False)[2]
    up = rl.DeviceBuffer.from_array
    dev = [up(x) for x in (c.arena, c.table, c.pos, cow, c.k, c.v)]
    rl.kv_append(rl.AppendArgs(arena_base=dev[0].ptr, arena_bytes=dev[0].nbytes, layout=rl.KvLayoutDesc.paged(16, 128),
                               block_table=dev[1].ptr, table_stride=c.stride, batch=b, kv_heads=kvh, positions=dev[2].ptr,
                               cow_src=dev[3].ptr, k_new=dev[4].ptr, v_new=dev[5].ptr))
    rl.sync()
    assert np.array_equal(got, dev[0].download(np.uint16, c.arena.shape))
    for x in dev:
        x.close()


def test_offsets_past_4_gib(rl, gpu):
    """A block behind 4 GiB of arena, and a token behind 4 GiB of rows."""
    d, tpb = 128, 16
    c = Case(41, [1, 1], [7, 20], 1, 1, d, tpb, "bf16", stride=2)
    blocks = (5 << 30) // (4 * tpb * d)
    big = rl.DeviceBuffer(blocks * 4 * tpb * d, zero=True)
    c.table[0, 0, 0], c.table[1, 0, 1] = blocks - 1, blocks - 2
    up = rl.DeviceBuffer.from_array
    rows = rl.DeviceBuffer((5 << 30), zero=True)
    stride = (9 << 29) // 2  # 4.5 GiB between the two rows
    rows.upload(c.k[0], 0)
    rows.upload(c.k[1], stride * 2)
    dev = [up(x) for x in (c.table, c.pos, rl.rope_freqs(d), c.v)]
    rl.rope_append(rl.RopeAppendArgs(
        arena_base=big.ptr, arena_bytes=big.nbytes, layout=rl.KvLayoutDesc.paged(tpb, d), block_table=dev[0].ptr,
        table_stride=2, batch=2, kv_heads=1, dtype=rl.DTYPE_BF16, positions=dev[1].ptr, tokens=2, freqs=dev[2].ptr,
        rot_dim=d, k_new=rows.ptr, k_stride=stride, v_new=dev[3].ptr))
    rl.sync()
    ref, mag = turned(k8.floats(c.k, "bf16"), c.pos.astype(np.int64), rl.rope_freqs(d), d, True)
    for t, (blk, slot) in enumerate(((blocks - 1, 7), (blocks - 2, 4))):
        got = big.download(np.uint16, (2, tpb, d), blk * 4 * tpb * d)
        close(got[0, slot], ref[t, 0], mag[t, 0], "bf16")
        assert np.array_equal(got[1, slot], c.v[t, 0])
    for x in dev + [big, rows]:
        x.close()

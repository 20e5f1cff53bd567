"""The 8-bit KV cache in numpy, in 64 bits: e4m3 values, the append's rule and
plain attention, and the device calls of the tests that compare with them."""
import numpy as np

import synth

LEAST = 2.0 ** -126


def _values():
    v = np.empty(256)
    for byte in range(256):
        e, m = byte >> 3 & 15, byte & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[byte] = np.nan if byte & 127 == 127 else -x if byte & 128 else x
    return v


E4M3 = _values()
_POS = E4M3[:127]  # 0 .. 448, ascending


def to_e4m3(x):
    """The byte nearest to each x (ties to the even byte), |x| <= 448; NaN: 0x7F."""
    a = np.abs(x)
    i = np.clip(np.searchsorted(_POS, a, side="right") - 1, 0, 126)
    up = np.minimum(i + 1, 126)
    low, high = a - _POS[i], _POS[up] - a
    take = (high < low) | ((high == low) & (up % 2 == 0) & (up != i))
    byte = np.where(take, up, i).astype(np.uint8) | (np.signbit(x).astype(np.uint8) << 7)
    return np.where(np.isnan(x), np.uint8(0x7F), byte)


def scale_of(x):
    """The smallest power of two of which 448 reach every finite |x|, 2^-126 at least."""
    a = np.abs(x[np.isfinite(x)]).max(initial=0.0)
    s = LEAST
    while s * 448.0 < a:
        s *= 2.0
    return s


class Arena8:
    """An arena of 8-bit blocks on the host."""

    def __init__(self, blocks, t, d, seed=0, fill=True):
        self.t, self.d, self.n = t, d, 2 * t * d
        self.bytes = np.zeros((blocks, self.n + 128), np.uint8)
        if fill:  # random finite bytes, scales from 2^-7 to 2^-3
            rng = np.random.default_rng(seed)
            b = rng.integers(0, 256, (blocks, self.n), dtype=np.uint8)
            self.bytes[:, :self.n] = np.where(b & 127 == 127, 0x40, b)
            self.scales()[:] = 2.0 ** rng.integers(-7, -2, (blocks, 2))

    def scales(self):
        return self.bytes[:, self.n:self.n + 8].view(np.float32)

    def planes(self, blk):
        return self.bytes[blk, :self.n].reshape(2, self.t, self.d)

    def tokens(self, blocks, ctx):
        """K and V of the first ctx tokens of a row, [2][ctx][d] in 64 bits."""
        out = np.zeros((2, len(blocks) * self.t, self.d))
        for j, blk in enumerate(blocks):
            out[:, j * self.t:(j + 1) * self.t] = E4M3[self.planes(blk)] * self.scales()[blk][:, None, None].astype(float)
        return out[:, :ctx]

    def append(self, blocks, pos, kv, cow=-1):
        """kv [2][n][d] at positions pos, pos + 1, ... of the row with these blocks."""
        t = self.t
        done = 0
        while done < kv.shape[1]:
            lb, lo = (pos + done) // t, (pos + done) % t
            m = min(t - lo, kv.shape[1] - done)
            if lb >= len(blocks):
                return
            blk = blocks[lb]
            if blk < len(self.bytes):
                src = cow if cow >= 0 and done == 0 and lo > 0 else blk
                for q in range(2):
                    x = kv[q, done:done + m]
                    s = scale_of(x)
                    if lo > 0:
                        s = max(s, float(self.scales()[src, q]))
                        old = E4M3[self.planes(src)[q, :lo]] * float(self.scales()[src, q])
                        self.planes(blk)[q, :lo] = self._same(self.planes(src)[q, :lo], old / s,
                                                              s == float(self.scales()[src, q]))
                    self.planes(blk)[q, lo:lo + m] = to_e4m3(np.where(np.isfinite(x), x, np.nan) / s)
                    self.scales()[blk, q] = s
            done += m

    @staticmethod
    def _same(held, x, unchanged):
        return held if unchanged else to_e4m3(x)


def attend(q, k, v, scale, seen):
    """softmax(scale q k^T) v over the first seen[i] keys of query i, in 64 bits: o and sum p |v|
    (both normalised); q [n][d], k and v [m][d]."""
    o, a = np.zeros(q.shape), np.zeros(q.shape)
    for i, s in enumerate(seen):
        if s <= 0:
            continue
        x = k[:s] @ q[i] * scale
        p = np.exp(x - x.max())
        p /= p.sum()
        o[i], a[i] = p @ v[:s], p @ np.abs(v[:s])
    return o, a


def bits(x, dtype):
    return synth.to_scalar16(np.asarray(x, np.float32), dtype)


def floats(h, dtype):
    return synth.from_scalar16(h, dtype).astype(np.float64)


def dtype_id(rl, dtype):
    return rl.DTYPE_BF16 if dtype == "bf16" else rl.DTYPE_FP16


HALF_STEP = {"bf16": 2.0 ** -8, "fp16": 2.0 ** -11}


def run_append(rl, arena, table, positions, k, v, dtype, starts=None, max_new=1, cow=None, k_stride=0, v_stride=0,
               tokens=None, arena_blocks=None, graph=0):
    """The call on copies; returns the arena's bytes afterwards. k, v: 16-bit [tokens][...]."""
    blocks = len(arena.bytes) if arena_blocks is None else arena_blocks
    up = rl.DeviceBuffer.from_array
    dev = dict(a=up(arena.bytes), t=up(np.asarray(table, np.uint32)), p=up(np.asarray(positions, np.uint32)), k=up(k), v=up(v))
    if starts is not None:
        dev["s"] = up(np.asarray(starts, np.uint32))
    if cow is not None:
        dev["c"] = up(np.asarray(cow, np.int32))
    args = rl.Kv8AppendArgs(
        arena_base=dev["a"].ptr, arena_bytes=blocks * arena.bytes.shape[1], layout=rl.KvLayoutDesc.paged8(arena.t, arena.d),
        block_table=dev["t"].ptr, table_stride=table.shape[2], batch=table.shape[0], kv_heads=table.shape[1],
        dtype=dtype_id(rl, dtype), positions=dev["p"].ptr, starts=dev["s"].ptr if starts is not None else None,
        tokens=len(k) if tokens is None else tokens, max_new=max_new, cow_src=dev["c"].ptr if cow is not None else None,
        k_new=dev["k"].ptr, v_new=dev["v"].ptr, k_stride=k_stride, v_stride=v_stride)
    if graph:
        gr = rl.Graph(lambda: rl.kv8_append(args))
        for _ in range(graph):
            gr.launch()
        rl.sync()
        gr.close()
    else:
        rl.kv8_append(args)
        rl.sync()
    out = dev["a"].download(np.uint8, arena.bytes.shape)
    for b in dev.values():
        b.close()
    return out


def run_decode(rl, arena, table, ctx, q, dtype, max_ctx, scale=0.0, arena_blocks=None, graph=0):
    """The call on copies; returns (16-bit out, fp32 out). q: 16-bit [batch][q_heads][d]."""
    blocks = len(arena.bytes) if arena_blocks is None else arena_blocks
    up = rl.DeviceBuffer.from_array
    a, t, c, qb = up(arena.bytes[:blocks]), up(np.asarray(table, np.uint32)), up(np.asarray(ctx, np.uint32)), up(q)
    out, out32 = rl.DeviceBuffer(q.size * 2, zero=True), rl.DeviceBuffer(q.size * 4, zero=True)
    args = rl.attn_args(a, rl.KvLayoutDesc.paged8(arena.t, arena.d), t, table.shape[2], q.shape[0], q.shape[1],
                        table.shape[1], dtype_id(rl, dtype), c, max_ctx, qb, out, out32, scale=scale)
    ws = rl.attn_kv8_workspace(args)
    if graph:
        gr = rl.Graph(lambda: rl.attn_decode_kv8(args))
        for _ in range(graph):
            rl.check(rl.lib().rl_hip_memset_d(ws.ptr, 0xFF, ws.nbytes), "memset")
            gr.launch()
        rl.sync()
        gr.close()
    else:
        rl.attn_decode_kv8(args)
        rl.sync()
    got = out.download(np.uint16, q.shape), out32.download(np.float32, q.shape)
    for b in (a, t, c, qb, out, out32, ws):
        b.close()
    return got


def run_prompt(rl, q, k, v, q_starts, q_heads, kv_heads, d, dtype, kv_starts=None, max_q=None, strides=(0, 0, 0, 0),
               offsets=(0, 0, 0), q_tokens=None, kv_tokens=None, out_fill=0x1234, scale=0.0, out_rows=None, graph=0):
    """The call on copies of the 16-bit arrays q, k, v ([tokens][elements]); offsets are element offsets of the
    three into their rows. Returns out [rows][out stride or row]."""
    up = rl.DeviceBuffer.from_array
    qb, kb, vb, sb = up(q), up(k), up(v), up(np.asarray(q_starts, np.uint32))
    ksb = up(np.asarray(kv_starts, np.uint32)) if kv_starts is not None else None
    ks = np.asarray(q_starts if kv_starts is None else kv_starts)
    width = strides[3] or q_heads * d
    rows = len(q) if out_rows is None else out_rows
    ob = up(np.full((rows, width), out_fill, np.uint16))
    args = rl.AttnPromptArgs(
        q=qb.ptr + 2 * offsets[0], k=kb.ptr + 2 * offsets[1], v=vb.ptr + 2 * offsets[2], out=ob.ptr, q_stride=strides[0],
        k_stride=strides[1], v_stride=strides[2], out_stride=strides[3], q_starts=sb.ptr,
        kv_starts=ksb.ptr if ksb is not None else None, seqs=len(q_starts) - 1,
        q_tokens=len(q) if q_tokens is None else q_tokens, kv_tokens=len(k) if kv_tokens is None else kv_tokens,
        max_q=int(np.diff(q_starts).max()) if max_q is None else max_q, max_kv=int(np.diff(ks).max()), q_heads=q_heads,
        kv_heads=kv_heads, head_dim=d, dtype=dtype_id(rl, dtype), scale=scale)
    ws = rl.attn_prompt_workspace(args)
    if graph:
        gr = rl.Graph(lambda: rl.attn_prompt(args))
        for _ in range(graph):
            rl.check(rl.lib().rl_hip_memset_d(ws.ptr, 0xFF, ws.nbytes), "memset")
            gr.launch()
        rl.sync()
        gr.close()
    else:
        rl.attn_prompt(args)
        rl.sync()
    out = ob.download(np.uint16, (rows, width))
    for b in (qb, kb, vb, sb, ksb, ob, ws):
        if b is not None:
            b.close()
    return out

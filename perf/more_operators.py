"""Chunks of tokens over the 16-bit paged cache, and the scoring of tokens, measured.

Four operators, in the order a rollout and its training meet them:

  append  new tokens' queries and keys turned by their positions, keys and
          values into the blocks of the paged arena (rl_hip_rope_append):
          whole prompts, pieces of them, or one token per rollout
  chunk   causal attention of each rollout's newest tokens over the blocks
          that hold all of its tokens (rl_hip_attn_chunk)
  score   the log probability of given tokens under a vocabulary projection,
          without keeping the logits (rl_hip_token_logprob)
  train   the same with the gradients of the hidden states and the projection
          (rl_hip_token_logprob, then rl_hip_token_logprob_grad)

listed() names the cases, draw() gives more of the same ranges, prepare()
makes a case's inputs from a seed, run() is one pass (the plain form, or the
framework's calls where `own` is set), work() what a pass cannot do without and
exact() the results in 64 bits.

A block is [2][block][head_dim] scalars of one KV head: the K plane, the V plane.
"""
import math
import os
import sys
from types import SimpleNamespace

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one token of each of 64 rollouts: latency counts
        dict(name="append_b64_token", kind="append", batch=64, new_lo=1, new_hi=1, ctx_lo=512, ctx_hi=1280, q_heads=32,
             kv_heads=8, head_dim=128, block=16, dtype="bf16", rot=128, pairing="halves", theta=500000.0),
        # the prompts of 64 GRPO groups into an empty cache
        dict(name="append_grpo_64", kind="append", batch=64, new_lo=512, new_hi=1024, ctx_lo=0, ctx_hi=0, q_heads=32,
             kv_heads=8, head_dim=128, block=16, dtype="bf16", rot=128, pairing="halves", theta=10000.0),
        # pieces of prompts of the small-head configuration behind odd numbers of cached tokens, 32-token blocks,
        # half of the dims turned, neighbours as pairs
        dict(name="append_b24_d64_fp16", kind="append", batch=24, new_lo=1, new_hi=301, ctx_lo=5, ctx_hi=555, q_heads=8,
             kv_heads=8, head_dim=64, block=32, dtype="fp16", rot=32, pairing="neighbours", theta=10000.0),
        # one rollout's short piece of a prompt: latency
        dict(name="chunk_b1_37", kind="chunk", batch=1, new_lo=37, new_hi=37, old_lo=480, old_hi=480, shared=0,
             members=1, q_heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # the members of 8 GRPO groups: up to 512 private prompt tokens behind the 512 tokens their group shares
        dict(name="chunk_grpo_64", kind="chunk", batch=64, new_lo=1, new_hi=512, old_lo=512, old_hi=512, shared=512,
             members=8, q_heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # four drafted tokens of each of 64 rollouts checked behind 512 to 4,096 tokens
        dict(name="chunk_b64_draft4", kind="chunk", batch=64, new_lo=4, new_hi=4, old_lo=512, old_hi=4096, shared=0,
             members=1, q_heads=32, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # a piece of one long prompt, GQA 8
        dict(name="chunk_b1_2048_of_32k", kind="chunk", batch=1, new_lo=2048, new_hi=2048, old_lo=30000, old_hi=30000,
             shared=0, members=1, q_heads=64, kv_heads=8, head_dim=128, block=16, dtype="bf16"),
        # the small-head configuration (MHA 8 x d64, fp16), odd lengths, 32-token blocks
        dict(name="chunk_b9_d64_fp16", kind="chunk", batch=9, new_lo=3, new_hi=700, old_lo=0, old_hi=1500, shared=0,
             members=1, q_heads=8, kv_heads=8, head_dim=64, block=32, dtype="fp16"),
        # the tokens of one step of 24 rollouts
        dict(name="score_24", kind="score", rows=24, vocab=32000, hidden=4096, scale=1.0),
        # the 256 generated tokens of each of 8 rollouts, over the large vocabulary
        dict(name="score_2048_v128k", kind="score", rows=2048, vocab=128256, hidden=4096, scale=1.0),
        # a short micro-batch, sampled at temperature 0.8
        dict(name="train_200", kind="train", rows=200, vocab=32000, hidden=4096, scale=1.25),
        # the 256 generated tokens of each of 16 rollouts (two GRPO groups)
        dict(name="train_4096", kind="train", rows=4096, vocab=32000, hidden=4096, scale=1.0),
    ]


HEADS = ((32, 8, 128), (64, 8, 128), (16, 8, 128), (8, 8, 128), (8, 8, 64), (32, 8, 64), (16, 8, 64), (12, 2, 128))


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("append", "chunk", "score", "train"))
    if kind in ("score", "train"):
        hidden, vocab = 64 * rng.randint(8, 64), _log_int(rng, 4000, 130000)
        most = (1 << 42) // ((1 if kind == "score" else 4) * hidden * vocab)
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(8192, most))), vocab=vocab, hidden=hidden,
                    scale=rng.choice((1.0, 1.0, 0.7, 1.25)))
    qh, kvh, d = rng.choice(HEADS)
    dtype, block = rng.choice(("bf16", "bf16", "fp16")), rng.choice((16, 16, 32))
    if kind == "append":
        batch = _log_int(rng, 1, 256)
        hi = 1 if rng.random() < 0.4 else _log_int(rng, 2, max(2, min(4096, 65536 // batch)))
        ctx = _log_int(rng, 8, max(8, min(100000, 400000 // batch)))
        return dict(kind=kind, batch=batch, new_lo=rng.randint(1, hi), new_hi=hi, ctx_lo=rng.randint(0, ctx),
                    ctx_hi=ctx, q_heads=qh, kv_heads=kvh, head_dim=d, block=block, dtype=dtype,
                    rot=rng.choice((d, d, d // 2)), pairing=rng.choice(("halves", "neighbours")),
                    theta=rng.choice((10000.0, 500000.0)))
    batch = _log_int(rng, 1, 64)
    old = _log_int(rng, 1, max(1, min(32000, 250000 // batch)))
    # at most 2^31 (head, query, key) triples once padded to the longest row
    pairs = (1 << 31) // (batch * qh)
    hi = _log_int(rng, 1, max(1, min(2048, int((math.sqrt(old * old + 4.0 * pairs) - old) / 2))))
    members, shared = 1, 0
    if rng.random() < 0.3 and old > 64:
        members, shared = rng.choice((2, 4, 8)), block * (old // 2 // block)
    return dict(kind=kind, batch=batch, new_lo=rng.randint(1, hi), new_hi=hi, old_lo=rng.randint(shared, old),
                old_hi=old, shared=shared, members=members, q_heads=qh, kv_heads=kvh, head_dim=d, block=block,
                dtype=dtype)


# ---------------------------------------------------------------- inputs
def _spread(lo, hi, n):
    """n whole numbers from lo to hi in even steps (hi alone for n = 1)."""
    return [hi] if n == 1 else [lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _shuffled(lo, hi, n, rng):
    return rng.permutation(np.array(_spread(lo, hi, n), np.int64))


def _starts(lens):
    return np.concatenate([[0], np.cumsum(lens)]).astype(np.int64)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, std=1.0):
    out = torch.empty(shape, dtype=dtype, device="cuda")
    rows = max(1, (1 << 28) // max(1, out[0].numel())) if len(out) else 1
    for at in range(0, len(out), rows):
        n = min(rows, len(out) - at)
        out[at:at + n] = torch.randn((n, *shape[1:]), generator=g, device="cuda").mul_(std)
    return out


def _table(g, tokens, kv_heads, block, shared=0, members=1, room=0):
    """Blocks for `tokens` tokens per row at random places of an arena: the table [batch][kv_heads][stride] and how
    many blocks the arena has (`room` for each KV head at least). The first `shared` tokens (whole blocks) of `members`
    neighbouring rows are the same blocks."""
    need = -(-np.asarray(tokens) // block)
    stride, sb = max(1, int(need.max())), shared // block
    ids = np.zeros((len(need), kv_heads, stride), np.int64)
    n = 0
    for b, m in enumerate(need):
        first = 0
        if sb and b % members:
            ids[b, :, :sb] = ids[b - 1, :, :sb]
            first = sb
        k = kv_heads * (int(m) - first)
        ids[b, :, first:m] = n + np.arange(k).reshape(kv_heads, -1)
        n += k
    n = max(1, n, room * kv_heads)
    perm = torch.randperm(n, generator=g, device="cuda")
    has = torch.from_numpy(np.arange(stride)[None, :] < need[:, None]).cuda()[:, None]
    return torch.where(has, perm[torch.from_numpy(ids).cuda()], 0).to(torch.int32).contiguous(), stride, n


def prepare(case, seed):
    s = SimpleNamespace(case=case)
    g, rng = _gen(seed), np.random.default_rng(seed)
    if case["kind"] in ("score", "train"):
        r, v, h = case["rows"], case["vocab"], case["hidden"]
        s.w = _normal(g, (v, h), torch.bfloat16, 1.28 / math.sqrt(h))
        target = torch.randint(0, v, (r,), generator=g, device="cuda")
        # hidden states that lean to the token that was generated, some little, some so that it is all but sure
        lean = torch.rand(r, 1, generator=g, device="cuda") * 7.0
        s.x = (torch.randn(r, h, generator=g, device="cuda") + lean * s.w[target].float()).to(torch.bfloat16)
        # the places behind the end of a rollout have no token
        none = torch.rand(r, generator=g, device="cuda") < (0.03 if r > 8 else 0.0)
        s.target = torch.where(none, -1, target).to(torch.int32)
        s.logprob, s.lse = torch.empty(r, device="cuda"), torch.empty(r, device="cuda")
        if case["kind"] == "train":
            # group advantages over the number of tokens
            s.grad = torch.randn(r, generator=g, device="cuda") / r
            s.dx, s.dw = torch.empty_like(s.x), torch.empty_like(s.w)
        if own:
            _plan(s)
        return s
    dt, d, qh, kvh, b, t = (DTYPES[case["dtype"]], case["head_dim"], case["q_heads"], case["kv_heads"], case["batch"],
                            case["block"])
    new = _shuffled(case["new_lo"], case["new_hi"], b, rng)
    st = _starts(new)
    s.starts, s.max_new, n = _i32(st), int(new.max()), int(st[-1])
    if case["kind"] == "append":
        ctx = _shuffled(case["ctx_lo"], case["ctx_hi"], b, rng)
        # whichever way the lengths are paired, the cached and the new tokens fit
        s.table, s.stride, s.blocks = _table(g, ctx + new, kvh, t, room=int((-(-ctx // t) - (-new // t)).sum()))
        s.arena = _normal(g, (s.blocks, 2, t, d), dt)
        s.positions, s.one_each = _i32(ctx), case["new_hi"] == 1
        s.freqs = case["theta"] ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"])
        s.q, s.k, s.v = _normal(g, (n, qh, d), dt), _normal(g, (n, kvh, d), dt), _normal(g, (n, kvh, d), dt)
        s.q_out = torch.empty_like(s.q)
    else:
        old = _shuffled(case["old_lo"], case["old_hi"], b, rng)
        s.table, s.stride, s.blocks = _table(g, old + new, kvh, t, case["shared"], case["members"])
        s.arena = _normal(g, (s.blocks, 2, t, d), dt)
        s.ctx, s.max_ctx = _i32(old + new), int((old + new).max())
        s.q = _normal(g, (n, qh, d), dt)
        s.out = torch.empty_like(s.q)
    if own:
        _plan(s)
    return s


# ---------------------------------------------------------------- the framework's calls
def _rlrt():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gb300-rl-runtime_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import rlrt
    if not rlrt.lib().rl_hip_is_open():
        rlrt.open_device(torch.cuda.current_device())
    return rlrt


def _workspace(s, args, nbytes):
    ws = torch.zeros(max(1, nbytes), dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = ws.data_ptr(), ws.numel()
    s.ws.append(ws)


def _plan(s):
    """The arguments and the workspaces that a program keeps from step to step."""
    rl, c = _rlrt(), s.case
    s.ws = []
    if c["kind"] in ("score", "train"):
        r, v, h = c["rows"], c["vocab"], c["hidden"]
        a = rl.TokenLogprobArgs(x=s.x.data_ptr(), w=s.w.data_ptr(), targets=s.target.data_ptr(), rows=r, vocab=v,
                                hidden=h, x_stride=h, w_stride=h, scale=c["scale"], logprob=s.logprob.data_ptr(),
                                lse=s.lse.data_ptr())
        _workspace(s, a, rl.token_logprob_workspace_bytes(a))
        s.calls = [(rl.token_logprob, a)]
        if c["kind"] == "train":
            a = rl.TokenLogprobGradArgs(x=s.x.data_ptr(), w=s.w.data_ptr(), targets=s.target.data_ptr(), rows=r,
                                        vocab=v, hidden=h, x_stride=h, w_stride=h, scale=c["scale"],
                                        lse=s.lse.data_ptr(), grad_logprob=s.grad.data_ptr(), dx=s.dx.data_ptr(),
                                        dw=s.dw.data_ptr(), dx_stride=h, dw_stride=h)
            _workspace(s, a, rl.token_logprob_grad_workspace_bytes(a))
            s.calls.append((rl.token_logprob_grad, a))
        return
    dt = {"bf16": rl.DTYPE_BF16, "fp16": rl.DTYPE_FP16}[c["dtype"]]
    layout = rl.KvLayoutDesc.paged(c["block"], c["head_dim"])
    both = dict(arena_base=s.arena.data_ptr(), arena_bytes=s.arena.numel() * 2, layout=layout,
                block_table=s.table.data_ptr(), table_stride=s.stride, batch=c["batch"], q_heads=c["q_heads"],
                kv_heads=c["kv_heads"], dtype=dt, q=s.q.data_ptr())
    if c["kind"] == "append":
        a = rl.RopeAppendArgs(positions=s.positions.data_ptr(), starts=None if s.one_each else s.starts.data_ptr(),
                              tokens=s.q.shape[0], freqs=s.freqs.data_ptr(), rot_dim=c["rot"],
                              pairing={"halves": rl.ROPE_HALVES, "neighbours": rl.ROPE_NEIGHBOURS}[c["pairing"]],
                              q_out=s.q_out.data_ptr(), k_new=s.k.data_ptr(), v_new=s.v.data_ptr(), **both)
        s.calls = [(rl.rope_append, a)]
        return
    a = rl.AttnChunkArgs(ctx_lens=s.ctx.data_ptr(), max_ctx=s.max_ctx, q_starts=s.starts.data_ptr(),
                         q_tokens=s.q.shape[0], max_q=s.max_new, out=s.out.data_ptr(), **both)
    _workspace(s, a, rl.attn_chunk_workspace_bytes(a))
    s.calls = [(rl.attn_chunk, a)]


# ---------------------------------------------------------------- one pass
def run(state):
    s, kind = state, state.case["kind"]
    if own:
        for call, args in s.calls:
            call(args)
    else:
        {"append": _append, "chunk": _chunk, "score": _score, "train": _train}[kind](s)
    if kind == "append":
        return {"q": s.q_out, "arena": s.arena}
    if kind == "chunk":
        return s.out
    if kind == "score":
        return {"logprob": s.logprob, "lse": s.lse}
    return {"logprob": s.logprob, "lse": s.lse, "dx": s.dx, "dw": s.dw}


def _turn(x, cos, sin, rot, pairing):
    """x [tokens][heads][d] in 32 bits, cos and sin [tokens][1][rot / 2]."""
    y = x.clone()
    if pairing == "halves":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y[..., :rot // 2], y[..., rot // 2:rot] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y[..., 0:rot:2], y[..., 1:rot:2] = a * cos - b * sin, a * sin + b * cos
    return y


def _append(s):
    c, st = s.case, s.starts.long()
    t, kvh = c["block"], c["kv_heads"]
    i = torch.arange(s.q.shape[0], device="cuda")
    row = torch.searchsorted(st[1:], i, right=True)
    pos = s.positions.long()[row] + i - st[row]
    angle = (pos.double()[:, None] * s.freqs)[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    s.q_out.copy_(_turn(s.q.float(), cos, sin, c["rot"], c["pairing"]))
    k = _turn(s.k.float(), cos, sin, c["rot"], c["pairing"]).to(s.k.dtype)
    ids = s.table.long()[row[:, None], torch.arange(kvh, device="cuda"), (pos // t)[:, None]]
    s.arena[ids, 0, (pos % t)[:, None]] = k
    s.arena[ids, 1, (pos % t)[:, None]] = s.v


def _chunk(s):
    c, qs = s.case, s.starts.long()
    n, d, kvh, grp = c["batch"], c["head_dim"], c["kv_heads"], c["q_heads"] // c["kv_heads"]
    lq, lk, most = qs[1:] - qs[:-1], s.ctx.long(), s.stride * c["block"]
    iq, ik = torch.arange(s.max_new, device="cuda"), torch.arange(most, device="cuda")
    tq = (qs[:-1, None] + iq).clamp(max=s.q.shape[0] - 1)
    kv = s.arena[s.table.long()].float()                                         # [row][head][block][plane][slot][d]
    q = s.q[tq].float().view(n, s.max_new, kvh, grp, d).permute(0, 2, 3, 1, 4).reshape(n * kvh, grp * s.max_new, d)
    k = kv[:, :, :, 0].reshape(n * kvh, most, d).transpose(1, 2).contiguous()
    x = torch.bmm(q.mul_(1.0 / math.sqrt(d)), k).view(n, kvh * grp, s.max_new, most)
    seen = (ik <= iq[:, None] + (lk - lq)[:, None, None]) & (ik < lk[:, None, None])
    x.masked_fill_(~seen[:, None], -math.inf)
    x -= x.amax(-1, keepdim=True)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    v = kv[:, :, :, 1].reshape(n * kvh, most, d)
    o = torch.bmm(x.view(n * kvh, grp * s.max_new, most), v).view(n, kvh * grp, s.max_new, d) / total
    t = torch.arange(s.q.shape[0], device="cuda")
    row = torch.searchsorted(qs[1:], t, right=True)
    s.out.copy_(o[row, :, t - qs[row]])


def _score(s):
    logits = (s.x.float() @ s.w.float().t()).mul_(s.case["scale"])
    top = logits.amax(-1, keepdim=True)
    lse = top + (logits - top).exp_().sum(-1, keepdim=True).log()
    has = s.target >= 0
    at = logits.gather(1, s.target.long().clamp(min=0)[:, None])
    s.lse.copy_(lse[:, 0])
    s.logprob.copy_(torch.where(has, (at - lse)[:, 0], 0.0))
    return logits


def _train(s):
    p = _score(s)
    p.sub_(s.lse[:, None]).exp_()
    has = s.target >= 0
    g = torch.where(has, s.grad, 0.0) * s.case["scale"]
    p.mul_(-g[:, None])
    p.scatter_add_(1, s.target.long().clamp(min=0)[:, None], g[:, None])
    s.dx.copy_(p @ s.w.float())
    s.dw.copy_(p.t() @ s.x.float())


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] in ("score", "train"):
        r, v, h = case["rows"], case["vocab"], case["hidden"]
        n = 1 if case["kind"] == "score" else 3
        return {"bytes": 2 * (v * h + r * h) * (2 if n == 3 else 1) + (16 if n == 3 else 12) * r,
                "flops": 2.0 * n * r * v * h}
    d, qh, kvh, b, t = case["head_dim"], case["q_heads"], case["kv_heads"], case["batch"], case["block"]
    news = _spread(case["new_lo"], case["new_hi"], b)
    new = sum(news)
    if case["kind"] == "append":
        blocks = max(b, new / t) * kvh
        return {"bytes": 4 * new * (qh + 2 * kvh) * d + 4 * blocks + 8 * b + 4 * case["rot"],
                "flops": 3.0 * new * (qh + kvh) * case["rot"]}
    # how the new and the old tokens are paired is the seed's: every pairing is as likely
    olds = _spread(case["old_lo"], case["old_hi"], b)
    pairs = sum(x * (x + 1) // 2 for x in news) + new * sum(olds) / b
    held = new + sum(olds) - case["shared"] * (b - -(-b // case["members"]))
    return {"bytes": 4 * new * qh * d + 4 * held * kvh * d + 4 * kvh * held / t + 8 * b, "flops": 4.0 * d * qh * pairs}


# ---------------------------------------------------------------- 64 bits
def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] in ("score", "train"):
        return _exact_loss(s)
    d, kvh, t, grp = case["head_dim"], case["kv_heads"], case["block"], case["q_heads"] // case["kv_heads"]
    st = s.starts.tolist()
    if case["kind"] == "append":
        arena, q = s.arena.double(), s.q.double()
        half = case["rot"] // 2
        at = [(i, i + half) if case["pairing"] == "halves" else (2 * i, 2 * i + 1) for i in range(half)]
        first, second = [a for a, _ in at], [b for _, b in at]
        for b, p in enumerate(s.positions.tolist()):
            pos = torch.arange(p, p + st[b + 1] - st[b], device="cuda")
            # a turn by the angle is a product with cos + i sin
            angle = torch.outer(pos.double(), s.freqs)[:, None]
            z = torch.polar(torch.ones_like(angle), angle)
            k, v = s.k[st[b]:st[b + 1]].double(), s.v[st[b]:st[b + 1]].double()
            for x in (q[st[b]:st[b + 1]], k):
                y = torch.complex(x[..., first], x[..., second]) * z
                x[..., first], x[..., second] = y.real, y.imag
            for h in range(kvh):
                ids = s.table[b, h].long()[pos // t]
                arena[ids, 0, pos % t], arena[ids, 1, pos % t] = k[:, h], v[:, h]
        return {"q": q, "arena": arena}
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s.ctx.tolist()):
        q = s.q[st[b]:st[b + 1]].double()
        hidden = torch.ones(len(q), length, dtype=torch.bool, device="cuda").triu(length - len(q) + 1)
        for h in range(kvh):
            kv = s.arena[s.table[b, h, :-(-length // t)].long()].transpose(0, 1).reshape(2, -1, d)[:, :length].double()
            k = kv[0].t().contiguous()
            for j in range(h * grp, (h + 1) * grp):
                x = (q[:, j] @ k) * d ** -0.5
                out[st[b]:st[b + 1], j] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ kv[1]
    return out


def _exact_loss(s):
    c, rows = s.case, max(64, (1 << 27) // s.case["vocab"])
    w, target = s.w.double(), s.target.long()
    train = c["kind"] == "train"
    out = {k: torch.zeros(c["rows"], dtype=torch.float64, device="cuda") for k in ("logprob", "lse")}
    if train:
        out["dx"], out["dw"] = s.x.double(), torch.zeros_like(w)
    for at in range(0, c["rows"], rows):
        x, t = s.x[at:at + rows].double(), target[at:at + rows]
        i = torch.arange(len(x), device="cuda")
        logits = c["scale"] * torch.matmul(x, w.t())
        lse = torch.logsumexp(logits, 1)
        out["lse"][at:at + rows] = lse
        out["logprob"][at:at + rows] = torch.where(t >= 0, logits[i, t.clamp(min=0)] - lse, 0.0)
        if train:
            hot = torch.zeros_like(logits)
            hot[i, t.clamp(min=0)] = 1.0
            g = c["scale"] * torch.where(t >= 0, s.grad[at:at + rows].double(), 0.0)
            delta = (hot - torch.softmax(logits, 1)) * g[:, None]
            out["dx"][at:at + rows] = torch.matmul(delta, w)
            out["dw"] += torch.matmul(delta.t().contiguous(), x)
    return out

"""Which kernel a call of rl_hip_attn_chunk takes, by the rules and the constants in attn_chunk.hip and prompt_core.h,
read from there: tests that mean a certain kernel say so and notice when a rule moves them."""
import os
import re

HIP = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gb300-rl-runtime_amd", "csrc", "hip")


def _up(n, d):
    return -(-n // d)


def _numbers(pattern, name):
    return [int(x) for x in re.search(pattern, open(os.path.join(HIP, name)).read()).groups()]


def kernel(cus, lens, max_ctx, q_heads, kv_heads, max_q=None):
    """"few": attn_chunk_few_kernel; "tiled": attn_prompt_kernel; "split": that, its keys shared by workgroups."""
    few_rows, = _numbers(r"kFewRows = (\d+);", "attn_chunk.hip")
    unit, share, joined = _numbers(r"(\d+) \* \(\(units \+ 3\) / 4\) < (\d+) \* per_share \+ \(pl.split > 1 \? (\d+) : 0\)",
                                   "attn_chunk.hip")
    least, long_least = _numbers(r"kShareTiles = (\d+), kLongShareTiles = (\d+);", "prompt_core.h")
    group, max_q = q_heads // kv_heads, max(lens) if max_q is None else max_q
    pairs = len(lens) * kv_heads
    blocks, keys = pairs * _up(max_q * group, 128), _up(max_ctx, 64)
    shares = 1
    if 0 < blocks <= cus:
        shares = cus // blocks
        if keys >= long_least * (2 * cus // blocks):
            shares = 2 * cus // blocks
    split = max(1, min(shares, keys // least))
    units = _up(max_ctx, 32)
    few = (max_q * group <= few_rows and _up(max_q * group, 32) * pairs <= cus and
           unit * _up(units, 4) < share * _up(_up(units, 2), split) + (joined if split > 1 else 0))
    return "few" if few else "split" if split > 1 else "tiled"

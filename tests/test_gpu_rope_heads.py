"""rl_hip_rope_append: every number of heads per wave, chosen by the waves that a compute unit gets."""
import os
import re

import pytest

from test_gpu_rope import Case

pytestmark = pytest.mark.gpu

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gb300-rl-runtime_amd", "csrc", "hip",
                      "rope_append.hip")


def heads_per_wave(cus, tokens, heads, d):
    """By rope_append.hip's rule, with the constant that stands there."""
    enough = int(re.search(r"enough = (\d+)ull \* rl_cu_count\(\)", open(SOURCE).read()).group(1)) * cus
    groups = -(-tokens * (d // 16) // 64)
    return 4 if groups * -(-heads // 4) >= enough else 2 if groups * -(-heads // 2) >= enough else 1


@pytest.mark.parametrize("qh, kvh, d, tpb", [(13, 3, 128, 16), (32, 1, 64, 32)])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("halves, part", [(True, 1), (True, 2), (False, 1), (False, 2)])
@pytest.mark.parametrize("per", [2, 4])
def test_heads_per_wave(rl, gpu, per, qh, kvh, d, tpb, dtype, halves, part):
    """Head counts that do not divide; a token count just above the least for so many heads per wave."""
    heads, tokens = qh + 2 * kvh, 64
    while heads_per_wave(gpu.cu_count, tokens, heads, d) != per:
        tokens += 64
    tokens += 37
    assert heads_per_wave(gpu.cu_count, tokens, heads, d) == per
    c = Case(tokens + d, [tokens // 3, 0, tokens - tokens // 3], [3, 9, 40], qh, kvh, d, tpb, dtype)
    c.check(*c.run(rl, rot=d // part, halves=halves, k_out=True), d // part, halves, k_out=True)

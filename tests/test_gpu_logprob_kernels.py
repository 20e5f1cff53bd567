"""rl_hip_token_logprob_grad: the kernels that only larger calls take."""
import numpy as np
import pytest

from logprob_rules import Rules
from test_gpu_logprob import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows, hidden, logits", [(60, 192, "Logits64x32"), (100, 192, "Logits64x32"), (130, 448, "Logits64x32"),
                                                  (200, 192, "Logits256")])
def test_largest_tiles_of_dw(rl, gpu, rows, hidden, logits):
    """256 x 256 tiles, the last ones partly filled along the entries and along hidden, with D in two parts and with what
    its rounding takes put back."""
    rules, vocab = Rules(gpu.cu_count), 33001
    c = Case(rows + hidden, rows, vocab, hidden, none=0.05)
    c.target[rows // 2:rows // 2 + 6] = c.target[0] = 33000
    assert rules.logits_kind(rows, vocab) == logits and rules.dw_kind(hidden, vocab) == "Dw256"
    out = c.run(rl)
    c.check(out, targets_whole=True)
    for a, b in zip(out, c.run(rl, graph=2)):
        assert np.array_equal(a, b)


@pytest.mark.parametrize("rows, vocab, hidden, logits, dw, shares", [
    (1025, 140000, 192, ["Logits256", "Logits128x256"], ["Dw256", "Dw128"], 32),
    (2049, 70001, 64, ["Logits256", "Logits256"], ["Dw128", "Dw128"], 12)])
def test_pieces_and_shares(rl, gpu, rows, vocab, hidden, logits, dw, shares):
    """The vocabulary in two pieces, and each in shares for dx: the second piece's sums are added to the first's."""
    rules = Rules(gpu.cu_count)
    pieces, split, parts = rules.grad(rows, vocab, hidden)
    assert len(pieces) == 2 and split == shares and parts == 1
    assert [rules.logits_kind(rows, n) for n in pieces] == logits and [rules.dw_kind(hidden, n) for n in pieces] == dw
    c = Case(rows, rows, vocab, hidden, none=0.02)
    c.target[:4] = [0, pieces[0] - 1, pieces[0], vocab - 1]
    out = c.run(rl)
    c.check(out, targets_whole=True)
    for a, b in zip(out, c.run(rl, graph=2)):
        assert np.array_equal(a, b)


def test_pieces_with_d_in_two_parts(rl, gpu):
    """Few rows of a vocabulary that D, in two parts, holds in two pieces."""
    rows, vocab, hidden = 70, 530000, 64
    pieces, split, parts = Rules(gpu.cu_count).grad(rows, vocab, hidden)
    assert len(pieces) == 2 and split > 1 and parts == 2
    c = Case(1, rows, vocab, hidden, none=0.05)
    c.target[:4] = [0, pieces[0] - 1, pieces[0], vocab - 1]
    c.check(c.run(rl), targets_whole=True)

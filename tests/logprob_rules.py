"""Which kernels a call of rl_hip_token_logprob or its gradient takes, by the rules and the constants in
token_logprob.hip, read from there: tests that mean a certain kernel say so and notice when a rule moves them."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "gb300-rl-runtime_amd", "csrc", "hip",
                      "token_logprob.hip")
LOGITS = ("Logits256", "Logits128x256", "Logits128", "Logits64", "Logits64x32")


def _up(n, d):
    return -(-n // d)


class Rules:
    def __init__(self, cus):
        self.cus = cus
        text = open(SOURCE).read()
        self.tile = {}  # name: (BN, BM)
        for name, tn, wn, tm, wm in re.findall(r"using (\w+) = Gemm<(\d+), (\d+), (\d+), (\d+),", text):
            self.tile[name] = (32 * int(tn) * int(wn), 32 * int(tm) * int(wm))
        self.logits = [(name, *[int(x) for x in re.search(rf"cost_of<{name}>\(vocab, rows, (\d+), (\d+)\)", text).groups()])
                       for name in LOGITS]
        self.dw = [(name, *[int(x) for x in re.search(rf"cost_of<{name}>\(dw.hidden, n, (\d+), (\d+)\)", text).groups()])
                   for name in ("Dw128", "Dw256")]
        self.delta = 1 << int(re.search(r"kDeltaElements = 1ull << (\d+)", text).group(1))
        self.two_parts = int(re.search(r"pl.parts = rows <= (\d+) \? 2 : 1", text).group(1))
        self.dx = {name: int(per) for name, per in re.findall(r"dx_shape<(\w+)>\(rows, hidden, (\d+), tiles", text)}

    def _cost(self, name, per_cu, duration, n, m):
        bn, bm = self.tile[name]
        return _up(_up(n, bn) * _up(m, bm), per_cu * self.cus) * duration

    def logits_kind(self, rows, entries):
        return min(self.logits, key=lambda k: self._cost(*k, entries, rows))[0]

    def dw_kind(self, hidden, entries):
        small, large = self.dw
        return (small if self._cost(*small, hidden, entries) < self._cost(*large, hidden, entries) else large)[0]

    def grad(self, rows, vocab, hidden):
        """(entries of each piece, shares of a piece's vocabulary for dx, parts of D)"""
        parts = 2 if rows <= self.two_parts else 1
        d_rows = parts * _up(rows, 64) * 64
        width = min(_up(vocab, 256) * 256, max(1024, self.delta // d_rows // 256 * 256))
        name = "Dx32" if rows <= 32 else "Dx64" if rows <= 64 else "Dx128" if rows <= 128 else "DxMany"
        bn, bm = self.tile[name]
        tiles = _up(rows, bm) * _up(hidden, bn)
        pieces = [min(width, vocab - at) for at in range(0, vocab, width)]
        return pieces, max(1, min(self.dx[name] * self.cus // tiles, pieces[-1] // 512)), parts

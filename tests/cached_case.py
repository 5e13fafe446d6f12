"""Seeded paged FP8 caches with ragged queries, and the error bounds of what is
computed from them, for the tests of tree attention and attention weights.

Bounds, eps = 2^-24 the rounding step of float32:
  * a score s = sum of 128 exact products in some order of float32 sums, times a
    scale rounded three times, plus one fused multiply-add: off by at most
    ds = eps (128 A + 8 max(|s|, 1)), A the largest sum |q~ K| of a score, scaled
    (the sums dominate: 128 terms, each rounding at most eps A);
  * a weight exp(s - m) is then off by a factor of at most exp(ds + 4 eps (1 + |s - m|))
    (the exponential's own error and its argument's rounding), the sum of K of
    them by K eps more.
"""

import numpy as np
import torch

EPS = 2.0 ** -24
NAMES = {torch.bfloat16: "bf16", torch.float16: "f16", torch.float32: "f32", torch.float8_e4m3fn: "fp8"}


def score_error(bound, most):
    return EPS * (128 * bound + 8 * max(most, 1.0))


class Case:
    """lens: cached tokens of each sequence; counts: query tokens of each (the last ones)."""

    def __init__(self, dev, seed, lens, counts, Hq, Hkv, ps, q_dtype=torch.bfloat16, descales=True, spare_rows=0,
                 holes=(), head_major=False, strided_q=False, spare_table=0, first_page=0, k_sign=1.0):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        need = [-(-x // ps) for x in lens]
        P = sum(need) + 3
        self.fused = torch.randn(P, 2, ps, Hkv, 128, generator=g).mul_(2.0).to(torch.float8_e4m3fn)
        W = max([1, *need]) + spare_table
        perm = torch.randperm(P, generator=g).to(torch.int32)
        # entries past a sequence's pages name pages too: they are not to be read
        self.bt = torch.randint(0, P, (B, W), generator=g, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.bt[b, :k] = perm[at:at + k]
            at += k
        for k, (b, page) in enumerate(holes):
            self.bt[b, page] = -3 if k % 2 else P + 5
        self.cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        TQ = int(self.cu[-1]) + spare_rows
        self.q = (torch.randn(TQ, Hq, 128, generator=g) * 3).clamp(-448, 448).to(q_dtype)
        rng = np.random.default_rng(seed)
        self.ds = [rng.uniform(0.25, 1.0, (B, Hkv)).astype(np.float32) if descales else None for _ in range(3)]
        if descales:
            self.ds[1] *= np.float32(k_sign)
        self.lens, self.counts, self.B, self.TQ, self.rows = list(lens), list(counts), B, TQ, int(self.cu[-1])
        self.Hq, self.Hkv, self.ps, self.name = Hq, Hkv, ps, NAMES[q_dtype]
        self.scale = 128 ** -0.5
        # on the device
        f = self.fused.to(dev)
        if head_major:
            f = f.transpose(2, 3).contiguous().transpose(2, 3)
        if strided_q:  # a column slice of a projection
            wide = torch.zeros(TQ, Hq * 128 + 256, dtype=torch.float32).to(q_dtype).to(dev)
            wide[:, 128:128 + Hq * 128] = self.q.view(TQ, -1).to(dev)
            self.qd = wide[:, 128:128 + Hq * 128].view(TQ, Hq, 128) if TQ else self.q.to(dev)
        else:
            self.qd = self.q.to(dev)
        self.k, self.v = f[:, 0], f[:, 1]
        self.btd, self.cud = self.bt.to(dev), torch.from_numpy(self.cu).to(dev)
        self.lensd = torch.tensor(self.lens, dtype=torch.int32, device=dev)
        self.dd = [None if d is None else torch.from_numpy(d).to(dev) for d in self.ds]
        self.max_q = max([1, *counts])

    def raw(self, t):
        t = t.contiguous()
        if t.dtype == torch.float8_e4m3fn:
            return t.view(torch.uint8).numpy()
        return t.view(torch.int16).numpy().view(np.uint16) if t.element_size() == 2 else t.numpy().view(np.uint32)

    def host(self):
        """(q bits of the owned rows, k bytes, v bytes)"""
        return self.raw(self.q[:self.rows]), self.raw(self.fused[:, 0]), self.raw(self.fused[:, 1])

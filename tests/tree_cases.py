"""Inputs and 64-bit references of the drafted-tree tests: random trees, their ancestor masks, paged pools, and the attention
of every row from the definition, with the bound that the types' roundings give it."""

from __future__ import annotations

import numpy as np
import torch


def random_parents(n: int, rng: np.random.RandomState, chain: bool = False) -> list[int]:
    """Parents of a random tree of n nodes (a chain: each node's parent is the one before it); some nodes are roots."""
    if chain:
        return list(range(-1, n - 1))
    return [-1 if i == 0 or rng.rand() < 0.1 else rng.randint(max(0, i - 6), i) for i in range(n)]


def ancestor_sets(parents: list[int]) -> list[set[int]]:
    """Each node's ancestors and itself."""
    sets: list[set[int]] = []
    for i, p in enumerate(parents):
        sets.append({i} | (sets[p] if p >= 0 else set()))
    return sets


def mask_tensor(sets: list[set[int]], words: int) -> torch.Tensor:
    """int64 [rows, words] with the sets' elements as bits."""
    m = np.zeros((len(sets), words), dtype=np.uint64)
    for r, s in enumerate(sets):
        for a in s:
            m[r, a // 64] |= np.uint64(1) << np.uint64(a % 64)
    return torch.from_numpy(m.view(np.int64))


class Case:
    """A batch of trees over a paged pool. seqs: [(cached tokens, nodes)]; everything seeded."""

    def __init__(self, seqs, heads=(14, 2, 64), block=16, int8=False, seed=0, device="cuda", sets=None, words=None,
                 spare=3, chain=False, scale_dtype=torch.float16):
        self.seqs, (self.Hq, self.Hkv, self.D), self.B = seqs, heads, block
        self.scale = self.D ** -0.5
        rng = np.random.RandomState(seed)
        g = torch.Generator().manual_seed(seed)
        counts = [n for _, n in seqs]
        need = [-(-(c + n) // block) for c, n in seqs]
        self.N = sum(need) + spare
        ids = rng.permutation(self.N)
        width = max(max(need), 1)
        bt = np.full((len(seqs), width), -1, dtype=np.int32)
        at = 0
        for i, k in enumerate(need):
            bt[i, :k] = ids[at:at + k]
            at += k
        T = sum(counts)
        self.parents = [random_parents(n, rng, chain) for n in counts]
        self.sets = sets if sets is not None else [s for p in self.parents for s in ancestor_sets(p)]
        self.max_nodes = max(max(counts), 1)
        self.words = words or -(-self.max_nodes // 64)
        shape = (self.Hkv, self.N, block, self.D)
        k, v = torch.randn(shape, generator=g).bfloat16(), torch.randn(shape, generator=g).bfloat16()
        self.ks = self.vs = None
        if int8:
            k, self.ks = quantize(k, scale_dtype)
            v, self.vs = quantize(v, scale_dtype)
            self.ks, self.vs = self.ks.to(device), self.vs.to(device)
        self.k, self.v = k.to(device), v.to(device)
        self.q = torch.randn(T, self.Hq, self.D, generator=g).bfloat16().to(device)
        self.bt = torch.from_numpy(bt).to(device)
        self.ctx = torch.tensor([c + n for c, n in seqs], dtype=torch.int32, device=device)
        self.qs = torch.tensor(np.concatenate([[0], np.cumsum(counts)]), dtype=torch.int32, device=device)
        self.masks = mask_tensor(self.sets, self.words).to(device) if T else \
            torch.zeros(0, self.words, dtype=torch.int64, device=device)
        self.max_ctx = max(max(c + n for c, n in seqs), 1)

    def quant(self):
        from engine.hip_decode import QuantKV

        return None if self.ks is None else QuantKV(1, self.ks, self.vs)

    def reference(self):
        """(out, tol) [T, Hq, D] float64 on the CPU. The kernel's result is within tol of out:
        - the probability of key j is rounded to bf16 (times V's scale over INT8 pools): half a step, 2^-8 of it, so 2^-8 of
          sum p |v| at most; its exponent's argument carries the score's error, an fp32 sum of D products and three further
          roundings, (D + 8) 2^-24 of sum |q k| scale, and the exponential 2^-22: all relative to p, and the same again in
          the denominator;
        - up to 300 keys' partial sums in fp32 add less than 2^-14 of sum p |v|;
        - the result is rounded to bf16: 2^-8 of it."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        tol = torch.zeros_like(out)
        q, k, v = self.q.cpu().double(), self.k.cpu().double(), self.v.cpu().double()
        if self.ks is not None:
            k, v = k * self.ks.cpu().double()[..., None], v * self.vs.cpu().double()[..., None]
        G, at = self.Hq // self.Hkv, 0
        for i, (c, n) in enumerate(self.seqs):
            ids = self.bt[i, :-(-(c + n) // self.B)].cpu().long()
            sees = torch.zeros(n, c + n, dtype=torch.bool)
            sees[:, :c] = True
            for r in range(n):
                for a in self.sets[at + r]:
                    if a < n:
                        sees[r, c + a] = True
            for h in range(self.Hq):
                kk = k[h // G, ids].reshape(-1, self.D)[:c + n]
                vv = v[h // G, ids].reshape(-1, self.D)[:c + n]
                for r in range(n):
                    on = sees[r]
                    if not on.any():
                        continue
                    qr = q[at + r, h]
                    z = kk[on] @ qr * self.scale
                    p = torch.softmax(z, 0)
                    out[at + r, h] = p @ vv[on]
                    size = (kk[on].abs() @ qr.abs()).max() * self.scale
                    eps = 2 * ((self.D + 8) * 2.0 ** -24 * size + 2.0 ** -22) + 2.0 ** -14
                    tol[at + r, h] = (2.0 ** -8 + eps) * (p @ vv[on].abs()) + 2.0 ** -8 * out[at + r, h].abs()
            at += n
        return out, tol


def quantize(x: torch.Tensor, scale_dtype=torch.float16):
    """Per-token INT8 codes of x and their scales, absmax / 127."""
    s = (x.abs().amax(-1).float() / 127).to(scale_dtype)
    q = (x.float() / s.float().clamp_min(1e-30)[..., None]).round().clamp(-127, 127)
    return q.to(torch.int8), s

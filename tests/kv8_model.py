"""Plain models of the 8-bit KV cache and of the sampler (include/qwen_b200_ops.h), written token by token in
numpy: the codes and scales in the fp32 operations of the definition, everything else in float64."""
from __future__ import annotations

import numpy as np

BLOCK, HEAD = 64, 128
F = np.float32


class Model:
    """Codes and scales of one of K and V, and the block table."""

    def __init__(self, codes: np.ndarray, scales: np.ndarray, table: np.ndarray):
        self.codes, self.scales, self.table = codes.copy(), scales.copy(), table

    def append(self, x: np.ndarray, seq: int, start: int) -> None:
        """x [n][heads][128] fp32 to positions start .. of `seq`."""
        pos = start
        with np.errstate(all="ignore"):
            while pos < start + len(x):
                slot = pos % BLOCK
                n = min(BLOCK - slot, start + len(x) - pos)
                block = self.table[seq, pos // BLOCK]
                for h in range(x.shape[1]):
                    self._block(block, h, slot, x[pos - start : pos - start + n, h].astype(F))
                pos += n

    def _block(self, block: int, h: int, slot: int, x: np.ndarray) -> None:
        codes, old = self.codes[block, h], self.scales[block, h]
        a = np.abs(x).max()
        if not np.isfinite(x).all() or (slot > 0 and not (old >= 0 and old <= F(3.4e38))):
            s = F(np.nan)
        else:
            need = F(0) if a == 0 else max(F(a) * F(1 / 127), F(2.0**-126))
            s = need
            if slot > 0 and old > 0:
                s, twice = F(old), 0
                while s < need:
                    s, twice = F(s * F(2)), twice + 1
                codes[:slot] = np.rint(codes[:slot] * 2.0**-twice)
        self.scales[block, h] = s
        codes[slot : slot + len(x)] = np.clip(np.rint(x / s), -127, 127) if s > 0 else 0

    def values(self, seq: int, n: int, start: int = 0) -> np.ndarray:
        """[n][heads][128] fp32 values of positions start .. start + n - 1."""
        pos = np.arange(start, start + n)
        b = self.table[seq, pos // BLOCK]
        return self.codes[b, :, pos % BLOCK].astype(F) * self.scales[b][:, :, None]


def attention(q, k, v, scale):
    """q [heads][128]; k, v [tokens][kv heads][128]: (out, lse, largest sum |scale q k|) in float64."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    group = q.shape[0] // k.shape[1]
    out, lse, mag = np.zeros(q.shape), np.full(q.shape[0], -np.inf), 0.0
    if k.shape[0] == 0:
        return out, lse, mag
    for h in range(q.shape[0]):
        kk, vv = k[:, h // group], v[:, h // group]
        s = kk @ q[h] * scale
        mag = max(mag, float((np.abs(kk) @ np.abs(q[h])).max() * abs(scale)))
        m = s.max()
        p = np.exp(s - m)
        out[h], lse[h] = p @ vv / p.sum(), m + np.log(p.sum())
    return out, lse, mag


def kept(x, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token ids, weights) that the filters leave of one row's logits, best first."""
    x = np.asarray(x, np.float64)
    ok = x > -np.inf  # false for NaN
    order = np.argsort(np.where(ok, -x, np.inf), kind="stable")[: ok.sum()]
    if len(order) == 0:
        return order, np.zeros(0)
    if not temperature >= 2.0**-126:
        return order[:1], np.ones(1)
    with np.errstate(all="ignore"):
        d = x[order] - x[order[0]]
    w = np.where(x[order] == x[order[0]], 1.0, np.exp(np.where(np.isnan(d), -np.inf, d) / np.float64(temperature)))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        n = 1 + int(np.searchsorted(np.cumsum(w), top_p * w.sum(), side="left"))
        order, w = order[:n], w[:n]
    n = max(1, int((w >= min_p).sum()))
    return order[:n], w[:n]


def sample(x, u, **filters):
    order, w = kept(x, **filters)
    if len(order) == 0:
        return -1, 0.0
    at = min(int(np.searchsorted(np.cumsum(w), max(u, 0.0) * w.sum(), side="right")), len(w) - 1)
    return int(order[at]), float(w[at] / w.sum())

"""Oracle of the KV cache held in 4 bits: the stated format in 32-bit steps, the attention in 64 bits.  Test infrastructure only.

The arithmetic between the projections follows attention.rs:344-398 (rotate, append, softmax(q K^T / sqrt(head_dim)) V over the
positions a query sees); what the cache stands for follows the rule in include/kv_attention_b200.h.
"""
import numpy as np

GROUP = 32


def to_bf16(x):
    """Nearest bf16 number, ties to even, as f32 (finite values and NaN)."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    bits = x.view(np.uint32).astype(np.uint64)
    out = ((bits + 0x7fff + ((bits >> 16) & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), out)


def quantise(x):
    """x [..., head_dim] f32 -> what the cache stands for, f32, with the codes."""
    g = np.ascontiguousarray(x, np.float32).reshape(x.shape[:-1] + (-1, GROUP))
    low, high = g.min(-1, keepdims=True), g.max(-1, keepdims=True)
    step, base = to_bf16((high - low) / np.float32(15)), to_bf16(low)
    with np.errstate(divide="ignore", invalid="ignore"):
        code = np.where(step > 0, np.clip(np.rint((g - base) / step), 0, 15), 0).astype(np.float32)
    return (code * step + base).astype(np.float32).reshape(x.shape), code.astype(np.int32)


class Q4CacheOracle:
    """One sequence."""

    def __init__(self, num_heads, kv_heads, head_dim, capacity, rope_base=10000.0, rope=True):
        self.H, self.Hkv, self.hd, self.rope = num_heads, kv_heads, head_dim, rope
        half = head_dim // 2
        angle = np.arange(capacity, dtype=np.float64)[:, None] * np.power(float(rope_base), -np.arange(half, dtype=np.float64) / half)
        self.cos, self.sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
        self.keys = np.zeros((0, kv_heads, head_dim), np.float32)
        self.values = np.zeros((0, kv_heads, head_dim), np.float32)

    def __len__(self):
        return self.keys.shape[0]

    def _rotate(self, x, first, dtype):
        if not self.rope:
            return x.astype(dtype)
        half = self.hd // 2
        c = self.cos[first:first + x.shape[0], None].astype(dtype)
        s = self.sin[first:first + x.shape[0], None].astype(dtype)
        lo, hi = x[..., :half].astype(dtype), x[..., half:].astype(dtype)
        return np.concatenate([lo * c - hi * s, hi * c + lo * s], axis=-1)

    def append(self, k, v):
        n = k.shape[0]
        with np.errstate(over="ignore", invalid="ignore"):
            k = self._rotate(np.asarray(k, np.float32).reshape(n, self.Hkv, self.hd), len(self), np.float32)
        v = np.asarray(v, np.float32).reshape(n, self.Hkv, self.hd)
        with np.errstate(invalid="ignore"):
            bad = ~(np.abs(k) <= 2.0 ** 40).all(-1, keepdims=True) | ~(np.abs(v) <= 2.0 ** 40).all(-1, keepdims=True)
        kq, _ = quantise(np.where(bad, 0, k).astype(np.float32))
        vq, _ = quantise(np.where(bad, 0, v).astype(np.float32))
        self.keys = np.concatenate([self.keys, np.where(bad, np.float32(np.nan), kq)])
        self.values = np.concatenate([self.values, np.where(bad, np.float32(np.nan), vq)])

    def truncate(self, n):
        self.keys, self.values = self.keys[:n], self.values[:n]

    def forward_cached(self, q, k, v):
        """-> (merged [rows, H * hd] f64, how far a bf16 result may be off, elementwise).

        The device rounds the rotated query to f16 (half a step: 2^-11 of it), the values to bf16 (2^-8 of each), the weights to two bf16
        numbers (2^-16), and the result to bf16.  A score is then off by at most d = 2^-11 sum |q_c k_c| / sqrt(hd), and a little for
        the sums in 32 bits; the weights by e^(2 d) - 1 of themselves, and the rest adds up.
        """
        first, n = len(self), q.shape[0]
        self.append(k, v)
        q = self._rotate(np.asarray(q, np.float32).reshape(n, self.H, self.hd), first, np.float64)
        group = self.H // self.Hkv
        out, tol = np.empty((n, self.H, self.hd)), np.empty((n, self.H, self.hd))
        for i in range(n):
            see = first + i + 1
            for h in range(self.H):
                keys, values = self.keys[:see, h // group].astype(np.float64), self.values[:see, h // group].astype(np.float64)
                s = keys @ q[i, h] / np.sqrt(self.hd)
                d = (np.abs(keys) @ np.abs(q[i, h]) / np.sqrt(self.hd) * (2.0 ** -11 + 2.0 ** -18)).max()
                p = np.exp(s - s.max())
                p /= p.sum()
                out[i, h] = p @ values
                tol[i, h] = (p @ np.abs(values)) * (np.expm1(2 * d) + 2.0 ** -8 + 2.0 ** -14) + np.abs(out[i, h]) * 2.0 ** -8 + 1e-30
        return out.reshape(n, -1), tol.reshape(n, -1)

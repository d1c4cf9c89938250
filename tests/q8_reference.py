"""A cache line in 8 bits in plain numpy, from its definition: what the tests of the kernels compare with.

`Line` plays a batch of sequences step by step: it is given the rotated rows that a step's append wrote (so that a rounding border
in the rotation, which is tested by itself, does not decide about the rest), stores blocks in 8 bits with the very operations of the
definition in float32 (so that pages can be compared bit by bit), and forms attention in float64."""
import numpy as np

PAGE = 64


def rotate(x, positions, inv_freq, rotary_dim, pairs, turn_scale=1.0):
    """x [N, heads, D] float64, turned; `pairs` 0: lanes (i, i + rotary_dim / 2), 1: (2 i, 2 i + 1), 2: (16 (i // 8) + i % 8, that + 8)."""
    x = x.copy()
    for i in range(rotary_dim // 2):
        a, b = ((i, i + rotary_dim // 2), (2 * i, 2 * i + 1), (16 * (i // 8) + i % 8, 16 * (i // 8) + i % 8 + 8))[pairs]
        angle = positions * inv_freq[i]
        c, s = (turn_scale * np.cos(angle))[:, None], (turn_scale * np.sin(angle))[:, None]
        x[:, :, a], x[:, :, b] = x[:, :, a] * c - x[:, :, b] * s, x[:, :, b] * c + x[:, :, a] * s
    return x


def in_eight(block):
    """block [64, D] float32 -> (whole numbers as float32, scale)."""
    top = np.float32(np.abs(block).max())
    scale = top / np.float32(127.0)
    if scale == 0:
        return np.zeros_like(block), scale
    return np.clip(np.rint(block / scale), -127, 127), scale


class Line:
    def __init__(self, n_seqs, n_kv, dim):
        self.n_kv, self.dim = n_kv, dim
        self.rows = [np.zeros((0, 2, n_kv, dim), np.float32) for _ in range(n_seqs)]      # every position's key and value as stored

    def append(self, seq, rows):
        """rows [n, 2, n_kv, D] float32."""
        self.rows[seq] = np.concatenate([self.rows[seq], rows])

    def block(self, seq, b):
        """(whole numbers [2, n_kv, 64, D], scales [n_kv, 2]) of a complete block."""
        rows = self.rows[seq][b * PAGE: (b + 1) * PAGE]
        assert len(rows) == PAGE
        out, scales = np.zeros((2, self.n_kv, PAGE, self.dim), np.float32), np.zeros((self.n_kv, 2), np.float32)
        for w in range(2):
            for h in range(self.n_kv):
                out[w, h], scales[h, w] = in_eight(rows[:, w, h])
        return out, scales

    def attend(self, seq, q, start, scale, window=0):
        """q [n, heads, D] float64 at positions start ..; (output [n, heads, D], and of every number what roundings of a query's
        probabilities are multiplied by: sum of p |v|, and the largest sum of |q k| of a score)."""
        n, heads, dim = q.shape
        length, group = start + n, heads // self.n_kv
        rows = self.rows[seq][:length].astype(np.float64)
        eight = np.zeros_like(rows)
        for b in range(length // PAGE):
            whole, scales = self.block(seq, b)
            eight[b * PAGE: (b + 1) * PAGE] = (whole.astype(np.float64) * scales.T[:, :, None, None].astype(np.float64)).transpose(2, 0, 1, 3)
        out, weight, reach = np.zeros((n, heads, dim)), np.zeros((n, heads, dim)), np.zeros((n, heads, 1))
        for t in range(n):
            p = start + t
            lo, own = max(0, p + 1 - window) if window else 0, p // PAGE * PAGE
            seen = np.concatenate([eight[lo: max(lo, own)], rows[max(lo, own): p + 1]])
            for h in range(heads):
                k, v = seen[:, 0, h // group], seen[:, 1, h // group]
                s = k @ q[t, h] * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h], weight[t, h] = w @ v, w @ np.abs(v)
                reach[t, h] = (np.abs(k) @ np.abs(q[t, h]) * scale).max()
        return out, weight, reach

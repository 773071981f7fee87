"""Answering token by token once more, with numpy's 64-bit integers and Python's: what the cache, attention, 4-bit weights and logits entry points are compared with."""
import math

import numpy as np

import valueshelp as ref

NONE = -(1 << 31)


class Softmax:
    """digits of radices bs, the lowest L dropped, the highest M zero or the weight is, the others mapped to exponentials (the tables of zkSoftmax)"""

    def __init__(self, bs=(1 << 8, 1 << 20, 1 << 20), L=1, M=0, sf_in=float(1 << 32), thetas=(float(1 << 18), float(1 << 22)), dim=1):
        self.bs, self.L, self.M, self.sf_in, self.thetas, self.dim = bs, L, M, sf_in, thetas, dim
        self.scale = sf_in * math.sqrt(dim)

    def shift(self, scores):
        """by the sum of the exponentials one after the other"""
        if len(scores) == 0:
            return 0
        total = np.cumsum(np.exp(scores.astype(np.float64) / self.scale))[-1]
        v = self.scale * math.log(total)
        return int(v + 0.5) if v >= 0 else int(v - 0.5)

    def weights(self, below):
        """of keys whose scores lie `below` the shift"""
        y, t, weight = np.ones(len(below), np.int64), np.asarray(below, np.int64).copy(), 1.0
        for i, b in enumerate(self.bs):
            digit = t % b
            t //= b
            if i >= len(self.bs) - self.M:
                y *= digit == 0
            elif i >= self.L:
                y *= np.floor(np.exp(math.log(self.thetas[i - self.L]) - weight / self.scale * digit) + 0.5).astype(np.int64)
            weight *= b
        return y


def attention(q, keys, values, softmax, sf_first, sf_second, shift=None):
    """one query's head over its keys in order: the output and the shift"""
    scores = np.asarray(keys, np.int64) @ np.asarray(q, np.int64)      # below 2^63 in every test that looks at the result
    s = softmax.shift(scores) if shift is None else shift
    y = softmax.weights(s - scores)
    # exact: the values' lowest 16 bits and the rest apart, each product's sums below 2^63
    v = np.asarray(values, np.int64).reshape(len(keys), len(q))
    sums = [(int(a) << 16) + int(b) for a, b in zip((y[:, None] * (v >> 16)).sum(0), (y[:, None] * (v & 0xFFFF)).sum(0))]
    out = [((t + sf_first // 2) // sf_first + sf_second // 2) // sf_second for t in sums]
    return np.array(out, np.int64), s


def q4_weight(codes, scales, zeros, N, P, group):
    """codes: [N][(P + 1) / 2] bytes"""
    q = np.empty((N, 2 * codes.shape[1]), np.int64)
    q[:, 0::2], q[:, 1::2] = codes & 15, codes >> 4
    at = np.arange(N) // group
    return (q[:, :P] - (8 if zeros is None else zeros.astype(np.int64)[at])) * scales.astype(np.int64)[at]


def logits(l, history, penalties, biases, mask, sf):
    """one row: history a list of tokens, biases a list of (token, value), mask a truth value a token or None"""
    out = [int(v) for v in l]
    counts = {}
    for t in history:
        counts[int(t)] = counts.get(int(t), 0) + 1
    more = {}
    for t, v in biases:
        more[int(t)] = more.get(int(t), 0) + int(v)
    for t in range(len(out)):
        if out[t] == NONE or (mask is not None and not mask[t]):
            out[t] = NONE
            continue
        if t in counts and penalties is not None:
            r, f, p = (int(v) for v in penalties)
            out[t] = int((out[t] * sf + r // 2) // r if out[t] > 0 else (out[t] * r + sf // 2) // sf) - f * counts[t] - p
        out[t] += more.get(t, 0)
    best = max(out)
    return np.array(out, np.int64), -1 if best == NONE else out.index(best)


__all__ = ["ref", "Softmax", "attention", "q4_weight", "logits", "NONE"]

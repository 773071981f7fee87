"""A decoder layer's values once more, with numpy's 64-bit integers and Python floats: what the int32 entry points are compared with."""
import numpy as np

RANGE, TABLE, POSITION = 1, 2, 4


def quotient(t, s):
    return (np.asarray(t, np.int64) + s // 2) // s


def rms_inverse(v, eps, scale):
    """row by row, the sum of squares in double precision and in index order"""
    out = []
    for row in np.asarray(v, np.int64):
        acc = 0.0
        for t in (row.astype(np.float64) / scale) ** 2:
            acc += float(t)
        out.append(np.rint(1.0 / np.sqrt(acc / row.size + eps) * scale))
    return np.array(out).astype(np.int64)


def norm(v, w, eps, scale, sf):
    v, r = np.asarray(v, np.int64), rms_inverse(v, eps, scale)
    return quotient(quotient(np.asarray(w, np.int64)[None] * r[:, None], sf) * v, sf), r


def residual_norm(x, b=None, post=None, gate=None, res=None, w=None, eps=1e-5, scale=65536.0, sf=65536):
    h = np.asarray(x, np.int64)
    if b is not None:
        q = np.asarray(b, np.int64)
        if post is not None:
            q = norm(q, post, eps, scale, sf)[0]
        if gate is not None:
            q = quotient(np.repeat(np.asarray(gate, np.int64), len(q) // len(gate), 0) * q, sf)
        h = h + quotient((sf if res is None else res) * q, sf)
    n, r = norm(h, w if w is not None else np.zeros(h.shape[1]), eps, scale, sf)
    return h, n, r


def rope(x, table, positions, rot, neighbours, sf):
    """x: [token][head][dim], table: [position][rot / 2][2]"""
    y = np.asarray(x, np.int64).copy()
    at = np.arange(rot).reshape(-1, 2).T if neighbours else np.arange(rot).reshape(2, -1)
    t = np.asarray(table, np.int64)[positions]
    c, s = t[:, None, :, 0], t[:, None, :, 1]
    x0, x1 = y[..., at[0]].copy(), y[..., at[1]].copy()
    y[..., at[0]], y[..., at[1]] = quotient(c * x0 - s * x1, sf), quotient(s * x0 + c * x1, sf)
    return y


def linear(x, w, sf):
    return quotient(np.asarray(x, np.int64) @ np.asarray(w, np.int64), sf)


def gated(x, g, u, sf_gate, sf_up, table, low, sf_hidden):
    at = linear(x, g, sf_gate) - low
    return quotient(np.asarray(table, np.int64)[at] * linear(x, u, sf_up), sf_hidden)


def elements(v):
    """integers as field elements: [..., 8] 32-bit limbs"""
    r = 0x73EDA753299D7D483339D80809A1D80553BDA402FFFE5BFEFFFFFFFF00000001
    v = np.asarray(v)
    return np.array([[(int(i) % r) >> 32 * k & 0xFFFFFFFF for k in range(8)] for i in v.reshape(-1)], np.uint32).reshape(v.shape + (8,))

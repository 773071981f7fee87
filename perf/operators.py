"""A decoder layer's values in the prover's own integers, without a witness or a proof: what the layer answers, and what the next layer is proved on.

A case is a dict with an "op" and that operator's sizes:

  norm    h = x + res * gate * norm(b), and norm(h): the residual stream with a block's output added, and the next block's input (norms before and after a block)
  rope    rotary positions of the heads of a query or key tensor, from a table of cosines and sines in fixed point
  linear  a projection with its rescaling: round(x W / 2^s)
  gated   the gated half of a feed-forward block: round(act(round(x G / 2^g)) * round(x U / 2^u) / 2^s), act a table of function values

Activations and weights are int32 in fixed point (scale 2^16), as the prover's .bin files hold them; "fr" tensors are field elements, eight 32-bit limbs each,
a negative integer v standing as r + v.  All results are whole numbers: a quotient is floor((v + s / 2) / s).
"""
import ctypes
import importlib

import numpy as np
import torch

own = False

SCALE = 65536
EPS = 1e-5
# the field's modulus r: its low 64 bits as a signed integer, and the six 32-bit limbs above them
R_LOW = 0xFFFFFFFF00000001 - (1 << 64)
R_HIGH = (0xFFFE5BFE - (1 << 32), 0x53BDA402, 0x09A1D805, 0x3339D808, 0x299D7D48, 0x73EDA753)


def listed():
    return [
        # between the blocks of one token: all of it is latency
        {"name": "norm_1x4096", "op": "norm", "rows": 1, "cols": 4096, "post": False, "gates": 0, "res": SCALE, "outliers": False},
        # a short prompt of odd sizes, every option of the operator, rows with activations a thousand times the others
        {"name": "norm_300x1000_post_gate", "op": "norm", "rows": 300, "cols": 1000, "post": True, "gates": 300, "res": 46341, "outliers": True},
        # the 7B-shape layer at 2048 tokens
        {"name": "norm_2048x4096", "op": "norm", "rows": 2048, "cols": 4096, "post": False, "gates": 0, "res": SCALE, "outliers": False},
        # one token at a far position, its queries and keys side by side
        {"name": "rope_1x64x128", "op": "rope", "tokens": 1, "heads": 64, "dim": 128, "rot": 128, "pairs": "half", "fr": False, "by_head": False, "factor": 8, "reach": 131072},
        # a prompt whose tokens have positions of their own, part of every head rotated, neighbours paired, written head by head for the attention behind it
        {"name": "rope_777x40x80_part", "op": "rope", "tokens": 777, "heads": 40, "dim": 80, "rot": 48, "pairs": "neighbours", "fr": False, "by_head": True, "factor": 1, "reach": 4096},
        # the 7B-shape layer's queries as field elements, the form that the attention's proof reads
        {"name": "rope_fr_2048x32x128", "op": "rope", "tokens": 2048, "heads": 32, "dim": 128, "rot": 128, "pairs": "half", "fr": True, "by_head": True, "factor": 1, "reach": 2048},
        # a long prompt
        {"name": "rope_16384x32x128", "op": "rope", "tokens": 16384, "heads": 32, "dim": 128, "rot": 128, "pairs": "half", "fr": False, "by_head": False, "factor": 4, "reach": 16384},
        # one token through the down projection of the 7B shape: the weights are read once
        {"name": "linear_1x11008x4096", "op": "linear", "rows": 1, "inner": 11008, "cols": 4096, "wide": False},
        # a 7B-shape projection at 2048 tokens
        {"name": "linear_2048x4096x4096", "op": "linear", "rows": 2048, "inner": 4096, "cols": 4096, "wide": False},
        # one token through both projections of the 7B shape
        {"name": "gated_1x4096x11008", "op": "gated", "rows": 1, "inner": 4096, "cols": 11008, "wide": False, "out_scale": 16},
        # a mid-sized block with no dimension a power of two, weights of more than 16 bits among them
        {"name": "gated_300x1000x2750_wide", "op": "gated", "rows": 300, "inner": 1000, "cols": 2750, "wide": True, "out_scale": 65536},
        # the 7B-shape block at 2048 tokens
        {"name": "gated_2048x4096x11008", "op": "gated", "rows": 2048, "inner": 4096, "cols": 11008, "wide": False, "out_scale": 16},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["norm", "rope", "linear", "gated"])
    if op == "norm":
        cols = size(64, 16384)
        rows = size(1, (2048 * 4096) // cols)
        return {"op": op, "rows": rows, "cols": cols, "post": rng.random() < 0.5, "gates": rng.choice([0, 1, rows]), "res": rng.choice([SCALE, rng.randrange(1, 2 * SCALE)]),
                "outliers": rng.random() < 0.5}
    if op == "rope":
        dim = 2 * size(16, 128)
        heads = size(1, 64)
        fr = rng.random() < 0.3
        tokens = size(1, (2048 if fr else 16384) * 4096 // (dim * heads))
        rot = dim if rng.random() < 0.5 else 2 * rng.randrange(1, dim // 2 + 1)
        return {"op": op, "tokens": tokens, "heads": heads, "dim": dim, "rot": rot, "pairs": rng.choice(["half", "neighbours"]), "fr": fr, "by_head": rng.random() < 0.5,
                "factor": rng.choice([1, 4, 8]), "reach": max(tokens, size(16, 131072))}
    inner, cols = size(64, 11008), size(64, 11008)
    rows = size(1, min(2048, 2048 * 4096 * 11008 // (inner * cols)))
    case = {"op": op, "rows": rows, "inner": inner, "cols": cols, "wide": rng.random() < 0.25}
    return case if op == "linear" else {**case, "out_scale": rng.choice([16, 4096, 65536])}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------
def _values(gen, shape, std, most):
    """whole numbers of a normal distribution, as int32"""
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).round_().clamp_(-most, most).to(torch.int32)


def _weights(gen, n, p, wide):
    """N(0, 0.02) at scale 2^16: 15 bits and a sign; wide: one in a thousand up to fifty times that, beyond 16 bits"""
    w = _values(gen, (n, p), 0.02 * SCALE, 32000)
    if wide:
        w = torch.where(torch.rand((n, p), device="cuda", generator=gen) < 1e-3, w * 50, w)
        w[0, 0] = 100000
    return w


def _activation(out_scale):
    """x * sigmoid(x) for x from -512 on in steps of 2^-12"""
    x = (torch.arange(1 << 22, device="cuda", dtype=torch.float64) - (1 << 21)) / 4096.0
    return torch.round(x / (1.0 + torch.exp(-x)) * out_scale).to(torch.int32)


def _angles(reach, rot, factor):
    """cosine and sine of position / factor * 10000^(-2 i / rot) at scale 2^16: [position][i][2]"""
    pos = torch.arange(reach, device="cuda", dtype=torch.float64)[:, None] / factor
    angle = pos * 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    return torch.round(torch.stack([torch.cos(angle), torch.sin(angle)], -1) * SCALE).to(torch.int32).contiguous()


def _elements(v):
    """int64 values below 2^62 as field elements: r's low 64 bits are above 2^62, so r + v borrows nothing from the limbs behind them"""
    below = (v < 0)[..., None]
    low = torch.where(below, v[..., None] + R_LOW, v[..., None]).view(torch.int32)
    return torch.cat([low, torch.where(below, torch.tensor(R_HIGH, dtype=torch.int32, device=v.device), 0)], -1)


def _integers(limbs):
    """field elements that stand for 64-bit integers, as int64"""
    low = (limbs[..., 0].to(torch.int64) & 0xFFFFFFFF) | (limbs[..., 1].to(torch.int64) << 32)
    return torch.where(limbs[..., 7] != 0, low - R_LOW, low)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case, "flag": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        s["x"] = _values(gen, (rows, cols), SCALE, 1 << 24)
        s["b"] = _values(gen, (rows, cols), 0.5 * SCALE, 1 << 24)
        if case["outliers"]:   # a row in eight has two channels with values in the hundreds
            s["x"][::8, cols // 3] = 700 * SCALE
            s["x"][::8, cols // 2] = -300 * SCALE
        s["w"] = _values(gen, (cols,), 0.1 * SCALE, 1 << 20) + SCALE
        s["post"] = _values(gen, (cols,), 0.1 * SCALE, 1 << 20) + SCALE if case["post"] else None
        s["gate"] = _values(gen, (case["gates"], cols), 0.5 * SCALE, 1 << 20) if case["gates"] else None
        s["h"], s["n"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
        s["rms_inv"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    elif case["op"] == "rope":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        x = _values(gen, (tokens, heads, dim), SCALE, 1 << 24)
        s["x"] = _elements(x.to(torch.int64)) if case["fr"] else x
        s["table"] = _angles(case["reach"], case["rot"], case["factor"])
        if tokens == 1:
            s["positions"] = torch.full((1,), case["reach"] - 1, dtype=torch.int32, device="cuda")
        else:   # sequences one after the other, each from a place of its own
            at = torch.randint(0, case["reach"], (tokens,), generator=gen, device="cuda")
            start = torch.where(torch.arange(tokens, device="cuda") % 100 == 0, at, torch.zeros_like(at)).cummax(0).values
            s["positions"] = ((start + torch.arange(tokens, device="cuda")) % case["reach"]).to(torch.int32)
        shape = (heads, tokens, dim) if case["by_head"] else (tokens, heads, dim)
        s["out"] = torch.empty(shape + ((8,) if case["fr"] else ()), dtype=torch.int32, device="cuda")
    else:
        rows, inner, cols = case["rows"], case["inner"], case["cols"]
        s["x"] = _values(gen, (rows, inner), SCALE, 1 << 20)
        w = [_weights(gen, inner, cols, case["wide"]) for _ in range(2 if case["op"] == "gated" else 1)]
        if case["op"] == "gated":
            s["table"] = _activation(case["out_scale"])
        s["out"] = torch.empty((rows, cols), dtype=torch.int32, device="cuda")
        # a program keeps its weights the way its products read them
        s["w"] = [_Rhs(t) for t in w] if own else [t.to(torch.float64) for t in w]
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------
def _round(v, bits):
    return (v + (1 << bits >> 1)) >> bits


def _plain_norm(v, w):
    mean = (v * v).sum(-1).to(torch.float64) / SCALE / SCALE / v.shape[-1]
    rms_inv = torch.round(1.0 / torch.sqrt(mean + EPS) * SCALE).to(torch.int64)
    return _round(_round(w * rms_inv[:, None], 16) * v, 16), rms_inv


def _plain_product(x, w):
    return torch.matmul(x.to(torch.float64), w).to(torch.int64)   # whole numbers below 2^53 throughout


def _plain(s):
    case = s["case"]
    if case["op"] == "norm":
        x, b, w = (s[k].to(torch.int64) for k in ("x", "b", "w"))
        if s["post"] is not None:
            b = _plain_norm(b, s["post"].to(torch.int64))[0]
        if s["gate"] is not None:
            b = _round(s["gate"].to(torch.int64) * b, 16)
        h = x + _round(case["res"] * b, 16)
        n, rms_inv = _plain_norm(h, w)
        return {"h": h.to(torch.int32), "n": n.to(torch.int32), "rms_inv": rms_inv.to(torch.int32)}
    if case["op"] == "rope":
        x = _integers(s["x"]) if case["fr"] else s["x"].to(torch.int64)
        rot, half = case["rot"], case["rot"] // 2
        angle = s["table"][s["positions"].long()].to(torch.int64)[:, None]
        c, sn = angle[..., 0], angle[..., 1]
        x0, x1 = (x[..., :half], x[..., half:rot]) if case["pairs"] == "half" else (x[..., 0:rot:2], x[..., 1:rot:2])
        y0, y1 = _round(c * x0 - sn * x1, 16), _round(sn * x0 + c * x1, 16)
        y = torch.cat([y0, y1], -1) if case["pairs"] == "half" else torch.stack([y0, y1], -1).flatten(-2)
        y = torch.cat([y, x[..., rot:]], -1)
        if case["by_head"]:
            y = y.transpose(0, 1).contiguous()
        return _elements(y) if case["fr"] else y.to(torch.int32)
    if case["op"] == "linear":
        return _round(_plain_product(s["x"], s["w"][0]), 16).to(torch.int32)
    gate, up = _round(_plain_product(s["x"], s["w"][0]), 20), _round(_plain_product(s["x"], s["w"][1]), 16)
    return _round(s["table"][gate + (1 << 21)].to(torch.int64) * up, 16).to(torch.int32)


# ---- the framework's calls -------------------------------------------------------------------------------------------------------------------
_hip = None


def _lib():
    global _hip
    if _hip is None:
        _hip = importlib.import_module("zkllm-ccs2024_amd").load_hip()
        _hip.zk_i32_linear_workspace.restype = ctypes.c_size_t
        _ok(_hip.zk_init(ctypes.c_int(torch.cuda.current_device())))
    return _hip


def _ok(rc):
    if rc != 0:
        raise RuntimeError(_hip.zk_last_error().decode())


def _p(t):
    return ctypes.c_void_p(None if t is None else t.data_ptr())


def _n(v):
    return ctypes.c_size_t(v)


def _u(v):
    return ctypes.c_uint32(v)


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class _Rhs:
    """a weight laid out for products, and what it was made from gone"""

    def __init__(self, w):
        self.h = ctypes.c_void_p()
        _ok(_lib().zk_i32_rhs_prepare(ctypes.byref(self.h), _p(w), _u(w.shape[0]), _u(w.shape[1]), _stream()))
        torch.cuda.synchronize()

    def __del__(self):
        _hip.zk_fr_matmul_rhs_free(self.h)


def _workspace(s):
    if "workspace" not in s:
        s["workspace"] = torch.empty(_lib().zk_i32_linear_workspace(_u(s["case"]["rows"]), _u(s["case"]["inner"])), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _framework(s):
    case, lib = s["case"], _lib()
    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        _ok(lib.zk_i32_residual_norm(_p(s["h"]), _p(s["n"]), _p(s["rms_inv"]), _p(s["x"]), _n(cols), _p(s["b"]), _n(cols), _p(s["post"]), _p(s["gate"]), _u(case["gates"]),
                                     ctypes.c_int32(case["res"]), _p(s["w"]), _u(rows), _u(cols), ctypes.c_double(EPS), ctypes.c_double(SCALE), _u(SCALE), _p(s["flag"]), _stream()))
        return {"h": s["h"], "n": s["n"], "rms_inv": s["rms_inv"]}
    if case["op"] == "rope":
        tokens, heads, dim = case["tokens"], case["heads"], case["dim"]
        by_token, by_head = (dim, tokens * dim) if case["by_head"] else (heads * dim, dim)
        call = lib.zk_fr_rope if case["fr"] else lib.zk_i32_rope
        _ok(call(_p(s["out"]), _n(by_token), _n(by_head), _p(s["x"]), _n(heads * dim), _n(dim), _u(tokens), _u(heads), _u(dim), _u(case["rot"]),
                 ctypes.c_int(case["pairs"] == "neighbours"), _p(s["table"]), _u(case["reach"]), _p(s["positions"]), _u(0), _u(SCALE), _p(s["flag"]), _stream()))
        return s["out"]
    rows, inner, ws = case["rows"], case["inner"], _workspace(s)
    if case["op"] == "linear":
        _ok(lib.zk_i32_linear(_p(s["out"]), _p(s["x"]), _n(inner), s["w"][0].h, _u(rows), _u(SCALE), _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
        return s["out"]
    _ok(lib.zk_i32_gated(_p(s["out"]), _p(s["x"]), _n(inner), s["w"][0].h, s["w"][1].h, _u(rows), _u(1 << 20), _u(SCALE), _p(s["table"]), ctypes.c_int32(-(1 << 21)),
                         _u(1 << 22), _u(SCALE), _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
    return s["out"]


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        gates = case["gates"] * case["cols"]
        return {"bytes": 4 * (4 * n + gates + 2 * case["cols"]), "flops": n * (20 if case["post"] else 12)}
    if case["op"] == "rope":
        n = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * n * (32 if case["fr"] else 4) + min(case["tokens"], case["reach"]) * case["rot"] * 4 + 4 * case["tokens"], "flops": 4 * n}
    matrices = 2 if case["op"] == "gated" else 1
    products = matrices * case["rows"] * case["inner"] * case["cols"]
    return {"bytes": 4 * case["rows"] * (case["inner"] + case["cols"]) + matrices * (3 if case["wide"] else 2) * case["inner"] * case["cols"], "flops": 2 * products}


# ---- the definitions once more, with numpy on the host -------------------------------------------------------------------------------------------
def _quotient(v, s):
    return (v + s // 2) // s


def _host_norm(v, w):
    squares = (v * v).sum(axis=1)
    rms_inv = np.rint(np.longdouble(SCALE) / np.sqrt(squares.astype(np.longdouble) / (np.longdouble(SCALE) ** 2 * v.shape[1]) + np.longdouble(EPS))).astype(np.int64)
    return _quotient(_quotient(w[None, :] * rms_inv[:, None], SCALE) * v, SCALE), rms_inv


def _host_product(x, w):
    """exact: x in two pieces of 11 bits and the rest, each product's sums below 2^53"""
    low = x & 2047
    return (low.astype(np.float64) @ w).astype(np.int64) + ((x >> 11).astype(np.float64) @ w).astype(np.int64) * 2048


def exact(case, seed):
    if case["op"] in ("linear", "gated") and case["rows"] * case["inner"] * case["cols"] > 10 ** 10:
        return None
    if case["op"] == "rope" and case["tokens"] * case["heads"] * case["dim"] > 10 ** 7:
        return None
    global own
    was, own = own, False   # inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = was
    a = {k: v.cpu().numpy().astype(np.int64) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "norm":
        b = a["b"]
        if case["post"]:
            b = _host_norm(b, a["post"])[0]
        if case["gates"]:
            b = _quotient(a["gate"] * b, SCALE)
        h = a["x"] + _quotient(case["res"] * b, SCALE)
        n, rms_inv = _host_norm(h, a["w"])
        return {"h": h.astype(np.int32), "n": n.astype(np.int32), "rms_inv": rms_inv.astype(np.int32)}
    if case["op"] == "rope":
        x = a["x"]
        if case["fr"]:
            x = (x[..., 0] & 0xFFFFFFFF) + (x[..., 1] << 32) + np.where(x[..., 7] != 0, (1 << 32) - 1, 0)
        rot = case["rot"]
        at = np.arange(rot).reshape(2, -1) if case["pairs"] == "half" else np.arange(rot).reshape(-1, 2).T
        t = a["table"][a["positions"]]
        y = x.copy()
        for j, (i0, i1) in enumerate(at.T):
            c, sn = t[:, None, j, 0], t[:, None, j, 1]
            y[..., i0], y[..., i1] = _quotient(c * x[..., i0] - sn * x[..., i1], SCALE), _quotient(sn * x[..., i0] + c * x[..., i1], SCALE)
        if case["by_head"]:
            y = np.ascontiguousarray(y.swapaxes(0, 1))
        if not case["fr"]:
            return y.astype(np.int32)
        r = 0x73EDA753299D7D483339D80809A1D80553BDA402FFFE5BFEFFFFFFFF00000001
        out = np.zeros(y.shape + (8,), np.int64)
        carry = np.zeros(y.shape, np.int64)
        for k in range(8):   # y + r where y is negative, limb by limb
            t = (y & 0xFFFFFFFF if k == 0 else y >> 32 if k == 1 else 0) + np.where(y < 0, r >> 32 * k & 0xFFFFFFFF, 0) + carry
            out[..., k], carry = t & 0xFFFFFFFF, t >> 32
        return out.astype(np.uint32).view(np.int32)
    w = [t.cpu().numpy() for t in s["w"]]
    if case["op"] == "linear":
        return _quotient(_host_product(a["x"], w[0]), SCALE).astype(np.int32)
    gate, up = _quotient(_host_product(a["x"], w[0]), 1 << 20), _quotient(_host_product(a["x"], w[1]), SCALE)
    return _quotient(a["table"][gate + (1 << 21)] * up, SCALE).astype(np.int32)

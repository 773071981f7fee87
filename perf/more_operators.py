"""Answering token by token in the prover's own integers: what a program that generates text with a model calls between the layers' other products, for many requests at once
that begin with the same text.

A case is a dict with an "op" and that operator's sizes:

  append     the keys and values of new tokens written into the pages of their sequences
  attention  queries over keys and values, those of a prefix that all sequences share and those of a sequence's own pages, by the softmax that the layer's proof is made of
  linear     a projection whose weight is kept in 4 bits with a scale (and a zero) for every group of rows: round(x W / 2^s), W = (code - zero) * scale
  gated      the gated half of a feed-forward block with two such weights
  logits     a row's logits after penalties for repeated tokens, biases and the mask of a grammar, and the best token that is left

Activations are int32 in fixed point (scale 2^16), as the prover's .bin files hold them.  All results are whole numbers: a quotient is floor((v + s / 2) / s).
"""
import ctypes
import importlib
import math

import numpy as np
import torch

own = False

SCALE = 65536
# the softmax of the layer's proof: digits of 8, 20 and 20 bits, the lowest dropped, the others mapped to exponentials of scale 2^18 and 2^22
RADICES, DROPPED, THETAS, SCORE_SCALE = (1 << 8, 1 << 20, 1 << 20), 1, (float(1 << 18), float(1 << 22)), float(1 << 32)
ATTN_SCALE = 1 << 20
NONE = -(1 << 31)      # a token that cannot be chosen


def listed():
    return [
        # one token of one request
        {"name": "append_1x8x128", "op": "append", "seqs": 1, "tokens": 1, "kv_heads": 8, "dim": 128, "own": 512, "page": 64},
        # prompts of 32 requests that came in together, heads and pages of odd sizes
        {"name": "append_32x100x5x80", "op": "append", "seqs": 32, "tokens": 100, "kv_heads": 5, "dim": 80, "own": 300, "page": 17},
        # one token of one request early in its answer: all of it is latency
        {"name": "attn_1x32x128_own200", "op": "attention", "seqs": 1, "tokens": 1, "heads": 32, "kv_heads": 32, "dim": 128, "prefix": 0, "own": 200, "page": 64, "causal": True},
        # one token of one request behind a long text
        {"name": "attn_1x32x128_own16000", "op": "attention", "seqs": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 0, "own": 16000, "page": 64, "causal": True},
        # 32 requests, each at its own place of its answer behind one long common instruction
        {"name": "attn_32x32x128_pre8192", "op": "attention", "seqs": 32, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 8192, "own": 512, "page": 64, "causal": True},
        # a few tokens of some requests at a time, heads and pages of odd sizes, a prefix that no tile divides
        {"name": "attn_7x5x6x80_odd", "op": "attention", "seqs": 7, "tokens": 5, "heads": 6, "kv_heads": 2, "dim": 80, "prefix": 333, "own": 150, "page": 17, "causal": True},
        # the 7B-shape layer at 2048 tokens, every token over all of them as the layer's proof has it
        {"name": "attn_prompt_2048x32x128", "op": "attention", "seqs": 1, "tokens": 2048, "heads": 32, "kv_heads": 32, "dim": 128, "prefix": 0, "own": 2048, "page": 2048, "causal": False},
        # one token through the down projection of the 7B shape: the weights are read once
        {"name": "linear4_1x11008x4096", "op": "linear", "rows": 1, "inner": 11008, "cols": 4096, "group": 128, "zeros": False, "wide": False},
        # a batch through both projections of the 7B shape
        {"name": "gated4_32x4096x11008", "op": "gated", "rows": 32, "inner": 4096, "cols": 11008, "group": 128, "zeros": True, "wide": False, "out_scale": 16},
        # a prompt through a block with no dimension a power of two, small groups, weights of more than 16 bits
        {"name": "gated4_300x1000x2750_wide", "op": "gated", "rows": 300, "inner": 1000, "cols": 2750, "group": 32, "zeros": True, "wide": True, "out_scale": 65536},
        # one request's next token
        {"name": "logits_1x32000", "op": "logits", "rows": 1, "vocab": 32000, "history": 200, "biases": 0, "masked": False},
        # many requests, long answers behind them, a large vocabulary whose rows begin anywhere
        {"name": "logits_64x128257", "op": "logits", "rows": 64, "vocab": 128257, "history": 8000, "biases": 300, "masked": True},
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))

    op = rng.choice(["append", "attention", "attention", "linear", "gated", "logits"])
    if op == "append":
        seqs, tokens = size(1, 64), size(1, 128)
        return {"op": op, "seqs": seqs, "tokens": tokens, "kv_heads": size(1, 8), "dim": size(16, 128), "own": tokens + size(1, 256), "page": size(8, 256)}
    if op == "attention":
        kv_heads = size(1, 32)
        heads = kv_heads * rng.choice([1, 2, 4, 8] if kv_heads <= 8 else [1])
        dim = size(16, 128)
        tokens, seqs = rng.choice([(1, 1), (1, size(1, 64)), (size(1, 16), size(1, 16)), (size(64, 2048), 1)])
        tokens = min(tokens, math.isqrt(2048 * 2048 * 32 * 128 // (heads * dim)))
        most = max(tokens, min(16000, 2048 * 32 * 2048 * 128 // (tokens * seqs * heads * dim)))
        prefix = 0 if rng.random() < 0.3 else min(size(16, 8192), most // 2)
        return {"op": op, "seqs": seqs, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim, "prefix": prefix,
                "own": max(tokens, min(size(tokens, 16000 if seqs == 1 else 2048), most - prefix)), "page": size(8, 1024), "causal": rng.random() < 0.7}
    if op == "logits":
        vocab = size(1000, 160000)
        rows = size(1, min(256, 64 * 128257 // vocab))
        return {"op": op, "rows": rows, "vocab": vocab, "history": size(1, 8000), "biases": rng.choice([0, size(1, 1000)]), "masked": rng.random() < 0.5}
    inner, cols = size(64, 11008), size(64, 11008)
    case = {"op": op, "rows": size(1, min(300, 32 * 4096 * 11008 // (inner * cols))), "inner": inner, "cols": cols, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
            "wide": rng.random() < 0.25}
    return case if op == "linear" else {**case, "out_scale": rng.choice([16, 4096, 65536])}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------
def _values(gen, shape, std, most):
    """whole numbers of a normal distribution, as int32"""
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).round_().clamp_(-most, most).to(torch.int32)


def _below(gen, n, shape):
    return torch.randint(0, n, shape, generator=gen, device="cuda", dtype=torch.int32)


def _pages(gen, case):
    """a pool of pages in no order, and each sequence's list of them"""
    each = -(-case["own"] // case["page"])
    pages = case["seqs"] * each
    table = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).reshape(case["seqs"], each).contiguous()
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    return _values(gen, shape, SCALE, 1 << 20), _values(gen, shape, SCALE, 1 << 20), table


def _lengths(gen, case):
    """tokens that a sequence has in its pages, the new ones among them: any number, for one sequence the most"""
    if case["seqs"] == 1:
        return torch.full((1,), case["own"], dtype=torch.int32, device="cuda")
    return (case["tokens"] + _below(gen, case["own"] - case["tokens"] + 1, (case["seqs"],))).to(torch.int32)


def _activation(out_scale):
    """x * sigmoid(x) for x from -512 on in steps of 2^-12"""
    x = (torch.arange(1 << 22, device="cuda", dtype=torch.float64) - (1 << 21)) / 4096.0
    return torch.round(x / (1.0 + torch.exp(-x)) * out_scale).to(torch.int32)


def _exponentials(dim):
    """the tables of the digits that are kept: round(theta exp(-digit * weight / (scale sqrt(dim))))"""
    out, weight = [], RADICES[0]
    for radix, theta in zip(RADICES[DROPPED:], THETAS):
        digit = torch.arange(radix, device="cuda", dtype=torch.float64)
        out.append(torch.floor(torch.exp(math.log(theta) - weight / (SCORE_SCALE * math.sqrt(dim)) * digit) + 0.5).to(torch.int64))
        weight *= radix
    return out


class _Weight:
    """4-bit codes, two neighbouring columns a byte, with a scale and a zero for every `group` rows of a column"""

    def __init__(self, gen, case):
        n, p, g = case["inner"], case["cols"], case["group"]
        groups = -(-n // g)
        codes = torch.empty((n, p + p % 2), device="cuda").normal_(8.0, 2.7, generator=gen).round_().clamp_(0, 15).to(torch.uint8)
        self.codes = (codes[:, 0::2] | codes[:, 1::2] << 4).contiguous()
        self.scales = 300 + _below(gen, 500, (groups, p))
        if case["wide"]:      # a group in a hundred has weights fifty times as large
            self.scales = torch.where(torch.rand((groups, p), device="cuda", generator=gen) < 0.01, self.scales * 50, self.scales)
            self.scales[0, 0] = 40000
        self.scales = self.scales.to(torch.int32).contiguous()
        self.zeros = _below(gen, 16, (groups, p)).to(torch.uint8).contiguous() if case["zeros"] else None
        self.case = case

    def values(self):
        n, p, g = self.case["inner"], self.case["cols"], self.case["group"]
        code = torch.stack([self.codes & 15, self.codes >> 4], -1).reshape(n, -1)[:, :p].to(torch.float64)
        at = torch.arange(n, device="cuda") // g
        return (code - (8.0 if self.zeros is None else self.zeros.to(torch.float64)[at])) * self.scales.to(torch.float64)[at]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    s = {"case": case, "flag": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["op"] in ("append", "attention"):
        s["k_pages"], s["v_pages"], s["table"] = _pages(gen, case)
        s["lengths"] = _lengths(gen, case)
        n = case["seqs"] * case["tokens"]
        s["starts"] = (torch.arange(case["seqs"] + 1, device="cuda") * case["tokens"]).to(torch.int32)
    if case["op"] == "append":
        # keys and values side by side, as one projection leaves them
        s["kv"] = _values(gen, (n, 2, case["kv_heads"], case["dim"]), SCALE, 1 << 20)
    elif case["op"] == "attention":
        s["q"] = _values(gen, (n, case["heads"], case["dim"]), SCALE, 1 << 20)
        s["prefix"] = [_values(gen, (case["prefix"], case["kv_heads"], case["dim"]), SCALE, 1 << 20) for _ in range(2)]
        s["out"] = torch.empty_like(s["q"])
        s["softmax"] = _Softmax(case["dim"]) if own else _exponentials(case["dim"])
    elif case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        s["logits"] = _values(gen, (rows, vocab), 3 * SCALE, 1 << 24)
        counts = [case["history"] * (1 + r % 4) // 4 for r in range(rows)]      # ragged
        s["history_starts"] = torch.tensor([0] + counts, device="cuda").cumsum(0).to(torch.int32)
        # few tokens make up most of a text
        s["history"] = (torch.rand(sum(counts), device="cuda", generator=gen) ** 4 * vocab).to(torch.int32).clamp_(max=vocab - 1)
        s["penalties"] = torch.tensor([[SCALE + r % 5 * 6554, r % 3 * 3277, r % 2 * 13107] for r in range(rows)], dtype=torch.int32, device="cuda")   # repeated 1.0 .. 1.4, by count, once
        s["bias_starts"] = (torch.arange(rows + 1, device="cuda") * case["biases"]).to(torch.int32)
        s["bias_tokens"] = _below(gen, vocab, (rows * case["biases"],))
        s["bias_values"] = _values(gen, (rows * case["biases"],), 2 * SCALE, 1 << 22)
        s["mask"] = None
        if case["masked"]:      # a grammar allows a few tokens in a hundred; here and there it allows all, or nothing
            part = torch.tensor([0.03, 1.0, 0.3, 0.003, 0.03, 0.03, 0.0, 0.1], device="cuda")[torch.arange(rows, device="cuda") % 8]
            allowed = torch.rand((rows, -(-vocab // 32) * 32), device="cuda", generator=gen) < part[:, None]
            bits = torch.ones(32, dtype=torch.int64, device="cuda") << torch.arange(32, device="cuda")
            s["mask"] = (allowed.reshape(rows, -1, 32).to(torch.int64) * bits).sum(-1).to(torch.int32).contiguous()
        s["out"] = torch.empty_like(s["logits"])
        s["token"] = torch.empty(rows, dtype=torch.int32, device="cuda")
    else:
        s["x"] = _values(gen, (case["rows"], case["inner"]), SCALE, 1 << 20)
        s["w"] = [_Weight(gen, case) for _ in range(2 if case["op"] == "gated" else 1)]
        if case["op"] == "gated":
            s["act"] = _activation(case["out_scale"])
        s["out"] = torch.empty((case["rows"], case["cols"]), dtype=torch.int32, device="cuda")
        if own:      # a program keeps its weights the way its products read them
            s["w"] = [_Rhs(w) for w in s["w"]]
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------------------------------
def _quotient(v, s):
    return torch.div(v + s // 2, s, rounding_mode="floor")


def _plain_append(s):
    case = s["case"]
    n = torch.arange(case["tokens"], device="cuda")
    at = (s["lengths"].long() - case["tokens"])[:, None] + n[None]      # each new token's place in its sequence
    page = torch.gather(s["table"].long(), 1, at // case["page"])
    new = s["kv"].reshape(case["seqs"], case["tokens"], 2, case["kv_heads"], case["dim"])
    s["k_pages"][page, at % case["page"]] = new[:, :, 0]
    s["v_pages"][page, at % case["page"]] = new[:, :, 1]
    return {"k": s["k_pages"], "v": s["v_pages"]}


def _plain_heads(case, tables, q, k, v, hidden):
    """q: [head][row][dim], k and v: [head][key][dim], hidden: [row][key] or none, all exact in 64-bit floating point"""
    scores = torch.bmm(q, k.transpose(1, 2).contiguous())      # whole numbers below 2^53
    scale = SCORE_SCALE * math.sqrt(case["dim"])
    terms = torch.exp(scores / scale)
    if hidden is not None:
        terms = terms.masked_fill(hidden, 0.0)
    shift = torch.round(torch.log(terms.sum(-1, keepdim=True)) * scale)
    del terms
    digits = (shift - scores).to(torch.int64)
    del scores
    y, digits = None, digits // RADICES[0]
    for radix, table in zip(RADICES[DROPPED:], tables):
        mapped = table[(digits % radix).clamp_(min=0)]
        y = mapped if y is None else y * mapped
        digits = digits // radix
    if hidden is not None:
        y = y.masked_fill(hidden, 0)
    # sums of products up to 2^60: the weights' upper and lower 20 bits apart
    upper, lower = torch.bmm((y >> 20).to(torch.float64), v), torch.bmm((y & 0xFFFFF).to(torch.float64), v)
    return upper.to(torch.int64) * (1 << 20) + lower.to(torch.int64)


def _plain_attention(s):
    case = s["case"]
    heads, kv_heads, dim, n, prefix = (case[k] for k in ("heads", "kv_heads", "dim", "tokens", "prefix"))
    group = heads // kv_heads
    out = torch.empty((case["seqs"], n, heads, dim), dtype=torch.int32, device="cuda")
    q = s["q"].reshape(case["seqs"], n, kv_heads, group, dim).permute(0, 2, 1, 3, 4).reshape(case["seqs"], kv_heads, n * group, dim).to(torch.float64)
    at = torch.arange(case["own"], device="cuda")
    for i in range(case["seqs"]):      # a sequence's keys: the prefix's, then its own, out of its pages
        # (positions behind its last are hidden: how many there are is known on the device alone)
        page = s["table"][i].long()[at // case["page"]]
        k, v = (torch.cat([p, own_[page, at % case["page"]]]).transpose(0, 1).to(torch.float64) for p, own_ in zip(s["prefix"], (s["k_pages"], s["v_pages"])))
        last = s["lengths"][i].long() - (n - 1 - torch.arange(n, device="cuda") if case["causal"] else torch.zeros(n, dtype=torch.int64, device="cuda"))
        hidden = None
        if case["causal"] or case["seqs"] > 1:
            hidden = torch.cat([torch.zeros((n, prefix), dtype=torch.bool, device="cuda"), at[None] >= last[:, None]], 1).repeat_interleave(group, 0)
        sums = _plain_heads(case, s["softmax"], q[i], k.contiguous(), v.contiguous(), hidden)
        values = _quotient(_quotient(sums, ATTN_SCALE), ATTN_SCALE)
        out[i] = values.reshape(kv_heads, n, group, dim).permute(1, 0, 2, 3).reshape(n, heads, dim).to(torch.int32)
    return out.reshape(-1, heads, dim)


def _plain_product(x, w):
    return torch.matmul(x.to(torch.float64), w).to(torch.int64)   # whole numbers below 2^53 throughout


def _plain_logits(s):
    case = s["case"]
    rows, vocab = case["rows"], case["vocab"]
    l = s["logits"].to(torch.int64)

    def by_token(starts, tokens, values):      # what a row's list holds, added up by token
        row = torch.searchsorted(starts[1:].long().contiguous(), torch.arange(tokens.numel(), device="cuda"), right=True)
        return torch.zeros(rows * vocab, dtype=torch.int64, device="cuda").index_add_(0, row * vocab + tokens.long(), values).reshape(rows, vocab)

    count = by_token(s["history_starts"], s["history"], torch.ones_like(s["history"], dtype=torch.int64))
    repeat, frequency, presence = (s["penalties"][:, i:i + 1].to(torch.int64) for i in range(3))
    repeated = torch.where(l > 0, torch.div(l * SCALE + repeat // 2, repeat, rounding_mode="floor"), _quotient(l * repeat, SCALE))
    l = torch.where(count > 0, repeated - frequency * count - presence, l)
    if case["biases"]:
        l = l + by_token(s["bias_starts"], s["bias_tokens"], s["bias_values"].to(torch.int64))
    if s["mask"] is not None:
        token = torch.arange(vocab, device="cuda")
        l = torch.where((s["mask"][:, token // 32] >> (token % 32).to(torch.int32) & 1) == 1, l, NONE)
    best = l.max(-1, keepdim=True).values
    first = torch.where(l == best, torch.arange(vocab, device="cuda"), vocab).min(-1).values      # the lowest of equals
    return {"logits": l.to(torch.int32), "token": torch.where(best[:, 0] == NONE, -1, first).to(torch.int32)}


def _plain(s):
    case = s["case"]
    if case["op"] == "append":
        return _plain_append(s)
    if case["op"] == "attention":
        return _plain_attention(s)
    if case["op"] == "logits":
        return _plain_logits(s)
    if case["op"] == "linear":
        return _quotient(_plain_product(s["x"], s["w"][0].values()), SCALE).to(torch.int32)
    gate, up = _quotient(_plain_product(s["x"], s["w"][0].values()), 1 << 20), _quotient(_plain_product(s["x"], s["w"][1].values()), SCALE)
    return _quotient(s["act"][gate + (1 << 21)].to(torch.int64) * up, SCALE).to(torch.int32)


# ---- the framework's calls -------------------------------------------------------------------------------------------------------------------
_hip = None


def _lib():
    global _hip
    if _hip is None:
        _hip = importlib.import_module("zkllm-ccs2024_amd").load_hip()
        for f in ("zk_i32_attention_workspace", "zk_i32_rhs_workspace", "zk_i32_logits_workspace"):
            getattr(_hip, f).restype = ctypes.c_size_t
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


class _Cache(ctypes.Structure):      # zk_i32_cache
    _fields_ = [("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("page_stride", ctypes.c_size_t), ("token_stride", ctypes.c_size_t), ("head_stride", ctypes.c_size_t),
                ("page_size", ctypes.c_uint32), ("pages", ctypes.c_uint32), ("page_table", ctypes.c_void_p), ("table_cols", ctypes.c_uint32)]


def _own_cache(s):
    case = s["case"]
    token = case["kv_heads"] * case["dim"]
    return _Cache(s["k_pages"].data_ptr(), s["v_pages"].data_ptr(), case["page"] * token, token, case["dim"], case["page"], s["k_pages"].shape[0], s["table"].data_ptr(), s["table"].shape[1])


def _prefix_cache(s):
    case = s["case"]
    token = case["kv_heads"] * case["dim"]
    return _Cache(s["prefix"][0].data_ptr(), s["prefix"][1].data_ptr(), case["prefix"] * token, token, case["dim"], case["prefix"], 1, None, 0)


class _Softmax:
    def __init__(self, dim):
        self.h = ctypes.c_void_p()
        _ok(_lib().zk_i32_softmax_prepare(ctypes.byref(self.h), (ctypes.c_uint32 * len(RADICES))(*RADICES), ctypes.c_int(len(RADICES)), ctypes.c_int(DROPPED), ctypes.c_int(0),
                                          ctypes.c_double(SCORE_SCALE), (ctypes.c_double * len(THETAS))(*THETAS), _u(dim), _stream()))

    def __del__(self):
        _hip.zk_i32_softmax_free(self.h)


class _Rhs:
    """a weight laid out for products, and what it was made from gone"""

    def __init__(self, w):
        self.h = ctypes.c_void_p()
        _ok(_lib().zk_i32_rhs_prepare_q4(ctypes.byref(self.h), _p(w.codes), _p(w.scales), _p(w.zeros), _u(w.case["inner"]), _u(w.case["cols"]), _u(w.case["group"]), _stream()))
        torch.cuda.synchronize()

    def __del__(self):
        _hip.zk_fr_matmul_rhs_free(self.h)


def _workspace(s):
    if "workspace" not in s:
        case, lib = s["case"], _lib()
        if case["op"] == "attention":
            size = lib.zk_i32_attention_workspace(*(_u(v) for v in (case["seqs"] * case["tokens"], case["heads"], case["kv_heads"], case["dim"], case["prefix"], case["seqs"], case["own"])))
        elif case["op"] == "logits":
            size = lib.zk_i32_logits_workspace(_u(case["rows"]), _u(case["vocab"]))
        else:
            size = sum(lib.zk_i32_rhs_workspace(w.h, _u(case["rows"])) for w in s["w"])
        s["workspace"] = torch.empty(max(size, 16), dtype=torch.uint8, device="cuda")
    return s["workspace"]


def _framework(s):
    case, lib = s["case"], _lib()
    if case["op"] == "append":
        token = case["kv_heads"] * case["dim"]
        cache = _own_cache(s)
        _ok(lib.zk_i32_cache_append(ctypes.byref(cache), _p(s["kv"]), _n(2 * token), _n(case["dim"]), _p(s["kv"][:, 1]), _n(2 * token), _n(case["dim"]), _u(len(s["kv"])),
                                    _u(case["kv_heads"]), _u(case["dim"]), _u(case["seqs"]), _p(s["starts"]), _p(s["lengths"]), _p(s["flag"]), _stream()))
        return {"k": s["k_pages"], "v": s["v_pages"]}
    ws = _workspace(s)
    if case["op"] == "attention":
        token = case["heads"] * case["dim"]
        cache, prefix = _own_cache(s), _prefix_cache(s)
        _ok(lib.zk_i32_attention(_p(s["out"]), _n(token), _n(case["dim"]), _p(s["q"]), _n(token), _n(case["dim"]), _u(len(s["q"])), _u(case["heads"]), _u(case["kv_heads"]), _u(case["dim"]),
                                 s["softmax"].h, ctypes.byref(prefix) if case["prefix"] else None, _u(case["prefix"]), ctypes.byref(cache), _u(case["seqs"]), _p(s["starts"]), _p(s["lengths"]),
                                 _u(case["own"]), ctypes.c_int(case["causal"]), _u(ATTN_SCALE), _u(ATTN_SCALE), None, _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
        return s["out"]
    if case["op"] == "logits":
        rows, vocab = case["rows"], case["vocab"]
        some = case["biases"] > 0
        _ok(lib.zk_i32_logits(_p(s["out"]), _n(vocab), _p(s["token"]), _p(s["logits"]), _n(vocab), _u(rows), _u(vocab), _p(s["history"]), _u(s["history"].numel()), _p(s["history_starts"]),
                              _p(s["penalties"]), _p(s["bias_tokens"] if some else None), _p(s["bias_values"] if some else None), _u(s["bias_tokens"].numel()),
                              _p(s["bias_starts"] if some else None), _p(s["mask"]), _n(0 if s["mask"] is None else s["mask"].shape[1]), _u(0 if s["mask"] is None else rows), _u(SCALE),
                              _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
        return {"logits": s["out"], "token": s["token"]}
    rows, inner = case["rows"], case["inner"]
    if case["op"] == "linear":
        _ok(lib.zk_i32_linear(_p(s["out"]), _p(s["x"]), _n(inner), s["w"][0].h, _u(rows), _u(SCALE), _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
        return s["out"]
    _ok(lib.zk_i32_gated(_p(s["out"]), _p(s["x"]), _n(inner), s["w"][0].h, s["w"][1].h, _u(rows), _u(1 << 20), _u(SCALE), _p(s["act"]), ctypes.c_int32(-(1 << 21)),
                         _u(1 << 22), _u(SCALE), _p(ws), _n(ws.numel()), _p(s["flag"]), _stream()))
    return s["out"]


def run(state):
    return _framework(state) if own else _plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "append":
        n = case["seqs"] * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": 4 * 4 * n, "flops": n}
    if case["op"] == "attention":
        tokens = case["seqs"] * case["tokens"]
        each = case["own"] if case["seqs"] == 1 else (case["tokens"] + case["own"]) // 2      # of ragged lengths the mean
        seen = case["prefix"] + each - (case["tokens"] // 2 if case["causal"] else 0)
        keys = case["prefix"] + case["seqs"] * each
        return {"bytes": 4 * (2 * tokens * case["heads"] * case["dim"] + 2 * keys * case["kv_heads"] * case["dim"]), "flops": 4 * tokens * case["heads"] * case["dim"] * seen}
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        return {"bytes": 8 * n + (n // 8 if case["masked"] else 0) + case["rows"] * (4 * case["history"] + 8 * case["biases"]), "flops": 4 * n}
    matrices = 2 if case["op"] == "gated" else 1
    n = case["inner"] * case["cols"]
    weight = n // 2 + -(-case["inner"] // case["group"]) * case["cols"] * (5 if case["zeros"] else 4)
    return {"bytes": 4 * case["rows"] * (case["inner"] + case["cols"]) + matrices * weight, "flops": 2 * matrices * case["rows"] * n}


# ---- the definitions once more, with numpy on the host -------------------------------------------------------------------------------------------
def _floor(v, s):
    return (v + s // 2) // s


def _host_attention(case, a):
    heads, kv_heads, dim, n, prefix, page = (case[k] for k in ("heads", "kv_heads", "dim", "tokens", "prefix", "page"))
    scale = SCORE_SCALE * math.sqrt(dim)
    out = np.zeros((case["seqs"] * n, heads, dim), np.int64)
    for i in range(case["seqs"]):
        length = int(a["lengths"][i])
        places = [(int(a["table"][i, t // page]), t % page) for t in range(length)]
        k = np.concatenate([a["prefix_k"]] + [a["k_pages"][p, t][None] for p, t in places])
        v = np.concatenate([a["prefix_v"]] + [a["v_pages"][p, t][None] for p, t in places])
        for t in range(n):
            seen = prefix + (length - n + t + 1 if case["causal"] else length)
            if seen <= 0:
                continue
            for h in range(heads):
                kh = h // (heads // kv_heads)
                scores = (k[:seen, kh].astype(np.float64) @ a["q"][i * n + t, h].astype(np.float64)).astype(np.int64)
                total = np.cumsum(np.exp(scores.astype(np.float64) / scale))[-1]      # one after the other
                shifted = int(math.floor(scale * math.log(total) + 0.5)) - scores
                weight, y = RADICES[0], np.ones(seen, np.int64)
                for radix, theta in zip(RADICES[DROPPED:], THETAS):
                    y *= np.floor(np.exp(math.log(theta) - weight / scale * (shifted // weight % radix)) + 0.5).astype(np.int64)
                    weight *= radix
                out[i * n + t, h] = _floor(_floor((y[:, None] * v[:seen, kh]).sum(0), ATTN_SCALE), ATTN_SCALE)
    return out.astype(np.int32)


def _host_logits(case, a):
    out, token = np.empty((case["rows"], case["vocab"]), np.int64), np.empty(case["rows"], np.int64)
    for r in range(case["rows"]):
        l = a["logits"][r].copy()
        count = np.bincount(a["history"][a["history_starts"][r]:a["history_starts"][r + 1]], minlength=case["vocab"])
        repeat, frequency, presence = (int(v) for v in a["penalties"][r])
        for t in np.nonzero(count)[0]:
            v = int(l[t])
            v = (v * SCALE + repeat // 2) // repeat if v > 0 else _floor(v * repeat, SCALE)
            l[t] = v - frequency * int(count[t]) - presence
        at = slice(a["bias_starts"][r], a["bias_starts"][r + 1])
        np.add.at(l, a["bias_tokens"][at], a["bias_values"][at])
        if case["masked"]:
            allowed = np.unpackbits(a["mask"][r].astype(np.uint32).view(np.uint8), bitorder="little")[:case["vocab"]]
            l[allowed == 0] = NONE
        out[r] = l
        token[r] = -1 if l.max() == NONE else int(np.argmax(l))
    return {"logits": out.astype(np.int32), "token": token.astype(np.int32)}


def _host_weight(w):
    case = w.case
    codes = w.codes.cpu().numpy()
    q = np.empty((case["inner"], 2 * codes.shape[1]), np.int64)
    q[:, 0::2], q[:, 1::2] = codes & 15, codes >> 4
    out = np.empty((case["inner"], case["cols"]))
    scales, zeros = w.scales.cpu().numpy().astype(np.int64), None if w.zeros is None else w.zeros.cpu().numpy().astype(np.int64)
    for g in range(len(scales)):
        rows = slice(g * case["group"], (g + 1) * case["group"])
        out[rows] = (q[rows, :case["cols"]] - (8 if zeros is None else zeros[g])) * scales[g]
    return out


def _host_product(x, w):
    """exact: x in two pieces of 11 bits and the rest, each product's sums below 2^53"""
    low = x & 2047
    return (low.astype(np.float64) @ w).astype(np.int64) + ((x >> 11).astype(np.float64) @ w).astype(np.int64) * 2048


def exact(case, seed):
    if case["op"] in ("linear", "gated") and case["rows"] * case["inner"] * case["cols"] > 10 ** 10:
        return None
    if case["op"] == "attention" and case["seqs"] * case["tokens"] * case["heads"] * (case["prefix"] + case["own"]) * (case["dim"] + 20) > 10 ** 9:
        return None
    global own
    was, own = own, False   # inputs alone
    try:
        s = prepare(case, seed)
    finally:
        own = was
    a = {k: v.cpu().numpy().astype(np.int64) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if case["op"] == "append":
        k, v = a["k_pages"], a["v_pages"]
        for i in range(case["seqs"]):
            for t in range(case["tokens"]):
                at = int(a["lengths"][i]) - case["tokens"] + t
                page, slot = int(a["table"][i, at // case["page"]]), at % case["page"]
                k[page, slot], v[page, slot] = a["kv"][i * case["tokens"] + t]
        return {"k": k.astype(np.int32), "v": v.astype(np.int32)}
    if case["op"] == "attention":
        a["prefix_k"], a["prefix_v"] = (t.cpu().numpy().astype(np.int64) for t in s["prefix"])
        return _host_attention(case, a)
    if case["op"] == "logits":
        return _host_logits(case, a)
    w = [_host_weight(t) for t in s["w"]]
    if case["op"] == "linear":
        return _floor(_host_product(a["x"], w[0]), SCALE).astype(np.int32)
    gate, up = _floor(_host_product(a["x"], w[0]), 1 << 20), _floor(_host_product(a["x"], w[1]), SCALE)
    return _floor(a["act"][gate + (1 << 21)] * up, SCALE).astype(np.int32)

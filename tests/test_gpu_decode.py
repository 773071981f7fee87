"""Answering token by token in the prover's integers (zk_i32_cache_append, zk_i32_attention, zk_i32_rhs_prepare_q4, zk_i32_logits): whole numbers, so every comparison is for equality."""
import ctypes

import numpy as np
import pytest

import decodehelp as dec
import valueshelp as ref
from valueshelp import POSITION, RANGE, TABLE

c_void_p, c_size_t, c_int, c_uint, c_double = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint32, ctypes.c_double
gpu = pytest.mark.gpu


class Cache(ctypes.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("page_stride", c_size_t), ("token_stride", c_size_t), ("head_stride", c_size_t), ("page_size", c_uint), ("pages", c_uint),
                ("page_table", c_void_p), ("table_cols", c_uint)]


@pytest.fixture(scope="module")
def hip():
    import torch
    from gpuhelp import Hip
    torch.cuda.init()
    h = Hip()
    for f in ("zk_i32_attention_workspace", "zk_i32_rhs_workspace", "zk_i32_logits_workspace", "zk_i32_linear_workspace"):
        getattr(h.lib, f).restype = c_size_t
    return h


def dev(a, dtype=np.int32):
    import torch
    return None if a is None else torch.as_tensor(np.ascontiguousarray(a, dtype=dtype).copy(), device="cuda")


def new_flag():
    import torch
    return torch.zeros(1, dtype=torch.int32, device="cuda")


def ptr(t):
    return c_void_p(None if t is None or t.numel() == 0 else t.data_ptr())


def host(t):
    import torch
    torch.cuda.synchronize()
    return t.cpu().numpy()


def normal(rng, shape, std=65536.0, most=1 << 24):
    return np.clip(np.round(rng.normal(0, std, shape)), -most, most).astype(np.int32)


# ---- caches --------------------------------------------------------------------------------------------------------------------------------
class Pages:
    """keys and values of sequences in pages in no order; by_head: [page][head][place][dim]; offset: elements before the first (rows that begin at no multiple of 16 bytes)"""

    def __init__(self, rng, seqs, most, kv_heads, dim, page, table=True, by_head=False, offset=0, fill=None, pad=0):
        self.page, self.kv_heads, self.dim, self.offset = page, kv_heads, dim, offset
        self.cols = -(-most // page) if table else 1
        self.table = rng.permutation(seqs * self.cols).reshape(seqs, self.cols).astype(np.int32) if table else np.arange(seqs, dtype=np.int32).reshape(seqs, 1)
        wide = dim + pad
        self.token, self.head = (wide, page * wide) if by_head else (kv_heads * wide, wide)
        self.stride = page * kv_heads * wide
        n = seqs * self.cols * self.stride + offset
        self.k, self.v = (normal(rng, n) if fill is None else np.full(n, fill, np.int32) for _ in range(2))
        self.dk, self.dv, self.dt = dev(self.k), dev(self.v), dev(self.table) if table else None

    def at(self, s, t, h):
        p = self.offset + int(self.table[s, t // self.page]) * self.stride + t % self.page * self.token + h * self.head
        return slice(p, p + self.dim)

    def put(self, s, t, h, k, v):
        self.k[self.at(s, t, h)], self.v[self.at(s, t, h)] = k, v

    def read(self, s, n, h):
        return tuple(np.array([a[self.at(s, t, h)] for t in range(n)], np.int64).reshape(n, self.dim) for a in (self.k, self.v))

    def c(self):
        return Cache(self.dk.data_ptr() + 4 * self.offset, self.dv.data_ptr() + 4 * self.offset, self.stride, self.token, self.head, self.page, self.table.size,
                     None if self.dt is None else self.dt.data_ptr(), 0 if self.dt is None else self.cols)


def append(hip, cache, k, v, heads, dim, seqs, starts, lengths, flag, stream=None):
    c = cache.c()
    hip.call("zk_i32_cache_append", ctypes.byref(c), ptr(k), c_size_t(k.stride(0)), c_size_t(k.stride(1)), ptr(v), c_size_t(v.stride(0)), c_size_t(v.stride(1)), c_uint(k.shape[0]), c_uint(heads),
             c_uint(dim), c_uint(seqs), ptr(starts), ptr(lengths), ptr(flag), stream)


@gpu
@pytest.mark.parametrize("counts,lengths,heads,dim,page,table,by_head,offset", [
    ([1], [1], 1, 1, 1, True, False, 0), ([1], [200], 8, 128, 64, True, False, 0), ([3, 0, 5], [3, 7, 5], 2, 80, 17, True, False, 0), ([3, 1, 5], [20, 33, 40], 2, 7, 16, True, True, 1),
    ([2, 2], [64, 2], 3, 64, 64, False, False, 0), ([4, 4, 4], [9, 40, 4], 5, 20, 5, True, True, 0), ([100], [130], 4, 256, 32, True, False, 4)])
def test_append(hip, counts, lengths, heads, dim, page, table, by_head, offset):
    rng = np.random.default_rng(sum(lengths) * 7 + dim)
    tokens = sum(counts) + 2                        # two behind the last sequence
    cache = Pages(rng, len(counts), max(lengths), heads, dim, page, table, by_head, offset, fill=-7, pad=4 if by_head else 0)
    kv = normal(rng, (tokens, 2, heads, dim))
    d = dev(kv)
    starts = np.cumsum([0] + counts)
    flag = new_flag()
    append(hip, cache, d[:, 0], d[:, 1], heads, dim, len(counts), dev(starts), dev(lengths), flag)
    for s, n in enumerate(counts):
        for i in range(n):
            for h in range(heads):
                cache.put(s, lengths[s] - n + i, h, kv[starts[s] + i, 0, h], kv[starts[s] + i, 1, h])
    assert host(flag)[0] == 0
    assert (host(cache.dk) == cache.k).all() and (host(cache.dv) == cache.v).all()


@gpu
def test_append_leaves_what_has_no_place(hip):
    """a length below the new tokens', one beyond the cache, a page that there is not, starts that descend: the others are written"""
    rng = np.random.default_rng(5)
    cache = Pages(rng, 5, 32, 2, 8, 16, fill=-7)
    cache.table[2, 0], cache.table[2, 1] = 99, -1
    cache.dt.copy_(dev(cache.table))
    kv = normal(rng, (10, 2, 2, 8))
    d, flag = dev(kv), new_flag()
    lengths = [1, 33, 17, 20, 5]                    # sequence 0 has two new tokens and one place
    append(hip, cache, d[:, 0], d[:, 1], 2, 8, 5, dev([0, 2, 4, 6, 8, 7]), dev(lengths), flag)
    for h in range(2):
        cache.put(0, 0, h, kv[1, 0, h], kv[1, 1, h])
        for i in range(2):
            cache.put(3, 18 + i, h, kv[6 + i, 0, h], kv[6 + i, 1, h])
    assert host(flag)[0] == POSITION
    assert (host(cache.dk) == cache.k).all() and (host(cache.dv) == cache.v).all()


# ---- attention -----------------------------------------------------------------------------------------------------------------------------
class Plan:
    def __init__(self, hip, softmax):
        self.hip, self.s, self.h = hip, softmax, c_void_p()
        s = softmax
        hip.call("zk_i32_softmax_prepare", ctypes.byref(self.h), (c_uint * len(s.bs))(*s.bs), c_int(len(s.bs)), c_int(s.L), c_int(s.M), c_double(s.sf_in), (c_double * len(s.thetas))(*s.thetas),
                 c_uint(s.dim), None)

    def __del__(self):
        self.hip.lib.zk_i32_softmax_free(self.h)


def attend(hip, q, plan, prefix, prefix_len, own, seqs, starts, lengths, most, causal, kv_heads, sf=(1 << 20, 1 << 20), out=None, shift=None, ws="caller", flag=None, stream=None, tokens=None, heads=None):
    """q: a tensor [token][head][dim], any strides with contiguous heads"""
    import torch
    n, h, dim = q.shape
    out = torch.full(q.shape, -77, dtype=torch.int32, device="cuda") if out is None else out
    size = hip.lib.zk_i32_attention_workspace(c_uint(n), c_uint(h), c_uint(kv_heads), c_uint(dim), c_uint(prefix_len), c_uint(seqs if own else 0), c_uint(most))
    if isinstance(ws, str):
        ws = torch.full((max(size, 16),), 0x5B, dtype=torch.uint8, device="cuda")
    pc, oc = prefix.c() if prefix else None, own.c() if own else None
    hip.call("zk_i32_attention", ptr(out), c_size_t(out.stride(0)), c_size_t(out.stride(1)), ptr(q), c_size_t(q.stride(0)), c_size_t(q.stride(1)), c_uint(n), c_uint(h), c_uint(kv_heads), c_uint(dim),
             plan.h, ctypes.byref(pc) if pc else None, c_uint(prefix_len), ctypes.byref(oc) if oc else None, c_uint(seqs), ptr(starts), ptr(lengths), c_uint(most), c_int(causal), c_uint(sf[0]),
             c_uint(sf[1]), ptr(shift), ptr(ws), c_size_t(0 if ws is None else ws.numel()), ptr(flag), stream)
    return out


def expected(q, softmax, prefix, prefix_len, own, counts, lengths, causal, kv_heads, sf=(1 << 20, 1 << 20), before=-77):
    out = np.full(q.shape, before, np.int64)
    shift = np.zeros(q.shape[:2], np.int64)
    group = q.shape[1] // kv_heads
    at = 0
    for s, n in enumerate(counts):
        for i in range(n):
            seen = 0 if not own else max(0, lengths[s] - n + i + 1) if causal else lengths[s]
            for h in range(q.shape[1]):
                keys = [np.zeros((0, q.shape[2]), np.int64)] * 2
                if prefix:
                    keys = prefix.read(0, prefix_len, h // group)
                if own:
                    keys = [np.concatenate(p) for p in zip(keys, own.read(s, seen, h // group))]
                out[at, h], shift[at, h] = dec.attention(q[at, h], keys[0], keys[1], softmax, *sf)
            at += 1
    return out, shift


ATTENTION = [
    # counts, lengths, heads, kv heads, dim, prefix, page, causal, options
    ([1], [1], 1, 1, 1, 0, 1, True, ""), ([1], [17], 4, 4, 64, 0, 16, True, ""), ([1], [200], 4, 1, 128, 0, 64, True, ""), ([1, 1, 1], [1, 40, 65], 8, 2, 64, 100, 32, True, ""),
    ([2, 5, 0, 1], [2, 30, 9, 0], 6, 3, 80, 33, 17, True, ""), ([2, 5, 0, 1], [2, 30, 9, 0], 6, 3, 80, 33, 17, False, ""), ([3, 4], [1, 0], 2, 2, 20, 0, 8, True, ""),
    ([20], [20], 3, 3, 48, 0, 20, False, "flat"), ([37], [50], 4, 2, 65, 16, 7, True, "odd"), ([1, 1], [70, 3], 40, 1, 16, 70, 9, True, ""), ([9], [9], 2, 1, 256, 260, 4, True, ""),
    ([2, 2], [300, 513], 2, 1, 200, 0, 128, True, "by head"), ([1, 2], [64, 256], 5, 5, 3, 64, 64, True, "odd by head"), ([4], [0], 2, 2, 32, 50, 16, False, "only prefix"),
    ([16, 17], [40, 40], 2, 2, 96, 0, 40, True, "flat strided"), ([33], [33], 1, 1, 128, 0, 33, True, "flat in place")]


@gpu
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,dim,prefix_len,page,causal,options", ATTENTION)
def test_attention(hip, counts, lengths, heads, kv_heads, dim, prefix_len, page, causal, options):
    import torch
    rng = np.random.default_rng(heads * 1000 + dim + sum(lengths))
    softmax = dec.Softmax(dim=dim)
    plan = Plan(hip, softmax)
    more = {"by_head": "by head" in options, "offset": 1 if "odd" in options else 0}
    prefix = Pages(rng, 1, prefix_len, kv_heads, dim, 48 if prefix_len > 64 else max(prefix_len, 1), prefix_len > 64, **more) if prefix_len else None
    own = None if options == "only prefix" else Pages(rng, len(counts), max(lengths), kv_heads, dim, page, "flat" not in options, **more)
    behind = 2 if len(counts) > 1 else 0
    n = sum(counts)
    q = normal(rng, (n + behind, heads, dim))
    if "strided" in options:                        # heads first, rows that hold more than their heads
        wide = dev(np.zeros((heads, n + behind, dim + 4), np.int32))
        dq = wide.transpose(0, 1)[:, :, :dim]
        dq.copy_(dev(q))
        out = torch.full((heads, n + behind, dim + 4), -77, dtype=torch.int32, device="cuda").transpose(0, 1)[:, :, :dim]
    else:
        dq = dev(q)
        out = dq if "in place" in options else None
    flag, shift = new_flag(), torch.full((n + behind, heads), -5, dtype=torch.int64, device="cuda")
    got = attend(hip, dq, plan, prefix, prefix_len, own, len(counts), dev(np.cumsum([0] + counts)), dev(lengths), max(lengths) if own else 0, causal, kv_heads, out=out, shift=shift, flag=flag)
    assert host(flag)[0] == 0
    exp, shifts = expected(q, softmax, prefix, prefix_len, own, counts, lengths, causal, kv_heads)
    rows = slice(0, n + behind) if not own else slice(0, n)
    if not own:
        exp, shifts = expected(q, softmax, prefix, prefix_len, None, [n + behind], [0], False, kv_heads)
    assert (host(got)[rows] == exp[rows]).all()
    assert (host(shift)[rows] == shifts[rows]).all()
    if own and behind:                              # rows behind the last sequence are left as they were
        assert (host(got)[n:] == -77).all() and (host(shift)[n:] == -5).all()


@gpu
@pytest.mark.parametrize("softmax", [
    dec.Softmax((100, 1000003, 999983), 1, 0, float(1 << 31), (250000.0, 4000000.0), 24), dec.Softmax((1 << 10, 1 << 12, 1 << 20, 16), 1, 1, float(1 << 30), (5000.0, 30000.0), 24),
    dec.Softmax((1 << 24, 1 << 20), 0, 0, float(1 << 32), (3000.0, 1000000.0), 24), dec.Softmax((4096, 7, 1 << 20, 1 << 16, 3), 2, 1, float(1 << 32), (1000.0, 900000.0), 24),
    dec.Softmax((1 << 20, 1 << 22), 1, 0, float(1 << 32), (1000000.0,), 24)])
@pytest.mark.parametrize("sf", [(1 << 20, 1 << 20), (1000003, 77), (1, 1 << 25)])
def test_attention_softmaxes(hip, softmax, sf):
    rng = np.random.default_rng(int(sum(softmax.bs)) + sf[0])
    plan = Plan(hip, softmax)
    own = Pages(rng, 2, 90, 2, 24, 13)
    q = normal(rng, (4, 2, 24), 40000.0)
    if sf[0] == 1:                                  # outputs of 16 bits more
        for a in (own.v, ):
            a[:] //= 4096
        own.dv.copy_(dev(own.v))
    flag = new_flag()
    got = attend(hip, dev(q), plan, None, 0, own, 2, dev([0, 1, 4]), dev([77, 90]), 90, True, 2, sf=sf, flag=flag)
    exp, _ = expected(q, softmax, None, 0, own, [1, 3], [77, 90], True, 2, sf)
    assert host(flag)[0] == 0
    assert (host(got) == exp).all()


@gpu
@pytest.mark.parametrize("factor", [0.9, 0.6, 0.45, 0.4, 0.1, 0.001])
@pytest.mark.parametrize("tokens,keys", [(3, 90), (3, 700), (300, 600)])
def test_attention_of_small_second_factors(hip, factor, tokens, keys):
    """Below 0.5 the second table holds zeros alone, from some e^-0.75 = 0.47 down no entry is reached by its bound: every output is 0, in one launch and in several, of few rows and of many"""
    import torch
    rng = np.random.default_rng(tokens + keys)
    dim = 64
    softmax = dec.Softmax(thetas=(float(1 << 18), factor), dim=dim)
    own = Pages(rng, 1, keys, 1, dim, 64)
    q = normal(rng, (tokens, 1, dim))
    flag, shift = new_flag(), torch.full((tokens, 1), -5, dtype=torch.int64, device="cuda")
    got = host(attend(hip, dev(q), Plan(hip, softmax), None, 0, own, 1, None, dev([keys]), keys, False, 1, sf=(1 << 10, 1 << 6), shift=shift, flag=flag))
    assert host(flag)[0] == 0
    k, v = own.read(0, keys, 0)
    for i in {0, 1, tokens // 2, tokens - 1}:
        exp, s = dec.attention(q[i, 0], k, v, softmax, 1 << 10, 1 << 6)
        assert host(shift)[i, 0] == s and (got[i, 0] == exp).all() and (factor > 0.5 or not exp.any()), i


@gpu
@pytest.mark.parametrize("big_q,big_k,big_v", [(1 << 27, 1 << 27, 1 << 16), (1 << 20, 0x7F7F7F7F, 1 << 20), (0x7F7F7F7F, 1 << 18, 0x7F7F7F7F), (1 << 10, 1 << 10, 0x7F7F7F7F)])
def test_attention_of_large_values(hip, big_q, big_k, big_v):
    """four digits in some places of the queries, keys and values; the weights are small so that sums fit"""
    rng = np.random.default_rng(big_q % 1000 + big_k % 999)
    dim = 4
    softmax = dec.Softmax((1 << 30 >> 2, 1 << 20, 1 << 13), 1, 0, float(big_q) * big_k / 4, (1000.0, 3000.0), dim)
    plan = Plan(hip, softmax)
    own = Pages(rng, 1, 150, 1, dim, 64)
    for a, big in ((own.k, big_k), (own.v, big_v)):
        a[:] = rng.integers(-big, big + 1, a.size)
        a[:8] = [big, -big, big, -big, 0, -1, 1, 127]
    own.dk.copy_(dev(own.k)), own.dv.copy_(dev(own.v))
    q = rng.integers(-big_q, big_q + 1, (3, 1, dim)).astype(np.int32)
    q[0] = [[big_q, -big_q, big_q, 128]]
    flag = new_flag()
    got = attend(hip, dev(q), plan, None, 0, own, 1, dev([0, 3]), dev([150]), 150, False, 1, sf=(3000, 1000), flag=flag)
    exp, _ = expected(q, softmax, None, 0, own, [3], [150], False, 1, (3000, 1000))
    # in the last case every score lies within the digit that is dropped, 2^28: all weights are the largest, and the sums of 150 values leave int32 here and there
    fits = (exp >= -(1 << 31)) & (exp < 1 << 31)
    assert fits.all() == (big_k != 1 << 10)
    assert host(flag)[0] == (0 if fits.all() else RANGE)
    assert (host(got)[fits] == exp[fits]).all()


def shifts_of(hip, scores, scale):
    """zk_softmax_shift's: scores [row][key] int64"""
    import torch
    rows, cols = scores.shape
    x, fr, out, sh, back = dev(scores, np.int64), *(torch.empty(n * 8, dtype=torch.int32, device="cuda") for n in (scores.size, scores.size, rows)), torch.empty(rows, dtype=torch.int64, device="cuda")
    hip.call("zk_fr_from_i64", ptr(fr), ptr(x), c_size_t(scores.size), None)
    hip.call("zk_softmax_shift", ptr(sh), ptr(out), ptr(fr), c_uint(rows), c_uint(cols), c_double(scale), None)
    hip.call("zk_fr_to_i64", ptr(back), ptr(sh), c_size_t(rows), None)
    return host(back)


@gpu
@pytest.mark.parametrize("kind", ["normal", "rising", "falling", "equal", "one large", "two levels", "tiny", "pairs"])
@pytest.mark.parametrize("keys,prefix_len", [(1, 0), (2, 0), (63, 0), (65, 0), (511, 0), (513, 100), (2048, 2047), (5000, 1), (20000, 9000)])
def test_shifts_are_the_sums_of_exponentials_in_order(hip, kind, keys, prefix_len):
    """At this scale a shift is some 2^53: it tells sums apart that differ by their last bit, and zk_softmax_shift's sum is taken one term after the other."""
    import torch
    rng = np.random.default_rng(keys)
    softmax = dec.Softmax((1 << 28, 1 << 28, 1 << 7), 1, 0, float(1 << 49), (1000.0, 1000.0), 1)
    k = {"normal": rng.normal(0, 1.0, keys), "rising": np.linspace(-20, 3, keys), "falling": np.linspace(3, -20, keys), "equal": np.zeros(keys), "one large": np.where(np.arange(keys) == keys // 2, 9.0, -3.0),
         "two levels": np.where(rng.random(keys) < 0.5, 0.0, -0.6931471805599453), "tiny": rng.normal(-30, 5.0, keys), "pairs": np.repeat(rng.normal(0, 4.0, (keys + 1) // 2), 2)[:keys]}[kind]
    k = np.round(k * (1 << 22)).astype(np.int32)
    q = np.array([[[1 << 27]], [[-(1 << 26) + 12345]], [[77777777]]], np.int32)
    prefix = Pages(rng, 1, prefix_len, 1, 1, prefix_len, False) if prefix_len else None
    own = Pages(rng, 1, keys - prefix_len, 1, 1, 100)
    if prefix:
        prefix.k[:], prefix.v[:] = k[:prefix_len], 1
        prefix.dk.copy_(dev(prefix.k)), prefix.dv.copy_(dev(prefix.v))
    for t in range(keys - prefix_len):
        own.put(0, t, 0, k[prefix_len + t], 1)
    own.dk.copy_(dev(own.k)), own.dv.copy_(dev(own.v))
    shift = torch.zeros((3, 1), dtype=torch.int64, device="cuda")
    attend(hip, dev(q), Plan(hip, softmax), prefix, prefix_len, own, 1, dev([0, 3]), dev([keys - prefix_len]), keys - prefix_len, False, 1, sf=(1, 1), shift=shift, flag=new_flag())
    scores = k.astype(np.int64)[None] * q.reshape(3, 1)
    assert (host(shift)[:, 0] == shifts_of(hip, scores, softmax.scale)).all()


@gpu
@pytest.mark.parametrize("kind", ["normal", "rising", "falling", "two levels"])
@pytest.mark.parametrize("keys", [600, 2048, 2500, 9001])
def test_shifts_of_many_rows(hip, kind, keys):
    """The same where rows are many: every one of them goes through both launches at this scale"""
    import torch
    rng, rows = np.random.default_rng(keys + 1), 300
    softmax = dec.Softmax((1 << 28, 1 << 28, 1 << 7), 1, 0, float(1 << 49), (1000.0, 1000.0), 1)
    k = {"normal": rng.normal(0, 1.0, keys), "rising": np.linspace(-20, 3, keys), "falling": np.linspace(3, -20, keys), "two levels": np.where(rng.random(keys) < 0.5, 0.0, -0.6931471805599453)}[kind]
    k = np.round(k * (1 << 22)).astype(np.int32)
    q = rng.integers(-(1 << 27), 1 << 27, (rows, 1, 1)).astype(np.int32)
    own = Pages(rng, 1, keys, 1, 1, keys, False)
    own.k[:], own.v[:] = k, 1
    own.dk.copy_(dev(own.k)), own.dv.copy_(dev(own.v))
    shift = torch.zeros((rows, 1), dtype=torch.int64, device="cuda")
    attend(hip, dev(q), Plan(hip, softmax), None, 0, own, 1, dev([0, rows]), dev([keys]), keys, False, 1, sf=(1, 1), shift=shift, flag=new_flag())
    assert (host(shift)[:, 0] == shifts_of(hip, k.astype(np.int64)[None] * q.reshape(rows, 1), softmax.scale)).all()


@gpu
@pytest.mark.parametrize("what,bit", [("query", RANGE), ("key", RANGE), ("value", RANGE), ("score", RANGE), ("output", RANGE), ("far", TABLE), ("page", POSITION), ("length", POSITION), ("negative", POSITION), ("starts", POSITION)])
def test_attention_raises_flags(hip, what, bit):
    """and leaves the other sequence right"""
    rng = np.random.default_rng(3)
    softmax = dec.Softmax(dim=8) if what != "far" else dec.Softmax((1 << 8, 1 << 10, 1 << 10), 1, 0, float(1 << 32), (1000.0, 1000.0), 8)
    plan = Plan(hip, softmax)
    own = Pages(rng, 2, 40, 1, 8, 16)
    q = normal(rng, (2, 1, 8), 30000.0) if what != "far" else normal(rng, (2, 1, 8), 3.0)
    lengths, starts = [40, 40], [0, 1, 2]
    at = own.at(0, 20, 0).start
    if what == "query":
        q[0, 0, 3] = 0x7F7F7F80
    elif what == "key":
        own.k[at] = 0x7FFFFFFF
    elif what == "value":
        own.v[at] = 0x7F7F7F80
    elif what == "score":
        own.k[at:at + 8], q[0, 0] = 0x70000000, 0x70000000
    elif what == "output":
        own.v[:] = 1 << 26
    elif what == "far":
        own.k[:] //= 64
        own.k[at:at + 8], q[0, 0] = -(1 << 24), 1 << 22
    elif what == "page":
        own.table[0, 1] = 6
    elif what == "length":
        lengths[0] = 41
    elif what == "negative":
        lengths[0] = -1
    elif what == "starts":
        starts = [-1, 1, 2]
    for d, h in ((own.dk, own.k), (own.dv, own.v), (own.dt, own.table)):
        d.copy_(dev(h))
    if what == "output":
        softmax_sf = (1 << 10, 1)
    flag = new_flag()
    got = host(attend(hip, dev(q), plan, None, 0, own, 2, dev(starts), dev(lengths), 40, True, 1, sf=softmax_sf if what == "output" else (1 << 20, 1 << 20) if what != "far" else (1000, 1000), flag=flag))
    assert host(flag)[0] & bit
    if what in ("length", "negative", "starts"):
        assert (got[0] == -77).all()
    if what not in ("output", "far"):
        own.table[0, 1] = own.table[0, 1] if what != "page" else 0
        exp, _ = expected(np.stack([q[1], q[1]]), softmax, None, 0, own, [1, 1], [1, 40], True, 1)
        assert (got[1] == exp[1]).all()


@gpu
def test_attention_without_a_flag_returns_the_error(hip):
    rng = np.random.default_rng(4)
    plan = Plan(hip, dec.Softmax(dim=8))
    own = Pages(rng, 1, 40, 1, 8, 16)
    q = normal(rng, (1, 1, 8), 30000.0)
    for ws in (None, "caller"):
        got = attend(hip, dev(q), plan, None, 0, own, 1, None, dev([40]), 40, True, 1, ws=ws)
        assert (host(got) == expected(q, plan.s, None, 0, own, [1], [40], True, 1)[0]).all()
        with pytest.raises(RuntimeError, match="zk_i32_attention: a position"):
            attend(hip, dev(q), plan, None, 0, own, 1, None, dev([41]), 40, True, 1, ws=ws)


@gpu
@pytest.mark.parametrize("tokens,heads,kv_heads,dim,prefix_len,most", [(3, 4, 2, 32, 9000, 20), (2, 2, 2, 64, 0, 17000), (130, 8, 2, 64, 40, 130), (300, 2, 2, 128, 0, 300)])
def test_attention_of_many_keys_and_many_tokens(hip, tokens, heads, kv_heads, dim, prefix_len, most):
    """parts of long rows joined, many tiles of queries, against the same in torch's 64-bit floating point and integers"""
    import torch
    rng = np.random.default_rng(most)
    softmax = dec.Softmax(dim=dim)
    prefix = Pages(rng, 1, prefix_len, kv_heads, dim, prefix_len, False) if prefix_len else None
    own = Pages(rng, 1, most, kv_heads, dim, most, False)
    q = normal(rng, (tokens, heads, dim))
    flag = new_flag()
    got = host(attend(hip, dev(q), Plan(hip, softmax), prefix, prefix_len, own, 1, None, dev([most]), most, True, kv_heads, flag=flag))
    assert host(flag)[0] == 0
    for i in {0, 1, tokens // 2, tokens - 1}:
        for h in range(heads):
            keys = own.read(0, most - tokens + i + 1, h * kv_heads // heads)
            if prefix:
                keys = [np.concatenate(p) for p in zip(prefix.read(0, prefix_len, h * kv_heads // heads), keys)]
            scores = keys[0] @ q[i, h].astype(np.int64)
            y = softmax.weights(softmax.shift(scores) - scores)
            sums = (y[:, None] >> 20) * keys[1], (y[:, None] & 0xFFFFF) * keys[1]
            v = sums[0].sum(0) * (1 << 20) + sums[1].sum(0)
            assert (got[i, h] == ref.quotient(ref.quotient(v, 1 << 20), 1 << 20)).all(), (i, h)


# Tiles of 64 rows: a prefix under few rows (whose values every tile splits), under many (split once), one sequence's prompt, prompts of several, rows that begin and end inside tiles, parts joined; heads of every
# number of blocks of dimensions and every way to read them; fourth digits here and there
TILES = [([40], [700], 4, 2, 128, 0, 64, True, ""), ([40, 3, 0, 70], [650, 3, 9, 90], 4, 1, 64, 100, 33, True, ""), ([9, 8], [20, 300], 4, 2, 80, 600, 16, True, ""), ([70], [700], 4, 2, 80, 130, 50, False, "wide"),
         ([130], [640], 2, 1, 65, 70, 64, True, "odd wide"), ([150], [150], 2, 2, 130, 600, 150, True, "flat"), ([64], [64], 8, 4, 200, 640, 64, True, "by head wide"), ([33, 100], [600, 610], 4, 2, 256, 0, 64, True, ""),
         ([129], [0], 2, 2, 96, 700, 16, False, "only prefix wide"), ([200], [777], 2, 2, 128, 0, 777, False, "flat lowest"), ([140], [600], 1, 1, 256, 64, 64, False, "lowest"), ([20], [9000], 8, 1, 32, 0, 100, True, ""),
         ([300], [300], 2, 2, 128, 640, 300, True, "flat wide far"), ([260, 20], [260, 300], 2, 2, 96, 700, 64, True, "wide"), ([150], [700], 2, 1, 256, 0, 700, False, "flat wide"), ([257], [64], 1, 1, 64, 577, 64, True, "lowest"),
         ([90], [640], 4, 1, 65, 70, 64, True, "odd wide"), ([260], [0], 2, 2, 200, 9000, 16, False, "only prefix")]


@gpu
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,dim,prefix_len,page,causal,options", TILES)
def test_attention_in_tiles(hip, counts, lengths, heads, kv_heads, dim, prefix_len, page, causal, options):
    rng = np.random.default_rng(heads * 1000 + dim + sum(lengths))
    large = "wide" in options or "lowest" in options
    softmax = dec.Softmax((1 << 20, 1 << 20, 1 << 14), 1, 0, float(1 << 44), (1000.0, 3000.0), dim) if large else dec.Softmax(dim=dim)
    sf = (3000, 1000) if large else (1 << 20, 1 << 20)
    more = {"by_head": "by head" in options, "offset": 1 if "odd" in options else 0}
    prefix = Pages(rng, 1, prefix_len, kv_heads, dim, 48, True, **more) if prefix_len else None
    own = None if "only prefix" in options else Pages(rng, len(counts), max(lengths), kv_heads, dim, page, "flat" not in options, **more)
    n = sum(counts)
    behind = 2 if own and len(counts) > 1 else 0
    q = normal(rng, (n + behind, heads, dim), 60000.0)
    for c in (prefix, own):
        if c is not None and "wide" in options:     # fourth digits, in some keys and values
            for a in (c.k, c.v):
                a[rng.integers(0, a.size, 40)] = rng.integers(-(1 << 27), 1 << 27, 40)
        if c is not None and "lowest" in options:   # three digits of -128 each
            c.k[:] = -8421504
            c.v[::2] = -8421504
        if c is not None:
            c.dk.copy_(dev(c.k)), c.dv.copy_(dev(c.v))
    if "wide" in options:
        q[rng.integers(0, n, 5), 0, rng.integers(0, dim, 5)] = rng.integers(-(1 << 27), 1 << 27, 5)
    if "lowest" in options:
        q[1::2] = -8421504
    flag = new_flag()
    got = host(attend(hip, dev(q), Plan(hip, softmax), prefix, prefix_len, own, len(counts), dev(np.cumsum([0] + counts)), dev(lengths), max(lengths) if own else 0, causal, kv_heads, sf=sf, flag=flag))
    # far: a query's fourth digit meets a key's: that product of up to 2^54 puts one score 1.008 x 2^54 below its row's shift, and the three tables hold 2^20 2^20 2^14 distances
    assert host(flag)[0] == (TABLE if "far" in options else 0)
    at = 0
    for s, count in enumerate(counts):
        for i in range(count):
            if i not in (0, 1, 2, 15, 16, 31, 63, 64, 65, count // 2, count - 2, count - 1):
                at += 1
                continue
            seen = 0 if not own else max(0, lengths[s] - count + i + 1) if causal else lengths[s]
            for h in range(heads):
                keys = [np.zeros((0, dim), np.int64)] * 2
                for c, m, j in ((prefix, prefix_len, 0), (own, seen, s)):
                    if c:
                        keys = [np.concatenate(p) for p in zip(keys, c.read(j, m, h * kv_heads // heads))]
                exp, _ = dec.attention(q[at, h], keys[0], keys[1], softmax, *sf)
                assert (got[at, h] == exp).all(), (s, i, h)
            at += 1
    if behind:
        assert (got[n:] == -77).all()


def smaller_workspaces(hip, lower, upper, call):
    """the smallest workspace that a call is not refused with, between a size that is too small and one that is enough; call(bytes, plan) with a plan for heads of another width ends at that"""
    other = Plan(hip, dec.Softmax(dim=1))
    while lower + 1 < upper:
        mid = (lower + upper) // 2
        with pytest.raises(RuntimeError) as e:
            call(mid, other)
        small = "the workspace is smaller" in str(e.value)
        assert small or "another width" in str(e.value)
        lower, upper = (mid, upper) if small else (lower, mid)
    return upper


# Workspaces below the one that is fastest: five heads of keys in passes of two, two and one or one by one, with parts that are joined, keys and values split before, many sequences of few tokens, a sequence's prompt
PASSES = [([300], [400], 5, 5, 32, 700, True), ([300], [700], 10, 5, 80, 0, True), ([1] * 70, list(range(560, 630)), 15, 5, 24, 1300, True), ([3, 40, 0, 2], [100, 640, 7, 2], 20, 5, 130, 600, False), ([280], [0], 5, 5, 16, 9000, False),
          ([9], [20000], 10, 5, 16, 8500, True)]


@gpu
@pytest.mark.parametrize("counts,lengths,heads,kv_heads,dim,prefix_len,causal", PASSES)
def test_attention_in_smaller_workspaces(hip, counts, lengths, heads, kv_heads, dim, prefix_len, causal):
    import torch
    rng = np.random.default_rng(heads * 1000 + dim + sum(lengths))
    softmax, n, most, group = dec.Softmax(dim=dim), sum(counts), max(lengths), heads // kv_heads
    prefix = Pages(rng, 1, prefix_len, kv_heads, dim, 48) if prefix_len else None
    own = Pages(rng, len(counts), most, kv_heads, dim, 64) if most else None
    q = normal(rng, (n, heads, dim))
    dq, starts, dl, plan = dev(q), dev(np.cumsum([0] + counts)), dev(lengths), Plan(hip, softmax)
    full = hip.lib.zk_i32_attention_workspace(c_uint(n), c_uint(heads), c_uint(kv_heads), c_uint(dim), c_uint(prefix_len), c_uint(len(counts) if own else 0), c_uint(most))
    guard = 4096
    memory = torch.empty(full + guard, dtype=torch.uint8, device="cuda")

    def call(size, p, out=None, shift=None, flag=None):
        return attend(hip, dq, p, prefix, prefix_len, own, len(counts), starts, dl, most, causal, kv_heads, out=out, shift=shift, ws=memory[:size], flag=flag)

    cols = -(-prefix_len // 64) * 64 + -(-most // 64) * 64
    least = smaller_workspaces(hip, n * group * cols * 14 - 1, full, call)
    results = []
    for size in (full, full * 2 // 5 + 4096, (full * 2 // 5 + least) // 2, least * 2 + 4096, least):
        memory.fill_(0x5B)
        flag, shift = new_flag(), torch.full((n, heads), -5, dtype=torch.int64, device="cuda")
        out = host(call(size, plan, shift=shift, flag=flag))
        assert host(flag)[0] == 0 and (host(memory)[size:] == 0x5B).all()
        results.append((out, host(shift)))
    for out, shift in results[1:]:
        assert (out == results[0][0]).all() and (shift == results[0][1]).all()
    at = 0
    for s, count in enumerate(counts):
        for i in range(count):
            if i in (0, 1, 17, 64, count // 2, count - 1) and (len(counts) < 10 or s in (0, 1, 30, 69)):
                seen = 0 if not own else max(0, lengths[s] - count + i + 1) if causal else lengths[s]
                for h in range(heads):
                    keys = [np.zeros((0, dim), np.int64)] * 2
                    for c, m, j in ((prefix, prefix_len, 0), (own, seen, s)):
                        if c:
                            keys = [np.concatenate(p) for p in zip(keys, c.read(j, m, h // group))]
                    exp, sh = dec.attention(q[at, h], keys[0], keys[1], softmax, 1 << 20, 1 << 20)
                    assert (results[0][0][at, h] == exp).all() and results[0][1][at, h] == sh, (s, i, h)
            at += 1


@gpu
@pytest.mark.parametrize("sequences,tokens,heads,kv_heads,dim,prefix_len,most,rows", [
    (1, 2048, 20, 20, 16, 0, 2048, (0, 1000, 2047)), (256, 256, 20, 5, 8, 9000, 64, (0, 100, 255)), (1, 6000, 3, 3, 4, 6000, 6000, (0, 63, 64, 5999)), (1, 3000, 5, 5, 70, 3500, 0, (0, 1500, 2999))])
def test_attention_of_more_heads_than_go_at_a_time(hip, sequences, tokens, heads, kv_heads, dim, prefix_len, most, rows):
    """Passes of eight heads of keys of twenty, three of five, one of three, three of five: one more would take more than 512 MB, or leave units idle"""
    import torch
    rng = np.random.default_rng(tokens)
    softmax, group = dec.Softmax(dim=dim), heads // kv_heads
    prefix = Pages(rng, 1, prefix_len, kv_heads, dim, prefix_len, False) if prefix_len else None
    own = Pages(rng, sequences, most, kv_heads, dim, 64) if most else None
    lengths = rng.integers(1, most + 1, sequences) if sequences > 1 else [most]
    q = normal(rng, (tokens, heads, dim))
    flag, shift = new_flag(), torch.full((tokens, heads), -5, dtype=torch.int64, device="cuda")
    assert hip.lib.zk_i32_attention_workspace(*(c_uint(i) for i in (tokens, heads, kv_heads, dim, prefix_len, sequences, most))) < kv_heads * tokens * group * (prefix_len + most) * 14
    got = host(attend(hip, dev(q), Plan(hip, softmax), prefix, prefix_len, own, sequences, None, dev(lengths), most, True, kv_heads, shift=shift, flag=flag))
    assert host(flag)[0] == 0
    for i in rows:
        s, n = (i, 1) if sequences > 1 else (0, tokens)
        seen = lengths[s] if sequences > 1 else i + 1 if most else 0
        for h in range(heads):
            keys = [np.zeros((0, dim), np.int64)] * 2
            for c, m, j in ((prefix, prefix_len, 0), (own, seen, s)):
                if c:
                    keys = [np.concatenate(p) for p in zip(keys, c.read(j, m, h // group))]
            exp, sh = dec.attention(q[i, h], keys[0], keys[1], softmax, 1 << 20, 1 << 20)
            assert (got[i, h] == exp).all() and host(shift)[i, h] == sh, (i, h)


@gpu
def test_attention_of_many_tokens_without_keys(hip):
    n, heads, dim = 600, 32, 64
    own = Pages(np.random.default_rng(3), 1, 1, heads, dim, 16)
    q = dev(normal(np.random.default_rng(4), (n + 1, heads, dim)))
    for causal in (True, False):
        flag = new_flag()
        out = host(attend(hip, q, Plan(hip, dec.Softmax(dim=dim)), None, 0, own, 1, dev([0, n]), dev([0]), 0, causal, heads, flag=flag))
        assert host(flag)[0] == 0 and (out[:n] == 0).all() and (out[n] == -77).all()


@gpu
@pytest.mark.parametrize("most", [9, 600])
def test_attention_of_as_many_sequences_as_there_are_tiles(hip, most):
    """61680 sequences of a token each, from none to `most` keys: 65535 tiles"""
    rng, n = np.random.default_rng(most), 61680
    softmax = dec.Softmax(dim=3)
    own = Pages(rng, n, most, 1, 3, 16 if most < 16 else most, most < 16)
    lengths, q = rng.integers(0, most + 1, n), normal(rng, (n, 1, 3))
    lengths[[0, n - 1]] = 0, most
    flag = new_flag()
    got = host(attend(hip, dev(q), Plan(hip, softmax), None, 0, own, n, None, dev(lengths), most, True, 1, flag=flag))
    assert host(flag)[0] == 0 and (got[lengths == 0] == 0).all()
    for i in [0, 1, 2, 15, 16, 17, n - 2, n - 1] + rng.integers(0, n, 200).tolist():
        k, v = own.read(i, int(lengths[i]), 0)
        assert (got[i, 0] == dec.attention(q[i, 0], k, v, softmax, 1 << 20, 1 << 20)[0]).all(), i


# ---- weights of 4 bits -----------------------------------------------------------------------------------------------------------------------
class Q4:
    def __init__(self, hip, rng, N, P, group, zeros=True, most=800):
        groups = -(-N // group)
        self.codes = rng.integers(0, 256, (N, (P + 1) // 2)).astype(np.uint8)
        self.scales = rng.integers(-most, most + 1, (groups, P)).astype(np.int32)
        self.zeros = rng.integers(0, 16, (groups, P)).astype(np.uint8) if zeros else None
        self.w = dec.q4_weight(self.codes, self.scales, self.zeros, N, P, group)
        self.hip, self.h = hip, c_void_p()
        codes, scales, zero = dev(self.codes, np.uint8), dev(self.scales), dev(self.zeros, np.uint8)
        hip.call("zk_i32_rhs_prepare_q4", ctypes.byref(self.h), ptr(codes), ptr(scales), ptr(zero), c_uint(N), c_uint(P), c_uint(group), None)

    def __del__(self):
        self.hip.lib.zk_fr_matmul_rhs_free(self.h)


def workspace(hip, weights, rows):
    import torch
    return torch.full((max(16, sum(hip.lib.zk_i32_rhs_workspace(w.h, c_uint(rows)) for w in weights)),), 0x5B, dtype=torch.uint8, device="cuda")


def linear(hip, x, w, rows, N, P, sf=65536, flag=None, ws="caller", stream=None, ldx=None):
    import torch
    out = torch.full((rows + 1, P), -77, dtype=torch.int32, device="cuda")
    ws = workspace(hip, [w], rows) if isinstance(ws, str) else ws
    hip.call("zk_i32_linear", ptr(out), ptr(x), c_size_t(ldx or N), w.h, c_uint(rows), c_uint(sf), ptr(ws), c_size_t(0 if ws is None else ws.numel()), ptr(flag), stream)
    return out


@gpu
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 16, 17, 33, 70, 130])
@pytest.mark.parametrize("N,P,group,zeros,most", [(1, 1, 16, True, 800), (64, 16, 64, False, 800), (63, 17, 16, True, 800), (129, 33, 32, True, 9000), (300, 100, 48, True, 800), (256, 64, 128, False, 2000),
                                                  (1000, 75, 128, True, 557047), (700, 50, 1024, True, 8), (512, 1000, 64, True, 0)])
def test_linear_of_4_bits(hip, rows, N, P, group, zeros, most):
    rng = np.random.default_rng(N * 31 + P + rows)
    w = Q4(hip, rng, N, P, group, zeros, most)
    x = normal(rng, (rows, N), 65536.0 if most < 100000 else 300.0)
    flag = new_flag()
    got = host(linear(hip, dev(x), w, rows, N, P, flag=flag))
    assert host(flag)[0] == 0
    assert (got[:rows] == ref.linear(x, w.w, 65536)).all() and (got[rows:] == -77).all()


@gpu
@pytest.mark.parametrize("rows,sf", [(1, 65536), (3, 1000003), (9, 1 << 20), (40, 77777)])
def test_linear_of_4_bits_on_large_values(hip, rows, sf):
    """inputs of four digits, rows wider than they are long, not at multiples of 16 bytes"""
    rng = np.random.default_rng(rows)
    N, P = 330, 41
    w = Q4(hip, rng, N, P, 64, True, 3)
    wide = rng.integers(-(1 << 31), 0x7F7F7F7F, (rows, N + 3), dtype=np.int64).astype(np.int32)
    flag = new_flag()
    got = host(linear(hip, dev(wide), w, rows, N, P, sf=sf, flag=flag, ldx=N + 3))
    exp = ref.linear(wide[:, :N], w.w, sf)
    assert host(flag)[0] == (RANGE if (np.abs(exp) > 0x7FFFFFFF).any() else 0)
    fits = np.abs(exp) <= 0x7FFFFFFF
    assert fits.mean() > 0.3 and (got[:rows][fits] == exp[fits]).all()


@gpu
@pytest.mark.parametrize("rows,N,P,group,most", [(1, 200, 40, 32, 500), (4, 1000, 130, 128, 500), (6, 129, 17, 16, 500), (16, 500, 300, 64, 500), (32, 512, 96, 128, 40000), (90, 300, 77, 48, 500), (150, 640, 200, 64, 500)])
def test_gated_of_4_bits(hip, rows, N, P, group, most):
    import torch
    rng = np.random.default_rng(N + rows)
    g, u = Q4(hip, rng, N, P, group, True, most if most < 1000 else 500), Q4(hip, rng, N, P, group, False, most)
    low, n = -(1 << 16), 1 << 17
    v = (np.arange(n) + low) / 4096.0
    table = np.round(v / (1 + np.exp(-v)) * 65536).astype(np.int32)
    x = normal(rng, (rows, N), 30000.0)
    out, flag, ws, dx, dt = torch.full((rows + 1, P), -77, dtype=torch.int32, device="cuda"), new_flag(), workspace(hip, [g, u], rows), dev(x), dev(table)
    hip.call("zk_i32_gated", ptr(out), ptr(dx), c_size_t(N), g.h, u.h, c_uint(rows), c_uint(1 << 18), c_uint(1 << 18), ptr(dt), c_int(low), c_uint(n), c_uint(1 << 18), ptr(ws),
             c_size_t(ws.numel()), ptr(flag), None)
    assert host(flag)[0] == 0
    got = host(out)
    assert (got[:rows] == ref.gated(x, g.w, u.w, 1 << 18, 1 << 18, table, low, 1 << 18)).all() and (got[rows:] == -77).all()


def with_four_digits(rng, x):
    """a few inputs of four digits, in the first and last columns as well"""
    rows, n = x.shape
    x[rng.integers(0, rows, 6), rng.integers(0, n, 6)] = rng.integers(-(1 << 29), 1 << 29, 6)
    x[0, 0], x[-1, -1] = 1 << 29, -(1 << 29)
    return x


# Where a workgroup takes two or four strips of 16 columns (from 5105 and 10225 columns), with fewer and more steps than there are buffers; where it has four waves (from 8193 columns) and where the inner
# dimension is more than LDS holds of x at a time (14336 of one row, 7168 of two, 3584 of four); groups of 64 and their multiples, powers of two and none
WIDE_Q4 = [(5, 130, 5201, 64), (16, 1100, 5121, 128), (13, 2300, 5201, 192), (5, 130, 10301, 64), (16, 1100, 10301, 192), (9, 2300, 10240, 128), (17, 130, 10301, 128), (32, 1100, 10301, 64), (32, 2300, 10301, 320),
           (17, 700, 5201, 64), (1, 1100, 8301, 64), (2, 300, 8301, 192), (3, 1100, 8301, 128), (4, 3700, 8301, 64), (1, 14500, 33, 64), (1, 29000, 17, 192), (2, 7300, 33, 128), (2, 14400, 8, 64), (3, 3700, 33, 192),
           (4, 11008, 40, 128), (4, 3585, 16, 64)]


@gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,N,P,group", WIDE_Q4)
def test_linear_of_4_bits_in_every_arrangement(hip, rows, N, P, group, four):
    rng = np.random.default_rng(N * 31 + P + rows)
    w = Q4(hip, rng, N, P, group, True, 8 if four else 400)
    x = normal(rng, (rows, N), 20000.0)
    if four:
        x = with_four_digits(rng, x)
    flag = new_flag()
    got = host(linear(hip, dev(x), w, rows, N, P, flag=flag))
    assert host(flag)[0] == 0
    assert (got[:rows] == ref.linear(x, w.w, 65536)).all() and (got[rows:] == -77).all()


@gpu
@pytest.mark.parametrize("four", [False, True])
@pytest.mark.parametrize("rows,N,P,group", WIDE_Q4[:1] + WIDE_Q4[2:9] + [(2, 300, 8301, 192), (4, 1100, 8301, 64), (1, 14500, 33, 64), (2, 7300, 33, 128), (4, 3700, 40, 192)])
def test_gated_of_4_bits_in_every_arrangement(hip, rows, N, P, group, four):
    import torch
    rng = np.random.default_rng(N + rows + P)
    g, u = Q4(hip, rng, N, P, group, True, 8 if four else 400), Q4(hip, rng, N, P, group, False, 8 if four else 400)
    low = -(1 << 23 if four else 1 << 18)          # eight inputs of four digits in one row reach 8 * 2^29 * 15 * 8 / 2^16
    n = -2 * low
    table = rng.integers(-(1 << 16), 1 << 16, n).astype(np.int32)
    x = normal(rng, (rows, N), 2000.0 if four else 10000.0)
    if four:
        x = with_four_digits(rng, x)
    sf = (1 << 16, 1 << 16, 1 << 10)
    assert (np.abs(ref.linear(x, g.w, sf[0])) < -low).all()
    out, flag, ws, dx, dt = torch.full((rows + 1, P), -77, dtype=torch.int32, device="cuda"), new_flag(), workspace(hip, [g, u], rows), dev(x), dev(table)
    hip.call("zk_i32_gated", ptr(out), ptr(dx), c_size_t(N), g.h, u.h, c_uint(rows), c_uint(sf[0]), c_uint(sf[1]), ptr(dt), c_int(low), c_uint(n), c_uint(sf[2]), ptr(ws), c_size_t(ws.numel()), ptr(flag), None)
    exp = ref.gated(x, g.w, u.w, sf[0], sf[1], table, low, sf[2])
    got = host(out)
    assert host(flag)[0] == 0 and (np.abs(exp) < 1 << 31).all()
    assert (got[:rows] == exp).all() and (got[rows:] == -77).all()


@gpu
def test_4_bits_refusals_with_a_device(hip):
    rng = np.random.default_rng(1)
    h = c_void_p()
    codes, ok = dev(rng.integers(0, 256, (32, 4)), np.uint8), np.ones((2, 8), np.int32)
    for scales, zeros in ((ok * 557048, None), (ok * -557048, None), (ok, np.full((2, 8), 16))):
        ds, dz = dev(scales), dev(zeros, np.uint8)
        with pytest.raises(RuntimeError, match="a scale beyond 557047 or a zero above 15"):
            hip.call("zk_i32_rhs_prepare_q4", ctypes.byref(h), ptr(codes), ptr(ds), ptr(dz), c_uint(32), c_uint(8), c_uint(16), None)
    w, plain = Q4(hip, rng, 32, 8, 16), c_void_p()
    dw = dev(w.w)
    hip.call("zk_i32_rhs_prepare", ctypes.byref(plain), ptr(dw), c_uint(32), c_uint(8), None)
    x, out, flag = dev(np.ones((6, 32))), dev(np.zeros((6, 8))), new_flag()
    for pair in ((w.h, plain), (plain, w.h)):
        with pytest.raises(RuntimeError, match="one weight of 4 bits"):
            hip.call("zk_i32_gated", ptr(out), ptr(x), c_size_t(32), *pair, c_uint(6), c_uint(1), c_uint(1), ptr(x), c_int(0), c_uint(4), c_uint(1), None, c_size_t(0), ptr(flag), None)
    with pytest.raises(RuntimeError, match="zk_i32_linear: the workspace is smaller than zk_i32_rhs_workspace says"):
        hip.call("zk_i32_linear", ptr(out), ptr(x), c_size_t(32), w.h, c_uint(6), c_uint(1), ptr(x), c_size_t(hip.lib.zk_i32_rhs_workspace(w.h, c_uint(6)) - 1), ptr(flag), None)
    path = c_int()
    with pytest.raises(RuntimeError, match="no field elements"):
        hip.call("zk_fr_matmul_rhs", ptr(out), ptr(x), w.h, c_uint(1), c_int(0), ctypes.byref(path), None)
    got = linear(hip, x, w, 6, 32, 8, sf=1, flag=flag, ws=None)      # the library's own memory
    assert (host(got)[:6] == np.ones((6, 32), np.int64) @ w.w).all()
    hip.lib.zk_fr_matmul_rhs_free(plain)


# ---- logits ----------------------------------------------------------------------------------------------------------------------------------
def lists(rows):
    return np.concatenate([np.asarray(r, np.int64).reshape(-1) for r in rows]) if rows else np.zeros(0), np.cumsum([0] + [len(r) for r in rows])


def call_logits(hip, l, history=None, penalties=None, biases=None, mask=None, sf=65536, want="lt", in_place=False, flag=None, ld=None, ws="caller", stream=None, starts=None):
    import torch
    rows, vocab = l.shape
    ld = ld or vocab
    d = torch.full((rows, ld), -(1 << 30), dtype=torch.int32, device="cuda")
    d[:, :vocab] = dev(l)
    out = d if in_place else torch.full((rows, ld), -77, dtype=torch.int32, device="cuda") if "l" in want else None
    token = torch.full((rows,), -9, dtype=torch.int32, device="cuda") if "t" in want else None
    h, hs = lists(history) if history is not None else (None, None)
    bt, bs = lists([[t for t, _ in r] for r in biases]) if biases is not None else (None, None)
    bv = lists([[v for _, v in r] for r in biases])[0] if biases is not None else None
    hs = starts if starts is not None else hs
    words = None
    if mask is not None:
        m = np.zeros((len(mask), (vocab + 31) // 32 * 32), np.uint8)
        m[:, :vocab] = mask
        words = np.packbits(m, axis=1, bitorder="little").view(np.uint32)
    if isinstance(ws, str):
        ws = torch.full((max(16, hip.lib.zk_i32_logits_workspace(c_uint(rows), c_uint(vocab))),), 0x5B, dtype=torch.uint8, device="cuda")
    keep = [dev(a) for a in (h, hs, penalties, bt, bv, bs)] + [dev(words, np.uint32) if words is not None else None]
    dh, dhs, dp, dbt, dbv, dbs, dm = keep
    hip.call("zk_i32_logits", ptr(out), c_size_t(ld), ptr(token), ptr(d), c_size_t(ld), c_uint(rows), c_uint(vocab), ptr(dh), c_uint(0 if h is None else len(h)), ptr(dhs), ptr(dp), ptr(dbt), ptr(dbv),
             c_uint(0 if bt is None else len(bt)), ptr(dbs), ptr(dm), c_size_t(0 if words is None else words.shape[1]), c_uint(0 if words is None else len(words)), c_uint(sf), ptr(ws),
             c_size_t(0 if ws is None else ws.numel()), ptr(flag), stream)
    return (host(out)[:, :vocab] if out is not None else None), (host(token) if token is not None else None), (host(out)[:, vocab:] if out is not None else None)


@gpu
@pytest.mark.parametrize("rows,vocab", [(1, 1), (2, 31), (3, 32), (2, 33), (4, 1000), (1, 4095), (2, 4096), (3, 4097), (2, 8200), (1, 32000), (5, 40001)])
@pytest.mark.parametrize("options", ["", "history", "biases", "mask", "history biases mask", "history biases one mask in place", "history mask wide odd", "history token only"])
def test_logits(hip, rows, vocab, options):
    rng = np.random.default_rng(rows * vocab + len(options))
    sf = 65521 if "odd" in options else 65536
    l = normal(rng, (rows, vocab), 200000.0)
    l[0, vocab // 2] = 0
    l[-1, vocab // 3] = dec.NONE
    history = [rng.integers(0, vocab, int(rng.integers(0, 400))).tolist() + [0, 0, vocab - 1] * (r % 2) for r in range(rows)] if "history" in options else None
    penalties = np.stack([rng.integers(30000, 130000, rows), rng.integers(-3000, 9000, rows), rng.integers(-3000, 60000, rows)], 1) if history is not None else None
    biases = [[(int(t), int(v)) for t, v in zip(rng.integers(0, vocab, n), rng.integers(-(1 << 22), 1 << 22, n))] + [(0, 5), (0, 7)] for n in rng.integers(0, 300, rows)] if "biases" in options else None
    mask = None
    if "mask" in options:
        mask = rng.random((1 if "one" in options else rows, vocab)) < 0.3
        if len(mask) > 1:
            mask[1] = False                         # nothing is left
    flag = new_flag()
    got, token, pad = call_logits(hip, l, history, penalties, biases, mask, sf, "t" if "only" in options else "lt", "in place" in options, flag, vocab + 5 if "wide" in options else None)
    assert host(flag)[0] == 0
    for r in range(rows):
        exp, best = dec.logits(l[r], history[r] if history else [], penalties[r] if history else None, biases[r] if biases else [], None if mask is None else mask[r if len(mask) > 1 else 0], sf)
        assert token[r] == best, r
        if got is not None:
            assert (got[r] == exp).all(), r
    if pad is not None:                             # what lies between rows is left
        assert (pad == (-(1 << 30) if "in place" in options else -77)).all()


@gpu
def test_logits_ties_and_lowest_values(hip):
    """equals go to the lowest token wherever the stretches begin; a logit of the lowest value is none"""
    vocab = 9000
    l = np.full((6, vocab), -5, np.int32)
    l[0, [8999, 4096, 4095]] = 7
    l[1, [8192, 8191]] = 7
    l[2, :] = dec.NONE
    l[3, :] = dec.NONE
    l[3, 8999] = dec.NONE + 1
    l[4, [1, 5000]] = 0x7FFFFFFF
    flag = new_flag()
    got, token, _ = call_logits(hip, l, flag=flag)
    assert host(flag)[0] == 0 and (got == l).all()
    assert token.tolist() == [4095, 8191, -1, 8999, 1, 0]


@gpu
@pytest.mark.parametrize("what,bit", [("token", POSITION), ("negative", POSITION), ("bias", POSITION), ("starts", POSITION), ("behind", POSITION), ("penalty", RANGE), ("high", RANGE), ("low", RANGE), ("sum", RANGE)])
def test_logits_raise_flags(hip, what, bit):
    """and the other row is right"""
    rng = np.random.default_rng(8)
    l = normal(rng, (2, 5000), 200000.0)
    history, penalties, biases = [[3, 3, 4], [4999, 1]], np.array([[80000, 100, 200], [90000, 10, 20]]), [[(3, 9)], [(1, 70), (1, -30)]]
    starts = None
    if what == "token":
        history[0][1] = 5000
    elif what == "negative":
        history[0][1] = -1
    elif what == "bias":
        biases[0][0] = (5000, 9)
    elif what == "starts":
        starts = np.array([-1, 3, 5])
    elif what == "behind":
        starts, history = np.array([9, 8, 8]), [[3, 3, 4], []]
    elif what == "penalty":
        penalties[0, 0] = 0
    elif what == "high":
        l[0, 3], biases[0] = 0x7FFFFFFF, [(3, 1)]
        penalties[0] = [1, 0, 0]
    elif what == "low":
        l[0, 77], biases[0] = dec.NONE + 1, [(77, -1)]
    elif what == "sum":
        biases[0] = [(3, 0x7FFFFFFF)] * 3
    flag = new_flag()
    got, token, _ = call_logits(hip, l, history, penalties, biases, flag=flag, starts=starts)
    assert host(flag)[0] & bit
    if what != "behind":
        exp, best = dec.logits(l[1], history[1], penalties[1], biases[1], None, 65536)
        assert (got[1] == exp).all() and token[1] == best
    if what in ("token", "negative"):               # the entry does not count
        exp, best = dec.logits(l[0], [3, 4], penalties[0], biases[0], None, 65536)
        assert (got[0] == exp).all() and token[0] == best


# ---- a step of many requests, as a program calls it -------------------------------------------------------------------------------------------
E, H, KV, D, HID, V, PRE, MOST, PAGE = 64, 4, 2, 16, 96, 5000, 50, 24, 7


class Model:
    """one block with weights of 4 bits, and a head"""

    def __init__(self, hip, rng):
        self.w = {k: Q4(hip, rng, n, p, 32, True, 400) for k, n, p in (("q", E, H * D), ("k", E, KV * D), ("v", E, KV * D), ("o", H * D, E), ("gate", E, HID), ("up", E, HID), ("down", HID, E), ("head", E, V))}
        self.norm = normal(rng, (3, E), 5000.0) + 65536
        self.emb = normal(rng, (V, E), 50000.0)
        at = np.arange(PRE + MOST)[:, None] * 10000.0 ** (-np.arange(0, D, 2) / D)
        self.angles = np.round(np.stack([np.cos(at), np.sin(at)], -1) * 65536).astype(np.int32)
        v = (np.arange(1 << 17) - (1 << 16)) / 4096.0
        self.act = np.round(v / (1 + np.exp(-v)) * 65536).astype(np.int32)
        self.softmax = dec.Softmax(dim=D)
        self.plan = Plan(hip, self.softmax)
        self.d = {"norm": dev(self.norm), "angles": dev(self.angles), "act": dev(self.act), "emb": dev(self.emb)}


class State:
    def __init__(self, hip, rng, m, S):
        import torch
        self.S, self.m = S, m
        new = lambda *s: torch.zeros(s, dtype=torch.int32, device="cuda")
        self.prefix, self.own = Pages(rng, 1, PRE, KV, D, PRE, False), Pages(rng, S, MOST, KV, D, PAGE)
        self.prefix.k[:], self.prefix.v[:] = normal(rng, self.prefix.k.size, 60000.0), normal(rng, self.prefix.k.size, 60000.0)
        self.prefix.dk.copy_(dev(self.prefix.k)), self.prefix.dv.copy_(dev(self.prefix.v))
        self.lengths_host = rng.integers(0, MOST - 4, S)
        self.lengths, self.positions, self.x, self.flag = dev(self.lengths_host), new(S), new(S, E), new_flag()
        self.n, self.q, self.k, self.v, self.a, self.o, self.h, self.hid, self.l, self.token = new(S, E), new(S, H, D), new(S, KV, D), new(S, KV, D), new(S, H, D), new(S, E), new(S, E), new(S, HID), new(S, V), new(S)
        self.history = [rng.integers(0, V, n).tolist() for n in rng.integers(1, 30, S)]
        h, hs = lists(self.history)
        self.dh, self.dhs, self.pen_host = dev(h), dev(hs), np.tile([80000, 500, 3000], (S, 1))
        self.pen = dev(self.pen_host)
        self.mask_host = rng.random((S, V)) < 0.5
        m_ = np.zeros((S, (V + 31) // 32 * 32), np.uint8)
        m_[:, :V] = self.mask_host
        self.mask = dev(np.packbits(m_, axis=1, bitorder="little").view(np.uint32), np.uint32)
        sizes = [2 * hip.lib.zk_i32_rhs_workspace(w.h, c_uint(S)) for w in m.w.values()] + [hip.lib.zk_i32_logits_workspace(c_uint(S), c_uint(V)),
                 hip.lib.zk_i32_attention_workspace(c_uint(S), c_uint(H), c_uint(KV), c_uint(D), c_uint(PRE), c_uint(S), c_uint(MOST))]
        self.ws = torch.full((max(sizes) + 16,), 0x5B, dtype=torch.uint8, device="cuda")


def step(hip, s, stream):
    """the tokens' rows in x, their lengths (with them) and positions: the block, the head and the next tokens"""
    m, S = s.m, s.S
    st = c_void_p(stream.cuda_stream)
    ws = (ptr(s.ws), c_size_t(s.ws.numel()), ptr(s.flag), st)
    lin = lambda out, x, k, n: hip.call("zk_i32_linear", ptr(out), ptr(x), c_size_t(n), m.w[k].h, c_uint(S), c_uint(65536), *ws)
    norm = lambda h, n, x, b, i: hip.call("zk_i32_residual_norm", ptr(h), ptr(n), None, ptr(x), c_size_t(E), ptr(b), c_size_t(E), None, None, c_uint(0), c_int(65536), c_void_p(m.d["norm"].data_ptr() + 4 * E * i),
                                          c_uint(S), c_uint(E), c_double(1e-5), c_double(65536.0), c_uint(65536), ptr(s.flag), st)
    rope = lambda x, heads: hip.call("zk_i32_rope", ptr(x), c_size_t(heads * D), c_size_t(D), ptr(x), c_size_t(heads * D), c_size_t(D), c_uint(S), c_uint(heads), c_uint(D), c_uint(D), c_int(0),
                                     ptr(m.d["angles"]), c_uint(PRE + MOST), ptr(s.positions), c_uint(0), c_uint(65536), ptr(s.flag), st)
    norm(None, s.n, s.x, None, 0)
    for out, k in ((s.q, "q"), (s.k, "k"), (s.v, "v")):
        lin(out, s.n, k, E)
    rope(s.q, H)
    rope(s.k, KV)
    append(hip, s.own, s.k, s.v, KV, D, S, None, s.lengths, s.flag, st)
    attend(hip, s.q, m.plan, s.prefix, PRE, s.own, S, None, s.lengths, MOST, True, KV, out=s.a, ws=s.ws, flag=s.flag, stream=st)
    lin(s.o, s.a, "o", H * D)
    norm(s.h, s.n, s.x, s.o, 1)
    hip.call("zk_i32_gated", ptr(s.hid), ptr(s.n), c_size_t(E), m.w["gate"].h, m.w["up"].h, c_uint(S), c_uint(1 << 20), c_uint(65536), ptr(m.d["act"]), c_int(-(1 << 16)), c_uint(1 << 17), c_uint(65536), *ws)
    lin(s.o, s.hid, "down", HID)
    norm(None, s.n, s.h, s.o, 2)
    lin(s.l, s.n, "head", E)
    hip.call("zk_i32_logits", ptr(s.l), c_size_t(V), ptr(s.token), ptr(s.l), c_size_t(V), c_uint(S), c_uint(V), ptr(s.dh), c_uint(s.dh.numel()), ptr(s.dhs), ptr(s.pen), None, None, c_uint(0), None,
             ptr(s.mask), c_size_t(s.mask.shape[1]), c_uint(S), c_uint(65536), *ws)


def step_expected(s, x):
    m, S = s.m, s.S
    n = ref.residual_norm(x, w=m.norm[0])[1]
    q, k, v = (ref.linear(n, m.w[i].w, 65536) for i in "qkv")
    at = PRE + s.lengths_host - 1
    q, k = ref.rope(q.reshape(S, H, D), m.angles, at, D, 0, 65536), ref.rope(k.reshape(S, KV, D), m.angles, at, D, 0, 65536)
    for i in range(S):
        for h in range(KV):
            s.own.put(i, int(s.lengths_host[i]) - 1, h, k[i, h], v.reshape(S, KV, D)[i, h])
    a, _ = expected(q, m.softmax, s.prefix, PRE, s.own, [1] * S, [int(i) for i in s.lengths_host], True, KV)
    h, n, _ = ref.residual_norm(x, ref.linear(a.reshape(S, H * D), m.w["o"].w, 65536), w=m.norm[1])
    hid = ref.gated(n, m.w["gate"].w, m.w["up"].w, 1 << 20, 65536, m.act, -(1 << 16), 65536)
    n = ref.residual_norm(h, ref.linear(hid, m.w["down"].w, 65536), w=m.norm[2])[1]
    l = ref.linear(n, m.w["head"].w, 65536)
    rows = [dec.logits(l[i], s.history[i], s.pen_host[i], [], s.mask_host[i], 65536) for i in range(S)]
    return np.stack([r[0] for r in rows]), np.array([r[1] for r in rows])


@gpu
@pytest.mark.parametrize("S", [1, 5, 20])
def test_steps_eager_and_captured(hip, S):
    """Two sets of requests with workspaces of their own, some steps each: eager on a side stream, then as graphs replayed in turn as their sequences grow, eager work in between"""
    import torch
    rng = np.random.default_rng(S)
    m = Model(hip, rng)
    states, stream = [State(hip, rng, m, S) for _ in range(2)], torch.cuda.Stream()

    def begin(s):
        s.lengths_host = s.lengths_host + 1
        tokens = rng.integers(0, V, S)
        s.lengths.copy_(dev(s.lengths_host)), s.positions.copy_(dev(PRE + s.lengths_host - 1)), s.x.copy_(dev(m.emb[tokens]))
        torch.cuda.synchronize()
        return m.emb[tokens]

    def check(s, x):
        l, token = step_expected(s, x)
        assert host(s.flag)[0] == 0
        assert (host(s.own.dk) == s.own.k).all() and (host(s.own.dv) == s.own.v).all()
        assert (host(s.l) == l).all() and (host(s.token) == token).all()

    x = begin(states[0])
    step(hip, s=states[0], stream=stream)
    check(states[0], x)
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            step(hip, s, stream)
        graphs.append(g)
    for turn in range(3):
        xs = [begin(s) for s in states]
        for g in graphs:
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        for s, x in zip(states, xs):
            check(s, x)
        step(hip, states[turn % 2], torch.cuda.current_stream())      # the same step again: nothing is left over from the first
        check(states[turn % 2], xs[turn % 2])


@gpu
def test_captured_calls_need_their_own_memory(hip):
    import torch
    rng = np.random.default_rng(2)
    plan, own, w = Plan(hip, dec.Softmax(dim=8)), Pages(rng, 1, 3000, 1, 8, 16), Q4(hip, rng, 64, 16, 32)
    q, lengths, l = dev(normal(rng, (1, 1, 8))), dev([3000]), normal(rng, (1, 5000))
    stream, g, flag = torch.cuda.Stream(), torch.cuda.CUDAGraph(), new_flag()
    x, out, dl = dev(normal(rng, (6, 64))), dev(np.zeros((6, 16))), dev(l)
    oc = own.c()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=stream):
        st, texts = c_void_p(stream.cuda_stream), []

        def refused(name, *args):
            rc = getattr(hip.lib, name)(*args)
            texts.append((name, rc, hip.lib.zk_last_error()))

        for f, ws in ((None, dl), (flag, None)):
            refused("zk_i32_attention", ptr(q), c_size_t(8), c_size_t(8), ptr(q), c_size_t(8), c_size_t(8), c_uint(1), c_uint(1), c_uint(1), c_uint(8), plan.h, None, c_uint(0), ctypes.byref(oc), c_uint(1), None,
                    ptr(lengths), c_uint(3000), c_int(1), c_uint(1), c_uint(1), None, ptr(ws), c_size_t(1 << 20 if ws is not None else 0), ptr(f), st)
            refused("zk_i32_linear", ptr(out), ptr(x), c_size_t(64), w.h, c_uint(6), c_uint(1), ptr(ws), c_size_t(1 << 20 if ws is not None else 0), ptr(f), st)
            refused("zk_i32_logits", ptr(dl), c_size_t(5000), ptr(out), ptr(dl), c_size_t(5000), c_uint(1), c_uint(5000), None, c_uint(0), None, None, None, None, c_uint(0), None, None, c_size_t(0), c_uint(0),
                    c_uint(1), ptr(ws), c_size_t(1 << 20 if ws is not None else 0), ptr(f), st)
        refused("zk_i32_cache_append", ctypes.byref(oc), ptr(q), c_size_t(8), c_size_t(8), ptr(q), c_size_t(8), c_size_t(8), c_uint(1), c_uint(1), c_uint(8), c_uint(1), None, ptr(lengths), None, st)
        h = c_void_p()
        refused("zk_i32_softmax_prepare", ctypes.byref(h), (c_uint * 2)(4, 4), c_int(2), c_int(1), c_int(0), c_double(4.0), (c_double * 1)(4.0), c_uint(8), st)
        refused("zk_i32_rhs_prepare_q4", ctypes.byref(h), ptr(x), ptr(x), None, c_uint(16), c_uint(4), c_uint(16), st)
    for name, rc, text in texts:
        assert rc == 10001 and name.encode() in text and b"a captured call needs" in text, (name, rc, text)


# ---- refusals: nothing here reaches a device ------------------------------------------------------------------------------------------------------
W = (ctypes.c_int32 * 64)()


def refused(name, args, text):
    from gpuhelp import pkg
    lib = pkg.load_hip()
    assert getattr(lib, name)(*args) == 10001
    assert text in lib.zk_last_error().decode()


def a_cache(**change):
    a = dict(k=ctypes.addressof(W), v=ctypes.addressof(W), page_stride=64, token_stride=8, head_stride=4, page_size=8, pages=4, page_table=None, table_cols=0) | change
    return Cache(**a)


CACHES = [({"k": None}, "without keys"), ({"v": None}, "without keys"), ({"page_size": 0}, "without pages"), ({"pages": 0}, "without pages"), ({"page_size": 1}, "fewer places"), ({"pages": 1}, "fewer places"),
          ({"page_table": ctypes.addressof(W)}, "fewer places"), ({"token_stride": 3}, "heads overlap"), ({"head_stride": 3}, "heads overlap"), ({"token_stride": 7}, "heads overlap"),
          ({"page_stride": 63}, "pages overlap")]


@pytest.mark.parametrize("change,text", [c for c in CACHES if c[0] != {"page_size": 1}] + [({"cache": None}, "null argument"), ({"k": None, "argument": 1}, "null argument"), ({"lengths": None}, "null argument"),
                                                                                        ({"sequences": 0}, "no sequences"), ({"tokens": 3}, "divide among"), ({"dim": 0}, "empty heads")])
def test_append_refusals(change, text):
    change = dict(change)
    arg = {"cache": 0, "lengths": W, "sequences": 2, "tokens": 2, "dim": 4} | {k: v for k, v in change.items() if k in ("cache", "lengths", "sequences", "tokens", "dim")}
    k = None if change.pop("argument", None) else W
    c = a_cache(**({} if k is None else {x: v for x, v in change.items() if x not in arg}))
    refused("zk_i32_cache_append", [None if arg["cache"] is None else ctypes.byref(c), k, c_size_t(8), c_size_t(4), W, c_size_t(8), c_size_t(4), c_uint(arg["tokens"]), c_uint(2), c_uint(arg["dim"]),
                                    c_uint(arg["sequences"]), None, arg["lengths"], W, None], text)


@pytest.mark.parametrize("args,text", [
    ((None, 3, 1, 0, 4.0, (4.0, 4.0), 8), "null argument"), (((4, 4, 4), 0, 0, 0, 4.0, (4.0,), 8), "1 to 8 digits"), (((4,) * 9, 9, 1, 0, 4.0, (4.0,) * 8, 8), "1 to 8 digits"),
    (((4, 4, 4), 3, 2, 1, 4.0, (4.0,), 8), "at least one"), (((4, 4, 4), 3, -1, 0, 4.0, (4.0,), 8), "1 to 8 digits"), (((4, 4, 4), 3, 1, 0, 0.5, (4.0, 4.0), 8), "scaling factor"),
    (((4, 4, 4), 3, 1, 0, float("nan"), (4.0, 4.0), 8), "scaling factor"), (((4, 0, 4), 3, 1, 0, 4.0, (4.0, 4.0), 8), "a radix"), (((4, (1 << 28) + 1, 4), 3, 1, 0, 4.0, (4.0, 4.0), 8), "a radix"),
    (((1 << 28, 1 << 28, 1 << 8), 3, 1, 0, 4.0, (4.0, 4.0), 8), "2^63"), (((4, 4, 4), 3, 1, 0, 4.0, (0.0, 4.0), 8), "a factor of the exponentials"),
    (((4, 4, 4), 3, 1, 0, 4.0, (float("nan"), 4.0), 8), "a factor of the exponentials"), (((4, 4, 4), 3, 1, 0, 4.0, (2147483647.0, 4.0), 8), "a factor of the exponentials"),
    (((4, 4, 4), 3, 1, 0, 4.0, (1e7, 2e7), 8), "1.4e14"), (((4, 4, 4), 3, 1, 0, 4.0, (4.0, 4.0), 0), "empty heads")])
def test_softmax_refusals(args, text):
    bs, K, L, M, sf, thetas, dim = args
    h = c_void_p()
    refused("zk_i32_softmax_prepare", [ctypes.byref(h), None if bs is None else (c_uint * len(bs))(*bs), c_int(K), c_int(L), c_int(M), c_double(sf), (c_double * len(thetas))(*thetas), c_uint(dim), None], text)


ATTENTION_REFUSALS = [
    ({"out": None}, "null argument"), ({"q": None}, "null argument"), ({"plan": None}, "null argument"), ({}, "another width"), ({"dim": 0}, "heads of 1 to 256"), ({"kv_heads": 0}, "divide among"),
    ({"kv_heads": 3}, "divide among"), ({"heads": 65536 * 2, "kv_heads": 65536 * 2}, "65535 heads"), ({"tokens": (1 << 20) + 1, "seqs": 1}, "2^20 queries"), ({"most": (1 << 24) + 1}, "2^24 keys"),
    ({"own": None, "most": 0}, "neither a prefix"), ({"own": None, "prefix_len": 4}, "neither a prefix"), ({"prefix_len": 4}, "no prefix"), ({"seqs": 0}, "need lengths"), ({"lengths": None}, "need lengths"),
    ({"own": None, "prefix": {}, "prefix_len": 4}, "own keys without"), ({"tokens": 5}, "divide among"), ({"sf": (0, 1)}, "factor of 0"), ({"sf": (1, 0)}, "factor of 0"), ({"q": "out", "q_token": 12}, "in place"),
    ({"out_token": 3}, "heads overlap"), ({"out_head": 3}, "heads overlap"), ({"out_token": 7}, "output's heads overlap"), ({"prefix": {"page_size": 3}, "prefix_len": 4}, "fewer places"),
    ({"own": {"page_size": 3}}, "fewer places"), ({"own": {"k": None}}, "without keys"), ({"own": {"page_stride": 63}}, "pages overlap"), ({"bytes": 5, "workspace": 16, "most": 5000, "own": {"page_size": 5000, "page_stride": 40000}}, "the workspace is smaller"),
    ({"bytes": 1 << 30, "workspace": 8}, "multiple of 16")]


@pytest.mark.parametrize("change,text", ATTENTION_REFUSALS)
def test_attention_refusals(change, text):
    plan = (ctypes.c_char * 4096)()                 # a handle for heads of no elements: a call that nothing else refuses ends at that
    other = (ctypes.c_int32 * 64)()
    a = dict(out=other, q=W, out_token=8, out_head=4, q_token=8, q_head=4, tokens=4, heads=2, kv_heads=2, dim=4, plan=plan, prefix=None, prefix_len=0, own={}, seqs=2, lengths=W, most=8, sf=(1, 1), workspace=None,
             bytes=0) | change
    if a["q"] == "out":
        a["q"] = a["out"]
    pc, oc = (None if a[k] is None else a_cache(**a[k]) for k in ("prefix", "own"))
    refused("zk_i32_attention", [a["out"], c_size_t(a["out_token"]), c_size_t(a["out_head"]), a["q"], c_size_t(a["q_token"]), c_size_t(a["q_head"]), c_uint(a["tokens"]), c_uint(a["heads"]), c_uint(a["kv_heads"]),
                                 c_uint(a["dim"]), a["plan"], None if pc is None else ctypes.byref(pc), c_uint(a["prefix_len"]), None if oc is None else ctypes.byref(oc), c_uint(a["seqs"]), None, a["lengths"],
                                 c_uint(a["most"]), c_int(1), c_uint(a["sf"][0]), c_uint(a["sf"][1]), None, c_void_p(a["workspace"]), c_size_t(a["bytes"]), W, None], text)


def test_attention_workspace_of_the_longest_caches():
    """Keys and values are split once for many rows as long as a launch can have as many workgroups"""
    from gpuhelp import pkg
    workspace_of, most = pkg.load_hip().zk_i32_attention_workspace, 65535 * 64
    workspace_of.restype = c_size_t
    size = [workspace_of(c_uint(256), c_uint(1), c_uint(1), c_uint(128), c_uint(keys), c_uint(0), c_uint(0)) for keys in (most, most + 64, 1 << 24)]
    # a key's row of scores and weights: 256 x 14 bytes, its digits: 128 x 8; parts of 8192 keys, one more for the longest by each as many
    assert size[0] >= most * (256 * 14 + 128 * 8) > size[1] >= (most + 64) * 256 * 14 and size[2] >= (1 << 24) * 256 * 14


def attention_takes(tokens, heads, kv_heads, dim, prefix_len, sequences, most, size):
    """whether zk_i32_attention takes a workspace of that size: a handle for heads of no elements is what it is refused for then"""
    from gpuhelp import pkg
    lib = pkg.load_hip()
    plan, other = (ctypes.c_char * 4096)(), (ctypes.c_int32 * 64)()
    caches = [Cache(ctypes.addressof(W), ctypes.addressof(W), kv_heads * dim << 24, kv_heads * dim, dim, 1 << 24, 1 << 21, None, 0) for _ in range(2)]
    rc = lib.zk_i32_attention(other, c_size_t(heads * dim), c_size_t(dim), W, c_size_t(heads * dim), c_size_t(dim), c_uint(tokens), c_uint(heads), c_uint(kv_heads), c_uint(dim), plan,
                              ctypes.byref(caches[0]) if prefix_len else None, c_uint(prefix_len), ctypes.byref(caches[1]) if sequences else None, c_uint(sequences), W, W, c_uint(most), c_int(1), c_uint(1),
                              c_uint(1), None, c_void_p(1 << 20), c_size_t(size), W, None)
    text = lib.zk_last_error().decode()
    assert rc == 10001 and any(i in text for i in ("another width", "the workspace is smaller", "65535 tiles")), text
    return "another width" in text


def attention_workspace(*sizes):
    from gpuhelp import pkg
    f = pkg.load_hip().zk_i32_attention_workspace
    f.restype = c_size_t
    return f(*(c_uint(i) for i in sizes))


@pytest.mark.parametrize("tokens,group,sequences,prefix_len,most,takes", [
    (61680, 1, 61680, 0, 100, True), (61681, 1, 61681, 0, 100, False), (7710 * 4, 32, 3855, 50, 9, True), (1 << 20, 1, 1, 0, 700, True), (1 << 20, 1, 31775, 0, 700, True), (1 << 20, 1, 31776, 0, 700, False),
    (1 << 20, 1, 31774, 0, 700, True), (65535 * 16 - 1, 1, 1, 0, 0, True), (65535 * 16, 1, 1, 0, 0, False), (65534 * 16 + 15, 1, 1, 0, 0, True), (1 << 20, 1, 0, 700, 0, True), (1 << 18, 4, 1, 0, 0, False), (1 << 18, 4, 1, 0, 9, True)])
def test_attention_takes_65535_tiles(tokens, group, sequences, prefix_len, most, takes):
    """of 16 or 64 queries, by the average of a sequence's queries and whether there are keys"""
    queries = tokens * group
    tiles = queries // (64 if most and queries // sequences > 32 else 16) + sequences if sequences else 0
    assert (tiles <= 65535) == takes
    assert attention_takes(tokens, group, 1, 16, prefix_len, sequences, most, 1 << 50) == takes


def test_a_workspace_serves_every_smaller_call():
    """tokens, sequences and both numbers of keys below those that a workspace was asked for, which may take more by itself: more parts, or keys split before"""
    import random
    rng = random.Random(1)
    log = lambda most: int(2 ** rng.uniform(0, np.log2(most + 1)))
    more = 0
    for _ in range(1500):
        kv_heads, dim, group = rng.choice([1, 2, 8, 32]), rng.choice([1, 16, 64, 80, 128, 200, 256]), rng.choice([1, 4, 5])
        tokens, prefix_len, most = log(5000), rng.choice([0, log(1 << 17), log(3000)]), rng.choice([0, log(1 << 17), log(3000)])
        sequences = rng.choice([1, min(tokens, log(300)), tokens]) if most or prefix_len == 0 else rng.choice([0, 1, tokens])
        large = (tokens, group * kv_heads, kv_heads, dim, prefix_len, sequences, most)
        size = attention_workspace(*large)
        assert attention_takes(*large, size)
        cols = (prefix_len + 63) // 64 * 64 + (most + 63) // 64 * 64
        if size:
            assert not attention_takes(*large, tokens * group * cols * 14)
        for _ in range(6):
            t, p, m = rng.choice([tokens, rng.randint(1, tokens)]), rng.choice([prefix_len, rng.randint(0, prefix_len)]), rng.choice([most, rng.randint(0, most)])
            s = rng.choice([sequences, rng.randint(0, sequences)])
            if s == 0:
                m = 0
                if p == 0:
                    continue
            small = (t, group * kv_heads, kv_heads, dim, p, s, m)
            assert attention_takes(*small, size), (large, small)
            more += attention_workspace(*small) > size
    assert more > 20                                # some of them would be faster with more


@pytest.mark.parametrize("large,small", [((33, 32, 8, 128, 8192, 33, 512), (32, 32, 8, 128, 8192, 32, 512)), ((599, 32, 32, 128, 0, 1, 16000), (260, 32, 32, 128, 0, 1, 16000)),
                                         ((256, 1, 1, 128, 65535 * 64 + 64, 0, 0), (256, 1, 1, 128, 65535 * 64, 0, 0)), ((256, 1, 1, 128, 1 << 24, 1, 1 << 24), (256, 1, 1, 128, 65535 * 64, 1, 65535 * 64))])
def test_a_workspace_serves_a_smaller_call_that_has_more(large, small):
    assert attention_workspace(*large) < attention_workspace(*small) or large[4] == 1 << 24
    assert attention_takes(*small, attention_workspace(*large))


@pytest.mark.parametrize("sizes", [(2048, 32, 32, 128, 0, 1, 2048), (260, 32, 32, 128, 0, 1, 16000), (300, 32, 8, 256, 30000, 1, 30000), (64, 32, 8, 128, 8192, 64, 4096)])
def test_a_workspace_of_more_than_one_head_stays_within_512_mb(sizes):
    tokens, heads, kv_heads, dim, prefix_len, sequences, most = sizes
    size, one = attention_workspace(*sizes), attention_workspace(tokens, heads // kv_heads, 1, dim, prefix_len, sequences, most)
    assert size <= max(512 << 20, one + 64)


def test_q4_refusals():
    h = c_void_p()
    for codes, scales, n, p, g, text in ((None, W, 2, 2, 16, "null argument"), (W, None, 2, 2, 16, "null argument"), (W, W, 0, 2, 16, "empty matrix"), (W, W, 2, 0, 16, "empty matrix"), (W, W, 43691, 1, 16, "above 43690"),
                                         (W, W, 1, (1 << 22) + 1, 16, "4194304 columns"), (W, W, 2, 2, 0, "multiples of 16"), (W, W, 2, 2, 8, "multiples of 16"), (W, W, 2, 2, 40, "multiples of 16")):
        refused("zk_i32_rhs_prepare_q4", [ctypes.byref(h), codes, scales, None, c_uint(n), c_uint(p), c_uint(g), None], text)


@pytest.mark.parametrize("change,text", [
    ({"logits": None}, "null logits"), ({"out": None, "token": None}, "no output"), ({"vocab": 0}, "no tokens"), ({"ld": 9}, "rows overlap"), ({"ld_out": 9}, "rows overlap"), ({"vocab": (1 << 30) + 1}, "2^30 tokens"),
    ({"rows": 65536}, "65535 rows"), ({"out": "logits", "ld": 12}, "in place"), ({"history_starts": W}, "a history needs"), ({"history_starts": W, "history": W}, "a history needs"),
    ({"history": W}, "without starts"), ({"penalties": W}, "without starts"), ({"bias_starts": W, "bias_len": 3}, "biases need"), ({"bias_tokens": W}, "biases without starts"), ({"mask": W}, "a mask has"),
    ({"mask": W, "mask_rows": 2}, "a mask has"), ({"mask_rows": 1}, "a mask has"), ({"mask": W, "mask_rows": 3, "ld_mask": 0}, "a mask has"), ({"sf": 0}, "a scaling factor of 0"), ({"sf": 1 << 31}, "2^31 and more"),
    ({"bytes": 5, "workspace": 16, "vocab": 5000, "ld": 5000, "ld_out": 5000}, "the workspace is smaller"), ({"bytes": 64, "workspace": 8}, "multiple of 16"),
    ({"history_starts": W, "history": W, "penalties": W, "history_len": 1 << 31}, "2^31 - 1")])
def test_logits_refusals(change, text):
    other = (ctypes.c_int32 * 64)()
    a = dict(out=other, ld_out=10, token=W, logits=W, ld=10, rows=3, vocab=10, history=None, history_len=0, history_starts=None, penalties=None, bias_tokens=None, bias_values=None, bias_len=0, bias_starts=None,
             mask=None, ld_mask=1, mask_rows=0, sf=1, workspace=None, bytes=0) | change
    if a["out"] == "logits":
        a["out"] = a["logits"]
    refused("zk_i32_logits", [a["out"], c_size_t(a["ld_out"]), a["token"], a["logits"], c_size_t(a["ld"]), c_uint(a["rows"]), c_uint(a["vocab"]), a["history"], c_uint(a["history_len"]), a["history_starts"],
                              a["penalties"], a["bias_tokens"], a["bias_values"], c_uint(a["bias_len"]), a["bias_starts"], a["mask"], c_size_t(a["ld_mask"]), c_uint(a["mask_rows"]), c_uint(a["sf"]),
                              c_void_p(a["workspace"]), c_size_t(a["bytes"]), W, None], text)


def test_no_tokens_is_no_error():
    from gpuhelp import pkg
    lib = pkg.load_hip()
    assert lib.zk_i32_cache_append(None, None, c_size_t(0), c_size_t(0), None, c_size_t(0), c_size_t(0), c_uint(0), c_uint(1), c_uint(4), c_uint(1), None, None, None, None) == 0
    assert lib.zk_i32_logits(None, c_size_t(0), None, None, c_size_t(0), c_uint(0), c_uint(4), None, c_uint(0), None, None, None, None, c_uint(0), None, None, c_size_t(0), c_uint(0), c_uint(1), None, c_size_t(0),
                             None, None) == 0
    assert lib.zk_i32_attention(None, c_size_t(0), c_size_t(0), None, c_size_t(0), c_size_t(0), c_uint(0), c_uint(1), c_uint(1), c_uint(4), None, None, c_uint(0), None, c_uint(0), None, None, c_uint(0), c_int(0),
                                c_uint(1), c_uint(1), None, None, c_size_t(0), None, None) == 0
    assert lib.zk_i32_softmax_free(None) == 0

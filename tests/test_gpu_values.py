"""A decoder layer's values without their witness (zk_i32_*, zk_fr_rope): whole numbers, so every comparison with the 64-bit restatement is for equality."""
import ctypes

import numpy as np
import pytest

import valueshelp as ref

c_void_p, c_size_t, c_int, c_uint, c_double = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint32, ctypes.c_double
gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def hip():
    from gpuhelp import Hip
    return Hip()


class Dev:
    """device copies of arrays that live until the object goes"""

    def __init__(self, hip):
        self.hip, self.held = hip, []

    def up(self, a, dtype=np.int32):
        if a is None:
            return c_void_p(None)
        self.held.append(self.hip.upload(np.ascontiguousarray(a, dtype=dtype)))
        return c_void_p(self.held[-1])

    def space(self, nbytes, fill=0x5A):
        self.held.append(self.hip.malloc(max(nbytes, 16)))
        self.hip.call("zk_memset", c_void_p(self.held[-1]), c_int(fill), c_size_t(max(nbytes, 16)), None)
        return c_void_p(self.held[-1])

    def down(self, p, shape, dtype=np.int32):
        return self.hip.download(p.value, shape, dtype)

    def flag(self):
        return self.space(4, 0)

    def free(self):
        self.hip.sync()
        for p in self.held:
            self.hip.free(p)


@pytest.fixture
def dev(hip):
    d = Dev(hip)
    yield d
    d.free()


def normal(rng, shape, std=65536.0, most=1 << 24):
    return np.clip(np.round(rng.normal(0, std, shape)), -most, most).astype(np.int32)


# ---- norms with the residual stream ------------------------------------------------------------------------------------------------------------
def call_norm(hip, dev, x, b=None, post=None, gate=None, res=65536, w=None, eps=1e-5, scale=65536.0, sf=65536, ldx=None, ldb=None, want="hnr", flag=None, stream=None, into=None):
    rows, cols = x.shape

    def strided(a, ld):
        if a is None or ld is None:
            return a
        wide = np.full((a.shape[0], ld), 12345678, np.int32)
        wide[:, :cols] = a
        return wide

    px, pb = dev.up(strided(x, ldx)), dev.up(strided(b, ldb))
    out = {k: dev.space(4 * rows * (1 if k == "r" else cols)) if k in want else c_void_p(None) for k in "hnr"}
    if into:
        out.update({k: px if v == "x" else pb for k, v in into.items()})
    f = dev.flag() if flag is None else flag
    hip.call("zk_i32_residual_norm", out["h"], out["n"], out["r"], px, c_size_t(ldx or cols), pb, c_size_t(ldb or cols), dev.up(post), dev.up(gate), c_uint(0 if gate is None else len(gate)),
             c_int(res), dev.up(w), c_uint(rows), c_uint(cols), c_double(eps), c_double(scale), c_uint(sf), f, stream)
    hip.sync()
    got = {k: dev.down(out[k], (rows,) if k == "r" else (rows, cols)) for k in "hnr" if out[k].value}
    return got, int(dev.down(f, (1,), np.uint32)[0]) if f.value else 0


def same(got, h, n, r):
    for k, e in zip("hnr", (h, n, r)):
        if k in got:
            assert (got[k].astype(np.int64) == e).all(), k


# one column, one row; rows below, at and above a wave's, a workgroup's and the register path's widths; odd widths
@gpu
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (1, 64), (5, 63), (2, 100), (7, 257), (4, 1000), (3, 1024), (2, 1025), (1, 4096), (3, 4097), (2, 8192), (1, 11008), (2, 16384), (1, 16388), (2, 20001)])
@pytest.mark.parametrize("options", ["", "b", "post gate"])
def test_norm_sizes(hip, dev, rows, cols, options):
    rng = np.random.default_rng(rows * 100003 + cols)
    x, w = normal(rng, (rows, cols)), normal(rng, cols, 6000.0) + 65536
    b = normal(rng, (rows, cols), 30000.0) if options else None
    post = normal(rng, cols, 6000.0) + 65536 if "post" in options else None
    gate = normal(rng, (rows, cols), 30000.0) if "gate" in options else None
    res = 46341 if "gate" in options else 65536
    got, flag = call_norm(hip, dev, x, b, post, gate, res, w)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, post, gate, res, w))


# Prompts: the kernel whose stores go past the caches (512 rows and more of 1025 to 4096 aligned columns), with every option, in the inputs' place, rows whose sums round among the others
@gpu
@pytest.mark.parametrize("rows,cols", [(512, 1028), (700, 2052), (513, 4096)])
@pytest.mark.parametrize("options", ["", "b", "post gate", "post gate in place"])
@pytest.mark.parametrize("sf", [65536, 65521])
def test_norm_of_prompts(hip, dev, rows, cols, options, sf):
    rng = np.random.default_rng(rows + sf)
    x, w = normal(rng, (rows, cols)), normal(rng, cols, 6000.0) + 65536
    b = normal(rng, (rows, cols), 30000.0) if options else None
    post = normal(rng, cols, 6000.0) + 65536 if "post" in options else None
    gate = normal(rng, ({512: 32, 700: 20, 513: 27}[rows], cols), 30000.0) if "gate" in options else None
    for at in ((0, 0), (rows // 2, 7), (rows - 1, cols - 1)):
        x[at] = 2000 * 65536
    x[3, 1:9] = -1500 * 65536
    if post is not None:
        b[5, 6] = b[rows - 2, cols - 4] = 1800 * 65536
    got, flag = call_norm(hip, dev, x, b, post, gate, 46341, w, sf=sf, into={"h": "x", "n": "b"} if "in place" in options else None)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, post, gate, 46341, w, sf=sf))


# as many rows through each of the other kernels: one column a lane and four, more of either, rows too long for registers
@gpu
@pytest.mark.parametrize("cols", [1021, 1024, 1030, 5120, 8192, 16390])
def test_norm_of_prompts_of_other_widths(hip, dev, cols):
    rng = np.random.default_rng(cols)
    x, b, w, post, gate = normal(rng, (512, cols)), normal(rng, (512, cols), 30000.0), normal(rng, cols, 6000.0) + 65536, normal(rng, cols, 6000.0) + 65536, normal(rng, (16, cols), 30000.0)
    x[100, cols // 2] = 2000 * 65536
    got, flag = call_norm(hip, dev, x, b, post, gate, 46341, w)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, post, gate, 46341, w))


# rows whose squares pass 2^53: the sum is then the one in index order, rounding and all
@gpu
@pytest.mark.parametrize("cols", [7, 300, 4096, 5000, 17000])
@pytest.mark.parametrize("scale", [65536.0, 1000.0, 0.75])
def test_norm_sums_that_round(hip, dev, cols, scale):
    rng = np.random.default_rng(cols)
    x = normal(rng, (6, cols))
    x[1, cols // 3] = (1 << 31) - 1
    x[2, cols // 2] = -(1 << 31)
    x[3] = rng.integers(-(1 << 28), 1 << 28, cols)
    x[4] = 0
    w = np.full(cols, 3, np.int32)
    got, flag = call_norm(hip, dev, x, w=w, scale=scale, eps=1e-3)
    assert flag == 0
    same(got, *ref.residual_norm(x, w=w, scale=scale, eps=1e-3))


@gpu
@pytest.mark.parametrize("sf", [1, 2, 3, 1000, 65536, (1 << 31) + 1, (1 << 32) - 1])
@pytest.mark.parametrize("cols", [129, 520])
def test_norm_scaling_factors(hip, dev, sf, cols):
    rng = np.random.default_rng(sf % 1000 + cols)
    std, scale = (3.0, 4.0) if sf < 1000 else (20000.0, 65536.0)
    x, b, w = normal(rng, (4, cols), std), normal(rng, (4, cols), std), normal(rng, cols, std)
    gate = normal(rng, (2, cols), std)
    got, flag = call_norm(hip, dev, x, b, None, gate, 2, w, sf=sf, scale=scale, eps=0.5)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, None, gate, 2, w, sf=sf, scale=scale, eps=0.5))


@gpu
@pytest.mark.parametrize("want", ["h", "n", "r", "hn", "nr"])
@pytest.mark.parametrize("cols", [96, 18000])
def test_norm_outputs_left_out(hip, dev, want, cols):
    rng = np.random.default_rng(5)
    x, b, w = normal(rng, (3, cols)), normal(rng, (3, cols)), normal(rng, cols)
    got, flag = call_norm(hip, dev, x, b, w=w if "n" in want else None, want=want)
    assert flag == 0 and set(got) == set(want)
    same(got, *ref.residual_norm(x, b, w=w))


@gpu
def test_norm_of_more_rows_than_a_launch_takes(hip, dev):
    rows = 2 * ((1 << 20) + 3)
    rng = np.random.default_rng(1)
    x, b, w, gate = normal(rng, (rows, 2)), normal(rng, (rows, 2)), normal(rng, 2), normal(rng, (rows // 2, 2))
    got, flag = call_norm(hip, dev, x, b, None, gate, 65536, w)
    h = x.astype(np.int64) + ref.quotient(np.repeat(gate.astype(np.int64), 2, 0) * b, 65536)
    r = np.rint(1.0 / np.sqrt((h.astype(np.float64) / 65536) [:, 0] ** 2 / 2 + (h.astype(np.float64) / 65536)[:, 1] ** 2 / 2 + 1e-5) * 65536)      # two squares below 2^50: no sum rounds
    assert flag == 0 and (got["h"] == h).all() and (np.abs(got["r"] - r) <= 1).all()
    some = np.concatenate([np.arange(5), np.arange((1 << 20) - 3, (1 << 20) + 3), np.arange(rows - 5, rows)])
    exp = ref.residual_norm(h[some], w=w)
    assert (got["n"][some] == exp[1]).all() and (got["r"][some] == exp[2]).all()


# strides that break the alignment of rows, and the outputs in the inputs' place
@gpu
@pytest.mark.parametrize("cols,ldx,ldb", [(64, 65, 64), (64, 68, 72), (1000, 1003, 1001), (4096, 4100, 4097)])
def test_norm_strides(hip, dev, cols, ldx, ldb):
    rng = np.random.default_rng(cols + ldx)
    x, b, w, post = normal(rng, (5, cols)), normal(rng, (5, cols)), normal(rng, cols), normal(rng, cols)
    got, flag = call_norm(hip, dev, x, b, post, w=w, ldx=ldx, ldb=ldb)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, post, w=w))


@gpu
@pytest.mark.parametrize("into", [{"h": "x"}, {"h": "b"}, {"n": "x"}, {"h": "x", "n": "b"}])
@pytest.mark.parametrize("cols", [77, 1024, 17001])
def test_norm_in_place(hip, dev, into, cols):
    rng = np.random.default_rng(cols)
    x, b, w, post, gate = normal(rng, (3, cols)), normal(rng, (3, cols)), normal(rng, cols), normal(rng, cols), normal(rng, (1, cols))
    x[1, 3] = 1 << 30
    got, flag = call_norm(hip, dev, x, b, post, gate, 70000, w, into=into)
    assert flag == 0
    same(got, *ref.residual_norm(x, b, post, gate, 70000, w))


@gpu
@pytest.mark.parametrize("cols", [70, 17000])
@pytest.mark.parametrize("what", ["sum", "weight", "gate", "product"])
def test_norm_values_that_do_not_fit_raise_the_flag(hip, dev, what, cols):
    x, b, w, gate = np.full((2, cols), 1 << 20, np.int32), np.full((2, cols), 1 << 20, np.int32), np.full(cols, 65536, np.int32), np.full((1, cols), 65536, np.int32)
    if what == "sum":
        x[1, 5], b[1, 5] = (1 << 31) - 1, 1
    elif what == "weight":      # w r / s of a row of zeros: 2^31 * 2.07e7 / 2^16
        x[1], b[1], w[5] = 0, 0, (1 << 31) - 1
    elif what == "gate":
        b[1, 5], gate[0, 5] = 1 << 30, 1 << 30
    else:                       # q(w r) = 2^26, times 2^21, by 2^16: 2^31
        w[5] = (1 << 31) - 1
    got, flag = call_norm(hip, dev, x, b, None, gate, 65536, w)
    assert flag == ref.RANGE
    # without a flag the call returns the error, and the next call is none the worse
    with pytest.raises(RuntimeError, match="zk_i32_residual_norm: a value does not fit"):
        call_norm(hip, dev, x, b, None, gate, 65536, w, flag=c_void_p(None))
    ok = np.full((2, cols), 1 << 16, np.int32)
    got, _ = call_norm(hip, dev, ok, w=np.full(cols, 65536, np.int32), flag=c_void_p(None))
    same(got, *ref.residual_norm(ok, w=np.full(cols, 65536)))


# ---- rotary positions ----------------------------------------------------------------------------------------------------------------------------------
def angles(rows, rot, sf, base=10000.0):
    a = np.arange(rows)[:, None] * base ** (-np.arange(0, rot, 2) / max(rot, 1))
    return np.round(np.stack([np.cos(a), np.sin(a)], -1) * sf).astype(np.int32)


def call_rope(hip, dev, x, table, rot, neighbours, positions=None, first=0, sf=65536, fr=False, by_head=False, pad=0, in_place=False, flag=None):
    """x: [token][head][dim]; pad: elements between heads, and twice as many behind a token's"""
    tokens, heads, dim = x.shape
    stored = np.full((tokens, heads * (dim + pad) + 2 * pad), 999, np.int64)
    stored[:, :heads * (dim + pad)].reshape(tokens, heads, dim + pad)[..., :dim] = x
    xs = (stored.shape[1], dim + pad)
    os = xs if in_place else (dim, tokens * dim) if by_head else (heads * dim, dim)
    px = dev.up(ref.elements(stored), np.uint32) if fr else dev.up(stored)
    size = stored.size if in_place else x.size
    out = px if in_place else dev.space(size * (32 if fr else 4))
    f = dev.flag() if flag is None else flag
    hip.call("zk_fr_rope" if fr else "zk_i32_rope", out, c_size_t(os[0]), c_size_t(os[1]), px, c_size_t(xs[0]), c_size_t(xs[1]), c_uint(tokens), c_uint(heads), c_uint(dim), c_uint(rot),
             c_int(neighbours), dev.up(table), c_uint(len(table)), dev.up(positions), c_uint(first), c_uint(sf), f, None)
    hip.sync()
    limbs = (8,) if fr else ()
    got = dev.down(out, (size,) + limbs, np.uint32 if fr else np.int32)
    if in_place:
        got = got.reshape(stored.shape + limbs)
        between = got[:, :heads * (dim + pad)].reshape((tokens, heads, dim + pad) + limbs)
        untouched = ref.elements(np.array(999)) if fr else 999
        assert (between[:, :, dim:] == untouched).all() and (got[:, heads * (dim + pad):] == untouched).all()
        got = between[:, :, :dim]
    elif by_head:
        got = got.reshape((heads, tokens, dim) + limbs).swapaxes(0, 1)
    else:
        got = got.reshape((tokens, heads, dim) + limbs)
    return got, int(dev.down(f, (1,), np.uint32)[0]) if f.value else 0


@gpu
@pytest.mark.parametrize("tokens,heads,dim,rot", [(1, 1, 2, 2), (1, 64, 128, 128), (5, 3, 8, 8), (7, 2, 9, 4), (6, 5, 20, 12), (3, 4, 6, 6), (33, 2, 80, 32), (9, 40, 80, 48), (70, 8, 64, 64), (4, 3, 16, 0),
                                                  (257, 1, 256, 250), (130, 32, 128, 128)])
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("fr", [False, True])
@pytest.mark.parametrize("layout", ["tokens", "heads", "in place", "gaps"])
def test_rope(hip, dev, tokens, heads, dim, rot, neighbours, fr, layout):
    if fr and tokens * heads * dim > 100000:
        pytest.skip("the restatement's field elements take minutes at this size")
    rng = np.random.default_rng(tokens + heads + dim + rot)
    x = normal(rng, (tokens, heads, dim))
    table = angles(300, rot, 65536)
    positions = rng.integers(0, 300, tokens).astype(np.int32)
    got, flag = call_rope(hip, dev, x, table, rot, neighbours, positions, fr=fr, by_head=layout == "heads", pad={"gaps": 3, "in place": 4}.get(layout, 0), in_place=layout == "in place")
    exp = ref.rope(x, table, positions, rot, neighbours, 65536)
    assert flag == 0 and (got == (ref.elements(exp) if fr else exp)).all()


def limbs64(v):
    """64-bit integers as field elements, without Python's: r's lowest 64 bits are above 2^63, so r + v borrows nothing from the limbs above for v down to -2^63"""
    v = np.asarray(v, np.int64)
    below, out = v < 0, np.zeros(v.shape + (8,), np.uint32)
    out[..., :2] = np.where(below, v + np.int64(-0xFFFFFFFF), v).astype(np.int64)[..., None].view(np.uint32)
    out[..., 2:] = np.where(below[..., None], ref.elements(np.array(-1))[2:], 0)
    return out


# field elements at the sizes of a prompt's heads
@gpu
@pytest.mark.parametrize("tokens,heads,dim,rot", [(130, 32, 128, 128), (70, 40, 80, 48), (300, 8, 126, 126)])
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("by_head", [False, True])
def test_rope_of_field_elements_of_a_prompt(hip, dev, tokens, heads, dim, rot, neighbours, by_head):
    rng = np.random.default_rng(tokens)
    x = normal(rng, (tokens, heads, dim))
    assert (limbs64(x[0, 0]) == ref.elements(x[0, 0])).all()
    table, positions = angles(500, rot, 65536), rng.integers(0, 500, tokens).astype(np.int32)
    out, f = dev.space(32 * x.size), dev.flag()
    to = (dim, tokens * dim) if by_head else (heads * dim, dim)
    hip.call("zk_fr_rope", out, c_size_t(to[0]), c_size_t(to[1]), dev.up(limbs64(x), np.uint32), c_size_t(heads * dim), c_size_t(dim), c_uint(tokens), c_uint(heads), c_uint(dim), c_uint(rot),
             c_int(neighbours), dev.up(table), c_uint(500), dev.up(positions), c_uint(0), c_uint(65536), f, None)
    hip.sync()
    exp = ref.rope(x, table, positions, rot, neighbours, 65536)
    assert dev.down(f, (1,), np.uint32)[0] == 0
    assert (dev.down(out, (heads, tokens, dim, 8) if by_head else (tokens, heads, dim, 8), np.uint32) == limbs64(exp.swapaxes(0, 1) if by_head else exp)).all()


@gpu
@pytest.mark.parametrize("sf", [1, 3, 1000, 1 << 30])
@pytest.mark.parametrize("fr", [False, True])
def test_rope_scales_and_consecutive_positions(hip, dev, sf, fr):
    rng = np.random.default_rng(sf)
    x = rng.integers(-(1 << 30), 1 << 30, (12, 2, 8)).astype(np.int32)
    table = angles(40, 6, sf)
    got, flag = call_rope(hip, dev, x, table, 6, 0, None, 28, sf, fr)
    exp = ref.rope(x, table, np.arange(28, 40), 6, 0, sf)
    assert flag == 0 and (got == (ref.elements(exp) if fr else exp)).all()


@gpu
@pytest.mark.parametrize("fr", [False, True])
@pytest.mark.parametrize("bad", ["negative", "behind", "first", "wraps"])
def test_rope_positions_outside_the_table_are_not_written(hip, dev, fr, bad):
    rng = np.random.default_rng(3)
    x = normal(rng, (5, 2, 8))
    table = angles(10, 8, 65536)
    positions = np.array([0, 9, 4, 9, 1], np.int32)
    where = [2]
    if bad == "negative":
        positions[2] = -1
    elif bad == "behind":
        positions[2] = 10
    first = {"first": 7, "wraps": 0xFFFFFFFE}.get(bad, 0)
    if first:
        positions, where = None, [3, 4] if bad == "first" else [0, 1, 2, 3, 4]
    got, flag = call_rope(hip, dev, x, table, 8, 0, positions, first, fr=fr)
    assert flag == ref.POSITION
    at = positions if positions is not None else np.minimum(first + np.arange(5), 9)
    exp = ref.rope(x, table, np.where((at < 0) | (at > 9), 0, at), 8, 0, 65536)
    exp = ref.elements(exp) if fr else exp
    for t in range(5):
        if t in where:
            assert (got[t].view(np.uint8 if not fr else np.uint32) == (0x5A if not fr else 0x5A5A5A5A)).all()
        else:
            assert (got[t] == exp[t]).all()
    with pytest.raises(RuntimeError, match="rope: a position lies outside the table"):
        call_rope(hip, dev, x, table, 8, 0, positions, first, fr=fr, flag=c_void_p(None))


@gpu
@pytest.mark.parametrize("fr", [False, True])
@pytest.mark.parametrize("dim", [7, 8])
def test_heads_that_are_only_copied_have_no_position(hip, dev, fr, dim):
    rng = np.random.default_rng(dim)
    x = normal(rng, (5, 2, dim))
    for positions, first in ((np.array([-1, 5, 1 << 30, -(1 << 31), 0], np.int32), 0), (None, 0xFFFFFFFE)):
        got, flag = call_rope(hip, dev, x, angles(2, 0, 65536), 0, 0, positions, first, fr=fr, by_head=True)
        assert flag == 0 and (got == (ref.elements(x) if fr else x)).all()


@gpu
def test_rope_values_that_do_not_fit_raise_the_flag(hip, dev):
    x = np.zeros((1, 2, 4), np.int32)
    x[0, 1] = (1 << 31) - 1
    table = np.full((1, 2, 2), 65536, np.int32)             # c = s = 1: the second sum is 2^32 - 2
    assert call_rope(hip, dev, x, table, 4, 0)[1] == ref.RANGE
    assert call_rope(hip, dev, x // 2, table // 2, 4, 1)[1] == 0
    assert call_rope(hip, dev, x // 2, np.full((1, 2, 2), (1 << 30) + 1, np.int32), 4, 1, sf=1 << 30)[1] == ref.RANGE
    # field elements: sums beyond int32 are elements like any other; elements that are no 32-bit integers are not
    got, flag = call_rope(hip, dev, x, table, 4, 0, fr=True)
    assert flag == 0 and (got == ref.elements(ref.rope(x, table, [0], 4, 0, 65536))).all()
    for v in ((1 << 31), -(1 << 31) - 1, 1 << 62, 1 << 62):
        y = np.zeros((1, 2, 4), np.int64)
        y[0, 1, 2] = v
        assert call_rope(hip, dev, y, table, 4, 0, fr=True)[1] == ref.RANGE


# integers as Python has them: what lies outside int32, the negatives beyond 64 bits among it, raises the flag and counts as 0
OUTSIDE = [1 << 31, -(1 << 31) - 1, 1 << 62, -(1 << 62), (1 << 63) - 1, -(1 << 63), 1 << 63, -(1 << 63) - 1, 5 - (1 << 64), 1 - (1 << 64), (1 << 31) - 1 - (1 << 64), (1 << 31) - (1 << 64), (1 << 62) - (1 << 64),
           (1 << 64) - 1, 1 << 64, -(1 << 64), -(1 << 64) - 5, 1 << 100, -(1 << 100), 7 - (1 << 200)]


def call_fr_rope(hip, dev, x, table, rot, neighbours, sf=65536):
    """x: [token][head][dim] of Python integers, positions 0, 1, ..."""
    tokens, heads, dim = x.shape
    out, f = dev.space(32 * x.size), dev.flag()
    strides = (c_size_t(heads * dim), c_size_t(dim))
    hip.call("zk_fr_rope", out, *strides, dev.up(ref.elements(x), np.uint32), *strides, c_uint(tokens), c_uint(heads), c_uint(dim), c_uint(rot), c_int(neighbours), dev.up(table), c_uint(len(table)), None,
             c_uint(0), c_uint(sf), f, None)
    hip.sync()
    return dev.down(out, x.shape + (8,), np.uint32), int(dev.down(f, (1,), np.uint32)[0])


@gpu
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("v", OUTSIDE)
def test_rope_of_elements_that_are_no_32_bit_integers(hip, dev, v, neighbours):
    x = normal(np.random.default_rng(1), (3, 2, 8)).astype(object)
    table = angles(3, 8, 65536)
    for at in ((0, 0, 1), (2, 1, 6)):
        y, zeroed = x.copy(), x.copy()
        y[at], zeroed[at] = v, 0
        got, flag = call_fr_rope(hip, dev, y, table, 8, neighbours)
        assert flag == ref.RANGE and (got == ref.elements(ref.rope(zeroed, table, np.arange(3), 8, neighbours, 65536))).all()
    for edge in ((1 << 31) - 1, -(1 << 31)):
        y = x.copy()
        y[1, 1, 3] = edge
        got, flag = call_fr_rope(hip, dev, y, table, 8, neighbours)
        assert flag == 0 and (got == ref.elements(ref.rope(y, table, np.arange(3), 8, neighbours, 65536))).all()


# the same in the part of a head that is not rotated, and where no part is
@gpu
@pytest.mark.parametrize("rot", [0, 2, 4])
@pytest.mark.parametrize("v", OUTSIDE)
def test_rope_copies_only_elements_that_are_32_bit_integers(hip, dev, v, rot):
    x = normal(np.random.default_rng(3), (3, 2, 7)).astype(object)
    table = angles(3, rot, 65536)
    for at in ((0, 0, 4), (2, 1, 6)):
        y, zeroed = x.copy(), x.copy()
        y[at], zeroed[at] = v, 0
        got, flag = call_fr_rope(hip, dev, y, table, rot, 0)
        assert flag == ref.RANGE and (got == ref.elements(ref.rope(zeroed, table, np.arange(3), rot, 0, 65536))).all()
    x[0, 1, 5], x[1, 0, 6], x[2, 1, 4] = (1 << 31) - 1, -(1 << 31), 0
    got, flag = call_fr_rope(hip, dev, x, table, rot, 0)
    assert flag == 0 and (got == ref.elements(ref.rope(x, table, np.arange(3), rot, 0, 65536))).all()


@gpu
@pytest.mark.parametrize("v", [v for v in OUTSIDE if abs(v) > 1 << 62])
def test_heads_of_elements_that_are_no_63_bit_integers(hip, dev, v):
    x = normal(np.random.default_rng(2), (2, 3, 4)).astype(object)
    out, f = dev.space(4 * x.size), dev.flag()

    def call(x):
        hip.call("zk_memset", f, c_int(0), c_size_t(4), None)
        hip.call("zk_i32_from_heads", out, dev.up(ref.elements(x), np.uint32), c_uint(2), c_uint(3), c_uint(4), c_uint(1 << 16), c_uint(1 << 16), f, None)
        return dev.down(out, (3, 2, 4)).astype(np.int64), int(dev.down(f, (1,), np.uint32)[0])

    for edge in (1 << 62, -(1 << 62)):
        x[1, 2, 3] = edge
        got, flag = call(x)
        assert flag == 0 and (got == ref.quotient(ref.quotient(x, 1 << 16), 1 << 16).swapaxes(0, 1)).all()
    x[1, 2, 3] = v
    assert call(x)[1] == ref.RANGE


# ---- products with a kept weight ---------------------------------------------------------------------------------------------------------------------------
class Weight:
    def __init__(self, hip, dev, w, from_fr=False):
        self.hip, self.h = hip, c_void_p()
        if from_fr:
            self.fr = dev.space(32 * w.size)
            hip.call("zk_fr_from_i32", self.fr, dev.up(w), c_size_t(w.size), None)
            hip.call("zk_fr_matmul_rhs_prepare", ctypes.byref(self.h), self.fr, c_uint(w.shape[0]), c_uint(w.shape[1]), None)
        else:
            p = dev.up(w)
            hip.call("zk_i32_rhs_prepare", ctypes.byref(self.h), p, c_uint(w.shape[0]), c_uint(w.shape[1]), None)
            hip.call("zk_memset", p, c_int(0x11), c_size_t(4 * w.size), None)      # what it was made from is not read again

    def __del__(self):
        if self.h:
            self.hip.lib.zk_fr_matmul_rhs_free(self.h)


def prepare_x(dev, x, ldx):
    wide = np.full((x.shape[0], ldx or x.shape[1]), 2147483647, np.int32)
    wide[:, :x.shape[1]] = x
    return dev.up(wide)


def workspace(hip, dev, rows, inner):
    hip.lib.zk_i32_linear_workspace.restype = c_size_t
    n = hip.lib.zk_i32_linear_workspace(c_uint(rows), c_uint(inner))
    return dev.space(n), n


def call_linear(hip, dev, x, weight, cols, sf, ldx=None, own_workspace=False, flag=None):
    rows, inner = x.shape
    out, f = dev.space(4 * rows * cols), dev.flag() if flag is None else flag
    ws, n = workspace(hip, dev, rows, inner) if own_workspace else (c_void_p(None), 0)
    hip.call("zk_i32_linear", out, prepare_x(dev, x, ldx), c_size_t(ldx or inner), weight.h, c_uint(rows), c_uint(sf), ws, c_size_t(n), f, None)
    hip.sync()
    return dev.down(out, (rows, cols)), int(dev.down(f, (1,), np.uint32)[0]) if f.value else 0


def call_gated(hip, dev, x, gate, up, cols, sf_gate, sf_up, table, low, sf_hidden, ldx=None, own_workspace=False, flag=None):
    rows, inner = x.shape
    out, f = dev.space(4 * rows * cols), dev.flag() if flag is None else flag
    ws, n = workspace(hip, dev, rows, inner) if own_workspace else (c_void_p(None), 0)
    hip.call("zk_i32_gated", out, prepare_x(dev, x, ldx), c_size_t(ldx or inner), gate.h, up.h, c_uint(rows), c_uint(sf_gate), c_uint(sf_up), dev.up(table), c_int(low), c_uint(len(table)),
             c_uint(sf_hidden), ws, c_size_t(n), f, None)
    hip.sync()
    return dev.down(out, (rows, cols)), int(dev.down(f, (1,), np.uint32)[0]) if f.value else 0


def swiglu(low, n, out_scale):
    v = (np.arange(n) + low) / 4096.0
    return np.round(v / (1 + np.exp(-v)) * out_scale).astype(np.int32)


SHAPES = [(1, 1, 1), (1, 7, 5), (1, 128, 64), (1, 1000, 129), (2, 33, 70), (3, 64, 1), (7, 129, 31), (8, 256, 96), (16, 200, 100), (17, 64, 65), (31, 300, 33), (32, 128, 128), (33, 97, 64), (64, 160, 64),
          (65, 31, 63), (100, 500, 130), (127, 128, 129), (128, 256, 64), (129, 130, 127), (200, 64, 300), (257, 96, 200), (300, 1000, 275)]


@gpu
@pytest.mark.parametrize("rows,inner,cols", SHAPES)
@pytest.mark.parametrize("weights", ["one digit", "two digits", "three digits"])
def test_linear(hip, dev, rows, inner, cols, weights):
    rng = np.random.default_rng(rows * 7919 + inner * 31 + cols)
    most = {"one digit": 127, "two digits": 32639, "three digits": 8355711}[weights]
    w = rng.integers(-most, most + 1, (inner, cols)).astype(np.int32)
    w[0, 0] = most
    x = normal(rng, (rows, inner))
    sf = 65536 if most > 127 else 1000
    got, flag = call_linear(hip, dev, x, Weight(hip, dev, w), cols, sf, own_workspace=rows % 2 == 0)
    assert flag == 0 and (got == ref.linear(x, w, sf)).all()


# rows of one, two, three and four digits beside each other, the largest and smallest that there are, and rows of zeros
@gpu
@pytest.mark.parametrize("rows", [1, 5, 40, 130, 260])
@pytest.mark.parametrize("inner", [40, 1000])
def test_linear_rows_of_every_magnitude(hip, dev, rows, inner):
    rng = np.random.default_rng(rows + inner)
    x = np.zeros((rows, inner), np.int32)
    for r in range(rows):
        most = [127, 32639, 8355711, 0x7F7F7F7F, 0][(r + rows) % 5]
        x[r] = rng.integers(-most, most + 1, inner)
        x[r, r % inner] = most
    x[rows // 2, 0] = -(1 << 31)
    w = rng.integers(-32000, 32000, (inner, 70)).astype(np.int32)
    got, flag = call_linear(hip, dev, x, Weight(hip, dev, w), 70, 1 << 24, ldx=inner + 5)
    assert flag == 0 and (got == ref.linear(x, w, 1 << 24)).all()


@gpu
@pytest.mark.parametrize("rows", [1, 4, 50, 150])
@pytest.mark.parametrize("sf", [1, 3, 1000, 1 << 16, (1 << 32) - 1])
def test_linear_scaling_factors_and_strides(hip, dev, rows, sf):
    rng = np.random.default_rng(rows)
    x, w = rng.integers(-100, 101, (rows, 66)).astype(np.int32) * (1 if sf < 1000 else 3000), rng.integers(-100, 101, (66, 40)).astype(np.int32)
    got, flag = call_linear(hip, dev, x, Weight(hip, dev, w), 40, sf, ldx=67, own_workspace=True)
    assert flag == 0 and (got == ref.linear(x, w, sf)).all()


@gpu
@pytest.mark.parametrize("rows", [1, 3, 70, 140])
def test_linear_values_that_do_not_fit_raise_the_flag(hip, dev, rows):
    rng = np.random.default_rng(1)
    x, w = normal(rng, (rows, 64)), rng.integers(-100, 101, (64, 48)).astype(np.int32)
    weight = Weight(hip, dev, w)
    exp = ref.linear(x, w, 65536)
    for v in (0x7F7F7F80, (1 << 31) - 1):                       # an element of x with no four digits
        y = x.copy()
        y[rows - 1, 63] = v
        assert call_linear(hip, dev, y, weight, 48, 1 << 30)[1] == ref.RANGE
    x2 = x.copy()                                               # a result beyond int32, one just within
    x2[rows - 1] = 0
    x2[rows - 1, 0] = 1 << 30
    w2 = np.zeros((64, 48), np.int32)
    w2[0, 47] = 4
    got, flag = call_linear(hip, dev, x2, Weight(hip, dev, w2), 48, 2)
    assert flag == ref.RANGE
    got, flag = call_linear(hip, dev, -x2, Weight(hip, dev, w2), 48, 2)
    assert flag == 0 and (got == ref.linear(-x2, w2, 2)).all()
    with pytest.raises(RuntimeError, match="zk_i32_linear: a value does not fit"):
        call_linear(hip, dev, x2, Weight(hip, dev, w2), 48, 2, flag=c_void_p(None))
    got, _ = call_linear(hip, dev, x, weight, 48, 65536, flag=c_void_p(None))
    assert (got == exp).all()


# sums of products around 2^62: below they are exact, from there on flagged
@gpu
@pytest.mark.parametrize("rows", [1, 40, 200])
def test_linear_sums_around_the_limit(hip, dev, rows):
    inner = 1024
    w = np.zeros((inner, 34), np.int32)
    w[:, 33] = 1 << 22
    x = np.zeros((rows, inner), np.int32)
    x[rows - 1] = 1 << 30                                       # 2^10 * 2^52 = 2^62
    weight = Weight(hip, dev, w)
    assert call_linear(hip, dev, x, weight, 34, 1 << 31)[1] == ref.RANGE
    x[rows - 1, 5] -= 1                                         # 2^62 - 2^22: by 2^32 - 1, 2^30 + 2^-2 - ...
    got, flag = call_linear(hip, dev, x, weight, 34, (1 << 32) - 1)
    assert flag == 0 and (got == ref.linear(x, w, (1 << 32) - 1)).all()
    x = -x
    got, flag = call_linear(hip, dev, x, weight, 34, (1 << 32) - 1)
    assert flag == 0 and (got == ref.linear(x, w, (1 << 32) - 1)).all()


@gpu
@pytest.mark.parametrize("rows,inner,cols", SHAPES)
@pytest.mark.parametrize("weights", [(32000, 32000), (100, 100), (120, 8355711), (8355711, 20000)])
def test_gated(hip, dev, rows, inner, cols, weights):
    rng = np.random.default_rng(rows * 104729 + inner * 13 + cols)
    g, u = (np.clip(np.round(rng.normal(0, 0.3 * m, (inner, cols))), -m, m).astype(np.int32) for m in weights)
    g[0, 0], u[0, 0] = weights
    x = normal(rng, (rows, inner), 3000.0)
    sf_gate = 1 << 20 if weights[0] > 100 else 1 << 10
    low, n = -(1 << 21), 1 << 22
    if weights[0] > 1 << 20:
        sf_gate = 1 << 28
    table = swiglu(low, n, 4096.0)
    got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u, from_fr=rows % 2 == 1), cols, sf_gate, 1 << 16, table, low, 1 << 20, own_workspace=rows % 3 == 0)
    assert flag == 0 and (got == ref.gated(x, g, u, sf_gate, 1 << 16, table, low, 1 << 20)).all()


@gpu
@pytest.mark.parametrize("rows", [1, 30, 131])
def test_gated_divisors_that_are_no_powers_of_two(hip, dev, rows):
    rng = np.random.default_rng(rows)
    x, g, u = normal(rng, (rows, 90), 500.0), normal(rng, (90, 61), 300.0), normal(rng, (90, 61), 300.0)
    table = rng.integers(-1000, 1000, 5001).astype(np.int32)
    got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), 61, 10007, 999, table, -2500, 12345, ldx=93)
    assert flag == 0 and (got == ref.gated(x, g, u, 10007, 999, table, -2500, 12345)).all()


@gpu
@pytest.mark.parametrize("rows", [1, 33, 150])
@pytest.mark.parametrize("side", ["below", "above"])
def test_gated_activations_outside_the_table(hip, dev, rows, side):
    x = np.ones((rows, 40), np.int32)
    g, u = np.zeros((40, 50), np.int32), np.ones((40, 50), np.int32)
    g[0] = 3
    g[0, 49] = 4 if side == "above" else -5
    table = np.arange(100, 108, dtype=np.int32)                  # -4 .. 3
    got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), 50, 1, 1, table, -4, 1)
    assert flag == ref.TABLE and (got[:, 49] == 0).all() and (got[:, :49] == 107 * 40).all()
    with pytest.raises(RuntimeError, match="zk_i32_gated: an activation lies outside the table"):
        call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), 50, 1, 1, table, -4, 1, flag=c_void_p(None))
    g[0, 49] = 3 if side == "above" else -4
    got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), 50, 1, 1, table, -4, 1)
    assert flag == 0 and (got == ref.gated(x, g, u, 1, 1, table, -4, 1)).all()


# Products of enough tiles for the kernel of many rows (1024 strips of 16 columns by 32 rows, 640 where there are two weights; 64 columns a tile up to 128 tiles, 128 rows from 256 on):
# ragged in every direction, one step of the contraction and several, rows of four digits in some tiles only, in the last row, in all
TILED = [(300, 40, 2100), (641, 128, 1030), (130, 300, 3650), (2100, 40, 2050), (2177, 140, 1921), (33, 70, 16600), (600, 33, 2000), (700, 260, 2111)]


def tiled_rows(rng, rows, inner, digits):
    x = normal(rng, (rows, inner))
    if digits == "some":
        for r in (3, rows // 2, rows - 1):
            x[r] = rng.integers(-(1 << 31), 0x7F7F7F80, inner)
            x[r, r % inner] = 0x7F7F7F7F
    elif digits == "all":
        x = rng.integers(-(1 << 31), 0x7F7F7F80, (rows, inner)).astype(np.int32)
    return x


@gpu
@pytest.mark.parametrize("rows,inner,cols", TILED)
@pytest.mark.parametrize("most,sf", [(127, 1 << 16), (32639, 1 << 24), (32639, 9999991), (8355711, 1 << 31)])
@pytest.mark.parametrize("digits", ["three", "some", "all"])
def test_linear_in_tiles(hip, dev, rows, inner, cols, most, sf, digits):
    rng = np.random.default_rng(rows + inner + cols + most % 1000)
    w = rng.integers(-most, most + 1, (inner, cols)).astype(np.int32)
    w[0, 0] = most
    x = tiled_rows(rng, rows, inner, digits)
    got, flag = call_linear(hip, dev, x, Weight(hip, dev, w), cols, sf, own_workspace=True, ldx=inner + (3 if digits == "some" else 4))
    exp = ref.linear(x, w, sf)
    assert flag == (0 if (exp == exp.astype(np.int32)).all() else ref.RANGE) and (got == exp.astype(np.int32)).all()


@gpu
@pytest.mark.parametrize("rows,inner,cols", [(300, 40, 1100), (641, 128, 517), (2100, 40, 1050), (2177, 140, 961)])
@pytest.mark.parametrize("weights", [(30000, 30000), (120, 8355711), (8355711, 20000)])
@pytest.mark.parametrize("general", [False, True])
def test_gated_in_tiles(hip, dev, rows, inner, cols, weights, general):
    rng = np.random.default_rng(rows + inner + cols + weights[0] % 1000)
    g, u = (np.clip(np.round(rng.normal(0, 0.3 * m, (inner, cols))), -m, m).astype(np.int32) for m in weights)
    g[0, 0], u[0, 0] = weights
    x = normal(rng, (rows, inner), 3000.0)
    if general:                                                 # a tile with rows of four digits: their activations leave the table
        x[rows - 1] = rng.integers(-(1 << 31), 0x7F7F7F80, inner)
    sfs = (1 << 20, 1 << 16, 1 << 20) if weights[0] < 1 << 20 else (1 << 28, 1 << 16, 1 << 20)
    if general:
        sfs = tuple(v - 1 for v in sfs)
    low, n = -(1 << 20), 1 << 21
    table = swiglu(low, n, 4096.0)
    got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), cols, sfs[0], sfs[1], table, low, sfs[2], own_workspace=True)
    at, up = ref.linear(x, g, sfs[0]) - low, ref.linear(x, u, sfs[1])
    inside = (at >= 0) & (at < n)
    exp = np.where(inside, ref.quotient(table.astype(np.int64)[np.clip(at, 0, n - 1)] * up.astype(np.int32), sfs[2]), 0)
    fits = (up == up.astype(np.int32)) & (exp == exp.astype(np.int32))
    assert flag == (0 if inside.all() else ref.TABLE) | (0 if fits.all() else ref.RANGE)
    assert (got == exp)[fits].all() and (general or flag == 0)


# Long contractions with few tiles, which are split over workgroups (more than 32 rows, two digits a weight), in parts of several lengths; and their neighbours, which are not
LONG = [(33, 8065, 70), (64, 11008, 130), (150, 8300, 650), (1000, 8200, 40), (32, 8200, 70), (33, 8064, 70)]


@gpu
@pytest.mark.parametrize("rows,inner,cols", LONG)
@pytest.mark.parametrize("most,sf", [(127, 1 << 16), (32639, 1 << 29), (32639, (1 << 29) - 3)])
@pytest.mark.parametrize("digits", ["three", "some", "all"])
def test_linear_of_long_rows(hip, dev, rows, inner, cols, most, sf, digits):
    test_linear_in_tiles(hip, dev, rows, inner, cols, most, sf, digits)


@gpu
@pytest.mark.parametrize("rows,inner,cols", LONG)
@pytest.mark.parametrize("weights", [(30000, 30000), (120, 8355711)])
@pytest.mark.parametrize("general", [False, True])
def test_gated_of_long_rows(hip, dev, rows, inner, cols, weights, general):
    test_gated_in_tiles(hip, dev, rows, inner, cols, weights, general)


# the parts of one sum: all of it in one part or another, and the largest that there is
@gpu
def test_edges_of_long_rows(hip, dev):
    inner, cols, rows = 16384, 70, 40
    w = np.full((inner, cols), 32639, np.int32)
    weight = Weight(hip, dev, w)
    x = np.zeros((rows, inner), np.int32)
    for r in range(rows):
        x[r, r * 420:r * 420 + 3] = (1 << 30, -(1 << 30), 1 + r)
    got, flag = call_linear(hip, dev, x, weight, cols, 1)
    assert flag == 0 and (got == ref.linear(x, w, 1)).all()
    x[rows - 1] = -(1 << 31)
    sf = 0xFFFFFFFF
    got, flag = call_linear(hip, dev, x, weight, cols, sf)           # 2^31 2^14 32639 is the largest sum that two digits of weights have at this length
    assert flag == 0 and (got == ref.linear(x, w, sf)).all()


@gpu
def test_products_in_place_are_refused(hip, dev):
    x = np.ones((6, 8), np.int32)
    w, p, f = Weight(hip, dev, np.eye(8, dtype=np.int32)), dev.up(x), dev.flag()
    with pytest.raises(RuntimeError, match="zk_i32_linear: in place"):
        hip.call("zk_i32_linear", p, p, c_size_t(8), w.h, c_uint(6), c_uint(1), None, c_size_t(0), f, None)
    with pytest.raises(RuntimeError, match="zk_i32_gated: in place"):
        hip.call("zk_i32_gated", p, p, c_size_t(8), w.h, w.h, c_uint(6), c_uint(1), c_uint(1), dev.up(np.ones(4, np.int32)), c_int(0), c_uint(4), c_uint(1), None, c_size_t(0), f, None)
    assert (dev.down(p, (6, 8)) == x).all()


# sums around 2^62 and values around the edges of int32 and the table, in the last row and column of the last tile; x's rows and the weight's columns beyond them do not count
@gpu
@pytest.mark.parametrize("rows", [321, 2200])
def test_edges_in_tiles(hip, dev, rows):
    inner, cols = 1024, 2050
    w = np.zeros((inner, cols), np.int32)
    w[:, cols - 1] = 1 << 22
    weight = Weight(hip, dev, w)
    x = np.zeros((rows, inner), np.int32)
    x[rows - 1] = 1 << 30
    assert call_linear(hip, dev, x, weight, cols, 1 << 31)[1] == ref.RANGE
    for sign in (1, -1):
        x[rows - 1] = sign * (1 << 30)
        x[rows - 1, 5] -= sign
        got, flag = call_linear(hip, dev, x, weight, cols, (1 << 32) - 1)
        exp = np.zeros((rows, cols), np.int64)
        exp[rows - 1, cols - 1] = ref.quotient(sign * ((1 << 62) - (1 << 22)), (1 << 32) - 1)
        assert flag == 0 and (got == exp).all()
    g = np.zeros((40, cols), np.int32)
    g[0, cols - 1] = 3
    x = np.ones((rows, 40), np.int32)
    u = np.ones((40, cols), np.int32)
    table = np.arange(100, 108, dtype=np.int32)                  # 1 .. 8: a sum of 0 lies outside
    for low, bad in ((-4, False), (0, False), (1, True)):
        got, flag = call_gated(hip, dev, x, Weight(hip, dev, g), Weight(hip, dev, u), cols, 1, 1, table, low, 1)
        assert flag == (ref.TABLE if bad else 0)
        assert (got[:, cols - 1] == (103 - low) * 40).all() and (got[:, :cols - 1] == (0 if bad else (100 - low) * 40)).all()


@gpu
def test_handles_from_field_elements_serve_both_and_those_from_int32_no_field_product(hip, dev):
    rng = np.random.default_rng(8)
    x, w = normal(rng, (5, 40)), normal(rng, (40, 30), 1300.0)
    of_fr, of_i32 = Weight(hip, dev, w, from_fr=True), Weight(hip, dev, w)
    for weight in (of_fr, of_i32):
        assert (call_linear(hip, dev, x, weight, 30, 65536)[0] == ref.linear(x, w, 65536)).all()
    C, path = dev.space(32 * 150), c_int()
    hip.call("zk_fr_matmul_rhs_ints", C, dev.up(x), of_fr.h, c_uint(5), c_int(0), ctypes.byref(path), None)
    assert (dev.down(C, (5, 30, 8), np.uint32) == ref.elements(x.astype(np.int64) @ w)).all()
    for name in ("zk_fr_matmul_rhs", "zk_fr_matmul_rhs_ints"):
        with pytest.raises(RuntimeError, match="made from int32"):
            hip.call(name, C, dev.up(x), of_i32.h, c_uint(5), c_int(0), ctypes.byref(path), None)
    large = np.full((3, 3), 8355712, np.int32)
    with pytest.raises(RuntimeError, match="8355711"):
        Weight(hip, dev, large)
    with pytest.raises(RuntimeError, match="8355711"):
        call_linear(hip, dev, x[:, :3], Weight(hip, dev, large, from_fr=True), 3, 65536)
    with pytest.raises(RuntimeError, match="different shapes"):
        call_gated(hip, dev, x, of_i32, Weight(hip, dev, w[:, :29]), 30, 1, 1, np.zeros(4), 0, 1)
    with pytest.raises(RuntimeError, match="workspace is smaller"):
        hip.call("zk_i32_linear", C, dev.up(x), c_size_t(40), of_i32.h, c_uint(33), c_uint(1), C, c_size_t(100), dev.flag(), None)      # 33 rows need more; up to four need none


def test_torch_and_the_library_have_one_runtime():
    """What hands torch's streams to the library needs that: two runtimes in a process, and a stream is a pointer into the other one's memory"""
    from gpuhelp import pkg
    pkg.load_hip()
    import torch  # noqa: F401
    with open("/proc/self/maps") as f:
        assert len({line.split()[-1] for line in f if "libamdhip64" in line}) == 1


@gpu
def test_calls_on_two_streams_without_workspaces_of_the_callers(hip, dev):
    """Handles made on one stream and used on others at once, the library's own scratch memory in every call: each result is its own"""
    import torch
    rng = np.random.default_rng(6)
    w = [normal(rng, (300, 500), 3000.0) for _ in range(2)]
    handles, streams, x, out, flags = [], [torch.cuda.Stream() for _ in range(4)], [], [], []
    for i, s in enumerate(streams):
        h, p = c_void_p(), dev.up(w[i % 2])
        hip.sync()
        hip.call("zk_i32_rhs_prepare", ctypes.byref(h), p, c_uint(300), c_uint(500), c_void_p(s.cuda_stream))
        handles.append(h)
        rows = [3, 20, 50, 200][i]
        x.append(normal(rng, (rows, 300)))
        out.append(dev.space(4 * rows * 500))
        flags.append(dev.flag())
    px = [dev.up(a) for a in x]
    hip.sync()
    for turn in range(5):
        for i in range(4):
            hip.call("zk_i32_linear", out[i], px[i], c_size_t(300), handles[(i + turn) % 4], c_uint(len(x[i])), c_uint(65536), None, c_size_t(0), flags[i], c_void_p(streams[(i * 3 + turn) % 4].cuda_stream))
        torch.cuda.synchronize()
        for i in range(4):
            assert (dev.down(out[i], (len(x[i]), 500)) == ref.linear(x[i], w[(i + turn) % 4 % 2], 65536)).all()
            assert dev.down(flags[i], (1,), np.uint32)[0] == 0
    for h in handles:
        hip.lib.zk_fr_matmul_rhs_free(h)


@gpu
@pytest.mark.parametrize("rows", [2, 40])
def test_handles_from_field_elements_serve_other_streams_at_once(hip, dev, rows):
    """Handles made from field elements, each on a stream of its own, and used on others right behind: the planes are there, for the int32 products and the field's"""
    n, p = 2048, 1536
    rng = np.random.default_rng(rows)
    w, x = normal(rng, (n, p), 3000.0), normal(rng, (rows, n))
    fr, px = dev.space(32 * n * p), dev.up(x)
    hip.call("zk_fr_from_i32", fr, dev.up(w), c_size_t(n * p), None)
    exp = x.astype(np.int64) @ w
    low = np.where(exp < 0, exp + np.int64(-0xFFFFFFFF), exp)         # the lowest 64 bits of r + v, modulo 2^64: r's are 2^64 - (2^32 - 1)
    streams = [c_void_p() for _ in range(3)]
    for s in streams:                        # of the runtime that the library runs on; non-blocking
        assert hip.lib.hipStreamCreateWithFlags(ctypes.byref(s), c_uint(1)) == 0
    outs, fields, flags = [dev.space(4 * rows * p) for _ in streams], [dev.space(32 * rows * p) for _ in streams], [dev.flag() for _ in streams]
    handles = []
    hip.sync()
    for i, s in enumerate(streams):
        h, path, other = c_void_p(), c_int(), streams[(i + 1) % 3]
        hip.call("zk_fr_matmul_rhs_prepare", ctypes.byref(h), fr, c_uint(n), c_uint(p), s)
        hip.call("zk_i32_linear", outs[i], px, c_size_t(n), h, c_uint(rows), c_uint(65536), None, c_size_t(0), flags[i], other)
        hip.call("zk_fr_matmul_rhs_ints", fields[i], px, h, c_uint(rows), c_int(0), ctypes.byref(path), other)
        handles.append(h)
    for s in streams:
        hip.call("zk_sync", s)
    for i in range(3):
        assert dev.down(flags[i], (1,), np.uint32)[0] == 0
        assert (dev.down(outs[i], (rows, p)) == ref.quotient(exp, 65536)).all()
        assert (dev.down(fields[i], (rows, p, 8), np.uint32)[..., :2].copy().view(np.int64)[..., 0] == low).all()
    for h, s in zip(handles, streams):
        hip.lib.zk_fr_matmul_rhs_free(h)
        assert hip.lib.hipStreamDestroy(s) == 0


# ---- as a program calls them: on a stream of its own, captured, one after the other -------------------------------------------------------------------------
def _step(hip, torch, s, stream):
    """one block: the residual stream and its norm, positions for the queries, a projection, the gated product and the way down; every buffer is the caller's"""
    p = lambda t: c_void_p(t.data_ptr())
    T, E, P = s["x"].shape[0], s["x"].shape[1], s["out"].shape[1]
    st = c_void_p(stream.cuda_stream)
    hip.call("zk_i32_residual_norm", p(s["h"]), p(s["n"]), None, p(s["x"]), c_size_t(E), p(s["b"]), c_size_t(E), None, None, c_uint(0), c_int(65536), p(s["nw"]), c_uint(T), c_uint(E), c_double(1e-5),
             c_double(65536.0), c_uint(65536), p(s["flag"]), st)
    hip.call("zk_i32_linear", p(s["q"]), p(s["n"]), c_size_t(E), s["wq"].h, c_uint(T), c_uint(65536), p(s["ws"]), c_size_t(s["ws"].numel()), p(s["flag"]), st)
    hip.call("zk_i32_rope", p(s["q"]), c_size_t(E), c_size_t(E // 4), p(s["q"]), c_size_t(E), c_size_t(E // 4), c_uint(T), c_uint(4), c_uint(E // 4), c_uint(E // 4), c_int(0), p(s["table"]),
             c_uint(s["table"].shape[0]), p(s["at"]), c_uint(0), c_uint(65536), p(s["flag"]), st)
    hip.call("zk_i32_gated", p(s["out"]), p(s["q"]), c_size_t(E), s["wg"].h, s["wu"].h, c_uint(T), c_uint(1 << 20), c_uint(65536), p(s["act"]), c_int(-(1 << 16)), c_uint(1 << 17), c_uint(4096), p(s["ws"]),
             c_size_t(s["ws"].numel()), p(s["flag"]), st)
    hip.call("zk_i32_linear", p(s["down"]), p(s["out"]), c_size_t(P), s["wd"].h, c_uint(T), c_uint(65536), p(s["ws"]), c_size_t(s["ws"].numel()), p(s["flag"]), st)


def _expected(host, w, at):
    h, n, _ = ref.residual_norm(host["x"], host["b"], w=w["nw"])
    T, E = h.shape
    q = ref.rope(ref.linear(n, w["wq"], 65536).reshape(T, 4, E // 4), w["table"], at, E // 4, 0, 65536).reshape(T, E)
    g = ref.gated(q, w["wg"], w["wu"], 1 << 20, 65536, w["act"], -(1 << 16), 4096)
    return h, g, ref.linear(g, w["wd"], 65536)


@gpu
@pytest.mark.parametrize("T", [1, 9, 150])
def test_a_block_on_its_own_stream_and_captured(hip, dev, T):
    """Two states with workspaces of their own: eager on a side stream, then as two graphs replayed in turn with new inputs and eager work in between."""
    import torch
    E, P = 128, 200
    rng = np.random.default_rng(T)
    w = {"nw": normal(rng, E, 5000.0) + 65536, "wq": normal(rng, (E, E), 4000.0), "wg": normal(rng, (E, P), 4000.0), "wu": normal(rng, (E, P), 4000.0), "wd": normal(rng, (P, E), 4000.0),
         "table": angles(64, E // 4, 65536), "act": swiglu(-(1 << 16), 1 << 17, 4096.0)}
    kept = {k: Weight(hip, dev, w[k]) for k in ("wq", "wg", "wu", "wd")}
    hip.lib.zk_i32_linear_workspace.restype = c_size_t
    room = max(hip.lib.zk_i32_linear_workspace(c_uint(T), c_uint(E)), hip.lib.zk_i32_linear_workspace(c_uint(T), c_uint(P)))
    t = lambda a: torch.as_tensor(np.ascontiguousarray(a), device="cuda")
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")

    def state():
        return {**kept, "x": new(T, E), "b": new(T, E), "h": new(T, E), "n": new(T, E), "q": new(T, E), "out": new(T, P), "down": new(T, E), "nw": t(w["nw"]), "table": t(w["table"]), "act": t(w["act"]),
                "at": new(T), "flag": torch.zeros(1, dtype=torch.int32, device="cuda"), "ws": torch.empty(room, dtype=torch.uint8, device="cuda")}

    def fill(s):
        host = {"x": normal(rng, (T, E)), "b": normal(rng, (T, E))}
        at = rng.integers(0, 64, T).astype(np.int32)
        for k in ("x", "b"):
            s[k].copy_(t(host[k]))
        s["at"].copy_(t(at))
        return _expected(host, w, at)

    def check(s, exp):
        torch.cuda.synchronize()
        assert int(s["flag"]) == 0
        for k, e in zip(("h", "out", "down"), exp):
            assert (s[k].cpu().numpy() == e).all(), k

    states, stream = [state(), state()], torch.cuda.Stream()
    for s in states:
        exp = fill(s)
        torch.cuda.synchronize()
        _step(hip, torch, s, stream)
        check(s, exp)
    graphs = []
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            _step(hip, torch, s, stream)
        graphs.append(g)
    for turn in range(3):
        exps = [fill(s) for s in states]
        torch.cuda.synchronize()
        for g in graphs:                         # one behind the other on two streams: nothing is shared
            with torch.cuda.stream(torch.cuda.Stream()):
                g.replay()
        for s, exp in zip(states, exps):
            check(s, exp)
        eager = state()
        exp = fill(eager)
        torch.cuda.synchronize()
        _step(hip, torch, eager, torch.cuda.current_stream())
        check(eager, exp)
    # a captured call without the caller's flag is refused, and the capture goes on
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        rc = hip.lib.zk_i32_residual_norm(c_void_p(states[0]["h"].data_ptr()), None, None, c_void_p(states[0]["x"].data_ptr()), c_size_t(E), None, c_size_t(0), None, None, c_uint(0), c_int(0), None,
                                          c_uint(T), c_uint(E), c_double(1e-5), c_double(65536.0), c_uint(65536), None, c_void_p(stream.cuda_stream))
        message = hip.lib.zk_last_error()
        _step(hip, torch, states[0], stream)
    assert rc == 10001 and b"a captured call needs" in message
    exp = fill(states[0])
    torch.cuda.synchronize()
    g.replay()
    check(states[0], exp)


@gpu
def test_long_rows_captured(hip, dev):
    """Products whose contraction is split, both kinds in one graph with one workspace, replayed with new inputs and eager calls in between"""
    import torch
    T, K, P = 70, 8200, 130
    rng = np.random.default_rng(1)
    g, u = normal(rng, (K, P), 300.0), normal(rng, (K, P), 3000.0)
    wg, wu = Weight(hip, dev, g), Weight(hip, dev, u)
    low, n = -(1 << 16), 1 << 17
    act = swiglu(low, n, 4096.0)
    t = lambda a: torch.as_tensor(np.ascontiguousarray(a), device="cuda")
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device="cuda")
    hip.lib.zk_i32_linear_workspace.restype = c_size_t
    room = hip.lib.zk_i32_linear_workspace(c_uint(T), c_uint(K))
    state = lambda: {"x": new(T, K), "a": new(T, P), "b": new(T, P), "flag": torch.zeros(1, dtype=torch.int32, device="cuda"), "ws": torch.empty(room, dtype=torch.uint8, device="cuda"), "act": t(act)}
    ptr = lambda a: c_void_p(a.data_ptr())

    def step(s, stream):
        st = c_void_p(stream.cuda_stream)
        hip.call("zk_i32_linear", ptr(s["a"]), ptr(s["x"]), c_size_t(K), wu.h, c_uint(T), c_uint(1 << 16), ptr(s["ws"]), c_size_t(room), ptr(s["flag"]), st)
        hip.call("zk_i32_gated", ptr(s["b"]), ptr(s["x"]), c_size_t(K), wg.h, wu.h, c_uint(T), c_uint(1 << 16), c_uint(1 << 16), ptr(s["act"]), c_int(low), c_uint(n), c_uint(1 << 16), ptr(s["ws"]),
                 c_size_t(room), ptr(s["flag"]), st)

    def turn(s, run):
        x = normal(rng, (T, K), 3000.0)
        s["x"].copy_(t(x))
        torch.cuda.synchronize()
        run()
        torch.cuda.synchronize()
        assert int(s["flag"]) == 0
        assert (s["a"].cpu().numpy() == ref.linear(x, u, 1 << 16)).all() and (s["b"].cpu().numpy() == ref.gated(x, g, u, 1 << 16, 1 << 16, act, low, 1 << 16)).all()

    stream, s, eager = torch.cuda.Stream(), state(), state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step(s, stream)
    for _ in range(3):
        turn(s, graph.replay)
        turn(eager, lambda: step(eager, torch.cuda.current_stream()))


# ---- refusals: nothing of these reaches a GPU ----------------------------------------------------------------------------------------------------------------
def refused(name, args, text):
    from gpuhelp import pkg
    lib = pkg.load_hip()
    assert getattr(lib, name)(*args) == 10001
    assert text in lib.zk_last_error().decode()


W = (ctypes.c_int32 * 64)()


@pytest.mark.parametrize("change,text", [
    ({"x": None}, "null x"), ({"cols": 0}, "empty rows"), ({"h": None, "n": None, "r": None}, "no output"), ({"w": None}, "needs a weight"), ({"ldx": 3}, "rows overlap"), ({"ldb": 3}, "rows overlap"),
    ({"b": None}, "needs the block's output"), ({"gate": None}, "gate_rows"), ({"gate_rows": 0}, "gate_rows"), ({"gate_rows": 4}, "gate_rows"), ({"sf": 0}, "scaling factor of 0"),
    ({"eps": 0.0}, "positive"), ({"eps": float("nan")}, "positive"), ({"scale": -1.0}, "positive"), ({"scale": float("inf")}, "positive"), ({"eps": 1e-10}, "below 2^31")])
def test_norm_refusals(change, text):
    a = {"h": W, "n": W, "r": W, "x": W, "ldx": 4, "b": W, "ldb": 4, "post": W, "gate": W, "gate_rows": 2, "res": 1, "w": W, "rows": 6, "cols": 4, "eps": 1e-5, "scale": 65536.0, "sf": 65536}
    a.update(change)
    refused("zk_i32_residual_norm", [a["h"], a["n"], a["r"], a["x"], c_size_t(a["ldx"]), a["b"], c_size_t(a["ldb"]), a["post"], a["gate"], c_uint(a["gate_rows"]), c_int(a["res"]), a["w"], c_uint(a["rows"]),
                                     c_uint(a["cols"]), c_double(a["eps"]), c_double(a["scale"]), c_uint(a["sf"]), W, None], text)


@pytest.mark.parametrize("name", ["zk_i32_rope", "zk_fr_rope"])
@pytest.mark.parametrize("change,text", [
    ({"out": None}, "null tensor"), ({"x": None}, "null tensor"), ({"dim": 0, "rot": 0}, "empty heads"), ({"rot": 10}, "within the head"), ({"rot": 3}, "even"), ({"table": None}, "no table"), ({"rows": 0}, "no table"),
    ({"sf": 0}, "scale"), ({"sf": (1 << 30) + 1}, "scale"), ({"x": "out", "xh": 9}, "in place with other strides"), ({"xt": 7}, "heads overlap"), ({"oh": 7}, "heads overlap"),
    ({"ot": 8, "oh": 8}, "output's heads overlap"), ({"ot": 15, "oh": 8}, "output's heads overlap"), ({"ot": 9, "oh": 16}, "output's heads overlap"), ({"heads": 1 << 28}, "2^30 elements")])
def test_rope_refusals(name, change, text):
    other = (ctypes.c_int32 * 64)()
    a = {"out": other, "x": W, "ot": 16, "oh": 8, "xt": 16, "xh": 8, "tokens": 2, "heads": 2, "dim": 8, "rot": 8, "table": W, "rows": 4, "sf": 65536}
    a.update(change)
    if a["x"] == "out":
        a["x"] = a["out"]
    refused(name, [a["out"], c_size_t(a["ot"]), c_size_t(a["oh"]), a["x"], c_size_t(a["xt"]), c_size_t(a["xh"]), c_uint(a["tokens"]), c_uint(a["heads"]), c_uint(a["dim"]), c_uint(a["rot"]), c_int(0), a["table"],
                   c_uint(a["rows"]), None, c_uint(0), c_uint(a["sf"]), W, None], name + ": ")
    from gpuhelp import pkg
    assert text in pkg.load_hip().zk_last_error().decode()


# tensors that one kernel would read and write at once, and sizes that its counters do not hold
@pytest.mark.parametrize("change,text", [
    ({"h": "x", "ldx": 5}, "cols apart"), ({"n": "x", "ldx": 5}, "cols apart"), ({"h": "b", "ldb": 5}, "cols apart"), ({"n": "b", "ldb": 5}, "cols apart"), ({"h": "n"}, "one tensor"),
    ({"cols": (1 << 24) + 1, "ldx": 1 << 25, "ldb": 1 << 25}, "2^24 columns"), ({"cols": 0xFFFFFFFF, "ldx": 1 << 32, "ldb": 1 << 32}, "2^24 columns")])
def test_norm_refuses_overlaps(change, text):
    a = {k: (ctypes.c_int32 * 64)() for k in ("h", "n", "r", "x", "b", "w")} | {"ldx": 4, "ldb": 4, "cols": 4}
    a.update({k: a[v] if isinstance(v, str) else v for k, v in change.items()})
    refused("zk_i32_residual_norm", [a["h"], a["n"], a["r"], a["x"], c_size_t(a["ldx"]), a["b"], c_size_t(a["ldb"]), None, None, c_uint(0), c_int(1), a["w"], c_uint(6), c_uint(a["cols"]), c_double(1e-5),
                                     c_double(65536.0), c_uint(65536), W, None], text)


@pytest.mark.parametrize("heads,tokens,dim", [(1 << 16, 1 << 16, 1), (0x80000000, 0x80000000, 4), (1, 1, 0xFFFFFF01), (1 << 31, 1 << 31, 1 << 31)])
def test_from_heads_refuses_sizes(heads, tokens, dim):
    refused("zk_i32_from_heads", [W, (ctypes.c_int32 * 64)(), c_uint(heads), c_uint(tokens), c_uint(dim), c_uint(1), c_uint(1), W, None], "more elements")


@pytest.mark.parametrize("rows,factor", [(2148, 1e-6), ((1 << 31) + 1, 1.0), (1 << 31, 0.5)])
def test_table_refuses_angles(rows, factor):
    refused("zk_rope_table", [W, c_uint(rows), c_uint(2), c_double(10000.0), c_double(factor), c_double(0.0), c_double(1.0), c_double(4.0), c_double(1.0), c_uint(65536), None], "zk_rope_table: ")


def test_product_refusals():
    refused("zk_i32_linear", [W, W, c_size_t(4), None, c_uint(1), c_uint(1), None, c_size_t(0), W, None], "zk_i32_linear: null weight")
    refused("zk_i32_gated", [W, W, c_size_t(4), None, None, c_uint(1), c_uint(1), c_uint(1), W, c_int(0), c_uint(4), c_uint(1), None, c_size_t(0), W, None], "zk_i32_gated: null weight")
    h = c_void_p()
    for B, n, p, text in ((None, 2, 2, "null argument"), (W, 0, 2, "empty matrix"), (W, 2, 0, "empty matrix"), (W, 43691, 1, "above 43690"), (W, 1, (1 << 22) + 1, "4194304 columns")):
        refused("zk_i32_rhs_prepare", [ctypes.byref(h), B, c_uint(n), c_uint(p), None], text)


def test_nothing_to_do_is_no_error():
    from gpuhelp import pkg
    lib = pkg.load_hip()
    assert lib.zk_i32_residual_norm(W, W, W, W, c_size_t(4), None, c_size_t(0), None, None, c_uint(0), c_int(0), W, c_uint(0), c_uint(4), c_double(1e-5), c_double(1.0), c_uint(1), W, None) == 0
    for name in ("zk_i32_rope", "zk_fr_rope"):
        assert getattr(lib, name)(W, c_size_t(8), c_size_t(8), W, c_size_t(8), c_size_t(8), c_uint(0), c_uint(1), c_uint(8), c_uint(8), c_int(0), W, c_uint(1), None, c_uint(0), c_uint(1), W, None) == 0

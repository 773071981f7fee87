"""The layer's values as a whole (LayerValues) against the layer's proof and the CPU oracle, and rotary positions in both: outputs equal element for element, transcripts entry for entry."""
import ctypes
import os

import numpy as np
import pytest

import layercfg
import valueshelp as ref
from test_gpu_drivers import TINY_ENV, run
from zkhelp import load_oracle, orc_check, orc_transcript

pytestmark = pytest.mark.gpu
c_void_p, c_size_t, c_int, c_uint, c_double = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_uint32, ctypes.c_double


@pytest.fixture(scope="module")
def pv():
    from gpuhelp import Prover
    p = Prover()
    for name in ("zkp_layer_values", "zkp_layer_attention"):
        getattr(p.lib, name).restype = c_void_p
    return p


@pytest.fixture(scope="module")
def hip():
    from gpuhelp import Hip
    return Hip()


def set_rope(pv, layer, base=10000.0, factor=1.0, original=0.0, low=1.0, high=4.0, magnitude=1.0, dim=0, neighbours=0, first=0, scale=65536):
    pv.lib.zkp_layer_set_rope(c_void_p(layer), (c_double * 6)(base, factor, original, low, high, magnitude), (c_uint * 4)(dim, neighbours, first, scale))


def values(pv, layer, X, repeats=1):
    x = pv.from_i32(X)
    return pv.H(pv.lib.zkp_layer_values(c_void_p(layer), c_void_p(x.h), c_int(repeats), None)).host()


def frequencies(rot, base, factor, original, low, high):
    f = base ** (-np.arange(0, rot, 2, dtype=np.longdouble) / max(rot, 1))
    if original:
        keep = np.clip((original * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return f * (keep + (1 - keep) / factor)
    return f / factor


def exact_table(rows, rot, base=10000.0, factor=1.0, original=0.0, low=1.0, high=4.0, magnitude=1.0, scale=65536, **_):
    a = np.arange(rows, dtype=np.longdouble)[:, None] * frequencies(rot, np.longdouble(base), factor, original, low, high)
    return np.stack([np.cos(a), np.sin(a)], -1) * (magnitude * scale)


def table(hip, rows, rot, base=10000.0, factor=1.0, original=0.0, low=1.0, high=4.0, magnitude=1.0, scale=65536, **_):
    p = hip.malloc(max(16, 4 * rows * rot))
    hip.call("zk_rope_table", c_void_p(p), c_uint(rows), c_uint(rot), c_double(base), c_double(factor), c_double(original), c_double(low), c_double(high), c_double(magnitude), c_uint(scale), None)
    t = hip.download(p, (rows, rot // 2, 2), np.int32)
    hip.free(p)
    return t


@pytest.mark.parametrize("rows,rot", [(1, 2), (300, 64), (2048, 128), (5, 250)])
@pytest.mark.parametrize("how", [{}, {"base": 500000.0, "factor": 8.0, "original": 1024.0, "high": 4.0}, {"factor": 4.0, "magnitude": 1.1386}, {"scale": 1 << 30, "base": 1.5}, {"original": 32.0, "low": 0.0, "high": 1.0, "factor": 0.5}])
def test_rope_table(hip, rows, rot, how):
    """Every entry is the nearest integer.  An angle carries a relative error of some 2^-50 (the power and two products in double precision), 2048 positions a tenth of a
    2^-39: times the scale that is below 2^-8 at 2^30 and nothing at 2^16, so an entry may only be the other neighbour of a value within that of a half."""
    got, exp = table(hip, rows, rot, **how), exact_table(rows, rot, **how)
    slack = rows * 2.0 ** -50 * how.get("scale", 65536) * how.get("magnitude", 1.0) + 1e-9
    assert (np.abs(got - exp) <= 0.5 + slack).all()


def test_rope_table_of_far_positions(hip):
    got, exp = table(hip, 131072, 8), exact_table(131072, 8)
    assert (np.abs(got - exp) <= 0.5 + 131072 * 2.0 ** -50 * 65536 + 1e-9).all()


@pytest.mark.parametrize("change,text", [({"rot": 3}, "odd part"), ({"base": 1.0}, "base"), ({"base": float("nan")}, "base"), ({"factor": 0.0}, "factor"), ({"original": -1.0}, "original"),
                                         ({"original": 10.0, "low": 4.0}, "low < high"), ({"scale": 0}, "scale"), ({"scale": 1 << 30, "magnitude": 1.5}, "2^30")])
def test_rope_table_refusals(hip, change, text):
    with pytest.raises(RuntimeError, match=text.replace("^", r"\^")):
        table(hip, 4, **{"rot": 8, **change})


@pytest.mark.parametrize("heads,tokens,dim", [(1, 1, 1), (3, 5, 7), (1, 1, 1000), (4, 33, 16)])
@pytest.mark.parametrize("sf", [(1, 1), (1 << 20, 1 << 20), (1000, 3)])
def test_i32_from_heads(hip, heads, tokens, dim, sf):
    rng = np.random.default_rng(heads + tokens + dim)
    v = rng.integers(-(1 << 30), 1 << 30, (heads, tokens, dim)) * (1 if sf[0] == 1 else sf[0] // 2 * sf[1])      # wraps for the second factors: any 64 bits
    v[0, 0, 0] = 0
    p, o, f = hip.upload(ref.elements(v)), hip.malloc(4 * v.size), hip.malloc(16)

    def call(v):
        hip.call("zk_memcpy_h2d", c_void_p(p), ref.elements(v), c_size_t(32 * v.size), None)
        hip.call("zk_memset", c_void_p(f), c_int(0), c_size_t(4), None)
        hip.call("zk_i32_from_heads", c_void_p(o), c_void_p(p), c_uint(heads), c_uint(tokens), c_uint(dim), c_uint(sf[0]), c_uint(sf[1]), c_void_p(f), None)
        return hip.download(o, (tokens, heads, dim), np.int32), int(hip.download(f, (1,), np.uint32)[0])

    most = 1 << 62
    for x in (v, v % most - most // 2 if sf[0] > 1 else v):
        got, flag = call(x)
        exp = ref.quotient(ref.quotient(x, sf[0]), sf[1]).swapaxes(0, 1)
        fits = (np.abs(x.swapaxes(0, 1)) <= most) & (x.swapaxes(0, 1) != -(1 << 63)) & (exp == exp.astype(np.int32))
        assert flag == (0 if fits.all() else ref.RANGE) and (got == exp)[fits].all()
    for wide in ((1 << 62) + 1, -(1 << 63), 1 << 64, -(1 << 100)):          # no integers of 63 bits
        v = v.astype(object)
        v[-1, -1, -1] = wide
        assert call(v)[1] == ref.RANGE
    for x in (p, o, f):
        hip.free(x)


ROPES = [None, {}, {"dim": 8, "neighbours": 1, "first": 5, "factor": 4.0, "original": 16.0, "magnitude": 1.1, "scale": 1 << 12}]


@pytest.mark.parametrize("head_group", [0, 1, 2])
@pytest.mark.parametrize("rope", ROPES)
def test_values_equal_the_proved_layer(pv, head_group, rope):
    """The proof's output is the oracle's where there are no positions; the values' is the proof's, with the layer's own tokens and after other numbers of them."""
    orc = load_oracle()
    cu, cf = layercfg.tiny(open_weights=True, head_group=head_group)
    ws = layercfg.tiny_weights(7, cu)
    S, E = int(cu[0]), int(cu[1])
    X = np.round(np.random.default_rng(17).normal(0, 1, (S, E)) * 256).astype(np.int32)
    layer = pv.layer_create(cu, cf, ws, 1)
    if rope is not None:
        set_rope(pv, layer, **rope)
    for tokens in (1, 3, 40):
        values(pv, layer, np.tile(X, (3, 1))[:tokens])
    got = values(pv, layer, X, repeats=3)
    pv.seed(5)
    out, _ = pv.layer_run(layer, pv.from_i32(X))
    assert (got == out.host()).all()
    assert (values(pv, layer, X) == got).all()
    pv.layer_free(layer)
    if rope is None:
        exp = np.zeros((S * E, 8), np.uint32)
        orc.orc_seed(5)
        orc_check(orc.orc_layer(cu, cf, *ws, 1, X, exp, None))
        assert (got == exp).all()


def test_values_of_a_wider_layer_with_kept_weights(pv):
    """Random weights as make_random_layer_weights keeps them (planes shared with the proof's products), widths that are no powers of two, more than 32 tokens: the kernels for many rows"""
    # weights of 0.02 at scale 2^16 and activations at 2^8: projections of some 256 * 1311 * 160^0.5 / 2^12 = 1000, scores of 2^25 to 2^28, no table longer than the tensor it serves
    cu, cf = layercfg.pack(64, 160, 4, 352, 1 << 12, 1 << 12, 1 << 8, [1 << 4, 1 << 12, 1 << 14], 1, 0, 1 << 20, [1 << 8, 1 << 8], -(1 << 13), 1 << 14, 256.0, value_scale=256.0, open_weights=False,
                           head_group=4)
    layer = pv.layer_create_random(cu, cf, 3, 1)
    set_rope(pv, layer)
    X = np.round(np.random.default_rng(1).normal(0, 1, (64, 160)) * 256).astype(np.int32)
    got = values(pv, layer, X)
    pv.seed(9)
    out, _ = pv.layer_run(layer, pv.from_i32(X))
    assert (got == out.host()).all() and (values(pv, layer, X) == got).all()
    with pytest.raises(RuntimeError, match="tokens x embed_dim"):
        values(pv, layer, X[:1, :5])
    with pytest.raises(RuntimeError, match="LayerValues: a value does not fit"):
        values(pv, layer, np.concatenate([np.full((1, 160), (1 << 31) - 1, np.int32), X[1:]]))          # the other rows' attention pushes some of the first over the edge
    set_rope(pv, layer, dim=41)
    with pytest.raises(RuntimeError, match="within the head"):
        values(pv, layer, X)
    pv.layer_free(layer)


@pytest.mark.parametrize("base", [-10000.0, 0.5, float("nan")])
def test_a_base_that_is_none_is_refused(pv, base):
    cu, cf = layercfg.tiny(open_weights=False)
    layer = pv.layer_create(cu, cf, layercfg.tiny_weights(1, cu), 1)
    set_rope(pv, layer, base=base)
    with pytest.raises(RuntimeError, match="the base must lie above 1"):
        values(pv, layer, np.zeros((int(cu[0]), int(cu[1])), np.int32))
    pv.layer_free(layer)


@pytest.mark.parametrize("head_group", [0, 1, 2])
@pytest.mark.parametrize("rope", ROPES[1:])
def test_positions_in_the_proof_are_those_of_rotated_queries_and_keys(pv, hip, head_group, rope):
    """The attention proof with positions is the oracle's for queries and keys that were rotated before."""
    orc = load_oracle()
    cu, cf = layercfg.tiny(open_weights=False, head_group=head_group)
    S, E, H = int(cu[0]), int(cu[1]), int(cu[2])
    d, first = E // H, rope.get("first", 0)
    rng = np.random.default_rng(8)
    Q, K, V = (np.round(rng.normal(0, 1.0, (S, E)) * 256).astype(np.int32) for _ in range(3))
    rot = rope.get("dim") or d
    t = table(hip, first + S, rot, **rope)
    turn = lambda x: ref.rope(x.reshape(S, H, d), t, np.arange(first, first + S), rot, rope.get("neighbours", 0), rope.get("scale", 65536)).reshape(S, E)
    exp = np.zeros((S * E, 8), np.uint32)
    orc.orc_seed(31)
    orc.orc_transcript_clear()
    orc_check(orc.orc_attn_block(cu, cf, 0, ref.elements(turn(Q)), ref.elements(turn(K)), ref.elements(V), exp, None))
    exp_t = orc_transcript(orc)
    layer = pv.layer_create(cu, cf, layercfg.tiny_weights(1, cu), 1)
    set_rope(pv, layer, **rope)
    pv.seed(31)
    pv.transcript_begin()
    q, k, v = (pv.from_i32(x) for x in (Q, K, V))
    out = pv.H(pv.lib.zkp_layer_attention(c_void_p(layer), c_void_p(q.h), c_void_p(k.h), c_void_p(v.h)))
    pv.lib.zkp_transcript_end()
    got_t = pv.transcript()
    pv.layer_free(layer)
    assert (out.host() == exp).all()
    assert got_t.shape == exp_t.shape and (got_t == exp_t).all()


def test_self_attn_executable_with_positions(tmp_path, hip):
    """ZKLLM_LAYER_CONFIG's rope_* keys: what the executable writes for queries and keys is what it writes, without them, for queries and keys that were rotated before; as one head it refuses."""
    cu, _ = layercfg.tiny()
    S, E, H = int(cu[0]), int(cu[1]), int(cu[2])
    d = E // H
    rng = np.random.default_rng(12)
    Q, K, V = (np.round(rng.normal(0, 1.0, (S, E)) * 256).astype(np.int32) for _ in range(3))
    how = {"base": 1000.0, "dim": 12, "neighbours": 1, "factor": 2.0, "original": 64.0, "low": 0.5, "high": 3.0, "magnitude": 1.25, "first": 3, "scale": 1 << 14}
    t = table(hip, 3 + S, 12, **{k: v for k, v in how.items() if k != "dim"})
    turn = lambda x: ref.rope(x.reshape(S, H, d), t, np.arange(3, 3 + S), 12, 1, 1 << 14).reshape(S, E).astype(np.int32)
    keys = "," + ",".join(f"rope_{k}={v}" for k, v in how.items())
    outs = []
    for config, q, k in ((TINY_ENV + keys, Q, K), (TINY_ENV, turn(Q), turn(K))):
        for n, x in zip("QKV", (q, k, V)):
            x.tofile(tmp_path / f"temp_{n}.bin")
        proof = tmp_path / f"p{len(outs)}.proof"
        run(tmp_path, 55, proof, "self-attn", "attn", "unused.bin", S, E, tmp_path, "layer-0", "out.bin", config=config, extra_env={"ZKLLM_ATTN_HEADS": "2", "ZKLLM_ATTN_HEAD_GROUP": "2"})
        outs.append((open(tmp_path / "out.bin", "rb").read(), open(proof, "rb").read()))
    assert outs[0] == outs[1]
    with pytest.raises(AssertionError, match="positions need heads"):
        run(tmp_path, 55, None, "self-attn", "attn", "unused.bin", S, E, tmp_path, "layer-0", "out.bin", config=TINY_ENV + keys)

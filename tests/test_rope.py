"""Frequencies of scaled rotary positions, and the refusals of the rotary and
block-scaled cache calls (no GPU: nothing is launched)."""
import ctypes
import math

import numpy as np
import pytest
import torch

import nvkv
import nvkv_oracle as O
from nvkv import NvkvError, ops
from nvkv._lib import (ERR_ALIGNMENT, ERR_INVALID_ARG, ERR_UNSUPPORTED, OK, RopeScaling, lib)

THETA, FACTOR, ORIG = 1e6, 4.0, 32768


def _plain(rot):
    return THETA ** (-2.0 * np.arange(rot // 2) / rot)


@pytest.mark.parametrize("rot", [2, 32, 64, 100, 128])
def test_frequencies(rot):
    """Every scaling against its formula; 1e-13: a handful of f64 roundings and
    a pow accurate to a few ulps."""
    f = _plain(rot)
    i = np.arange(rot // 2)

    def got(kind, **kw):
        x, a = ops.rope_frequencies(rot, THETA, kind, FACTOR, ORIG, **kw)
        return x.numpy()[:rot // 2], a

    x, a = got("plain")
    np.testing.assert_allclose(x, f, rtol=1e-13)
    assert a == 1.0
    np.testing.assert_allclose(got("linear")[0], f / FACTOR, rtol=1e-13)
    base = THETA * FACTOR ** (rot / (rot - 2)) if rot > 2 else THETA
    np.testing.assert_allclose(got("ntk")[0], base ** (-2.0 * i / rot), rtol=1e-13)
    x, a = got("yarn")
    assert a == pytest.approx(0.1 * math.log(FACTOR) + 1, rel=1e-15)
    turns = ORIG * f / (2 * math.pi)  # over the original context
    np.testing.assert_allclose(x[turns > 32 * 4], f[turns > 32 * 4], rtol=1e-13)
    np.testing.assert_allclose(x[turns < 0.25], f[turns < 0.25] / FACTOR, rtol=1e-13)
    assert np.all(x <= f * (1 + 1e-13)) and np.all(x >= f / FACTOR * (1 - 1e-13))
    x, _ = got("bands")
    keep = np.clip((turns - 1) / 3, 0, 1)
    np.testing.assert_allclose(x, f / FACTOR * (1 - keep) + f * keep, rtol=1e-13)
    assert got("yarn", attention_factor=1.25)[1] == 1.25


def test_yarn_ramp():
    """The pairs between the two turn counts: a linear ramp over the index."""
    rot = 128
    x = ops.rope_frequencies(rot, THETA, "yarn", FACTOR, ORIG)[0].numpy()
    f = _plain(rot)

    def pair(turns):
        return rot * math.log(ORIG / (turns * 2 * math.pi)) / (2 * math.log(THETA))
    lo, hi = math.floor(pair(32.0)), math.ceil(pair(1.0))
    share = np.clip((np.arange(64) - lo) / (hi - lo), 0, 1)
    np.testing.assert_allclose(x, f / FACTOR * share + f * (1 - share), rtol=1e-13)


@pytest.mark.parametrize("kw", [dict(rot_dim=0), dict(rot_dim=7), dict(theta=0.0),
                                dict(theta=float("inf")), dict(scaling="linear", factor=0.5),
                                dict(scaling="yarn", factor=2.0),
                                dict(scaling="yarn", factor=2.0, original_max_position=64,
                                     beta_fast=1.0, beta_slow=32.0),
                                dict(scaling="bands", factor=2.0, original_max_position=64,
                                     low_freq_factor=4.0, high_freq_factor=4.0),
                                dict(scaling="dynamic")])
def test_frequencies_refused(kw):
    args = dict(dict(rot_dim=64, theta=1e4), **kw)
    with pytest.raises(NvkvError):
        ops.rope_frequencies(**args)


def test_frequencies_null_and_unknown_type():
    out = (ctypes.c_double * 32)()
    a = ctypes.c_double()
    assert lib.nvkv_rope_frequencies(64, 1e4, None, out, ctypes.byref(a)) == OK
    assert lib.nvkv_rope_frequencies(64, 1e4, None, None, ctypes.byref(a)) == ERR_INVALID_ARG
    sc = RopeScaling(9, 2.0, 64, 32.0, 1.0, 1.0, 4.0, 0.0)
    assert lib.nvkv_rope_frequencies(64, 1e4, ctypes.byref(sc), out,
                                     ctypes.byref(a)) == ERR_UNSUPPORTED


def P(x):
    return ctypes.c_void_p(x)


BIG = 1 << 32


def _rope(**kw):
    a = dict(q=P(BIG), qs=256, k=P(2 * BIG), ks=256, qo=P(3 * BIG), qos=256, ko=P(4 * BIG),
             kos=256, T=4, hq=2, hkv=2, d=128, pos=P(5 * BIG), f=P(6 * BIG), rot=64, a=1.0,
             inter=0, dt=1)
    a.update(kw)
    return lib.nvkv_rope(a["q"], a["qs"], a["k"], a["ks"], a["qo"], a["qos"], a["ko"], a["kos"],
                         a["T"], a["hq"], a["hkv"], a["d"], a["pos"], a["f"], a["rot"], a["a"],
                         a["inter"], a["dt"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=2), ERR_UNSUPPORTED), (dict(T=-1), ERR_INVALID_ARG), (dict(rot=7), ERR_UNSUPPORTED),
    (dict(rot=130), ERR_UNSUPPORTED), (dict(rot=0), ERR_UNSUPPORTED), (dict(d=2048), ERR_UNSUPPORTED),
    (dict(hq=0, hkv=0), ERR_INVALID_ARG), (dict(q=None), ERR_INVALID_ARG),
    (dict(ko=None), ERR_INVALID_ARG), (dict(pos=None), ERR_INVALID_ARG),
    (dict(f=None), ERR_INVALID_ARG), (dict(qs=255), ERR_INVALID_ARG),
    (dict(kos=128), ERR_INVALID_ARG), (dict(q=P(BIG + 1)), ERR_ALIGNMENT),
    (dict(f=P(BIG + 4)), ERR_ALIGNMENT),
    (dict(qo=P(BIG + 16)), ERR_INVALID_ARG),           # shifted onto its own input
    (dict(qo=P(BIG), qos=512), ERR_INVALID_ARG),       # the same start, other rows
    (dict(qo=P(2 * BIG)), ERR_INVALID_ARG),            # onto k
    (dict(qo=P(4 * BIG + 256)), ERR_INVALID_ARG),      # onto k_out
])
def test_rope_refused(kw, code):
    assert _rope(**kw) == code
    assert lib.nvkv_last_error()


def test_rope_nothing_to_do():
    assert _rope(T=0, q=None, k=None, qo=None, ko=None, pos=None, f=None) == OK


def _append(**kw):
    a = dict(q=P(BIG), qs=768, k=P(BIG + 512), ks=768, v=P(BIG + 1024), vs=768, T=4, hq=2, hkv=2,
             d=128, pos=P(5 * BIG), f=P(6 * BIG), rot=128, a=1.0, inter=0, qw=None, kw=None,
             eps=1e-6, qo=P(7 * BIG), kc=P(8 * BIG), vc=P(9 * BIG), sc=P(10 * BIG),
             slots=P(11 * BIG), nb=4, page=256, dt=1)
    a.update(kw)
    return lib.nvkv_rope_append(a["q"], a["qs"], a["k"], a["ks"], a["v"], a["vs"], a["T"],
                                a["hq"], a["hkv"], a["d"], a["pos"], a["f"], a["rot"], a["a"],
                                a["inter"], a["qw"], a["kw"], a["eps"], a["qo"], a["kc"], a["vc"],
                                a["sc"], a["slots"], a["nb"], a["page"], a["dt"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(dt=2), ERR_UNSUPPORTED), (dict(d=64), ERR_UNSUPPORTED), (dict(rot=12), ERR_UNSUPPORTED),
    (dict(rot=136), ERR_UNSUPPORTED), (dict(T=-1), ERR_INVALID_ARG), (dict(hkv=0), ERR_INVALID_ARG),
    (dict(nb=0), ERR_INVALID_ARG), (dict(page=24), ERR_UNSUPPORTED), (dict(k=None), ERR_INVALID_ARG),
    (dict(slots=None), ERR_INVALID_ARG), (dict(qo=None), ERR_INVALID_ARG),
    (dict(qw=P(BIG)), ERR_INVALID_ARG), (dict(ks=128), ERR_INVALID_ARG),
    (dict(qs=770), ERR_ALIGNMENT), (dict(kc=P(8 * BIG + 8)), ERR_ALIGNMENT),
    (dict(sc=P(10 * BIG + 4)), ERR_ALIGNMENT), (dict(q=P(BIG + 2)), ERR_ALIGNMENT),
    (dict(qo=P(BIG)), ERR_INVALID_ARG),        # dense rows over the fused buffer
    (dict(qo=P(BIG + 512)), ERR_INVALID_ARG),  # over k
    (dict(vc=P(8 * BIG)), ERR_INVALID_ARG),    # one pool for both
    (dict(vc=P(8 * BIG + 4 * 256 * 256 - 16)), ERR_INVALID_ARG),
    (dict(k=P(8 * BIG + 4096), ks=256), ERR_INVALID_ARG),  # rows of the pool itself
    (dict(qo=P(9 * BIG + 512)), ERR_INVALID_ARG),
])
def test_rope_append_refused(kw, code):
    assert _append(**kw) == code
    assert lib.nvkv_last_error()


def test_rope_append_nothing_to_do():
    assert _append(T=0, q=None, k=None, v=None, qo=None, slots=None, pos=None) == OK


def test_load_refused():
    def call(kc=P(BIG), sc=P(2 * BIG), slots=P(3 * BIG), n=4, hkv=2, d=128, nb=4, page=256,
             ko=P(4 * BIG), vo=P(5 * BIG), dt=1):
        return lib.nvkv_load_kvcache_fp8b(kc, kc, sc, slots, n, hkv, d, nb, page, ko, vo, dt, None)
    assert call(dt=2) == ERR_UNSUPPORTED
    assert call(d=64) == ERR_UNSUPPORTED
    assert call(page=8) == ERR_UNSUPPORTED
    assert call(n=-1) == ERR_INVALID_ARG
    assert call(hkv=0) == ERR_INVALID_ARG
    assert call(ko=None) == ERR_INVALID_ARG
    assert call(ko=P(4 * BIG + 8)) == ERR_ALIGNMENT
    assert call(vo=P(4 * BIG + 1024)) == ERR_INVALID_ARG  # onto k_out
    assert call(ko=P(BIG + 1024)) == ERR_INVALID_ARG      # into the pool
    assert call(vo=P(2 * BIG)) == ERR_INVALID_ARG         # onto the scales
    assert call(n=0, kc=None, sc=None, slots=None, ko=None, vo=None) == OK


def test_attention_fp8b_refused():
    def call(**kw):
        a = dict(q=P(BIG), qs=4 * 128, T=2, kc=P(2 * BIG), sc=P(3 * BIG), nb=8, out=P(4 * BIG),
                 cu=P(5 * BIG), bt=P(6 * BIG), bts=4, B=2, mq=1, mk=1000, hq=4, hkv=2, d=128,
                 page=256, sm=0.1, rows=0, ws=None, wsb=0, dt=1)
        a.update(kw)
        return lib.nvkv_paged_attention_fp8b(
            a["q"], a["qs"], a["T"], a["kc"], a["kc"], a["sc"], a["nb"], a["out"], a["cu"],
            a["cu"], a["bt"], a["bts"], a["B"], a["mq"], a["mk"], a["hq"], a["hkv"], a["d"],
            a["page"], a["sm"], 1, a["rows"], a["ws"], a["wsb"], a["dt"], None)
    assert call(dt=2) == ERR_UNSUPPORTED
    assert call(d=64) == ERR_UNSUPPORTED
    assert call(hq=34) == ERR_UNSUPPORTED  # group 17
    assert call(hq=3) == ERR_INVALID_ARG
    assert call(page=64) == ERR_UNSUPPORTED
    assert call(bts=3) == ERR_INVALID_ARG
    assert call(bt=None) == ERR_INVALID_ARG
    assert call(sm=0.0) == ERR_INVALID_ARG
    assert call(sm=float("nan")) == ERR_INVALID_ARG
    assert call(qs=4 * 128 + 4) == ERR_ALIGNMENT
    assert call(sc=P(3 * BIG + 8)) == ERR_ALIGNMENT
    assert call(nb=1 << 24, page=256) == ERR_UNSUPPORTED  # 2^32 cache rows
    assert call(rows=-1) == ERR_INVALID_ARG
    assert call(mk=(1 << 30) + 1, bts=1 << 23) == ERR_UNSUPPORTED
    assert call(out=P(BIG + 16)) == ERR_INVALID_ARG  # shifted onto q
    assert call(mq=17, rows=0) == ERR_INVALID_ARG    # prompts without their key count
    assert call(B=0) == OK
    assert call(T=0) == OK
    assert call(mq=0) == OK


def test_python_calls_refuse_host_tensors_and_bad_shapes():
    q = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    pos = torch.zeros(4, dtype=torch.int64)
    f = torch.ones(64, dtype=torch.float64)
    pool = torch.zeros(2, 256, 2, 128, dtype=torch.uint8)
    sc = torch.zeros(2, 2, 16, 2)
    for call in (lambda: nvkv.rope(q, q, pos, f),
                 lambda: nvkv.rope(q, q, pos[:3], f),
                 lambda: nvkv.rope(q, q, pos, f.float()),
                 lambda: nvkv.rope(q, q[:3], pos, f),
                 lambda: nvkv.rope(q.transpose(1, 2), None, pos, f),
                 lambda: nvkv.rope_append(q, q, q, pos, f, pool, pool, pos, kv_scale=sc),
                 lambda: nvkv.rope_append(q, q, q, pos, f, pool, pool, pos),
                 lambda: nvkv.rope_append(q, q, q, pos, f, pool, pool, pos, kv_scale=sc[:, :, :8]),
                 lambda: nvkv.load_kvcache_fp8b(pool, pool, sc, pos),
                 lambda: nvkv.load_kvcache_fp8b(pool, pool, sc, pos.int())):
        with pytest.raises(NvkvError):
            call()


def test_oracle_exponent_is_the_least():
    for amax in (1e-40, 2.0 ** -92, 0.3, 1.0, 1.75, 1.7500001, 447.9, 448.0, 448.1, 3e38):
        e = O.fp8b_exponent(amax)
        assert amax <= 448 * 2.0 ** e
        assert e == O.FP8B_MIN_EXP or amax > 448 * 2.0 ** (e - 1)
    assert O.fp8b_exponent(0.0) == O.FP8B_MIN_EXP

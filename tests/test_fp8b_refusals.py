"""Overlaps and sizes that nvkv_rope, nvkv_rope_append, nvkv_load_kvcache_fp8b and
nvkv_paged_attention_fp8b refuse before anything is launched: a buffer that a call
writes may not share memory with another of its buffers (but for the rows that the
header allows), metadata among them."""
import ctypes

import pytest

import nvkv  # noqa: F401
from nvkv._lib import lib
from test_rope import BIG, ERR_INVALID_ARG, OK, P, _append, _rope

POS, FREQ, KC, VC, SC, SLOTS = (i * BIG for i in (5, 6, 8, 9, 10, 11))


@pytest.mark.parametrize("kw", [
    dict(qo=P(POS - 512)),              # its last row onto the positions
    dict(ko=P(POS + 24 - 24 % 16)),     # onto their last entries
    dict(qo=P(FREQ + 8 * 24)),          # onto the frequencies
])
def test_rope_output_over_metadata(kw):
    assert _rope(**kw) == ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [
    dict(qo=P(POS)), dict(qo=P(FREQ + 256)), dict(qo=P(SLOTS + 16)),
    dict(qw=P(12 * BIG), kw=P(13 * BIG), qo=P(13 * BIG + 128)),
    dict(qo=P(SC)), dict(qo=P(SC + 4 * 2 * 16 * 8 - 16)),      # over the scales
    dict(sc=P(KC + 1024)), dict(sc=P(VC - 64)),                # scales in a cache
    dict(sc=P(BIG + 512)),                                     # scales over k
    dict(sc=P(POS)), dict(sc=P(SLOTS + 8)), dict(sc=P(FREQ)),
    dict(pos=P(KC)), dict(slots=P(VC + 64)), dict(f=P(KC + 8)),
    dict(qw=P(KC), kw=P(13 * BIG)),
    dict(sc=None, slots=P(KC)),                                # the dtype pool
])
def test_append_output_over_metadata(kw):
    assert _append(**kw) == ERR_INVALID_ARG


@pytest.mark.parametrize("nb", [1 << 61, (1 << 63) - 1, (1 << 63) // (256 * 256) + 1])
def test_pool_sizes_past_64_bits(nb):
    assert _append(nb=nb) == ERR_INVALID_ARG
    assert lib.nvkv_load_kvcache_fp8b(P(BIG), P(BIG), P(2 * BIG), P(3 * BIG), 4, 2, 128, nb, 256,
                                      P(4 * BIG), P(5 * BIG), 1, None) == ERR_INVALID_ARG


def test_load_output_over_slots():
    assert lib.nvkv_load_kvcache_fp8b(P(BIG), P(BIG), P(2 * BIG), P(3 * BIG), 4, 2, 128, 4, 256,
                                      P(4 * BIG), P(3 * BIG + 16), 1, None) == ERR_INVALID_ARG


def _attend(**kw):
    a = dict(q=P(BIG), qs=4 * 128, T=2, kc=P(2 * BIG), vc=P(3 * BIG), sc=P(4 * BIG), nb=8,
             out=P(5 * BIG), cq=P(6 * BIG), ck=P(7 * BIG), bt=P(8 * BIG), ws=P(9 * BIG))
    a.update(kw)
    n = ctypes.c_size_t(0)
    assert lib.nvkv_paged_attention_fp8b_workspace_size(2, 4, 2, 128, 1, 1000, 0,
                                                        ctypes.byref(n)) == OK
    return lib.nvkv_paged_attention_fp8b(
        a["q"], a["qs"], a["T"], a["kc"], a["vc"], a["sc"], a["nb"], a["out"], a["cq"], a["ck"],
        a["bt"], 4, 2, 1, 1000, 4, 2, 128, 256, 0.1, 1, 0, a["ws"], n.value, 1, None)


POOL = 8 * 256 * 2 * 128  # bytes of a cache


@pytest.mark.parametrize("kw", [
    dict(out=P(2 * BIG + POOL - 16)), dict(out=P(3 * BIG)), dict(out=P(4 * BIG + 64)),
    dict(out=P(6 * BIG)), dict(out=P(7 * BIG - 2032)), dict(out=P(8 * BIG + 16)),
    dict(ws=P(BIG)), dict(ws=P(2 * BIG + 256)), dict(ws=P(3 * BIG)), dict(ws=P(4 * BIG)),
    dict(ws=P(5 * BIG + 1024)), dict(ws=P(6 * BIG)), dict(ws=P(7 * BIG)), dict(ws=P(8 * BIG)),
])
def test_attention_output_or_workspace_over_inputs(kw):
    assert _attend(**kw) == ERR_INVALID_ARG
    assert lib.nvkv_last_error()


@pytest.mark.parametrize("theta", [1.0, 0.5])
def test_yarn_needs_falling_frequencies(theta):
    """Its ramp runs from fast pairs to slow ones: theta <= 1 has none."""
    out = (ctypes.c_double * 32)()
    a = ctypes.c_double()
    sc = nvkv._lib.RopeScaling(nvkv._lib.ROPE_YARN, 4.0, 4096, 32.0, 1.0, 1.0, 4.0, 0.0)
    assert lib.nvkv_rope_frequencies(64, theta, ctypes.byref(sc), out,
                                     ctypes.byref(a)) == ERR_INVALID_ARG

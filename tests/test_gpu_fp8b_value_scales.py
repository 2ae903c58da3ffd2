"""Block-scaled decode where the scales of V differ by many powers of two: a key
whose values are small or zero counts in the softmax's sum as any other.

Tolerance (one rounding of the result, and of sum p |v|): scores are sums of exact
products in f32, at most 60 in the exponent here, so their rounding is 2^-18 of a
weight; the approximate exponentials add 2^-21; weights keep 12 significant bits,
2^-13 each, down to 2^-17 of a row's largest, and below that lose at most 2^-30 of
it each, 2^-15 for 20000 keys: 2^-12 covers them."""
import numpy as np
import pytest
import torch

import nvkv
import nvkv_oracle as O
from fp8b import D, G, attend64, check_attention, empty_pool, filled, slots_of, tables
from helpers import cu
from nvkv import ops

pytestmark = pytest.mark.gpu

ERR = 2.0 ** -12
LOG2E = 1.4426950408889634


def _pool(k, v, hkv, P=256, seed=0):
    """A pool of one sequence with these rows [L, Hkv, D], and its f64 values."""
    L = k.size(0)
    bt, nb = tables([L], P, seed)
    pool = empty_pool(nb, P, hkv)
    s = slots_of(bt, 0, 0, L, P)
    ops.rope_append(None, k.cuda(), v.cuda(), torch.zeros(L, dtype=torch.int64, device="cuda"),
                    torch.ones(4, dtype=torch.float64, device="cuda"), pool[0], pool[1],
                    torch.from_numpy(s).cuda(), kv_scale=pool[2])
    torch.cuda.synchronize()
    c, sc = [t.cpu().numpy() for t in pool[:2]], pool[2].cpu().numpy()
    rows = [O.e4m3_decode(x[s // P, s % P]).astype(np.float64) *
            sc[s // P, :, s % P // G, w][..., None].astype(np.float64) for w, x in enumerate(c)]
    return pool, torch.from_numpy(bt).cuda(), rows


def _attend(q, pool, bt, L):
    n = q.size(0)
    out = nvkv.paged_attention_fp8b(q, *pool, cu([n]), cu([L]), bt, n, L, D ** -0.5)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    return out


@pytest.mark.parametrize("mode", ["equal", "random", "seesaw"])
@pytest.mark.parametrize("L", [40, 700, 20000])
@pytest.mark.parametrize("new,hq,hkv", [(1, 4, 1), (1, 16, 2), (4, 8, 2), (2, 16, 1)])
def test_value_scales_far_apart(new, hq, hkv, L, mode):
    """Blocks of V from 2^-90 to 2^90, a quarter of them zero.  equal: every key
    weighs the same; seesaw: small values have large weights and the other way
    round, so that all contribute."""
    g = torch.Generator().manual_seed(L + hq)
    nblk = (L + G - 1) // G
    gain = torch.randint(-90, 91, (nblk,), generator=g)
    if mode == "seesaw":  # 2^gain goes with a score of -gain / 3 in log2
        gain = gain // 2
    block = torch.arange(L) // G
    v = torch.randn(L, hkv, D, generator=g) * torch.exp2(gain.float())[block][:, None, None]
    v[(torch.rand(nblk, generator=g) < 0.25)[block]] = 0.0
    q = torch.randn(new, hq, D, generator=g)
    k = torch.randn(L, hkv, D, generator=g)
    if mode == "equal":
        q.zero_()
    elif mode == "seesaw":
        q.fill_(1.0)
        k[:] = (-gain.float() / 3 / LOG2E / D ** 0.5)[block][:, None, None]
    q = q.bfloat16().cuda()
    pool, bt, rows = _pool(k.bfloat16(), v.bfloat16(), hkv, seed=L)
    check_attention(_attend(q, pool, bt, L), q, [rows], [new], [L], D ** -0.5, ERR)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L", [17, 700, 32785])
def test_zero_values_count_in_the_sum(L, dtype):
    """The first key has a large value, the others (in other blocks) none: each of
    them still takes its share of the weight, 1 / L with equal scores and, with the
    first key 2^20 above them, 2^-20 of it."""
    big = 2.0 ** 40 if dtype == torch.bfloat16 else 65504.0
    hq, hkv = 4, 1
    v = torch.zeros(L, hkv, D)
    v[0] = big
    k = torch.zeros(L, hkv, D)
    k[0] = 1.0
    pool, bt, rows = _pool(k.to(dtype), v.to(dtype), hkv, seed=L)
    q = torch.zeros(1, hq, D)
    q[0, 1:] = 20 / LOG2E / D ** 0.5  # heads 1 .. : scores of 20 and 0 in log2
    q = q.to(dtype).cuda()
    out = _attend(q, pool, bt, L)
    check_attention(out, q, [rows], [1], [L], D ** -0.5, ERR)
    alone = rows[1][0, 0, 0]
    assert abs(float(out[0, 0, 0]) / alone * L - 1) < torch.finfo(dtype).eps


@pytest.mark.parametrize("lead", [30, 100, 120])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("L,hq", [(300, 4), (300, 16), (9000, 8)])
def test_sink_of_zero_values(L, hq, first, lead):
    """A key whose values are zero takes all but 2^-lead of the weight; the others'
    values, 2^lead times as large, are the answer.  Scores of up to 120 in
    the exponent: an f32 sum of 128 products of one sign is off by at most 128 x 60 x
    2^-24 there, 2^-11.6 of a weight, and weights keep 2^-13: 2^-11 in all."""
    hkv = 1
    g = torch.Generator().manual_seed(L)
    at = slice(0, 16) if first else slice((L - 1) // 16 * 16, L)
    v = torch.randn(L, hkv, D, generator=g) * 2.0 ** lead
    v[at] = 0.0
    k = torch.zeros(L, hkv, D)
    k[at.start] = 8.0
    q = torch.full((1, hq, D), lead / 8 / LOG2E / D ** 0.5).bfloat16().cuda()
    pool, bt, rows = _pool(k.bfloat16(), v.bfloat16(), hkv, seed=L)
    check_attention(_attend(q, pool, bt, L), q, [rows], [1], [L], D ** -0.5, 2.0 ** -11)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("q_gain,k_gain,v_gain", [(8.0, 1.0, 1.0), (1e-3, 1e3, 1e-4),
                                                  (1.0, 1.0, 3e4), (30.0, 1.0, 1e-30)])
def test_peaked_softmaxes_and_far_ranges(q_gain, k_gain, v_gain, dtype):
    """Scores of a few hundred, keys and values far from 1; what is compared is what
    the kernel wrote, with no term but its one rounding and the weights'.  A score of
    up to 400 in the exponent is joined from three pieces' products in four steps
    each: 16 roundings of 2^-24 x 400 are 2^-11.4 of a weight; weights keep 2^-12: 2^-10
    covers them."""
    if dtype == torch.float16 and not 1e-4 <= v_gain <= 1e3:
        v_gain = 1e-3 if v_gain < 1 else 50.0  # (f16 holds up to 65504)
    k_lens = [1, 100, 1300, 4000]
    hq, hkv = 8, 2
    g = torch.Generator().manual_seed(12)
    q = (torch.randn(4, hq, D, generator=g) * q_gain).to(dtype).cuda()
    if dtype == torch.float16 and k_gain > 100:
        k_gain = 100.0
    pool, bt, rows = filled(k_lens, hkv, seed=11, dtype=dtype, k_gain=k_gain, v_gain=v_gain)
    out = nvkv.paged_attention_fp8b(q, *pool, cu([1] * 4), cu(k_lens), bt, 1, 4000, D ** -0.5)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    got, qn = out.double().cpu().numpy(), q.double().cpu().numpy()
    f = torch.finfo(dtype)
    for b in range(4):
        want, bound = attend64(qn[b:b + 1], *rows[b], D ** -0.5)
        tol = abs(want) * f.eps / 2 * (1 + 2.0 ** -10) + bound * 2.0 ** -10 + f.smallest_normal * f.eps
        assert (abs(got[b:b + 1] - want) <= tol).all(), k_lens[b]

"""Prompts beside memory that holds no keys: rows behind a sequence's last key
(the next sequence's, stale pages, workspace that was never written) may hold NaN
and infinities, and no query sees them.

Every form of the prefill kernel is run: the model-dtype pool, contiguous K/V, the
row-scaled and the block-scaled e4m3 pools, head pairs and single heads.
Tolerance: weights are rounded to the dtype (eps / 2), some exponentials come from
a polynomial (7.5e-5), sums are f32: eps / 2 + 2^-12 of sum p |v|, and one rounding
of the result."""
import numpy as np
import pytest
import torch

import nvkv
from fp8b import D, check_attention, filled, slots_of, tables
from helpers import cu
from nvkv import ops
from nvkv._lib import DEVERR_SEQLEN

pytestmark = pytest.mark.gpu

Q_LENS, K_LENS = [130, 1, 200, 64], [130, 300, 701, 127]  # (one single row beside the prompts)
NAN_BITS = 0xFF  # as bf16, f16, f32 and e4m3 a NaN


def _err(dtype):
    return torch.finfo(dtype).eps / 2 + 2.0 ** -12


def _q(hq, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(sum(Q_LENS), hq, D, generator=g).to(dtype).cuda()


def _poisoned(n):
    return torch.full((n,), NAN_BITS, dtype=torch.uint8, device="cuda")


def _prompts():
    return sum(k for a, k in zip(Q_LENS, K_LENS) if a > 1)


def _rows(hkv, seed, dtype):
    g = torch.Generator().manual_seed(seed)
    return [[torch.randn(L, hkv, D, generator=g).to(dtype) for _ in "kv"] for L in K_LENS]


def _f64(rows):
    return [[t.double().numpy() for t in kv] for kv in rows]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 1), (12, 1)])
@pytest.mark.parametrize("spare", [0, 1000])
def test_block_scaled_prompts_in_unwritten_workspace(hq, hkv, spare, dtype):
    """A workspace full of NaN, prompt_kv_tokens at and above the sum."""
    pool, bt, rows = filled(K_LENS, hkv, seed=hq, dtype=dtype)
    q = _q(hq, dtype, hq)
    for causal in (True, False):
        ws = _poisoned(nvkv.workspace_size_fp8b(4, hq, hkv, 200, 701, _prompts() + spare))
        out = nvkv.paged_attention_fp8b(q, *pool, cu(Q_LENS), cu(K_LENS), bt, 200, 701, D ** -0.5,
                                        prompt_kv_tokens=_prompts() + spare, workspace=ws,
                                        causal=causal)
        torch.cuda.synchronize()
        assert nvkv.device_error() == 0
        check_attention(out, q, rows, Q_LENS, K_LENS, D ** -0.5, _err(dtype), causal)


def test_block_scaled_prompt_that_does_not_fit_in_unwritten_workspace():
    """The prompt left out is recorded and its rows stay; those before it are right."""
    pool, bt, rows = filled(K_LENS, 2, seed=3)
    q = _q(4, torch.bfloat16, 3)
    ws = _poisoned(nvkv.workspace_size_fp8b(4, 4, 2, 200, 701, 800))
    out = torch.full_like(q, 7.0)
    nvkv.device_error()
    nvkv.paged_attention_fp8b(q, *pool, cu(Q_LENS), cu(K_LENS), bt, 200, 701, D ** -0.5,
                              prompt_kv_tokens=800, workspace=ws, out=out)
    torch.cuda.synchronize()
    assert nvkv.device_error() == DEVERR_SEQLEN and bool((out[131:] == 7).all())
    check_attention(out[:131], q[:131], rows[:2], Q_LENS[:2], K_LENS[:2], D ** -0.5,
                    _err(q.dtype))


@pytest.mark.parametrize("what", [0, 1])
def test_block_scaled_nan_prompt_stays_alone(what):
    """NaN codes in a prompt's first K (0) or V (1) rows: the prompts before and
    behind it do not see them."""
    pool, bt, rows = filled(K_LENS, 2, seed=4)
    pool[what][int(bt[2, 0]), :3] = 0x7F
    q = _q(8, torch.bfloat16, 4)
    out = nvkv.paged_attention_fp8b(q, *pool, cu(Q_LENS), cu(K_LENS), bt, 200, 701, D ** -0.5,
                                    prompt_kv_tokens=_prompts())
    torch.cuda.synchronize()
    assert bool(out[131:331].isnan().any())
    keep = [0, 1, 3]
    for b in keep:
        s = slice(sum(Q_LENS[:b]), sum(Q_LENS[:b + 1]))
        check_attention(out[s], q[s], [rows[b]], [Q_LENS[b]], [K_LENS[b]], D ** -0.5,
                        _err(q.dtype))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1)])
@pytest.mark.parametrize("stale", [float("nan"), float("inf")])
def test_dtype_pool_with_stale_pages(hq, hkv, stale, dtype):
    P = 256
    bt, nb = tables(K_LENS, P, 9)
    rows = _rows(hkv, 9, dtype)
    pool = [torch.full((nb, P, hkv, D), stale, dtype=dtype) for _ in "kv"]
    for b, L in enumerate(K_LENS):
        s = torch.from_numpy(slots_of(bt, b, 0, L, P))
        for w in (0, 1):
            pool[w].view(-1, hkv, D)[s] = rows[b][w]
    q = _q(hq, dtype, 9)
    for causal in (True, False):
        out = nvkv.paged_attention(q, pool[0].cuda(), pool[1].cuda(), cu(Q_LENS), cu(K_LENS),
                                   torch.from_numpy(bt).cuda(), 200, 701, D ** -0.5, causal=causal)
        torch.cuda.synchronize()
        assert nvkv.device_error() == 0
        check_attention(out, q, _f64(rows), Q_LENS, K_LENS, D ** -0.5, _err(dtype), causal)


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1)])
def test_contiguous_rows_beside_a_nan_sequence(hq, hkv):
    """The third sequence's first rows are NaN; the others are right, and rows
    behind the last sequence (the buffer goes on) do not count."""
    rows = _rows(hkv, 10, torch.bfloat16)
    kv = [torch.cat([r[w] for r in rows] + [torch.full((200, hkv, D), float("nan")).bfloat16()])
          for w in (0, 1)]
    at = sum(K_LENS[:2])
    kv[1][at:at + 2] = float("nan")
    q = _q(hq, torch.bfloat16, 10)
    out = nvkv.paged_attention(q, kv[0].cuda(), kv[1].cuda(), cu(Q_LENS), cu(K_LENS), None, 200,
                               701, D ** -0.5)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    assert bool(out[131:331].isnan().any())
    for b in (0, 1, 3):
        s = slice(sum(Q_LENS[:b]), sum(Q_LENS[:b + 1]))
        check_attention(out[s], q[s], _f64(rows[b:b + 1]), [Q_LENS[b]], [K_LENS[b]], D ** -0.5,
                        _err(q.dtype))


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1)])
def test_row_scaled_prompts_in_unwritten_workspace(hq, hkv):
    P = 256
    bt, nb = tables(K_LENS, P, 11)
    rows = _rows(hkv, 11, torch.bfloat16)
    codes = [torch.full((nb, P, hkv, D), 0x7F, dtype=torch.uint8, device="cuda") for _ in "kv"]
    scales = [torch.full((nb, hkv, P), float("nan"), device="cuda") for _ in "kv"]
    slots = np.concatenate([slots_of(bt, b, 0, L, P) for b, L in enumerate(K_LENS)])
    ops.store_kvcache_fp8(torch.cat([r[0] for r in rows]).cuda(),
                          torch.cat([r[1] for r in rows]).cuda(), *codes, *scales,
                          torch.from_numpy(slots).cuda())
    q = _q(hq, torch.bfloat16, 11)
    # the values of the pool, rounded to the dtype as prompts see them
    held = []
    for b, L in enumerate(K_LENS):
        s = torch.from_numpy(slots_of(bt, b, 0, L, P)).cuda()
        held.append([(c.view(-1, hkv, D)[s].view(torch.float8_e4m3fn).float() *
                      sc[s // P, :, s % P][..., None]).bfloat16().double().cpu().numpy()
                     for c, sc in zip(codes, scales)])
    for spare in (0, 1000):
        n = _prompts() + spare
        ws = _poisoned(ops.workspace_size_fp8(4, hq, hkv, 200, 701, n))
        out = ops.paged_attention_fp8(q, *codes, *scales, cu(Q_LENS), cu(K_LENS),
                                      torch.from_numpy(bt).cuda(), 200, 701, D ** -0.5,
                                      prompt_kv_tokens=n, workspace=ws)
        torch.cuda.synchronize()
        assert nvkv.device_error() == 0
        for b in (0, 2, 3):  # the prompts
            s = slice(sum(Q_LENS[:b]), sum(Q_LENS[:b + 1]))
            check_attention(out[s], q[s], held[b:b + 1], [Q_LENS[b]], [K_LENS[b]], D ** -0.5,
                            _err(q.dtype))
        assert bool(out[130:131].isfinite().all())

"""nvkv_rope_append takes a call's tokens in windows whose width follows their number;
the rows of a call do not depend on it: bit by bit those of calls of 100 tokens."""
import pytest
import torch

import nvkv
from fp8b import D
from nvkv import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1183, 1184, 1500, 1775, 1776, 2400])
def test_dtype_pool_rows_do_not_depend_on_the_call(T, dtype):
    hq, hkv, P = 6, 2, 128
    g = torch.Generator().manual_seed(T)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, generator=g).to(dtype).cuda()
    q, k, v = (x.view(T, -1, D) for x in qkv.split([hq * D, hkv * D, hkv * D], 1))
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() for _ in "qk"]
    f, a = ops.rope_frequencies(D, 1e6, "yarn", 4.0, 32768)
    f, nb = f.cuda(), T // P + 2
    slots = torch.randperm(nb * P, generator=g)[:T].cuda()
    pos = torch.randint(0, 100000, (T,), generator=g).cuda()
    got = []
    for step in (T, 100):
        pool = [torch.zeros(nb, P, hkv, D, dtype=dtype, device="cuda") for _ in "kv"]
        out = torch.empty(T, hq, D, dtype=dtype, device="cuda")
        for lo in range(0, T, step):
            s = slice(lo, min(lo + step, T))
            nvkv.rope_append(q[s], k[s], v[s], pos[s], f, *pool, slots[s], attn_factor=a,
                             q_norm_w=w[0], k_norm_w=w[1], q_out=out[s])
        got.append([out, *pool])
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    assert all(torch.equal(x, y) for x, y in zip(*got))

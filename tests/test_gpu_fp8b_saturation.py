"""Rows at the top of the dtype's range: their e4m3 codes round up past it (65504 to
65536, 1.99 x 2^127 to 2^128), and come back from the block-scaled pool as the
dtype's largest value, read or attended, not as infinities."""
import numpy as np
import pytest
import torch

import nvkv
from fp8b import D, empty_pool, slots_of, tables
from helpers import cu
from nvkv import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("L,new", [(20, 1), (300, 3), (9000, 1)])  # (one CTA, several rows, parts)
def test_largest_values_stay_finite(L, new, dtype):
    hkv, hq, P, top = 2, 8, 256, torch.finfo(dtype).max
    bt, nb = tables([L], P, 1)
    pool = empty_pool(nb, P, hkv)
    sign = torch.where(torch.arange(D) % 3 == 0, -1.0, 1.0)
    rows = (top * sign).expand(L, hkv, D).to(dtype).contiguous()
    slots = torch.from_numpy(slots_of(bt, 0, 0, L, P)).cuda()
    zero = torch.zeros(L, dtype=torch.int64, device="cuda")
    one = torch.ones(4, dtype=torch.float64, device="cuda")
    ops.rope_append(None, rows.cuda(), rows.cuda(), zero, one, *pool[:2], slots, kv_scale=pool[2])
    for t in nvkv.load_kvcache_fp8b(*pool, slots, dtype=dtype):
        assert torch.equal(t.cpu(), rows)
    q = torch.zeros(new, hq, D, dtype=dtype, device="cuda")
    out = nvkv.paged_attention_fp8b(q, *pool, cu([new]), cu([L]), torch.from_numpy(bt).cuda(), new,
                                    L, D ** -0.5)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    # equal weights: the average is the value itself, within the weights' 2^-12
    want = rows[0, 0].double().numpy()
    err = np.abs(out.double().cpu().numpy() / want - 1)
    assert np.isfinite(err).all() and err.max() <= torch.finfo(dtype).eps / 2 + 2.0 ** -12

"""nvkv_paged_attention_fp8b against f64 attention over the dequantised rows.

Decode and short batches: scores are sums of exact products in f32 (an error of
2^-17 in the exponent at the sizes here, so 2^-17 of a weight), exponentials off
by 2^-21, weights held to 2^-12: 2^-11 of sum p |v| covers them.  Prompts: the
prefill kernel rounds weights to the dtype (eps / 2) and takes some exponentials
from a polynomial (7.5e-5): eps / 2 + 2^-12."""
import numpy as np
import pytest
import torch

import nvkv
from fp8b import D, G, check_attention, empty_pool, filled, slots_of, tables
from helpers import cu
from nvkv import ops
from nvkv._lib import DEVERR_BLOCK_RANGE, DEVERR_SEQLEN

pytestmark = pytest.mark.gpu

SHORT = 2.0 ** -11


def prompt_err(dtype):
    return torch.finfo(dtype).eps / 2 + 2.0 ** -12


def _q(T, hq, dtype, seed, gain=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, hq, D, generator=g) * gain).to(dtype).cuda()


def _run(q, pool, bt, q_lens, k_lens, **kw):
    prompts = sum(k for a, k in zip(q_lens, k_lens) if a > 1)
    out = nvkv.paged_attention_fp8b(q, *pool, cu(q_lens), cu(k_lens), bt, max(q_lens), max(k_lens),
                                    D ** -0.5, prompt_kv_tokens=prompts, **kw)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 8, 9, 16])
def test_decode_groups(group, dtype):
    """Every group size; lengths of one key, tiles that end inside, on and after
    a page."""
    k_lens = [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 700, 1025]
    hkv = 2
    pool, bt, rows = filled(k_lens, hkv, seed=group, dtype=dtype)
    q = _q(len(k_lens), hkv * group, dtype, group)
    q_lens = [1] * len(k_lens)
    out = _run(q, pool, bt, q_lens, k_lens)
    assert nvkv.device_error() == 0
    check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, SHORT)


@pytest.mark.parametrize("k_lens,hq,hkv,P", [
    ([20000, 300, 1, 4096], 16, 1, 256),          # split over many CTAs
    ([9000], 8, 8, 128), ([5000] * 3, 40, 8, 512),
    (np.random.default_rng(1).integers(1, 1500, 180).tolist(), 4, 1, 256)])
def test_decode_long_and_many(k_lens, hq, hkv, P):
    pool, bt, rows = filled(k_lens, hkv, P=P, seed=7)
    q_lens = [1] * len(k_lens)
    q = _q(len(k_lens), hq, torch.bfloat16, 3)
    out = _run(q, pool, bt, q_lens, k_lens)
    assert nvkv.device_error() == 0
    check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, SHORT, every=max(1, len(k_lens) // 40))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,q_hi", [(8, 2, 8), (16, 1, 2), (3, 3, 32), (5, 1, 6), (32, 8, 4)])
def test_short_batches(hq, hkv, q_hi, dtype):
    """A few tokens a sequence, ragged, causal and not."""
    rng = np.random.default_rng(hq + q_hi)
    q_lens = rng.integers(1, q_hi + 1, 9).tolist() + [q_hi, q_hi, 1]
    k_lens = [int(rng.integers(a, 1400)) for a in q_lens[:-3]] + [q_hi, 2000, 1]
    pool, bt, rows = filled(k_lens, hkv, seed=q_hi, dtype=dtype)
    q = _q(sum(q_lens), hq, dtype, 5)
    for causal in (True, False):
        out = _run(q, pool, bt, q_lens, k_lens, causal=causal)
        assert nvkv.device_error() == 0
        check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, SHORT, causal)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [True, False])
def test_prompts_and_decode_rows(dtype, causal):
    """Fresh prompts, chunks on a cached context and decode rows in one call."""
    q_lens = [1, 300, 64, 1, 130, 129, 1, 2]
    k_lens = [900, 300, 700, 1, 131, 1000, 256, 2]
    hq, hkv = 10, 2
    pool, bt, rows = filled(k_lens, hkv, seed=2, dtype=dtype)
    q = _q(sum(q_lens), hq, dtype, 6)
    out = _run(q, pool, bt, q_lens, k_lens, causal=causal)
    assert nvkv.device_error() == 0
    for b, (a, k) in enumerate(zip(q_lens, k_lens)):
        s = slice(sum(q_lens[:b]), sum(q_lens[:b + 1]))
        check_attention(out[s], q[s], [rows[b]], [a], [k], D ** -0.5,
                        SHORT if a == 1 else prompt_err(dtype), causal)


@pytest.mark.parametrize("q_gain,k_gain,v_gain", [(8.0, 1.0, 1.0), (1e-3, 1e3, 1e-4),
                                                  (1.0, 1.0, 3e4), (30.0, 1.0, 1e-30)])
def test_decode_value_ranges(q_gain, k_gain, v_gain):
    """Peaked softmaxes, and keys and values far from 1.  The exponent of a
    weight is off by 2^-24 of the scores' partial sums (up to a few hundred
    here): 2^-10 of a weight more."""
    k_lens = [1, 100, 1300, 4000]
    hq, hkv = 8, 2
    pool, bt, rows = filled(k_lens, hkv, seed=11, k_gain=k_gain, v_gain=v_gain)
    q = _q(4, hq, torch.bfloat16, 12, q_gain)
    out = _run(q, pool, bt, [1] * 4, k_lens)
    assert nvkv.device_error() == 0
    scaled = [[k, v / v_gain] for k, v in rows]
    check_attention((out.double() / v_gain).to(torch.float32), q, scaled, [1] * 4, k_lens,
                    D ** -0.5, SHORT + 2.0 ** -10 + 2.0 ** -8)


def test_sink_and_spread():
    """One key takes most of the weight and has a tiny value; thousands of small
    weights carry the answer.  Their precision must not depend on the sink."""
    L, hkv, hq = 5000, 1, 4
    bt, nb = tables([L], 256, 4)
    pool = empty_pool(nb, 256, hkv)
    g = torch.Generator().manual_seed(4)
    k = torch.randn(L, hkv, D, generator=g) * 0.05
    k[0] = 1.0
    v = torch.randn(L, hkv, D, generator=g)
    v[:16] *= 1e-4
    v[16:] += 0.5
    slots = torch.from_numpy(slots_of(bt, 0, 0, L, 256)).cuda()
    ops.rope_append(None, k.bfloat16().cuda(), v.bfloat16().cuda(),
                    torch.zeros(L, dtype=torch.int64).cuda(),
                    torch.ones(4, dtype=torch.float64).cuda(), pool[0], pool[1], slots,
                    kv_scale=pool[2])
    kd, vd = nvkv.load_kvcache_fp8b(*pool, slots)
    q = torch.full((1, hq, D), 1.0)
    q *= torch.tensor([0.2, 0.5, 0.9, 1.1])[None, :, None]
    q = q.half().cuda()
    out = _run(q, pool, torch.from_numpy(bt).cuda(), [1], [L])
    check_attention(out, q, [[kd.double().cpu().numpy(), vd.double().cpu().numpy()]], [1], [L],
                    D ** -0.5, SHORT)


def test_malformed_sequences_are_skipped():
    """k_len above the maximum, k_len below q_len, rows past q: skipped and
    recorded, their out rows and those behind the last sequence as they were;
    k_len 0: zeros, recorded; a page past the pool: recorded, memory-safe."""
    k_lens = [300, 700, 5, 40]
    hq, hkv = 4, 2
    pool, bt, rows = filled(k_lens, hkv, seed=3)
    q = _q(12, hq, torch.bfloat16, 1)

    def run(q_lens, ks, max_k, bt_=bt, prompts=0):
        out = torch.full_like(q, 7.0)
        nvkv.paged_attention_fp8b(q, *pool, cu(q_lens), cu(ks), bt_, max(q_lens), max_k, D ** -0.5,
                                  out=out, prompt_kv_tokens=prompts)
        torch.cuda.synchronize()
        return out, nvkv.device_error()
    nvkv.device_error()
    out, err = run([1, 1, 1, 1], [300, 700, 5, 40], 512)
    assert err == DEVERR_SEQLEN and bool((out[1] == 7).all()) and bool((out[4:] == 7).all())
    check_attention(out[[0, 2, 3]], q[[0, 2, 3]], [rows[i] for i in (0, 2, 3)], [1] * 3,
                    [300, 5, 40], D ** -0.5, SHORT)
    out, err = run([2, 6, 1, 1], [300, 5, 5, 40], 700)
    assert err == DEVERR_SEQLEN and bool((out[2:8] == 7).all()) and bool((out[10:] == 7).all())
    out, err = run([1, 1, 1, 1], [300, 0, 5, 40], 700)
    assert err == DEVERR_SEQLEN and bool((out[1] == 0).all())
    out, err = run([8, 1, 4, 1], [300, 700, 5, 40], 700)  # 14 rows asked of 12
    assert err == DEVERR_SEQLEN
    assert bool((out[9:] == 7).all()) and not bool((out[:9] == 7).all())
    bad = bt.clone()
    bad[1, 1] = 1 << 30
    out, err = run([1, 1, 1, 1], k_lens, 700, bad)
    assert err == DEVERR_BLOCK_RANGE
    check_attention(out[[0]], q[[0]], [rows[0]], [1], [300], D ** -0.5, SHORT)


def test_nan_keys_stay_with_their_sequence():
    """A NaN in one sequence's keys or values reaches that sequence's heads alone."""
    k_lens = [200, 200, 200]
    pool, bt, rows = filled(k_lens, 2, seed=9)
    page = int(bt[1, 0])
    pool[0][page, 7, 1, 3] = 0x7F
    q = _q(3, 4, torch.bfloat16, 2)
    out = _run(q, pool, bt, [1] * 3, k_lens)
    assert bool(out[1, 2:].isnan().any()) and not bool(out[1, :2].isnan().any())
    check_attention(out[[0, 2]], q[[0, 2]], [rows[0], rows[2]], [1] * 2, [200] * 2, D ** -0.5, SHORT)


def test_strided_q_streams_and_shared_graph_pool():
    """q as a slice of a fused buffer, a side stream, and two graphs with a
    workspace each replayed in turn."""
    k_lens = [3000, 10, 800]
    hq, hkv = 8, 2
    pool, bt, rows = filled(k_lens, hkv, seed=13)
    g = torch.Generator().manual_seed(1)
    buf = torch.randn(3, (hq + 2 * hkv) * D, generator=g).bfloat16().cuda()
    q = buf[:, :hq * D].view(3, hq, D)
    want = _run(q, pool, bt, [1] * 3, k_lens)
    check_attention(want, q, rows, [1] * 3, k_lens, D ** -0.5, SHORT)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(q, pool, bt, [1] * 3, k_lens)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    cq, ck = cu([1] * 3), cu(k_lens)
    graphs, outs = [], []
    for _ in range(2):
        ws = torch.empty(max(16, nvkv.workspace_size_fp8b(3, hq, hkv, 1, 3000)), device="cuda",
                         dtype=torch.uint8)
        out = torch.empty_like(want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            nvkv.paged_attention_fp8b(q, *pool, cq, ck, bt, 1, 3000, D ** -0.5, out=out,
                                      workspace=ws)
        graphs.append((graph, ws))
        outs.append(out)
    buf.mul_(0.5)
    want = _run(q, pool, bt, [1] * 3, k_lens)
    for _ in range(3):
        for (graph, _), out in zip(graphs, outs):
            out.zero_()
            graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_append_then_attend_steps():
    """The operators as they are used together: a prompt and decode steps, each
    appended and attended, against f64 over the rows that the pool holds."""
    P, hq, hkv = 128, 8, 2
    lens = [130, 5, 64]
    total = [L + 20 for L in lens]
    bt, nb = tables(total, P, 5)
    pool = empty_pool(nb, P, hkv)
    f, a = ops.rope_frequencies(128, 1e6, "yarn", 4.0, 32768)
    f = f.cuda()
    bt_d = torch.from_numpy(bt).cuda()
    have = [0] * 3
    for step in range(12):
        new = lens if step == 0 else [1] * 3 if step % 3 else [2, 3, 1]
        k_lens = [h + n for h, n in zip(have, new)]
        slots = np.concatenate([slots_of(bt, b, have[b], k_lens[b], P) for b in range(3)])
        pos = np.concatenate([np.arange(have[b], k_lens[b]) for b in range(3)])
        qkv = torch.randn(len(slots), (hq + 2 * hkv) * D,
                          generator=torch.Generator().manual_seed(step)).bfloat16().cuda()
        q, k, v = (x.view(len(slots), -1, D) for x in
                   qkv.split([hq * D, hkv * D, hkv * D], 1))
        q = nvkv.rope_append(q, k, v, torch.from_numpy(pos).cuda(), f, pool[0], pool[1],
                             torch.from_numpy(slots).cuda(), kv_scale=pool[2], attn_factor=a)
        out = _run(q, pool, bt_d, list(new), k_lens)
        rows = []
        for b in range(3):
            s = torch.from_numpy(slots_of(bt, b, 0, k_lens[b], P)).cuda()
            rows.append([t.double().cpu().numpy() for t in nvkv.load_kvcache_fp8b(*pool, s)])
        check_attention(out, q, rows, list(new), k_lens, D ** -0.5,
                        SHORT if max(new) <= 8 else prompt_err(q.dtype))
        have = k_lens
    assert nvkv.device_error() == 0


def test_many_kv_heads_and_many_sequences():
    """More kv heads than a wave has CTAs; more sequences than a CTA has threads,
    empty ones among them (q_len 0: padding of a batch)."""
    k_lens = [70, 3]
    pool, bt, rows = filled(k_lens, 301, P=128, seed=21)
    q = _q(2, 301, torch.bfloat16, 8)
    out = _run(q, pool, bt, [1, 1], k_lens)
    assert nvkv.device_error() == 0
    check_attention(out, q, rows, [1, 1], k_lens, D ** -0.5, SHORT)
    rng = np.random.default_rng(6)
    k_lens = rng.integers(1, 200, 700).tolist()
    q_lens = (rng.random(700) < 0.8).astype(int).tolist()
    pool, bt, rows = filled(k_lens, 2, P=128, seed=22)
    q = _q(sum(q_lens) + 3, 6, torch.float16, 9)  # three rows behind the last sequence
    out = torch.full_like(q, 7.0)
    nvkv.paged_attention_fp8b(q, *pool, cu(q_lens), cu(k_lens), bt, 1, 199, D ** -0.5, out=out)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0 and bool((out[-3:] == 7).all())
    check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, SHORT, every=7)


def test_prompt_that_does_not_fit_is_reported():
    """prompt_kv_tokens below the prompts' keys: that prompt's rows stay as they
    were, the others are right."""
    q_lens, k_lens = [300, 1, 200], [300, 900, 450]
    pool, bt, rows = filled(k_lens, 2, seed=23)
    q = _q(sum(q_lens), 4, torch.bfloat16, 3)
    out = torch.full_like(q, 7.0)
    nvkv.device_error()
    nvkv.paged_attention_fp8b(q, *pool, cu(q_lens), cu(k_lens), bt, 300, 900, D ** -0.5,
                              prompt_kv_tokens=500, out=out)
    torch.cuda.synchronize()
    assert nvkv.device_error() == DEVERR_SEQLEN and bool((out[301:] == 7).all())
    check_attention(out[:300], q[:300], rows[:1], [300], [300], D ** -0.5, prompt_err(q.dtype))
    check_attention(out[300:301], q[300:301], rows[1:2], [1], [900], D ** -0.5, SHORT)


def test_two_streams_at_once_and_in_place():
    """Calls that overlap on the GPU, each with its own workspace, and out = q:
    the bits of a call alone."""
    cases = []
    for seed, k_lens in ((31, [4000, 100, 9]), (32, [700] * 40)):
        pool, bt, _ = filled(k_lens, 2, seed=seed)
        q = _q(len(k_lens), 8, torch.bfloat16, seed)
        want = _run(q, pool, bt, [1] * len(k_lens), k_lens)
        ws = torch.empty(nvkv.workspace_size_fp8b(len(k_lens), 8, 2, 1, max(k_lens)),
                         device="cuda", dtype=torch.uint8)
        cases.append((q, pool, bt, cu([1] * len(k_lens)), cu(k_lens), max(k_lens), want, ws,
                      torch.cuda.Stream(), torch.empty_like(q)))
    torch.cuda.synchronize()
    for _ in range(30):
        for q, pool, bt, cq, ck, mk, _, ws, stream, out in cases:
            with torch.cuda.stream(stream):
                nvkv.paged_attention_fp8b(q, *pool, cq, ck, bt, 1, mk, D ** -0.5, out=out,
                                          workspace=ws)
    torch.cuda.synchronize()
    for q, pool, bt, cq, ck, mk, want, ws, _, out in cases:
        assert torch.equal(out, want)
        nvkv.paged_attention_fp8b(q, *pool, cq, ck, bt, 1, mk, D ** -0.5, out=q, workspace=ws)
        assert torch.equal(q, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_mixed_batch_in_place_with_padding(dtype):
    """Prompts, chunks, single rows and padded entries, out = q: the bits of a call
    into another buffer, and rows behind the last sequence as they were."""
    q_lens = [150, 1, 0, 300, 1, 17, 0]
    k_lens = [150, 2000, 5, 1100, 1, 17, 1]
    pool, bt, rows = filled(k_lens, 2, seed=41, dtype=dtype)
    q = _q(sum(q_lens) + 5, 8, dtype, 41)
    out = torch.full_like(q, 7.0)
    kw = dict(prompt_kv_tokens=150 + 1100 + 17)
    args = (*pool, cu(q_lens), cu(k_lens), bt, 300, 2000, D ** -0.5)
    nvkv.paged_attention_fp8b(q, *args, out=out, **kw)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0 and bool((out[-5:] == 7).all())
    check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, prompt_err(dtype))
    before = q.clone()
    nvkv.paged_attention_fp8b(q, *args, out=q, **kw)
    torch.cuda.synchronize()
    assert torch.equal(q[:-5], out[:-5]) and torch.equal(q[-5:], before[-5:])


@pytest.mark.parametrize("n,skew", [(148, 0), (200, 700), (296, 300), (296, 2500), (297, 300)])
def test_about_as_many_sequences_as_shares(n, skew):
    """One kv head: sequences that get a share each (equal or nearly), others that
    are cut, empty ones among them, one more than the shares."""
    rng = np.random.default_rng(n + skew)
    k_lens = (300 + rng.integers(0, skew + 1, n)).tolist()
    q_lens = (np.arange(n) % 11 != 3).astype(int).tolist()
    pool, bt, rows = filled(k_lens, 1, P=128, seed=n)
    q = _q(sum(q_lens) + 2, 4, torch.bfloat16, n)
    out = torch.full_like(q, 7.0)
    nvkv.paged_attention_fp8b(q, *pool, cu(q_lens), cu(k_lens), bt, 1, max(k_lens), D ** -0.5,
                              out=out)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0 and bool((out[-2:] == 7).all())
    check_attention(out, q, rows, q_lens, k_lens, D ** -0.5, SHORT)

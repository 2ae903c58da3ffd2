"""nvkv_rope_append and nvkv_load_kvcache_fp8b against the 64-bit definition.

The fp8b pool is compared exactly: K is normalised and rotated in f64 and
rounded once, so codes and scales are functions of the formulas (a difference
needs an f64 value within some 1e-12 of a rounding border).  q and the
model-dtype pool: one rounding (eps / 2) plus f32 arithmetic, 2^-20 of |x0| +
|x1|, the norm's f32 sum among it (its 7 additions and a square root stay below
2^-21 relative)."""
import numpy as np
import pytest
import torch

import nvkv
import nvkv_oracle as O
from fp8b import D, G, empty_pool, slots_of, tables
from nvkv import ops
from nvkv._lib import DEVERR_SLOT_ORDER, DEVERR_SLOT_RANGE

pytestmark = pytest.mark.gpu


def _inputs(T, hq, hkv, dtype, seed, norm):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randn(T, (hq + 2 * hkv) * D + 8, generator=g)
    buf *= torch.exp(torch.randn(T, 1, generator=g))  # rows of very different size
    buf = buf.to(dtype).cuda()
    q = buf[:, :hq * D].view(T, hq, D)
    k = buf[:, hq * D:(hq + hkv) * D].view(T, hkv, D)
    v = buf[:, (hq + hkv) * D:(hq + 2 * hkv) * D].view(T, hkv, D)
    w = [(1 + 0.2 * torch.randn(D, generator=g)).to(dtype).cuda() if norm else None
         for _ in range(2)]
    return q, k, v, w


def _n(t):
    return None if t is None else t.double().cpu().numpy()


def _rotated(x, w, pos, f, a, inter):
    return O.rope_rotate(O.head_rms_norm(_n(x), _n(w), 1e-6), pos.cpu().numpy(),
                         f.cpu().numpy(), a, inter)


def _check_rows(got, x, w, pos, f, a, inter):
    want = _rotated(x, w, pos, f, a, inter)
    xn, n = O.head_rms_norm(_n(x), _n(w), 1e-6), f.numel()
    size = np.zeros_like(xn)
    i0 = slice(0, 2 * n, 2) if inter else slice(0, n)
    i1 = slice(1, 2 * n, 2) if inter else slice(n, 2 * n)
    size[:] = abs(xn)
    size[..., i0] = size[..., i1] = (abs(xn[..., i0]) + abs(xn[..., i1])) * a
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0
    tol = abs(want) * torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -20) + size * 2.0 ** -20 + tiny
    assert (abs(_n(got) - want) <= tol).all()


def _same_pool(pool, want):
    kc, vc, sc = (t.cpu().numpy() for t in pool)
    assert np.array_equal(sc, want[2], equal_nan=True)
    for c, w in ((kc, want[0]), (vc, want[1])):  # +0 and -0 are the same value
        bad = ~((c == w) | ((c & 0x7F) == 0) & ((w & 0x7F) == 0))
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:4], c[bad][:4], w[bad][:4])


def _freq(rot, kind="yarn"):
    f, a = ops.rope_frequencies(rot, 1e6, kind, 4.0, 32768)
    return f.cuda(), a


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,rot,inter,norm,P", [
    (4, 1, 128, False, True, 256), (2, 2, 64, True, False, 128), (5, 1, 8, False, True, 16),
    (0, 3, 24, True, True, 64), (16, 8, 120, False, False, 256)])
def test_append_fp8b_steps(hq, hkv, rot, inter, norm, P, dtype):
    """Prompts, then ragged chunks, then single tokens into the blocks that are
    being filled: pool and scales bit by bit after every call."""
    rng = np.random.default_rng(rot + P)
    B, steps = 7, 6
    lens = np.zeros(B, int)
    bt, nb = tables([160] * B, P, 3)
    pool = empty_pool(nb, P, hkv)
    want = [t.cpu().numpy().copy() for t in pool]
    f, a = _freq(rot)
    for step in range(steps):
        new = rng.integers(0, 40, B) if step < 2 else np.ones(B, int)
        if step == 0:
            new[:4] = [16, 33, 1, 15]
        slots = np.concatenate([slots_of(bt, b, lens[b], lens[b] + new[b], P) for b in range(B)])
        pos = np.concatenate([np.arange(lens[b], lens[b] + new[b]) for b in range(B)])
        T = len(slots)
        q, k, v, w = _inputs(T, hq, hkv, dtype, step * 31 + rot, norm)
        pos = torch.from_numpy(pos).cuda() * 37
        q_out = nvkv.rope_append(q if hq else None, k, v, pos, f, pool[0], pool[1],
                                 torch.from_numpy(slots).cuda(), kv_scale=pool[2], attn_factor=a,
                                 interleaved=inter, q_norm_w=w[0], k_norm_w=w[1])
        torch.cuda.synchronize()
        assert nvkv.device_error() == 0
        O.append_fp8b(_rotated(k, w[1], pos, f, a, inter), _n(v), *want, slots)
        _same_pool(pool, want)
        if hq:
            _check_rows(q_out, q, w[0], pos, f, a, inter)
        lens += new


def test_append_fp8b_large_batch_and_windows():
    """Windows of several tokens whose blocks straddle them, padded tokens in
    between: 5000 tokens."""
    rng = np.random.default_rng(5)
    P, hkv = 256, 2
    lens = [1800, 1, 777, 900, 30, 1200, 292]
    bt, nb = tables(lens, P, 1)
    slots = np.concatenate([slots_of(bt, b, 0, L, P) for b, L in enumerate(lens)])
    pads = np.sort(rng.integers(0, len(slots), 60))
    slots = np.insert(slots, pads, -1)
    T = len(slots)
    pool = empty_pool(nb, P, hkv)
    want = [t.cpu().numpy().copy() for t in pool]
    q, k, v, w = _inputs(T, 4, hkv, torch.bfloat16, 8, True)
    pos = torch.from_numpy(rng.integers(0, 100000, T)).cuda()
    f, a = _freq(128)
    # a padding in the middle of a block would split its tokens: the block's
    # second half is then a run of its own that starts past row 0
    clean = slots.copy()
    for t in range(1, T):
        if slots[t] >= 0 and slots[t - 1] < 0 and slots[t] % G:
            clean[t:][clean[t:] // G == slots[t] // G] = -1
    q_out = nvkv.rope_append(q, k, v, pos, f, pool[0], pool[1], torch.from_numpy(clean).cuda(),
                             kv_scale=pool[2], attn_factor=a, q_norm_w=w[0], k_norm_w=w[1])
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    O.append_fp8b(_rotated(k, w[1], pos, f, a, False), _n(v), *want, clean)
    _same_pool(pool, want)
    _check_rows(q_out, q, w[0], pos, f, a, False)


def test_append_fp8b_special_values():
    """Infinities saturate, NaN stays NaN, zeros and tiny rows take the least
    scale, a block's scale grows by more than e4m3's range."""
    P, hkv = 128, 1
    rows = torch.zeros(16, hkv, D)
    rows[0] = 1e-37
    rows[2] = torch.linspace(-1e-3, 1e-3, D)
    rows[3, 0, 5] = float("inf")
    rows[4, 0, 6] = float("-inf")
    rows[5, 0, 7] = float("nan")
    rows[6] = 1.0
    rows[7] = 448.0
    rows[8] = 3e30
    rows = rows.bfloat16()
    f = torch.ones(4, dtype=torch.float64).cuda()
    pool = empty_pool(2, P, hkv)
    want = [t.cpu().numpy().copy() for t in pool]
    for lo, hi in ((0, 1), (1, 2), (2, 3), (3, 7), (7, 8), (8, 16)):
        x = rows[lo:hi].cuda()
        slots = torch.arange(lo, hi).cuda()
        nvkv.rope_append(None, x, x, torch.zeros(hi - lo, dtype=torch.int64).cuda(), f, pool[0],
                         pool[1], slots, kv_scale=pool[2])
        torch.cuda.synchronize()
        # dims 8 .. are not rotated; inf and NaN sit at 5 .. 7 of V and, by the
        # rotation with angle 0, inf * 0 = NaN spreads over K's pair
        xn = _n(x)
        with np.errstate(invalid="ignore"):
            O.append_fp8b(O.rope_rotate(xn, np.zeros(hi - lo), np.ones(4)), xn, *want, slots.tolist())
        _same_pool(pool, want)
    assert nvkv.device_error() == 0


def test_append_slot_errors_are_recorded():
    """Slots past the pool and slots that do not ascend are not stored; the
    others are; rows of no slot stay as they were."""
    P, hkv, nb = 128, 2, 3
    pool = empty_pool(nb, P, hkv)
    want = [t.cpu().numpy().copy() for t in pool]
    q, k, v, _ = _inputs(8, 2, hkv, torch.bfloat16, 1, False)
    f, a = _freq(64)
    pos = torch.arange(8).cuda()
    slots = [0, 1, nb * P, 64, 64, 65, 32, 1 << 40]
    nvkv.device_error()
    nvkv.rope_append(q, k, v, pos, f, pool[0], pool[1], torch.tensor(slots).cuda(),
                     kv_scale=pool[2], attn_factor=a)
    torch.cuda.synchronize()
    assert nvkv.device_error() in (DEVERR_SLOT_RANGE, DEVERR_SLOT_ORDER)
    O.append_fp8b(_rotated(k, None, pos, f, a, False), _n(v), *want,
                  [0, 1, -1, 64, -1, -1, 32, -1])
    _same_pool(pool, want)
    nvkv.rope_append(q, k, v, pos, f, pool[0], pool[1],
                     torch.tensor([5, 4, -1, -1, -1, -1, -1, -1]).cuda(), kv_scale=pool[2])
    torch.cuda.synchronize()
    assert nvkv.device_error() == DEVERR_SLOT_ORDER
    dt = [torch.zeros(nb, P, hkv, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    nvkv.rope_append(q, k, v, pos, f, *dt, torch.tensor([0, -1, nb * P, 7, 6, 5, 9, 8]).cuda())
    torch.cuda.synchronize()
    assert nvkv.device_error() == DEVERR_SLOT_RANGE
    assert torch.equal(dt[1][0, 7], v[3]) and torch.equal(dt[1][0, 8], v[7])
    assert int((dt[1] != 0).any(-1).any(-1).sum()) == 6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,hq,hkv,rot,inter,norm", [
    (1, 4, 1, 128, False, True), (300, 3, 2, 64, True, True), (2500, 2, 1, 40, False, False)])
def test_append_dtype_pool(T, hq, hkv, rot, inter, norm, dtype):
    P = 48  # any page size: no scales
    nb = (T + P - 1) // P + 1
    q, k, v, w = _inputs(T, hq, hkv, dtype, T, norm)
    g = torch.Generator().manual_seed(T)
    slots = torch.randperm(nb * P, generator=g)[:T]
    slots[::7] = -1
    pos = torch.randint(0, 131072, (T,), generator=g).cuda()
    f, a = _freq(rot, "bands")
    kc = torch.full((nb, P, hkv, D), 3.0, dtype=dtype, device="cuda")
    vc = kc.clone()
    q_out = nvkv.rope_append(q, k, v, pos, f, kc, vc, slots.cuda(), attn_factor=a,
                             interleaved=inter, q_norm_w=w[0], k_norm_w=w[1])
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    _check_rows(q_out, q, w[0], pos, f, a, inter)
    put = (slots >= 0).nonzero().flatten()
    at = slots[put].cuda()
    _check_rows(kc.view(-1, hkv, D)[at], k[put.cuda()], w[1], pos[put.cuda()], f, a, inter)
    assert torch.equal(vc.view(-1, hkv, D)[at], v[put.cuda()])
    rest = torch.ones(nb * P, dtype=torch.bool)
    rest[slots[put]] = False
    assert bool((kc.view(-1, hkv, D)[rest.cuda()] == 3).all())


def test_append_q_in_place_and_graph():
    """q_out = q on a dense q; a captured decode step replays on new inputs."""
    P, hkv, hq, B = 256, 2, 8, 40
    bt, nb = tables([64] * B, P, 2)
    f, a = _freq(128)
    pools = [empty_pool(nb, P, hkv) for _ in range(2)]
    q, k, v, w = (t if isinstance(t, list) else t.contiguous()
                  for t in _inputs(B, hq, hkv, torch.bfloat16, 4, True))
    pos = torch.zeros(B, dtype=torch.int64).cuda()
    slots = torch.zeros(B, dtype=torch.int64).cuda()
    out = torch.empty_like(q)

    def call(pool, **kw):
        return nvkv.rope_append(q, k, v, pos, f, pool[0], pool[1], slots, kv_scale=pool[2],
                                attn_factor=a, q_norm_w=w[0], k_norm_w=w[1], **kw)
    slots.copy_(torch.from_numpy(np.concatenate([slots_of(bt, b, 0, 1, P) for b in range(B)])))
    call(pools[0], q_out=out)
    call(pools[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(pools[1], q_out=out)
    for step in range(1, 6):
        slots.copy_(torch.from_numpy(np.concatenate([slots_of(bt, b, step, step + 1, P)
                                                     for b in range(B)])))
        pos.fill_(step)
        k.mul_(1.5)
        graph.replay()
        want = call(pools[0])
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for x, y in zip(*pools):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    want = call(pools[0])
    q2 = q.clone()
    nvkv.rope_append(q2, k, v, pos, f, pools[1][0], pools[1][1], slots, kv_scale=pools[1][2],
                     attn_factor=a, q_norm_w=w[0], k_norm_w=w[1], q_out=q2)
    assert torch.equal(q2, want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_load(dtype):
    """code * scale is exact before the rounding to the dtype; f16 saturates."""
    P, hkv, nb = 32, 3, 4
    g = torch.Generator().manual_seed(2)
    codes = [torch.randint(0, 256, (nb, P, hkv, D), generator=g, dtype=torch.uint8) for _ in "kv"]
    sc = torch.exp2(torch.randint(-12, 12, (nb, hkv, P // G, 2), generator=g).float())
    slots = torch.randint(0, nb * P, (77,), generator=g)
    slots[3], slots[9] = -1, nb * P
    nvkv.device_error()
    got = nvkv.load_kvcache_fp8b(codes[0].cuda(), codes[1].cuda(), sc.cuda(), slots.cuda(), dtype)
    torch.cuda.synchronize()
    assert nvkv.device_error() == DEVERR_SLOT_RANGE
    for which in (0, 1):
        vals = O.dequantize_pages_fp8b(codes[which].numpy(), sc.numpy(), which)
        want = vals.reshape(nb * P, hkv, D)[np.clip(slots.numpy(), 0, nb * P - 1)]
        want[[3, 9]] = 0.0
        want = torch.from_numpy(want)
        if dtype == torch.float16:
            want = torch.where(want.isnan(), want, want.clamp(-65504, 65504))
        assert torch.equal(got[which].cpu().nan_to_num(nan=7e4), want.to(dtype).nan_to_num(nan=7e4))
    none = nvkv.load_kvcache_fp8b(codes[0].cuda(), codes[1].cuda(), sc.cuda(),
                                  torch.zeros(0, dtype=torch.int64).cuda())
    assert none[0].shape == (0, hkv, D)

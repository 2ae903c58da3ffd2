"""nvkv_rope against the 64-bit rotation, and its transpose.

Tolerance: one rounding to the dtype (half a step, eps / 2 relative) plus the
f32 arithmetic: two products and a sum of f32 cos / sin, each within 2^-22 of
|x0| + |x1| times the factor (cos and sin themselves are off by up to 2^-23: the
f32 fraction of a turn, sincospif, the factor)."""
import numpy as np
import pytest
import torch

import nvkv
import nvkv_oracle as O
from nvkv import ops

pytestmark = pytest.mark.gpu


def _freq(rot, kind="yarn"):
    f, a = ops.rope_frequencies(rot, 1e6, kind, 4.0, 32768)
    return f.cuda(), a


def _check(got, x, pos, f, a, inter, rot):
    xn, y = x.double().cpu().numpy(), got.double().cpu().numpy()
    want = O.rope_rotate(xn, pos.cpu().numpy(), f.cpu().numpy(), a, inter)
    n = rot // 2
    pair = np.zeros_like(xn)
    i0 = slice(0, rot, 2) if inter else slice(0, n)
    i1 = slice(1, rot, 2) if inter else slice(n, rot)
    pair[..., i0] = pair[..., i1] = (abs(xn[..., i0]) + abs(xn[..., i1])) * a
    tiny = 2.0 ** -24 if got.dtype == torch.float16 else 0.0  # f16 subnormals' half step
    tol = abs(want) * torch.finfo(got.dtype).eps / 2 * (1 + 2.0 ** -20) + pair * 2.0 ** -21 + tiny
    bad = abs(y - want) > tol
    assert not bad.any(), (np.argwhere(bad)[:4], y[bad][:4], want[bad][:4])
    assert np.array_equal(y[..., rot:], xn[..., rot:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,hq,hkv,d,rot", [
    (1, 1, 1, 8, 2), (1, 32, 8, 128, 128), (5, 3, 1, 96, 64), (257, 16, 8, 128, 32),
    (33, 7, 2, 80, 20), (9, 5, 5, 50, 50), (1000, 4, 1, 256, 256), (7, 2, 1, 1024, 1024),
    (4001, 9, 3, 72, 24), (9000, 1, 1, 1024, 1024), (20000, 2, 1, 16, 6)])
def test_rope(T, hq, hkv, d, rot, inter, dtype):
    g = torch.Generator().manual_seed(T * 7 + d)
    q = torch.randn(T, hq, d, generator=g).to(dtype).cuda()
    k = (torch.randn(T, hkv, d, generator=g) * 8).to(dtype).cuda()
    pos = torch.randint(0, 200000, (T,), generator=g).cuda()
    pos[0] = 0
    f, a = _freq(rot)
    qo, ko = nvkv.rope(q, k, pos, f, a, inter)
    _check(qo, q, pos, f, a, inter, rot)
    _check(ko, k, pos, f, a, inter, rot)
    q2, k2 = q.clone(), k.clone()  # in place: the same bits
    nvkv.rope(q2, k2, pos, f, a, inter, q_out=q2, k_out=k2)
    assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("inter", [False, True])
def test_rope_views_of_a_fused_buffer(inter):
    """Strided views, odd strides and offsets (single pairs), in place; the rest
    of the buffer stays."""
    for width, lead in ((16 * 128 + 8, 0), (16 * 128 + 7, 0), (16 * 128 + 9, 1)):
        g = torch.Generator().manual_seed(width)
        buf = torch.randn(65, width, generator=g).bfloat16().cuda()
        before = buf.clone()
        q = buf[:, lead:lead + 8 * 128].view(65, 8, 128)
        k = buf[:, lead + 8 * 128:lead + 12 * 128].view(65, 4, 128)
        q0, k0 = q.clone(), k.clone()
        pos = torch.arange(65).cuda() * 1001
        f, a = _freq(64, "plain")
        nvkv.rope(q, k, pos, f, a, inter, q_out=q, k_out=k)
        _check(q, q0, pos, f, a, inter, 64)
        _check(k, k0, pos, f, a, inter, 64)
        assert torch.equal(buf[:, lead + 12 * 128:], before[:, lead + 12 * 128:])
        assert torch.equal(buf[:, :lead], before[:, :lead])


def test_rope_q_alone_and_far_positions():
    g = torch.Generator().manual_seed(3)
    q = torch.randn(6, 2, 128, generator=g).half().cuda()
    pos = torch.tensor([0, 1, -1, 1 << 20, (1 << 22) + 1, -(1 << 21)]).cuda()
    f, _ = _freq(128, "plain")
    out, none = nvkv.rope(q, None, pos, f)
    assert none is None
    _check(out, q, pos, f, 1.0, False, 128)


@pytest.mark.parametrize("inter", [False, True])
def test_rope_negated_positions_transpose(inter):
    """<R x, y> = <x, R^T y>, R^T the call with negated positions: each side is
    off by its rows' roundings, eps / 2 of |x| |y| a row (Cauchy-Schwarz), and
    the f32 part below."""
    g = torch.Generator().manual_seed(5)
    x, y = (torch.randn(64, 4, 96, generator=g).bfloat16().cuda() for _ in range(2))
    pos = torch.randint(0, 131072, (64,), generator=g).cuda()
    f, a = _freq(64)
    rx, _ = nvkv.rope(x, None, pos, f, a, inter)
    ty, _ = nvkv.rope(y, None, -pos, f, a, inter)
    lhs = (rx.double() * y.double()).sum(-1)
    rhs = (x.double() * ty.double()).sum(-1)
    tol = x.double().norm(dim=-1) * y.double().norm(dim=-1) * a * (2.0 ** -8 * 2 + 2.0 ** -19)
    assert bool(((lhs - rhs).abs() <= tol).all())


def test_rope_gradient_against_differences():
    """The map is linear: (R (x + h) - R x) = R h for h a power of two along one
    dim, up to both roundings; R^T e_i gives the same numbers."""
    T, d, rot = 3, 16, 8
    pos = torch.tensor([1, 77, 5000]).cuda()
    f, a = _freq(rot, "linear")
    eye = torch.eye(d).half().cuda().view(1, d, d).expand(T, d, d).contiguous()  # head i = e_i
    cols, _ = nvkv.rope(eye, None, pos, f, a, True)      # cols[t, i] = R e_i
    rows, _ = nvkv.rope(eye, None, -pos, f, a, True)     # rows[t, j] = R^T e_j
    diff = (cols.double() - rows.double().transpose(1, 2)).abs()
    assert float(diff.max()) <= 2 * (2.0 ** -11 * 1.0) + 2.0 ** -20
    x = torch.randn(T, 1, d, generator=torch.Generator().manual_seed(1)).half().cuda()
    h = 4.0
    for i in range(d):
        up, down = x.clone(), x.clone()
        up[..., i] += h
        down[..., i] -= h
        du = (up[..., i] - down[..., i]).double()  # the step as f16 holds it
        yu, _ = nvkv.rope(up, None, pos, f, a, True)
        yd, _ = nvkv.rope(down, None, pos, f, a, True)
        slope = (yu.double() - yd.double()) / du[..., None]
        big = float(torch.maximum(yu.abs().max(), yd.abs().max()))
        tol = 2 * big * 2.0 ** -11 / float(du.min()) + 2.0 ** -11 + 2.0 ** -18
        assert float((slope[:, 0] - cols[:, i].double()).abs().max()) <= tol


def test_rope_on_a_side_stream_and_in_a_graph():
    g = torch.Generator().manual_seed(9)
    q = torch.randn(300, 8, 128, generator=g).bfloat16().cuda()
    pos = torch.arange(300).cuda()
    f, a = _freq(128)
    want, _ = nvkv.rope(q, None, pos, f, a)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got, _ = nvkv.rope(q, None, pos, f, a)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        nvkv.rope(q, None, pos, f, a, q_out=out)
    q.mul_(2)
    pos.add_(1000)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, nvkv.rope(q, None, pos, f, a)[0])

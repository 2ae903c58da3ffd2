"""Pools, tables and checks shared by the tests of the block-scaled e4m3 cache."""
import numpy as np
import torch

import nvkv_oracle as O
from nvkv import ops

D, G = 128, 16


def empty_pool(nb, P, hkv, fill=0x7F):
    """A pool of stale memory: NaN codes, NaN scales."""
    kc = torch.full((nb, P, hkv, D), fill, dtype=torch.uint8, device="cuda")
    sc = torch.full((nb, hkv, P // G, 2), float("nan"), device="cuda")
    return kc, kc.clone(), sc


def tables(k_lens, P, seed, spare=2):
    """A seeded permutation of the pool's pages as block tables [B, W]."""
    need = [(L + P - 1) // P for L in k_lens]
    perm = np.random.default_rng(seed).permutation(sum(need) + spare)
    bt = np.zeros((len(need), max(1, max(need))), np.int32)
    u = 0
    for i, n in enumerate(need):
        bt[i, :n] = perm[u:u + n]
        u += n
    return bt, sum(need) + spare


def slots_of(bt, b, lo, hi, P):
    t = np.arange(lo, hi)
    return bt[b, t // P].astype(np.int64) * P + t % P


def filled(k_lens, hkv, P=256, seed=0, dtype=torch.bfloat16, k_gain=1.0, v_gain=1.0):
    """A pool holding k_lens keys per sequence, written by nvkv_rope_append with
    positions 0 (no rotation); every other row is NaN codes.  Returns the pool,
    the tables and the dequantised f64 rows per sequence."""
    bt, nb = tables(k_lens, P, seed)
    pool = empty_pool(nb, P, hkv)
    g = torch.Generator().manual_seed(seed + 1)
    n = sum(k_lens)
    k = (torch.randn(n, hkv, D, generator=g) * torch.exp(torch.randn(hkv, D, generator=g) / 2) *
         k_gain).to(dtype)
    v = (torch.randn(n, hkv, D, generator=g) * torch.exp(torch.randn(n, hkv, 1, generator=g)) *
         v_gain).to(dtype)
    slots = np.concatenate([slots_of(bt, b, 0, L, P) for b, L in enumerate(k_lens)] or
                           [np.zeros(0, np.int64)])
    f = torch.ones(4, dtype=torch.float64, device="cuda")
    ops.rope_append(None, k.cuda(), v.cuda(), torch.zeros(n, dtype=torch.int64, device="cuda"), f,
                    pool[0], pool[1], torch.from_numpy(slots).cuda(), kv_scale=pool[2])
    torch.cuda.synchronize()
    kn, vn, sn = (t.cpu().numpy() for t in pool)
    rows = []
    for b, L in enumerate(k_lens):
        s = slots_of(bt, b, 0, L, P)
        pg, off = s // P, s % P
        rows.append([O.e4m3_decode(c[pg, off]).astype(np.float64) *
                     sn[pg, :, off // G, w][..., None].astype(np.float64)
                     for w, c in ((0, kn), (1, vn))])
    return pool, torch.from_numpy(bt).cuda(), rows


def attend64(q, k, v, scale, causal=True):
    """(softmax(scale q k^T) v, softmax(..) |v|) in f64: q [n, Hq, D], k / v
    [L, Hkv, D]; the second bounds what errors of the weights can do."""
    n, hq, _ = q.shape
    L, hkv = k.shape[0], k.shape[1]
    qh = q.astype(np.float64).reshape(n, hkv, hq // hkv, D)
    s = np.einsum("ihgd,jhd->hgij", qh, k) * scale
    if causal:
        s = np.where(np.arange(L) <= np.arange(n)[:, None] + (L - n), s, -np.inf)
    p = np.exp(s - s.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return [np.einsum("hgij,jhd->ihgd", p, x).reshape(n, hq, D) for x in (v, np.abs(v))]


def check_attention(got, q, rows, q_lens, k_lens, scale, weight_err, causal=True, every=1):
    """got against f64 on the dequantised rows.  Tolerance: one rounding to the
    dtype (eps / 2 of the value) plus weight_err of sum p |v|, the relative error
    that the kernel's softmax weights may have."""
    qn, gn = q.double().cpu().numpy(), got.double().cpu().numpy()
    at = np.cumsum([0] + list(q_lens))
    eps = torch.finfo(got.dtype).eps
    for b in range(0, len(q_lens), every):
        if q_lens[b] == 0:
            continue
        s = slice(at[b], at[b + 1])
        want, bound = attend64(qn[s], *rows[b], scale, causal)
        tol = abs(want) * eps / 2 * (1 + 2.0 ** -10) + bound * weight_err + 2.0 ** -25
        err = abs(gn[s] - want)
        assert np.isfinite(gn[s]).all(), f"seq {b}: not finite"
        assert (err <= tol).all(), (f"seq {b} (q {q_lens[b]}, k {k_lens[b]}): off by "
                                    f"{float((err / tol).max()):.2f} tolerances")

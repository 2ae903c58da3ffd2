"""Operators of the 8-bit paged KV cache for long contexts: what they compute,
in plain torch, and the calls a user makes of them.

  rope     rotary positions on q and k: half / interleaved layout, part of the
           head, frequencies scaled for long contexts.
  append   q/k RMSNorm + rotation + append of K and V to a paged cache: the
           model-dtype pool, or e4m3 codes with one power-of-two scale for each
           block of 16 tokens and kv head (then the blocks' rows are read back).
  attend   paged attention over that 8-bit cache: decode, short multi-token
           batches and prompts.

A pool has pages of 256 slots: codes [Nb, 256, Hkv, 128] uint8 (e4m3),
scales [Nb, Hkv, 16, 2] f32 (K, V).
"""
import math
import os
import sys

import torch

own = False

D = 128  # head size of the cache
P = 256  # slots a page
G = 16  # tokens that share a scale
MIN_E = -100  # smallest scale exponent
DT = {"bf16": torch.bfloat16, "f16": torch.float16}


def _ops():
    pkg = os.path.join(os.getcwd(), "nanovllm-rs_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from nvkv import ops
    return ops


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def _rope(name, tokens, hq, hkv, head, rot, inter, scaling, dtype, lo, hi):
    return dict(name=name, op="rope", tokens=tokens, hq=hq, hkv=hkv, head=head, rot=rot,
                interleaved=inter, scaling=scaling, dtype=dtype, pos_lo=lo, pos_hi=hi)


def _append(name, seqs, q_lo, q_hi, k_lo, k_hi, hq, hkv, rot, inter, scaling, norm, pool, dtype):
    return dict(name=name, op="append", seqs=seqs, q_lo=q_lo, q_hi=q_hi, k_lo=k_lo, k_hi=k_hi,
                hq=hq, hkv=hkv, rot=rot, interleaved=inter, scaling=scaling, norm=norm, pool=pool,
                dtype=dtype)


def _attend(name, seqs, q_lo, q_hi, k_lo, k_hi, hq, hkv, dtype):
    return dict(name=name, op="attend", seqs=seqs, q_lo=q_lo, q_hi=q_hi, k_lo=k_lo, k_hi=k_hi,
                hq=hq, hkv=hkv, dtype=dtype)


def listed():
    return [
        # a decode step of 256 sequences, plain frequencies: latency
        _rope("rope_decode_256", 256, 32, 8, 128, 128, False, "none", "bf16", 1024, 1536),
        # a full 16384-token prefill step with long-context (yarn) frequencies
        _rope("rope_prefill_16384", 16384, 32, 8, 128, 128, False, "yarn", "bf16", 0, 131072),
        # part of a smaller head, interleaved pairs, an odd number of rows
        _rope("rope_partial_1001", 1001, 16, 8, 96, 64, True, "linear", "f16", 0, 65536),
        # decode: one row each into the blocks that 256 sequences are filling
        _append("append_decode_256", 256, 1, 1, 1025, 1536, 32, 8, 128, False, "none", True,
                "block8", "bf16"),
        # 16 fresh prompts of 1024 tokens: whole blocks
        _append("append_prompts_16x1024", 16, 1024, 1024, 1024, 1024, 32, 8, 128, False, "yarn",
                True, "block8", "bf16"),
        # ragged chunks on cached contexts, model-dtype pool, interleaved part of the head
        _append("append_chunks_dtype", 24, 1, 300, 40, 1500, 16, 8, 64, True, "bands", False,
                "dtype", "f16"),
        # one short sequence: the smallest decode call
        _attend("attend_one_1000", 1, 1, 1, 1000, 1000, 32, 8, "bf16"),
        # a decode step of the 256-request workload, one layer
        _attend("attend_decode_256", 256, 1, 1, 1025, 1536, 32, 8, "bf16"),
        # long-context decode at one kv head a GPU
        _attend("attend_long_64x32768", 64, 1, 1, 32768, 32768, 8, 1, "bf16"),
        # four tokens a sequence (speculative verification) over ragged contexts
        _attend("attend_verify_64x4", 64, 4, 4, 512, 4096, 16, 8, "f16"),
        # fresh prompts
        _attend("attend_prompts_16x1024", 16, 1024, 1024, 1024, 1024, 32, 8, "bf16"),
        # chunks of long prompts next to decode rows
        _attend("attend_chunks_5", 5, 1, 511, 5000, 16000, 32, 8, "f16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attend"])
    dtype = rng.choice(["bf16", "f16"])
    inter = rng.random() < 0.5
    scaling = rng.choice(["none", "linear", "ntk", "yarn", "bands"])
    hkv = rng.choice([1, 2, 4, 8])
    hq = hkv * rng.choice([1, 2, 4, 5, 8])
    if op == "rope":
        head = rng.choice([64, 80, 96, 128, 256])
        rot = rng.choice([head, head // 2, 32])
        hi = _log_int(rng, 2, 131072)
        return _rope(None, _log_int(rng, 1, 8000), hq, hkv, head, rot, inter, scaling, dtype, 0,
                     hi) | {"name": "rope"}
    if op == "append":
        seqs = _log_int(rng, 1, 200)
        q_hi = _log_int(rng, 1, max(1, 8000 // seqs)) if rng.random() < 0.5 else 1
        k_hi = _log_int(rng, max(q_hi, 17), max(q_hi, 3000))
        return _append(None, seqs, max(1, q_hi // 4), q_hi, max(1, q_hi // 2), k_hi, hq, hkv,
                       rng.choice([128, 64, 32]), inter, scaling, rng.random() < 0.5,
                       rng.choice(["block8", "dtype"]), dtype) | {"name": "append"}
    kind = rng.choice(["decode", "short", "prompt"])
    if kind == "decode":
        seqs = _log_int(rng, 1, 256)
        k_hi = _log_int(rng, 1, max(1, min(40000, 3_000_000 // (seqs * hkv))))
        return _attend(None, seqs, 1, 1, max(1, k_hi // 3), k_hi, hq, hkv, dtype) | {"name": "attend"}
    if kind == "short":
        seqs, q = _log_int(rng, 1, 64), rng.randint(2, 8)
        k_hi = _log_int(rng, 2 * q, max(2 * q, min(20000, 1_000_000 // (seqs * hkv))))
        return _attend(None, seqs, 1, q, k_hi // 2, k_hi, hq, hkv, dtype) | {"name": "attend"}
    seqs = rng.randint(1, 6)
    q = _log_int(rng, 9, 800)
    k_hi = _log_int(rng, q + 10, max(q + 10, min(12000, 250_000_000 // (seqs * hq * q))))
    return _attend(None, seqs, 1, q, min(q, k_hi), k_hi, hq, hkv, dtype) | {"name": "attend"}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _frequencies(scaling, rot):
    """(inv_freq f64 [rot / 2], attention factor) of theta = 1e6; contexts of
    32768 stretched by 4."""
    theta, factor, orig = 1e6, 4.0, 32768
    i = torch.arange(rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        theta = theta * factor ** (rot / (rot - 2)) if rot > 2 else theta
    f = theta ** (-2.0 * i / rot)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "yarn":
        def turn_dim(turns):
            return rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(theta))
        low, high = max(math.floor(turn_dim(32.0)), 0), min(math.ceil(turn_dim(1.0)), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    if scaling == "bands":
        lo_f, hi_f = 1.0, 4.0
        wave = 2 * math.pi / f
        mix = ((orig / wave - lo_f) / (hi_f - lo_f)).clamp(0, 1)
        return f / factor * (1 - mix) + f * mix, 1.0
    return f, 1.0


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ints(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda")


def _encode_blocks(x, live):
    """Codes and scales of rows x [n * 16, Hkv, D] f32 in blocks of 16; `live`
    [n * 16] rows count (the others become NaN codes, as stale memory may)."""
    n, hkv = x.size(0) // G, x.size(1)
    xb = torch.where(live[:, None, None], x, 0.0).view(n, G, hkv, D)
    m, e = torch.frexp(xb.abs().amax(dim=(1, 3)))
    e = torch.where(m > 0, e - 9 + (m > 0.875).int(), MIN_E).clamp(min=MIN_E)
    codes = torch.ldexp(xb, -e[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(live.view(n, G, 1, 1), codes, 0x7F)
    return codes.view(n * G, hkv, D), torch.ldexp(torch.ones_like(m), e)


def _lens(case):
    """Query and key lengths of every sequence (q <= k): the case's own, so that
    every seed has the same shapes."""
    g = torch.Generator().manual_seed(case["seqs"] * 100003 + case["k_hi"] * 11 + case["q_hi"])
    n = case["seqs"]
    q = torch.randint(case["q_lo"], case["q_hi"] + 1, (n,), generator=g)
    k = torch.randint(case["k_lo"], case["k_hi"] + 1, (n,), generator=g)
    if case["q_hi"] > 1:  # at least one sequence of the longest chunk
        q[0] = case["q_hi"]
    return q.cuda(), torch.maximum(k, q).cuda()


def _tables(k, g):
    """Pages of every sequence, a permutation of the pool: [B, W], pool size."""
    need = (k + P - 1) // P
    total, width = int(need.sum()), int(need.max())
    perm = torch.randperm(total + 2, generator=g, device="cuda")
    start = torch.cumsum(need, 0) - need
    col = torch.arange(width, device="cuda")
    idx = (start[:, None] + col).clamp(max=total + 1)
    return torch.where(col < need[:, None], perm[idx], 0).to(torch.int32), total + 2


def _pool(nb, hkv, live, g, dtype_pool=None):
    """A pool whose live slots [Nb * P] hold rows: keys with a few loud
    channels, values of varying size."""
    n = nb * P
    gain = torch.exp(0.5 * _rand(g, hkv, D))
    if dtype_pool is not None:
        k = (_rand(g, n, hkv, D) * gain).to(dtype_pool)
        v = _rand(g, n, hkv, D).to(dtype_pool)
        return k.view(nb, P, hkv, D), v.view(nb, P, hkv, D), None
    codes, scales = [], []
    for what in ("k", "v"):
        c, s = [], []
        for lo in range(0, nb, 512):  # bounded temporaries
            rows = slice(lo * P, min(lo + 512, nb) * P)
            x = _rand(g, rows.stop - rows.start, hkv, D)
            x = x * gain if what == "k" else x * torch.exp(0.5 * _rand(g, x.size(0), hkv, 1))
            a, b = _encode_blocks(x, live[rows])
            c.append(a)
            s.append(b)
        codes.append(torch.cat(c).view(nb, P, hkv, D))
        scales.append(torch.cat(s).view(nb, P // G, hkv))
    scale = torch.stack(scales, -1).permute(0, 2, 1, 3).contiguous()
    return codes[0], codes[1], scale


def _cu(lens):
    z = torch.zeros(1, dtype=torch.int64, device="cuda")
    return torch.cat([z, torch.cumsum(lens, 0)]).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    dt = DT[case["dtype"]]
    if case["op"] == "rope":
        f, a = _frequencies(case["scaling"], case["rot"])
        T = case["tokens"]
        qkv = _rand(g, T, (case["hq"] + 2 * case["hkv"]) * case["head"]).to(dt)
        qw, kw = case["hq"] * case["head"], case["hkv"] * case["head"]
        pos = _ints(g, case["pos_lo"], case["pos_hi"] - 1, T)
        return dict(case=case, q=qkv[:, :qw].view(T, case["hq"], case["head"]),
                    k=qkv[:, qw:qw + kw].view(T, case["hkv"], case["head"]), pos=pos,
                    f=f.cuda(), a=a)
    q_len, k_len = _lens(case)
    tables, nb = _tables(k_len, g)
    hq, hkv, T = case["hq"], case["hkv"], int(q_len.sum())
    seq = torch.repeat_interleave(torch.arange(case["seqs"], device="cuda"), q_len)
    cu_q = _cu(q_len)
    i = torch.arange(T, device="cuda") - cu_q.long()[seq]
    pos = (k_len - q_len)[seq] + i
    # which slots hold a key: before the call (append) or at the call (attend)
    limit = k_len - q_len if case["op"] == "append" else k_len
    t = torch.arange(tables.size(1) * P, device="cuda")
    slots = tables.long().repeat_interleave(P, 1) * P + t % P
    live = torch.zeros(nb * P, dtype=torch.bool, device="cuda")
    live[slots[t < limit[:, None]]] = True
    if case["op"] == "append":
        f, a = _frequencies(case["scaling"], case["rot"])
        qkv = _rand(g, T, (hq + 2 * hkv) * D).to(dt)
        qkv[:, hq * D:(hq + hkv) * D] *= 2
        q, k, v = qkv.split([hq * D, hkv * D, hkv * D], 1)
        slot = slots[seq, pos]
        kc, vc, sc = _pool(nb, hkv, live, g, None if case["pool"] == "block8" else dt)
        w = (1 + 0.1 * _rand(g, 2, D)).to(dt) if case["norm"] else (None, None)
        # the blocks that the call reaches, each by its first token, and their rows in use
        first = torch.ones(T, dtype=torch.bool, device="cuda")
        first[1:] = slot[1:] // G != slot[:-1] // G
        lead = first.nonzero().flatten()
        rows = slot[lead][:, None] // G * G + torch.arange(G, device="cuda")
        end = (pos[lead] // G + 1) * G
        used = torch.minimum(end, k_len[seq[lead]]) - pos[lead] // G * G
        back = rows[torch.arange(G, device="cuda") < used[:, None]]
        return dict(case=case, q=q.view(T, hq, D), k=k.view(T, hkv, D), v=v.view(T, hkv, D),
                    pos=pos, f=f.cuda(), a=a, kc=kc, vc=vc, sc=sc, slot=slot, qw=w[0], kw=w[1],
                    lead=lead, back=back)
    kc, vc, sc = _pool(nb, hkv, live, g)
    prompts = int(k_len[q_len > 1].sum())
    return dict(case=case, q=_rand(g, T, hq, D).to(dt), kc=kc, vc=vc, sc=sc, tables=tables,
                cu_q=cu_q, cu_k=_cu(k_len), max_q=int(q_len.max()), max_k=int(k_len.max()),
                q_len=q_len, k_len=k_len, seq=seq, i=i, prompts=prompts, scale=D ** -0.5)


# ---------------------------------------------------------------------------
# the operators, plain
# ---------------------------------------------------------------------------

def _rotate(x, pos, f, a, inter):
    """x [T, H, d] f32 rotated by pos * f (angles in 64 bits)."""
    r = 2 * f.numel()
    ang = pos.double()[:, None] * f
    c = (a * ang.cos()).float()[:, None]
    s = (a * ang.sin()).float()[:, None]
    y = x.clone()
    if inter:
        x0, x1 = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = x0 * c - x1 * s, x1 * c + x0 * s
    else:
        x0, x1 = x[..., :r // 2], x[..., r // 2:r]
        y[..., :r // 2], y[..., r // 2:r] = x0 * c - x1 * s, x1 * c + x0 * s
    return y


def _norm(x, w):
    x = x.float()
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


def _append_plain(s, c):
    dt, inter = s["q"].dtype, c["interleaved"]
    q = _rotate(_norm(s["q"], s["qw"]), s["pos"], s["f"], s["a"], inter).to(dt)
    k = _rotate(_norm(s["k"], s["kw"]), s["pos"], s["f"], s["a"], inter)
    hkv, slot = c["hkv"], s["slot"]
    if s["sc"] is None:
        s["kc"].view(-1, hkv, D)[slot] = k.to(dt)
        s["vc"].view(-1, hkv, D)[slot] = s["v"]
        return [q, s["kc"], s["vc"]]
    rows = torch.stack([k, s["v"].float()], 2)  # [T, Hkv, 2, D]
    kc, vc = s["kc"].view(-1, hkv, D), s["vc"].view(-1, hkv, D)
    nblk, blk = kc.size(0) // G, slot // G
    amax = torch.zeros(nblk, hkv, 2, device="cuda")
    amax.index_reduce_(0, blk, rows.abs().amax(-1), "amax")
    low = torch.full((nblk,), G, device="cuda").index_reduce_(0, blk, slot % G, "amin")
    m, e = torch.frexp(amax)
    e = torch.where(m > 0, e - 9 + (m > 0.875).int(), MIN_E).clamp(min=MIN_E)
    lb = blk[s["lead"]]  # the blocks reached, once each
    old = torch.frexp(s["sc"][lb // (P // G), :, lb % (P // G)])[1] - 1
    e[lb] = torch.where((low[lb] > 0)[:, None, None], torch.maximum(e[lb], old), e[lb])
    value = torch.ldexp(torch.ones_like(amax), e)
    s["sc"][lb // (P // G), :, lb % (P // G)] = value[lb]
    at = lb[:, None] * G + torch.arange(G, device="cuda")
    codes = torch.stack([kc[at], vc[at]], 3)  # the blocks' rows, [n, 16, Hkv, 2, D]
    shift = torch.exp2((old - e[lb]).float())[:, None, :, :, None]
    again = (codes.view(torch.float8_e4m3fn).float() * shift).to(torch.float8_e4m3fn)
    stay = (torch.arange(G, device="cuda") < low[lb][:, None])[..., None, None, None]
    codes = torch.where(stay, again.view(torch.uint8), codes)
    fresh = torch.ldexp(rows, -e[blk][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    kc[at], vc[at] = codes[..., 0, :], codes[..., 1, :]
    kc[slot], vc[slot] = fresh[:, :, 0], fresh[:, :, 1]
    back = torch.stack([kc[s["back"]], vc[s["back"]]], 2).view(torch.float8_e4m3fn).float()
    back = (back * value[s["back"] // G][..., None]).to(dt)
    return [q, back[:, :, 0].contiguous(), back[:, :, 1].contiguous()]


def _values(codes, scale, tables, which):
    """Rows of every sequence as f32, [B, W * P, Hkv, D]."""
    B, W = tables.shape
    hkv = codes.size(2)
    x = codes[tables.long()].view(torch.float8_e4m3fn).float()  # [B, W, P, Hkv, D]
    sc = scale[tables.long()][..., which].transpose(2, 3)  # [B, W, P / G, Hkv]
    return (x.view(B, W, P // G, G, hkv, D) * sc[:, :, :, None, :, None]).view(B, W * P, hkv, D)


def _attend_plain(s, c):
    hq, hkv = c["hq"], c["hkv"]
    B, n = s["tables"].size(0), s["tables"].size(1) * P
    q = torch.zeros(B, s["max_q"], hq, D, device="cuda")
    q[s["seq"], s["i"]] = s["q"].float()
    q = q.view(B, s["max_q"], hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, -1, D)
    k = _values(s["kc"], s["sc"], s["tables"], 0).permute(0, 2, 3, 1)
    j = torch.arange(n, device="cuda")
    sc = torch.matmul(q, k) * s["scale"]
    del k
    sc = sc.view(B, hkv, hq // hkv, s["max_q"], n)
    i = torch.arange(s["max_q"], device="cuda")
    seen = j <= (i + (s["k_len"] - s["q_len"])[:, None])[..., None]  # [B, max_q, n]
    seen &= (j < s["k_len"][:, None])[:, None]
    sc = torch.where(seen[:, None, None], sc, -math.inf)
    p = torch.exp(sc - sc.amax(-1, keepdim=True).clamp(min=-3e38))
    del sc
    total = p.sum(-1, keepdim=True)
    v = _values(s["vc"], s["sc"], s["tables"], 1)
    v = torch.where((j < s["k_len"][:, None])[..., None, None], v, 0.0).permute(0, 2, 1, 3)
    o = torch.matmul(p.view(B, hkv, -1, n), v).view(B, hkv, hq // hkv, s["max_q"], D)
    o = (o / total).permute(0, 3, 1, 2, 4).reshape(B, s["max_q"], hq, D)
    return o[s["seq"], s["i"]].to(s["q"].dtype)


def run(state):
    s, c = state, state["case"]
    if own:
        ops = _ops()
        if c["op"] == "rope":
            return list(ops.rope(s["q"], s["k"], s["pos"], s["f"], attn_factor=s["a"],
                                 interleaved=c["interleaved"]))
        if c["op"] == "append":
            q = ops.rope_append(s["q"], s["k"], s["v"], s["pos"], s["f"], s["kc"], s["vc"],
                                s["slot"], kv_scale=s["sc"], attn_factor=s["a"],
                                interleaved=c["interleaved"], q_norm_w=s["qw"], k_norm_w=s["kw"],
                                eps=1e-6)
            if s["sc"] is None:
                return [q, s["kc"], s["vc"]]
            return [q, *ops.load_kvcache_fp8b(s["kc"], s["vc"], s["sc"], s["back"],
                                              dtype=s["q"].dtype)]
        return ops.paged_attention_fp8b(s["q"], s["kc"], s["vc"], s["sc"], s["cu_q"], s["cu_k"],
                                        s["tables"], s["max_q"], s["max_k"], s["scale"],
                                        prompt_kv_tokens=s["prompts"])
    if c["op"] == "rope":
        x = [_rotate(t.float(), s["pos"], s["f"], s["a"], c["interleaved"]) for t in (s["q"], s["k"])]
        return [t.to(s["q"].dtype) for t in x]
    return _append_plain(s, c) if c["op"] == "append" else _attend_plain(s, c)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------

def _mean_lens(case):
    """Expected sums of the ragged lengths: tokens, keys, (query, key) pairs."""
    n = case["seqs"]
    q = (case["q_lo"] + case["q_hi"]) / 2
    k = max((case["k_lo"] + case["k_hi"]) / 2, q)
    return n * q, n * k, n * q * (k - (q - 1) / 2)


def work(case):
    if case["op"] == "rope":
        n = case["tokens"] * (case["hq"] + case["hkv"])
        return {"bytes": 4 * n * case["head"] + 8 * case["tokens"], "flops": 3 * n * case["rot"]}
    hq, hkv = case["hq"], case["hkv"]
    T, keys, pairs = _mean_lens(case)
    if case["op"] == "append":
        one = 1 if case["pool"] == "block8" else 2
        b = 2 * T * (hq + 2 * hkv) * D + 2 * T * hq * D + one * 2 * T * hkv * D + 16 * T
        if case["pool"] == "block8":  # the blocks' rows come back as values
            b += max(T, 8 * case["seqs"]) * hkv * D * 2 * (1 + 2)
        return {"bytes": b, "flops": 3 * T * (hq + hkv) * D + 2 * T * hkv * D}
    return {"bytes": keys * hkv * 2 * (D + 4 / G) + 4 * T * hq * D, "flops": 4 * D * hq * pairs}


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------

def _turn64(x, pos, f, a, inter):
    """The rotation as a product with e^(i angle)."""
    n = f.numel()
    w = torch.polar(torch.full((pos.numel(), n), a, dtype=torch.float64, device=pos.device),
                    pos.double()[:, None] * f)[:, None]
    head, rest = x[..., :2 * n], x[..., 2 * n:]
    pair = head.unflatten(-1, (n, 2)) if inter else head.unflatten(-1, (2, n)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * w)
    z = z.flatten(-2) if inter else z.transpose(-1, -2).flatten(-2)
    return torch.cat([z, rest], -1)


def _normed64(x, w):
    x = x.double()
    return x if w is None else x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()


def _append64(s, c):
    q = _turn64(_normed64(s["q"], s["qw"]), s["pos"], s["f"], s["a"], c["interleaved"])
    k = _turn64(_normed64(s["k"], s["kw"]), s["pos"], s["f"], s["a"], c["interleaved"])
    v, hkv, slot = s["v"].double(), c["hkv"], s["slot"]
    if s["sc"] is None:
        kc, vc = s["kc"].double(), s["vc"].double()
        kc.view(-1, hkv, D)[slot], vc.view(-1, hkv, D)[slot] = k, v
        return [q, kc, vc]
    out, blocks = [], slot // G
    for x, codes, which in ((k, s["kc"], 0), (v, s["vc"], 1)):
        val = codes.view(-1, hkv, D)[s["back"]].view(torch.float8_e4m3fn).double()
        b = s["back"] // G
        sc = s["sc"][b // (P // G), :, b % (P // G), which].double()
        val = val * sc[..., None]
        # position of each written token among the rows that come back
        order = torch.full((codes.size(0) * P,), -1, device=slot.device)
        order[s["back"]] = torch.arange(b.numel(), device=slot.device)
        low = torch.full((codes.size(0) * P // G,), G, device=slot.device)
        low.scatter_reduce_(0, blocks, slot % G, "amin")
        keep = s["back"] % G < low[b]
        top = torch.zeros(codes.size(0) * P // G, hkv, dtype=torch.float64, device=slot.device)
        top.index_reduce_(0, blocks, x.abs().amax(-1), "amax")
        step = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=MIN_E))
        step = torch.where(step * 448 < top, step * 2, step)
        step = torch.where((step * 224 >= top) & (step > 2.0 ** MIN_E), step / 2, step)
        unit = torch.where((low[b] > 0)[:, None], torch.maximum(step[b], sc), step[b])
        val = torch.where(keep[:, None, None], val, 0.0)
        val[order[slot]] = x
        out.append((val / unit[..., None]).to(torch.float8_e4m3fn).double() * unit[..., None])
    return [q, *out]


def _attend64(s, c):
    hq, hkv = c["hq"], c["hkv"]
    g = hq // hkv
    out = torch.zeros(s["q"].size(0), hq, D, dtype=torch.float64, device="cuda")
    q_at, q_n, k_n = s["cu_q"].tolist(), s["q_len"].tolist(), s["k_len"].tolist()
    for b in range(len(q_n)):
        L, n = k_n[b], q_n[b]
        t = torch.arange(L, device="cuda")
        page = s["tables"][b].long()[t // P]
        unit = s["sc"][page, :, t % P // G].double()  # [L, Hkv, 2]
        k = s["kc"][page, t % P].view(torch.float8_e4m3fn).double() * unit[..., :1]
        v = s["vc"][page, t % P].view(torch.float8_e4m3fn).double() * unit[..., 1:]
        q = s["q"][q_at[b]:q_at[b] + n].double().view(n, hkv, g, D)
        logit = torch.einsum("ihgd,jhd->hgij", q, k) * s["scale"]
        hide = t[None] > torch.arange(n, device="cuda")[:, None] + (L - n)
        logit.masked_fill_(hide, -math.inf)
        logit -= torch.logsumexp(logit, -1, keepdim=True)
        out[q_at[b]:q_at[b] + n] = torch.einsum("hgij,jhd->ihgd", logit.exp_(), v).reshape(n, hq, D)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rope":
        return [_turn64(t.double(), s["pos"], s["f"], s["a"], case["interleaved"])
                for t in (s["q"], s["k"])]
    return _append64(s, case) if case["op"] == "append" else _attend64(s, case)

"""The Qwen3 driver and the serving loop over the block-scaled e4m3 pool, and with
scaled rotary frequencies over the model-dtype pool.

* Plain frequencies through nvkv_rope_append (one rounding) against the prologue
  (the reference's rounding points): the same logit direction, cosine >= 0.99.
* The block-scaled pool against the model-dtype pool, teacher forced: cosine >=
  0.98 at every step, as the row-scaled pool's test asks.
* The engine over the block-scaled pool: graph replays give the tokens of eager
  steps, through prompts, ragged lengths and preemption.
"""
from dataclasses import replace

import numpy as np
import pytest
import torch

import nvkv
import nvkv_oracle as O
import test_gpu_greedy as G
from nvkv.decoder import Qwen3TP, RopeScaling, Step
from nvkv.engine import Engine

pytestmark = pytest.mark.gpu

CFG = replace(G.CFG, num_hidden_layers=6)


def _run(model, forced=None, steps=6):
    """Logits of `steps` steps (a prompt step, then decode) and the tokens fed."""
    seqs, free = G.make_seqs(11)
    logits, toks = [], []
    for step in range(steps):
        ids, pos, ctx = O.prepare_model_input(seqs, G.P)
        bt = O.prepare_block_tables(seqs)
        cu_q = torch.from_numpy(ctx.cu_seqlens_q.view(np.int32)).cuda()
        q_lens = np.diff(ctx.cu_seqlens_q.astype(np.int64))
        k_lens = np.diff(ctx.cu_seqlens_k.astype(np.int64))
        st = Step(torch.from_numpy(ids).cuda(), torch.from_numpy(pos).cuda(),
                  torch.from_numpy(ctx.slot_mapping).cuda(), cu_q,
                  torch.from_numpy(ctx.cu_seqlens_k.view(np.int32)).cuda(),
                  torch.from_numpy(bt.view(np.int32)).cuda(), (cu_q[1:] - 1).long(),
                  ctx.max_seqlen_q, ctx.max_seqlen_k,
                  prompt_kv_tokens=int(k_lens[q_lens > 1].sum()))
        lg = model.forward(st).float()
        logits.append(lg)
        toks.append(lg.argmax(-1).cpu().numpy() if forced is None else forced[step])
        G.Q.advance(seqs, toks[-1], free, G.P)
    torch.cuda.synchronize()
    assert nvkv.device_error() == 0
    return logits, toks


def _cos(a, b):
    return min(float(torch.nn.functional.cosine_similarity(x, y, dim=-1).min())
               for x, y in zip(a, b))


@pytest.mark.parametrize("scaling", [None, RopeScaling("yarn", 4.0, 128)])
def test_block_scaled_pool_against_dtype_pool(scaling):
    model = Qwen3TP(replace(CFG, rope_scaling=scaling), seed=3, device="cuda", **G.INIT)
    model.allocate_kv_cache(G.NB, G.P)
    base, toks = _run(model)
    model.allocate_kv_cache(G.NB, G.P, kv_fp8b=True)
    got, _ = _run(model, toks)
    assert all(torch.isfinite(x).all() for x in got)
    assert _cos(base, got) >= 0.98


def test_plain_frequencies_through_the_append():
    base = Qwen3TP(CFG, seed=3, device="cuda", **G.INIT)
    base.allocate_kv_cache(G.NB, G.P)
    want, toks = _run(base)
    model = Qwen3TP(replace(CFG, rope_scaling=RopeScaling("plain")), seed=3, device="cuda",
                    **G.INIT)
    model.allocate_kv_cache(G.NB, G.P)
    got, _ = _run(model, toks)
    assert _cos(want, got) >= 0.99


def test_random_fill_is_readable():
    model = Qwen3TP(replace(CFG, num_hidden_layers=1), seed=3, device="cuda", **G.INIT)
    model.allocate_kv_cache(3, 256, fill_random=True, kv_fp8b=True)
    k, v = nvkv.load_kvcache_fp8b(model.k_caches[0], model.v_caches[0], model.kv_scales[0],
                                  torch.arange(3 * 256).cuda())
    for t in (k, v):  # unit normal rows, up to e4m3's 2^-4
        assert abs(float(t.float().std()) - 1) < 0.02


def test_engine_graphs_and_preemption():
    """A small pool, so that sequences are preempted and resumed; the tokens do
    not depend on graph replay."""
    model = Qwen3TP(replace(CFG, num_hidden_layers=2), seed=4, device="cuda", **G.INIT)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, 1000, int(n)).tolist() for n in rng.integers(3, 200, 9)]
    outs = []
    for graphs in (False, True):
        model.allocate_kv_cache(10, 128, kv_fp8b=True)
        eng = Engine(model, 10, 128, max_num_seqs=8, max_num_batched_tokens=600,
                     max_model_len=512, cuda_graphs=graphs)
        outs.append(eng.generate(prompts, 40))
        steps = eng.graph_steps
        eng.close()
    assert nvkv.device_error() == 0
    assert steps > 0
    assert outs[0] == outs[1]

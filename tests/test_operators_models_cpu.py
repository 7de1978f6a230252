"""Branch norms, rotary positions with several axes, moves of pages and log probabilities where models, the pool, the engine and the
server use them (CPU)."""
import copy
import math

import pytest
import torch
from fastapi.testclient import TestClient

from mlxcel_b200.cache.kv_pool import KVPool
from mlxcel_b200.config import preset
from mlxcel_b200.engine import Engine, EngineConfig, SamplingParams
from mlxcel_b200.engine.scoring import prefill_hidden, sequence_logprobs, sequence_scores
from mlxcel_b200.models.decoder import DecoderModel, StepBatch
from mlxcel_b200.models.weights import random_weights
from mlxcel_b200.server.app import ServerState, create_app
from mlxcel_b200.server.worker import ModelWorker
from mlxcel_b200.tokenizer import ByteTokenizer


def _model(post_norms=False, sections=None, seed=0, **extra):
    """A tiny model with per-head q/k norms whose norm weights are not all alike."""
    cfg = copy.deepcopy(preset("tiny-qwen3"))
    cfg.post_norms = post_norms
    if sections:
        cfg.extra["mrope_section"] = sections
    cfg.extra.update(extra)
    w = random_weights(cfg, seed=seed, dtype=torch.float32, std=0.08)
    g = torch.Generator().manual_seed(seed + 1)
    for lw in w.layers:
        for n in ("q_norm", "k_norm", "ln1", "ln2", "post_attn_norm", "post_mlp_norm"):
            if getattr(lw, n) is not None:
                setattr(lw, n, 1.0 + 0.5 * torch.randn(getattr(lw, n).shape, generator=g))
    return cfg, DecoderModel(cfg, w)


def _prefill(cfg, model, ids, positions3=None, pool=None, table=None):
    T, bs = len(ids), 8
    nb = -(-T // bs)
    pool = pool or KVPool(cfg, nb, bs, dtype=torch.float32)
    i32 = dict(dtype=torch.int32)
    b = StepBatch(token_ids=torch.tensor(ids, **i32), positions=torch.arange(T, **i32), slot_mapping=torch.arange(T, **i32), num_prefill_seqs=1,
                  pf_block_tables=torch.arange(nb, **i32)[None], pf_cu_q=torch.tensor([0, T], **i32), pf_context_lens=torch.tensor([T], **i32),
                  pf_max_q_len=T, pf_max_len=T, pf_cu_q_host=[0, T], logits_rows=torch.arange(T))
    b.positions3 = positions3
    return model.forward(b, pool.layers), pool


def test_three_equal_axes_give_the_plain_positions():
    """With q/k norms whose weights differ along a head: the norm comes before the rotation in both paths."""
    ids = torch.randint(0, 1000, (21,), generator=torch.Generator().manual_seed(3)).tolist()
    for post in (False, True):
        cfg, model = _model(post)
        plain, pool = _prefill(cfg, model, ids)
        cfg.extra["mrope_section"] = [12, 10, 10]
        three, pool3 = _prefill(cfg, model, ids, torch.arange(21, dtype=torch.int32).expand(3, -1).contiguous())
        assert torch.allclose(plain, three, atol=2e-4)
        assert all(torch.allclose(a.k, b.k, atol=1e-4) and torch.equal(a.v, b.v) for a, b in zip(pool.layers[:1], pool3.layers[:1]))
        apart = torch.stack([torch.arange(21), torch.arange(21) % 5, torch.arange(21) % 7]).int()
        other, _ = _prefill(cfg, model, ids, apart)
        assert not torch.allclose(plain, other, atol=1e-2)


@pytest.mark.parametrize("post,scale,bias", [(True, 1.0, 0.0), (False, 0.3, 0.0), (True, 0.7, 1.0)])
def test_norms_around_sub_layers_in_the_layer_loop(post, scale, bias):
    """The joined steps against the layer loop written out."""
    cfg, model = _model(post, residual_multiplier=scale)
    cfg.norm_weight_bias = bias
    ids = list(range(1, 18))
    got, _ = _prefill(cfg, model, ids)
    rms = lambda x, w: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + cfg.rms_norm_eps) * (w + bias)    # noqa: E731
    pool = KVPool(cfg, 3, 8, dtype=torch.float32)
    i32 = dict(dtype=torch.int32)
    b = StepBatch(token_ids=torch.tensor(ids, **i32), positions=torch.arange(17, **i32), slot_mapping=torch.arange(17, **i32), num_prefill_seqs=1,
                  pf_block_tables=torch.arange(3, **i32)[None], pf_cu_q=torch.tensor([0, 17], **i32), pf_context_lens=torch.tensor([17], **i32),
                  pf_max_q_len=17, pf_max_len=17, pf_cu_q_host=[0, 17])
    h = model.w.embed[torch.tensor(ids)] * cfg.embed_scale
    for li, lw in enumerate(model.w.layers):
        o = model._attention(li, lw, rms(h, lw.ln1), b, pool.layers[li]) @ lw.wo.t()
        h = h + scale * (rms(o, lw.post_attn_norm) if post else o)
        o = model._mlp(lw, rms(h, lw.ln2)) @ lw.w_down.t()
        h = h + scale * (rms(o, lw.post_mlp_norm) if post else o)
    want = rms(h, model.w.final_norm) @ model.w.lm_head.t()
    assert torch.allclose(got, want, atol=1e-3 * want.abs().max().item())


# ----------------------------------------------------------------------------- pages of the pool
@pytest.mark.parametrize("bits", [16, 8, 4])
def test_pool_copies_snapshots_and_restores(bits, monkeypatch):
    from mlxcel_b200.cache import kv_pool
    cfg = preset("tiny-llama")
    pool = KVPool(cfg, 9, 8, kv_bits=bits, dtype=torch.float32)
    names = [(l, n) for l in pool.layers for n in kv_pool.SLABS if getattr(l, n) is not None]
    g = torch.Generator().manual_seed(1)
    for l, n in names:
        t = getattr(l, n)
        t.copy_(torch.randint(0, 200, t.shape, generator=g).to(t.dtype))
    first = [getattr(l, n).clone() for l, n in names]
    pool.copy_blocks([(0, 1), (1, 2), (2, 0), (3, 4), (3, 5)])          # a cycle and a fork
    want = list(range(9))
    for s, d in [(0, 1), (1, 2), (2, 0), (3, 4), (3, 5)]:
        want[d] = s
    for (l, n), f in zip(names, first):
        assert torch.equal(getattr(l, n), f[want])
    for limit in (1 << 30, 3000, 1):                                    # one staging buffer, a few slabs at a time, one by one
        monkeypatch.setattr(kv_pool, "STAGING_BYTES", limit)
        data = pool.extract_blocks([8, 0, 3])
        assert [sorted(d) for d in data] == [sorted(n for n in kv_pool.SLABS if getattr(l, n) is not None) for l in pool.layers]
        assert all(torch.equal(d[n], getattr(l, n)[[8, 0, 3]]) for l, d in zip(pool.layers, data) for n in d)
        other = KVPool(cfg, 5, 8, kv_bits=bits, dtype=torch.float32)
        other.restore_blocks([4, 1, 2], data)
        for a, b in zip(other.layers, data):
            assert all(torch.equal(getattr(a, n)[[4, 1, 2]], b[n]) and not getattr(a, n)[[0, 3]].any() for n in b)
    assert pool.extract_blocks([]) and pool.restore_blocks([], pool.extract_blocks([])) is None and pool.copy_blocks([]) is None
    for bad in ([(0, 9)], [(-1, 0)], [(0, 1), (2, 1)]):
        with pytest.raises(ValueError):
            pool.copy_blocks(bad)
    with pytest.raises(ValueError):
        pool.restore_blocks([1, 1, 2], data)
    pool.layers[0].k = pool.layers[0].k.clone()                         # a slab that was put in another's place
    before = pool.layers[0].k.clone()
    pool.copy_blocks([(7, 6)])
    assert torch.equal(pool.layers[0].k[6], before[7])


def test_snapshot_of_the_latent_pool_keeps_its_empty_slabs():
    cfg = copy.deepcopy(preset("tiny-llama"))
    cfg.extra.update(mla_latent=True, mla=dict(kv_lora_rank=24, rope=8))
    pool = KVPool(cfg, 4, 8, dtype=torch.float32)
    data = pool.extract_blocks([1, 2])
    assert data[0]["v"].shape == (2, 1, 8, 0) and data[0]["k"].shape == (2, 1, 8, 32)
    pool.restore_blocks([0, 3], data)


# ----------------------------------------------------------------------------- log probabilities
def test_scores_of_a_text():
    cfg, model = _model()
    ids = torch.randint(0, 1000, (40,), generator=torch.Generator().manual_seed(5)).tolist()
    h = prefill_hidden(model, cfg, ids, 8)
    lp = torch.log_softmax(model.logits(h, torch.arange(39)).double(), -1)
    for chunk in (7, 512):
        got = sequence_scores(model, cfg, ids, 8, row_chunk=chunk, top=5)
        assert torch.allclose(got.logprob.double(), lp.gather(1, torch.tensor(ids[1:])[:, None])[:, 0], atol=1e-4)
        assert torch.allclose(got.entropy.double(), -(lp.exp() * lp).sum(-1), atol=1e-4)
        want = lp.topk(5, -1)
        assert torch.equal(got.top_ids.long(), want.indices) and torch.allclose(got.top_logprobs.double(), want.values, atol=1e-4)
    assert torch.allclose(sequence_logprobs(model, cfg, ids, 8), got.logprob, atol=1e-5)
    assert sequence_scores(model, cfg, ids[:1], top=3).top_ids.shape == (0, 3)
    cfg.final_logit_softcap, cfg.extra["logits_scaling"] = 5.0, 2.0
    lp = torch.log_softmax(model.logits(h, torch.arange(39)).double(), -1)
    assert torch.allclose(sequence_logprobs(model, cfg, ids, 8).double(), lp.gather(1, torch.tensor(ids[1:])[:, None])[:, 0], atol=1e-4)


def test_alternatives_of_generated_tokens():
    cfg, model = _model()
    eng = Engine(model, cfg, EngineConfig(max_batch=4, max_num_batched_tokens=64, num_blocks=32, max_model_len=128, cuda_graphs=False))
    ask = [SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True, logprobs=True, top_logprobs=3),
           SamplingParams(max_tokens=4, temperature=0.9, seed=3, ignore_eos=True, logprobs=True, top_logprobs=6, logit_bias={5: float("-inf"), 9: 2.0}),
           SamplingParams(max_tokens=4, temperature=0.0, ignore_eos=True, logprobs=True)]
    sids = [eng.add_request([1, 2, 3, 4 + i], p) for i, p in enumerate(ask)]
    while eng.has_work():
        eng.step()
    for sid, p in zip(sids, ask):
        s = eng.seqs[sid]
        assert len(s.logprobs) == 4
        for tok, lp in zip(s.output, s.logprobs):
            top = getattr(lp, "top", None)
            if not p.top_logprobs:
                assert top is None
                continue
            assert len(top) == p.top_logprobs and [v for _, v in top] == sorted((v for _, v in top), reverse=True)
            assert all(math.isclose(v, float(lp), abs_tol=1e-5) for t, v in top if t == tok) and 5 not in [t for t, _ in top][:0 if p.greedy else None]
            if p.greedy:
                assert top[0][0] == tok


def test_server_returns_alternatives():
    cfg = preset("tiny-llama")
    w = random_weights(cfg, seed=0, dtype=torch.float32, std=0.05)
    eng = Engine(DecoderModel(cfg, w), cfg, EngineConfig(max_batch=4, max_num_batched_tokens=256, num_blocks=128, max_model_len=512, cuda_graphs=False))
    tk = ByteTokenizer(cfg.vocab_size)
    worker = ModelWorker(eng, tk, "tiny")
    try:
        with TestClient(create_app(ServerState(worker, tk, "tiny"))) as c:
            body = {"messages": [{"role": "user", "content": "hi"}], "max_tokens": 3, "temperature": 0, "ignore_eos": True, "logprobs": True}
            plain = c.post("/v1/chat/completions", json=body).json()["choices"][0]
            got = c.post("/v1/chat/completions", json={**body, "top_logprobs": 4}).json()["choices"][0]
            assert got["message"] == plain["message"] and all("top_logprobs" not in e for e in plain["logprobs"]["content"])
            for a, b in zip(got["logprobs"]["content"], plain["logprobs"]["content"]):
                assert len(a["top_logprobs"]) == 4 and a["top_logprobs"][0]["token"] == a["token"]
                assert math.isclose(a["logprob"], b["logprob"], abs_tol=1e-4) and math.isclose(a["top_logprobs"][0]["logprob"], a["logprob"], abs_tol=1e-5)
            # fewer tokens allowed than alternatives asked for: masked ones are not listed (and the answer stays JSON)
            few = c.post("/v1/chat/completions", json={**body, "top_logprobs": 10, "logit_bias": {str(i): False for i in range(3, cfg.vocab_size)}})
            assert few.status_code == 200
            t = c.post("/v1/completions", json={"prompt": "abc", "max_tokens": 2, "temperature": 0, "ignore_eos": True, "logprobs": True, "top_logprobs": 2}).json()
            # (a mapping by token text: the tiny vocabulary has ids of one text, of which the most likely stays)
            assert all(1 <= len(x) <= 2 for x in t["choices"][0]["logprobs"]["top_logprobs"]) and len(t["choices"][0]["logprobs"]["top_logprobs"]) == 2
            e = c.post("/v1/completions", json={"prompt": "hello", "max_tokens": 0, "echo": True, "logprobs": 3}).json()["choices"][0]["logprobs"]
            assert e["top_logprobs"][0] is None and len(e["top_logprobs"]) == len(e["token_logprobs"])
            for lp, top in zip(e["token_logprobs"][1:], e["top_logprobs"][1:]):
                assert 1 <= len(top) <= 3 and max(top.values()) >= lp - 1e-5
            e = c.post("/v1/completions", json={"prompt": "hello", "max_tokens": 0, "echo": True, "logprobs": True}).json()["choices"][0]["logprobs"]
            assert "top_logprobs" not in e
    finally:
        worker.shutdown()


@pytest.mark.parametrize("through_logits", [False, True])
def test_scores_hold_few_rows_of_logits(through_logits):
    """Logits of a long text are never held for more rows than asked for, with a head that scores hidden rows and with one that cannot."""
    cfg, model = _model()
    if through_logits:
        class Wrapped(DecoderModel):
            def logits(self, h, rows):
                return super().logits(h, rows)
        model = Wrapped(cfg, model.w)
    assert model.scores_from_hidden is not through_logits
    ids = [(7 * i) % cfg.vocab_size for i in range(90)]
    want = sequence_scores(model, cfg, ids, 8, row_chunk=89)
    rows, own = [], model.token_logprobs
    model.token_logprobs = lambda h, r, i, top=0: (rows.append(r.numel()), own(h, r, i, top))[1]
    got = sequence_scores(model, cfg, ids, 8, row_chunk=32)
    assert rows == [32, 32, 25]
    # the same sums of the same numbers, in products of 32 rows and of 89: fp32 rounding of 64 additions each
    torch.testing.assert_close(got.logprob, want.logprob, rtol=0, atol=1e-4)

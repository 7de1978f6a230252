"""Calls at the edge of what the branch norms, the rotary positions with several axes, the moves of pages and the log probabilities
take, and the paths of models, pool, engine and server around them (CPU)."""
import copy
import math
import os
import socket
import struct
import subprocess
import sys
import textwrap
import threading

import pytest
import torch
from fastapi.testclient import TestClient

from mlxcel_b200.cache import kv_pool
from mlxcel_b200.cache.kv_pool import KVPool
from mlxcel_b200.config import preset
from mlxcel_b200.engine import Engine, EngineConfig, SamplingParams
from mlxcel_b200.engine.scoring import prefill_hidden, sequence_scores
from mlxcel_b200.models.decoder import DecoderModel, StepBatch
from mlxcel_b200.models.depth_anything import Dinov2Backbone
from mlxcel_b200.models.weights import random_weights
from mlxcel_b200.multimodal.qwen2_vision import Glm4vVisionTower, Qwen2VisionTower
from mlxcel_b200.ops import KVLayer, _lib, logprobs, pages, rotary
from mlxcel_b200.server.app import ServerState, create_app
from mlxcel_b200.server.worker import ModelWorker
from mlxcel_b200.tokenizer import ByteTokenizer


# ----------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("heads", [dict(Hq=0, Hkv=0), dict(Hq=2, Hkv=-1), dict(Hq=-2, Hkv=1), dict(Hq=1, Hkv=1, D=0)])
def test_mrope_append_refuses_a_projection_without_heads(heads):
    kw = dict(D=64) | heads
    hkv, D = max(kw["Hkv"], 0), kw["D"]
    slab = lambda: torch.zeros(4, hkv, 8, D)    # noqa: E731
    with pytest.raises(ValueError):
        rotary.mrope_append(torch.zeros(5, max(0, (kw["Hq"] + 2 * kw["Hkv"]) * D)), torch.zeros(3, 5, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                            torch.ones(0), torch.zeros(0, dtype=torch.int32), KVLayer(slab(), slab(), None, None, 8), rot_dim=0, **kw)


def test_mrope_entry_refuses_no_heads_before_it_launches():
    """The C entry checks this itself (it returns before it asks for a device)."""
    args = rotary._ARGS.pack(*([16, 0] * 3), 16, 16, 64, *[16] * 5, 0, 0, 3, 5, 0, 0, 64, 64, 16, 0, 16, 1e-6, 1.0)
    assert len(args) == struct.calcsize(rotary._ARGS.format) and _lib.load().mx_mrope_append(args, None) == -1


@pytest.mark.parametrize("rows,heads", [(0, 2), (3, 0), (0, 0)])
def test_axial_rope_of_nothing(rows, heads):
    got = rotary.axial_rope(torch.zeros(rows, 3 * heads * 8), torch.zeros(2, rows, dtype=torch.int32), torch.ones(4), torch.zeros(4, dtype=torch.int32), heads=heads, D=8)
    assert [t.shape for t in got] == [(heads, rows, 8)] * 3


# ----------------------------------------------------------------------------- pages of the pool
def test_slabs_that_share_memory_are_refused():
    """A chain of copies would be taken once per slab: pages 0, 1, 2 in place of 0, 0, 1 became 0, 0, 0."""
    t, wide = torch.arange(12).view(4, 3), torch.arange(24)
    for bad in ([t, t], [t, t.view(4, 3)], [wide[:12].view(4, 3), wide[9:21].view(4, 3)], [wide[:8].view(4, 2), torch.zeros(4, 1), wide[7:11].view(4, 1)]):
        with pytest.raises(ValueError):
            pages.PageSlabs(bad)
    near = [wide[:12].view(4, 3), torch.zeros(4, 0), wide[12:].view(4, 3)]                    # (side by side is apart)
    pages.PageSlabs(near).copy([0, 1], [1, 2])
    assert wide.view(8, 3)[:, 0].tolist() == [0, 0, 3, 9, 12, 12, 15, 21]


@pytest.mark.parametrize("limit", [1 << 30, 5000, 1])
@pytest.mark.parametrize("bits", [16, 8])
def test_pool_restores_what_a_snapshot_has(bits, limit, monkeypatch):
    monkeypatch.setattr(kv_pool, "STAGING_BYTES", limit)
    cfg = copy.deepcopy(preset("tiny-llama"))
    cfg.num_hidden_layers = 4
    pool, g = KVPool(cfg, 6, 8, kv_bits=bits, dtype=torch.float32), torch.Generator().manual_seed(1)
    slabs = [(i, n) for i, l in enumerate(pool.layers) for n in kv_pool.SLABS if getattr(l, n) is not None]
    for i, n in slabs:
        t = getattr(pool.layers[i], n)
        t.copy_(torch.randint(1, 200, t.shape, generator=g).to(t.dtype))
    data = pool.extract_blocks([5, 1])
    whole = [dict(d) for d in data]
    del data[1]["v"], data[2]["k"], data[3]                    # slabs and a layer are not there
    other = KVPool(cfg, 6, 8, kv_bits=bits, dtype=torch.float32)
    other.restore_blocks([0, 4], data)
    for i, n in slabs:
        t = getattr(other.layers[i], n)
        there = i < len(data) and n in data[i]
        assert torch.equal(t[[0, 4]], whole[i][n] if there else torch.zeros_like(whole[i][n])) and not t[[1, 2, 3, 5]].any()
    other.restore_blocks([2, 3], [])
    assert not any(getattr(l, n)[[2, 3]].any() for l in other.layers for n in kv_pool.SLABS if getattr(l, n) is not None)


def test_pool_refuses_blocks_of_another_layout():
    cfg = preset("tiny-llama")
    pools = {bits: KVPool(cfg, 4, 8, kv_bits=bits, dtype=torch.float32) for bits in (16, 8, 4)}
    snaps = {bits: p.extract_blocks([1, 2]) for bits, p in pools.items()}
    for to, p in pools.items():
        for t in (getattr(l, n) for l in p.layers for n in kv_pool.SLABS if getattr(l, n) is not None):
            t.fill_(3)
        for frm, s in snaps.items():
            if frm != to:
                with pytest.raises(ValueError):
                    p.restore_blocks([0, 3], s)
        for bad in ([0], [0, 1, 2]):                           # another number of blocks than the snapshot has
            with pytest.raises(ValueError):
                p.restore_blocks(bad, snaps[to])
        assert all((getattr(l, n) == 3).all() for l in p.layers for n in kv_pool.SLABS if getattr(l, n) is not None)


# ----------------------------------------------------------------------------- models of other types
NORMS = ("ln1", "ln2", "post_attn_norm", "post_mlp_norm")


def _tiny(seed=0, dtype=torch.float32, post_norms=False, norms=None, **extra):
    """A tiny model whose weights are the same bf16 numbers in any type; ``norms``: the type of its norms around sub-layers."""
    cfg = copy.deepcopy(preset("tiny-qwen3"))
    cfg.post_norms = post_norms
    cfg.extra.update(extra)
    w = random_weights(cfg, seed=seed, dtype=torch.bfloat16, std=0.08)
    same = w.lm_head is w.embed
    for lw in w.layers:
        for n, v in vars(lw).items():
            if isinstance(v, torch.Tensor):
                setattr(lw, n, v.to(norms if norms and n in NORMS else dtype))
    w.embed, w.final_norm = w.embed.to(dtype), w.final_norm.to(dtype)
    w.lm_head = w.embed if same else w.lm_head.to(dtype)
    return cfg, DecoderModel(cfg, w)


@pytest.mark.parametrize("extra", [dict(post_norms=True), dict(residual_multiplier=0.3)])
def test_norms_around_sub_layers_in_other_types(extra):
    """On the CPU models run in any type, and norm weights may be of another than the rows."""
    ids = [(37 * i) % 1000 for i in range(21)]
    hidden = lambda **kw: prefill_hidden(*reversed(_tiny(**extra, **kw)), ids, 8)    # noqa: E731
    want = hidden().double()
    for dtype, u in ((torch.float16, 2.0 ** -11), (torch.float64, 2.0 ** -24)):
        got = hidden(dtype=dtype)
        # 2 layers, each of some 8 roundings to the row type (fp32 within): relative to the spread of the rows
        assert got.dtype == dtype and (got.double() - want).norm() < 16 * max(u, 2.0 ** -20) * want.norm()
    assert torch.equal(hidden(dtype=torch.bfloat16), hidden(dtype=torch.bfloat16, norms=torch.float32))


def test_image_positions_with_head_norms_of_another_type():
    """bf16 rows whose per-head norm weights are the same numbers in fp32."""
    def run(norms):
        cfg, model = _tiny(dtype=torch.bfloat16, mrope_section=[12, 10, 10])
        for lw in model.w.layers:
            lw.q_norm, lw.k_norm = (1.0 + torch.arange(64) / 64).to(norms), (2.0 - torch.arange(64) / 64).to(norms)
        T, i32 = 9, dict(dtype=torch.int32)
        pool = KVPool(cfg, 2, 8, dtype=torch.bfloat16)
        b = StepBatch(token_ids=torch.arange(3, 3 + T, **i32), positions=torch.arange(T, **i32), slot_mapping=torch.arange(T, **i32), num_prefill_seqs=1,
                      pf_block_tables=torch.arange(2, **i32)[None], pf_cu_q=torch.tensor([0, T], **i32), pf_context_lens=torch.tensor([T], **i32),
                      pf_max_q_len=T, pf_max_len=T, pf_cu_q_host=[0, T], logits_rows=torch.arange(T))
        b.positions3 = torch.stack([torch.arange(T), torch.arange(T) // 3, torch.arange(T) % 3]).int()
        return model.forward(b, pool.layers)
    assert torch.equal(run(torch.bfloat16), run(torch.float32))


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_vision_backbone_in_other_types(dtype):
    hid, cfg = 32, dict(hidden_size=32, num_hidden_layers=2, num_attention_heads=4, patch_size=4)
    g = torch.Generator().manual_seed(0)
    rn = lambda *s, scale=0.2: (torch.randn(*s, generator=g) * scale).to(torch.float16)    # noqa: E731
    t = {"embeddings.patch_embeddings.projection.weight": rn(hid, 3, 4, 4), "embeddings.patch_embeddings.projection.bias": rn(hid),
         "embeddings.cls_token": rn(1, 1, hid), "embeddings.position_embeddings": rn(1, 10, hid), "layernorm.weight": 1 + rn(hid), "layernorm.bias": rn(hid)}
    for i in range(2):
        p = f"encoder.layer.{i}."
        for n, shape in (("attention.attention.query", (hid, hid)), ("attention.attention.key", (hid, hid)), ("attention.attention.value", (hid, hid)),
                         ("attention.output.dense", (hid, hid)), ("mlp.fc1", (64, hid)), ("mlp.fc2", (hid, 64))):
            t[p + n + ".weight"], t[p + n + ".bias"] = rn(*shape), rn(shape[0])
        for n in ("norm1", "norm2"):
            t[p + n + ".weight"], t[p + n + ".bias"] = 1 + rn(hid), rn(hid)
        t[p + "layer_scale1.lambda1"], t[p + "layer_scale2.lambda1"] = rn(hid), rn(hid)
    x = rn(2, 3, 12, 12, scale=1.0)
    want = Dinov2Backbone(cfg, t, dtype=torch.float32).forward(x)[0].double()
    got = Dinov2Backbone(cfg, t, dtype=dtype).forward(x)[0]
    assert got.dtype == dtype and (got.double() - want).norm() < 24 * 2.0 ** -11 * want.norm()


def _tower(kind, dim=64, heads=2, dtype=torch.float32, device="cpu", blocks=3, head_norms=True, scale=0.2):
    """A small tower of random weights: Qwen2-VL's, or GLM-4V's (with norms of the heads, GLM-OCR's)."""
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: torch.randn(*s, generator=g) * scale    # noqa: E731
    t = {"patch_embed.proj.weight": rn(dim, 3, 2, 2, 2)}
    if kind is Qwen2VisionTower:
        for n in ("merger.ln_q", *(f"blocks.{i}.norm{j}" for i in range(blocks) for j in (1, 2))):
            t[n + ".weight"], t[n + ".bias"] = 1 + rn(dim), rn(dim)
        shapes = [(f"blocks.{i}.{n}", s) for i in range(blocks) for n, s in (("attn.qkv", (3 * dim, dim)), ("attn.proj", (dim, dim)), ("mlp.fc1", (2 * dim, dim)),
                                                                            ("mlp.fc2", (dim, 2 * dim)))]
        for n, s in shapes + [("merger.mlp.0", (4 * dim, 4 * dim)), ("merger.mlp.2", (dim, 4 * dim))]:
            t[n + ".weight"], t[n + ".bias"] = rn(*s), rn(s[0])
        return kind(dict(depth=blocks, embed_dim=dim, num_heads=heads, patch_size=2), t, dtype, device)
    t.update({"patch_embed.proj.bias": rn(dim), "post_layernorm.weight": 1 + rn(dim), "downsample.weight": rn(dim, dim, 2, 2), "downsample.bias": rn(dim),
              "merger.proj.weight": rn(dim, dim), "merger.post_projection_norm.weight": 1 + rn(dim), "merger.post_projection_norm.bias": rn(dim),
              "merger.gate_proj.weight": rn(dim, dim), "merger.up_proj.weight": rn(dim, dim), "merger.down_proj.weight": rn(dim, dim)})
    for i in range(blocks):
        b = f"blocks.{i}."
        t.update({b + "norm1.weight": 1 + rn(dim), b + "norm2.weight": 1 + rn(dim), b + "attn.qkv.weight": rn(3 * dim, dim), b + "attn.proj.weight": rn(dim, dim),
                  b + "mlp.gate_proj.weight": rn(dim, dim), b + "mlp.up_proj.weight": rn(dim, dim), b + "mlp.down_proj.weight": rn(dim, dim)})
        if head_norms:
            t.update({b + "attn.q_norm.weight": 1 + rn(dim // heads), b + "attn.k_norm.weight": 1 + rn(dim // heads)})
    return kind(dict(depth=blocks, hidden_size=dim, num_heads=heads, patch_size=2), t, dtype, device)


@pytest.mark.parametrize("kind,head_norms", [(Qwen2VisionTower, False), (Glm4vVisionTower, True), (Glm4vVisionTower, False)])
def test_towers_make_their_angles_once(kind, head_norms, monkeypatch):
    """The cosines of a forward are those of its grids, for all blocks, and the rows are those of angles made at every use."""
    tower, grids = _tower(kind, head_norms=head_norms), [(1, 4, 6), (1, 2, 2)]
    rows = torch.randn(28, 24, generator=torch.Generator().manual_seed(1))
    calls, cos = [], torch.Tensor.cos
    monkeypatch.setattr(torch.Tensor, "cos", lambda t: (calls.append(t.shape), cos(t))[1])
    got = tower.forward(rows, grids)
    assert len(calls) == 1
    # written out: each block's q and k turned as pairs (i, i + 16), i < 8 by the patch's row, else by its column
    angles = []
    for _, gh, gw in grids:
        hp = torch.arange(gh)[:, None].expand(gh, gw).reshape(gh // 2, 2, gw // 2, 2).permute(0, 2, 1, 3).flatten()
        wp = torch.arange(gw)[None].expand(gh, gw).reshape(gh // 2, 2, gw // 2, 2).permute(0, 2, 1, 3).flatten()
        angles.append(torch.cat([hp[:, None] * tower.inv_freq, wp[:, None] * tower.inv_freq], 1))
    c, s = (f(torch.cat(angles).double()).repeat(1, 2).float()[:, None] for f in (torch.cos, torch.sin))

    def turn(z):
        return z * c + torch.cat([-z[..., 16:], z[..., :16]], -1) * s

    def heads(qkv):
        q, k, v = qkv.view(28, 3, 2, 32).float().unbind(1)
        return [z.transpose(0, 1) for z in (turn(q), turn(k), v)]
    tower._axial = lambda grids: (heads, turn)
    want = tower.forward(rows, grids)
    assert torch.allclose(got, want, atol=1e-4 * want.abs().max().item())


# ----------------------------------------------------------------------------- log probabilities of requests


@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
@pytest.mark.parametrize("top", [0, 3])
def test_scores_of_models_in_other_types(dtype, top):
    """The log probabilities of the logits that the model makes, in whatever type: as an fp32 log softmax has them."""
    ids = [(37 * i) % 1000 for i in range(30)]
    cfg, model = _tiny(dtype=dtype)
    want = torch.log_softmax(model.logits(prefill_hidden(model, cfg, ids, 8), torch.arange(29)).float(), -1)
    got = sequence_scores(model, cfg, ids, 8, top=top)
    assert torch.allclose(got.logprob, want.gather(1, torch.tensor(ids[1:])[:, None])[:, 0], atol=1e-5)
    assert got.top_ids.shape == (29, top) and torch.allclose(got.top_logprobs, want.sort(dim=-1, descending=True, stable=True).values[:, :top], atol=1e-5)

    class Bare:                                      # a model that offers logits alone
        device = model.device

        def logits(self, h, rows):
            return model.logits(h, rows)

        def __getattr__(self, name):
            if name == "token_logprobs":
                raise AttributeError(name)
            return getattr(model, name)
    assert all(torch.equal(a, b) for a, b in zip(sequence_scores(Bare(), cfg, ids, 8, top=top), got))


def test_scores_with_a_head_or_bias_of_another_type():
    ids = [(37 * i) % 1000 for i in range(30)]
    for head, bias in ((torch.float16, None), (torch.bfloat16, None), (None, torch.float16), (None, torch.float64)):
        cfg, model = _tiny()
        if head:
            model.w.lm_head = model.w.lm_head.to(head)
        if bias:
            model.w.extra["lm_head_b"] = (torch.randn(cfg.vocab_size, generator=torch.Generator().manual_seed(1)) * 0.5).to(torch.bfloat16).to(bias)
        want = torch.log_softmax(model.logits(prefill_hidden(model, cfg, ids, 8), torch.arange(29)).double(), -1).gather(1, torch.tensor(ids[1:])[:, None])[:, 0]
        assert torch.allclose(sequence_scores(model, cfg, ids, 8).logprob.double(), want, atol=1e-4), (head, bias)


def test_log_probabilities_alone_order_no_vocabulary(monkeypatch):
    """Sorting every row costs thirty times what its log softmax does; alternatives come without it too, ties by index."""
    x = torch.randn(6, 3001, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).float() * 3
    x[1, 7:], x[2], x[3, 5], x[4, 100], x[5] = float("-inf"), float("-inf"), float("nan"), float("inf"), torch.finfo(torch.float32).min
    x[0, ::2], x[0, 1::2] = 0.0, -0.0
    z = torch.where(x.isnan(), torch.full_like(x, float("-inf")), x)
    want = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :64]
    ids = torch.randint(0, 3001, (6, 4), generator=torch.Generator().manual_seed(2))

    def never(*a, **k):
        raise AssertionError("a vocabulary was sorted")
    for name in ("sort", "argsort"):
        monkeypatch.setattr(torch, name, never)
        monkeypatch.setattr(torch.Tensor, name, never)
    r, alone = logprobs.token_logprobs(x, ids, top=64), logprobs.token_logprobs(x, ids)
    assert torch.equal(r.top_ids.long(), want) and alone.top_ids.shape == (6, 0)
    assert all(torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0)) for a, b in zip(r[:3], alone[:3]))
    assert torch.allclose(r.top_logprobs[5], torch.full((64,), -math.log(3001)), atol=1e-5) and r.top_logprobs[4, 0] == 0
    assert (r.top_logprobs[1, 7:] == float("-inf")).all() and (r.top_logprobs[2] == float("-inf")).all() and r.entropy[2] == 0


def test_alternatives_change_no_draw():
    """Seeded requests, alone and beside others, draw the same tokens whether or not they ask for alternatives."""
    cfg, model = _tiny()
    base = [dict(temperature=0.9, top_p=0.9, seed=3), dict(temperature=1.3, top_k=50, seed=4), dict(temperature=0.7, min_p=0.05, typical_p=0.9, seed=5),
            dict(temperature=0.0)]

    def run(extra):
        eng = Engine(model, cfg, EngineConfig(max_batch=4, max_num_batched_tokens=64, num_blocks=32, max_model_len=128, cuda_graphs=False))
        sids = [eng.add_request([1, 2, 3, 4 + i], SamplingParams(max_tokens=8, ignore_eos=True, **b, **e)) for i, (b, e) in enumerate(zip(base, extra))]
        while eng.has_work():
            eng.step()
        return [eng.seqs[s] for s in sids]
    want = run([{}] * 4)
    for extra in ([dict(logprobs=True, top_logprobs=5)] * 4, [dict(logprobs=True, top_logprobs=1 + 3 * i) if i % 2 else {} for i in range(4)],
                  [dict(top_logprobs=4)] * 4):
        for s, w, e in zip(run(extra), want, extra):
            assert s.output == w.output, e
            assert [len(lp.top) for lp in s.logprobs] == ([e["top_logprobs"]] * 8 if e.get("logprobs") else [])


def _serve(allowed=None):
    """A client of a tiny model, whose head allows all tokens or those of a text."""
    cfg = preset("tiny-llama")
    w, tk = random_weights(cfg, seed=0, dtype=torch.float32, std=0.05), ByteTokenizer(cfg.vocab_size)
    if allowed:
        w.extra["lm_head_b"] = torch.full((cfg.vocab_size,), float("-inf")).index_fill_(0, torch.tensor(tk.encode(allowed)), 0.0)
    eng = Engine(DecoderModel(cfg, w), cfg, EngineConfig(max_batch=4, max_num_batched_tokens=256, num_blocks=128, max_model_len=512, cuda_graphs=False))
    worker = ModelWorker(eng, tk, "tiny")
    try:
        with TestClient(create_app(ServerState(worker, tk, "tiny"))) as c:
            yield c
    finally:
        worker.shutdown()


@pytest.fixture(scope="module")
def client():
    yield from _serve()


def _complete(client, **body):
    r = client.post("/v1/completions", json={"prompt": "hello", "max_tokens": 3, "temperature": 0, "ignore_eos": True, **body})
    assert r.status_code == 200
    return r.json()["choices"][0].get("logprobs")


@pytest.mark.parametrize("ask", [dict(logprobs=4), dict(logprobs=True, top_logprobs=4), dict(logprobs=2, top_logprobs=4)])
def test_echo_lists_alternatives_of_prompt_and_generated_tokens_alike(client, ask):
    e = _complete(client, echo=True, **ask)
    n = len(e["tokens"])
    assert len(e["token_logprobs"]) == len(e["top_logprobs"]) == n and e["top_logprobs"][0] is None
    for lp, top in zip(e["token_logprobs"][1:], e["top_logprobs"][1:]):
        assert 1 <= len(top) <= 4 and max(top.values()) >= lp - 1e-5
    for lp, top in zip(e["token_logprobs"][-3:], e["top_logprobs"][-3:]):           # (drawn greedily: the most likely)
        assert math.isclose(max(top.values()), lp, abs_tol=1e-5)


def test_echo_without_log_probabilities_of_generated_tokens(client):
    e = _complete(client, echo=True, top_logprobs=4)
    assert len(e["top_logprobs"]) == len(e["token_logprobs"]) == len(e["tokens"])
    assert e["top_logprobs"][-3:] == e["token_logprobs"][-3:] == [None] * 3 and all(e["top_logprobs"][1:-3])


def test_echo_scores_between_steps_of_the_engine(client, monkeypatch):
    """A forward of the model beside the engine's would share the buffers that both keep in the model: one thread makes both."""
    threads, forward = [], DecoderModel.forward_hidden
    monkeypatch.setattr(DecoderModel, "forward_hidden", lambda self, *a, **k: (threads.append(threading.current_thread()), forward(self, *a, **k))[1])
    _complete(client, echo=True, logprobs=True)
    assert len(threads) >= 4 and len(set(threads)) == 1


def test_echo_behind_the_end_of_the_worker():
    """A worker that has ended makes no more calls: the request is answered with an error instead of waiting for it."""
    cfg, tk = preset("tiny-llama"), ByteTokenizer(preset("tiny-llama").vocab_size)
    eng = Engine(DecoderModel(cfg, random_weights(cfg, seed=0, dtype=torch.float32, std=0.05)), cfg, EngineConfig(num_blocks=32, max_model_len=128, cuda_graphs=False))
    worker = ModelWorker(eng, tk, "tiny")
    with TestClient(create_app(ServerState(worker, tk, "tiny"))) as c:
        def late():
            raise TimeoutError("its own")
        with pytest.raises(TimeoutError, match="its own"):
            worker.run_exclusive(late)
        worker.shutdown()
        r = c.post("/v1/completions", json={"prompt": "hello", "max_tokens": 0, "echo": True, "logprobs": True})
        assert r.status_code == 400 and "ended" in r.text


def test_a_number_of_log_probabilities_gives_alternatives_without_echo_too(client):
    got, want = _complete(client, logprobs=3), _complete(client, logprobs=True, top_logprobs=3)
    assert got == want and len(got["top_logprobs"]) == 3 and all(got["top_logprobs"])
    assert "top_logprobs" not in _complete(client, logprobs=True)


def test_echo_lists_no_alternatives_without_probability():
    """Fewer tokens have a probability than alternatives are asked for: the answer stays JSON and lists those."""
    served = _serve("hello")
    try:
        e = _complete(next(served), echo=True, logprobs=20)
        assert all(set(top) == set("helo") for top in e["top_logprobs"][1:])
    finally:
        served.close()


PIPELINE = """
import sys, torch, torch.distributed as dist
sys.path.insert(0, %r)
dist.init_process_group("gloo")
rank, world = dist.get_rank(), dist.get_world_size()
from mlxcel_b200.cache import kv_pool
from mlxcel_b200.cache.kv_pool import KVPool
from mlxcel_b200.config import preset
from mlxcel_b200.engine import Engine, EngineConfig, SamplingParams
from mlxcel_b200.engine.scoring import prefill_hidden, sequence_scores
from mlxcel_b200.models.decoder import DecoderModel, StepBatch
from mlxcel_b200.models.depth_anything import Dinov2Backbone
from mlxcel_b200.models.weights import random_weights
from mlxcel_b200.loading.shard import shard_weights, partition_layers
from mlxcel_b200.parallel.pp import PipelineContext, PipelineModel
cfg = preset("tiny-qwen3")
cfg.num_hidden_layers = 4
full = random_weights(cfg, seed=9, dtype=torch.float32, std=0.05)
asks = [dict(logprobs=True, top_logprobs=3), {}, dict(logprobs=True), dict(logprobs=True, top_logprobs=100, temperature=0.8, seed=4)]
def run(model):
    eng = Engine(model, cfg, EngineConfig(max_batch=4, max_num_batched_tokens=64, num_blocks=64, max_model_len=128, cuda_graphs=False))
    sids = [eng.add_request([5, 6, 7 + i], SamplingParams(**(dict(max_tokens=4, temperature=0.0, ignore_eos=True) | a))) for i, a in enumerate(asks)]
    while eng.has_work():
        eng.step()
    return [eng.seqs[s] for s in sids]
want = run(DecoderModel(cfg, full))
ranges = partition_layers(cfg.num_hidden_layers, world)
w = shard_weights(cfg, full, 0, 1, layers=ranges[rank], vocab_parallel=False)
got = run(PipelineModel(cfg, w, PipelineContext(dist.group.WORLD, rank, world), num_micro=2, layer_range=ranges[rank]))
for g, o, a, count in zip(got, want, asks, (3, None, None, 64)):
    assert g.output == o.output and len(g.logprobs) == len(o.logprobs) == (4 if a.get("logprobs") else 0), (rank, a)
    for x, y in zip(g.logprobs, o.logprobs):
        assert abs(x - y) < 1e-4 and hasattr(x, "top") == hasattr(y, "top") == (count is not None), (rank, a)
        if count:
            assert len(x.top) == count and [i for i, _ in x.top][:3] == [i for i, _ in y.top][:3], (rank, a)
            assert all(abs(u - v) < 1e-4 for (_, u), (_, v) in zip(x.top, y.top)), (rank, a)
dist.barrier()
if rank == 0:
    print("ALTERNATIVES_OK")
"""


def test_alternatives_cross_a_pipeline(tmp_path):
    """Two stages (gloo): every rank's requests have the alternatives that the last one found."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    script = tmp_path / "pipeline.py"
    script.write_text(textwrap.dedent(PIPELINE % root))
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        port = s.getsockname()[1]
    cmd = [sys.executable, "-m", "torch.distributed.run", "--nnodes=1", "--nproc-per-node=2", "--master-addr", "127.0.0.1", "--master-port", str(port), str(script)]
    r = subprocess.run(cmd, capture_output=True, text=True, timeout=600, env=dict(os.environ, MASTER_ADDR="127.0.0.1", OMP_NUM_THREADS="2"))
    assert r.returncode == 0 and "ALTERNATIVES_OK" in r.stdout, (r.stdout + r.stderr)[-3000:]

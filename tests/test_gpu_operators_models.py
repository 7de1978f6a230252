"""A request's path over the branch norms, the rotary positions with several axes, the moves of pages and the log probabilities
together, on the kernels (bf16) against the CPU (fp32): a model with norms around its sub-layers reads a prompt with image positions,
its pages are copied, snapshot and restored, it goes on decoding from the copies, and the text is scored."""
import copy

import pytest
import torch

from mlxcel_b200.cache.kv_pool import KVPool
from mlxcel_b200.config import preset
from mlxcel_b200.engine import Engine, EngineConfig, SamplingParams
from mlxcel_b200.engine.scoring import sequence_logprobs, sequence_scores
from mlxcel_b200.models.decoder import DecoderModel, StepBatch
from mlxcel_b200.models.weights import random_weights
from mlxcel_b200.ops import _lib

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    torch.cuda.synchronize()
    assert _lib.read_status(torch.device("cuda")) == 0


def _models(traditional=False, seed=0):
    """One model on the CPU in fp32 and on the GPU in bf16, from the same bf16 weights."""
    cfg = copy.deepcopy(preset("tiny-qwen3"))
    cfg.post_norms, cfg.rope_traditional = True, traditional
    if traditional:
        cfg.partial_rotary_factor = 0.5
    cfg.extra["mrope_section"] = [4, 6, 6] if traditional else [8, 12, 12]
    out = []
    for dev, dt in (("cpu", torch.float32), ("cuda", torch.bfloat16)):
        w = random_weights(cfg, seed=seed, dtype=torch.bfloat16, device="cpu", std=0.06)
        g = torch.Generator().manual_seed(seed + 1)
        for lw in w.layers:
            for n in ("q_norm", "k_norm", "ln1", "ln2", "post_attn_norm", "post_mlp_norm"):
                setattr(lw, n, (1.0 + 0.3 * torch.randn(getattr(lw, n).shape, generator=g)).to(torch.bfloat16))
            for n, v in vars(lw).items():
                if isinstance(v, torch.Tensor):
                    setattr(lw, n, v.to(dev, dt))
        same = w.lm_head is w.embed
        w.embed, w.final_norm = w.embed.to(dev, dt), w.final_norm.to(dev, dt)
        w.lm_head = w.embed if same else w.lm_head.to(dev, dt)
        out.append(DecoderModel(copy.deepcopy(cfg), w))
    return cfg, out


def _path(cfg, model, dev, dt, bits):
    """Logits of the prompt's rows and of a token decoded from copied, restored pages of another pool."""
    i32 = dict(dtype=torch.int32, device=dev)
    T, bs, nb = 37, 16, 3
    g = torch.Generator().manual_seed(7)
    ids = torch.randint(0, 1000, (T + 1,), generator=g)
    pos = torch.arange(T)
    pos3 = torch.stack([torch.where(pos < 25, 0 * pos, pos), torch.where(pos < 25, pos // 5, pos), torch.where(pos < 25, pos % 5, pos)])
    pool = KVPool(cfg, 8, bs, kv_bits=bits, device=dev, dtype=dt)
    b = StepBatch(token_ids=ids[:T].to(**i32), positions=pos.to(**i32), slot_mapping=torch.arange(T, **i32), num_prefill_seqs=1,
                  pf_block_tables=torch.arange(nb, **i32)[None], pf_cu_q=torch.tensor([0, T], **i32), pf_context_lens=torch.tensor([T], **i32),
                  pf_max_q_len=T, pf_max_len=T, pf_cu_q_host=[0, T], logits_rows=torch.arange(T, device=dev))
    b.positions3 = pos3.to(**i32).contiguous()
    prompt = model.forward(b, pool.layers).float().cpu()
    pool.copy_blocks([(0, 5), (1, 0), (5, 1), (2, 7)])                  # page 0 to 5, 1 to 0, what was in 5 to 1, 2 to 7
    data = pool.extract_blocks([5, 0, 7])
    other = KVPool(cfg, 11, bs, kv_bits=bits, device=dev, dtype=dt)
    other.restore_blocks([9, 2, 4], data)
    table = torch.tensor([[9, 2, 4]], **i32)
    d = StepBatch(token_ids=ids[T:].to(**i32), positions=torch.tensor([T], **i32), slot_mapping=torch.tensor([4 * bs + T - 2 * bs], **i32), num_decode=1,
                  dec_block_tables=table, dec_context_lens=torch.tensor([T + 1], **i32), dec_max_len=T + 1, logits_rows=torch.arange(1, device=dev))
    return prompt, model.forward(d, other.layers).float().cpu()


@pytest.mark.parametrize("traditional", [False, True])
@pytest.mark.parametrize("bits", [16, 8])
def test_prompt_pages_and_decode_together(traditional, bits):
    cfg, (cpu, gpu) = _models(traditional)
    want = _path(cfg, cpu, "cpu", torch.float32, bits)
    got = _path(cfg, gpu, "cuda", torch.bfloat16, bits)
    # 2 layers of bf16 rows: each sub-layer rounds its input, its products and the stream (half a step of 2^-8 each, some 8 of them a
    # layer), against fp32 rows; relative to the spread of the logits
    for g, w in zip(got, want):
        assert (g - w).norm() / w.norm() < 16 * 2.0 ** -8, ((g - w).norm() / w.norm()).item()


def test_scores_against_logits_and_the_cpu():
    cfg, (cpu, gpu) = _models()
    ids = torch.randint(0, 1000, (700,), generator=torch.Generator().manual_seed(2)).tolist()
    want = sequence_scores(cpu, cfg, ids[:120], top=5)
    got = sequence_scores(gpu, cfg, ids[:120], top=5)
    assert (got.logprob - want.logprob).abs().mean() < 16 * 2.0 ** -8 * want.logprob.abs().mean()
    assert ((got.entropy - want.entropy).abs() < 0.05 * want.entropy).all()
    # rows that keep their logits on the chip (more than 256) against those through memory: fp32 sums of 256 products in other orders
    long = sequence_logprobs(gpu, cfg, ids)
    short = sequence_logprobs(gpu, cfg, ids[:200])
    assert torch.isfinite(long).all() and (long[:199] - short).abs().max() < 0.05 * short.abs().max()


def test_alternatives_of_generated_tokens_and_an_unchanged_answer():
    cfg, (_, gpu) = _models()

    def run(p):
        eng = Engine(gpu, cfg, EngineConfig(max_batch=2, max_num_batched_tokens=64, num_blocks=32, max_model_len=128))
        sid = eng.add_request([5, 6, 7, 8], p)
        while eng.has_work():
            eng.step()
        return eng.seqs[sid]
    a = run(SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True))
    b = run(SamplingParams(max_tokens=6, temperature=0.0, ignore_eos=True, logprobs=True, top_logprobs=4))
    assert a.output == b.output and all(lp.top[0][0] == t and len(lp.top) == 4 and lp.top[0][1] == pytest.approx(float(lp), abs=1e-5)
                                        for t, lp in zip(b.output, b.logprobs))

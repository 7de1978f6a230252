"""Calls at the edge of what the kernels of the branch norms, the rotary positions with several axes, the moves of pages and the log
probabilities take, and the forms that their dispatch chooses for large calls."""
import math

import pytest
import torch
from test_gpu_operators import F64, _check_head, _check_mrope, _check_norm, _turned

from mlxcel_b200.ops import _lib, linear, logprobs, norms, recurrent, rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    torch.cuda.synchronize()
    assert _lib.read_status(torch.device(DEV)) == 0


def _rn(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


# ----------------------------------------------------------------------------- norms
def test_layernorm_refuses_types_that_its_kernel_would_misread():
    x, w, b = _rn(3, 64, seed=1), _rn(64, seed=2), _rn(64, seed=3)
    assert recurrent.layernorm(x, w, b).dtype == torch.bfloat16
    for bad in ((x.float(), w, b), (x, w.float(), b), (x, w, b.half()), (x.half(), w.half(), None)):
        with pytest.raises(ValueError):
            recurrent.layernorm(*bad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("dim", [1003, 4096, 5119, 5120, 8192])
def test_branch_norm_several_accesses_of_a_thread(dim, layer, dtype):
    """More than two rows an SM: a thread takes several vectors of a row; 1003 and 5119 elements by the vectors that hold them."""
    rows = 400
    x, res = _rn(rows, dim, seed=1, scale=3, dtype=dtype), _rn(rows, dim, seed=2, scale=8, shift=2, dtype=dtype)
    w1, w2, g, b = (_rn(dim, seed=3 + i, scale=0.3, shift=0.5, dtype=dtype) for i in range(4))
    kw = dict(post_w=None if layer else w1, gate=g if layer else None, pre_w=w2, pre_b=b if layer else None, layer_norm=layer, scale=0.22, w_bias=1.0)
    y, h = norms.branch_norm(x, res, **kw)
    _check_norm(x, res, y, h, **kw)


@pytest.mark.parametrize("layer", [False, True])
@pytest.mark.parametrize("dim", [1003, 4096])
def test_branch_norm_many_rows_element_by_element(dim, layer):
    """Rows that lie differently within 16 bytes; what is between and behind them stays as it was."""
    wide = [_rn(400, dim + 9, seed=s) for s in (1, 2, 3)]
    before = [t.clone() for t in wide]
    x, res, out = wide[0][:, 1:1 + dim], wide[1][:, 2:2 + dim], wide[2][:, 5:5 + dim]
    w, g = _rn(dim, seed=4, shift=1), _rn(dim, seed=5)
    kw = dict(post_w=w, gate=g, pre_w=w, layer_norm=layer)
    y, h = norms.branch_norm(x, res, out=out, **kw)
    _check_norm(x, res, y, h, **kw)
    before[2][:, 5:5 + dim] = h
    assert all(torch.equal(a, b) for a, b in zip(wide, before))


# ----------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("T", [1184, 1185, 2368, 2371, 4099])
def test_mrope_append_several_tokens_of_a_cta(T, bits):
    """From 8 tokens an SM on a CTA takes two, from 16 on four (and 16-bit pools accesses of 16 bytes); the last CTA has fewer. With few
    heads a warp's are of several tokens."""
    for i, (hq, hkv, D, rot, pairs, norm) in enumerate([(2, 1, 64, 64, False, True), (1, 1, 128, 64, True, False), (6, 2, 128, 128, False, True),
                                                        (3, 1, 256, 64, False, False), (2, 1, 64, 32, True, True)]):
        _check_mrope(T, hq, hkv, D, rot, pairs, bits, norm, far=70000, inplace=i % 2 == 0, strided=i == 2, seed=i, dead=((T - 1, -1), (T - 2, 2 ** 31 - 1), (5, -3)))


@pytest.mark.parametrize("D", [64, 72, 80])
@pytest.mark.parametrize("R", [1184, 1185, 2368, 2369, 2371])
def test_axial_rope_several_rows_of_a_cta(R, D):
    for H in (1, 5):
        qkv = _rn(R, 3 * H * D, seed=R)
        pos = torch.randint(0, 200, (2, R), generator=torch.Generator().manual_seed(2)).int().to(DEV)
        inv = (1.0 / 1e4 ** (torch.arange(D // 2).double() / D)).float().to(DEV)
        axes = (torch.arange(D // 2) % 2).int().to(DEV)
        got = rotary.axial_rope(qkv, pos, inv, axes, heads=H, D=D)
        q, k, v = qkv.to(F64).reshape(R, 3, H, D).unbind(1)
        for t, w in zip(got[:2], (q, k)):
            want, mag = _turned(w, pos, inv, axes, D, False)
            # (12 roundings of fp32: the reduced angle, its sine and cosine, two products and their sum)
            assert ((t.to(F64) - want.transpose(0, 1)).abs() <= 12 * 2.0 ** -24 * mag.transpose(0, 1)).all()
        assert torch.equal(got[2].to(F64), v.transpose(0, 1))


@pytest.mark.parametrize("off", [(0, 0, 0), (2, 0, 0), (0, 2, 0), (0, 0, 2), (1, 2, 3)])
def test_axial_entry_with_results_off_16_bytes(off):
    """The C entry with results on any boundary of 4 bytes: what the wrapper's own (aligned) results hold."""
    R, H, D = 9, 2, 16
    qkv = _rn(R, 3 * H * D, seed=1)
    pos = torch.arange(2 * R, device=DEV, dtype=torch.int32).view(2, R)
    inv, axes = torch.rand(D // 2, device=DEV), torch.arange(D // 2, device=DEV, dtype=torch.int32) % 2
    want = rotary.axial_rope(qkv, pos, inv, axes, heads=H, D=D)
    flat = [torch.zeros(R * H * D + 4, device=DEV) for _ in off]
    got = [t[o:o + R * H * D] for t, o in zip(flat, off)]
    assert [t.data_ptr() % 16 for t in got] == [4 * o for o in off]
    _lib.launch_on(qkv.device, "mx_axial_rope", qkv.data_ptr(), qkv.stride(0), *(t.data_ptr() for t in got), pos.data_ptr(), pos.stride(0), 2,
                   axes.data_ptr(), inv.data_ptr(), R, H, D)
    for f, g, w, o in zip(flat, got, want, off):
        # (two kernels with one formula each: their products and sums may be contracted differently, half a step of each term)
        assert ((g.view(H, R, D) - w).abs() <= 2.0 ** -22 * w.abs().amax().clamp(min=1.0)).all()
        assert not f[:o].any() and not f[o + R * H * D:].any()


@pytest.mark.parametrize("head_norms", [False, True])
@pytest.mark.parametrize("dim,heads", [(528, 2), (128, 2)])
def test_tower_on_the_gpu_against_the_cpu(dim, heads, head_norms):
    """GLM-4V's tower with and without norms of the heads, whose heads the kernel takes (64) and does not (264), bf16 against fp32."""
    from test_operators_edges_cpu import Glm4vVisionTower, _tower
    kw = dict(head_norms=head_norms, scale=dim ** -0.5)
    grids, rows = [(1, 4, 6), (1, 2, 2)], torch.randn(28, 24, generator=torch.Generator().manual_seed(1))
    want = _tower(Glm4vVisionTower, dim, heads, **kw).forward(rows, grids).double()
    got = _tower(Glm4vVisionTower, dim, heads, torch.bfloat16, DEV, **kw).forward(rows, grids)
    assert got.dtype == torch.bfloat16
    # weights and inputs rounded to bf16, then some 10 rounded steps in each of 3 blocks and 8 behind them: each moves the rows by up to
    # 2^-8 of their size, at random; twice the root of their number
    assert (got.double().cpu() - want).norm() < 2 * 48 ** 0.5 * 2.0 ** -8 * want.norm()


# ----------------------------------------------------------------------------- log probabilities
@pytest.mark.parametrize("K", [1024, 1032, 2048, 2056, 3080, 4096])
@pytest.mark.parametrize("R", [257, 1100])
def test_head_logprobs_wide_rows(R, K):
    """Sums leave the tensor core every 1024 of K: tiles of one and several such parts, the last one short or whole, a pair of SMs with
    several tiles, logits that are the products and logits that are not."""
    V = 20011
    x, w = _rn(R, K, seed=R), _rn(V, K, seed=V, scale=2.5 / K ** 0.5)
    ids = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV)
    ids[-1] = V - 1
    _check_head(x, w, ids)
    _check_head(x, w, ids, bias=_rn(V, seed=4, scale=0.5), scale=0.5, softcap=30.0)


@pytest.mark.parametrize("K", [2048, 4096])
def test_head_logprobs_long_sums_are_rounded_in_between(K):
    """A vocabulary of one token has the logit as its normaliser. Of positive products the tensor core's truncated sums come out low, each
    addition by the same part of a step of the partial sum on average: in proportion to the sum times its additions. Sums over 1024 of K
    that are added up rounded are therefore all low by one part of themselves, b, and so is their total (the few rounded additions,
    half a step each, are off either way); a sum over all of K is low by K / 1024 times b. The root of that ratio tells the two apart."""
    x, w = _rn(1100, K, seed=1).abs(), _rn(1, K, seed=2).abs()

    def off(n):
        got = logprobs.head_logprobs(x[:, :n], w[:, :n], torch.zeros(1100, dtype=torch.long, device=DEV)).lse.to(F64)
        want = (x[:, :n].to(F64) @ w[:, :n].to(F64).T)[:, 0]
        return (got - want) / want
    # 64 steps of a sum and the additions of sums, each off by at most a step of fp32
    assert off(K).abs().max() <= 2.0 ** -23 * (64 + 4 + K / 1024)
    assert off(K).mean().abs() <= math.sqrt(K / 1024) * off(1024).mean().abs()


@pytest.mark.parametrize("R", [1, 40, 300])
def test_head_logprobs_on_the_chip_and_through_memory(R, monkeypatch):
    V, K = 9001, 1032
    x, w = _rn(R, K, seed=R), _rn(V, K, seed=V, scale=2.5 / K ** 0.5)
    ids = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV)
    chip = _check_head(x, w, ids)
    monkeypatch.setattr(logprobs, "LARGE_WEIGHTS", 0)
    monkeypatch.setattr(logprobs, "FEW_ROWS", R)
    seen = []
    monkeypatch.setattr(logprobs, "linear", lambda *a, **k: (seen.append(a[0].shape[0]), linear(*a, **k))[1])
    memory = _check_head(x, w, ids)
    assert seen == [R] and all(a.shape == b.shape for a, b in zip(chip, memory))


# ----------------------------------------------------------------------------- models
def test_scores_on_the_chip_and_through_memory(monkeypatch):
    """A model's scores of a text by either route: logits are fp32 sums of 256 products in other orders."""
    from test_gpu_operators_models import _models

    from mlxcel_b200.engine.scoring import sequence_logprobs
    cfg, (_, gpu) = _models()
    ids = torch.randint(0, 1000, (700,), generator=torch.Generator().manual_seed(2)).tolist()
    chip = sequence_logprobs(gpu, cfg, ids)
    monkeypatch.setattr(logprobs, "LARGE_WEIGHTS", 0)
    monkeypatch.setattr(logprobs, "FEW_ROWS", 700)
    seen = []
    monkeypatch.setattr(logprobs, "linear", lambda *a, **k: (seen.append(a[0].shape[0]), linear(*a, **k))[1])
    memory = sequence_logprobs(gpu, cfg, ids)
    # hidden rows are normed (elements of about 1) and weights about 0.06: the magnitudes of a logit's products add up to about 10, each of
    # 256 additions is off by 2^-23 of that at most, and a log probability has that of two logits
    assert seen == [699] and (chip - memory).abs().max() <= 2 * 256 * 2.0 ** -23 * 16


def test_vision_backbone_in_bf16_against_the_cpu():
    from test_operators_edges_cpu import Dinov2Backbone
    hid, depth, heads = 128, 3, 4
    cfg = dict(hidden_size=hid, num_hidden_layers=depth, num_attention_heads=heads, patch_size=4, out_features=["stage1", "stage3"])
    g = torch.Generator().manual_seed(0)
    rn = lambda *s: (torch.randn(*s, generator=g) / math.sqrt(s[-1])).to(torch.bfloat16)    # noqa: E731
    t = {"embeddings.patch_embeddings.projection.weight": rn(hid, 48).view(hid, 3, 4, 4), "embeddings.patch_embeddings.projection.bias": rn(hid),
         "embeddings.cls_token": rn(1, 1, hid), "embeddings.position_embeddings": rn(1, 82, hid), "layernorm.weight": 1 + rn(hid), "layernorm.bias": rn(hid)}
    for i in range(depth):
        p = f"encoder.layer.{i}."
        for n, shape in (("attention.attention.query", (hid, hid)), ("attention.attention.key", (hid, hid)), ("attention.attention.value", (hid, hid)),
                         ("attention.output.dense", (hid, hid)), ("mlp.fc1", (2 * hid, hid)), ("mlp.fc2", (hid, 2 * hid))):
            t[p + n + ".weight"], t[p + n + ".bias"] = rn(*shape), rn(shape[0])
        for n in ("norm1", "norm2"):
            t[p + n + ".weight"], t[p + n + ".bias"] = 1 + rn(hid), rn(hid)
        t[p + "layer_scale1.lambda1"], t[p + "layer_scale2.lambda1"] = (0.5 + rn(hid).abs() for _ in range(2))
    x = torch.randn(2, 3, 36, 36, generator=g).to(torch.bfloat16)
    want = Dinov2Backbone(cfg, t, dtype=torch.float32).forward(x)
    got = Dinov2Backbone(cfg, t, dtype=torch.bfloat16, device=DEV).forward(x)
    assert len(got) == len(want) == 2
    for a, b in zip(got, want):
        # some 12 steps a block and 3 around them round the rows to bf16 (half a step, 2^-8, of their size), at random: twice the root
        assert a.dtype == torch.bfloat16 and a.shape == b.shape
        assert (a.double().cpu() - b.double()).norm() < 2 * math.sqrt(12 * depth + 3) * 2.0 ** -8 * b.double().norm()


def test_alternatives_change_no_draw():
    """Seeded requests of a mixed batch draw the same tokens, with the same log probabilities, whether or not they ask for alternatives."""
    from test_gpu_operators_models import _models

    from mlxcel_b200.engine import Engine, EngineConfig, SamplingParams
    cfg, (_, gpu) = _models()
    base = [dict(temperature=0.9, top_p=0.9, seed=3), dict(temperature=1.3, top_k=50, seed=4), dict(temperature=0.7, min_p=0.05, seed=5), dict(temperature=0.0)]

    def run(tops):
        eng = Engine(gpu, cfg, EngineConfig(max_batch=4, max_num_batched_tokens=64, num_blocks=32, max_model_len=128))
        sids = [eng.add_request([5, 6, 7, 8 + i], SamplingParams(max_tokens=8, ignore_eos=True, logprobs=True, top_logprobs=t, **b))
                for i, (b, t) in enumerate(zip(base, tops))]
        while eng.has_work():
            eng.step()
        return [eng.seqs[s] for s in sids]
    want = run([0] * 4)
    for tops in ([5] * 4, [0, 64, 0, 1]):
        for s, w, t in zip(run(tops), want, tops):
            assert s.output == w.output and [len(getattr(lp, "top", [])) for lp in s.logprobs] == [t] * 8
            # (the sampler's normaliser and the alternatives': fp32 sums of the same logits)
            assert all(abs(a - b) <= 1e-5 * (1 + abs(b)) for a, b in zip(s.logprobs, w.logprobs))

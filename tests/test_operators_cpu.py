"""Branch norms, rotary positions with several axes, moves of pages and log probabilities on the CPU: the plain statements against
their definitions in 64 bits, the copy tables, and what is refused."""
import random

import numpy as np
import pytest
import torch

from mlxcel_b200 import host_runtime
from mlxcel_b200.ops import KVLayer, logprobs, norms, pages, reference as ref, rotary

F64 = torch.float64


def _rn(*shape, seed=0, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


# ----------------------------------------------------------------------------- norms
@pytest.mark.parametrize("layer", [False, True])
def test_branch_norm_definition(layer):
    x, res, w, g, p, b = _rn(5, 37, seed=1), _rn(5, 37, seed=2, scale=4), *(_rn(37, seed=3 + i) for i in range(4))
    y, h = norms.branch_norm(x, res, post_w=w, gate=g, scale=0.5, pre_w=p, pre_b=b if layer else None, layer_norm=layer, eps=1e-5, w_bias=1.0)
    d = x.to(F64)
    d = d / torch.sqrt(d.pow(2).mean(1, True) + 1e-5) * (w.to(F64) + 1) * g.to(F64) * 0.5 + res.to(F64)
    assert torch.allclose(h.to(F64), d, rtol=1e-5, atol=1e-5)
    z = d - d.mean(1, True) if layer else d
    want = z / torch.sqrt(z.pow(2).mean(1, True) + 1e-5) * (p.to(F64) + 1) + (b.to(F64) if layer else 0)
    assert torch.allclose(y.to(F64), want, rtol=1e-4, atol=1e-4)
    assert norms.branch_norm(x)[0] is None and torch.equal(norms.branch_norm(x)[1], x)
    out = torch.empty_like(x)
    assert norms.branch_norm(x, res, out=out)[1] is out and torch.equal(out, x + res)


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(3)), dict(x=torch.zeros(3, 8, dtype=torch.float16)), dict(residual=torch.zeros(3, 7)), dict(residual=torch.zeros(3, 8, dtype=torch.bfloat16)),
    dict(post_w=torch.zeros(7)), dict(post_w=torch.zeros(8, dtype=torch.bfloat16)), dict(gate=torch.zeros(3, 8)), dict(pre_w=torch.zeros(16)[::2]),
    dict(pre_b=torch.zeros(8)), dict(pre_b=torch.zeros(8), pre_w=torch.zeros(8)), dict(out=torch.zeros(4, 8)), dict(x=torch.zeros(1, 32769))])
def test_branch_norm_refusals(bad):
    kw = dict(x=torch.zeros(3, 8)) | bad
    with pytest.raises(ValueError):
        norms.branch_norm(kw.pop("x"), kw.pop("residual", None), **kw)


# ----------------------------------------------------------------------------- rotary positions
def test_section_axes():
    assert rotary.section_axes([2, 3, 3], 8).tolist() == [0, 0, 1, 1, 1, 2, 2, 2]
    assert rotary.section_axes([1, 1, 1, 1, 2], 6).tolist() == [0, 1, 2, 0, 1, 1]
    assert rotary.section_axes([4, 2, 2], 8, interleaved=True).tolist() == [0, 1, 2, 0, 1, 2, 0, 0]
    with pytest.raises(ValueError):
        rotary.section_axes([2, 2], 8)


def _args(T=5, Hq=4, Hkv=2, D=64, rot=64, bits=16, dtype=torch.float32):
    kv = KVLayer(torch.zeros(4, Hkv, 8, D, dtype=dtype), torch.zeros(4, Hkv, 8, D, dtype=dtype), None, None, 8)
    if bits != 16:
        kv = KVLayer(*(torch.zeros(4, Hkv, 8, D * bits // 8, dtype=torch.uint8) for _ in range(2)),
                     *(torch.zeros(4, Hkv, 8, D // 64, 2, dtype=torch.bfloat16) for _ in range(2)), 8, bits)
    pos = torch.randint(0, 500, (3, T), generator=torch.Generator().manual_seed(1)).int()
    inv = (1.0 / 1e4 ** (torch.arange(rot // 2).double() * 2 / max(rot, 1))).float()
    return dict(qkv=_rn(T, (Hq + 2 * Hkv) * D, seed=2).to(dtype), positions=pos, slot_mapping=torch.tensor([9, -1, 31, 0, 32][:T], dtype=torch.int32),
                inv_freq=inv, axes=torch.arange(rot // 2).int() % 3, kv=kv, Hq=Hq, Hkv=Hkv, D=D, rot_dim=rot)


@pytest.mark.parametrize("pairs,rot", [(False, 64), (True, 64), (False, 32), (True, 16), (False, 0)])
def test_mrope_append_definition(pairs, rot):
    a = _args(rot=rot)
    w = _rn(64, seed=3)
    q = rotary.mrope_append(**a, traditional=pairs, q_norm_w=w, k_norm_w=w, norm_eps=1e-5, mscale=1.5)
    x = a["qkv"].to(F64).view(5, 8, 64).clone()
    x[:, :6] = x[:, :6] / torch.sqrt(x[:, :6].pow(2).mean(2, True) + 1e-5) * w.to(F64)            # the norm comes before the rotation
    for i in range(rot // 2):
        i1, i2 = (2 * i, 2 * i + 1) if pairs else (i, i + rot // 2)
        ang = (a["positions"][i % 3].to(F64) * a["inv_freq"][i].to(F64))[:, None]
        u, v = x[:, :6, i1].clone(), x[:, :6, i2].clone()
        x[:, :6, i1], x[:, :6, i2] = 1.5 * (u * ang.cos() - v * ang.sin()), 1.5 * (v * ang.cos() + u * ang.sin())
    assert torch.allclose(q.to(F64).view(5, 4, 64), x[:, :4], atol=1e-5)
    k, v = torch.zeros(4, 2, 8, 64, dtype=F64), torch.zeros(4, 2, 8, 64, dtype=F64)
    for t, s in enumerate([9, -1, 31, 0, 32]):                  # (-1 and 32 are outside the pool of 32 slots)
        if 0 <= s < 32:
            k[s // 8, :, s % 8], v[s // 8, :, s % 8] = x[t, 4:6], x[t, 6:]
    assert torch.allclose(a["kv"].k.to(F64), k, atol=1e-5) and torch.allclose(a["kv"].v.to(F64), v, atol=1e-5)


def test_mrope_append_agrees_with_the_sectioned_rotation_and_the_plain_append():
    """With chunks and interleaved sections it is `apply_mrope`; with equal axes it is `rope_append`."""
    for inter in (False, True):
        x, pos = _rn(6, 3, 32, seed=1), torch.randint(0, 90, (3, 6)).int()
        inv, ms = ref.rope_inv_freq(32, 1e4, None)
        want = ref.apply_mrope(x, pos, inv, [6, 5, 5], 1.0, interleaved=inter)
        got = ref.rotate_axes(x, pos, inv, ref.section_axes([6, 5, 5], 16, inter), 32)
        assert torch.allclose(got, want, atol=2e-5)
    for bits in (16, 8, 4):
        a, b = _args(bits=bits), _args(bits=bits)
        a["positions"] = a["positions"][:1].expand(3, -1).contiguous()
        a["slot_mapping"] = b["slot_mapping"] = torch.tensor([9, -1, 31, 0, 3], dtype=torch.int32)
        w = _rn(64, seed=4)
        q = rotary.mrope_append(**a, q_norm_w=w, k_norm_w=w)
        ref.rope_append(b["qkv"], a["positions"][0], b["slot_mapping"], b["inv_freq"], b["kv"], Hq=4, Hkv=2, D=64, rot_dim=64, traditional=False,
                        q_norm_w=w, k_norm_w=w)
        assert torch.allclose(q, b["qkv"][:, :256], atol=1e-4)
        if bits == 16:
            assert torch.allclose(a["kv"].k, b["kv"].k, atol=1e-4) and torch.equal(a["kv"].v, b["kv"].v)
        else:
            assert (a["kv"].k.int() - b["kv"].k.int()).abs().max() <= 17 and torch.equal(a["kv"].v, b["kv"].v)      # (a code or two apart at a border)


@pytest.mark.parametrize("bad", [
    dict(qkv=torch.zeros(5, 8 * 64 - 1)), dict(rot_dim=66), dict(rot_dim=31), dict(positions=torch.zeros(3, 4, dtype=torch.int32)),
    dict(positions=torch.zeros(3, 5, dtype=torch.int64)), dict(positions=torch.zeros(5, dtype=torch.int32)), dict(axes=torch.zeros(8, dtype=torch.int32)),
    dict(axes=torch.zeros(32, dtype=torch.int64)), dict(inv_freq=torch.zeros(32, dtype=torch.float64)), dict(inv_freq=torch.zeros(31)),
    dict(slot_mapping=torch.zeros(5, dtype=torch.int64)), dict(slot_mapping=torch.zeros(4, dtype=torch.int32)), dict(q_norm_w=torch.zeros(63)),
    dict(k_norm_w=torch.zeros(64, dtype=torch.bfloat16)), dict(out=torch.zeros(5, 255)), dict(Hkv=1, Hq=6),
    dict(kv=KVLayer(torch.zeros(4, 2, 8, 32), torch.zeros(4, 2, 8, 32), None, None, 8)),
    dict(kv=KVLayer(torch.zeros(4, 2, 8, 64, dtype=torch.uint8), torch.zeros(4, 2, 8, 64, dtype=torch.uint8), None, None, 8, 8))])
def test_mrope_append_refusals(bad):
    with pytest.raises(ValueError):
        rotary.mrope_append(**(_args() | bad))


def test_axial_rope_definition_and_refusals():
    x, pos = _rn(7, 3 * 2 * 8, seed=1), torch.randint(0, 30, (2, 7)).int()
    inv, axes = torch.tensor([1.0, 0.1, 1.0, 0.1]), torch.tensor([0, 0, 1, 1], dtype=torch.int32)
    q, k, v = rotary.axial_rope(x, pos, inv, axes, heads=2, D=8)
    z = x.view(7, 3, 2, 8).to(F64)
    ang = torch.stack([pos[a].to(F64) * float(f) for a, f in zip(axes.tolist(), inv)], 1)[:, None]
    for got, t in ((q, z[:, 0]), (k, z[:, 1])):
        a, b = t[..., :4], t[..., 4:]
        want = torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1)
        assert torch.allclose(got.to(F64), want.transpose(0, 1), atol=1e-5)
    assert torch.equal(v, z[:, 2].float().transpose(0, 1))
    for bad in (dict(D=7), dict(heads=3), dict(positions=pos[:, :6]), dict(inv_freq=inv[:3]), dict(axes=axes.long())):
        kw = dict(qkv=x, positions=pos, inv_freq=inv, axes=axes, heads=2, D=8) | bad
        with pytest.raises(ValueError):
            rotary.axial_rope(**kw)


# ----------------------------------------------------------------------------- pages
def _play(table, n, chains, pool):
    """The copy kernel's reading of a table, one unit of a page per entry."""
    t = table.tolist()
    starts = t[2 * n:]
    assert len(starts) == chains + 1 and starts[0] == 0 and starts[-1] == n
    spans = list(zip(starts, starts[1:]))
    wrote = [{t[2 * i + 1] for i in range(a, b)} for a, b in spans]
    for c, (a, b) in enumerate(spans):                      # chains may run in any order: none writes what another touches
        assert a < b and not any(wrote[c] & ({t[2 * i] for i in range(*s)} | wrote[d]) for d, s in enumerate(spans) if d != c)
        cycle = next((i for i in range(a, b) if b - a > 1 and t[2 * i + 1] == t[2 * (b - 1)]), b)
        for i in range(a, b):
            if i == cycle:
                held = pool[t[2 * i + 1]]
            pool[t[2 * i + 1]] = held if i == b - 1 and cycle < b else pool[t[2 * i]]
    return pool


def test_page_copies_give_what_a_copy_from_an_untouched_pool_would():
    r = random.Random(0)
    for _ in range(3000):
        P = r.randint(1, 14)
        dst = r.sample(range(P), r.randint(0, P))
        src = [r.randrange(P) for _ in dst]
        want = list(range(P))
        for s, d in zip(src, dst):
            want[d] = s
        assert _play(*host_runtime.page_copies(src, dst, P), list(range(P))) == want, (src, dst)
    n = 5000
    table, pairs, chains = host_runtime.page_copies(list(range(1, n)), list(range(n - 1)), n)
    assert (pairs, chains) == (n - 1, 1) and _play(table, pairs, chains, list(range(n))) == [*range(1, n), n - 1]
    assert host_runtime.page_copies([3, 3], [3, 3], 4)[1:] == (0, 0)


@pytest.mark.parametrize("src,dst", [([0], [4]), ([4], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2]), ([0, 1], [2, 2])])
def test_page_copy_refusals(src, dst):
    slabs = [torch.arange(8).view(4, 2), torch.arange(4).view(4, 1)]
    before = [t.clone() for t in slabs]
    with pytest.raises(ValueError):
        pages.PageSlabs(slabs).copy(src, dst)
    assert all(torch.equal(a, b) for a, b in zip(slabs, before))


def test_pages_on_the_cpu():
    slabs = [_rn(6, 2, 3, seed=1), _rn(6, 5, seed=2).to(torch.bfloat16), torch.zeros(6, 0)]
    p = pages.PageSlabs(slabs)
    assert p.bytes_per_page == 24 + 10 and len(p.slabs) == 2
    first = [t.clone() for t in slabs]
    data = p.gather(np.array([5, 0, 0]))
    assert data.dtype == torch.uint8 and data.numel() == 3 * 34 and torch.equal(data[:72].view(torch.float32).view(3, 2, 3), slabs[0][[5, 0, 0]])
    assert torch.equal(p.gather([5, 0, 0], out=torch.empty_like(data)), data) and torch.equal(p.gather([1], first=1), slabs[1][1].view(torch.uint8))
    p.scatter(torch.tensor([1, 2, 3]), data)
    for t, f in zip(slabs, first):
        f[[1, 2, 3]] = f[[5, 0, 0]]
        assert torch.equal(t, f)
    p.copy([0, 1], [1, 0])
    assert all(torch.equal(t[[1, 0]], f[[0, 1]]) for t, f in zip(slabs, first))
    for call in (lambda: p.gather([6]), lambda: p.gather([-1]), lambda: p.scatter([1, 1], data[:68]), lambda: p.scatter([1], data[:33]),
                 lambda: p.scatter([1], data[:34].to(torch.int8)), lambda: p.gather([1], out=torch.empty(35, dtype=torch.uint8)),
                 lambda: p.gather([1], first=3), lambda: p.gather([1], first=1, count=2), lambda: pages.PageSlabs([]),
                 lambda: pages.PageSlabs([torch.zeros(3, 2), torch.zeros(4, 2)]), lambda: pages.PageSlabs([torch.zeros(3, 4)[:, ::2]])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        p.copy([0.5], [1])


# ----------------------------------------------------------------------------- log probabilities
def test_token_logprobs_definition():
    x = _rn(6, 50, seed=1, scale=3)
    x[1, 5:] = float("-inf")
    x[2] = float("-inf")
    x[3, 7] = float("nan")
    x[4, 9] = float("inf")
    ids = torch.tensor([[0, 49], [3, 20], [1, 2], [7, 8], [9, 8], [-1, 50]])
    r = logprobs.token_logprobs(x, ids, top=4)
    z = torch.where(x.isnan(), torch.full_like(x, float("-inf")), x).to(F64)
    for i in (0, 1, 3, 5):
        p = torch.softmax(z[i], 0)
        assert torch.allclose(r.entropy[i].to(F64), -torch.special.xlogy(p, p).sum(), atol=1e-5)
        assert torch.allclose(r.lse[i].to(F64), torch.logsumexp(z[i], 0), atol=1e-5)
        order = torch.argsort(z[i], descending=True, stable=True)[:4]
        assert r.top_ids[i].tolist() == order.tolist() and torch.allclose(r.top_logprobs[i].to(F64), p[order].log(), atol=1e-5)
        for j in (0, 1):
            if 0 <= ids[i, j] < 50:
                assert torch.allclose(r.logprob[i, j].to(F64), p[ids[i, j]].log(), atol=1e-5)
    assert r.logprob[5].isnan().all() and r.logprob[3, 0] == float("-inf")
    assert r.lse[2] == float("-inf") and r.entropy[2] == 0 and (r.logprob[2] == float("-inf")).all() and r.top_ids[2].tolist() == [0, 1, 2, 3]
    assert r.logprob[4].tolist() == [0.0, float("-inf")] and r.entropy[4] == 0 and r.top_ids[4, 0] == 9
    b = _rn(50, seed=2)
    got = logprobs.token_logprobs(x[:1], ids[:1], bias=b, scale=0.5, softcap=2.0)
    want = torch.log_softmax(2.0 * torch.tanh((x[:1] + b) * 0.5 / 2.0), -1)
    assert torch.allclose(got.logprob, want[:, [0, 49]], atol=1e-5)
    assert logprobs.token_logprobs(x[:0], ids[:0], top=3).top_ids.shape == (0, 3)


def test_head_logprobs_definition():
    x, w, b = _rn(5, 16, seed=1), _rn(30, 16, seed=2), _rn(30, seed=3)
    ids = torch.tensor([0, 29, 4, 4, 7])
    r = logprobs.head_logprobs(x, w, ids, bias=b, scale=0.5, softcap=3.0)
    want = logprobs.token_logprobs(x @ w.t(), ids, bias=b, scale=0.5, softcap=3.0)
    assert all(torch.allclose(a, c, atol=1e-5) for a, c in zip(r[:3], want[:3])) and r.top_ids.shape == (5, 0)


@pytest.mark.parametrize("bad", [
    dict(logits=torch.zeros(3)), dict(logits=torch.zeros(3, 8, dtype=torch.float16)), dict(logits=torch.zeros(3, 0)), dict(ids=torch.zeros(2, dtype=torch.long)),
    dict(ids=torch.zeros(3)), dict(ids=torch.zeros(3, 1, 1, dtype=torch.long)), dict(top=9), dict(top=-1), dict(logits=torch.zeros(3, 100), top=65),
    dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8, dtype=torch.float64)), dict(scale=0.0), dict(scale=float("nan")), dict(softcap=-1.0)])
def test_token_logprobs_refusals(bad):
    with pytest.raises(ValueError):
        logprobs.token_logprobs(**(dict(logits=torch.zeros(3, 8), ids=torch.zeros(3, dtype=torch.long)) | bad))


@pytest.mark.parametrize("bad", [
    dict(x=torch.zeros(3, 5)), dict(w=torch.zeros(8, 4, dtype=torch.bfloat16)), dict(x=torch.zeros(4)), dict(w=torch.zeros(0, 4)),
    dict(x=torch.zeros(3, 4, dtype=torch.float16), w=torch.zeros(8, 4, dtype=torch.float16)), dict(ids=torch.zeros(3, 1, dtype=torch.long)),
    dict(ids=torch.zeros(4, dtype=torch.long)), dict(bias=torch.zeros(9)), dict(scale=-1.0)])
def test_head_logprobs_refusals(bad):
    with pytest.raises(ValueError):
        logprobs.head_logprobs(**(dict(x=torch.zeros(3, 4), w=torch.zeros(8, 4), ids=torch.zeros(3, dtype=torch.long)) | bad))

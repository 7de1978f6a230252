"""Kernels of the branch norms, the rotary positions with several axes, the moves of pages and the log probabilities against their
definitions in 64 bits.

Tolerances count roundings. U[t] is half a step of a type relative to the value (one rounding), and SUM bounds what fp32 sums and
functions add, relative to the magnitudes that went into them: a sum over n elements goes through at most n / 256 + 16 additions of
one partial sum and the functions (rsqrt, exp2, log, sine) are off by at most 4 ulp each."""
import itertools

import pytest
import torch

from mlxcel_b200.ops import KVLayer, _lib, logprobs, norms, pages, rotary

pytestmark = pytest.mark.gpu
DEV = "cuda"
F64 = torch.float64
U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
E32 = 2.0 ** -24
NEG, INF, NAN = float("-inf"), float("inf"), float("nan")


@pytest.fixture(autouse=True)
def _status_clean():
    yield
    torch.cuda.synchronize()
    assert _lib.read_status(torch.device(DEV)) == 0


def _rn(*shape, seed=0, scale=1.0, shift=0.0, dtype=torch.bfloat16):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(dtype)


def _within(got, want, tol, what=""):
    got = got.to(F64)
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        i = bad.flatten().nonzero()[0, 0]
        t = tol.expand_as(want).flatten()[i] if torch.is_tensor(tol) else tol
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first {got.flatten()[i]} for {want.flatten()[i]}, allowed {t}")


def _sums(n):
    return E32 * (n / 256 + 80)


# ----------------------------------------------------------------------------- norms around a sub-layer
def _check_norm(x, res, y, h, *, post_w=None, gate=None, scale=1.0, pre_w=None, pre_b=None, layer_norm=False, eps=1e-6, w_bias=0.0):
    dim, u = x.shape[1], U[x.dtype]
    b = x.to(F64)
    if post_w is not None:
        b = b / torch.sqrt(b.pow(2).mean(1, True) + eps) * (post_w.to(F64) + w_bias)
    if gate is not None:
        b = b * gate.to(F64)
    b = b * scale
    r = torch.zeros_like(b) if res is None else res.to(F64)
    slop = _sums(dim) * (b.abs() + r.abs())
    _within(h, r + b, u * ((r + b).abs() + slop) + slop, "h")
    if pre_w is None:
        assert y is None
        return
    z, w = h.to(F64), pre_w.to(F64) + w_bias                # y is the norm of the stored h
    mean = z.mean(1, True) if layer_norm else torch.zeros_like(z[:, :1])
    rstd = 1 / torch.sqrt((z - mean).pow(2).mean(1, True) + eps)
    want = (z - mean) * rstd * w + (0 if pre_b is None else pre_b.to(F64))
    # the fp32 mean is off by _sums(dim) of the mean magnitude, which moves every element and adds to the spread
    off = _sums(dim) * z.abs().mean(1, True) if layer_norm else 0.0
    slop = (w.abs() * rstd * (off * (1 + (z - mean).abs() * rstd) + _sums(dim) * ((z - mean).abs() + z.abs() * layer_norm))
            + E32 * want.abs() + (0 if pre_b is None else E32 * pre_b.to(F64).abs()))
    _within(y, want, u * (want.abs() + slop) + slop, "y")


DIMS = [1, 2, 7, 8, 33, 64, 1003, 2560, 4104, 5120, 8191, 8192, 20480, 32761, 32768]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("layer", [False, True])
def test_branch_norm(dim, dtype, layer):
    for rows in (1, 5):
        x, res = _rn(rows, dim, seed=1, scale=3, dtype=dtype), _rn(rows, dim, seed=2, scale=8, shift=2, dtype=dtype)
        w1, w2, g, b = (_rn(dim, seed=3 + i, scale=0.3, shift=0.5, dtype=dtype) for i in range(4))
        kw = dict(post_w=None if layer else w1, gate=g if layer else None, pre_w=w2, pre_b=b if layer else None, layer_norm=layer, scale=0.22,
                  eps=1e-6, w_bias=0.0 if layer else 1.0)
        y, h = norms.branch_norm(x, res, **kw)
        _check_norm(x, res, y, h, **kw)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim", [40, 1001, 4096])
def test_branch_norm_operands_left_out(dim, dtype):
    x, res = _rn(3, dim, seed=1, dtype=dtype), _rn(3, dim, seed=2, dtype=dtype)
    w, g = _rn(dim, seed=3, shift=1, dtype=dtype), _rn(dim, seed=4, dtype=dtype)
    for has_res, post, gate, pre, layer in itertools.product((False, True), repeat=5):
        kw = dict(post_w=w if post else None, gate=g if gate else None, pre_w=w if pre else None, layer_norm=layer)
        y, h = norms.branch_norm(x, res if has_res else None, **kw)
        _check_norm(x, res if has_res else None, y, h, **kw)


@pytest.mark.parametrize("dim", [96, 1000])
def test_branch_norm_strided_rows_in_place_and_neighbours(dim):
    """Rows inside wider matrices, at any offset; what lies between them stays as it was."""
    for offset in (0, 1, 8):
        wide = [_rn(4, dim + 24, seed=s) for s in (1, 2)]
        x, res = (t[:, offset:offset + dim] for t in wide)
        before = [t.clone() for t in wide]
        w = _rn(dim, seed=3, shift=1)
        want = norms.branch_norm(x.contiguous(), res.contiguous(), post_w=w, pre_w=w)
        y, h = norms.branch_norm(x, res, post_w=w, pre_w=w, out=res)
        assert h.data_ptr() == res.data_ptr() and torch.equal(h, want[1]) and torch.equal(y, want[0])
        assert torch.equal(wide[0], before[0])
        before[1][:, offset:offset + dim] = want[1]
        assert torch.equal(wide[1], before[1])


def test_branch_norm_rows_are_independent_and_bad_values_stay_in_theirs():
    x, res, w = _rn(300, 768, seed=1), _rn(300, 768, seed=2), _rn(768, seed=3, shift=1)
    y, h = norms.branch_norm(x, res, post_w=w, pre_w=w)
    x2, res2 = x.clone(), res.clone()
    x2[7, 5], res2[100, 0], x2[200] = NAN, INF, 0
    y2, h2 = norms.branch_norm(x2, res2, post_w=w, pre_w=w)
    keep = [i for i in range(300) if i not in (7, 100, 200)]
    assert torch.equal(y[keep], y2[keep]) and torch.equal(h[keep], h2[keep])
    assert y2[7].isnan().all() and torch.equal(h2[200], res[200])
    y0, h0 = norms.branch_norm(torch.zeros_like(x), None, post_w=w, pre_w=w)
    assert not y0.any() and not h0.any()
    big = torch.full((1, 4096), 3e4, device=DEV, dtype=torch.float32)            # squares near 1e9: no overflow of the sum
    y, _ = norms.branch_norm(big, None, pre_w=torch.ones(4096, device=DEV))
    _within(y, torch.ones(1, 4096, device=DEV, dtype=F64), _sums(4096) + 2 * E32)


def test_branch_norm_no_rows():
    y, h = norms.branch_norm(_rn(0, 64), _rn(0, 64), pre_w=_rn(64))
    assert y.shape == h.shape == (0, 64)


def test_branch_norm_many_rows():
    x, res, w = _rn(9001, 256, seed=1), _rn(9001, 256, seed=2), _rn(256, seed=3, shift=1)
    y, h = norms.branch_norm(x, res, post_w=w, pre_w=w)
    _check_norm(x, res, y, h, post_w=w, pre_w=w)


# ----------------------------------------------------------------------------- rotary positions with several axes
def _pool(pages_, hkv, bs, D, bits):
    if bits == 16:
        return KVLayer(_rn(pages_, hkv, bs, D, seed=90), _rn(pages_, hkv, bs, D, seed=91), None, None, bs)
    z = [torch.full((pages_, hkv, bs, D * bits // 8), 77, dtype=torch.uint8, device=DEV) for _ in range(2)]
    return KVLayer(*z, *(_rn(pages_, hkv, bs, D // 64, 2, seed=92 + i) for i in range(2)), bs, bits)


def _turned(x, pos, inv, axes, rot, pairs, mscale=1.0):
    """x [T, H, D] in 64 bits → (turned, |a| + |b| of each element's pair)."""
    x, half = x.clone(), rot // 2
    ang = torch.stack([pos[a].to(F64) * inv[i].to(F64) for i, a in enumerate(axes[:half].tolist())], 1)[:, None] if half else None
    mag = x.abs()
    if half:
        i1 = torch.arange(half, device=DEV) * (2 if pairs else 1)
        i2 = i1 + (1 if pairs else half)
        a, b = x[..., i1], x[..., i2]
        x[..., i1], x[..., i2] = (a * ang.cos() - b * ang.sin()) * mscale, (b * ang.cos() + a * ang.sin()) * mscale
        mag[..., i1] = mag[..., i2] = (a.abs() + b.abs()) * mscale
    return x, mag


def _check_mrope(T, hq, hkv, D, rot, pairs, bits, norm, *, bs=16, far=0, mscale=1.0, strided=False, inplace=False, dead=(), seed=0):
    width = (hq + 2 * hkv) * D
    base = _rn(T, width + (40 if strided else 0), seed=seed + 1)
    qkv = base[:, 16:16 + width] if strided else base
    x0 = qkv.to(F64).reshape(T, -1, D)
    g = torch.Generator().manual_seed(seed)
    pos = (far + torch.randint(0, 3000, (3, T), generator=g)).int().to(DEV)
    half = rot // 2
    axes = torch.randint(0, 3, (max(half, 1),), generator=g).int().to(DEV)
    inv = (1.0 / 1e5 ** (torch.arange(max(half, 1)).double() / max(half, 1))).float().to(DEV)
    n_pages = (T + bs - 1) // bs + 3
    slots = torch.randperm(n_pages * bs, generator=g)[:T].int()
    for i, s in dead:
        slots[i] = s
    kv = _pool(n_pages, hkv, bs, D, bits)
    old = [None if t is None else t.clone() for t in (kv.k, kv.v, kv.k_meta, kv.v_meta)]
    qw, kw = (_rn(D, seed=seed + 5, scale=0.4, shift=1), _rn(D, seed=seed + 6, scale=0.4, shift=1)) if norm else (None, None)
    before = base.clone()
    q = rotary.mrope_append(qkv, pos, slots.to(DEV), inv, axes, kv, Hq=hq, Hkv=hkv, D=D, rot_dim=rot, traditional=pairs, mscale=mscale,
                            q_norm_w=qw, k_norm_w=kw, out=qkv[:, :hq * D] if inplace else None)
    if inplace:
        at = 16 if strided else 0
        before[:, at:at + hq * D] = q
    assert torch.equal(base, before)
    xq, xk, xv = x0.split([hq, hkv, hkv], 1)
    if norm:
        xq, xk = (t / torch.sqrt(t.pow(2).mean(2, True) + 1e-6) * w.to(F64) for t, w in ((xq, qw), (xk, kw)))
    want, mag = _turned(xq, pos, inv, axes, rot, pairs, mscale)
    slop = E32 * 64 * mag
    _within(q.view(T, hq, D), want, 2.0 ** -8 * (want.abs() + slop) + slop, "q")
    kw_, kmag = _turned(xk, pos, inv, axes, rot, pairs, mscale)
    live = (slots >= 0) & (slots < n_pages * bs)
    at = slots[live].long()
    page, off, live = (at // bs).to(DEV), (at % bs).to(DEV), live.to(DEV)
    for name, pool, meta, was, was_m, new, nmag in (("k", kv.k, kv.k_meta, old[0], old[2], kw_[live], kmag[live]),
                                                    ("v", kv.v, kv.v_meta, old[1], old[3], xv[live], xv[live].abs())):
        slop = E32 * 64 * nmag
        got = pool[page, :, off]
        if bits == 16:
            _within(got, new, 2.0 ** -8 * (new.abs() + slop) + slop, name)
        else:
            if bits == 4:
                got = torch.stack([got & 15, got >> 4], -1).flatten(-2)
            m = meta[page, :, off].to(F64)
            z, s64 = new.unflatten(-1, (-1, 64)), slop.unflatten(-1, (-1, 64)).amax(-1, True)
            low, high, top = z.amin(-1, True), z.amax(-1, True), 2 ** bits - 1
            # the stored pair: one bf16 rounding of each
            _within(m[..., 1:2], low, 2.0 ** -8 * (low.abs() + s64) + s64, name + " offset")
            step = (high - low) / top
            _within(torch.where(step == 0, torch.zeros_like(step), m[..., 0:1]), step, 2.0 ** -8 * (step + 2 * s64) + 2 * s64 / top + E32 * step, name + " step")
            # the codes: the nearest to the value on the stored grid; either neighbour where fp32 cannot tell
            exact = ((z - m[..., 1:2]) / m[..., 0:1]).clamp(0, top)
            _within(got.unflatten(-1, (-1, 64)), exact, 0.5 + s64 / m[..., 0:1] + E32 * 4 * top, name + " codes")
            was_m = was_m.clone()
            was_m[page, :, off] = meta[page, :, off]
            assert torch.equal(meta, was_m)
        was = was.clone()
        was[page, :, off] = pool[page, :, off]
        assert torch.equal(pool, was), f"{name}: a slot that no row named has changed"


@pytest.mark.parametrize("bits", [16, 8, 4])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,rot,pairs", [(64, 64, False), (128, 128, False), (128, 64, True), (128, 64, False), (256, 256, False), (192, 64, True),
                                         (64, 32, True), (128, 0, False), (256, 64, False), (64, 2, True), (128, 120, False)])
def test_mrope_append(D, rot, pairs, bits, norm):
    _check_mrope(19, 6, 2, D, rot, pairs, bits, norm, dead=((3, -1), (18, -7)))


@pytest.mark.parametrize("D,rot,pairs", [(16, 16, False), (16, 8, True), (40, 40, False), (72, 72, False), (80, 80, False), (96, 96, False), (98, 34, True),
                                         (80, 40, True), (112, 48, False), (2, 2, False), (250, 250, True)])
def test_mrope_append_other_heads(D, rot, pairs):
    for norm in (False, True):
        _check_mrope(7, 3, 1, D, rot, pairs, 16, norm, bs=4)


@pytest.mark.parametrize("T,hq,hkv", [(1, 1, 1), (1, 64, 8), (5, 28, 4), (33, 32, 2), (600, 8, 8), (257, 16, 1), (3, 0, 2)])
@pytest.mark.parametrize("bits", [16, 8])
def test_mrope_append_shapes(T, hq, hkv, bits):
    _check_mrope(T, hq, hkv, 128, 128, False, bits, True, far=70000, seed=3)


@pytest.mark.parametrize("far", [0, 1 << 17, 1 << 24, (1 << 31) - 3001])
def test_mrope_append_far_positions(far):
    for pairs in (False, True):
        _check_mrope(9, 2, 1, 128, 128, pairs, 16, False, far=far, seed=4)


@pytest.mark.parametrize("strided,inplace", [(True, False), (False, True), (True, True)])
@pytest.mark.parametrize("D", [64, 72, 128])
def test_mrope_append_strides_and_in_place(D, strided, inplace):
    _check_mrope(21, 4, 2, D, D, False, 16, True, strided=strided, inplace=inplace, bs=8, mscale=1.25)


def test_mrope_append_slots_outside_the_pool():
    n = ((40 + 15) // 16 + 3) * 16
    _check_mrope(40, 4, 2, 128, 128, False, 16, False, dead=[(i, s) for i, s in zip(range(8), (-1, n, n + 5, -2 ** 31, 2 ** 31 - 1, -16, n + 16 * 1000, -1))])
    _check_mrope(3, 4, 2, 128, 128, False, 8, False, dead=[(0, -1), (1, -1), (2, -1)])


def test_mrope_append_no_rows():
    kv = _pool(2, 1, 16, 64, 16)
    z = torch.zeros(3, 0, dtype=torch.int32, device=DEV)
    q = rotary.mrope_append(_rn(0, 64 * 4), z, z[0], torch.ones(32, device=DEV), torch.zeros(32, dtype=torch.int32, device=DEV), kv, Hq=2, Hkv=1, D=64, rot_dim=64)
    assert q.shape == (0, 128)


@pytest.mark.parametrize("R,H,D", [(1, 1, 2), (4, 16, 80), (129, 12, 64), (257, 16, 72), (1000, 3, 128), (37, 5, 6), (12, 2, 256), (50, 16, 16)])
@pytest.mark.parametrize("strided", [False, True])
def test_axial_rope(R, H, D, strided):
    base = _rn(R, 3 * H * D + 24, seed=1)
    qkv = base[:, 8:8 + 3 * H * D] if strided else base[:, :3 * H * D].contiguous()
    pos = torch.randint(0, 200, (2, R), generator=torch.Generator().manual_seed(2)).int().to(DEV)
    inv = (1.0 / 1e4 ** (torch.arange(D // 2).double() / D)).float().to(DEV)
    axes = (torch.arange(D // 2) % 2).int().to(DEV)
    got = rotary.axial_rope(qkv, pos, inv, axes, heads=H, D=D)
    q, k, v = qkv.to(F64).reshape(R, 3, H, D).unbind(1)
    for t, w in zip(got[:2], (q, k)):
        want, mag = _turned(w, pos, inv, axes, D, False)
        assert t.dtype == torch.float32 and t.shape == (H, R, D) and t.is_contiguous()
        _within(t, want.transpose(0, 1), E32 * 12 * mag.transpose(0, 1))
    assert torch.equal(got[2].to(F64), v.transpose(0, 1))


# ----------------------------------------------------------------------------- pages
def _slabs(P, shapes, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return [torch.randint(0, 256, (P, *s), generator=g, device=DEV, dtype=torch.uint8) for s in shapes]


SHAPES = {"16": [(2, 16, 64), (2, 16, 64), (3 * 16,)], "4": [(20,), (4096 * 5 + 4,), (1024,)], "1": [(7,), (16384 + 3,), (1,), (0,)],
          "many": [(32 + 16 * (i % 3),) for i in range(300)], "large": [(1 << 16,), (1 << 17,)]}


@pytest.mark.parametrize("kind", list(SHAPES))
def test_pages_copy_gather_scatter(kind):
    P = 40
    slabs = _slabs(P, SHAPES[kind], 1)
    handle = pages.PageSlabs(slabs)
    want = [t.clone() for t in slabs]
    for src, dst in (([1, 5, 7], [2, 3, 39]),                   # apart
                     ([0, 0, 0, 4], [1, 2, 3, 5]),              # a fork
                     ([1, 2, 3, 4, 5], [0, 1, 2, 3, 4]),        # a chain towards the front
                     ([0, 1, 2, 3], [1, 2, 3, 4]),              # and away from it
                     ([3, 4], [4, 3]),                          # an exchange
                     ([0, 1, 2, 3, 0, 9, 12, 12], [1, 2, 3, 0, 9, 10, 12, 13]),     # a cycle with pages hanging off it, a page onto itself
                     ([6, 6, 6], [7, 7, 7]), ([], []), (list(range(40)), list(reversed(range(40))))):
        handle.copy(src, dst)
        for w in want:
            if w.numel() and src:
                w[torch.tensor(dst)] = w.clone()[torch.tensor(src)]
        assert all(torch.equal(a, b) for a, b in zip(slabs, want)), (src, dst)
    ids = [39, 0, 0, 17, 5]
    got = handle.gather(ids)
    assert torch.equal(got, torch.cat([t[torch.tensor(ids)].flatten() for t in want]))
    back = [1, 30, 2, 3, 39]
    handle.scatter(back, got)
    for w in want:
        if w.numel():
            w[torch.tensor(back)] = w.clone()[torch.tensor(ids)]
    assert all(torch.equal(a, b) for a, b in zip(slabs, want))


def test_pages_long_tables():
    """More pairs than travel in the parameters: random maps (forks, chains, cycles) of a pool onto itself, one long cycle."""
    P = 1500
    slabs = _slabs(P, [(48,), (16,)], 2)
    handle = pages.PageSlabs(slabs)
    g = torch.Generator().manual_seed(3)
    for src, dst in ((torch.randint(0, P, (P,), generator=g), torch.arange(P)), (torch.randperm(P, generator=g), torch.randperm(P, generator=g)),
                     (torch.arange(P), (torch.arange(P) + 1) % P), (torch.arange(1, P), torch.arange(P - 1))):
        want = [t.clone() for t in slabs]
        for w in want:
            w[dst] = w.clone()[src]
        handle.copy(src, dst)
        assert all(torch.equal(a, b) for a, b in zip(slabs, want))
    ids = torch.randint(0, P, (3 * P,), generator=g)
    assert torch.equal(handle.gather(ids), torch.cat([t[ids].flatten() for t in slabs]))
    ids = torch.randperm(P, generator=g)
    data = torch.randint(0, 256, (64 * P,), dtype=torch.uint8, device=DEV)
    handle.scatter(ids, data)
    assert torch.equal(handle.gather(ids), data)


def test_pages_part_of_the_slabs_and_offsets_past_32_bits():
    slabs = _slabs(9, [(32,), (7,), (64,)], 4)
    handle = pages.PageSlabs(slabs)
    got = handle.gather([8, 2], first=1, count=1)
    assert torch.equal(got, slabs[1][[8, 2]].flatten())
    handle.scatter([0, 1], got, first=1, count=1)
    assert torch.equal(slabs[1][:2].flatten(), got)
    wide = torch.zeros(5, 1 << 30, dtype=torch.uint8, device=DEV)               # the last page begins 4 GB into the slab
    wide[1, -5:] = torch.arange(1, 6, dtype=torch.uint8, device=DEV)
    h = pages.PageSlabs([wide])
    h.copy([1], [4])
    assert torch.equal(wide[4, -5:], wide[1, -5:]) and not wide[0].any() and not wide[2:4].any()


# ----------------------------------------------------------------------------- log probabilities
def _definition(z, ids, top):
    """In 64 bits, and the slack of an fp32 evaluation per row."""
    z = torch.where(z.isnan(), torch.full_like(z, NEG), z)
    m = z.amax(1, True)
    gap = torch.where(z == m, torch.zeros_like(z), z - m)
    e = torch.where(z == NEG, torch.zeros_like(z), gap.exp())
    s = e.sum(1)
    gone = s == 0
    log_s = s.log()
    logp = torch.where(z == NEG, z, gap - log_s[:, None])
    p = torch.where(gone[:, None], torch.zeros_like(e), e / s[:, None])
    spread = torch.where(p > 0, p * gap.abs(), torch.zeros_like(p)).sum(1)
    entropy = torch.where(gone, torch.zeros_like(s), log_s + spread)
    lse = torch.where(gone, m[:, 0], m[:, 0] + log_s)
    order = torch.argsort(z, dim=1, descending=True, stable=True)[:, :top]
    i2 = ids if ids.dim() == 2 else ids[:, None]
    lp = torch.where((i2 < 0) | (i2 >= z.shape[1]), torch.full_like(i2, NAN, dtype=F64), logp.gather(1, i2.clamp(0, z.shape[1] - 1)))
    big = torch.where(m[:, 0].isinf(), torch.zeros_like(s), m[:, 0].abs())
    second = torch.where(p > 0, p * gap.abs() ** 2, torch.zeros_like(p)).sum(1)
    slack = _sums(z.shape[1]) * (1 + spread) + E32 * 4 * (big + torch.where(gone, torch.zeros_like(s), log_s))
    slack_h = _sums(z.shape[1]) * (1 + 3 * spread + second) + E32 * 4 * torch.where(gone, torch.zeros_like(s), log_s)
    return lp.view(ids.shape), entropy, lse, order.int(), logp.gather(1, order), slack, slack_h


def _check_scores(logits, ids, top, **kw):
    r = logprobs.token_logprobs(logits, ids, top=top, **kw)
    z = logits.to(F64)
    bias, scale, cap = kw.get("bias"), kw.get("scale", 1.0), kw.get("softcap", 0.0)
    extra = 0.0
    if bias is not None or scale != 1.0 or cap:
        z = (z + (0 if bias is None else bias.to(F64))) * scale
        extra = E32 * 4 * torch.where(z.isinf() | z.isnan(), torch.zeros_like(z), z).abs().amax(1)
        if cap:
            z = cap * torch.tanh(z / cap)
            extra = extra + E32 * 8 * cap
    lp, en, lse, order, best, slack, slack_h = _definition(z, ids, top)
    slack, slack_h = slack + 2 * extra, slack_h + 2 * extra * (1 + en)
    col = lambda t, like: t if like.dim() == 1 else t[:, None]    # noqa: E731
    fin = lambda t: torch.where(t.isfinite(), t, torch.zeros_like(t)).abs()    # noqa: E731
    _within(r.logprob, lp, col(slack, lp) + 4 * E32 * fin(lp), "logprob")
    _within(r.entropy, en, slack_h + 4 * E32 * en, "entropy")
    _within(r.lse, lse, slack + 4 * E32 * fin(lse), "lse")
    if top:
        if bias is None and not cap and scale == 1.0:
            assert torch.equal(r.top_ids, order)
        else:                                   # (values of fp32 may tie or change places where those of 64 bits are as near)
            picked = torch.where(z.isnan(), torch.full_like(z, NEG), z).gather(1, r.top_ids.long())
            sorted_ = torch.where(z.isnan(), torch.full_like(z, NEG), z).gather(1, order.long())
            _within(picked, sorted_, extra[:, None] if torch.is_tensor(extra) else extra, "top values")
        _within(r.top_logprobs, best, slack[:, None] + 4 * E32 * fin(best), "top")
    return r


@pytest.mark.parametrize("V", [1, 2, 5, 31, 32, 33, 100, 1023, 1024, 4097, 8191, 32000, 50257, 151936, 262145])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs(V, dtype):
    for R, top in ((1, 20), (3, 64), (2, 1), (5, 0)):
        x = _rn(R, V, seed=V + R, scale=3, dtype=dtype)
        ids = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV)
        _check_scores(x, ids, min(top, V))


@pytest.mark.parametrize("R", [7, 37, 148, 300, 700])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_many_rows(R, dtype):
    x = _rn(R, 5003, seed=R, scale=2, dtype=dtype)
    for top in (0, 5, 50):
        _check_scores(x, torch.randint(0, 5003, (R, 3)).to(DEV), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [64, 4999, 70000])
def test_token_logprobs_masks_and_bad_values(V, dtype):
    x = _rn(14, V, seed=2, scale=3, dtype=dtype)
    x[0] = NEG                                   # nothing left
    x[1, torch.rand(V, device=DEV) < 0.95] = NEG
    x[2], x[2, V // 3] = NEG, 1.5                # one token left
    x[3] = torch.finfo(dtype).min                # every token at the type's lowest value: uniform
    x[4, :V // 2] = torch.finfo(dtype).min
    x[5, 7] = INF                                # takes all the mass
    x[6, 5], x[6, V - 1] = INF, INF              # two that share it
    x[7, V // 2] = NAN                           # counts as masked
    x[8] = NAN
    x[9] = 0.0                                   # all equal: ties by index
    x[10, ::2], x[10, 1::2] = 0.0, -0.0          # zeros of either sign are equal
    x[11] = torch.arange(V, device=DEV).to(dtype) / 100        # ever larger (in bf16 with many ties)
    x[12] = -torch.arange(V, device=DEV).to(dtype) / 100
    x[13, 0] = 200.0                             # all the mass on the first
    ids = torch.stack([torch.zeros(14, dtype=torch.long), torch.full((14,), V - 1), torch.full((14,), V // 3), torch.tensor([-1, V] * 7),
                       torch.full((14,), 7)], 1).to(DEV)
    for top in (0, 20, 64):
        r = _check_scores(x, ids, min(top, V))
    assert r.entropy[0] == 0 and r.lse[0] == NEG and (r.logprob[0, :3] == NEG).all() and r.top_ids[0].tolist() == list(range(64))
    assert r.logprob[:, 3].isnan().all() and r.logprob[2, 2] == 0 and r.entropy[2] == 0
    assert r.lse[5] == INF and r.logprob[5, 4] == 0 and r.logprob[5, 0] == NEG and r.top_ids[9].tolist() == list(range(64))


def test_token_logprobs_strided_rows_ids_and_transforms():
    wide = _rn(9, 1200, seed=3, scale=4, dtype=torch.float32)
    for lo in (0, 1, 2, 3):
        for V in (1000, 1001, 1003):
            x = wide[::2, lo:lo + V]
            _check_scores(x, torch.randint(0, V, (5, 2), dtype=torch.int32).to(DEV), 10)
            y = wide.to(torch.bfloat16)[::2, lo:lo + V]
            _check_scores(y, torch.randint(0, V, (5,), dtype=torch.int32).to(DEV), 3)
    x = wide[:, :1000]
    ids = torch.randint(0, 1000, (9,)).to(DEV)
    for bias in (None, _rn(1000, seed=4), _rn(1000, seed=4, dtype=torch.float32)):
        for scale, cap in ((1.0, 0.0), (0.125, 0.0), (1.0, 30.0), (2.0, 5.0)):
            _check_scores(x, ids, 7, bias=bias, scale=scale, softcap=cap)
    r = logprobs.token_logprobs(x, torch.empty(9, 0, dtype=torch.long, device=DEV))
    assert r.logprob.shape == (9, 0) and r.entropy.isfinite().all()
    r = logprobs.token_logprobs(x[:0], ids[:0], top=4)
    assert r.logprob.shape == (0,) and r.top_ids.shape == (0, 4)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_token_logprobs_many_of_the_largest_in_few_threads(dtype):
    """Large values only where the first 126 of a row's 256 threads look (vectors of 16 bytes, thread after thread): more of them than
    candidates are kept, with and without ties."""
    E, V, R = 16 // dtype.itemsize, 40000, 150
    j = torch.arange(V, device=DEV)
    for values in (torch.rand(R, V, device=DEV) * 50 + 100, torch.full((R, V), 100.0, device=DEV), (j % 97).float().expand(R, V) + 100):
        x = torch.where((j // E % 256 < 126)[None], values, _rn(R, V, seed=1, dtype=torch.float32)).to(dtype)
        for top in (5, 64):
            _check_scores(x, torch.randint(0, V, (R,)).to(DEV), top)
    one = x[:1].repeat(1, 4)[:, :151936].contiguous()                          # one row in parts
    _check_scores(one, torch.zeros(1, dtype=torch.long, device=DEV), 64)


def test_token_logprobs_repeat_bit_for_bit():
    x = _rn(3, 151936, seed=5, dtype=torch.bfloat16)
    ids = torch.zeros(3, dtype=torch.long, device=DEV)
    first = logprobs.token_logprobs(x, ids, top=40)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, logprobs.token_logprobs(x, ids, top=40)))


def _check_head(x, w, ids, bias=None, scale=1.0, softcap=0.0):
    r = logprobs.head_logprobs(x, w, ids, bias=bias, scale=scale, softcap=softcap)
    x64, w64 = x.to(F64), w.to(F64)
    z = x64 @ w64.T
    # an fp32 sum of K products, whatever the order and if every step truncates
    err = x.shape[1] * 2.0 ** -23 * (x64.abs() @ w64.abs().T)
    if bias is not None:
        z, err = z + bias.to(F64), err + E32 * (z.abs() + bias.to(F64).abs())
    z, err = z * scale, err * scale + E32 * (z * scale).abs()
    if softcap:
        z, err = softcap * torch.tanh(z / softcap), err + E32 * 8 * softcap
    lp, en, lse, _, _, slack, slack_h = _definition(z, ids, 0)
    p = torch.exp(z - lse[:, None])
    moved = (p * err).sum(1) + err.amax(1) * 1e-3                          # (first order, and the curvature)
    at = err.gather(1, ids.long().clamp(0, w.shape[0] - 1)[:, None])[:, 0]
    _within(r.logprob, lp, slack + moved + at + 4 * E32 * torch.where(lp.isfinite(), lp, torch.zeros_like(lp)).abs(), "logprob")
    _within(r.lse, lse, slack + moved + 4 * E32 * lse.abs(), "lse")
    mean = (p * z).sum(1, True)
    _within(r.entropy, en, slack_h + (p * (z - mean).abs() * err).sum(1) + err.amax(1) * (en + 1) * 1e-2 + 4 * E32 * en, "entropy")
    assert r.top_ids.shape == (x.shape[0], 0)
    return r


@pytest.mark.parametrize("R", [1, 2, 17, 128, 255, 256, 257, 300, 511, 513, 1100])
@pytest.mark.parametrize("V,K", [(1, 64), (7, 8), (255, 128), (256, 200), (1000, 512), (5003, 72), (20011, 256)])
def test_head_logprobs(R, V, K):
    x, w = _rn(R, K, seed=R), _rn(V, K, seed=V, scale=2.5 / K ** 0.5)
    ids = torch.randint(0, V, (R,), generator=torch.Generator().manual_seed(1)).to(DEV)
    ids[-1] = V - 1
    _check_head(x, w, ids)


@pytest.mark.parametrize("R", [40, 600])
def test_head_logprobs_transforms_and_layouts(R):
    V, K = 3001, 136
    x, w = _rn(R, K + 24, seed=1)[:, 8:8 + K], _rn(V, K + 8, seed=2, scale=0.2)[:, :K]
    ids = torch.randint(0, V, (R,), dtype=torch.int32).to(DEV)
    for bias in (None, _rn(V, seed=4), _rn(V, seed=4, dtype=torch.float32)):
        for scale, cap in ((1.0, 0.0), (0.125, 0.0), (1.0, 30.0), (3.0, 2.0)):
            _check_head(x, w, ids, bias, scale, cap)
    bad = ids.clone()
    bad[0], bad[1], bad[-1] = -1, V, 2 ** 31 - 1
    r = logprobs.head_logprobs(x, w, bad)
    good = logprobs.head_logprobs(x, w, ids)
    assert r.logprob[[0, 1, -1]].isnan().all() and torch.equal(r.logprob[2:-1], good.logprob[2:-1]) and torch.equal(r.lse, good.lse)
    odd = _rn(R, 131, seed=6), _rn(500, 131, seed=7, scale=0.2)                  # a width that TMA does not take
    _check_head(*odd, ids % 500)
    _check_head(*(t.float() for t in odd), ids % 500)
    shifted = _rn(R, K + 3, seed=8)[:, 1:1 + K]                                 # rows that do not start on 16 bytes
    _check_head(shifted, w, ids)
    r = logprobs.head_logprobs(x[:0], w, ids[:0])
    assert r.logprob.shape == r.entropy.shape == (0,)


def test_head_logprobs_in_parts_and_single_rows(monkeypatch):
    x, w = _rn(1500, 128, seed=1), _rn(900, 128, seed=2, scale=0.2)
    ids = torch.randint(0, 900, (1500,)).to(DEV)
    whole = logprobs.head_logprobs(x, w, ids)
    monkeypatch.setattr(logprobs, "PARTIAL_BYTES", 1)
    parts = logprobs.head_logprobs(x, w, ids)
    assert all(torch.equal(a, b) for a, b in zip(whole[:3], parts[:3]))
    one = x[3].as_strided((1, 128), (0, 1))                                      # (a row stride of 0)
    assert one.stride(0) == 0
    r = logprobs.head_logprobs(one, w, ids[3:4])
    assert all(torch.allclose(a[0], b[3], atol=1e-5) for a, b in zip(r[:3], whole[:3]))
    r = logprobs.head_logprobs(x, w[:1], ids * 0)                                # one token: certain
    assert not r.logprob.any() and not r.entropy.any()


@pytest.mark.parametrize("K", [128, 131])
def test_head_logprobs_single_row_of_any_stride_through_logits(K, monkeypatch):
    monkeypatch.setattr(logprobs, "LARGE_WEIGHTS", 0)
    x, w = _rn(2, K, seed=1), _rn(900, K, seed=2, scale=0.2)
    ids = torch.tensor([17], device=DEV)
    for stride in (0, 1, K - 3, K + 5):
        _check_head(x[0].as_strided((1, K), (stride, 1)), w, ids)


def test_head_logprobs_masked_by_bias_and_bad_rows():
    R, V, K = 400, 2000, 128
    x, w = _rn(R, K, seed=1), _rn(V, K, seed=2, scale=0.2)
    ids = torch.full((R,), 300, device=DEV)
    bias = torch.zeros(V, device=DEV)
    bias[torch.arange(V, device=DEV) != 300] = NEG
    r = logprobs.head_logprobs(x, w, ids, bias=bias)                             # one token left, in the second tile of columns
    assert not r.logprob.any() and not r.entropy.any()
    r = logprobs.head_logprobs(x, w, ids, bias=torch.full((V,), NEG, device=DEV))
    assert (r.logprob == NEG).all() and (r.lse == NEG).all() and not r.entropy.any()
    good = logprobs.head_logprobs(x, w, ids)
    x[7, 3] = NAN
    r = logprobs.head_logprobs(x, w, ids)                                        # NaN logits: nothing left in that row alone
    keep = torch.arange(R, device=DEV) != 7
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(r[:3], good[:3])) and r.logprob[7] == NEG and r.entropy[7] == 0


# ----------------------------------------------------------------------------- streams, graphs, devices
def _all_operators(seed):
    """One call of each on inputs of its own: (run, buffers to fill, outputs to read)."""
    x, res, w = _rn(65, 768, seed=seed), _rn(65, 768, seed=seed + 1), _rn(768, seed=seed + 2, shift=1)
    qkv, kv = _rn(65, 8 * 64, seed=seed + 3), _pool(8, 2, 16, 64, 16)
    kv.k.zero_(), kv.v.zero_()
    pos, slots = torch.arange(195, device=DEV, dtype=torch.int32).view(3, 65), torch.arange(65, device=DEV, dtype=torch.int32)
    inv, axes = torch.rand(32, device=DEV, generator=torch.Generator(device=DEV).manual_seed(seed)), torch.arange(32, device=DEV, dtype=torch.int32) % 3
    handle = pages.PageSlabs([kv.k, kv.v])
    head, ids = _rn(4000, 768, seed=seed + 4, scale=0.1), torch.arange(65, device=DEV)

    def run():
        y, h = norms.branch_norm(x, res, post_w=w, pre_w=w)
        q = rotary.mrope_append(qkv, pos, slots, inv, axes, kv, Hq=4, Hkv=2, D=64, rot_dim=64)
        handle.copy([0, 1, 2], [5, 6, 7])
        data = handle.gather([7, 0])
        big = logprobs.head_logprobs(y.repeat(5, 1), head, ids.repeat(5))
        few = logprobs.token_logprobs(h.float(), ids, top=5)
        return [y, h, q, kv.k, kv.v, data, *big[:3], *few, *rotary.axial_rope(qkv[:, :6 * 64], pos, inv, axes, heads=2, D=64)]
    return run, x, [kv.k, kv.v]


def test_side_streams_and_concurrent_calls():
    jobs = [_all_operators(s) for s in (10, 20)]
    want = [[t.clone() for t in run()] for run, _, _ in jobs]
    torch.cuda.synchronize()
    for _, _, pools in jobs:
        for t in pools:
            t.zero_()
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [None, None]
    for _ in range(3):
        for i, (run, _, _) in enumerate(jobs):
            with torch.cuda.stream(streams[i]):
                got[i] = run()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_captured_and_replayed_beside_another_graph():
    """Two graphs over the same operators, replayed in turn and with other inputs in the same buffers."""
    jobs = [_all_operators(s) for s in (30, 40)]
    for run, _, _ in jobs:
        run()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for run, _, _ in jobs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run())
        graphs.append(g)
    for seed in (50, 60):
        for run, x, _ in jobs:
            x.copy_(_rn(*x.shape, seed=seed))
        for _ in range(2):
            for g in graphs:
                g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for (run, _, _), o in zip(jobs, got):
            assert all(torch.equal(a, b) for a, b in zip(run(), o))

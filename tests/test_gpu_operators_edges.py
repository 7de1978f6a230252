"""Calls at the edge of what the kernels of the branch norms, the rotary positions with several axes, the moves of pages and the log
probabilities take, and the forms that their dispatch chooses for large calls."""
import pytest
import torch

from mlxcel_b200.ops import _lib, recurrent, rotary

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


# ----------------------------------------------------------------------------- rotary positions
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

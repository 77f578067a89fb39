"""Gated blocks in half precision whose intermediates are beyond the type's range (65504) or below what it holds with all its bits
(6e-5), while inputs and outputs are ordinary: every row against the formula in 64 bits.

A row's 2-norm error: the output's rounding (2^-11 at most, 2^-11 / sqrt 3 in the mean) and that of one operand on the way (the
same), 2.3e-4 of the row's norm together, as without the range's ends; the bound is twice that and a little, 5e-4."""
import math

import pytest
import torch

from test_gpu_ops import ACTS, BOUND, Layer, choices, ffn64, gen, guarded, mat, room, stream, untouched

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    from tierstream_amd import ops
    return ops


def near_rows(got, want, what="", sums=True):
    """sums: False where a row may be one product, so that an operand's rounding is the whole row's: 2^-11 for it and for the output."""
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), f"{what}: not finite"
    off, norm = (got.double() - want).norm(dim=-1), want.norm(dim=-1)
    if not sums:
        off = off / 2 - 2.0 ** -25 * math.sqrt(want.shape[-1])  # (and the type's own spacing)
    worst = int((off / norm.clamp_min(1e-30)).argmax())
    assert bool((off <= BOUND[got.dtype] * norm + 1e-30).all()), f"{what}: row {worst} off by {float(off.flatten()[worst] / norm.flatten()[worst]):.3g}"


def scaled(ops, g, n, d, f, kind, gate, up, down):
    """A stacked layer whose parts are multiplied by powers of two."""
    from test_gpu_ops import weight64
    layer = Layer(ops, g, "stacked", n, d, f, kind)
    for p, by in zip(layer.keep, (gate, up, down)):
        if kind == "q4":
            b = p.view(-1, 18)
            b[:, :2] = (b[:, :2].contiguous().view(torch.float16) * by).view(torch.uint8)
        else:
            p.mul_(by)
    layer.w64 = [weight64(p) for p in layer.keep]
    return layer


SIZES = [(1, 3, 2, 256, 512, 0), (1, 4, 3, 96, 160, 0), (1, 4, 4, 64, 9000, 0), (1, 3, 2, 70, 90, 1), (2, 3, 2, 256, 128, 0), (40, 3, 2, 128, 200, 0),
         (90, 3, 2, 131, 77, 1), (150, 2, 2, 192, 256, 1), (300, 2, 1, 160, 264, 0), (2501, 3, 2, 768, 776, 0)]


@pytest.mark.parametrize("rows,n,k,d,f,shift", SIZES)
@pytest.mark.parametrize("weights", ["f16", "q4"])
@pytest.mark.parametrize("large", [True, False])
def test_block(ops, rows, n, k, d, f, shift, weights, large):
    if weights == "q4":
        d, f = -(-d // 32) * 32, -(-f // 32) * 32
    g = gen(rows + d + large)
    # 4-bit values are up to 8 scales of 0.01: about 0.05, as 2 / sqrt(1600)
    wide = math.sqrt(1600 / d) if weights == "q4" else 1.0
    up, down = (2.0 ** 13, 2.0 ** -10) if large else (2.0 ** -11, 2.0 ** (12 if weights == "q4" else 9))
    layer = scaled(ops, g, n, d, f, weights, 2.0 ** 4 if large else 2.0 ** -8, 2.0 ** round(math.log2(up * wide)), down)
    x = mat(g, rows, d, "f16", pad=8 if shift == 0 else 3, shift=shift)
    ids, w = choices(g, rows, n, k, holes=False)
    w = w.abs() + 0.25
    want = ffn64(layer, x, ids, w, None, "silu")
    gate, u = (x[:1].double() @ p[ids[0, 0].long()].T for p in layer.w64[:2])
    h = (gate * torch.sigmoid(gate) * u).abs()
    assert float(h.max()) > 1e5 if large else float(h.median()) < 4e-6  # (what the test is about)
    assert float(want.abs().max()) < 6e4 and float(want.norm(dim=1).min()) > 64 * 6e-8 * math.sqrt(d) / BOUND[torch.float16] / 20
    t, y = guarded(rows, d, "f16")
    ops.ffn(layer.e, x, y, ids=ids, weights=w, act="silu", workspace=room(ops.ffn_workspace(layer.e, rows, k)), stream=stream())
    near_rows(y, want, f"{rows} rows")
    untouched(t, rows, d)


@pytest.mark.parametrize("kind", ["f16", "q4"])
def test_a_row_alone_and_among_others(ops, kind):
    """Rows of very different sizes, each by itself (one row's kernels) and all together; one holds an infinity, which stays in it."""
    g = gen(9)
    layer = scaled(ops, g, 3, 128, 256, kind, 4.0, 2.0 ** (14 if kind == "q4" else 12), 2.0 ** (-8 if kind == "q4" else -9))
    x = mat(g, 24, 128, "f16") * torch.tensor([2.0 ** -(i % 7) for i in range(24)], device="cuda").half()[:, None]
    ids, w = choices(g, 24, 3, 2, holes=False)
    w = w.abs() + 0.25
    want = ffn64(layer, x, ids, w, None, "silu")
    x[5, 3] = math.inf
    ws = room(ops.ffn_workspace(layer.e, 24, 2))
    y, alone = torch.empty_like(x), torch.empty_like(x)
    ops.ffn(layer.e, x, y, ids=ids, weights=w, workspace=ws, stream=stream())
    for i in range(24):
        ops.ffn(layer.e, x[i:i + 1], alone[i:i + 1], ids=ids[i:i + 1], weights=w[i:i + 1], workspace=ws, stream=stream())
    keep = torch.arange(24, device="cuda") != 5
    near_rows(y[keep], want[keep], "together")
    near_rows(alone[keep], want[keep], "alone")
    assert not bool(torch.isfinite(y[5]).any()) and not bool(torch.isfinite(alone[5]).any())


@pytest.mark.parametrize("act", ACTS)
def test_a_row_without_experts_beside_large_ones(ops, act):
    """Ids that add nothing leave no trace in the row's common power of two."""
    g = gen(10)
    layer = scaled(ops, g, 4, 64, 96, "f16", 8.0, 2.0 ** 13, 2.0 ** -10)
    x = mat(g, 1, 64, "f16")
    for ids in ([-1, -1, -1], [2, -1, 9], [-1, 0, 1], [4, 3, -7]):
        i = torch.tensor([ids], dtype=torch.int32, device="cuda")
        w = torch.tensor([[0.5, 1.0, 2.0]], device="cuda")
        y = torch.full_like(x, 7.0)
        ops.ffn(layer.e, x, y, ids=i, weights=w, act=act, workspace=room(ops.ffn_workspace(layer.e, 1, 3)), stream=stream())
        near_rows(y, ffn64(layer, x, i, w, None, act), str(ids))


@pytest.mark.parametrize("rows", [3, 200])
def test_a_column_beyond_32_bits_in_a_ragged_tile(ops, rows):
    """act(gate x) (up x) of the last column is infinite in 32 bits: so is the weight's gradient, of its own sign, and not NaN."""
    g = gen(12)
    d, f = 64, 40
    layer = Layer(ops, g, "stacked", 1, d, f, "bf16")
    x, dy = mat(g, rows, d, "bf16").abs() + 0.5, mat(g, rows, d, "bf16").abs() + 0.5
    for p in layer.keep[:2]:
        p[0, -1] = 1e20
    layer.keep[2][0, :, -1] = 0.5
    dw = torch.full((rows, 1), 7.0, device="cuda")
    ops.ffn_backward(layer.e, x, dy, None, dweights=dw, workspace=room(ops.ffn_backward_workspace(layer.e, rows)), stream=stream())
    assert bool((dw == math.inf).all())


# Powers of two of gate, up, down, x, dy and the range of the experts' weights; what is looked at besides the weights' gradient.
BACK = {
    "w h beyond 65504": (4, 13, -10, 0, -11, (0.25, 1.0), ("ddown",)),
    "dg beyond 65504": (-7, 10, 2, -8, 12, (0.25, 1.0), ("dgate", "dx")),
    "du beyond 65504": (7, -5, 3, -6, 10, (0.25, 1.0), ("dup",)),
    "all below 6e-5": (-10, -17, -12, 8, 8, (0.0025, 0.01), ("dgate", "dup", "ddown")),
    "dg below 6e-5": (10, -6, -2, -10, 0, (0.0125, 0.05), ("dx",)),
}


@pytest.mark.parametrize("what", BACK)
@pytest.mark.parametrize("rows,n,k,d,f,shift", [(1, 3, 2, 256, 128, 0), (37, 4, 2, 128, 200, 0), (90, 3, 2, 131, 77, 1), (300, 2, 1, 160, 264, 0),
                                                (3001, 2, 2, 256, 1672, 0)])
def test_block_backward(ops, rows, n, k, d, f, shift, what):
    gate, up, down, xs, dys, (low, high), looked = BACK[what]
    g = gen(rows + d)
    layer = scaled(ops, g, n, d, f, "f16", 2.0 ** gate, 2.0 ** up, 2.0 ** down)
    pad = 8 if shift == 0 else 3
    x, dy = (mat(g, rows, d, "f16", pad=pad, shift=shift, sigma=2.0 ** s) for s in (xs, dys))
    ids, w = choices(g, rows, n, k, holes=False)
    w = low + (high - low) * torch.rand(w.shape, device="cuda", generator=g)
    want_dx, want_dw, want = ffn64(layer, x, ids, w, None, "silu", dy)
    want = {"dx": want_dx, **dict(zip(("dgate", "dup", "ddown"), want))}
    got = {name: torch.full(t.shape, 7.0, dtype=torch.float16, device="cuda") for name, t in want.items()}
    dw = torch.full((rows, k), 7.0, device="cuda")
    ops.ffn_backward(layer.e, x, dy, got["dx"], ids=ids, weights=w, dweights=dw, dgate=got["dgate"], dup=got["dup"], ddown=got["ddown"],
                     workspace=room(ops.ffn_backward_workspace(layer.e, rows, k)), stream=stream())
    for name in looked:
        assert float(want[name].abs().max()) < 6e4 and float(want[name].abs().max()) > 1e-3, name
        near_rows(got[name], want[name], name, sums=name == "dx")
    assert float((dw.double() - want_dw).norm()) <= BOUND[torch.float32] * float(want_dw.norm())

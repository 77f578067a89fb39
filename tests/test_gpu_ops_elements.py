"""The model operators element by element, on the paths that sizes, alignment and types choose: every element of an output that was
full of NaN before, against the formula in 64 bits, so that one wrong or unwritten value in a ragged corner fails.

With e the largest rounding of a type (2^-8 bf16, 2^-11 half precision) and Q the root of the sum of squares of an element's terms:
rounding an operand once on the way adds 0.4 e Q in the mean, and e times the sum of the terms' sizes at most, which is below 6 e Q up
to 36 terms; beyond them 6 e Q is fifteen times the mean. The output's own rounding is e of the element. A sum in 32 bits loses
sqrt(n) 2^-24 Q, 4e-6 Q at the longest here, ten times that bounds it (the 4-bit form's offset cancels to a tenth); such a loss in a
factor that is near zero itself is not small beside its own Q, but beside the largest: 1e-6 of that."""
import math

import pytest
import torch

from test_gpu_ops import ACTS, KINDS, Layer, act64, choices, gen, linear64, mat, q4, room, stream, weight64

pytestmark = pytest.mark.gpu

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


@pytest.fixture(scope="module")
def ops(gpu):
    from tierstream_amd import ops
    return ops


def every(got, want, q, what="", operand=None):
    """q: each element's Q; operand: the type that operands were rounded to on the way, if they were."""
    assert got.shape == want.shape == q.shape, what
    bound = STEP[got.dtype] * want.abs() + (4e-5 + (6 * STEP[operand] if operand else 0)) * q + 1e-6 * q.max() + (2.0 ** -25 if got.dtype == torch.float16 else 1e-38)
    bad = ~((got.double() - want).abs() <= bound)
    if bool(bad.any()):
        at = tuple(int(i) for i in torch.nonzero(bad)[0])
        pytest.fail(f"{what}: {int(bad.sum())} of {bad.numel()} elements, first {at}: {float(got[at])} for {float(want[at])}, {float(bound[at]):.3g} allowed")


def block64(layer, x, ids, w, residual, act, dy=None):
    """The block in 64 bits, or its gradients: name -> (values, their Q)."""
    gate, up, down = layer.w64
    n, x, w = len(gate), x.double(), w.double()
    out = {"y": torch.zeros_like(x)} if dy is None else {"dx": torch.zeros_like(x), "dweights": torch.zeros_like(w), "dgate": torch.zeros_like(gate),
                                                         "dup": torch.zeros_like(up), "ddown": torch.zeros_like(down)}
    q = {name: torch.zeros_like(t) for name, t in out.items()}

    def put(name, at, left, right):
        if name in ("dgate", "dup", "ddown"):
            out[name][at], q[name][at] = left @ right, left.square() @ right.square()
        else:
            out[name].index_add_(0, at, left @ right)
            q[name].index_add_(0, at, left.square() @ right.square())

    for e in range(n):
        row, col = torch.nonzero(ids == e, as_tuple=True)
        if not len(row):
            continue
        a, slope = act64(act, x[row] @ gate[e].T)
        u, we = x[row] @ up[e].T, w[row, col][:, None]
        if dy is None:
            put("y", row, we * a * u, down[e].T)
            continue
        dye = dy[row].double()
        b = dye @ down[e]
        out["dweights"][row, col], q["dweights"][row, col] = (b * a * u).sum(1), (b * a * u).square().sum(1)
        dg, du = we * b * u * slope, we * b * a
        put("dx", row, dg, gate[e])
        put("dx", row, du, up[e])
        put("dgate", e, dg.T, x[row])
        put("dup", e, du.T, x[row])
        put("ddown", e, dye.T, we * a * u)
    if residual is not None:
        out["y"] += residual.double()
    return {name: (t, q[name].sqrt()) for name, t in out.items()}


class Output:
    """A matrix of NaN between values that must stay as they are."""

    def __init__(self, rows, cols, kind, pad=5):
        self.all = torch.full((rows + 2, cols + pad), 7.0, dtype=KINDS[kind], device="cuda")
        self.y = self.all[1:1 + rows, :cols]
        self.y.fill_(math.nan)

    def untouched(self):
        rows, cols = self.y.shape
        t = self.all
        assert bool((t[0] == 7).all()) and bool((t[1 + rows:] == 7).all()) and bool((t[:, cols:] == 7).all()), "written outside"


def moved(w, offset):
    """The same bytes, `offset` further on."""
    flat = torch.empty(w.numel() + 128, dtype=w.dtype, device="cuda")
    at = (-flat.data_ptr() // w.element_size()) % (64 // w.element_size()) + offset // w.element_size()
    out = flat[at:at + w.numel()].view(w.shape)
    out.copy_(w)
    assert out.data_ptr() % 16 == offset % 16
    return out


# ---- products ---------------------------------------------------------------------------------------------------------
def product_q(x, w):
    return (x.double().square() @ weight64(w).square().T).sqrt()


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 4096, 37), (1, 200, 33), (3, 264, 70), (16, 512, 96), (19, 2048, 520), (65, 96, 128), (129, 320, 385),
                                             (515, 1096, 777), (2050, 136, 3601), (1793, 72, 4096)])
@pytest.mark.parametrize("pad,shift", [(0, 0), (8, 0), (3, 1)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_linear(ops, rows, n_in, n_out, pad, shift, kind):
    g = gen(rows + n_out)
    x, w, bias = mat(g, rows, n_in, kind, pad, shift), mat(g, n_out, n_in, kind, pad, shift, sigma=0.1), mat(g, 1, n_out, kind)[0]
    for y_kind, act, b, r in ((kind, "none", None, False), ("f32", "gelu_tanh", bias, True), (kind, "silu", bias, True)):
        res = mat(g, rows, n_out, y_kind, pad=1) if r else None
        out = Output(rows, n_out, y_kind, pad=4 if shift == 0 else 3)
        ops.linear(x, w, out.y, bias=b, residual=res, act=act, workspace=room(ops.linear_workspace(x, w, out.y)), stream=stream())
        every(out.y, linear64(x, w, b, res, act), product_q(x, w), f"{y_kind} {act}")
        out.untouched()


@pytest.mark.parametrize("rows,n_in,n_out", [(1, 256, 16), (1, 1280, 37), (1, 96, 50), (20, 2048, 200), (40, 96, 33), (200, 32, 16), (449, 1056, 2501),
                                             (200, 160, 40000), (20, 64, 40001)])
@pytest.mark.parametrize("shift,offset", [(0, 0), (0, 4), (1, 0), (1, 8)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_linear_4_bits(ops, rows, n_in, n_out, shift, offset, kind):
    """x at any alignment, and packed where tiles take it; weights at any 4 bytes."""
    g = gen(rows + n_in)
    x, w = mat(g, rows, n_in, kind, pad=3 * shift, shift=shift), moved(q4(g, n_out, n_in), offset)
    out = Output(rows, n_out, "f32")
    ops.linear(x, w, out.y, workspace=room(ops.linear_workspace(x, w, out.y)), stream=stream())
    every(out.y, linear64(x, w, None, None, "none"), product_q(x, w))
    out.untouched()


@pytest.mark.parametrize("rows", [1, 20, 200])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("n_in", [256, 96])
def test_linear_4_bit_scales_at_their_limits(ops, rows, kind, n_in):
    """Rows of weights whose scales are half precision's largest, its smallest, negative, or zero."""
    g = gen(rows)
    n_out = 48
    w, x = q4(g, n_out, n_in), mat(g, rows, n_in, kind)
    scales = torch.tensor([65504.0, -65504.0, 2.0 ** -24, -3 * 2.0 ** -24, 2.0 ** -14, 0.0], device="cuda").half()
    w.view(n_out, -1, 18)[:, :, :2] = scales[torch.arange(n_out, device="cuda") % 6].view(torch.uint8).view(n_out, 1, 2)
    out = Output(rows, n_out, "f32")
    ops.linear(x, w, out.y, workspace=room(ops.linear_workspace(x, w, out.y)), stream=stream())
    every(out.y, linear64(x, w, None, None, "none"), product_q(x, w))


# ---- blocks -------------------------------------------------------------------------------------------------------------
def shifted(layer, where, offset):
    """The layer's weights `offset` bytes further on (stacked or in slots)."""
    if where == "stacked":
        layer.keep = [moved(p, offset) for p in layer.keep]
        for i, p in enumerate(layer.keep):
            layer.e.s.part[i] = p.data_ptr()
    else:
        parts = [moved(p, offset) for p in layer.keep[3]]
        layer.keep[3] = parts
        for i, p in enumerate(parts):
            layer.e.keep.parts[i].base = p.data_ptr()


BLOCKS = [(1, 5, 3, 256, 256), (1, 5, 3, 96, 160), (2, 3, 2, 96, 64), (20, 4, 2, 128, 96), (90, 16, 4, 64, 160), (200, 3, 2, 160, 96), (333, 2, 1, 96, 288),
          (1100, 3, 2, 256, 320)]


@pytest.mark.parametrize("rows,n,k,d,f", BLOCKS)
@pytest.mark.parametrize("kind,weights", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "q4"), ("f16", "q4")])
@pytest.mark.parametrize("shift,offset", [(0, 0), (1, 0), (0, 4), (1, 4)])
@pytest.mark.parametrize("where", ["stacked", "arena"])
def test_block(ops, rows, n, k, d, f, kind, weights, shift, offset, where):
    """x off its 16 bytes and weights off theirs, each and both, up to several hundred pairs an expert."""
    g = gen(rows + f + shift)
    layer = Layer(ops, g, where, n, d, f, weights)
    if offset:
        shifted(layer, where, offset)
    x, res = mat(g, rows, d, kind, pad=3 * shift, shift=shift), mat(g, rows, d, kind, pad=1)
    ids, w = choices(g, rows, n, k)
    act = ACTS[(rows + n) % 4]
    out = Output(rows, d, kind)
    ops.ffn(layer.e, x, out.y, ids=ids, weights=w, residual=res, act=act, workspace=room(ops.ffn_workspace(layer.e, rows, k)), stream=stream())
    every(out.y, *block64(layer, x, ids, w, res, act)["y"], act, operand=KINDS[kind])
    out.untouched()


@pytest.mark.parametrize("rows,n,k,d,f", [(2501, 3, 2, 768, 776), (700, 2, 1, 1032, 2088)])
@pytest.mark.parametrize("kind,weights", [("bf16", "bf16"), ("f16", "f16")])
def test_block_many_tiles(ops, rows, n, k, d, f, kind, weights):
    test_block(ops, rows, n, k, d, f, kind, weights, 0, 0, "arena")


@pytest.mark.parametrize("rows,n,k,d,f", [(1100, 1, 1, 1024, 1024), (701, 3, 2, 992, 1056)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_block_many_4_bit_tiles(ops, rows, n, k, d, f, kind):
    test_block(ops, rows, n, k, d, f, kind, "q4", 0, 0, "stacked")


def backward(ops, layer, kind, rows, n, k, d, f, g, act, pad=8, shift=0, unused=True):
    x, dy = (mat(g, rows, d, kind, pad=pad, shift=shift) for _ in range(2))
    ids, w = choices(g, rows, n, k)
    if unused and n > 1:
        ids[ids == n - 1] = -1  # an expert without rows
    out = Output(rows, d, kind)
    dw = torch.full((rows, k), math.nan, device="cuda")
    grads = [torch.full(s, math.nan, dtype=KINDS[kind], device="cuda") for s in ((n, f, d), (n, f, d), (n, d, f))]
    ops.ffn_backward(layer.e, x, dy, out.y, ids=ids, weights=w, dweights=dw, dgate=grads[0], dup=grads[1], ddown=grads[2], act=act,
                     workspace=room(ops.ffn_backward_workspace(layer.e, rows, k)), stream=stream())
    want = block64(layer, x, ids, w, None, act, dy)
    check_gradients(dict(dx=out.y, dweights=dw, **dict(zip(("dgate", "dup", "ddown"), grads))), want, ids, n, KINDS[kind])
    out.untouched()


def check_gradients(got, want, ids, n, operand):
    for name, t in got.items():
        every(t, *want[name], name, operand=None if name == "dweights" else operand)
        if name == "dweights":
            assert bool((t[(ids < 0) | (ids >= n)] == 0).all())
        elif name != "dx":
            for e in range(n):
                if not bool((ids == e).any()):
                    assert bool((t[e] == 0).all()), name


@pytest.mark.parametrize("rows,n,k,d,f", [(1, 3, 2, 67, 130), (37, 5, 3, 67, 130), (90, 3, 2, 131, 77), (300, 4, 2, 33, 70), (200, 3, 2, 64, 96)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("where", ["stacked", "arena", "table"])
def test_backward_at_any_alignment(ops, rows, n, k, d, f, kind, where):
    g = gen(rows + f)
    layer = Layer(ops, g, where, n, d, f, kind)
    backward(ops, layer, kind, rows, n, k, d, f, g, ACTS[(rows + k) % 4], pad=3, shift=1)


@pytest.mark.parametrize("rows,n,k,d,f", [(37, 8, 2, 320, 256), (64, 3, 2, 96, 160), (300, 2, 1, 160, 264), (3001, 2, 2, 512, 840)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_backward_through_a_table(ops, rows, n, k, d, f, kind):
    g = gen(rows)
    backward(ops, Layer(ops, g, "table", n, d, f, kind), kind, rows, n, k, d, f, g, "silu")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows", [2049, 5003])
def test_backward_small_experts_of_many_rows(ops, kind, rows):
    """Small tiles over sums of more pairs than one filling of a tile's map of rows holds."""
    g = gen(rows)
    backward(ops, Layer(ops, g, "stacked", 1, 128, 72, kind), kind, rows, 1, 1, 128, 72, g, "gelu", unused=False)


# ---- what is masked is not read ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("rows", [1, 4, 40, 300])
@pytest.mark.parametrize("kind,weights", [("bf16", "bf16"), ("f16", "f16"), ("f16", "q4")])
def test_nan_behind_a_mask(ops, rows, kind, weights):
    """Ids that add nothing have NaN for a weight, a row without experts has NaN for x (and dy), an expert that nobody asks for NaN in
    its weights: none of it shows."""
    g = gen(rows)
    n, k, d, f = 4, 3, 64, 96
    layer = Layer(ops, g, "stacked", n, d, f, weights)
    x, dy, res = mat(g, rows, d, kind).contiguous(), mat(g, rows, d, kind).contiguous(), mat(g, rows, d, kind)
    ids, w = choices(g, rows, n - 1, k, holes=False)
    ids[torch.rand(ids.shape, device="cuda", generator=g) < 0.3] = -1
    ids[rows // 2] = torch.tensor([-1, n, -5], dtype=torch.int32, device="cuda")
    empty = (ids < 0).logical_or(ids >= n)
    clean = w.masked_fill(empty, 0.0), x.clone(), dy.clone()
    want = block64(layer, clean[1], ids, clean[0], res, "silu")["y"]
    if weights != "q4":
        want_grads = block64(layer, clean[1], ids, clean[0], None, "silu", clean[2])
    w[empty] = math.nan
    x[empty.all(1)], dy[empty.all(1)] = math.nan, math.inf
    for p in layer.keep:
        if weights == "q4":
            p[n - 1].view(-1, 18)[:, :2] = torch.tensor([math.nan], device="cuda").half().view(torch.uint8)
        else:
            p[n - 1] = math.nan
    out = Output(rows, d, kind)
    ops.ffn(layer.e, x, out.y, ids=ids, weights=w, residual=res, workspace=room(ops.ffn_workspace(layer.e, rows, k)), stream=stream())
    every(out.y, *want, operand=KINDS[kind])
    assert torch.equal(out.y[empty.all(1)], res[empty.all(1)])
    if weights == "q4":
        return
    back, dw = Output(rows, d, kind), torch.full((rows, k), math.nan, device="cuda")
    grads = [torch.full(s, math.nan, dtype=KINDS[kind], device="cuda") for s in ((n, f, d), (n, f, d), (n, d, f))]
    ops.ffn_backward(layer.e, x, dy, back.y, ids=ids, weights=w, dweights=dw, dgate=grads[0], dup=grads[1], ddown=grads[2],
                     workspace=room(ops.ffn_backward_workspace(layer.e, rows, k)), stream=stream())
    check_gradients(dict(dx=back.y, dweights=dw, **dict(zip(("dgate", "dup", "ddown"), grads))), want_grads, ids, n, KINDS[kind])


@pytest.mark.parametrize("rows", [2, 40, 300])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_an_infinite_row_stays_alone(ops, rows, kind):
    """One row of x holds an infinity and one NaN: the other rows are what they are without them, to the bit."""
    g = gen(rows)
    layer = Layer(ops, g, "stacked", 2, 64, 96, kind)
    x = mat(g, rows, 64, kind).contiguous()
    ids, w = choices(g, rows, 2, 2, holes=False)
    y, y2 = torch.empty_like(x), torch.empty_like(x)
    ws = room(ops.ffn_workspace(layer.e, rows, 2))
    ops.ffn(layer.e, x, y, ids=ids, weights=w, workspace=ws, stream=stream())
    x[0, 7], x[rows - 1, 63] = math.inf, math.nan
    ops.ffn(layer.e, x, y2, ids=ids, weights=w, workspace=ws, stream=stream())
    assert torch.equal(y[1:rows - 1], y2[1:rows - 1])
    assert not bool(torch.isfinite(y2[0]).any()) and bool(torch.isnan(y2[rows - 1]).all())


@pytest.mark.parametrize("rows", [2, 20, 300])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_an_infinite_row_stays_alone_with_4_bit_weights(ops, rows, kind):
    g = gen(rows)
    x, w = mat(g, rows, 96, kind).contiguous(), q4(g, 48, 96)
    y, y2 = torch.empty((rows, 48), device="cuda"), torch.empty((rows, 48), device="cuda")
    layer = Layer(ops, g, "stacked", 2, 96, 64, "q4")
    ids, weights = choices(g, rows, 2, 2, holes=False)
    z, z2 = torch.empty_like(x), torch.empty_like(x)
    for out, block in ((y, z), (y2, z2)):
        ops.linear(x, w, out, workspace=room(ops.linear_workspace(x, w, out)), stream=stream())
        ops.ffn(layer.e, x, block, ids=ids, weights=weights, workspace=room(ops.ffn_workspace(layer.e, rows, 2)), stream=stream())
        x[0, 7], x[rows - 1, 95] = math.inf, math.nan
    assert torch.equal(y[1:rows - 1], y2[1:rows - 1]) and torch.equal(z[1:rows - 1], z2[1:rows - 1])
    assert not bool(torch.isfinite(y2[0]).any()) and bool(torch.isnan(y2[rows - 1]).all())
    assert not bool(torch.isfinite(z2[0]).any()) and bool(torch.isnan(z2[rows - 1]).all())

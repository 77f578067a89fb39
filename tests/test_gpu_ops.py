"""The model operators (include/tierstream_amd/tsa_ops.h) on an MI355X against plain implementations in 64 bits, at the sizes
and masks where they can go wrong: one row and many, odd widths, unaligned strides, rows without experts and experts
without rows, every type and activation, the three places weights are read from.

Tolerances, by the sums' lengths. Products of 16-bit values are exact in 32 bits; a sum of n of them in 32 bits is off by
at most about sqrt(n) 2^-24 of the terms' root-sum-square, 2e-6 at the longest used here (2-norms of the whole result).
An output rounded to bf16 (2^-9 at most, 2^-9 / sqrt(3) in the 2-norm) is off by 1.2e-3, to half precision by 1.5e-4; a
result behind one rounded intermediate carries sqrt(2) of that, and where a term's rounding and the output's combine with
both halves of dx, at most sqrt(3). The bounds are twice those: 4e-3 (bf16), 5e-4 (f16), 1e-5 (f32)."""
import ctypes as C
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BOUND = {torch.bfloat16: 4e-3, torch.float16: 5e-4, torch.float32: 1e-5}
ACTS = ["silu", "gelu", "gelu_tanh", "relu"]


@pytest.fixture(scope="module")
def ops(gpu):
    from tierstream_amd import ops
    return ops


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def near(got, want, what=""):
    assert got.shape == want.shape, what
    assert bool(torch.isfinite(got.double()).all()), f"{what}: not finite"
    norm = float(want.norm())
    off = float((got.double() - want).norm())
    assert off <= BOUND[got.dtype] * norm + 1e-30, f"{what}: off by {off / max(norm, 1e-30):.3g}"


def act64(name, v):
    """act(v) and its slope, 64 bits."""
    if name == "silu":
        s = torch.sigmoid(v)
        return v * s, s * (1 + v * (1 - s))
    if name == "gelu":
        p = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v ** 3))
        return 0.5 * v * (1 + t), 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    if name == "relu":
        return v.clamp_min(0), (v > 0).double()
    return v, torch.ones_like(v)


def mat(g, rows, cols, kind, pad=0, shift=0, sigma=1.0):
    """A matrix whose rows are cols + pad apart and start `shift` values into the buffer."""
    flat = torch.randn(rows * (cols + pad) + shift + 1, device="cuda", generator=g) * sigma
    return flat.to(KINDS[kind])[shift:].as_strided((rows, cols), (cols + pad, 1))


def q4(g, rows, cols):
    raw = torch.randint(0, 256, (rows * cols // 32, 18), dtype=torch.uint8, device="cuda", generator=g)
    raw[:, :2] = (torch.randn(len(raw), 1, device="cuda", generator=g) * 0.01).half().view(torch.uint8)
    return raw.view(rows, -1)


def weight64(w):
    if w.dtype != torch.uint8:
        return w.double()
    b = w.reshape(-1, 18)
    q = torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], 1).double() - 8
    return (q * b[:, :2].contiguous().view(torch.float16).double()).reshape(*w.shape[:-1], -1)


def stream():
    return torch.cuda.current_stream().cuda_stream


def room(n, fill=0xFF):
    return torch.full((max(n, 16),), fill, dtype=torch.uint8, device="cuda")


def guarded(rows, cols, kind, pad=5):
    """An output between values that must stay as they are."""
    t = torch.full((rows + 2, cols + pad), 7.0, dtype=KINDS[kind], device="cuda")
    return t, t[1:1 + rows, :cols]


def untouched(t, rows, cols):
    assert bool((t[0] == 7).all()) and bool((t[1 + rows:] == 7).all()) and bool((t[:, cols:] == 7).all()), "written outside"


# ---- route ----------------------------------------------------------------------------------------------------------
def route64(logits, k, renorm, scale):
    v = logits.double()
    v = torch.where(torch.isnan(v), -math.inf, v)
    order = torch.argsort(-v, dim=1, stable=True)[:, :k]
    top = torch.gather(v, 1, order)
    there = top > -math.inf
    best = v.max(1, keepdim=True).values
    e = torch.where(v == best, 1.0, torch.exp(v - best)).masked_fill(v == -math.inf, 0.0)
    chosen = torch.gather(e, 1, order)
    total = (chosen if renorm else e).sum(1, keepdim=True)
    w = torch.where(there, scale * chosen / total, 0.0)
    return torch.where(there, order, -1).int(), w


@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (1, 256, 8), (3, 7, 7), (5, 64, 64), (33, 65, 2), (130, 128, 8),
                                      (9, 512, 16), (4, 1000, 64), (2, 1024, 1)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route(ops, kind, rows, n, k, renorm):
    g = gen(rows * 1000 + n)
    logits = mat(g, rows, n, kind, pad=3, shift=1, sigma=2)
    logits[torch.rand(rows, n, device="cuda", generator=g) < 0.2] = -math.inf
    if rows > 2:
        logits[1] = -math.inf      # nothing to choose from
        logits[2] = 0.25           # all equal: the lowest ids
        logits[2, n // 2] = math.nan
    if rows > 3:
        logits[3, : n // 3 + 1] = torch.finfo(logits.dtype).min  # the lowest value is no mask
    if rows > 4:
        logits[4, n - 1] = math.inf
    ids = torch.full((rows, k), 77, dtype=torch.int32, device="cuda")
    w = torch.full((rows, k), 77.0, device="cuda")
    ops.route(logits, ids, w, renorm=renorm, scale=1.5, stream=stream())
    want_ids, want_w = route64(logits, k, renorm, 1.5)
    assert torch.equal(ids, want_ids)
    near(w, want_w, "weights")


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,n,k", [(1, 5, 2), (7, 128, 8), (65, 300, 16), (2, 1024, 64)])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_backward(ops, kind, rows, n, k, renorm):
    g = gen(n + k)
    logits = mat(g, rows, n, kind, pad=1)
    logits[torch.rand(rows, n, device="cuda", generator=g) < 0.3] = -math.inf
    if rows > 1:
        logits[1] = -math.inf
    ids, _ = route64(logits, k, renorm, 1.0)
    dw = torch.randn((rows, k), device="cuda", generator=g)
    t, out = guarded(rows, n, kind)
    ops.route_backward(logits, ids, dw, out, renorm=renorm, scale=0.5, stream=stream())
    # by differentiation: autograd through the formula in 64 bits
    v = logits.double().requires_grad_()
    pick = ids.long().clamp_min(0)
    e = torch.exp(v - v.detach().max(1, keepdim=True).values.clamp_min(-1e300))
    chosen = torch.gather(e, 1, pick) * (ids >= 0)
    total = (chosen if renorm else e).sum(1, keepdim=True)
    (0.5 * chosen / total.clamp_min(1e-300) * dw).sum().backward()
    near(out, torch.nan_to_num(v.grad), "dlogits")
    assert bool((out[logits == -math.inf] == 0).all())
    untouched(t, rows, n)


def test_route_backward_against_differences(ops):
    g = gen(5)
    logits = torch.randn((1, 12), device="cuda", generator=g)
    dw = torch.randn((1, 3), device="cuda", generator=g)
    for renorm in (True, False):
        ids, _ = route64(logits, 3, renorm, 1.0)
        out = torch.empty_like(logits)
        ops.route_backward(logits, ids, dw, out, renorm=renorm, stream=stream())

        def value(v):
            e = torch.exp(v)
            c = torch.gather(e, 1, ids.long())
            return (c / (c if renorm else e).sum(1, keepdim=True) * dw.double()).sum()

        for i in range(12):
            step = torch.zeros((1, 12), dtype=torch.float64, device="cuda")
            step[0, i] = 1e-5
            slope = float(value(logits.double() + step) - value(logits.double() - step)) / 2e-5
            assert abs(slope - float(out[0, i])) < 1e-6


# ---- linear ---------------------------------------------------------------------------------------------------------
def linear64(x, w, bias, residual, act):
    z = x.double() @ weight64(w).T
    y = act64(act, z if bias is None else z + bias.double())[0]
    return y if residual is None else y + residual.double()


LINEAR = [(1, 64, 16), (1, 4096, 4096), (1, 1280, 37), (1, 256, 16), (1, 2560, 200), (2, 200, 33), (7, 72, 257), (16, 512, 96), (17, 1000, 130), (33, 256, 64),
          (64, 2048, 520), (65, 96, 128), (129, 320, 384), (300, 640, 256), (515, 1096, 776), (200, 32, 16)]


@pytest.mark.parametrize("rows,n_in,n_out", LINEAR)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("weights", ["same", "q4"])
def test_linear(ops, rows, n_in, n_out, kind, weights):
    g = gen(rows + n_in)
    if weights == "q4":
        n_in = -(-n_in // 32) * 32
    x = mat(g, rows, n_in, kind, pad=8)
    w = q4(g, n_out, n_in) if weights == "q4" else mat(g, n_out, n_in, kind, sigma=0.05)
    for y_kind, act, with_bias, with_residual in ((kind, "none", False, True), ("f32", "gelu", True, False),
                                                  (kind, "silu", True, True), ("f32", "none", False, False)):
        bias = mat(g, 1, n_out, kind)[0] if with_bias else None
        res = mat(g, rows, n_out, y_kind, pad=2) if with_residual else None
        t, y = guarded(rows, n_out, y_kind)
        ws = room(ops.linear_workspace(x, w, y))
        ops.linear(x, w, y, bias=bias, residual=res, act=act, workspace=ws, stream=stream())
        near(y, linear64(x, w, bias, res, act), f"{y_kind} {act}")
        untouched(t, rows, n_out)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("rows,n_in,n_out,weights", [(2050, 136, 3601, "same"), (1793, 72, 4096, "same"), (290, 96, 4096, "q4"),
                                                     (449, 1056, 2501, "q4")])
def test_linear_many_tiles(ops, rows, n_in, n_out, weights, kind):
    """Enough tiles for the largest ones: ragged in both directions, short and long sums."""
    test_linear(ops, rows, n_in, n_out, kind, weights)


@pytest.mark.parametrize("n_in", [32767, 32768, 32769, 40000])
def test_linear_long_rows(ops, n_in):
    """One row of x up to what is staged of it, and beyond."""
    test_linear(ops, 1, n_in, 37, "bf16", "same")


@pytest.mark.parametrize("pad,shift", [(0, 0), (1, 0), (3, 1), (8, 4), (0, 1)])
@pytest.mark.parametrize("rows,n_in,n_out", [(1, 1, 1), (1, 129, 40), (5, 63, 17), (33, 515, 70), (64, 255, 33), (70, 1001, 65), (140, 264, 300)])
def test_linear_any_alignment(ops, pad, shift, rows, n_in, n_out):
    g = gen(pad * 10 + shift)
    x, w = mat(g, rows, n_in, "bf16", pad, shift), mat(g, n_out, n_in, "bf16", pad, shift, sigma=0.1)
    t, y = guarded(rows, n_out, "bf16", pad=1 + pad)
    ops.linear(x, w, y, workspace=room(ops.linear_workspace(x, w, y)), stream=stream())
    near(y, linear64(x, w, None, None, "none"))
    untouched(t, rows, n_out)


def test_linear_residual_in_place_and_activations(ops):
    g = gen(3)
    for rows in (3, 200):
        for act in ["none"] + ACTS:
            x, w = mat(g, rows, 160, "f16"), mat(g, 96, 160, "f16", sigma=0.1)
            y = mat(g, rows, 96, "f32")
            want = linear64(x, w, None, y.clone(), act)
            ops.linear(x, w, y, residual=y, act=act, workspace=room(ops.linear_workspace(x, w, y)), stream=stream())
            near(y, want, act)


def test_linear_special_values(ops):
    """Infinities and NaN stay in their rows; what lies behind a row's end is not read into the sums."""
    g = gen(4)
    for rows in (2, 80):
        buf = torch.full((rows, 104), math.nan, device="cuda", dtype=torch.bfloat16)
        buf[:, :96] = mat(g, rows, 96, "bf16")
        x, w = buf[:, :96], mat(g, 48, 96, "bf16")
        x[1, 5] = math.inf
        y = torch.empty((rows, 48), dtype=torch.float32, device="cuda")
        ops.linear(x, w, y, act="relu", workspace=room(ops.linear_workspace(x, w, y)), stream=stream())
        assert bool(torch.isfinite(y[0]).all()) and bool(((y[1] == math.inf) | (y[1] == 0)).all())
        keep = torch.arange(rows, device="cuda") != 1
        near(y[keep], linear64(x, w, None, None, "relu")[keep])


# ---- ffn --------------------------------------------------------------------------------------------------------------
class Layer:
    """An expert layer's weights in one of the three places."""

    def __init__(self, ops, g, where, n, d, f, kind):
        from tierstream_amd import ss
        make = (lambda r, c: q4(g, r, c)) if kind == "q4" else (lambda r, c: mat(g, r, c, kind, sigma=2 / math.sqrt(c)).contiguous())
        slots = n + 2
        parts = [make(slots * r, c).view(slots, r, -1) for r, c in ((f, d), (f, d), (d, f))]
        order = torch.randperm(slots, device="cuda", generator=g)[:n]
        self.w64 = [weight64(p[order]) for p in parts]
        if where == "stacked":
            self.keep = [p[order].contiguous() for p in parts]
            self.e = ops.Experts.stacked(*self.keep)
        elif where == "table":
            units = torch.cat([p.reshape(slots, -1) for p in parts], 1)
            table = units.data_ptr() + order * units.shape[1] * units.element_size()
            self.keep = [units, table]
            self.e = ops.Experts.in_table(table, d, f, kind)
        else:
            words = torch.zeros(2, dtype=torch.int32, device="cuda")
            slot_of = torch.cat([torch.full((5,), -1, device="cuda"), order]).to(torch.int32)  # gated layer 1 of two
            base = torch.tensor([0, 5, 5 + n], dtype=torch.int32, device="cuda")
            v = ss.SsDgDeviceView(struct_size=C.sizeof(ss.SsDgDeviceView), n_gated=2, n_parts=3, guard_slot=slots - 1, slots=slots,
                                  slot_of=slot_of.data_ptr(), unit_base=base.data_ptr(), abort=words.data_ptr(),
                                  absent_err=words.data_ptr() + 4)
            for i, p in enumerate(parts):
                size = p[0].numel() * p.element_size()
                v.parts[i].base, v.parts[i].stride, v.parts[i].bytes = p.data_ptr(), size, size
            self.keep = [words, slot_of, base, parts]
            self.e = ops.Experts.in_arena(v, 1, n, d, f, kind)


def choices(g, rows, n, k, holes=True):
    ids = torch.rand((rows, n), device="cuda", generator=g).topk(k, 1).indices.int()
    if holes and rows > 1:
        ids[torch.rand((rows, k), device="cuda", generator=g) < 0.2] = -1
        ids[rows // 2] = -1   # a row without experts
        ids[0, 0] = n         # out of range: nothing, as below 0
        ids[rows - 1] = 0     # one expert k times
    return ids.contiguous(), torch.randn((rows, k), device="cuda", generator=g)


def ffn64(layer, x, ids, weights, residual, act, dy=None):
    gate, up, down = layer.w64
    n, x, w = len(gate), x.double(), weights.double()
    y = torch.zeros_like(x) if residual is None else residual.double().clone()
    if dy is not None:
        dy, dx, dw = dy.double(), torch.zeros_like(x), torch.zeros_like(w)
        grads = [torch.zeros_like(t) for t in layer.w64]
    for e in range(n):
        row, col = torch.nonzero(ids == e, as_tuple=True)
        if not len(row):
            continue
        a, s = act64(act, x[row] @ gate[e].T)
        u, we = x[row] @ up[e].T, w[row, col][:, None]
        if dy is None:
            y.index_add_(0, row, we * ((a * u) @ down[e].T))
            continue
        b = dy[row] @ down[e]
        dw[row, col] = (b * a * u).sum(1)
        dg, du = we * b * u * s, we * b * a
        dx.index_add_(0, row, dg @ gate[e] + du @ up[e])
        grads[0][e], grads[1][e], grads[2][e] = dg.T @ x[row], du.T @ x[row], dy[row].T @ (we * a * u)
    return y if dy is None else (dx, dw, grads)


FFN = [(1, 1, 1, 64, 64), (1, 6, 3, 1280, 768), (1, 9, 8, 768, 2304), (1, 3, 2, 256, 1024),(1, 8, 2, 256, 512), (1, 4, 3, 96, 160), (2, 8, 2, 512, 128), (5, 16, 4, 128, 96), (32, 40, 8, 256, 192),
       (37, 8, 2, 320, 256), (64, 2, 2, 128, 416), (200, 3, 2, 160, 288), (300, 5, 3, 512, 256), (700, 2, 1, 256, 320)]


@pytest.mark.parametrize("rows,n,k,d,f", FFN)
@pytest.mark.parametrize("kind,weights", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "q4"), ("f16", "q4")])
@pytest.mark.parametrize("where", ["stacked", "table", "arena"])
def test_ffn(ops, rows, n, k, d, f, kind, weights, where):
    g = gen(rows + d)
    layer = Layer(ops, g, where, n, d, f, weights)
    x, res = mat(g, rows, d, kind, pad=8), mat(g, rows, d, kind, pad=1)
    ids, w = choices(g, rows, n, k)
    t, y = guarded(rows, d, kind)
    act = ACTS[(rows + n) % 4]
    ops.ffn(layer.e, x, y, ids=ids, weights=w, residual=res, act=act, workspace=room(ops.ffn_workspace(layer.e, rows, k)),
            stream=stream())
    near(y, ffn64(layer, x, ids, w, res, act), act)
    untouched(t, rows, d)
    y2 = torch.empty((rows, d), dtype=y.dtype, device="cuda")  # the same bits again, in another workspace
    ops.ffn(layer.e, x, y2, ids=ids, weights=w, residual=res, act=act, workspace=room(ops.ffn_workspace(layer.e, rows, k), 0),
            stream=stream())
    assert torch.equal(y, y2)


@pytest.mark.parametrize("rows,d,f", [(1, 33, 47), (1, 1001, 65), (9, 67, 70), (130, 99, 131), (3, 8, 1)])
def test_ffn_odd_sizes(ops, rows, d, f):
    g = gen(d)
    layer = Layer(ops, g, "stacked", 3, d, f, "bf16")
    x = mat(g, rows, d, "bf16", pad=1, shift=1)
    ids, w = choices(g, rows, 3, 2)
    t, y = guarded(rows, d, "bf16")
    ops.ffn(layer.e, x, y, ids=ids, weights=w, workspace=room(ops.ffn_workspace(layer.e, rows, 2)), stream=stream())
    near(y, ffn64(layer, x, ids, w, None, "silu"))
    untouched(t, rows, d)


@pytest.mark.parametrize("rows", [1, 3, 90, 400])
def test_ffn_without_ids(ops, rows):
    """A dense block: every row through expert 0 with weight 1, the residual in place."""
    g = gen(rows)
    layer = Layer(ops, g, "stacked", 1, 192, 320, "bf16")
    x, y = mat(g, rows, 192, "bf16"), mat(g, rows, 192, "bf16").contiguous()
    ids, ones = torch.zeros((rows, 1), dtype=torch.int32, device="cuda"), torch.ones((rows, 1), device="cuda")
    want = ffn64(layer, x, ids, ones, y.clone(), "silu")
    ops.ffn(layer.e, x, y, residual=y, workspace=room(ops.ffn_workspace(layer.e, rows)), stream=stream())
    near(y, want)


@pytest.mark.parametrize("rows,n,k,d,f,weights", [(2501, 3, 2, 768, 776, "same"), (1100, 1, 1, 1024, 1024, "q4"), (701, 3, 2, 992, 1056, "q4")])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("where", ["stacked", "arena"])
def test_ffn_many_tiles(ops, rows, n, k, d, f, kind, weights, where):
    """Enough tiles for the largest ones."""
    test_ffn(ops, rows, n, k, d, f, kind, kind if weights == "same" else weights, where)


@pytest.mark.parametrize("n,k,d,f", [(4, 3, 72, 10880), (4, 3, 64, 10923), (4, 4, 128, 8192), (2, 1, 33000, 48)])
def test_ffn_one_long_row(ops, n, k, d, f):
    """One row whose x, or whose h of all experts, is as long as what is staged of it, or longer."""
    test_ffn(ops, 1, n, k, d, f, "bf16", "bf16", "stacked")


@pytest.mark.parametrize("rows,n,k,where", [(1025, 3, 2, "stacked"), (5003, 400, 7, "table"), (70001, 5, 2, "arena")])
def test_ffn_many_pairs(ops, rows, n, k, where):
    """Pairs for more than one workgroup to group: a few over one's share, a ragged last one, more than 64 shares."""
    g = gen(n)
    layer = Layer(ops, g, where, n, 64, 72, "bf16")
    x = mat(g, rows, 64, "bf16")
    ids, w = choices(g, rows, n, k)
    t, y = guarded(rows, 64, "bf16")
    ops.ffn(layer.e, x, y, ids=ids, weights=w, workspace=room(ops.ffn_workspace(layer.e, rows, k)), stream=stream())
    near(y, ffn64(layer, x, ids, w, None, "silu"))
    untouched(t, rows, 64)


def test_ffn_absent_table_entries_and_empty_calls(ops):
    g = gen(1)
    layer = Layer(ops, g, "table", 4, 128, 96, "bf16")
    layer.keep[1][2] = 0  # not acquired
    for rows in (1, 40):
        x = mat(g, rows, 128, "bf16")
        ids, w = choices(g, rows, 4, 3, holes=False)
        y = torch.empty((rows, 128), dtype=torch.bfloat16, device="cuda")
        ops.ffn(layer.e, x, y, ids=ids, weights=w, workspace=room(ops.ffn_workspace(layer.e, rows, 3)), stream=stream())
        near(y, ffn64(layer, x, ids.masked_fill(ids == 2, -1), w, None, "silu"))
    nothing = torch.full((5, 2), -1, dtype=torch.int32, device="cuda")
    x, y = mat(g, 5, 128, "bf16"), torch.ones((5, 128), dtype=torch.bfloat16, device="cuda")
    ops.ffn(layer.e, x, y, ids=nothing, workspace=room(ops.ffn_workspace(layer.e, 5, 2)), stream=stream())
    assert bool((y == 0).all())
    ops.ffn(layer.e, x[:0], y[:0], ids=nothing[:0], workspace=None, stream=stream())
    ops.linear(x[:0], x, y[:0, :5], stream=stream())
    ops.route(x[:0].float(), nothing[:0], torch.empty((0, 2), device="cuda"), stream=stream())


def test_ffn_aborted_view_reads_the_guard_slot(ops):
    g = gen(2)
    layer = Layer(ops, g, "arena", 3, 64, 96, "bf16")
    words, _, _, parts = layer.keep
    for p in parts:
        p[-1].zero_()  # the guard slot
    words[0] = 1
    x, res = mat(g, 1, 64, "bf16"), mat(g, 1, 64, "bf16")
    ids = torch.tensor([[0, 2]], dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    ops.ffn(layer.e, x, y, ids=ids, residual=res, workspace=room(ops.ffn_workspace(layer.e, 1, 2)), stream=stream())
    assert torch.equal(y, res)


@pytest.mark.parametrize("rows,n,k,d,f", [(1, 1, 1, 64, 64), (1, 8, 2, 256, 128), (37, 8, 2, 320, 256), (64, 3, 2, 96, 160),
                                          (90, 4, 3, 128, 200), (300, 2, 1, 160, 264), (530, 3, 2, 256, 136)])
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("where", ["stacked", "arena"])
def test_ffn_backward(ops, rows, n, k, d, f, kind, where):
    g = gen(rows + f)
    layer = Layer(ops, g, where, n, d, f, kind)
    x, dy = mat(g, rows, d, kind, pad=8), mat(g, rows, d, kind, pad=16)
    ids, w = choices(g, rows, n, k)
    act = ACTS[(rows + k) % 4]
    t, dx = guarded(rows, d, kind)
    dw = torch.full((rows, k), 7.0, device="cuda")
    grads = [torch.full(s, 7.0, dtype=KINDS[kind], device="cuda") for s in ((n, f, d), (n, f, d), (n, d, f))]
    ws = room(ops.ffn_backward_workspace(layer.e, rows, k))
    ops.ffn_backward(layer.e, x, dy, dx, ids=ids, weights=w, dweights=dw, dgate=grads[0], dup=grads[1], ddown=grads[2], act=act,
                     workspace=ws, stream=stream())
    want_dx, want_dw, want = ffn64(layer, x, ids, w, None, act, dy)
    near(dx, want_dx, "dx")
    near(dw, want_dw, "dweights")
    for got, wanted, what in zip(grads, want, ("dgate", "dup", "ddown")):
        near(got, wanted, what)
        for e in range(n):
            if not bool((ids == e).any()):
                assert bool((got[e] == 0).all()), what
    untouched(t, rows, d)
    dx2 = torch.empty((rows, d), dtype=dx.dtype, device="cuda")  # the input's alone: the same bits
    ops.ffn_backward(layer.e, x, dy, dx2, ids=ids, weights=w, act=act, workspace=ws.zero_(), stream=stream())
    assert torch.equal(dx, dx2)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
def test_ffn_backward_many_tiles(ops, kind):
    """Enough tiles for the largest ones, and sums over more pairs than one filling of a tile's map of rows holds."""
    test_ffn_backward(ops, 3001, 2, 2, 1024, 1672, kind, "arena")


def test_ffn_backward_odd_sizes_and_dense(ops):
    g = gen(8)
    layer = Layer(ops, g, "stacked", 1, 45, 77, "bf16")
    x, dy = mat(g, 70, 45, "bf16", pad=1, shift=1), mat(g, 70, 45, "bf16", pad=2)
    ids, ones = torch.zeros((70, 1), dtype=torch.int32, device="cuda"), torch.ones((70, 1), device="cuda")
    dx = torch.empty((70, 45), dtype=torch.bfloat16, device="cuda")
    grads = [torch.empty(s, dtype=torch.bfloat16, device="cuda") for s in ((1, 77, 45), (1, 77, 45), (1, 45, 77))]
    ops.ffn_backward(layer.e, x, dy, dx, dgate=grads[0], dup=grads[1], ddown=grads[2],
                     workspace=room(ops.ffn_backward_workspace(layer.e, 70)), stream=stream())
    want_dx, _, want = ffn64(layer, x, ids, ones, None, "silu", dy)
    near(dx, want_dx)
    for got, wanted in zip(grads, want):
        near(got, wanted)
    empty = [t.fill_(7) for t in grads]  # no rows: zero gradients
    ops.ffn_backward(layer.e, x[:0], dy[:0], None, dgate=empty[0], dup=empty[1], ddown=empty[2],
                     workspace=room(ops.ffn_backward_workspace(layer.e, 0)), stream=stream())
    assert all(bool((t == 0).all()) for t in empty)


@pytest.mark.parametrize("act", ACTS)
def test_ffn_backward_against_differences(ops, act):
    """The slope of <y, dy> along random directions of x and of each weight, from the 64-bit forward formula. The
    gradients carry the operands' rounding (2^-11 each in half precision, two of them at most): 2e-3 of the product of
    the norms' typical size, sqrt(count) times smaller than their largest."""
    g = gen(11)
    rows, n, k, d, f = 6, 2, 2, 64, 96
    layer = Layer(ops, g, "stacked", n, d, f, "f16")
    x, dy = mat(g, rows, d, "f16"), mat(g, rows, d, "f16")
    ids, w = choices(g, rows, n, k, holes=False)
    dx = torch.empty_like(x)
    grads = [torch.empty(s, dtype=torch.float16, device="cuda") for s in ((n, f, d), (n, f, d), (n, d, f))]
    ops.ffn_backward(layer.e, x, dy, dx, ids=ids, weights=w, dgate=grads[0], dup=grads[1], ddown=grads[2], act=act,
                     workspace=room(ops.ffn_backward_workspace(layer.e, rows, k)), stream=stream())

    class Moved:
        pass

    def value(x64, w64):
        m = Moved()
        m.w64 = w64
        return float((ffn64(m, x64, ids, w, None, act) * dy.double()).sum())

    for which in range(4):
        grad = dx if which == 0 else grads[which - 1]
        way = torch.randn(grad.shape, device="cuda", generator=g).double()
        eps = 1e-6
        moved = [(x.double() + (s * way if which == 0 else 0), [t + (s * way if which == i + 1 else 0) for i, t in enumerate(layer.w64)])
                 for s in (eps, -eps)]
        slope = (value(*moved[0]) - value(*moved[1])) / (2 * eps)
        assert abs(slope - float((grad.double() * way).sum())) <= 2e-3 * float(grad.double().norm()) + 1e-6


# ---- together, on another stream, in a graph --------------------------------------------------------------------------
def test_layer_in_a_graph_on_another_stream(ops):
    """A decode layer (the router's product, the choice, the blocks) captured once on a stream of its own and replayed
    with new inputs between eager work: every replay gives what the eager calls give."""
    g = gen(21)
    n, k, d, f = 16, 4, 256, 192
    layer = Layer(ops, g, "arena", n, d, f, "bf16")
    router = mat(g, n, d, "bf16", sigma=0.1)
    s = torch.cuda.Stream()
    for rows in (1, 24):
        x = mat(g, rows, d, "bf16").contiguous()
        logits, ids = torch.empty((rows, n), device="cuda"), torch.empty((rows, k), dtype=torch.int32, device="cuda")
        w, y = torch.empty((rows, k), device="cuda"), torch.empty_like(x)
        ws = room(max(ops.ffn_workspace(layer.e, rows, k), ops.linear_workspace(x, router, logits)))

        def step():
            h = torch.cuda.current_stream().cuda_stream
            ops.linear(x, router, logits, workspace=ws, stream=h)
            ops.route(logits, ids, w, stream=h)
            ops.ffn(layer.e, x, y, ids=ids, weights=w, residual=x, workspace=ws, stream=h)

        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            step()
            s.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=s):
                step()
            for turn in range(4):
                x.copy_(mat(g, rows, d, "bf16"))
                step()
                s.synchronize()
                eager = [t.clone() for t in (logits, ids, w, y)]
                for t in (logits, ids, w, y):
                    t.zero_()
                ws.fill_(turn)
                graph.replay()
                s.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(eager, (logits, ids, w, y)))
        want = ffn64(layer, x, ids, w, x, "silu")
        near(y, want)

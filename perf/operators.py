"""The model operators that run between the library's serving calls, as cases that can be timed and compared.

A decode step that streams its experts does, at every layer: a product with the weights of the layer (a streamed block of
dense weights, or the router's), the choice of the experts by the router's logits, and the gated feed-forward blocks of
the chosen experts, read where the library put their units (the slots of a device-gated arena, the addresses of the host
contract's table, or weights that lie one after the other). Training adds the gradients of the choice and of the blocks.

Every case is a dict of plain values; "op" names the operator:

  route     ids and weights of the top_k largest logits of each row ("grad": the logits' gradient too)
  linear    y = act(x W^T + bias) + residual
  ffn       y_t = residual_t + sum_j w_tj Wd_e (act(Wg_e x_t) * (Wu_e x_t)), e = ids_tj
  ffn_grad  the gradients of ffn with respect to x, w and the three weights

`own` chooses who computes: False, elementary torch operations in 32 bits; True, the library.
"""
import ctypes as C
import math

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
Q4_BLOCK, Q4_BYTES = 32, 18  # values per block; its bytes: a half-precision scale, then 16 bytes of 4-bit values


def listed():
    return [
        # One token's choice among 256 experts: what a decode step waits for before it can export its ids (latency).
        {"name": "route-token", "op": "route", "rows": 1, "experts": 256, "top_k": 8, "type": "f32", "renorm": True,
         "masked": 0.0, "grad": False},
        # A training step's choice and its gradient: the qwen3-moe layer, many rows, some experts masked out.
        {"name": "route-train", "op": "route", "rows": 8191, "experts": 128, "top_k": 8, "type": "bf16", "renorm": True,
         "masked": 0.2, "grad": True},
        # The router's own product for one token of the deepseek-q4 shape: few weights, all latency.
        {"name": "linear-logits", "op": "linear", "rows": 1, "n_in": 7168, "n_out": 256, "type": "bf16", "w": "bf16",
         "y": "f32", "act": "none", "bias": False, "residual": False, "pad": 0},
        # One token through a whole block of the dense-prefix workload (4096 x 28672): the weights' bytes.
        {"name": "linear-token", "op": "linear", "rows": 1, "n_in": 4096, "n_out": 28672, "type": "bf16", "w": "bf16",
         "y": "bf16", "act": "silu", "bias": True, "residual": False, "pad": 0},
        # A prompt of odd length through the same block, with the whole epilogue: matrix instructions.
        {"name": "linear-prompt", "op": "linear", "rows": 2047, "n_in": 4096, "n_out": 28672, "type": "bf16", "w": "bf16",
         "y": "bf16", "act": "gelu_tanh", "bias": True, "residual": True, "pad": 8},
        # A small batch over 4-bit weights of the deepseek-q4 part's size.
        {"name": "linear-q4-batch", "op": "linear", "rows": 19, "n_in": 2048, "n_out": 7168, "type": "f16", "w": "q4",
         "y": "f16", "act": "none", "bias": False, "residual": True, "pad": 0},
        # A decode token of the mixtral workload: two experts of 352 MB in the slots of the arena.
        {"name": "ffn-token", "op": "ffn", "rows": 1, "experts": 8, "top_k": 2, "d": 4096, "f": 14336, "type": "bf16",
         "w": "bf16", "where": "arena", "act": "silu", "holes": 0.0, "zipf": 1.1},
        # A decode token of the deepseek-q4 workload: eight experts of 24.8 MB in 4-bit blocks.
        {"name": "ffn-q4-token", "op": "ffn", "rows": 1, "experts": 64, "top_k": 8, "d": 7168, "f": 2048, "type": "bf16",
         "w": "q4", "where": "arena", "act": "silu", "holes": 0.0, "zipf": 1.2},
        # A decode step of the qwen3-moe workload: 32 rows, top 8 of 128 experts, through the host contract's table.
        {"name": "ffn-step", "op": "ffn", "rows": 32, "experts": 128, "top_k": 8, "d": 2048, "f": 768, "type": "bf16",
         "w": "bf16", "where": "table", "act": "silu", "holes": 0.0, "zipf": 1.1},
        # A prompt of the mixtral workload: the largest products, groups of unlike sizes.
        {"name": "ffn-prompt", "op": "ffn", "rows": 4001, "experts": 8, "top_k": 2, "d": 4096, "f": 14336, "type": "bf16",
         "w": "bf16", "where": "arena", "act": "silu", "holes": 0.0, "zipf": 1.1},
        # A small, ragged training step of the moe-small shape: rows without experts, experts without rows.
        {"name": "ffn-train-small", "op": "ffn_grad", "rows": 37, "experts": 8, "top_k": 2, "d": 1024, "f": 512,
         "type": "f16", "w": "f16", "where": "stacked", "act": "gelu", "holes": 0.2, "zipf": 1.1},
        # A training step of a qwen3-moe layer: every gradient, 16 k pairs of a row and an expert.
        {"name": "ffn-train", "op": "ffn_grad", "rows": 2048, "experts": 128, "top_k": 8, "d": 2048, "f": 768,
         "type": "bf16", "w": "bf16", "where": "stacked", "act": "silu", "holes": 0.0, "zipf": 1.1},
    ]


def _spread(rng, lo, hi, unit=1):
    """A multiple of `unit` between lo and hi, spread over the logarithm."""
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))) // unit * unit


def draw(rng):
    op = rng.choice(["route", "linear", "linear", "ffn", "ffn", "ffn", "ffn_grad", "ffn_grad"])
    if op == "route":
        experts = _spread(rng, 4, 512)
        return {"op": op, "rows": _spread(rng, 1, 16384), "experts": experts, "top_k": rng.randint(1, min(16, experts)),
                "type": rng.choice(["f32", "bf16", "f16"]), "renorm": rng.random() < 0.6,
                "masked": rng.choice([0.0, 0.0, 0.3, 0.97]), "grad": rng.random() < 0.5}
    if op == "linear":
        w = rng.choice(["same", "same", "q4"])
        n_in = _spread(rng, 64, 8192, rng.choice([64, 8, 1]) if w == "same" else 32)
        n_out, kind = _spread(rng, 16, 32768, rng.choice([16, 1])), rng.choice(["bf16", "f16"])
        rows = min(_spread(rng, 1, 4096), max(1, int(2e11 / (n_in * n_out))))
        return {"op": op, "rows": rows, "n_in": n_in, "n_out": n_out, "type": kind, "w": kind if w == "same" else w,
                "y": rng.choice([kind, kind, "f32"]), "act": rng.choice(["none", "silu", "gelu", "gelu_tanh", "relu"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "pad": rng.choice([0, 0, 8, 3])}
    experts = rng.choice([1, _spread(rng, 2, 128), _spread(rng, 2, 128)])
    d, f = _spread(rng, 256, 7168, 32), _spread(rng, 256, 14336, 32)
    if experts * d * f > 1.3e8:
        experts = max(1, int(1.3e8 / (d * f)))
    kind = rng.choice(["bf16", "bf16", "f16"])
    if op == "ffn":
        w, where = rng.choice([kind, kind, "q4"]), rng.choice(["arena", "table", "stacked"])
        rows = min(_spread(rng, 1, 4096), max(1, int(1e12 / (6.0 * experts * d * f))))
    else:
        w, where = kind, rng.choice(["arena", "stacked"])
        rows = min(_spread(rng, 1, 2048), max(1, int(6e11 / (16.0 * experts * d * f))))
    return {"op": op, "rows": rows, "experts": experts, "top_k": rng.randint(1, min(8, experts)), "d": d, "f": f,
            "type": kind, "w": w, "where": where, "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]),
            "holes": rng.choice([0.0, 0.0, 0.2]), "zipf": rng.choice([0.0, 1.1])}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, kind, sigma=1.0):
    return (torch.randn(shape, device="cuda", generator=g, dtype=TYPES[kind] if kind != "f32" else torch.float32) * sigma)


def _q4(g, rows, cols):
    """[rows][cols / 32 * 18] bytes: blocks of a half-precision scale and 32 4-bit values."""
    blocks = rows * (cols // Q4_BLOCK)
    raw = torch.randint(0, 256, (blocks, Q4_BYTES), dtype=torch.uint8, device="cuda", generator=g)
    raw[:, :2] = (torch.randn(blocks, 1, device="cuda", generator=g) * 0.005).to(torch.float16).view(torch.uint8)
    return raw.view(rows, -1)


def _weights(g, rows, cols, kind):
    return _q4(g, rows, cols) if kind == "q4" else _normal(g, (rows, cols), kind, 0.02)


def _part_width(cols, kind):
    return cols // Q4_BLOCK * Q4_BYTES if kind == "q4" else cols


def _choices(g, case):
    """ids [rows][top_k] without repetition in a row, experts drawn by a power law; a share of them absent (-1), and of
    the rows whole."""
    rows, n, k = case["rows"], case["experts"], case["top_k"]
    rank = torch.randperm(n, device="cuda", generator=g).float() + 1
    u = torch.rand((rows, n), device="cuda", generator=g).clamp_(1e-7, 1 - 1e-7)
    ids = (-case["zipf"] * rank.log() - (-u.log()).log()).topk(k, dim=1).indices.to(torch.int32)
    weights = torch.randn((rows, k), device="cuda", generator=g).softmax(1)
    if case["holes"]:
        gone = torch.rand((rows, k), device="cuda", generator=g) < case["holes"]
        gone |= torch.rand((rows, 1), device="cuda", generator=g) < case["holes"] / 2
        ids = ids.masked_fill(gone, -1)
    return ids.contiguous(), weights.contiguous()


def prepare(case, seed):
    g = _generator(seed)
    s = dict(case)
    if case["op"] == "route":
        logits = torch.randn((case["rows"], case["experts"]), device="cuda", generator=g) * 2
        logits = logits.masked_fill(torch.rand(logits.shape, device="cuda", generator=g) < case["masked"], -math.inf)
        s["logits"] = logits.to(TYPES[case["type"]])
        s["dweights"] = torch.randn((case["rows"], case["top_k"]), device="cuda", generator=g)
        return s
    if case["op"] == "linear":
        rows, n_in, n_out = case["rows"], case["n_in"], case["n_out"]
        s["x"] = _normal(g, (rows, n_in + case["pad"]), case["type"])[:, :n_in]
        s["weight"] = _weights(g, n_out, n_in, case["w"])
        s["bias_v"] = _normal(g, (n_out,), case["type"]) if case["bias"] else None
        s["residual_v"] = _normal(g, (rows, n_out), case["y"]) if case["residual"] else None
        return s
    rows, n, d, f = case["rows"], case["experts"], case["d"], case["f"]
    s["x"] = _normal(g, (rows, d), case["type"])
    s["ids"], s["weights"] = _choices(g, case)
    shapes = [(f, d), (f, d), (d, f)]
    slots = n if case["where"] == "stacked" else n + 3  # a few slots hold nothing that is asked for
    parts = [_weights(g, slots * r, c, case["w"]).view(slots, r, -1) for r, c in shapes]
    if case["where"] == "table":  # whole units, a unit's parts back to back
        s["units"] = torch.cat([p.reshape(slots, -1) for p in parts], 1)
        parts = None
    else:
        s["parts"] = parts
    slot_of = torch.randperm(slots, device="cuda", generator=g)[:n].to(torch.int32)
    if case["where"] == "stacked":
        slot_of = torch.arange(n, dtype=torch.int32, device="cuda")
    s["slot_of"] = slot_of
    if case["where"] == "arena":
        s["unit_base"] = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        s["abort"] = torch.zeros(2, dtype=torch.int32, device="cuda")
        s["slots"] = slots
    elif case["where"] == "table":
        unit = s["units"].shape[1] * s["units"].element_size()
        s["table"] = s["units"].data_ptr() + slot_of.to(torch.int64) * unit
    if case["op"] == "ffn":
        s["residual_v"] = _normal(g, (rows, d), case["type"])
    else:
        s["dy"] = _normal(g, (rows, d), case["type"])
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------
def _act(name, v):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v.clamp_min(0) if name == "relu" else v


def _act_slope(name, v):
    if name == "silu":
        t = torch.sigmoid(v)
        return t * (1 + v * (1 - t))
    if name == "gelu":
        return 0.5 * (1 + torch.erf(v * math.sqrt(0.5))) + v * torch.exp(-0.5 * v * v) * (1 / math.sqrt(2 * math.pi))
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (v + 0.044715 * v * v * v))
        return 0.5 * (1 + t) + 0.5 * v * (1 - t * t) * c * (1 + 3 * 0.044715 * v * v)
    return (v > 0).to(v.dtype)


def _values(w, wide):
    """Weights (the last axis a row) as numbers; 4-bit ones from their blocks: low halves of the 16 bytes, then high."""
    if w.dtype != torch.uint8:
        return w.to(wide)
    b = w.reshape(-1, Q4_BYTES)
    q = torch.cat([b[:, 2:] & 15, b[:, 2:] >> 4], 1).to(wide) - 8
    return (q * b[:, :2].contiguous().view(torch.float16).to(wide)).reshape(*w.shape[:-1], -1)


def _plain_route(s):
    v = s["logits"].float()
    v = torch.where(torch.isnan(v), torch.full_like(v, -math.inf), v)
    top, ids = torch.sort(v, dim=1, descending=True, stable=True)
    top, ids, k = top[:, :s["top_k"]], ids[:, :s["top_k"]], s["top_k"]
    best = top[:, :1]
    exps = torch.where(v == best, 1.0, torch.exp(v - best)).masked_fill(v == -math.inf, 0)
    chosen = torch.gather(exps, 1, ids)
    total = chosen.sum(1, keepdim=True) if s["renorm"] else exps.sum(1, keepdim=True)
    there = top > -math.inf
    weights = torch.where(there, chosen / total, 0.0)
    out = {"ids": torch.where(there, ids, -1).to(torch.int32), "weights": weights}
    if s["grad"]:
        mean = (weights * s["dweights"]).sum(1, keepdim=True)
        pull = torch.zeros_like(v).scatter_(1, ids, torch.where(there, s["dweights"], 0.0))
        if s["renorm"]:
            share = torch.zeros_like(v).scatter_(1, ids, weights)
        else:
            share = torch.where(total > 0, exps / total, 0.0)
        out["dlogits"] = (share * (pull - mean)).to(s["logits"].dtype)
    return out


def _plain_linear(s):
    y = _act(s["act"], s["x"].float() @ _values(s["weight"], torch.float32).T + (0 if s["bias_v"] is None else s["bias_v"].float()))
    if s["residual_v"] is not None:
        y = y + s["residual_v"].float()
    return {"y": y.to(TYPES[s["y"]])}


def _live(s):
    """The experts that some row asks for: their weights [n][rows][columns] in 32 bits, and the weight of each for each row."""
    ids = s["ids"].long()
    live = torch.unique(ids[ids >= 0])
    d, f, kind = s["d"], s["f"], s["w"]
    at = s["slot_of"].long()[live]
    if "units" in s:
        first = f * _part_width(d, kind)
        unit = s["units"][at]
        parts = [unit[:, :first].view(-1, f, _part_width(d, kind)), unit[:, first:2 * first].view(-1, f, _part_width(d, kind)),
                 unit[:, 2 * first:].view(-1, d, _part_width(f, kind))]
    else:
        parts = [p[at] for p in s["parts"]]
    asks = (ids[:, :, None] == live).float()  # [rows][top_k][live]
    return [_values(p, torch.float32) for p in parts], live, asks


def _plain_ffn(s):
    (gate, up, down), live, asks = _live(s)
    x, n = s["x"].float(), len(live)
    c = (asks * s["weights"][:, :, None]).sum(1)
    h = _act(s["act"], x @ gate.reshape(-1, s["d"]).T) * (x @ up.reshape(-1, s["d"]).T)
    h = (h.view(-1, n, s["f"]) * c[:, :, None]).reshape(-1, n * s["f"])
    y = h @ down.permute(0, 2, 1).reshape(-1, s["d"]) + s["residual_v"].float()
    return {"y": y.to(s["x"].dtype)}


def _plain_ffn_grad(s):
    (gate, up, down), live, asks = _live(s)
    x, dy, n, d, f = s["x"].float(), s["dy"].float(), len(live), s["d"], s["f"]
    kind = s["x"].dtype
    c = (asks * s["weights"][:, :, None]).sum(1)[:, :, None]
    gate2, up2 = gate.reshape(-1, d), up.reshape(-1, d)
    g, u = (x @ gate2.T).view(-1, n, f), (x @ up2.T).view(-1, n, f)
    back = (dy @ down.permute(1, 0, 2).reshape(d, -1)).view(-1, n, f)
    a = _act(s["act"], g)
    dweights = (asks * (a * u * back).sum(2)[:, None, :]).sum(2)
    dg = (c * back * u * _act_slope(s["act"], g)).reshape(-1, n * f)
    du = (c * back * a).reshape(-1, n * f)
    h = (c * a * u).reshape(-1, n * f)
    out = {"dx": (dg @ gate2 + du @ up2).to(kind), "dweights": dweights}
    every = {"dgate": (dg.T @ x).view(n, f, d), "dup": (du.T @ x).view(n, f, d), "ddown": (dy.T @ h).view(d, n, f).permute(1, 0, 2)}
    out.update({k: torch.zeros((s["experts"], *v.shape[1:]), dtype=kind, device=v.device).index_copy_(0, live, v.to(kind))
                for k, v in every.items()})
    return out


# ---- the library's calls --------------------------------------------------------------------------------------------
def _stream():
    return torch.cuda.current_stream().cuda_stream


def _room(n):
    return torch.empty(n, dtype=torch.uint8, device="cuda")


def _own_route(s):
    from tierstream_amd import ops
    logits = s["logits"]
    ids = torch.empty((s["rows"], s["top_k"]), dtype=torch.int32, device="cuda")
    weights = torch.empty((s["rows"], s["top_k"]), dtype=torch.float32, device="cuda")
    ops.route(logits, ids, weights, renorm=s["renorm"], stream=_stream())
    out = {"ids": ids, "weights": weights}
    if s["grad"]:
        out["dlogits"] = torch.empty_like(logits)
        ops.route_backward(logits, ids, s["dweights"], out["dlogits"], renorm=s["renorm"], stream=_stream())
    return out


def _own_linear(s):
    from tierstream_amd import ops
    y = torch.empty((s["rows"], s["n_out"]), dtype=TYPES[s["y"]], device="cuda")
    ws = _room(ops.linear_workspace(s["x"], s["weight"], y))
    ops.linear(s["x"], s["weight"], y, bias=s["bias_v"], residual=s["residual_v"], act=s["act"], workspace=ws, stream=_stream())
    return {"y": y}


def _experts(s):
    from tierstream_amd import ops, ss
    if s["where"] == "stacked":
        return ops.Experts.stacked(*s["parts"])
    kind = "q4" if s["w"] == "q4" else s["type"]
    if s["where"] == "table":
        return ops.Experts.in_table(s["table"], s["d"], s["f"], kind)
    v = ss.SsDgDeviceView(struct_size=C.sizeof(ss.SsDgDeviceView), n_gated=1, n_parts=3, guard_slot=s["slots"] - 1,
                          slots=s["slots"], slot_of=s["slot_of"].data_ptr(), unit_base=s["unit_base"].data_ptr(),
                          abort=s["abort"].data_ptr(), absent_err=s["abort"].data_ptr() + 4)
    for p, part in enumerate(s["parts"]):
        size = part[0].numel() * part.element_size()
        v.parts[p].base, v.parts[p].stride, v.parts[p].bytes = part.data_ptr(), size, size
    return ops.Experts.in_arena(v, 0, s["experts"], s["d"], s["f"], kind)


def _own_ffn(s):
    from tierstream_amd import ops
    e, y = _experts(s), torch.empty_like(s["x"])
    ws = _room(ops.ffn_workspace(e, s["rows"], s["top_k"]))
    ops.ffn(e, s["x"], y, ids=s["ids"], weights=s["weights"], residual=s["residual_v"], act=s["act"], workspace=ws,
            stream=_stream())
    return {"y": y}


def _own_ffn_grad(s):
    from tierstream_amd import ops
    e, dx, dweights = _experts(s), torch.empty_like(s["x"]), torch.empty_like(s["weights"])
    n, d, f = s["experts"], s["d"], s["f"]
    dgate, dup, ddown = (torch.empty(shape, dtype=s["x"].dtype, device="cuda") for shape in ((n, f, d), (n, f, d), (n, d, f)))
    ws = _room(ops.ffn_backward_workspace(e, s["rows"], s["top_k"]))
    ops.ffn_backward(e, s["x"], s["dy"], dx, ids=s["ids"], weights=s["weights"], dweights=dweights, dgate=dgate, dup=dup,
                     ddown=ddown, act=s["act"], workspace=ws, stream=_stream())
    return {"dx": dx, "dweights": dweights, "dgate": dgate, "dup": dup, "ddown": ddown}


_PLAIN = {"route": _plain_route, "linear": _plain_linear, "ffn": _plain_ffn, "ffn_grad": _plain_ffn_grad}
_OWN = {"route": _own_route, "linear": _own_linear, "ffn": _own_ffn, "ffn_grad": _own_ffn_grad}


def run(state):
    return (_OWN if own else _PLAIN)[state["op"]](state)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------
def _weight_bytes(values, kind):
    return values // Q4_BLOCK * Q4_BYTES if kind == "q4" else 2 * values


def work(case):
    rows = case["rows"]
    if case["op"] == "route":
        size, n, k = 4 if case["type"] == "f32" else 2, rows * case["experts"], rows * case["top_k"]
        return {"bytes": n * size + 8 * k + (n * size + 4 * k if case["grad"] else 0), "flops": n * (8 if case["grad"] else 4)}
    if case["op"] == "linear":
        n_in, n_out, wide = case["n_in"], case["n_out"], 4 if case["y"] == "f32" else 2
        return {"bytes": 2 * rows * n_in + _weight_bytes(n_in * n_out, case["w"]) + 2 * n_out * case["bias"]
                + wide * rows * n_out * (1 + case["residual"]), "flops": 2 * rows * n_in * n_out}
    d, f, n, k = case["d"], case["f"], case["experts"], case["top_k"]
    keep = (1 - case["holes"]) * (1 - case["holes"] / 2)
    share = [(i + 1.0) ** -case["zipf"] for i in range(n)]
    taken = [1 - (1 - min(1.0, k * keep * p / sum(share))) ** rows for p in share]  # an expert is asked for by some row
    live = min(float(n), max(k * keep, sum(taken)))
    unit = _weight_bytes(3 * d * f, case["w"])
    if case["op"] == "ffn":
        return {"bytes": live * unit + 6 * rows * d + 8 * rows * k, "flops": 6 * rows * k * keep * d * f}
    return {"bytes": live * unit + n * unit + 6 * rows * d + 12 * rows * k, "flops": 16 * rows * k * keep * d * f}


# ---- in 64 bits, expert by expert and formula by formula ------------------------------------------------------------
def _exact_act(name, v):
    """The activation and its slope."""
    if name == "silu":
        e = 1 / (1 + torch.exp(-v))
        return v * e, e + v * e * (1 - e)
    if name == "gelu":
        p = 0.5 * torch.erfc(-v / math.sqrt(2))
        return v * p, p + v * torch.exp(-v * v / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":  # 0.5 (1 + tanh z) = 1 / (1 + exp(-2 z))
        z = math.sqrt(8 / math.pi) * (v + 0.044715 * v ** 3)
        e = 1 / (1 + torch.exp(-z))
        return v * e, e + v * e * (1 - e) * math.sqrt(8 / math.pi) * (1 + 0.134145 * v * v)
    if name == "relu":
        return torch.where(v > 0, v, 0.0), torch.where(v > 0, 1.0, 0.0).to(v.dtype)
    return v, torch.ones_like(v)


def _exact_q4(raw):
    blocks = raw.reshape(raw.shape[0], -1, Q4_BYTES)
    scale = blocks[:, :, 0:2].contiguous().view(torch.float16).double()
    low = (blocks[:, :, 2:] % 16).double() - 8
    high = torch.div(blocks[:, :, 2:], 16, rounding_mode="floor").double() - 8
    return torch.cat([low * scale, high * scale], 2).reshape(raw.shape[0], -1)


def _exact_weight(w):
    return _exact_q4(w) if w.dtype == torch.uint8 else w.double()


def _exact_route(s):
    v, k = s["logits"].double(), s["top_k"]
    order = torch.argsort(-v, dim=1, stable=True)[:, :k]
    top = torch.gather(v, 1, order)
    there = torch.isfinite(top)
    p = torch.softmax(v, 1) if not s["renorm"] else torch.softmax(torch.full_like(v, -math.inf).scatter(1, order, top), 1)
    p = torch.nan_to_num(p, nan=0.0)  # a row with nothing to choose from
    weights = torch.gather(p, 1, order) * there
    out = {"ids": torch.where(there, order, -1).to(torch.int32), "weights": weights}
    if s["grad"]:  # d w_j / d l_i = p_i (delta_ij - w_j)
        dw = s["dweights"].double() * there
        full = torch.zeros_like(v).scatter(1, order, dw)
        out["dlogits"] = p * full - p * (weights * dw).sum(1, keepdim=True)
    return out


def _exact_linear(s):
    z = torch.matmul(s["x"].double(), _exact_weight(s["weight"]).T)
    if s["bias_v"] is not None:
        z = z + s["bias_v"].double()
    y = _exact_act(s["act"], z)[0]
    return {"y": y if s["residual_v"] is None else y + s["residual_v"].double()}


def _exact_unit(s, e):
    at, d, f = int(s["slot_of"][e]), s["d"], s["f"]
    if "units" in s:
        wd, wf = _part_width(d, s["w"]), _part_width(f, s["w"])
        parts = [t.view(r, c) for t, r, c in zip(s["units"][at].split([f * wd, f * wd, d * wf]), (f, f, d), (wd, wd, wf))]
    else:
        parts = [p[at] for p in s["parts"]]
    return [_exact_weight(p) for p in parts]


def _exact_ffn(s):
    grad = s["op"] == "ffn_grad"
    x, w = s["x"].double(), s["weights"].double()
    y = torch.zeros_like(x) if grad else s["residual_v"].double().clone()
    d, f, n = s["d"], s["f"], s["experts"]
    if grad:
        dy, dx, dweights = s["dy"].double(), torch.zeros_like(x), torch.zeros_like(w)
        kept = {"dgate": (n, f, d), "dup": (n, f, d), "ddown": (n, d, f)}
        kept = {k: torch.zeros(v, dtype=torch.float64, device="cuda") for k, v in kept.items()}
    for e in range(n):
        row, col = torch.nonzero(s["ids"] == e, as_tuple=True)
        if not len(row):
            continue
        gate, up, down = _exact_unit(s, e)
        xe, we = x[row], w[row, col][:, None]
        u = xe @ up.T
        a, slope = _exact_act(s["act"], xe @ gate.T)
        if not grad:
            y.index_add_(0, row, we * ((a * u) @ down.T))
            continue
        dh = dy[row] @ down
        dweights[row, col] = (dh * a * u).sum(1)
        dgate, dup = we * dh * u * slope, we * dh * a
        dx.index_add_(0, row, dgate @ gate + dup @ up)
        kept["dgate"][e], kept["dup"][e] = dgate.T @ xe, dup.T @ xe
        kept["ddown"][e] = dy[row].T @ (we * a * u)
    return {"dx": dx, "dweights": dweights, **kept} if grad else {"y": y}


def exact(case, seed):
    s = prepare(case, seed)
    return {"route": _exact_route, "linear": _exact_linear, "ffn": _exact_ffn, "ffn_grad": _exact_ffn}[case["op"]](s)

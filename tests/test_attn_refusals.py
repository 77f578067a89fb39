"""What the attention operators refuse (include/tierstream_amd/tsa_attn.h, tierstream_amd/attn.py), before any launch: no GPU is
needed."""
import ctypes as C
import math
from pathlib import Path

import pytest

import tierstream_amd as tsa
from test_abi import declared
from test_ops_refusals import P, changed, refused
from tierstream_amd import attn, ops

ROOT = Path(__file__).resolve().parent.parent


def heads(n=4, dim=128, tokens=8, **kw):
    h = attn.TsaHeads(P, n * dim, dim, n, 0)
    for k, v in kw.items():
        setattr(h, k, v)
    return h


def call(name, *args, says, **kw):
    refused(getattr(attn._attn(), name), *args, says=says, **kw)


def test_every_declared_operator_is_exported():
    names = declared(ROOT / "include" / "tierstream_amd" / "tsa_attn.h")
    assert len(names) == 11
    assert [n for n in names if not hasattr(tsa.lib(), n)] == []


def test_struct_sizes_are_the_headers(tmp_path):
    """The ctypes structs against the compiler's."""
    import subprocess
    pairs = {"tsa_heads": attn.TsaHeads, "tsa_rotary_params": attn.TsaRotaryParams, "tsa_rotary": attn.TsaRotary, "tsa_rotate_args": attn.TsaRotateArgs,
             "tsa_cache": attn.TsaCache, "tsa_cache_plan_args": attn.TsaCachePlanArgs, "tsa_cache_rows_args": attn.TsaCacheRowsArgs,
             "tsa_attend_cached_args": attn.TsaAttendCachedArgs, "tsa_attend_args": attn.TsaAttendArgs, "tsa_attend_grad_args": attn.TsaAttendGradArgs}
    lines = []
    for name, cls in pairs.items():
        lines.append(f"_Static_assert(sizeof({name}) == {C.sizeof(cls)}, \"{name}\");")
        lines += [f"_Static_assert(offsetof({name}, {f[0]}) == {getattr(cls, f[0]).offset}, \"{name}.{f[0]}\");" for f in cls._fields_]
    src = tmp_path / "sizes.c"
    src.write_text("#include <stddef.h>\n#include \"tierstream_amd/tsa_attn.h\"\n" + "\n".join(lines) + "\nint main(void) { return 0; }\n")
    packed = {attn._ROTATE: attn.TsaRotateArgs, attn._PLAN: attn.TsaCachePlanArgs, attn._ROWS: attn.TsaCacheRowsArgs, attn._CACHED: attn.TsaAttendCachedArgs,
              attn._ATTEND: attn.TsaAttendArgs, attn._GRAD: attn.TsaAttendGradArgs}
    assert all(p.size == C.sizeof(cls) for p, cls in packed.items())
    r = subprocess.run(["gcc", f"-I{ROOT / 'include'}", "-c", str(src), "-o", str(tmp_path / "sizes.o")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_rotary():
    good = attn.TsaRotaryParams(10000.0, 4.0, 8192.0, 1.0, 4.0, 1.0, 128, 0)
    out = attn.TsaRotary()
    call("tsa_rotary_init", None, out, says="null")
    call("tsa_rotary_init", good, None, says="null")
    for bad in (dict(rotated=0), dict(rotated=3), dict(rotated=258), dict(interleaved=2), dict(base=0.0), dict(base=math.inf), dict(factor=0.0),
                dict(factor=math.nan), dict(amplitude=math.inf), dict(trained=-1.0), dict(high=1.0), dict(low=math.nan)):
        call("tsa_rotary_init", changed(good, **bad), out, says="tsa_rotary_init")
    assert attn._attn().tsa_rotary_init(good, out) == tsa.SS_OK and out.pairs == 64


@pytest.mark.parametrize("factor,trained", [(1.0, 0), (8.0, 0), (4.0, 8192), (0.5, 100)])
def test_frequencies(factor, trained):
    r = attn.Rotary(96, base=5e5, factor=factor, trained=trained, low=1.0, high=4.0, amplitude=1.25)
    for i in range(48):
        f = 5e5 ** (-2 * i / 96)
        if factor != 1:
            keep = min(1.0, max(0.0, (trained * f / (2 * math.pi) - 1) / 3))
            f = keep * f + (1 - keep) * f / factor
        assert abs(r.s.turns[i] * 2 * math.pi / f - 1) < 1e-14
    assert r.s.amplitude == 1.25 and r.s.pairs == 48


def test_rotate():
    r = attn.Rotary(128).s
    a = attn.TsaRotateArgs(positions=P, tokens=8, head_dim=128, type=ops.BF16)
    a.x[0], a.y[0], a.x[1], a.y[1] = heads(), heads(), heads(2), heads(2)
    call("tsa_rotate", None, a, None, says="null")
    call("tsa_rotate", r, None, None, says="null")
    for bad in (dict(type=ops.Q4), dict(head_dim=64), dict(head_dim=1032), dict(backward=2), dict(tokens=1 << 24), dict(positions=None), dict(positions=P + 2)):
        call("tsa_rotate", r, changed(a, **bad), None, says="tsa_rotate")
    call("tsa_rotate", changed(r, pairs=0), a, None, says="tsa_rotary_init")
    for i in range(2):
        for what, h in (("x", heads(p=None)), ("x", heads(p=P + 1)), ("x", heads(heads=0)), ("x", heads(heads=3)), ("x", heads(token_stride=1 << 40)),
                        ("y", heads(token_stride=100)), ("y", heads(head_stride=127)), ("y", heads(p=None)), ("x", heads(token_stride=1024))):
            b = changed(a)
            getattr(b, what)[i] = h
            call("tsa_rotate", r, b, None, says="tsa_rotate")
    assert attn._attn().tsa_rotate(r, changed(a, tokens=0), None) == tsa.SS_OK


def plan_args(**kw):
    names = ("lengths", "fresh", "table", "free", "n_free", "ends", "left", "first", "positions", "slots", "status")
    a = attn.TsaCachePlanArgs(requests=4, width=8, table_stride=8, pages=32, rows=16, **dict.fromkeys(names, P))
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_plan_and_slots():
    call("tsa_cache_plan", None, None, says="null")
    call("tsa_cache_slots", None, None, says="null")
    for name in ("lengths", "fresh", "table", "free", "n_free", "ends", "left", "first", "positions", "slots", "status"):
        for v in (None, P + 2):
            call("tsa_cache_plan", plan_args(**{name: v}), None, says="tsa_cache_plan")
            if name in ("table", "ends", "first", "positions", "slots"):
                call("tsa_cache_slots", plan_args(**{name: v}), None, says="tsa_cache_slots")
    for bad in (dict(requests=4097), dict(width=0), dict(width=1 << 25), dict(table_stride=7), dict(table_stride=1 << 40), dict(rows=1 << 24)):
        call("tsa_cache_plan", plan_args(**bad), None, says="tsa_cache_plan")
        call("tsa_cache_slots", plan_args(**bad), None, says="tsa_cache_slots")
    call("tsa_cache_plan", plan_args(pages=1 << 25), None, says="pages")
    assert attn._attn().tsa_cache_slots(plan_args(rows=0, slots=None), None) == tsa.SS_OK


CACHE = attn.TsaCache(P, 16, 4, 128, 0)
BAD_CACHES = [dict(head_dim=0), dict(head_dim=16), dict(head_dim=160), dict(head_dim=48), dict(kv_heads=0), dict(kv_heads=1025),
              dict(n_pages=1 << 25), dict(pages=None), dict(pages=P + 8)]


@pytest.mark.parametrize("name", ["tsa_cache_store", "tsa_cache_load"])
def test_store_and_load(name):
    a = attn.TsaCacheRowsArgs(heads(), heads(), P, 8, ops.BF16)
    call(name, None, a, None, says="null")
    call(name, CACHE, None, None, says="null")
    for bad in BAD_CACHES:
        call(name, changed(CACHE, **bad), a, None, says=name)
    for bad in (dict(type=ops.F32), dict(tokens=1 << 24), dict(slots=None), dict(slots=P + 1), dict(k=heads(p=None)), dict(v=heads(3)), dict(k=heads(p=P + 1)),
                dict(v=heads(head_stride=1 << 40))):
        call(name, CACHE, changed(a, **bad), None, says=name)
    call(name, changed(CACHE, kv_heads=1024), changed(a, tokens=1 << 23, k=heads(1024), v=heads(1024)), None, says="2^33")
    if name == "tsa_cache_load":
        call(name, CACHE, changed(a, v=heads(head_stride=100)), None, says="overlap")
    assert getattr(attn._attn(), name)(CACHE, changed(a, tokens=0, slots=None), None) == tsa.SS_OK


def test_attend_cached():
    a = attn.TsaAttendCachedArgs(heads(8), heads(8), P, 4, P, P, 8, 4, 4, ops.BF16, 0.1)
    size = attn._attn().tsa_attend_cached_workspace
    for bad in BAD_CACHES:
        call("tsa_attend_cached", changed(CACHE, **bad), a, P, 1 << 40, None, says="tsa_attend_cached")
    call("tsa_attend_cached", None, a, P, 1 << 40, None, says="null")
    call("tsa_attend_cached", CACHE, None, P, 1 << 40, None, says="null")
    for bad in (dict(type=ops.F32), dict(q=heads(6)), dict(q=heads(0)), dict(q=heads(8, p=None)), dict(out=heads(4)), dict(out=heads(8, head_stride=64)),
                dict(table=None), dict(table_stride=3), dict(ends=None), dict(ends=P + 1), dict(first=None), dict(tokens=1 << 24), dict(requests=4097),
                dict(width=0), dict(scale=math.inf)):
        call("tsa_attend_cached", CACHE, changed(a, **bad), P, 1 << 40, None, says="tsa_attend_cached")
    need = size(CACHE, a)
    if need:
        call("tsa_attend_cached", CACHE, a, P, need - 1, None, says="workspace")
        call("tsa_attend_cached", CACHE, a, P + 8, need, None, says="workspace")
    assert size(CACHE, changed(a, width=0)) == 0
    assert attn._attn().tsa_attend_cached(CACHE, changed(a, tokens=0), None, 0, None) == tsa.SS_OK
    assert attn._attn().tsa_attend_cached(CACHE, changed(a, requests=0), None, 0, None) == tsa.SS_OK


def attend_args(**kw):
    a = attn.TsaAttendArgs(heads(8), heads(), heads(), heads(8), P, P, P, 8, 8, 2, 128, ops.BF16, 1, 0.1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


BAD_ATTEND = [dict(type=ops.F32), dict(head_dim=0), dict(head_dim=12), dict(head_dim=136), dict(tokens=1 << 24), dict(k_tokens=1 << 24),
              dict(sequences=1 << 24), dict(q=heads(6)), dict(q=heads(0)), dict(v=heads(2)), dict(causal=2), dict(scale=math.nan), dict(first=None),
              dict(first=None, k_first=None), dict(k_first=None, k_tokens=9), dict(first=P + 2), dict(lse=P + 1), dict(q=heads(8, p=None)),
              dict(k=heads(4, p=P + 1)), dict(out=heads(4))]


def test_attend():
    call("tsa_attend", None, None, says="null")
    for bad in [*BAD_ATTEND, dict(out=heads(8, token_stride=512))]:
        call("tsa_attend", attend_args(**bad), None, says="tsa_attend")
    assert attn._attn().tsa_attend(attend_args(tokens=0, k_first=P), None) == tsa.SS_OK
    assert attn._attn().tsa_attend(attend_args(sequences=0), None) == tsa.SS_OK


def test_attend_backward():
    f, size = "tsa_attend_backward", attn._attn().tsa_attend_backward_workspace
    g = attn.TsaAttendGradArgs(attend_args(), heads(8), heads(8), heads(), heads())
    call(f, None, P, 1 << 40, None, says="null")
    for bad in BAD_ATTEND:
        call(f, changed(g, f=attend_args(**bad)), P, 1 << 40, None, says=f)
    for bad in (dict(dout=heads(4)), dict(dout=heads(8, p=None)), dict(dq=heads(4)), dict(dq=heads(8, head_stride=8)), dict(dk=heads(4, p=None)),
                dict(dv=heads(4, p=None)), dict(dk=heads(8)), dict(dv=heads(4, head_stride=0)), dict(f=attend_args(lse=None))):
        call(f, changed(g, **bad), P, 1 << 40, None, says=f)
    need = size(attend_args())
    if need:
        call(f, g, P, need - 1, None, says="workspace")
        call(f, g, None, need, None, says="workspace")
    assert size(attend_args(head_dim=12)) == 0
    none = heads(4, p=None)
    assert getattr(attn._attn(), f)(changed(g, dq=heads(8, p=None), dk=none, dv=none), None, 0, None) == tsa.SS_OK


# ---- arrays -----------------------------------------------------------------------------------------------------------------
class Fake:
    is_cuda, device = True, "cuda:0"

    def __init__(self, *shape, dtype="torch.bfloat16", **kw):
        self.shape, self.dtype = shape, dtype
        self.__dict__.update(kw)

    def stride(self):
        s = [1]
        for n in self.shape[:0:-1]:
            s.insert(0, s[0] * n)
        return tuple(s)

    def is_contiguous(self):
        return True

    def data_ptr(self):
        return P

    def numel(self):
        return math.prod(self.shape)

    def element_size(self):
        return 2


def i32(*shape, **kw):
    return Fake(*shape, dtype="torch.int32", **kw)


def cache():
    return attn.Cache(Fake(16, 4, 72 * 128, dtype="torch.uint8"), 4, 128)


CALLS = {
    "q": lambda m: attn.rotate(attn.Rotary(128), i32(8), m(8, 4, 128)),
    "positions": lambda m: attn.rotate(attn.Rotary(128), m(8, dtype="torch.int32"), Fake(8, 4, 128)),
    "k_out": lambda m: attn.rotate(attn.Rotary(128), i32(8), Fake(8, 4, 128), Fake(8, 4, 128), None, m(8, 4, 128)),
    "pages": lambda m: attn.Cache(m(16, 4, 72 * 128, dtype="torch.uint8"), 4, 128),
    "table": lambda m: attn.slots(m(4, 8, dtype="torch.int32"), i32(4), i32(5), i32(9), i32(9)),
    "free": lambda m: attn.plan(i32(4), i32(4), i32(4, 8), m(9, dtype="torch.int32"), i32(1), i32(5), i32(9), i32(9), i32(1)),
    "slots": lambda m: attn.store(cache(), Fake(8, 4, 128), Fake(8, 4, 128), m(8, dtype="torch.int32")),
    "v": lambda m: attn.load(cache(), i32(8), Fake(8, 4, 128), m(8, 4, 128)),
    "ends": lambda m: attn.attend_cached(cache(), Fake(4, 8, 128), Fake(4, 8, 128), i32(4, 8), m(4, dtype="torch.int32"), i32(5)),
    "out": lambda m: attn.attend(Fake(4, 8, 128), Fake(4, 4, 128), Fake(4, 4, 128), m(4, 8, 128)),
    "lse": lambda m: attn.attend(Fake(4, 8, 128), Fake(4, 4, 128), Fake(4, 4, 128), Fake(4, 8, 128), lse=m(8, 4, dtype="torch.float32")),
    "dk": lambda m: attn.attend_backward(*[Fake(4, 4, 128)] * 5, Fake(4, 4, dtype="torch.float32"), None, m(4, 4, 128), Fake(4, 4, 128)),
}


@pytest.mark.parametrize("name", CALLS)
def test_an_array_of_the_host_is_refused(name):
    with pytest.raises(ValueError, match=f"{name}.*device memory"):
        CALLS[name](lambda *shape, **kw: Fake(*shape, is_cuda=False, **kw))


@pytest.mark.parametrize("name", CALLS)
def test_another_shape_or_type_is_refused(name):
    with pytest.raises(ValueError, match={"q": "positions|q", "ends": "ends|table"}.get(name, name)):
        CALLS[name](lambda *shape, **kw: Fake(shape[0] + 1, *shape[1:], 1, **kw))


@pytest.mark.parametrize("name", [n for n in CALLS if n not in ("pages",)])
def test_an_array_of_another_device_is_refused(name):
    with pytest.raises(ValueError, match="cuda:0"):
        CALLS[name](lambda *shape, **kw: Fake(*shape, device="cuda:1", **kw))


def test_values_of_a_head_lie_together():
    spaced = Fake(8, 4, 128)
    spaced.stride = lambda: (1024, 256, 2)
    with pytest.raises(ValueError, match="next to each other"):
        attn.rotate(attn.Rotary(128), i32(8), spaced)


@pytest.mark.parametrize("head_dim", [32, 128])
@pytest.mark.parametrize("kind", [ops.BF16, ops.F16])
def test_workspaces_grow(head_dim, kind):
    """One that holds a batch holds every smaller one."""
    c = attn.TsaCache(P, 16, 4, head_dim, 0)
    at = [1, 2, 3, 15, 16, 17, 63, 64, 65, 127, 500, 1024, 4096]
    size = lambda t, n, w: attn._attn().tsa_attend_cached_workspace(  # noqa: E731
        c, attn.TsaAttendCachedArgs(q=heads(8), tokens=t, requests=n, width=w, type=kind))
    for n in at:
        for w in at:
            sizes = [size(t, n, w) for t in at]
            assert sizes == sorted(sizes)
    for t in at:
        for w in at:
            sizes = [size(t, n, w) for n in at]
            assert sizes == sorted(sizes)
        for n in at:
            sizes = [size(t, n, w) for w in at]
            assert sizes == sorted(sizes)
    back = lambda t, k: attn._attn().tsa_attend_backward_workspace(attend_args(tokens=t, k_tokens=k, head_dim=head_dim, type=kind))  # noqa: E731
    for k in at:
        sizes = [back(t, k) for t in at]
        assert sizes == sorted(sizes)
        sizes = [back(k, t) for t in at]
        assert sizes == sorted(sizes)

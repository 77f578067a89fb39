"""What a decoder of tierstream_amd.moe keeps while its model is trained on: the tensors whose addresses its graph holds."""
import contextlib
import gc
import types
import weakref

import pytest

torch = pytest.importorskip("torch")


def test_the_captured_weights_outlive_the_models(monkeypatch):
    """No GPU: the calls that are captured are recorded instead. After the model's own tensors are replaced, as a step does, every
    tensor that a captured product reads is still there."""
    from tierstream_amd import moe
    s = moe.Shape(layers=2, experts=4, top_k=2, d_model=32, d_ff=32, vocab=16)
    model = moe.Model.__new__(moe.Model)
    model.s, model.embedding = s, torch.zeros(s.vocab, s.d_model)
    model.w = {"head": torch.zeros(s.vocab, s.d_model), **{f"router{L}": torch.zeros(s.experts, s.d_model) for L in range(s.layers)}}
    read = []

    class Ctx:
        def __getattr__(self, name):
            return lambda *a, **k: 0

    monkeypatch.setattr(moe, "ss", types.SimpleNamespace(Desc=lambda *a: None, Plan=lambda *a: None, Ctx=lambda *a: Ctx(),
                                                         budget=lambda **k: None, options=lambda **k: None))
    monkeypatch.setattr(moe, "_empty", lambda *shape, dtype=moe.BF16: torch.empty(shape, dtype=dtype))
    monkeypatch.setattr(moe.ops.Experts, "in_arena", classmethod(lambda cls, *a: types.SimpleNamespace(s=types.SimpleNamespace(gated=0))))
    monkeypatch.setattr(moe.ops, "linear", lambda x, w, y, **k: read.append(weakref.ref(w)))
    for name in ("linear_workspace", "ffn_workspace"):
        monkeypatch.setattr(moe.ops, name, lambda *a: 0)
    for name in ("route", "ffn"):
        monkeypatch.setattr(moe.ops, name, lambda *a, **k: None)
    for name, value in (("Stream", lambda: None), ("CUDAGraph", lambda: None), ("synchronize", lambda: None),
                        ("graph", lambda *a, **k: contextlib.nullcontext()),
                        ("current_stream", lambda: types.SimpleNamespace(cuda_stream=0))):
        monkeypatch.setattr(torch.cuda, name, value)
    decoder = moe.Decoder(model, "")
    assert len(read) == s.layers + 1
    model.w = {}
    gc.collect()
    assert all(r() is not None for r in read)
    del decoder


@pytest.mark.gpu
def test_decode_after_a_step_gives_what_it_gave_before(gpu, tmp_path):
    from tierstream_amd import moe
    s = moe.Shape(layers=2, experts=8, top_k=2, d_model=128, d_ff=128, vocab=96)
    m = moe.Model(s, seed=6)
    d = moe.Decoder(m, m.write(tmp_path / "experts.bin"))
    try:
        before = []
        for t in range(12):
            d.token(t)
            before.append(d.logits.clone())
        tokens = torch.arange(64, device="cuda")
        for _ in range(2):
            m.step(tokens, (tokens + 1) % s.vocab, 0.5)
        others = [torch.full((s.vocab, s.d_model), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(64)]  # what was freed is used
        for t in range(12):
            d.token(t)
            assert torch.equal(d.logits, before[t]), t
        assert not torch.equal(m.forward(tokens[:1])[0], before[0])
        del others
    finally:
        d.close()

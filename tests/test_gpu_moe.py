"""The routed layers of tierstream_amd.moe: the gradient step against autograd of the same formulas in 64 bits, and decode from
a device-gated context against the same weights resident."""
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe(gpu):
    from tierstream_amd import moe
    return moe


def test_step_follows_the_gradient(moe):
    """rate x gradient (over its length, where that is above 1) is what the step takes off the 32-bit weights. 64-bit autograd uses the operators' own choice of experts;
    16-bit rounding of activations and their gradients (2^-9 each, a few in a row) stays below 3e-2 of each gradient's norm."""
    s = moe.Shape(layers=2, experts=6, top_k=2, d_model=64, d_ff=96, vocab=48)
    m = moe.Model(s, seed=3)
    tokens = torch.arange(40, device="cuda") % 31
    targets = (tokens * 7 + 1) % s.vocab
    kept = m.forward(tokens)[2]
    w = {k: v.double().requires_grad_() for k, v in m.w.items()}
    x = m.embedding[tokens].double()
    for L in range(s.layers):
        ids = kept[L][2].long()
        weights = torch.softmax((x @ w[f"router{L}"].T).gather(1, ids), 1)
        add = torch.zeros_like(x)
        for j in range(s.top_k):
            gate, up, down = (w[f"{p}{L}"][ids[:, j]] for p in ("gate", "up", "down"))
            h = torch.nn.functional.silu((gate * x[:, None]).sum(2)) * (up * x[:, None]).sum(2)
            add = add + weights[:, j:j + 1] * (down * h[:, None]).sum(2)
        x = x + add
    loss = torch.nn.functional.cross_entropy(x @ w["head"].T, targets)
    loss.backward()
    before = {k: v.clone() for k, v in m.master.items()}
    got = m.step(tokens, targets, 0.5)
    long = max(1.0, float(sum(t.grad.square().sum() for t in w.values()).sqrt()))
    assert abs(got - float(loss.detach())) < 3e-2 * float(loss.detach())
    for name, t in w.items():
        grad = (before[name] - m.master[name]).double() / 0.5
        assert float((grad - t.grad / long).norm()) <= 3e-2 * float(t.grad.norm()) / long, name


def test_decode_from_the_arena_equals_resident_weights(moe, tmp_path):
    s = moe.Shape(layers=3, experts=8, top_k=2, d_model=128, d_ff=256, vocab=96)
    m = moe.Model(s, seed=5)
    want = [m.forward(torch.tensor([t], device="cuda")) for t in range(24)]
    torch.cuda.synchronize()
    d = moe.Decoder(m, m.write(tmp_path / "experts.bin"))
    try:
        for t, (logits, top, kept) in enumerate(want):
            got = d.token(t)
            assert torch.equal(d.logits, logits) and torch.equal(d.x[-1], top), t
            assert all(torch.equal(a, k[2]) for a, k in zip(d.ids, kept)) and got == int(logits.argmax())
        stats = d.ctx.dg_stats()
        assert stats["fetched"] > 0 and stats["evicted"] > 0 and d.ctx.verify_failures() == 0
    finally:
        d.close()


def test_command_learns_and_decodes(moe, capsys):
    moe.main(["--layers", "2", "--experts", "8", "--d-model", "128", "--d-ff", "128", "--vocab", "64", "--steps", "40", "--tokens", "16"])
    lines = capsys.readouterr().out.splitlines()
    losses = [float(line.split()[-1]) for line in lines[:-1]]
    assert losses[-1] < losses[0] / 2 and "failed checks 0" in lines[-1]

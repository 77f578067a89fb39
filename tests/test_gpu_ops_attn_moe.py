"""The routed layers of tierstream_amd.moe with attention before them: the gradient step against autograd of the same formulas in 64
bits, and decode through the 4-bit cache, a token a captured graph, against those formulas over what the cache holds."""
import gc
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def moe(gpu):
    from tierstream_amd import moe
    yield moe
    gc.collect()              # graphs and tensors go now, not in the middle of another module's token,
    torch.cuda.synchronize()  # and the null stream is idle: streams of a device-gated context wait for what it still has


def turned(x, positions, turns):
    """[rows][heads][dim], halves as pairs."""
    angle = (positions.double()[:, None] * turns.cuda() * 2 * math.pi)[:, None]
    a, b = x.chunk(2, -1)
    return torch.cat([a * torch.cos(angle) - b * torch.sin(angle), a * torch.sin(angle) + b * torch.cos(angle)], -1)


def attended(s, x, qkv, mix, positions, lengths, turns):
    rows = (x @ qkv.T).view(len(x), -1, s.head_dim)
    q, k, v = rows.split([s.heads, s.kv_heads, s.kv_heads], 1)
    q, k = turned(q, positions, turns), turned(k, positions, turns)
    k, v = (t.repeat_interleave(s.heads // s.kv_heads, 1) for t in (k, v))
    outs, at = [], 0
    for n in lengths:
        i = slice(at, at + n)
        scores = torch.einsum("qhd,khd->hqk", q[i], k[i]) * s.head_dim ** -0.5
        scores = scores.masked_fill(torch.ones((n, n), dtype=torch.bool, device="cuda").triu(1), -math.inf)
        outs.append(torch.einsum("hqk,khd->qhd", torch.softmax(scores, -1), v[i]))
        at += n
    return x + torch.cat(outs).reshape(len(x), -1) @ mix.T


def test_step_follows_the_gradient(moe):
    """As without attention: 16-bit rounding of activations and their gradients (2^-9 each, some more in a row) stays below 4e-2 of each
    gradient's norm. 64-bit autograd uses the operators' own choice of experts."""
    s = moe.Shape(layers=2, experts=6, top_k=2, d_model=64, d_ff=96, vocab=48, heads=4, kv_heads=2, head_dim=32)
    m, lengths = moe.Model(s, seed=3), [17, 1, 22]
    tokens = torch.arange(40, device="cuda") * 5 % 31
    targets = (tokens * 7 + 1) % s.vocab
    packed = moe.Packed(40, lengths)
    kept = m.forward(tokens, packed)[2]
    turns = torch.tensor(list(m.rotary.s.turns)[:16], dtype=torch.float64)
    w = {k: v.double().requires_grad_() for k, v in m.w.items()}
    x = m.embedding[tokens].double()
    for L in range(s.layers):
        x = attended(s, x, w[f"qkv{L}"], w[f"mix{L}"], packed.positions, lengths, turns)
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
    got = m.step(tokens, targets, 0.5, lengths)
    long = max(1.0, float(sum(t.grad.square().sum() for t in w.values()).sqrt()))
    assert abs(got - float(loss.detach())) < 4e-2 * float(loss.detach())
    for name, t in w.items():
        grad = (before[name] - m.master[name]).double() / 0.5
        assert float((grad - t.grad / long).norm()) <= 4e-2 * float(t.grad.norm()) / long, name


def test_decode_attends_to_what_its_cache_holds(moe, tmp_path):
    """Every layer's output of attention, from its input and the keys and values that the cache gives back: a product's rounding of
    queries, one of the output and one of the sum to bf16, 2^-9 each, stay below 1e-2. Then from the first token again."""
    from tierstream_amd import attn
    s = moe.Shape(layers=2, experts=8, top_k=2, d_model=128, d_ff=256, vocab=96, heads=4, kv_heads=2, head_dim=32)
    m = moe.Model(s, seed=5)
    turns = torch.tensor(list(m.rotary.s.turns)[:16], dtype=torch.float64)
    d = moe.Decoder(m, m.write(tmp_path / "experts.bin"), context=128)
    try:
        firsts = []
        for again in range(2):
            for t in range(70):
                got = d.token(t * 3 % s.vocab)
                torch.cuda.synchronize()
                assert int(d.length) == t + 1 and got == int(d.logits.argmax())
                if t in (0, 1, 40, 63, 64, 69):
                    rows = torch.arange(t + 1, device="cuda")
                    slots = (d.table[0].long()[rows // 64] * 64 + rows % 64).to(torch.int32)
                    for L in range(s.layers):
                        k, v = (torch.empty((t + 1, s.kv_heads, s.head_dim), dtype=torch.bfloat16, device="cuda") for _ in range(2))
                        attn.load(d.caches[L], slots, k, v, stream=torch.cuda.current_stream().cuda_stream)
                        x = d.x[L].double()
                        q = (x @ m.w[f"qkv{L}"].double().T).view(1, -1, s.head_dim)[:, :s.heads]
                        q = turned(q, torch.tensor([t], device="cuda"), turns)
                        kk, vv = (z.double().repeat_interleave(2, 1) for z in (k, v))
                        p = torch.softmax(torch.einsum("qhd,khd->hqk", q, kk) * s.head_dim ** -0.5, -1)
                        want = x + torch.einsum("hqk,khd->qhd", p, vv).reshape(1, -1) @ m.w[f"mix{L}"].double().T
                        assert float((d.mid[L].double() - want).norm()) <= 1e-2 * float(want.norm()), (again, t, L)
                if t == 5:
                    firsts.append(d.logits.clone())
            d.forget()
            torch.cuda.synchronize()
            assert int(d.length) == 0 and int(d.n_free) == 2
        assert torch.equal(*firsts)
        for t in range(128):
            d.token(t % s.vocab)
        with pytest.raises(RuntimeError, match="no place"):
            d.token(1)
        d.forget()
        d.token(1)
        assert d.ctx.verify_failures() == 0
    finally:
        d.close()


def test_work_left_on_the_null_stream(moe, tmp_path):
    """A token begins behind what its caller left there, however long that takes."""
    s = moe.Shape(layers=2, experts=8, top_k=2, d_model=128, d_ff=128, vocab=64, heads=4, kv_heads=2, head_dim=32)
    d = moe.Decoder(moe.Model(s, seed=6), moe.Model(s, seed=6).write(tmp_path / "experts.bin"), context=64)
    try:
        want = [d.token(3 * t % s.vocab) for t in range(8)]
        d.forget()
        x = torch.randn((2048, 2048), device="cuda")
        for t in range(8):
            for _ in range(20):
                x = torch.tanh(x @ x)
            assert d.token(3 * t % s.vocab) == want[t]
        assert bool(torch.isfinite(x).all()) and d.ctx.verify_failures() == 0
    finally:
        d.close()


def test_command_runs_with_attention(moe, capsys):
    moe.main(["--layers", "2", "--experts", "8", "--d-model", "128", "--d-ff", "128", "--vocab", "64", "--steps", "3", "--tokens", "16", "--heads", "4"])
    assert "failed checks 0" in capsys.readouterr().out.splitlines()[-1]


def test_sequences_are_the_rows(moe):
    with pytest.raises(ValueError, match="lengths"):
        moe.Packed(5, [2, 2])

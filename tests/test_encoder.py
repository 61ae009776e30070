"""The query encoder: its gradients against autograd in 64 bits, and its training against a fixed index (needs a B200)."""
import pytest

pytestmark = pytest.mark.gpu


def test_encoder_gradients_match_autograd_in_64_bits():
    """forward and backward of a float32 encoder; every sum has fewer than 2^10 terms of size about 1, so float32
    leaves 2^-24 * 2^10 of the largest magnitudes, far below the 1e-4 asked."""
    import torch

    from trident_b200.encoder import QueryEncoder

    enc = QueryEncoder(50, 24, seed=3)
    gen = torch.Generator(device="cuda").manual_seed(4)
    enc.weight += 0.2 * torch.randn(24, generator=gen, device="cuda")
    tokens = torch.randint(-1, 50, (40, 7), generator=gen, device="cuda")
    tokens[3] = -1  # a query without tokens
    grad = torch.randn((40, 24), generator=gen, device="cuda")
    q = enc.forward(tokens)
    got = enc.backward(grad)

    table, weight, bias = (t.double().requires_grad_() for t in (enc.table, enc.weight, enc.bias))
    x = torch.where((tokens >= 0)[:, :, None], table[tokens.clamp(min=0)], 0.0) * enc.scale
    y = torch.nn.functional.layer_norm(x, (24,), weight, bias, enc.eps)
    share = (tokens >= 0).double()
    share = share / share.sum(1, keepdim=True).clamp(min=1)
    want_q = (share[:, :, None] * y).sum(1)
    want = torch.autograd.grad((want_q * grad).sum(), (table, weight, bias))
    assert bool((q[3] == 0).all())
    for g, w in ((q, want_q), *zip(got, want)):
        assert float((g - w).abs().max()) <= 1e-4 * float(w.abs().max())


@pytest.mark.parametrize("state_bits", [32, 8])
def test_training_finds_the_documents(state_bits):
    """From chance (10 of 2,000 documents) to most queries; the same seeds give the same losses."""
    from trident_b200.encoder import train

    kw = dict(docs=2000, vocab=300, dim=64, steps=60, batch=256, nlist=16, nprobe=8, state_bits=state_bits)
    res = train(**kw)
    assert res["recall_before"] < 0.1
    assert res["recall_after"] > 0.6
    assert res["losses"][-1] < 0.7 * res["losses"][0]


def test_a_step_repeats_bit_for_bit():
    import torch

    from trident_b200 import AdamW
    from trident_b200.encoder import QueryEncoder

    ends = []
    for _ in range(2):
        enc = QueryEncoder(200, 32, seed=1, dtype=torch.bfloat16)
        opt = AdamW(enc.parameters, state_bits=8, master=True)
        gen = torch.Generator(device="cuda").manual_seed(5)
        for _ in range(3):
            tokens = torch.randint(-1, 200, (500, 9), generator=gen, device="cuda")
            q = enc.forward(tokens)
            opt.step(enc.backward(q - 1.0))
        ends.append([p.clone() for p in enc.parameters])
    assert all(torch.equal(a, b) for a, b in zip(*ends))

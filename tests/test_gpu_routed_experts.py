"""The operators together: a routed layer's passes against 64 bits, captured, and the example that trains a block.

Each result passes at most seven roundings to bf16 (rows of gate, up, activation, down, their gradients), each 2^-8 of what it
rounds; a result that is a sum of many such terms lies within 7 x 2^-8 of its norm."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BF16, F32 = torch.bfloat16, torch.float32
BOUND = 7 * 2.0 ** -8


def layer(seed, experts, expert_hidden, hidden):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[-1] ** -0.5).to(BF16)  # noqa: E731
    return normal(experts, expert_hidden, hidden), normal(experts, expert_hidden, hidden), normal(experts, hidden, expert_hidden)


def batch(seed, tokens, experts, top_k, hidden):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(BF16)
    ids = (torch.randn(tokens, experts, generator=g, device="cuda") - torch.arange(experts, device="cuda") * 0.2).topk(top_k, 1).indices
    weights = torch.rand(tokens, top_k, generator=g, device="cuda") + 0.2
    return x, ids.to(torch.int32), weights, torch.randn(tokens, hidden, generator=g, device="cuda").to(BF16)


def reference(kind, w1, w3, w2, x, ids, weights, d_out):
    """Output and gradients in 64 bits, by torch's own differentiation of the definition."""
    leaves = [t.double().requires_grad_() for t in (x, weights, w1, w3, w2)]
    x, weights, w1, w3, w2 = leaves
    gate = torch.einsum("td,trid->tri", x, w1[ids.long()])
    up = torch.einsum("td,trid->tri", x, w3[ids.long()])
    if kind == "swiglu":
        act = gate * torch.sigmoid(gate) * up
    else:
        act = 4 * torch.tanh(gate / 4) * torch.sigmoid(gate) * 25 * torch.tanh(up / 25)
    out = torch.einsum("tri,trdi,tr->td", act, w2[ids.long()], weights)
    (out * d_out.double()).sum().backward()
    return out.detach(), grouped.ExpertGradients(*(t.grad for t in leaves))


def near(got, want, name):
    rel = float((got.double() - want).norm() / want.norm().clamp(min=1e-30))
    assert rel <= BOUND, (name, rel)


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
@pytest.mark.parametrize("tokens,experts,top_k,expert_hidden,hidden", [(1, 8, 2, 64, 96), (37, 16, 4, 40, 72), (500, 8, 3, 128, 136), (24, 6, 2, 7, 40)])
def test_against_64_bits(kind, tokens, experts, top_k, expert_hidden, hidden):
    w = layer(tokens, experts, expert_hidden, hidden)
    x, ids, weights, d_out = batch(tokens + 1, tokens, experts, top_k, hidden)
    call = grouped.RoutedExperts(*w, top_k, activation=kind)
    out, saved = call.forward(x, ids, weights)
    got = call.backward(d_out, saved)
    want_out, want = reference(kind, *w, x, ids, weights, d_out)
    near(out, want_out, "out")
    for name, a, b in zip(got._fields, got, want):
        assert a.shape == b.shape
        near(a, b, name)
    assert ops.k3_moe_device_status() == 0


def test_captured_and_replayed_with_other_routes():
    w = layer(3, 8, 64, 128)
    call = grouped.RoutedExperts(*w, 2)
    x, ids, weights, d_out = batch(4, 60, 8, 2, 128)

    def both():
        out, saved = call.forward(x, ids, weights)
        return (out, *call.backward(d_out, saved))
    both()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    big = batch(5, 900, 8, 2, 128)                                          # larger workspaces in between
    call.backward(big[3], call.forward(*big[:3])[1])
    for old, new in zip((x, ids, weights, d_out), batch(6, 60, 8, 2, 128)):
        old.copy_(new)
    graph.replay()
    for a, b in zip(out, both()):
        assert torch.equal(a, b)


def test_no_tokens():
    w = layer(7, 4, 16, 24)
    call = grouped.RoutedExperts(*w, 2)
    x, ids, weights = (torch.empty(0, n, dtype=d, device="cuda") for n, d in ((24, BF16), (2, torch.int32), (2, F32)))
    out, saved = call.forward(x, ids, weights)
    got = call.backward(x, saved)
    assert out.shape == got.x.shape == (0, 24) and got.weights.shape == (0, 2)
    assert got.w1.shape == w[0].shape and not got.w1.any() and not got.w3.any() and not got.w2.any()


def test_refusals():
    w1, w3, w2 = layer(8, 4, 16, 24)
    with pytest.raises(ValueError, match="w1, w3 and w2: expected"):
        grouped.RoutedExperts(w1, w3, w1, 2)
    for top_k in (0, 5):
        with pytest.raises(ValueError, match="top_k: 1 to 4"):
            grouped.RoutedExperts(w1, w3, w2, top_k)
    with pytest.raises(ValueError, match="w1: expected a multiple of 8 columns"):
        grouped.RoutedExperts(*layer(8, 6, 7, 33), 2)                       # k3_moe_combine takes no such rows
    call = grouped.RoutedExperts(w1, w3, w2, 2)
    x, ids, weights, d_out = batch(9, 5, 4, 2, 24)
    with pytest.raises(ValueError, match=r"ids: expected torch.int32 \[5, 2\]"):
        call.forward(x, ids.long(), weights)
    with pytest.raises(ValueError, match=r"weights: expected torch.float32 \[5, 2\]"):
        call.forward(x, ids, weights[:4])
    _, saved = call.forward(x, ids, weights)
    with pytest.raises(ValueError, match="d_out: expected 5 tokens, got 4"):
        call.backward(d_out[:4], saved)


def example():
    spec = importlib.util.spec_from_file_location("train_experts", os.path.join(ROOT, "examples", "train_experts.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_runs():
    losses = example().main(steps=3, tokens=200, quiet=True)
    assert len(losses) == 3 and all(torch.isfinite(torch.tensor(losses)))


def test_the_examples_gradients():
    """Those of the whole block against torch's, in 64 bits, for the routes that the block took."""
    m = example()
    block = m.RoutedBlock(5)
    g = torch.Generator(device="cuda").manual_seed(6)
    x, residual, d_routed, d_sum = (torch.randn(120, m.HIDDEN, generator=g, device="cuda").to(BF16) for _ in range(4))
    routed, kept = block.forward(x, residual)
    gradients, dx = block.backward(d_routed, d_sum, kept)
    normed, logits, ids, _ = kept
    leaves = {name: t.double().requires_grad_() for name, t in block.read.items()}
    s = normed.sum.double().requires_grad_()
    y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + block.norm.epsilon) * leaves["norm"]
    scores = torch.sigmoid(y @ leaves["router"].t())
    chosen = scores.gather(1, ids.long())
    weights = chosen / (1e-20 + chosen.sum(1, keepdim=True))
    gate, up = (torch.einsum("td,trid->tri", y, leaves[n][ids.long()]) for n in ("w1", "w3"))
    out = torch.einsum("tri,trdi,tr->td", gate * torch.sigmoid(gate) * up, leaves["w2"][ids.long()], weights)
    counts = torch.bincount(ids.reshape(-1), minlength=m.EXPERTS).double()
    share = counts * m.EXPERTS / (m.TOP_K * x.shape[0])
    balance = m.BALANCE * (share * (scores / scores.sum(1, keepdim=True)).mean(0)).sum()
    near(routed, out.detach(), "routed")
    ((out * d_routed.double()).sum() + (s * d_sum.double()).sum() + balance).backward()
    near(dx, s.grad, "dx")
    for name, got in gradients.items():
        near(got, leaves[name].grad, name)

"""Routed experts where some ids are no expert's: such a route has no row."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, I32 = torch.bfloat16, torch.int32


def layer(seed, experts, expert_hidden, hidden):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: (torch.randn(*s, generator=g, device="cuda") * s[-1] ** -0.5).to(BF16)  # noqa: E731
    return normal(experts, expert_hidden, hidden), normal(experts, expert_hidden, hidden), normal(experts, hidden, expert_hidden)


@pytest.mark.parametrize("tokens", [1, 5, 200, 3000])
def test_an_id_that_is_no_experts_adds_nothing(tokens):
    """Against the same call with an expert in its place whose matrices are zeros: the same bits, and the status word says so."""
    experts, top_k, hidden = 6, 3, 40
    w1, w3, w2 = layer(tokens, experts + 1, 24, hidden)
    for w in (w1, w3, w2):
        w[experts] = 0
    call = grouped.RoutedExperts(w1, w3, w2, top_k)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x, d_out = (torch.randn(tokens, hidden, generator=g, device="cuda").to(BF16) for _ in range(2))
    ids = torch.rand(tokens, experts, generator=g, device="cuda").topk(top_k, 1).indices.to(I32)
    weights = torch.rand(tokens, top_k, generator=g, device="cuda") + 0.2
    ids[0] = torch.tensor([experts + 1, -1, 2 ** 31 - 1], dtype=I32)              # a token without any row
    ids[tokens // 2, 1], ids[tokens - 1, 2] = experts + 1, -5
    bad = (ids < 0) | (ids > experts)
    of_zeros = torch.where(bad, experts, ids)
    weights[bad] = float("inf")                                             # what belongs to no row enters nothing
    want, saved = call.forward(x, of_zeros, torch.where(bad, 1.0, weights))
    want_back = call.backward(d_out, saved)
    assert ops.k3_moe_device_status_clear()
    try:
        got, saved = call.forward(x, ids, weights)
        back = call.backward(d_out, saved)
        assert ops.k3_moe_device_status() & 2
    finally:
        assert ops.k3_moe_device_status_clear()
    assert torch.equal(got, want) and torch.equal(back.x, want_back.x)
    assert not got[0].any() and not back.x[0].any()
    assert torch.equal(back.weights, want_back.weights) and not back.weights[bad].any()
    for a, b in ((back.w1, want_back.w1), (back.w3, want_back.w3), (back.w2, want_back.w2)):
        assert torch.equal(a[:experts], b[:experts]) and not a[experts].any()


def test_the_weighted_sum_passes_over_a_route_without_a_row():
    tokens, top_k, hidden, none = 3, 4, 16, -1
    g = torch.Generator(device="cuda").manual_seed(2)
    rows = torch.randn(tokens * top_k, hidden, generator=g, device="cuda").to(BF16)
    weights = torch.rand(tokens, top_k, generator=g, device="cuda")
    index = torch.randperm(tokens * top_k, generator=g, device="cuda").to(I32)
    index[1], index[8:] = none, none
    weights.view(-1)[1], weights[2, 0] = float("nan"), float("inf")
    out = torch.empty(tokens, hidden, dtype=BF16, device="cuda")
    assert ops.k3_moe_combine(out, rows, index, weights, None, tokens, top_k, hidden)
    want = torch.zeros(tokens, hidden, device="cuda")
    for t in range(tokens):
        for r in range(top_k):
            if int(index[t * top_k + r]) != none:
                want[t] = torch.addcmul(want[t], weights[t, r], rows[int(index[t * top_k + r])].float())
    assert float((out.float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max()) and not out[2].any()

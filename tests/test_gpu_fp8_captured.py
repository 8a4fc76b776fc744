"""A captured call of the E4M3 and balance forms, replayed after its object has served larger calls."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import balance, fp8        # noqa: E402


def table(g, rows, columns, *lead):
    codes, scales = fp8.quantize_blocks(torch.randn(rows, columns, generator=g, device="cuda", dtype=torch.bfloat16) * 0.05)
    return (codes.expand(*lead, *codes.shape).contiguous(), scales.expand(*lead, *scales.shape).contiguous()) if lead else (codes, scales)


def calls(g):
    """(name, call of some tokens, tokens of the graph, tokens of the larger call)"""
    linear = fp8.Fp8Linear(*table(g, 300, 520), 300, 520)
    gradient = fp8.Fp8LinearGradient(*table(g, 520, 300), 300, 520)
    experts = fp8.Fp8Experts(*table(g, 128, 256, 8), *table(g, 128, 256, 8), *table(g, 256, 128, 8), top_k=2)
    router = balance.RouterBalance(96, 4)

    def inputs(tokens):
        x = lambda n, scale=1.0: (torch.randn(tokens, n, generator=g, device="cuda") * scale).to(torch.bfloat16)  # noqa: E731
        ids = lambda n, k: torch.rand(tokens, n, generator=g, device="cuda").topk(k, 1).indices.to(torch.int32)  # noqa: E731
        return {"linear": (x(520),), "by_input": (x(300, 1e-3),), "by_weight": (x(300, 1e-3), x(520)),
                "experts": (x(256), ids(8, 2), torch.rand(tokens, 2, generator=g, device="cuda")),
                "balance": (torch.randn(tokens, 96, generator=g, device="cuda"), ids(96, 4))}
    forms = {"linear": linear.forward, "by_input": gradient.by_input, "by_weight": gradient.by_weight, "experts": experts.forward,
             "balance": router.forward}
    return forms, inputs


@pytest.mark.parametrize("name", ["linear", "by_input", "by_weight", "experts", "balance"])
def test_replay_after_a_larger_call(name):
    g = torch.Generator(device="cuda").manual_seed(1)
    forms, inputs = calls(g)
    call, args = forms[name], inputs(600)[name]
    as_list = lambda out: [t.clone() for t in out] if isinstance(out, tuple) else [out.clone()]  # noqa: E731
    want = as_list(call(*args))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(*args)
    large = inputs(5000)[name]
    want_large = as_list(call(*large))                                      # the object takes a larger workspace
    # memory that the allocator hands out now, of all sizes that an old workspace could be cut into
    others = [torch.full((n,), 77, dtype=torch.uint8, device="cuda") for n in [1 << 12, 1 << 16, 1 << 18, 1 << 20, 3 << 20, 1 << 22] * 8]
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    for got, w in zip(out if isinstance(out, tuple) else (out,), want):
        assert torch.equal(got, w)
    assert all(bool((t == 77).all()) for t in others)
    for got, w in zip(as_list(call(*large)), want_large):
        assert torch.equal(got, w)

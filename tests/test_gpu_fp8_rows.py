"""The expert rows behind the weighted sum: as exact for many tokens as for few."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8                 # noqa: E402
from tests import fp8_reference as R           # noqa: E402

# Of the norm: the output's rounding to bf16, uniform within half a unit of 2^-7, is 2^-8 / sqrt(3) = 2.26e-3 of a
# binade's start, and 1.53e-3 of values whose mantissas m have the density 1 / m (mean square 2.16); activations that
# fall on the other side between two codes than in 64 bits, a part in 1e4 by 2^-4 of their value: 6e-4.  Together 1.65e-3.
# Rows rounded to bf16 before their sum would add 1.53e-3 once more: 2.25e-3.
LIMIT = 1.95e-3


@pytest.mark.parametrize("kind", ["swiglu", "situ"])
@pytest.mark.parametrize("tokens,experts,top_k", [(40, 4, 2), (300, 4, 2), (700, 3, 1), (1000, 8, 8)])
def test_rows_are_not_rounded_before_their_sum(tokens, experts, top_k, kind):
    hidden, expert_hidden = 640, 256
    g = torch.Generator().manual_seed(tokens)
    tables = []
    for r, c in ((expert_hidden, hidden), (expert_hidden, hidden), (hidden, expert_hidden)):
        per = [fp8.quantize_blocks((torch.randn(r, c, generator=g) * 1.5 * c ** -0.5).cuda()) for _ in range(experts)]
        tables.append((torch.stack([p[0] for p in per]), torch.stack([p[1] for p in per])))
    x = torch.randn(tokens, hidden, generator=g).to(torch.bfloat16)
    ids = torch.rand(tokens, experts, generator=g).topk(top_k, 1).indices.to(torch.int32)
    weights = torch.rand(tokens, top_k, generator=g) + 0.1
    layer = fp8.Fp8Experts(*tables[0], *tables[1], *tables[2], top_k=top_k, activation=kind)
    out = layer.forward(x.cuda(), ids.cuda(), weights.cuda()).cpu().double()
    want = R.experts(x, ids, weights, [(c.cpu(), s.cpu()) for c, s in tables], kind)
    assert float((out - want).norm() / want.norm()) <= LIMIT

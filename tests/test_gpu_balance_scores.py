"""Scores, and the gradient where they are nearly certain, against 64 bits: over the whole range of finite logits,
relative to each value."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import balance             # noqa: E402


def means_of_single_tokens(logits, kind):
    """Each token a sequence of its own: its scores over their total."""
    tokens, experts = logits.shape
    ids = torch.zeros(tokens, 1, dtype=torch.int32, device="cuda")
    offsets = torch.arange(tokens + 1, dtype=torch.int32, device="cuda")
    return balance.RouterBalance(experts, 1, kind).forward(logits.cuda(), ids, offsets)[2].cpu().double()


# The exponential is within 2^-22 of itself, the reciprocal within 2^-23, and with the sums and products around them a
# score lies within 6e-7; a mean is a score over a sum of such.
SCORE = 6e-7
# few tokens go through one launch, others through two; rows of 16-byte units and others
SHAPES = [(40, 128), (50, 77), (700, 256), (600, 129)]


@pytest.mark.parametrize("tokens,experts", SHAPES)
def test_sigmoid_scores_of_any_size(tokens, experts):
    g = torch.Generator().manual_seed(tokens)
    logits = torch.rand(tokens, experts, generator=g) * 110 - 80
    p = torch.sigmoid(logits.double())
    want = p / (1e-20 + p.sum(1, keepdim=True))
    assert float(p.min()) < 1e-33
    assert bool(((means_of_single_tokens(logits, "sigmoid") - want).abs() <= (2 * SCORE + experts ** 0.5 * 2.0 ** -24) * want).all())


@pytest.mark.parametrize("tokens,experts", SHAPES)
def test_softmax_scores_of_any_size(tokens, experts):
    """Logits on a grid of 1/64, so that their differences are exact (elsewhere they are f32 differences)."""
    g = torch.Generator().manual_seed(tokens + 1)
    logits = torch.floor(torch.rand(tokens, experts, generator=g) * 80 * 64) / 64 - 75
    want = torch.softmax(logits.double(), 1)
    assert float(want.min()) < 1e-33
    assert bool(((means_of_single_tokens(logits, "softmax") - want).abs() <= (2 * SCORE + experts ** 0.5 * 2.0 ** -24) * want).all())

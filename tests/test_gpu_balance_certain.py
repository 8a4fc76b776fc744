"""The router's gradient where scores are nearly certain or the weights' gradients cancel, against 64 bits and
relative to what is left."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import balance             # noqa: E402

TINY, ALPHA, SCALE = 1e-20, 1e-2, 2.5
# A score and a derivative lie within 6e-7, a sum of chosen scores and its reciprocal within 8e-7, which enters twice;
# the products around them add 2^-24 each.
LIMIT = 6e-6


def cuda(*tensors):
    return [t.cuda() for t in tensors]


@pytest.mark.parametrize("experts", [64, 129])
def test_weights_gradient_of_large_logits(experts):
    """Both chosen logits between 8 and 30, where 1 - s is 3e-4 to 1e-13."""
    tokens, g = 300, torch.Generator().manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g)
    ids = torch.rand(tokens, experts, generator=g).topk(2, 1).indices.to(torch.int32)
    logits.scatter_(1, ids.long(), torch.rand(tokens, 2, generator=g) * 22 + 8)
    sizes = torch.rand(tokens, 2, generator=g) + 0.5
    d_weights = sizes * torch.tensor([1.0, -1.0])                           # their difference does not cancel
    router = balance.RouterBalance(experts, 2, "sigmoid", ALPHA, SCALE)
    got = router.backward(*cuda(logits, ids), d_weights=d_weights.cuda()).cpu().double()
    x, w = logits.double().gather(1, ids.long()), d_weights.double()
    s = torch.sigmoid(x)
    d = TINY + s.sum(1, keepdim=True)
    want = SCALE * (w - (w * s).sum(1, keepdim=True) / d) / d * s * torch.sigmoid(-x)
    off = (got.gather(1, ids.long()) - want).abs()
    assert bool((off <= LIMIT * want.abs()).all())
    assert int((got != 0).sum()) == 2 * tokens                              # and nothing at the others


@pytest.mark.parametrize("top_k", [1, 4])
def test_weights_gradients_that_cancel(top_k):
    """One choice, or equal gradients: w tiny / D^2 of the score is all that is left."""
    tokens, experts, g = 200, 48, torch.Generator().manual_seed(top_k)
    logits = torch.randn(tokens, experts, generator=g) * 3
    ids = torch.rand(tokens, experts, generator=g).topk(top_k, 1).indices.to(torch.int32)
    w = torch.randn(tokens, 1, generator=g)
    router = balance.RouterBalance(experts, top_k, "sigmoid", ALPHA, SCALE)
    got = router.backward(*cuda(logits, ids), d_weights=w.expand(tokens, top_k).contiguous().cuda()).cpu().double()
    s = torch.sigmoid(logits.double()).gather(1, ids.long())
    d = TINY + s.sum(1, keepdim=True)
    want = SCALE * w.double() * TINY / d ** 2 * s * torch.sigmoid(-logits.double()).gather(1, ids.long())
    assert bool(((got.gather(1, ids.long()) - want).abs() <= LIMIT * want.abs()).all())


def test_weights_gradient_of_scores_below_the_tiny_term():
    """Chosen logits of -80 to -60: the weights are s / (tiny + sum), far from normalised."""
    tokens, experts, g = 100, 32, torch.Generator().manual_seed(9)
    logits = torch.randn(tokens, experts, generator=g)
    ids = torch.rand(tokens, experts, generator=g).topk(3, 1).indices.to(torch.int32)
    logits.scatter_(1, ids.long(), torch.rand(tokens, 3, generator=g) * 20 - 80)
    d_weights = torch.rand(tokens, 3, generator=g) + 0.5
    router = balance.RouterBalance(experts, 3, "sigmoid", ALPHA, SCALE)
    got = router.backward(*cuda(logits, ids), d_weights=d_weights.cuda()).cpu().double()
    s, w = torch.sigmoid(logits.double()).gather(1, ids.long()), d_weights.double()
    d = TINY + s.sum(1, keepdim=True)
    want = SCALE * (w - (w * s).sum(1, keepdim=True) / d) / d * s
    assert bool(((got.gather(1, ids.long()) - want).abs() <= LIMIT * want.abs()).all())


def shares(ids, tokens, experts, top_k):
    n = torch.bincount(ids.reshape(-1).long(), minlength=experts)
    return n, n.double() * experts / (top_k * tokens)


def test_loss_gradient_of_large_logits():
    """Some logits between 8 and 30; relative to the terms f and sum f s / Z of the difference."""
    tokens, experts, top_k, g = 400, 96, 4, torch.Generator().manual_seed(5)
    logits = torch.randn(tokens, experts, generator=g)
    large = torch.rand(tokens, experts, generator=g) < 0.1
    logits = torch.where(large, torch.rand(tokens, experts, generator=g) * 22 + 8, logits)
    ids = (logits + torch.randn(tokens, experts, generator=g)).topk(top_k, 1).indices.to(torch.int32)
    router = balance.RouterBalance(experts, top_k, "sigmoid", ALPHA, SCALE)
    counts = router.forward(*cuda(logits, ids))[0]
    got = router.backward(*cuda(logits, ids), counts, d_loss=torch.ones(1, device="cuda")).cpu().double()
    n, f = shares(ids, tokens, experts, top_k)
    assert torch.equal(counts.cpu().long()[0], n)
    s = torch.sigmoid(logits.double())
    z = TINY + s.sum(1, keepdim=True)
    by = ALPHA / tokens / z * s * torch.sigmoid(-logits.double())
    mean = (f * s).sum(1, keepdim=True) / z
    off = (got - by * (f - mean)).abs()
    assert bool((off <= LIMIT * by * (f + mean)).all())


@pytest.mark.parametrize("experts", [48, 200, 1000])
def test_softmax_gradient_of_a_nearly_certain_expert(experts):
    """One logit 12 to 25 above the others: its gradient is the small sum of theirs.  The gradient by a score is a
    share f of counts up to n, with three roundings; two that differ do so by 1 / n of themselves at least."""
    tokens, top_k, g = 300, 4, torch.Generator().manual_seed(experts)
    logits = torch.randn(tokens, experts, generator=g) * 0.5
    logits.scatter_(1, torch.randint(0, experts, (tokens, 1), generator=g), torch.rand(tokens, 1, generator=g) * 13 + 14)
    ids = (logits + 2 * torch.randn(tokens, experts, generator=g)).topk(top_k, 1).indices.to(torch.int32)
    router = balance.RouterBalance(experts, top_k, "softmax", ALPHA, SCALE)
    counts = router.forward(*cuda(logits, ids))[0]
    got = router.backward(*cuda(logits, ids), counts, d_loss=torch.ones(1, device="cuda")).cpu().double()
    n, f = shares(ids, tokens, experts, top_k)
    p = torch.softmax(logits.double(), 1)
    d = ALPHA / tokens * f.expand_as(p)
    top = d.gather(1, p.argmax(1, keepdim=True))
    others = ((d - top).abs() * p).sum(1, keepdim=True)
    off = (got - p * ((d - top) - ((d - top) * p).sum(1, keepdim=True))).abs()
    limit = LIMIT + 2 * 3 * 2.0 ** -24 * int(n.max())
    assert bool((off <= limit * p * ((d - top).abs() + others)).all())

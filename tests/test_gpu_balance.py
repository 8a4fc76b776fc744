"""Counts, balance loss and router gradient against the formulas in 64 bits and against differences of them."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import balance, ops        # noqa: E402

TINY, ALPHA, SCALE = 1e-20, 1e-2, 2.5


def scores(logits, kind):
    if kind == "sigmoid":
        return 1 / (1 + torch.exp(-logits))
    top = logits.amax(1, keepdim=True)
    p = torch.exp(logits - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    return p / p.sum(1, keepdim=True).clamp(min=1e-300)


def count(ids, cuts, experts):
    out = torch.zeros(len(cuts) - 1, experts, dtype=torch.float64)
    for s in range(len(cuts) - 1):
        part = ids[cuts[s]:cuts[s + 1]].reshape(-1).long()
        part = part[(part >= 0) & (part < experts)]
        out[s] = torch.bincount(part, minlength=experts)
    return out


def losses(logits, counts, cuts, top_k, kind):
    """(loss, means) of each sequence; a function of the logits with the counts given."""
    loss, means = [], []
    for s in range(len(cuts) - 1):
        length = cuts[s + 1] - cuts[s]
        if length == 0:
            loss.append(logits.new_zeros(()))
            means.append(logits.new_zeros(logits.shape[1]))
            continue
        p = scores(logits[cuts[s]:cuts[s + 1]], kind)
        if kind == "sigmoid":
            p = p / (TINY + p.sum(1, keepdim=True))
        means.append(p.mean(0))
        loss.append(ALPHA * (counts[s] * (logits.shape[1] / (top_k * length)) * means[-1]).sum())
    return torch.stack(loss), torch.stack(means)


def routing_weights(logits, ids, kind):
    chosen = scores(logits, kind).gather(1, ids.long())
    return SCALE * chosen / (TINY + chosen.sum(1, keepdim=True))


def case(seed, tokens, experts, top_k, sequences):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(tokens, experts, generator=g) * 1.5
    ids = (logits + 0.5 * torch.randn(tokens, experts, generator=g)).topk(top_k, 1).indices.to(torch.int32)
    cuts = [0] + sorted(torch.randint(0, tokens + 1, (sequences - 1,), generator=g).tolist()) + [tokens]
    d_loss = torch.rand(sequences, generator=g) + 0.5
    d_weights = torch.randn(tokens, top_k, generator=g) * 1e-2
    return logits, ids, cuts, d_loss, d_weights


def device(cuts):
    return torch.tensor(cuts, dtype=torch.int32, device="cuda")


def gradient(logits, ids, counts, cuts, d_loss, d_weights, top_k, kind):
    """The formula's gradient, by automatic differentiation in 64 bits."""
    x = logits.double().requires_grad_(True)
    total = (losses(x, counts, cuts, top_k, kind)[0] * d_loss.double()).sum() if d_loss is not None else 0
    if d_weights is not None:
        total = total + (routing_weights(x, ids, kind) * d_weights.double()).sum()
    total.backward()
    return x.grad


# A score is within a few 2^-24 of itself, sums of E scores and of a chunk's tokens within their number's root of
# roundings; 3e-6 covers both at these sizes.  The gradient is a difference of two such terms, so its limit is that
# of the row's larger term: 1e-5 of the row's norm, besides itself.
REL = 3e-6

SHAPES = [(1, 1, 1, 1), (1, 896, 16, 1), (5, 7, 3, 2), (33, 64, 6, 4), (257, 160, 6, 5), (100, 129, 8, 9), (500, 1024, 32, 3),
          (1000, 384, 8, 1), (700, 255, 4, 40), (3000, 896, 16, 7)]


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
@pytest.mark.parametrize("tokens,experts,top_k,sequences", SHAPES)
def test_against_the_formulas(tokens, experts, top_k, sequences, kind):
    logits, ids, cuts, d_loss, d_weights = case(tokens + experts, tokens, experts, top_k, sequences)
    router = balance.RouterBalance(experts, top_k, kind, ALPHA, SCALE)
    dl, di, do = logits.cuda(), ids.cuda(), device(cuts)
    counts, loss, means = router.forward(dl, di, do)
    want_counts = count(ids, cuts, experts)
    want_loss, want_means = losses(logits.double(), want_counts, cuts, top_k, kind)
    assert torch.equal(counts.cpu().double(), want_counts)
    assert bool(((loss.cpu().double() - want_loss).abs() <= REL * want_loss.abs()).all())
    assert bool(((means.cpu().double() - want_means).abs() <= REL * want_means).all())
    assert torch.equal(router.forward(None, di, do), counts)                # counts alone
    for a, b in zip(router.forward(dl, di, do), (counts, loss, means)):
        assert torch.equal(a, b)                                            # the same bits again
    for by_loss, by_weights in ((d_loss, d_weights), (d_loss, None), (None, d_weights)):
        got = router.backward(dl, di, counts, do, *(None if t is None else t.cuda() for t in (by_loss, by_weights)))
        want = gradient(logits, ids, want_counts, cuts, by_loss, by_weights, top_k, kind)
        off = (got.cpu().double() - want).abs()
        # terms that cancel (softmax and normalised weights leave differences): the size they had
        size = 2 * ((0 if by_loss is None else ALPHA * float(by_loss.max()) * experts / max(1, min(b - a for a, b in zip(cuts, cuts[1:]) if b > a)))
                    + (0 if by_weights is None else SCALE * by_weights.abs().double().max(1, keepdim=True).values * 2))
        p = scores(logits.double(), kind)
        chosen = p.gather(1, ids.long()).sum(1, keepdim=True)
        assert bool((off <= 1e-5 * want.abs() + REL * size * p / torch.minimum(chosen, torch.ones(()).double())).all())


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_gradient_against_differences(kind):
    logits, ids, cuts, d_loss, d_weights = case(11, 40, 24, 4, 3)
    router = balance.RouterBalance(24, 4, kind, ALPHA, SCALE)
    counts, _, _ = router.forward(logits.cuda(), ids.cuda(), device(cuts))
    got = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), d_loss.cuda(), d_weights.cuda()).cpu().double()
    c = count(ids, cuts, 24)

    def total(x):
        return float((losses(x, c, cuts, 4, kind)[0] * d_loss.double()).sum()
                     + (routing_weights(x, ids, kind) * d_weights.double()).sum())
    h = 1e-4                                     # the quotient is off by h^2 / 6 of a third derivative, about 1e-9 here
    for seed in range(5):
        d = torch.randn(40, 24, generator=torch.Generator().manual_seed(seed)).double()
        slope = (total(logits.double() + h * d) - total(logits.double() - h * d)) / (2 * h)
        assert abs(float((got * d).sum()) - slope) <= 1e-5 * float((got * d).norm()) + 1e-8


def test_one_sequence_without_offsets():
    logits, ids, _, _, d_weights = case(3, 200, 128, 8, 1)
    router = balance.RouterBalance(128, 8, "sigmoid", ALPHA, SCALE)
    with_offsets = router.forward(logits.cuda(), ids.cuda(), device([0, 200]))
    for a, b in zip(router.forward(logits.cuda(), ids.cuda()), with_offsets):
        assert torch.equal(a, b)


def test_empty_sequences_and_tokens_past_the_last():
    logits, ids, _, _, _ = case(4, 60, 32, 4, 1)
    cuts = [0, 0, 20, 20, 20, 45, 45]            # 15 tokens belong to none
    router = balance.RouterBalance(32, 4, "sigmoid", ALPHA, SCALE)
    counts, loss, means = router.forward(logits.cuda(), ids.cuda(), device(cuts))
    assert torch.equal(counts.cpu().double(), count(ids, cuts, 32))
    for s in (0, 2, 3, 5):
        assert float(loss[s]) == 0 and not means[s].any()
    d = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), torch.ones(6, device="cuda"))
    assert not d[45:].any() and bool(d[:45].any())


@pytest.mark.parametrize("kind", ["sigmoid", "softmax"])
def test_masked_experts_and_rows(kind):
    """Logits of -inf mask an expert, or a whole row; the lowest finite value does too."""
    logits, ids, cuts, d_loss, d_weights = case(5, 50, 40, 4, 2)
    logits[:, 7] = -math.inf
    logits[:, 8] = torch.finfo(torch.float32).min
    logits[9] = -math.inf
    ids = torch.where(ids == 7, 0, ids)
    ids = torch.where(ids == 8, 1, ids)
    router = balance.RouterBalance(40, 4, kind, ALPHA, SCALE)
    counts, loss, means = router.forward(logits.cuda(), ids.cuda(), device(cuts))
    want_loss, want_means = losses(logits.double(), count(ids, cuts, 40), cuts, 4, kind)
    assert bool(((loss.cpu().double() - want_loss).abs() <= REL * want_loss).all())
    assert bool(((means.cpu().double() - want_means).abs() <= REL * want_means).all())
    assert not means[:, 7:9].any()
    d = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), d_loss.cuda()).cpu()
    assert bool(torch.isfinite(d).all()) and not d[:, 7:9].any() and not d[9].any()


def test_a_row_that_is_not_finite_stays_alone():
    logits, ids, cuts, d_loss, d_weights = case(6, 50, 64, 4, 2)
    for kind in ("sigmoid", "softmax"):
        router = balance.RouterBalance(64, 4, kind, ALPHA, SCALE)
        counts, _, _ = router.forward(logits.cuda(), ids.cuda(), device(cuts))
        clean = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), d_loss.cuda(), d_weights.cuda())
        bad = logits.clone()
        bad[20, 3] = math.nan
        got = router.backward(bad.cuda(), ids.cuda(), counts, device(cuts), d_loss.cuda(), d_weights.cuda())
        assert bool(torch.isnan(got[20]).all()) and torch.equal(got[:20], clean[:20]) and torch.equal(got[21:], clean[21:])


def test_ids_that_are_no_expert_or_named_twice():
    logits, ids, cuts, d_loss, d_weights = case(7, 30, 16, 4, 1)
    ids[3, 1], ids[8, 0] = 16, -5
    ids[5, 2] = ids[5, 1]
    router = balance.RouterBalance(16, 4, "sigmoid", ALPHA, SCALE)
    counts, _, _ = router.forward(logits.cuda(), ids.cuda(), device(cuts))
    assert torch.equal(counts.cpu().double(), count(ids, cuts, 16))
    d = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), None, d_weights.cuda())
    assert ops.k3_moe_device_status() & 2
    assert ops.k3_moe_device_status_clear() and ops.k3_moe_device_status() == 0
    # an id that is no expert has the score 0; twice the same is the sum of both
    x = logits.double().requires_grad_(True)
    p = 1 / (1 + torch.exp(-x))
    real = (ids >= 0) & (ids < 16)
    chosen = p.gather(1, torch.where(real, ids, 0).long()) * real
    (SCALE * chosen / (TINY + chosen.sum(1, keepdim=True)) * d_weights.double()).sum().backward()
    assert bool(((d.cpu().double() - x.grad).abs() <= 1e-5 * x.grad.abs() + REL * SCALE * 0.1).all())


def test_unaligned_rows():
    """Logits that start between 16-byte boundaries."""
    logits, ids, cuts, d_loss, d_weights = case(8, 70, 128, 4, 2)
    store = torch.empty(70 * 128 + 1, device="cuda")
    view = store[1:].view(70, 128)
    view.copy_(logits)
    router = balance.RouterBalance(128, 4, "softmax", ALPHA, SCALE)
    counts, loss, means = router.forward(view, ids.cuda(), device(cuts))
    want = router.forward(logits.cuda(), ids.cuda(), device(cuts))
    assert torch.equal(counts, want[0])
    assert bool(((means - want[2]).abs() <= REL * want[2]).all())
    d = router.backward(view, ids.cuda(), counts, device(cuts), d_loss.cuda(), d_weights.cuda())
    e = router.backward(logits.cuda(), ids.cuda(), counts, device(cuts), d_loss.cuda(), d_weights.cuda())
    assert bool(((d - e).abs() <= 1e-5 * e.abs() + 1e-8).all())


def test_logits_of_more_than_four_billion_values():
    """The last tokens of a long batch give what they give alone."""
    tokens, experts, tail = 4_300_001, 1000, 9
    logits, ids, _, d_loss, d_weights = case(12, tail, experts, 2, 1)
    long_logits = torch.zeros(tokens, experts, device="cuda")
    long_ids = torch.zeros(tokens, 2, dtype=torch.int32, device="cuda")
    long_ids[:, 1] = 1
    long_logits[-tail:], long_ids[-tail:] = logits.cuda(), ids.cuda()
    assert long_logits.numel() > 1 << 32
    router = balance.RouterBalance(experts, 2, "sigmoid", ALPHA, SCALE)
    cuts = device([0, tokens - tail, tokens])
    counts, loss, means = router.forward(long_logits, long_ids, cuts)
    alone = router.forward(logits.cuda(), ids.cuda())
    assert torch.equal(counts[1:], alone[0])
    assert bool(((means[1:] - alone[2]).abs() <= REL * alone[2]).all())
    assert counts[0].tolist()[:3] == [tokens - tail, tokens - tail, 0]
    both = torch.cat([torch.ones(1), d_loss]).cuda()
    long_weights = torch.zeros(tokens, 2, device="cuda")
    long_weights[-tail:] = d_weights.cuda()
    d = router.backward(long_logits, long_ids, counts, cuts, both, long_weights)
    e = router.backward(logits.cuda(), ids.cuda(), alone[0], None, d_loss.cuda(), d_weights.cuda())
    assert torch.equal(d[-tail:], e)

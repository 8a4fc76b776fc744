"""Offsets that no dispatch writes: past the rows, descending, overlapping.  Outputs lie between guards, all groups have one
matrix and the values are integers, so that a row has the same bits whichever of its groups writes it."""
import random

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
GUARD = 4096


def integers(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-3, 4, shape, generator=g, device="cuda").to(BF16)


def cuts_of(offsets, rows):
    """The groups' rows: an offset past the rows counts as their number, one below its predecessor ends an empty group."""
    cut = [min(o & 0xffffffff, rows) for o in offsets]
    return [(a, max(a, b)) for a, b in zip(cut, cut[1:])]


def guarded(shape, dtype):
    elements = 1
    for s in shape:
        elements *= s
    buffer = torch.full((elements + 2 * GUARD,), 7.5, dtype=dtype, device="cuda")
    return buffer, buffer[GUARD:GUARD + elements].view(shape)


def guards_stand(buffer):
    return bool((buffer[:GUARD] == 7.5).all()) and bool((buffer[-GUARD:] == 7.5).all())


def run_rows(form, offsets, rows, n, k, dtype):
    depth, wide = (k, n) if form == "forward" else (n, k)
    a, matrix = integers(rows, rows, depth), integers(n + k, n, k)
    product = grouped.GroupedProduct(matrix.expand(len(offsets) - 1, n, k).contiguous())
    buffer, out = guarded((rows, wide), dtype)
    dev = torch.tensor([o if o < 2 ** 31 else o - 2 ** 32 for o in offsets], dtype=torch.int32, device="cuda")
    (product.forward if form == "forward" else product.by_input)(a, dev, out=out)
    torch.cuda.synchronize()
    assert guards_stand(buffer) and ops.k3_moe_device_status() == 0
    want = a.float() @ (matrix.float().t() if form == "forward" else matrix.float())
    return out, want.to(dtype)


FEW = [[0, 50, 300, 2 ** 31, 2 ** 32 - 1], [0, 40, 20, 20, 60], [90, 100, 101, 5, 5], [2 ** 32 - 1] * 5, [100, 70, 40, 10, 0], [30, 20, 60, 10, 15]]


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
@pytest.mark.parametrize("offsets", FEW)
def test_few_groups(form, dtype, n, k, offsets):
    rows = 100
    out, want = run_rows(form, offsets, rows, n, k, dtype)
    covered = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, b in cuts_of(offsets, rows):
        covered[a:b] = True
    assert torch.equal(out[covered], want[covered]) and bool((out[~covered] == 7.5).all())


def many(kind, groups, rows):
    r = random.Random(groups + rows)
    if kind == "saw":                                                       # every second group has all rows
        return [0 if g % 2 == 0 else rows for g in range(groups + 1)]
    if kind == "random":
        return [r.choice([r.randrange(rows + 1), r.randrange(2 ** 32)]) for _ in range(groups + 1)]
    return sorted((r.randrange(rows + 1) for _ in range(groups + 1)), reverse=True)


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("n,k", [(264, 136), (2048, 64), (33, 7)])
@pytest.mark.parametrize("groups,rows", [(200, 100), (200, 5000), (1024, 3000), (129, 129 * 600)])
@pytest.mark.parametrize("kind", ["saw", "random", "falling"])
def test_more_tiles_than_there_is_room_for(form, n, k, groups, rows, kind):
    """A row of several groups, or of one where others overlap, has its result or is left as it was."""
    offsets = many(kind, groups, rows)
    out, want = run_rows(form, offsets, rows, n, k, F32)
    covered = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for a, b in cuts_of(offsets, rows):
        covered[a:b] = True
    assert bool((out[~covered] == 7.5).all())
    assert bool(((out == want) | (out == 7.5)).all())
    if kind == "falling":
        assert not covered.any()
    else:
        assert bool((out[covered] == want[covered]).any())


@pytest.mark.parametrize("n,k", [(264, 136), (33, 7)])
@pytest.mark.parametrize("kind", ["saw", "random", "falling"])
@pytest.mark.parametrize("groups,rows", [(4, 100), (200, 1500), (896, 40)])
def test_by_weight(n, k, kind, groups, rows):
    offsets = many(kind, groups, rows)
    dy, x = integers(1, rows, n), integers(2, rows, k)
    dev = torch.tensor([o if o < 2 ** 31 else o - 2 ** 32 for o in offsets], dtype=torch.int32, device="cuda")
    want = torch.stack([dy[a:b].float().t() @ x[a:b].float() for a, b in cuts_of(offsets, rows)])
    for dtype in (F32, BF16):
        buffer, out = guarded((groups, n, k), dtype)
        grouped.GroupedWeightGradient(groups, n, k).forward(dy, x, dev, out=out)
        torch.cuda.synchronize()
        assert guards_stand(buffer) and ops.k3_moe_device_status() == 0
        assert torch.equal(out, want.to(dtype))


@pytest.mark.parametrize("n,k", [(8, 8), (7, 7)])
def test_more_than_2_to_32_tiles(n, k):
    """512 groups of about 2^29 rows each, which overlap: their tiles' places pass 32 bits."""
    rows = (1 << 29) + (1 << 20)
    r = random.Random(n)
    offsets = [r.randrange(1000) if g % 2 == 0 else rows - r.randrange(1000) for g in range(1025)]
    a, matrix = integers(3, 1 << 20, k).repeat(rows >> 20, 1), integers(4, n, k)
    buffer, out = guarded((rows, n), BF16)
    grouped.GroupedProduct(matrix.expand(1024, n, k).contiguous()).forward(a, torch.tensor(offsets, dtype=torch.int32, device="cuda"), out=out)
    torch.cuda.synchronize()
    assert guards_stand(buffer) and ops.k3_moe_device_status() == 0
    want = (a[:1 << 20].float() @ matrix.float().t()).to(BF16)
    for i in range(rows >> 20):
        part = out[i << 20:(i + 1) << 20]
        inside = torch.ones(1 << 20, dtype=torch.bool, device="cuda")
        if i == 0:
            inside[:offsets[0]] = False                                     # the first group's rows have room for all of their tiles
        if i == (rows >> 20) - 1:
            inside[(1 << 20) - (rows - offsets[1]):] = False
        assert torch.equal(part[inside], want[inside])
        assert bool(((part == want) | (part == 7.5)).all())
    del a, out, buffer
    torch.cuda.empty_cache()

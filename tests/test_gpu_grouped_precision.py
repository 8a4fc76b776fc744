"""How far f32 outputs of the grouped products lie from 64 bits at large depths, in the norm.

Tensor cores: an accumulator takes 32 additions of 16 products (512 of the depth) before it is added to the others.  An addition
cuts off half a unit on average, at most 2^-24 of the sum so far, always towards zero; the sum after i of 32 random additions is
sqrt(i / 32) of the segment's, so a segment loses at most 32 x 2/3 x 2^-24 of itself.  Without segments the same count gives 2.5e-6
at a depth of 2048 and 9e-6 at 7168.

FMA pipes: each of a segment's 512 additions is rounded, 2^-23 / sqrt(12) of the sum so far at most; independent errors make that
sqrt(512 / 2) of it.  One sum over the whole depth would lose sqrt(depth / 2).

Segments are added with rounding in both: sqrt(segments / 2) x 2^-23 / sqrt(12)."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32
ROUNDED = 2.0 ** -23 / math.sqrt(12)


def tensor_core_bound(depth):
    return 32 * 2 / 3 * 2.0 ** -24 + math.sqrt(math.ceil(depth / 512) / 2) * ROUNDED


def fma_bound(depth):
    return (math.sqrt(512 / 2) + math.sqrt(math.ceil(depth / 512) / 2)) * ROUNDED


def normal(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(BF16)


def on_device(offsets):
    return torch.tensor(list(offsets), dtype=torch.int32, device="cuda")


def off(got, want):
    return float((got.double() - want).norm() / want.norm())


def by_rows(form, rows, wide, depth):
    a = normal(depth + rows, rows, depth)
    w = normal(depth, 1, *((wide, depth) if form == "forward" else (depth, wide)))
    call = grouped.GroupedProduct(w)
    got = (call.forward if form == "forward" else call.by_input)(a, on_device([0, rows]), dtype=F32)
    return off(got, a.double() @ (w[0].double().t() if form == "forward" else w[0].double()))


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("rows,wide", [(8, 264), (300, 520), (2500, 2048), (2500, 520)])
@pytest.mark.parametrize("depth", [2048, 7168, 16392])
def test_tensor_cores_by_rows(form, rows, wide, depth):
    # (8 rows: parts of the depth in a cluster; the others: one block or a pair per item)
    assert by_rows(form, rows, wide, depth) <= tensor_core_bound(depth)


@pytest.mark.parametrize("form", ["forward", "by_input"])
@pytest.mark.parametrize("depth", [2049, 7169, 16387])
def test_fma_pipes_by_rows(form, depth):
    assert by_rows(form, 40, 130, depth) <= fma_bound(depth)


def by_weight(n, k, sizes):
    offsets = [0]
    for size in sizes:
        offsets.append(offsets[-1] + size)
    dy, x = normal(n, offsets[-1], n), normal(k, offsets[-1], k)
    got = grouped.GroupedWeightGradient(len(sizes), n, k).forward(dy, x, on_device(offsets))
    assert ops.k3_moe_device_status() == 0
    return [off(got[g], dy[a:b].double().t() @ x[a:b].double()) if b > a else 0.0
            for g, (a, b) in enumerate(zip(offsets, offsets[1:]))]


# the second: large groups among empty and small ones; the last two: deep ones among hundreds, groups on the average small
@pytest.mark.parametrize("n,k", [(520, 264), (2048, 1032), (384, 2048)])
@pytest.mark.parametrize("sizes", [[2048] * 8, [3000, 40, 0, 20] * 5, [8192], [2500, 16, 4096, 1] + [3] * 300, [20000] + [0] * 60])
def test_tensor_cores_by_weight(n, k, sizes):
    for size, error in zip(sizes, by_weight(n, k, sizes)):
        if size:
            assert error <= tensor_core_bound(size), (size, error)


@pytest.mark.parametrize("groups,n,k", [(32, 2048, 1032), (40, 520, 2056), (300, 264, 520)])
@pytest.mark.parametrize("segments", [2, 3])
def test_every_512_rows_of_a_group_are_summed_by_themselves(groups, n, k, segments):
    """So a group's gradient is the f32 sum of those of its parts of 512 rows, to the last bit, whatever the group's size."""
    rows = groups * segments * 512
    dy, x = normal(n, rows, n), normal(k, rows, k)
    whole, parts = (grouped.GroupedWeightGradient(g, n, k).forward(dy, x, on_device(range(0, rows + 1, rows // g)))
                    for g in (groups, groups * segments))
    want = parts[::segments].clone()
    for i in range(1, segments):
        want += parts[i::segments]
    assert torch.equal(whole, want)


def test_fma_pipes_by_weight():
    sizes = [2049, 17, 0, 32770, 7168]
    for size, error in zip(sizes, by_weight(130, 65, sizes)):
        if size:
            assert error <= fma_bound(size), (size, error)

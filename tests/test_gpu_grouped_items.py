"""Grouped products of many short items per block, so that item slots, stages and accumulators are taken again and again, with
integers whose sums f32 holds exactly: every element has to be equal."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import grouped, ops        # noqa: E402

BF16, F32 = torch.bfloat16, torch.float32


def integers(seed, *shape):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(-3, 4, shape, generator=g, device="cuda").to(BF16)


# rows per group: many tiles of up to 64, 128 and 256 rows, even and not, of one to nine blocks of the depth
@pytest.mark.parametrize("sizes", [[512] * 64, [300, 0, 811, 1, 256] * 20, [2048] * 16, [130] * 200, [40] * 200, [1000, 5] * 32])
@pytest.mark.parametrize("depth,wide", [(64, 2048), (136, 1032), (576, 2048)])
@pytest.mark.parametrize("form", ["forward", "by_input"])
def test_many_short_items(form, sizes, depth, wide):
    offsets = torch.tensor([0] + sizes, device="cuda").cumsum(0)
    rows = int(offsets[-1])
    a = integers(depth, rows, depth)
    w = integers(wide, len(sizes), *((wide, depth) if form == "forward" else (depth, wide)))
    product = grouped.GroupedProduct(w)
    call = product.forward if form == "forward" else product.by_input
    want = torch.cat([x.float() @ (m.float().t() if form == "forward" else m.float()) for x, m in zip(a.split(sizes), w)])
    assert float(want.abs().max()) < 2 ** 24
    for dtype in (F32, BF16):
        for _ in range(3):
            assert torch.equal(call(a, offsets.to(torch.int32), dtype=dtype), want.to(dtype))
    assert ops.k3_moe_device_status() == 0


@pytest.mark.parametrize("sizes", [[64] * 300, [70, 0, 130, 17] * 40, [1030, 5, 600] * 8])
@pytest.mark.parametrize("n,k", [(520, 264), (1032, 512)])
def test_many_short_items_by_weight(sizes, n, k):
    offsets = torch.tensor([0] + sizes, device="cuda").cumsum(0)
    rows = int(offsets[-1])
    dy, x = integers(n, rows, n), integers(k, rows, k)
    want = torch.stack([a.float().t() @ b.float() for a, b in zip(dy.split(sizes), x.split(sizes))])
    gradient = grouped.GroupedWeightGradient(len(sizes), n, k)
    for dtype in (F32, BF16):
        for _ in range(3):
            assert torch.equal(gradient.forward(dy, x, offsets.to(torch.int32), dtype=dtype), want.to(dtype))
    assert ops.k3_moe_device_status() == 0

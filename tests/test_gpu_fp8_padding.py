"""Codes past the end of a row are zeros also where the last block holds an infinity or a NaN."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
if not torch.cuda.is_available():
    pytest.skip("no CUDA device", allow_module_level=True)

from moonshine_b200 import fp8                 # noqa: E402
from tests.test_gpu_fp8 import check_quantized  # noqa: E402


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
@pytest.mark.parametrize("rows,columns", [(260, 260), (1, 1), (129, 264), (7, 33), (264, 129), (200, 136), (131, 250)])
def test_padding_of_a_block_that_is_not_finite(form, rows, columns, dtype):
    x = torch.randn(rows, columns, generator=torch.Generator().manual_seed(rows)).to(dtype)
    x[rows - 1, :] = float("nan")                # the last block of every row or column, partial in both
    x[:, columns - 1] = float("inf")
    if rows > 1:
        x[0, 0] = -float("inf")
    x = x.cuda()
    check_quantized(form, x, *getattr(fp8, "quantize_" + form)(x))

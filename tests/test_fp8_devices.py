"""Where the tensors of the E4M3 and balance forms lie, and that each check of shapes and types is made: every
refusal by its own message.  Nothing here reaches a launch."""
import pytest
import torch

from moonshine_b200 import balance, fp8, ops

F8, BF16, F32, I32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32, torch.int32
CUDA0 = torch.device("cuda", 0)


class Placed:
    """What the checks look at of a tensor on a GPU."""
    def __init__(self, *shape, dtype=BF16, device=CUDA0):
        self.shape, self.dtype, self.device = torch.Size(shape), dtype, device

    def get_device(self):
        return self.device.index

    def dim(self):
        return len(self.shape)


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    monkeypatch.setattr(fp8, "_current_device", lambda: 0)
    for name in vars(ops).copy():
        if name.startswith(("k3_moe_fp8_", "k3_moe_balance", "k3_moe_router_backward")) and "workspace" not in name:
            monkeypatch.setattr(ops, name, lambda *a, name=name, **k: pytest.fail(name + " was called"))


def table(rows, columns, *lead, device="cpu", scales_device=None):
    codes = torch.zeros(*lead, rows, fp8.pitch(columns), dtype=F8, device=device)
    return codes, torch.ones(*lead, fp8.blocks(rows), fp8.blocks(columns), device=scales_device or device)


def on_the_gpu(monkeypatch, *objects):
    """As if the objects' tables lay on the GPU."""
    for o in objects:
        monkeypatch.setattr(o, "_device", CUDA0)


def test_tables_on_the_host_are_not_multiplied():
    linear = fp8.Fp8Linear(*table(64, 128), 64, 128)
    with pytest.raises(ValueError, match="x: on cuda:0, the tables are on cpu"):
        linear.forward(Placed(2, 128))
    gradient = fp8.Fp8LinearGradient(*table(128, 64), 64, 128)
    with pytest.raises(ValueError, match="x: on cuda:0, the tables are on cpu"):
        gradient.by_input(Placed(2, 64))
    experts = fp8.Fp8Experts(*table(64, 128, 2), *table(64, 128, 2), *table(128, 64, 2), top_k=1)
    with pytest.raises(ValueError, match="x: on cuda:0, the tables are on cpu"):
        experts.forward(Placed(3, 128), Placed(3, 1, dtype=I32), Placed(3, 1, dtype=F32))
    with pytest.raises(ValueError, match="table: expected a tensor on the current CUDA device, got one on cpu"):
        fp8.transpose_blocks(*table(64, 128), 64, 128)


def test_a_table_lies_on_one_device():
    with pytest.raises(ValueError, match="table: codes on cpu, scales on meta"):
        fp8.Fp8Linear(*table(64, 128, scales_device="meta"), 64, 128)
    with pytest.raises(ValueError, match="table: codes on meta, scales on cpu"):
        fp8.transpose_blocks(*table(64, 128, device="meta", scales_device="cpu"), 64, 128)
    for at in range(3):
        shapes = ((64, 128, 2), (64, 128, 2), (128, 64, 2))
        tables = [t for i, s in enumerate(shapes) for t in table(*s, scales_device="meta" if i == at else None)]
        with pytest.raises(ValueError, match=f"w{(1, 3, 2)[at]}: codes on cpu, scales on meta"):
            fp8.Fp8Experts(*tables, top_k=1)
        if at:
            tables = [t for i, s in enumerate(shapes) for t in table(*s, device="meta" if i == at else "cpu")]
            with pytest.raises(ValueError, match=f"w{(1, 3, 2)[at]}: on meta, w1 on cpu"):
                fp8.Fp8Experts(*tables, top_k=1)


HOST = "expected a tensor on the current CUDA device, got one on cpu"


def test_inputs_lie_on_the_current_device(monkeypatch):
    host = lambda *s, dtype=BF16: torch.zeros(*s, dtype=dtype)              # noqa: E731
    other = lambda *s, dtype=BF16: Placed(*s, dtype=dtype, device=torch.device("cuda", 1))  # noqa: E731
    for form in (fp8.quantize_rows, fp8.quantize_columns, fp8.quantize_blocks):
        with pytest.raises(ValueError, match="x: " + HOST):
            form(host(4, 4))
        with pytest.raises(ValueError, match="x: .* got one on cuda:1"):
            form(other(4, 4))
    linear = fp8.Fp8Linear(*table(64, 128), 64, 128)
    gradient = fp8.Fp8LinearGradient(*table(128, 64), 64, 128)
    experts = fp8.Fp8Experts(*table(64, 128, 2), *table(64, 128, 2), *table(128, 64, 2), top_k=1)
    on_the_gpu(monkeypatch, linear, gradient._by_input, experts)
    for wrong, message in ((host, HOST), (other, ".* got one on cuda:1")):
        with pytest.raises(ValueError, match="x: " + message):
            linear.forward(wrong(2, 128))
        with pytest.raises(ValueError, match="dy: " + message):
            gradient.by_weight(wrong(2, 64), Placed(2, 128))
        with pytest.raises(ValueError, match="x: " + message):
            gradient.by_weight(Placed(2, 64), wrong(2, 128))
        with pytest.raises(ValueError, match="into: " + message):
            gradient.by_weight(Placed(2, 64), Placed(2, 128), into=wrong(64, 128, dtype=F32))
        good = [Placed(3, 128), Placed(3, 1, dtype=I32), Placed(3, 1, dtype=F32), Placed(3, 128)]
        for at, name in enumerate(("x", "ids", "weights", "shared")):
            args = list(good)
            args[at] = wrong(*good[at].shape, dtype=good[at].dtype)
            with pytest.raises(ValueError, match=name + ": " + message):
                experts.forward(*args)
        router = balance.RouterBalance(8, 2)
        good = [Placed(3, 8, dtype=F32), Placed(3, 2, dtype=I32), Placed(2, dtype=I32)]
        for at, name in enumerate(("logits", "ids", "offsets")):
            args = list(good)
            args[at] = wrong(*good[at].shape, dtype=good[at].dtype)
            with pytest.raises(ValueError, match=name + ": " + message):
                router.forward(*args)
        good = [Placed(3, 8, dtype=F32), Placed(3, 2, dtype=I32), Placed(1, 8, dtype=I32), Placed(2, dtype=I32), Placed(1, dtype=F32),
                Placed(3, 2, dtype=F32)]
        for at, name in enumerate(("logits", "ids", "counts", "offsets", "d_loss", "d_weights")):
            args = list(good)
            args[at] = wrong(*good[at].shape, dtype=good[at].dtype)
            with pytest.raises(ValueError, match=name + ": " + message):
                router.backward(*args)


def test_shapes_and_types_of_inputs(monkeypatch):
    linear = fp8.Fp8Linear(*table(64, 128), 64, 128)
    gradient = fp8.Fp8LinearGradient(*table(128, 64), 64, 128)
    experts = fp8.Fp8Experts(*table(64, 128, 2), *table(64, 128, 2), *table(128, 64, 2), top_k=1)
    on_the_gpu(monkeypatch, linear, gradient._by_input, experts)
    for bad in (Placed(2, 127), Placed(2, 128, dtype=F32), Placed(128)):
        with pytest.raises(ValueError, match=r"x: expected \[rows, 128\]"):
            linear.forward(bad)
        with pytest.raises(ValueError, match=r"x: expected \[rows, 128\]"):
            gradient.by_weight(Placed(2, 64), bad)
        with pytest.raises(ValueError, match=r"x: expected \[rows, 128\]"):
            experts.forward(bad, Placed(2, 1, dtype=I32), Placed(2, 1, dtype=F32))
        with pytest.raises(ValueError, match=r"shared: expected \[rows, 128\]"):
            experts.forward(Placed(2, 128), Placed(2, 1, dtype=I32), Placed(2, 1, dtype=F32), bad)
    with pytest.raises(ValueError, match="dy and x: different numbers of tokens"):
        gradient.by_weight(Placed(3, 64), Placed(2, 128))
    with pytest.raises(ValueError, match=r"into: expected \[64, 128\], got \[63, 128\]"):
        gradient.by_weight(Placed(2, 64), Placed(2, 128), into=Placed(63, 128, dtype=F32))
    with pytest.raises(ValueError, match="into: .*float32"):
        gradient.by_weight(Placed(2, 64), Placed(2, 128), into=Placed(64, 128))
    for bad in (Placed(2, 2, dtype=I32), Placed(3, 1, dtype=I32), Placed(2, 1, dtype=torch.int64)):
        with pytest.raises(ValueError, match=r"ids: expected torch.int32 \[2, 1\]"):
            experts.forward(Placed(2, 128), bad, Placed(2, 1, dtype=F32))
    with pytest.raises(ValueError, match=r"weights: expected torch.float32 \[2, 1\]"):
        experts.forward(Placed(2, 128), Placed(2, 1, dtype=I32), Placed(2, 1))
    with pytest.raises(ValueError, match="shared: another number of tokens"):
        experts.forward(Placed(2, 128), Placed(2, 1, dtype=I32), Placed(2, 1, dtype=F32), Placed(3, 128))
    for form in (fp8.quantize_rows, fp8.quantize_columns, fp8.quantize_blocks):
        with pytest.raises(ValueError, match=r"x: expected \[rows, columns\]"):
            form(Placed(4, 4, dtype=torch.float16))
    router = balance.RouterBalance(8, 2)
    good = [Placed(3, 8, dtype=F32), Placed(3, 2, dtype=I32), Placed(1, 8, dtype=I32), Placed(2, dtype=I32), Placed(1, dtype=F32),
            Placed(3, 2, dtype=F32)]
    for at, bad, message in ((0, Placed(3, 9, dtype=F32), "logits: expected torch.float32"), (0, Placed(3, 8), "logits: expected"),
                             (1, Placed(3, 2, dtype=torch.int64), "ids: expected torch.int32"), (1, Placed(3, 3, dtype=I32), "ids: "),
                             (2, None, "d_loss wants the counts"), (2, Placed(2, 8, dtype=I32), r"counts: expected torch.int32 \[1, 8\]"),
                             (3, Placed(2, dtype=F32), r"offsets: expected int32 \[sequences \+ 1\]"), (3, Placed(1, dtype=I32), "offsets: "),
                             (4, Placed(2, dtype=F32), r"d_loss: expected torch.float32 \[1\]"),
                             (5, Placed(3, 3, dtype=F32), r"d_weights: expected torch.float32 \[3, 2\]")):
        args = list(good)
        args[at] = bad
        with pytest.raises(ValueError, match=message):
            router.backward(*args)
    for args in ((good[0], good[1], Placed(2, 2, dtype=I32)), (Placed(2, 8, dtype=F32), good[1], good[3])):
        with pytest.raises(ValueError, match="offsets: |logits: "):
            router.forward(*args)

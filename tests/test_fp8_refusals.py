"""What the E4M3 and balance entry points refuse, before any launch; their Python forms' checks."""
import ctypes as C
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def native():
    from moonshine_b200 import build, _native
    build.build()
    return _native


P = 0x1000          # never dereferenced: every call below fails validation first


def test_description_matches_header(native):
    text = open(os.path.join(ROOT, "include", "k3_moe_fp8.h")).read()
    body = text[text.index("typedef struct k3_moe_fp8_experts_desc {"):text.index("} k3_moe_fp8_experts_desc;")]
    fields = re.findall(r"^\s+(?:const void \*|uint32_t\s+|int32_t\s+|float\s+)(\w+);", body, re.M)
    assert fields == [f[0] for f in native.Fp8ExpertsDesc._fields_]


@pytest.mark.parametrize("form", ["rows", "columns", "blocks"])
def test_quantisers(native, form):
    fn = getattr(native.lib(), "k3_moe_fp8_quantize_" + form)
    good = [P, P, P, 4, 64, 0, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, 0), (4, 0), (5, 2), (5, -1), (0, P + 8), (1, P + 4), (2, P + 1),
                    (3, (1 << 30) + 1)):
        args = list(good)
        args[at] = bad
        assert fn(*args) is False, (at, bad)
    assert fn(P, P, P + 2, 4, 64, 1, None) is False                        # f32 between its words


def test_transposed_table(native):
    fn = native.lib().k3_moe_fp8_transpose_blocks
    good = [2 * P, P, P, P, 4, 64, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, 0), (5, 0), (0, P + 8), (2, P + 4), (0, P)):
        args = list(good)
        args[at] = bad
        assert fn(*args) is False, (at, bad)


def test_product(native):
    fn = native.lib().k3_moe_fp8_product
    good = [P, P, P, P, P, 4, 64, 64, 0, 0, 0, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, 0), (6, 0), (7, 0), (8, 2), (9, 2), (10, 1), (1, P + 8),
                    (2, P + 4), (3, P + 1), (4, P + 2), (0, P + 1)):
        args = list(good)
        args[at] = bad
        assert fn(*args) is False, (at, bad)
    assert fn(P, P, P, P, P + 4, 4, 64, 64, 1, 0, 0, None) is False        # scales per row want 16 bytes
    assert fn(P + 2, P, P, P, P, 4, 64, 64, 0, 1, 0, None) is False        # f32 between its words


def test_linear_and_weight_gradient(native):
    lib = native.lib()
    need = lib.k3_moe_fp8_linear_workspace_bytes(4, 64)
    assert need > 0 and lib.k3_moe_fp8_linear_workspace_bytes(0, 64) == 0 and lib.k3_moe_fp8_linear_workspace_bytes(4, 0) == 0
    good = [P, P, P, P, 4, 64, 64, P, need, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, 0), (5, 0), (6, 0), (7, None), (8, need - 1), (7, P + 8),
                    (2, P + 8), (0, P + 1), (1, P + 1)):
        args = list(good)
        args[at] = bad
        assert lib.k3_moe_fp8_linear(*args) is False, (at, bad)
    need = lib.k3_moe_fp8_weight_gradient_workspace_bytes(4, 64, 64)
    assert need > 0 and lib.k3_moe_fp8_weight_gradient_workspace_bytes(4, 64, 0) == 0
    good = [P, P, P, 4, 64, 64, 0, P, need, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, 0), (4, 0), (5, 0), (7, None), (8, need - 1), (0, P + 2), (1, P + 1)):
        args = list(good)
        args[at] = bad
        assert lib.k3_moe_fp8_weight_gradient(*args) is False, (at, bad)


def experts_desc(native, **changed):
    d = dict(hidden=256, expert_hidden=128, experts=8, top_k=2, activation=1, beta=4.0, linear_beta=25.0, w1=P, w1_scales=P,
             w3=P, w3_scales=P, w2=P, w2_scales=P)
    d.update(changed)
    return native.Fp8ExpertsDesc(**d)


def test_experts(native):
    lib = native.lib()
    for changed in (dict(hidden=0), dict(hidden=250), dict(expert_hidden=0), dict(expert_hidden=120), dict(experts=0),
                    dict(experts=1025), dict(top_k=0), dict(top_k=33), dict(top_k=9), dict(activation=2),
                    dict(activation=0, beta=0.0), dict(activation=0, linear_beta=-1.0)):
        d = experts_desc(native, **changed)
        assert lib.k3_moe_fp8_experts_workspace_bytes(d, 4) == 0, changed
        assert lib.k3_moe_fp8_experts_forward(d, P, P, P, P, None, 4, P, 1 << 40, None) is False, changed
    d = experts_desc(native)
    need = lib.k3_moe_fp8_experts_workspace_bytes(d, 4)
    assert need > 0 and lib.k3_moe_fp8_experts_workspace_bytes(d, 0) == 0 and lib.k3_moe_fp8_experts_workspace_bytes(None, 4) == 0
    good = [d, P, P, P, P, None, 4, P, need, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (6, 0), (7, None), (8, need - 1), (1, P + 8), (5, P + 8),
                    (7, P + 8), (2, P + 1), (3, P + 2), (4, P + 1)):
        args = list(good)
        args[at] = bad
        assert lib.k3_moe_fp8_experts_forward(*args) is False, (at, bad)
    for name in ("w1", "w1_scales", "w3", "w3_scales", "w2", "w2_scales"):
        assert lib.k3_moe_fp8_experts_forward(experts_desc(native, **{name: None}), *good[1:]) is False
        assert lib.k3_moe_fp8_experts_forward(experts_desc(native, **{name: P + 2}), *good[1:]) is False


def test_balance(native):
    lib = native.lib()
    need = lib.k3_moe_balance_workspace_bytes(10, 2, 64)
    assert need > 0
    for bad in ((0, 2, 64), (10, 0, 64), (10, 2, 0), (10, 2, 1025)):
        assert lib.k3_moe_balance_workspace_bytes(*bad) == 0
    good = [P, P, P, P, P, P, 10, 2, 64, 4, 0, 0.1, P, need, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (5, None), (6, 0), (7, 0), (8, 1025), (9, 0), (9, 33),
                    (8, 3), (10, 2), (12, None), (13, need - 1), (12, P + 8), (0, P + 2), (3, P + 1), (4, P + 3)):
        args = list(good)
        args[at] = bad
        assert lib.k3_moe_balance(*args) is False, (at, bad)
    good = [P, P, P, P, P, P, P, 10, 2, 64, 4, 0, 0.1, 1.0, None]
    for at, bad in ((0, None), (1, None), (2, None), (3, None), (4, None), (7, 0), (8, 0), (9, 0), (10, 0), (11, 5), (13, 0.0),
                    (13, float("nan")), (0, P + 2)):
        args = list(good)
        args[at] = bad
        assert lib.k3_moe_router_backward(*args) is False, (at, bad)
    args = list(good)
    args[5] = args[6] = None
    assert lib.k3_moe_router_backward(*args) is False                      # no gradient comes in


def test_python_forms_check_shapes_and_types(native):
    from moonshine_b200 import balance, fp8
    f8 = torch.float8_e4m3fn
    table, scales = torch.zeros(64, 128, dtype=f8), torch.ones(1, 1)
    lin = fp8.Fp8Linear(table, scales, 64, 128)
    for x in (torch.zeros(2, 127, dtype=torch.bfloat16), torch.zeros(2, 128), torch.zeros(128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            lin.forward(x)
    for args in ((table, scales, 64, 100), (table.float(), scales, 64, 128), (table, torch.ones(2, 1), 64, 128),
                 (table, scales.double(), 64, 128)):
        with pytest.raises(ValueError):
            fp8.Fp8Linear(*args)
    for form in (fp8.quantize_rows, fp8.quantize_columns, fp8.quantize_blocks):
        with pytest.raises(ValueError):
            form(torch.zeros(4, 4, dtype=torch.float16))
    w1, w2, s = torch.zeros(2, 64, 128, dtype=f8), torch.zeros(2, 128, 64, dtype=f8), torch.ones(2, 1, 1)
    with pytest.raises(ValueError):
        fp8.Fp8Experts(w1, s, w1, s, w1, s, top_k=1)
    with pytest.raises(ValueError):
        fp8.Fp8Experts(w1, s, w1, s, w2, s, top_k=1, activation="gelu")
    layer = fp8.Fp8Experts(w1, s, w1, s, w2, s, top_k=1)
    with pytest.raises(ValueError):
        layer.forward(torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, 2))
    with pytest.raises(ValueError):
        balance.RouterBalance(8, 2, "tanh")
    router = balance.RouterBalance(8, 2)
    ids = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError):
        router.forward(torch.zeros(3, 9), ids)
    with pytest.raises(ValueError):
        router.forward(torch.zeros(3, 8), ids.long())
    with pytest.raises(ValueError):
        router.forward(torch.zeros(3, 8), ids, torch.zeros(2))
    with pytest.raises(ValueError):
        router.backward(torch.zeros(3, 8), ids, None, None, torch.zeros(1))

"""What shapes and types the adapters of a batch take does not depend on the number of rows."""
import pytest
import torch

from polyrl_b200 import ops

from .requests_oracle import adapters64, check_near, swiglu64
from .test_requests_cpu import adapters_case
from .test_requests_gpu import near64, run_adapters

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
ROWS = [40, 300, 700]


@pytest.mark.parametrize("t", ROWS)
@pytest.mark.parametrize("way", [True, False])
def test_shapes_are_refused_for_any_number_of_rows(t, way, monkeypatch):
    monkeypatch.setattr(ops.adapters, "_together", lambda a, b: way)
    for k, widths, rank in ((64, (64,), 8), (64, (48, 16), 16), (72, (64,), 16), (64, (64, 64, 64), 144), (64, (64,), 400)):
        c = adapters_case(t, k, widths, rank, 2, 0, BF, "cuda")
        with pytest.raises(ValueError):
            run_adapters(c, widths, 2)
    for k, f, rank in ((64, 128, 8), (72, 128, 16), (64, 128, 200)):
        c = adapters_case(t, k, (f, f), rank, 2, 0, BF, "cuda", extra=False)
        with pytest.raises(ValueError):
            ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], ops.adapter_plan(c["ids"], 2))
    c = adapters_case(t, 64, (64, 64, 64), 128, 2, 1, BF, "cuda")                    # the most that is taken
    check_near(run_adapters(c, (64, 64, 64), 2), *near64(c, (64, 64, 64)))


@pytest.mark.parametrize("t", [3, *ROWS])
def test_a_weight_of_another_type_is_converted(t):
    c = adapters_case(t, 128, (256,), 16, 3, t, BF, "cuda")
    assert torch.equal(run_adapters(dict(c, w=c["w"].float()), (256,), 3), run_adapters(c, (256,), 3))
    c = adapters_case(t, 128, (256, 256), 16, 3, t, BF, "cuda", extra=False)
    plan = ops.adapter_plan(c["ids"], 3)
    y = ops.adapter_linear_swiglu(c["x"], c["w"].float(), c["a"], c["b"], c["scales"], plan)
    assert torch.equal(y, ops.adapter_linear_swiglu(c["x"], c["w"], c["a"], c["b"], c["scales"], plan))
    check_near(y, *swiglu64(*adapters64(**c, widths=(256, 256), interleaved=True)))

"""The serving operators' checks that need no GPU, beyond those of test_serving_cpu.py."""
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType


class UnlaunchedRuntime(tb.Runtime):
    def __init__(self):
        self.session, self.stream, self.autotuner = object(), None, None


@pytest.mark.parametrize("operator,dtype,shape", [("kv_cache.append", DType.BF16, (6, 16, 2, 64)),
                                                  ("attention.varlen", DType.BF16, (6, 16, 64))])
def test_an_output_has_to_be_its_spec(operator, dtype, shape):
    rt = UnlaunchedRuntime()
    handle = lambda dtype, shape, strides=None: tb.TensorHandle(  # noqa: E731
        rt.session, None, dtype, shape, strides or tb.runtime.contiguous_strides(shape))
    count = 2 if operator == "kv_cache.append" else 1
    inputs = [handle(dtype, (4, 2, 64))] * (3 if count == 2 else 4)

    def outputs(spec, tensor):
        return rt._checked(tb.OpRequest(operator, inputs, [spec] * count), [tensor] * count)

    plain = tb.runtime.contiguous_strides(shape)
    turned = tuple(2 * x for x in plain[:-1]) + (1,)
    # A spec without strides takes the tensor's; equal ones and those of an extent of one pass.
    request, _ = outputs(tb.TensorSpec(dtype, shape), handle(dtype, shape, turned))
    assert [s.resolved_strides() for s in request.outputs] == [turned] * count
    outputs(tb.TensorSpec(dtype, shape, turned), handle(dtype, shape, turned))
    single = (1,) + shape[1:]
    outputs(tb.TensorSpec(dtype, single, (7,) + plain[1:]), handle(dtype, single))
    for spec, tensor in [(tb.TensorSpec(dtype, shape, plain), handle(dtype, shape, turned)),
                         (tb.TensorSpec(dtype, shape), handle(DType.F16, shape)),
                         (tb.TensorSpec(dtype, shape), handle(dtype, (5,) + shape[1:])),
                         (tb.TensorSpec(dtype, shape), handle(dtype, shape[1:]))]:
        with pytest.raises(tb.ExecutionError, match="their specs' dtype, shape and strides"):
            outputs(spec, tensor)

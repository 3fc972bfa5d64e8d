"""Host threads that enqueue on one stream: operators that take the stream's scratch memory."""
import threading

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import rows

pytestmark = pytest.mark.gpu


def bound_gemm(session, rt, m, n, k, seed):
    a, b = (upload(session, rt.stream, rows((x, k), DType.BF16, seed + i), DType.BF16) for i, x in enumerate((m, n)))
    request = tb.OpRequest("gemm", [a, b], [tb.TensorSpec(DType.BF16, (m, n))], {"transpose_rhs": True})
    return rt.bind(request, tb.TensorHandle.allocate(session, DType.BF16, (m, n)))


def test_bound_gemms_from_two_threads():
    """Split-K partials and staged operands of different sizes on one stream: the scratch grows while
    the other thread enqueues, and each result is what it is alone."""
    session = tb.Session(0)
    for sizes in (((128, 128, 4096), (256, 512, 4096)), ((512, 512, 513), (1024, 1024, 513))):
        alone, together = tb.Runtime(session), tb.Runtime(session)
        want = []
        for i, size in enumerate(sizes):
            one = bound_gemm(session, alone, *size, 10 * i)
            one.enqueue()
            want.append(one.outputs[0].to_numpy(alone.stream))
        both = [bound_gemm(session, together, *size, 10 * i) for i, size in enumerate(sizes)]
        threads = [threading.Thread(target=lambda r=r: [r.enqueue() for _ in range(200)]) for r in both]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        for r, w in zip(both, want):
            np.testing.assert_array_equal(r.outputs[0].to_numpy(together.stream), w)
    session.close()

"""The serving operators at sizes, bounds and arguments between those of the other tests."""
import math

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import as_f64, assert_attention, paged_reference, plan_reference, rows
from test_attention_serving_gpu import check_varlen, ints, make_cache, prefix, run_paged, view
from test_kv_cache_gpu import assert_plan, random_plan, spec_of

pytestmark = pytest.mark.gpu


@pytest.fixture()
def session():
    s = tb.Session(0)
    yield s
    s.close()


@pytest.fixture()
def rt(session):
    return tb.Runtime(session)


def test_plan_of_every_batch_launches(session, rt):
    """Batches whose shared memory is 48 KB with the kernel's static bytes, the smaller ones first."""
    for batch in (6109, 6110, 6143, 6144, 16384, 6120):
        rng = np.random.default_rng(batch)
        ctx, new, free, table = random_plan(rng, batch, 9, 2, 4)
        got = assert_plan(session, rt, ctx, new, free, table, int(new.sum()) + 1, 4)
        assert got[4][1] == 0

"""The library's host side on a stand-in driver: what threads, sizes and requests make of a
stream's memory and a kernel's limits."""
import pytest

import host_driver

pytestmark = host_driver.needs_compiler


@pytest.fixture(scope="module")
def driver(tmp_path_factory):
    return host_driver.build_driver(tmp_path_factory.mktemp("driver"))


SCRATCH_USERS = """
def gemm(m, n, k, **attrs):
    a, b = (tb.TensorHandle.allocate(session, DType.BF16, s) for s in ((m, k), (n, k)))
    c = tb.TensorHandle.allocate(session, DType.BF16, (m, n))
    return rt.bind(tb.OpRequest("gemm", [a, b], [spec_of(c)], {"transpose_rhs": True, **attrs}), c)

def sdpa(t):
    x = tb.TensorHandle.allocate(session, DType.BF16, (1, 1, t, 128))
    return rt.bind(tb.OpRequest("scaled_dot_product_attention", [x] * 3, [spec_of(x)],
                                {"candidate": "sdpa_fwd_bf16_d128_persist"}), x)

def hammer(*requests):
    fake.fake_slow(3)
    in_threads(*[lambda r=r: [r.enqueue() for _ in range(8)] for r in requests])
    fake.fake_slow(0)
    seen = lines()
    assert not [x for x in seen if x.startswith("error")], [x for x in seen if x.startswith("error")]
    return [x.split()[1:] for x in seen]
"""


def test_threads_share_a_stream_s_scratch(driver):
    """Requests of several threads on one stream, of operators that take its scratch memory: none is
    launched on memory that a larger one replaced, and none comes between another's kernels."""
    host_driver.run(driver, SCRATCH_USERS + """
small, large = gemm(128, 128, 4096), gemm(256, 512, 4096)
launches = hammer(small, large)
assert {x[0] for x in launches} == {"gemm_bf16_tn_splitk", "splitk_reduce_bf16"}
for first, second in zip(launches[::2], launches[1::2]):
    assert first[0] == "gemm_bf16_tn_splitk" and second[0] == "splitk_reduce_bf16" and first[1:] == second[1:]

rt = tb.Runtime(session)
launches = hammer(gemm(512, 512, 513), gemm(1024, 1024, 513), sdpa(300))
names = [x[0] for x in launches]
for i, name in enumerate(names):  # two staged operands, then their product
    if name == "stage_bf16_pad_rows":
        if names[i - 1] != name:
            assert names[i + 1] == name and names[i + 2].startswith("gemm_bf16_tn"), names[i:i + 4]
""")


def test_every_plan_has_its_shared_memory(driver):
    """kv_cache.plan's dynamic shared memory grows with the batch, beside static bytes: around 48 KB
    together, and from threads whose batches differ."""
    host_driver.run(driver, """
def plan(runtime, batch):
    ints = lambda *shape: tb.TensorHandle.allocate(session, DType.I32, shape)
    outs = [ints(batch, 2), ints(batch), ints(batch + 1), ints(batch), ints(2)]
    return runtime.bind(tb.OpRequest("kv_cache.plan", [ints(batch), ints(batch), ints(4)],
                                     [spec_of(t) for t in outs], {"page_size": 16}), outs)

for batch in (6109, 6110, 6143, 6144, 16384, 6120):
    plan(rt, batch).enqueue()
fake.fake_slow(2)
requests = [plan(tb.Runtime(session), batch) for batch in (6500, 9000, 12000, 16000)]
in_threads(*[lambda r=r: [r.enqueue() for _ in range(20)] for r in requests])
session.close()
session = tb.Session(0)  # (a fresh limit)
requests = [plan(tb.Runtime(session), batch) for batch in (6500, 9000, 12000, 16000)]
in_threads(*[lambda r=r: [r.enqueue() for _ in range(20)] for r in requests])
""")


def test_an_omitted_attention_output_begins_as_zeros(driver):
    """Rows of no request are left as they were: in an output that the runtime makes they are zeros."""
    host_driver.run(driver, """
x = tb.TensorHandle.allocate(session, DType.BF16, (70, 4, 64))
cu = tb.TensorHandle.allocate(session, DType.I32, (2,))
assert x.to_numpy(rt.stream).any()  # (memory that something was in)
cache = tb.TensorHandle.allocate(session, DType.BF16, (6, 16, 4, 64))
table, lens = (tb.TensorHandle.allocate(session, DType.I32, s) for s in ((1, 6), (1,)))
for request in (tb.OpRequest("attention.varlen", [x, x, x, cu], [spec_of(x)]),
                tb.OpRequest("attention.paged", [x, cache, cache, table, lens, cu], [spec_of(x)])):
    assert not rt.execute(request).outputs[0].to_numpy(rt.stream).any()
    assert not rt.bind(request).outputs[0].to_numpy(rt.stream).any()
    given = tb.TensorHandle.allocate(session, DType.BF16, (70, 4, 64))
    assert rt.execute(request, output=given).outputs[0].to_numpy(rt.stream).all()
""")


def test_clear_checks_its_buffer(driver):
    host_driver.run(driver, """
b = session.allocate(64)
def raised(call, text):
    try:
        call()
    except tb.HalError as e:
        assert text in str(e), e
        return True
assert raised(lambda: session.clear(rt.stream, b, 65), "exceeds allocation")
other = tb.Session(0)
assert raised(lambda: other.clear(other.create_stream(), b, 8), "foreign buffer")
assert raised(lambda: other.clear(rt.stream, other.allocate(8), 8), "stream")
x = tb.TensorHandle(session, b, DType.I32, (16,), (1,))
session.wait(session.clear(rt.stream, b, 12))
assert (x.to_numpy(rt.stream)[:3] == 0).all() and x.to_numpy(rt.stream)[3:].all()
""")


def test_a_graph_keeps_the_scratch_that_it_was_captured_on(driver):
    """A larger operator on the stream, and the stream's release, leave a captured one's scratch memory."""
    host_driver.run(driver, SCRATCH_USERS + """
small, large = gemm(128, 128, 4096), gemm(256, 512, 4096)
small.enqueue()
session.capture_begin(rt.stream)
small.enqueue()
graph = session.capture_end(rt.stream)
lines()
large.enqueue()
other = session.create_stream()
for step in range(2):
    graph.launch(other)
    seen = lines()
    assert [x.split()[1] for x in seen[-2:]] == ["gemm_bf16_tn_splitk", "splitk_reduce_bf16"], seen
    assert not [x for x in seen if x.startswith("error")], seen
    if step == 0:  # the larger one, captured too, outlives its stream
        session.capture_begin(rt.stream)
        large.enqueue()
        second = session.capture_end(rt.stream)
        rt.stream.release()
        del small, large
        import gc; gc.collect()
second.launch(other)
seen = lines()
assert len(seen) == 2 and not [x for x in seen if x.startswith("error")], seen
""")

"""The paged cache's plan and append on the GPU, and a serving run that uses them with the
attention operators: prompts, chunks and tokens, eager, bound and captured."""
import math

import numpy as np
import pytest

import titan_rs_b200 as tb
from titan_rs_b200.kernel_abi import DType

from gpu_util import upload
from serving_util import as_f64, assert_attention, one_request, plan_reference, rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def session():
    s = tb.Session(0)
    yield s
    s.close()


@pytest.fixture(scope="module")
def rt(session):
    return tb.Runtime(session)


def ints(session, rt, values):
    return upload(session, rt.stream, np.asarray(values, np.int32), DType.I32)


def spec_of(t):
    return tb.TensorSpec(t.dtype, t.shape, t.strides)


def run_plan(session, rt, ctx, new, free, table, tokens, page):
    batch = len(ctx)
    outs = [ints(session, rt, table), ints(session, rt, np.full(batch, -9)), ints(session, rt, np.full(batch + 1, -9)),
            ints(session, rt, np.full(tokens, -9)), ints(session, rt, [-9, -9])]
    rt.execute(tb.OpRequest("kv_cache.plan", [ints(session, rt, x) for x in (ctx, new, free)],
                            [spec_of(t) for t in outs], {"page_size": page}), output=outs).wait()
    return [t.to_numpy(rt.stream) for t in outs]


def assert_plan(session, rt, ctx, new, free, table, tokens, page):
    got = run_plan(session, rt, ctx, new, free, table, tokens, page)
    want = plan_reference(ctx, new, free, np.asarray(table, np.int32), tokens, page)
    for name, g, w in zip(("block_table", "seq_lens", "cu_seqlens", "slot_map", "status"), got, want):
        np.testing.assert_array_equal(g, w, err_msg=name)
    return got


def random_plan(rng, batch, ctx_high, new_high, page, width_extra=0):
    ctx, new = rng.integers(0, ctx_high + 1, batch), rng.integers(0, new_high + 1, batch)
    width = max(1, -(-(ctx_high + new_high) // page)) + width_extra
    held = -(-ctx // page)
    table = np.full((batch, width), -1, np.int32)
    order = rng.permutation(int(held.sum()) + 1000).astype(np.int32)
    at = 0
    for b in range(batch):
        table[b, :held[b]] = order[at:at + held[b]]
        at += held[b]
    need = int((-(-(ctx + new) // page) - held).sum())
    return ctx, new, np.concatenate([order[at:], np.arange(need, dtype=np.int32) + len(order)])[:need + 3], table


@pytest.mark.parametrize("batch,ctx_high,new_high,page", [
    (1, 0, 1, 16), (1, 100, 1, 16), (3, 50, 40, 8), (33, 300, 1, 16), (64, 0, 500, 64), (257, 90, 30, 7),
    (1000, 60, 3, 1), (1025, 100, 9, 16), (4097, 33, 5, 24), (16384, 9, 2, 4)])
def test_plan_matches_the_restatement(session, rt, batch, ctx_high, new_high, page):
    rng = np.random.default_rng(batch + page)
    ctx, new, free, table = random_plan(rng, batch, ctx_high, new_high, page)
    tokens = max(1, int(new.sum())) + (batch % 3)
    got = assert_plan(session, rt, ctx, new, free, table, tokens, page)
    assert got[4][1] == 0


def test_plan_refuses_requests_and_says_how_many(session, rt):
    page = 16
    # Negative lengths, a row too short, and a free list that ends: in one step.
    ctx = [5, -1, 16, 30, 40, 10, 31, 64]
    new = [1, 4, 20, -2, 60, 30, 1, 40]
    table = np.arange(8 * 6, dtype=np.int32).reshape(8, 6)
    for n_free in (1, 2, 3, 6, 30):
        got = assert_plan(session, rt, ctx, new, np.arange(100, 100 + n_free), table, 200, page)
        assert got[4][1] >= 3
    # More tokens than the slot map holds, and page ids whose slots pass 32 bits.
    assert_plan(session, rt, [0, 0, 0], [10, 10, 10], [1, 2, 3, 4], np.zeros((3, 2), np.int32), 15, page)
    assert_plan(session, rt, [3, 3], [2, 2], [7], np.array([[2 ** 31 - 1], [-4]], np.int32), 4, page)
    assert_plan(session, rt, [2 ** 31 - 1], [2 ** 31 - 1], [7], np.array([[1, 1]], np.int32), 4, 2 ** 31 - 1)
    assert_plan(session, rt, [2 ** 31 - 2, 2 ** 31 - 3], [3, 2], [7, 8], np.array([[1, 1], [0, 5]], np.int32), 9,
                2 ** 31 - 1)


def test_plan_refuses_outputs_that_share_memory(session, rt):
    ctx, new, free = (ints(session, rt, x) for x in ([5, 6], [1, 1], [7, 8, 9]))
    outs = [ints(session, rt, np.full((2, 3), -1)), ints(session, rt, [0, 0]), ints(session, rt, [0, 0, 0]),
            ints(session, rt, [0, 0]), ints(session, rt, [0, 0])]
    for i, other in ((1, ctx), (3, new), (3, outs[4]), (4, outs[1])):
        bad = list(outs)
        bad[i] = other
        with pytest.raises(tb.ExecutionError, match="share no memory"):
            rt.execute(tb.OpRequest("kv_cache.plan", [ctx, new, free], [spec_of(x) for x in outs], {"page_size": 16}),
                       output=bad)


def test_plan_strided_table(session, rt):
    rng = np.random.default_rng(3)
    ctx, new, free, table = random_plan(rng, 20, 60, 20, 8)
    wide = np.full((20, table.shape[1] + 5), -77, np.int32)
    wide[:, :table.shape[1]] = table
    base = ints(session, rt, wide)
    tokens = int(new.sum())
    t = tb.TensorHandle(session, base.buffer, DType.I32, table.shape, (wide.shape[1], 1))
    outs = [t, ints(session, rt, np.zeros(20)), ints(session, rt, np.zeros(21)), ints(session, rt, np.zeros(tokens)),
            ints(session, rt, [0, 0])]
    rt.execute(tb.OpRequest("kv_cache.plan", [ints(session, rt, x) for x in (ctx, new, free)],
                            [spec_of(x) for x in outs], {"page_size": 8}), output=outs).wait()
    want = plan_reference(ctx, new, free, table, tokens, 8)
    after = base.to_numpy(rt.stream)
    np.testing.assert_array_equal(after[:, :table.shape[1]], want[0])
    np.testing.assert_array_equal(after[:, table.shape[1]:], -77)
    np.testing.assert_array_equal(outs[3].to_numpy(rt.stream), want[3])


_NP = {DType.F32: np.float32, DType.F16: np.float16, DType.BF16: np.uint16}


@pytest.mark.parametrize("dtype", [DType.F32, DType.F16, DType.BF16])
@pytest.mark.parametrize("t,h,d,page,pages", [(1, 1, 1, 1, 1), (5, 2, 7, 3, 9), (64, 8, 128, 16, 40),
                                              (300, 2, 80, 24, 20), (17, 3, 64, 8, 4)])
def test_append_writes_the_named_rows_only(session, rt, dtype, t, h, d, page, pages):
    rng = np.random.default_rng(t + d)
    shape = (pages, page, h, d)
    k, v = (rng.standard_normal((t, h, d)).astype(np.float32) for _ in range(2))
    kc, vc = (rng.standard_normal(shape).astype(np.float32) for _ in range(2))
    k, v, kc, vc = ((tb.f32_to_bf16_bits(x) if dtype == DType.BF16 else x.astype(_NP[dtype])) for x in (k, v, kc, vc))
    slots = rng.permutation(pages * page)[:t].astype(np.int64)
    slots = np.concatenate([slots, np.full(max(0, t - len(slots)), -1)])
    slots[rng.random(t) < 0.2] = rng.choice([-1, -2 ** 31, pages * page, 2 ** 31 - 1])
    ins = [upload(session, rt.stream, x, dtype) for x in (k, v)] + [ints(session, rt, slots)]
    outs = [upload(session, rt.stream, x, dtype) for x in (kc, vc)]
    h_ = rt.execute(tb.OpRequest("kv_cache.append", ins, [tb.TensorSpec(dtype, shape)] * 2), output=outs).wait()
    for rows_, cache, got in ((k, kc, h_.outputs[0]), (v, vc, h_.outputs[1])):
        want = cache.reshape(-1, h, d).copy()
        ok = (slots >= 0) & (slots < pages * page)
        want[slots[ok]] = rows_[ok]
        np.testing.assert_array_equal(got.to_numpy(rt.stream).view(np.uint8), want.reshape(shape).view(np.uint8))


def test_append_strided_rows_and_caches(session, rt):
    """K and V as slices of one projection, the caches [pages, Hkv, page, D] inside one tensor, and
    rows that start at odd elements."""
    dtype, t, hk, d, page, pages = DType.BF16, 37, 2, 64, 16, 8
    for odd in (0, 1):
        rng = np.random.default_rng(odd)
        step = 5 * d + odd
        flat = rows((t * step + 8,), dtype, 600 + odd)
        base = upload(session, rt.stream, flat, dtype)
        both = rows((2, pages, hk, page, d), dtype, 610)
        store = upload(session, rt.stream, both, dtype)

        def part(owner, offset, shape, strides):
            extent = 1 + sum((n - 1) * st for n, st in zip(shape, strides))
            buf = session.wrap(owner.buffer.device_ptr + 2 * offset, 2 * extent)
            return tb.TensorHandle(session, buf, dtype, shape, strides)

        k, v = (part(base, odd + i * hk * d, (t, hk, d), (step, d, 1)) for i in range(2))
        caches = [part(store, i * pages * hk * page * d, (pages, page, hk, d), (hk * page * d, d, page * d, 1))
                  for i in range(2)]
        slots = rng.permutation(pages * page)[:t]
        rt.execute(tb.OpRequest("kv_cache.append", [k, v, ints(session, rt, slots)], [spec_of(c) for c in caches]),
                   output=caches).wait()
        want = both.copy()
        for i in range(2):
            for n, slot in enumerate(slots):
                at = n * step + odd + i * hk * d
                want[i, slot // page, :, slot % page] = flat[at:at + hk * d].reshape(hk, d)
        np.testing.assert_array_equal(store.to_numpy(rt.stream), want)


class Server:
    """A small serving loop over the four operators, with the sequences kept on the host beside it."""

    def __init__(self, session, batch, h, hk, d, page, pages, width, tokens, dtype, seed):
        self.s, self.rt = session, tb.Runtime(session)
        self.h, self.hk, self.d, self.page, self.dtype = h, hk, d, page, dtype
        self.batch, self.tokens, self.seed = batch, tokens, seed
        z = lambda *shape: upload(session, self.rt.stream, np.zeros(shape, np.int32), DType.I32)  # noqa: E731
        bits = np.uint16 if dtype == DType.BF16 else np.float16
        e = lambda *shape: upload(session, self.rt.stream, np.zeros(shape, bits), dtype)  # noqa: E731
        self.ctx, self.new, self.free = z(batch), z(batch), z(pages)
        self.table, self.lens, self.cu, self.slots, self.status = z(batch, width), z(batch), z(batch + 1), z(tokens), z(2)
        self.q, self.k, self.v, self.o = e(tokens, h, d), e(tokens, hk, d), e(tokens, hk, d), e(tokens, h, d)
        self.kc, self.vc = e(pages, page, hk, d), e(pages, page, hk, d)
        self.pool = list(range(pages))
        self.lengths = np.zeros(batch, np.int64)
        self.keys = [np.zeros((0, hk, d)) for _ in range(batch)]
        self.values = [np.zeros((0, hk, d)) for _ in range(batch)]

    def requests(self):
        outs = [self.table, self.lens, self.cu, self.slots, self.status]
        yield tb.OpRequest("kv_cache.plan", [self.ctx, self.new, self.free], [spec_of(t) for t in outs],
                           {"page_size": self.page}), outs
        caches = [self.kc, self.vc]
        yield tb.OpRequest("kv_cache.append", [self.k, self.v, self.slots], [spec_of(t) for t in caches]), caches
        yield tb.OpRequest("attention.paged", [self.q, self.kc, self.vc, self.table, self.lens, self.cu],
                           [spec_of(self.o)]), [self.o]

    def put(self, tensor, array):
        self.s.wait(self.s.upload(self.rt.stream, tensor.buffer, array))

    def inputs(self, new, seed):
        """Uploads a step's inputs; returns what check() needs."""
        free = np.full(self.free.shape, -1, np.int32)
        free[:len(self.pool)] = self.pool
        for t, a in ((self.ctx, self.lengths.astype(np.int32)), (self.new, np.asarray(new, np.int32)), (self.free, free)):
            self.put(t, a)
        q, k, v = (rows((self.tokens, n, self.d), self.dtype, seed + i) for i, n in enumerate((self.h, self.hk, self.hk)))
        for t, a in ((self.q, q), (self.k, k), (self.v, v)):
            self.put(t, a)
        return new, q, k, v

    def check(self, new, q, k, v):
        status = self.status.to_numpy(self.rt.stream)
        assert status[1] == 0
        self.pool = self.pool[status[0]:]
        got = self.o.to_numpy(self.rt.stream)
        at = 0
        for b, n in enumerate(new):
            sl = slice(at, at + n)
            at += n
            self.keys[b] = np.concatenate([self.keys[b], as_f64(k[sl])])
            self.values[b] = np.concatenate([self.values[b], as_f64(v[sl])])
            self.lengths[b] += n
            if n:
                ref, mag = one_request(as_f64(q[sl]), self.keys[b], self.values[b], True, 1 / math.sqrt(self.d))
                assert_attention(got[sl], ref, mag, self.dtype, len(self.keys[b]), np.abs(self.values[b]).max())


STEPS = [[130, 0, 7, 33], [1, 60, 1, 1], [1, 1, 0, 90], [3, 1, 1, 1], [1, 1, 1, 1], [0, 0, 1, 0]]


@pytest.mark.parametrize("dtype,d", [(DType.BF16, 128), (DType.F16, 64)])
@pytest.mark.parametrize("mode", ["eager", "bound", "captured"])
def test_serving_steps(session, dtype, d, mode):
    """Prompts, chunks and single tokens of four requests, step after step: plan, append, attend. As a
    captured graph one recording serves every step, since lengths and tables are read on the device."""
    srv = Server(session, 4, 8, 2, d, 16, 40, 12, 176, dtype, 700)
    rt = srv.rt
    bound = [rt.bind(r, o) for r, o in srv.requests()]
    if mode == "captured":
        srv.inputs([1, 1, 1, 1], 690)
        session.capture_begin(rt.stream)
        for b in bound:
            b.enqueue()
        graph = session.capture_end(rt.stream)
    for i, new in enumerate(STEPS):
        data = srv.inputs(new, 700 + 10 * i)
        if mode == "eager":
            for r, o in srv.requests():
                rt.execute(r, output=o)
        elif mode == "bound":
            for b in bound:
                b.enqueue()
        else:
            graph.launch(rt.stream)
        session.synchronize(rt.stream)
        srv.check(*data)


def test_prompt_attention_agrees_with_the_cache_path(session, rt):
    """The same prompts through attention.varlen and through append + attention.paged."""
    new = [70, 129, 1]
    srv = Server(session, 3, 4, 2, 128, 16, 30, 9, 200, DType.BF16, 800)
    _, q, k, v = srv.inputs(new, 800)
    for r, o in srv.requests():
        srv.rt.execute(r, output=o)
    paged = srv.o.to_numpy(srv.rt.stream)
    out = srv.rt.execute(tb.OpRequest("attention.varlen", [srv.q, srv.k, srv.v, srv.cu], [spec_of(srv.o)],
                                      {"causal": True})).wait().outputs[0].to_numpy(srv.rt.stream)
    a, b = as_f64(paged[:200]), as_f64(out[:200])
    # Both are within attention_tolerance of one value: 2 x (2^-8 + 2^-8 + 2^-11) of the largest |v| at most.
    assert np.abs(a - b).max() <= 2 * (2.0 ** -7 + 2.0 ** -11) * np.abs(as_f64(v)).max()


def test_bound_requests_hold_their_buffers(session):
    rt = tb.Runtime(session)
    x = upload(session, rt.stream, np.random.default_rng(1).standard_normal((4, 64)).astype(np.float32))
    y = tb.TensorHandle.allocate(session, DType.F32, (4, 64))
    want = np.exp(x.to_numpy(rt.stream).astype(np.float64))
    want /= want.sum(1, keepdims=True)
    b = rt.bind(tb.OpRequest("softmax", [x], [tb.TensorSpec(DType.F32, (4, 64))]), y)
    x.buffer.release()
    b.enqueue()
    np.testing.assert_allclose(y.to_numpy(rt.stream), want, rtol=1e-5)
    rt.stream.release()
    b.enqueue()  # and their stream
    other = tb.Session(0)
    foreign = upload(other, other.create_stream(), np.ones((4, 64), np.float32))
    foreign.session = session
    with pytest.raises(tb.ExecutionError, match="foreign buffer"):
        tb.Runtime(session).bind(tb.OpRequest("softmax", [foreign], [tb.TensorSpec(DType.F32, (4, 64))]), y)
    with pytest.raises(tb.ExecutionError, match="same shape"):  # an operator's checks run at every enqueue
        tb.Runtime(session).bind(tb.OpRequest("softmax", [y], [tb.TensorSpec(DType.F32, (2, 64))]), y).enqueue()


def test_bound_requests_from_two_threads(session):
    """Two host threads on one stream, with an operator that takes the stream's workspace."""
    import threading
    rt = tb.Runtime(session)
    batch, h, hk, d, page = 3, 8, 2, 128, 16
    lens = [3000, 70, 1100]
    need = [-(-n // page) for n in lens]
    table = np.full((batch, max(need)), -1, np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = np.arange(at, at + n)
        at += n
    cache = [upload(session, rt.stream, rows((at, page, hk, d), DType.BF16, 900 + i), DType.BF16) for i in range(2)]
    ins = cache + [ints(session, rt, table), ints(session, rt, lens)]
    bound = []
    for tokens in (1, 20):  # the token kernel and the tile kernel, whose workspaces differ in size
        q = upload(session, rt.stream, rows((batch * tokens, h, d), DType.BF16, 910), DType.BF16)
        cu = ints(session, rt, np.arange(batch + 1) * tokens)
        request = tb.OpRequest("attention.paged", [q, *ins, cu], [spec_of(q)], {"max_query_len": tokens})
        bound.append(rt.bind(request, tb.TensorHandle.allocate(session, DType.BF16, q.shape)))
        bound[-1].enqueue()
    session.synchronize(rt.stream)
    want = [b.outputs[0].to_numpy(rt.stream) for b in bound]
    threads = [threading.Thread(target=lambda b=b: [b.enqueue() for _ in range(200)]) for b in bound]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    session.synchronize(rt.stream)
    for b, w in zip(bound, want):
        np.testing.assert_array_equal(b.outputs[0].to_numpy(rt.stream), w)


@pytest.mark.parametrize("tokens", [1, 40])
def test_graphs_of_one_stream_replay_side_by_side(session, tokens):
    """Two graphs captured on one stream, and eager calls, keep their partial results apart: replayed at
    the same time on three streams, each gives its own inputs' result every time."""
    rt = tb.Runtime(session)
    batch, h, hk, d, page, n = 2, 8, 2, 128, 16, 5000
    pages = -(-n // page)
    table = ints(session, rt, np.arange(batch * pages).reshape(batch, pages))
    lens, cu = ints(session, rt, [n, n - 700]), ints(session, rt, np.arange(batch + 1) * tokens)
    graphs, outs, want, bound = [], [], [], []
    for g in range(3):
        cache = [upload(session, rt.stream, rows((batch * pages, page, hk, d), DType.F16, 950 + 3 * g + i), DType.F16)
                 for i in range(2)]
        q = upload(session, rt.stream, rows((batch * tokens, h, d), DType.F16, 960 + g), DType.F16)
        out = tb.TensorHandle.allocate(session, DType.F16, q.shape)
        request = tb.OpRequest("attention.paged", [q, *cache, table, lens, cu], [spec_of(out)],
                               {"max_query_len": tokens})
        bound.append(rt.bind(request, out))
        bound[-1].enqueue()
        want.append(out.to_numpy(rt.stream))
        outs.append(out)
        if g < 2:
            session.capture_begin(rt.stream)
            bound[-1].enqueue()
            graphs.append(session.capture_end(rt.stream))
    session.synchronize(rt.stream)
    zero = np.zeros(outs[0].shape, np.float16)
    for t in outs:
        session.wait(session.upload(rt.stream, t.buffer, zero))
    streams = [session.create_stream() for _ in range(2)]
    for _ in range(100):
        graphs[0].launch(streams[0])
        graphs[1].launch(streams[1])
        bound[2].enqueue()
    for st in (*streams, rt.stream):
        session.synchronize(st)
    for t, w in zip(outs, want):
        np.testing.assert_array_equal(t.to_numpy(rt.stream), w)
    for g in graphs:
        g.release()


def test_an_invalid_capture_leaves_the_stream_usable(session):
    rt = tb.Runtime(session)
    x = upload(session, rt.stream, rows((40, 4, 64), DType.BF16, 1), DType.BF16)
    cu = ints(session, rt, [0, 40])
    b = rt.bind(tb.OpRequest("attention.varlen", [x, x, x, cu], [spec_of(x)], {}),
                tb.TensorHandle.allocate(session, DType.BF16, x.shape))
    b.enqueue()
    want = b.outputs[0].to_numpy(rt.stream)
    session.capture_begin(rt.stream)
    b.enqueue()
    with pytest.raises(tb.HalError):  # a host wait on a capturing stream invalidates the capture
        session.synchronize(rt.stream)
    with pytest.raises(tb.HalError):
        session.capture_end(rt.stream)
    b.enqueue()
    np.testing.assert_array_equal(b.outputs[0].to_numpy(rt.stream), want)


def test_workspaces_come_and_go_beside_a_capture(session):
    """While one stream is captured, another's workspace grows (its old one is freed) and an older
    graph of attention operators is released: the capture stays valid, and nothing is put into it."""
    rt = tb.Runtime(session)
    other = tb.Runtime(session)
    batch, h, hk, d, page, n = 2, 8, 2, 128, 16, 5000
    pages = -(-n // page)
    cache = [upload(session, rt.stream, rows((batch * pages, page, hk, d), DType.BF16, 980 + i), DType.BF16)
             for i in range(2)]
    table = ints(session, rt, np.arange(batch * pages).reshape(batch, pages))
    lens = ints(session, rt, [n, n - 700])

    def bind(runtime, tokens):
        q = upload(session, rt.stream, rows((batch * tokens, h, d), DType.BF16, 990 + tokens), DType.BF16)
        cu = ints(session, rt, np.arange(batch + 1) * tokens)
        request = tb.OpRequest("attention.paged", [q, *cache, table, lens, cu], [spec_of(q)],
                               {"max_query_len": tokens})
        return runtime.bind(request, tb.TensorHandle.allocate(session, DType.BF16, q.shape))

    small, large, mine = bind(other, 1), bind(other, 40), bind(rt, 3)
    reference = bind(rt, 40)
    for b in (small, mine, reference):  # (and their modules are loaded before the capture)
        b.enqueue()
    session.synchronize(rt.stream)
    session.synchronize(other.stream)
    want, want_large = (b.outputs[0].to_numpy(rt.stream) for b in (mine, reference))
    session.capture_begin(rt.stream)
    mine.enqueue()
    old = session.capture_end(rt.stream)
    old.launch(rt.stream)
    session.synchronize(rt.stream)

    session.capture_begin(rt.stream)
    mine.enqueue()
    with pytest.raises(tb.HalError, match="into a capture"):
        old.launch(rt.stream)
    large.enqueue()
    old.release()
    graph = session.capture_end(rt.stream)
    session.synchronize(other.stream)
    session.wait(session.upload(rt.stream, mine.outputs[0].buffer, np.zeros(want.shape, np.uint16)))
    graph.launch(rt.stream)
    session.synchronize(rt.stream)
    np.testing.assert_array_equal(mine.outputs[0].to_numpy(rt.stream), want)
    np.testing.assert_array_equal(large.outputs[0].to_numpy(other.stream), want_large)
    graph.release()

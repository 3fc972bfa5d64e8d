"""Serving operators of the library as measurable cases: attention over packed prompts
("attention.varlen"), attention of new tokens over a paged cache ("attention.paged"), the
cache write ("kv_cache.append") and the page and slot assignment of a step ("kv_cache.plan").

`run` computes a case with elementary torch operations, or, where `own` is true, with the
library's operators. Both take what `prepare` made.
"""
import math
import random

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
_runtime = None


# ---------------------------------------------------------------- cases
def listed():
    return [
        # Four short questions packed into one call of a small model: the launch counts.
        dict(name="varlen_short_d64", op="varlen", type="bf16", heads=8, kv_heads=2, dim=64, batch=4, low=7, high=190,
             cross=False, causal=True, packed=True, pad=0, shape_seed=11),
        # A prompt step of a server: sixteen ragged prompts, grouped heads, Q, K and V in one projection's output.
        dict(name="varlen_prompts_gqa", op="varlen", type="bf16", heads=32, kv_heads=8, dim=128, batch=16, low=33,
             high=2048, cross=False, causal=True, packed=True, pad=13, shape_seed=12),
        # Training-sized prompts of up to 4096 tokens, 32 heads each with keys of its own.
        dict(name="varlen_long_mha", op="varlen", type="bf16", heads=32, kv_heads=32, dim=128, batch=8, low=2900,
             high=4096, cross=False, causal=True, packed=False, pad=0, shape_seed=13),
        # Decoder tokens over encoder states of other lengths, every key seen, half precision.
        dict(name="varlen_cross_f16_d64", op="varlen", type="f16", heads=16, kv_heads=16, dim=64, batch=24, low=40,
             high=1500, cross=True, causal=False, packed=False, pad=0, shape_seed=14),
        # One user waiting for the next token of a short chat.
        dict(name="paged_token_one", op="paged", type="bf16", heads=32, kv_heads=8, dim=128, batch=1, ctx_low=1017,
             ctx_high=1017, new_low=1, new_high=1, page=16, pad=0, shape_seed=21),
        # The decode step of a busy server: 64 chats of very different lengths.
        dict(name="paged_token_batch", op="paged", type="bf16", heads=64, kv_heads=8, dim=128, batch=64, ctx_low=300,
             ctx_high=8192, new_low=1, new_high=1, page=16, pad=0, shape_seed=22),
        # Four long documents being answered token by token, a cache of about 2 GB.
        dict(name="paged_token_long_f16", op="paged", type="f16", heads=32, kv_heads=8, dim=128, batch=4,
             ctx_low=110000, ctx_high=131071, new_low=1, new_high=1, page=32, pad=0, shape_seed=23),
        # A chunk of each prompt while others only add a token: prompts processed in pieces.
        dict(name="paged_chunk_mixed", op="paged", type="bf16", heads=32, kv_heads=8, dim=128, batch=8, ctx_low=900,
             ctx_high=8192, new_low=1, new_high=1024, page=64, pad=5, shape_seed=24),
        # The cache write of a decode step.
        dict(name="append_tokens", op="append", type="bf16", kv_heads=8, dim=128, tokens=64, page=16, pages=4096,
             packed=True, shape_seed=31),
        # The cache write of a prompt step, 16384 tokens.
        dict(name="append_prompts", op="append", type="bf16", kv_heads=8, dim=128, tokens=16384, page=16, pages=4096,
             packed=True, shape_seed=32),
        # Pages and slots of a decode step of 64 chats.
        dict(name="plan_tokens", op="plan", batch=64, ctx_low=1, ctx_high=8192, new_low=1, new_high=1, page=16, pad=0,
             shape_seed=41),
        # Pages and slots of a step that admits many prompts at once.
        dict(name="plan_prompts", op="plan", batch=700, ctx_low=1, ctx_high=4096, new_low=1, new_high=400, page=16,
             pad=100, shape_seed=42),
    ]


def _log_uniform(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))))))


def draw(rng):
    op = rng.choice(["varlen", "paged", "paged", "append", "plan"])
    seed = rng.randrange(1 << 30)
    if op == "varlen":
        kv = rng.choice([1, 2, 4, 8, 16])
        group = rng.choice([1, 2, 3, 4, 6, 8])
        case = dict(op=op, type=rng.choice(["bf16", "f16"]), heads=kv * group, kv_heads=kv,
                    dim=rng.choice([64, 128]), batch=_log_uniform(rng, 1, 32), low=1,
                    high=_log_uniform(rng, 1, 4096), cross=rng.random() < 0.3, causal=rng.random() < 0.7,
                    packed=False, pad=rng.choice([0, 0, 1, 29]), shape_seed=seed)
        case["packed"] = not case["cross"] and rng.random() < 0.5
        while case["batch"] * case["heads"] * case["high"] ** 2 > 8 * 32 * 4096 ** 2 // 4:
            case["high"] = max(1, case["high"] // 2)
        return case
    if op == "paged":
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 4, 5, 8])
        case = dict(op=op, type=rng.choice(["bf16", "f16"]), heads=kv * group, kv_heads=kv,
                    dim=rng.choice([64, 128]), batch=_log_uniform(rng, 1, 96), ctx_low=1,
                    ctx_high=_log_uniform(rng, 1, 65536), new_low=1, new_high=rng.choice([1, 1, 3, 8, 100, 700]),
                    page=rng.choice([8, 16, 16, 32, 64, 128]), pad=rng.choice([0, 0, 3]), shape_seed=seed)
        while case["batch"] * case["ctx_high"] * kv * case["dim"] > 1 << 28 or \
                case["batch"] * case["heads"] * case["new_high"] * case["ctx_high"] > 1 << 30:
            case["ctx_high"] = max(1, case["ctx_high"] // 2)
        return case
    if op == "append":
        page = rng.choice([8, 16, 32, 64])
        return dict(op=op, type=rng.choice(["bf16", "f16"]), kv_heads=rng.choice([1, 2, 4, 8]),
                    dim=rng.choice([64, 80, 128]), tokens=_log_uniform(rng, 1, 16384), page=page, pages=32768 // page,
                    packed=rng.random() < 0.5, shape_seed=seed)
    return dict(op=op, batch=_log_uniform(rng, 1, 700), ctx_low=1, ctx_high=_log_uniform(rng, 1, 4096), new_low=1,
                new_high=_log_uniform(rng, 1, 400), page=rng.choice([1, 8, 16, 24, 64]), pad=rng.choice([0, 7]),
                shape_seed=seed)


def _lengths(case, low, high, salt):
    """The lengths of the case's requests: spread over their logarithm, the longest one among them."""
    rng = random.Random(case["shape_seed"] * 16 + salt)
    n = case["batch"]
    got = [_log_uniform(rng, low, high) for _ in range(n)]
    got[rng.randrange(n)] = high
    return got


def _varlen_lengths(case):
    q = _lengths(case, case["low"], case["high"], 0)
    return q, (_lengths(case, case["low"], case["high"], 1) if case["cross"] else q)


def _paged_lengths(case):
    """Tokens already cached, and new ones, of each request."""
    return (_lengths(case, case["ctx_low"], case["ctx_high"], 2), _lengths(case, case["new_low"], case["new_high"], 3))


def _prefix(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


# ---------------------------------------------------------------- inputs
def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _rows(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 7919 + case["shape_seed"])
    state = {"varlen": _prepare_varlen, "paged": _prepare_paged, "append": _prepare_append,
             "plan": _prepare_plan}[case["op"]](case, gen)
    state["case"] = case
    if own:
        _bind(state)
    return state


def _prepare_varlen(case, gen):
    dtype, h, hk, d = _TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"]
    lq, lk = _varlen_lengths(case)
    tq, tk = sum(lq) + case["pad"], sum(lk) + (0 if case["cross"] else case["pad"])
    if case["packed"]:  # one projection's output, [token, (heads + 2 kv_heads) x dim]
        qkv = _rows(gen, (tq, h + 2 * hk, d), dtype)
        q, k, v = qkv[:, :h], qkv[:, h:h + hk], qkv[:, h + hk:]
    else:
        q, k, v = _rows(gen, (tq, h, d), dtype), _rows(gen, (tk, hk, d), dtype), _rows(gen, (tk, hk, d), dtype)
    return dict(q=q, k=k, v=v, cu_q=_int32(_prefix(lq)), cu_k=_int32(_prefix(lk)), max_q=max(lq), max_k=max(lk),
                out=torch.zeros(tq, h, d, dtype=dtype, device="cuda"))


def _page_tables(lengths, page, gen, spare=3):
    """A block table over shuffled pages for caches of these lengths; unused entries hold -1."""
    need = torch.tensor([-(-n // page) for n in lengths])
    total, width = int(need.sum()), int(need.max())
    pages = total + spare
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    used = torch.arange(width)[None, :] < need[:, None]
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    table[used.cuda()] = order[:total]
    return table, pages


def _prepare_paged(case, gen):
    dtype, h, hk, d, page = _TYPES[case["type"]], case["heads"], case["kv_heads"], case["dim"], case["page"]
    ctx, new = _paged_lengths(case)
    lengths = [a + b for a, b in zip(ctx, new)]
    table, pages = _page_tables(lengths, page, gen)
    tq = sum(new) + case["pad"]
    return dict(q=_rows(gen, (tq, h, d), dtype), k_cache=_rows(gen, (pages, page, hk, d), dtype),
                v_cache=_rows(gen, (pages, page, hk, d), dtype), table=table, lens=_int32(lengths),
                cu_q=_int32(_prefix(new)), max_q=max(new), max_k=max(lengths),
                out=torch.zeros(tq, h, d, dtype=dtype, device="cuda"))


def _prepare_append(case, gen):
    dtype, hk, d, t, page = _TYPES[case["type"]], case["kv_heads"], case["dim"], case["tokens"], case["page"]
    if case["packed"]:
        kv = _rows(gen, (t, 2 * hk, d), dtype)
        k, v = kv[:, :hk], kv[:, hk:]
    else:
        k, v = _rows(gen, (t, hk, d), dtype), _rows(gen, (t, hk, d), dtype)
    slots = torch.randperm(case["pages"] * page, generator=gen, device="cuda")[:t].to(torch.int32)
    slots[torch.rand(t, generator=gen, device="cuda") < 0.02] = -1  # rows that pad the batch
    shape = (case["pages"], page, hk, d)
    return dict(k=k, v=v, slots=slots, k_cache=_rows(gen, shape, dtype), v_cache=_rows(gen, shape, dtype))


def _prepare_plan(case, gen):
    ctx, new = _paged_lengths(case)
    page = case["page"]
    width = max(-(-(a + b) // page) for a, b in zip(ctx, new))
    held, _ = _page_tables(ctx, page, gen)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    table[:, :held.shape[1]] = held
    first = int(held.max()) + 1
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(ctx, new))
    free = torch.randperm(need + 5, generator=gen, device="cuda").to(torch.int32) + first
    tokens = sum(new) + case["pad"]
    lens = torch.zeros(case["batch"], dtype=torch.int32, device="cuda")
    return dict(ctx=_int32(ctx), new=_int32(new), free=free, table=table, lens=lens,
                cu=torch.zeros(case["batch"] + 1, dtype=torch.int32, device="cuda"),
                slots=torch.zeros(tokens, dtype=torch.int32, device="cuda"),
                status=torch.zeros(2, dtype=torch.int32, device="cuda"))


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        state["bound"].enqueue()
        return state["outputs"]
    return {"varlen": _run_varlen, "paged": _run_paged, "append": _run_append,
            "plan": _run_plan}[state["case"]["op"]](state)


def _attend(q, k, v, visible, scale):
    """softmax(scale q k^T) v in 32 bits for padded q [B, I, H, D] and k, v [B, J, K, D]; row i of
    request b sees its first visible[b, i] keys, and a row that sees none gives zeros."""
    b, i, h, d = q.shape
    kv = k.shape[2]
    scores = torch.einsum("bikgd,bjkd->bkgij", q.float().view(b, i, kv, h // kv, d) * scale, k.float())
    hidden = torch.arange(k.shape[1], device=q.device) >= visible[:, None, None, :, None]
    scores.masked_fill_(hidden, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    weights = scores.sub_(top).exp_()
    total = weights.sum(-1).clamp_min(torch.finfo(torch.float32).tiny)
    out = torch.einsum("bkgij,bjkd->bkgid", weights, v.float()) / total[..., None]
    return out.permute(0, 3, 1, 2, 4).reshape(b, i, h, d)


def _padded(rows, cu, longest):
    """Packed rows [T, ...] as [B, longest, ...]; the places behind a request repeat some row."""
    at = cu[:-1, None].long() + torch.arange(longest, device=rows.device)
    return rows[at.clamp_max(rows.shape[0] - 1)]


def _into(out, cu, padded):
    """`out` with each request's rows of `padded` [B, I, H, D] at their packed places."""
    lengths = (cu[1:] - cu[:-1]).long()
    steps = torch.arange(padded.shape[1], device=out.device)
    here = steps < lengths[:, None]
    result = out.clone()
    result[(cu[:-1, None].long() + steps)[here]] = padded[here].to(out.dtype)
    return result


def _visible(lq, lk, longest, causal):
    steps = torch.arange(longest, device=lq.device)
    seen = lk[:, None].long().expand(-1, longest)
    return (lk - lq)[:, None].long() + steps + 1 if causal else seen


def _run_varlen(s):
    cu_q, cu_k = s["cu_q"], s["cu_k"]
    visible = _visible(cu_q[1:] - cu_q[:-1], cu_k[1:] - cu_k[:-1], s["max_q"], s["case"]["causal"])
    out = _attend(_padded(s["q"], cu_q, s["max_q"]), _padded(s["k"], cu_k, s["max_k"]),
                  _padded(s["v"], cu_k, s["max_k"]), visible, 1.0 / math.sqrt(s["q"].shape[2]))
    return _into(s["out"], cu_q, out)


def _run_paged(s):
    page, cu_q = s["case"]["page"], s["cu_q"]
    steps = torch.arange(s["max_k"], device="cuda")
    slots = s["table"].long().clamp_min(0)[:, steps // page] * page + steps % page
    visible = _visible(cu_q[1:] - cu_q[:-1], s["lens"], s["max_q"], True)
    out = _attend(_padded(s["q"], cu_q, s["max_q"]), s["k_cache"].flatten(0, 1)[slots],
                  s["v_cache"].flatten(0, 1)[slots], visible, 1.0 / math.sqrt(s["q"].shape[2]))
    return _into(s["out"], cu_q, out)


def _run_append(s):
    kept = s["slots"] >= 0
    at = s["slots"][kept].long()
    s["k_cache"].flatten(0, 1)[at] = s["k"][kept]
    s["v_cache"].flatten(0, 1)[at] = s["v"][kept]
    return s["k_cache"], s["v_cache"]


def _run_plan(s):
    page, tokens = s["case"]["page"], s["slots"].shape[0]
    ctx, new, free, width = s["ctx"].long(), s["new"].long(), s["free"].long(), s["table"].shape[1]
    held, wanted = -(-ctx // page), -(-(ctx + new) // page)
    end = new.cumsum(0)
    fits = (wanted <= width) & (end <= tokens)
    need = torch.where(fits, wanted - held, 0)
    last = need.cumsum(0)
    served = fits & (last <= free.shape[0])
    first = last - need
    column = torch.arange(width, device="cuda")
    fresh = (column >= held[:, None]) & (column < wanted[:, None]) & served[:, None]
    from_free = free[(first[:, None] + column - held[:, None]).clamp(0, free.shape[0] - 1)]
    table = torch.where(fresh, from_free, s["table"].long())
    lens = torch.where(served, ctx + new, ctx)
    step = torch.arange(tokens, device="cuda")
    owner = torch.searchsorted(end, step, right=True)
    inside = owner.clamp_max(ctx.shape[0] - 1)
    position = ctx[inside] + step - (end - new)[inside]
    slots = table[inside, (position // page).clamp_max(width - 1)] * page + position % page
    slots = torch.where((owner < ctx.shape[0]) & served[inside], slots, -1)
    cu = torch.cat([end.new_zeros(1), end])
    status = torch.stack([torch.where(served, need, 0).sum(), (~served).sum()])
    return tuple(x.to(torch.int32) for x in (table, lens, cu, slots, status))


# ---------------------------------------------------------------- the library's operators
def _handle(session, tensor):
    """A torch tensor as a tensor of the session: the same memory, its strides kept."""
    from titan_rs_b200 import TensorHandle
    from titan_rs_b200.kernel_abi import DType
    kinds = {torch.bfloat16: DType.BF16, torch.float16: DType.F16, torch.int32: DType.I32}
    extent = 1 + sum((n - 1) * st for n, st in zip(tensor.shape, tensor.stride()))
    return TensorHandle(session, session.wrap(tensor.data_ptr(), extent * tensor.element_size()),
                        kinds[tensor.dtype], tuple(tensor.shape), tuple(tensor.stride()))


_CALLS = {
    "varlen": ("attention.varlen", ("q", "k", "v", "cu_q", "cu_k"), ("out",)),
    "paged": ("attention.paged", ("q", "k_cache", "v_cache", "table", "lens", "cu_q"), ("out",)),
    "append": ("kv_cache.append", ("k", "v", "slots"), ("k_cache", "v_cache")),
    "plan": ("kv_cache.plan", ("ctx", "new", "free"), ("table", "lens", "cu", "slots", "status")),
}


def _bind(state):
    """The request that a serving loop builds once over its buffers and enqueues every step."""
    global _runtime
    import titan_rs_b200 as tb
    if _runtime is None:
        _runtime = tb.Runtime(tb.Session(0))
    session, case = _runtime.session, state["case"]
    name, inputs, outputs = _CALLS[case["op"]]
    attrs = {}
    if case["op"] == "varlen":
        attrs = {"causal": case["causal"]}
    elif case["op"] == "paged":
        attrs = {"max_query_len": case["new_high"]}
    elif case["op"] == "plan":
        attrs = {"page_size": case["page"]}
    ins, outs = ([_handle(session, state[key]) for key in keys] for keys in (inputs, outputs))
    specs = [tb.TensorSpec(t.dtype, t.shape, t.strides) for t in outs]
    state["bound"] = _runtime.bind(tb.OpRequest(name, ins, specs, attrs), output=outs)
    state["outputs"] = state["out"] if len(outputs) == 1 else tuple(state[key] for key in outputs)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "append":
        return {"bytes": 8 * case["tokens"] * case["kv_heads"] * case["dim"] + 4 * case["tokens"], "flops": 0}
    if op == "plan":
        ctx, new = _paged_lengths(case)
        page = case["page"]
        fresh = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(ctx, new))
        partial = sum(a % page != 0 for a in ctx)
        return {"bytes": 4 * (4 * case["batch"] + 1 + 2 * fresh + partial + sum(new) + case["pad"] + 2), "flops": 0}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if op == "varlen":
        lq, lk = _varlen_lengths(case)
        causal = case["causal"]
    else:
        ctx, lq = _paged_lengths(case)
        lk = [a + b for a, b in zip(ctx, lq)]
        causal = True
    pairs = sum(_pairs(a, b) if causal else a * b for a, b in zip(lq, lk))
    moved = 4 * h * d * sum(lq) + 4 * hk * d * sum(lk)
    index = 4 * (2 * case["batch"] + 2)
    if op == "paged":
        index += 4 * sum(-(-n // case["page"]) for n in lk)
    return {"bytes": moved + index, "flops": 4 * h * d * pairs}


def _pairs(lq, lk):
    """Query and key pairs under the causal mask: row i sees max(0, lk - lq + i + 1) keys."""
    hidden = max(lk - lq, 0)
    return (lk * (lk + 1) - hidden * (hidden + 1)) // 2


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "append":
        k, v = s["k_cache"].double().flatten(0, 1), s["v_cache"].double().flatten(0, 1)
        rows = (s["slots"] >= 0).nonzero()[:, 0]
        at = s["slots"].long()[rows]
        k.index_copy_(0, at, s["k"].double()[rows])
        v.index_copy_(0, at, s["v"].double()[rows])
        return k.view(s["k_cache"].shape), v.view(s["v_cache"].shape)
    if op == "plan":
        return None
    out = s["out"].double()
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    cu_q = s["cu_q"].tolist()
    cu_k = s["cu_k"].tolist() if op == "varlen" else None
    for b in range(case["batch"]):
        q = s["q"][cu_q[b]:cu_q[b + 1]].double()
        if op == "varlen":
            k, v = (s[key][cu_k[b]:cu_k[b + 1]].double() for key in ("k", "v"))
        else:
            n = int(s["lens"][b])
            pages = s["table"][b, :-(-n // case["page"])].long()
            k, v = (s[key][pages].reshape(-1, hk, d)[:n].double() for key in ("k_cache", "v_cache"))
        lq, lk = q.shape[0], k.shape[0]
        keep = torch.ones(lq, lk, dtype=torch.bool, device="cuda")
        if op == "paged" or case["causal"]:
            keep = keep.tril(lk - lq)
        empty = ~keep.any(1)
        for g in range(hk):
            heads = slice(g * (h // hk), (g + 1) * (h // hk))
            a = torch.matmul(q[:, heads].transpose(0, 1), k[:, g].t()) / math.sqrt(d)
            p = torch.softmax(a.masked_fill(~keep, -math.inf), -1).masked_fill(empty[:, None], 0.0)
            out[cu_q[b]:cu_q[b + 1], heads] = torch.matmul(p, v[:, g]).transpose(0, 1)
    return out

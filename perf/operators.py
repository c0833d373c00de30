"""What the operators of a serving step with a shared prompt are measured on.

Four kinds of calls, each through an ``InferenceSession`` with bound buffers, the way the serving loop makes them:

* ``layout``: com.ortb200.PagedBatchLayout - block table, packing, positions and cache slots of a batch out of the lengths of its requests;
* ``attention``: com.ortb200.SharedPrefixPagedAttention - rotary, cache append and attention over paged caches for a batch whose sequences begin with
  the same tokens (a system prompt, a document that many questions are asked about);
* ``score``: com.ortb200.TokenLogProbs - log probabilities of given tokens, entropy and the best alternatives out of logits;
* ``train``: the same and its backward half, com.ortb200.TokenLogProbsGrad, as a policy-gradient step has them.

Lengths belong to the case, values to the seed.
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FUSED = "com.ortb200"


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a small chat server: one token for each of 24 requests, the call whose latency every step pays
        dict(name="layout_24", kind="layout", requests=24, blocks=64, block=256, past=9000, single=1.0, new=1),
        # a step that admits prompts and continues others, small blocks
        dict(name="layout_mixed_160", kind="layout", requests=160, blocks=640, block=16, past=7000, single=0.8, new=900),
        # a large offline batch with long tables
        dict(name="layout_1000", kind="layout", requests=1000, blocks=4096, block=16, past=60000, single=0.9, new=600),
        # two users of one short system prompt
        dict(name="attention_2x300", kind="attention", dtype="bf16", heads=32, kv=8, head=128, block=256, batch=2, prefix=300, past=60, new=1, cap=0.0),
        # a chat server: 24 requests behind a system prompt of 2000 tokens
        dict(name="attention_24x2000", kind="attention", dtype="bf16", heads=32, kv=8, head=128, block=256, batch=24, prefix=2000, past=400, new=1, cap=0.0),
        # samples of one long problem: 64 continuations of 8192 tokens
        dict(name="attention_64x8192", kind="attention", dtype="bf16", heads=64, kv=8, head=128, block=128, batch=64, prefix=8192, past=700, new=1, cap=0.0),
        # many readers of one document, heads of 64 that share no key head, small blocks
        dict(name="attention_180x20011", kind="attention", dtype="fp16", heads=16, kv=16, head=64, block=16, batch=180, prefix=20011, past=333, new=1, cap=0.0),
        # questions about one document: prompts of up to 150 tokens join, groups of seven heads
        dict(name="attention_questions_24x6000", kind="attention", dtype="bf16", heads=28, kv=4, head=128, block=64, batch=24, prefix=6000, past=90, new=150, cap=0.0),
        # answers of a small step with five alternatives each
        dict(name="score_6", kind="score", dtype="bf16", rows=6, vocab=128256, top=5),
        # log probabilities of a prompt's own tokens, a vocabulary of odd size, 32-bit logits
        dict(name="score_2000", kind="score", dtype="fp32", rows=2000, vocab=50257, top=1),
        # a small policy-gradient step
        dict(name="train_300", kind="train", dtype="fp16", rows=300, vocab=32000, top=0),
        # a large one: 4096 tokens over a long vocabulary
        dict(name="train_4096", kind="train", dtype="bf16", rows=4096, vocab=128256, top=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["layout", "attention", "attention", "questions", "score", "train"])
    if kind == "layout":
        block, requests = rng.choice([16, 32, 64, 256]), _log(rng, 1, 1000)
        past = _log(rng, 30, 60000)
        new = rng.choice([1, _log(rng, 2, 600)])
        return dict(kind=kind, requests=requests, blocks=(past + new) // block + 1 + rng.randint(0, 40), block=block, past=past,
                    single=rng.choice([0.5, 0.9]), new=new)
    if kind in ("attention", "questions"):
        heads, kv, head = rng.choice([(32, 8, 128), (64, 8, 128), (16, 16, 64), (28, 4, 128), (24, 8, 64), (32, 2, 128)])
        several = kind == "questions"
        batch, new = (_log(rng, 1, 40), _log(rng, 2, 150)) if several else (_log(rng, 1, 200), 1)
        prefix = _log(rng, 64, max(100, min(20000, 300000000 // (batch * new * heads))))
        return dict(kind="attention", dtype=rng.choice(["bf16", "fp16"]), heads=heads, kv=kv, head=head, block=rng.choice([16, 32, 64, 128, 256]), batch=batch,
                    prefix=prefix, past=_log(rng, 1, 700), new=new, cap=rng.choice([0.0, 0.0, 30.0]))
    dtype, vocab = rng.choice(["bf16", "fp16", "fp32"]), rng.choice([_log(rng, 1000, 200000), 32000, 50257, 128256])
    most = 4096 * 128256 // (2 * vocab) if kind == "train" else 60000000 // vocab
    return dict(kind=kind, dtype=dtype, rows=_log(rng, 1, min(8000, most)), vocab=vocab, top=0 if kind == "train" else rng.choice([0, 1, 5, 20]))


# ---------------------------------------------------------------------------------------------------------- shapes of a case
def _lengths(case):
    """[(tokens held, new tokens)] of the requests; for attention the tokens held are those behind the shared prefix."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["kind"] == "layout":
        new = lambda: 1 if r.random() < case["single"] else r.randint(1, case["new"])  # noqa: E731
        return [(r.randint(0, case["past"]), new()) for _ in range(case["requests"])]
    return [(r.randint(case["past"] // 4, case["past"]), r.randint((case["new"] + 3) // 4, case["new"])) for _ in range(case["batch"])]


def work(case):
    if case["kind"] == "layout":
        pairs, s = _lengths(case), case["block"]
        tokens = sum(n for _, n in pairs)
        fresh = sum((p + n + s - 1) // s - (p + s - 1) // s for p, n in pairs)
        return {"bytes": 8 * case["requests"] * case["blocks"] + 16 * tokens + 12 * case["requests"] + 4 * fresh + 8, "flops": 4 * tokens}
    if case["kind"] == "attention":
        pairs, size, entry = _lengths(case), 2, 2 * case["kv"] * case["head"] * 2
        tokens = sum(n for _, n in pairs)
        own_keys = sum(p + n for p, n in pairs)
        seen = sum(n * case["prefix"] + n * p + n * (n + 1) // 2 for p, n in pairs)
        return {"bytes": entry * (case["prefix"] + own_keys + tokens) + 2 * size * tokens * case["heads"] * case["head"],
                "flops": 4 * case["heads"] * case["head"] * seen}
    size = 4 if case["dtype"] == "fp32" else 2
    passes = 2 if case["kind"] == "train" else 1
    values = case["rows"] * case["vocab"]
    return {"bytes": passes * size * values + case["rows"] * (20 + 12 * case["top"]), "flops": 4 * passes * values}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _normal(gen, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _layout_inputs(case, seed):
    g, pairs, s = _gen(seed, 1), _lengths(case), case["block"]
    past, new = _ints([p for p, _ in pairs]), _ints([n for _, n in pairs])
    held, total = (past.long() + s - 1) // s, (past.long() + new + s - 1) // s
    pool = int(total.sum()) + 64
    order = torch.randperm(pool, generator=g, device="cuda").int()
    column = torch.arange(case["blocks"], device="cuda").unsqueeze(0)
    index = (held.cumsum(0) - held).unsqueeze(1) + column
    table = torch.where(column < held.unsqueeze(1), order[index.clamp(max=pool - 1)], torch.zeros_like(order[:1]))
    ids = torch.randint(0, 32000, (sum(n for _, n in pairs),), generator=g, device="cuda")
    return dict(past=past, new=new, table=table.contiguous(), free=order[int(held.sum()):].contiguous(), ids=ids)


def _attention_inputs(case, seed):
    g, pairs, dt = _gen(seed, 2), _lengths(case), DTYPES[case["dtype"]]
    s, prefix, n = case["block"], case["prefix"], case["heads"] + 2 * case["kv"]
    past, new = [prefix + p for p, _ in pairs], [n for _, n in pairs]
    shared = prefix // s                                   # whole blocks of the prefix are the same ones in every row of the table
    mine = [(p + n + s - 1) // s - shared for p, n in zip(past, new)]
    pool = shared + sum(mine) + 8
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.zeros(len(pairs), shared + max(mine), dtype=torch.int32, device="cuda")
    table[:, :shared] = order[:shared]
    at = shared
    for b, m in enumerate(mine):
        table[b, shared:shared + m] = order[at:at + m]
        at += m
    caches = [_normal(g, (pool, s, case["kv"], case["head"]), dt) for _ in range(2)]
    rest = prefix - shared * s                             # the tokens of a block that the prefix fills in part: a copy per sequence
    if rest:
        blocks = table[:, shared].long()
        for c in caches:
            c[blocks, :rest] = c[blocks[0], :rest].clone()
    tokens = sum(new)
    cum = torch.tensor([0] + new).cumsum(0)
    positions = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).cuda()
    seq = torch.repeat_interleave(torch.arange(len(new)), torch.tensor(new)).cuda()
    slots = table[seq, positions // s].long() * s + positions % s
    qkv = _normal(g, (tokens, n * case["head"]), dt)
    rows = max(p + n for p, n in zip(past, new))
    angle = torch.arange(rows, device="cuda").double().unsqueeze(1) * 10000.0 ** (-torch.arange(case["head"] // 2, device="cuda").double() * 2 / case["head"])
    return dict(qkv=qkv, key_cache=caches[0], value_cache=caches[1], cum=cum.int().cuda(), past=_ints(past), table=table, prefix=_ints([prefix]),
                cos=angle.cos().to(dt), sin=angle.sin().to(dt), positions=positions, slots=slots, seq=seq)


def _score_inputs(case, seed):
    """Logits of a language model: a broad bulk and a few tokens far above it in every row; most given tokens are likely ones."""
    g, rows, vocab = _gen(seed, 3), case["rows"], case["vocab"]
    logits = _normal(g, (rows, vocab), DTYPES[case["dtype"]], 2.0)
    likely = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
    logits.scatter_(1, likely, (_normal(g, (rows, 8), torch.float32, 1.5) + 11).to(logits.dtype))
    other = torch.randint(0, vocab, (rows,), generator=g, device="cuda")
    tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.8, likely[:, 0], other)
    grads = [torch.randn(rows, generator=g, device="cuda") for _ in range(2)]
    return dict(logits=logits, tokens=tokens, d_log_prob=grads[0], d_entropy=grads[1] * 0.1)


# ------------------------------------------------------------------------------------------------------------ prepare and run
def _bound(nodes, ins, outs):
    """A session over one operator (or a forward and its backward half) with every input and output bound to a device tensor."""
    import onnxruntime_b200 as ort
    from onnxruntime_b200 import onnx_lite as ol
    T = ol.TensorProto
    types = {torch.bfloat16: T.BFLOAT16, torch.float16: T.FLOAT16, torch.float32: T.FLOAT, torch.int32: T.INT32, torch.int64: T.INT64}
    info = lambda n, t: ol.make_tensor_value_info(n, types[t.dtype], list(t.shape))  # noqa: E731
    graph = ol.make_graph([ol.make_node(op, i, o, domain=FUSED, **attrs) for op, i, o, attrs in nodes], "step", [info(n, t) for n, t in ins.items()],
                          [info(n, t) for n, t in outs.items()])
    sess = ort.InferenceSession(ol.make_model(graph, opset=17, extra_opsets={FUSED: 1}).serialize(), providers=[("CUDAExecutionProvider", {"device_id": "0"})])
    binding = sess.io_binding()
    for n, t in ins.items():
        binding.bind_torch_input(n, t)
    for n, t in outs.items():
        binding.bind_torch_output(n, t)
    return dict(sess=sess, binding=binding, out=outs)


def _prepare_layout(case, state):
    B, rows, dev = case["requests"], len(state["ids"]), "cuda"
    outs = dict(block_table=torch.empty_like(state["table"]), cumulative_sequence_length=torch.empty(B + 1, dtype=torch.int32, device=dev),
                positions=torch.empty(rows, dtype=torch.int64, device=dev), slot_mapping=torch.empty(rows, dtype=torch.int64, device=dev),
                blocks_used=torch.empty(1, dtype=torch.int32, device=dev))
    names = ["past", "new", "table", "free", "ids"]
    return _bound([("PagedBatchLayout", names, list(outs), dict(block_size=case["block"]))], {n: state[n] for n in names}, outs)


def _prepare_attention(case, state):
    names = ["qkv", "key_cache", "value_cache", "cum", "past", "table", "prefix", "cos", "sin", "positions", "slots"]
    outs = dict(out=torch.empty(len(state["qkv"]), case["heads"] * case["head"], dtype=state["qkv"].dtype, device="cuda"),
                key_cache_out=state["key_cache"], value_cache_out=state["value_cache"])
    attrs = dict(num_heads=case["heads"], kv_num_heads=case["kv"], do_rotary=1)
    if case["cap"]:
        attrs["softcap"] = case["cap"]
    return _bound([("SharedPrefixPagedAttention", ["qkv", "", ""] + names[1:], list(outs), attrs)], {n: state[n] for n in names}, outs)


def _prepare_score(case, state):
    rows, top = case["rows"], case["top"]
    f32 = lambda *s: torch.empty(s, dtype=torch.float32, device="cuda")  # noqa: E731
    ins = {n: state[n] for n in ("logits", "tokens")}
    outs = dict(log_prob=f32(rows), entropy=f32(rows))
    if top:
        outs.update(top_log_probs=f32(rows, top), top_tokens=torch.empty(rows, top, dtype=torch.int64, device="cuda"))
    tops = ["top_log_probs", "top_tokens"] if top else ["", ""]
    nodes = [("TokenLogProbs", ["logits", "tokens"], ["log_prob", "entropy"] + tops + ["lse"], dict(top_k=top))]
    if case["kind"] == "train":
        ins.update(d_log_prob=state["d_log_prob"], d_entropy=state["d_entropy"])
        outs.update(d_logits=torch.empty_like(state["logits"]))
        nodes.append(("TokenLogProbsGrad", ["logits", "tokens", "lse", "entropy", "d_log_prob", "d_entropy"], ["d_logits"], {}))
    return _bound(nodes, ins, outs)


def prepare(case, seed):
    state = {"layout": _layout_inputs, "attention": _attention_inputs, "score": _score_inputs, "train": _score_inputs}[case["kind"]](case, seed)
    if own:
        made = {"layout": _prepare_layout, "attention": _prepare_attention, "score": _prepare_score, "train": _prepare_score}[case["kind"]]
        state.update(made(case, state))
    return dict(state, case=case)


def run(state):
    if own:
        state["sess"].run_with_iobinding(state["binding"])
        return state["out"]
    return {"layout": _layout, "attention": _attention, "score": _score, "train": _train}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _layout(s):
    size, past, new, table = s["case"]["block"], s["past"].long(), s["new"].long(), s["table"]
    held = (past + size - 1) // size
    need = (past + new + size - 1) // size - held
    start = need.cumsum(0) - need
    column = torch.arange(table.shape[1], device="cuda").unsqueeze(0)
    fresh = (column >= held.unsqueeze(1)) & (column < (held + need).unsqueeze(1))
    index = (start - held).unsqueeze(1) + column
    table = torch.where(fresh, s["free"][index.clamp(0, len(s["free"]) - 1)], table)
    ends = new.cumsum(0)
    row = torch.arange(len(s["ids"]), device="cuda")
    seq = torch.searchsorted(ends, row, right=True).clamp(max=len(past) - 1)
    pos = past[seq] + row - (ends - new)[seq]
    slot = table[seq, pos // size].long() * size + pos % size
    inside = row < ends[-1]
    cum = torch.cat([torch.zeros_like(ends[:1]), ends]).int()
    return dict(block_table=table, cumulative_sequence_length=cum, positions=torch.where(inside, pos, -1), slot_mapping=torch.where(inside, slot, -1),
                blocks_used=need.sum().int().reshape(1))


def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _attention(s):
    """The prefix once for all rows, the own keys per sequence (padded), and both put together by their maxima and sums."""
    c = s["case"]
    kv, head, group, size, dt = c["kv"], c["head"], c["heads"] // c["kv"], c["block"], s["qkv"].dtype
    tokens, B = len(s["qkv"]), len(s["past"])
    x = s["qkv"].float().reshape(tokens, -1, head)
    cos, sin = (s[n][s["positions"]].float().unsqueeze(1) for n in ("cos", "sin"))
    q, k = _rotated(x[:, :c["heads"]], cos, sin), _rotated(x[:, c["heads"]:c["heads"] + kv], cos, sin)
    caches = s["key_cache"], s["value_cache"]
    for cache, new in zip(caches, (k, x[:, c["heads"] + kv:])):
        cache.view(-1, kv, head)[s["slots"]] = new.to(dt)
    capped = lambda t: c["cap"] * torch.tanh(t / c["cap"]) if c["cap"] else t  # noqa: E731
    scale = head ** -0.5
    # prefix: [kv, tokens * group, prefix]
    blocks = (c["prefix"] + size - 1) // size
    pk, pv = (t[s["table"][0, :blocks].long()].reshape(-1, kv, head)[:c["prefix"]].float().transpose(0, 1) for t in caches)
    qg = q.reshape(tokens, kv, group, head)
    score = capped(qg.transpose(0, 1).reshape(kv, tokens * group, head) @ pk.transpose(1, 2) * scale)
    m1 = score.amax(-1, keepdim=True)
    e = torch.exp(score - m1)
    o1 = (e @ pv).reshape(kv, tokens, group, head).transpose(0, 1)
    m1, l1 = (t.reshape(kv, tokens, group, 1).transpose(0, 1) for t in (m1, e.sum(-1, keepdim=True)))
    # own keys: [B, kv, new * group, keys]
    lengths = _lengths(c)
    most, keys = max(n for _, n in lengths), max(p + n for p, n in lengths)
    place = s["positions"] - s["past"].long()[s["seq"]]
    padded = torch.zeros(B, most, kv, group, head, device="cuda")
    padded[s["seq"], place] = qg
    at = c["prefix"] + torch.arange(keys, device="cuda")
    entry = s["table"][:, (at // size).clamp(max=s["table"].shape[1] - 1)].long() * size + at % size
    ok, ov = (t.view(-1, kv, head)[entry].float().transpose(1, 2) for t in caches)
    score = capped(padded.transpose(1, 2).reshape(B, kv, most * group, head) @ ok.transpose(2, 3) * scale).reshape(B, kv, most, group, keys)
    last = s["past"].long().reshape(B, 1, 1, 1, 1) + torch.arange(most, device="cuda").reshape(1, 1, most, 1, 1)
    score = torch.where(at <= last, score, -math.inf)
    m2 = score.amax(-1, keepdim=True)
    e = torch.exp(score - m2)
    o2 = (e.reshape(B, kv, most * group, keys) @ torch.where((at < (s["past"] + s["cum"].diff()).reshape(B, 1)).reshape(B, 1, keys, 1), ov, 0.0))
    o2 = o2.reshape(B, kv, most, group, head).transpose(1, 2)[s["seq"], place]
    m2, l2 = (t.transpose(1, 2)[s["seq"], place] for t in (m2, e.sum(-1, keepdim=True)))
    m = torch.maximum(m1, m2)
    w1, w2 = torch.exp(m1 - m), torch.exp(m2 - m)
    out = (o1 * w1 + o2 * w2) / (l1 * w1 + l2 * w2)
    return dict(out=out.reshape(tokens, -1).to(dt), key_cache_out=caches[0], value_cache_out=caches[1])


def _statistics(x, tokens):
    """(log probability of the tokens, entropy, log sum exp, probabilities, log probabilities) of 32-bit logits."""
    m = x.amax(-1, keepdim=True)
    lse = m + torch.exp(x - m).sum(-1, keepdim=True).log()
    logp = x - lse
    p = torch.exp(logp)
    return logp.gather(1, tokens.unsqueeze(1)).squeeze(1), -(p * logp).sum(-1), p, logp


def _score(s):
    x = s["logits"].float()
    log_prob, entropy, _, logp = _statistics(x, s["tokens"])
    out = dict(log_prob=log_prob, entropy=entropy)
    if s["case"]["top"]:
        order = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :s["case"]["top"]]
        out.update(top_log_probs=logp.gather(1, order), top_tokens=order)
    return out


def _train(s):
    log_prob, entropy, p, logp = _statistics(s["logits"].float(), s["tokens"])
    g, h = s["d_log_prob"].unsqueeze(1), s["d_entropy"].unsqueeze(1)
    dx = -p * (g + h * (logp + entropy.unsqueeze(1)))
    dx = dx.scatter_add(1, s["tokens"].unsqueeze(1), g)
    return dict(log_prob=log_prob, entropy=entropy, d_logits=dx.to(s["logits"].dtype))


# -------------------------------------------------------------------------------------------------------------- 64-bit results
def _exact_attention(case, seed):
    """PagedAttention's definition, sequence by sequence over its own row of the block table."""
    s, kv, head, group = _attention_inputs(case, seed), case["kv"], case["head"], case["heads"] // case["kv"]
    qkv, dt, size = s["qkv"].double().reshape(len(s["qkv"]), -1, head), s["qkv"].dtype, case["block"]
    keys, values = s["key_cache"].double().view(-1, kv, head), s["value_cache"].double().view(-1, kv, head)
    out, t0 = torch.empty(len(qkv), case["heads"], head, dtype=torch.float64, device="cuda"), 0
    for b, (held, new) in enumerate(_lengths(case)):
        past, rows = case["prefix"] + held, slice(t0, t0 + new)
        t0 += new
        where = torch.arange(past + new, device="cuda")
        entry = s["table"][b].long()[where // size] * size + where % size
        cos, sin = s["cos"][past:past + new].double().unsqueeze(1), s["sin"][past:past + new].double().unsqueeze(1)
        turn = lambda t: torch.cat([t[..., :head // 2] * cos - t[..., head // 2:] * sin, t[..., head // 2:] * cos + t[..., :head // 2] * sin], -1)  # noqa: E731
        q = turn(qkv[rows, :case["heads"]])
        keys[entry[past:]] = turn(qkv[rows, case["heads"]:case["heads"] + kv]).to(dt).double()
        values[entry[past:]] = qkv[rows, case["heads"] + kv:]
        hidden = where > torch.arange(past, past + new, device="cuda").unsqueeze(1)
        for j in range(kv):
            score = q[:, j * group:(j + 1) * group].transpose(0, 1) @ keys[entry, j].t() / math.sqrt(head)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            out[rows, j * group:(j + 1) * group] = (score.masked_fill(hidden, -math.inf).softmax(-1) @ values[entry, j]).transpose(0, 1)
    shape = s["key_cache"].shape
    return dict(out=out.reshape(len(qkv), -1), key_cache_out=keys.view(shape), value_cache_out=values.view(shape))


def _exact_score(case, seed):
    s, top, rows = _score_inputs(case, seed), case["top"], case["rows"]
    f64 = lambda *n: torch.empty(n, dtype=torch.float64, device="cuda")  # noqa: E731
    out = dict(log_prob=f64(rows), entropy=f64(rows))
    if top:
        out["top_log_probs"] = f64(rows, top)
        out["top_tokens"] = None
    if case["kind"] == "train":
        out["d_logits"] = f64(rows, case["vocab"])
    for r in range(0, rows, 256):                          # a portion of the rows at a time: 64-bit logits take much room
        part = slice(r, min(r + 256, rows))
        logp = torch.log_softmax(s["logits"][part].double(), -1)
        p, tokens = logp.exp(), s["tokens"][part]
        entropy = -torch.special.xlogy(p, p).sum(-1)
        out["log_prob"][part], out["entropy"][part] = logp[torch.arange(len(tokens), device="cuda"), tokens], entropy
        if top:
            out["top_log_probs"][part] = logp.topk(top, -1)[0]
        if case["kind"] == "train":
            g, h = s["d_log_prob"][part].double().unsqueeze(1), s["d_entropy"][part].double().unsqueeze(1)
            one = torch.nn.functional.one_hot(tokens, case["vocab"])
            out["d_logits"][part] = g * (one - p) - h * p * (logp + entropy.unsqueeze(1))
    return out


def exact(case, seed):
    if case["kind"] == "layout":
        return None                                        # whole numbers: equal, or wrong
    return _exact_attention(case, seed) if case["kind"] == "attention" else _exact_score(case, seed)

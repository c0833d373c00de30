"""What the operators of a decode step with drafted tokens are measured on.

Three kinds of calls, each through an ``InferenceSession`` with bound buffers, the way the serving loop makes them:

* ``tree``: com.ortb200.TreePagedAttention - rotary, cache append and attention over paged caches for sequences that bring a tree of drafted tokens
  each: a token sees what its sequence holds, and its own ancestors;
* ``move``: com.ortb200.PagedCacheMove - the entries of accepted tokens, or whole blocks, to other places of all layers' caches;
* ``logits``: com.ortb200.ProcessLogits - penalties for repeated tokens, biases, grammar masks and temperatures, row by row.

Lengths and trees belong to the case, values to the seed.
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
        # one user of a chat, eight drafted tokens: the call whose latency every layer of every step pays
        dict(name="tree_1x900", kind="tree", dtype="bf16", heads=32, kv=8, head=128, block=256, batch=1, past=900, nodes=8, chain=0.5, cap=0.0),
        # a chat server: 24 conversations with up to 16 drafted tokens each
        dict(name="tree_24x4000", kind="tree", dtype="bf16", heads=32, kv=8, head=128, block=256, batch=24, past=4000, nodes=16, chain=0.5, cap=0.0),
        # long documents, large trees, eight query heads to a key head
        dict(name="tree_6x30000", kind="tree", dtype="bf16", heads=64, kv=8, head=128, block=128, batch=6, past=30000, nodes=64, chain=0.4, cap=0.0),
        # many requests without drafts: one token each
        dict(name="tree_single_90x1500", kind="tree", dtype="bf16", heads=28, kv=4, head=128, block=64, batch=90, past=1500, nodes=1, chain=1.0, cap=0.0),
        # chains of five, heads of 64 that share no key head, small blocks
        dict(name="tree_chain_64x1211", kind="tree", dtype="fp16", heads=16, kv=16, head=64, block=16, batch=64, past=1211, nodes=5, chain=1.0, cap=30.0),
        # accepted tokens of a small server, 32 layers
        dict(name="move_accept_6", kind="move", dtype="bf16", kv=8, head=128, block=256, caches=64, what="accept", moves=6, nodes=8),
        # accepted tokens of a large one, small blocks
        dict(name="move_accept_200", kind="move", dtype="fp16", kv=8, head=128, block=16, caches=32, what="accept", moves=200, nodes=24),
        # beams that go on from other beams: whole blocks of twelve layers
        dict(name="move_beams_40", kind="move", dtype="bf16", kv=8, head=128, block=256, caches=24, what="blocks", moves=40, nodes=0),
        # a small step, all penalties, a history each
        dict(name="logits_4", kind="logits", dtype="bf16", lists=4, nodes=1, vocab=128256, history=700, bias=20, masks=0, row_params="all"),
        # one very long history, 32-bit logits of an odd vocabulary
        dict(name="logits_40_long", kind="logits", dtype="fp32", lists=40, nodes=1, vocab=50257, history=60000, bias=0, masks=0, row_params="repetition"),
        # structured answers: a grammar's mask for every row
        dict(name="logits_grammar_150", kind="logits", dtype="fp16", lists=150, nodes=1, vocab=32000, history=1000, bias=3, masks=40, row_params="temperature"),
        # the drafted trees of 32 requests: every node's row has its request's history and its own ancestors
        dict(name="logits_tree_32x16", kind="logits", dtype="bf16", lists=32, nodes=16, vocab=128256, history=3000, bias=8, masks=32, row_params="all"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "move", "logits", "logits"])
    if kind == "tree":
        heads, kv, head = rng.choice([(32, 8, 128), (64, 8, 128), (16, 16, 64), (28, 4, 128), (24, 8, 64), (32, 2, 128)])
        nodes = rng.choice([1, _log(rng, 2, 64), _log(rng, 2, 64)])
        batch = _log(rng, 1, 100)
        most = min(30000, 360000000 // (batch * nodes * heads), 3000000 // (batch * kv))   # within the cost of the largest listed case
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), heads=heads, kv=kv, head=head, block=rng.choice([16, 32, 64, 128, 256]), batch=batch,
                    past=_log(rng, 30, max(60, most)), nodes=nodes, chain=rng.choice([0.2, 0.5, 0.8, 1.0]), cap=rng.choice([0.0, 0.0, 30.0]))
    if kind == "move":
        what = rng.choice(["accept", "accept", "blocks"])
        kv, head = rng.choice([(8, 128), (16, 64), (4, 128), (1, 576), (2, 80)])
        if what == "accept":
            return dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), kv=kv, head=head, block=rng.choice([16, 32, 64, 256]), caches=rng.randint(1, 64), what=what,
                        moves=_log(rng, 1, 200), nodes=rng.randint(8, 32))
        return dict(kind=kind, dtype=rng.choice(["bf16", "fp16"]), kv=kv, head=head, block=rng.choice([16, 64, 256]), caches=rng.randint(1, 24), what=what, moves=_log(rng, 1, 40),
                    nodes=0)
    vocab = rng.choice([_log(rng, 1000, 200000), 32000, 50257, 128256])
    nodes = rng.choice([1, 1, rng.randint(2, 32)])
    lists = _log(rng, 1, max(1, min(500, 512 * 128256 // (vocab * nodes))))
    return dict(kind=kind, dtype=rng.choice(["bf16", "fp16", "fp32"]), lists=lists, nodes=nodes, vocab=vocab, history=_log(rng, 1, min(60000, 2400000 // lists)),
                bias=rng.choice([0, _log(rng, 1, 300)]), masks=rng.choice([0, rng.randint(1, 40)]), row_params=rng.choice(["all", "repetition", "temperature"]))


# ---------------------------------------------------------------------------------------------------------- shapes of a case
def _own_random(case):
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _trees(case):
    """[(tokens held, parents of the new tokens)] of the sequences; the first new token is the one that the step before chose."""
    r, out = _own_random(case), []
    for _ in range(case["batch"]):
        past, nodes = r.randint((case["past"] + 1) // 2, case["past"]), r.randint((case["nodes"] + 1) // 2, case["nodes"])
        out.append((past, [-1] + [i - 1 if r.random() < case["chain"] else r.randint(max(0, i - 8), i - 1) for i in range(1, nodes)]))
    return out


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _moves(case):
    """(sources, targets, tokens or blocks in the pool); accepted tokens come from places behind those that they take."""
    r = _own_random(case)
    if case["what"] == "blocks":
        order = list(range(2 * case["moves"] + 3))
        r.shuffle(order)
        targets = order[:case["moves"]]
        return [r.choice(order[case["moves"]:]) for _ in targets], targets, len(order)
    sources, targets, at, nodes = [], [], r.randint(0, case["block"]), case["nodes"]
    while len(sources) < case["moves"]:
        accepted = min(r.randint(1, nodes // 2 - 1), case["moves"] - len(sources))
        sources += [at + i for i in sorted(r.sample(range(nodes // 2, nodes), accepted))]
        targets += [at + 1 + i for i in range(accepted)]
        at += nodes + r.randint(0, 4 * case["block"])
    return sources, targets, at // case["block"] + 1


def _histories(case):
    r = _own_random(case)
    lengths = [r.randint(case["history"] // 2, case["history"]) for _ in range(case["lists"])]
    nodes = [r.randint((case["nodes"] + 1) // 2, case["nodes"]) if case["nodes"] > 1 else 1 for _ in range(case["lists"])]
    parents = [[-1] + [r.randint(max(0, i - 6), i - 1) for i in range(1, n)] for n in nodes]
    return lengths, parents


def work(case):
    if case["kind"] == "tree":
        entry, held, tokens, seen = 2 * case["kv"] * case["head"] * 2, 0, 0, 0
        for past, parents in _trees(case):
            held += past
            tokens += len(parents)
            seen += sum(past + d + 1 for d in _depths(parents))
        return {"bytes": entry * (held + 2 * tokens) + 2 * 2 * tokens * case["heads"] * case["head"], "flops": 4 * case["heads"] * case["head"] * seen}
    if case["kind"] == "move":
        entry = case["kv"] * case["head"] * 2 * (case["block"] if case["what"] == "blocks" else 1)
        return {"bytes": case["moves"] * (2 * entry * case["caches"] + 16), "flops": 0}
    lengths, parents = _histories(case)
    rows = sum(len(p) for p in parents)
    size = 4 if case["dtype"] == "fp32" else 2
    told = sum(lengths) if case["row_params"] != "temperature" else 0
    return {"bytes": rows * case["vocab"] * (size + 4) + 8 * told + case["masks"] * case["vocab"] // 8 + rows * (32 + 12 * case["bias"]), "flops": 6 * rows * case["vocab"]}


# ------------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed, salt):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + salt) % (1 << 62))


def _normal(gen, shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0, std, generator=gen)


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _tree_inputs(case, seed):
    g, trees, dt, size = _gen(seed, 1), _trees(case), DTYPES[case["dtype"]], case["block"]
    past, new = [p for p, _ in trees], [len(t) for _, t in trees]
    need = [(p + n + size - 1) // size for p, n in zip(past, new)]
    pool = sum(need) + 8
    order = torch.randperm(pool, generator=g, device="cuda").int()
    table = torch.zeros(len(trees), max(need), dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    caches = [_normal(g, (pool, size, case["kv"], case["head"]), dt) for _ in range(2)]
    qkv = _normal(g, (sum(new), (case["heads"] + 2 * case["kv"]) * case["head"]), dt)
    rows = max(p + n for p, n in zip(past, new))
    angle = torch.arange(rows, device="cuda").double().unsqueeze(1) * 10000.0 ** (-torch.arange(case["head"] // 2, device="cuda").double() * 2 / case["head"])
    return dict(qkv=qkv, key_cache=caches[0], value_cache=caches[1], cum=torch.tensor([0] + new).cumsum(0).int().cuda(), past=_ints(past), table=table,
                parents=_ints([p for _, t in trees for p in t]), cos=angle.cos().to(dt), sin=angle.sin().to(dt))


def _move_inputs(case, seed):
    g, dt = _gen(seed, 2), DTYPES[case["dtype"]]
    sources, targets, pool = _moves(case)
    s = {f"cache.{i}": _normal(g, (pool, case["block"], case["kv"], case["head"]), dt) for i in range(case["caches"])}
    return dict(s, sources=_ints(sources, torch.int64), targets=_ints(targets, torch.int64))


def _logits_inputs(case, seed):
    """Logits of a language model: a broad bulk and a few tokens far above it in every row; likely tokens are often in the history."""
    g, vocab, dev = _gen(seed, 3), case["vocab"], "cuda"
    lengths, parents = _histories(case)
    rows, total = sum(len(p) for p in parents), sum(lengths)
    logits = _normal(g, (rows, vocab), DTYPES[case["dtype"]], 2.0)
    favourites = torch.randint(0, vocab, (64,), generator=g, device=dev)
    likely = favourites[torch.randint(0, 64, (rows, 8), generator=g, device=dev)]
    logits.scatter_(1, likely, (_normal(g, (rows, 8), torch.float32, 1.5) + 11).to(logits.dtype))
    history = torch.where(torch.rand(total, generator=g, device=dev) < 0.3, favourites[torch.randint(0, 64, (total,), generator=g, device=dev)],
                          torch.randint(0, vocab, (total,), generator=g, device=dev))
    s = dict(logits=logits)
    if case["row_params"] != "temperature":
        s.update(history=history, history_starts=torch.tensor([0] + lengths).cumsum(0).cuda())
    uniform = lambda lo, hi: lo + (hi - lo) * torch.rand(rows, generator=g, device=dev)  # noqa: E731
    if case["nodes"] > 1 and "history" in s:               # the rows of a request's tree: its history, then the node's ancestors
        lists, drafted, deepest = [], [], max(max(_depths(p)) for p in parents) + 1
        tokens = favourites[torch.randint(0, 64, (rows,), generator=g, device=dev)].tolist()
        for i, tree in enumerate(parents):
            first = len(lists)
            for j in range(len(tree)):
                path, k = [], j
                while k >= 0:
                    path.append(tokens[first + k])
                    k = tree[k]
                lists.append(i)
                drafted.append(path + [-1] * (deepest - len(path)))
        s.update(row_list=_ints(lists), drafted=_ints(drafted, torch.int64))
    if case["row_params"] in ("all", "repetition"):
        s.update(repetition=uniform(1.0, 1.3))
    if case["row_params"] == "all":
        prompt = (s["history_starts"].diff().float() * torch.rand(case["lists"], generator=g, device=dev)).long()
        s.update(generated_starts=s["history_starts"][:-1] + prompt, presence=uniform(0.0, 0.8), frequency=uniform(0.0, 0.3))
    if case["row_params"] in ("all", "temperature"):
        s.update(temperature=uniform(0.5, 1.5))
    if case["bias"]:
        pick = torch.rand(rows, max(vocab // 4, case["bias"]), generator=g, device=dev).topk(case["bias"], -1)[1]    # distinct within a row
        s.update(bias_tokens=pick.reshape(-1), bias_values=3 * torch.randn(rows * case["bias"], generator=g, device=dev),
                 bias_starts=torch.arange(rows + 1, device=dev) * case["bias"])
    if case["masks"]:
        words = torch.randint(-(1 << 31), 1 << 31, (2, case["masks"], (vocab + 31) // 32), generator=g, device=dev)
        s.update(allowed=(words[0] & words[1]).int(), row_mask=torch.randint(-1, case["masks"], (rows,), generator=g, device=dev).int())
    return s


# ------------------------------------------------------------------------------------------------------------ prepare and run
def _bound(node, ins, outs, attrs):
    """A session over one operator with every input and output bound to a device tensor."""
    import onnxruntime_b200 as ort
    from onnxruntime_b200 import onnx_lite as ol
    T = ol.TensorProto
    types = {torch.bfloat16: T.BFLOAT16, torch.float16: T.FLOAT16, torch.float32: T.FLOAT, torch.int32: T.INT32, torch.int64: T.INT64}
    info = lambda n, t: ol.make_tensor_value_info(n, types[t.dtype], list(t.shape))  # noqa: E731
    graph = ol.make_graph([ol.make_node(node[0], node[1], list(outs), domain=FUSED, **attrs)], "step", [info(n, t) for n, t in ins.items()],
                          [info(n, t) for n, t in outs.items()])
    sess = ort.InferenceSession(ol.make_model(graph, opset=17, extra_opsets={FUSED: 1}).serialize(), providers=[("CUDAExecutionProvider", {"device_id": "0"})])
    binding = sess.io_binding()
    for n, t in ins.items():
        binding.bind_torch_input(n, t)
    for n, t in outs.items():
        binding.bind_torch_output(n, t)
    return dict(sess=sess, binding=binding, out=outs)


def _prepare_tree(case, s):
    names = ["qkv", "key_cache", "value_cache", "cum", "past", "table", "parents", "cos", "sin"]
    outs = dict(out=torch.empty(len(s["qkv"]), case["heads"] * case["head"], dtype=s["qkv"].dtype, device="cuda"), key_cache_out=s["key_cache"],
                value_cache_out=s["value_cache"])
    attrs = dict(num_heads=case["heads"], kv_num_heads=case["kv"], do_rotary=1)
    if case["cap"]:
        attrs["softcap"] = case["cap"]
    return _bound(("TreePagedAttention", ["qkv", "", ""] + names[1:]), {n: s[n] for n in names}, outs, attrs)


def _prepare_move(case, s):
    names = ["sources", "targets"] + [n for n in s if n.startswith("cache.")]
    return _bound(("PagedCacheMove", names), {n: s[n] for n in names}, {n + ".out": s[n] for n in names[2:]}, dict(whole_blocks=int(case["what"] == "blocks")))


LOGITS_INPUTS = ["logits", "history", "history_starts", "generated_starts", "row_list", "drafted", "repetition", "presence", "frequency", "bias_tokens", "bias_values",
                 "bias_starts", "allowed", "row_mask", "temperature"]


def _prepare_logits(case, s):
    names = [n if n in s else "" for n in LOGITS_INPUTS]
    while not names[-1]:
        names.pop()
    outs = dict(scores=torch.empty(s["logits"].shape, dtype=torch.float32, device="cuda"))
    return _bound(("ProcessLogits", names), {n: s[n] for n in names if n}, outs, {})


def prepare(case, seed):
    state = {"tree": _tree_inputs, "move": _move_inputs, "logits": _logits_inputs}[case["kind"]](case, seed)
    if own:
        made = {"tree": _prepare_tree, "move": _prepare_move, "logits": _prepare_logits}[case["kind"]]
        state.update(made(case, state))
    elif case["kind"] == "tree":
        state.update(_tree_plan(case))
    return dict(state, case=case)


def run(state):
    if own:
        state["sess"].run_with_iobinding(state["binding"])
        return state["out"]
    return {"tree": _tree, "move": _move, "logits": _logits}[state["case"]["kind"]](state)


# ---------------------------------------------------------------------------------------------------------------- plain forms
def _rotated(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _tree_plan(case):
    """What the plain form knows of the lengths on the host: which sequence and place a row has, and how far keys go."""
    trees = _trees(case)
    seq = torch.tensor([b for b, (_, t) in enumerate(trees) for _ in t]).cuda()
    place = torch.tensor([i for _, t in trees for i in range(len(t))]).cuda()
    return dict(seq=seq, place=place, most=max(len(t) for _, t in trees), keys=max(p + len(t) for p, t in trees))


def _tree(s):
    """Ancestors by following parents, keys of all sequences padded to the longest."""
    c = s["case"]
    kv, head, group, size, dt = c["kv"], c["head"], c["heads"] // c["kv"], c["block"], s["qkv"].dtype
    tokens, B, past, seq, place, most, keys = len(s["qkv"]), len(s["past"]), s["past"].long(), s["seq"], s["place"], s["most"], s["keys"]
    parents = torch.full((B, most), -1, device="cuda", dtype=torch.int64)
    parents[seq, place] = s["parents"].long()
    sees = torch.zeros(B, most, most, dtype=torch.bool, device="cuda")
    at, depth = torch.arange(most, device="cuda").expand(B, most), torch.full((B, most), -1, device="cuda")
    for _ in range(most):
        sees |= torch.nn.functional.one_hot(at.clamp(min=0), most).bool() & (at >= 0).unsqueeze(-1)
        depth = depth + (at >= 0)
        at = torch.where(at >= 0, parents.gather(1, at.clamp(min=0)), at)
    x = s["qkv"].float().reshape(tokens, -1, head)
    pos = past[seq] + depth[seq, place]
    cos, sin = (s[n][pos].float().unsqueeze(1) for n in ("cos", "sin"))
    q, k = _rotated(x[:, :c["heads"]], cos, sin), _rotated(x[:, c["heads"]:c["heads"] + kv], cos, sin)
    spot = past[seq] + place
    slots = s["table"][seq, spot // size].long() * size + spot % size
    caches = s["key_cache"], s["value_cache"]
    for cache, new in zip(caches, (k, x[:, c["heads"] + kv:])):
        cache.view(-1, kv, head)[slots] = new.to(dt)
    padded = torch.zeros(B, most, kv, group, head, device="cuda")
    padded[seq, place] = q.reshape(tokens, kv, group, head)
    where = torch.arange(keys, device="cuda")
    held = where < (past + s["cum"].diff()).unsqueeze(1)                    # [B, keys]
    entry = s["table"][:, where // size].long() * size + where % size
    ok, ov = (t.view(-1, kv, head)[entry].float().transpose(1, 2) for t in caches)
    score = padded.transpose(1, 2).reshape(B, kv, most * group, head) @ ok.transpose(2, 3) * head ** -0.5
    if c["cap"]:
        score = c["cap"] * torch.tanh(score / c["cap"])
    node = (where.unsqueeze(0) - past.unsqueeze(1))                          # [B, keys]: which new token a key is
    seen = sees.gather(2, node.clamp(0, most - 1).unsqueeze(1).expand(B, most, keys)) | (node < 0).unsqueeze(1)
    seen = (seen & held.unsqueeze(1)).reshape(B, 1, most, 1, keys)
    score = torch.where(seen, score.reshape(B, kv, most, group, keys), -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    weights = (e / e.sum(-1, keepdim=True)).reshape(B, kv, most * group, keys)
    out = weights @ torch.where(held.reshape(B, 1, keys, 1), ov, 0.0)
    out = out.reshape(B, kv, most, group, head).transpose(1, 2)[seq, place]
    return dict(out=out.reshape(tokens, -1).to(dt), key_cache_out=caches[0], value_cache_out=caches[1])


def _move(s):
    blocks, out = s["case"]["what"] == "blocks", {}
    for n in [n for n in s if n.startswith("cache.")]:
        t = s[n] if blocks else s[n].view(-1, *s[n].shape[2:])
        t[s["targets"]] = t[s["sources"]]
        out[n + ".out"] = s[n]
    return out


def _counts(s, rows, vocab, first):
    """How often each row's history, from the places `first` of the lists on, and its drafted tokens have each token."""
    starts, total = s["history_starts"], len(s["history"])
    place = torch.arange(total, device="cuda")
    lists = torch.searchsorted(starts[1:], place, right=True)
    counted = (place >= first[lists]).float()
    count = torch.zeros(len(starts) - 1, vocab, device="cuda").view(-1).index_add_(0, lists * vocab + s["history"], counted).view(-1, vocab)
    if "drafted" in s:
        count = count[s["row_list"].long()]
        inside = s["drafted"] >= 0
        count.scatter_add_(1, s["drafted"].clamp(min=0), inside.float())
    return count


def _logits(s):
    x, vocab = s["logits"].float(), s["logits"].shape[1]
    rows, column = len(x), lambda n: s[n].unsqueeze(1)  # noqa: E731
    if "repetition" in s:
        seen = _counts(s, rows, vocab, s["history_starts"][:-1]) > 0
        x = torch.where(seen, torch.where(x < 0, x * column("repetition"), x / column("repetition")), x)
    if "frequency" in s:
        count = _counts(s, rows, vocab, s["generated_starts"])
        x = x - (column("frequency") * count + column("presence") * (count > 0))
    if "bias_tokens" in s:
        row = torch.repeat_interleave(torch.arange(rows, device="cuda"), s["bias_starts"].diff(), output_size=len(s["bias_tokens"]))
        x = x.index_put((row, s["bias_tokens"]), s["bias_values"], accumulate=True)
    if "allowed" in s:
        bit = torch.arange(vocab, device="cuda")
        allowed = (s["allowed"][:, bit // 32] >> (bit % 32).int()) & 1
        x = torch.where((s["row_mask"] < 0).unsqueeze(1) | (allowed[s["row_mask"].long().clamp(min=0)] == 1), x, -math.inf)
    if "temperature" in s:
        x = x / column("temperature")
    return dict(scores=x)


# -------------------------------------------------------------------------------------------------------------- 64-bit results
def _exact_tree(case, seed):
    """Sequence by sequence over its own row of the block table, a token at a time for what it may see."""
    s, kv, head, group, size = _tree_inputs(case, seed), case["kv"], case["head"], case["heads"] // case["kv"], case["block"]
    qkv, dt = s["qkv"].double().reshape(len(s["qkv"]), -1, head), s["qkv"].dtype
    keys, values = s["key_cache"].double().view(-1, kv, head), s["value_cache"].double().view(-1, kv, head)
    out, t0 = torch.empty(len(qkv), case["heads"], head, dtype=torch.float64, device="cuda"), 0
    for b, (past, parents) in enumerate(_trees(case)):
        new = len(parents)
        rows = slice(t0, t0 + new)
        t0 += new
        depth = torch.tensor(_depths(parents)).cuda() + past
        where = torch.arange(past + new, device="cuda")
        entry = s["table"][b].long()[where // size] * size + where % size
        cos, sin = s["cos"][depth].double().unsqueeze(1), s["sin"][depth].double().unsqueeze(1)
        turn = lambda t: torch.cat([t[..., :head // 2] * cos - t[..., head // 2:] * sin, t[..., head // 2:] * cos + t[..., :head // 2] * sin], -1)  # noqa: E731
        q = turn(qkv[rows, :case["heads"]])
        keys[entry[past:]] = turn(qkv[rows, case["heads"]:case["heads"] + kv]).to(dt).double()
        values[entry[past:]] = qkv[rows, case["heads"] + kv:]
        hidden = torch.ones(new, past + new, dtype=torch.bool)
        hidden[:, :past] = False
        for i, p in enumerate(parents):
            if p >= 0:
                hidden[i, past:] = hidden[p, past:]
            hidden[i, past + i] = False
        hidden = hidden.cuda()
        for j in range(kv):
            score = q[:, j * group:(j + 1) * group].transpose(0, 1) @ keys[entry, j].t() / math.sqrt(head)
            if case["cap"]:
                score = case["cap"] * torch.tanh(score / case["cap"])
            out[rows, j * group:(j + 1) * group] = (score.masked_fill(hidden, -math.inf).softmax(-1) @ values[entry, j]).transpose(0, 1)
    shape = s["key_cache"].shape
    return dict(out=out.reshape(len(qkv), -1), key_cache_out=keys.view(shape), value_cache_out=values.view(shape))


def _exact_logits(case, seed):
    s, vocab = _logits_inputs(case, seed), case["vocab"]
    x, starts = s["logits"].double(), s["history_starts"].tolist() if "history" in s else None
    for r in range(len(x)):
        if "history" in s:
            i = int(s["row_list"][r]) if "row_list" in s else r
            drafted = s["drafted"][r][s["drafted"][r] >= 0] if "drafted" in s else s["history"][:0]
            text = torch.cat([s["history"][starts[i]:starts[i + 1]], drafted])
        if "repetition" in s:
            ids, rep = text.unique(), s["repetition"][r].double()
            v = x[r, ids]
            x[r, ids] = torch.where(v < 0, v * rep, v / rep)
        if "frequency" in s:
            ids, n = text[int(s["generated_starts"][i]) - starts[i]:].unique(return_counts=True)
            x[r, ids] -= s["frequency"][r].double() * n + s["presence"][r].double()
        if "bias_tokens" in s:
            part = slice(int(s["bias_starts"][r]), int(s["bias_starts"][r + 1]))
            x[r, s["bias_tokens"][part]] += s["bias_values"][part].double()
        if "allowed" in s and int(s["row_mask"][r]) >= 0:
            words = s["allowed"][int(s["row_mask"][r])]
            bits = torch.stack([(words >> b) & 1 for b in range(32)], -1).reshape(-1)[:vocab]
            x[r, bits == 0] = -math.inf
        if "temperature" in s:
            x[r] /= s["temperature"][r].double()
    return dict(scores=x)


def _exact_move(case, seed):
    """Entry by entry; values are copied, so that their own type holds them."""
    s, out = _move_inputs(case, seed), {}
    pairs = list(zip(s["sources"].tolist(), s["targets"].tolist()))
    for n in [n for n in s if n.startswith("cache.")]:
        before, after = s[n], s[n].clone()
        for source, target in pairs:
            if case["what"] == "blocks":
                after[target] = before[source]
            else:
                after[target // case["block"], target % case["block"]] = before[source // case["block"], source % case["block"]]
        out[n + ".out"] = after
    return out


def exact(case, seed):
    return {"tree": _exact_tree, "move": _exact_move, "logits": _exact_logits}[case["kind"]](case, seed)

"""Edges of the decode step with drafted tokens: what its operators, the pool and the generation loop make of infinities, shared blocks, drafts
that a grammar forbids, and limits.  The definitions are draft_oracle.py's."""
import math

import pytest
import torch

import draft_oracle as oracle

from onnxruntime_b200.capi import EPFail, InvalidArgument
from onnxruntime_b200.models.decoder_cache import CachePool, CacheTensor
from onnxruntime_b200.models.generation import GenerationConfig, LogitsProcessor, draft_tree, generate, generate_requests
from test_draft_generation import PROVIDERS, decoder, pool
from test_draft_ops import KINDS, LOGITS_KINDS, LogitsCase, TreeCase, tree


# ----------------------------------------------------------------------------------------------------------------------- bans
HARD = [math.inf, -math.inf, math.nan, 0.0]


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("biases", [4, 400])
@pytest.mark.parametrize("twice", [False, True])
def test_banned_tokens_of_any_logit(kind, biases, twice):
    """A token whose biases sum to -inf has -inf, whatever its logit is: infinities, NaN, the type's largest number; on rows with few biases and
    with more than are listed, named once and twice, inside and outside of the text."""
    vocab, tokens = 3001, torch.arange(biases) * 7 + 1
    case = LogitsCase(kind[1], 2, vocab, without=["row_list", "drafted", "allowed", "row_mask"], seed=biases)
    hard = torch.tensor([*HARD, torch.finfo(kind[1]).max])
    case.t["logits"][:, tokens] = hard[torch.arange(biases) % 5].to(kind[1])
    named = torch.cat([tokens, tokens[::2]]) if twice else tokens
    per = len(named)
    case.t.update(history=torch.arange(2 * 50) % 50, history_starts=torch.tensor([0, 50, 100]), generated_starts=torch.tensor([20, 60]), bias_tokens=named.repeat(2),
                  bias_values=torch.full((2 * per,), -math.inf), bias_starts=torch.tensor([0, per, 2 * per]), repetition=torch.tensor([1.0, 1.5]), presence=torch.tensor([0.5, 0.0]),
                  frequency=torch.tensor([0.25, 0.0]), temperature=torch.tensor([0.5, 1.0]))
    got = case.call(kind[0])()["scores"]
    assert (got[:, tokens] == -math.inf).all()
    free = torch.ones(vocab, dtype=torch.bool)
    free[tokens] = False
    assert got[:, free].isfinite().all()


@pytest.mark.parametrize("kind", LOGITS_KINDS)
def test_masked_and_banned_tokens_under_an_infinite_temperature(kind):
    """x / inf is 0 for every finite logit; what is masked or banned stays -inf, on every provider."""
    case = LogitsCase(kind[1], 2, 300, without=["history", "history_starts", "generated_starts", "row_list", "drafted", "repetition", "presence", "frequency"], seed=3)
    case.t.update(temperature=torch.full((2,), math.inf), bias_tokens=torch.tensor([1, 2, 1, 2]), bias_values=torch.tensor([-math.inf, 1.0] * 2), bias_starts=torch.tensor([0, 2, 4]),
                  allowed=torch.full((1, 10), 0x5555555f, dtype=torch.int32), row_mask=torch.tensor([0, -1], dtype=torch.int32))
    got = case.call(kind[0])()["scores"]
    want = torch.zeros(2, 300)
    want[:, 1] = -math.inf
    want[0, [v for v in range(300) if not 0x5555555f >> (v % 32) & 1]] = -math.inf
    assert torch.equal(got, want)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("hard", [math.inf, math.nan])
@pytest.mark.parametrize("kw", [dict(eos_token_id=5, min_new_tokens=4), dict(no_repeat_ngram_size=2), dict(no_repeat_ngram_size=1), dict(logit_bias={5: -math.inf})], ids=str)
def test_a_banned_token_is_not_chosen(provider, hard, kw):
    """An end token before its time, and one that would repeat an n-gram, are not the best of a row whatever the model says of them."""
    device = torch.device("cuda" if provider == "CUDAExecutionProvider" else "cpu")
    logits = torch.linspace(-1, 1, 40).repeat(2, 1)
    logits[:, 5] = hard
    scores = LogitsProcessor(40, torch.float32, device, GenerationConfig(**kw))(logits.to(device), [([1, 2, 5, 1, 2], 1, [[]]), ([2, 5, 3, 2], 0, [[]])]).cpu()
    assert (scores[:, 5] == -math.inf).all() and scores.argmax(-1).tolist() == [39, 39]


# ------------------------------------------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,Nk,H,past,nodes", [(4, 2, 64, 0, 3), (8, 2, 64, 57, 7), (6, 3, 128, 130, 40), (32, 2, 128, 100, 100), (2, 2, 128, 70, 300), (40, 40, 64, 9, 3), (64, 64, 64, 70, 2),
                                              (35, 5, 64, 200, 60), (6, 3, 40, 20, 9), (2, 2, 256, 65, 270)])
@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_a_value_that_is_not_finite_reaches_its_key_head(kind, N, Nk, H, past, nodes, bad):
    """One element of one key head of one drafted token: the query heads that read it, in the rows that see the token, become NaN; all other results are,
    to the bit, what they are without it, on every provider and in every form of the kernels."""
    parents = [-1] + [(i - 1) // 2 if nodes <= 256 else i - 1 for i in range(1, nodes)]
    case = TreeCase(kind[1], N, Nk, H, 16, [past, 33], [parents, tree(6, 3)], seed=nodes)
    token, head, group = nodes // 2, Nk // 2, N // Nk
    case.qkv[token, N + Nk + head] = 0.0
    want = case.call(kind[0])()["out"].reshape(-1, N, H)
    case.qkv[token, N + Nk + head, H // 3] = bad
    got = case.call(kind[0])()["out"].reshape(-1, N, H)
    spoilt = torch.zeros(nodes + 6, N, dtype=torch.bool)
    sees = oracle.sees(parents)[:, token] if nodes <= 256 else torch.arange(nodes) >= token
    spoilt[:nodes, head * group:(head + 1) * group] = sees.unsqueeze(1)
    assert got[spoilt].isnan().all() and torch.equal(got[~spoilt], want[~spoilt])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,H,nodes", [(4, 64, 3), (32, 64, 40), (32, 128, 100), (4, 40, 3)])
def test_a_value_that_is_not_finite_behind_a_score_of_minus_infinity(kind, N, H, nodes):
    """A token that a row sees is seen, also with a weight of 0 because its score is -inf."""
    case = TreeCase(kind[1], N, 2, H, 16, [20], [[-1, 0] + [1] * (nodes - 2)], rotary=0.0, seed=nodes)
    case.qkv[:, :N] = case.qkv[:, :N].abs() + 0.125
    case.qkv[1, N:N + 2] = -math.inf
    case.qkv[1, N + 2, 3] = math.inf
    got = case.call(kind[0])()["out"].reshape(nodes, N, H)
    assert got[1:, :N // 2].isnan().all() and got[0].isfinite().all() and got[:, N // 2:].isfinite().all()


# -------------------------------------------------------------------------------------------------------------------- biases
def sums_in_order(vocab, tokens, values):
    """Of each token its biases, added in 32 bits one after the other, and whether it has one."""
    sums, some = torch.zeros(vocab), torch.zeros(vocab, dtype=torch.bool)
    for t, v in zip(tokens.tolist(), values):
        if 0 <= t < vocab:
            sums[t] = sums[t] + v if some[t] else v
            some[t] = True
    return sums, some


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("vocab,biases,pool_of", [(50257, 30000, 20000), (1000, 3001, 40), (9001, 33, 2), (300, 64, 1), (20000, 1025, 1024)])
def test_biases_of_the_same_tokens(kind, vocab, biases, pool_of):
    """Thousands of biases, tokens named again side by side and far apart: each sum in its order, to the bit; magnitudes so far apart that another
    order shows."""
    g = torch.Generator().manual_seed(biases)
    case = LogitsCase(kind[1], 3, vocab, without=["row_list", "drafted", "allowed", "row_mask", "temperature", "history", "history_starts", "generated_starts", "repetition", "presence",
                                                  "frequency"], seed=1)
    tokens = torch.randint(-1, pool_of, (2 * biases,), generator=g) * (vocab // pool_of)
    tokens[:64] = tokens[0]
    tokens[5::97] = vocab
    values = torch.randn(2 * biases, generator=g) * 10.0 ** torch.randint(-3, 6, (2 * biases,), generator=g)
    case.t.update(bias_tokens=tokens, bias_values=values, bias_starts=torch.tensor([0, biases, biases, 2 * biases]))
    got, x = case.call(kind[0])()["scores"], case.t["logits"].float()
    for row, part in ((0, slice(0, biases)), (1, slice(0, 0)), (2, slice(biases, 2 * biases))):
        sums, some = sums_in_order(vocab, tokens[part], values[part])
        assert torch.equal(got[row], torch.where(some, x[row] + sums, x[row]))


@pytest.mark.parametrize("kind", LOGITS_KINDS)
def test_biases_of_the_same_tokens_beside_texts(kind):
    case = LogitsCase(kind[1], 3, 5003, length=3000, biases=900, drafted=3, seed=8)
    case.run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("starts", [[0, 1, 0, 0], [0, 0, 0, 5], [-1, 0, 0, 0]])
@pytest.mark.parametrize("texts", [False, True])
def test_starts_of_no_biases(kind, starts, texts):
    """Starts that leave a list of biases are an error for an empty list, too; those of an empty list are none."""
    left_out = ["row_list", "drafted", "allowed", "row_mask"] + ([] if texts else ["history", "history_starts", "generated_starts"])
    case = LogitsCase(kind[1], 3, 40, biases=0, without=left_out)
    assert len(case.t["bias_tokens"]) == 0
    case.run(kind[0])
    case.t["bias_starts"] = torch.tensor(starts)
    with pytest.raises((InvalidArgument, EPFail)):
        case.call(kind[0])()


# ---------------------------------------------------------------------------------------------------------------------- texts
@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("vocab,lengths,place", [(50257, [20000, 8193, 9001], None), (50257, [20000, 8193, 9001], 1), (300007, [9000, 12001, 8200], None), (4099, [30000, 1, 12000], None),
                                                 (16384, [8193, 8193, 8193], 1)])
def test_texts_of_more_than_64_kilobytes(kind, vocab, lengths, place):
    """Texts of more than 8192 tokens to a list on average, which a form of its own reads: fewer tokens than are listed and more, parts that count and
    parts that do not, at odd places; with drafted tokens, biases and masks, and rows that share a list."""
    g = torch.Generator().manual_seed(vocab)
    case = LogitsCase(kind[1], 5, vocab, lists=3, drafted=4, biases=300, seed=vocab)
    starts = torch.tensor([0, *lengths]).cumsum(0)
    tokens = torch.randint(-1, vocab + 1, (sum(lengths),), generator=g)
    tokens[::3] = torch.randint(0, 50, (len(tokens[::3]),), generator=g)
    case.t.update(history=tokens, history_starts=starts, generated_starts=starts[:-1] + torch.tensor([lengths[0] // 3, 0, lengths[2]]),
                  row_list=torch.tensor([1, 0, 2, -1, 0], dtype=torch.int32), repetition=torch.tensor([1.2, 1.0, 1.5, 1.3, 1.1]))
    case.run(kind[0], place=place)


# ------------------------------------------------------------------------------------------------------------------- the pool
def hold(p, seq, tokens):
    if seq not in p.sequences:
        p.open(seq)
    p.reserve(seq, tokens)
    p.advance(seq, tokens)


@pytest.mark.parametrize("held,path", [(2, [1, 3]), (0, []), (6, [0]), (8, []), (8, [1]), (7, [0, 1])])
def test_pool_keeps_no_path_in_shared_blocks(held, path):
    """What another sequence holds, or would see written by the tokens that follow a shorter path, stays: the call is refused before anything moves."""
    p = pool()
    hold(p, "a", 12)
    p.fork("b", "a")
    hold(p, "c", 3)
    before = {n: t.clone() for n, t in p.tensors.items()}
    with pytest.raises(ValueError):
        p.keep({"c": (0, [1]), "a": (held, path)})
    assert p.sequences["a"].length == 12 and p.sequences["c"].length == 3
    assert all(torch.equal(t, before[n]) for n, t in p.tensors.items())


def test_pool_keeps_paths_behind_shared_blocks():
    p = pool()
    hold(p, "a", 8)
    p.fork("b", "a")
    hold(p, "a", 3)
    last = {n: t[p.sequences["a"].blocks[2], 2].clone() for n, t in p.tensors.items()}
    p.keep({"a": (8, [2]), "b": (2, range(6))})       # (all of b's tokens: nothing moves)
    assert p.sequences["a"].length == 9 and p.sequences["b"].length == 8
    assert all(torch.equal(t[p.sequences["a"].blocks[2], 0], last[n]) for n, t in p.tensors.items())
    p.close("b")
    p.keep({"a": (1, [4])})                           # nobody else's any more
    assert p.sequences["a"].length == 2


def test_pool_keeps_no_path_of_state_in_slots():
    spec = [CacheTensor("k", "k_out", "paged", (2,), torch.float32), CacheTensor("s", "s_out", "slot", (3,), torch.float32)]
    p = CachePool(spec, 4, 4, 2, torch.device("cpu"))
    hold(p, "a", 5)
    with pytest.raises(ValueError):
        p.keep({"a": (3, [1])})
    p.keep({"a": (3, [0, 1])})
    assert p.sequences["a"].length == 5


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.float8_e5m2, torch.bool, torch.int16, torch.bfloat16, torch.complex64, torch.complex128], ids=str)
@pytest.mark.parametrize("shape", [(3,), (2, 8), ()])
def test_pools_of_any_type(provider, dtype, shape):
    """Forks, kept paths and beams move bytes: caches of 8-bit floats, truth values and complex numbers, beside one of another type."""
    device = torch.device("cuda:0" if provider == "CUDAExecutionProvider" else "cpu")
    p = CachePool([CacheTensor("k", "k_out", "paged", shape, dtype), CacheTensor("v", "v_out", "paged", (2,), torch.float32)], 8, 4, 3, device)
    for t in p.tensors.values():
        raw = t.view(torch.uint8)
        raw.copy_(torch.randint(0, 2 if dtype == torch.bool else 256, raw.shape, generator=torch.Generator().manual_seed(1)))
    entries = lambda n, s: p.tensors[n].view(torch.uint8).reshape(8, 4, -1)[p.sequences[s].blocks].flatten(0, 1)[:p.sequences[s].length].clone()  # noqa: E731
    hold(p, "a", 7)
    hold(p, "c", 6)
    before = {n: entries(n, "a") for n in "kv"}
    p.fork("b", "a", 6)
    assert all(torch.equal(entries(n, "b"), before[n][:6]) for n in "kv")
    p.close("b")
    p.copy_sequence_state(["a"], ["c"])
    p.keep({"a": (1, [2, 5])})
    assert all(torch.equal(entries(n, "a"), before[n][[0, 3, 6]]) and torch.equal(entries(n, "c"), before[n]) for n in "kv")


def test_pool_moves_in_the_tensors_that_it_has_now():
    """A pool's tensor may be another one than in the call before."""
    p = pool()
    hold(p, "a", 6)
    p.fork("b", "a")
    p.close("b")
    old, p.tensors["k"] = p.tensors["k"], torch.randn(p.tensors["k"].shape)
    untouched = old.clone()
    e = p.fork("b", "a")
    assert torch.equal(old, untouched) and torch.equal(p.tensors["k"][e.blocks[1]], p.tensors["k"][p.sequences["a"].blocks[1]])


# --------------------------------------------------------------------------------------------------------------- grammars
class Strict:
    """Even and odd tokens by turns, as a state machine: a text that it has not allowed is an error."""

    def __init__(self, end=None, kind=list):
        self.end, self.kind, self.asked = end, kind, 0

    def __call__(self, done):
        self.asked += 1
        assert self.end not in done, "nothing follows the end"
        for i, t in enumerate(done):
            assert t % 2 == i % 2, "never allowed: %s" % done
        return self.kind(t for t in range(40) if t % 2 == len(done) % 2 or t == self.end)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("end", [None, 7])
@pytest.mark.parametrize("kind", [list, set, lambda g: torch.tensor(list(g)), lambda g: g], ids=["list", "set", "tensor", "iterator"])
def test_a_grammar_is_asked_only_about_what_it_allows(provider, end, kind):
    """Drafts out of prompts that break the grammar everywhere, and that repeat an end token."""
    prompts = [[1, 3, 7, 1, 3, 8, 1, 3, 9, 1] * 2, [4, 4, 5, 5, 4, 4, 7, 5, 5], [0, 1, 2, 3] * 5]
    r = decoder(provider, dtype="fp32", batch=2, vocab=40)
    want = generate_requests(r, prompts, GenerationConfig(max_new_tokens=20, eos_token_id=end, grammar=Strict(end, kind)))
    for drafts in (1, 6, 30):
        steps, whole = [], r.draft_step
        r.draft_step = lambda entries: steps.extend((e[1], e[2]) for e in entries) or whole(entries)
        got = generate_requests(r, prompts, GenerationConfig(max_new_tokens=20, eos_token_id=end, grammar=Strict(end, kind), draft_tokens=drafts))
        r.draft_step = whole
        assert got == want
        assert any(len(tokens) > 1 for tokens, _ in steps)
        for tokens, parents in steps:     # what is drafted could be chosen
            assert all(p < 0 or (tokens[p] % 2 != t % 2 and t != end) for t, p in zip(tokens, parents) if p > 0)
            assert end not in tokens[1:]


@pytest.mark.parametrize("provider", PROVIDERS)
def test_a_grammar_that_names_what_is_no_token(provider):
    """-1 is not the last token of the vocabulary, and what lies behind it is none."""
    device = torch.device("cuda" if provider == "CUDAExecutionProvider" else "cpu")
    named = [[3, -1], [40, 5, 1 << 40], [], [-41, 39], None]
    processor = LogitsProcessor(40, torch.float32, device, GenerationConfig(grammar=lambda done: named[done[0]]))
    scores = processor(torch.zeros(5, 40, device=device), [([i], 1, [[]]) for i in range(5)]).cpu()
    assert [(row == 0).nonzero().flatten().tolist() for row in scores] == [[3], [5], [], [39], list(range(40))]


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("vocab", [1, 7, 8, 31, 32, 33, 77, 1000])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("kind", [torch.bool, torch.float32, torch.bfloat16, torch.int64])
def test_masks_of_grammars_and_vocabularies(provider, vocab, masked, kind):
    """Rows with equal masks, with masks of their own and with none, under a constant mask of any type; that one is laid out once."""
    device, g = torch.device("cuda" if provider == "CUDAExecutionProvider" else "cpu"), torch.Generator().manual_seed(vocab)
    keep = torch.rand(vocab, generator=g) < 0.7 if masked else torch.ones(vocab, dtype=torch.bool)
    named = [torch.randint(0, vocab, (n,), generator=g).tolist() for n in (0, 1, 9, 300)] + [None]
    rows = [4, 2, 2, 0, 3, 4, 1, 2]
    processor = LogitsProcessor(vocab, torch.float32, device, GenerationConfig(grammar=lambda done: named[done[0]], vocab_mask=keep.to(kind) if masked else None))
    scores = processor(torch.zeros(len(rows), vocab, device=device), [([r], 1, [[]]) for r in rows]).cpu()
    for r, row in zip(rows, scores):
        want = keep.clone()
        if named[r] is not None:
            want &= torch.isin(torch.arange(vocab), torch.tensor(named[r], dtype=torch.int64))
        assert torch.equal(row == 0, want) and (row[~want] == -math.inf).all()
    if masked:
        alone = LogitsProcessor(vocab, torch.float32, device, GenerationConfig(vocab_mask=keep.to(kind)))
        alone._words = None
        assert torch.equal(alone(torch.zeros(2, vocab, device=device), [([1], 1, [[]]), ([2], 0, [[]])]).cpu() == 0, keep.expand(2, -1))


@pytest.mark.parametrize("drafts", [0, 6])
def test_requests_of_a_call_that_fails_are_given_back(drafts):
    """A grammar that raises ends its call; the next one starts anew, with all blocks, and does not go on behind what the first one left."""
    r = decoder("CPUExecutionProvider", dtype="fp32", batch=2, vocab=40)
    prompts = [[1, 2, 3, 1, 2, 3, 1, 2], [5, 6, 5, 6, 5]]
    want = generate_requests(r, prompts, GenerationConfig(max_new_tokens=8, draft_tokens=drafts))

    def broken(done):
        if len(done) >= 3:
            raise KeyError(done[-1])
    with pytest.raises(KeyError):
        generate_requests(r, prompts, GenerationConfig(max_new_tokens=8, draft_tokens=drafts, grammar=broken))
    assert not r.pool.sequences and len(r.pool.free_blocks) == r.pool.num_blocks and r._drafted == {}
    assert generate_requests(r, prompts, GenerationConfig(max_new_tokens=8, draft_tokens=drafts)) == want


@pytest.mark.parametrize("kw", [dict(repetition_penalty=1.2), dict(logit_bias={1: 1.0}), dict(grammar=lambda done: [1]), dict(temperature=0.5), dict()], ids=lambda k: " ".join(k) or "idle")
def test_no_rows(kw):
    """A batch without a request."""
    processor = LogitsProcessor(40, torch.bfloat16, torch.device("cpu"), GenerationConfig(**kw))
    got = processor(torch.zeros(0, 40, dtype=torch.bfloat16), [])
    assert got.shape == (0, 40) and got.dtype == torch.float32
    assert processor(torch.zeros(1, 40, dtype=torch.bfloat16), [([1], 0, [[]])]).shape == (1, 40)


# ----------------------------------------------------------------------------------------------------------------- limits of drafts
def test_drafts_of_a_text_that_overlaps_itself():
    """The longest tail first, of its occurrences the latest first, each with half as many tokens as there may be: worked out by hand."""
    assert draft_tree([5, 5, 5, 5], 3) == ([5, 5, 5], [-1, 0, 1])
    assert draft_tree([5, 5, 5, 5], 1) == ([5, 5], [-1, 0])
    assert draft_tree([5, 5, 5, 5, 5], 6, 2) == ([5, 5, 5, 5], [-1, 0, 1, 2])
    assert draft_tree([1, 2, 1, 2, 1], 4, 2) == ([1, 2, 1], [-1, 0, 1])


@pytest.mark.parametrize("drafts", [255, 256, 300, 1 << 40])
def test_drafts_beyond_the_largest_tree(drafts):
    """A text that offers more drafts than a tree has: the step takes the largest tree, and the call goes on."""
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, 4, (500,), generator=g).tolist()
    r = decoder("CPUExecutionProvider", dtype="fp32", batch=1, max_len=1024, vocab=40)
    want = generate_requests(r, [prompt], GenerationConfig(max_new_tokens=400, vocab_mask=torch.arange(40) < 4, repetition_penalty=1.5))
    sizes, whole = [], r.draft_step
    r.draft_step = lambda entries: sizes.extend(len(e[1]) for e in entries) or whole(entries)
    got = generate_requests(r, [prompt], GenerationConfig(max_new_tokens=400, vocab_mask=torch.arange(40) < 4, repetition_penalty=1.5, draft_tokens=drafts))
    assert got == want and max(sizes) == 256


# --------------------------------------------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("provider", PROVIDERS)
def test_sampled_drafts_of_a_request_that_runs_alone(provider):
    """One request's draws come in the order of its tokens, whether a step gives one or several: a seed gives the same tokens with and without drafts."""
    prompt = [1, 2, 3, 4, 1, 2, 3, 4, 1, 2]
    kw = dict(max_new_tokens=24, top_k=2, temperature=0.2, vocab_mask=torch.arange(40) < 5)
    r = decoder(provider, dtype="fp32", batch=1, vocab=40)
    for seed in range(3):
        want = generate_requests(r, [prompt], GenerationConfig(seed=seed, **kw))
        assert generate_requests(r, [prompt], GenerationConfig(seed=seed, draft_tokens=6, **kw)) == want


@pytest.mark.parametrize("provider", PROVIDERS)
def test_sampled_drafts_of_requests_that_run_together(provider):
    """They share the draws, in another order than without drafts; a seed gives the same tokens again, and none that may not be chosen."""
    prompts = [[1, 2, 3, 4, 1, 2, 3, 4, 1, 2], [3, 2, 3, 2, 3], [4, 4, 4]]
    cfg = GenerationConfig(max_new_tokens=24, top_k=2, temperature=0.5, vocab_mask=torch.arange(40) < 5, seed=1, draft_tokens=6)
    r = decoder(provider, dtype="fp32", batch=2, vocab=40)
    first = generate_requests(r, prompts, cfg)
    assert generate_requests(r, prompts, cfg) == first and all(len(t) == 24 and max(t) < 5 for t in first)


# ---------------------------------------------------------------------------------------------------------------------- options
@pytest.mark.parametrize("option", [dict(presence_penalty=0.5), dict(frequency_penalty=-0.1), dict(logit_bias={3: 1.0}), dict(grammar=lambda done: None), dict(draft_tokens=2)], ids=lambda o: list(o)[0])
@pytest.mark.parametrize("beams", [1, 2])
def test_a_fixed_batch_refuses_options_that_it_does_not_have(option, beams):
    """What only generate_requests() applies is an error in generate(), and not without effect."""
    r = decoder("CPUExecutionProvider", trees=False, dtype="fp32", batch=beams, vocab=40)
    with pytest.raises(ValueError, match=list(option)[0]):
        generate(r, torch.tensor([[1, 2, 3]]), GenerationConfig(max_new_tokens=2, num_beams=beams, **option))
    assert generate(r, torch.tensor([[1, 2, 3]]), GenerationConfig(max_new_tokens=2, num_beams=beams, logit_bias={}, draft_ngram=2)).shape == (1, 5)


def test_drafts_of_the_fixed_batch_wait_for_accept():
    """The rows of prefill() and decode_step() are sequences like others: a step behind drafts that wait is refused, and new prompts forget them."""
    r = decoder("CPUExecutionProvider", dtype="fp32", batch=2, max_len=32, vocab=40)
    row = ("row", 0)
    first = r.prefill([[1, 2, 3], [4, 5]]).clone()
    want = r.decode_step(first).clone()
    r.prefill([[1, 2, 3], [4, 5]])
    r.draft_step([(row, [7, 8], [-1, 0], [1])])
    for call in (lambda: r.decode_step(first), lambda: r.reorder_cache(torch.tensor([1, 0])), lambda: r.step([(row, [1], [0])]), lambda: r.fork("x", row)):
        with pytest.raises(ValueError, match="accept"):
            call()
    r.accept({row: []})
    assert torch.equal(r.decode_step(first), want)
    r.draft_step([(row, [7, 8], [-1, 0], [1])])
    r.prefill([[1, 2, 3], [4, 5]])
    assert torch.equal(r.decode_step(first), want)
    with pytest.raises(ValueError):
        r.accept({row: [0]})
    r.draft_step([(row, [7], [-1], [0])])
    r.assume_context(9)
    r.decode_step(first)


@pytest.mark.parametrize("kind", KINDS)
def test_key_and_value_caches_in_the_same_memory(kind):
    """New values would be written over new keys."""
    case = TreeCase(kind[1], 4, 2, 64, 16, [20, 40], [[-1, 0], [-1, 0, 0]])
    call = case.call(kind[0])
    both = torch.cat([call.ins["kc"], call.ins["vc"]])
    n = len(call.ins["kc"])
    for first, second in ((0, 0), (0, 1), (n - 1, 0)):
        for name, at in (("kc", first), ("vc", second)):
            call.binding.bind_torch_input(name, both[at:at + n])
            call.binding.bind_torch_output(name + "_out", both[at:at + n])
        with pytest.raises(InvalidArgument):
            call()
    for name, at in (("kc", 0), ("vc", n)):
        call.binding.bind_torch_input(name, both[at:at + n])
        call.binding.bind_torch_output(name + "_out", both[at:at + n])
    got = call()
    case.check({**got, "kc_out": both[:n].cpu(), "vc_out": both[n:].cpu()})


# ------------------------------------------------------------------------------------------------------------ buffers by address
def by_address(call, provider, shared):
    """Runs with output `shared[0]` bound, by its address, to the memory of input `shared[1]`; returns the outputs as they are there."""
    out, into = shared
    gpu = provider == "CUDAExecutionProvider"
    t = call.ins[into].clone()
    call.binding.bind_input(into, "cuda" if gpu else "cpu", 0, t.dtype, list(t.shape), t.data_ptr())
    call.binding.bind_output(out, "cuda" if gpu else "cpu", 0, t.dtype, list(call.outs[out].shape), t.data_ptr())
    call.sess.run_with_iobinding(call.binding)
    if gpu:
        torch.cuda.synchronize()
        call.sess.check_device_status()
    return {**{n: v.cpu() for n, v in call.outs.items()}, out: t.cpu().reshape(call.outs[out].shape)}


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("vocab", [200, 50257])
def test_scores_in_the_memory_of_the_logits(provider, vocab):
    """32-bit scores bound, by their address, where the logits are: touched tokens are worked out of the logits, not of scores."""
    case = LogitsCase(torch.float32, 6, vocab, length=300, seed=2)
    case.check(by_address(case.call(provider), provider, ("scores", "logits")))


@pytest.mark.parametrize("kind", KINDS)
def test_results_in_the_memory_of_the_queries(kind):
    case = TreeCase(kind[1], 4, 2, 64, 16, [90, 80, 120], [tree(1, 0), tree(3, 1), tree(20, 2)], separate=True, seed=3)
    case.check(by_address(case.call(kind[0]), kind[0], ("out", "q")))

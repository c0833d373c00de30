"""Steps with drafted tokens, as the runner, the generation loop and the tool use the operators together: trees over a paged cache, the logits
processors of all their rows, and the move of what is accepted."""
import json

import pytest
import torch

import onnxruntime_b200 as ort
from onnxruntime_b200.models.decoder_cache import CacheFull, CachePool, CacheTensor
from onnxruntime_b200.models.generation import (GenerationConfig, LogitsProcessor, PagedDecoderRunner, draft_tree, generate_requests,
                                                process_logits)
from onnxruntime_b200.models.llama import LlamaConfig, build_llama
from onnxruntime_b200.models.registry import create_decoder

CPU, GPU = "CPUExecutionProvider", "CUDAExecutionProvider"
PROVIDERS = [pytest.param(CPU, id="cpu"), pytest.param(GPU, marks=pytest.mark.gpu, id="gpu")]


def decoder(provider, trees=True, dtype=None, batch=4, max_len=256, size=16, vocab=512, num_blocks=None):
    gpu = provider == GPU
    cfg = LlamaConfig.tiny(dtype=dtype or ("bf16" if gpu else "fp32"), max_seq_len=max_len, vocab_size=vocab, **(dict(head_dim=64) if gpu else {}))
    model, w = build_llama(cfg, weight_std=0.05, paged=True, draft_trees=trees, device="cuda" if gpu else "cpu", external_weights=True)
    so = ort.SessionOptions()
    so.add_external_initializers(list(w), list(w.values()))
    graph = "1" if trees or cfg.dtype != "fp32" else "0"      # (32-bit PagedAttention reads lengths on the host)
    sess = ort.InferenceSession(model, so, providers=[(provider, {"enable_cuda_graph": graph, "use_tf32": "0"}) if gpu else provider], **({"enable_fallback": False} if gpu else {}))
    return PagedDecoderRunner(sess, cfg, batch, max_len, block_size=size, num_slots=batch + 1, num_blocks=num_blocks)


def close(a, b, provider):
    """16-bit layers: two computations of the same values differ by a few roundings of 2^-8 through the layers of the tiny model."""
    assert (a.float() - b.float()).abs().max() <= (2.0 ** -4 if provider == GPU else 1e-5) * b.float().abs().max()


# ------------------------------------------------------------------------------------------------------------------ the pool
def pool(blocks=8, size=4, slots=4):
    spec = [CacheTensor(n, n + "_out", "paged", shape, d) for n, shape, d in (("k", (2,), torch.float32), ("v", (3, 2), torch.float16))]
    p = CachePool(spec, blocks, size, slots, torch.device("cpu"))
    for t in p.tensors.values():
        t.copy_(torch.arange(t.numel()).reshape(t.shape))
    return p


def test_pool_keeps_a_path():
    p = pool()
    for seq, n in (("a", 11), ("b", 6)):
        p.open(seq)
        p.reserve(seq, n)
        p.advance(seq, n)
    rows = {n: lambda seq, n=n: torch.stack([p.tensors[n][p.sequences[seq].blocks[i // 4], i % 4] for i in range(p.sequences[seq].length)]) for n in ("k", "v")}
    before = {(n, s): rows[n](s) for n in rows for s in "ab"}
    p.keep({"a": (3, [0, 2, 3, 7]), "b": (5, [])})
    assert p.sequences["a"].length == 7 and p.sequences["b"].length == 5
    for n in rows:
        assert torch.equal(rows[n]("a"), before[n, "a"][[0, 1, 2, 3, 5, 6, 10]]) and torch.equal(rows[n]("b"), before[n, "b"][:5])
    for chosen in (dict(a=(3, [4])), dict(a=(3, [1, 1])), dict(a=(8, [])), dict(a=(3, [-1])), dict(a=(-1, [0]))):
        with pytest.raises(ValueError):
            p.keep(chosen)
    assert p.sequences["a"].length == 7


def test_pool_copies_of_sequences_that_exchange_places():
    """Beams that swap: blocks are read before any is written, in all tensors."""
    p = pool()
    for seq in "abc":
        p.open(seq)
        p.reserve(seq, 8)
    for seq, n in zip("abc", (5, 8, 7)):
        p.advance(seq, n)
    before = {n: {s: t[p.sequences[s].blocks].clone() for s in "abc"} for n, t in p.tensors.items()}
    p.copy_sequence_state(["b", "a", "a"], ["a", "b", "c"])
    assert [p.sequences[s].length for s in "abc"] == [8, 5, 5]
    for n, t in p.tensors.items():
        for s, source in zip("abc", "baa"):
            assert torch.equal(t[p.sequences[s].blocks], before[n][source])


# ---------------------------------------------------------------------------------------------------------------------- drafts
def test_draft_trees():
    assert draft_tree([7], 4) == ([7], [-1]) and draft_tree([7, 8], 0) == ([8], [-1])
    # what followed "1 2" before, latest first, then what followed "2" alone
    tokens, parents = draft_tree([1, 2, 3, 4, 9, 1, 2, 5, 6, 2, 8, 1, 2], 6, 2)
    assert tokens == [2, 5, 6, 2, 3, 4, 9] and parents == [-1, 0, 1, 2, 0, 4, 5]
    tokens, parents = draft_tree([1, 2, 3, 4, 9, 1, 2, 5, 6, 2, 8, 1, 2], 9, 2)
    assert tokens[:4] == [2, 5, 6, 2] and len(tokens) <= 10 and all(p < i for i, p in enumerate(parents)) and len(set(zip(tokens, parents))) == len(tokens)
    assert draft_tree([5, 5, 5, 5], 3) == ([5, 5, 5], [-1, 0, 1]) or len(draft_tree([5, 5, 5, 5], 3)[0]) <= 4
    # many occurrences of a token that always goes on the same way
    assert draft_tree([1, 2] * 5000 + [1], 3, 1) == ([1, 2, 1], [-1, 0, 1])
    for most in range(1, 20):
        tokens, parents = draft_tree([i * i % 7 for i in range(60)], most)
        assert 1 < len(tokens) <= most + 1 and parents[0] == -1 and all(0 <= p < i for i, p in enumerate(parents) if i)


# ------------------------------------------------------------------------------------------------------------ logits processors
@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("kw", [dict(), dict(repetition_penalty=1.3), dict(temperature=0.7), dict(no_repeat_ngram_size=2), dict(no_repeat_ngram_size=1), dict(no_repeat_ngram_size=3, repetition_penalty=1.1),
                                dict(eos_token_id=5, min_new_tokens=4), dict(vocab_mask=True, repetition_penalty=1.2, temperature=1.4, eos_token_id=3, min_new_tokens=9, no_repeat_ngram_size=2)], ids=str)
def test_logits_processor_equals_the_processors_of_one_row(provider, kw):
    """To the bit on the CPU, also where drafted tokens are part of the text.  On the GPU the tensor library divides by a number by multiplying with its
    reciprocal: with u = 2^-24 the reciprocal is off by u and the product by u, the operator's quotient by u, so the two differ by 3 u of the quotient at
    most, and by twice that (with a little for products of the terms) where a penalty and a temperature divide."""
    vocab, device = 77, torch.device("cuda" if provider == GPU else "cpu")
    g = torch.Generator().manual_seed(1)
    if kw.get("vocab_mask"):
        kw = {**kw, "vocab_mask": torch.rand(vocab, generator=g) < 0.6}
    cfg = GenerationConfig(**kw)
    texts = [torch.randint(0, 12, (n,), generator=g).tolist() for n in (4, 9, 30)]
    requests = [(texts[0], 0, [[]]), (texts[1], 3, [[], [4], [4, 2]]), (texts[2], 10, [[], [7, 7, 7]])]
    logits = (3 * torch.randn(6, vocab, generator=g)).to(torch.bfloat16 if provider == GPU else torch.float32).to(device)
    got = LogitsProcessor(vocab, logits.dtype, device, cfg)(logits, requests)
    row = 0
    for text, new, paths in requests:
        for path in paths:
            want = process_logits(logits[row:row + 1], torch.tensor([text + path], device=device), new + len(path), cfg)
            if provider == CPU:
                assert torch.equal(got[row:row + 1], want)
            else:
                finite = want.isfinite()
                assert torch.equal(got[row:row + 1][~finite], want[~finite])
                assert ((got[row:row + 1] - want).abs()[finite] <= 6.01 * 2.0 ** -24 * want.abs()[finite]).all()
            row += 1


@pytest.mark.parametrize("provider", PROVIDERS)
def test_logits_processor_penalties_biases_and_grammar(provider):
    device = torch.device("cuda" if provider == GPU else "cpu")
    cfg = GenerationConfig(presence_penalty=0.5, frequency_penalty=0.25, logit_bias={3: 2.0, 9: -1.0}, grammar=lambda done: None if not done else [3, 4, done[-1]])
    logits = torch.zeros(3, 40, device=device)
    got = LogitsProcessor(40, torch.float32, device, cfg)(logits, [([1, 2], 0, [[]]), ([1, 6, 6], 2, [[], [8]])]).cpu()
    want = torch.zeros(3, 40)
    want[:, 3], want[:, 9] = 2.0, -1.0
    keep = [list(range(40)), [3, 4, 6], [3, 4, 8]]
    want[1:, 6] -= 0.5 + 2 * 0.25
    want[2, 8] -= 0.75
    for r, k in enumerate(keep):
        want[r, [v for v in range(40) if v not in k]] = -torch.inf
    assert torch.equal(got, want)


# ------------------------------------------------------------------------------------------------------------------ the runner
@pytest.mark.parametrize("provider", PROVIDERS)
def test_rows_of_a_tree_equal_sequences_of_their_own(provider):
    """Every path of a tree has the logits of a sequence that brings the same tokens; what is accepted goes on like one that never drafted."""
    r, plain = decoder(provider), decoder(provider, trees=False)
    g = torch.Generator().manual_seed(2)
    ids = lambda n: torch.randint(0, 512, (n,), generator=g).tolist()  # noqa: E731
    prompts = [ids(37), ids(5)]
    close(r.step([(b, p, [len(p) - 1]) for b, p in enumerate(prompts)]), plain.step([(b, p, [len(p) - 1]) for b, p in enumerate(prompts)]), provider)
    trees = [(ids(7), [-1, 0, 0, 1, 1, 2, 5]), (ids(4), [-1, 0, 1, 0])]
    for _ in range(3):
        logits = r.draft_step([(b, *t, range(len(t[0]))) for b, t in enumerate(trees)])
        row = 0
        for b, (tokens, parents) in enumerate(trees):
            for i in range(len(tokens)):
                path, j = [], i
                while j >= 0:
                    path.insert(0, j)
                    j = parents[j]
                plain.fork("one", b)
                want = plain.step([("one", [tokens[p] for p in path], [len(path) - 1])])
                plain.release("one")
                close(logits[row:row + 1], want, provider)
                row += 1
        with pytest.raises(ValueError):
            r.step([(0, [1], [0])])                       # waits for accept()
        with pytest.raises(ValueError):
            r.accept({0: [0, 3]})
        with pytest.raises(ValueError):
            r.fork("two", 0)
        r.accept({0: [0, 2, 5, 6], 1: [0, 3]})
        plain.step([(0, [trees[0][0][p] for p in (0, 2, 5, 6)], []), (1, [trees[1][0][p] for p in (0, 3)], [])])
        assert [r.pool.sequences[b].length for b in (0, 1)] == [plain.pool.sequences[b].length for b in (0, 1)]
        for step in range(2):
            one = ids(2)
            close(r.step([(b, [one[b]], [0]) for b in (0, 1)]), plain.step([(b, [one[b]], [0]) for b in (0, 1)]), provider)
    r.release(0)
    r.release(1)
    assert len(r.pool.free_blocks) == r.pool.num_blocks


def test_draft_step_refusals():
    r = decoder(CPU, batch=2)
    r.step([(0, [1, 2, 3], [])])
    for entry in ((0, [1, 2], [-1], [0]), (0, [1, 2], [-1, 1], [0]), (0, [1, 2], [-2, 0], [0]), (0, [1, 2], [-1, 0], [2]), (0, [1] * 300, [-1] * 300, [])):
        with pytest.raises((ValueError, CacheFull)):
            r.draft_step([entry])
    with pytest.raises(ValueError):
        r.draft_step([(0, [1], [-1], [0]), (0, [2], [-1], [0])])
    with pytest.raises(ValueError):
        r.accept({0: [0]})
    assert r.pool.sequences[0].length == 3 and r.draft_step([]).shape == (0, 512)
    with pytest.raises(ValueError):
        decoder(CPU, trees=False).draft_step([(0, [1], [-1], [0])])
    with pytest.raises(ValueError):
        generate_requests(decoder(CPU, trees=False), [[1, 2]], GenerationConfig(draft_tokens=2))
    with pytest.raises(ValueError):
        generate_requests(r, [[1, 2]], GenerationConfig(draft_tokens=-1))


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("kw", [dict(), dict(repetition_penalty=1.2, frequency_penalty=0.1), dict(no_repeat_ngram_size=2, temperature=0.8), dict(eos_token_id=7, min_new_tokens=5),
                                dict(presence_penalty=0.3, logit_bias={4: 1.0}, grammar=lambda done: range(0, 40, 2) if len(done) % 2 else None)],
                         ids=["greedy", "repetition", "ngrams", "end", "grammar"])
def test_drafted_requests_equal_requests_without(provider, kw):
    """Greedy tokens, with 32-bit layers, in which rows of a tree and single rows differ far less than the best tokens do; a small vocabulary, so
    that drafts are often right; more requests than run at a time."""
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, 40, (n,), generator=g).tolist() for n in (20, 3, 45, 11)] + [[1, 2, 3, 4] * 6]
    want = generate_requests(decoder(provider, trees=False, dtype="fp32", batch=3, vocab=40), prompts, GenerationConfig(max_new_tokens=24, **kw))
    r = decoder(provider, dtype="fp32", batch=3, vocab=40)
    for drafts in (1, 6, 30):
        steps = []
        whole = r.draft_step
        r.draft_step = lambda entries: steps.append([len(e[1]) for e in entries]) or whole(entries)
        got = generate_requests(r, prompts, GenerationConfig(max_new_tokens=24, draft_tokens=drafts, **kw))
        r.draft_step = whole
        assert got == want and steps and max(map(max, steps)) <= drafts + 1
        assert len(r.pool.free_blocks) == r.pool.num_blocks and r._drafted == {}


@pytest.mark.parametrize("provider", PROVIDERS)
def test_drafted_requests_report_log_probabilities_and_sample(provider):
    r = decoder(provider, dtype="fp32", batch=2, vocab=40)
    prompts = [[1, 2, 3, 4, 1, 2, 3, 4, 1, 2], [5, 6, 5, 6, 5]]
    a = generate_requests(r, prompts, GenerationConfig(max_new_tokens=12, logprobs=2))
    b = generate_requests(r, prompts, GenerationConfig(max_new_tokens=12, logprobs=2, draft_tokens=5))
    for x, y in zip(a, b):
        assert x.tokens == y.tokens and x.top_tokens == y.top_tokens and torch.allclose(torch.tensor(x.log_probs), torch.tensor(y.log_probs), atol=1e-4)
    for text in generate_requests(r, prompts, GenerationConfig(max_new_tokens=12, draft_tokens=5, top_k=4, seed=1)):
        assert len(text) == 12 and all(0 <= t < 40 for t in text)


def test_drafts_stay_within_the_room_that_is_kept():
    """A pool with just the blocks that the requests need."""
    r = decoder(CPU, batch=1, max_len=32, size=4, vocab=40, num_blocks=7)
    got = generate_requests(r, [[1, 2, 3, 4] * 4], GenerationConfig(max_new_tokens=12, draft_tokens=20))
    assert len(got[0]) == 12 and len(r.pool.free_blocks) == 7


def test_registry_and_tool(tmp_path, capsys):
    from onnxruntime_b200.safetensors_lite import save_file
    from onnxruntime_b200.tools.generate import main
    config = dict(architectures=["LlamaForCausalLM"], vocab_size=64, hidden_size=32, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, intermediate_size=48,
                  rms_norm_eps=1e-5, rope_theta=10000.0, max_position_embeddings=128)
    g = torch.Generator().manual_seed(0)
    w = {"model.embed_tokens.weight": (64, 32), "lm_head.weight": (64, 32), "model.norm.weight": (32,)}
    for i in range(2):
        p = f"model.layers.{i}."
        w.update({p + "self_attn.q_proj.weight": (32, 32), p + "self_attn.k_proj.weight": (16, 32), p + "self_attn.v_proj.weight": (16, 32), p + "self_attn.o_proj.weight": (32, 32),
                  p + "mlp.gate_proj.weight": (48, 32), p + "mlp.up_proj.weight": (48, 32), p + "mlp.down_proj.weight": (32, 48), p + "input_layernorm.weight": (32,),
                  p + "post_attention_layernorm.weight": (32,)})
    tensors = {n: 0.3 * torch.randn(s, generator=g) + (1.0 if len(s) == 1 else 0.0) for n, s in w.items()}
    with open(tmp_path / "config.json", "w") as f:
        json.dump(config, f)
    save_file(tensors, str(tmp_path / "model.safetensors"))
    args = ["--model", str(tmp_path), "--dtype", "float32", "--provider", "cpu", "--max-new-tokens", "9", "--frequency-penalty", "0.2", "--presence-penalty", "0.1"]
    prompts = ["--prompt-ids", "1,2,3,1,2,3,1", "--prompt-ids", "9,9,9"]
    assert main(args + prompts) == 0
    want = capsys.readouterr().out
    assert main(args + prompts + ["--draft-tokens", "4"]) == 0
    assert capsys.readouterr().out == want
    runner = create_decoder(config, tensors, "float32", batch=1, max_len=64, provider=CPU, draft_trees=True)
    assert "TreePagedAttention" in {n["op_type"] for n in runner.sess.graph_nodes()}
    with pytest.raises(ValueError):
        create_decoder(config, tensors, "float32", batch=1, max_len=64, provider=CPU, draft_trees=True, shared_prefix=True)
    with pytest.raises(ValueError):
        create_decoder(dict(architectures=["Fegilix"], vocab_size=64, hidden_size=64, num_hidden_layers=2, num_attention_heads=2), None, provider=CPU, draft_trees=True)

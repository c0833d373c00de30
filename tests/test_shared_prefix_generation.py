"""Sequences that begin with the same tokens: cache blocks in common, the decoder form that attends to them once, log probabilities of what is
generated and of given texts, and the gradient of log probabilities in a training graph."""
import json
import math

import numpy as np
import pytest
import torch

import onnxruntime_b200 as ort
from onnxruntime_b200 import onnx_lite as ol
from onnxruntime_b200.models.decoder_cache import CacheFull, CachePool, CacheTensor
from onnxruntime_b200.models.generation import GenerationConfig, Generated, PagedDecoderRunner, generate_requests, score_requests
from onnxruntime_b200.models.llama import LlamaConfig, build_llama
from onnxruntime_b200.models.registry import create_decoder
from onnxruntime_b200.training.gradient_builder import build_gradient_graph

CPU, GPU = "CPUExecutionProvider", "CUDAExecutionProvider"
PROVIDERS = [pytest.param(CPU, id="cpu"), pytest.param(GPU, marks=pytest.mark.gpu, id="gpu")]


# ------------------------------------------------------------------------------------------------------------------ the pool
def pool(blocks=8, size=4, slots=4, slot_state=False):
    spec = [CacheTensor("k", "k_out", "paged", (2,), torch.float32)]
    if slot_state:
        spec.append(CacheTensor("s", "s_out", "slot", (3,), torch.float32))
    return CachePool(spec, blocks, size, slots, torch.device("cpu"))


def hold(p, seq, tokens):
    if seq not in p.sequences:
        p.open(seq)
    p.reserve(seq, tokens)
    p.advance(seq, tokens)


def test_pool_fork_shares_whole_blocks_and_copies_the_rest():
    p = pool()
    hold(p, "a", 10)
    p.tensors["k"].copy_(torch.arange(8 * 4 * 2).reshape(8, 4, 2).float())
    a = p.sequences["a"]
    b = p.fork("b", "a")
    assert b.blocks[:2] == a.blocks[:2] and b.blocks[2] not in a.blocks and b.length == 10
    assert torch.equal(p.tensors["k"][b.blocks[2]], p.tensors["k"][a.blocks[2]])
    c = p.fork("c", "b", 8)
    assert c.blocks == a.blocks[:2] and p.common_tokens(["a", "b", "c"]) == 8 == p.common_tokens(["b", "c"]) and p.common_tokens(["a"]) == 10
    assert len(p.free_blocks) == 8 - 4
    shared = list(a.blocks[:2])
    p.close("a")
    assert not set(shared) & set(p.free_blocks) and len(p.free_blocks) == 5
    p.close("c")
    assert not set(shared) & set(p.free_blocks)
    p.close("b")
    assert sorted(p.free_blocks) == list(range(8)) and p.owners == {} and len(p.free_slots) == 4
    assert p.common_tokens([]) == 0


def test_pool_fork_of_nothing_and_refusals():
    p = pool(blocks=3, slots=3, slot_state=True)
    hold(p, "a", 9)
    with pytest.raises(CacheFull):
        p.fork("b", "a")                       # the copy of the third block has no room
    assert "b" not in p.sequences and p.owners == {} and len(p.free_slots) == 2
    with pytest.raises(ValueError):
        p.fork("b", "a", 8)                    # recurrent state is that of all nine tokens
    with pytest.raises(ValueError):
        p.fork("b", "a", 10)
    with pytest.raises(ValueError):
        p.fork("a", "a", 9)
    q = pool(slot_state=True)
    hold(q, "a", 8)
    q.tensors["s"][q.sequences["a"].slot] = 5.0
    e = q.fork("b", "a")
    assert (q.tensors["s"][e.slot] == 5.0).all() and e.slot != q.sequences["a"].slot
    with pytest.raises(ValueError):
        q.copy_sequence_state(["a"], ["b"])    # would write into blocks of both
    r = pool()
    hold(r, "a", 6)
    assert r.fork("b", "a", 0).blocks == [] and r.common_tokens(["a", "b"]) == 0


# ----------------------------------------------------------------------------------------------------------------- the decoder
def decoders(provider, size, batch, max_len, num_blocks=None):
    """The plain paged form and the one with a shared prefix, same weights."""
    gpu = provider == GPU
    cfg = LlamaConfig.tiny(dtype="bf16" if gpu else "fp32", max_seq_len=256, **(dict(head_dim=64) if gpu else {}))
    got = []
    for shared in (False, True):
        model, w = build_llama(cfg, weight_std=0.05, paged=True, shared_prefix=shared, block_size=size, device="cuda" if gpu else "cpu", external_weights=True)
        so = ort.SessionOptions()
        so.add_external_initializers(list(w), list(w.values()))
        sess = ort.InferenceSession(model, so, providers=[(provider, {"enable_cuda_graph": "1"}) if gpu else provider], **({"enable_fallback": False} if gpu else {}))
        got.append(PagedDecoderRunner(sess, cfg, batch, max_len, block_size=size, num_blocks=num_blocks, num_slots=batch + 1))
    assert {n["op_type"] for n in got[1].sess.graph_nodes()} >= {"PagedBatchLayout", "SharedPrefixPagedAttention"}
    return cfg, got[0], got[1]


def close(a, b, provider):
    """16-bit layers: two computations of the same values differ by a few roundings of 2^-8 through the layers of the tiny model."""
    scale = b.float().abs().max()
    assert (a.float() - b.float()).abs().max() <= (2.0 ** -4 if provider == GPU else 1e-5) * scale


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("prefix", [64, 70, 150])
def test_steps_of_forked_sequences_equal_steps_without_sharing(provider, prefix):
    size = 16
    cfg, plain, shared = decoders(provider, size, 4, 256)
    g = torch.Generator().manual_seed(prefix)
    ids = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()  # noqa: E731
    common, own = ids(prefix), [ids(3), ids(40), ids(1)]
    shared.step([("common", common, [])])
    for b in range(3):
        shared.fork(b, "common")
    want = plain.step([(b, common + own[b], [prefix + len(own[b]) - 1]) for b in range(3)])
    got = shared.step([(b, own[b], [len(own[b]) - 1]) for b in range(3)])
    close(got, want, provider)
    for step in range(20):                       # crosses block borders; a sequence leaves and another one joins on the way
        if step == 7:
            for r in (plain, shared):
                r.release(1)
            shared.fork(3, "common")
            new = ids(5)
            close(shared.step([(3, new, [4])]), plain.step([(3, common + new, [prefix + 4])]), provider)
        live = [0, 1, 2] if step < 7 else [0, 2, 3]
        tokens = ids(3)
        entries = [(b, [t], [0]) for b, t in zip(live, tokens)]
        want, got = plain.step(entries), shared.step(entries)
        close(got, want, provider)
    shared.release("common")
    for b in live:
        shared.release(b)
    assert len(shared.pool.free_blocks) == shared.pool.num_blocks


@pytest.mark.parametrize("provider", PROVIDERS)
def test_fixed_batch_of_the_shared_form(provider):
    cfg, plain, shared = decoders(provider, 16, 3, 96)
    g = torch.Generator().manual_seed(3)
    prompts = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (5, 33, 16)]
    for r in (plain, shared):
        r.prefill(prompts)
    close(shared.prefill_logits, plain.prefill_logits, provider)
    for _ in range(20):
        tokens = torch.randint(0, cfg.vocab_size, (3,), generator=g)
        plain.decode_step(tokens)
        shared.decode_step(tokens)
        close(shared.step_logits, plain.step_logits, provider)


def test_requests_behind_a_shared_prompt():
    """The same tokens as without sharing, with log probabilities; fewer blocks are in use, and all come back."""
    cfg, plain, shared = decoders(CPU, 8, 3, 96, num_blocks=40)
    g = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()  # noqa: E731
    common, prompts = ids(29), [ids(n) for n in (1, 7, 12, 4, 9)]
    want = generate_requests(plain, [common + p for p in prompts], GenerationConfig(max_new_tokens=6))
    assert generate_requests(shared, prompts, GenerationConfig(max_new_tokens=6), common) == want
    assert generate_requests(plain, prompts, GenerationConfig(max_new_tokens=6), common) == want      # any model can share blocks
    got = generate_requests(shared, prompts, GenerationConfig(max_new_tokens=6, logprobs=3), common)
    assert [d.tokens for d in got] == want and all(isinstance(d, Generated) for d in got)
    for r in (plain, shared):
        assert len(r.pool.free_blocks) == 40 and not r.pool.sequences and r.pool.owners == {}
    for prompt, d in zip(prompts, got):          # against the model's own logits
        logits = plain.step([("check", common + prompt + d.tokens[:-1], range(len(common) + len(prompt) - 1, len(common) + len(prompt) + 5))])
        plain.release("check")
        logp = torch.log_softmax(logits.double(), -1)
        # two computations of the same 32-bit logits, of size below 10: 1e-4
        np.testing.assert_allclose(d.log_probs, logp[torch.arange(6), d.tokens], atol=1e-4)
        np.testing.assert_allclose(d.entropies, -(logp.exp() * logp).sum(-1), atol=1e-4)
        assert [t[0] for t in d.top_tokens] == d.tokens and all(len(t) == 3 for t in d.top_tokens)
        np.testing.assert_allclose(d.top_log_probs, logp.topk(3, -1)[0], atol=1e-4)


@pytest.mark.parametrize("form", ["plain", "shared"])
@pytest.mark.parametrize("rows", [4, 1024])
def test_scores_of_given_texts(form, rows):
    cfg, plain, shared = decoders(CPU, 8, 2, 96)
    runner = plain if form == "plain" else shared
    g = torch.Generator().manual_seed(2)
    ids = lambda n: torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist()  # noqa: E731
    common, texts = ids(11), [ids(9), [], ids(1), ids(20)]
    for prompt in (common, []):
        got = score_requests(runner, texts, 2, prompt, rows)
        for text, d in zip(texts, got):
            whole = prompt + text
            first = len(prompt) if prompt else 1
            assert d.tokens == whole[first:] and len(d.log_probs) == len(d.entropies) == len(d.top_tokens) == len(d.tokens)
            if not d.tokens:
                continue
            logits = plain.step([("check", whole, range(len(whole)))])
            plain.release("check")
            logp = torch.log_softmax(logits.double(), -1)[first - 1:-1]
            np.testing.assert_allclose(d.log_probs, logp[torch.arange(len(d.tokens)), d.tokens], atol=1e-4)
            np.testing.assert_allclose(d.top_log_probs, logp.topk(2, -1)[0], atol=1e-4)
    assert not runner.pool.sequences


def test_a_shared_prompt_needs_room_and_prompts():
    cfg, plain, shared = decoders(CPU, 8, 2, 32)
    with pytest.raises(ValueError):
        generate_requests(shared, [[1], []], GenerationConfig(max_new_tokens=2), [1, 2])
    with pytest.raises(CacheFull):
        generate_requests(shared, [[1]], GenerationConfig(max_new_tokens=2), [1] * 33)
    assert not shared.pool.sequences


def test_a_call_that_is_given_up_leaves_nothing_open():
    """The second request outgrows the longest sequence when it joins; the first is under way."""
    shared = decoders(CPU, 16, 2, 64)[2]
    free = len(shared.pool.free_blocks)
    with pytest.raises(CacheFull):
        generate_requests(shared, [[3], [4] * 60], GenerationConfig(max_new_tokens=5), shared_prompt=[1] * 20)
    assert shared.pool.sequences == {} and len(shared.pool.free_blocks) == free and shared.pool.owners == {}
    assert [len(r) for r in generate_requests(shared, [[3], [4]], GenerationConfig(max_new_tokens=5), shared_prompt=[1] * 20)] == [5, 5]


def test_registry_and_tool(tmp_path, capsys):
    from onnxruntime_b200.safetensors_lite import save_file
    from onnxruntime_b200.tools.generate import main
    config = dict(architectures=["LlamaForCausalLM"], vocab_size=64, hidden_size=32, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                  intermediate_size=48, rms_norm_eps=1e-5, rope_theta=10000.0, max_position_embeddings=128)
    g = torch.Generator().manual_seed(0)
    w = {"model.embed_tokens.weight": (64, 32), "lm_head.weight": (64, 32), "model.norm.weight": (32,)}
    for i in range(2):
        p = f"model.layers.{i}."
        w.update({p + "self_attn.q_proj.weight": (32, 32), p + "self_attn.k_proj.weight": (16, 32), p + "self_attn.v_proj.weight": (16, 32),
                  p + "self_attn.o_proj.weight": (32, 32), p + "mlp.gate_proj.weight": (48, 32), p + "mlp.up_proj.weight": (48, 32),
                  p + "mlp.down_proj.weight": (32, 48), p + "input_layernorm.weight": (32,), p + "post_attention_layernorm.weight": (32,)})
    tensors = {n: 0.3 * torch.randn(s, generator=g) + (1.0 if len(s) == 1 else 0.0) for n, s in w.items()}
    with open(tmp_path / "config.json", "w") as f:
        json.dump(config, f)
    save_file(tensors, str(tmp_path / "model.safetensors"))
    args = ["--model", str(tmp_path), "--dtype", "float32", "--provider", "cpu", "--max-new-tokens", "4"]
    assert main(args + ["--prompt-ids", "1,2,3,4,5", "--prompt-ids", "1,2,3,9"]) == 0
    want = [json.loads(line)["generated"] for line in capsys.readouterr().out.splitlines()]
    assert main(args + ["--prompt-ids", "4,5", "--prompt-ids", "9", "--shared-prompt-ids", "1,2,3", "--logprobs", "2"]) == 0
    got = [json.loads(line) for line in capsys.readouterr().out.splitlines()]
    assert [d["generated"] for d in got] == want
    assert all(len(d["log_probs"]) == 4 and all(a[0][0] == t for a, t in zip(d["alternatives"], d["generated"])) for d in got)
    with pytest.raises(ValueError):
        _family_without_a_shared_form()


def _family_without_a_shared_form():
    import onnxruntime_b200.models.registry as registry
    family = registry.DecoderFamily(registry.FAMILIES["LlamaForCausalLM"].config, registry.FAMILIES["LlamaForCausalLM"].build)
    registry.register_family("Plain", family)
    try:
        create_decoder(dict(architecture="Plain", vocab_size=64, hidden_size=32, num_hidden_layers=1, num_attention_heads=4, num_key_value_heads=2, intermediate_size=48),
                       None, "float32", provider=CPU, shared_prefix=True)
    finally:
        del registry.FAMILIES["Plain"]


# ------------------------------------------------------------------------------------------------------------ training graphs
@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("outputs", [["lp"], ["lp", "h"], ["", "h"], ["", "", "top"], ["", "", "", "", "lse"], ["lp", "h", "top", "index", "lse"]])
def test_gradient_graph_of_log_probs(provider, outputs):
    """d (sum of the outputs) / d (input of the product in front of the logits) by the gradient builder, against autograd on the definitions."""
    rows, width, V, k = 4, 6, 40, 3
    g = torch.Generator().manual_seed(1)
    x, w, tokens = torch.randn(rows, width, generator=g), torch.randn(width, V, generator=g), torch.tensor([1, 39, 0, 7])
    T = ol.TensorProto
    nodes = [ol.make_node("MatMul", ["x", "w"], ["logits"]), ol.make_node("TokenLogProbs", ["logits", "tokens"], outputs, domain="com.ortb200", top_k=k)]
    parts = []
    for o in outputs:
        if o in ("lp", "h", "lse", "top"):
            nodes.append(ol.make_node("ReduceSum", [o], [o + "_sum"], keepdims=0))
            parts.append(o + "_sum")
    nodes.append(ol.make_node("Sum", parts, ["loss"]))
    info = ol.make_tensor_value_info
    graph = ol.make_graph(nodes, "g", [info("x", T.FLOAT, [rows, width]), info("w", T.FLOAT, [width, V]), info("tokens", T.INT64, [rows])], [info("loss", T.FLOAT, [])])
    model = build_gradient_graph(ol.make_model(graph, opset=17, extra_opsets={"com.ortb200": 1}), ["w"], "loss", recompute_fallback=False)
    sess = ort.InferenceSession(model.serialize(), providers=[provider])
    assert "TokenLogProbsGrad" in {n["op_type"] for n in sess.graph_nodes()}
    loss, grad = sess.run(["loss", "w_grad"], {"x": x.numpy(), "w": w.numpy(), "tokens": tokens.numpy()})
    wd = w.double().requires_grad_(True)
    logp = torch.log_softmax(x.double() @ wd, -1)
    lse = torch.logsumexp(x.double() @ wd, -1)
    want = {"lp": logp.gather(1, tokens[:, None]).sum(), "h": -(logp.exp() * logp).sum(), "top": logp.topk(k, -1)[0].sum(), "lse": lse.sum()}
    total = sum(want[o] for o in outputs if o in want)
    total.backward()
    total = total.detach()
    # 32-bit products of six terms and sums over 40: relative 2^-18 of the largest
    assert abs(float(loss) - float(total)) < 1e-4 * max(1.0, abs(float(total)))
    assert np.abs(grad - wd.grad.numpy()).max() < 1e-5 * max(1.0, float(wd.grad.abs().max())) * (64 if provider == GPU else 1)

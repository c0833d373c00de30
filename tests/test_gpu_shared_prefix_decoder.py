"""The shared-prefix decoder as ``create_decoder`` makes it for a GPU (launches that overlap, captured single-token steps): requests behind a shared prompt,
log probabilities of what is generated and of given texts."""
import numpy as np
import pytest
import torch

from onnxruntime_b200.models.generation import GenerationConfig, generate_requests, score_requests
from onnxruntime_b200.models.registry import create_decoder

CPU, GPU = "CPUExecutionProvider", "CUDAExecutionProvider"
CONFIG = dict(architectures=["LlamaForCausalLM"], vocab_size=512, hidden_size=256, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2,
              intermediate_size=384, rms_norm_eps=1e-5, rope_theta=10000.0, max_position_embeddings=512)


def weights():
    g = torch.Generator().manual_seed(0)
    w = {"model.embed_tokens.weight": (512, 256), "lm_head.weight": (512, 256), "model.norm.weight": (256,)}
    for i in range(3):
        p = f"model.layers.{i}."
        w.update({p + "self_attn.q_proj.weight": (256, 256), p + "self_attn.k_proj.weight": (128, 256), p + "self_attn.v_proj.weight": (128, 256),
                  p + "self_attn.o_proj.weight": (256, 256), p + "mlp.gate_proj.weight": (384, 256), p + "mlp.up_proj.weight": (384, 256),
                  p + "mlp.down_proj.weight": (256, 384), p + "input_layernorm.weight": (256,), p + "post_attention_layernorm.weight": (256,)})
    return {n: 0.1 * torch.randn(s, generator=g) + (1.0 if len(s) == 1 else 0.0) for n, s in w.items()}


def decoder(provider, dtype, shared=True, **entries):
    return create_decoder(CONFIG, weights(), dtype, batch=4, max_len=320, block_size=16, provider=provider, shared_prefix=shared, session_entries=entries)


def texts():
    g = torch.Generator().manual_seed(7)
    ids = lambda n: torch.randint(0, 512, (n,), generator=g).tolist()  # noqa: E731
    return ids(150), [ids(n) for n in (1, 30, 5, 90, 2, 17)]


def against_own_logits(plain, whole, d, first, tol):
    """Reported values against the logits that the form without sharing gives to the same tokens."""
    logits = plain.step([("check", whole[:-1], range(first - 1, len(whole) - 1))]).float().cpu()
    plain.release("check")
    logp = torch.log_softmax(logits.double(), -1)
    tol = 2 * tol * float(logits.abs().max())     # a difference of two logits
    np.testing.assert_allclose(d.log_probs, logp[torch.arange(len(d.tokens)), d.tokens], atol=tol)
    np.testing.assert_allclose(np.array(d.top_log_probs), logp.topk(3, -1)[0], atol=tol)
    # the entropy H moves by at most the logits' error times sum p |log p + H| <= 2 H <= 2 log 512 = 12.5
    np.testing.assert_allclose(d.entropies, -(logp.exp() * logp).sum(-1), atol=tol * 20)
    assert max(d.log_probs) <= 0 and all(a >= b for top in d.top_log_probs for a, b in zip(top, top[1:]))


# 16-bit layers: two computations of the same values differ by a few roundings of 2^-8; 32-bit ones by sums over 384 terms
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 2.0 ** -4), ("float16", 2.0 ** -7)])
def test_requests_behind_a_shared_prompt(dtype, tol):
    prompt, prompts = texts()
    shared, plain = decoder(GPU, dtype), decoder(GPU, dtype, shared=False)
    got = generate_requests(shared, prompts, GenerationConfig(max_new_tokens=25, logprobs=3), prompt)
    shared.sess.check_device_status()
    for p, d in zip(prompts, got):
        assert len(d.tokens) == 25 and [t[0] for t in d.top_tokens] == d.tokens
        against_own_logits(plain, prompt + p + d.tokens, d, len(prompt) + len(p), tol)
    assert generate_requests(shared, prompts, GenerationConfig(max_new_tokens=25), prompt) == [d.tokens for d in got]      # nothing is left from the first time
    if dtype == "float32":
        want = generate_requests(decoder(CPU, dtype), prompts, GenerationConfig(max_new_tokens=25, logprobs=3), prompt)
        assert [d.tokens for d in got] == [d.tokens for d in want]
    assert not shared.pool.sequences and len(shared.pool.free_blocks) == shared.pool.num_blocks


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 2.0 ** -4)])
@pytest.mark.parametrize("rows", [7, 1024])
def test_scores_of_given_texts(dtype, tol, rows):
    prompt, given = texts()
    shared, plain = decoder(GPU, dtype), decoder(GPU, dtype, shared=False)
    for text, d in zip(given, score_requests(shared, given, 3, prompt, rows)):
        assert d.tokens == text
        against_own_logits(plain, prompt + text, d, len(prompt), tol)
    shared.sess.check_device_status()
    assert not shared.pool.sequences


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("graph", [False, True])
def test_overlapping_launches_change_nothing(dtype, graph):
    """Every step of a growing batch, with launches that overlap and without: the same bits."""
    prompt, prompts = texts()
    runners = [create_decoder(CONFIG, weights(), dtype, batch=4, max_len=320, block_size=16, provider=GPU, shared_prefix=True, cuda_graph=graph,
                              session_entries={"ortb200.pdl": pdl}) for pdl in ("0", "1")]
    for r in runners:
        r.step([("common", prompt, [])])
        for b in range(3):
            r.fork(b, "common")
    g = torch.Generator().manual_seed(1)
    for step in range(40):
        new = [prompts[b + 1] for b in range(3)] if step == 0 else [torch.randint(0, 512, (1,), generator=g).tolist() for _ in range(3)]
        a, b = (r.step([(s, t, [len(t) - 1]) for s, t in enumerate(new)]) for r in runners)
        assert torch.equal(a, b), step
    for r in runners:
        r.sess.check_device_status()

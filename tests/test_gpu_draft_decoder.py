"""The decoder for drafted tokens as ``create_decoder`` makes it for a GPU (launches that overlap, captured single-token steps): trees, what is accepted
of them, and requests with drafts."""
import pytest
import torch

from onnxruntime_b200.models.generation import GenerationConfig, draft_tree, generate_requests
from onnxruntime_b200.models.registry import create_decoder
from test_gpu_shared_prefix_decoder import CONFIG, CPU, GPU, against_own_logits, weights


def decoder(provider, dtype, trees=True, batch=4, **how):
    return create_decoder(CONFIG, weights(), dtype, batch=batch, max_len=512, block_size=16, provider=provider, draft_trees=trees, **how)


def prompts():
    g = torch.Generator().manual_seed(7)
    ids = lambda n: torch.randint(0, 512, (n,), generator=g).tolist()  # noqa: E731
    return [ids(n) for n in (1, 30, 5, 290)] + [ids(6) * 5, ids(3) * 20]


# 16-bit layers: two computations of the same values differ by a few roundings of 2^-8; 32-bit ones by sums over 384 terms
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 2.0 ** -4), ("float16", 2.0 ** -7)])
def test_requests_with_drafts(dtype, tol):
    trees, plain = decoder(GPU, dtype), decoder(GPU, dtype, trees=False, cuda_graph=False)   # (32-bit PagedAttention reads lengths on the host)
    cfg = GenerationConfig(max_new_tokens=40, logprobs=3, draft_tokens=12)
    got = generate_requests(trees, prompts(), cfg)
    trees.sess.check_device_status()
    for p, d in zip(prompts(), got):
        assert len(d.tokens) == 40 and [t[0] for t in d.top_tokens] == d.tokens
        against_own_logits(plain, p + d.tokens, d, len(p), tol)
    assert [d.tokens for d in generate_requests(trees, prompts(), cfg)] == [d.tokens for d in got]      # nothing is left from the first time
    if dtype == "float32":
        assert [d.tokens for d in got] == generate_requests(plain, prompts(), GenerationConfig(max_new_tokens=40))
        assert [d.tokens for d in got] == generate_requests(decoder(CPU, dtype), prompts(), GenerationConfig(max_new_tokens=40, draft_tokens=12))
    assert not trees.pool.sequences and len(trees.pool.free_blocks) == trees.pool.num_blocks


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("graph", [False, True])
def test_overlapping_launches_change_nothing(dtype, graph):
    """Prompts, trees of one to 64 tokens, accepted paths and captured single-token steps in turn, with launches that overlap and without: the same bits."""
    runners = [decoder(GPU, dtype, cuda_graph=graph, session_entries={"ortb200.pdl": pdl}) for pdl in ("0", "1")]
    texts = [p[:60] for p in prompts()[:2] + prompts()[4:]]
    g = torch.Generator().manual_seed(1)
    for step in range(24):
        if step == 0:
            a, b = (r.step([(s, t, [len(t) - 1]) for s, t in enumerate(texts)]) for r in runners)
        elif step % 3 == 2:
            a, b = (r.step([(s, [t[-1]], [0]) for s, t in enumerate(texts)]) for r in runners)
        else:
            trees = [draft_tree(t, (0, 3, 15, 63)[(step + s) % 4]) for s, t in enumerate(texts)]
            a, b = (r.draft_step([(s, *tree, range(len(tree[0]))) for s, tree in enumerate(trees)]) for r in runners)
            paths = {}
            for s, (tokens, parents) in enumerate(trees):
                node = int(torch.randint(0, len(tokens), (), generator=g))
                paths[s] = []
                while node >= 0:
                    paths[s].insert(0, node)
                    node = parents[node]
                texts[s] = texts[s] + [tokens[j] for j in paths[s][1:]]
            for r in runners:
                r.accept(paths)
        assert torch.equal(a, b), step
        texts = [t + [int(torch.randint(0, 512, (), generator=g))] for t in texts]
    for r in runners:
        r.sess.check_device_status()
        for one, other in zip(runners[0].pool.tensors.values(), r.pool.tensors.values()):
            assert torch.equal(one, other)

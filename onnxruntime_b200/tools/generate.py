"""``python -m onnxruntime_b200.tools.generate --model DIR --prompt-ids 5,17,3 [--prompt-ids ...]``

Generates continuations of token-id prompts with a model folder (config.json + model.safetensors) of any family the
registry knows.  Prompts of different lengths run as one batch.  Prints one JSON line per prompt.
"""
from __future__ import annotations

import argparse
import json
import sys


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(prog="generate", description="generate token ids with a decoder")
    ap.add_argument("--model", required=True, help="folder with config.json and model.safetensors")
    ap.add_argument("--prompt-ids", action="append", required=True, help="comma-separated token ids; repeat for a batch")
    ap.add_argument("--dtype", default="bfloat16", choices=["bfloat16", "float16", "float32"])
    ap.add_argument("--provider", default="cuda", choices=["cuda", "cpu"])
    ap.add_argument("--max-new-tokens", type=int, default=32)
    ap.add_argument("--batch", type=int, default=8, help="requests that run at a time, at most")
    ap.add_argument("--eos-token-id", type=int, default=None)
    ap.add_argument("--temperature", type=float, default=1.0)
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--repetition-penalty", type=float, default=1.0)
    ap.add_argument("--presence-penalty", type=float, default=0.0)
    ap.add_argument("--frequency-penalty", type=float, default=0.0)
    ap.add_argument("--draft-tokens", type=int, default=0, help="tokens that a step may draft from the request's own text (255 at most)")
    ap.add_argument("--seed", type=int, default=None, help="sampling with this seed (greedy without it, top-k and top-p)")
    ap.add_argument("--shared-prompt-ids", default="", help="comma-separated token ids in front of every prompt; they run once")
    ap.add_argument("--logprobs", type=int, default=None, help="also report log probabilities, entropies and that many alternatives")
    a = ap.parse_args(argv)

    from onnxruntime_b200.models.generation import GenerationConfig, generate_requests
    from onnxruntime_b200.models.registry import load_decoder
    prompts = [[int(t) for t in p.split(",")] for p in a.prompt_ids]
    shared = [int(t) for t in a.shared_prompt_ids.split(",") if t]
    longest = len(shared) + max(len(p) for p in prompts) + a.max_new_tokens
    runner = load_decoder(a.model, a.dtype, batch=min(a.batch, len(prompts)), max_len=longest,
                          provider="CUDAExecutionProvider" if a.provider == "cuda" else "CPUExecutionProvider", shared_prefix=bool(shared),
                          draft_trees=a.draft_tokens > 0)
    outs = generate_requests(runner, prompts, GenerationConfig(
        max_new_tokens=a.max_new_tokens, eos_token_id=a.eos_token_id, temperature=a.temperature, top_k=a.top_k, top_p=a.top_p,
        repetition_penalty=a.repetition_penalty, seed=a.seed, logprobs=a.logprobs,
        presence_penalty=a.presence_penalty, frequency_penalty=a.frequency_penalty, draft_tokens=a.draft_tokens), shared)
    for prompt, out in zip(prompts, outs):
        if a.logprobs is None:
            print(json.dumps({"prompt": prompt, "generated": out}), flush=True)
        else:
            print(json.dumps({"prompt": prompt, "generated": out.tokens, "log_probs": out.log_probs, "entropies": out.entropies,
                              "alternatives": [list(zip(t, p)) for t, p in zip(out.top_tokens, out.top_log_probs)]}), flush=True)
    return 0


if __name__ == "__main__":
    sys.exit(main())

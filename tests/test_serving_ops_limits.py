"""The operators around a serving step at the ends of their ranges: masks of any size, logits far from zero, confident rows, lengths that fit no batch,
sizes next to 32 bits, buffers on odd addresses, and the paths of the decoder that use them on a GPU."""
import math

import pytest
import torch

from test_serving_ops import GPU, SCORE_KINDS, score_call


# ---------------------------------------------------------------------------------------------------- token log probabilities
def exact_rows(x, tokens):
    """In 64 bits, of rows of finite logits and -inf that are not all -inf: log probability of the tokens, entropy, log sum exp, log probabilities, and a
    bound on what 32-bit arithmetic may do to the sum S = sum exp(x - max), as a factor.

    With d = max - x: a running sum adds at most V / 256 + 64 terms before it is joined, each addition and joining factor rounds by 2^-24; an
    exponential is off by 2^-22, and its argument by 2^-23 d in all (difference and product), so r = (V / 256 + 64) 2^-24 + 2^-22 + 2^-23 sum p d."""
    x = x.double()
    V = x.shape[-1]
    top = x.amax(-1, keepdim=True)
    log_s = torch.log(torch.exp(x - top).sum(-1, keepdim=True))
    logp = (x - top) - log_s
    p = logp.exp()
    d = (top - x).masked_fill(p == 0, 0)
    mean = (p * d).sum(-1)
    r = (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23 * mean
    inside = (tokens >= 0) & (tokens < V)
    lp = torch.where(inside, logp.gather(-1, tokens.clamp(0, V - 1).unsqueeze(-1)).squeeze(-1), 0.0)
    # S rounds r, W = sum p d rounds r W and what d^2 adds to its exponents
    h_off = r * (1 + 2 * mean) + 2.0 ** -23 * (p * d * d).sum(-1) + 2.0 ** -22 * (1 + log_s.squeeze(-1) + mean)
    return lp, log_s.squeeze(-1) + mean, (top + log_s).squeeze(-1), logp, r, h_off


def near(name, got, want, tol):
    """Where the result fits 32 bits, within tol; where it is beyond them, -inf."""
    got, narrow = got.double(), want.float().double()
    assert torch.equal(got == -math.inf, narrow == -math.inf) and torch.isfinite(got[narrow != -math.inf]).all(), name
    keep = narrow != -math.inf
    off = ((got - want).abs() / tol)[keep]
    assert (off <= 1).all(), "%s: %g of the bound" % (name, float(off.max()))


def check_rows(kind, x, tokens, k, relative=True):
    """``relative``: log probabilities are as near as a difference to the largest logit allows; otherwise as near as one to log sum exp."""
    got = score_call(kind[0], x, tokens, k)()
    lp, h, lse, logp, r, h_off = exact_rows(x, tokens)
    size = x.double().masked_fill(x == -math.inf, 0).abs().amax(-1)
    near("lse", got["lse"], lse, r + 2.0 ** -23 * size)
    near("h", got["h"], h, h_off)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(got["index"], order)
    top = logp.gather(1, order)
    # the sum's factor, then the roundings of the difference, of log S and of their difference
    off = lambda v: r.reshape([-1] + [1] * (v.dim() - 1)) + 2.0 ** -22 * (v.abs().clamp(max=1e38) + 1) + (0 if relative else 2.0 ** -21 * size.reshape([-1] + [1] * (v.dim() - 1)))  # noqa: E731
    near("lp", got["lp"], lp, off(lp))
    near("top", got["top"], top, off(top))
    return got


def masked_rows(V, mask, dtype):
    """Rows of ordinary logits in which a finite mask takes whole rows, whole vectors, ends, beginnings and single places."""
    g = torch.Generator().manual_seed(V)
    x, at = 2 * torch.randn(12, V, generator=g), torch.arange(V)
    x[0] = -mask
    x[1, :max(V - 7, 1)] = -mask
    x[2, V // 2:] = -mask
    x[3, at != V // 3] = -mask
    x[4, at != V - 1] = -mask
    x[5, ::2] = -mask
    x[6, (at < 8) | (at >= 16)] = -mask
    x[7, at % 3 == 0], x[7, at % 3 == 1] = -mask, -math.inf
    x[8, V // 4:3 * V // 4] = -mask
    x[9, V // 5] = mask
    x[10] = mask
    x[11, at // 4096 % 2 == 0] = -mask
    return x.to(dtype)


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("V,k,times", [(40, 0, 1), (40, 3, 1), (1031, 5, 60), (50257, 0, 1), (50257, 5, 1), (20000, 0, 60)])
@pytest.mark.parametrize("mask", [1e4, 6e4, 1e6, 1e9, 2e9, 1e10, 1e15, 1e20, 1e30, 1e37, 1e38, 2.5e38, math.inf])
def test_log_probs_with_finite_masks(kind, V, k, times, mask):
    """Masks of every size up to the type's lowest value (``inf`` stands for that)."""
    most, times = torch.finfo(kind[1]).max, times if kind[0] == GPU else 1   # (many rows are another division of the work on a GPU alone)
    if mask > most and mask != math.inf:
        pytest.skip("beyond the type")
    x = masked_rows(V, min(mask, most), kind[1]).repeat(times, 1)
    tokens = torch.tensor([0, V - 1, 1, V // 3, V - 1, 3, 9, 2, 0, V // 5, 7, V - 1]).repeat(times)
    check_rows(kind, x, tokens, k, relative=False)


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("V,times", [(40, 1), (50257, 1), (20000, 60)])
@pytest.mark.parametrize("mask", [1e4, 1e6, 1e10, 1e30, math.inf])
def test_log_probs_relative_to_the_largest_logit(kind, V, times, mask):
    """A row of equal logits has the log probability -log V whatever their size."""
    most, times = torch.finfo(kind[1]).max, times if kind[0] == GPU else 1   # (many rows are another division of the work on a GPU alone)
    if mask > most and mask != math.inf:
        pytest.skip("beyond the type")
    x = masked_rows(V, min(mask, most), kind[1]).repeat(times, 1)
    tokens = torch.tensor([0, V - 1, 1, V // 3, V - 1, 3, 9, 2, 0, V // 5, 7, V - 1]).repeat(times)
    got = check_rows(kind, x, tokens, 3)
    assert (got["lp"][::12] + math.log(V)).abs().max() < 1e-4


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("base", [0.0, 5.0, 23.7, 60.0, 333.3, 1000.0, -1000.0, 30000.0])
def test_log_probs_of_confident_rows(kind, base):
    """Tokens of nearly all the probability: no log probability above 0, and each as near as the difference to the largest logit allows."""
    V, rows = 3001, 200
    g = torch.Generator().manual_seed(int(abs(base)))
    x = base + torch.randn(rows, V, generator=g)
    tokens = torch.randint(0, V, (rows,), generator=g)
    margin = torch.linspace(5, 40, rows)
    x[torch.arange(rows), tokens] = base + margin + torch.rand(rows, generator=g)
    x = x.to(kind[1])
    got = check_rows(kind, x, tokens, 4)
    assert (got["lp"] <= 0).all() and (got["top"] <= 0).all()

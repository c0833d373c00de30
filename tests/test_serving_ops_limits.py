"""The operators around a serving step at the ends of their ranges: masks of any size, logits far from zero, confident rows, lengths that fit no batch,
sizes next to 32 bits, buffers on odd addresses, and the paths of the decoder that use them on a GPU."""
import ctypes
import math

import pytest
import torch

import onnxruntime_b200 as ort
import serving_oracle as oracle
from onnxruntime_b200 import onnx_lite as ol
from onnxruntime_b200.capi import EPFail, InvalidArgument
from onnxruntime_b200.ops import _kernels as kernels
from onnxruntime_b200.training.gradient_builder import build_gradient_graph
from test_serving_ops import FUSED, GPU, KINDS, ONNX, PROVIDERS, SCORE_KINDS, Call, PrefixCase, half_step, i32, score_call


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


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("outputs", [["lp"], ["", "h"], ["", "", "top"], ["", "", "", "", "lse"], ["lp", "h", "top", "index", "lse"]])
@pytest.mark.parametrize("base", [0.0, 30.0, -2000.0, 60000.0, 1e7, -1e30, -math.inf])
def test_gradient_graph_of_log_probs_far_from_zero(kind, outputs, base):
    """The probabilities that a gradient is made of do not depend on where the logits lie (``-inf`` stands for the type's lowest value)."""
    rows, V, k, dt = 6, 333, 3, kind[1]
    g = torch.Generator().manual_seed(1)
    base = torch.finfo(dt).min if base == -math.inf else base
    if abs(base) > torch.finfo(dt).max:
        pytest.skip("beyond the type")
    x, tokens = base + 2 * torch.randn(rows, V, generator=g), torch.tensor([1, 332, 0, 7, -1, 200])
    x[1] = base
    x[2, ::3] = torch.finfo(dt).min
    x[3] = torch.finfo(dt).min
    x[4, 1::2] = -math.inf
    x = x.clamp(min=torch.finfo(dt).min).to(dt) if base > -1e30 else x.double().clamp(min=torch.finfo(dt).min).to(dt)
    x[4, 1::2] = -math.inf
    weights = {n: torch.randn(rows, *([k] if n == "top" else []), generator=g) for n in ("lp", "h", "top", "lse")}
    T = ol.TensorProto
    nodes, parts = [ol.make_node("TokenLogProbs", ["x", "tokens"], outputs, domain=FUSED, top_k=k)], []
    for o in outputs:
        if o in weights:
            nodes += [ol.make_node("Mul", [o, "c_" + o], [o + "_c"]), ol.make_node("ReduceSum", [o + "_c"], [o + "_sum"], keepdims=0)]
            parts.append(o + "_sum")
    nodes.append(ol.make_node("Sum", parts, ["loss"]))
    info = ol.make_tensor_value_info
    used = [o for o in outputs if o in weights]
    graph = ol.make_graph(nodes, "g", [info("x", ONNX[dt], [rows, V]), info("tokens", T.INT64, [rows])] + [info("c_" + o, T.FLOAT, list(weights[o].shape)) for o in used],
                          [info("loss", T.FLOAT, [])])
    model = build_gradient_graph(ol.make_model(graph, opset=17, extra_opsets={FUSED: 1}), ["x"], "loss", recompute_fallback=False)
    sess = ort.InferenceSession(model.serialize(), providers=[kind[0]])
    dev = "cuda" if kind[0] == GPU else "cpu"
    binding, dx = sess.io_binding(), torch.full((rows, V), 7.0, dtype=dt, device=dev)
    for n, t in dict(x=x, tokens=tokens, **{"c_" + o: weights[o] for o in used}).items():
        binding.bind_torch_input(n, t.to(dev))
    binding.bind_torch_output("x_grad", dx)
    binding.bind_torch_output("loss", torch.zeros((), device=dev))
    sess.run_with_iobinding(binding)
    c = {n: w.double() if n in used else torch.zeros_like(w).double() for n, w in weights.items()}
    index = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :k]
    want = oracle.token_log_probs_grad(x.double(), tokens, c["lp"], c["h"], index, c["top"], c["lse"])
    _, h, _, logp, r, _ = exact_rows(x, tokens)
    # p carries r, and its exponent (formed from a difference, rounded three times) 2^-22 |log p|; its factor is a sum of the coefficients and, with the
    # entropy, of |log p| + h; the result is rounded once
    size = sum(w.abs().reshape(rows, -1).sum(1) for w in c.values())[:, None]
    p, far = logp.exp(), logp.clamp(min=-1e4).abs()
    off = (r[:, None] + 2.0 ** -22 * (1 + far)) * p * (size + c["h"].abs()[:, None] * (far + h[:, None]) * 2) + 2.0 ** -21 * p * size * (1 + far)
    bound = half_step(dt) * want.abs() + off + 2.0 ** -22 * size * (want.abs() > 0) + torch.finfo(dt).tiny
    got = dx.cpu().double()
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all(), "%g of the bound" % float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("kind", SCORE_KINDS)
def test_log_probs_gradient_of_an_excluded_token_by_a_large_factor(kind):
    """An impossible token has no part in the entropy, however large the entropy's gradient."""
    x = torch.tensor([[0.0, 1.0, -math.inf, 2.0]]).to(kind[1])
    got = score_call(kind[0], x, torch.tensor([3]), 0, dict(g_h=torch.tensor([1e9])))()["dx"]
    want = oracle.token_log_probs_grad(x.double(), torch.tensor([3]), torch.zeros(1), torch.tensor([1e9]), torch.zeros(1, 0), torch.zeros(1, 0), torch.zeros(1))
    assert got[0, 2] == 0
    if kind[1] != torch.float16:
        assert ((got.double() - want).abs() <= (half_step(kind[1]) + 2.0 ** -19) * 1e9).all()


@pytest.mark.parametrize("kind", SCORE_KINDS)
def test_log_probs_gradient_of_logits_as_far_apart_as_the_type_allows(kind):
    most = torch.finfo(kind[1]).max
    x = torch.tensor([[most, -most, 0.0, most], [-most, most, -math.inf, -most]]).to(kind[1])
    tokens, grads = torch.tensor([0, 1]), dict(g_lp=torch.tensor([1.0, 2.0]), g_h=torch.tensor([3.0, -1.0]))
    every = score_call(kind[0], x, tokens, 0, grads)()
    got = every["dx"]
    assert abs(float(every["h"][0]) - math.log(2)) < 1e-6 and every["h"][1] == 0
    assert torch.isfinite(got).all() and (got[:, 1:3] == 0).all()      # no possible token there, or the only one


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("V,k", [(40, 12), (1031, 32), (5000, 7)])
def test_log_probs_of_hard_rows_row_by_row(kind, V, k):
    """Ties, zeros of both signs, impossible tokens, one certain token, steep and flat rows, rows of extreme values: each row against a bound from its
    own differences, which a large logit of another row does not widen."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(14, V, generator=g)
    x[0] = 0.0
    x[1] = torch.randint(-2, 3, (V,), generator=g).float()
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    x[3, 1:] = -math.inf
    x[4, :-1] = -math.inf
    x[5, 5:] = -math.inf
    x[6] = torch.arange(V).float()
    x[7] = -torch.arange(V).float() - 1000
    x[8] = -torch.finfo(torch.float16).max
    x[9] = -torch.finfo(torch.float16).max
    x[9, 7] = torch.finfo(torch.float16).max
    x[10] = torch.where(torch.arange(V) % 3 == 0, -math.inf, 5.0)
    x[11] = torch.linspace(-1e-3, 1e-3, V)
    x[12] = torch.linspace(20, -20, V) ** 3
    tokens = torch.tensor([0, 1, V - 1, 0, V - 1, 3, V - 1, 0, 2, 7, 4, 5, 0, 6])
    check_rows(kind, x.to(kind[1]), tokens, k)


# ---------------------------------------------------------------------------------------------------- shared prefix attention
def unchanged(case, got):
    """What the caches held before the call, NaN among it, is there still."""
    return all(torch.equal(got[n].nan_to_num(77.0), c.nan_to_num(77.0)) for n, c in zip(("kc_out", "vc_out"), case.caches))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("first", [0, 2])
def test_prefix_without_sequences(kind, first):
    """Tokens that no sequence has, whatever the only cumulative length says: zeros, and no access to lengths or tables that are empty."""
    c = PrefixCase(kind[1], 4, 2, 64, 16, 20, [3], [3])
    c.lengths, c.cum, c.table = [], i32(first), torch.zeros(0, 4, dtype=torch.int32)
    got = c.call(kind[0])()
    assert (got["out"] == 0).all() and unchanged(c, got)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("placed", [False, True])
@pytest.mark.parametrize("H", [64, 24])
@pytest.mark.parametrize("first", [1, 2, 40])
def test_prefix_rows_in_front_of_the_first_sequence(kind, placed, H, first):
    """They are nobody's, like those behind the last one: zeros, and neither the cache nor the other rows feel them, whatever their slots say."""
    base, c = (PrefixCase(kind[1], 4, 2, H, 16, 70, [30, 5, 0], [1, 3, 12], placed=placed, seed=first, behind=2) for _ in range(2))
    lead = torch.full((first, 4 + 2 * 2, H), math.nan, dtype=kind[1])
    c.qkv, c.cum = torch.cat([lead, c.qkv]), c.cum + first
    # with slots of the first sequence's oldest tokens, and a position of no table
    c.pos = torch.cat([torch.arange(first) - 1, c.pos])
    c.slot = torch.cat([c.table[0, 0].long() * 16 + torch.arange(first) % 16, c.slot])
    got = c.call(kind[0])()
    assert (got["out"][:first] == 0).all()
    base.check(dict(got, out=got["out"][first:]))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", [dict(H=64), dict(H=24), dict(H=64, size=10)])
@pytest.mark.parametrize("cum,past", [([0, 4, 2], None), ([0, 2, 9], None), ([-1, 2, 5], None), ([0, 2, 5], [75, 190]), ([0, 2, 5], [75, -1])])
@pytest.mark.parametrize("placed", [False, True])
def test_prefix_lengths_that_fit_no_batch_or_table_are_an_error_in_every_form(kind, form, cum, past, placed):
    """Cumulative lengths that run backwards, beyond the tokens or below 0, and tokens beyond the table, with slots given and without."""
    c = PrefixCase(kind[1], 4, 2, form["H"], form.get("size", 16), 70, [5, 30], [2, 3], placed=placed)
    c.cum = i32(*cum)
    if past:
        c.lengths = [(p, 1) for p in past]
        assert max(past) > c.table.shape[1] * c.size - 3 or min(past) < 0
    with pytest.raises((InvalidArgument, EPFail)):
        c.call(kind[0])()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H,new", [(64, [1, 3]), (128, [1, 3]), (128, [40, 1]), (24, [1, 3])])
@pytest.mark.parametrize("shift", [1, 2, 4])
def test_prefix_buffers_on_odd_addresses(kind, H, new, shift):
    """Queries and the bound result start ``shift`` elements behind an aligned address."""
    c = PrefixCase(kind[1], 4, 2, H, 16, 70, [5, 30], new)
    call = c.call(kind[0])
    for n, bind in (("q", call.binding.bind_torch_input), ("out", call.binding.bind_torch_output)):
        t = (call.ins if n == "q" else call.outs)[n]
        moved = torch.empty(t.numel() + shift, dtype=t.dtype, device=t.device)[shift:].view(t.shape)
        moved.copy_(t)
        (call.ins if n == "q" else call.outs)[n] = moved
        bind(n, moved)
    c.check(call())


class PrefixArgs(ctypes.Structure):
    """ortb200_prefix_attn_args"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("qkv", "k", "v", "k_cache", "v_cache", "cu_seqlens", "past_seqlens", "block_table", "shared_prefix", "cos_cache", "sin_cache",
                                               "positions", "slot_mapping", "out", "workspace")] + [("workspace_bytes", ctypes.c_int64), ("T", ctypes.c_int64)] + [
        (n, ctypes.c_int) for n in ("B", "N", "Nk", "H", "block_size", "max_blocks", "num_blocks", "cos_rows", "rot_dim", "interleaved")] + [
        ("scale", ctypes.c_float), ("softcap", ctypes.c_float)] + [(n, ctypes.c_int) for n in ("dtype", "tensor_cores", "use_pdl")] + [("status", ctypes.c_void_p)]


def refused(name, args):
    """What a C entry answers to arguments that it has to refuse on the host: the addresses are none, so a call that were let through would fault."""
    if torch.cuda.is_available():
        pytest.skip("never launched with addresses that are none")
    return getattr(ctypes.CDLL(kernels.lib_path()), name)(ctypes.byref(args), None)


@pytest.mark.parametrize("field", ["out", "k_cache", "v_cache", "workspace"])
def test_prefix_c_entry_refuses_addresses_that_vectors_do_not_take(field):
    place = {n: 1 << 20 for n in ("qkv", "k_cache", "v_cache", "cu_seqlens", "past_seqlens", "block_table", "shared_prefix", "out", "workspace")}
    place[field] += 4
    assert refused("ortb200_prefix_attn", PrefixArgs(**place, workspace_bytes=1 << 40, T=2, B=1, N=2, Nk=1, H=64, block_size=16, max_blocks=4, num_blocks=9, dtype=1, tensor_cores=1)) == -3


# ------------------------------------------------------------------------------------------------------ sizes next to 32 bits
class LogProbsArgs(ctypes.Structure):
    """ortb200_token_log_probs_args"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "tokens", "log_prob", "entropy", "log_sum_exp", "top_log_probs", "top_tokens", "log_sum_exp_rest")] + [
        ("rows", ctypes.c_int64)] + [(n, ctypes.c_int) for n in ("vocab", "top_k", "dtype", "use_pdl")]


class LogProbsGradArgs(ctypes.Structure):
    """ortb200_token_log_probs_grad_args"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("logits", "tokens", "log_sum_exp", "entropy", "d_log_prob", "d_entropy", "top_tokens", "d_top_log_probs", "d_log_sum_exp",
                                               "log_sum_exp_rest", "d_logits")] + [("rows", ctypes.c_int64)] + [(n, ctypes.c_int) for n in ("vocab", "top_k", "dtype", "use_pdl")]


@pytest.mark.parametrize("name,args", [("ortb200_token_log_probs", LogProbsArgs), ("ortb200_token_log_probs_grad", LogProbsGradArgs)])
def test_log_probs_c_entry_refuses_vocabularies_next_to_32_bits(name, args):
    place = {n: 1 << 20 for n, t in args._fields_ if t is ctypes.c_void_p}
    assert refused(name, args(**place, rows=1, vocab=2 ** 31 - 1, top_k=0, dtype=1)) == -2


class LayoutArgs(ctypes.Structure):
    """ortb200_batch_layout_args"""
    _fields_ = [(n, ctypes.c_void_p) for n in ("past_seqlens", "new_tokens", "table_in", "free_blocks", "table_out", "cum", "positions", "slot_mapping", "blocks_used")] + [
        (n, ctypes.c_int) for n in ("B", "max_blocks", "block_size")] + [("num_free", ctypes.c_int64), ("rows", ctypes.c_int64), ("status", ctypes.c_void_p)]


def test_layout_c_entry_refuses_rows_next_to_32_bits():
    place = {n: 1 << 20 for n, t in LayoutArgs._fields_ if t is ctypes.c_void_p}
    assert refused("ortb200_batch_layout", LayoutArgs(**place, B=1, max_blocks=2 ** 31 - 1, block_size=1, num_free=2 ** 31 - 1, rows=2 ** 31 - 1)) == -2


@pytest.mark.parametrize("sizes", [dict(max_blocks=2 ** 23, block_size=256, N=2, Nk=1), dict(max_blocks=4, block_size=16, N=2 ** 25, Nk=1)])
@pytest.mark.parametrize("tensor_cores", [0, 1])
def test_prefix_c_entry_refuses_sizes_next_to_32_bits(sizes, tensor_cores):
    """A table for 2^31 tokens of a sequence, and a token of 2^31 elements."""
    place = {n: 1 << 20 for n in ("qkv", "k_cache", "v_cache", "cu_seqlens", "past_seqlens", "block_table", "shared_prefix", "out", "workspace")}
    assert refused("ortb200_prefix_attn", PrefixArgs(**place, workspace_bytes=1 << 60, T=2, B=1, H=64, num_blocks=9, dtype=1, tensor_cores=tensor_cores, **sizes)) == -2


# --------------------------------------------------------------------------------------------------------------- refused layouts
LAYOUT_REFUSALS = [([4, 9], [1, 4], 1, 5), ([4, 29], [1, 4], 9, 5), ([4, 9], [1, 4], 9, 4), ([4, -1], [1, 4], 9, 5)]   # blocks, table, rows, a negative length


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("past,new,free,rows", LAYOUT_REFUSALS)
def test_strict_layout_makes_a_refusal_an_error(provider, past, new, free, rows):
    table = torch.arange(16, dtype=torch.int32).reshape(2, 8)
    ins = dict(past=i32(*past), new=i32(*new), table=table, free=i32(*range(50, 50 + free)), rows=torch.zeros(rows, dtype=torch.int64))
    outs = dict(block_table=table, cum=i32(0, 0, 0), positions=torch.zeros(rows, dtype=torch.int64), slots=torch.zeros(rows, dtype=torch.int64), used=i32(7))
    call = Call(provider, [("PagedBatchLayout", list(ins), list(outs), dict(block_size=4, strict=1))], ins, outs)
    with pytest.raises((InvalidArgument, EPFail)):
        call()
    call.ins["past"].copy_(i32(4, 9))
    call.binding.bind_torch_input("new", i32(1, 1).to(call.ins["new"].device))
    assert call()["used"].tolist() == [1]            # 4 and 9 tokens in blocks of 4: the first one enters a block; the session goes on


@pytest.mark.parametrize("provider", PROVIDERS)
def test_a_decoder_step_whose_layout_is_refused_is_an_error(provider):
    """The shared-prefix form of the decoder with fewer blocks than its tokens need: not logits out of attention to nothing."""
    from test_shared_prefix_generation import decoders
    shared = decoders(provider, 16, 2, 64)[2]
    shared._granted = lambda seqs, new: []
    with pytest.raises((InvalidArgument, EPFail)):
        shared.step([(0, [1, 2, 3], [2]), (1, [4], [0])])
        shared.sess.check_device_status()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", [dict(), dict(H=24), dict(H=128, new=[40, 1]), dict(size=10), dict(size=128, H=128)])
@pytest.mark.parametrize("bad", [-1, 10 ** 6])
@pytest.mark.parametrize("placed", [False, True])
def test_prefix_blocks_outside_the_cache(kind, form, bad, placed):
    """Where a sequence has tokens they are an error, be it in the prefix or in its own keys; behind its end they may be anything."""
    size, H, new = form.get("size", 16), form.get("H", 64), form.get("new", [2, 3])
    make = lambda: PrefixCase(kind[1], 4, 2, H, size, 70, [5, 130], new, placed=placed)  # noqa: E731
    c = make()
    for b, (past, n) in enumerate(c.lengths):
        c.table[b, oracle.blocks_of(past + n, size):] = bad
    c.run(kind[0])
    for b, column in ((0, 0), (1, (70 + 129) // size)):
        c = make()
        c.table[b, column] = bad
        with pytest.raises((InvalidArgument, EPFail)):
            c.call(kind[0])()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [64, 24])
@pytest.mark.parametrize("slot", [-1, 10 ** 7])
def test_prefix_slots_outside_the_cache_are_an_error(kind, H, slot):
    c = PrefixCase(kind[1], 4, 2, H, 16, 70, [5, 30], [2, 3])
    c.slot[3] = slot
    with pytest.raises((InvalidArgument, EPFail)):
        c.call(kind[0])()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("H", [64, 24])
@pytest.mark.parametrize("position", [-1, 10 ** 7])
def test_prefix_positions_outside_the_rotary_tables_are_an_error(kind, H, position):
    c = PrefixCase(kind[1], 4, 2, H, 16, 70, [5, 30], [2, 3])
    c.pos[3] = position
    with pytest.raises((InvalidArgument, EPFail)):
        c.call(kind[0])()

"""The operators around a decode step with drafted tokens against draft_oracle.py: TreePagedAttention, PagedCacheMove and ProcessLogits, each on the
CPU provider and (marked gpu) on the GPU, with what they refuse."""
import ctypes
import math
import random

import pytest
import torch

import draft_oracle as oracle
import serving_oracle
from onnxruntime_b200.capi import EPFail, InvalidArgument
from onnxruntime_b200.ops import _kernels as kernels
from test_serving_ops import GPU, KINDS, PROVIDERS, Call, half_step, i32

i64 = lambda *v: torch.tensor(v, dtype=torch.int64)  # noqa: E731


def tree(nodes, seed, wide=0.5):
    """Parents of a tree with a bit of everything: chains, siblings, several roots."""
    r = random.Random(seed)
    return [-1] + [-1 if r.random() < 0.1 else i - 1 if r.random() > wide else r.randint(max(0, i - 9), i - 1) for i in range(1, nodes)] if nodes else []


# --------------------------------------------------------------------------------------------------------- attention of trees
class TreeCase:
    """A batch over its own caches: sequences of ``pasts`` tokens that bring the trees ``trees`` (parents by row)."""

    def __init__(self, dt, N, Nk, H, size, pasts, trees, rotary=1.0, interleaved=False, separate=False, cap=0.0, scale=0.0, behind=0, seed=0, spread=1.0, stale=math.nan):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: (spread * torch.randn(*s, generator=g)).to(dt)  # noqa: E731
        self.__dict__.update(locals())
        need = [serving_oracle.blocks_of(p + len(t), size) for p, t in zip(pasts, trees)]
        tokens = sum(len(t) for t in trees)
        order = torch.randperm(sum(need) + 2, generator=g).int()
        self.table = torch.full((len(pasts), max(need, default=0) + 1), int(order[-1]), dtype=torch.int32)   # entries behind the end name a stale block
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        self.caches = [torch.full((len(order), size, Nk, H), stale, dtype=dt) for _ in range(2)]   # what no sequence holds may be anything
        for c in self.caches:
            for b, past in enumerate(pasts):
                p = torch.arange(past)
                c[self.table[b].long()[p // size], p % size] = rand(past, Nk, H)
        self.qkv = rand(tokens + behind, N + 2 * Nk, H)
        self.qkv[tokens:] = math.nan
        r = int(H * rotary) // 2
        rows = max([p + len(t) for p, t in zip(pasts, trees)], default=1) or 1
        angle = torch.arange(rows).double()[:, None] * 100.0 ** (-torch.arange(r).double() / max(r, 1))
        self.cos, self.sin = angle.cos().to(dt), angle.sin().to(dt)
        self.parents = i32(*[p for t in trees for p in t], *[-1] * behind)
        self.pos = torch.tensor([p + d for p, t in zip(pasts, trees) for d in oracle.depths(t)], dtype=torch.int64)
        spots = [(b, p + i) for b, (p, t) in enumerate(zip(pasts, trees)) for i in range(len(t))]
        self.slot = torch.tensor([int(self.table[b, p // size]) * size + p % size for b, p in spots], dtype=torch.int64)
        self.cum = torch.tensor([0] + [len(t) for t in trees]).cumsum(0).int()

    def call(self, provider, graph=False):
        n, k, tokens = self.N, self.Nk, len(self.qkv)
        flat = lambda t: t.flatten(1).contiguous()  # noqa: E731
        ins = dict(q=flat(self.qkv[:, :n]), k=flat(self.qkv[:, n:n + k]), v=flat(self.qkv[:, n + k:])) if self.separate else dict(q=flat(self.qkv))
        names = list(ins) + ([] if self.separate else ["", ""]) + ["kc", "vc", "cum", "past", "table", "parents"]
        ins.update(kc=self.caches[0].clone(), vc=self.caches[1].clone(), cum=self.cum, past=i32(*self.pasts), table=self.table, parents=self.parents)
        if self.rotary:
            names += ["cos", "sin"]
            ins.update(cos=self.cos, sin=self.sin)
        attrs = dict(num_heads=n, kv_num_heads=k, do_rotary=int(self.rotary > 0), rotary_interleaved=int(self.interleaved))
        if self.cap:
            attrs["softcap"] = self.cap
        if self.scale:
            attrs["scale"] = self.scale
        outs = dict(out=torch.full((tokens, n * self.H), 3.0, dtype=self.dt), kc_out=ins["kc"], vc_out=ins["vc"])
        return Call(provider, [("TreePagedAttention", names, list(outs), attrs)], ins, outs, graph)

    def check(self, got):
        tokens, u, n = len(self.slot), half_step(self.dt), self.N
        x = self.qkv[:tokens].double()
        turn = lambda t: serving_oracle.rotate(t, self.cos[self.pos].double(), self.sin[self.pos].double(), self.interleaved) if self.rotary else t  # noqa: E731
        for c, before, want in zip((got["kc_out"], got["vc_out"]), self.caches, (turn(x[:, n:n + self.Nk]), x[:, n + self.Nk:])):
            flat, old = c.reshape(-1, self.Nk, self.H), before.reshape(-1, self.Nk, self.H)
            # a rotated element is a rounded sum of two products, each at most as large as its pair
            assert ((flat[self.slot].double() - want).abs() <= u * want.abs() + 2.0 ** -22 * (x[:, n:].abs().amax() if tokens else 0)).all()
            rest = torch.ones(len(flat), dtype=torch.bool)
            rest[self.slot] = False
            assert torch.equal(flat[rest].nan_to_num(77.0), old[rest].nan_to_num(77.0))          # nothing else was touched
        scale = self.scale or self.H ** -0.5
        want, bound = oracle.tree_attention(turn(x[:, :n]), got["kc_out"], got["vc_out"], self.table, self.pasts, self.trees, self.size, scale, self.cap, u)
        out = got["out"].reshape(-1, n, self.H).double()
        off = (out[:tokens] - want).abs()
        assert torch.isfinite(out).all() and (off <= bound).all(), "%g of the bound" % float((off / bound).max())
        assert (out[tokens:] == 0).all()

    def run(self, provider):
        self.check(self.call(provider)())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past", [0, 1, 60, 63, 64, 65, 127, 130])
@pytest.mark.parametrize("nodes", [1, 2, 7, 33])
def test_tree_lengths(kind, past, nodes):
    """Tiles of 64 keys that hold old keys, old and new ones, and new ones alone."""
    TreeCase(kind[1], 4, 2, 64, 16, [past, past + 3], [tree(nodes, past), tree(nodes, past + 1)], seed=past).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nodes", [31, 32, 33, 63, 64, 65, 128, 200, 255, 256])
def test_tree_sizes(kind, nodes):
    """Words of a row's bits, several tiles of new keys, several tiles of rows; the largest tree."""
    TreeCase(kind[1], 2, 1, 64, 32, [70, 5], [tree(nodes, nodes), tree(nodes // 2, 1)], seed=nodes).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parents", [[-1, -1, -1, -1], [-1, 0, 1, 2, 3, 4, 5, 6, 7, 8], [-1] + [0] * 20, [-1, 0, 0, 1, 1, 2, 2, 3, 3, 4, 4], list(range(-1, 255))],
                         ids=["roots", "chain", "star", "binary", "deep"])
def test_tree_shapes(kind, parents):
    TreeCase(kind[1], 4, 1, 64, 16, [50, 0], [parents, parents[:3]], seed=len(parents)).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,Nk,H", [(1, 1, 64), (2, 2, 128), (6, 2, 64), (7, 1, 128), (16, 1, 64), (8, 2, 128), (4, 2, 24), (2, 1, 256), (5, 5, 40)])
def test_tree_head_layouts(kind, N, Nk, H):
    TreeCase(kind[1], N, Nk, H, 32, [103, 29, 70], [tree(1, 0), tree(6, 1), tree(19, 2)], seed=N).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [8, 16, 32, 64, 128, 192, 10])
def test_tree_block_sizes(kind, size):
    TreeCase(kind[1], 4, 2, 128, size, [81, 250], [tree(9, 3), tree(40, 4)], seed=size).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nodes", [[1], [0, 1, 0], [33, 1, 0, 64, 31], [150], [129, 1], [2] * 40, [0], [300, 5, 257]])
def test_tree_batches(kind, nodes):
    """Sequences without tokens between others, single tokens beside trees, and prompts of more rows than a tree has."""
    trees = [tree(n, i) if n <= 256 else list(range(-1, n - 1)) for i, n in enumerate(nodes)]
    TreeCase(kind[1], 4, 1, 64, 16, [90 + (37 * i) % 90 for i in range(len(nodes))], trees, seed=len(nodes)).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", [dict(rotary=0.0), dict(rotary=0.5), dict(interleaved=True), dict(separate=True), dict(cap=5.0), dict(cap=100.0), dict(scale=0.3), dict(behind=5),
                                  dict(behind=130), dict(rotary=0.25, interleaved=True, separate=True, cap=2.0)])
def test_tree_forms(kind, form):
    TreeCase(kind[1], 4, 2, 64, 32, [90, 80, 120], [tree(1, 0), tree(3, 1), tree(20, 2)], seed=3, **form).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
def test_tree_large_scores(kind):
    """Scores far apart: the running maximum moves between tiles, most weights vanish, also where the largest scores are hidden ones."""
    TreeCase(kind[1], 2, 1, 64, 16, [300, 3], [tree(20, 1), tree(70, 2)], spread=2.0, seed=5).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
def test_tree_chain_is_causal(kind):
    """A chain has the results of SharedPrefixPagedAttention without a prefix, to the bit where the same kernel computes both."""
    from test_serving_ops import PrefixCase
    a = PrefixCase(kind[1], 8, 2, 64, 16, 0, [130, 7], [5, 3], placed=False)
    b = TreeCase(kind[1], 8, 2, 64, 16, [130, 7], [list(range(-1, 4)), list(range(-1, 2))])
    b.table, b.caches, b.qkv, b.cos, b.sin = a.table, a.caches, a.qkv, a.cos, a.sin
    assert torch.equal(a.call(kind[0])()["out"], b.call(kind[0])()["out"])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Nk,H,past,nodes", [(32, 8, 128, 2000, [8] * 9), (64, 8, 128, 1330, [64, 50, 1]), (16, 16, 64, 4100, [5] * 20), (28, 4, 128, 700, [60, 1, 90, 17])])
def test_tree_sizes_of_models(dt, N, Nk, H, past, nodes):
    TreeCase(dt, N, Nk, H, 64, [past - (40 * i) % 311 for i in range(len(nodes))], [tree(n, i) for i, n in enumerate(nodes)], seed=1, stale=0.0).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Nk,H,size", [(8, 2, 64, 16), (8, 2, 128, 64), (4, 4, 128, 8)])
def test_tree_units_of_few_and_of_many_rows(dt, N, Nk, H, size):
    nodes = [(1, 2, 3, 40, 1, 0, 2, 8, 9)[i % 9] for i in range(130)]
    TreeCase(dt, N, Nk, H, size, [100 + (29 * i) % 83 for i in range(130)], [tree(n, i) for i, n in enumerate(nodes)], seed=4).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", [0.0, 7.0, 90.0])
@pytest.mark.parametrize("N,Nk,H,size", [(16, 2, 64, 16), (16, 2, 128, 64), (64, 4, 128, 32), (128, 1, 64, 64)])
def test_tree_units_of_two_row_tiles(dt, cap, N, Nk, H, size):
    """Batches whose sequences bring many rows: units of up to 256 rows, with fewer, with one tile's and with very few rows between them."""
    nodes = [60, 1, 0, 33, 16, 17, 120, 2, 250, 31, 32, 5, 64, 1]
    TreeCase(dt, N, Nk, H, size, [(29 * i) % 183 + (900 if i == 3 else 0) for i in range(len(nodes))], [tree(n, i) for i, n in enumerate(nodes)], seed=4, cap=cap).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [[256], [300, 256], [128, 129, 127], [64] * 50, [200] * 9 + [1] * 9])
@pytest.mark.parametrize("N,Nk,H", [(8, 4, 128), (24, 3, 64)])
def test_tree_batches_of_many_rows(N, Nk, H, nodes):
    trees = [tree(n, i) if n <= 256 else list(range(-1, n - 1)) for i, n in enumerate(nodes)]
    TreeCase(torch.bfloat16, N, Nk, H, 64, [(211 * i) % 700 for i in range(len(nodes))], trees, seed=5).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Nk,H", [(24, 8, 64), (32, 8, 128), (32, 32, 64), (16, 1, 128)])
@pytest.mark.parametrize("long", [0, 6000])
def test_tree_units_of_one_and_of_several_ctas(dt, N, Nk, H, long):
    """Units of every size, most of which one CTA has; with a long sequence some are spread over many."""
    pasts = [(97 * i) % 400 + (long if i == 9 else 0) for i in range(45)]
    TreeCase(dt, N, Nk, H, 32, pasts, [tree((37 * i) % 61, i) for i in range(45)], seed=11, behind=3).run(GPU)


@pytest.mark.gpu
def test_tree_wide_units_of_many_sequences():
    """More units of two row tiles than a CTA keeps the running sums of."""
    TreeCase(torch.bfloat16, 64, 1, 128, 16, [i % 67 for i in range(300)], [tree(4 + (i % 5 == 0), i) for i in range(300)], seed=8).run(GPU)


@pytest.mark.parametrize("kind", KINDS)
def test_tree_tokens_without_a_sequence(kind):
    """Rows that belong to no sequence: nothing is cached, and their results are 0."""
    case = TreeCase(kind[1], 4, 2, 64, 16, [], [], behind=5)
    case.table = torch.zeros(0, 3, dtype=torch.int32)
    got = case.call(kind[0])()
    assert (got["out"] == 0).all() and torch.equal(got["kc_out"].nan_to_num(7.0), case.caches[0].nan_to_num(7.0))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("past,nodes", [(0, 3), (70, 9), (130, 40)])
def test_tree_hidden_scores_of_any_size(kind, past, nodes):
    """What a row does not see has no say, however large its scores are: keys of infinities, NaN and the type's largest numbers in siblings."""
    trees = [[-1] + [0] * (nodes - 1)]
    case = TreeCase(kind[1], 4, 2, 64, 16, [past], trees, rotary=0.0, seed=nodes)
    want = case.call(kind[0])()["out"]
    for i, v in ((1, math.inf), (2, math.nan)) if nodes < 9 else ((1, math.inf), (2, math.nan), (5, torch.finfo(kind[1]).max), (8, -math.inf)):
        case.qkv[i, 4:6] = v
    got = case.call(kind[0])()["out"]
    rows = [0] + [i for i in range(3, nodes) if i not in (5, 8)]
    assert torch.equal(got[rows], want[rows])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,H,past,nodes", [(4, 64, 0, 3), (4, 64, 57, 7), (4, 128, 130, 40), (16, 128, 100, 100), (2, 128, 70, 300), (2, 40, 20, 9)])
def test_tree_hidden_values_of_any_size(kind, N, H, past, nodes):
    """A drafted token whose values overflow spoils the rows that see it, and no others: to the bit, these are what they are without it."""
    parents = [-1] + [(i - 1) // 2 if nodes <= 256 else i - 1 for i in range(1, nodes)]
    other = tree(6, 3)
    case = TreeCase(kind[1], N, 2, H, 16, [past, 33], [parents, other], seed=nodes)
    bad = {1: math.inf, 2: math.nan} if nodes < 40 else {5: -math.inf, nodes // 2: math.nan, nodes - 1: math.inf}
    # what is not finite counts as 0 for all others
    for i in bad:
        case.qkv[i, -2:, ::3] = 0.0
    whole = [case.qkv[i, -2:].clone() for i in bad]
    for i in bad:
        case.qkv[i, -2:] = 0.0
    want = case.call(kind[0])()["out"]
    for (i, v), row in zip(bad.items(), whole):
        case.qkv[i, -2:] = row
        case.qkv[i, -2:, 1::3] = v
    got = case.call(kind[0])()["out"]
    sees = oracle.sees(parents) if nodes <= 256 else torch.ones(nodes, nodes, dtype=torch.bool).tril()
    spoilt = sees[:, list(bad)].any(1)
    assert torch.equal(got[:nodes][~spoilt], want[:nodes][~spoilt]) and torch.equal(got[nodes:], want[nodes:])
    assert not got[:nodes][spoilt].isfinite().all(1).any()


@pytest.mark.gpu
def test_tree_many_sequences_and_long_prompts():
    """More row tiles than a CTA keeps the running sums of, trees and a prompt among them."""
    trees = [tree((1, 9, 0, 2)[i % 4], i) for i in range(900)] + [list(range(-1, 699))]
    TreeCase(torch.bfloat16, 16, 1, 64, 16, [i % 9 for i in range(901)], trees, seed=7).run(GPU)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("parents", [[-1, 1, 0], [-1, 2, 0], [-2, 0, 1], [0, 0, 1]])
def test_tree_parents_that_are_none(kind, parents):
    case = TreeCase(kind[1], 4, 2, 64, 16, [20, 40], [[-1, 0], [-1, 0, 1]])
    case.parents = i32(-1, 0, *parents)
    with pytest.raises((InvalidArgument, EPFail)):
        case.call(kind[0])()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_beyond_its_size(kind):
    """257 rows that are no chain are no prompt and too many for a tree."""
    case = TreeCase(kind[1], 2, 2, 64, 64, [20], [list(range(-1, 256))])
    case.parents[200] = 100
    with pytest.raises((InvalidArgument, EPFail)):
        case.call(kind[0])()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("change", [dict(past=i32(20, 5000)), dict(past=i32(-3, 40)), dict(cum=i32(0, 2, 90)), dict(table="outside")])
def test_tree_lengths_and_tables_that_fit_nothing(kind, change):
    case = TreeCase(kind[1], 4, 2, 64, 16, [20, 40], [[-1, 0], [-1, 0, 0]])
    call = case.call(kind[0])
    if change.get("table") == "outside":
        call.ins["table"][1, 0] = 1 << 20
    else:
        for n, t in change.items():
            call.ins[n].copy_(t)
    with pytest.raises((InvalidArgument, EPFail)):
        call()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,Nk", [(4, 2), (64, 2)])
def test_tree_lengths_that_run_backwards(kind, N, Nk):
    call = TreeCase(kind[1], N, Nk, 64, 16, [20, 40, 70], [[-1, 0], [-1, 0, 0], [-1, 0, 1, 1]]).call(kind[0])
    call.ins["cum"].copy_(i32(0, 6, 2, 9))
    with pytest.raises((InvalidArgument, EPFail)):
        call()


@pytest.mark.parametrize("kind", KINDS)
def test_tree_refusals(kind):
    def build(**change):
        case = TreeCase(kind[1], 4, 2, 64, 16, [20, 40], [[-1, 0], [-1, 0, 0]])
        for n, v in change.items():
            setattr(case, n, v)
        return case.call(kind[0])
    for change in (dict(parents=i32(-1, 0)), dict(parents=i64(-1, 0, -1, 0, 0)), dict(cum=i32(0, 2)), dict(table=torch.zeros(3, 4, dtype=torch.int32)), dict(cap=-1.0),
                   dict(cap=math.inf), dict(scale=-0.5), dict(cos=torch.zeros(60, 40, dtype=kind[1]), sin=torch.zeros(60, 40, dtype=kind[1])),
                   dict(caches=[torch.zeros(9, 16, 2, 64, dtype=torch.float64)] * 2)):
        with pytest.raises(InvalidArgument):
            build(**change)()


@pytest.mark.gpu
def test_tree_in_captured_graphs():
    """Replays follow the trees and lengths in the bound buffers; two graphs of two sessions, replayed by turns, share no workspace."""
    trees = [tree(6, 1), tree(9, 2)]
    cases = [TreeCase(torch.bfloat16, 8, 2, 128, 64, [200, 77], trees, seed=s) for s in (1, 2)]
    calls = [c.call(GPU, graph=True) for c in cases]
    for _ in range(3):
        for case, call in zip(cases, calls):
            case.check(call())
    other = [tree(9, 5), tree(6, 6)]
    for seed, call in zip((1, 2), calls):
        case = TreeCase(torch.bfloat16, 8, 2, 128, 64, [200, 77], other, seed=seed, behind=0)
        case.table = case.table[:, :calls[0].ins["table"].shape[1]]
        call.ins["kc"].copy_(case.caches[0])
        call.ins["vc"].copy_(case.caches[1])
        for n, t in (("q", case.qkv.reshape(15, -1)), ("cum", case.cum), ("parents", case.parents), ("table", case.table)):
            call.ins[n].copy_(t)
        call.sess.run_with_iobinding(call.binding)
    torch.cuda.synchronize()
    for seed, call in zip((1, 2), calls):
        case = TreeCase(torch.bfloat16, 8, 2, 128, 64, [200, 77], other, seed=seed)
        case.check({n: t.cpu() for n, t in call.outs.items()})
        assert call.sess.num_captured_graphs() == 1


@pytest.mark.gpu
def test_tree_on_another_stream():
    case = TreeCase(torch.float16, 8, 2, 64, 16, [90, 33], [tree(9, 1), tree(4, 2)])
    call = case.call(GPU)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call.sess.run_with_iobinding(call.binding)
    stream.synchronize()
    case.check({n: t.cpu() for n, t in call.outs.items()})


# ----------------------------------------------------------------------------------------------------------------- cache moves
def move_call(provider, sources, targets, caches, blocks=False, graph=False, keep=False):
    ins = dict(s=i64(*sources), t=i64(*targets), **{"c%d" % i: c for i, c in enumerate(caches)})
    outs = {"c%d_out" % i: c for i, c in enumerate(caches)}
    return Call(provider, [("PagedCacheMove", list(ins), list(outs), dict(whole_blocks=int(blocks)))], ins, outs, graph)


def moved(caches, sources, targets, blocks):
    want = []
    for c in caches:
        before, after = (t if blocks else t.flatten(0, 1) for t in (c, c.clone()))
        for s, t in zip(sources, targets):
            if t >= 0:
                after[t] = before[s]
        want.append(after.reshape(c.shape))
    return want


def some_caches(num, blocks=9, size=16, inner=(2, 24), dt=torch.float16, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(blocks, size, *inner, generator=g).to(dt) for _ in range(num)]


def check_move(provider, sources, targets, caches, blocks=False):
    got = move_call(provider, sources, targets, [c.clone() for c in caches], blocks)()
    for i, want in enumerate(moved(caches, sources, targets, blocks)):
        assert torch.equal(got["c%d_out" % i], want)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("sources,targets", [([], []), ([3], [3]), ([5], [7]), ([2, 3], [1, 2]), ([0, 1], [1, 0]), ([1, 2, 3, 0], [0, 1, 2, 3]), ([4, 4, 4], [0, 1, 4]),
                                             ([9, 0, 77], [-1, 5, -3]), ([-5], [-1])],
                         ids=["none", "itself", "one", "close_up", "swap", "cycle", "spread", "padding", "padding_alone"])
@pytest.mark.parametrize("blocks", [False, True])
def test_move_orders(provider, sources, targets, blocks):
    """Every source is read before any target is written."""
    sources = [min(s, 8) for s in sources] if blocks else sources
    check_move(provider, sources, targets, some_caches(3), blocks)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("moves", [1, 31, 32, 33, 300, 749, 750, 751, 2999, 3000, 3001, 4000])
def test_move_numbers(provider, moves):
    """Permutations with cycles of all lengths, up to what one pass of the kernel holds and beyond."""
    caches = some_caches(2, blocks=260, inner=(1, 40))
    r = random.Random(moves)
    places = r.sample(range(260 * 16), moves)
    check_move(provider, places, r.sample(places, moves), caches)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("inner,dt", [((8, 128), torch.bfloat16), ((1, 1), torch.uint8), ((3, 5), torch.uint8), ((7,), torch.float16), ((1, 3), torch.float32), ((), torch.float32),
                                      ((576,), torch.float16), ((2, 2, 9), torch.int8), ((1, 2), torch.float64)], ids=str)
@pytest.mark.parametrize("blocks", [False, True])
def test_move_entries(provider, inner, dt, blocks):
    """Entries of any size and type: vectors of 16, 4, 2 and 1 bytes, ranges that end inside an entry."""
    from test_serving_ops import ONNX
    ONNX.setdefault(torch.uint8, 2)
    ONNX.setdefault(torch.int8, 3)
    g = torch.Generator().manual_seed(1)
    caches = [torch.randint(-100, 100, (7, 10, *inner), generator=g).to(dt) for _ in range(2)]
    check_move(provider, [0, 1, 6, 5], [1, 0, 5, 2], caches, blocks)


@pytest.mark.parametrize("provider", PROVIDERS)
def test_move_caches_of_different_entries(provider):
    """Keys wider than values, a cache without elements, more caches than one launch takes."""
    caches = some_caches(70, inner=(2, 24)) + some_caches(70, inner=(1, 16), dt=torch.float32, seed=1) + some_caches(1, inner=(0, 4))
    check_move(provider, [20, 3, 21], [3, 20, 100], caches)


@pytest.mark.parametrize("provider", PROVIDERS)
def test_move_caches_that_are_not_dense(provider):
    """Views of one tensor that holds keys and values side by side."""
    both = some_caches(1, inner=(2, 2, 8))[0]
    before = [both[:, :, i].clone() for i in range(2)]
    dev = "cuda" if provider == GPU else "cpu"
    placed = both.to(dev)
    import onnxruntime_b200 as ort
    from onnxruntime_b200 import onnx_lite as ol
    names = ["s", "t", "k", "v"]
    info = lambda n, t, d: ol.make_tensor_value_info(n, t, ["%s%d" % (n, i) for i in range(d)])  # noqa: E731
    T = ol.TensorProto
    graph = ol.make_graph([ol.make_node("PagedCacheMove", names, ["ko", "vo"], domain="com.ortb200")], "g",
                          [info("s", T.INT64, 1), info("t", T.INT64, 1), info("k", T.FLOAT16, 4), info("v", T.FLOAT16, 4)], [info("ko", T.FLOAT16, 4), info("vo", T.FLOAT16, 4)])
    sess = ort.InferenceSession(ol.make_model(graph, opset=17, extra_opsets={"com.ortb200": 1}).serialize(), providers=[provider])
    binding = sess.io_binding()
    out = [torch.zeros_like(before[0], device=dev) for _ in range(2)]
    for n, t in (("s", i64(4, 2).to(dev)), ("t", i64(2, 9).to(dev)), ("k", placed[:, :, 0]), ("v", placed[:, :, 1])):
        binding.bind_torch_input(n, t)
    for n, t in zip(("ko", "vo"), out):
        binding.bind_torch_output(n, t)
    sess.run_with_iobinding(binding)
    for got, want in zip(out, moved(before, [4, 2], [2, 9], False)):
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("sources,targets", [([0], [9 * 16]), ([9 * 16], [0]), ([-1], [0]), ([1 << 40], [0]), ([0, 1], [5, 5]), ([0, 1, 2, 3], [6, 5, 7, 6])])
def test_move_places_that_are_none(provider, sources, targets):
    """Reported; what lies outside the cache is neither read nor written, and the other moves take place on the GPU."""
    with pytest.raises((InvalidArgument, EPFail)):
        move_call(provider, sources, targets, some_caches(3))()


@pytest.mark.parametrize("provider", PROVIDERS)
def test_move_in_a_cache_of_nothing(provider):
    """Caches without a block have no place that a move could name."""
    move_call(provider, [], [], some_caches(2, blocks=0))()
    move_call(provider, [3], [-1], some_caches(2, blocks=0))()
    with pytest.raises((InvalidArgument, EPFail)):
        move_call(provider, [0], [0], some_caches(2, blocks=0))()


@pytest.mark.parametrize("provider", PROVIDERS)
def test_move_refusals(provider):
    caches = some_caches(2)
    same = caches[0].to("cuda") if provider == GPU else caches[0]
    for call in (lambda: move_call(provider, [0, 1], [2], caches), lambda: move_call(provider, [0], [2], [caches[0], some_caches(1, blocks=8)[0]]),
                 lambda: move_call(provider, [0], [2], [caches[0], some_caches(1, size=8)[0]]), lambda: move_call(provider, [0], [2], [same, same]),
                 lambda: move_call(provider, [0], [2], [torch.zeros(4)])):
        with pytest.raises(InvalidArgument):
            call()()


@pytest.mark.gpu
def test_move_in_a_captured_graph():
    caches = some_caches(4)
    call = move_call(GPU, [1, 2, -1], [0, 1, -1], [c.clone() for c in caches], graph=True)
    want = caches
    for sources, targets in (([1, 2, -1], [0, 1, -1]), ([5, 100, 3], [3, 5, 100]), ([0, 0, 0], [-1, -1, -1])):
        call.ins["s"].copy_(i64(*sources))
        call.ins["t"].copy_(i64(*targets))
        got = call()
        want = moved(want, sources, targets, False)
        assert all(torch.equal(got["c%d_out" % i], w) for i, w in enumerate(want))
    assert call.sess.num_captured_graphs() == 1


@pytest.mark.gpu
def test_move_beyond_32_bit_offsets():
    """Entries behind 2^32 bytes of a cache."""
    cache = torch.zeros(70000, 256, 1, 128, dtype=torch.float16, device="cuda")
    units, g = 70000 * 256, torch.Generator().manual_seed(0)
    cache.view(units, 128)[-3:] = torch.randn(3, 128, generator=g).half().cuda()
    want = cache.view(units, 128)[-3:].clone()
    call = move_call(GPU, [units - 3, units - 1], [0, units - 2], [cache])
    call.sess.run_with_iobinding(call.binding)
    torch.cuda.synchronize()
    call.sess.check_device_status()
    flat = cache.view(units, 128)
    assert torch.equal(flat[0], want[0]) and torch.equal(flat[-2], want[2]) and torch.equal(flat[-1], want[2]) and torch.equal(flat[-3], want[0])


# -------------------------------------------------------------------------------------------------------------- process logits
LOGITS_KINDS = [pytest.param((p.values[0], d), marks=p.marks, id="%s-%s" % (p.id, n)) for p in PROVIDERS
                for n, d in (("fp32", torch.float32), ("bf16", torch.bfloat16), ("fp16", torch.float16))]
NAMES = ["logits", "history", "history_starts", "generated_starts", "row_list", "drafted", "repetition", "presence", "frequency", "bias_tokens", "bias_values", "bias_starts",
         "allowed", "row_mask", "temperature"]


class LogitsCase:
    """Rows of logits with everything that may be asked of them; ``without`` names what is left out."""

    def __init__(self, dt, rows, vocab, lists=None, length=40, drafted=0, biases=6, masks=3, without=(), seed=0, shift=0):
        r, g = random.Random(seed), torch.Generator().manual_seed(seed)
        self.dt, self.rows, self.vocab = dt, rows, vocab
        t = dict(logits=(4 * torch.randn(rows * vocab + shift, generator=g)).to(dt)[shift:].reshape(rows, vocab))
        self.lists = rows if lists is None else lists
        texts = [[r.randint(-1, vocab) if r.random() < 0.3 else r.randint(0, min(vocab, 9) - 1) for _ in range(r.choice([0, 1, length, r.randint(0, length)]))] for _ in range(self.lists)]
        starts = [0]
        for text in texts:
            starts.append(starts[-1] + len(text))
        t.update(history=i64(*[v for x in texts for v in x]), history_starts=i64(*starts))
        t.update(generated_starts=i64(*[starts[i] + r.randint(0, len(x)) for i, x in enumerate(texts)]))
        if lists is not None:
            t.update(row_list=i32(*[r.randint(-1, lists - 1) for _ in range(rows)]))
        if drafted:
            t.update(drafted=torch.tensor([[r.randint(-1, vocab - 1) for _ in range(drafted)] for _ in range(rows)], dtype=torch.int64).reshape(rows, drafted))
        uniform = lambda lo, hi: torch.tensor([r.choice([lo, r.uniform(lo, hi)]) for _ in range(rows)], dtype=torch.float32)  # noqa: E731
        t.update(repetition=uniform(1.0, 1.5), presence=uniform(0.0, 1.0), frequency=uniform(0.0, 0.5), temperature=uniform(1.0, 2.0))
        per = [r.randint(0, biases) for _ in range(rows)]
        t.update(bias_tokens=i64(*[r.choice([r.randint(-1, vocab), r.randint(0, min(vocab, 5) - 1)]) for n in per for _ in range(n)]),
                 bias_values=torch.randn(sum(per), generator=g), bias_starts=torch.tensor([0] + per).cumsum(0))
        if len(t["bias_values"]):
            t["bias_values"][::5] = -math.inf
        words = (vocab + 31) // 32
        t.update(allowed=torch.randint(-(1 << 31), 1 << 31, (masks, words), generator=g).int(), row_mask=i32(*[r.randint(-1, masks - 1) for _ in range(rows)]))
        self.t = {n: v for n, v in t.items() if n not in without}

    def call(self, provider, graph=False, place=None):
        dev = "cuda" if provider == GPU else "cpu"
        names = [n if n in self.t else "" for n in NAMES]
        while not names[-1]:
            names.pop()
        outs = dict(scores=torch.full((self.rows, self.vocab), 3.0))
        if place is not None:   # logits and scores on addresses that are no multiple of 16 bytes
            shifted = lambda t: torch.cat([t.reshape(-1)[:1].expand(place), t.reshape(-1)]).to(dev)[place:].view(t.shape)  # noqa: E731
            return Call(provider, [("ProcessLogits", names, ["scores"], {})], {**self.t, "logits": shifted(self.t["logits"])}, dict(scores=shifted(outs["scores"])), graph)
        return Call(provider, [("ProcessLogits", names, ["scores"], {})], {n: self.t[n] for n in names if n}, outs, graph)

    def want(self, row):
        t, of = self.t, lambda n, d: float(self.t[n][row]) if n in self.t else d  # noqa: E731
        text, counted = [], []
        if "history" in t:
            i = int(t["row_list"][row]) if "row_list" in t else row
            if i >= 0:
                lo, hi = int(t["history_starts"][i]), int(t["history_starts"][i + 1])
                text = t["history"][lo:hi].tolist()
                counted = t["history"][max(lo, int(t["generated_starts"][i])) if "generated_starts" in t else lo:hi].tolist()
        extra = t["drafted"][row].tolist() if "drafted" in t else []
        biases = []
        if "bias_tokens" in t:
            lo, hi = int(t["bias_starts"][row]), int(t["bias_starts"][row + 1])
            biases = list(zip(t["bias_tokens"][lo:hi].tolist(), t["bias_values"][lo:hi].tolist()))
        allowed = None
        if "allowed" in t and int(t["row_mask"][row]) >= 0:
            words = t["allowed"][int(t["row_mask"][row])].tolist()
            allowed = [v for v in range(self.vocab) if words[v // 32] >> (v % 32) & 1]
        return oracle.process_logits(t["logits"][row], text + extra, counted + extra, of("repetition", 1.0), of("presence", 0.0), of("frequency", 0.0), biases, allowed,
                                     of("temperature", 1.0))

    def check(self, got):
        for row in range(self.rows):
            want, bound = self.want(row)
            out = got["scores"][row].double()
            finite = want.isfinite()
            assert torch.equal(out[~finite].nan_to_num(5.0, 7.0, 9.0), want[~finite].nan_to_num(5.0, 7.0, 9.0))
            assert ((out - want)[finite].abs() <= bound[finite]).all(), row

    def run(self, provider, **how):
        self.check(self.call(provider, **how)())


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("vocab", [1, 2, 5, 7, 8, 9, 31, 32, 33, 64, 127, 1000, 4099, 32000])
def test_logits_vocabularies(kind, vocab):
    LogitsCase(kind[1], 5, vocab, seed=vocab).run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("without", [["history", "history_starts", "generated_starts"], ["generated_starts"], ["bias_tokens", "bias_values", "bias_starts"], ["allowed", "row_mask"],
                                     ["repetition"], ["presence"], ["frequency"], ["temperature"], ["repetition", "presence", "frequency"],
                                     [n for n in NAMES if n not in ("logits", "temperature")], [n for n in NAMES if n not in ("logits", "allowed", "row_mask")], NAMES[1:]], ids=str)
def test_logits_forms(kind, without):
    LogitsCase(kind[1], 4, 203, without=without, seed=len(without)).run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
def test_logits_rows_of_trees(kind):
    """Rows share the texts of their requests and have drafted tokens of their own."""
    LogitsCase(kind[1], 23, 301, lists=4, drafted=5).run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("rows", [0, 1, 2, 40, 200])
def test_logits_rows(kind, rows):
    LogitsCase(kind[1], rows, 77, seed=rows).run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
def test_logits_long_texts(kind):
    LogitsCase(kind[1], 3, 5003, length=9000, biases=700, seed=2).run(kind[0])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
def test_logits_that_are_no_numbers(kind):
    """Infinities and NaN, also in places that a mask takes out: masked is -inf whatever was there."""
    case = LogitsCase(kind[1], 6, 120, seed=4, without=["bias_tokens", "bias_values", "bias_starts"])
    x = case.t["logits"]
    x[:, ::7], x[:, 1::7], x[:, 2::7], x[:, 3::7] = math.inf, -math.inf, math.nan, torch.finfo(kind[1]).min
    case.t["repetition"].fill_(1.0)   # (what a penalty makes of the largest numbers leaves 32 bits)
    case.t["presence"].fill_(0.5)
    case.run(kind[0])


@pytest.mark.parametrize("provider", PROVIDERS)
def test_logits_neutral_values(provider):
    """A temperature that is not above 0 leaves a row; a row without penalties has no use for its text."""
    case = LogitsCase(torch.float32, 6, 50, without=["bias_tokens", "bias_values", "bias_starts", "allowed", "row_mask"])
    case.t["temperature"] = torch.tensor([0.0, -1.0, math.nan, 1.0, 0.5, 1.0])
    case.t["repetition"].fill_(1.0)
    case.t["presence"].fill_(0.0)
    case.t["frequency"].fill_(0.0)
    got = case.call(provider)()["scores"]
    x = case.t["logits"]
    assert torch.equal(got[[0, 1, 2, 3, 5]], x[[0, 1, 2, 3, 5]]) and torch.equal(got[4], x[4] / 0.5)


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("text,biases", [(2000, 0), (0, 2000), (1023, 300), (1500, 1500)])
def test_logits_touched_tokens_side_by_side(kind, text, biases):
    """More touched tokens of one part of the vocabulary than are listed, whether by texts that are short for the whole of it or by biases."""
    case = LogitsCase(kind[1], 3, 20000, without=["drafted", "row_list"], seed=text)
    case.t.update(history=torch.arange(3 * text) % max(text, 1) + 5, history_starts=torch.arange(4) * text, generated_starts=torch.arange(3) * text + text // 2,
                  bias_tokens=(torch.arange(3 * biases) * 2) % max(2 * biases, 1), bias_values=torch.linspace(-3, 3, 3 * biases), bias_starts=torch.arange(4) * biases,
                  repetition=torch.full((3,), 1.25))
    case.run(kind[0])


@pytest.mark.parametrize("provider", PROVIDERS)
def test_logits_quotients(provider):
    """Temperatures and penalties of any size: quotients are rounded once, also where they overflow, underflow or divide infinities."""
    g = torch.Generator().manual_seed(6)
    by = torch.cat([torch.rand(40, generator=g) * 3 + 0.01, 10.0 ** torch.linspace(-44, 38, 40), torch.tensor([2 - 2.0 ** -23, 1 + 2.0 ** -23, 3.0, torch.finfo(torch.float32).max, 2.0 ** -149])])
    x = torch.cat([torch.randn(3000, generator=g) * 10.0 ** (torch.rand(3000, generator=g) * 76 - 38), torch.tensor([0.0, -0.0, math.inf, -math.inf, math.nan, 2.0 ** -149, 3.4e38, -3.4e38])])
    case = LogitsCase(torch.float32, len(by), len(x), without=NAMES[1:])
    case.t.update(logits=x.expand(len(by), -1).contiguous(), temperature=by)
    for repeated in (False, True):
        if repeated:   # the same as penalties: only what is not below 0 is divided
            case.t.pop("temperature")
            case.t.update(history=torch.arange(len(x)), history_starts=i64(0, len(x)), row_list=torch.zeros(len(by), dtype=torch.int32), repetition=by)
        got, exact = case.call(provider)()["scores"].double(), x.double() / by.double().unsqueeze(1)
        if repeated:
            exact = torch.where(x < 0, x.double() * by.double().unsqueeze(1), exact)
        want = exact.float().double()
        same = (got == want) | (got.isnan() & want.isnan())
        # Half a unit in the last place of 32 bits (u = 2^-24 of the value), or of the smallest numbers.  A quotient q that is off by 1.5 u is mended with its
        # remainder x - q d, which is exact unless it falls below what 32 bits hold, 2^-149: that takes |x| < 2^-100 (the remainder is at most 1.5 u |x|, and its
        # last bit 2^-48 |x|).  There it is rounded to a multiple of 2^-149: to 0 while it is below 2^-150, which leaves 1.5 u, and otherwise
        # |x| > 2^-150 / (1.5 u), so that an error of 2^-150 is 1.5 u of x.  With the last rounding that is within 3 u for such numbers.
        units = torch.where(x.abs() < 2.0 ** -100, 3.0, 1.0).double()
        assert (same | ((got - exact).abs() <= torch.clamp(units * exact.abs() * 2.0 ** -24, min=2.0 ** -149))).all()


@pytest.mark.parametrize("provider", PROVIDERS)
def test_logits_biases_of_one_token_count_in_their_order(provider):
    case = LogitsCase(torch.float32, 2, 64, without=NAMES[1:9] + ["allowed", "row_mask", "temperature"])
    case.t.update(bias_tokens=i64(*[3, 9, 3, 3, 9], *[5] * 300), bias_values=torch.cat([torch.tensor([1e8, 2.0, 1.0, -1e8, 0.5]), torch.full((300,), 0.25)]), bias_starts=i64(0, 5, 305))
    got, x = case.call(provider)()["scores"], case.t["logits"]
    # 1e8 + 1 is 1e8 in 32 bits, so that nothing is left of the first token's
    assert float(got[0, 3]) == float(x[0, 3]) and float(got[0, 9]) == float(x[0, 9] + torch.tensor(2.5))
    assert float(got[1, 5]) == float(x[1, 5] + torch.tensor(75.0))
    rest = torch.ones(2, 64, dtype=torch.bool)
    rest[0, [3, 9]], rest[1, 5] = False, False
    assert torch.equal(got[rest], x[rest])


@pytest.mark.parametrize("kind", LOGITS_KINDS)
@pytest.mark.parametrize("change", [dict(row_list=i32(0, 4, 1)), dict(history_starts=i64(0, 5, 3, 9)), dict(history_starts=i64(0, 5, 9, 1 << 40)), dict(history_starts=i64(-4, 5, 9, 9)),
                                    dict(row_mask=i32(0, 3, -1)), dict(bias_starts=i64(0, 2, 1, 4)), dict(bias_starts=i64(0, 2, 3, 5000))])
def test_logits_places_that_are_none(kind, change):
    case = LogitsCase(kind[1], 3, 40, lists=3)
    case.t.update(history=i64(*range(9)), history_starts=i64(0, 5, 7, 9), generated_starts=i64(0, 5, 7), row_list=i32(0, 1, 2), bias_tokens=i64(1, 2, 3, 4), bias_values=torch.ones(4),
                  bias_starts=i64(0, 2, 3, 4), repetition=torch.full((3,), 1.2))
    case.t.update(change)
    with pytest.raises((InvalidArgument, EPFail)):
        case.call(kind[0])()


@pytest.mark.parametrize("provider", PROVIDERS)
def test_logits_refusals(provider):
    whole = LogitsCase(torch.float32, 4, 100, lists=2, drafted=2).t
    changes = [dict(repetition=torch.ones(3)), dict(presence=torch.ones(4, dtype=torch.float64)), dict(row_list=i64(0, 0, 0, 0)), dict(drafted=torch.zeros(3, 2, dtype=torch.int64)),
               dict(allowed=torch.zeros(3, 5, dtype=torch.int32)), dict(allowed=torch.zeros(3, 4, dtype=torch.int64)), dict(bias_starts=i64(0, 0)), dict(bias_values=torch.ones(99)),
               dict(generated_starts=i64(0)), dict(logits=torch.zeros(4, 100, dtype=torch.int32)), dict(logits=torch.zeros(4, 5, 20)), dict(history=None), dict(row_mask=None),
               dict(bias_values=None), dict(row_list=None)]
    for change in changes:
        case = LogitsCase(torch.float32, 4, 100, lists=2, drafted=2)
        case.t = {n: v for n, v in {**whole, **change}.items() if v is not None}
        with pytest.raises(InvalidArgument):
            case.call(provider)()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("vocab", [64, 203, 9001])
def test_logits_on_odd_addresses(dt, vocab):
    LogitsCase(dt, 5, vocab, seed=3).run(GPU, place=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rows,vocab", [(torch.bfloat16, 3, 128256), (torch.float32, 5, 50257), (torch.float16, 150, 32000), (torch.bfloat16, 2, 262144), (torch.float32, 1, 458752),
                                           (torch.float32, 1, 458753)])
def test_logits_sizes_of_models(dt, rows, vocab):
    """Up to what a cluster's counters hold, and one more."""
    LogitsCase(dt, rows, vocab, length=3000, biases=30, seed=1).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rows,vocab,how", [(torch.bfloat16, 132, 128256, dict(lists=9, drafted=5)), (torch.float32, 335, 50257, dict(length=200, biases=300)),
                                               (torch.float16, 525, 32003, dict(length=5500, lists=20)), (torch.bfloat16, 17000, 1000, dict(length=60)),
                                               (torch.float32, 335, 50257, dict(without=NAMES[1:9])), (torch.float16, 525, 32003, dict(length=300, place=1))])
def test_logits_of_large_batches(dt, rows, vocab, how):
    """What rows touch is gathered in front of the stream; some of the texts of 5500 tokens touch more than is gathered."""
    how = dict(how)
    place = how.pop("place", None)
    case = LogitsCase(dt, rows, vocab, seed=9, **{"biases": 12, **how})
    got = case.call(GPU, place=place)()
    rest = case.rows
    assert rest * vocab >= 1 << 24
    case.rows = min(rest, 100)                              # (the oracle takes its time)
    case.check(got)


@pytest.mark.gpu
def test_logits_in_captured_graphs():
    """Replays follow the texts and rules in the bound buffers."""
    first, second = (LogitsCase(torch.bfloat16, 6, 1000, lists=3, drafted=2, seed=s) for s in (1, 2))
    call = first.call(GPU, graph=True)
    first.check(call())
    for n in ("logits", "repetition", "presence", "frequency", "temperature", "row_list", "drafted", "row_mask", "allowed"):
        call.ins[n].copy_(second.t[n])
        first.t[n] = second.t[n]
    for _ in range(2):
        first.check(call())
    assert call.sess.num_captured_graphs() == 1


# ------------------------------------------------------------------------------------------------------------------ C interface
class MoveArgs(ctypes.Structure):
    """ortb200_cache_move_args"""
    _fields_ = [("caches", ctypes.c_void_p), ("unit_bytes", ctypes.c_void_p), ("num_caches", ctypes.c_int), ("units", ctypes.c_int64), ("sources", ctypes.c_void_p),
                ("targets", ctypes.c_void_p), ("moves", ctypes.c_int64), ("use_pdl", ctypes.c_int), ("status", ctypes.c_void_p)]


def test_c_interface_refuses_what_it_cannot_take():
    """Arguments that are missing or impossible end in an error code before anything is launched."""
    lib = ctypes.CDLL(kernels.lib_path())
    addresses, sizes = (ctypes.c_void_p * 1)(1 << 20), (ctypes.c_int64 * 1)(64)
    good = dict(caches=ctypes.addressof(addresses), unit_bytes=ctypes.addressof(sizes), num_caches=1, units=10, sources=1 << 20, targets=1 << 20, moves=4)
    for change, code in ((dict(moves=-1), -1), (dict(units=-1), -1), (dict(sources=None), -1), (dict(caches=None), -1), (dict(moves=1 << 20), -2), (dict(moves=0), 0)):
        assert lib.ortb200_cache_move(ctypes.byref(MoveArgs(**{**good, **change})), None) == code
    assert lib.ortb200_cache_move(None, None) == -1 and lib.ortb200_tree_attn(None, None) == -1 and lib.ortb200_process_logits(None, None) == -1
    size = lib.ortb200_tree_attn_workspace_bytes
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int64] + [ctypes.c_int] * 5
    assert size(8, 2, 4, 0, 64, 1) == -1 and size(8, 2, 4, 2, 64, 1) > 0 and size(0, 0, 4, 2, 64, 0) >= 0

"""The operators around one step of a serving batch against serving_oracle.py: PagedBatchLayout, SharedPrefixPagedAttention,
TokenLogProbs and its gradient, each on the CPU provider and (marked gpu) on the GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

import onnxruntime_b200 as ort
import serving_oracle as oracle
from onnxruntime_b200 import onnx_lite as ol
from onnxruntime_b200.capi import EPFail, InvalidArgument

CPU, GPU = "CPUExecutionProvider", "CUDAExecutionProvider"
PROVIDERS = [pytest.param(CPU, id="cpu"), pytest.param(GPU, marks=pytest.mark.gpu, id="gpu")]
FUSED = "com.ortb200"
T = ol.TensorProto
ONNX = {torch.float32: T.FLOAT, torch.float16: T.FLOAT16, torch.bfloat16: T.BFLOAT16, torch.float64: T.DOUBLE, torch.int32: T.INT32, torch.int64: T.INT64}
i32 = lambda *v: torch.tensor(v, dtype=torch.int32)  # noqa: E731


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Call:
    """A session over nodes [(op, inputs, outputs, attributes)] with named tensors bound; an output of an input's name with "_out" behind it
    is that input, updated in place."""

    def __init__(self, provider, nodes, ins, outs, graph=False):
        dev = "cuda" if provider == GPU else "cpu"
        self.ins = {n: t.to(dev) for n, t in ins.items()}
        self.outs = {n: self.ins[n[:-4]] if n.endswith("_out") and n[:-4] in ins else t.to(dev) for n, t in outs.items()}
        info = lambda n, t: ol.make_tensor_value_info(n, ONNX[t.dtype], ["d%s%d" % (n, i) for i in range(t.dim())])  # noqa: E731
        model = ol.make_graph([ol.make_node(op, i, o, name=op, domain=FUSED, **attrs) for op, i, o, attrs in nodes], "g",
                              [info(n, t) for n, t in self.ins.items()], [info(n, t) for n, t in self.outs.items()])
        options = {"enable_fallback": False} if provider == GPU else {}
        self.sess = ort.InferenceSession(ol.make_model(model, opset=17, extra_opsets={FUSED: 1}).serialize(),
                                         providers=[(GPU, {"enable_cuda_graph": "1" if graph else "0"}) if provider == GPU else CPU], **options)
        self.binding = self.sess.io_binding()
        for n, t in self.ins.items():
            self.binding.bind_torch_input(n, t)
        for n, t in self.outs.items():
            self.binding.bind_torch_output(n, t)
        self.provider = provider

    def __call__(self):
        self.sess.run_with_iobinding(self.binding)
        if self.provider == GPU:
            torch.cuda.synchronize()
            self.sess.check_device_status()
        return {n: t.cpu() for n, t in self.outs.items()}


# ------------------------------------------------------------------------------------------------------------- batch layout
LAYOUT_OUT = ["block_table", "cum", "positions", "slots", "used"]


def layout_call(provider, past, new, table, free, rows, size, in_place=False, graph=False):
    B = len(past)
    ins = dict(past=i32(*past), new=i32(*new), table=table, free=i32(*free), rows=torch.zeros(rows, dtype=torch.int64))
    outs = {("table_out" if in_place else "block_table"): table.clone(), "cum": torch.full((B + 1,), 7, dtype=torch.int32),
            "positions": torch.full((rows,), 7, dtype=torch.int64), "slots": torch.full((rows,), 7, dtype=torch.int64), "used": i32(7)}
    return Call(provider, [("PagedBatchLayout", list(ins), list(outs), dict(block_size=size))], ins, outs, graph)


def check_layout(provider, past, new, table, free, rows, size, in_place=False):
    want = oracle.batch_layout(past, new, table.tolist() if table.numel() else [[] for _ in past], free, rows, size)
    got = layout_call(provider, past, new, table, free, rows, size, in_place)()
    for (name, g), w in zip(got.items(), want):
        assert g.reshape(-1).tolist() == torch.tensor(w).reshape(-1).tolist(), name
    return want


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("size,past,new", [
    (16, [0], [1]), (16, [15], [1]), (16, [16], [1]), (16, [17], [0]), (4, [0, 3, 4, 5, 9], [4, 1, 0, 7, 13]), (1, [3, 0], [2, 5]), (7, [20, 6, 13], [1, 1, 1]),
    (256, [255, 256, 0, 1000], [1, 1, 700, 1]), (2, [0] * 9, [0] * 9)])
def test_layout(provider, in_place, size, past, new):
    g = torch.Generator().manual_seed(1)
    M = max(oracle.blocks_of(p + n, size) for p, n in zip(past, new)) + 3
    table = torch.randint(0, 99, (len(past), M), generator=g).int()
    check_layout(provider, past, new, table, list(range(500, 500 + 400)), sum(new) + 5, size, in_place)
    check_layout(provider, past, new, table, list(range(500, 500 + 400)), sum(new), size, in_place)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("B", [255, 256, 257, 1500])
def test_layout_of_many_requests(provider, B):
    g = torch.Generator().manual_seed(B)
    past, new = torch.randint(0, 40, (B,), generator=g).tolist(), torch.randint(0, 6, (B,), generator=g).tolist()
    table = torch.randint(0, 10000, (B, 13), generator=g).int()
    want = check_layout(provider, past, new, table, torch.randperm(9000, generator=g).tolist(), sum(new) + 300, 4)
    assert want[4] > B // 2


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("B", [6119, 6120, 6143, 6144, 16384])
def test_layout_around_48_kb_of_running_sums(provider, B):
    check_layout(provider, [i % 5 for i in range(B)], [(i + 1) % 2 for i in range(B)], torch.arange(3 * B, dtype=torch.int32).reshape(B, 3), list(range(7, 3 * B)), B, 2)


@pytest.mark.parametrize("provider", PROVIDERS)
def test_layout_of_more_requests_than_one_launch_takes(provider):
    B = 16400
    check_layout(provider, [i % 5 for i in range(B)], [(i + 1) % 2 for i in range(B)], torch.arange(3 * B, dtype=torch.int32).reshape(B, 3), list(range(7, 3 * B)), B, 2)


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("past,new,free,rows,code", [
    ([4, 9], [1, 4], 1, 5, -1),                 # two blocks wanted, one free
    ([4, 29], [1, 4], 9, 5, -2),                # the second request outgrows its eight blocks of four
    ([4, 9], [1, 4], 9, 4, -3), ([4, -1], [1, 4], 9, 5, -4), ([4, 9], [1, -4], 9, 5, -4), ([-5, 40], [9, 9], 0, 1, -4),
    ([0, 0], [2 ** 31 - 1, 2 ** 31 - 1], 9, 5, -3)])
def test_layout_refuses_a_batch_that_does_not_fit(provider, past, new, free, rows, code):
    table = torch.arange(16, dtype=torch.int32).reshape(2, 8)
    got = {n: t.tolist() for n, t in layout_call(provider, past, new, table, list(range(50, 50 + free)), rows, 4)().items()}
    assert got["used"] == [code] and got["cum"] == [0, 0, 0] and got["positions"] == [-1] * rows == got["slots"] and got["block_table"] == table.tolist()


@pytest.mark.parametrize("provider", PROVIDERS)
def test_layout_without_requests_rows_or_free_blocks(provider):
    got = layout_call(provider, [], [], torch.zeros(0, 4, dtype=torch.int32), [], 3, 16)()
    assert got["cum"].tolist() == [0] and got["positions"].tolist() == [-1] * 3 and got["used"].tolist() == [0]
    check_layout(provider, [5, 3], [0, 0], torch.arange(6, dtype=torch.int32).reshape(2, 3), [], 0, 4)
    check_layout(provider, [5, 3], [1, 1], torch.arange(6, dtype=torch.int32).reshape(2, 3), [], 2, 4)


@pytest.mark.parametrize("provider", PROVIDERS)
def test_layout_argument_checks(provider):
    table = torch.zeros(2, 8, dtype=torch.int32)
    bad = [dict(size=0), dict(new=[1]), dict(table=torch.zeros(3, 8, dtype=torch.int32)), dict(table=torch.zeros(2, 8, dtype=torch.int64))]
    for change in bad:
        with pytest.raises(InvalidArgument):
            layout_call(provider, **{**dict(past=[1, 2], new=[1, 1], table=table, free=[5], rows=2, size=4), **change})()


@pytest.mark.gpu
def test_layout_in_a_captured_graph():
    """Replays follow the lengths in the bound buffers; a table that is updated in place grows from replay to replay."""
    size, table = 4, torch.full((3, 8), -1, dtype=torch.int32)
    past, new = [0, 3, 4], [1, 1, 1]
    call = layout_call(GPU, past, new, table, [9, 8, 7], 3, size, in_place=True, graph=True)
    free = list(range(100, 103))
    call.ins["table"][1, 0], call.ins["table"][2, 0] = 50, 51
    want = call.ins["table"].tolist()
    for step in range(6):
        call.ins["free"].copy_(i32(*free))
        call.ins["past"].copy_(i32(*past))
        got = call()
        want, cum, pos, slot, used = oracle.batch_layout(past, new, want, free, 3, size)
        assert got["table_out"].tolist() == want and got["positions"].tolist() == pos and got["slots"].tolist() == slot and got["used"].tolist() == [used]
        past = [p + 1 for p in past]
        free = free[used:] + list(range(110 + 3 * step, 110 + 3 * step + used))
    assert call.sess.num_captured_graphs() == 1


# -------------------------------------------------------------------------------------------------- shared prefix attention
KINDS = [pytest.param((CPU, torch.float32), id="cpu-fp32")] + [
    pytest.param((GPU, d), marks=pytest.mark.gpu, id="gpu-" + n) for n, d in (("fp32", torch.float32), ("bf16", torch.bfloat16), ("fp16", torch.float16))]


class PrefixCase:
    """A batch over its own caches.  ``held``: tokens of every sequence behind the prefix before the call; ``new``: tokens it brings."""

    def __init__(self, dt, N, Nk, H, size, prefix, held, new, rotary=1.0, interleaved=False, separate=False, cap=0.0, scale=0.0, placed=True,
                 behind=0, seed=0, spread=1.0, promised=None, stale=math.nan):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: (spread * torch.randn(*s, generator=g)).to(dt)  # noqa: E731
        self.__dict__.update(locals())
        self.lengths = [(prefix + h, n) for h, n in zip(held, new)]
        tokens, B = sum(new), len(held)
        shared = prefix // size
        mine = [oracle.blocks_of(p + n, size) - shared for p, n in self.lengths]
        order = torch.randperm(shared + sum(mine) + 2, generator=g).int()
        self.table = torch.full((B, max([shared + m for m in mine], default=1) + 1), int(order[-1]), dtype=torch.int32)   # entries behind the end name a stale block
        self.table[:, :shared] = order[:shared]
        at = shared
        for b, m in enumerate(mine):
            self.table[b, shared:shared + m] = order[at:at + m]
            at += m
        self.caches = [torch.full((len(order), size, Nk, H), stale, dtype=dt) for _ in range(2)]   # what no sequence holds may be anything
        copies = [rand(prefix, Nk, H) for _ in range(2)]
        for c, whole in zip(self.caches, copies):
            for b, (past, n) in enumerate(self.lengths):
                for p in range(past):
                    blk = int(self.table[b, p // size])
                    c[blk, p % size] = whole[p] if p < prefix else rand(Nk, H)
        self.qkv = rand(tokens + behind, N + 2 * Nk, H)
        if behind:
            self.qkv[tokens:] = math.nan
        r = int(H * rotary) // 2
        rows = max([p + n for p, n in self.lengths], default=1)
        angle = torch.arange(rows).double()[:, None] * 100.0 ** (-torch.arange(r).double() / max(r, 1))
        self.cos, self.sin = angle.cos().to(dt), angle.sin().to(dt)
        self.pos = torch.cat([torch.arange(p, p + n) for p, n in self.lengths] + [torch.full((behind,), -1)]).long()
        seq = torch.cat([torch.full((n,), b) for b, n in enumerate(new)] + [torch.zeros(behind)]).long()
        self.slot = torch.where(self.pos < 0, -1, self.table[seq, self.pos.clamp_min(0) // size].long() * size + self.pos % size)
        self.cum = torch.tensor([0] + new).cumsum(0).int()

    def call(self, provider, graph=False):
        n, k, tokens = self.N, self.Nk, len(self.qkv)
        flat = lambda t: t.reshape(tokens, -1).contiguous()  # noqa: E731
        ins = dict(q=flat(self.qkv[:, :n]), k=flat(self.qkv[:, n:n + k]), v=flat(self.qkv[:, n + k:])) if self.separate else dict(q=flat(self.qkv))
        names = list(ins) + ([] if self.separate else ["", ""]) + ["kc", "vc", "cum", "past", "table", "prefix"]
        ins.update(kc=self.caches[0].clone(), vc=self.caches[1].clone(), cum=self.cum, past=i32(*[p for p, _ in self.lengths]), table=self.table,
                   prefix=i32(self.prefix if self.promised is None else self.promised))
        names += ["cos", "sin"] if self.rotary else ["", ""]
        if self.rotary:
            ins.update(cos=self.cos, sin=self.sin)
        if self.placed:
            names += ["pos", "slot"]
            ins.update(pos=self.pos, slot=self.slot)
        while not names[-1]:
            names.pop()
        attrs = dict(num_heads=n, kv_num_heads=k, do_rotary=int(self.rotary > 0), rotary_interleaved=int(self.interleaved))
        if self.cap:
            attrs["softcap"] = self.cap
        if self.scale:
            attrs["scale"] = self.scale
        outs = dict(out=torch.full((tokens, n * self.H), 3.0, dtype=self.dt), kc_out=ins["kc"], vc_out=ins["vc"])
        return Call(provider, [("SharedPrefixPagedAttention", names, list(outs), attrs)], ins, outs, graph)

    def check(self, got):
        tokens, u, n = sum(self.new), half_step(self.dt), self.N
        x = self.qkv[:tokens].double()
        turn = lambda t: oracle.rotate(t, self.cos[self.pos[:tokens]].double(), self.sin[self.pos[:tokens]].double(), self.interleaved) if self.rotary else t  # noqa: E731
        slot = self.slot[:tokens]
        for c, before, want in zip((got["kc_out"], got["vc_out"]), self.caches, (turn(x[:, n:n + self.Nk]), x[:, n + self.Nk:])):
            flat, old = c.reshape(-1, self.Nk, self.H), before.reshape(-1, self.Nk, self.H)
            # a rotated element is a rounded sum of two products, each at most as large as its pair
            assert ((flat[slot].double() - want).abs() <= u * want.abs() + 2.0 ** -22 * x[:, n:].abs().amax()).all()
            rest = torch.ones(len(flat), dtype=torch.bool)
            rest[slot] = False
            assert torch.equal(flat[rest].nan_to_num(77.0), old[rest].nan_to_num(77.0))          # nothing else was touched
        scale = self.scale or self.H ** -0.5
        want, bound = oracle.paged_attention(turn(x[:, :n]), got["kc_out"], got["vc_out"], self.table, self.lengths, self.size, scale, self.cap, u)
        out = got["out"].reshape(-1, n, self.H).double()
        off = (out[:tokens] - want).abs()
        assert torch.isfinite(out).all() and (off <= bound).all(), "%g of the bound" % float((off / bound).max())
        assert (out[tokens:] == 0).all()

    def run(self, provider):
        self.check(self.call(provider)())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 130, 192])
@pytest.mark.parametrize("size", [16, 64])
def test_prefix_lengths(kind, prefix, size):
    PrefixCase(kind[1], 4, 2, 64, size, prefix, [0, 5, 64, 130], [1, 1, 1, 1], seed=prefix).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("N,Nk,H", [(1, 1, 64), (2, 2, 128), (6, 2, 64), (7, 1, 128), (16, 1, 64), (8, 2, 128), (4, 2, 24), (2, 1, 256), (5, 5, 40)])
def test_prefix_head_layouts(kind, N, Nk, H):
    PrefixCase(kind[1], N, Nk, H, 32, 100, [3, 29, 70], [1, 4, 2], seed=N).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", [8, 16, 32, 64, 128, 192, 10])
def test_prefix_block_sizes(kind, size):
    PrefixCase(kind[1], 4, 2, 128, size, 70, [11, 250], [2, 1], seed=size).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [[1], [0, 1, 0], [33, 1, 0, 64, 31], [150], [129, 1], [2] * 40])
def test_prefix_new_tokens(kind, new):
    """Rows of one tile and of several, sequences without tokens, single rows between long ones."""
    held = [(37 * i) % 90 for i in range(len(new))]
    PrefixCase(kind[1], 4, 1, 64, 16, 90, held, new, seed=len(new)).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("form", [dict(rotary=0.0), dict(rotary=0.5), dict(interleaved=True), dict(separate=True), dict(cap=5.0), dict(scale=0.3), dict(placed=False),
                                  dict(placed=False, behind=5), dict(behind=130), dict(rotary=0.25, interleaved=True, separate=True, cap=2.0)])
def test_prefix_forms(kind, form):
    PrefixCase(kind[1], 4, 2, 64, 32, 80, [10, 0, 40], [1, 3, 2], seed=3, **form).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("promised", [0, 10, 100, 127, 5000, -3])
def test_prefix_promise_is_cut_to_the_shortest_past(kind, promised):
    """128 tokens are shared.  Less may be promised; more is cut: the first sequence holds no more than the prefix."""
    PrefixCase(kind[1], 4, 2, 64, 64, 128, [0, 77], [2, 1], promised=promised).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_large_scores(kind):
    """Scores far apart: the running maximum moves between parts, most weights vanish."""
    PrefixCase(kind[1], 2, 1, 64, 16, 200, [100, 3], [1, 2], spread=2.0, seed=5).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
def test_prefix_many_sequences(kind):
    PrefixCase(kind[1], 4, 2, 64, 16, 140, [(7 * i) % 23 for i in range(70)], [1] * 70, seed=8).run(kind[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Nk,H,prefix,held,new", [(32, 8, 128, 2000, 40, [1] * 9), (64, 8, 128, 1030, 300, [1] * 3), (16, 16, 64, 4100, 9, [1] * 20), (28, 4, 128, 700, 20, [60, 1, 90, 17])])
def test_prefix_sizes_of_models(dt, N, Nk, H, prefix, held, new):
    PrefixCase(dt, N, Nk, H, 64, prefix, [(held * (i + 1)) % 311 for i in range(len(new))], new, seed=1, stale=0.0).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,Nk,H,size", [(8, 2, 64, 16), (8, 2, 128, 64), (4, 4, 128, 8)])
def test_prefix_units_of_few_and_of_many_rows(dt, N, Nk, H, size):
    """Sequences of 1 to 40 tokens by turns: units of up to eight rows and of more follow one another on every SM."""
    new = [(1, 2, 3, 40, 1, 0, 2, 8, 9)[i % 9] for i in range(130)]
    PrefixCase(dt, N, Nk, H, size, 100, [(29 * i) % 83 for i in range(130)], new, seed=4).run(GPU)


@pytest.mark.gpu
@pytest.mark.parametrize("N,H,held,new", [(128, 64, [5] * 8, [100] * 8), (2, 128, [i % 7 for i in range(780)], [1] * 780), (64, 128, [0, 3, 0], [900, 1, 700]),
                                          (2, 128, [i % 7 for i in range(400)], [(1, 1, 0, 2)[i % 4] for i in range(400)]),
                                          (16, 64, [i % 9 for i in range(300)], [(1, 9, 0, 2)[i % 4] for i in range(300)])])
def test_prefix_batches_of_many_row_tiles(N, H, held, new):
    """More row tiles than a CTA keeps the running sums of (long prompts, many sequences), and more than it has threads."""
    PrefixCase(torch.bfloat16, N, 1, H, 16, 70, held, new, seed=7).run(GPU)


@pytest.mark.gpu
def test_prefix_of_a_cache_beyond_32_bit_offsets():
    """The same blocks behind 2^31 elements of cache give the same bits."""
    a = PrefixCase(torch.bfloat16, 4, 2, 128, 64, 100, [5, 70], [1, 3], stale=0.0)
    near = a.call(GPU)()
    first, used = 2 ** 31 // (64 * 2 * 128) + 3, len(a.caches[0])
    caches = [torch.zeros(first + used, 64, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    for c, mine in zip(caches, a.caches):
        c[first:].copy_(mine)
    a.caches, a.table, a.slot = caches, a.table + first, a.slot + first * 64
    call = a.call(GPU)
    call.sess.run_with_iobinding(call.binding)
    torch.cuda.synchronize()
    call.sess.check_device_status()
    assert torch.equal(call.outs["out"].cpu(), near["out"])
    for name in ("kc_out", "vc_out"):
        assert torch.equal(call.outs[name][first:].cpu(), near[name]) and not call.outs[name][:first].any()


@pytest.mark.parametrize("provider", PROVIDERS)
@pytest.mark.parametrize("cum", [[0, 4, 2], [0, 2, 9], [-1, 2, 5]])
def test_prefix_lengths_that_fit_no_batch_are_an_error(provider, cum):
    c = PrefixCase(torch.float32 if provider == CPU else torch.bfloat16, 4, 2, 64, 16, 70, [5, 30], [2, 3])
    c.cum = i32(*cum)
    with pytest.raises((InvalidArgument, EPFail)):
        c.call(provider)()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("new", [[1], [5, 4]])
def test_prefix_of_one_key_head_in_hundreds_of_parts(dt, new):
    PrefixCase(dt, 1, 1, 64, 64, 22000, [5, 70][:len(new)], new, seed=6, stale=0.0).run(GPU)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cap", [0.5, 30.0, 64.0, 65.0, 1e6])
def test_prefix_caps(kind, cap):
    """Caps below the scores, near them, and so large that they change nothing."""
    PrefixCase(kind[1], 4, 1, 64, 16, 70, [60, 0, 190], [3, 1, 1], spread=2.0, cap=cap, seed=2).run(kind[0])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows", [1, 2, 3])
def test_prefix_scores_far_apart_within_a_tile(kind, rows):
    """Each quarter of a tile has a maximum of its own, and most weights vanish beside one."""
    PrefixCase(kind[1], 4, 2, 128, 16, 70, [60, 0, 190], [rows, 1, rows], scale=2.0, seed=rows).run(kind[0])


@pytest.mark.gpu
def test_prefix_captured_graph_follows_the_lengths():
    """One captured step is replayed for other lengths, another shared prefix and other queries."""
    a = PrefixCase(torch.bfloat16, 8, 2, 128, 64, 192, [5, 70, 200], [1, 1, 1], seed=1)
    call = a.call(GPU, graph=True)
    a.check(call())
    for prefix, held in ((64, [1, 300, 2]), (0, [9, 1, 0]), (300, [100, 0, 70])):
        b = PrefixCase(torch.bfloat16, 8, 2, 128, 64, prefix, held, [1, 1, 1], seed=prefix)
        width, blocks = call.ins["table"].shape[1], len(call.ins["kc"])
        if b.table.shape[1] > width or len(b.caches[0]) > blocks or len(b.cos) > len(a.cos):
            b = PrefixCase(torch.bfloat16, 8, 2, 128, 64, 128, [1, 0, 130], [1, 1, 1], seed=9)
        table = torch.zeros_like(a.table)
        table[:, :b.table.shape[1]] = b.table
        for c, mine in zip(("kc", "vc"), b.caches):
            call.ins[c][:len(mine)].copy_(mine)
        angle_rows = len(b.cos)
        b.cos, b.sin = a.cos, a.sin
        assert angle_rows <= len(a.cos)
        for name, t in dict(q=b.qkv.reshape(3, -1), past=i32(*[p for p, _ in b.lengths]), table=table, prefix=i32(b.prefix), pos=b.pos, slot=b.slot).items():
            call.ins[name].copy_(t)
        got = call()
        got = dict(out=got["out"], kc_out=got["kc_out"][:len(b.caches[0])], vc_out=got["vc_out"][:len(b.caches[1])])
        b.check(got)
    assert call.sess.num_captured_graphs() == 1


@pytest.mark.gpu
def test_prefix_two_captured_graphs_of_one_session_by_turns():
    a = PrefixCase(torch.bfloat16, 8, 2, 128, 64, 192, [5, 70], [1, 1], seed=1)
    b = PrefixCase(torch.bfloat16, 8, 2, 128, 64, 320, [300, 9, 64, 0, 31], [1, 1, 1, 1, 1], seed=2)
    first, second = a.call(GPU, graph=True), b.call(GPU, graph=True)
    second.sess = first.sess
    second.binding = first.sess.io_binding()
    for n, t in second.ins.items():
        second.binding.bind_torch_input(n, t)
    for n, t in second.outs.items():
        second.binding.bind_torch_output(n, t)
    for _ in range(3):
        for i, (case, call) in enumerate(((a, first), (b, second))):
            call.outs["out"].fill_(3.0)
            options = ort.RunOptions()
            options.add_run_config_entry("gpu_graph_id", str(i + 1))
            call.sess.run_with_iobinding(call.binding, options)
            torch.cuda.synchronize()
            call.sess.check_device_status()
            case.check({n: t.cpu() for n, t in call.outs.items()})
    assert first.sess.num_captured_graphs() == 2


@pytest.mark.gpu
def test_prefix_two_sessions_at_once():
    cases = [PrefixCase(torch.float16, 16, 4, 64, 16, 700, [(31 * i) % 290 for i in range(40)], [1] * 40, seed=s, stale=0.0) for s in (1, 2)]
    calls = [c.call(GPU) for c in cases]
    alone = [call()["out"] for call in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for _ in range(20):
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                call.sess.run_with_iobinding(call.binding)
    torch.cuda.synchronize()
    for call, want in zip(calls, alone):
        call.sess.check_device_status()
        assert torch.equal(call.outs["out"].cpu(), want)


@pytest.mark.gpu
def test_prefix_on_another_stream_and_twice():
    a = PrefixCase(torch.bfloat16, 8, 2, 128, 64, 192, [5, 70], [1, 1], seed=1)
    call = a.call(GPU)
    first = call()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = call()
    assert torch.equal(first["out"], second["out"])      # no order of arrival decides a sum


@pytest.mark.parametrize("provider", PROVIDERS)
def test_prefix_argument_checks(provider):
    base = dict(dt=torch.float32, N=4, Nk=2, H=64, size=16, prefix=20, held=[3], new=[1])

    def broken(change):
        c = PrefixCase(**base)
        change(c)
        with pytest.raises(InvalidArgument):
            c.call(provider)()
    broken(lambda c: setattr(c, "Nk", 3))
    broken(lambda c: setattr(c, "table", c.table.long()))
    broken(lambda c: setattr(c, "cum", i32(0, 1, 1)))
    broken(lambda c: setattr(c, "cos", c.cos.half()))
    broken(lambda c: setattr(c, "pos", c.pos[:0]))
    broken(lambda c: setattr(c, "qkv", c.qkv[:, :-1]))
    broken(lambda c: setattr(c, "cap", -1.0))
    broken(lambda c: setattr(c, "cap", math.inf))
    broken(lambda c: setattr(c, "scale", -0.5))
    broken(lambda c: setattr(c, "scale", math.nan))
    broken(lambda c: setattr(c, "table", c.table[:, :0]))
    broken(lambda c: setattr(c, "caches", [c.caches[0], c.caches[1][:-1]]))


# ---------------------------------------------------------------------------------------------------- token log probabilities
SCORE_KINDS = [pytest.param((CPU, torch.float32), id="cpu-fp32"), pytest.param((CPU, torch.bfloat16), id="cpu-bf16")] + [
    pytest.param((GPU, d), marks=pytest.mark.gpu, id="gpu-" + n) for n, d in (("fp32", torch.float32), ("bf16", torch.bfloat16), ("fp16", torch.float16))]


def score_call(provider, x, tokens, k, grads=None, graph=False, in_place=False):
    lead = list(x.shape[:-1])
    f32 = lambda *s: torch.full(s, 7.0)  # noqa: E731
    ins = dict(x=x, tokens=tokens)
    outs = dict(lp=f32(*lead), h=f32(*lead), top=f32(*lead, k), index=torch.full((*lead, k), 7, dtype=torch.int64), lse=f32(*lead))
    nodes = [("TokenLogProbs", ["x", "tokens"], list(outs), dict(top_k=k))]
    if grads is not None:
        ins.update({n: g for n, g in grads.items() if g is not None})
        name = lambda n: n if grads.get(n) is not None else ""  # noqa: E731
        out = "x_out" if in_place else "dx"
        nodes.append(("TokenLogProbsGrad", ["x", "tokens", "lse", "h" if name("g_h") else "", name("g_lp"), name("g_h"), "index" if name("g_top") else "", name("g_top"), name("g_lse")], [out], {}))
        outs[out] = torch.full_like(x, 7.0)
    return Call(provider, nodes, ins, outs, graph)


def check_score(provider, x, tokens, k):
    """Sums of V terms in 32 bits: a running sum of at most V terms is off by V 2^-24 relative at worst, an exponential by 2^-21; a difference
    x - lse by 2^-23 of the larger.  The entropy adds a sum of terms p log p, each bounded by p (|x| + |lse|)."""
    rows, V = x.reshape(-1, x.shape[-1]).shape
    got = score_call(provider, x, tokens, k)()
    lp, h, top, index, lse = oracle.token_log_probs(x.double().reshape(rows, V), tokens.reshape(-1), k)
    finite = x.double().masked_fill(~torch.isfinite(x.double()), 0).abs().amax() if x.numel() else 0.0
    off = (V + 64) * 2.0 ** -24 * (1 + (1 + math.log(V)))
    eps = off + 2.0 ** -20 + 2.0 ** -22 * float(finite)
    assert got["index"].reshape(rows, k).tolist() == index.tolist()
    for name, want, tol in (("lp", lp, eps), ("lse", lse, eps), ("top", top, eps), ("h", h, eps * (2 + 2 * float(finite)))):
        g = got[name].reshape(want.shape).double()
        assert torch.equal(g.isnan(), want.isnan()) and torch.equal(g == -math.inf, want == -math.inf), name
        keep = torch.isfinite(want)
        assert (g[keep] - want[keep]).abs().le(tol).all(), (name, float((g[keep] - want[keep]).abs().max()), tol)


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("rows,V,k", [(1, 1, 1), (1, 7, 3), (3, 32, 32), (2, 33, 5), (5, 257, 20), (2, 1000, 0), (1, 4099, 32), (300, 65, 2), (7, 2048, 1), (2, 9000, 8)])
def test_log_probs(kind, rows, V, k):
    g = torch.Generator().manual_seed(V)
    x = (3 * torch.randn(rows, V, generator=g)).to(kind[1])
    check_score(kind[0], x, torch.randint(0, V, (rows,), generator=g), k)


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("V,k", [(40, 12), (1031, 32)])
def test_log_probs_of_hard_rows(kind, V, k):
    """Ties, zeros of both signs, impossible tokens, rows without any possible token, one certain token, steep and flat rows, NaN and infinity."""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(16, V, generator=g)
    x[0] = 0.0
    x[1] = torch.randint(-2, 3, (V,), generator=g).float()
    x[2, ::2], x[2, 1::2] = 0.0, -0.0
    x[3] = -math.inf
    x[4, 1:] = -math.inf
    x[5, :-1] = -math.inf
    x[6, 5:] = -math.inf
    x[7] = torch.arange(V).float()
    x[8] = -torch.arange(V).float() - 1000
    x[9, 3] = math.nan
    x[10, V - 1] = math.inf
    x[11] = -torch.finfo(torch.float16).max
    x[12] = -torch.finfo(torch.float16).max
    x[12, 7] = torch.finfo(torch.float16).max
    x[13] = torch.where(torch.arange(V) % 3 == 0, -math.inf, 5.0)
    x[14, V // 2] = -math.nan
    tokens = torch.tensor([0, 1, V - 1, 2, 0, 0, 3, V - 1, 0, 1, 2, 3, 7, 0, 5, 6])
    check_score(kind[0], x.to(kind[1]), tokens, k)


@pytest.mark.parametrize("kind", SCORE_KINDS)
def test_log_probs_padding_tokens_and_shapes(kind):
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 50, generator=g).to(kind[1])
    check_score(kind[0], x, torch.tensor([[-1, -100, 50], [2 ** 40, 0, 49]]), 4)
    check_score(kind[0], x[0, 0], torch.tensor(3), 2)
    check_score(kind[0], x[:, :0], torch.zeros(2, 0, dtype=torch.int64), 2)
    got = score_call(kind[0], x, torch.tensor([[1, 2, 3], [4, 5, -1]], dtype=torch.int32), 0)()
    assert got["lp"].shape == (2, 3) and got["lp"][1, 2] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V", [(1, 128256), (6, 50257), (37, 32000), (333, 50257)])
def test_log_probs_sizes_of_models(dt, rows, V):
    """Against torch in 64 bits (the oracle's loops are slow here)."""
    g = torch.Generator().manual_seed(rows)
    x = (2.5 * torch.randn(rows, V, generator=g)).to(dt)
    tokens = torch.randint(0, V, (rows,), generator=g)
    grads = dict(g_lp=torch.randn(rows, generator=g), g_h=0.1 * torch.randn(rows, generator=g))
    got = score_call(GPU, x, tokens, 20, grads)()
    logp = torch.log_softmax(x.double(), -1)
    p = logp.exp()
    h = -(p * logp).sum(-1)
    order = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :20]
    assert torch.equal(got["index"], order)
    tol = 4e-6 * 20           # sums in 32 bits, as in check_score but for random errors: 2^-18 of values up to 20
    for name, want in (("lp", logp.gather(1, tokens[:, None])[:, 0]), ("h", h), ("top", logp.gather(1, order)), ("lse", torch.logsumexp(x.double(), -1))):
        assert (got[name].double() - want).abs().max() < tol, name
    one = torch.nn.functional.one_hot(tokens, V).double()
    want = grads["g_lp"].double()[:, None] * (one - p) - grads["g_h"].double()[:, None] * p * (logp + h[:, None])
    # p carries the error of lse (tol) as a factor; the output is rounded once (fp16: also below its normal range)
    bound = half_step(dt) * want.abs() + tol * (p * (grads["g_lp"].abs() + 40 * grads["g_h"].abs())[:, None]) + torch.finfo(dt).tiny * half_step(dt) + 1e-9
    assert ((got["dx"].double() - want).abs() <= bound).all()


@pytest.mark.gpu
def test_log_probs_beyond_32_bit_offsets():
    """The last of so many rows that their logits are more than 2^31; tolerances as above."""
    rows, V = 2 ** 31 // 50257 + 7, 50257
    g = torch.Generator().manual_seed(1)
    last = (2.5 * torch.randn(V, generator=g)).bfloat16()
    x = torch.zeros(rows, V, dtype=torch.bfloat16, device="cuda")
    x[-1] = last.cuda()
    grads = dict(g_lp=torch.ones(rows), g_h=torch.zeros(rows))
    call = score_call(GPU, x, torch.full((rows,), 5), 3, grads)
    call.sess.run_with_iobinding(call.binding)
    torch.cuda.synchronize()
    logp = torch.log_softmax(last.double(), -1)
    tol = 4e-6 * 20
    assert abs(float(call.outs["lp"][-1]) - float(logp[5])) < tol and abs(float(call.outs["h"][-1]) + float((logp.exp() * logp).sum())) < tol
    assert (call.outs["lse"][:-1].cpu().double() - math.log(V)).abs().max() < tol and (call.outs["index"][:-1].cpu() == torch.arange(3)).all()
    assert torch.equal(call.outs["index"][-1].cpu(), torch.sort(last.float(), descending=True, stable=True)[1][:3])
    want = -logp.exp()
    want[5] += 1
    assert ((call.outs["dx"][-1].cpu().double() - want).abs() <= half_step(torch.bfloat16) * want.abs() + tol * logp.exp() + 1e-9).all()


GRADS = ["g_lp", "g_h", "g_top", "g_lse"]


@pytest.mark.parametrize("kind", SCORE_KINDS)
@pytest.mark.parametrize("which", [GRADS, ["g_lp"], ["g_h"], ["g_top"], ["g_lse"], ["g_lp", "g_h"]])
@pytest.mark.parametrize("V,k", [(9, 3), (300, 5), (1027, 32)])
def test_log_probs_gradient(kind, which, V, k):
    g = torch.Generator().manual_seed(V)
    rows = 9
    x = (2 * torch.randn(rows, V, generator=g))
    x[1, ::2] = -math.inf
    x[2] = -math.inf
    x[3, 1:] = -math.inf
    x = x.to(kind[1])
    tokens = torch.tensor([0, 1, 2, 0, -1, V, V - 1, 3, 4])
    index = oracle.token_log_probs(x.double(), tokens, k)[3]
    # a token that a row excludes has the log probability -inf: it gets no gradient here
    every = dict(g_lp=torch.randn(rows, generator=g), g_h=torch.randn(rows, generator=g), g_top=torch.randn(rows, k, generator=g), g_lse=torch.randn(rows, generator=g))
    got = score_call(kind[0], x, tokens, k, {n: every[n] for n in which})()["dx"].double()
    use = {n: every[n].double() if n in which else torch.zeros_like(every[n]).double() for n in GRADS}
    want = oracle.token_log_probs_grad(x.double(), tokens, use["g_lp"], use["g_h"], index, use["g_top"], use["g_lse"])
    size = sum(v.abs().reshape(rows, -1).sum(1) for v in use.values())[:, None]
    # coefficients of p up to size * 20 carry 32-bit errors of sums over V terms, and the result is rounded once
    p = x.double().softmax(-1).nan_to_num(0)
    bound = half_step(kind[1]) * want.abs() + (V + 64) * 2.0 ** -22 * 20 * size * p + 2.0 ** -22 * size + torch.finfo(kind[1]).tiny
    assert torch.isfinite(got).all() and ((got - want).abs() <= bound).all(), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("provider", PROVIDERS)
def test_log_probs_gradient_against_differences(provider):
    """Central differences of the operator's own outputs, step 2^-5: their error is h^2 / 6 times a third derivative (below 10 for these) plus
    2^-21 / h of 32-bit values."""
    g = torch.Generator().manual_seed(4)
    rows, V, k, h = 3, 21, 2, 2.0 ** -5
    x, tokens = torch.randn(rows, V, generator=g), torch.tensor([2, 20, 7])
    x[:, 11], x[:, 5] = 4.0, 3.0                                 # the alternatives stay the same ones
    grads = dict(g_lp=torch.randn(rows, generator=g), g_h=torch.randn(rows, generator=g), g_top=torch.randn(rows, k, generator=g), g_lse=torch.randn(rows, generator=g))
    dx = score_call(provider, x, tokens, k, grads)()["dx"].double()
    bumped = torch.cat([(x + s * h * torch.eye(V)[v]) for v in range(V) for s in (1, -1)])
    got = score_call(provider, bumped, tokens.repeat(2 * V), k)()
    value = sum((got[o].double().reshape(V, 2, rows, -1) * grads[n].double().reshape(rows, -1)).sum(-1) for o, n in (("lp", "g_lp"), ("h", "g_h"), ("top", "g_top"), ("lse", "g_lse")))
    diff = ((value[:, 0] - value[:, 1]) / (2 * h)).T
    size = sum(v.abs().reshape(rows, -1).sum(1) for v in grads.values()).max()
    assert (dx - diff).abs().max() < size * (10 * h * h / 6 + 2.0 ** -21 * 8 / h)


@pytest.mark.parametrize("kind", SCORE_KINDS)
def test_log_probs_gradient_over_the_logits(kind):
    """The gradient may be written over the logits it is formed from."""
    g = torch.Generator().manual_seed(2)
    x, tokens = torch.randn(4, 300, generator=g).to(kind[1]), torch.tensor([1, 2, 3, -1])
    grads = dict(g_lp=torch.randn(4, generator=g), g_h=torch.randn(4, generator=g))
    apart = score_call(kind[0], x, tokens, 2, grads)()
    over = score_call(kind[0], x.clone(), tokens, 2, grads, in_place=True)()
    assert torch.equal(apart["dx"], over["x_out"]) and torch.equal(apart["lp"], over["lp"])


@pytest.mark.parametrize("kind", SCORE_KINDS)
def test_log_probs_of_a_view(kind):
    """Rows that start on odd addresses, and logits that are columns of a wider tensor."""
    g = torch.Generator().manual_seed(6)
    wide = torch.randn(5, 1003, generator=g).to(kind[1])
    tokens = torch.tensor([0, 1, 500, 998, -1])
    want = score_call(kind[0], wide[:, 3:1002].contiguous(), tokens, 6, dict(g_lp=torch.ones(5)))()
    call = score_call(kind[0], wide[:, 3:1002].contiguous(), tokens, 6, dict(g_lp=torch.ones(5)))
    moved = wide.to(call.ins["x"].device)
    call.binding.bind_torch_input("x", moved[:, 3:1002])
    got = call()
    base = torch.empty(5 * 999 + 1, dtype=kind[1], device=moved.device)
    base[1:].copy_(moved[:, 3:1002].reshape(-1))
    call.binding.bind_torch_input("x", base[1:].view(5, 999))
    again = call()
    for n in want:
        assert torch.equal(want[n], got[n]), n
        tol = 0 if want[n].dtype == torch.int64 else 2.0 ** -18     # another split of the same sums
        assert (want[n].double() - again[n].double()).abs().max() <= tol * max(1.0, float(want[n].double().abs().max())) + (half_step(kind[1]) if n == "dx" else 0), n


@pytest.mark.parametrize("provider", PROVIDERS)
def test_log_probs_argument_checks(provider):
    x, tokens = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int64)
    for args in ((x, tokens, 11), (x, tokens, 33), (x, tokens, -1), (x, tokens[:2], 1), (x.long(), tokens, 1), (torch.zeros(3, 0), tokens, 0), (x, tokens.float(), 1)):
        with pytest.raises(Exception) as e:
            score_call(provider, args[0], args[1], max(args[2], 0) if args[2] != -1 else 0)() if args[2] >= 0 else \
                Call(provider, [("TokenLogProbs", ["x", "tokens"], ["lp"], dict(top_k=-1))], dict(x=x, tokens=tokens), dict(lp=torch.zeros(3)))()
        assert isinstance(e.value, (InvalidArgument, RuntimeError)), e.value


@pytest.mark.gpu
def test_log_probs_in_a_captured_graph():
    g = torch.Generator().manual_seed(0)
    x, tokens = torch.randn(3, 5000, generator=g).bfloat16(), torch.tensor([1, 2, 3])
    call = score_call(GPU, x, tokens, 5, dict(g_lp=torch.ones(3)), graph=True)
    for _ in range(4):
        got = call()
        want = score_call(GPU, call.ins["x"].cpu(), call.ins["tokens"].cpu(), 5, dict(g_lp=torch.ones(3)))()
        assert all(torch.equal(got[n], want[n]) for n in want)
        call.ins["x"].copy_(torch.randn(3, 5000, generator=g).bfloat16())
        call.ins["tokens"].add_(700)
    assert call.sess.num_captured_graphs() == 1


# ----------------------------------------------------------------------------------------------------------- all of them in a row
@pytest.mark.parametrize("kind", KINDS)
def test_layout_attention_and_log_probs_in_one_graph(kind):
    """A step as a decoder has it: the layout's outputs place the tokens, a product makes logits of the attention's result, the step answers with
    log probabilities.  Two steps: the second one needs a new block."""
    provider, dt = kind
    N, Nk, H, size, V, prefix = 4, 2, 64, 16, 97, 64
    g = torch.Generator().manual_seed(11)
    c = PrefixCase(dt, N, Nk, H, size, prefix, [15, 3], [1, 1], seed=2, stale=0.0)
    table = torch.full((2, 8), 0, dtype=torch.int32)
    held = [oracle.blocks_of(p, size) for p, _ in c.lengths]
    for b in range(2):
        table[b, :held[b]] = c.table[b, :held[b]]
    spare = [i for i in range(len(c.caches[0])) if i not in set(c.table[0, :held[0]].tolist() + c.table[1, :held[1]].tolist())]
    w = (0.2 * torch.randn(N * H, V, generator=g)).to(dt)
    angle = torch.arange(200).double()[:, None] * 100.0 ** (-torch.arange(H // 2).double() / (H // 2))
    ins = dict(past=i32(*[p for p, _ in c.lengths]), new=i32(1, 1), table=table, free=i32(*spare[:2]), ids=torch.zeros(2, dtype=torch.int64), q=c.qkv.reshape(2, -1),
               kc=c.caches[0], vc=c.caches[1], prefix=i32(prefix), cos=angle.cos().to(dt), sin=angle.sin().to(dt), w=w, tokens=torch.tensor([5, 90]))
    outs = dict(table_out=table, cum=i32(0, 0, 0), pos=torch.zeros(2, dtype=torch.int64), slot=torch.zeros(2, dtype=torch.int64), used=i32(0),
                a=torch.zeros(2, N * H, dtype=dt), kc_out=c.caches[0], vc_out=c.caches[1], logits=torch.zeros(2, V, dtype=dt), lp=torch.zeros(2), h=torch.zeros(2))
    dev = "cuda" if provider == GPU else "cpu"
    nodes = [ol.make_node("PagedBatchLayout", ["past", "new", "table", "free", "ids"], ["table_out", "cum", "pos", "slot", "used"], domain=FUSED, block_size=size),
             ol.make_node("SharedPrefixPagedAttention", ["q", "", "", "kc", "vc", "cum", "past", "table_out", "prefix", "cos", "sin", "pos", "slot"],
                          ["a", "kc_out", "vc_out"], domain=FUSED, num_heads=N, kv_num_heads=Nk, do_rotary=1),
             ol.make_node("MatMul", ["a", "w"], ["logits"]), ol.make_node("TokenLogProbs", ["logits", "tokens"], ["lp", "h"], domain=FUSED)]
    info = lambda n, t: ol.make_tensor_value_info(n, ONNX[t.dtype], list(t.shape))  # noqa: E731
    graph = ol.make_graph(nodes, "step", [info(n, t) for n, t in ins.items()], [info(n, t) for n, t in outs.items()])
    sess = ort.InferenceSession(ol.make_model(graph, opset=17, extra_opsets={FUSED: 1}).serialize(), providers=[provider])
    ins = {n: t.to(dev) for n, t in ins.items()}
    outs = {n: ins[n[:-4]] if n.endswith("_out") else t.to(dev) for n, t in outs.items()}
    binding = sess.io_binding()
    for n, t in ins.items():
        binding.bind_torch_input(n, t)
    for n, t in outs.items():
        binding.bind_torch_output(n, t)
    u, lengths, free = half_step(dt), list(c.lengths), spare[:2]
    for step in range(2):
        want = oracle.batch_layout([p for p, _ in lengths], [1, 1], ins["table"].tolist(), free, 2, size)
        sess.run_with_iobinding(binding)
        got = {n: t.cpu() for n, t in outs.items()}
        assert got["table_out"].tolist() == want[0] and got["slot"].tolist() == want[3] and got["used"].tolist() == [want[4]]
        x = ins["q"].cpu().double().reshape(2, N + 2 * Nk, H)
        cos, sin = (ins[n].cpu()[got["pos"]].double() for n in ("cos", "sin"))
        attn, bound = oracle.paged_attention(oracle.rotate(x[:, :N], cos, sin), got["kc_out"], got["vc_out"], got["table_out"], lengths, size, H ** -0.5, 0.0, u)
        assert ((got["a"].reshape(2, N, H).double() - attn).abs() <= bound).all()
        lp, h, *_ = oracle.token_log_probs(got["logits"].double(), ins["tokens"].cpu(), 0)
        assert (got["lp"].double() - lp).abs().max() < 2e-5 and (got["h"].double() - h).abs().max() < 1e-4
        free = free[want[4]:] + [0] * want[4]
        lengths = [(p + 1, 1) for p, _ in lengths]
        ins["past"].add_(1)
        ins["free"].copy_(i32(*free))
        ins["q"].copy_(torch.randn(2, (N + 2 * Nk) * H, generator=g).to(dt))


# ------------------------------------------------------------------------------------------------------------- the C interface
def test_c_entries_refuse_what_is_missing():
    """A return code, on a machine without a GPU too."""
    from onnxruntime_b200.ops import _kernels as K
    lib = ctypes.CDLL(K.lib_path())
    for name in ("ortb200_batch_layout", "ortb200_prefix_attn", "ortb200_token_log_probs", "ortb200_token_log_probs_grad"):
        assert getattr(lib, name)(None, None) == -1, name
    size = lib.ortb200_prefix_attn_workspace_bytes
    size.restype, size.argtypes = ctypes.c_int64, [ctypes.c_int64] + [ctypes.c_int] * 5
    assert size(10, 2, 8, 0, 64, 1) == size(-1, 2, 8, 2, 64, 1) == size(10, 2, 8, 2, 0, 0) == -1
    assert size(10, 2, 8, 2, 64, 1) > size(10, 2, 8, 2, 64, 0) > 0

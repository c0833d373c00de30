"""Greedy generation drivers for decoder graphs with GroupQueryAttention or PagedAttention.

Mirrors how the reference's tooling drives an exported LLM
(onnxruntime/python/tools/transformers/models/llama/benchmark_e2e.py:120-148,
435-512): inputs and outputs are bound once with ``IOBinding``; ``past`` and
``present`` of every layer are bound to the SAME pre-allocated cache buffer so
the KV cache never moves; the prompt runs once, then one token per step.  The
decode step has fixed shapes and addresses, so with ``enable_cuda_graph`` the
session captures it on the first step and replays it afterwards.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Callable, Dict, Hashable, List, Optional, Sequence, Tuple, Union

import numpy as np
import torch

from .. import onnx_lite as ol
from ..capi import InferenceSession, RunOptions
from .decoder_cache import CacheFull, CachePool
from .llama import LlamaConfig, empty_kv_cache


MOST_DRAFTED = 256   # tokens of a sequence's tree (com.ortb200.TreePagedAttention)


class DecoderRunner:
    """Owns the KV cache and the bindings of one (session, batch size, cache capacity)."""

    def __init__(self, session: InferenceSession, cfg: LlamaConfig, batch: int, max_len: int, tp_size: int = 1,
                 device: Optional[torch.device] = None, prefill_graph: bool = False):
        """``prefill_graph``: also capture the prompt run in a CUDA graph (one graph per prompt shape; worthwhile when the
        same prompt shape recurs, e.g. fixed-size prefill chunks).  Needs a session created with ``enable_cuda_graph``."""
        self.sess = session
        self.cfg = cfg
        self.batch = batch
        self.max_len = max_len
        self.device = device if device is not None else (
            torch.device("cuda", torch.cuda.current_device()) if "CUDAExecutionProvider" in session.get_providers() else torch.device("cpu"))
        self.cache = empty_kv_cache(cfg, batch, max_len, self.device, tp_size)
        self.out_names = [o.name for o in session.get_outputs()]
        self.has_argmax = "next_tokens" in self.out_names
        # static device buffers for the decode step (addresses must not change between graph replays)
        self.step_ids = torch.zeros(batch, 1, dtype=torch.int64, device=self.device)
        self.step_seqlens = torch.zeros(batch, dtype=torch.int32, device=self.device)
        self.step_next = torch.zeros(batch, 1, dtype=torch.int64, device=self.device)
        self.step_logits = torch.zeros(batch, 1, cfg.vocab_size, dtype=self.cache[0][0].dtype, device=self.device)
        self._decode_binding = None
        self._decode_total = None
        self._ro_decode = RunOptions()
        self._ro_decode.add_run_config_entry("gpu_graph_id", "1")
        self._ro_prefill = RunOptions()
        self._ro_prefill.add_run_config_entry("gpu_graph_id", "-1")
        self._prefill_graph = prefill_graph
        self._prefill_graph_ids: Dict[Tuple[int, int], int] = {}

    def _bind_common(self, binding, ids: torch.Tensor, seqlens: torch.Tensor, total: torch.Tensor, logits, next_tokens) -> None:
        binding.bind_torch_input("input_ids", ids)
        binding.bind_torch_input("seqlens_k", seqlens)
        binding.bind_torch_input("total_sequence_length", total)
        for i, (k, v) in enumerate(self.cache):
            binding.bind_torch_input(f"past_key_values.{i}.key", k)
            binding.bind_torch_input(f"past_key_values.{i}.value", v)
            binding.bind_torch_output(f"present.{i}.key", k)
            binding.bind_torch_output(f"present.{i}.value", v)
        binding.bind_torch_output("logits", logits)
        if self.has_argmax:
            binding.bind_torch_output("next_tokens", next_tokens)

    def prefill(self, input_ids: torch.Tensor) -> torch.Tensor:
        """Run the prompt [B, S]; returns the first generated token per sequence [B, 1] (device tensor)."""
        B, S = input_ids.shape
        assert B == self.batch and S <= self.max_len
        ids = input_ids.to(self.device)
        seqlens = torch.full((B,), S - 1, dtype=torch.int32, device=self.device)
        total = torch.tensor(S, dtype=torch.int32)
        logits = torch.empty(B, 1, self.cfg.vocab_size, dtype=self.cache[0][0].dtype, device=self.device)
        nxt = torch.empty(B, 1, dtype=torch.int64, device=self.device)
        binding = self.sess.io_binding()
        self._bind_common(binding, ids, seqlens, total, logits, nxt)
        ro = self._ro_prefill
        if self._prefill_graph:
            gid = self._prefill_graph_ids.setdefault((B, S), 2 + len(self._prefill_graph_ids))
            ro = RunOptions()
            ro.add_run_config_entry("gpu_graph_id", str(gid))
        try:
            self.sess.run_with_iobinding(binding, ro)
        except Exception:
            if ro is self._ro_prefill:
                raise
            # the prompt graph holds something that cannot be captured: run it eagerly from now on
            self._prefill_graph = False
            self.sess.run_with_iobinding(binding, self._ro_prefill)
        self.cur_len = S
        self.prefill_logits = logits
        if not self.has_argmax:
            nxt = logits.float().argmax(-1)
        return nxt

    def reorder_cache(self, rows: torch.Tensor) -> None:
        """Row i of every cache takes the content of row rows[i] (beam search: beams follow their parents)."""
        rows = rows.to(self.device)
        for k, v in self.cache:
            k.copy_(k.index_select(0, rows))
            v.copy_(v.index_select(0, rows))

    def _ensure_decode_binding(self) -> None:
        if self._decode_binding is not None:
            return
        binding = self.sess.io_binding()
        # the capacity bound is a host scalar: the cache capacity, so the captured graph stays valid every step
        self._decode_total = torch.tensor(self.max_len, dtype=torch.int32)
        self._bind_common(binding, self.step_ids, self.step_seqlens, self._decode_total, self.step_logits, self.step_next)
        self._decode_binding = binding

    def decode_step(self, tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One decode step.  ``tokens`` [B, 1] (device or pinned host); None re-uses the previous step's output,
        which already sits in the bound input buffer."""
        self._ensure_decode_binding()
        if tokens is not None:
            self.step_ids.copy_(tokens, non_blocking=True)
        else:
            self.step_ids.copy_(self.step_next)
        self.step_seqlens.fill_(self.cur_len)  # total length - 1 after appending this token
        self.sess.run_with_iobinding(self._decode_binding, self._ro_decode)
        self.cur_len += 1
        if not self.has_argmax:
            self.step_next.copy_(self.step_logits.float().argmax(-1))
        return self.step_next

    def decode_step_host(self, ids_pinned: torch.Tensor, seqlens_pinned: torch.Tensor, out_pinned: torch.Tensor) -> None:
        """One decode step driven from the host: inputs come from pinned host memory, the sampled tokens are
        copied back to pinned host memory and the call returns after they have arrived."""
        self._ensure_decode_binding()
        seqlens_pinned.fill_(self.cur_len)
        self.step_ids.copy_(ids_pinned, non_blocking=True)
        self.step_seqlens.copy_(seqlens_pinned, non_blocking=True)
        self.sess.run_with_iobinding(self._decode_binding, self._ro_decode)
        self.cur_len += 1
        if not self.has_argmax:
            self.step_next.copy_(self.step_logits.float().argmax(-1))
        out_pinned.copy_(self.step_next, non_blocking=True)
        torch.cuda.current_stream().synchronize() if self.device.type == "cuda" else None

    def generate(self, input_ids: torch.Tensor, max_new_tokens: int) -> torch.Tensor:
        out = [self.prefill(input_ids).clone()]
        for _ in range(max_new_tokens - 1):
            nxt = self.decode_step(out[-1])
            out.append(nxt.clone())
        return torch.cat(out, dim=1)


class PagedDecoderRunner:
    """Decoding over pooled caches: the serving form of a decoder.  Tokens of all sequences of a step are packed along
    one axis; all sequences share one pool of cache blocks (``block_table[b, j]`` names the block that holds tokens
    [j * block_size, (j + 1) * block_size) of sequence b, as in com.microsoft.PagedAttention,
    onnxruntime/contrib_ops/cuda/bert/paged_attention.cc) and one pool of state slots for models with recurrent layers
    (``state_slots[b]``).  What a model keeps is declared by ``cfg.cache_tensors()``.

    ``step`` runs one batch of any composition - whole prompts, portions of prompts, single tokens - for sequences named
    by the caller and returns the wanted logits; ``release`` gives a sequence's blocks and slot back.  ``prefill`` /
    ``decode_step`` drive a fixed batch of ``batch`` rows on top of the same pool.  A step that brings one token per
    sequence has fixed shapes and addresses and is captured as one CUDA graph per batch size.

    ``draft_step`` (models built with ``draft_trees``) runs a tree of drafted tokens for each sequence, ``accept`` keeps one of
    its paths.

    ``fork`` opens a sequence behind the tokens of another one, with the blocks that these fill in common.  A model built with
    ``shared_prefix`` attends to what all sequences of a batch have in common once for all of them, and extends its block
    tables on the device."""

    def __init__(self, session: InferenceSession, cfg, batch: int, max_len: int, block_size: int = 256,
                 tp_size: int = 1, device: Optional[torch.device] = None, graph_id: int = 1, num_blocks: Optional[int] = None,
                 num_slots: Optional[int] = None):
        """``num_blocks``: size of the block pool (default: ``batch`` sequences of ``max_len`` tokens); ``max_len`` bounds
        one sequence; ``num_slots`` (default ``batch``) bounds the sequences that are open at a time."""
        self.sess, self.cfg, self.batch, self.max_len, self.block_size = session, cfg, batch, max_len, block_size
        self.device = device if device is not None else (
            torch.device("cuda", torch.cuda.current_device()) if "CUDAExecutionProvider" in session.get_providers() else torch.device("cpu"))
        self.blocks_per_seq = (max_len + block_size - 1) // block_size
        self.pool = CachePool(cfg.cache_tensors(tp_size), num_blocks or batch * self.blocks_per_seq, block_size, num_slots or batch, self.device)
        out_info = {o.name: o for o in session.get_outputs()}
        in_names = {i.name for i in session.get_inputs()}
        self.has_argmax = "next_tokens" in out_info
        self.has_slots = "state_slots" in in_names
        self.has_key_starts = "key_starts" in in_names
        self.has_layout = "free_blocks" in in_names
        self.has_trees = "parents" in in_names
        self._drafted: Dict[Hashable, Tuple[int, List[int]]] = {}   # sequences with drafted tokens: tokens held before, parents
        self.logits_dtype = {"tensor(float)": torch.float32, "tensor(float16)": torch.float16,
                             "tensor(bfloat16)": torch.bfloat16}[out_info["logits"].type]
        self._steps: Dict[int, "_DecodeBuffers"] = {}
        self._graph_id = graph_id             # graph ids graph_id, graph_id + 1, ...: one captured graph per batch size
        self._ro_prefill = RunOptions()
        self._ro_prefill.add_run_config_entry("gpu_graph_id", "-1")
        self._rows: List[Tuple[str, int]] = [("row", b) for b in range(batch)]   # sequences of prefill / decode_step
        self.prefill_logits = self.step_logits = None

    @property
    def cur_len(self) -> int:
        """Tokens held by the longest row of the fixed batch."""
        return max((self.pool.sequences[r].length for r in self._rows if r in self.pool.sequences), default=0)

    @cur_len.setter
    def cur_len(self, length: int) -> None:
        self.assume_context(length)

    @property
    def cache(self) -> List[Tuple[torch.Tensor, torch.Tensor]]:
        """(key, value) block pools of the attention layers that own them (models that cache keys and values in every layer)."""
        paged = [self.pool.tensors[c.input] for c in self.pool.spec if c.kind == "paged"]
        return list(zip(paged[::2], paged[1::2]))

    @property
    def block_table(self) -> torch.Tensor:
        """Block table of the fixed batch."""
        return self._table(self._rows).to(self.device)

    def _table(self, seqs) -> torch.Tensor:
        t = torch.zeros(len(seqs), self.blocks_per_seq, dtype=torch.int32)
        for b, s in enumerate(seqs):
            blocks = self.pool.sequences[s].blocks
            t[b, :len(blocks)] = torch.tensor(blocks, dtype=torch.int32)
        return t

    def _slots(self, seqs) -> torch.Tensor:
        return torch.tensor([self.pool.sequences[s].slot for s in seqs], dtype=torch.int32)

    def _granted(self, seqs, new) -> List[int]:
        """The blocks that the batch enters with these new tokens, in its order."""
        got = []
        for s, n in zip(seqs, new):
            e = self.pool.sequences[s]
            got += e.blocks[-(-e.length // self.block_size):-(-(e.length + n) // self.block_size)]
        return got

    def _bind(self, binding, ids, cum, past, table, slots, key_starts, rows, logits, nxt, free=None, shared=None, used=None, parents=None) -> None:
        binding.bind_torch_input("input_ids", ids)
        if self.has_trees:
            binding.bind_torch_input("parents", parents)
        if self.has_layout:      # `cum` holds the new tokens of every sequence; the extended table goes where the table is
            binding.bind_torch_input("new_tokens", cum)
            binding.bind_torch_input("free_blocks", free)
            binding.bind_torch_input("shared_prefix", shared)
            binding.bind_torch_output("block_table_out", table)
            binding.bind_torch_output("blocks_used", used)
        else:
            binding.bind_torch_input("cumulative_sequence_length", cum)
        binding.bind_torch_input("past_seqlens", past)
        binding.bind_torch_input("block_table", table)
        binding.bind_torch_input("logits_indices", rows)
        if self.has_slots:
            binding.bind_torch_input("state_slots", slots)
        if self.has_key_starts:
            binding.bind_torch_input("key_starts", key_starts)
        for c in self.pool.spec:
            binding.bind_torch_input(c.input, self.pool.tensors[c.input])
            binding.bind_torch_output(c.output, self.pool.tensors[c.input])
        binding.bind_torch_output("logits", logits)
        if self.has_argmax:
            binding.bind_torch_output("next_tokens", nxt)

    # ------------------------------------------------------------------------------------------------- general steps
    def step(self, entries: Sequence[Tuple[Hashable, Sequence[int], Sequence[int]]]) -> torch.Tensor:
        """One batch: ``entries`` = (sequence, its next tokens, places among them whose logits are wanted).  A sequence
        seen for the first time is opened.  Returns the logits [wanted, vocab] in the order of the entries."""
        entries = [e for e in entries if len(e[1]) > 0]
        self._make_room(entries)
        if not entries:
            return torch.empty(0, self.cfg.vocab_size, dtype=self.logits_dtype, device=self.device)
        seqs = [e[0] for e in entries]
        if all(len(e[1]) == 1 for e in entries):
            buf = self._decode_buffers(len(entries))
            buf.ids.copy_(torch.tensor([int(e[1][0]) for e in entries], dtype=torch.int64))
            self._run_decode(buf, seqs)
            wanted = [b for b, e in enumerate(entries) for _ in e[2]]
            return buf.logits[torch.tensor(wanted, dtype=torch.int64, device=self.device)]
        return self._run_wanted(entries, None)

    def draft_step(self, entries: Sequence[Tuple[Hashable, Sequence[int], Sequence[int], Sequence[int]]]) -> torch.Tensor:
        """One batch of trees: ``entries`` = (sequence, its tokens, the place of each token's parent among them or -1, places whose
        logits are wanted).  A parent stands in front of its children; a token sees what the sequence holds, its ancestors and
        itself.  Returns the logits [wanted, vocab] in the order of the entries.  ``accept`` has to follow for every sequence."""
        if not self.has_trees:
            raise ValueError("the model has no form for drafted tokens (draft_trees)")
        entries = [e for e in entries if len(e[1]) > 0]
        if len({e[0] for e in entries}) != len(entries):
            raise ValueError("a sequence comes twice in a batch")
        for seq, tokens, parents, _ in entries:
            if len(parents) != len(tokens) or any(not -1 <= p < i for i, p in enumerate(parents)):
                raise ValueError(f"sequence {seq!r}: every token has one parent, in front of it")
            if len(tokens) > MOST_DRAFTED and any(p != i - 1 for i, p in enumerate(parents)):
                raise ValueError(f"sequence {seq!r}: a tree of more than {MOST_DRAFTED} tokens")
        plain = [(seq, tokens, want) for seq, tokens, _, want in entries]
        self._make_room(plain)
        if not entries:
            return torch.empty(0, self.cfg.vocab_size, dtype=self.logits_dtype, device=self.device)
        before = {seq: self.pool.sequences[seq].length for seq, *_ in entries}
        logits = self._run_wanted(plain, [int(p) for _, _, parents, _ in entries for p in parents])
        for seq, _, parents, _ in entries:
            self._drafted[seq] = (before[seq], [int(p) for p in parents])
        return logits

    def accept(self, paths: Dict[Hashable, Sequence[int]]) -> None:
        """What sequences keep of their drafted tokens: for each a path of its tree, the places of its tokens from a root on.  The
        others are forgotten."""
        for seq, path in paths.items():
            if seq not in self._drafted:
                raise ValueError(f"sequence {seq!r} has no drafted tokens")
            parents = self._drafted[seq][1]
            if any(not 0 <= p < len(parents) or parents[p] != q for p, q in zip(path, [-1, *path])):
                raise ValueError(f"sequence {seq!r}: {list(path)} is no path of its tree")
        self.pool.keep({seq: (self._drafted[seq][0], list(path)) for seq, path in paths.items()})
        for seq in paths:
            del self._drafted[seq]

    def _want_accepted(self, seqs) -> None:
        for seq in seqs if self._drafted else ():
            if seq in self._drafted:
                raise ValueError(f"the drafted tokens of sequence {seq!r} wait for accept()")

    def _make_room(self, entries) -> None:
        opened = []
        try:
            for seq, tokens, want in entries:
                self._want_accepted([seq])
                if any(not 0 <= w < len(tokens) for w in want):
                    raise ValueError(f"sequence {seq!r}: a wanted place lies outside its {len(tokens)} tokens")
                if seq not in self.pool.sequences:
                    self.pool.open(seq)
                    opened.append(seq)
                if self.pool.sequences[seq].length + len(tokens) > self.max_len:
                    raise CacheFull(f"sequence {seq!r} would exceed {self.max_len} tokens")
                self.pool.reserve(seq, len(tokens))
        except Exception:
            for seq in opened:
                self.pool.close(seq)
            raise

    def _run_wanted(self, entries, parents) -> torch.Tensor:
        ids = torch.cat([torch.as_tensor(e[1], dtype=torch.int64).reshape(-1).cpu() for e in entries])
        starts, rows = [0], []
        for _, tokens, want in entries:
            rows += [starts[-1] + int(w) for w in want]
            starts.append(starts[-1] + len(tokens))
        logits, _ = self._run_packed(ids, starts, [e[0] for e in entries], rows or [0], parents)
        return logits if rows else logits[:0]

    def fork(self, seq: Hashable, source: Hashable, tokens: Optional[int] = None) -> None:
        """Opens ``seq`` behind the first ``tokens`` (default: all) tokens that ``source`` holds."""
        self._want_accepted([source])
        self.pool.fork(seq, source, tokens)

    def release(self, seq: Hashable) -> None:
        """The sequence is finished: its blocks and slot go back to the pool."""
        self.pool.close(seq)
        self._drafted.pop(seq, None)

    def _run_packed(self, ids: torch.Tensor, starts, seqs, rows, parents=None) -> Tuple[torch.Tensor, torch.Tensor]:
        dev = self.device
        lengths = [self.pool.sequences[s].length for s in seqs]
        past = torch.tensor(lengths, dtype=torch.int32)
        # host tensor: the keys of sequence b, cached and new, are rows [key_starts[b], key_starts[b + 1]) of an expansion
        key_starts = torch.tensor([starts[b] + sum(lengths[:b]) for b in range(len(seqs) + 1)], dtype=torch.int32)
        logits = torch.empty(len(rows), self.cfg.vocab_size, dtype=self.logits_dtype, device=dev)
        nxt = torch.empty(len(rows), dtype=torch.int64, device=dev)
        binding = self.sess.io_binding()
        i32 = lambda v: torch.tensor(v, dtype=torch.int32).to(dev)  # noqa: E731
        cum, layout = starts, {}
        if self.has_trees:
            layout = dict(parents=i32(parents if parents is not None else [i - 1 for a, b in zip(starts, starts[1:]) for i in range(b - a)]))
        if self.has_layout:
            cum = [starts[b + 1] - starts[b] for b in range(len(seqs))]
            layout = dict(free=i32(self._granted(seqs, cum)), shared=i32([self.pool.common_tokens(seqs)]), used=i32([0]))
        self._bind(binding, ids.to(dev), i32(cum), past.to(dev), self._table(seqs).to(dev),
                   self._slots(seqs).to(dev), key_starts, torch.tensor(rows, dtype=torch.int64).to(dev), logits, nxt, **layout)
        self.sess.run_with_iobinding(binding, self._ro_prefill)
        for b, s in enumerate(seqs):
            self.pool.advance(s, starts[b + 1] - starts[b])
        if not self.has_argmax:
            nxt = logits.float().argmax(-1)
        return logits, nxt

    def _decode_buffers(self, rows: int) -> "_DecodeBuffers":
        if rows not in self._steps:
            buf = _DecodeBuffers(rows, self.blocks_per_seq, self.cfg.vocab_size, self.logits_dtype, self.device)
            buf.binding = self.sess.io_binding()
            self._bind(buf.binding, buf.ids, buf.new if self.has_layout else buf.cum, buf.past, buf.table, buf.slots, buf.key_starts, buf.rows, buf.logits, buf.next,
                       buf.free, buf.shared, buf.used, buf.parents)
            buf.options.add_run_config_entry("gpu_graph_id", str(self._graph_id + len(self._steps)))
            self._steps[rows] = buf
        return self._steps[rows]

    def _run_decode(self, buf: "_DecodeBuffers", seqs) -> None:
        """One token per sequence, ids already in ``buf.ids``; room has been reserved."""
        entries = [self.pool.sequences[s] for s in seqs]
        if self.has_layout:
            # New blocks reach the table in the step that enters them; another batch, or one that has moved since, has its table
            # sent.  (A sequence that was closed and opened again has another entry.)
            granted = self._granted(seqs, [1] * len(seqs))
            if granted:
                buf.free[:len(granted)].copy_(torch.tensor(granted, dtype=torch.int32))
            found = [e.length for e in entries]
            if buf.layout is None or any(a is not b for a, b in zip(buf.layout, entries)) or buf.tokens != found:
                buf.table.copy_(self._table(seqs))
                buf.slots.copy_(self._slots(seqs))
                buf.shared.fill_(self.pool.common_tokens(seqs))
                buf.layout = entries
            buf.tokens = [n + 1 for n in found]
        else:
            layout = [(s, e.slot, tuple(e.blocks)) for s, e in zip(seqs, entries)]
            if layout != buf.layout:
                buf.table.copy_(self._table(seqs))
                buf.slots.copy_(self._slots(seqs))
                buf.layout = layout
        lengths = [self.pool.sequences[s].length for s in seqs]
        if lengths.count(lengths[0]) == len(lengths):
            buf.past.fill_(lengths[0])
        else:
            buf.past.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.sess.run_with_iobinding(buf.binding, buf.options)
        for s in seqs:
            self.pool.advance(s, 1)
        if not self.has_argmax:
            buf.next.copy_(buf.logits.float().argmax(-1))

    # ------------------------------------------------------------------------------------------- the fixed batch of rows
    def _reopen_rows(self) -> None:
        for r in self._rows:
            if r in self.pool.sequences:
                self.release(r)
        for r in self._rows:
            self.pool.open(r)
        # full capacity at once, one block per row in turn: the block table of a row is fixed from here on, and no row owns
        # a contiguous range
        for j in range(self.blocks_per_seq):
            for r in self._rows:
                self.pool.reserve(r, min((j + 1) * self.block_size, self.max_len))

    def prefill(self, input_ids) -> torch.Tensor:
        """Prompts of the fixed batch: a tensor [B, S] or a list of B prompts of any lengths, packed without padding.
        Returns the first generated token of every row [B]."""
        prompts = [torch.as_tensor(p, dtype=torch.int64).reshape(-1) for p in input_ids]
        assert len(prompts) == self.batch and all(1 <= len(p) <= self.max_len for p in prompts)
        self._reopen_rows()
        starts = [0]
        for p in prompts:
            starts.append(starts[-1] + len(p))
        self.prefill_logits, nxt = self._run_packed(torch.cat(prompts), starts, self._rows, [s - 1 for s in starts[1:]])
        self._decode_buffers(self.batch).next.copy_(nxt)
        return nxt

    def assume_context(self, length: int) -> None:
        """Treat the caches as holding ``length`` tokens per sequence (benchmarks that time decode over a cache
        filled with arbitrary values instead of running a prompt first)."""
        assert 0 <= length < self.max_len
        if any(r not in self.pool.sequences for r in self._rows):
            self._reopen_rows()
        for r in self._rows:
            self.pool.sequences[r].length = length
            self._drafted.pop(r, None)

    def decode_step(self, tokens: Optional[torch.Tensor] = None) -> torch.Tensor:
        """One token per sequence; ``tokens`` [B] or None to feed back the previous step's output."""
        self._want_accepted(self._rows)
        buf = self._decode_buffers(self.batch)
        buf.ids.copy_(tokens.reshape(-1) if tokens is not None else buf.next, non_blocking=True)
        self._run_decode(buf, self._rows)
        self.step_logits = buf.logits
        return buf.next

    def reorder_cache(self, rows: torch.Tensor) -> None:
        """Row i takes the content of row rows[i] (beam search: beams follow their parents)."""
        self._want_accepted(self._rows)
        self.pool.copy_sequence_state([self._rows[int(r)] for r in rows.tolist()], self._rows)

    def generate(self, input_ids, max_new_tokens: int) -> torch.Tensor:
        out = [self.prefill(input_ids).clone()]
        for _ in range(max_new_tokens - 1):
            out.append(self.decode_step(out[-1]).clone())
        return torch.stack(out, dim=1)


class _DecodeBuffers:
    """Device buffers of the one-token step of one batch size; their addresses are frozen into its CUDA graph."""

    def __init__(self, rows: int, max_blocks: int, vocab: int, logits_dtype: torch.dtype, device: torch.device):
        self.ids = torch.zeros(rows, dtype=torch.int64, device=device)
        self.cum = torch.arange(rows + 1, dtype=torch.int32, device=device)
        self.past = torch.zeros(rows, dtype=torch.int32, device=device)
        self.table = torch.zeros(rows, max_blocks, dtype=torch.int32, device=device)
        self.slots = torch.zeros(rows, dtype=torch.int32, device=device)
        self.key_starts = torch.zeros(rows + 1, dtype=torch.int32)     # one-token steps read the cache as it lies
        self.rows = torch.arange(rows, dtype=torch.int64, device=device)
        self.logits = torch.zeros(rows, vocab, dtype=logits_dtype, device=device)
        self.next = torch.zeros(rows, dtype=torch.int64, device=device)
        self.new = torch.ones(rows, dtype=torch.int32, device=device)
        self.free = torch.zeros(rows, dtype=torch.int32, device=device)     # a token enters one new block at most
        self.shared = torch.zeros(1, dtype=torch.int32, device=device)
        self.used = torch.zeros(1, dtype=torch.int32, device=device)
        self.parents = torch.full((rows,), -1, dtype=torch.int32, device=device)
        self.layout = None
        self.tokens = None       # lengths that the next step of the same batch finds
        self.binding = None
        self.options = RunOptions()


# ----------------------------------------------------------------------------------------------------------------
# Logits processors, sampling and beam search on top of DecoderRunner.  The knobs are the attributes / inputs of the
# reference's generation operators (com.microsoft GreedySearch, Sampling, BeamSearch:
# onnxruntime/contrib_ops/cpu/transformers/{greedy_search.cc, sampling.cc, beam_search.cc, logits_processor.h});
# here the loop runs in Python over the session's bound decode step and all tensor work stays on the device.
class GenerationConfig:
    def __init__(self, max_new_tokens: int = 32, min_new_tokens: int = 0, eos_token_id: Optional[int] = None,
                 pad_token_id: int = 0, temperature: float = 1.0, top_k: int = 0, top_p: float = 1.0,
                 repetition_penalty: float = 1.0, no_repeat_ngram_size: int = 0, num_beams: int = 1,
                 length_penalty: float = 1.0, early_stopping: bool = False, num_return_sequences: int = 1,
                 vocab_mask: Optional[torch.Tensor] = None, seed: Optional[int] = None, logprobs: Optional[int] = None,
                 presence_penalty: float = 0.0, frequency_penalty: float = 0.0, logit_bias: Optional[Dict[int, float]] = None,
                 grammar: Optional[Callable[[List[int]], Optional[Sequence[int]]]] = None, draft_tokens: int = 0, draft_ngram: int = 3):
        """For ``generate_requests``: ``logprobs``: report log probabilities, entropies and that many best alternatives.
        ``presence_penalty`` and ``frequency_penalty`` are subtracted from the logits of generated tokens, once and as often as they
        occur; ``logit_bias`` is added to tokens' logits; ``grammar`` names the tokens that may follow the generated ones (None: all; what lies
        outside the vocabulary is no token), and is asked only about tokens that it has named.
        ``draft_tokens`` (runners with ``draft_trees``): up to so many tokens a step, and 255 at most, are drafted from what followed
        the last ``draft_ngram`` tokens, or fewer, earlier in the request's own text; the step keeps those that it would have chosen."""
        self.__dict__.update(locals())
        del self.__dict__["self"]


def process_logits(logits: torch.Tensor, sequences: torch.Tensor, step: int, cfg: GenerationConfig) -> torch.Tensor:
    """logits [rows, vocab] (fp32), sequences [rows, len] = every token so far (prompt included).  Order of the
    reference's LogitsProcessorList: min length, repetition penalty, no-repeat n-gram, vocabulary mask, temperature."""
    logits = logits.float().clone()
    if cfg.eos_token_id is not None and step < cfg.min_new_tokens:
        logits[:, cfg.eos_token_id] = float("-inf")
    if cfg.repetition_penalty != 1.0:
        seen = torch.gather(logits, 1, sequences)
        seen = torch.where(seen < 0, seen * cfg.repetition_penalty, seen / cfg.repetition_penalty)
        logits.scatter_(1, sequences, seen)
    n = cfg.no_repeat_ngram_size
    if n > 0 and sequences.shape[1] + 1 >= n:
        L = sequences.shape[1]
        if n == 1:
            logits.scatter_(1, sequences, float("-inf"))
        else:
            grams = sequences.unfold(1, n, 1)                      # [rows, L - n + 1, n]
            tail = sequences[:, L - (n - 1):].unsqueeze(1)          # [rows, 1, n - 1]
            hit = (grams[:, :, : n - 1] == tail).all(-1)            # n-grams whose prefix equals the current tail
            banned = torch.where(hit, grams[:, :, n - 1], torch.full_like(grams[:, :, n - 1], -1))
            rows = torch.arange(logits.shape[0], device=logits.device).unsqueeze(1).expand_as(banned)
            keep = banned >= 0
            logits[rows[keep], banned[keep]] = float("-inf")
    if cfg.vocab_mask is not None:
        logits = logits.masked_fill(cfg.vocab_mask.to(logits.device).view(1, -1) == 0, float("-inf"))
    if cfg.temperature != 1.0 and cfg.temperature > 0:
        logits = logits / cfg.temperature
    return logits


def top_k_top_p_filter(logits: torch.Tensor, top_k: int, top_p: float) -> torch.Tensor:
    if top_k > 0:
        kth = torch.topk(logits, min(top_k, logits.shape[-1]), dim=-1).values[:, -1:]
        logits = logits.masked_fill(logits < kth, float("-inf"))
    if top_p < 1.0:
        sorted_logits, idx = torch.sort(logits, descending=True, dim=-1)
        cum = torch.softmax(sorted_logits, -1).cumsum(-1)
        drop = cum - torch.softmax(sorted_logits, -1) > top_p       # keep the token that crosses the threshold
        sorted_logits = sorted_logits.masked_fill(drop, float("-inf"))
        logits = torch.full_like(logits, float("-inf")).scatter(1, idx, sorted_logits)
    return logits


def generate(runner: Union[DecoderRunner, PagedDecoderRunner], input_ids: torch.Tensor, cfg: GenerationConfig) -> torch.Tensor:
    """Greedy (``num_beams == 1``, ``top_k == 0``, ``top_p == 1``, temperature 1), sampling or beam search.
    Returns [batch * num_return_sequences, prompt + generated] token ids, padded with ``pad_token_id`` after EOS.
    For beam search the runner must have been created with ``batch = prompts * num_beams``."""
    for name in ("presence_penalty", "frequency_penalty", "logit_bias", "grammar", "draft_tokens"):
        if getattr(cfg, name):
            raise ValueError(f"{name} is an option of generate_requests()")
    if cfg.num_beams > 1:
        return _beam_search(runner, input_ids, cfg)
    dev = runner.device
    sampling = cfg.top_k > 0 or cfg.top_p < 1.0 or cfg.seed is not None
    gen = torch.Generator(device=dev)
    if cfg.seed is not None:
        gen.manual_seed(cfg.seed)
    seqs = input_ids.to(dev)
    done = torch.zeros(seqs.shape[0], dtype=torch.bool, device=dev)
    runner.prefill(input_ids)
    logits = _last_logits(runner, prefill=True)
    for step in range(cfg.max_new_tokens):
        scores = process_logits(logits, seqs, step, cfg)
        if sampling:
            probs = torch.softmax(top_k_top_p_filter(scores, cfg.top_k, cfg.top_p), -1)
            nxt = torch.multinomial(probs, 1, generator=gen).squeeze(1)
        else:
            nxt = scores.argmax(-1)
        nxt = torch.where(done, torch.full_like(nxt, cfg.pad_token_id), nxt)
        seqs = torch.cat([seqs, nxt.unsqueeze(1)], 1)
        if cfg.eos_token_id is not None:
            done = done | (nxt == cfg.eos_token_id)
            if bool(done.all()):
                break
        if step + 1 < cfg.max_new_tokens:
            runner.decode_step(nxt.view(-1, 1))
            logits = _last_logits(runner, prefill=False)
    return seqs


class LogitsProcessor:
    """The logits processors of ``generate_requests`` for all rows of a step at once: ``com.ortb200.ProcessLogits`` as a session of its
    own on the provider of the logits' device, with the inputs that the configuration needs.  ``vocab_mask`` is laid out when the
    processor is made."""

    def __init__(self, vocab_size: int, dtype: torch.dtype, device: torch.device, cfg: GenerationConfig):
        T, info = ol.TensorProto, ol.make_tensor_value_info
        kind = {torch.float32: T.FLOAT, torch.float16: T.FLOAT16, torch.bfloat16: T.BFLOAT16}[dtype]
        self.vocab_size, self.device, self.cfg = vocab_size, device, cfg
        self.text = cfg.repetition_penalty != 1.0 or cfg.presence_penalty != 0.0 or cfg.frequency_penalty != 0.0
        self.biased = (cfg.eos_token_id is not None and cfg.min_new_tokens > 0) or cfg.no_repeat_ngram_size > 0 or bool(cfg.logit_bias)
        self.masked = cfg.vocab_mask is not None or cfg.grammar is not None
        self.warm = cfg.temperature != 1.0 and cfg.temperature > 0
        self._vocab_words = None if cfg.vocab_mask is None else self._words((cfg.vocab_mask.reshape(-1).cpu() != 0).expand(vocab_size).numpy())
        self._vocab_mask = None if cfg.vocab_mask is None else torch.from_numpy(self._vocab_words.reshape(1, -1).copy()).to(device)
        self.idle = not (self.text or self.biased or self.masked or self.warm)
        ins = [info("logits", kind, ["rows", vocab_size])]
        names = ["logits"] + [""] * 14

        def add(place: int, name: str, onnx_type: int, shape) -> None:
            names[place] = name
            ins.append(info(name, onnx_type, shape))
        if self.text:
            for i, (name, shape) in enumerate((("history", ["total"]), ("history_starts", ["ends"]), ("generated_starts", ["lists"]))):
                add(1 + i, name, T.INT64, shape)
            add(4, "row_list", T.INT32, ["rows"])
            add(5, "drafted", T.INT64, ["rows", "depth"])
            for i, name in enumerate(("repetition", "presence", "frequency")):
                add(6 + i, name, T.FLOAT, ["rows"])
        if self.biased:
            add(9, "bias_tokens", T.INT64, ["biases"])
            add(10, "bias_values", T.FLOAT, ["biases"])
            add(11, "bias_starts", T.INT64, ["bias_ends"])
        if self.masked:
            add(12, "allowed", T.INT32, ["masks", (vocab_size + 31) // 32])
            add(13, "row_mask", T.INT32, ["rows"])
        if self.warm:
            add(14, "temperature", T.FLOAT, ["rows"])
        while not names[-1]:
            names.pop()
        graph = ol.make_graph([ol.make_node("ProcessLogits", names, ["scores"], domain="com.ortb200")], "logits", ins, [info("scores", T.FLOAT, ["rows", vocab_size])])
        gpu = device.type == "cuda"
        self.sess = None if self.idle else InferenceSession(
            ol.make_model(graph, opset=17, extra_opsets={"com.ortb200": 1}).serialize(),
            providers=[("CUDAExecutionProvider", {"device_id": str(device.index or 0)}) if gpu else "CPUExecutionProvider"])

    def _biases(self, text: Sequence[int], path: Sequence[int], generated: int) -> Dict[int, float]:
        """Of one row: a request's text, of which ``generated`` tokens are generated, and the drafted tokens behind it."""
        cfg, bias = self.cfg, dict(self.cfg.logit_bias or {})
        if cfg.eos_token_id is not None and generated + len(path) < cfg.min_new_tokens:
            bias[cfg.eos_token_id] = -math.inf
        n = cfg.no_repeat_ngram_size
        if n > 0:
            whole = np.concatenate([np.asarray(text, dtype=np.int64), np.asarray(path, dtype=np.int64)])
            if len(whole) >= n:
                bias.update(dict.fromkeys(whole[_places_of(whole[:-1], whole[len(whole) - (n - 1):])].tolist(), -math.inf))
        return bias

    def _words(self, keep: np.ndarray) -> np.ndarray:
        """A truth value for each token as bits of 32-bit words."""
        packed = np.zeros((self.vocab_size + 31) // 32 * 4, dtype=np.uint8)
        packed[:(self.vocab_size + 7) // 8] = np.packbits(keep, bitorder="little")
        return packed.view("<i4")

    def _masks(self, named: Sequence[Optional[Sequence[int]]]) -> Tuple[np.ndarray, List[int]]:
        """The different masks of rows for which a grammar names these tokens, and the mask of each row (-1: none)."""
        places: Dict[bytes, int] = {}
        rows = []
        for tokens in named:
            words = self._vocab_words
            if tokens is not None:
                tokens = _token_array(tokens)
                keep = np.zeros(self.vocab_size, dtype=bool)
                keep[tokens[(tokens >= 0) & (tokens < self.vocab_size)]] = True
                words = self._words(keep) if words is None else self._words(keep) & words
            rows.append(-1 if words is None else places.setdefault(words.tobytes(), len(places)))
        return np.frombuffer(bytearray(b"".join(places)), dtype="<i4").reshape(len(places), (self.vocab_size + 31) // 32), rows

    def __call__(self, logits: torch.Tensor, requests: Sequence[Tuple[Sequence[int], int, Sequence[Sequence[int]]]],
                 named: Optional[Sequence[Optional[Sequence[int]]]] = None) -> torch.Tensor:
        """logits [rows, vocab] -> scores [rows, vocab] in 32 bits.  ``requests``: (text, how many tokens of it are generated, for each of
        the request's rows the drafted tokens behind the text).  ``named``: what the grammar names for each row, where it has been asked."""
        if self.idle or not len(logits):
            return logits.float()
        cfg, dev, rows = self.cfg, self.device, logits.shape[0]
        ints = lambda v, t=torch.int64: torch.tensor(v, dtype=t).to(dev)  # noqa: E731
        same = lambda v: torch.full((rows,), v, dtype=torch.float32, device=dev)  # noqa: E731
        feeds = {"logits": logits}
        if self.text:
            starts, generated, lists = [0], [], []
            for i, (text, new, paths) in enumerate(requests):
                starts.append(starts[-1] + len(text))
                generated.append(starts[-1] - new)
                lists += [i] * len(paths)
            deepest = max(len(p) for _, _, paths in requests for p in paths)
            drafted = [list(p) + [-1] * (deepest - len(p)) for _, _, paths in requests for p in paths]
            feeds.update(history=torch.from_numpy(np.concatenate([np.asarray(text, dtype=np.int64) for text, _, _ in requests])).to(dev), history_starts=ints(starts), generated_starts=ints(generated), row_list=ints(lists, torch.int32),
                         drafted=ints(drafted).reshape(rows, deepest), repetition=same(cfg.repetition_penalty), presence=same(cfg.presence_penalty),
                         frequency=same(cfg.frequency_penalty))
        if self.biased:
            bias = [self._biases(text, p, new) for text, new, paths in requests for p in paths]
            ends = [0]
            for b in bias:
                ends.append(ends[-1] + len(b))
            feeds.update(bias_tokens=ints([t for b in bias for t in b]), bias_values=torch.tensor([v for b in bias for v in b.values()], dtype=torch.float32).to(dev), bias_starts=ints(ends))
        if self.masked:
            if cfg.grammar is None:
                feeds.update(allowed=self._vocab_mask, row_mask=torch.zeros(rows, dtype=torch.int32, device=dev))
            else:
                if named is None:
                    named = [cfg.grammar([int(t) for t in (*text[len(text) - new:], *p)]) for text, new, paths in requests for p in paths]
                masks, of_row = self._masks(named)
                feeds.update(allowed=torch.from_numpy(masks).to(dev), row_mask=ints(of_row, torch.int32))
        if self.warm:
            feeds.update(temperature=same(cfg.temperature))
        scores = torch.empty(rows, self.vocab_size, dtype=torch.float32, device=dev)
        binding = self.sess.io_binding()
        for name, t in feeds.items():
            binding.bind_torch_input(name, t)
        binding.bind_torch_output("scores", scores)
        self.sess.run_with_iobinding(binding)
        return scores


def draft_tree(text: Sequence[int], most: int, ngram: int = 3) -> Tuple[List[int], List[int]]:
    """A tree of the last token of ``text`` and up to ``most`` drafted ones: what followed earlier occurrences of the last ``ngram`` tokens, then
    of fewer; the latest occurrences first, 64 at most, and of each up to half as many tokens as there may be.  Returns the tokens and their parents."""
    text = np.asarray(text, dtype=np.int64)
    tokens, parents, children = [int(text[-1])], [-1], {}
    depth, end = max(1, (most + 1) // 2), len(text)
    for n in range(min(ngram, end - 1) if most > 0 else 0, 0, -1):
        for at in _places_of(text[:-1], text[end - n:])[:-65:-1].tolist():
            if len(tokens) > most:
                return tokens, parents
            node = 0
            for t in text[at:min(at + depth, end)].tolist():
                if (node, t) not in children:
                    if len(tokens) > most:
                        break
                    children[node, t] = len(tokens)
                    tokens.append(t)
                    parents.append(node)
                node = children[node, t]
    return tokens, parents


def _permitted(cfg: GenerationConfig, generated: Sequence[int], tokens: Sequence[int], parents: Sequence[int]):
    """Of a tree of drafted tokens behind ``generated`` those that can be chosen: tokens that the grammar names behind their parent, and no end
    token, behind which nothing is.  The grammar is so asked for texts alone that it allows.  Returns the tokens, their parents, and for each what
    the grammar names behind it (None: all)."""
    kept: Dict[int, int] = {}
    left, up, named, texts = [], [], [], []   # (texts: for a grammar)
    for j, (token, parent) in enumerate(zip(tokens, parents)):
        if parent >= 0:
            if parent not in kept or token == cfg.eos_token_id:
                continue
            if named[kept[parent]] is not None and not (named[kept[parent]] == token).any():
                continue
        kept[j] = len(left)
        left.append(token)
        up.append(kept[parent] if parent >= 0 else -1)
        if cfg.grammar is not None:
            texts.append([*texts[up[-1]], token] if parent >= 0 else [int(t) for t in generated])
        named.append(None if cfg.grammar is None else _token_array(cfg.grammar(list(texts[-1]))))
    return left, up, named


def _token_array(tokens: Optional[Sequence[int]]) -> Optional[np.ndarray]:
    if tokens is None:
        return None
    if isinstance(tokens, torch.Tensor):
        tokens = tokens.cpu().numpy()
    return np.asarray(tokens if isinstance(tokens, np.ndarray) else list(tokens), dtype=np.int64).reshape(-1)


def _places_of(text: np.ndarray, tail: np.ndarray) -> np.ndarray:
    """The places behind every occurrence of ``tail`` in ``text``, ascending (of an empty tail: all places of tokens and the one behind)."""
    starts = len(text) - len(tail) + 1
    found = np.ones(max(starts, 0), dtype=bool)
    for k, t in enumerate(tail):
        found &= text[k:starts + k] == t
    return np.flatnonzero(found) + len(tail)


class TokenScorer:
    """Log probabilities of chosen tokens, entropies and the ``top_k`` best alternatives out of logits:
    ``com.ortb200.TokenLogProbs`` as a session of its own on the provider of the logits' device."""

    def __init__(self, vocab_size: int, top_k: int, dtype: torch.dtype, device: torch.device):
        T = ol.TensorProto
        kind = {torch.float32: T.FLOAT, torch.float16: T.FLOAT16, torch.bfloat16: T.BFLOAT16}[dtype]
        info = ol.make_tensor_value_info
        outs = [info("log_prob", T.FLOAT, ["rows"]), info("entropy", T.FLOAT, ["rows"]), info("top_log_probs", T.FLOAT, ["rows", top_k]),
                info("top_tokens", T.INT64, ["rows", top_k])]
        graph = ol.make_graph([ol.make_node("TokenLogProbs", ["logits", "tokens"], [o.name for o in outs], domain="com.ortb200", top_k=top_k)], "scores",
                              [info("logits", kind, ["rows", vocab_size]), info("tokens", T.INT64, ["rows"])], outs)
        gpu = device.type == "cuda"
        self.sess = InferenceSession(ol.make_model(graph, opset=17, extra_opsets={"com.ortb200": 1}).serialize(),
                                     providers=[("CUDAExecutionProvider", {"device_id": str(device.index or 0)}) if gpu else "CPUExecutionProvider"])
        self.top_k, self.device = top_k, device

    def __call__(self, logits: torch.Tensor, tokens: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        """logits [rows, vocab], tokens [rows] -> log probabilities [rows], entropies [rows], and of the alternatives log
        probabilities and tokens [rows, top_k], the best first."""
        rows = logits.shape[0]
        outs = [torch.empty(s, dtype=d, device=self.device) for s, d in
                (((rows,), torch.float32), ((rows,), torch.float32), ((rows, self.top_k), torch.float32), ((rows, self.top_k), torch.int64))]
        binding = self.sess.io_binding()
        binding.bind_torch_input("logits", logits)
        binding.bind_torch_input("tokens", tokens.to(self.device))
        for name, t in zip(("log_prob", "entropy", "top_log_probs", "top_tokens"), outs):
            binding.bind_torch_output(name, t)
        self.sess.run_with_iobinding(binding)
        return tuple(outs)


@dataclass
class Generated:
    """A request's tokens and, for each, what the model thought of it: its log probability and the entropy of the distribution it
    comes from (before any logits processor), and the best alternatives."""
    tokens: List[int] = field(default_factory=list)
    log_probs: List[float] = field(default_factory=list)
    entropies: List[float] = field(default_factory=list)
    top_tokens: List[List[int]] = field(default_factory=list)
    top_log_probs: List[List[float]] = field(default_factory=list)


def score_requests(runner: PagedDecoderRunner, texts: Sequence[Sequence[int]], top_k: int = 0, shared_prompt: Sequence[int] = (),
                   rows: int = 1024) -> List[Generated]:
    """Log probabilities that the model gives to every token of ``texts`` but the first (with ``shared_prompt`` in front of all
    of them: to every token).  A text runs in portions of ``rows`` tokens at most, alone, behind the shared prompt's blocks."""
    scorer = TokenScorer(runner.cfg.vocab_size, top_k, runner.logits_dtype, runner.device)
    results = []
    prompt_logits = None
    try:
        if len(shared_prompt):
            prompt_logits = runner.step([(("shared prompt",), shared_prompt, [len(shared_prompt) - 1])]).clone()
        for i, text in enumerate(texts):
            text, seq, got = [int(t) for t in text], ("text", i), Generated()
            results.append(got)
            if not text:
                continue

            def note(logits: torch.Tensor, tokens: List[int]) -> None:
                lp, h, top_lp, top = (t.tolist() for t in scorer(logits, torch.tensor(tokens, dtype=torch.int64)))
                got.tokens += tokens
                got.log_probs += lp
                got.entropies += h
                got.top_log_probs += top_lp
                got.top_tokens += top
            if prompt_logits is not None:
                runner.fork(seq, ("shared prompt",))
                note(prompt_logits, text[:1])
            try:
                for start in range(0, len(text) - 1, rows):
                    portion = text[start:min(start + rows, len(text) - 1)]
                    note(runner.step([(seq, portion, range(len(portion)))]), text[start + 1:start + 1 + len(portion)])
            finally:
                if seq in runner.pool.sequences:
                    runner.release(seq)
    finally:
        if ("shared prompt",) in runner.pool.sequences:
            runner.release(("shared prompt",))
    return results


def generate_requests(runner: PagedDecoderRunner, prompts: Sequence[Sequence[int]], cfg: GenerationConfig,
                      shared_prompt: Sequence[int] = ()) -> Union[List[List[int]], List[Generated]]:
    """Greedy or sampled continuations of prompts of any lengths, with the processors and knobs of ``generate``.  At most
    ``runner.batch`` requests run at a time; a finished one frees its blocks and slot, and the next waiting prompt joins
    the running batch in a step of its own.  Returns the generated tokens of every request (end token included).

    ``shared_prompt`` stands in front of every prompt: it runs once, the requests share the cache blocks that it fills, and it
    takes one of the runner's sequences.  With ``cfg.logprobs`` the requests come back as ``Generated``.  With ``cfg.draft_tokens``
    a step may give a request several tokens.  Without sampling they are the same as without drafts, as far as rows of a tree and single rows
    round alike.  Sampled tokens have the same distribution; as all requests draw from one generator, a seed gives the same ones as without
    drafts only to a request that runs alone."""
    if cfg.draft_tokens < 0 or cfg.draft_ngram < 1:
        raise ValueError("draft_tokens is not negative, and draft_ngram positive")
    if cfg.draft_tokens and not runner.has_trees:
        raise ValueError("drafted tokens need a decoder with draft_trees")
    key = None
    if len(shared_prompt):
        if any(len(p) == 0 for p in prompts):
            raise ValueError("a request behind a shared prompt has a token of its own at least")
        if len(shared_prompt) > runner.max_len:
            raise CacheFull(f"the shared prompt exceeds {runner.max_len} tokens")
        key = ("shared prompt",)
        runner.step([(key, shared_prompt, [])])
    try:
        return _generate_requests(runner, prompts, cfg, [int(t) for t in shared_prompt], key)
    finally:
        for i in range(len(prompts)):   # of a call that was given up, or a grammar that raised: a later call starts anew
            if ("request", i) in runner.pool.sequences:
                runner.release(("request", i))
        if key is not None:
            runner.release(key)


def _generate_requests(runner: PagedDecoderRunner, prompts, cfg: GenerationConfig, shared: List[int], key):
    if cfg.num_beams > 1:
        raise ValueError("beam search needs a fixed batch: use generate()")
    sampling = cfg.top_k > 0 or cfg.top_p < 1.0 or cfg.seed is not None
    gen = torch.Generator(device=runner.device)
    if cfg.seed is not None:
        gen.manual_seed(cfg.seed)
    texts = [shared + [int(t) for t in p] for p in prompts]
    flat = [np.array(t + [0] * max(cfg.max_new_tokens, 1), dtype=np.int64) for t in texts]   # the same, and what is generated
    done: List[Optional[List[int]]] = [None] * len(texts)
    new: Dict[int, List[int]] = {}
    held_by_all = len(shared) // runner.block_size     # blocks that a request does not need for itself
    scorer = TokenScorer(runner.cfg.vocab_size, cfg.logprobs, runner.logits_dtype, runner.device) if cfg.logprobs is not None else None
    details = [Generated() for _ in texts]
    processor = LogitsProcessor(runner.cfg.vocab_size, runner.logits_dtype, runner.device, cfg)
    waiting, running = list(range(len(texts))), []

    def pick(i: int, logits: torch.Tensor, scores: torch.Tensor, best: int) -> int:
        """The request's next token out of a row of logits, noted; a request that is finished leaves."""
        tok = best
        if sampling:
            tok = int(torch.multinomial(torch.softmax(top_k_top_p_filter(scores.reshape(1, -1), cfg.top_k, cfg.top_p), -1), 1, generator=gen))
        flat[i][len(texts[i]) + len(new[i])] = tok
        new[i].append(tok)
        if scorer is not None:
            lp, h, top_lp, top = (t.tolist() for t in scorer(logits.reshape(1, -1), torch.tensor([tok], dtype=torch.int64)))
            d = details[i]
            d.tokens.append(tok)
            d.log_probs += lp
            d.entropies += h
            d.top_log_probs += top_lp
            d.top_tokens += top
        if len(new[i]) >= cfg.max_new_tokens or tok == cfg.eos_token_id:
            done[i] = new.pop(i)
            running.remove(i)
            runner.release(("request", i))
        return tok

    while waiting or running:
        joining = waiting[:min(runner.batch - len(running), len(runner.pool.free_slots))]
        while joining:   # prompts that fit into the free blocks together with the tokens they will generate
            room = len(runner.pool.free_blocks)
            need = [(len(texts[i]) + cfg.max_new_tokens + runner.block_size - 1) // runner.block_size - held_by_all for i in joining]
            held = sum(max(0, (len(texts[i]) + cfg.max_new_tokens + runner.block_size - 1) // runner.block_size
                           - len(runner.pool.sequences[("request", i)].blocks)) for i in running)
            if sum(need) + held <= room:
                break
            joining.pop()
        if joining:
            if key is not None:
                for i in joining:
                    runner.fork(("request", i), key)
            logits = runner.step([(("request", i), texts[i][len(shared):], [len(texts[i]) - len(shared) - 1]) for i in joining])
            waiting = waiting[len(joining):]
            running += joining
            for i in joining:
                new[i] = []
            trees = {i: _permitted(cfg, [], [-1], [-1]) for i in joining}   # a row for the last token of each
            drafted = False
        elif running:
            joining = list(running)
            # room has been kept for the tokens that a request will generate: no more of them are drafted
            trees = {i: draft_tree(flat[i][:len(texts[i]) + len(new[i])], min(cfg.draft_tokens, MOST_DRAFTED - 1, cfg.max_new_tokens - len(new[i]) - 1), cfg.draft_ngram) if cfg.draft_tokens else ([new[i][-1]], [-1])
                     for i in joining}
            trees = {i: _permitted(cfg, new[i], *tree) for i, tree in trees.items()}
            drafted = any(len(tokens) > 1 for tokens, _, _ in trees.values())
            if drafted:
                logits = runner.draft_step([(("request", i), *trees[i][:2], range(len(trees[i][0]))) for i in joining])
            else:
                logits = runner.step([(("request", i), [new[i][-1]], [0]) for i in joining])
        else:
            raise CacheFull(f"request {waiting[0]} does not fit into the cache")
        paths = {i: _paths(*trees[i][:2]) for i in joining}
        scores = processor(logits, [(flat[i][:len(texts[i]) + len(new[i])], len(new[i]), [[trees[i][0][j] for j in path[1:]] for path in paths[i]]) for i in joining],
                           [allowed for i in joining for allowed in trees[i][2]])
        best = [0] * len(scores) if sampling else scores.argmax(-1).tolist()
        row, kept = 0, {}
        for i in joining:   # from the root on, as far as the tree has what is chosen
            tokens, parents, _ = trees[i]
            node = 0
            while True:
                tok = pick(i, logits[row + node], scores[row + node], best[row + node])
                child = [j for j in range(node + 1, len(tokens)) if parents[j] == node and tokens[j] == tok]
                if i not in running or not child:
                    break
                node = child[0]
            if drafted and i in running:
                kept[("request", i)] = paths[i][node]
            row += len(tokens)
        if drafted:
            runner.accept(kept)
    return done if scorer is None else details


def _paths(tokens: Sequence[int], parents: Sequence[int]) -> List[List[int]]:
    """Of every token of a tree, the places from its root to it."""
    paths: List[List[int]] = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [i])
    return paths


def _last_logits(runner: DecoderRunner, prefill: bool) -> torch.Tensor:
    src = runner.prefill_logits if prefill else runner.step_logits
    return src.reshape(src.shape[0], -1).float()


def _beam_search(runner: DecoderRunner, input_ids: torch.Tensor, cfg: GenerationConfig) -> torch.Tensor:
    """Beam search with the scorer of the reference (beam_search_scorer.cc): hypotheses are ranked by
    sum(log p) / length ** length_penalty, 2 * num_beams candidates are examined per step so that finished beams
    can be replaced, and the KV cache rows follow their beams."""
    dev = runner.device
    B, K = input_ids.shape[0], cfg.num_beams
    assert runner.batch == B * K, "beam search needs a runner with batch = prompts * num_beams"
    seqs = input_ids.to(dev).repeat_interleave(K, 0)
    prompt_len = seqs.shape[1]
    runner.prefill(seqs)
    logits = _last_logits(runner, prefill=True)
    beam_scores = torch.zeros(B, K, device=dev)
    beam_scores[:, 1:] = -1e9                    # all beams of a prompt start identical: keep one alive
    finished: List[List[Tuple[float, torch.Tensor]]] = [[] for _ in range(B)]
    done = [False] * B
    V = logits.shape[-1]
    for step in range(cfg.max_new_tokens):
        logp = torch.log_softmax(process_logits(logits, seqs, step, cfg), -1)
        cand = (beam_scores.view(B * K, 1) + logp).view(B, K * V)
        top_scores, top_idx = torch.topk(cand, 2 * K, dim=1)
        src_beam, token = top_idx // V, top_idx % V
        new_scores = torch.full((B, K), -1e9, device=dev)
        new_src = torch.zeros(B, K, dtype=torch.long, device=dev)
        new_tok = torch.full((B, K), cfg.pad_token_id, dtype=torch.long, device=dev)
        ts, sb, tk = top_scores.tolist(), src_beam.tolist(), token.tolist()
        cur_len = seqs.shape[1] + 1 - prompt_len
        for b in range(B):
            if done[b]:
                continue
            filled = 0
            for rank in range(2 * K):
                if cfg.eos_token_id is not None and tk[b][rank] == cfg.eos_token_id:
                    if rank < K:   # only candidates that would have survived may finish
                        hyp = torch.cat([seqs[b * K + sb[b][rank]], torch.tensor([cfg.eos_token_id], device=dev)])
                        finished[b].append((ts[b][rank] / (cur_len ** cfg.length_penalty), hyp))
                    continue
                new_scores[b, filled], new_src[b, filled], new_tok[b, filled] = ts[b][rank], sb[b][rank], tk[b][rank]
                filled += 1
                if filled == K:
                    break
            if len(finished[b]) >= K:
                best_open = float(new_scores[b].max()) / (cur_len ** cfg.length_penalty)
                worst_kept = sorted(f[0] for f in finished[b])[-K]
                if cfg.early_stopping or worst_kept >= best_open:
                    done[b] = True
        rows = (torch.arange(B, device=dev).unsqueeze(1) * K + new_src).view(-1)
        seqs = torch.cat([seqs.index_select(0, rows), new_tok.view(-1, 1)], 1)
        beam_scores = new_scores
        if all(done):
            break
        if step + 1 < cfg.max_new_tokens:
            runner.reorder_cache(rows)
            runner.decode_step(new_tok.view(-1, 1))
            logits = _last_logits(runner, prefill=False)
    out = []
    gen_len = seqs.shape[1] - prompt_len
    for b in range(B):
        hyps = list(finished[b])
        for k in range(K):   # open beams count as hypotheses of the current length
            hyps.append((float(beam_scores[b, k]) / (max(gen_len, 1) ** cfg.length_penalty), seqs[b * K + k]))
        hyps.sort(key=lambda h: -h[0])
        out.extend(h[1] for h in hyps[: cfg.num_return_sequences])
    width = max(h.shape[0] for h in out)
    return torch.stack([torch.nn.functional.pad(h, (0, width - h.shape[0]), value=cfg.pad_token_id) for h in out])

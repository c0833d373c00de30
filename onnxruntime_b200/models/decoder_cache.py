"""Cache and state memory of packed decoders: pools of cache blocks and state slots shared by all sequences.

A model declares what it keeps per sequence as a list of ``CacheTensor``: "paged" tensors grow with the sequence and
live in blocks of ``block_size`` tokens named by a block table; "slot" tensors have a fixed size per sequence (recurrent
state) and live in one slot.  ``CachePool`` owns the device tensors and hands blocks and slots to sequences; the graph
updates both in place.  Slots are not cleared between owners: an operator starts from the zero state when a sequence's
past length is 0.  Sequences that begin with the same tokens share the blocks that these fill (``fork``); a block goes back
to the pool with its last owner.  Entries and blocks move in all paged tensors at once (``CacheMover``).
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import Dict, Hashable, List, Optional, Sequence, Tuple

import torch

from .. import onnx_lite as ol
from ..capi import InferenceSession


@dataclass(frozen=True)
class CacheTensor:
    input: str                    # graph input that receives the pool tensor
    output: str                   # graph output bound to the same tensor
    kind: str                     # "paged": [num_blocks, block_size, *shape]; "slot": [num_slots, *shape]
    shape: Tuple[int, ...]
    dtype: torch.dtype


class CacheFull(RuntimeError):
    """No free block or slot is left for a sequence."""


@dataclass
class SequenceEntry:
    slot: int
    blocks: List[int] = field(default_factory=list)
    length: int = 0


class CacheMover:
    """``com.ortb200.PagedCacheMove`` over given cache tensors, as a session of its own: one launch moves entries of tokens, or whole
    blocks, in all of them.  All sources are read before any target is written."""

    # bytes are moved, whatever type they are of: by the size of an element
    _TYPES = {1: (torch.uint8, ol.TensorProto.UINT8), 2: (torch.int16, ol.TensorProto.INT16), 4: (torch.int32, ol.TensorProto.INT32), 8: (torch.int64, ol.TensorProto.INT64)}

    def __init__(self, tensors: Sequence[torch.Tensor], whole_blocks: bool):
        self.tensors, self.device = list(tensors), tensors[0].device
        info = ol.make_tensor_value_info
        tensors = [torch.view_as_real(t) if t.is_complex() else t for t in tensors]
        types = [self._TYPES[t.element_size()] for t in tensors]
        tensors, kinds = [t.view(dtype) for t, (dtype, _) in zip(tensors, types)], [kind for _, kind in types]
        places = [info(n, ol.TensorProto.INT64, ["moves"]) for n in ("sources", "targets")]
        names = ["cache.%d" % i for i in range(len(tensors))]
        graph = ol.make_graph([ol.make_node("PagedCacheMove", ["sources", "targets"] + names, [n + ".out" for n in names], domain="com.ortb200", whole_blocks=int(whole_blocks))],
                              "move", places + [info(n, k, list(t.shape)) for n, k, t in zip(names, kinds, tensors)],
                              [info(n + ".out", k, list(t.shape)) for n, k, t in zip(names, kinds, tensors)])
        gpu = self.device.type == "cuda"
        self.sess = InferenceSession(ol.make_model(graph, opset=17, extra_opsets={"com.ortb200": 1}).serialize(),
                                     providers=[("CUDAExecutionProvider", {"device_id": str(self.device.index or 0)}) if gpu else "CPUExecutionProvider"])
        self.binding = self.sess.io_binding()
        for n, t in zip(names, tensors):
            self.binding.bind_torch_input(n, t)
            self.binding.bind_torch_output(n + ".out", t)

    def __call__(self, sources: Sequence[int], targets: Sequence[int]) -> None:
        moves = [(s, t) for s, t in zip(sources, targets) if s != t]
        if not moves:
            return
        both = torch.tensor(moves, dtype=torch.int64).t().contiguous().to(self.device)
        self.binding.bind_torch_input("sources", both[0])
        self.binding.bind_torch_input("targets", both[1])
        self.sess.run_with_iobinding(self.binding)


class CachePool:
    def __init__(self, spec: Sequence[CacheTensor], num_blocks: int, block_size: int, num_slots: int, device: torch.device):
        self.spec = list(spec)
        self.num_blocks, self.block_size, self.num_slots = num_blocks, block_size, num_slots
        # zero-filled once: attention kernels read whole tiles and multiply what lies beyond a sequence's end by zero, so
        # every entry has to be finite
        self.tensors = {c.input: torch.zeros((num_blocks, block_size, *c.shape) if c.kind == "paged" else (num_slots, *c.shape),
                                             dtype=c.dtype, device=device) for c in self.spec}
        self.free_blocks = list(range(num_blocks - 1, -1, -1))   # popped from the end: block 0 first, freed blocks first
        self.free_slots = list(range(num_slots - 1, -1, -1))
        self.sequences: Dict[Hashable, SequenceEntry] = {}
        self.owners: Dict[int, int] = {}                         # blocks of more than one sequence: how many
        self._movers: Dict[bool, CacheMover] = {}

    def _move(self, sources: Sequence[int], targets: Sequence[int], whole_blocks: bool) -> None:
        """Entries or blocks of the paged tensors to other places."""
        paged = [self.tensors[c.input] for c in self.spec if c.kind == "paged"]
        if not paged or not sources:
            return
        mover = self._movers.get(whole_blocks)
        if mover is None or any(a is not b for a, b in zip(mover.tensors, paged)):   # (another tensor may have taken one's place)
            self._movers[whole_blocks] = CacheMover(paged, whole_blocks)
        self._movers[whole_blocks](sources, targets)

    def open(self, seq: Hashable) -> SequenceEntry:
        if seq in self.sequences:
            raise ValueError(f"sequence {seq!r} is already open")
        if not self.free_slots:
            raise CacheFull(f"all {self.num_slots} sequence slots are in use")
        entry = SequenceEntry(self.free_slots.pop())
        self.sequences[seq] = entry
        return entry

    def fork(self, seq: Hashable, source: Hashable, tokens: Optional[int] = None) -> SequenceEntry:
        """Opens ``seq`` as a continuation of the first ``tokens`` (default: all) tokens of ``source``.  Blocks that these fill are
        shared, a block that they fill in part is copied; state in slots is copied, and has no memory of fewer tokens than all."""
        if seq in self.sequences:
            raise ValueError(f"sequence {seq!r} is already open")
        src = self.sequences[source]
        tokens = src.length if tokens is None else tokens
        if not 0 <= tokens <= src.length:
            raise ValueError(f"sequence {source!r} holds {src.length} tokens, not {tokens}")
        if tokens < src.length and any(c.kind == "slot" for c in self.spec):
            raise ValueError(f"the state of sequence {source!r} is that of all its {src.length} tokens")
        whole, rest = divmod(tokens, self.block_size)
        if rest and not self.free_blocks:
            raise CacheFull(f"sequence {seq!r} needs a cache block for a copy, none is free")
        entry = self.open(seq)
        entry.length = tokens
        entry.blocks = src.blocks[:whole]
        for block in entry.blocks:
            self.owners[block] = self.owners.get(block, 1) + 1
        if rest:
            entry.blocks.append(self.free_blocks.pop())
        if rest:
            self._move([src.blocks[whole]], [entry.blocks[-1]], True)
        for c in self.spec:
            if c.kind == "slot":
                t = self.tensors[c.input]
                t[entry.slot].copy_(t[src.slot])
        return entry

    def keep(self, chosen: Dict[Hashable, Tuple[int, Sequence[int]]]) -> None:
        """Of the tokens behind the first ``held`` of a sequence, only those at the places ``path`` (ascending, counted from
        ``held``), which close up: ``chosen`` names (held, path) for each sequence.  Blocks that several sequences share are not
        written, now or by the tokens that follow, and state in slots has no memory of fewer tokens than all."""
        sources, targets = [], []
        for seq, (held, path) in chosen.items():
            entry = self.sequences[seq]
            if not 0 <= held <= held + len(path) <= entry.length or any(not 0 <= p < entry.length - held for p in path) or any(a >= b for a, b in zip(path, path[1:])):
                raise ValueError(f"sequence {seq!r} holds no such tokens")
            if held + len(path) == entry.length:
                continue
            if any(b in self.owners for b in entry.blocks[held // self.block_size:]):
                raise ValueError(f"sequence {seq!r}: blocks that several sequences share are not written")
            if any(c.kind == "slot" for c in self.spec):
                raise ValueError(f"the state of sequence {seq!r} is that of all its {entry.length} tokens")
        for seq, (held, path) in chosen.items():
            entry = self.sequences[seq]
            place = lambda t: entry.blocks[t // self.block_size] * self.block_size + t % self.block_size  # noqa: E731, B023
            sources += [place(held + p) for p in path]
            targets += [place(held + i) for i in range(len(path))]
            entry.length = held + len(path)
        self._move(sources, targets, False)

    def common_tokens(self, seqs: Sequence[Hashable]) -> int:
        """How many leading tokens of all ``seqs`` lie in the same blocks."""
        entries = [self.sequences[s] for s in seqs]
        blocks = 0
        for column in zip(*(e.blocks for e in entries)):
            if any(b != column[0] for b in column):
                break
            blocks += 1
        return min([blocks * self.block_size] + [e.length for e in entries]) if entries else 0

    def reserve(self, seq: Hashable, tokens: int) -> bool:
        """Room for ``tokens`` more tokens of ``seq``; True when blocks were added.  All or nothing."""
        entry = self.sequences[seq]
        need = (entry.length + tokens + self.block_size - 1) // self.block_size - len(entry.blocks)
        if need > len(self.free_blocks):
            raise CacheFull(f"sequence {seq!r} needs {need} more cache blocks, {len(self.free_blocks)} are free")
        for _ in range(max(need, 0)):
            entry.blocks.append(self.free_blocks.pop())
        return need > 0

    def advance(self, seq: Hashable, tokens: int) -> None:
        self.sequences[seq].length += tokens

    def close(self, seq: Hashable) -> None:
        entry = self.sequences.pop(seq)
        for block in reversed(entry.blocks):
            left = self.owners.pop(block, 1) - 1
            if left == 0:
                self.free_blocks.append(block)
            elif left > 1:
                self.owners[block] = left
        self.free_slots.append(entry.slot)

    def copy_sequence_state(self, sources: Sequence[Hashable], targets: Sequence[Hashable]) -> None:
        """Content of ``targets[i]`` becomes that of ``sources[i]`` (beam search); all open, with equally many blocks."""
        src, dst = [self.sequences[s] for s in sources], [self.sequences[t] for t in targets]
        if any(b in self.owners for e in dst for b in e.blocks):
            raise ValueError("blocks that several sequences share are not written")
        src_blocks = [b for e in src for b in e.blocks]
        dst_blocks = [b for e in dst for b in e.blocks]
        if any(len(a.blocks) != len(b.blocks) for a, b in zip(src, dst)):
            raise ValueError("sequences hold different numbers of blocks")
        lengths = [e.length for e in src]
        self._move(src_blocks, dst_blocks, True)
        for c in self.spec:
            if c.kind == "slot":
                t = self.tensors[c.input]
                a, b = (torch.tensor([e.slot for e in entries], device=t.device) for entries in (src, dst))
                t.index_copy_(0, b, t.index_select(0, a))
        for e, n in zip(dst, lengths):
            e.length = n

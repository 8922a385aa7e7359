"""A paged KV cache in fp32, fp16 or INT8, and attention of new tokens over it.

The reference keeps no cache: ``generate`` recomputes the whole prefix for
every token (generate.py:313-315).  ``KVCache`` (model.py) holds sequences of
one length in one fp32 block per layer.  Here sequences of any length share a
pool of pages, so a serving program can add, extend and drop them one by one:

* ``PagedKV``      one layer's pages (a key or value of a head is 24 values:
                   fp32, fp16, or INT8 codes with an fp32 scale of their own);
* ``PagedBatch``   what a step brings: how many new tokens of which sequences,
                   and in which pages those live;
* ``paged_write``  the new tokens' keys (normalised by ``k_ln``) and values
                   quantised into their slots; ``paged_read`` back to fp32;
* ``paged_attention``  causal attention of the new tokens, one per sequence,
                   chunks of prompts or both in one step, over the pages
                   (PolluxCausalAttention, pollux.py:613-626, with q_ln fused);
* ``PagedKVCache`` every layer's pages, with the sequences' tables and the
                   free pages kept on the host.

Inference only: no entry point records a gradient.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass, field
from typing import Sequence

import torch

from . import _lib
from .castor import H24_DIM

_X_TYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_KV_TYPES = {torch.float32: _lib.KV_F32, torch.float16: _lib.KV_F16, torch.int8: _lib.KV_INT8}


@dataclass(frozen=True)
class PagedKV:
    """One layer's pages: k, v [pages, heads, page_size, 24] (fp32, fp16 or int8), for int8 with fp32 scales
    [pages, heads, page_size].  page_size is a power of two from 8 to 4,096."""

    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor | None = None
    v_scale: torch.Tensor | None = None
    _c: _lib.PagedKVStruct = field(init=False, repr=False, compare=False)
    _index: int = field(init=False, repr=False, compare=False)  # the device's

    def __post_init__(self) -> None:
        k = self.k
        if k.dim() != 4 or k.shape[3] != H24_DIM or k.dtype not in _KV_TYPES:
            raise ValueError("PagedKV: pages are [pages, heads, page_size, 24] in float32, float16 or int8")
        size = k.shape[2]
        if not 8 <= size <= 4096 or size & (size - 1):
            raise ValueError(f"PagedKV: page size {size} is not a power of two from 8 to 4096")
        if k.shape[0] < 1 or k.shape[1] < 1:
            raise ValueError("PagedKV needs at least one page and one head")
        scales = (self.k_scale, self.v_scale)
        if (k.dtype == torch.int8) != all(s is not None for s in scales) or (scales[0] is None) != (scales[1] is None):
            raise ValueError("PagedKV: int8 pages come with both scales, others with none")
        for name, t, shape, dtype in (("k", k, k.shape, k.dtype), ("v", self.v, k.shape, k.dtype),
                                      ("k_scale", scales[0], k.shape[:3], torch.float32),
                                      ("v_scale", scales[1], k.shape[:3], torch.float32)):
            if t is None:
                continue
            _lib.require_device(t, f"PagedKV {name}")
            if t.shape != shape or t.dtype != dtype or t.device != k.device or not t.is_contiguous():
                raise ValueError(f"PagedKV: {name} must be contiguous {dtype} of shape {tuple(shape)} on {k.device}")
        object.__setattr__(self, "_c", _lib.PagedKVStruct(
            _lib.ptr(k), _lib.ptr(self.v), _lib.ptr(scales[0]), _lib.ptr(scales[1]), k.shape[0], k.shape[1], size,
            _KV_TYPES[k.dtype]))
        object.__setattr__(self, "_index", k.get_device())

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int, kv_dtype: torch.dtype, device) -> PagedKV:
        # uninitialised: a position is only ever read after it is written (positions < its sequence's length)
        shape = (pages, heads, page_size, H24_DIM)
        k, v = (torch.empty(shape, dtype=kv_dtype, device=device) for _ in range(2))
        if kv_dtype != torch.int8:
            return cls(k, v)
        return cls(k, v, *(torch.empty(shape[:3], dtype=torch.float32, device=device) for _ in range(2)))

    @property
    def heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]


@dataclass(frozen=True)
class PagedBatch:
    """The new tokens of a step, as rows of one flat [tokens, ...] array.

    Rows cu_q[r] .. cu_q[r + 1] - 1 are sequence r's, the last of its
    kv_len[r] positions; position j lies in page table[r, j // page_size].
    The tensors (int32) are read on the device when a kernel runs, so a
    captured graph may be replayed on new contents; the host's numbers bound
    them: tokens in all, max_q new tokens and max_kv positions of a sequence.
    Contents outside those bounds, or a page outside the cache, write nothing
    and give NaN outputs.  ``singles``: how many sequences are known to bring
    one token beside others that bring more (they then take the one-token kernel).
    ``order`` (int32, a permutation of the sequences): attention begins with its
    first ones; its last ``singles``, beside others that bring more, must
    bring one token at most (NaN outputs otherwise).
    """

    table: torch.Tensor
    cu_q: torch.Tensor
    kv_len: torch.Tensor
    tokens: int
    max_q: int
    max_kv: int
    singles: int = 0
    order: torch.Tensor | None = None
    _c: _lib.PagedBatchStruct = field(init=False, repr=False, compare=False)
    _index: int = field(init=False, repr=False, compare=False)
    _needs: dict = field(init=False, repr=False, compare=False)  # (heads, cache type) -> workspace bytes

    def __post_init__(self) -> None:
        seqs = self.kv_len.shape[0] if self.kv_len.dim() == 1 else -1
        if seqs < 0 or self.table.dim() != 2 or self.table.shape[0] != seqs or tuple(self.cu_q.shape) != (seqs + 1,):
            raise ValueError("PagedBatch: table [seqs, pages], cu_q [seqs + 1], kv_len [seqs]")
        if self.order is not None and tuple(self.order.shape) != (seqs,):
            raise ValueError("PagedBatch: order [seqs]")
        for name, t in (("table", self.table), ("cu_q", self.cu_q), ("kv_len", self.kv_len), ("order", self.order)):
            if t is None:
                continue
            _lib.require_device(t, f"PagedBatch {name}")
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.table.device:
                raise ValueError(f"PagedBatch: {name} must be contiguous int32 on one device")
        if min(self.tokens, self.max_q, self.max_kv, self.singles) < 0:
            raise ValueError("PagedBatch: negative bounds")
        object.__setattr__(self, "_c", _lib.PagedBatchStruct(
            _lib.ptr(self.table), self.table.shape[1], seqs, _lib.ptr(self.cu_q), _lib.ptr(self.kv_len), self.tokens,
            self.max_q, self.max_kv, self.singles, _lib.ptr(self.order)))
        object.__setattr__(self, "_index", self.table.get_device())
        object.__setattr__(self, "_needs", {})

    @classmethod
    def build(cls, table: torch.Tensor | Sequence[Sequence[int]], kv_lens: Sequence[int], q_lens: Sequence[int],
              device=None) -> PagedBatch:
        """The batch of sequences of kv_lens positions, of which the last q_lens are this step's.

        table: int32 [seqs, pages] on the device, or each sequence's list of pages (then ``device`` says where;
        positions past the end of a list have no page).
        """
        if len(kv_lens) != len(q_lens) or len(table) != len(kv_lens):
            raise ValueError("PagedBatch.build: one table row, length and number of new tokens per sequence")
        if any(q < 0 for q in q_lens) or any(n < 0 for n in kv_lens):
            raise ValueError("PagedBatch.build: negative lengths")
        starts = [0]
        for n in q_lens:
            starts.append(starts[-1] + n)
        seqs, top = len(kv_lens), max(q_lens, default=0)
        # those that bring more than one token first, and of either kind the most work
        order = sorted(range(seqs), key=lambda r: (q_lens[r] > 1, q_lens[r] * kv_lens[r]), reverse=True)
        small = [*starts, *kv_lens, *order]
        if isinstance(table, torch.Tensor):
            device = table.device
            table = table.to(torch.int32).contiguous()
            small = torch.tensor(small, dtype=torch.int32).to(device)
        else:  # the rows, starts, lengths and order in one copy
            width = max((len(t) for t in table), default=0)
            # (-1 is no page: a list that ends before its sequence does is read as NaN and written nowhere)
            rows = [p for t in table for p in (*t, *([-1] * (width - len(t))))]
            both = torch.tensor([*rows, *small], dtype=torch.int32).to(device)
            table, small = both[:seqs * width].view(seqs, width), both[seqs * width:]
        return cls(table, small[:seqs + 1], small[seqs + 1:2 * seqs + 1], starts[-1], top, max(kv_lens, default=0),
                   sum(n <= 1 for n in q_lens) if top > 1 else 0, small[2 * seqs + 1:])


def _rows(name: str, x: torch.Tensor, kv: PagedKV, batch: PagedBatch) -> torch.Tensor:
    """x as [rows, heads * 24] on the pages' device, with the batch's rows at least."""
    c = kv._c.heads * H24_DIM
    if x.dtype not in _X_TYPES:
        raise ValueError(f"{name} must be float32, float16 or bfloat16")
    if x.dim() < 2 or x.shape[-1] != c:
        raise ValueError(f"{name} must have rows of {c} values ({kv.heads} heads), got {tuple(x.shape)}")
    if x.dim() > 2:
        x = x.reshape(-1, c)
    if x.shape[0] < batch.tokens:
        raise ValueError(f"{name} has {x.shape[0]} rows for the batch's {batch.tokens} tokens")
    if x.get_device() != kv._index or batch._index != kv._index:
        _lib.require_device(x, name)
        raise ValueError(f"{name}, the batch and the pages must be on one device")
    return x


def _strided(x: torch.Tensor) -> torch.Tensor:
    """x with rows as the kernels read them: 16-byte pieces, rows a multiple of 8 elements apart."""
    row, step = x.stride()
    if step == 1 and row >= x.shape[1] and row % 8 == 0 and x.data_ptr() % 16 == 0:
        return x
    x = x.contiguous()
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _norm(name: str, ln, index: int) -> tuple[int | None, float]:
    """The address of a norm's weight (held by the module) and its epsilon."""
    if ln is None:
        return None, 0.0
    w = ln.weight
    if w.dtype != torch.float32 or w.dim() != 1 or w.shape[0] != H24_DIM or w.get_device() != index or w.stride(0) != 1:
        raise ValueError(f"{name}: the norm's weight must be contiguous float32 [24] on the pages' device")
    return w.data_ptr(), ln.eps


def paged_write(k: torch.Tensor, v: torch.Tensor, kv: PagedKV, batch: PagedBatch, k_ln=None) -> None:
    """The new tokens' keys (through ``k_ln``, an RMSNorm, if given) and values into their slots (plx_paged_write).

    k, v: [tokens, heads * 24] projections (fp32, fp16 or bf16; column slices of
    one stacked projection are read in place).  INT8 slots: per key and value of
    a head code = rint(x * (127 / max|x|)) and scale = max|x| / 127; one with a
    NaN or an infinity reads back as NaN.
    """
    kk, vv = _rows("paged_write k", k, kv, batch), _rows("paged_write v", v, kv, batch)
    if kk.dtype != vv.dtype:
        raise ValueError("paged_write: k and v of one dtype")
    kk, vv = _strided(kk), _strided(vv)
    if kk.stride(0) != vv.stride(0):
        kk, vv = _strided(kk.contiguous()), _strided(vv.contiguous())
    w, eps = _norm("paged_write", k_ln, kv._index)
    device = kv.k.device
    with _lib.on_device(device):
        st = _lib.lib().plx_paged_write(ctypes.byref(kv._c), ctypes.byref(batch._c), kk.data_ptr(), vv.data_ptr(),
                                        _X_TYPES[kk.dtype], kk.stride(0) if kk.shape[0] > 1 else 0, w, eps,
                                        _lib.stream_of(device))
    _lib.check(st, "paged_write")


def paged_read(kv: PagedKV, batch: PagedBatch) -> tuple[torch.Tensor, torch.Tensor]:
    """What the slots of the batch's tokens hold: (keys, values), fp32 [tokens, heads * 24] (plx_paged_read).

    A batch whose sequences bring all their positions (q_lens = kv_lens) reads them whole.
    Rows that cu_q gives to no sequence are not written: they hold anything.
    """
    if batch._index != kv._index:
        raise ValueError("paged_read: the batch and the pages must be on one device")
    device = kv.k.device
    k, v = torch.empty(2, batch.tokens, kv._c.heads * H24_DIM, dtype=torch.float32, device=device).unbind()
    with _lib.on_device(device):
        st = _lib.lib().plx_paged_read(ctypes.byref(kv._c), ctypes.byref(batch._c), k.data_ptr(), v.data_ptr(),
                                       _lib.stream_of(device))
    _lib.check(st, "paged_read")
    return k, v


def paged_attention(q: torch.Tensor, kv: PagedKV, batch: PagedBatch, q_ln=None,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """Causal attention of the batch's new tokens over the pages, which hold them already (plx_paged_attention).

    q: [tokens, heads * 24] projections, normalised by ``q_ln`` (an RMSNorm) if
    given; returns the same shape and dtype (into ``out`` if given, which must
    not overlap q).  A token
    sees its sequence's positions up to its own; one before position 0 (a
    sequence shorter than its new tokens) sees none and gives zeros.  Rows past
    the batch's tokens are left as they are in ``out``, and zeros without it;
    rows among them that cu_q gives to no sequence are not written.
    """
    qq = _strided(_rows("paged_attention q", q, kv, batch))
    w, eps = _norm("paged_attention", q_ln, kv._index)
    device = kv.k.device
    if out is None:
        make = torch.empty if qq.shape[0] == batch.tokens else torch.zeros
        out = make(q.shape, dtype=q.dtype, device=device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.device != device or not out.is_contiguous():
        raise ValueError("paged_attention: out must be contiguous, of q's shape, dtype and device")
    key = (kv._c.heads, kv._c.kv_type)
    with _lib.on_device(device):
        lib, kc, bc = _lib.lib(), ctypes.byref(kv._c), ctypes.byref(batch._c)
        need = batch._needs.get(key)
        if need is None:
            need = batch._needs[key] = lib.plx_paged_attention_workspace_bytes(kc, bc)
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        st = lib.plx_paged_attention(kc, bc, qq.data_ptr(), _X_TYPES[qq.dtype], qq.stride(0) if qq.shape[0] > 1 else 0,
                                     w, eps, out.data_ptr(), _lib.ptr(ws), need, _lib.stream_of(device))
    _lib.check(st, "paged_attention")
    return out


@dataclass(frozen=True)
class PagedStep:
    """A step's batch on every layer's pages: what a model's blocks take in place of a KVCache."""

    layers: Sequence[PagedKV]
    batch: PagedBatch


class PagedKVCache:
    """Every layer's pages; the sequences' page tables, their lengths and the free pages, on the host.

    ``add`` opens a sequence, ``extend`` makes room for a step's new tokens and
    returns the step, ``drop`` closes a sequence and frees its pages.  All
    layers use one table, so a page stands for the same positions in each.
    """

    def __init__(self, layers: Sequence[PagedKV]) -> None:
        if not layers:
            raise ValueError("PagedKVCache needs at least one layer")
        if any(kv.k.shape[:3] != layers[0].k.shape[:3] or kv.k.device != layers[0].k.device for kv in layers):
            raise ValueError("PagedKVCache: every layer has the same pages, heads and page size, on one device")
        self.layers = list(layers)
        self.page_size = layers[0].page_size
        self._free = list(range(layers[0].k.shape[0] - 1, -1, -1))
        self._tables: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0

    @classmethod
    def allocate(cls, cfg, pages: int, device, *, page_size: int = 64, kv_dtype: torch.dtype = torch.int8) -> PagedKVCache:
        """``pages`` pages of ``page_size`` positions for each of a PolluxConfig's layers."""
        if int(cfg.d_head) != H24_DIM:
            raise ValueError(f"PagedKVCache: heads of {cfg.d_head} values (the pages hold {H24_DIM})")
        return cls([PagedKV.allocate(pages, int(cfg.n_heads), page_size, kv_dtype, device)
                    for _ in range(int(cfg.n_layers))])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _known(self, *seqs: int) -> None:
        if any(s not in self._tables for s in seqs):
            raise ValueError("PagedKVCache: no such sequence")

    def length(self, seq: int) -> int:
        """Positions that sequence ``seq`` holds."""
        self._known(seq)
        return self._lengths[seq]

    def add(self) -> int:
        """A new, empty sequence's number."""
        seq, self._next = self._next, self._next + 1
        self._tables[seq], self._lengths[seq] = [], 0
        return seq

    def drop(self, seq: int) -> None:
        """Closes ``seq``; its pages are free for others (work already enqueued on this stream may still read them)."""
        self._known(seq)
        self._free.extend(reversed(self._tables.pop(seq)))
        del self._lengths[seq]

    def extend(self, seqs: Sequence[int], counts: Sequence[int]) -> PagedStep:
        """The step that appends counts[i] tokens to sequence seqs[i]; nothing changes if the free pages do not suffice."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs):
            raise ValueError("PagedKVCache.extend: one count per sequence, every sequence once")
        if any(n < 1 for n in counts):
            raise ValueError("PagedKVCache.extend: at least one new token per sequence")
        self._known(*seqs)
        size = self.page_size
        lengths = [self._lengths[s] + n for s, n in zip(seqs, counts)]
        need = [-(-t // size) - len(self._tables[s]) for s, t in zip(seqs, lengths)]
        if sum(need) > len(self._free):
            raise ValueError(f"PagedKVCache: {sum(need)} pages needed, {len(self._free)} free")
        for s, t, n in zip(seqs, lengths, need):
            self._tables[s].extend(self._free.pop() for _ in range(n))
            self._lengths[s] = t
        batch = PagedBatch.build([self._tables[s] for s in seqs], lengths, list(counts), self.layers[0].k.device)
        return PagedStep(self.layers, batch)

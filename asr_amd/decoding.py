"""Decoding with beams: the operators around the decoder's own layers.

The reference decodes through HF ``generate`` (src/modeling.py:329-334), whose beam search keeps one bf16 cache per beam
and moves all of it at every step.  Here

* ``beam_select`` picks the best continuations over beams and vocabulary on the device,
* ``PagedKVCache`` holds keys and values in 8 bits on pages of 64 tokens that beams share; a change of beams only moves
  page numbers (``reorder``), and a page is copied when two beams that share it both go on (``extend``),
* ``PagedKVCache.attend`` is the attention over it, for prompts and for single tokens; pages that the beams of an
  utterance share (its whole audio prompt) are read once for all of them,
* ``reorder_states`` moves any other per-beam state.

``asr_amd.evaluation.beam_generate`` is the loop that uses them together.  Nothing here synchronises with the host (but
``PagedKVCache.check``), so a step can be captured into a HIP graph.  All of it is for inference: no gradients.  Runs in
libasrk.so; there is no CPU path.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Dict, List, NamedTuple, Optional, Tuple, Union

import torch

from . import _lib

_DT = {torch.float32: _lib.ASRK_F32, torch.bfloat16: _lib.ASRK_BF16}
PAGE = _lib.KV_PAGE
MAX_BEAMS = 16


class BeamStep(NamedTuple):
    """One step of a beam search over B utterances on K beams."""

    scores: torch.Tensor  # f32 [B, K]: log-probabilities of the beams that go on, best first
    tokens: torch.Tensor  # int64 [B, K]: their new tokens
    parents: torch.Tensor  # int64 [B, K]: the beams (0 .. K-1 of the same utterance) they continue
    cand_scores: torch.Tensor  # f32 [B, 2K]: the best 2K continuations, those that end the utterance among them
    cand_tokens: torch.Tensor
    cand_parents: torch.Tensor


def _call(name: str, device: torch.device, *args) -> None:
    """One entry point of libasrk.so on the current stream of ``device`` (a step makes hundreds of calls: no context manager
    and no Stream object where the device is current anyway)."""
    fn = getattr(_lib.load(), name)
    if torch.cuda.current_device() == device.index:
        rc = fn(*args, _lib.stream_of(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _lib.stream_of(device))
    if rc:
        _lib.check(rc, name)


def _address(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _gpu(name: str, *tensors: torch.Tensor) -> torch.device:
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise _lib.AsrkError(f"{name} runs on a ROCm GPU only (there is no CPU fallback)")
        if t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")
        if t.requires_grad and torch.is_grad_enabled():
            raise ValueError(f"{name} has no backward: call it under torch.no_grad() or detach its inputs")
    return dev


@functools.lru_cache(maxsize=64)
def _select_workspace(B: int, K: int, V: int) -> int:
    return _lib.load().asrk_beam_select_workspace_bytes(B, K, V)


def beam_select(logits: torch.Tensor, scores: torch.Tensor, eos_token_id: Optional[int] = None) -> BeamStep:
    """The best 2K of the K * V continuations of every utterance, and the first K of them that go on.

    ``logits`` [B*K, V] or [B, K, V] (float32 or bfloat16; rows may lie at any stride, as those of a padded output layer
    or of the last position of a longer run), ``scores`` float32 [B, K] (-inf: no beam).  A continuation's value is
    ``scores[b, k] + log_softmax(logits[b, k])[v]``, ordered best first, ties to the lowest ``k * V + v`` (values are
    compared in 64 bits; of two words of one beam the larger logit is ahead even where 64 bits cannot tell them apart).  -inf
    logits are words that cannot follow.  A beam whose score or largest logit is not finite, or that has a NaN logit, offers only
    -inf.  Continuations with ``eos_token_id`` are among the 2K candidates but do not go on.  1 <= K <= 16, V >= 2."""
    if scores.dim() != 2 or scores.dtype != torch.float32:
        raise ValueError("scores must be a float32 [B, K] tensor")
    B, K = scores.shape
    if logits.dim() == 3 and tuple(logits.shape[:2]) == (B, K):
        V = logits.shape[2]
        if logits.stride(0) != K * logits.stride(1) and B > 1 or logits.stride(2) != 1:
            logits = logits.contiguous()
        ld = logits.stride(1) if K > 1 else logits.stride(0)
    elif logits.dim() == 2 and logits.shape[0] == B * K:
        V = logits.shape[1]
        if logits.stride(1) != 1:
            logits = logits.contiguous()
        ld = logits.stride(0)
    else:
        raise ValueError("logits must be [B * K, V] or [B, K, V] for scores [B, K]")
    if logits.dtype not in _DT:
        raise ValueError("logits must be float32 or bfloat16")
    if not 1 <= K <= MAX_BEAMS or V < 2:
        raise ValueError(f"beam_select takes 1 to {MAX_BEAMS} beams and at least 2 words, got {K} and {V}")
    if B * K > 65535 or K * V > 0x7FFFFFFF or K * (-(-V // 8192)) > 2048:
        raise ValueError(f"beam_select: {B} x {K} beams over {V} words are more than one call takes")
    eos = -1 if eos_token_id is None else int(eos_token_id)
    dev = _gpu("beam_select", logits, scores)
    scores = scores.contiguous()
    if ld < V:  # a single row, or rows that overlap
        logits, ld = logits.contiguous(), V
    # six tensors in one allocation (an as_strided is 0.8 us, an allocation 1.4): 6 B K integers, then 3 B K floats
    ints, m = scores.new_empty((8 * B * K,), dtype=torch.int64), B * K
    floats = ints.view(torch.float32)
    one, two, ones, twos = (B, K), (B, 2 * K), (K, 1), (2 * K, 1)
    out = (floats.as_strided(one, ones, 12 * m), ints.as_strided(one, ones, 0), ints.as_strided(one, ones, m),
           floats.as_strided(two, twos, 13 * m), ints.as_strided(two, twos, 2 * m), ints.as_strided(two, twos, 4 * m))
    if B:
        need = _select_workspace(B, K, V)
        ws = scores.new_empty((need,), dtype=torch.uint8)
        _call("asrk_beam_select", dev, logits.data_ptr(), _DT[logits.dtype], ld, scores.data_ptr(), B, K, V, eos, *[t.data_ptr() for t in out],
              ws.data_ptr(), need)
    return BeamStep(*out)


def _check_parents(name: str, parents: torch.Tensor) -> torch.Tensor:
    if parents.dim() != 2 or parents.dtype != torch.int64:
        raise ValueError(f"{name}: parents must be an int64 [B, K] tensor")
    return parents if parents.is_contiguous() else parents.contiguous()


def reorder_states(states: torch.Tensor, parents: torch.Tensor) -> torch.Tensor:
    """``out[b, k] = states[b, parents[b, k]]``: any per-beam state, [B, K, ...] or [B*K, ...] of any type, goes to the beams
    that continue it (a new tensor of the same shape).  A parent that is no beam leaves the row as it is."""
    parents = _check_parents("reorder_states", parents)
    B, K = parents.shape
    if not (states.dim() >= 2 and tuple(states.shape[:2]) == (B, K)) and not (states.dim() >= 1 and states.shape[0] == B * K):
        raise ValueError(f"states must be [{B}, {K}, ...] or [{B * K}, ...], got {list(states.shape)}")
    if B * K > 65535:
        raise ValueError("reorder_states takes at most 65535 beams in all")
    dev = _gpu("reorder_states", states, parents)
    states = states.resolve_conj().resolve_neg().contiguous()  # x.conj() is the memory of x
    out = torch.empty_like(states)
    if out.numel():
        _call("asrk_reorder_rows", dev, states.data_ptr(), parents.data_ptr(), B, K, states.numel() // (B * K) * states.element_size(),
              out.data_ptr())
    return out


class PagedKVCache:
    """Keys and values of ``num_seqs`` sequences in 8 bits, on pages of 64 tokens.

    A page of one key/value head holds e4m3 values with one power-of-two scale ``2**e`` for its keys and one for its values: the
    smallest that fits its tokens.  A value is off by at most 2**-4 of itself, or where it is that small by 2**-10 of ``2**e``.
    When a later token of the page needs a larger scale, the older ones are rounded to it again: exactly, but for the small
    ones, whose roundings add up to less than 2**-9 of ``2**e``.  ``e`` lies in -64 .. 119: magnitudes above 1.75 * 2**127
    become that.  NaN and infinities are kept as NaN.

        cache = PagedKVCache(B * K, max_len, kv_heads, head_dim, num_layers=L, device="cuda")
        prompts = cache.leaders(K)                # every K-th sequence: one per utterance
        prompts.extend(prompt_lens)               # room for the prompts
        for l, layer in enumerate(layers):        # k, v [B, n, kv_heads, head_dim], q [B, n, q_heads, head_dim]
            prompts.write(k, v, layer=l); o = prompts.attend(q, layer=l)
        cache.reorder(zeros)                      # all beams of an utterance start from its prompt, on the same pages
        while ...:
            step = beam_select(logits, scores, eos)
            cache.reorder(step.parents)
            cache.extend(1)
            ... cache.write(k, v, layer=l); o = cache.attend(q, layer=l, num_beams=K) ...

    ``max_len`` is rounded up to whole pages; ``num_pages`` is room for all sequences at that length unless it is given.
    The cache and its views belong to one stream at a time.  Its tensors (``kv``, ``exps``, ``table``, ``lens``, ``starts``,
    ``refs``: the layout is that of ``asrk_kv_cache`` in include/asrk.h) may be read, and overwritten in place by what they
    held before, all of them together; they are never replaced, so a captured step stays valid.  Calls that cannot be
    carried out on the device (no free page, a sequence longer than ``max_len``) add nothing and set ``status``:
    ``check()`` raises for it."""

    def __init__(self, num_seqs: int, max_len: int, kv_heads: int, head_dim: int, *, num_layers: int = 1,
                 num_pages: Optional[int] = None, device: Union[str, torch.device] = "cuda"):
        if min(num_seqs, max_len, kv_heads, num_layers) < 1 or num_seqs > 65535 or kv_heads > 65535 or num_layers > 65535:
            raise ValueError("num_seqs, max_len, kv_heads and num_layers must be positive (and at most 65535 but for max_len)")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim must be 64 or 128, got {head_dim}")
        max_pages = -(-max_len // PAGE)
        num_pages = num_seqs * max_pages if num_pages is None else num_pages
        if num_pages < 1 or num_pages > 0x3FFFFFFF or max_pages > 0x7FFFFFFF // PAGE or num_seqs * max_pages > 0x7FFFFFFF:
            raise ValueError(f"num_pages {num_pages} / max_len {max_len} out of range")
        device = torch.device(device)
        if device.type != "cuda":
            raise _lib.AsrkError("PagedKVCache lives on a ROCm GPU only (there is no CPU fallback)")
        if device.index is None:
            device = torch.device("cuda", torch.cuda.current_device())
        lib = _lib.load()
        self.num_seqs, self.max_len, self.kv_heads, self.head_dim = num_seqs, max_pages * PAGE, kv_heads, head_dim
        self.num_layers, self.num_pages, self.device = num_layers, num_pages, device
        i32 = dict(dtype=torch.int32, device=device)
        self.kv = torch.zeros((num_layers, num_pages, kv_heads, 2, PAGE * head_dim), dtype=torch.uint8, device=device)
        self.exps = torch.zeros((num_layers, num_pages, kv_heads, 4), dtype=torch.int8, device=device)
        self.table = torch.full((num_seqs, max_pages), -1, **i32)
        self.lens, self.starts = torch.zeros((num_seqs,), **i32), torch.zeros((num_seqs,), **i32)
        self.refs = torch.zeros((num_pages,), **i32)
        self.status = torch.zeros((2,), **i32)
        self._scratch = torch.zeros((lib.asrk_kv_scratch_bytes(num_pages, num_seqs) // 4,), **i32)
        self._seq_stride = 1
        self._bind()

    def _bind(self):
        ptrs = (self.kv, self.exps, self.table, self.lens, self.starts, self.refs, self.status, self._scratch)
        self._c = _lib.KVCache(self.num_layers, self.num_pages, self.kv_heads, self.head_dim, self.num_seqs, self.max_len // PAGE,
                               self._seq_stride, *[ctypes.c_void_p(t.data_ptr()) for t in ptrs])
        self._ref = ctypes.byref(self._c)
        self._workspace: Dict[Tuple[int, int, int], int] = {}  # bytes that attend needs, by new tokens, heads and beams

    def leaders(self, num_beams: int) -> "PagedKVCache":
        """A view of every ``num_beams``-th sequence (beam 0 of each utterance), on the same pages."""
        if num_beams < 1 or self.num_seqs % num_beams:
            raise ValueError(f"{self.num_seqs} sequences are not groups of {num_beams}")
        view = object.__new__(PagedKVCache)
        view.__dict__.update(self.__dict__)
        view.num_seqs, view._seq_stride = self.num_seqs // num_beams, self._seq_stride * num_beams
        view.table, view.lens, view.starts = self.table[::num_beams], self.lens[::num_beams], self.starts[::num_beams]
        view._bind()
        return view

    # ---- pages

    def extend(self, n: Union[int, torch.Tensor]) -> None:
        """Room for ``n`` more tokens of every sequence (an int, or an integer [num_seqs] tensor: 0 for those that do not go
        on): ``starts`` becomes ``lens`` and ``lens`` grows.  Once per step, before the layers' ``write`` and ``attend``."""
        each = None
        if isinstance(n, torch.Tensor):
            if n.dim() != 1 or n.shape[0] != self.num_seqs or n.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"n must be an int or an integer [{self.num_seqs}] tensor")
            self._mine("extend", n)
            each, n = self._int32(n), 0
        elif not 0 <= n <= self.max_len:
            raise ValueError(f"cannot add {n} tokens to sequences of at most {self.max_len}")
        _call("asrk_kv_extend", self.device, self._ref, _address(each), n)

    def reorder(self, parents: torch.Tensor) -> None:
        """Beam k of utterance b goes on as a copy of its beam ``parents[b, k]``; -1 empties it and gives its pages back.
        int64 [B, K], B * K == num_seqs, K <= 32.  Only page numbers move.  No token of any sequence is new afterwards: ``extend``
        comes next."""
        parents = _check_parents("reorder", parents)
        if parents.numel() != self.num_seqs or parents.shape[1] > 32:
            raise ValueError(f"parents must be [B, K] with B * K == {self.num_seqs} and K <= 32, got {list(parents.shape)}")
        self._mine("reorder", parents)
        _call("asrk_kv_reorder", self.device, self._ref, parents.data_ptr(), parents.shape[1])

    def compact(self) -> torch.Tensor:
        """Moves pages so that those in use are the first ones of the pool; returns their number (int32 [], on the device)."""
        if self._seq_stride != 1:
            raise ValueError("compact the cache itself, not a view of some of its sequences")
        _call("asrk_kv_compact", self.device, self._ref)
        return self.status[1].clone()  # the word itself is the next compaction's

    def check(self) -> None:
        """Raises if any call since the last ``check`` could not be carried out (one host synchronisation)."""
        bits = int(self.status[0].item())
        if bits:
            self.status[0] = 0
            raise _lib.AsrkError("PagedKVCache: " + ", ".join(s for b, s in _lib.KV_STATUS.items() if bits & b))

    # ---- tokens

    def _mine(self, name: str, *tensors: torch.Tensor) -> None:
        if _gpu(name, *tensors) != self.device:
            raise ValueError(f"{name}: the cache is on {self.device}, the tensors are on {tensors[0].device}")

    @staticmethod
    def _int32(x: torch.Tensor) -> torch.Tensor:
        if x.dtype == torch.int64:
            x = x.clamp(-0x80000000, 0x7FFFFFFF).to(torch.int32)  # what does not fit stays out of range
        return x.contiguous()

    def _layer(self, layer: int) -> int:
        if not 0 <= layer < self.num_layers:
            raise ValueError(f"layer {layer} of a cache of {self.num_layers}")
        return layer

    @staticmethod
    def _rows(x: torch.Tensor) -> Tuple[torch.Tensor, List[int]]:
        """x [S, n, heads, dim] with dense last dimension and rows at 16 bytes, and its other strides."""
        mask = 16 // x.element_size() - 1
        *lds, one = x.stride()
        if one != 1 or (lds[0] | lds[1] | lds[2]) & mask or x.data_ptr() & 15:  # a dimension of size 1 may have any stride
            lds = [0 if size == 1 else st for size, st in zip(x.shape, lds)]
            if one != 1 or (lds[0] | lds[1] | lds[2]) & mask or x.data_ptr() & 15:
                x = x.clone(memory_format=torch.contiguous_format)
                lds = list(x.stride()[:3])
        return x, lds

    def write(self, k: torch.Tensor, v: torch.Tensor, layer: int = 0) -> None:
        """The new tokens' keys and values of one layer: ``k``, ``v`` [num_seqs, n, kv_heads, head_dim] (float32 or bfloat16, any
        strides).  Row i of sequence s is its token ``starts[s] + i``; rows behind ``lens[s]`` are not looked at.  New tokens that
        no row is given for are not written, and hold nothing defined until they are (also if an earlier call wrote them: a page's
        scale is that of the rows it was given last)."""
        shape = k.shape
        if len(shape) != 4 or shape != v.shape or shape[0] != self.num_seqs or shape[2] != self.kv_heads or shape[3] != self.head_dim:
            raise ValueError(f"k and v must be [{self.num_seqs}, n, {self.kv_heads}, {self.head_dim}], got {list(shape)} and {list(v.shape)}")
        if k.dtype not in _DT or v.dtype != k.dtype:
            raise ValueError("k and v must both be float32 or bfloat16")
        self._mine("write", k, v)
        layer = self._layer(layer)
        n = shape[1]
        if n == 0:
            return
        if n > 65534 * PAGE:
            raise ValueError(f"cannot write {n} tokens in one call")
        (k, lds), (v, v_lds) = self._rows(k), self._rows(v)
        if lds != v_lds:
            k, v = k.contiguous(), v.contiguous()
            row = self.kv_heads * self.head_dim
            lds = (n * row, row, self.head_dim)  # not k.stride(): a dimension of 1 may have any
        _call("asrk_kv_write", self.device, self._ref, layer, k.data_ptr(), v.data_ptr(), _DT[k.dtype], *lds, n)

    def read(self, first: Union[int, torch.Tensor], count: int, layer: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Tokens ``first`` .. ``first + count - 1`` of every sequence (an int, or an integer [num_seqs] tensor) as they are
        held: keys and values, bfloat16 [num_seqs, count, kv_heads, head_dim] of one layer, or [num_layers, ...] of all; zeros
        where a sequence has no such token."""
        each = None
        if isinstance(first, torch.Tensor):
            if first.dim() != 1 or first.shape[0] != self.num_seqs or first.dtype not in (torch.int32, torch.int64):
                raise ValueError(f"first must be an int or an integer [{self.num_seqs}] tensor")
            self._mine("read", first)
            each, first = self._int32(first), 0
        elif not 0 <= first <= self.max_len:
            raise ValueError(f"first {first} of sequences of at most {self.max_len}")
        if not 0 <= count <= 65534 * PAGE:
            raise ValueError(f"cannot read {count} tokens in one call")
        layers = self.num_layers if layer is None else 1
        if layers * self.num_seqs > 65535:
            raise ValueError("read one layer at a time: layers * num_seqs passes 65535")
        shape = (self.num_seqs, count, self.kv_heads, self.head_dim)
        k = torch.empty(shape if layer is not None else (layers, *shape), dtype=torch.bfloat16, device=self.device)
        v = torch.empty_like(k)
        layer = 0 if layer is None else self._layer(layer)
        if count:
            _call("asrk_kv_read", self.device, self._ref, layer, layers, _address(each), first, count, k.data_ptr(), v.data_ptr())
        return k, v

    def attend(self, q: torch.Tensor, layer: int = 0, *, scale: Optional[float] = None, num_beams: int = 1) -> torch.Tensor:
        """Attention of the new tokens over one layer of the cache: bfloat16 [num_seqs, n, q_heads, head_dim] for ``q`` of that
        shape (any strides; query head j reads key/value head ``j // (q_heads // kv_heads)``).  Row i of sequence s sees the
        tokens up to its own, ``starts[s] + i``; rows behind ``lens[s]`` are zero.  Tokens that a row sees have to have been written;
        those behind the last row's own need not be yet.  ``scale`` (positive) is ``head_dim ** -0.5`` by default.

        The weights of the tokens are held to 2**-11 of themselves, and below 2**-27 of a row's largest to 2**-38 of that.

        ``num_beams`` consecutive sequences are worked on together, and pages that they share are read once.  It changes
        no result but for rounding: the beams may share any pages, or none."""
        shape = q.shape
        if len(shape) != 4 or shape[0] != self.num_seqs or shape[3] != self.head_dim or shape[2] < 1 or shape[2] % self.kv_heads:
            raise ValueError(f"q must be [{self.num_seqs}, n, a multiple of {self.kv_heads}, {self.head_dim}], got {list(shape)}")
        if q.dtype != torch.bfloat16:
            raise ValueError("q must be bfloat16")
        if not 1 <= num_beams <= 32 or self.num_seqs % num_beams:
            raise ValueError(f"{self.num_seqs} sequences are not groups of {num_beams} (at most 32)")
        scale = self.head_dim ** -0.5 if scale is None else float(scale)
        if not 1e-30 < scale < 1e30:
            raise ValueError(f"scale must be positive, got {scale}")
        self._mine("attend", q)
        layer = self._layer(layer)
        n, heads = shape[1], shape[2]
        if num_beams * n * (heads // self.kv_heads) > 65535 * 128:
            raise ValueError(f"cannot attend {n} tokens of {num_beams} beams in one call")
        out = q.new_empty(shape)
        if n == 0:
            return out
        q, lds = self._rows(q)
        need = self._workspace.get((n, heads, num_beams))
        if need is None:
            need = self._workspace[n, heads, num_beams] = _lib.load().asrk_kv_attention_workspace_bytes(self._ref, n, heads, num_beams)
        ws = q.new_empty((need,), dtype=torch.uint8) if need else None
        _call("asrk_kv_attention", self.device, self._ref, layer, q.data_ptr(), *lds, n, heads, num_beams, scale, out.data_ptr(), _address(ws), need)
        return out

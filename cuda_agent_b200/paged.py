"""A paged latent cache for serving: storage, page tables and the operators that go with them.

``PagedLatentCache`` holds the rows (512 latent + 64 rotary columns) of many sequences over several layers in pages of
equal size, and the bookkeeping that says which page holds what: a table row, a length and reference counts on the
device. Its methods are the extension's ``mla_pages_*``, ``mla_rope_append_forward``, ``mla_paged_attention_forward``
and ``mla_sparse_decode_forward``; what is computed in torch are the batch's own small tables and, for ``attend_sparse``, the
rows of the selected positions. A program serves with it as

    cache = PagedLatentCache(layers, pages, 64, slots=256, max_rows=32768)
    freq, mscale = rope_frequencies(64, scaling="yarn", factor=16.0, mscale=1.0, mscale_all_dim=1.0)
    scale = head_dim ** -0.5 * rope_score_factor(16.0, 1.0)
    cache.extend(seqs, new_length)                       # pages for the new tokens of every sequence
    batch = cache.batch(seqs, q_start)                   # once per step, for all layers
    for layer in range(layers):
        cache.append(layer, batch, q_pe, c_kv, k_pe, freq, q[..., 512:], mscale=mscale)
        out, lse = cache.attend(layer, batch, q, scale)

and ``fork``, ``free`` and ``compact`` between steps. ``extend`` and ``fork`` change everything or nothing; they raise
when the pool has too few free pages, which costs a synchronisation (``check=False`` leaves it out).
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

from . import load_extension

ROW = 576


def rope_frequencies(rot: int, base: float = 10000.0, scaling: str = "none", factor: float = 1.0,
                     original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0, device="cuda",
                     mscale: float = 1.0, mscale_all_dim: float = 0.0):
    """(freq, factor on the rotated columns): radians per position of the rot / 2 pairs (64-bit), and what ``append`` takes as
    ``mscale``.

    ``scaling`` stretches a model's positions from ``original_length`` to ``factor`` times it:
      none    base^(-2i / rot)
      linear  every frequency divided by the factor
      ntk     the base raised to base * factor^(rot / (rot - 2)): fast pairs stay, the slowest is divided by the factor
      yarn    pairs that turn more than beta_fast times within original_length stay, those that turn less than beta_slow
              times are divided by the factor, a ramp over the pair's number in between. The factor on the rotated
              columns is m(mscale) / m(mscale_all_dim), m(c) = 0.1 c ln(factor) + 1

    YaRN means m as a temperature of the whole score, m^2 times it. On the rotated columns alone, as without
    ``mscale_all_dim``, that is so only for a head all of whose columns are rotated. Of the rows of this cache 64 of 576 are: a
    checkpoint says by its two coefficients (mostly equal, so that the factor is 1) what the rotated columns get, and the whole
    score takes ``rope_score_factor(factor, mscale_all_dim)``, which belongs into the softmax scale.
    """
    if rot <= 0 or rot % 2:
        raise ValueError("rot must be a positive even number")
    if base <= 1.0 or factor < 1.0 or original_length < 1:
        raise ValueError("base must be above 1, factor and original_length at least 1")
    if mscale < 0 or mscale_all_dim < 0:
        raise ValueError("mscale and mscale_all_dim must not be negative")
    i = torch.arange(rot // 2, dtype=torch.float64)
    on_rotated = 1.0
    if scaling == "ntk":
        if rot == 2:
            raise ValueError("ntk scaling needs more than one pair")
        base = base * factor ** (rot / (rot - 2))
    freq = base ** (-2.0 * i / rot)
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def pair_of(turns):
            return rot * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))
        low = min(max(math.floor(pair_of(beta_fast)), 0), rot - 1)
        high = min(max(math.ceil(pair_of(beta_slow)), 0), rot - 1)
        ramp = ((i - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        on_rotated = _yarn_m(factor, mscale) / _yarn_m(factor, mscale_all_dim)
    elif scaling not in ("none", "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}: none, linear, ntk or yarn")
    return freq.to(device), on_rotated


def _yarn_m(factor: float, coefficient: float) -> float:
    return 0.1 * coefficient * math.log(factor) + 1.0


def rope_score_factor(factor: float, mscale_all_dim: float) -> float:
    """What yarn scaling by ``factor`` multiplies the softmax scale by, for a checkpoint with the coefficient ``mscale_all_dim``."""
    if factor < 1.0 or mscale_all_dim < 0:
        raise ValueError("factor must be at least 1, mscale_all_dim must not be negative")
    return _yarn_m(factor, mscale_all_dim) ** 2


@dataclass
class PagedBatch:
    """The sequences of one step: their rows of the page table, where their new tokens begin, their lengths."""
    page_table: torch.Tensor
    q_start: torch.Tensor
    kv_len: torch.Tensor


class PagedLatentCache:
    """``layers`` x ``pages`` pages of ``page_size`` rows; up to ``slots`` sequences of up to ``max_rows`` rows."""

    def __init__(self, layers: int, pages: int, page_size: int, slots: int, max_rows: int, dtype=torch.bfloat16,
                 device="cuda"):
        if min(layers, pages, page_size, slots, max_rows) < 1:
            raise ValueError("layers, pages, page_size, slots and max_rows must be positive")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("the cache holds bfloat16 or float16")
        ints = dict(dtype=torch.int32, device=device)
        self.rows = torch.zeros(layers, pages, page_size, ROW, dtype=dtype, device=device)
        self.page_table = torch.full((slots, -(-max_rows // page_size)), -1, **ints)
        self.length = torch.zeros(slots, **ints)
        self.refcount = torch.zeros(pages, **ints)
        self.page_size = page_size
        self._ops = load_extension()

    def _list(self, x) -> torch.Tensor:
        return torch.as_tensor(x, dtype=torch.int32, device=self.length.device)

    # ------------------------------------------------------------------------------------------ pages
    def extend(self, seqs, new_length, check: bool = True) -> None:
        """Pages for sequences ``seqs`` up to ``new_length`` rows each; the lengths become these."""
        self._ops.mla_pages_extend(self.page_table, self.length, self.refcount, self._list(seqs), self._list(new_length),
                                   self.page_size, check)

    def fork(self, src, dst, check: bool = True) -> None:
        """Sequences ``dst``, empty before, become copies of ``src``: full pages shared, a partly filled last one copied."""
        self._ops.mla_pages_fork(self.rows, self.page_table, self.length, self.refcount, self._list(src), self._list(dst), check)

    def free(self, seqs, check: bool = False) -> None:
        self._ops.mla_pages_free(self.page_table, self.length, self.refcount, self._list(seqs), self.page_size, check)

    def compact(self, check: bool = False) -> None:
        """Moves the pages in use to the front of the pool. Batches made before no longer hold."""
        self._ops.mla_pages_compact(self.rows, self.page_table, self.length, self.refcount, check)

    def pages_free(self) -> int:
        """Free pages (synchronises)."""
        return int((self.refcount == 0).sum())

    # ------------------------------------------------------------------------------------------ steps
    def batch(self, seqs, q_start) -> PagedBatch:
        """The batch of sequences ``seqs``, whose new tokens are [q_start[i], q_start[i + 1]) of the step's and whose lengths
        (the new tokens among them) are the present ones. A sequence stands in a batch once: two would write the same rows.
        Of a list that is checked here. A tensor is not read by the host: there a sequence that is out of range gets no pages
        and length 0, so ``append`` writes nothing for it and reports it, and attention sees nothing; whether one stands there
        twice is not looked at."""
        slots = self.length.numel()
        if torch.is_tensor(seqs):
            seqs = seqs.to(self.length.device, torch.int64)
            at = seqs.clamp(0, slots - 1)
            inside = at == seqs
            return PagedBatch(torch.where(inside[:, None], self.page_table[at], -1), self._list(q_start), self.length[at] * inside)
        seqs = list(seqs)
        if not all(0 <= s < slots for s in seqs):
            raise ValueError(f"sequences must lie in [0, {slots})")
        if len(set(seqs)) < len(seqs):
            raise ValueError("a sequence is listed twice")
        seqs = self._list(seqs).long()
        return PagedBatch(self.page_table[seqs], self._list(q_start), self.length[seqs])

    def append(self, layer: int, batch: PagedBatch, q_pe, c_kv, k_pe, freq, q_out=None, interleaved: bool = False,
               mscale: float = 1.0, check: bool = False):
        """Writes the new rows of ``layer`` and returns the rotated q_pe (in ``q_out``, a view such as q[..., 512:], if given)."""
        return self._ops.mla_rope_append_forward(q_pe, c_kv, k_pe, self.rows[layer], batch.page_table, batch.q_start,
                                                 batch.kv_len, freq, q_out, interleaved, mscale, check)

    def attend(self, layer: int, batch: PagedBatch, q, softmax_scale: float, causal: bool = True, window: int = 0,
               check: bool = False):
        """(out [T, H, 512], lse [T, H]) of the new tokens over all their sequences' rows."""
        return self._ops.mla_paged_attention_forward(q, self.rows[layer], batch.page_table, batch.q_start, batch.kv_len,
                                                     softmax_scale, causal, window, check=check)

    def attend_sparse(self, layer: int, batch: PagedBatch, q, idx, softmax_scale: float, check: bool = False):
        """Top-k sparse decode on the same pages: one new token per sequence, q [B, H, 576], idx [B, topk] the selected
        positions of each sequence (-1: none). The pool is one run of rows to ``mla_sparse_decode_forward``, whose limits hold
        here: bfloat16 and a multiple of 64 heads, where ``attend`` takes either type and any number. The positions become rows by
        some ten small torch operations in every call."""
        layers, pages, size, _ = self.rows.shape
        B, topk = idx.shape
        at = idx.clamp_min(0).long()
        page = torch.gather(batch.page_table, 1, (at // size).clamp_max(batch.page_table.shape[1] - 1))
        live = (idx >= 0) & (idx < batch.kv_len[:, None]) & (page >= 0)
        rows = torch.where(live, page * size + (at % size).to(torch.int32), torch.full_like(page, -1))
        ends = torch.full((1, B), pages * size, dtype=torch.int32, device=idx.device)
        out = self._ops.mla_sparse_decode_forward(q.reshape(1, B, q.shape[1], ROW), self.rows[layer].view(1, pages * size, ROW),
                                                  ends, rows.reshape(1, B, topk).contiguous(), softmax_scale, 0, check)
        return out.reshape(B, q.shape[1], 512)

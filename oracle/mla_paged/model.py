"""Eager oracle for one serving step on a paged latent cache (TEST INFRASTRUCTURE).

File shape follows the reference's eager-model slot (agent_workdir/model.py:9-26). The reference ships no attention model,
test or vector, so parity of this path is UNPINNED by the reference; this file restates the operator definitions and the
tests pin them with float64 statements of their own.

The new tokens of a batch of sequences (one each in a decode step, many in a prompt's chunk):

  q          bf16 [T, Hh, 576]         512 latent columns, and 64 that q_pe's rotation replaces
  q_pe       bf16 [T, Hh, 64]          before rotation
  c_kv, k_pe bf16 [T, 512], [T, 64]    the new cache rows, k_pe before rotation
  cache      bf16 [P, page, 576]       pages of rows; rows of earlier tokens are there already
  page_table int32 [B, max_pages]      the pages of every sequence in order, -1 behind them
  q_start    int32 [B + 1]             sequence b has tokens [q_start[b], q_start[b + 1])
  kv_len     int32 [B]                 rows of sequence b, its new ones among them: its tokens' positions end at kv_len - 1

  rotation   pairs (2i, 2i + 1) by position * 10000^(-i / 32)                  fp64 angles, fp32 products -> bf16
  cache      the new rows are written to their pages
  out        softmax over j <= position of (q . row_j / sqrt(192)) . row_j[:512]   fp32 -> bf16   [T, Hh, 512]
  lse        log of the softmax's sum                                           fp32 [T, Hh]

forward returns (out, lse, cache). ``CAB_MLA_PAGED_CONFIG``: 0 = 3 sequences of a few tokens, 16 heads, pages of 16;
1 = a decode step of 64 sequences of up to 8192 rows, 128 heads, pages of 64; 2 = one chunk of 1024 tokens behind 7168
rows, 128 heads (an eager step of 40 TFLOP in fp32).
"""
import os

import torch
import torch.nn as nn

D_QK, D_V, R = 576, 512, 64
SCALE = 192 ** -0.5
CONFIGS = {
    0: dict(new=[5, 1, 40], rows=[5, 77, 130], heads=16, page=16),
    1: dict(new=[1] * 64, rows=[8192 - 97 * b for b in range(64)], heads=128, page=64),
    2: dict(new=[1024], rows=[8192], heads=128, page=64),
}
CONFIG = int(os.environ.get("CAB_MLA_PAGED_CONFIG", "0"))

OUTPUT_POLICY = [("atol", 2e-2), ("atol", 2e-2), ("atol", 2e-2)]


def rotate(x, pos, freq):
    """x [T, ..., 64], pos [T]: interleaved pairs, in x's type."""
    a = pos.double()[:, None] * freq
    shape = (x.shape[0],) + (1,) * (x.dim() - 2) + (freq.numel(),)
    cos, sin = a.cos().float().reshape(shape), a.sin().float().reshape(shape)
    x0, x1 = x.float()[..., 0::2], x.float()[..., 1::2]
    return torch.stack((x0 * cos - x1 * sin, x1 * cos + x0 * sin), -1).flatten(-2).to(x.dtype)


class Model(nn.Module):
    """forward(q, q_pe, c_kv, k_pe, cache, page_table, q_start, kv_len) -> (out, lse, cache)."""

    def __init__(self, heads: int, page: int) -> None:
        super().__init__()
        self.heads, self.page = heads, page
        self.register_buffer("freq", 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) / (R // 2)))

    def forward(self, q, q_pe, c_kv, k_pe, cache, page_table, q_start, kv_len):
        cache, q = cache.clone(), q.clone()
        outs, lses = [], []
        for b in range(kv_len.numel()):
            t0, t1, n = int(q_start[b]), int(q_start[b + 1]), int(kv_len[b])
            pos = torch.arange(n - (t1 - t0), n, device=q.device)
            page = page_table[b, pos // self.page].long()
            cache[page, pos % self.page] = torch.cat((c_kv[t0:t1], rotate(k_pe[t0:t1], pos, self.freq)), -1)
            q[t0:t1, :, D_V:] = rotate(q_pe[t0:t1], pos, self.freq)
            rows = cache[page_table[b, : -(-n // self.page)].long()].reshape(-1, D_QK)[:n].float()
            scores = torch.einsum("thd,jd->thj", q[t0:t1].float(), rows) * SCALE
            hidden = torch.arange(n, device=q.device)[None] > pos[:, None]
            scores = scores.masked_fill(hidden[:, None], float("-inf"))
            lses.append(torch.logsumexp(scores, -1))
            outs.append(torch.einsum("thj,jd->thd", torch.softmax(scores, -1), rows[:, :D_V]))
        return torch.cat(outs).to(q.dtype), torch.cat(lses), cache


_GEN = None


def reseed(seed=None) -> None:
    global _GEN
    _GEN = torch.Generator().manual_seed(1234 + CONFIG if seed is None else seed)


def make_inputs(new, rows, heads, page, gen):
    T, bf = sum(new), torch.bfloat16
    need = [-(-n // page) for n in rows]
    pool = sum(need) + 1
    cache = torch.empty(pool, page, D_QK, dtype=bf)
    for p in range(pool):                                               # keeps the fp32 staging small
        cache[p] = torch.randn(page, D_QK, generator=gen).to(bf)
    order = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    q = torch.randn(T, heads, D_QK, generator=gen).to(bf)
    q_pe = torch.randn(T, heads, R, generator=gen).to(bf)
    c_kv, k_pe = torch.randn(T, D_V, generator=gen).to(bf), torch.randn(T, R, generator=gen).to(bf)
    q_start = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    return [q, q_pe, c_kv, k_pe, cache, table, q_start, torch.tensor(rows, dtype=torch.int32)]


def get_inputs():
    if _GEN is None:
        reseed()
    c = CONFIGS[CONFIG]
    return make_inputs(c["new"], c["rows"], c["heads"], c["page"], _GEN)


def get_init_inputs():
    c = CONFIGS[CONFIG]
    return [c["heads"], c["page"]]

"""The paged latent cache as a serving program uses it: prompts in chunks, forks, decode steps (dense and top-k sparse),
sequences that end, compaction, over two layers; and the task's reference-style loops.

Beside the GPU's cache the test keeps every sequence's rows as a plain tensor, made from the 64-bit rotation rounded once;
attention is compared with the 64-bit statement on the rows that the pages hold.
"""
import random

import pytest
import torch

import paged_reference as ref
from conftest import ROOT

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


class Program:
    def __init__(self, dev, dtype, heads, page):
        from cuda_agent_b200.paged import PagedLatentCache, rope_frequencies
        self.dev, self.dtype, self.heads = dev, dtype, heads
        self.cache = PagedLatentCache(2, 400 * 16 // page, page, slots=24, max_rows=2000, dtype=dtype, device=dev)
        self.freq, self.mscale = rope_frequencies(64, scaling="yarn", factor=8.0, device=dev)
        self.rows = {}                               # sequence -> [layer] -> [n, 576] as expected
        self.g = torch.Generator(device=dev).manual_seed(page)

    def rand(self, *shape):
        return torch.randn(*shape, generator=self.g, device=self.dev).to(self.dtype)

    def step(self, new, sparse=False):
        """new: {sequence: tokens}."""
        seqs, T = list(new), sum(new.values())
        before = {s: (self.rows[s][0].shape[0] if s in self.rows else 0) for s in seqs}
        self.cache.extend(seqs, [before[s] + new[s] for s in seqs])
        start = [0]
        for s in seqs:
            start.append(start[-1] + new[s])
        batch = self.cache.batch(seqs, start)
        pos = torch.cat([torch.arange(before[s], before[s] + new[s]) for s in seqs]).to(self.dev, torch.int32)
        for layer in range(2):
            q, q_pe = self.rand(T, self.heads, 576), self.rand(T, self.heads, 64)
            joint = self.rand(T, 576)
            self.cache.append(layer, batch, q_pe, joint[:, :512], joint[:, 512:], self.freq, q[..., 512:], True, self.mscale, check=True)
            turned, tol = ref.rotate(q_pe, pos, self.freq, True, self.mscale)
            assert ((q[..., 512:].double() - turned).abs() <= tol).all()
            k, k_tol = ref.rotate(joint[:, None, 512:], pos, self.freq, True, self.mscale)
            for i, s in enumerate(seqs):
                held = self.held(s, layer)
                mine = held[before[s]:]
                assert torch.equal(mine[:, :512], joint[start[i]:start[i + 1], :512])
                assert ((mine[:, 512:].double() - k[start[i]:start[i + 1], 0]).abs() <= k_tol[start[i]:start[i + 1], 0]).all()
                old = self.rows.setdefault(s, [torch.empty(0, 576, dtype=self.dtype, device=self.dev)] * 2)
                assert torch.equal(held[:before[s]], old[layer])
                self.rows[s] = [held if e == layer else old[e] for e in range(2)]
            out, lse = self.cache.attend(layer, batch, q, SCALE, check=True)
            want, want_lse, tol, tol_lse = ref.attention(q, self.cache.rows[layer], batch.page_table, batch.q_start, batch.kv_len, SCALE)
            assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()
            if sparse:
                idx = torch.full((len(seqs), 128), -1, dtype=torch.int32, device=self.dev)
                for i, s in enumerate(seqs):
                    n = self.rows[s][layer].shape[0]
                    some = torch.randperm(n, generator=self.g, device=self.dev)[:100].to(torch.int32)
                    idx[i, :len(some)] = some
                idx[0, 120], idx[0, 121] = 1999, 2 ** 31 - 1             # behind the sequence's end: not selected
                got = self.cache.attend_sparse(layer, batch, q, idx, SCALE, check=True)
                for i, s in enumerate(seqs):
                    picked = idx[i][(idx[i] >= 0) & (idx[i] < self.rows[s][layer].shape[0])].long()
                    r = self.rows[s][layer][picked].double()
                    p = torch.softmax(q[i].double() @ r.T * SCALE, -1)
                    assert ((got[i].double() - p @ r[:, :512]).abs() <= 2e-2).all()

    def held(self, s, layer):
        """The rows of a sequence as its pages hold them now."""
        n = int(self.cache.length[s])
        pages = self.cache.page_table[s, :-(-n // self.cache.page_size)].long()
        return self.cache.rows[layer][pages].reshape(-1, 576)[:n].clone()

    def check_all(self):
        for s, layers in self.rows.items():
            for layer in range(2):
                assert torch.equal(self.held(s, layer), layers[layer]), (s, layer)
        need = sum(int(n > 0) for n in self.cache.refcount.tolist())
        assert self.cache.pages_free() == self.cache.refcount.numel() - need


@pytest.mark.parametrize("dtype,heads,page", [(torch.bfloat16, 64, 16), (torch.float16, 5, 64), (torch.bfloat16, 128, 40)])
def test_serving(cuda_device, dtype, heads, page):
    rng = random.Random(page)
    p = Program(cuda_device, dtype, heads, page)
    sparse = dtype == torch.bfloat16 and heads % 64 == 0
    p.step({0: 37})                                   # a prompt in three chunks, other sequences beside it
    p.step({0: 100, 1: 1, 2: 64})
    p.step({0: 13, 3: 150})
    p.cache.fork([0, 0, 2], [10, 11, 12])             # three answers from two prompts
    for a, b in ((0, 10), (0, 11), (2, 12)):
        p.rows[b] = list(p.rows[a])
    p.check_all()
    for _ in range(3):                                # decode: every sequence goes its own way
        p.step({s: 1 for s in sorted(p.rows)}, sparse=sparse)
    p.check_all()
    p.cache.free([0, 2])
    for s in (0, 2):
        del p.rows[s]
    p.check_all()
    p.cache.compact(check=True)
    used = int((p.cache.refcount > 0).sum())
    assert (p.cache.refcount[:used] > 0).all() and (p.cache.refcount[used:] == 0).all()
    p.check_all()
    p.step({10: 3, 0: 20, 12: 1, 5: 300})             # verification of drafted tokens, freed places used again
    p.check_all()
    with pytest.raises(RuntimeError, match="free pages"):
        p.cache.extend([15, 16, 17, 18], [2000] * 4)
    p.check_all()
    p.cache.free(sorted(p.rows) + [23])
    assert p.cache.pages_free() == p.cache.refcount.numel() and (p.cache.page_table == -1).all()


def test_decode_step_as_one_graph(cuda_device):
    """Append and attention of a step recorded once and replayed while the lengths grow (pages taken before)."""
    p = Program(cuda_device, torch.bfloat16, 16, 64)
    p.step({0: 60, 1: 130})
    p.cache.extend([0, 1], [80, 150])
    p.cache.length.copy_(torch.tensor([60, 130] + [0] * 22, dtype=torch.int32))
    batch = p.cache.batch([0, 1], [0, 1, 2])
    q, q_pe, joint = p.rand(2, 16, 576), p.rand(2, 16, 64), p.rand(2, 576)

    def step():
        batch.kv_len.add_(1)
        p.cache.append(0, batch, q_pe, joint[:, :512], joint[:, 512:], p.freq, q[..., 512:])
        return p.cache.attend(0, batch, q, SCALE)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = step()
    for i in range(1, 9):
        for t in (q, q_pe, joint):
            t.copy_(p.rand(*t.shape))
        graph.replay()
        torch.cuda.synchronize()
        assert batch.kv_len.tolist() == [60 + i, 130 + i]
        want, want_lse, tol, tol_lse = ref.attention(q, p.cache.rows[0], batch.page_table, batch.q_start, batch.kv_len, SCALE)
        assert ((out.double() - want).abs() <= tol).all() and ((lse.double() - want_lse).abs() <= tol_lse).all()
        turned, tol = ref.rotate(q_pe, batch.kv_len - 1, p.freq)
        assert ((q[..., 512:].double() - turned).abs() <= tol).all()


@pytest.mark.parametrize("config", ["0", "1"])
def test_task_loops(cuda_device, built_libs, capsys, monkeypatch, config):
    monkeypatch.setenv("CAB_MLA_PAGED_CONFIG", config)
    monkeypatch.syspath_prepend(str(built_libs.WORKDIR))
    from utils import profiling, verification
    args = ["--task", str(built_libs.WORKDIR / "tasks" / "mla_paged"), "--model-dir", str(ROOT / "oracle" / "mla_paged")]
    assert verification.main(args + ["--checks", "5" if config == "0" else "1"]) == 0
    assert "[PASS] verify success" in capsys.readouterr().out
    if config == "0":
        assert profiling.main(args + ["--iters", "3", "--no-compile"]) == 0
        assert "CUDA Extension:" in capsys.readouterr().out


def test_batch_from_numbers_on_the_gpu(cuda_device):
    """A place of the batch that names no sequence: reported by the append, nothing written for it, nothing seen by its tokens;
    also in a captured step, and where the step counts the lengths up."""
    p = Program(cuda_device, torch.bfloat16, 16, 64)
    p.step({0: 60, 1: 130, 2: 7})
    p.cache.extend([0, 1, 2], [61, 131, 8])
    seqs = torch.tensor([0, 24, 1, 2 ** 31 - 1, -3, 2], dtype=torch.int32, device=cuda_device)
    fine = [0, 2, 5]
    joint, q_pe, q = p.rand(6, 576), p.rand(6, 16, 64), p.rand(6, 16, 576)
    start = torch.arange(7, dtype=torch.int32, device=cuda_device)

    before = p.cache.rows.clone()
    batch = p.cache.batch(seqs, start)
    for _ in range(2):
        with pytest.raises(RuntimeError, match="page table"):
            p.cache.append(0, batch, q_pe, joint[:, :512], joint[:, 512:], p.freq, q[..., 512:], check=True)
        batch.kv_len[[1, 3, 4]] += 1                  # a step that counts the lengths up itself: still no page of anyone's
    changed = (p.cache.rows != before).any(-1).nonzero().tolist()
    assert sorted(changed) == sorted([0, int(p.cache.page_table[s, n // 64]), n % 64] for s, n in ((0, 60), (1, 130), (2, 7)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        batch = p.cache.batch(seqs, start)
        p.cache.append(0, batch, q_pe, joint[:, :512], joint[:, 512:], p.freq, q[..., 512:])
        out, lse = p.cache.attend(0, batch, q, SCALE)
    graph.replay()
    torch.cuda.synchronize()
    want, want_lse, tol, tol_lse = ref.attention(q, p.cache.rows[0], batch.page_table, start, batch.kv_len, SCALE)
    assert ((out.double() - want).abs() <= tol).all() and torch.isinf(lse[[1, 3, 4]]).all() and (out[[1, 3, 4]] == 0).all()
    assert ((lse.double() - want_lse)[fine].abs() <= tol_lse[fine]).all() and torch.isfinite(lse[fine]).all()

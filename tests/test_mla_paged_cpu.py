"""The paged latent cache without a GPU: the eager model against float64 loops, rotary frequencies, refusals that come
before anything touches a device."""
import ctypes
import math

import pytest
import torch

from conftest import load_oracle


@pytest.fixture(scope="module")
def capi(built_libs):
    from cuda_agent_b200 import capi
    capi.lib()
    return capi


def test_eager_model_against_loops():
    m = load_oracle("mla_paged", {"CAB_MLA_PAGED_CONFIG": 0})
    new, rows, heads, page = [3, 1], [3, 9], 2, 4
    q, q_pe, c_kv, k_pe, cache, table, start, kv = m.make_inputs(new, rows, heads, page, torch.Generator().manual_seed(1))
    out, lse, after = m.Model(heads, page)(q, q_pe, c_kv, k_pe, cache, table, start, kv)
    want = cache.clone()
    t = 0
    for b, n in enumerate(new):
        for i in range(n):
            pos = rows[b] - n + i
            turn = [pos * 10000.0 ** (-e / 32) for e in range(32)]

            def rot(x):
                y = []
                for e, a in enumerate(turn):
                    u, v = float(x[2 * e]), float(x[2 * e + 1])
                    y += [u * math.cos(a) - v * math.sin(a), v * math.cos(a) + u * math.sin(a)]
                return torch.tensor(y, dtype=torch.float64).to(torch.bfloat16)
            want[table[b, pos // page].long(), pos % page] = torch.cat((c_kv[t], rot(k_pe[t])))
            for h in range(heads):
                x = torch.cat((q[t, h, :512], rot(q_pe[t, h]))).double()
                seen = torch.stack([want[table[b, j // page].long(), j % page].double() for j in range(pos + 1)])
                s = (seen @ x) * 192 ** -0.5
                w = torch.exp(s - s.max())
                got = out[t, h].double()
                exact = (w / w.sum()) @ seen[:, :512]
                # bf16 roundings of the result, and of rotated values by another last bit at most
                assert ((got - exact).abs() <= 2.0 ** -8 * exact.abs() + 2e-2).all()
                assert abs(float(lse[t, h]) - float(s.max() + torch.log(w.sum()))) <= 2e-2
            t += 1
    assert ((after.double() - want.double()).abs() <= 2.0 ** -7 * want.double().abs()).all()


def test_frequencies():
    from cuda_agent_b200.paged import rope_frequencies
    f, m = rope_frequencies(64, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0 and f[0] == 1.0
    assert abs(float(f[31]) - 10000.0 ** (-62 / 64)) < 1e-15
    lin, _ = rope_frequencies(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, f / 4)
    ntk, _ = rope_frequencies(64, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and abs(float(ntk[31] / f[31]) - 0.25) < 1e-12 and (ntk[1:] < f[1:]).all()
    yarn, m = rope_frequencies(64, scaling="yarn", factor=40.0, original_length=4096, device="cpu")
    assert abs(m - (0.1 * math.log(40.0) + 1)) < 1e-15
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(yarn[turns > 32 * 1.4], f[turns > 32 * 1.4], rtol=1e-14)
    assert torch.allclose(yarn[turns < 1 / 1.4], f[turns < 1 / 1.4] / 40, rtol=1e-14)
    assert ((yarn <= f * (1 + 1e-15)) & (yarn >= f / 40 * (1 - 1e-15))).all()
    same, m = rope_frequencies(64, scaling="yarn", factor=1.0, device="cpu")
    assert torch.allclose(same, f, rtol=1e-15) and m == 1.0
    for bad in (dict(rot=63), dict(rot=0), dict(rot=64, scaling="log"), dict(rot=64, factor=0.5), dict(rot=64, base=1.0),
                dict(rot=2, scaling="ntk"), dict(rot=64, original_length=0)):
        with pytest.raises(ValueError):
            rope_frequencies(**bad, device="cpu")


def batch(capi, **kw):
    fake = 0x10000                                   # aligned, never dereferenced: the checks fail first
    b = capi.MlaPagedBatch(fake, 64 * 576, 576, 10, 64, fake, fake, fake, 2, 4, 0)
    for k, v in kw.items():
        setattr(b, k, v)
    return ctypes.byref(b)


OK, BAD, MISALIGNED, LARGE = 0, 1, 2, 4


def test_attention_refuses_before_the_device(capi):
    f, p = capi.lib().mla_paged_attention_launcher, 0x10000
    need = capi.mla_paged_workspace_bytes(8, 16)

    def call(out=p, lse=p, q=p, b=None, T=8, H=16, scale=0.07, window=0, ws=p, nbytes=need):
        return f(out, lse, q, b if b is not None else batch(capi), T, H, scale, 1, window, ws, nbytes, None, 0, None)

    assert call(T=0) == OK and call(b=batch(capi, batch=0)) == OK
    for kw in (dict(T=-1), dict(H=0), dict(out=None), dict(q=None), dict(ws=None), dict(nbytes=need - 1), dict(scale=0.0),
               dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1)):
        assert call(**kw) == BAD, kw
    assert f(p, p, p, None, 8, 16, 0.07, 1, 0, p, need, None, 0, None) == BAD
    for kw in (dict(rows=None), dict(page_table=None), dict(q_start=None), dict(kv_len=None), dict(batch=-1), dict(num_pages=0),
               dict(page_size=0), dict(max_pages=0), dict(dtype=2), dict(dtype=7), dict(token_stride=575), dict(token_stride=580),
               dict(page_stride=4), dict(page_stride=64 * 576 + 1)):
        assert call(b=batch(capi, **kw)) == BAD, kw
    for kw in (dict(out=p + 8), dict(q=p + 2), dict(ws=p + 4), dict(b=batch(capi, rows=p + 8))):
        assert call(**kw) == MISALIGNED, kw
    assert call(T=1 << 24, H=128, nbytes=1 << 40) == LARGE
    assert call(b=batch(capi, batch=16385)) == LARGE
    assert call(b=batch(capi, max_pages=1 << 26, page_size=64)) == LARGE


def test_rope_refuses_before_the_device(capi):
    f, p = capi.lib().mla_rope_launcher, 0x10000

    def call(out=p, x=p, pos=p, freq=p, T=4, H=2, R=64, st=128, sh=64, dtype=0, inter=0):
        return f(out, x, pos, freq, T, H, R, st, sh, st, sh, dtype, inter, 0, 1.0, 0, None)

    assert call(T=0) == OK and call(H=0) == OK
    for kw in (dict(T=-1), dict(R=63), dict(R=0), dict(out=None), dict(x=None), dict(pos=None), dict(freq=None), dict(dtype=3)):
        assert call(**kw) == BAD, kw
    assert call(R=2050) == LARGE
    for kw in (dict(x=p + 1), dict(x=p + 2, inter=1), dict(sh=63, inter=1), dict(x=p + 2, dtype=2), dict(x=p + 4, dtype=2, inter=1)):
        assert call(**kw) == MISALIGNED, kw
    g = capi.lib().mla_rope_append_launcher

    def append(qo=p, q=p, c=p, k=p, b=None, freq=p, T=4, H=2, inter=0, kt=64):
        return g(qo, q, c, k, b if b is not None else batch(capi), freq, T, H, 128, 64, 128, 64, 512, kt, inter, 1.0, None, 0, None)

    assert append(T=0) == OK and append(b=batch(capi, batch=0)) == OK
    for kw in (dict(T=-1), dict(H=-1), dict(qo=None), dict(q=None), dict(c=None), dict(k=None), dict(freq=None),
               dict(b=batch(capi, token_stride=570)), dict(b=batch(capi, page_size=0)), dict(b=batch(capi, dtype=2))):
        assert append(**kw) == BAD, kw
    assert append(b=batch(capi, rows=p + 8)) == MISALIGNED and append(k=p + 2, inter=1) == MISALIGNED
    assert append(inter=1, kt=65) == MISALIGNED


def test_pages_refuse_before_the_device(capi):
    lib, p = capi.lib(), 0x10000
    assert lib.mla_pages_scratch_bytes(0, 4) == 0 and lib.mla_pages_scratch_bytes(10, 4) >= 4 * (16 + 30 + 15)

    def copy(pages=p, ls=1000, layers=2, P=10, pb=100, src=p, dst=p, n=3, scratch=p):
        return lib.mla_pages_copy_launcher(pages, ls, layers, P, pb, src, dst, n, scratch, None, 0, None)

    assert copy(n=0) == OK and copy(layers=0) == OK
    for kw in (dict(n=-1), dict(P=0), dict(pages=None), dict(pb=0), dict(ls=999), dict(src=None), dict(dst=None),
               dict(scratch=None), dict(layers=-1)):
        assert copy(**kw) == BAD, kw
    assert copy(n=(1 << 20) + 1) == LARGE and copy(scratch=p + 4) == MISALIGNED

    def extend(t=p, le=p, rc=p, slots=4, mp=4, P=10, ps=16, seqs=p, new=p, n=3, scratch=p):
        return lib.mla_pages_extend_launcher(t, le, rc, slots, mp, P, ps, seqs, new, n, scratch, None, 0, None)

    assert extend(n=0) == OK
    for kw in (dict(n=-1), dict(t=None), dict(le=None), dict(rc=None), dict(slots=0), dict(mp=0), dict(P=0), dict(ps=0),
               dict(seqs=None), dict(new=None), dict(scratch=None)):
        assert extend(**kw) == BAD, kw
    assert extend(n=(1 << 20) + 1) == LARGE and extend(scratch=p + 8) == MISALIGNED
    free = lib.mla_pages_free_launcher
    assert free(p, p, p, 4, 4, 10, 16, p, 0, None, 0, None) == OK
    assert free(p, p, p, 4, 4, 10, 16, None, 1, None, 0, None) == BAD
    assert free(p, p, p, 4, 4, 10, 0, p, 1, None, 0, None) == BAD
    fork = lib.mla_pages_fork_launcher
    assert fork(p, 1000, 2, 100, p, p, p, 4, 4, 10, 16, p, p, 0, p, None, 0, None) == OK
    assert fork(None, 1000, 2, 100, p, p, p, 4, 4, 10, 16, p, p, 1, p, None, 0, None) == BAD
    assert fork(p, 1000, 2, 100, p, p, p, 4, 4, 10, 16, p, None, 1, p, None, 0, None) == BAD
    compact = lib.mla_pages_compact_launcher
    assert compact(p, 1000, 2, 100, p, p, p, 4, 4, 10, 16, None, None, 0, None) == BAD
    assert compact(p, 999, 2, 100, p, p, p, 4, 4, 10, 16, p, None, 0, None) == BAD


def test_extension_refuses_cpu_tensors(built_libs):
    import cuda_agent_b200
    ext = cuda_agent_b200.load_extension()
    i = lambda *s: torch.zeros(*s, dtype=torch.int32)
    x, cache = torch.zeros(2, 3, 64), torch.zeros(4, 16, 576, dtype=torch.bfloat16)
    for bad in (lambda: ext.mla_rope_forward(x, i(2), torch.zeros(32, dtype=torch.float64)),
                lambda: ext.mla_rope_append_forward(x, x, x, cache, i(1, 4), i(2), i(1), x),
                lambda: ext.mla_paged_attention_forward(cache, cache, i(1, 4), i(2), i(1), 0.07),
                lambda: ext.mla_pages_copy(cache[None], i(1), i(1)), lambda: ext.mla_pages_extend(i(2, 4), i(2), i(4), i(1), i(1), 16),
                lambda: ext.mla_pages_fork(cache[None], i(2, 4), i(2), i(4), i(1), i(1)),
                lambda: ext.mla_pages_free(i(2, 4), i(2), i(4), i(1), 16),
                lambda: ext.mla_pages_compact(cache[None], i(2, 4), i(2), i(4))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            bad()


def test_cache_class_refuses(built_libs):
    from cuda_agent_b200.paged import PagedLatentCache
    for kw in (dict(layers=0), dict(pages=0), dict(page_size=0), dict(slots=0), dict(max_rows=0), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            PagedLatentCache(**{**dict(layers=1, pages=4, page_size=16, slots=2, max_rows=64, device="cpu"), **kw})
    c = PagedLatentCache(2, 5, 16, 3, 70, device="cpu")
    assert c.page_table.shape == (3, 5) and (c.page_table == -1).all() and c.pages_free() == 5
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        c.extend([0], [4])


def test_yarn_temperature_of_the_whole_score():
    """A checkpoint's two coefficients (a, b): the rotated columns' part of a score is multiplied by m(a)^2 in all, the latent
    part by m(b)^2; with equal ones that is one temperature of the whole score. In 64 bits, on rows of 512 + 64 columns."""
    from cuda_agent_b200.paged import rope_frequencies, rope_score_factor
    g = torch.Generator().manual_seed(0)
    q, k = torch.randn(576, generator=g, dtype=torch.float64), torch.randn(576, generator=g, dtype=torch.float64)
    plain, _ = rope_frequencies(64, scaling="yarn", factor=40.0, device="cpu")

    def rot(x, position, freq, factor):
        a, b = x[0::2], x[1::2]
        c, s = (position * freq).cos(), (position * freq).sin()
        return factor * torch.stack((a * c - b * s, b * c + a * s), -1).flatten()

    for a, b in ((1.0, 1.0), (0.707, 0.707), (1.0, 0.0), (0.5, 0.8), (0.0, 0.0)):
        freq, mscale = rope_frequencies(64, scaling="yarn", factor=40.0, device="cpu", mscale=a, mscale_all_dim=b)
        assert torch.equal(freq, plain)
        score = lambda ms: (q[:512] @ k[:512], rot(q[512:], 5000, freq, ms) @ rot(k[512:], 77, freq, ms))
        latent, turned = (v * rope_score_factor(40.0, b) for v in score(mscale))
        m_a, m_b = (0.1 * c * math.log(40.0) + 1 for c in (a, b))
        want = score(1.0)
        assert abs(latent - m_b ** 2 * want[0]) <= 1e-12 * abs(want[0]) and abs(turned - m_a ** 2 * want[1]) <= 1e-12 * abs(want[1])
        if a == b:
            assert abs(mscale - 1) < 1e-15
    assert rope_score_factor(1.0, 1.0) == 1.0
    for bad in (lambda: rope_score_factor(0.5, 1.0), lambda: rope_score_factor(2.0, -1.0),
                lambda: rope_frequencies(64, scaling="yarn", factor=2.0, device="cpu", mscale=-1.0)):
        with pytest.raises(ValueError):
            bad()


def test_batch_of_sequences_that_are_not_there_or_twice(built_libs):
    """A list raises; a tensor, which the host does not read, gives a place out of range no pages and length 0."""
    from cuda_agent_b200.paged import PagedLatentCache
    c = PagedLatentCache(1, 8, 16, 4, 64, device="cpu")
    c.page_table[:] = torch.arange(16, dtype=torch.int32).view(4, 4)
    c.length[:] = torch.tensor([5, 6, 7, 8], dtype=torch.int32)
    for bad in ([4], [0, -1], [1, 2, 1], [2 ** 40]):
        with pytest.raises(ValueError):
            c.batch(bad, [0] * (len(bad) + 1))
    for seqs, fine in (([2, 0], [1, 1]), ([3, 4, 0], [1, 0, 1]), ([-1, 3], [0, 1]), ([1, 2, 0, -5], [1, 1, 1, 0]),
                       ([9, 2 ** 40, -2 ** 40, 3, 0], [0, 0, 0, 1, 1]), ([2 ** 32 + 1, 2 ** 32, 1], [0, 0, 1]), ([], [])):
        b = c.batch(torch.tensor(seqs, dtype=torch.int64), list(range(len(seqs) + 1)))
        assert b.page_table.dtype == b.kv_len.dtype == b.q_start.dtype == torch.int32
        assert b.page_table.tolist() == [c.page_table[s].tolist() if f else [-1] * 4 for s, f in zip(seqs, fine)]
        assert b.kv_len.tolist() == [5 + s if f else 0 for s, f in zip(seqs, fine)]
        if all(fine):
            same = c.batch(seqs, list(range(len(seqs) + 1)))
            assert torch.equal(same.page_table, b.page_table) and torch.equal(same.kv_len, b.kv_len)


class OnTheGpu:
    """What the wrappers ask of a tensor, said of one that is on a GPU; its address is never used."""

    def __init__(self, t, cuda=True):
        self.t, self.is_cuda, self.shape, self.dtype = t, cuda, t.shape, t.dtype

    def __getattr__(self, name):
        return getattr(self.t, name)


def test_c_wrappers_pass_on_device_pointers_only(capi, monkeypatch):
    """A host address, or columns that are not next to one another, never reach a launcher."""
    calls = []

    class Lib:
        def __getattr__(self, name):
            return lambda *a: calls.append(name) or 0
    monkeypatch.setattr(capi, "lib", lambda: Lib())
    monkeypatch.setattr(capi, "_stream", lambda: 0)
    bf, i32 = torch.bfloat16, torch.int32
    gpu = lambda *s, dtype=bf: OnTheGpu(torch.zeros(*s, dtype=dtype))
    freq, table, start, kv = gpu(32, dtype=torch.float64), gpu(2, 4, dtype=i32), gpu(3, dtype=i32), gpu(2, dtype=i32)
    rope = dict(out=gpu(3, 2, 64), x=gpu(3, 2, 64), positions=gpu(3, dtype=i32), freq=freq)
    append = dict(q_out=gpu(3, 2, 64), q_pe=gpu(3, 2, 64), c_kv=gpu(3, 512), k_pe=gpu(3, 64), freq=freq)
    cache = dict(cache=gpu(4, 16, 576), page_table=table, q_start=start, kv_len=kv)
    batch = capi.mla_paged_batch(**cache)
    capi.mla_rope(**rope)
    capi.mla_rope_append(batch=batch, **append)
    assert calls == ["mla_rope_launcher", "mla_rope_append_launcher"]
    apart = lambda t: OnTheGpu(torch.zeros(*t.shape, 2, dtype=t.dtype)[..., 0])
    for f, args in ((capi.mla_rope, rope), (capi.mla_rope_append, {**append, "batch": batch}), (capi.mla_paged_batch, cache)):
        for name, t in args.items():
            if isinstance(t, OnTheGpu):
                for bad in (OnTheGpu(t.t, cuda=False), apart(t)):
                    with pytest.raises(ValueError):
                        f(**{**args, name: bad})
    assert len(calls) == 2


def test_attention_refuses_a_scale_beyond_float(capi):
    """The scale is taken in powers of two, which may pass the largest float where the scale itself does not."""
    p, need = 0x10000, capi.mla_paged_workspace_bytes(8, 16)

    def call(scale):                                 # rows not aligned: what comes after the look at the scale
        return capi.lib().mla_paged_attention_launcher(p, p, p, batch(capi, rows=p + 8), 8, 16, scale, 1, 0, p, need, None, 0, None)

    assert [call(scale) for scale in (2.4e38, 2.9e38, 3.4e38)] == [BAD] * 3 and call(2.3e38) == MISALIGNED

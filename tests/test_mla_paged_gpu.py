"""The paged latent cache on a GPU: rotary positions, the write of new rows, dense attention of new tokens.

Every result is compared with a statement in 64 bits (tests/paged_reference.py, where the tolerances are derived).
"""
import math
import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu
SCALE = 192 ** -0.5


@pytest.fixture(scope="module")
def ext(cuda_device):
    import cuda_agent_b200
    return cuda_agent_b200.load_extension()


def ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def make_batch(lens, heads, page, dtype, dev, seed=0, extra_tokens=0, spread=3.0, garbage=None, layers=None, pad=0,
               more_pages=0):
    """lens: [(new tokens, cached rows)]. Rows behind a sequence's end and unused pages hold `garbage` if given."""
    g = torch.Generator(device=dev).manual_seed(seed)
    need = [-(-max(k, 0) // page) for _, k in lens]
    pool = sum(need) + 2
    shape = (pool, page, 576 + pad) if layers is None else (pool, layers, page, 576 + pad)
    store = torch.randn(shape, generator=g, device=dev).to(dtype)
    cache = (store if layers is None else store[:, layers - 1])[..., :576]
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(lens), max(need + [1]) + more_pages), -1, dtype=torch.int32, device=dev)
    at = 0
    live = torch.zeros(pool, page, dtype=torch.bool, device=dev)
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        for i in range(n):
            live[order[at + i].long(), :min(page, lens[b][1] - i * page)] = True
        at += n
    if garbage is not None:
        cache[~live] = garbage
    start = [0]
    for n, _ in lens:
        start.append(start[-1] + n)
    q = (spread * math.sqrt(192 / 576) * torch.randn(start[-1] + extra_tokens, heads, 576, generator=g, device=dev)).to(dtype)
    return q, cache, table, ints(start, dev), ints([k for _, k in lens], dev)


def check_attention(ext, args, causal=True, window=0, scale=SCALE, **kw):
    out, lse = ext.mla_paged_attention_forward(*args, scale, causal, window, check=True, **kw)
    want, want_lse, tol, tol_lse = ref.attention(*args, scale, causal, window)
    off = (out.double() - want).abs() - tol
    assert out.dtype == args[0].dtype and lse.dtype == torch.float32
    assert torch.isfinite(out).all()
    assert (off <= 0).all(), (off.max().item(), off.argmax().item())
    dead = want_lse == -math.inf
    assert torch.equal(dead, lse == -math.inf)
    assert ((lse.double() - want_lse)[~dead].abs() <= tol_lse[~dead]).all()
    assert (out[dead] == 0).all()
    return out, lse


# ------------------------------------------------------------------------------------------------ rotary positions
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("T,H,R", [(1, 1, 2), (1, 128, 64), (3, 5, 6), (7, 3, 24), (33, 16, 64), (300, 1, 128), (2, 9, 2048),
                                   (1200, 4, 64)])
def test_rope_matches_the_formula(ext, cuda_device, dtype, interleaved, inverse, T, H, R):
    g = torch.Generator(device=cuda_device).manual_seed(T * H + R)
    x = torch.randn(T, H, R, generator=g, device=cuda_device).to(dtype)
    pos = torch.randint(0, 1 << 20, (T,), generator=g, device=cuda_device, dtype=torch.int32)
    pos[0] = 2 ** 31 - 1
    freq = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64, device=cuda_device) * 2 / R)
    got = ext.mla_rope_forward(x, pos, freq, interleaved, 1.25, inverse)
    want, tol = ref.rotate(x, pos, freq, interleaved, 1.25, inverse)
    assert ((got.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("offset", [512, 8, 3, 2])
def test_rope_on_a_part_of_the_head(ext, cuda_device, interleaved, offset):
    """A view as input, the same view as output, another part of the same rows as output; what is beside stays."""
    if interleaved and offset % 2:
        pytest.skip("refused: see test_rope_refusals")
    g = torch.Generator(device=cuda_device).manual_seed(offset)
    full = torch.randn(37, 6, 640, generator=g, device=cuda_device).to(torch.bfloat16)
    pos = torch.arange(37, dtype=torch.int32, device=cuda_device) * 1000
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    x = full[..., offset:offset + 64]
    want, tol = ref.rotate(x, pos, freq, interleaved)
    assert ((ext.mla_rope_forward(x, pos, freq, interleaved).double() - want).abs() <= tol).all()
    before = full.clone()
    other = full[..., 576:640] if offset == 512 else full[..., 512:576]
    ext.mla_rope_forward(x, pos, freq, interleaved, out=other)
    assert ((other.double() - want).abs() <= tol).all()
    ext.mla_rope_forward(x, pos, freq, interleaved, out=x)
    assert ((x.double() - want).abs() <= tol).all()
    keep = torch.ones(640, dtype=torch.bool, device=cuda_device)
    keep[offset:offset + 64] = False
    keep[576:640] = keep[576:640] & (offset != 512)
    keep[512:576] = keep[512:576] & (offset == 512)
    assert torch.equal(full[..., keep], before[..., keep])


def test_rope_broadcast_transposed_and_empty(ext, cuda_device):
    pos = torch.arange(5, dtype=torch.int32, device=cuda_device)
    freq = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64, device=cuda_device)
    one = torch.randn(5, 1, 8, device=cuda_device).expand(5, 12, 8)
    want, tol = ref.rotate(one, pos, freq)
    assert ((ext.mla_rope_forward(one, pos, freq).double() - want).abs() <= tol).all()
    x = torch.randn(12, 5, 8, device=cuda_device).transpose(0, 1)
    out = torch.empty(12, 5, 8, device=cuda_device).transpose(0, 1)
    want, tol = ref.rotate(x, pos, freq)
    ext.mla_rope_forward(x, pos, freq, out=out)
    assert ((out.double() - want).abs() <= tol).all()
    assert ext.mla_rope_forward(x[:0], pos[:0], freq).shape == (0, 12, 8)


def test_rope_inverse_is_the_gradient(ext, cuda_device):
    """Against differences in 64 bits of the rotation, and <y, R x> = <R' y, x> of the kernels themselves."""
    g = torch.Generator(device=cuda_device).manual_seed(3)
    x = torch.randn(9, 4, 16, generator=g, device=cuda_device)
    dy = torch.randn(9, 4, 16, generator=g, device=cuda_device)
    pos = torch.randint(0, 5000, (9,), generator=g, device=cuda_device, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(8, dtype=torch.float64, device=cuda_device) / 8)
    for interleaved in (False, True):
        dx = ext.mla_rope_forward(dy, pos, freq, interleaved, 1.5, True)
        step = 1e-6 * torch.randn(9, 4, 16, generator=g, device=cuda_device, dtype=torch.float64)
        up, _ = ref.rotate(x.double() + step, pos, freq, interleaved, 1.5)
        down, _ = ref.rotate(x.double() - step, pos, freq, interleaved, 1.5)
        slope = ((up - down) * dy.double()).sum((1, 2)) / 2
        size = (dx.double().abs() * step.abs()).sum((1, 2))
        assert ((slope - (dx.double() * step).sum((1, 2))).abs() <= 1e-5 * size + 1e-12).all()


# ------------------------------------------------------------------------------------------------ new rows
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lens,heads,page", [([(1, 1)], 1, 1), ([(1, 300), (1, 17), (1, 64)], 128, 16),
                                             ([(70, 90), (0, 50), (3, 3), (0, 0)], 5, 48), ([(513, 1000)], 16, 64)])
def test_append_writes_rows_and_rotates(ext, cuda_device, dtype, interleaved, lens, heads, page):
    _, cache, table, start, kv = make_batch(lens, 1, page, dtype, cuda_device, layers=2)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    T = start[-1].item() + 3                       # three tokens behind the last sequence
    joint = torch.randn(T, 576 + 8, generator=g, device=cuda_device).to(dtype)
    c_kv, k_pe = joint[:, :512], joint[:, 520:]
    q_pe = torch.randn(T, heads, 64, generator=g, device=cuda_device).to(dtype)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    q = torch.randn(T, heads, 576, generator=g, device=cuda_device).to(dtype)
    q0, cache0 = q.clone(), cache.clone()
    ext.mla_rope_append_forward(q_pe, c_kv, k_pe, cache, table, start, kv, freq, q[..., 512:], interleaved, 1.1, check=True)
    pos, touched = torch.zeros(T, dtype=torch.int32), torch.zeros(cache.shape[:2], dtype=torch.bool)
    n_live = start[-1].item()
    place = []
    for b, (n, k) in enumerate(lens):
        for i in range(n):
            p = k - n + i
            pos[start[b].item() + i] = p
            place.append((table[b, p // page].item(), p % page))
    pos = pos.to(cuda_device)
    want, tol = ref.rotate(q_pe, pos, freq, interleaved, 1.1)
    assert ((q[..., 512:].double() - want).abs() <= tol)[:n_live].all()
    assert torch.equal(q[..., :512], q0[..., :512]) and torch.equal(q[n_live:], q0[n_live:])
    want, tol = ref.rotate(k_pe[:, None], pos, freq, interleaved, 1.1)
    for t, (a, r) in enumerate(place):
        touched[a, r] = True
        assert torch.equal(cache[a, r, :512], c_kv[t])
        assert ((cache[a, r, 512:].double() - want[t, 0]).abs() <= tol[t, 0]).all()
    assert torch.equal(cache[~touched], cache0[~touched])
    # a fresh output: the same rotation, zeros behind the last sequence
    fresh = ext.mla_rope_append_forward(q_pe, c_kv, k_pe, cache, table, start, kv, freq, None, interleaved, 1.1)
    assert torch.equal(fresh[:n_live], q[:n_live, :, 512:]) and (fresh[n_live:] == 0).all()


def test_append_unaligned_views_and_bad_pages(ext, cuda_device):
    dtype = torch.bfloat16
    _, cache, table, start, kv = make_batch([(5, 40), (4, 20)], 1, 8, dtype, cuda_device)
    T = 9
    base = torch.randn(T, 3, 67, device=cuda_device).to(dtype)
    joint = torch.randn(T, 600, device=cuda_device).to(dtype)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    q = ext.mla_rope_append_forward(base[..., 3:], joint[:, 5:517], joint[:, 519:583], cache, table, start, kv, freq)
    pos = torch.cat((torch.arange(35, 40), torch.arange(16, 20))).to(cuda_device, torch.int32)
    want, tol = ref.rotate(base[..., 3:], pos, freq)
    assert ((q.double() - want).abs() <= tol).all()
    assert torch.equal(cache[table[1, 2].long(), 3, :512], joint[8, 5:517])
    # entries outside the pool and tables that are too short: nothing is written there, and the call says so
    before = cache.clone()
    for bad in (-1, cache.shape[0], 2 ** 31 - 1):
        broken = table.clone()
        broken[0, 4] = bad
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_rope_append_forward(base[..., 3:], joint[:, 5:517], joint[:, 519:583], cache, broken, start, kv, freq,
                                        check=True)
        assert torch.equal(cache, before)
    for lens in ([1000, 20], [2, 20]):               # beyond the table; before the first position
        moved = cache.clone()
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_rope_append_forward(base[..., 3:], joint[:, 5:517], joint[:, 519:583], moved, table, start,
                                        ints(lens, cuda_device), freq, check=True)
        assert torch.equal(moved[table[1, :3].long()], before[table[1, :3].long()])


# ------------------------------------------------------------------------------------------------ attention
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads", [1, 16, 128])
@pytest.mark.parametrize("kv", [1, 2, 63, 64, 65, 128, 129, 1000])
def test_attention_one_token(ext, cuda_device, dtype, heads, kv):
    check_attention(ext, make_batch([(1, kv)], heads, 16, dtype, cuda_device, seed=kv, garbage=math.nan))


@pytest.mark.parametrize("page", [1, 2, 3, 8, 16, 48, 64, 100, 128, 256])
def test_attention_page_sizes(ext, cuda_device, page):
    check_attention(ext, make_batch([(3, 200), (1, 257), (70, 70)], 20, page, torch.bfloat16, cuda_device, seed=page,
                                    garbage=math.inf))


@pytest.mark.parametrize("heads", [1, 3, 7, 24, 64, 127, 130, 200])
def test_attention_head_counts(ext, cuda_device, heads):
    check_attention(ext, make_batch([(5, 100), (0, 40), (1, 333), (37, 150)], heads, 32, torch.bfloat16, cuda_device, seed=heads))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 100, 2 ** 31 - 1])
def test_attention_masks(ext, cuda_device, causal, window):
    args = make_batch([(130, 400), (64, 64), (1, 500), (9, 9)], 9, 16, torch.float16, cuda_device, seed=window % 97, garbage=math.nan)
    check_attention(ext, args, causal, window)


def test_attention_rows_that_see_nothing(ext, cuda_device):
    """More new tokens than rows, empty histories, empty places of the batch, tokens of no sequence."""
    args = make_batch([(10, 4), (3, 0), (0, 0), (200, 130), (0, 12), (1, 1)], 40, 16, torch.bfloat16, cuda_device,
                      extra_tokens=5, garbage=math.nan)
    out, lse = check_attention(ext, args)
    assert (out[-5:] == 0).all() and (lse[-5:] == -math.inf).all()
    mine, mine_lse = torch.full_like(out, 7.0), torch.full_like(lse, 7.0)
    ext.mla_paged_attention_forward(*args, SCALE, out=mine, lse=mine_lse)
    assert torch.equal(mine[:-5], out[:-5]) and (mine[-5:] == 7).all()
    assert torch.equal(mine_lse[:-5], lse[:-5]) and (mine_lse[-5:] == 7).all()
    check_attention(ext, args, causal=False, window=3)


def test_attention_empty_calls(ext, cuda_device):
    q, cache, table, start, kv = make_batch([(2, 5)], 4, 16, torch.bfloat16, cuda_device)
    out, lse = ext.mla_paged_attention_forward(q[:0], cache, table, start * 0, kv, SCALE)
    assert out.shape == (0, 4, 512) and lse.shape == (0, 4)
    out, lse = ext.mla_paged_attention_forward(q, cache, table[:0], start[:1], kv[:0], SCALE)
    assert (out == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("lens", [[(1, 20000)], [(1, 9000)] * 5 + [(1, 3)], [(4, 5000), (300, 700), (1, 1), (2, 4097)],
                                  [(1, 1 + 7 * b) for b in range(300)], [(b % 3, b % 50) for b in range(1000)]])
def test_attention_work_division(ext, cuda_device, lens):
    check_attention(ext, make_batch(lens, 16, 64, torch.bfloat16, cuda_device, seed=len(lens)))


def test_attention_strided_cache(ext, cuda_device):
    check_attention(ext, make_batch([(20, 300), (1, 90)], 16, 32, torch.bfloat16, cuda_device, layers=3, pad=64, garbage=math.nan))


@pytest.mark.parametrize("spread", [0.0, 40.0])
def test_attention_score_ranges(ext, cuda_device, spread):
    """Equal scores; scores hundreds apart whose maximum comes late (the reference maximum moves, O is rescaled)."""
    q, cache, table, start, kv = make_batch([(40, 900), (1, 700)], 16, 16, torch.bfloat16, cuda_device, spread=spread)
    for b in range(2):
        n = -(-kv[b].item() // 16)
        cache[table[b, :n].long()] *= torch.linspace(0.05, 1.0, n, device=cuda_device)[:, None, None].to(torch.bfloat16)
    check_attention(ext, (q, cache, table, start, kv))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("blocks", ["even", "odd", "any"])
def test_attention_maxima_that_rise_in_some_blocks(ext, cuda_device, blocks, dtype):
    """Runs of 64 rows with keys up to 40 times as long: a row's maximum rises far in the keys of one CTA of a pair or of
    the other, in some lane quadrants and not in others, early and late in a run."""
    q, cache, table, start, kv = make_batch([(3, 3000), (50, 1500), (1, 130)], 50, 32, dtype, cuda_device, seed=9)
    g = torch.Generator().manual_seed(3)
    for b in range(3):
        for i in range(0, kv[b].item(), 64):
            long_one = torch.rand((), generator=g).item() < 0.3 and (blocks == "any" or (i // 64) % 2 == (blocks == "odd"))
            if long_one:
                for page in table[b, i // 32:min(i // 32 + 2, -(-kv[b].item() // 32))].tolist():
                    cache[page] *= 1 + 39 * torch.rand((), generator=g).item()
    check_attention(ext, (q, cache, table, start, kv), scale=SCALE / 4)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("scale", [1e3, 1e5, 1e7, 1e30])
def test_attention_scores_beyond_whole_numbers(ext, cuda_device, scale, dtype):
    """Scores so large that fp32 holds them to whole units or worse: the key that each query repeats wins alone (another
    key's score is smaller by some 400 of 576, so far more than any rounding; 1e30 times 2^10 stays finite). From 1e5 on
    its score in powers of two, 8e7 and more, is a whole number, as is the reference: the weight is a power of two and the
    values come back as they are. At 1e3 it is 8e5 with a fraction f: the weight 2^-f is rounded to the 16-bit type on its
    way into the product, half a step, and not in the sum that it is divided by, and the result is rounded once more:
    two half steps, and the fp32 product and quotient (2^-22 is ample)."""
    q, cache, table, start, kv = make_batch([(7, 300), (2, 150)], 16, 16, dtype, cuda_device, seed=5)
    picked = torch.randint(0, 140, (9, 16), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    b = (torch.arange(9, device=cuda_device) >= 7).long()
    rows = cache[table[b[:, None], picked // 16].long(), picked % 16]
    out, _ = ext.mla_paged_attention_forward(rows, cache, table, start, kv, scale, check=True)
    if scale >= 1e5:
        assert torch.equal(out, rows[..., :512])
    want = rows[..., :512].double()
    assert ((out.double() - want).abs() <= want.abs() * ((1 + torch.finfo(dtype).eps / 2) ** 2 - 1 + 2.0 ** -22)).all()


def test_attention_nan_and_inf_in_a_query_stay_in_its_row(ext, cuda_device):
    args = make_batch([(6, 200), (1, 150)], 16, 16, torch.bfloat16, cuda_device)
    clean, _ = ext.mla_paged_attention_forward(*args, SCALE)
    args[0][2, 3, 10] = math.nan
    args[0][6, 1, 570] = math.inf
    out, lse = ext.mla_paged_attention_forward(*args, SCALE, check=True)
    assert out[2, 3].isnan().all() and lse[2, 3].isnan() and out[6, 1].isnan().all()
    same = torch.ones(7, 16, dtype=torch.bool, device=cuda_device)
    same[2, 3] = same[6, 1] = False
    assert torch.equal(out[same], clean[same])


def test_attention_bad_pages_and_long_lengths(ext, cuda_device):
    args = list(make_batch([(3, 200), (2, 150)], 16, 16, torch.bfloat16, cuda_device))
    for bad in (-1, args[1].shape[0], 2 ** 31 - 1, -2 ** 31):
        table = args[2].clone()
        table[0, 5] = bad
        broken = (args[0], args[1], table, args[3], args[4])
        with pytest.raises(RuntimeError, match="page table"):
            ext.mla_paged_attention_forward(*broken, SCALE, check=True)
        out, _ = ext.mla_paged_attention_forward(*broken, SCALE)
        want, _, tol, _ = ref.attention(*broken, SCALE)
        assert ((out.double() - want).abs() <= tol).all()
    args[4] = ints([2 ** 31 - 1, -5], cuda_device)    # read as 208 (13 pages of 16) and as 0
    args[2][0] = args[2][0].clamp_min(0)
    out, lse = ext.mla_paged_attention_forward(*args, SCALE, check=True)
    want, _, tol, _ = ref.attention(*args, SCALE)
    assert ((out.double() - want).abs() <= tol).all() and (out[3:] == 0).all()


def test_attention_far_pages(ext, cuda_device):
    """Rows whose offset in the cache passes 2^31 elements and 2^32 bytes."""
    page, pool = 64, 60000                            # 2.2e9 elements, 4.4e9 bytes
    cache = torch.empty(pool, page, 576, dtype=torch.bfloat16, device=cuda_device)
    ids = [59999, 1, 59000, 58255]
    g = torch.Generator(device=cuda_device).manual_seed(4)
    for i in ids:
        cache[i] = torch.randn(page, 576, generator=g, device=cuda_device).to(torch.bfloat16)
    q = torch.randn(2, 16, 576, generator=g, device=cuda_device).to(torch.bfloat16)
    args = (q, cache, ints([ids], cuda_device), ints([0, 2], cuda_device), ints([250], cuda_device))
    small = (q, cache[ids], ints([[0, 1, 2, 3]], cuda_device), args[3], args[4])
    out, _ = ext.mla_paged_attention_forward(*args, SCALE, check=True)
    want, _, tol, _ = ref.attention(*small, SCALE)
    assert ((out.double() - want).abs() <= tol).all()
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    c_kv = torch.randn(2, 512, generator=g, device=cuda_device).to(torch.bfloat16)
    ext.mla_rope_append_forward(q[..., :64].contiguous(), c_kv, c_kv[:, :64].contiguous(), *args[1:], freq, check=True)
    assert torch.equal(cache[58255, 56:58, :512], c_kv)


def test_attention_repeats_exactly_on_streams_and_in_graphs(ext, cuda_device):
    """The same bits again, on another stream beside other work, and replayed from a graph with other lengths."""
    args = make_batch([(1, 3000), (20, 900), (1, 77), (0, 5)], 16, 64, torch.bfloat16, cuda_device)
    first = ext.mla_paged_attention_forward(*args, SCALE)
    second = make_batch([(2, 1500), (5, 800)], 16, 64, torch.bfloat16, cuda_device, seed=9)
    want2 = ext.mla_paged_attention_forward(*second, SCALE)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(10):
        with torch.cuda.stream(s1):
            a = ext.mla_paged_attention_forward(*args, SCALE)
        with torch.cuda.stream(s2):
            b = ext.mla_paged_attention_forward(*second, SCALE)
        got.append((a, b))
    torch.cuda.synchronize()
    for a, b in got:
        assert all(torch.equal(x, y) for x, y in zip(a, first)) and all(torch.equal(x, y) for x, y in zip(b, want2))
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = ext.mla_paged_attention_forward(*args, SCALE)
    with torch.cuda.graph(g2):
        o2 = ext.mla_paged_attention_forward(*second, SCALE)
    for s, g in ((s1, g1), (s2, g2)) * 3:
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o1[0], first[0]) and torch.equal(o2[0], want2[0])
    args[4].copy_(ints([2000, 850, 70, 1], cuda_device))
    g1.replay()
    torch.cuda.synchronize()
    want, _, tol, _ = ref.attention(*args, SCALE)
    assert ((o1[0].double() - want).abs() <= tol).all()


def test_attention_through_the_c_abi(ext, cuda_device):
    from cuda_agent_b200 import capi
    q, cache, table, start, kv = make_batch([(4, 100), (1, 300)], 16, 16, torch.bfloat16, cuda_device)
    out = torch.full((5, 16, 512), math.nan, dtype=q.dtype, device=cuda_device)
    lse = torch.empty(5, 16, device=cuda_device)
    status = torch.ones(1, dtype=torch.int32, device=cuda_device)
    work = torch.empty(capi.mla_paged_workspace_bytes(5, 16), dtype=torch.uint8, device=cuda_device)
    batch = capi.mla_paged_batch(cache, table, start, kv)
    capi.mla_paged_attention(out, lse, q, batch, SCALE, workspace=work, status=status)
    want = ext.mla_paged_attention_forward(q, cache, table, start, kv, SCALE)
    assert status.item() == 0 and torch.equal(out, want[0]) and torch.equal(lse, want[1])
    capi.mla_paged_attention(out, None, q, batch, SCALE, workspace=work)      # no lse wanted
    assert torch.equal(out, want[0])
    with pytest.raises(capi.CabError):
        capi.mla_paged_attention(out, lse, q, batch, SCALE, workspace=work[:64])
    x = torch.randn(5, 3, 8, device=cuda_device)
    freq = torch.ones(4, dtype=torch.float64, device=cuda_device)
    y = torch.empty_like(x)
    capi.mla_rope(y, x, start[:1].expand(5).contiguous(), freq)
    assert torch.equal(y, x)                          # position 0


# ------------------------------------------------------------------------------------------------ refusals
def test_rope_refusals(ext, cuda_device):
    x = torch.randn(4, 2, 8, device=cuda_device)
    pos = torch.zeros(4, dtype=torch.int32, device=cuda_device)
    freq = torch.ones(4, dtype=torch.float64, device=cuda_device)
    for bad in (lambda: ext.mla_rope_forward(x[..., :7], pos, freq), lambda: ext.mla_rope_forward(x, pos[:3], freq),
                lambda: ext.mla_rope_forward(x, pos, freq[:3]), lambda: ext.mla_rope_forward(x, pos, freq.float()),
                lambda: ext.mla_rope_forward(x, pos.long(), freq), lambda: ext.mla_rope_forward(x.double(), pos, freq),
                lambda: ext.mla_rope_forward(x.cpu(), pos, freq), lambda: ext.mla_rope_forward(x, pos.cpu(), freq),
                lambda: ext.mla_rope_forward(x.transpose(1, 2), pos, freq[:1]),
                lambda: ext.mla_rope_forward(x, pos, freq, out=x[:, :1].expand(4, 2, 8)),
                lambda: ext.mla_rope_forward(x, pos, freq, out=x[:3]), lambda: ext.mla_rope_forward(x, pos, freq, out=x.half()),
                lambda: ext.mla_rope_forward(torch.randn(4, 1, 4098, device=cuda_device), pos,
                                             torch.ones(2049, dtype=torch.float64, device=cuda_device))):
        with pytest.raises(RuntimeError):
            bad()
    wide = torch.randn(4, 2, 20, device=cuda_device)
    with pytest.raises(RuntimeError, match="overlap"):
        ext.mla_rope_forward(wide[..., :8], pos, freq, out=wide[..., 4:12])
    with pytest.raises(RuntimeError, match="aligned"):
        ext.mla_rope_forward(wide[..., 1:9], pos, freq, True)


def test_attention_and_append_refusals(ext, cuda_device):
    q, cache, table, start, kv = make_batch([(2, 40)], 4, 16, torch.bfloat16, cuda_device)
    f = ext.mla_paged_attention_forward
    for bad in (lambda: f(q.half(), cache, table, start, kv, SCALE), lambda: f(q[..., :512].contiguous(), cache, table, start, kv, SCALE),
                lambda: f(q, cache[..., :512], table, start, kv, SCALE), lambda: f(q.float(), cache.float(), table, start, kv, SCALE),
                lambda: f(q, cache, table.long(), start, kv, SCALE), lambda: f(q, cache, table, start[:1], kv, SCALE),
                lambda: f(q, cache, table.repeat(2, 1), start, kv, SCALE), lambda: f(q, cache, table, start, kv, 0.0),
                lambda: f(q, cache, table, start, kv, -1.0), lambda: f(q, cache, table, start, kv, math.nan),
                lambda: f(q, cache, table, start, kv, SCALE, True, -1), lambda: f(q, cache, table.cpu(), start, kv, SCALE),
                lambda: f(q.transpose(0, 1), cache, table, start, kv, SCALE), lambda: f(q, cache, table[:, :0], start, kv, SCALE),
                lambda: f(q, cache, table, start, kv, SCALE, out=q[..., :512]),
                lambda: f(q, cache, table, start, kv, SCALE, lse=torch.empty(2, 4, device=cuda_device)),
                lambda: f(q, torch.empty(40, 16, 580, dtype=q.dtype, device=cuda_device)[..., :576], table, start, kv, SCALE),
                lambda: f(q, torch.empty(40, 16, 640, dtype=q.dtype, device=cuda_device)[..., 1:577], table, start, kv, SCALE)):
        with pytest.raises(RuntimeError):
            bad()
    freq = torch.ones(32, dtype=torch.float64, device=cuda_device)
    q_pe, c_kv, k_pe = q[..., :64], q[:, 0, :512], q[:, 0, 512:]
    a = ext.mla_rope_append_forward
    for bad in (lambda: a(q_pe, c_kv[:1], k_pe, cache, table, start, kv, freq), lambda: a(q_pe, c_kv, k_pe[:, :32], cache, table, start, kv, freq),
                lambda: a(q_pe, c_kv, k_pe, cache, table, start, kv, freq[:31]), lambda: a(q_pe.half(), c_kv, k_pe, cache, table, start, kv, freq),
                lambda: a(q_pe, c_kv, k_pe, cache, table, start, kv, freq, q[..., 32:96]),
                lambda: a(q_pe, cache[0, :2, :512], k_pe, cache, table, start, kv, freq)):
        with pytest.raises(RuntimeError):
            bad()


def test_attention_outputs_in_one_buffer_with_the_inputs(ext, cuda_device):
    """Views of one buffer are fine as long as no byte is shared; out or lse over an input, or over each other, is refused."""
    args = make_batch([(3, 40)], 4, 16, torch.bfloat16, cuda_device)
    q, T, H = args[0], 3, 4
    store = torch.zeros(T * H * (576 + 512 + 2), dtype=torch.bfloat16, device=cuda_device)
    q2 = store[:T * H * 576].view(T, H, 576)
    out = store[T * H * 576:T * H * 1088].view(T, H, 512)
    lse = store[T * H * 1088:].view(torch.float32).view(T, H)
    q2.copy_(q)
    want, want_lse = ext.mla_paged_attention_forward(*args, SCALE)
    ext.mla_paged_attention_forward(q2, *args[1:], SCALE, out=out, lse=lse, check=True)
    assert torch.equal(out, want) and torch.equal(lse, want_lse) and torch.equal(q2, q)
    half = T * H * 512
    for bad in (dict(out=store[:half].view(T, H, 512)), dict(out=store[T * H * 576 - 8:][:half].view(T, H, 512)),
                dict(out=args[1].reshape(-1)[:half].view(T, H, 512)),
                dict(out=out, lse=store[:2 * T * H].view(torch.float32).view(T, H)),
                dict(out=out, lse=out.view(-1)[:2 * T * H].view(torch.float32).view(T, H))):
        with pytest.raises(RuntimeError, match="overlap"):
            ext.mla_paged_attention_forward(q2, *args[1:], SCALE, **bad)
    assert torch.equal(out, want) and torch.equal(q2, q)


@pytest.mark.parametrize("batch", [3, 32, 40, 500])
def test_attention_with_starts_that_descend_does_nothing(ext, cuda_device, batch):
    """They would give tokens to several sequences at once. The outputs stay as they were, and the next call is sound."""
    args = make_batch([(2, 40)] * batch, 4, 16, torch.bfloat16, cuda_device)
    q, cache, table, start, kv = args
    wrong = start.clone()
    wrong[batch // 2] = 2 * batch
    out = torch.full((2 * batch, 4, 512), 7.0, dtype=q.dtype, device=cuda_device)
    lse = torch.full((2 * batch, 4), 7.0, device=cuda_device)
    with pytest.raises(RuntimeError, match="q_start descends"):
        ext.mla_paged_attention_forward(q, cache, table, wrong, kv, SCALE, out=out, lse=lse, check=True)
    assert (out == 7).all() and (lse == 7).all()
    check_attention(ext, args)


WRONG_STARTS = {"begin_late": (0, 1), "begin_below": (0, -1), "descend": (1, 10 ** 6), "end_low": (-1, -3), "end_early": (-1, 1),
                "end_late": (-1, 10 ** 6)}


def wrong_starts(start, kind):
    at, value = WRONG_STARTS[kind]
    wrong = start.clone()
    wrong[at] = min(value, start[-1].item() + 1)
    return wrong


@pytest.mark.parametrize("batch", [2, 32, 300])
@pytest.mark.parametrize("kind", list(WRONG_STARTS))
def test_append_with_wrong_starts_writes_nothing(ext, cuda_device, kind, batch):
    """Starts that do not begin at 0, descend or pass the tokens: rows of earlier tokens and of other sequences stay, as do the
    queries; a call with the right ones goes through after it."""
    _, cache, table, start, kv = make_batch([(2, 40)] * batch, 1, 16, torch.bfloat16, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(2)
    T, heads = 2 * batch, 3
    joint = torch.randn(T, 576, generator=g, device=cuda_device).to(torch.bfloat16)
    q_pe = torch.randn(T, heads, 64, generator=g, device=cuda_device).to(torch.bfloat16)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    q = torch.full((T, heads, 64), 7.0, dtype=torch.bfloat16, device=cuda_device)
    before, wrong = cache.clone(), wrong_starts(start, kind)
    with pytest.raises(RuntimeError, match="q_start"):
        ext.mla_rope_append_forward(q_pe, joint[:, :512], joint[:, 512:], cache, table, wrong, kv, freq, q, check=True)
    assert torch.equal(cache, before) and (q == 7).all()
    fresh = ext.mla_rope_append_forward(q_pe, joint[:, :512], joint[:, 512:], cache, table, wrong, kv, freq)
    assert torch.equal(cache, before) and (fresh == 0).all()
    ext.mla_rope_append_forward(q_pe, joint[:, :512], joint[:, 512:], cache, table, start, kv, freq, q, check=True)
    at = table[:, 2].long()
    assert torch.equal(cache[at, 6:8, :512].reshape(T, 512), joint[:, :512]) and not (q == 7).all()


@pytest.mark.parametrize("batch", [2, 32, 300])
@pytest.mark.parametrize("kind", list(WRONG_STARTS))
def test_attention_with_wrong_starts_returns_no_old_memory(ext, cuda_device, kind, batch):
    """Fresh outputs come from memory that held something else: zeros and -infinity, also where nobody asks for the status.
    Outputs that are given stay as they were."""
    args = make_batch([(2, 40)] * batch, 4, 16, torch.bfloat16, cuda_device)
    q, cache, table, start, kv = args
    wrong = wrong_starts(start, kind)
    for check in (False, True):
        poison = [torch.full((2 * batch, 4, 512), 7.0, dtype=q.dtype, device=cuda_device) for _ in range(4)]
        poison += [torch.full((2 * batch, 4), 7.0, device=cuda_device) for _ in range(4)]
        del poison
        if check:
            with pytest.raises(RuntimeError, match="q_start"):
                ext.mla_paged_attention_forward(q, cache, table, wrong, kv, SCALE, check=True)
        else:
            out, lse = ext.mla_paged_attention_forward(q, cache, table, wrong, kv, SCALE)
            assert (out == 0).all() and (lse == -math.inf).all()
    out = torch.full((2 * batch, 4, 512), 7.0, dtype=q.dtype, device=cuda_device)
    lse = torch.full((2 * batch, 4), 7.0, device=cuda_device)
    ext.mla_paged_attention_forward(q, cache, table, wrong, kv, SCALE, out=out, lse=lse)
    assert (out == 7).all() and (lse == 7).all()
    check_attention(ext, args)


def test_rope_between_views_of_one_buffer(ext, cuda_device):
    """Inputs and outputs anywhere in one buffer, with any strides: what shares bytes without being the same view is refused,
    what is accepted is right. Which bytes a view has is counted element by element."""
    rng, accepted, refused = random.Random(7), 0, 0
    freq = torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64, device=cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(1)
    base = torch.randn(1000, generator=g, device=cuda_device)
    places = [((2, 3, 8), (100, 30, 1), 0, (100, 30, 1), 40), ((2, 3, 8), (100, 30, 1), 0, (100, 30, 1), 8),
              ((3, 4, 8), (64, 16, 1), 8, (64, 16, 1), 0), ((1, 3, 8), (100, 16, 1), 0, (48, 16, 1), 0),
              ((2, 1, 8), (16, 50, 1), 4, (16, 8, 1), 4)]
    for _ in range(1500):
        shape = (rng.randint(1, 4), rng.randint(1, 4), 8)
        strides = [(rng.choice([8, 16, 24, 30, 48, 64, 100, 120]), rng.choice([8, 9, 16, 24, 30, 40]), 1) for _ in range(2)]
        if rng.random() < 0.7:
            strides[1] = strides[0]
        places.append((shape, strides[0], rng.randint(0, 200), strides[1], rng.randint(0, 200)))
    for shape, sx, ox, so, oo in places:
        def elements(strides, offset):
            return [offset + i * strides[0] + j * strides[1] + c for i in range(shape[0]) for j in range(shape[1]) for c in range(8)]
        a, b = elements(sx, ox), elements(so, oo)
        same = a == b
        if len(set(b)) < len(b):
            continue                                  # an output whose own rows overlap: another refusal
        store = base.clone()
        x, out = torch.as_strided(store, shape, sx, ox), torch.as_strided(store, shape, so, oo)
        pos = torch.arange(shape[0], dtype=torch.int32, device=cuda_device) + 5
        want, tol = ref.rotate(x.clone(), pos, freq)
        try:
            ext.mla_rope_forward(x, pos, freq, out=out)
        except RuntimeError as e:
            assert "overlap" in str(e) and not same, (shape, sx, ox, so, oo)
            refused += 1
            assert torch.equal(store, base)
            continue
        assert same or not set(a) & set(b), (shape, sx, ox, so, oo)
        assert ((out.double() - want).abs() <= tol).all(), (shape, sx, ox, so, oo)
        rest = torch.ones(1000, dtype=torch.bool, device=cuda_device)
        rest[torch.tensor(b, device=cuda_device)] = False
        assert torch.equal(store[rest], base[rest])
        accepted += 1
    assert accepted > 100 and refused > 100


def test_outputs_over_other_inputs_are_refused(ext, cuda_device):
    """Rotation and append: an output over anything that another block still reads. Columns of one joint projection, and one
    buffer for everything, are fine where no byte is shared."""
    T, H, bf = 6, 3, torch.bfloat16
    _, cache, table, start, kv = make_batch([(4, 40), (2, 20)], 1, 16, bf, cuda_device)
    g = torch.Generator(device=cuda_device).manual_seed(3)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    joint = torch.randn(T, H * 576 + 576, generator=g, device=cuda_device).to(bf)          # queries, latent row, k_pe
    q, c_kv, k_pe = joint[:, :H * 576].view(T, H, 576), joint[:, H * 576:H * 576 + 512], joint[:, H * 576 + 512:]
    first, before = cache.clone(), joint.clone()
    call = lambda out, cache=cache, freq=freq, table=table, start=start, kv=kv, q_pe=q[..., 512:]: ext.mla_rope_append_forward(
        q_pe, c_kv, k_pe, cache, table, start, kv, freq, out, check=True)
    flat = joint.view(-1)
    ints64 = torch.zeros(4096, dtype=torch.float64, device=cuda_device)
    ints64[:32] = freq
    as_rows = lambda t: t.view(bf)[:T * H * 64].view(T, H, 64)
    tables = torch.zeros(4096, dtype=torch.int32, device=cuda_device)
    for i, t in enumerate((table, start, kv)):
        tables[i * 64:i * 64 + t.numel()] = t.reshape(-1)
    inside = [tables[i * 64:i * 64 + t.numel()].view(t.shape) for i, t in enumerate((table, start, kv))]
    for bad in (lambda: call(k_pe[:, None].expand(T, 1, 64), q_pe=q[:, :1, 512:]), lambda: call(c_kv[:, None, 448:], q_pe=q[:, :1, 512:]),
                lambda: call(flat[H * 576 - 64:][:T * H * 64].view(T, H, 64)),
                lambda: call(as_rows(ints64), freq=ints64[:32]), lambda: call(as_rows(tables), table=inside[0]),
                lambda: call(as_rows(tables), start=inside[1]), lambda: call(as_rows(tables), kv=inside[2]),
                lambda: call(None, freq=cache.view(-1)[:128].view(torch.float64)),
                lambda: call(None, kv=cache.view(-1)[:4].view(torch.int32))):
        with pytest.raises(RuntimeError, match="overlap"):
            bad()
    assert torch.equal(cache, first) and torch.equal(joint, before)
    # in place in the joint projection
    want = ext.mla_rope_append_forward(q[..., 512:].clone(), c_kv.clone(), k_pe.clone(), first, table, start, kv, freq)
    call(q[..., 512:])
    assert torch.equal(q[..., 512:], want) and torch.equal(cache, first) and torch.equal(c_kv, before[:, H * 576:H * 576 + 512])
    x = torch.randn(4, 2, 8, generator=g, device=cuda_device)
    pos = torch.arange(64, dtype=torch.int32, device=cuda_device)
    f = torch.ones(64, dtype=torch.float64, device=cuda_device)
    for bad in (lambda: ext.mla_rope_forward(x, pos[:4], f[:4], out=pos.view(torch.float32).view(4, 2, 8)),
                lambda: ext.mla_rope_forward(x, pos[:4], f[:4], out=f.view(torch.float32)[4:68].view(4, 2, 8))):
        with pytest.raises(RuntimeError, match="overlap"):
            bad()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_forward_and_inverse_are_adjoint(ext, cuda_device, dtype, interleaved):
    """<dy, R x> = <R' dy, x> between the two directions of the kernel, on 64 columns of wider heads. Either side is off by at most
    its results' tolerance (derived in paged_reference) times the other factor, summed."""
    g = torch.Generator(device=cuda_device).manual_seed(11)
    x, dy = (torch.randn(37, 6, 192, generator=g, device=cuda_device).to(dtype)[..., o:o + 64] for o in (128, 64))
    pos = torch.randint(0, 1 << 20, (37,), generator=g, device=cuda_device, dtype=torch.int32)
    freq = 10000.0 ** (-torch.arange(32, dtype=torch.float64, device=cuda_device) / 32)
    y = ext.mla_rope_forward(x, pos, freq, interleaved, 1.5)
    dx = ext.mla_rope_forward(dy, pos, freq, interleaved, 1.5, True)
    _, tol_y = ref.rotate(x, pos, freq, interleaved, 1.5)
    _, tol_dx = ref.rotate(dy, pos, freq, interleaved, 1.5, True)
    left, right = (dy.double() * y.double()).sum(2), (dx.double() * x.double()).sum(2)
    assert ((left - right).abs() <= (dy.double().abs() * tol_y + x.double().abs() * tol_dx).sum(2)).all()
    assert (left.abs() > 1).any()                     # not all lost in the tolerance

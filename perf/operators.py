"""The operators of the paged latent cache, as cases that can be measured.

Three operators that a serving program runs one after the other on a cache of latent rows
(512 latent + 64 rotary columns per token) kept in pages:

* ``attention``  dense causal attention of each sequence's new tokens over its cached rows;
* ``rope`` / ``append``  rotary positions on a part of the head, and the same fused with the write of the new
  rows into their pages;
* ``fork`` / ``compact`` / ``free`` / ``copy``  what is done with whole pages.

``run`` computes them with elementary torch operations where ``own`` is false and calls the package's operators
where it is true. Lengths follow from a case alone, values from the seed.
"""
import math
import random

import torch

own = False

D, DV, R = 576, 512, 64          # row of the cache, its value part, its rotary part
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

_ext = None


def _ops():
    global _ext
    if _ext is None:
        import cuda_agent_b200
        _ext = cuda_agent_b200.load_extension()
    return _ext


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one user, one new token, a short history: what counts is the latency of a call
        dict(name="attention one user", kind="attention", batch=1, new=1, kv=1000, heads=16, page=64, dtype="bf16",
             ragged=False, window=0),
        # a decode step of a full batch on one GPU that holds all heads
        dict(name="attention decode batch", kind="attention", batch=64, new=1, kv=8192, heads=128, page=64,
             dtype="bf16", ragged=True, window=0),
        # verification of a few drafted tokens, heads split over GPUs, small pages
        dict(name="attention verify", kind="attention", batch=32, new=5, kv=4096, heads=24, page=16, dtype="bf16",
             ragged=True, window=0),
        # a long prompt taken in chunks: the last chunk, all heads
        dict(name="attention prompt chunk", kind="attention", batch=1, new=1024, kv=8192, heads=128, page=64,
             dtype="bf16", ragged=False, window=0),
        # several prompts of odd lengths at once, pages that are no power of two, a sliding window
        dict(name="attention ragged prompts", kind="attention", batch=6, new=300, kv=2048, heads=64, page=48,
             dtype="fp16", ragged=True, window=1024),
        # the new rows of a decode step
        dict(name="append decode", kind="append", batch=32, new=1, kv=2048, heads=128, page=64, dtype="bf16",
             interleaved=True, scaled=True),
        # the new rows of prompt chunks
        dict(name="append chunk", kind="append", batch=4, new=1024, kv=4096, heads=128, page=64, dtype="bf16",
             interleaved=True, scaled=True),
        # the rotary part of the queries, where it stands in the head, at far positions
        dict(name="rope part of head", kind="rope", tokens=4096, heads=128, rot=64, head=576, positions=131072,
             dtype="bf16", interleaved=False, scaled=True, inverse=False),
        # the gradient of a rotation of half of the head, in 32 bits
        dict(name="rope gradient", kind="rope", tokens=2047, heads=16, rot=64, head=128, positions=8192,
             dtype="fp32", interleaved=False, scaled=False, inverse=True),
        # four more answers from one prompt
        dict(name="fork few", kind="fork", live=1, slots=8, kv=1500, moved=4, layers=4, pool=64, page=64),
        # a fragmented pool put in order
        dict(name="compact pool", kind="compact", live=64, slots=128, kv=2500, moved=0, layers=8, pool=2048, page=64),
        # most answers of a batch have ended
        dict(name="free batch", kind="free", live=256, slots=256, kv=8192, moved=200, layers=1, pool=24576, page=64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "append", "rope", "fork", "compact", "free", "copy"])
    if kind == "attention":
        while True:
            c = dict(kind=kind, batch=_log_int(rng, 1, 64), new=_log_int(rng, 1, 1024), kv=_log_int(rng, 1, 8192),
                     heads=rng.choice([1, 7, 8, 16, 20, 32, 64, 128]), page=rng.choice([1, 8, 16, 24, 32, 64, 100, 128]),
                     dtype=rng.choice(["bf16", "bf16", "fp16"]), ragged=rng.random() < 0.7,
                     window=rng.choice([0, 0, 0, _log_int(rng, 1, 4096)]))
            c["kv"] = max(c["kv"], c["new"])
            if c["batch"] * c["new"] * c["heads"] * c["kv"] <= 1 << 29 and c["batch"] * c["kv"] <= 1 << 19:
                return c
    if kind == "append":
        while True:
            c = dict(kind=kind, batch=_log_int(rng, 1, 64), new=_log_int(rng, 1, 4096), kv=_log_int(rng, 1, 8192),
                     heads=rng.choice([1, 5, 16, 64, 128]), page=rng.choice([1, 16, 40, 64]),
                     dtype=rng.choice(["bf16", "fp16"]), interleaved=rng.random() < 0.5, scaled=rng.random() < 0.5)
            c["kv"] = max(c["kv"], c["new"])
            if c["batch"] * c["new"] * c["heads"] <= 1 << 19 and c["batch"] * c["kv"] <= 1 << 18:
                return c
    if kind == "rope":
        rot = rng.choice([8, 32, 64, 96, 128])
        return dict(kind=kind, tokens=_log_int(rng, 1, 4096), heads=_log_int(rng, 1, 128), rot=rot,
                    head=rot + rng.choice([0, 0, 64, 512]), positions=_log_int(rng, 16, 1 << 20),
                    dtype=rng.choice(["bf16", "fp16", "fp32"]), interleaved=rng.random() < 0.5,
                    scaled=rng.random() < 0.5, inverse=rng.random() < 0.4)
    live = _log_int(rng, 2, 64)
    kv, page, layers = _log_int(rng, 1, 1500), rng.choice([1, 16, 64]), rng.choice([1, 2, 6])
    moved = rng.randint(1, live - 1)
    most = live * -(-kv // page) + 2 * live + moved
    return dict(kind=kind, live=live, slots=2 * live + rng.randint(0, 9), kv=kv, moved=moved, layers=layers,
                pool=int(most * rng.uniform(1.0, 1.6)) + 1, page=page)


def _lengths(c):
    """New tokens and cached rows (the new ones among them) of every sequence."""
    r = random.Random("%(batch)d %(new)d %(kv)d %(page)d %(heads)d" % c)
    new, kv = [c["new"]] * c["batch"], [c["kv"]] * c["batch"]
    if c.get("ragged"):
        for b in range(1, c["batch"]):
            new[b] = r.randint(1, c["new"])
            kv[b] = r.randint(max(new[b], c["kv"] // 4), c["kv"])
        if c["batch"] >= 4:
            new[-1] = 0              # a place of the batch that has nothing to do now
    return new, kv


def _visible(n, kv, window):
    """Pairs of a new token and a row that it sees."""
    total = 0
    for i in range(n):
        p = kv - n + i
        total += p + 1 - (max(0, p + 1 - window) if window else 0)
    return total


def _pool(c):
    """Lengths of the live sequences, the pages in use, and who shares them: sequence 1 begins as sequence 0 does."""
    r = random.Random("%(live)d %(kv)d %(pool)d %(page)d %(moved)d" % c)
    kv = [c["kv"]] + [r.randint(1, c["kv"]) for _ in range(c["live"] - 1)]
    need = [-(-n // c["page"]) for n in kv]
    shared = min(kv[0], kv[1]) // c["page"] // 2 if c["live"] > 1 else 0
    used = sorted(r.sample(range(c["pool"]), sum(need) - shared))
    picked = r.sample(range(c["live"]), c["live"])
    picked = (picked * (c["moved"] // c["live"] + 1))[:c["moved"]]
    return kv, need, shared, used, picked


def work(case):
    c = case
    if c["kind"] == "attention":
        new, kv = _lengths(c)
        rows = sum(new) * c["heads"]
        pairs = sum(_visible(n, k, c["window"]) for n, k in zip(new, kv)) * c["heads"]
        reach = [min(k, c["window"] + n) if c["window"] else k for n, k in zip(new, kv)]
        cached = sum(k for n, k in zip(new, reach) if n)
        return {"bytes": cached * D * 2 + rows * (D * 2 + DV * 2 + 4), "flops": 2 * (D + DV) * pairs}
    if c["kind"] == "append":
        t = c["batch"] * c["new"]
        return {"bytes": t * c["heads"] * R * 2 * 2 + t * D * 2 * 2, "flops": 6 * t * (c["heads"] + 1) * R // 2}
    if c["kind"] == "rope":
        n = c["tokens"] * c["heads"] * c["rot"]
        return {"bytes": 2 * n * TYPES[c["dtype"]].itemsize, "flops": 3 * n}
    kv, need, shared, used, picked = _pool(c)
    one = 2 * c["layers"] * c["page"] * D * 2
    if c["kind"] == "fork":
        moves, ints = sum(kv[s] % c["page"] != 0 for s in picked), 3 * sum(need[s] for s in picked)
    elif c["kind"] == "compact":
        moves, ints = sum(u >= len(used) for u in used), 2 * sum(need) + 2 * c["pool"]
    elif c["kind"] == "free":
        moves, ints = 0, 4 * sum(need[s] for s in picked)
    else:
        moves, ints = min(c["moved"], c["pool"] - len(used)), 2 * c["moved"]
    return {"bytes": moves * one + 4 * ints, "flops": 0}


# ------------------------------------------------------------------------------------------------ inputs
def _frequencies(rot, scaled, device):
    """Radians per position of each pair, in 64 bits; `scaled` stretches the slow ones for a context 16 times as long."""
    i = torch.arange(rot // 2, dtype=torch.float64, device=device)
    f = 10000.0 ** (-2.0 * i / rot)
    if not scaled:
        return f, 1.0
    turns = 4096 * f / (2 * math.pi)
    keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0, 1)
    return f * keep + f / 16.0 * (1 - keep), 0.1 * math.log(16.0) + 1.0


def _paged(c, new, kv, g, dev, dtype):
    """A pool with the rows of every sequence in pages in no order, and the batch's tables."""
    ps = c["page"]
    need = [-(-k // ps) for k in kv]
    pool = sum(need) + max(1, sum(need) // 10)
    cache = torch.randn(pool, ps, D, generator=g, device=dev).to(dtype)
    order = torch.randperm(pool, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(kv), max(need)), -1, dtype=torch.int32, device=dev)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    return dict(cache=cache, table=table, q_start=torch.tensor(start, dtype=torch.int32, device=dev),
                kv_len=torch.tensor(kv, dtype=torch.int32, device=dev), tokens=start[-1], max_new=max(new), max_kv=max(kv))


def prepare(case, seed):
    c, dev = case, torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    s = {"case": c}
    if c["kind"] == "attention":
        new, kv = _lengths(c)
        dtype = TYPES[c["dtype"]]
        s.update(_paged(c, new, kv, g, dev, dtype))
        # scores with a spread of about three: some rows of the cache count much more than others
        s["q"] = (3 * math.sqrt(192 / D) * torch.randn(s["tokens"], c["heads"], D, generator=g, device=dev)).to(dtype)
        s["scale"] = 192 ** -0.5
    elif c["kind"] == "append":
        new, kv = _lengths(c)
        dtype = TYPES[c["dtype"]]
        s.update(_paged(c, new, kv, g, dev, dtype))
        t = s["tokens"]
        s["q_pe"] = torch.randn(t, c["heads"], R, generator=g, device=dev).to(dtype)
        joint = torch.randn(t, D, generator=g, device=dev).to(dtype)     # one projection gives both
        s["c_kv"], s["k_pe"] = joint[:, :DV], joint[:, DV:]
        s["q"] = torch.randn(t, c["heads"], D, generator=g, device=dev).to(dtype)
        s["freq"], s["mscale"] = _frequencies(R, c["scaled"], dev)
    elif c["kind"] == "rope":
        x = torch.randn(c["tokens"], c["heads"], c["head"], generator=g, device=dev).to(TYPES[c["dtype"]])
        s["x"] = x[..., c["head"] - c["rot"]:]
        s["positions"] = torch.randint(0, c["positions"], (c["tokens"],), generator=g, device=dev, dtype=torch.int32)
        s["freq"], s["mscale"] = _frequencies(c["rot"], c["scaled"], dev)
    else:
        kv, need, shared, used, picked = _pool(c)
        width = max(need) + 1
        order = torch.tensor(used, dtype=torch.int32, device=dev)[torch.randperm(len(used), generator=g, device=dev)]
        table = torch.full((c["slots"], width), -1, dtype=torch.int32, device=dev)
        length = torch.zeros(c["slots"], dtype=torch.int32, device=dev)
        length[:c["live"]] = torch.tensor(kv, dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(need):
            own_pages = n - (shared if b == 1 else 0)
            if b == 1:
                table[1, :shared] = table[0, :shared]
            table[b, n - own_pages:n] = order[at:at + own_pages]
            at += own_pages
        held = table[table >= 0].long()
        s["refcount"] = torch.bincount(held, minlength=c["pool"]).to(torch.int32)
        s["pages"] = torch.randn(c["layers"], c["pool"], c["page"], D, generator=g, device=dev, dtype=torch.float32) \
            .to(torch.bfloat16) if c["kind"] != "free" else None
        s["table"], s["length"] = table, length
        # who is forked or freed: any order; a fork's children take the empty places
        shuffle = torch.randperm(len(picked), generator=g, device=dev)
        s["picked"] = torch.tensor(picked, dtype=torch.int32, device=dev)[shuffle]
        s["children"] = c["live"] + torch.arange(len(picked), dtype=torch.int32, device=dev)
        if c["kind"] == "copy":
            spare = torch.nonzero(s["refcount"] == 0)[:, 0].to(torch.int32)
            n = min(c["moved"], len(spare))
            s["src"] = order[torch.randint(0, len(order), (n,), generator=g, device=dev)]
            s["dst"] = spare[torch.randperm(len(spare), generator=g, device=dev)[:n]]
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _slots(s, pos):
    """Rows of the pool that hold positions `pos` [B, n] of every sequence."""
    ps = s["case"]["page"]
    page = torch.gather(s["table"], 1, (pos // ps).clamp(0, s["table"].shape[1] - 1)).clamp_min(0).long()
    return page * ps + pos % ps


def _attention(s):
    c, dev = s["case"], s["q"].device
    b, h, n, m, t = len(s["kv_len"]), c["heads"], s["max_new"], s["max_kv"], s["tokens"]
    start, kv = s["q_start"].long(), s["kv_len"].long()
    count = start[1:] - start[:-1]
    j = torch.arange(m, device=dev)
    rows = s["cache"].reshape(-1, D)[_slots(s, j.expand(b, m))].float()
    rows.masked_fill_((j >= kv[:, None])[..., None], 0.0)
    i = torch.arange(n, device=dev)
    q = s["q"].float()[(start[:-1, None] + i).clamp_max(t - 1)]                       # [b, n, h, D]
    scores = (q.reshape(b, n * h, D) @ rows.transpose(1, 2)).mul_(s["scale"]).reshape(b, n, h, m)
    pos = (kv - count)[:, None] + i
    seen = (j <= pos[..., None]) & (j < kv[:, None, None])
    if c["window"]:
        seen &= j > pos[..., None] - c["window"]
    scores.masked_fill_(~seen[:, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.reshape(b, n * h, m) @ rows[..., :DV]).reshape(b, n, h, DV)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    lse = (top + total.log())[..., 0]
    tok = torch.arange(t, device=dev)
    at = torch.searchsorted(start[1:].contiguous(), tok, right=True)
    return out[at, tok - start[at]].to(s["q"].dtype), lse[at, tok - start[at]]


def _rotate(x, positions, freq, mscale, interleaved, inverse):
    angle = positions.double()[:, None] * freq
    cos, sin = (angle.cos() * mscale).float(), (angle.sin() * mscale).float()
    if inverse:
        sin = -sin
    cos, sin = (v.reshape(v.shape[0], *[1] * (x.dim() - 2), v.shape[1]) for v in (cos, sin))
    f, half = x.float(), x.shape[-1] // 2
    if interleaved:
        a, b = f[..., 0::2], f[..., 1::2]
        out = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = f[..., :half], f[..., half:]
        out = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return out.to(x.dtype)


def _append(s):
    c = s["case"]
    start, kv = s["q_start"].long(), s["kv_len"].long()
    tok = torch.arange(s["tokens"], device=kv.device)
    at = torch.searchsorted(start[1:].contiguous(), tok, right=True)
    pos = kv[at] - (start[at + 1] - start[at]) + tok - start[at]
    ps = c["page"]
    slot = s["table"][at, pos // ps].long() * ps + pos % ps
    rows = s["cache"].view(-1, D)
    rows[slot, :DV] = s["c_kv"]
    rows[slot, DV:] = _rotate(s["k_pe"], pos, s["freq"], s["mscale"], c["interleaved"], False)
    s["q"][..., DV:] = _rotate(s["q_pe"], pos, s["freq"], s["mscale"], c["interleaved"], False)
    return s["q"], s["cache"]


def _held(table, length, page):
    return torch.arange(table.shape[1], device=table.device) < ((length + page - 1) // page)[:, None]


def _fork(s, table, length, refcount):
    ps, src, dst = s["case"]["page"], s["picked"].long(), s["children"].long()
    rows, n = table[src], length[src]
    full = torch.arange(rows.shape[1], device=rows.device) < (n // ps)[:, None]
    refcount.index_add_(0, rows[full].long(), torch.ones_like(rows[full]))
    part = torch.nonzero(n % ps)[:, 0]
    fresh = torch.nonzero(refcount == 0)[:len(part), 0]
    last = (n // ps).long()[part]
    old = rows[part, last].long()
    rows = torch.where(full, rows, torch.full_like(rows, -1))
    rows[part, last] = fresh.to(rows.dtype)
    refcount[fresh] = 1
    table[dst], length[dst] = rows, n
    s["pages"][:, fresh] = s["pages"][:, old]
    return s["pages"], table, length, refcount


def _compact(s, table, length, refcount):
    used = refcount > 0
    ids = torch.arange(len(refcount), device=refcount.device)
    below = ids < used.sum()
    src, dst = torch.nonzero(used & ~below)[:, 0], torch.nonzero(~used & below)[:, 0]
    to = ids.to(torch.int32)
    to[src] = dst.to(torch.int32)
    held = _held(table, length, s["case"]["page"])
    table = torch.where(held, to[table.clamp_min(0).long()], table)
    refcount[dst] = refcount[src]
    refcount[src] = 0
    s["pages"][:, dst] = s["pages"][:, src]
    return s["pages"], table, length, refcount


def _free(s, table, length, refcount):
    seq = s["picked"].long()
    rows = table[seq]
    held = _held(rows, length[seq], s["case"]["page"])
    refcount.index_add_(0, rows.clamp_min(0).long().reshape(-1), -held.to(torch.int32).reshape(-1))
    table[seq] = -1
    length[seq] = 0
    return table, length, refcount


def run(state):
    s, c = state, state["case"]
    kind = c["kind"]
    if kind == "attention":
        if own:
            return _ops().mla_paged_attention_forward(s["q"], s["cache"], s["table"], s["q_start"], s["kv_len"],
                                                      s["scale"], True, c["window"])
        return _attention(s)
    if kind == "append":
        if own:
            _ops().mla_rope_append_forward(s["q_pe"], s["c_kv"], s["k_pe"], s["cache"], s["table"], s["q_start"],
                                           s["kv_len"], s["freq"], s["q"][..., DV:], c["interleaved"], s["mscale"])
            return s["q"], s["cache"]
        return _append(s)
    if kind == "rope":
        if own:
            return _ops().mla_rope_forward(s["x"], s["positions"], s["freq"], c["interleaved"], s["mscale"], c["inverse"])
        return _rotate(s["x"], s["positions"], s["freq"], s["mscale"], c["interleaved"], c["inverse"])
    if kind == "copy":
        if own:
            return _ops().mla_pages_copy(s["pages"], s["src"], s["dst"])
        s["pages"][:, s["dst"].long()] = s["pages"][:, s["src"].long()]
        return s["pages"]
    table, length, refcount = s["table"].clone(), s["length"].clone(), s["refcount"].clone()
    if kind == "fork":
        if own:
            _ops().mla_pages_fork(s["pages"], table, length, refcount, s["picked"], s["children"])
            return s["pages"], table, length, refcount
        return _fork(s, table, length, refcount)
    if kind == "compact":
        if own:
            _ops().mla_pages_compact(s["pages"], table, length, refcount)
            return s["pages"], table, length, refcount
        return _compact(s, table, length, refcount)
    if own:
        _ops().mla_pages_free(table, length, refcount, s["picked"], c["page"])
        return table, length, refcount
    return _free(s, table, length, refcount)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attention(s):
    c = s["case"]
    ps, h = c["page"], c["heads"]
    outs, lses = [], []
    table, start, kvs = s["table"].tolist(), s["q_start"].tolist(), s["kv_len"].tolist()
    for b, kv in enumerate(kvs):
        n = start[b + 1] - start[b]
        if not n:
            continue
        held = torch.tensor(table[b][:-(-kv // ps)], device=s["q"].device)
        rows = s["cache"][held].reshape(-1, D)[:kv].double()
        step = max(1, (1 << 28) // (kv * h))
        for i0 in range(0, n, step):
            q = s["q"][start[b] + i0:start[b] + min(n, i0 + step)].double()
            x = torch.einsum("nhd,kd->nhk", q, rows) * s["scale"]
            p = kv - n + i0 + torch.arange(len(q), device=x.device)
            j = torch.arange(kv, device=x.device)
            hide = j[None] > p[:, None]
            if c["window"]:
                hide = hide | (j[None] + c["window"] <= p[:, None])
            x = x.masked_fill(hide[:, None], -math.inf)
            lses.append(torch.logsumexp(x, -1))
            outs.append(torch.einsum("nhk,kd->nhd", torch.softmax(x, -1), rows[:, :DV]))
    return torch.cat(outs), torch.cat(lses)


def _exact_rotate(x, positions, freq, mscale, interleaved, inverse):
    """As multiplication by exp(i angle) of complex numbers."""
    half = x.shape[-1] // 2
    f = x.double()
    z = torch.view_as_complex(f.reshape(*f.shape[:-1], half, 2).contiguous()) if interleaved \
        else torch.complex(f[..., :half].contiguous(), f[..., half:].contiguous())
    angle = torch.outer(positions.double(), freq)
    turn = mscale * torch.exp(1j * (-angle if inverse else angle))
    z = z * turn.reshape(turn.shape[0], *[1] * (x.dim() - 2), half)
    return torch.view_as_real(z).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)


def _exact_pages(s):
    c = s["case"]
    ps = c["page"]
    pages = s["pages"].double() if s["pages"] is not None else None
    if c["kind"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            pages[:, b] = s["pages"][:, a].double()
        return pages
    table, length, count = s["table"].tolist(), s["length"].tolist(), s["refcount"].tolist()
    moves = []
    if c["kind"] == "fork":
        for a, b in zip(s["picked"].tolist(), s["children"].tolist()):
            n = length[a]
            for i in range(n // ps):
                table[b][i] = table[a][i]
                count[table[a][i]] += 1
            length[b] = n
        for a, b in zip(s["picked"].tolist(), s["children"].tolist()):
            if length[a] % ps:
                new = count.index(0)
                count[new] = 1
                table[b][length[a] // ps] = new
                moves.append((table[a][length[a] // ps], new))
    elif c["kind"] == "free":
        for a in s["picked"].tolist():
            for i in range(-(-length[a] // ps)):
                count[table[a][i]] -= 1
            table[a], length[a] = [-1] * len(table[a]), 0
    else:
        used = sum(n > 0 for n in count)
        holes = [i for i in range(used) if not count[i]]
        high = [i for i in range(used, len(count)) if count[i]]
        moves = list(zip(high, holes))
        to = dict(moves)
        for b, n in enumerate(length):
            for i in range(-(-n // ps)):
                table[b][i] = to.get(table[b][i], table[b][i])
        for a, b in moves:
            count[b], count[a] = count[a], 0
    for a, b in moves:
        pages[:, b] = pages[:, a]
    made = tuple(torch.tensor(v, dtype=torch.int32) for v in (table, length, count))
    return made if pages is None else (pages, *made)


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["kind"] == "attention":
        return _exact_attention(s)
    if c["kind"] == "rope":
        return _exact_rotate(s["x"], s["positions"], s["freq"], s["mscale"], c["interleaved"], c["inverse"])
    if c["kind"] == "append":
        q, cache, ps = s["q"].double(), s["cache"].double(), c["page"]
        start, kv, table = s["q_start"].tolist(), s["kv_len"].tolist(), s["table"].cpu()
        place, pos = [], []
        for b in range(len(kv)):
            n = start[b + 1] - start[b]
            p = torch.arange(kv[b] - n, kv[b])
            pos.append(p)
            place.append(table[b].long()[p // ps] * ps + p % ps)
        pos, place = (torch.cat(v).to(q.device) for v in (pos, place))
        turn = (pos, s["freq"], s["mscale"], c["interleaved"], False)
        q[..., DV:] = _exact_rotate(s["q_pe"], *turn)
        cache.view(-1, D)[place] = torch.cat((s["c_kv"].double(), _exact_rotate(s["k_pe"], *turn)), -1)
        return q, cache
    return _exact_pages(s)

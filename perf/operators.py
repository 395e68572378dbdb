"""Operators of a paged key-value cache, as timed cases.

Four kinds, each one call of a serving program:

  append   norms of queries and keys per head, rotation, keys and values into their pages: a decode batch, packed prompts
  attn     attention of one new token per sequence over its pages, behind a window with first tokens or not, with the attention
           weight that every cached token received added up or not
  evict    rows that hold more than ``keep`` tokens keep the first, the newest and the most attended ones, closed up in place
  gather   rows of pages as dense caches, which prompt attention reads

Keys and values lie in pages [P, key heads, page, D]; ``mass`` [P, key heads, page] holds the weight received; ``table``
[rows, width] names each row's pages (-1: none).  Head counts are those of this repository's configurations (synth.CONFIGS) and
generic ones; with ``own`` the framework's kernels run, without it elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-6
THETA = 500000.0


def listed():
    return [
        # one user's chat: a single token, nothing but latency
        dict(name="append-1", kind="append", heads=32, kv_heads=8, dim=128, page=16, dtype="f16", norm=False, pairs=0, rot=64, batch=1, tokens=1,
             context=1000, ahead=0),
        # a server's decode batch; sequences that have lost tokens to eviction stand at far positions
        dict(name="append-64", kind="append", heads=40, kv_heads=8, dim=128, page=64, dtype="bf16", norm=True, pairs=0, rot=64, batch=64, tokens=1,
             context=500, ahead=100000),
        # prompts of several users, packed
        dict(name="append-4x1501", kind="append", heads=64, kv_heads=8, dim=128, page=128, dtype="bf16", norm=False, pairs=0, rot=64, batch=4,
             tokens=1501, context=77, ahead=0),
        # one user's chat: latency, and one sequence's keys spread over the GPU
        dict(name="attn-1x1000", kind="attn", heads=32, kv_heads=8, dim=128, page=16, dtype="f16", batch=1, context=1000, ragged=False, first=0,
             window=0, mass=False),
        # a full server batch of short conversations of unequal lengths
        dict(name="attn-64x500", kind="attn", heads=40, kv_heads=8, dim=128, page=16, dtype="bf16", batch=64, context=500, ragged=True, first=0,
             window=0, mass=False),
        # long contexts: the cache stream
        dict(name="attn-16x8192", kind="attn", heads=32, kv_heads=8, dim=128, page=64, dtype="f16", batch=16, context=8192, ragged=False, first=0,
             window=0, mass=False),
        # endless conversations: four first tokens and the last 1024 stay visible
        dict(name="attn-window-48x6000", kind="attn", heads=32, kv_heads=8, dim=128, page=32, dtype="bf16", batch=48, context=6000, ragged=True,
             first=4, window=1024, mass=False),
        # a batch whose cache will be cut: the weights are added up on the way
        dict(name="attn-mass-12x3333", kind="attn", heads=64, kv_heads=8, dim=128, page=64, dtype="bf16", batch=12, context=3333, ragged=True, first=0,
             window=0, mass=True),
        # a batch cut to half of its cache
        dict(name="evict-16x4096", kind="evict", kv_heads=8, dim=128, page=64, dtype="bf16", batch=16, context=4096, ragged=False, keep=2048, first=4,
             recent=256),
        # one long document cut to an eighth
        dict(name="evict-1x40001", kind="evict", kv_heads=8, dim=128, page=16, dtype="f16", batch=1, context=40001, ragged=False, keep=5000, first=16,
             recent=1000),
        # a prompt's portion behind a long shared beginning
        dict(name="gather-1x7777", kind="gather", kv_heads=8, dim=128, page=128, dtype="bf16", batch=1, context=7777, ragged=False),
        # portions of several float32 sequences of a small model
        dict(name="gather-9x2000-f32", kind="gather", kv_heads=2, dim=64, page=16, dtype="f32", batch=9, context=2000, ragged=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["append", "attn", "attn", "attn", "evict", "gather"])
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (40, 8, 128), (64, 8, 128), (32, 32, 96), (4, 2, 64), (16, 2, 256), (12, 1, 64), (25, 5, 80)])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    case = dict(kind=kind, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    # cached tokens in all, so that a pass reads no more than the largest listed one
    room = min(131072, 16 * 8192 * 8 * 128 * 2 // (kv_heads * dim * SIZE[dtype]))
    if kind == "append":
        batch = _log(rng, 1, 64)
        tokens = rng.choice([1, _log(rng, 2, max(2, 4000 // batch))])
        rot = rng.choice([dim // 2, dim // 4])
        return dict(case, heads=heads, norm=rng.random() < 0.5, pairs=rng.choice([0, 1]), rot=rot, batch=batch, tokens=tokens,
                    context=_log(rng, 1, 1000), ahead=rng.choice([0, _log(rng, 100, 1000000)]))
    batch = _log(rng, 1, 64)
    if kind == "attn":
        context = _log(rng, 1, room // batch)
        window = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(case, heads=heads, batch=batch, context=context, ragged=rng.random() < 0.7, window=window,
                    first=rng.choice([4, _log(rng, 1, 64)]) if window else 0, mass=rng.random() < 0.3)
    if kind == "evict":
        context = _log(rng, 64, min(room, 65536) // batch)
        keep = rng.randint(context // 8 + 2, context - 1)
        return dict(case, batch=batch, context=context, ragged=rng.random() < 0.5, keep=keep, first=rng.randint(0, min(16, keep // 4)),
                    recent=rng.randint(0, keep // 2))
    return dict(case, batch=batch, context=_log(rng, 1, min(room, 65536) // batch), ragged=rng.random() < 0.7)


def _lengths(case):
    """Cached tokens of every row: ``context``, or (ragged) spread unevenly from a quarter of it up."""
    n = case["context"]
    return [max(1, int(n * (1.0 - 0.75 * (i * 0.618034 % 1.0)))) if case.get("ragged") else n for i in range(case["batch"])]


def _visible(case, n):
    return n if case["window"] == 0 else min(n, case["window"] + min(case["first"], max(n - case["window"], 0)))


def work(case):
    G, D, size = case["kv_heads"], case["dim"], SIZE[case["dtype"]]
    n = _lengths(case)
    if case["kind"] == "append":
        M, H = case["batch"] * case["tokens"], case["heads"]
        return {"bytes": 2 * M * (H + 2 * G) * D * size + 4 * M * G + 12 * M, "flops": M * (H + G) * (6 * case["rot"] + (4 * D if case["norm"] else 0))}
    if case["kind"] == "attn":
        M, H = case["batch"], case["heads"]
        seen = sum(_visible(case, x) for x in n)
        pages = sum(-(-_visible(case, x) // case["page"]) for x in n)
        return {"bytes": 2 * seen * G * D * size + 2 * M * H * D * size + 4 * pages + (8 * seen * G if case["mass"] else 0), "flops": 4 * seen * H * D}
    if case["kind"] == "evict":
        cut = [x for x in n if x > case["keep"]]
        moved = len(cut) * max(0, case["keep"] - case["first"]) * G
        return {"bytes": 4 * sum(cut) * G + moved * (4 * D * size + 8) + 4 * len(n) * case["keep"] * G, "flops": sum(cut) * G}
    return {"bytes": 4 * sum(n) * G * D * size, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# what a program holds before the call
class _Source:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 7919 + 29)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def table(self, counts, page):
        """Pages dealt to the rows in no order; -1 behind a row's last."""
        need = [-(-n // page) for n in counts]
        ids = torch.randperm(sum(need), generator=self.g, device=DEV).to(torch.int32)
        t = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEV)
        at = 0
        for i, k in enumerate(need):
            t[i, :k] = ids[at:at + k]
            at += k
        return t, sum(need)

    def pages(self, P, case):
        shape = (P, case["kv_heads"], case["page"], case["dim"])
        return self.normal(*shape).to(DT[case["dtype"]]), self.normal(*shape).to(DT[case["dtype"]])

    def mass(self, P, case):
        """Received weight: few tokens have much, many have none."""
        x = torch.exp(2.0 * self.normal(P, case["kv_heads"], case["page"]) - 4.0)
        return torch.where(x < 0.01, torch.zeros_like(x), x)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    src, dt, G, D = _Source(seed), DT[case["dtype"]], case["kv_heads"], case["dim"]
    n = _lengths(case)
    B = case["batch"]
    if case["kind"] == "append":
        H, L = case["heads"], case["tokens"]
        table, P = src.table([x + L for x in n], case["page"])
        k, v = src.pages(P, case)
        slots = torch.arange(L, dtype=torch.int32, device=DEV)[None, :] + _i32(n)[:, None]
        i = torch.arange(case["rot"], dtype=torch.float64, device=DEV)
        norm = (lambda: (1.0 + 0.1 * src.normal(D)).to(dt)) if case["norm"] else (lambda: None)
        return dict(case=case, qkv=src.normal(B * L, (H + 2 * G) * D).to(dt), q=torch.empty((B * L, H * D), dtype=dt, device=DEV), k=k, v=v,
                    mass=src.mass(P, case), table=table, row=torch.arange(B, dtype=torch.int32, device=DEV).repeat_interleave(L),
                    slot=slots.reshape(-1).contiguous(), pos=(slots + case["ahead"]).reshape(-1).contiguous(),
                    rates=torch.exp(-i / case["rot"] * math.log(THETA)).float(), q_norm=norm(), k_norm=norm())
    table, P = src.table(n, case["page"])
    k, v = src.pages(P, case)
    s = dict(case=case, k=k, v=v, table=table, lengths=_i32(n))
    if case["kind"] == "attn":
        H = case["heads"]
        s.update(q=(1.5 * src.normal(B, H * D)).to(dt), out=torch.empty((B, H * D), dtype=dt, device=DEV), mass=src.mass(P, case) if case["mass"] else None,
                 row=torch.arange(B, dtype=torch.int32, device=DEV), slot=s["lengths"] - 1, scale=D ** -0.5, ws=None)
        if own:
            from mlx_parallm_b200 import ops
            keys = (table.shape[1] * case["page"]) if case["mass"] else 0
            s["ws"] = torch.zeros((max(16, ops.paged_attn_workspace_bytes(B, H, D, keys)),), dtype=torch.uint8, device=DEV)
    elif case["kind"] == "evict":
        s.update(mass=src.mass(P, case), kept=torch.full((B, G, case["keep"]), -1, dtype=torch.int32, device=DEV))
    else:
        shape = (B, G, -(-max(n) // 256) * 256, D)
        s.update(rows=torch.arange(B, dtype=torch.int32, device=DEV), dk=torch.zeros(shape, dtype=dt, device=DEV),
                 dv=torch.zeros(shape, dtype=dt, device=DEV))
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
def _flat(table, slots, page):
    """Place of a slot in the pages laid end to end, by row: page id * page + offset (ids of absent pages read as 0)."""
    return table.clamp(min=0).long().gather(1, slots // page) * page + slots % page


def _by_slot(pages):
    """[P, G, page, ...] as [P * page, G, ...]: one line per place."""
    return pages.transpose(1, 2).reshape(pages.shape[0] * pages.shape[2], pages.shape[1], *pages.shape[3:])


def _put(pages, places, values):
    """pages[place // page, :, place % page] = values [n, G, ...]"""
    page = pages.shape[2]
    pages[places // page, :, places % page] = values.to(pages.dtype)


def _plain_append(s):
    c = s["case"]
    H, G, D, n = c["heads"], c["kv_heads"], c["dim"], c["rot"]
    M = s["qkv"].shape[0]
    x = s["qkv"].float().view(M, H + 2 * G, D)
    q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
    angle = s["pos"].double()[:, None] * s["rates"].double()[None, :]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x, w):
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
        a, b = (x[..., :n], x[..., n:2 * n]) if c["pairs"] == 0 else (x[..., 0:2 * n:2], x[..., 1:2 * n:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        both = torch.cat([a, b], -1) if c["pairs"] == 0 else torch.stack([a, b], -1).flatten(-2)
        return torch.cat([both, x[..., 2 * n:]], -1)

    s["q"].copy_(turned(q, s["q_norm"]).reshape(M, H * D))
    places = s["table"][s["row"].long(), (s["slot"] // c["page"]).long()].long() * c["page"] + (s["slot"] % c["page"]).long()
    _put(s["k"], places, turned(k, s["k_norm"]))
    _put(s["v"], places, v)
    _put(s["mass"], places, torch.zeros((M, G), device=DEV))


def _plain_attn(s):
    c = s["case"]
    H, G, D, B = c["heads"], c["kv_heads"], c["dim"], c["batch"]
    T = s["table"].shape[1] * c["page"]
    j = torch.arange(T, device=DEV)[None, :].expand(B, T)
    n = s["slot"].long()[:, None] + 1
    seen = j < n
    if c["window"]:
        seen = seen & ((j < c["first"]) | (j >= n - c["window"]))
    places = _flat(s["table"], j, c["page"])
    k = _by_slot(s["k"])[places].permute(0, 2, 3, 1).float()                  # [B, G, D, T]
    scores = s["q"].float().view(B, G, H // G, D) @ k * s["scale"]
    scores = torch.where(seen[:, None, None], scores, torch.full((), -math.inf, device=DEV))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    s["out"].copy_((p @ _by_slot(s["v"])[places].transpose(1, 2).float()).reshape(B, H * D))
    if c["mass"]:
        page, w = c["page"], p.sum(2).transpose(1, 2)[seen]                   # [seen places, G]
        at = places[seen]
        _put(s["mass"], at, s["mass"][at // page, :, at % page] + w)


def _plain_evict(s):
    c = s["case"]
    B, G, page, keep = c["batch"], c["kv_heads"], c["page"], c["keep"]
    T = s["table"].shape[1] * page
    j = torch.arange(T, device=DEV)[None, :].expand(B, T)
    n = s["lengths"].long()[:, None]
    places = _flat(s["table"], j, page)
    score = _by_slot(s["mass"])[places].transpose(1, 2)                       # [B, G, T]
    always = (j < c["first"]) | (j >= n - c["recent"])
    score = torch.where(always[:, None], torch.full((), math.inf, device=DEV), score)
    score = torch.where((j >= n)[:, None], torch.full((), -1.0, device=DEV), score)
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :keep]
    best = torch.nn.functional.pad(best, (0, keep - best.shape[-1]), value=T)
    best = torch.where(best < n[:, None], best, torch.full((), T, dtype=best.dtype, device=DEV)).sort(-1).values
    s["kept"].copy_(torch.where(best < T, best, torch.full((), -1, dtype=best.dtype, device=DEV)))
    b, g, i = torch.nonzero((n[:, None] > keep) & (best < T) & (best != torch.arange(keep, device=DEV)), as_tuple=True)
    at = places[b, best[b, g, i]], places[b, i]
    for t in (s["k"], s["v"], s["mass"]):
        t[at[1] // page, g, at[1] % page] = t[at[0] // page, g, at[0] % page]


def _plain_gather(s):
    c = s["case"]
    B, cap = c["batch"], s["dk"].shape[2]
    T = min(cap, s["table"].shape[1] * c["page"])
    j = torch.arange(T, device=DEV)[None, :].expand(B, T)
    places = _flat(s["table"], j, c["page"])
    here = (j < s["lengths"].long()[:, None])[:, None, :, None]
    for pages, dense in ((s["k"], s["dk"]), (s["v"], s["dv"])):
        dense[:, :, :T] = torch.where(here, _by_slot(pages)[places].transpose(1, 2), dense[:, :, :T])


PLAIN = {"append": _plain_append, "attn": _plain_attn, "evict": _plain_evict, "gather": _plain_gather}


def _own(s):
    from mlx_parallm_b200 import ops
    c = s["case"]
    if c["kind"] == "append":
        ops.paged_append(s["qkv"], s["q"], s["k"], s["v"], s["table"], s["row"], s["slot"], s["pos"], c["heads"], rates=s["rates"], pairs=c["pairs"],
                         q_norm_w=s["q_norm"], k_norm_w=s["k_norm"], eps=EPS, mass=s["mass"])
    elif c["kind"] == "attn":
        ops.paged_attn(s["q"], s["k"], s["v"], s["table"], s["row"], s["slot"], s["out"], s["scale"], first=c["first"], window=c["window"],
                       mass=s["mass"], workspace=s["ws"])
    elif c["kind"] == "evict":
        ops.paged_evict(s["k"], s["v"], s["mass"], s["table"], s["lengths"], s["kept"], first=c["first"], recent=c["recent"])
    else:
        ops.paged_gather(s["k"], s["v"], s["table"], s["rows"], s["lengths"], s["dk"], s["dv"])


def run(s):
    kind = s["case"]["kind"]
    if own:
        _own(s)
    else:
        PLAIN[kind](s)
    if kind == "append":
        return {"q": s["q"], "k": s["k"], "v": s["v"], "mass": s["mass"]}
    if kind == "attn":
        return {"out": s["out"], "mass": s["mass"]} if s["case"]["mass"] else {"out": s["out"]}
    if kind == "evict":
        return {"kept": s["kept"], "k": s["k"], "v": s["v"], "mass": s["mass"]}
    return {"k": s["dk"], "v": s["dv"]}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits, sequence by sequence
def exact(case, seed):
    s = prepare(case, seed)
    G, D, page = case["kv_heads"], case["dim"], case["page"]
    table = s["table"].tolist()

    def line(pages, r, n):
        """The first n slots of row r: [G, n, ...]."""
        ids = [p for p in table[r] if p >= 0][:-(-n // page)]
        return torch.cat([pages[p] for p in ids], 1)[:, :n]

    def write(pages, r, n, values):
        """The first n slots of row r take values [G, n, ...]."""
        for i in range(-(-n // page)):
            part = values[:, i * page:min(n, (i + 1) * page)]
            pages[table[r][i], :, :part.shape[1]] = part

    if case["kind"] == "append":
        H, L, r = case["heads"], case["tokens"], case["rot"]
        x = s["qkv"].double().view(-1, H + 2 * G, D)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * s["rates"].double())[:, None]
        parts = []
        for part, w in ((x[:, :H], s["q_norm"]), (x[:, H:H + G], s["k_norm"])):
            if w is not None:
                part = part / (part.square().sum(-1, keepdim=True) / D + EPS).sqrt() * w.double()
            part = part.clone()
            lo, hi = (slice(0, r), slice(r, 2 * r)) if case["pairs"] == 0 else (slice(0, 2 * r, 2), slice(1, 2 * r, 2))
            z = torch.complex(part[..., lo].contiguous(), part[..., hi].contiguous()) * turn
            part[..., lo], part[..., hi] = z.real, z.imag
            parts.append(part)
        k, v, mass = s["k"].double(), s["v"].double(), s["mass"].double()
        for b, n in enumerate(_lengths(case)):
            new = slice(b * L, (b + 1) * L)
            for pages, values in ((k, parts[1][new]), (v, x[new, H + G:]), (mass, torch.zeros((L, G), dtype=torch.float64, device=DEV))):
                write(pages, b, n + L, torch.cat([line(pages, b, n), values.transpose(0, 1)], 1))
        return {"q": parts[0].reshape(-1, H * D), "k": k, "v": v, "mass": mass}
    if case["kind"] == "attn":
        H = case["heads"]
        out, mass = [], s["mass"].double() if case["mass"] else None
        for b, n in enumerate(_lengths(case)):
            j = torch.arange(n, device=DEV)
            shown = j[(j < case["first"]) | (j >= n - case["window"])] if case["window"] else j
            k, v = line(s["k"], b, n)[:, shown].double(), line(s["v"], b, n)[:, shown].double()
            p = torch.softmax(torch.einsum("ghd,gjd->ghj", s["q"][b].double().view(G, H // G, D), k) * s["scale"], -1)
            out.append(torch.einsum("ghj,gjd->ghd", p, v).reshape(H * D))
            if mass is not None:
                m = line(mass, b, n).clone()
                m[:, shown] += p.sum(1)
                write(mass, b, n, m)
        return {"out": torch.stack(out), "mass": mass} if case["mass"] else {"out": torch.stack(out)}
    if case["kind"] == "evict":
        keep, kept = case["keep"], s["kept"].clone().fill_(-1)
        k, v, mass = s["k"].double(), s["v"].double(), s["mass"].double()
        for b, n in enumerate(_lengths(case)):
            if n <= keep:
                kept[b, :, :n] = torch.arange(n, dtype=torch.int32, device=DEV)
                continue
            lo, hi = case["first"], n - case["recent"]
            old, new = [line(t, b, n).clone() for t in (k, v, mass)], []
            for g in range(G):
                order = torch.argsort(old[2][g, lo:hi], descending=True, stable=True)[:keep - lo - case["recent"]] + lo
                at = torch.cat([torch.arange(lo, device=DEV), order.sort().values, torch.arange(hi, n, device=DEV)])
                kept[b, g] = at
                new.append([t[g, at] for t in old])
            for t, values in zip((k, v, mass), zip(*new)):
                write(t, b, keep, torch.stack(values))
        return {"kept": kept, "k": k, "v": v, "mass": mass}
    dk, dv = s["dk"].double(), s["dv"].double()
    for b, n in enumerate(_lengths(case)):
        dk[b, :, :n], dv[b, :, :n] = line(s["k"], b, n).double(), line(s["v"], b, n).double()
    return {"k": dk, "v": dv}

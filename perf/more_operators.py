"""Operators of sampling several answers to a prompt, under adapters, and of scoring them, as timed cases.

Three kinds, each one call of a serving program:

  score   log probabilities of given tokens out of a step's or a prompt's logits, the entropy of every row, its most likely tokens
  lora    low-rank updates of a projection's output, every row under an adapter of its own or none
  shared  attention of one new token per sequence over a paged cache in which groups of sequences have their first pages in common

Head counts, widths and vocabularies are those of this repository's configurations (synth.CONFIGS) and generic ones; with ``own`` the
framework's kernels run, without it elementary torch operations in 32 bits.
"""
import math

import torch

own = False

DEV = "cuda"
DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
SIZE = {"f16": 2, "bf16": 2, "f32": 4}


def listed():
    return [
        # one user's chat that shows the five most likely tokens: nothing but latency
        dict(name="score-1x32000", kind="score", rows=1, vocab=32000, dtype="f32", top=5, temperature=1.0, allowed=0),
        # a server's decode batch with the most alternatives that clients may ask for
        dict(name="score-64x128256", kind="score", rows=64, vocab=128256, dtype="f32", top=20, temperature=0.7, allowed=0),
        # a prompt's portion: how likely its own tokens were
        dict(name="score-1500x151936", kind="score", rows=1500, vocab=151936, dtype="f32", top=0, temperature=1.0, allowed=0),
        # 16-bit logits of an odd vocabulary in which a grammar allows few tokens
        dict(name="score-333x50257-bf16", kind="score", rows=333, vocab=50257, dtype="bf16", top=8, temperature=1.0, allowed=700),
        # one user's chat under an adapter
        dict(name="lora-1", kind="lora", rows=1, segment=1, adapters=1, none=False, rank=16, inner=4096, q_width=4096, v_width=1024, gap=1024,
             dtype="f16", out="f32"),
        # a server's decode batch, every request under an adapter of its own
        dict(name="lora-64x64", kind="lora", rows=64, segment=1, adapters=64, none=False, rank=16, inner=4096, q_width=4096, v_width=1024, gap=1024,
             dtype="f16", out="f32"),
        # a decode batch of few adapters of a small rank, some requests without one
        dict(name="lora-100x5", kind="lora", rows=100, segment=1, adapters=5, none=True, rank=8, inner=5120, q_width=5120, v_width=1024, gap=1024,
             dtype="bf16", out="f32"),
        # prompts of several requests, packed
        dict(name="lora-8x1000", kind="lora", rows=8000, segment=1000, adapters=7, none=True, rank=64, inner=4096, q_width=4096, v_width=1024, gap=1024,
             dtype="bf16", out="bf16"),
        # four answers to a question
        dict(name="shared-4x900", kind="shared", heads=32, kv_heads=8, dim=128, page=16, dtype="f16", batch=4, groups=1, alone=0, prefix=900, tail=60),
        # a batch behind one long system prompt
        dict(name="shared-64x4000", kind="shared", heads=32, kv_heads=8, dim=128, page=64, dtype="bf16", batch=64, groups=1, alone=0, prefix=4000, tail=300),
        # rollouts: groups of answers to prompts of unequal lengths, some requests by themselves
        dict(name="shared-96x1500", kind="shared", heads=40, kv_heads=8, dim=128, page=64, dtype="bf16", batch=96, groups=9, alone=5, prefix=1500, tail=700),
        # a long document that many ask about
        dict(name="shared-128x16000", kind="shared", heads=64, kv_heads=8, dim=128, page=128, dtype="f16", batch=128, groups=2, alone=0, prefix=16000,
             tail=100),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["score", "lora", "shared"])
    if kind == "score":
        vocab = rng.choice([32000, 128256, 151936, 50257, 1024, _log(rng, 300, 150000)])
        top = rng.choice([0, 1, 5, 20, rng.randint(2, 32)])
        # (the plain form sorts whole rows where alternatives are asked for)
        rows = _log(rng, 1, max(1, (20000000 if top else 200000000) // vocab))
        return dict(kind=kind, rows=min(rows, 4096), vocab=vocab, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), top=top,
                    temperature=rng.choice([1.0, 1.0, 0.7, round(rng.uniform(0.3, 2.0), 2)]),
                    allowed=rng.choice([0, 0, 0, _log(rng, 40, vocab)]))
    if kind == "lora":
        inner, first, last = rng.choice([(4096, 4096, 1024), (5120, 5120, 1024), (8192, 8192, 1024), (512, 512, 128), (128, 128, 64), (2048, 2048, 2048)])
        rank = rng.choice([8, 16, 32, 64, rng.randint(1, 64)])
        adapters = _log(rng, 1, 64)
        segment = rng.choice([1, 1, _log(rng, 2, 1000)])
        rows = _log(rng, 1, 256) if segment == 1 else segment * rng.randint(1, max(1, min(16, 6000 // segment)))
        return dict(kind=kind, rows=rows, segment=segment, adapters=adapters, none=rng.random() < 0.5, rank=rank, inner=inner, q_width=first, v_width=last,
                    gap=rng.choice([last, 0]), dtype=rng.choice(["f16", "bf16"]), out="f32" if rows <= 128 else "16")
    heads, kv_heads, dim = rng.choice([(32, 8, 128), (40, 8, 128), (64, 8, 128), (32, 32, 96), (4, 2, 64), (16, 2, 256), (12, 1, 64), (25, 5, 80)])
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    batch = _log(rng, 2, 128)
    groups = rng.randint(1, max(1, min(16, batch // 3)))
    # no more products than the largest listed case
    room = min(16000, 128 * 16000 * 64 * 128 // (batch * heads * dim) // (4 if dtype == "f32" else 1))
    return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 48, 64, 128, 256]), dtype=dtype, batch=batch, groups=groups,
                alone=rng.choice([0, 0, rng.randint(0, max(0, batch // 4))]), prefix=_log(rng, 16, room), tail=_log(rng, 1, 1000))


# ---------------------------------------------------------------------------------------------------------------------
# the cases' sizes
def _adapter_of(case):
    """Every row's adapter; -1: none."""
    out = []
    for i in range(case["rows"]):
        s = i // case["segment"]
        out.append(-1 if case["none"] and s % 5 == 3 else s * 7 % case["adapters"])
    return out


def _out_dtype(case):
    return "f32" if case["out"] == "f32" else case["dtype"]


def _groups(case):
    """(group of every sequence, -1: alone; shared slots of every group; slots of every sequence).  Groups and prompts are of unequal sizes, prompts are
    shared by whole pages, and what follows them has unequal lengths."""
    B, N, page = case["batch"], case["groups"], case["page"]
    joined = B - case["alone"]
    group = [min(N - 1, int(N * (i / max(1, joined)) ** 1.3)) if i < joined else -1 for i in range(B)]
    prefix = [max(1, int(case["prefix"] * (1.0 - 0.4 * (g * 0.618034 % 1.0))) // page) * page for g in range(N)]
    tail = [max(1, int(case["tail"] * (1.0 - 0.75 * (i * 0.618034 % 1.0)))) for i in range(B)]
    return group, prefix, [(prefix[group[i]] if group[i] >= 0 else case["prefix"]) + tail[i] for i in range(B)]


def work(case):
    if case["kind"] == "score":
        R, V, k = case["rows"], case["vocab"], case["top"]
        return {"bytes": R * (V * SIZE[case["dtype"]] + 12 + 8 * k), "flops": 6 * R * V}
    if case["kind"] == "lora":
        index = _adapter_of(case)
        R, K, N, r = sum(i >= 0 for i in index), case["inner"], case["q_width"] + case["v_width"], case["rank"]
        used, size = len({i for i in index if i >= 0}), SIZE[case["dtype"]]
        return {"bytes": R * K * size + used * r * (2 * K + N) * size + 2 * R * N * SIZE[_out_dtype(case)], "flops": 2 * R * r * (2 * K + N)}
    G, D, H, size = case["kv_heads"], case["dim"], case["heads"], SIZE[case["dtype"]]
    group, prefix, n = _groups(case)
    own_slots = sum(x - (prefix[g] if g >= 0 else 0) for g, x in zip(group, n))
    slots = own_slots + sum(prefix[g] for g in set(group) if g >= 0)
    return {"bytes": 2 * slots * G * D * size + 2 * len(n) * H * D * size, "flops": 4 * sum(n) * H * D}


# ---------------------------------------------------------------------------------------------------------------------
# what a program holds before the call
class _Source:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) * 6007 + 11)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g, device=DEV)

    def below(self, n, *shape):
        return torch.randint(0, n, shape, generator=self.g, device=DEV)

    def order(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    src = _Source(seed)
    return dict({"score": _prepare_score, "lora": _prepare_lora, "shared": _prepare_shared}[case["kind"]](case, src), case=case)


def _prepare_score(case, src):
    R, V, dt = case["rows"], case["vocab"], DT[case["dtype"]]
    x = src.normal(R, V).mul_(2.5)
    tokens = src.below(V, R)
    # two thirds of the tokens are likely ones, as sampled text has them
    x[torch.arange(R, device=DEV), tokens] += torch.where(src.below(3, R) > 0, 12.0, 0.0)
    if case["allowed"]:                                             # a grammar leaves a run of tokens and the given one
        lo = src.below(max(1, V - case["allowed"]), R)[:, None]
        j = torch.arange(V, device=DEV)[None]
        for r in range(0, R, 256):
            hide = (j < lo[r:r + 256]) | (j >= lo[r:r + 256] + case["allowed"])
            hide.scatter_(1, tokens[r:r + 256, None], False)
            x[r:r + 256].masked_fill_(hide, -math.inf)
    if R > 1:
        tokens[0] = -1                                              # a text's first token follows nothing
    return dict(logits=x.to(dt), tokens=tokens.to(torch.int32))


def _prepare_lora(case, src):
    dt, n, K, r = DT[case["dtype"]], case["adapters"], case["inner"], case["rank"]
    pad = -(-r // 16) * 16                                          # adapters lie with their rank filled up to a multiple of 16
    widths = (case["q_width"], case["v_width"])
    N = sum(widths)
    a = torch.zeros((n, len(widths), pad, K), dtype=dt, device=DEV)
    a[:, :, :r] = (src.normal(n, len(widths), r, K) / math.sqrt(K)).to(dt)
    b = torch.zeros((n, N, pad), dtype=dt, device=DEV)
    b[:, :, :r] = (src.normal(n, N, r) / math.sqrt(r)).to(dt)
    index = _adapter_of(case)
    columns, at = [], 0
    for w in widths:
        columns.append((at, w))
        at += w + case["gap"]
    base = src.normal(case["rows"], at).to(DT[_out_dtype(case)])
    s = dict(x=src.normal(case["rows"], K).to(dt), a=a, b=b, scales=0.5 + src.normal(n).abs(), columns=columns, base=base, y=torch.empty_like(base),
             index=_i32(index), rows_of=[torch.tensor([i for i, v in enumerate(index) if v == k], device=DEV, dtype=torch.int64) for k in range(n)])
    if own:
        from mlx_parallm_b200 import ops
        s["plan"] = ops.row_groups(s["index"], n, ops.lora_tile(case["rows"], n))
    return s


def _prepare_shared(case, src):
    dt, G, D, H, B, page = DT[case["dtype"]], case["kv_heads"], case["dim"], case["heads"], case["batch"], case["page"]
    group, prefix, n = _groups(case)
    order = src.order(B).tolist()                                   # members of a group stand anywhere in the batch
    group, n = [group[i] for i in order], [n[i] for i in order]
    need = [-(-x // page) for x in n]
    P = sum(p // page for p in prefix) + sum(k - (prefix[g] // page if g >= 0 else 0) for g, k in zip(group, need))
    ids = src.order(P).tolist()
    heads = [[ids.pop() for _ in range(p // page)] for p in prefix]
    table = torch.full((B, max(need)), -1, dtype=torch.int32)
    for i, (g, k) in enumerate(zip(group, need)):
        row = heads[g][:] if g >= 0 else []
        row += [ids.pop() for _ in range(k - len(row))]
        table[i, :k] = torch.tensor(row, dtype=torch.int32)
    shape = (P, G, page, D)
    s = dict(k=src.normal(*shape).to(dt), v=src.normal(*shape).to(dt), table=table.to(DEV), row=torch.arange(B, dtype=torch.int32, device=DEV),
             slot=_i32(n) - 1, q=(1.5 * src.normal(B, H * D)).to(dt), out=torch.empty((B, H * D), dtype=dt, device=DEV), scale=D ** -0.5, n=n, group=group,
             prefix=_i32(prefix), index=_i32(group), ws=None)
    if own:
        from mlx_parallm_b200 import ops
        s["plan"] = ops.row_groups(s["index"], case["groups"], ops.paged_attn_shared_tile(H, G))
        s["ws"] = torch.zeros((ops.paged_attn_shared_workspace_bytes(B, H, G, D, case["groups"]),), dtype=torch.uint8, device=DEV)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
def _plain_score(s):
    c = s["case"]
    x, t = s["logits"].float(), s["tokens"].long()
    V, k = c["vocab"], c["top"]
    y = x if c["temperature"] == 1.0 else x / c["temperature"]
    m = y.amax(-1, keepdim=True)
    d = y - m
    e = torch.exp(d)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    weighted = torch.where(e > 0, e * d, torch.zeros_like(e)).sum(-1, keepdim=True)
    entropy = (log_total - weighted / total)[:, 0]
    given = (d.gather(1, t.clamp(0, V - 1)[:, None]) - log_total)[:, 0]
    out = {"logprob": torch.where(t < 0, torch.zeros_like(given), given), "entropy": entropy}
    if k:
        ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
        out["top_ids"], out["top_logprobs"] = ids.to(torch.int32), d.gather(1, ids) - log_total
    return out


def _plain_lora(s):
    s["y"].copy_(s["base"])                                         # what the projection has left
    R = s["a"].shape[2]
    for i, rows in enumerate(s["rows_of"]):
        if rows.numel() == 0:
            continue
        x, at = s["x"][rows].float(), 0
        for t, (col0, n) in enumerate(s["columns"]):
            z = x @ s["a"][i, t].float().t() * s["scales"][i]
            update = z @ s["b"][i, at:at + n].float().t()
            at += n
            s["y"][rows, col0:col0 + n] = (s["y"][rows, col0:col0 + n].float() + update).to(s["y"].dtype)
    return {"y": s["y"]}


def _plain_shared(s):
    c = s["case"]
    H, G, D, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    T = s["table"].shape[1] * page
    j = torch.arange(T, device=DEV)[None, :]
    q = s["q"].float().view(-1, G, H // G, D)
    for r in range(0, c["batch"], 8):                               # rows whose keys are in hand at a time
        part = slice(r, r + 8)
        ids = s["table"][part].clamp(min=0).long()
        k = s["k"][ids].permute(0, 2, 1, 3, 4).reshape(ids.shape[0], G, T, D).float()
        scores = q[part] @ k.transpose(2, 3) * s["scale"]
        seen = (j <= s["slot"][part].long()[:, None])[:, None, None]
        scores = torch.where(seen, scores, torch.full((), -math.inf, device=DEV))
        p = torch.exp(scores - scores.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        v = s["v"][ids].permute(0, 2, 1, 3, 4).reshape(ids.shape[0], G, T, D).float()
        s["out"][part] = (p @ v).reshape(ids.shape[0], H * D).to(s["out"].dtype)
    return {"out": s["out"]}


def _own(s):
    from mlx_parallm_b200 import ops
    c = s["case"]
    if c["kind"] == "score":
        r = ops.token_logprobs(s["logits"], s["tokens"], top=c["top"], temperature=c["temperature"])
        out = {"logprob": r.logprob, "entropy": r.entropy}
        if c["top"]:
            out["top_ids"], out["top_logprobs"] = r.top_ids, r.top_logprobs
        return out
    if c["kind"] == "lora":
        s["y"].copy_(s["base"])
        ops.lora_rows(s["x"], s["plan"], s["a"], s["b"], s["scales"], s["columns"], s["y"])
        return {"y": s["y"]}
    ops.paged_attn_shared(s["q"], s["k"], s["v"], s["table"], s["row"], s["slot"], s["out"], s["scale"], s["index"], s["prefix"], s["plan"],
                          workspace=s["ws"])
    return {"out": s["out"]}


def run(s):
    if own:
        return _own(s)
    return {"score": _plain_score, "lora": _plain_lora, "shared": _plain_shared}[s["case"]["kind"]](s)


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "score":
        parts = {"logprob": [], "entropy": [], "top_ids": [], "top_logprobs": []}
        for r in range(0, case["rows"], 128):
            x, t = s["logits"][r:r + 128].double(), s["tokens"][r:r + 128].tolist()
            lp = torch.log_softmax(x / case["temperature"], -1)
            parts["logprob"].append(torch.stack([lp[i, v] if v >= 0 else lp.new_zeros(()) for i, v in enumerate(t)]))
            parts["entropy"].append(torch.special.entr(lp.exp()).sum(-1))
            if case["top"]:
                ids = torch.argsort(x, dim=-1, descending=True, stable=True)[:, :case["top"]]
                parts["top_ids"].append(ids.to(torch.int32))
                parts["top_logprobs"].append(torch.take_along_dim(lp, ids, 1))
        return {k: torch.cat(v) for k, v in parts.items() if v}
    if case["kind"] == "lora":
        y = s["base"].double()
        a, b = s["a"].double(), s["b"].double()
        index = _adapter_of(case)
        start = 0
        while start < len(index):                                   # runs of rows under one adapter
            end = start
            while end < len(index) and index[end] == index[start]:
                end += 1
            i = index[start]
            if i >= 0:
                x = s["x"][start:end].double()
                low = torch.einsum("mk,trk->tmr", x, a[i]) * float(s["scales"][i])
                at = 0
                for t, (col0, n) in enumerate(s["columns"]):
                    y[start:end, col0:col0 + n] += torch.einsum("mr,nr->mn", low[t], b[i, at:at + n])
                    at += n
            start = end
        return {"y": y}
    G, D, H, page = case["kv_heads"], case["dim"], case["heads"], case["page"]
    table, out = s["table"].tolist(), []
    for i, n in enumerate(s["n"]):
        ids = table[i][:-(-n // page)]
        k = s["k"][ids].double().transpose(0, 1).reshape(G, -1, D)[:, :n]
        v = s["v"][ids].double().transpose(0, 1).reshape(G, -1, D)[:, :n]
        p = torch.softmax(torch.einsum("ghd,gjd->ghj", s["q"][i].double().view(G, H // G, D), k) * s["scale"], -1)
        out.append(torch.einsum("ghj,gjd->ghd", p, v).reshape(H * D))
    return {"out": torch.stack(out)}

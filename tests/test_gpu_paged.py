"""The paged key-value cache against the formulas in 64 bits (tests/paged_oracle.py): append, attention, eviction, dense view, and runs of
them together.  Tolerances: half a step of the storage type for each rounding to it, plus the oracle's bound for 32-bit arithmetic."""
import math

import pytest
import torch

import paged_oracle as po

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ops():
    from mlx_parallm_b200 import ops as o, _lib
    _lib.require_device()
    o.paged_fault_count(reset=True)
    return o


class Cache:
    """Pages dealt to rows in no order, every place that no row owns full of NaN."""

    def __init__(self, lengths, page, G, D, dtype, seed, spare=3, mass=True, width=None):
        g = torch.Generator().manual_seed(seed)
        need = [-(-max(n, 1) // page) for n in lengths]
        P = sum(need) + spare
        ids = torch.randperm(P, generator=g)
        self.table = torch.full((len(lengths), width or max(need)), -1, dtype=torch.int32)
        self.k = torch.full((P, G, page, D), math.nan).to(dtype)
        self.v = self.k.clone()
        self.mass = torch.full((P, G, page), math.nan) if mass else None
        self.page, self.G, self.D, self.P, self.dtype, self.g = page, G, D, P, dtype, g
        at = 0
        for r, (n, c) in enumerate(zip(lengths, need)):
            self.table[r, :c] = ids[at:at + c].to(torch.int32)
            at += c
            for i in range(c):
                here = max(0, min(page, n - i * page))
                p = int(self.table[r, i])
                self.k[p, :, :here] = torch.randn((G, here, D), generator=g).to(dtype)
                self.v[p, :, :here] = torch.randn((G, here, D), generator=g).to(dtype)
                if mass:
                    self.mass[p, :, :here] = torch.rand((G, here), generator=g)

    def normal(self, *shape):
        return torch.randn(shape, generator=self.g)

    def cuda(self):
        return self.k.cuda(), self.v.cuda(), self.table.cuda(), None if self.mass is None else self.mass.cuda()


def i32(v):
    return torch.tensor(v, dtype=torch.int32)


def same(a, b):
    """Bit by bit, NaN like NaN."""
    a, b = a.cpu().contiguous(), b.cpu().contiguous()
    kind = {4: torch.int32, 2: torch.int16}[a.element_size()]
    return torch.equal(a.view(kind), b.view(kind))


# ---------------------------------------------------------------- append
APPEND = [
    # dtype, H, G, D, page, rot, pairs, norms, f32 accumulator, tokens per row, context per row, ahead, mass
    ("f16", 32, 8, 128, 16, 64, 0, "", False, [1], [1000], 0, True),
    ("bf16", 40, 8, 128, 64, 64, 0, "qk", False, [1] * 9, [0, 1, 15, 16, 17, 63, 64, 65, 500], 1000000, True),
    ("f32", 4, 2, 64, 32, 32, 0, "qk", False, [3, 1, 40], [5, 0, 31], 0, True),
    ("bf16", 12, 1, 64, 48, 16, 1, "q", False, [7, 50], [40, 3], 77, False),
    ("f16", 5, 5, 96, 16, 48, 1, "k", False, [33], [0], 0, True),
    ("f16", 16, 2, 256, 256, 128, 0, "qk", True, [2, 5], [255, 9], 4, True),
    ("bf16", 32, 8, 128, 128, 64, 0, "qk", True, [1] * 33, list(range(33)), 0, True),
    ("bf16", 25, 5, 80, 16, 20, 0, "", False, [300], [11], 0, True),
    ("f16", 32, 8, 128, 64, 0, 0, "qk", False, [600], [100], 0, False),
    ("bf16", 64, 8, 128, 128, 64, 0, "", False, [700, 1, 333], [0, 12, 128], 0, True),
    ("f32", 3, 1, 8, 16, 4, 1, "qk", False, [20], [0], 0, True),
    ("bf16", 16, 8, 128, 16, 64, 0, "qk", False, [650, 0, 31], [3, 8, 100], 0, True),      # prompts: norms, neighbours, an accumulation buffer
    ("f16", 9, 3, 64, 64, 30, 1, "", False, [1203], [60], 5, True),
    ("bf16", 16, 4, 96, 32, 24, 1, "k", True, [601, 20], [0, 31], 0, True),
    ("f16", 7, 7, 72, 16, 32, 0, "q", True, [640], [1], 0, False),
    ("f32", 6, 2, 256, 16, 128, 0, "qk", False, [600], [0], 0, True),
]


def _append_inputs(case, seed=3, idle=()):
    dtype, H, G, D, page, rot, pairs, norms, acc, tokens, context, ahead, mass = case
    dt = DT[dtype]
    c = Cache([a + b for a, b in zip(tokens, context)], page, G, D, dt, seed, mass=mass)
    row = [r for r, n in enumerate(tokens) for _ in range(n)]
    slot = [s + i for n, s in zip(tokens, context) for i in range(n)]
    for t in idle:
        row[t] = -1 - t
    M = len(row)
    qkv = c.normal(M, (H + 2 * G) * D + 8)                  # rows wider than the heads: a column slice
    qkv = qkv if acc else qkv.to(dt)
    w = lambda: (1 + 0.2 * c.normal(D)).to(dt)
    rates = None if rot == 0 else torch.exp(-torch.arange(rot, dtype=torch.float64) / max(rot, 1) * math.log(1e4)).float()
    return c, i32(row), i32(slot), i32([s + ahead for s in slot]), qkv, w() if "q" in norms else None, w() if "k" in norms else None, rates


def _on(x):
    return None if x is None else x.cuda()


def _check_append(ops, case, idle=()):
    dtype, H, G, D, page, rot, pairs, norms, acc, tokens, context, ahead, mass = case
    dt = DT[dtype]
    c, row, slot, pos, qkv, qw, kw, rates = _append_inputs(case, idle=idle)
    M = row.numel()
    k, v, table, ms = c.cuda()
    q = torch.full((M, H * D), 7.0, dtype=dt, device="cuda")
    dev = qkv.cuda()
    ops.paged_append(dev, q, k, v, table, row.cuda(), slot.cuda(), pos.cuda(), H, rates=_on(rates), pairs=pairs, q_norm_w=_on(qw), k_norm_w=_on(kw),
                     eps=1e-5, mass=ms)
    eq, ek, ev, em, off = po.append(qkv.to(dt), c.k, c.v, c.mass, c.table, row, slot, pos, H, rates, pairs, qw, kw, 1e-5)
    tol = lambda e: po.half_step(dt) * e.abs() * (1 + 1e-3) + off + (2.0 ** -25 if dt is torch.float16 else 0)   # f16 below its smallest normal: half of 2^-24
    idle_rows = torch.isnan(eq[:, 0, 0])
    got = q.cpu().double().view(M, H, D)
    assert bool((got[idle_rows] == 7.0).all()), "idle tokens are left as they were"
    live = ~idle_rows
    assert bool(((got - eq).abs() <= tol(eq))[live].all())
    for name, g, e in (("k", k, ek), ("v", v, ev)):
        g = g.cpu().double()
        assert torch.equal(torch.isnan(g), torch.isnan(e)), name
        assert bool(((g - e).abs() <= tol(e))[~torch.isnan(e)].all()), name
    assert same(v, ev.to(dt)), "values are copied"
    if mass:
        assert same(ms, em.float())
    if acc:
        used = (H + 2 * G) * D
        assert bool((dev[:, :used] == 0).all()) and torch.equal(dev[:, used:].cpu(), qkv[:, used:])
    else:
        assert same(dev, qkv)
    assert ops.paged_fault_count(reset=True) == 0


@pytest.mark.parametrize("case", APPEND, ids=lambda c: f"{c[0]}-{c[1]}.{c[2]}.{c[3]}-p{c[4]}-{sum(c[9])}")
def test_append(ops, case):
    _check_append(ops, case)


@pytest.mark.parametrize("case", [APPEND[1], APPEND[6], APPEND[9]], ids=["decode", "accumulator", "prompts"])
def test_append_idle_tokens(ops, case):
    M = sum(case[9])
    _check_append(ops, case, idle=sorted({0, 3, 5, M // 2, M - 1}))


def test_append_nothing(ops):
    c, row, slot, pos, qkv, qw, kw, rates = _append_inputs(APPEND[0])
    k, v, table, ms = c.cuda()
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    ops.paged_append(qkv[:0].cuda(), torch.zeros((0, 32 * 128), dtype=torch.float16, device="cuda"), k, v, table, none, none, none, 32, rates=rates.cuda(), mass=ms)
    assert same(k, c.k) and same(v, c.v) and same(ms, c.mass)


def test_append_places_that_do_not_exist(ops):
    """A slot behind the table, a negative one, a page id of -1 and one behind the pool, a row behind the table: the others go on, the queries of
    tokens with a row are written all the same, every miss is counted."""
    dt, H, G, D = torch.bfloat16, 8, 2, 128
    c = Cache([64, 64, 64], 16, G, D, dt, 5)
    c.table[1, 1], c.table[2, 2] = -1, c.P
    row, slot = i32([0, 0, 1, 2, 3, 0, 1]), i32([64, -1, 20, 40, 0, 5, 40])
    qkv = c.normal(7, (H + 2 * G) * D).to(dt)
    k, v, table, ms = c.cuda()
    q = torch.full((7, H * D), 7.0, dtype=dt, device="cuda")
    ops.paged_append(qkv.cuda(), q, k, v, table, row.cuda(), slot.cuda(), slot.cuda(), H, mass=ms)
    eq, ek, ev, em, _ = po.append(qkv, c.k, c.v, c.mass, c.table, row, slot, slot, H, None, 0, None, None, 0.0)
    assert same(k, ek.to(dt)) and same(v, ev.to(dt)) and same(ms, em.float())
    assert bool((q[4] == 7.0).all())
    live = [0, 1, 2, 3, 5, 6]
    assert torch.equal(q.cpu()[live], eq.view(7, -1)[live].to(dt))
    assert ops.paged_fault_count() == 5 and ops.paged_fault_count(reset=True) == 5 and ops.paged_fault_count() == 0


# ---------------------------------------------------------------- attention
ATTN = [
    # dtype, H, G, D, page, slots of the tokens (row by row), first, window
    ("f16", 32, 8, 128, 16, [999], 0, 0),
    ("bf16", 40, 8, 128, 64, [0, 1, 14, 15, 16, 17, 62, 63, 64, 65, 127, 128, 500], 0, 0),
    ("f16", 4, 4, 128, 32, [3000, 5], 0, 0),
    ("bf16", 16, 1, 128, 16, [777, 2100], 0, 0),
    ("f16", 20, 1, 128, 48, [300, 47, 48], 0, 0),
    ("bf16", 64, 2, 64, 16, [400, 33], 0, 0),
    ("bf16", 32, 32, 96, 64, [130, 77], 0, 0),
    ("f16", 16, 2, 256, 128, [900, 0, 31], 0, 0),
    ("bf16", 25, 5, 80, 16, [513, 16], 0, 0),
    ("f16", 6, 3, 8, 16, [70], 0, 0),
    ("f32", 8, 2, 64, 32, [600, 31, 32], 0, 0),
    ("f32", 3, 1, 256, 16, [200], 0, 0),
    ("f32", 32, 8, 128, 64, [1000, 3], 0, 0),
    ("bf16", 32, 8, 128, 32, [2999, 1000, 1023, 1024, 1027, 1028, 1029, 1043, 50], 4, 1024),
    ("f16", 8, 2, 128, 16, [0, 1, 2, 15, 16, 17, 31, 32, 33, 100], 1, 1),
    ("f16", 8, 2, 128, 16, [15, 16, 17, 47, 48, 60, 200], 20, 16),
    ("bf16", 8, 2, 64, 48, [500, 40], 0, 100),
    ("f32", 8, 2, 128, 16, [300, 90], 17, 33),
    ("f16", 8, 2, 256, 16, [300, 90], 500, 7),
    ("bf16", 8, 2, 128, 64, [20000, 40, 9000], 0, 0),
    ("bf16", 32, 32, 64, 64, [15000, 299, 0, 1500], 0, 0),          # work enough for small shares at its end, in each engine
    ("f16", 64, 32, 80, 48, [3, 8000, 9000], 100, 8500),
    ("f32", 32, 32, 8, 16, [12000, 77, 5000], 0, 0),
]


def _check_attn(ops, c, q, row, slot, H, first, window, mass, scale, perm=False):
    dt, G, D = c.dtype, c.G, c.D
    M = row.numel()
    k, v, table, ms = c.cuda()
    ms = ms if mass else None
    out = torch.full((M, H * D), 7.0, dtype=dt, device="cuda")
    keys = c.table.shape[1] * c.page if mass else 0
    n = ops.paged_attn_workspace_bytes(M, H, D, keys)
    ws = torch.full((n,), 0xa5, dtype=torch.uint8, device="cuda")
    ops.paged_attn(q.cuda(), k, v, table, row.cuda(), slot.cuda(), out, scale, first=first, window=window, mass=ms, workspace=ws, out_perm=perm)
    exp, tol, em, off = po.attn(q, c.k, c.v, c.mass if mass else None, c.table, row, slot, H, scale, first, window,
                                0.0 if dt is torch.float32 else po.half_step(dt) ** 2)
    got = out.cpu().double().view(M, H, D)
    if perm:
        got = got.view(M, H, D // 8, 8)[..., [0, 2, 4, 6, 1, 3, 5, 7]].reshape(M, H, D)
    idle = torch.isnan(exp[:, 0, 0])
    assert bool((got[idle] == 7.0).all()), "idle tokens are left as they were"
    err = (got - exp).abs() - (tol + po.half_step(dt) * exp.abs() * (1 + 1e-3) + (2.0 ** -25 if dt is torch.float16 else 0))
    assert bool((err[~idle] <= 0).all()), float(err[~idle].max())
    if mass:
        g = ms.cpu().double()
        assert torch.equal(torch.isnan(g), torch.isnan(em))
        e = ((g - em).abs() - off)[~torch.isnan(em)]
        assert bool((e <= 0).all()), float(e.max())
    return out, ms


@pytest.mark.parametrize("mass", [False, True], ids=["plain", "mass"])
@pytest.mark.parametrize("case", ATTN, ids=lambda c: f"{c[0]}-{c[1]}.{c[2]}.{c[3]}-p{c[4]}-{max(c[5])}-w{c[6]}.{c[7]}")
def test_attention(ops, case, mass):
    dtype, H, G, D, page, slots, first, window = case
    c = Cache([s + 1 for s in slots], page, G, D, DT[dtype], 11, mass=mass)
    q = (2 * c.normal(len(slots), H * D)).to(c.dtype)
    _check_attn(ops, c, q, torch.arange(len(slots), dtype=torch.int32), i32(slots), H, first, window, mass, D ** -0.5)
    assert ops.paged_fault_count(reset=True) == 0


@pytest.mark.parametrize("dtype,H,G,D", [("bf16", 32, 8, 128), ("f16", 6, 3, 24), ("f32", 8, 2, 64)])
def test_attention_padded_batch(ops, dtype, H, G, D):
    """Idle tokens between the others, tokens before their row's beginning (they see nothing: zeros), several tokens of one row, a row whose
    table is wider than it needs."""
    c = Cache([300, 20, 5], 16, G, D, DT[dtype], 12, width=64)
    row, slot = i32([-1, 0, 0, 1, -5, 2, 0, 1, 1]), i32([3, 299, 298, 19, 0, 4, 0, -1, -7])
    q = c.normal(9, H * D).to(c.dtype)
    for mass in (False, True):
        out, _ = _check_attn(ops, c, q, row, slot, H, 0, 0, mass, 0.3)
        assert bool((out[7:] == 0).all())
    _check_attn(ops, c, q, row, slot, H, 2, 10, True, 0.3)
    assert ops.paged_fault_count(reset=True) == 0


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f16", 40), ("f32", 64)])
def test_attention_pages_that_do_not_exist(ops, dtype, D):
    """Ids of -1 and behind the pool: their keys count as masked and are counted; a row of nothing else gives zeros; a slot behind the table sees what
    the table holds."""
    c = Cache([100, 100, 40, 64], 16, 2, D, DT[dtype], 13, width=7)
    c.table[0, 1], c.table[1, 0], c.table[1, 6] = -1, c.P + 5, -(1 << 31)
    c.table[2] = -1
    c.table[3, 4:] = c.table[0, 2:5]
    row, slot = i32([0, 1, 2, 3]), i32([99, 99, 39, 5000])
    q = c.normal(4, 8 * D).to(c.dtype)
    for mass in (False, True):
        out, _ = _check_attn(ops, c, q, row, slot, 8, 0, 0, mass, 0.2)
        assert bool((out[2] == 0).all())
        assert ops.paged_fault_count(reset=True) > 0


def test_attention_rows_behind_the_table(ops):
    """Their tokens are left as idle ones are, and counted, however many tokens the call has."""
    c = Cache([50, 20], 16, 2, 64, torch.float16, 32)
    for n in (3, 700):
        row, slot = i32([0, 2, 1] + [-1] * (n - 3)), i32([49, 5, 19] + [0] * (n - 3))
        q = c.normal(n, 8 * 64).to(c.dtype)
        for mass in (False, True):
            _check_attn(ops, c, q, row, slot, 8, 0, 0, mass, 0.2)
            assert ops.paged_fault_count(reset=True) == 1


def test_attention_rows_share_pages(ops):
    """A common beginning: two rows and two tokens of one of them add their weights to the same places."""
    c = Cache([200, 90, 64], 16, 2, 128, torch.bfloat16, 14)
    c.table[1, :4] = c.table[0, :4]
    c.table[2, :4] = c.table[0, :4]
    q = c.normal(4, 8 * 128).to(c.dtype)
    _check_attn(ops, c, q, i32([0, 1, 2, 0]), i32([199, 89, 63, 150]), 8, 0, 0, True, 0.1)


@pytest.mark.parametrize("dtype,H,G,D,first,window", [("bf16", 8, 2, 128, 0, 0), ("f16", 40, 1, 64, 3, 50), ("f32", 9, 1, 24, 0, 33), ("bf16", 16, 2, 256, 30, 20)])
def test_received_weights_of_many_tokens_have_one_order(ops, dtype, H, G, D, first, window):
    """Portions of three rows, as runs and woven into one another: every slot's mass is the 64-bit sum, and has the same bits each time."""
    lengths = [400, 290, 64]
    rows = [r for r, n in enumerate(lengths) for _ in range(n - 40)] + [i % 3 for i in range(90)] + [-1, 2, 0]
    at, slots = [0, 0, 0], []
    for r in rows:
        slots.append(at[r] if r >= 0 else 5)
        at[max(r, 0)] += r >= 0
    row, slot = i32(rows), i32(slots)
    assert all(a <= n for a, n in zip(at, lengths))
    c = Cache(lengths, 16, G, D, DT[dtype], 31)
    q = c.normal(len(rows), H * D).to(c.dtype)
    _check_attn(ops, c, q, row, slot, H, first, window, True, D ** -0.5)
    k, v, table, qd = c.k.cuda(), c.v.cuda(), c.table.cuda(), q.cuda()
    ws = torch.empty((ops.paged_attn_workspace_bytes(len(rows), H, D, c.table.shape[1] * 16),), dtype=torch.uint8, device="cuda")
    seen = []
    for _ in range(3):
        mass, out = c.mass.cuda(), torch.empty_like(qd)
        ops.paged_attn(qd, k, v, table, row.cuda(), slot.cuda(), out, D ** -0.5, first=first, window=window, mass=mass, workspace=ws)
        seen.append(mass.cpu())
    assert torch.equal(seen[0].view(torch.int32), seen[1].view(torch.int32)) and torch.equal(seen[0].view(torch.int32), seen[2].view(torch.int32))


def test_attention_of_more_tokens_than_a_cta_keeps(ops):
    """A portion of several rows as single tokens, more of them than a CTA holds in shared memory, idle ones among them."""
    c = Cache([500, 150], 16, 2, 64, torch.bfloat16, 18)
    row = i32([0] * 500 + [-1] * 7 + [1] * 150)
    slot = i32(list(range(500)) + [3] * 7 + list(range(150)))
    q = c.normal(row.numel(), 8 * 64).to(c.dtype)
    for first, window, mass in ((0, 0, True), (5, 40, False)):
        _check_attn(ops, c, q, row, slot, 8, first, window, mass, 0.125)


def test_attention_of_many_key_heads(ops):
    c = Cache([70, 33, 1], 32, 130, 8, torch.float16, 19)
    q = c.normal(3, 260 * 8).to(c.dtype)
    _check_attn(ops, c, q, i32([0, 1, 2]), i32([69, 32, 0]), 260, 0, 0, True, 0.3)


def test_attention_in_very_wide_tables(ops):
    """Tables of 2^30 tokens and a row at their end: tiles, pages and offsets beyond 16 million; only what is visible is looked up."""
    G, D, H, page = 1, 64, 4, 16
    width = (1 << 30) // page - 1
    c = Cache([64, 64], page, G, D, torch.bfloat16, 20)
    table = torch.full((1, width), -7, dtype=torch.int32, device="cuda")
    table[0, :4] = c.table[0].cuda()
    table[0, width - 4:] = c.table[1].cuda()
    n = width * page
    k, v = c.k.cuda(), c.v.cuda()
    q = c.normal(1, H * D).to(c.dtype)
    out = torch.empty((1, H * D), dtype=c.dtype, device="cuda")
    ws = torch.empty((ops.paged_attn_workspace_bytes(1, H, D, 0),), dtype=torch.uint8, device="cuda")
    ops.paged_attn(q.cuda(), k, v, table, i32([0]).cuda(), i32([n - 1]).cuda(), out, 0.125, first=30, window=50, workspace=ws)
    # the same 30 first and 50 last tokens as a short row's: 30 of the first 64, then the last 50 of the other 64
    near = torch.cat([c.table[0], c.table[1]])[None]
    exp, tol, _, _ = po.attn(q, c.k, c.v, None, near, i32([0]), i32([127]), H, 0.125, 30, 50, po.half_step(c.dtype) ** 2)
    err = (out.cpu().double().view(1, H, D) - exp).abs() - tol - po.half_step(c.dtype) * exp.abs() * 1.001
    assert bool((err <= 0).all()) and ops.paged_fault_count(reset=True) == 0


def test_attention_perm8_output(ops):
    c = Cache([200, 90], 16, 2, 128, torch.float16, 15)
    q = c.normal(2, 8 * 128).to(c.dtype)
    _check_attn(ops, c, q, i32([0, 1]), i32([199, 89]), 8, 0, 0, False, 0.1, perm=True)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_attention_extreme_scores(ops, dtype):
    """Scores of +-1000, one key far above the others, and equal scores throughout: the maximum is taken out before anything is raised."""
    D, H, G = 128, 8, 2
    c = Cache([700, 700, 33], 16, G, D, DT[dtype], 16)
    q = c.normal(3, H * D)
    q[0] *= 40
    q[2] = 0
    _check_attn(ops, c, q.to(c.dtype), i32([0, 1, 2]), i32([699, 699, 32]), H, 0, 0, True, 1.0)


def test_attention_over_more_than_two_giga_elements(ops):
    """Pages behind the 2^31st element and the 2^32nd byte."""
    G, page, D, H = 8, 128, 128, 32
    P = (1 << 31) // (G * page * D) + 64
    k = torch.empty((P, G, page, D), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    c = Cache([500, 130], page, G, D, torch.bfloat16, 17, spare=0)
    far = torch.arange(P - c.P, P)
    k[far], v[far] = c.k.cuda(), c.v.cuda()
    mass = torch.zeros((P, G, page), device="cuda")
    row, slot = i32([0, 1]), i32([499, 129])
    q = c.normal(2, H * D).to(c.dtype)
    table = torch.where(c.table >= 0, c.table + (P - c.P), c.table)
    out = torch.empty((2, H * D), dtype=torch.bfloat16, device="cuda")
    ws = torch.empty((ops.paged_attn_workspace_bytes(2, H, D, table.shape[1] * page),), dtype=torch.uint8, device="cuda")
    ops.paged_attn(q.cuda(), k, v, table.cuda(), row.cuda(), slot.cuda(), out, 0.1, mass=mass, workspace=ws)
    near, nearest = _check_attn(ops, c, q, row, slot, H, 0, 0, True, 0.1)
    assert same(out, near)
    assert float(mass[:P - c.P].abs().max()) == 0.0 and abs(float(mass.sum()) - 2 * H) < 1e-3
    # append and gather there
    c2 = table.cuda()
    qkv = c.normal(2, (H + 2 * G) * D).to(c.dtype).cuda()
    ops.paged_append(qkv, torch.empty_like(out), k, v, c2, row.cuda(), slot.cuda(), slot.cuda(), H, mass=mass)
    dense = torch.zeros((2, G, 512, D), dtype=torch.bfloat16, device="cuda")
    dv = torch.zeros_like(dense)
    ops.paged_gather(k, v, c2, row.cuda(), i32([500, 130]).cuda(), dense, dv)
    x = qkv.view(2, H + 2 * G, D)
    assert torch.equal(dense[0, :, 499], x[0, H:H + G]) and torch.equal(dv[1, :, 129], x[1, H + G:])
    assert float(mass[int(table[1, 1]), :, 1].abs().max()) == 0.0


# ---------------------------------------------------------------- eviction
EVICT = [
    # dtype, G, D, page, lengths, keep, first, recent
    ("bf16", 2, 128, 16, [100, 40, 41, 0, 1], 40, 4, 8),
    ("f16", 1, 64, 48, [500, 499], 100, 0, 0),
    ("f32", 3, 80, 16, [300], 299, 10, 200),
    ("bf16", 8, 128, 64, [2000, 1500, 700], 1000, 16, 256),
    ("f16", 2, 256, 32, [90, 70], 64, 32, 32),
    ("bf16", 1, 8, 16, [33, 17], 1, 0, 0),
    ("f16", 1, 128, 16, [9000, 3], 4500, 1, 1000),
    ("f32", 2, 96, 128, [700, 300], 77, 0, 77),
    ("bf16", 8, 16, 16, [100, 60, 61, 99, 0] * 8, 60, 3, 20),          # more rows and heads than two for every SM
]


@pytest.mark.parametrize("weights", ["spread", "ties", "odd"])
@pytest.mark.parametrize("case", EVICT, ids=lambda c: f"{c[0]}-{c[1]}.{c[2]}-p{c[3]}-{c[4][0]}to{c[5]}")
def test_evict(ops, case, weights):
    """The kept slots are those of the definition exactly, and every moved line arrives unchanged."""
    dtype, G, D, page, lengths, keep, first, recent = case
    c = Cache(lengths, page, G, D, DT[dtype], 21)
    if weights == "ties":
        c.mass = torch.where(torch.isnan(c.mass), c.mass, (c.mass * 3).floor())
    if weights == "odd":                                    # negative numbers, both zeros, infinities, NaN among the candidates
        pick = torch.randint(0, 12, c.mass.shape, generator=c.g)
        for i, x in enumerate((math.nan, math.inf, -math.inf, 0.0, -0.0, -1.0, 1e-40)):
            c.mass[pick == i] = x
    ln = i32(lengths)
    k, v, table, ms = c.cuda()
    kept = torch.full((len(lengths), G, keep), 99, dtype=torch.int32, device="cuda")
    ops.paged_evict(k, v, ms, table, ln.cuda(), kept, first=first, recent=recent)
    exp = po.select(c.mass, c.table, ln, keep, first, recent)
    assert torch.equal(kept.cpu().long(), exp)
    ek, ev, em = po.compact(c.k, c.v, c.mass, c.table, ln, exp)
    assert same(k, ek) and same(v, ev) and same(ms, em)
    assert ops.paged_fault_count(reset=True) == 0


def test_evict_long_rows(ops):
    """Rows longer than the selection can hold at once, checked against a stable sort."""
    G, keep, first, recent = 2, 30000, 7, 1000
    lengths = [150001, 60000]
    c = Cache([1, 1], 4096, G, 8, torch.float16, 22, spare=80)
    P = c.P
    ids = torch.randperm(P, generator=c.g).to(torch.int32)
    table = torch.full((2, 37), -1, dtype=torch.int32)
    table[0], table[1, :15] = ids[:37], ids[37:52]
    mass = (torch.rand((P, G, 4096), generator=c.g) * 5000).floor() / 5000        # many ties
    kept = torch.empty((2, G, keep), dtype=torch.int32, device="cuda")
    ops.paged_select(mass.cuda(), table.cuda(), i32(lengths).cuda(), kept, first, recent)
    for r, n in enumerate(lengths):
        line = mass[table[r][table[r] >= 0].long()].transpose(0, 1).reshape(G, -1)[:, :n]
        for g in range(G):
            order = torch.sort(line[g, first:n - recent], descending=True, stable=True).indices[:keep - first - recent] + first
            exp = torch.cat([torch.arange(first), order.sort().values, torch.arange(n - recent, n)])
            assert torch.equal(kept[r, g].cpu().long(), exp)


def test_evict_rows_longer_than_shared_memory(ops):
    """So many rows that each has one CTA, one of them with more weights than it holds: they are read anew in every pass."""
    G, keep, first, recent, rows, width = 2, 5000, 3, 500, 80, 15
    P = 3 * width
    g = torch.Generator().manual_seed(25)
    table = torch.full((rows, width), -1, dtype=torch.int32)
    for r, at in ((0, 0), (41, width), (79, 2 * width)):
        table[r] = torch.randperm(width, generator=g).to(torch.int32) + at
    lengths = torch.zeros(rows, dtype=torch.int32)
    lengths[0], lengths[41], lengths[79] = 61000, 5000, 50001
    mass = torch.rand((P, G, 4096), generator=g)
    mass[2 * width:] = (mass[2 * width:] * 7).floor()
    kept = torch.empty((rows, G, keep), dtype=torch.int32, device="cuda")
    ops.paged_select(mass.cuda(), table.cuda(), lengths.cuda(), kept, first, recent)
    for r in (0, 79):
        n = int(lengths[r])
        line = mass[table[r].long()].transpose(0, 1).reshape(G, -1)[:, :n]
        for h in range(G):
            order = torch.sort(line[h, first:n - recent], descending=True, stable=True).indices[:keep - first - recent] + first
            assert torch.equal(kept[r, h].cpu().long(), torch.cat([torch.arange(first), order.sort().values, torch.arange(n - recent, n)]))
    assert torch.equal(kept[41].cpu(), torch.arange(5000, dtype=torch.int32).expand(2, -1)) and bool((kept[1] == -1).all())


def test_evict_pages_that_do_not_exist(ops):
    c = Cache([200, 100], 16, 2, 64, torch.bfloat16, 23)
    c.table[0, 3], c.table[1, 0] = -1, c.P
    ln, keep = i32([200, 100]), 60
    k, v, table, ms = c.cuda()
    kept = torch.empty((2, 2, keep), dtype=torch.int32, device="cuda")
    ops.paged_evict(k, v, ms, table, ln.cuda(), kept, first=4, recent=20)
    exp = po.select(c.mass, c.table, ln, keep, 4, 20)
    assert torch.equal(kept.cpu().long(), exp)
    ek, ev, em = po.compact(c.k, c.v, c.mass, c.table, ln, exp)
    assert same(k, ek) and same(v, ev) and same(ms, em)
    assert ops.paged_fault_count(reset=True) > 0


def test_compact_slots_of_the_callers_choice(ops):
    """Fewer kept slots than the list has room for, per head; slots that the row does not have are not read."""
    c = Cache([100, 64], 16, 2, 64, torch.float32, 24)
    kept = torch.full((2, 2, 40), -1, dtype=torch.int32)
    kept[0, 0, :3] = i32([5, 50, 99])
    kept[0, 1, :40] = torch.arange(60, 100, dtype=torch.int32)
    kept[1, 0, :2] = i32([63, 64])
    ln = i32([100, 64])
    for mass in (True, False):
        k, v, table, ms = c.cuda()
        ops.paged_compact(k, v, table, ln.cuda(), kept.cuda(), mass=ms if mass else None)
        ek, ev, em = po.compact(c.k, c.v, c.mass if mass else None, c.table, ln, kept)
        assert same(k, ek) and same(v, ev) and same(ms, em if mass else c.mass)
    ops.paged_fault_count(reset=True)


# ---------------------------------------------------------------- dense view
@pytest.mark.parametrize("dtype,G,D,page,lengths,rows,extra,cap", [
    ("bf16", 8, 128, 128, [777, 1, 128, 129], [0, 1, 2, 3], 0, 1024),
    ("f32", 2, 64, 16, [100, 50], [1, 0, 1], 7, 64),
    ("f16", 3, 80, 48, [100, 0, 47], [2, -1, 1, 0], 1, 256),
    ("bf16", 1, 8, 16, [33], [0], -3, 16),
    ("f16", 1, 256, 256, [1000], [0], 100000, 1100),
])
def test_gather(ops, dtype, G, D, page, lengths, rows, extra, cap):
    c = Cache([n + max(0, min(extra, 20)) for n in lengths], page, G, D, DT[dtype], 31)
    k, v, table, _ = c.cuda()
    dk = torch.full((len(rows), G, cap, D), 3.0, dtype=c.dtype)
    dv = torch.full((len(rows), G, cap, D), 4.0, dtype=c.dtype)
    gk, gv = dk.cuda(), dv.cuda()
    ops.paged_gather(k, v, table, i32(rows).cuda(), i32(lengths).cuda(), gk, gv, extra=extra)
    assert same(gk, po.gather(c.k, c.table, i32(rows), i32(lengths), dk, extra))
    assert same(gv, po.gather(c.v, c.table, i32(rows), i32(lengths), dv, extra))
    assert ops.paged_fault_count(reset=True) == 0


def test_gather_pages_that_do_not_exist(ops):
    c = Cache([100, 40], 16, 2, 64, torch.float16, 32)
    c.table[0, 2] = c.P
    k, v, table, _ = c.cuda()
    dk = torch.full((3, 2, 112, 64), 3.0, dtype=c.dtype)
    gk, gv = dk.cuda(), dk.cuda()
    ops.paged_gather(k, v, table, i32([0, 1, 2]).cuda(), i32([100, 40]).cuda(), gk, gv)
    assert same(gk, po.gather(c.k, c.table, i32([0, 1, 2]), i32([100, 40]), dk, 0))
    assert same(gv, po.gather(c.v, c.table, i32([0, 1, 2]), i32([100, 40]), dk, 0))
    assert ops.paged_fault_count(reset=True) > 0


# ---------------------------------------------------------------- runs of them together
def _decode(ops, dtype, steps, graph):
    """Prompts appended in one call, then decode steps of append and attention with the weights added up; when a row is full it is cut, its tokens keep
    their rotations and the next ones go on at their positions in the text.  -> (device caches, oracle caches, outputs)."""
    H, G, D, page, keep, budget = 8, 2, 64, 16, 40, 56
    dt = DT[dtype]
    c = Cache([budget] * 3, page, G, D, dt, 41, spare=0)
    c.k.fill_(0), c.v.fill_(0), c.mass.fill_(0)
    rates = torch.exp(-torch.arange(32, dtype=torch.float64) / 32 * math.log(1e4)).float()
    k, v, table, ms = c.cuda()
    lengths, texts = i32([50, 30, 47]), i32([50, 30, 47])
    row = i32([r for r, n in enumerate(lengths.tolist()) for _ in range(n)])
    slot = i32([s for n in lengths.tolist() for s in range(n)])
    qkv = c.normal(row.numel(), (H + 2 * G) * D).to(dt)
    ops.paged_append(qkv.cuda(), torch.empty((row.numel(), H * D), dtype=dt, device="cuda"), k, v, table, row.cuda(), slot.cuda(), slot.cuda(), H,
                     rates=rates.cuda(), mass=ms)
    ok, ov, om = k.cpu(), v.cpu(), ms.cpu()                 # the oracle goes on from what the device stored
    rows = torch.arange(3, dtype=torch.int32)
    d = dict(x=torch.empty((3, (H + 2 * G) * D), dtype=dt, device="cuda"), q=torch.empty((3, H * D), dtype=dt, device="cuda"),
             out=torch.empty((3, H * D), dtype=dt, device="cuda"), slot=torch.zeros(3, dtype=torch.int32, device="cuda"),
             pos=torch.zeros(3, dtype=torch.int32, device="cuda"), row=rows.cuda(), rates=rates.cuda(),
             ws=torch.empty((ops.paged_attn_workspace_bytes(3, H, D, table.shape[1] * page),), dtype=torch.uint8, device="cuda"))

    def step():
        ops.paged_append(d["x"], d["q"], k, v, table, d["row"], d["slot"], d["pos"], H, rates=d["rates"], mass=ms)
        ops.paged_attn(d["q"], k, v, table, d["row"], d["slot"], d["out"], 0.25, mass=ms, workspace=d["ws"])

    captured = None
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                       # warm-up of idle tokens: writes nothing
            d["row"].fill_(-1)
            step()
            d["row"].copy_(rows)
        torch.cuda.current_stream().wait_stream(side)
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            step()
    worst = 0.0
    for i in range(steps):
        x = c.normal(3, (H + 2 * G) * D).to(dt)
        d["x"].copy_(x), d["slot"].copy_(lengths), d["pos"].copy_(texts)
        if captured is not None:
            captured.replay()
        else:
            step()
        q = d["q"].cpu()
        at = [po.place(c.table, c.P, page, r, int(lengths[r])) for r in range(3)]
        for p, o in at:                                     # what the device stored is checked by the append's tests
            ok[p, :, o], ov[p, :, o], om[p, :, o] = k.cpu()[p, :, o], v.cpu()[p, :, o], 0.0
        exp, tol, em, off = po.attn(q, ok, ov, om, c.table, rows, lengths, H, 0.25, 0, 0, 0.0 if dt is torch.float32 else po.half_step(dt) ** 2)
        err = (d["out"].cpu().double().view(3, H, D) - exp).abs()
        assert bool((err <= tol + po.half_step(dt) * exp.abs() * 1.001 + 2.0 ** -25).all()), i
        assert bool(((ms.cpu().double() - em).abs() <= off).all()), i
        om = ms.cpu()
        lengths, texts = lengths + 1, texts + 1
        if int(lengths.max()) == budget:
            kept = torch.empty((3, G, keep), dtype=torch.int32, device="cuda")
            ops.paged_evict(k, v, ms, table, lengths.cuda(), kept, first=2, recent=10)
            sel = po.select(om, c.table, lengths, keep, 2, 10)
            assert torch.equal(kept.cpu().long(), sel)
            ok, ov, om = po.compact(ok, ov, om, c.table, lengths, sel)
            assert same(k, ok) and same(v, ov) and same(ms, om)
            lengths = lengths.clamp(max=keep)
    assert ops.paged_fault_count(reset=True) == 0



@pytest.mark.parametrize("graph", [False, True], ids=["eager", "captured"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_decode_with_eviction(ops, dtype, graph):
    _decode(ops, dtype, 40, graph)


def test_two_graphs_share_a_workspace(ops):
    """Captured calls of different sizes on one workspace, replayed in turn and mixed with an eager call."""
    c = Cache([3000, 500, 64], 16, 2, 128, torch.bfloat16, 42)
    k, v, table, ms = c.cuda()
    H = 8
    n = ops.paged_attn_workspace_bytes(3, H, 128, table.shape[1] * 16)
    ws = torch.full((n,), 0x7f, dtype=torch.uint8, device="cuda")
    q = c.normal(3, H * 128).to(c.dtype).cuda()
    calls = [(i32([0, 1, 2]), i32([2999, 499, 63])), (i32([1]), i32([300])), (i32([2, 0]), i32([10, 1500]))]
    calls = [(a.cuda(), b.cuda(), torch.empty((a.numel(), H * 128), dtype=c.dtype, device="cuda")) for a, b in calls]

    def go(i):
        a, b, out = calls[i]
        ops.paged_attn(q[:a.numel()].contiguous(), k, v, table, a, b, out, 0.1, mass=None, workspace=ws)

    exp = []
    for i in range(3):
        go(i)
        exp.append(calls[i][2].clone())
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            go(i)
        graphs.append(g)
    for _ in range(3):
        for x in calls:
            x[2].fill_(math.nan)
        graphs[0].replay(), go(2), graphs[1].replay(), graphs[0].replay()
        torch.cuda.synchronize()
        for i in range(3):
            assert same(calls[i][2], exp[i]), i


def test_on_a_stream_of_its_own(ops):
    c = Cache([3000, 500], 16, 2, 128, torch.bfloat16, 43)
    k, v, table, ms = c.cuda()
    q = c.normal(2, 8 * 128).to(c.dtype).cuda()
    row, slot = i32([0, 1]).cuda(), i32([2999, 499]).cuda()
    outs = [torch.zeros((2, 8 * 128), dtype=c.dtype, device="cuda") for _ in range(3)]
    ws = [torch.empty((max(16, ops.paged_attn_workspace_bytes(2, 8, 128, 0)),), dtype=torch.uint8, device="cuda") for _ in range(3)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ops.paged_attn(q, k, v, table, row, slot, outs[2], 0.1, workspace=ws[2])
    for _ in range(20):                                     # two calls at once, a workspace each
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                ops.paged_attn(q, k, v, table, row, slot, outs[i], 0.1, workspace=ws[i])
    torch.cuda.synchronize()
    assert same(outs[0], outs[2]) and same(outs[1], outs[2])


def test_prompt_through_the_dense_view(ops):
    """A prompt in two portions: append, dense view, prompt attention; the same as the attention of single tokens over the pages."""
    H, G, D, page, n = 8, 2, 128, 64, 200
    dt = torch.float16
    c = Cache([n], page, G, D, dt, 44)
    k, v, table, ms = c.cuda()
    rates = torch.exp(-torch.arange(64, dtype=torch.float64) / 64 * math.log(1e4)).float().cuda()
    row0 = i32([0]).cuda()
    for lo, hi in ((0, 77), (77, n)):
        L = hi - lo
        qkv = c.normal(L, (H + 2 * G) * D).to(dt).cuda()
        row, slot = torch.zeros(L, dtype=torch.int32, device="cuda"), torch.arange(lo, hi, dtype=torch.int32, device="cuda")
        q = torch.empty((L, H * D), dtype=dt, device="cuda")
        ops.paged_append(qkv, q, k, v, table, row, slot, slot, H, rates=rates, mass=ms)
        before = i32([lo]).cuda()
        dk = torch.zeros((1, G, 256, D), dtype=dt, device="cuda")
        dv = torch.zeros_like(dk)
        ops.paged_gather(k, v, table, row0, before, dk, dv, extra=L)
        a, b = torch.empty_like(q), torch.empty_like(q)
        ws = torch.empty((max(16, ops.attn_workspace_bytes(1, L, H, D)),), dtype=torch.uint8, device="cuda")
        ops.attn(q, dk, dv, before, a, 1, L, H, G, D, D ** -0.5, workspace=ws)
        ws2 = torch.empty((max(16, ops.paged_attn_workspace_bytes(L, H, D, 0)),), dtype=torch.uint8, device="cuda")
        ops.paged_attn(q, k, v, table, row, slot, b, D ** -0.5, workspace=ws2)
        # weights and results rounded to f16 on either side: 2 x (2^-11 + 2^-11) of sums of at most sum p |v|
        bound = 4 * 2.0 ** -11 * float(v[~torch.isnan(v)].abs().max()) 
        assert float((a.float() - b.float()).abs().max()) <= bound


# ---------------------------------------------------------------- refusals
def test_refusals(ops):
    from mlx_parallm_b200._lib import B200PError
    c = Cache([100, 50], 16, 2, 64, torch.bfloat16, 51)
    k, v, table, ms = c.cuda()
    q = torch.zeros((2, 8 * 64), dtype=torch.bfloat16, device="cuda")
    out, row, slot = torch.zeros_like(q), i32([0, 1]).cuda(), i32([99, 49]).cuda()
    ws = torch.empty((ops.paged_attn_workspace_bytes(2, 8, 64, 0) + 16,), dtype=torch.uint8, device="cuda")
    x = torch.zeros((2, 12 * 64), dtype=torch.bfloat16, device="cuda")
    ln, kept = i32([100, 50]).cuda(), torch.zeros((2, 2, 20), dtype=torch.int32, device="cuda")
    dk = torch.zeros((2, 2, 128, 64), dtype=torch.bfloat16, device="cuda")
    A = lambda **kw: ops.paged_attn(**{**dict(q=q, kpages=k, vpages=v, table=table, t_row=row, t_slot=slot, out=out, scale=0.1, workspace=ws), **kw})
    W = lambda **kw: ops.paged_append(**{**dict(qkv=x, q_out=out, kpages=k, vpages=v, table=table, t_row=row, t_slot=slot, t_pos=slot, H=8), **kw})
    E = lambda **kw: ops.paged_evict(**{**dict(kpages=k, vpages=v, mass=ms, table=table, lengths=ln, kept=kept), **kw})
    Gt = lambda **kw: ops.paged_gather(**{**dict(kpages=k, vpages=v, table=table, rows=row, lengths=ln, kcache=dk, vcache=dk.clone()), **kw})
    A(), W(), E(), Gt()
    f32 = torch.zeros((2, 8 * 64), device="cuda")
    bad = [
        (A, dict(q=f32)), (A, dict(out=f32)), (A, dict(q=q[:1])), (A, dict(q=q.cpu())), (A, dict(kpages=k[:1])), (A, dict(vpages=v.half())),
        (A, dict(kpages=k.transpose(1, 2))), (A, dict(table=table.long())), (A, dict(table=table[0])), (A, dict(t_row=row.long())),
        (A, dict(t_slot=slot[:1])), (A, dict(mass=ms[:1])), (A, dict(mass=ms)), (A, dict(mass=ms.double())), (A, dict(first=-1)), (A, dict(window=-1)),
        (A, dict(q=torch.zeros((2, 7 * 64), dtype=torch.bfloat16, device="cuda"), out=torch.zeros((2, 7 * 64), dtype=torch.bfloat16, device="cuda"))),
        (A, dict(kpages=k[:, :, :8].contiguous(), vpages=v[:, :, :8].contiguous())),
        (A, dict(kpages=k[:, :, :, :60].contiguous(), vpages=v[:, :, :, :60].contiguous())),
        (W, dict(qkv=x[:, :-1])), (W, dict(qkv=x.half())), (W, dict(qkv=x.t())), (W, dict(qkv=x[:1])), (W, dict(q_out=f32)), (W, dict(t_pos=slot.long())),
        (W, dict(rates=torch.zeros(33, device="cuda"))), (W, dict(rates=torch.zeros(32, device="cuda").double())), (W, dict(pairs=2)),
        (W, dict(q_norm_w=torch.ones(32, dtype=torch.bfloat16, device="cuda"))), (W, dict(k_norm_w=torch.ones(64, device="cuda"))), (W, dict(qkv=x.cpu())),
        (W, dict(H=7)), (W, dict(qkv=x[:1].expand(2, -1))),
        (E, dict(first=15, recent=6)), (E, dict(first=-1)), (E, dict(recent=-1)), (E, dict(kept=kept[:, :1].contiguous())), (E, dict(kept=kept.long())),
        (E, dict(lengths=ln.long())), (E, dict(mass=ms[:, :1].contiguous())), (E, dict(mass=None)), (E, dict(kept=kept[:, :, :0])),
        (Gt, dict(rows=row.long())), (Gt, dict(lengths=ln[:1])), (Gt, dict(kcache=dk[:1])), (Gt, dict(kcache=dk.half())), (Gt, dict(vcache=dk[:, :, :64])),
    ]
    before = [t.clone() for t in (k, v, ms, out)]
    for i, (f, kw) in enumerate(bad):
        with pytest.raises((ValueError, B200PError, AttributeError)):
            f(**kw)
            pytest.fail(f"not refused: {i} {list(kw)}")
    assert all(same(a, b) for a, b in zip(before, (k, v, ms, out)))
    small = torch.empty((16,), dtype=torch.uint8, device="cuda")
    with pytest.raises(B200PError):
        A(mass=ms, workspace=small)


def test_advance_of_the_rows_in_use(ops):
    """Counters of rows whose index is negative stay; one launch, captured and replayed."""
    n = 700
    rows = torch.arange(n, dtype=torch.int32)
    rows[torch.tensor([0, 5, 255, 256, 699])] = i32([-1, -7, -1, -2, -1])
    a, b = torch.arange(n, dtype=torch.int32).cuda(), (3 * torch.arange(n, dtype=torch.int32)).cuda()
    rows = rows.cuda()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.paged_advance(a, b, rows, 7)
    g.replay()
    ops.paged_advance(a, b, rows, -2)
    up = torch.where(rows.cpu() < 0, 0, 5)
    assert torch.equal(a.cpu(), torch.arange(n) + up) and torch.equal(b.cpu(), 3 * torch.arange(n) + up)
    for bad in (dict(lengths=a[:5]), dict(positions=b.long()), dict(rows=rows[::2])):
        with pytest.raises(ValueError):
            ops.paged_advance(**{**dict(lengths=a, positions=b, rows=rows, delta=1), **bad})


def test_plan_of_idle_entries(ops):
    """An entry of a negative row (next to others): its tokens are idle, its history is not looked at."""
    cu, rows, lengths = i32([0, 3, 5, 9]).cuda(), i32([1, -1, 0]).cuda(), i32([40, 7]).cuda()
    row, pos, off = (torch.full((9,), 99, dtype=torch.int32, device="cuda") for _ in range(3))
    ops.ragged_plan(cu, rows, lengths, row, pos, off, 3, 9)
    assert row.tolist() == [1] * 3 + [-1] * 2 + [0] * 4 and pos.tolist() == [7, 8, 9, 0, 1, 40, 41, 42, 43] and off.tolist() == [0, 1, 2, 0, 1, 0, 1, 2, 3]


@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("f32", 40)])
def test_slots_behind_the_table_are_counted(ops, dtype, D):
    """A token whose slot is behind the table sees what its row holds, and each is counted once; one at the last slot, and a negative one, are not."""
    c = Cache([64, 64, 64, 64], 16, 2, D, DT[dtype], 61)
    for n in (0, 600):                                              # few tokens, and more than a CTA keeps
        row, slot = i32([0, 1, 2, 3] + [-1] * n), i32([64, 63, (1 << 31) - 1, -1] + [1 << 20] * n)
        q = c.normal(4 + n, 8 * D).to(c.dtype)
        for mass in (False, True):
            _check_attn(ops, c, q, row, slot, 8, 0, 0, mass, 0.2)
            assert ops.paged_fault_count(reset=True) == 2
    _check_attn(ops, c, c.normal(3, 8 * D).to(c.dtype), i32([0, 1, 2]), i32([63, 62, -3]), 8, 1, 5, True, 0.2)
    assert ops.paged_fault_count(reset=True) == 0


def test_lengths_behind_the_table_are_counted(ops):
    """Selection, closing up and the dense view take such a row for full, once counted in each call; ``extra`` behind the table's end is not."""
    c = Cache([64, 64, 40], 16, 2, 64, torch.bfloat16, 62)
    ln, keep = i32([65, 64, 1 << 30]), 30
    k, v, table, ms = c.cuda()
    kept = torch.empty((3, 2, keep), dtype=torch.int32, device="cuda")
    c.table[2, 3] = c.table[2, 2]                                   # (a page for each of row 2's slots)
    table.copy_(c.table)
    ops.paged_select(ms, table, ln.cuda(), kept, first=2, recent=4)
    assert ops.paged_fault_count(reset=True) == 2
    exp = po.select(c.mass, c.table, ln, keep, 2, 4)
    assert torch.equal(kept.cpu().long(), exp)
    kept[2] = torch.arange(keep, dtype=torch.int32)                 # (nothing moves in the row with a page twice)
    ops.paged_compact(k, v, table, ln.cuda(), kept, mass=ms)
    assert ops.paged_fault_count(reset=True) == 2
    ek, ev, em = po.compact(c.k, c.v, c.mass, c.table, ln.clamp(max=64), kept.cpu().long())
    assert same(k, ek) and same(v, ev) and same(ms, em)
    dk = torch.full((4, 2, 80, 64), 3.0, dtype=c.dtype)
    gk, gv = dk.cuda(), dk.cuda()
    ops.paged_gather(k, v, table, i32([0, 1, 0, -1]).cuda(), ln.cuda(), gk, gv, extra=9)
    assert ops.paged_fault_count(reset=True) == 2                   # (row 0, twice)
    assert same(gk, po.gather(ek, c.table, i32([0, 1, 0, -1]), ln, dk, 9))

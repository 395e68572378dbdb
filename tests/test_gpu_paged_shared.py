"""b200p_paged_attn_shared against the definition in 64 bits, token by token over its own table row."""
import pytest
import torch

from mlx_parallm_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(autouse=True)
def by_groups():
    """The kernels for groups, whatever the sizes."""
    _lib.lib().b200p_paged_attn_shared_set_path(1)
    yield
    _lib.lib().b200p_paged_attn_shared_set_path(0)


class Case:
    """Rows of ``lengths`` slots; rows of group g have their first ``prefix[g]`` slots (whole pages) in common."""

    def __init__(self, group, prefix, lengths, H=32, G=8, D=128, page=16, dtype="bf16", seed=0, spread=1.5, spare=3, poison=True):
        gen = torch.Generator().manual_seed(seed)
        B = len(group)
        need = [-(-n // page) for n in lengths]
        heads = [p // page for p in prefix]
        P = sum(heads) + sum(max(0, k - (heads[g] if 0 <= g < len(heads) else 0)) for g, k in zip(group, need)) + spare
        ids = torch.randperm(P, generator=gen).tolist()
        common = [[ids.pop() for _ in range(k)] for k in heads]
        table = torch.full((B, max(need) + 2), -1, dtype=torch.int32)
        for i, (g, k) in enumerate(zip(group, need)):
            row = common[g][:k] if 0 <= g < len(heads) else []
            row = row + [ids.pop() for _ in range(k - len(row))]
            table[i, :k] = torch.tensor(row, dtype=torch.int32)
        dev, dt = torch.Generator(device="cuda").manual_seed(seed), DT[dtype]
        normal = lambda *s: torch.randn(s, generator=dev, device="cuda")
        self.k, self.v = normal(P, G, page, D).to(dt), normal(P, G, page, D).to(dt)
        if poison:                                                  # what nobody may look at: pages of nobody, slots behind a row's last
            used = torch.zeros((P, page), dtype=torch.bool)
            for i, n in enumerate(lengths):
                for j in range(-(-n // page)):
                    if table[i, j] >= 0:
                        used[table[i, j], :min(page, n - j * page)] = True
            hide = ~used.cuda()[:, None, :, None]
            self.k.masked_fill_(hide, float("nan")), self.v.masked_fill_(hide, float("inf"))
        self.q = (spread * normal(B, H * D)).to(dt)
        self.table, self.H, self.G, self.D, self.page, self.P = table.cuda(), H, G, D, page, P
        self.row = torch.arange(B, dtype=torch.int32, device="cuda")
        self.slot = torch.tensor(lengths, dtype=torch.int32, device="cuda") - 1
        self.group = torch.tensor(group, dtype=torch.int32, device="cuda")
        self.prefix = torch.tensor(prefix, dtype=torch.int32, device="cuda")
        self.scale = D ** -0.5

    def workspace(self):
        n = ops.paged_attn_shared_workspace_bytes(self.row.numel(), self.H, self.G, self.D, self.prefix.numel())
        return torch.randint(0, 256, (n,), dtype=torch.uint8, device="cuda")

    def plan(self):
        return ops.row_groups(self.group, self.prefix.numel(), ops.paged_attn_shared_tile(self.H, self.G))

    def run(self, out=None, ws=None, plan=None, **kw):
        out = torch.full_like(self.q, 7.0) if out is None else out
        return ops.paged_attn_shared(self.q, self.k, self.v, self.table, self.row, self.slot, out, self.scale, self.group, self.prefix,
                                     self.plan() if plan is None else plan, workspace=self.workspace() if ws is None else ws, **kw)

    def want(self):
        """(outputs, their slack): idle tokens stay as they are."""
        H, G, D, page = self.H, self.G, self.D, self.page
        out = torch.full(self.q.shape, 7.0, dtype=torch.float64, device="cuda")
        slack = torch.zeros_like(out)
        half = torch.finfo(self.q.dtype).eps / 2
        table = self.table.tolist()
        for t, (r, s) in enumerate(zip(self.row.tolist(), self.slot.tolist())):
            if not 0 <= r < len(table):
                continue
            n = min(s + 1, len(table[r]) * page)
            keys = [j for j in range(max(n, 0)) if 0 <= table[r][j // page] < self.P]
            if not keys:
                out[t] = 0
                continue
            j = torch.tensor(keys, device="cuda")
            ids = self.table[r].long()[j // page]
            k, v = self.k[ids, :, j % page].double(), self.v[ids, :, j % page].double()           # [n, G, D]
            q = self.q[t].double().view(G, H // G, D)
            score = torch.einsum("ghd,jgd->ghj", q, k) * self.scale
            p = torch.softmax(score, -1)
            o = torch.einsum("ghj,jgd->ghd", p, v)
            size = torch.einsum("ghd,jgd->ghj", q.abs(), k.abs()).amax(-1, keepdim=True) * self.scale
            spread = torch.einsum("ghj,jgd->ghd", p, v.abs())
            # the output's rounding; a weight's, half a step of its type, in the numerator and its sum; the score's sums in fp32 (D / 16 products and some joins
            # of a unit of 2^-23 each), which the exponential turns into relative errors, in both; 2^x, the joins
            tol = half * o.abs() + spread * (2 * half + 2 * (D / 16 + 8) * 2.0 ** -23 * size + 2.0 ** -19)
            out[t], slack[t] = o.reshape(-1), tol.reshape(-1)
        return out, slack

    def check(self, got=None, **kw):
        got = self.run(**kw) if got is None else got
        out, slack = self.want()
        diff = (got.double() - out).abs()
        assert diff.le(slack).all(), (float(diff.max()), float((diff - slack).max()), (diff > slack).any(-1).nonzero()[:8, 0].tolist())
        return got


SHAPES = [(32, 8, 128), (40, 8, 128), (64, 8, 128), (32, 32, 96), (4, 2, 64), (16, 2, 256), (12, 1, 64), (25, 5, 80), (64, 4, 128), (128, 1, 64), (130, 1, 64),
          (9, 1, 256), (24, 1, 96), (6, 2, 72), (4, 2, 8)]


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,G,D", SHAPES)
def test_heads_and_sizes(H, G, D, dtype):
    Case([0, 0, 1, -1, 0, 1], [96, 160], [97, 130, 161, 50, 200, 333], H=H, G=G, D=D, dtype=dtype).check()


@pytest.mark.parametrize("page", [16, 32, 48, 64, 112, 256, 1024])
@pytest.mark.parametrize("pages", [1, 2, 3, 5])
def test_pages(page, pages):
    Case([0] * 5, [page * pages], [page * pages + i for i in (1, 15, 16, 17, 40)], H=8, G=2, D=64, page=page).check()


@pytest.mark.parametrize("B", [1, 2, 3, 31, 32, 33, 64, 65, 100])
def test_group_sizes(B):
    Case([0] * B, [208], [209 + 7 * i % 90 for i in range(B)], H=8, G=2, dtype="f16").check()


@pytest.mark.parametrize("B", [127, 128, 129, 300, 600])
def test_groups_of_many_tokens(B):
    Case([i % 2 for i in range(B)], [128, 64], [129 + i % 50 for i in range(B)], H=4, G=4, D=64).check()


def test_many_groups():
    Case([i // 3 if i % 7 else -1 for i in range(200)], [16 * (1 + g % 9) for g in range(67)], [160 + i % 33 for i in range(200)], H=8, G=2, D=64).check()
    Case(list(range(40)), [16 * (1 + g % 9) for g in range(40)], [150 + g for g in range(40)], H=8, G=2, D=64).check()      # one row each
    Case([5, 5, 900], [160] * 1024, [161, 170, 180], H=8, G=2, D=64).check()


@pytest.mark.parametrize("prefix", [4000, 16000])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_long_shared_slots(prefix, dtype):
    Case([0] * 20 + [1] * 3 + [-1], [prefix, 512], [prefix + 1 + 37 * i for i in range(20)] + [600, 700, 513] + [90], dtype=dtype).check()


def test_own_slots_from_none_to_many():
    Case([0] * 8, [320], [320, 321, 336, 352, 1000, 5000, 320, 20000], H=8, G=2).check()


def test_a_token_among_the_shared_slots_reads_what_it_sees():
    c = Case([0] * 6, [256], [300, 256, 255, 1, 100, 257], H=8, G=2)
    c.check()
    c = Case([0] * 3, [256], [255, 17, 1], H=8, G=2)                # none holds all of them
    c.check()


@pytest.mark.parametrize("prefix", [1, 5, 16, 17, 63, 64, 65, 100, 160])
def test_shared_slots_that_end_inside_a_page(prefix):
    c = Case([0] * 5, [160], [161, 170, 190, 200, 210], H=8, G=2, page=32)
    c.prefix.fill_(prefix)
    c.check()


def test_rows_that_are_the_same_row():
    c = Case([0] * 40, [160], [200] * 40, H=8, G=2)
    c.row.fill_(3)
    c.check()


def test_no_shared_slots():
    for prefix in (0, -5, -2 ** 31):
        c = Case([0, 0, 1], [64, 64], [70, 80, 90], H=8, G=2)
        c.prefix.fill_(prefix)
        c.check()
    c = Case([-1, -1], [64], [70, 80], H=8, G=2)
    c.check()


def test_more_shared_slots_than_the_table_has():
    c = Case([0, 0], [64], [90, 100], H=8, G=2)
    c.prefix.fill_(2 ** 31 - 1)
    c.check()


def test_idle_tokens_and_strange_groups():
    c = Case([0, 0, 0, 1, 1, 2, 7, -9, 0], [64, 64, 64], [70, 80, 90, 100, 70, 80, 90, 66, 67], H=8, G=2)
    c.row[0] = -1                                                   # a group's first member
    c.row[3], c.row[4] = -1, -7                                     # all of a group
    ops.paged_fault_count(reset=True)
    c.check()
    assert ops.paged_fault_count(reset=True) == 0
    c.row[1] = 9                                                    # behind the table
    c.check()
    assert ops.paged_fault_count(reset=True) > 0
    c.slot[2], c.row[1] = -1, 1                                     # sees nothing
    c.check()
    assert ops.paged_fault_count(reset=True) == 0
    c.row.fill_(-1)
    c.check()


@pytest.mark.parametrize("bad", [-1, -2 ** 31, 2 ** 31 - 1])
def test_ids_that_name_no_page(bad):
    c = Case([0] * 4, [160], [161, 170, 200, 230], H=8, G=2, poison=False)
    c.table[:, 4] = bad                                             # shared
    c.table[2, 11] = bad                                            # own
    ops.paged_fault_count(reset=True)
    c.check()
    assert ops.paged_fault_count(reset=True) > 0
    c.table[:, :10] = bad                                           # all shared ones
    c.check()
    c.table.fill_(bad)
    assert (c.run() == 0).all()
    ops.paged_fault_count(reset=True)


@pytest.mark.parametrize("spread", [0.0, 1e-3, 30.0])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_flat_and_sharp_weights(spread, dtype):
    Case([0] * 9, [2048], [2049 + 100 * i for i in range(9)], H=8, G=2, spread=spread, dtype=dtype).check()


def test_growing_scores():
    """Every tile has a new maximum."""
    c = Case([0] * 9, [1024], [1025 + 30 * i for i in range(9)], H=8, G=2, D=64, dtype="f16", poison=False)
    c.q.fill_(0.5)
    order = torch.arange(c.table.shape[1] * c.page, device="cuda").float() / 400
    for r in range(9):
        for j, i in enumerate(c.table[r].tolist()):
            if i >= 0:
                c.k[i] = order[j * c.page:(j + 1) * c.page, None].half()
    c.check()


def test_scores_of_minus_infinity():
    c = Case([0] * 3, [128], [129, 150, 170], H=8, G=2, D=64, poison=False)
    c.q.abs_()
    for j in range(8):
        c.k[c.table[0, j].item()] = float("-inf")
    got = c.run()
    c.table[:, :8] = -1                                             # the same as no shared slot
    out, slack = c.want()
    assert (got.double() - out).abs().le(slack).all()
    ops.paged_fault_count(reset=True)


@pytest.mark.parametrize("H,G,D,page", [(32, 8, 128, 256), (32, 8, 64, 512)])
def test_pages_behind_32_bits(H, G, D, page):
    """A pool of more than 2^31 elements, whose last pages are the ones in use."""
    c = Case([0] * 9 + [1, 1, -1], [2 * page, page], [2 * page + 1 + 9 * i for i in range(9)] + [page + 5, page + 300, 70], H=H, G=G, D=D, page=page, dtype="f16",
             poison=False)
    room = (2 ** 31 + 2 ** 28) // (G * page * D)
    for name in ("k", "v"):
        small = getattr(c, name)
        large = torch.empty((room + c.P, G, page, D), dtype=small.dtype, device="cuda")
        large[room:] = small
        setattr(c, name, large)
    c.table = torch.where(c.table >= 0, c.table + room, c.table)
    c.P += room
    c.check()


def test_as_paged_attn_does():
    c = Case([0] * 30, [1600], [1601 + 11 * i for i in range(30)])
    got = c.check()
    ws = torch.empty((ops.paged_attn_workspace_bytes(30, 32, 128, 0, 8),), dtype=torch.uint8, device="cuda")
    plain = ops.paged_attn(c.q, c.k, c.v, c.table, c.row, c.slot, torch.empty_like(c.q), c.scale, workspace=ws)
    out, slack = c.want()
    assert (plain.double() - out).abs().le(slack).all() and (got.double() - plain.double()).abs().le(2 * slack).all()


def test_permuted_outputs():
    c = Case([0] * 5, [160], [161, 170, 190, 200, 210])
    plain, perm = c.run(), c.run(out_perm=True)
    order = torch.tensor([0, 4, 1, 5, 2, 6, 3, 7], device="cuda")
    assert torch.equal(plain.view(-1, 8)[:, order], perm.view(-1, 8))


def test_same_bits_every_time():
    c = Case([i % 3 for i in range(40)], [640, 320, 1600], [1601 + 11 * i for i in range(40)])
    first, plan, ws = c.run(), c.plan(), c.workspace()
    for _ in range(5):
        assert torch.equal(first, c.run(plan=plan, ws=ws))


def test_graph_rows_that_grow_and_other_groups():
    c = Case([i % 2 for i in range(12)], [160, 320], [400] * 12, H=8, G=2)
    plan, ws, out = c.plan(), c.workspace(), torch.full_like(c.q, 7.0)
    c.run(out=out, plan=plan, ws=ws)
    c.slot.fill_(330)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(2):                                          # layers, one after the other in one workspace
            c.run(out=out, plan=plan, ws=ws)
    for slots in (330, 350, 399):
        c.slot.fill_(slots)
        g.replay()
        c.check(got=out)
    c.group[::4] = -1                                               # rows that leave their group: the plan's buffer is written anew
    ops.row_groups(c.group, 2, plan.tile, out=plan)
    c.prefix.copy_(torch.tensor([64, 0], dtype=torch.int32))
    c.row[3] = -1
    out.fill_(7.0)
    g.replay()
    c.check(got=out)


def test_two_streams():
    cases = [Case([0] * 20, [800], [801 + i for i in range(20)], seed=s, H=8, G=2) for s in (1, 2)]
    streams = [torch.cuda.Stream() for _ in cases]
    kept = [(c.plan(), c.workspace(), torch.full_like(c.q, 7.0)) for c in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, s, (plan, ws, out) in zip(cases, streams, kept):
            with torch.cuda.stream(s):
                c.run(out=out, plan=plan, ws=ws)
    torch.cuda.synchronize()
    for c, (_, _, out) in zip(cases, kept):
        c.check(got=out)


def test_refusals():
    c = Case([0, 0, 1], [64, 64], [70, 80, 90], H=8, G=2)
    keep = torch.full_like(c.q, 7.0)
    args = dict(q=c.q, kpages=c.k, vpages=c.v, table=c.table, t_row=c.row, t_slot=c.slot, out=keep, scale=c.scale, group=c.group, prefix=c.prefix, plan=c.plan(),
                workspace=c.workspace())
    for bad in (dict(q=c.q.float()), dict(q=c.q[:2]), dict(out=keep[:2]), dict(kpages=c.k.half()), dict(table=c.table.long()), dict(t_row=c.row.long()),
                dict(t_slot=c.slot[:2]), dict(group=c.group.long()), dict(group=c.group[:2]), dict(prefix=c.prefix.long()), dict(prefix=c.prefix[:1]),
                dict(plan=c.plan()._replace(rows=4)), dict(plan=ops.row_groups(c.group, 2, 7)), dict(plan=ops.row_groups(c.group, 3, args["plan"].tile)),
                dict(workspace=None), dict(workspace=c.workspace()[:-256]), dict(workspace=c.workspace()[1:]), dict(group=c.group.cpu()), dict(q=c.q.cpu())):
        with pytest.raises((ValueError, RuntimeError)):
            ops.paged_attn_shared(**dict(args, **bad))
    assert (keep == 7.0).all()


@pytest.mark.parametrize("path", [0, 2])
def test_by_the_rule_and_by_tokens(path):
    """The rule sends small calls past the groups; by tokens the bits are paged_attn's."""
    _lib.lib().b200p_paged_attn_shared_set_path(path)
    small = Case([0] * 5, [160], [161, 170, 190, 200, 210])
    ws = torch.empty((ops.paged_attn_workspace_bytes(5, 32, 128, 0, 8),), dtype=torch.uint8, device="cuda")
    plain = ops.paged_attn(small.q, small.k, small.v, small.table, small.row, small.slot, torch.empty_like(small.q), small.scale, workspace=ws)
    assert torch.equal(small.check(), plain)
    Case([0] * 12, [1600], [1601 + i for i in range(12)]).check()


def fine_slack(c, out):
    """How far outputs may be off when their own rounding is the only one to fewer than 32 bits that shows (``out`` [M, H D] the definition): a weight is two 16-bit
    numbers, off by half a step of what the first lost, half * half, and in f16 by 2^-25 at least where the largest weight is 2^8 or more; products of 16 keys
    are added up in fp32, a unit of 2^-23 each; a score's sums as in Case.want; 2^x and the joins."""
    H, G, D, page, half = c.H, c.G, c.D, c.page, torch.finfo(c.q.dtype).eps / 2
    tol = half * out.abs() + torch.finfo(c.q.dtype).tiny * half      # (half a step of the type's smallest numbers)
    for t, (r, s) in enumerate(zip(c.row.tolist(), c.slot.tolist())):
        n = s + 1
        j = torch.arange(n, device="cuda")
        ids = c.table[r].long()[j // page]
        k, v = c.k[ids, :, j % page].double(), c.v[ids, :, j % page].double()
        q = c.q[t].double().view(G, H // G, D)
        p = torch.softmax(torch.einsum("ghd,jgd->ghj", q, k) * c.scale, -1)
        size = torch.einsum("ghd,jgd->ghj", q.abs(), k.abs()).amax(-1, keepdim=True) * abs(c.scale)
        spread = torch.einsum("ghj,jgd->ghd", p, v.abs())
        lost = spread * (half * half + (n / 16 + 2 * (D / 16 + 8) * size) * 2.0 ** -23 + 2.0 ** -19) + n * 2.0 ** -33 * v.abs().amax(0)[:, None]
        tol[t] += lost.reshape(-1)
    return tol


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("H,G,D", [(32, 8, 128), (40, 8, 128), (4, 2, 64), (25, 5, 80), (32, 32, 96), (16, 2, 256)])
@pytest.mark.parametrize("spread,scale", [(0.2, 1.0), (1.5, 1.0), (0.2, -1.0)])
def test_outputs_carry_their_own_rounding_only(H, G, D, dtype, spread, scale):
    c = Case([0, 0, 1, 0, 0, 1], [160, 640], [161, 170, 641, 165, 163, 650], H=H, G=G, D=D, dtype=dtype, spread=spread)
    c.scale *= scale                                                # (a negative one goes through the mma.sync kernel for all sizes)
    got, (out, _) = c.run(), c.want()
    diff, tol = (got.double() - out).abs(), fine_slack(c, out)
    assert diff.le(tol).all(), (float((diff - tol).max()), float((diff > tol).double().mean()))


@pytest.mark.parametrize("H,G,D,dtype", [(32, 8, 128, "bf16"), (12, 1, 64, "f16"), (9, 9, 80, "f16"), (130, 1, 64, "bf16")])
def test_parts_stay_in_the_workspace(H, G, D, dtype):
    """Groups of one to thirty rows, each cut over several CTAs: every part in a place of its own, and nothing behind the workspace."""
    sizes = [1, 30, 2, 7, 1, 1, 16, 3]
    group = [g for g, n in enumerate(sizes) for _ in range(n)] + [-1]
    prefix = [2048 - 240 * g for g in range(len(sizes))]
    c = Case(group, prefix, [(prefix[g] if g >= 0 else 40) + 1 + 11 * i % 50 for i, g in enumerate(group)], H=H, G=G, D=D, dtype=dtype)
    n = ops.paged_attn_shared_workspace_bytes(len(group), H, G, D, len(sizes))
    ws = torch.randint(0, 256, (n + (1 << 20),), dtype=torch.uint8, device="cuda")
    behind = ws[n:].clone()
    c.check(ws=ws[:n])
    assert torch.equal(ws[n:], behind)


def test_few_shared_slots_are_read_by_every_token():
    """Where the table has no room for 64 MiB in common (here 63 and 47 MiB) a call is paged_attn's, bit by bit."""
    _lib.lib().b200p_paged_attn_shared_set_path(0)
    for B, prefix, tail in ((2, 16000, 40), (20, 512, 50)):
        c = Case([0] * B, [prefix], [prefix + 1 + i * tail // B for i in range(B)], page=64, poison=False)
        room = (B - 1) * c.table.shape[1] * 64 * 8 * 128 * 4
        assert 32 << 20 <= room < 64 << 20
        n = ops.paged_attn_workspace_bytes(B, 32, 128, 0, 8)
        alone = ops.paged_attn(c.q, c.k, c.v, c.table, c.row, c.slot, torch.empty_like(c.q), c.scale, workspace=torch.empty((n,), dtype=torch.uint8, device="cuda"))
        assert torch.equal(c.run(), alone)

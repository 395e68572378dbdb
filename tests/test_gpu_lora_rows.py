"""b200p_row_groups and b200p_lora_rows against their definitions in 64 bits."""
import pytest
import torch

from mlx_parallm_b200 import ops

pytestmark = pytest.mark.gpu
DT = {"f16": torch.float16, "bf16": torch.bfloat16}


def index_of(M, n, seed=0, none=True):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-1 if none else 0, n, (M,), generator=g, dtype=torch.int32)


# ---------------------------------------------------------------------------------------------------------------- plans
def check_plan(index, groups, tile):
    M = index.numel()
    plan = ops.row_groups(index.cuda(), groups, tile)
    d, want = plan.data.cpu().tolist(), index.tolist()
    order = [i for g in range(groups) for i in range(M) if want[i] == g] if groups < 50 else sorted((i for i in range(M) if 0 <= want[i] < groups),
                                                                                                      key=lambda i: (want[i], i))
    sizes = [0] * groups
    for i in order:
        sizes[want[i]] += 1
    tiles, at = [], 0
    for g, k in enumerate(sizes):
        tiles += [[g, at + x, min(tile, k - x), at] for x in range(0, k, tile)]
        at += k
    assert d[:4] == [len(tiles), len(order), sum(v >= groups for v in want), tile]
    assert d[4:4 + len(order)] == order
    base = 4 + (M + 3) // 4 * 4
    assert len(d) == base + 4 * (M // tile + min(M, groups)) and len(d) - base >= 4 * len(tiles)
    assert [d[base + 4 * k:base + 4 * k + 4] for k in range(len(tiles))] == tiles


@pytest.mark.parametrize("tile", [1, 7, 16, 64])
@pytest.mark.parametrize("M", [0, 1, 2, 3, 31, 32, 33, 500, 511, 512, 513, 1500, 9001])
@pytest.mark.parametrize("groups", [1, 2, 33, 1024])
def test_plans(M, groups, tile):
    check_plan(index_of(M, groups, seed=M + groups), groups, tile)


def test_plans_of_strange_indexes():
    for groups in (1, 5, 700):
        check_plan(torch.full((77,), -1, dtype=torch.int32), groups, 16)
        check_plan(torch.full((77,), groups - 1, dtype=torch.int32), groups, 16)
        check_plan(torch.full((77,), groups, dtype=torch.int32), groups, 16)
        check_plan(torch.tensor([2 ** 31 - 1, -2 ** 31, 0, groups, groups - 1, -5] * 9, dtype=torch.int32), groups, 16)
        check_plan(torch.arange(2000, dtype=torch.int32) % groups, groups, 16)


def test_a_plan_is_rewritten_in_a_graph():
    index = index_of(200, 6).cuda()
    plan = ops.row_groups(index, 6, 16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert ops.row_groups(index, 6, 16, out=plan) is plan
    index.copy_(index_of(200, 6, seed=5))
    g.replay()
    fresh = ops.row_groups(index, 6, 16)
    n = 4 + int(plan.data[1])
    assert torch.equal(plan.data[:n], fresh.data[:n])
    at, tiles = 4 + 200, int(plan.data[0])
    assert torch.equal(plan.data[at:at + 4 * tiles], fresh.data[at:at + 4 * tiles])


# ---------------------------------------------------------------------------------------------------------------- updates
def make(M, n, K, R, widths, dtype, gap=8, out="f32", seed=0, rank=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device="cuda")
    dt, rank = DT[dtype], R if rank is None else rank
    a = torch.zeros((n, len(widths), R, K), dtype=dt, device="cuda")
    a[:, :, :rank] = (normal(n, len(widths), rank, K) / K ** 0.5).to(dt)
    b = torch.zeros((n, sum(widths), R), dtype=dt, device="cuda")
    b[:, :, :rank] = normal(n, sum(widths), rank).to(dt)
    columns, at = [], gap
    for w in widths:
        columns.append((at, w))
        at += w + gap
    y = normal(M, at).to(torch.float32 if out == "f32" else dt)
    return normal(M, K).to(dt), a, b, 0.5 + normal(n).abs(), tuple(columns), y


def check(index, x, a, b, scales, columns, y, tile):
    n, T, R, K = a.shape
    M = x.shape[0]
    dt, before = x.dtype, y.double().clone()
    want, slack = before.clone(), torch.zeros_like(before)
    index = index.cuda()
    for i in sorted({v for v in index.tolist() if 0 <= v < n}):
        rows = (index == i).nonzero()[:, 0]
        at = 0
        for t, (c, w) in enumerate(columns):
            A, B, X = a[i, t].double(), b[i, at:at + w].double(), x[rows].double()
            z, s = X @ A.t(), float(scales[i])
            want[rows, c:c + w] += s * (z @ B.t())
            # z: every product of 16 adds at most a unit of 2^-23 of what has been summed in absolute values, and so do the joins of the parts; the second
            # product keeps z to 2^-21 of its row's largest, and adds R / 16 * 3 sums
            ez = (K / 16 + 32) * 2.0 ** -23 * (X.abs() @ A.abs().t()) + 2.0 ** -21 * z.abs().amax(-1, keepdim=True)
            slack[rows, c:c + w] += s * (ez @ B.abs().t() + (3 * R / 16 + 4) * 2.0 ** -23 * (z.abs() @ B.abs().t()))
            at += w
    slack += want.abs() * (torch.finfo(y.dtype).eps / 2 * 1.001) + torch.where(want != before, torch.finfo(y.dtype).tiny, 0.0)
    plan = ops.row_groups(index, n, tile)
    assert ops.lora_rows(x, plan, a, b, scales, columns, y) is y
    diff = (y.double() - want).abs()
    assert diff.le(slack).all(), (float(diff.max()), float((diff - slack).max()))
    idle = (index < 0) | (index >= n)
    assert torch.equal(y[idle].double(), before[idle])
    left = torch.ones(y.shape[1], dtype=torch.bool, device="cuda")
    for c, w in columns:
        left[c:c + w] = False
    assert torch.equal(y[:, left].double(), before[:, left])


@pytest.mark.parametrize("dtype,out", [("f16", "f32"), ("f16", "16"), ("bf16", "f32"), ("bf16", "16")])
@pytest.mark.parametrize("tile", [16, 128])
@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 63, 64, 65, 130, 300])
def test_rows(M, tile, dtype, out):
    for n in (1, 3, 40):
        check(index_of(M, n, seed=M), *make(M, n, 256, 16, (64, 24), dtype, out=out, seed=M + n), tile)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tile", [16, 128])
@pytest.mark.parametrize("K", [8, 16, 24, 32, 40, 64, 136, 248, 520, 4096, 8200])
def test_inner_sizes(K, tile, dtype):
    check(index_of(37, 3), *make(37, 3, K, 16, (128, 8, 40), dtype, seed=K), tile)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("tile", [16, 128])
@pytest.mark.parametrize("R,targets", [(16, 1), (16, 2), (16, 3), (16, 4), (32, 1), (32, 2), (32, 4), (48, 1), (48, 2), (48, 3), (64, 1), (64, 2), (64, 3), (64, 4)])
def test_ranks_and_targets(R, targets, tile, dtype):
    check(index_of(50, 2), *make(50, 2, 320, R, (72, 8, 16, 200)[:targets], dtype, out="16" if R % 32 else "f32", seed=R), tile)


@pytest.mark.parametrize("rank", [1, 3, 8, 17, 31])
def test_ranks_that_are_filled_up(rank):
    check(index_of(20, 4), *make(20, 4, 512, 32, (512, 128), "bf16", rank=rank), 16)


@pytest.mark.parametrize("width", [8, 16, 24, 56, 1000, 4096])
def test_widths(width):
    for tile in (16, 128):
        check(index_of(33, 3), *make(33, 3, 128, 16, (width,), "f16", out="16"), tile)


def test_sizes_of_a_model():
    check(index_of(64, 64, none=False), *make(64, 64, 4096, 16, (4096, 1024), "f16", gap=1024), 16)
    check(torch.arange(64, dtype=torch.int32), *make(64, 64, 4096, 16, (4096, 1024), "f16", gap=1024), 16)
    check(torch.arange(2100, dtype=torch.int32) // 300 - 1, *make(2100, 6, 5120, 64, (5120, 1024), "bf16", gap=1024, out="16"), ops.lora_tile(2100, 6))
    check(torch.arange(300, dtype=torch.int32), *make(300, 1000, 128, 16, (128,), "bf16"), 16)      # more adapters than rows


def test_slices_of_wider_tensors():
    x, a, b, s, columns, y = make(21, 3, 256, 16, (64, 32), "f16")
    wide, tall = torch.randn((21, 300), device="cuda").half(), torch.randn((21, 400), device="cuda")
    with pytest.raises(RuntimeError, match="16-byte aligned"):      # rows of 300
        ops.lora_rows(wide[:, 8:264], ops.row_groups(index_of(21, 3).cuda(), 3, 16), a, b, s, columns, tall[:, 4:204])
    wide = torch.randn((21, 304), device="cuda").half()
    check(index_of(21, 3), wide[:, 8:264], a, b, s, columns, tall[:, 4:204], 16)
    check(index_of(1, 3), wide[3:4, 16:272], a, b, s, columns, tall[:1, :y.shape[1]], 16)


@pytest.mark.parametrize("tile", [16, 128])
def test_rows_farther_apart_than_32_bits_reach(tile):
    x, a, b, s, columns, y = make(3, 2, 128, 16, (64, 32), "bf16", out="16")
    far = lambda n: torch.zeros((2 ** 31 + 4096,), dtype=torch.bfloat16, device="cuda").as_strided((3, n), (2 ** 30 + 64, 1))
    wide_x, wide_y = far(128), far(y.shape[1])
    wide_x.copy_(x), wide_y.copy_(y)
    check(torch.tensor([1, 0, 1], dtype=torch.int32), wide_x, a, b, s, columns, wide_y, tile)


def test_many_rows():
    check(index_of(5000, 30), *make(5000, 30, 256, 32, (128, 64), "f16", out="16"), 128)
    check(index_of(5000, 30), *make(5000, 30, 256, 32, (128, 64), "bf16"), 128)
    check(index_of(5000, 1024), *make(5000, 1024, 128, 16, (64,), "f16"), 16)


def test_no_row_has_an_adapter():
    x, a, b, s, columns, y = make(40, 3, 256, 16, (64,), "f16")
    for v in (-1, 3, 2 ** 31 - 1, -2 ** 31):
        check(torch.full((40,), v, dtype=torch.int32), x, a, b, s, columns, y, 16)
    ops.lora_rows(x[:0], ops.row_groups(torch.empty((0,), dtype=torch.int32, device="cuda"), 3, 16), a, b, s, columns, y[:0])


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 1.0, 300.0])
def test_small_and_large_inner_values(scale):
    """z beyond f16's range, or below its smallest numbers, keeps its bits."""
    x, a, b, s, columns, y = make(20, 2, 512, 16, (64,), "f16")
    x = (x.float() * scale).half()
    a *= 20.0 if scale > 1 else 1.0
    y.zero_()
    check(index_of(20, 2, none=False), x, a, b, s * (1.0 / scale if scale < 1 else 1.0), columns, y, 16)


def test_what_is_not_a_number_stays_in_its_row():
    x, a, b, s, columns, y = make(24, 2, 256, 16, (64, 8), "bf16")
    index = index_of(24, 2, none=False).cuda()
    plan = ops.row_groups(index, 2, 16)
    clean = ops.lora_rows(x, plan, a, b, s, columns, y.clone())
    x[5, 7] = float("nan")
    got = ops.lora_rows(x, plan, a, b, s, columns, y.clone())
    others = torch.arange(24, device="cuda") != 5
    assert torch.equal(got[others], clean[others])
    assert all(got[5, c:c + w].isnan().all() for c, w in columns)


def test_same_bits_every_time():
    """Nor does a row's update depend on the rows beside it (as long as the calls split K alike)."""
    x, a, b, s, columns, y = make(100, 5, 1024, 32, (256, 64), "bf16")
    index = index_of(100, 5).cuda()
    first = ops.lora_rows(x, ops.row_groups(index, 5, 16), a, b, s, columns, y.clone())
    for _ in range(3):
        assert torch.equal(first, ops.lora_rows(x, ops.row_groups(index, 5, 16), a, b, s, columns, y.clone()))
    for m in (0, 50, 99):
        alone = ops.lora_rows(x[m:m + 1], ops.row_groups(index[m:m + 1], 5, 16), a, b, s, columns, y[m:m + 1].clone())
        assert torch.equal(alone[0], first[m])


def test_graph_and_streams():
    x, a, b, s, columns, y = make(30, 4, 512, 16, (128, 64), "f16")
    index = index_of(30, 4).cuda()
    plan, base, out = ops.row_groups(index, 4, 16), y.clone(), y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out.copy_(base)
        ops.row_groups(index, 4, 16, out=plan)
        ops.lora_rows(x, plan, a, b, s, columns, out)
    side = torch.cuda.Stream()
    for seed in (1, 2):
        index.copy_(index_of(30, 4, seed=seed))
        g.replay()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = ops.lora_rows(x, ops.row_groups(index, 4, 16), a, b, s, columns, base.clone())
        torch.cuda.synchronize()
        assert torch.equal(out, other) and not torch.equal(out, base)


def test_refusals():
    x, a, b, s, columns, y = make(8, 2, 64, 16, (32, 8), "f16")
    index = index_of(8, 2).cuda()
    plan = ops.row_groups(index, 2, 16)
    keep = y.clone()
    for bad in (dict(x=x.float()), dict(x=x[:, ::2]), dict(x=x[:7]), dict(x=x[:, 1:]), dict(a=a.bfloat16()), dict(a=a[:, :, :8]), dict(a=a[:1]), dict(a=torch.zeros((2, 2, 80, 64), device="cuda").half(), b=torch.zeros((2, 40, 80), device="cuda").half()),
                dict(b=b[:, :39]), dict(b=b.float()), dict(scales=s.half()), dict(scales=s[:1]), dict(y=y.bfloat16()), dict(y=y[:7]), dict(y=y[:, :40]),
                dict(columns=columns[:1]), dict(columns=((0, 32), (30, 8))), dict(columns=((0, 36), (40, 4))), dict(columns=((2, 32), (40, 8))),
                dict(columns=((0, 32), (60, 8))), dict(columns=((-8, 32), (40, 8))), dict(x=x.cpu()), dict(plan=plan._replace(rows=9)),
                dict(plan=plan._replace(groups=3)), dict(plan=plan._replace(tile=8)), dict(plan=plan._replace(data=plan.data[:8])),
                dict(plan=ops.row_groups(index, 2, 32))):
        kw = dict(dict(x=x, plan=plan, a=a, b=b, scales=s, columns=columns, y=y), **bad)
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.lora_rows(**kw)
    assert torch.equal(y, keep)
    for bad in ((index.long(), 2, 16), (index.cpu(), 2, 16), (index, 0, 16), (index, 1025, 16), (index, 2, 0), (index[::2], 2, 16)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.row_groups(*bad)
    with pytest.raises(ValueError):
        ops.row_groups(index, 2, 16, out=ops.row_groups(index, 3, 16))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R,targets", [(32, 1), (32, 2), (32, 3), (64, 1), (64, 2), (64, 3)])
def test_prompt_tiles_of_higher_ranks(R, targets, dtype):
    """Blocks of columns that end inside a target, whole tiles and parts of one, at each size of the inner product's room."""
    columns = (264, 8, 1000)[:targets]
    check(index_of(300, 2), *make(300, 2, 4096 if R == 64 else 136, R, columns, dtype, out="16", seed=R + targets), 128)


@pytest.mark.parametrize("scale", [1e-3, 1.0, 300.0])
def test_prompt_tiles_of_small_and_large_inner_values(scale):
    x, a, b, s, columns, y = make(200, 2, 512, 32, (64, 136), "f16", out="16")
    x, a = (x.float() * scale).half(), a * (20.0 if scale > 1 else 1.0)
    y.zero_()
    check(index_of(200, 2, none=False), x, a, b / 64 if scale > 1 else b, s / max(scale, 1.0), columns, y, 128)


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("targets", [2, 3])
def test_prompt_tiles_keep_what_is_not_a_number_in_its_row(value, targets):
    x, a, b, s, columns, y = make(300, 2, 1024, 32, (264, 8, 72)[:targets], "bf16", out="16")
    plan = ops.row_groups(index_of(300, 2, none=False).cuda(), 2, 128)
    clean = ops.lora_rows(x, plan, a, b, s, columns, y.clone())
    x[77, 7] = value
    got = ops.lora_rows(x, plan, a, b, s, columns, y.clone())
    others = torch.arange(300, device="cuda") != 77
    assert torch.equal(got[others], clean[others])
    assert not any(got[77, c:c + w].isfinite().any() for c, w in columns)


@pytest.mark.parametrize("targets", [1, 3])
def test_prompt_tiles_in_graphs_on_two_streams(targets):
    """Two calls at once, rewritten plans, the same bits every time."""
    x, a, b, s, columns, y = make(1700, 4, 2048, 64, (512, 256, 64)[:targets], "f16", out="16")
    index = index_of(1700, 4).cuda()
    plan, base, out = ops.row_groups(index, 4, 128), y.clone(), y.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out.copy_(base)
        ops.row_groups(index, 4, 128, out=plan)
        ops.lora_rows(x, plan, a, b, s, columns, out)
    side = torch.cuda.Stream()
    for seed in (1, 2):
        index.copy_(index_of(1700, 4, seed=seed))
        other, plans = base.clone(), ops.row_groups(index, 4, 128)
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            ops.lora_rows(x, plans, a, b, s, columns, other)
        torch.cuda.synchronize()
        assert torch.equal(out, other) and not torch.equal(out, base)
        ops.check_waits()


@pytest.mark.parametrize("shift,gap", [(4, 0), (0, 4), (8, 0)])
def test_prompt_tiles_of_y_at_odd_places(shift, gap):
    """y whose rows or columns are no multiple of 16 bytes."""
    x, a, b, s, columns, y = make(260, 3, 256, 16, (64, 32), "bf16", gap=gap, out="16")
    wide = torch.randn((260, y.shape[1] + 16), device="cuda").bfloat16()
    check(index_of(260, 3), x, a, b, s, columns, wide[:, shift:shift + y.shape[1]], 128)


@pytest.mark.parametrize("M,n", [(900, 2), (2100, 6), (5000, 30), (9000, 40)])
@pytest.mark.parametrize("R,targets", [(16, 2), (64, 3)])
def test_prompt_tiles_of_clusters_of_every_size(M, n, R, targets):
    check(index_of(M, n, seed=M), *make(M, n, 520, R, (136, 264, 8)[:targets], "f16", out="16", seed=n), 128)


@pytest.mark.parametrize("out", ["f32", "16"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("R", [16, 64])
@pytest.mark.parametrize("tile,M", [(16, 40), (128, 200)])
def test_a_small_z_beside_a_large_one_keeps_its_bits(tile, M, R, dtype, out):
    """z is one exact product here, from 60 in the first rank, which b leaves out, down to 6e-6 in the others.  Two f16 numbers are off by 2^-22 of z or 2^-39 of
    the row's largest, three bf16 ones by 2^-24, two (where y is bf16) by 2^-16; the second product adds 3 R / 16 sums in fp32, and y is rounded once."""
    g = torch.Generator(device="cuda").manual_seed(R + M)
    rand = lambda *s: torch.rand(s, generator=g, device="cuda")
    K, N, dt = 64, 128, DT[dtype]
    x = (60 * 10 ** (-7 * rand(M, K))).to(dt)
    x[:, 0] = 60
    a = torch.zeros((2, 1, R, K), dtype=dt, device="cuda")
    a[:, 0, torch.arange(R), torch.arange(R)] = (1 + rand(2, R)).to(dt)
    for keep in (1, R // 2, R - 1):                                  # ranks that b looks at: small ones by themselves
        b = (torch.randn((2, N, R), generator=g, device="cuda")).to(dt)
        b[:, :, :R - keep] = 0
        index = (torch.arange(M, dtype=torch.int32) % 2).cuda()
        scales, columns = torch.ones(2, device="cuda"), ((0, N),)
        y = torch.zeros((M, N), dtype=torch.float32 if out == "f32" else dt, device="cuda")
        ops.lora_rows(x, ops.row_groups(index, 2, tile), a, b, scales, columns, y)
        z = x.double()[:, :R] * a[:, 0].double().diagonal(dim1=1, dim2=2)[index.long()]
        B = b.double()[index.long()]
        want = torch.einsum("mr,mnr->mn", z, B)
        part = 2.0 ** -22 * z.abs() + 2.0 ** -39 * z.abs().amax(-1, keepdim=True) if dtype == "f16" else 2.0 ** (-24 if out == "f32" else -16) * z.abs()
        slack = torch.einsum("mr,mnr->mn", part + (3 * R / 16 + 4) * 2.0 ** -23 * z.abs(), B.abs())
        eps = torch.finfo(y.dtype)
        slack += want.abs() * eps.eps / 2 + (0.0 if out == "f32" else eps.tiny * eps.eps / 2)      # (half of a smallest number)
        diff = (y.double() - want).abs()
        assert diff.le(slack).all(), (keep, float((diff / want.abs().clamp(min=1e-30)).max()))

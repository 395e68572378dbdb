"""Refusals of the operators of scoring, adapters and shared prompts that need no device."""
import pytest
import torch

from mlx_parallm_b200 import _lib, ops


def test_token_logprobs_refuses_before_it_launches():
    f = _lib.lib().b200p_token_logprobs
    ok = dict(logits=256, tokens=256, logprob=256, entropy=256, ids=256, alts=256, M=4, V=100, ld=100, top=2, T=1.0, dtype=_lib.F32)

    def call(**kw):
        a = dict(ok, **kw)
        return f(a["logits"], a["tokens"], a["logprob"], a["entropy"], a["ids"], a["alts"], a["M"], a["V"], a["ld"], a["top"], a["T"], a["dtype"], 0)

    for bad in (dict(M=-1), dict(M=1 << 27), dict(V=0), dict(V=1 << 30, ld=1 << 30), dict(ld=99), dict(top=-1), dict(top=33), dict(top=5, V=4), dict(T=0.0),
                dict(T=-1.0), dict(T=float("nan")), dict(T=float("inf")), dict(dtype=3), dict(dtype=-1), dict(logits=0), dict(tokens=0), dict(ids=0),
                dict(alts=0)):
        assert call(**bad) == -1, bad
    assert call(logits=258) == -2 and call(logits=257, dtype=_lib.BF16) == -2
    assert call(M=0) == 0 and call(M=0, logits=0) == 0              # nothing to do


def test_no_cpu_fallback():
    with pytest.raises(_lib.B200PError):
        ops.token_logprobs(torch.zeros((2, 8)), torch.zeros((2,), dtype=torch.int32))


def test_row_groups_refuses_before_it_launches():
    L = _lib.lib()
    assert L.b200p_row_groups_ints(10, 3, 16) == 4 + 12 + 4 * 3 and L.b200p_row_groups_ints(100, 3, 16) == 4 + 100 + 4 * (6 + 3)
    for bad in ((-1, 3, 16), ((1 << 20) + 1, 3, 16), (10, 0, 16), (10, 1025, 16), (10, 3, 0)):
        assert L.b200p_row_groups_ints(*bad) == 0
    ok = dict(index=256, plan=256, M=10, groups=3, tile=16, ints=1000)

    def call(**kw):
        a = dict(ok, **kw)
        return L.b200p_row_groups(a["index"], a["plan"], a["M"], a["groups"], a["tile"], a["ints"], 0)

    for bad in (dict(M=-1), dict(M=(1 << 20) + 1), dict(groups=0), dict(groups=1025), dict(tile=0), dict(plan=0), dict(index=0), dict(ints=27)):
        assert call(**bad) == -1, bad
    assert call(plan=260) == -2 and call(index=258) == -2


def test_lora_rows_refuses_before_it_launches():
    import ctypes as C
    f = _lib.lib().b200p_lora_rows
    ok = dict(x=256, plan=256, a=256, b=256, scales=256, y=256, columns=(0, 64, 128, 8), M=4, adapters=2, tile=16, targets=2, R=16, K=64, ldx=64, ldy=136,
              dtype=_lib.F16, f32=1)

    def call(**kw):
        a = dict(ok, **kw)
        held = (C.c_int32 * len(a["columns"]))(*a["columns"])
        return f(a["x"], a["plan"], a["a"], a["b"], a["scales"], a["y"], C.addressof(held), a["M"], a["adapters"], a["tile"], a["targets"], a["R"], a["K"],
                 a["ldx"], a["ldy"], a["dtype"], a["f32"], 0)

    for bad in (dict(dtype=_lib.F32), dict(dtype=7), dict(M=-1), dict(M=(1 << 20) + 1), dict(adapters=0), dict(adapters=1025), dict(tile=32), dict(targets=0),
                dict(targets=5, columns=(0, 8) * 5), dict(R=0), dict(R=24), dict(R=80), dict(K=0), dict(K=12), dict(ldx=56), dict(columns=(0, 64, 128, 16)),
                dict(columns=(0, 64, 60, 8)), dict(columns=(0, 0, 64, 8)), dict(columns=(-8, 64, 64, 8)), dict(columns=(0, 60, 64, 8)), dict(x=0), dict(plan=0),
                dict(a=0), dict(b=0), dict(scales=0), dict(y=0)):
        assert call(**bad) == -1, bad
    for bad in (dict(columns=(2, 64, 128, 8)), dict(x=264), dict(a=264), dict(b=264), dict(plan=264), dict(ldx=68), dict(y=264), dict(ldy=137)):
        assert call(**bad) == -2, bad
    assert call(M=0) == 0


def test_paged_attn_shared_refuses_before_it_launches():
    L = _lib.lib()
    assert [L.b200p_paged_attn_shared_tile(*x) for x in ((32, 8), (40, 8), (8, 8), (64, 1), (129, 1), (300, 1), (7, 2), (4, 0))] == [64, 51, 256, 4, 1, 1, 0, 0]
    assert L.b200p_paged_attn_shared_set_path(3) == -1 and L.b200p_paged_attn_shared_set_path(-1) == -1 and L.b200p_paged_attn_shared_set_path(0) == 0
    size = L.b200p_paged_attn_shared_workspace_bytes
    assert size(4, 8, 2, 64, 1) > 0 and [size(*x) for x in ((0, 8, 2, 64, 1), (4, 7, 2, 64, 1), (4, 8, 2, 64, 0), (4, 8, 2, 64, 1025))] == [0] * 4
    ok = dict(q=256, k=256, v=256, table=256, row=256, slot=256, out=256, index=256, prefix=256, plan=256, M=4, H=8, G=2, D=64, groups=1, tile=64, P=9, page=16,
              rows=4, width=8, dtype=_lib.F16, flags=0, ws=256, bytes=1 << 30)

    def call(**kw):
        a = dict(ok, **kw)
        return L.b200p_paged_attn_shared(a["q"], a["k"], a["v"], a["table"], a["row"], a["slot"], a["out"], a["index"], a["prefix"], a["plan"], a["M"], a["H"],
                                         a["G"], a["D"], a["groups"], a["tile"], a["P"], a["page"], a["rows"], a["width"], 1.0, a["dtype"], a["flags"], a["ws"],
                                         a["bytes"], 0)

    for bad in (dict(q=0), dict(k=0), dict(table=0), dict(row=0), dict(slot=0), dict(out=0), dict(index=0), dict(prefix=0), dict(plan=0), dict(M=-1), dict(M=65536),
                dict(H=7), dict(G=0), dict(D=12), dict(D=264), dict(groups=0), dict(groups=1025), dict(tile=16), dict(P=0), dict(page=24), dict(page=8192),
                dict(rows=0), dict(width=0), dict(width=1 << 27), dict(dtype=9), dict(flags=2), dict(ws=0), dict(ws=128), dict(bytes=1000),
                dict(dtype=_lib.F32, bytes=1000)):
        assert call(**bad) == -1, bad
    for bad in (dict(q=264), dict(out=264), dict(k=264), dict(plan=264)):
        assert call(**bad) == -2, bad


def test_pages_of_rows_that_share_a_prompt():
    """Counting of shared pages, on the CPU: whole pages belong to all rows of a group, the last one's tokens are copied, the last row gives pages back."""
    from mlx_parallm_b200.models.paged import PageBook, PagedLayer, PagesExhausted
    book = PageBook(5, 64, "cpu", page=16, pages=12)
    layer = PagedLayer(book, 4, 2, 8)
    layer.kpages, layer.vpages = torch.randn((12, 2, 16, 8)), torch.randn((12, 2, 16, 8))

    def read(n, tokens):
        side = PageBook(n, tokens, "cpu", page=16, pages=12, of=book)
        PagedLayer(side, 4, 2, 8)
        side.room_for([tokens] * n)
        return side

    side = read(1, 40)
    assert len(book.free) == 9 and side.free is book.free
    held = list(side.owned[0])
    book.adopt(side, [[0, 2, 3]], 40)
    side.shrink([0])
    assert layer._offsets == [40, 0, 40, 40, 0] and book.lengths.tolist() == [40, 0, 40, 40, 0]
    assert [o[:2] for o in (book.owned[0], book.owned[2], book.owned[3])] == [held[:2]] * 3 and book.owned[0][2] == held[2]
    assert len({o[2] for o in (book.owned[0], book.owned[2], book.owned[3])}) == 3 and len(book.free) == 7
    for r in (2, 3):
        assert book.table[r].tolist() == book.owned[r] + [-1]
        assert torch.equal(layer.kpages[book.owned[r][2]], layer.kpages[held[2]]) and torch.equal(layer.vpages[book.owned[r][2]], layer.vpages[held[2]])
    assert book.held == {p: 3 for p in held[:2]} and book.groups == [[0, 2, 3]] and book.prefixes == [32] and not book.by_groups
    side = read(1, 32)                                              # no rest: nothing is copied
    book.adopt(side, [[1, 4]], 32)
    assert book.owned[1] == book.owned[4] and len(book.free) == 5
    layer.release_rows_host([2])
    assert book.groups[0] == [0, 3] and len(book.free) == 6 and book.held[held[0]] == 2
    book.room_for([50, 0, 0, 0, 0])
    assert len(book.free) == 5
    layer.release_rows_host([0])
    assert book.held.keys() == set(book.owned[1]) and len(book.free) == 7
    layer.release_rows_host([3])
    assert len(book.free) == 10
    layer.reset()
    assert sorted(book.free) == list(range(12)) and not book.held and book.groups == [] and (book.table == -1).all()
    side = read(2, 40)                                              # 6 pages; 7 rows more want 5 for their rests, and 6 are free
    book.free[:] = book.free[:2]
    with pytest.raises(PagesExhausted):
        book.adopt(side, [[0, 1, 2], [3, 4]], 40)
    assert all(not o for o in book.owned) and book.groups == [] and len(book.free) == 2


def test_workspace_of_shared_slots_goes_by_query_rows_not_by_groups():
    """Parts are M H query rows and 256 more per SM at most, of outputs, maximum and sum in fp32, beside one row each of the own slots."""
    size = _lib.lib().b200p_paged_attn_shared_workspace_bytes
    for M, H, G, D in ((1024, 32, 8, 128), (1024, 32, 32, 96), (2048, 32, 32, 128), (64, 32, 8, 128), (3, 9, 1, 256)):
        base = ops.paged_attn_workspace_bytes(M, H, D, 0, G)
        assert size(M, H, G, D, 1) == size(M, H, G, D, 1024)
        assert size(M, H, G, D, 7) <= base + (2 * M * H + 256 * 160) * (D + 8) * 4 + 16 * M + 2048


def _state(book, layer):
    return (list(layer._offsets), [list(o) for o in book.owned], dict(book.held), [list(g) for g in book.groups], list(book.prefixes), list(book.free),
            book.table.tolist(), book.lengths.tolist(), book.positions.tolist(), book.by_groups)


@pytest.mark.parametrize("fails", ["copy", "group"])
def test_a_shared_prompt_that_finds_no_memory_leaves_the_book_as_it_was(fails, monkeypatch):
    """What fails on the device (the copies of last pages; what a step by groups needs, here refused without a device) fails before the book changes."""
    from mlx_parallm_b200.models import paged
    book = paged.PageBook(4, 64, "cpu", page=16, pages=14)
    layers = [paged.PagedLayer(book, 4, 2, 8) for _ in range(2)]
    for layer in layers:
        layer.kpages, layer.vpages = torch.randn((14, 2, 16, 8)), torch.randn((14, 2, 16, 8))
    side = paged.PageBook(1, 40, "cpu", page=16, pages=14, of=book)
    paged.PagedLayer(side, 4, 2, 8)
    side.room_for([40])
    if fails == "group":
        monkeypatch.setattr(paged, "SHARED_BYTES", 0)
    else:
        layers[1].vpages = torch.randn((1, 2, 16, 8))               # no page to copy
    before, theirs = _state(book, layers[0]), list(side.owned[0])
    with pytest.raises(_lib.B200PError if fails == "group" else IndexError):
        book.adopt(side, [[0, 1, 3]], 40)
    assert _state(book, layers[0]) == before and side.owned[0] == theirs
    side.shrink([0])
    assert sorted(book.free) == list(range(14))


def test_pages_that_empty_rows_have_go_back_when_they_share_a_prompt():
    """A step that fails behind room_for leaves its rows pages; adopted rows give them back, and no page is lost or has two places."""
    from mlx_parallm_b200.models.paged import PageBook, PagedLayer
    book = PageBook(3, 64, "cpu", page=16, pages=10)
    layer = PagedLayer(book, 4, 2, 8)
    layer.kpages, layer.vpages = torch.zeros((10, 2, 16, 8)), torch.zeros((10, 2, 16, 8))
    book.room_for([50, 10, 20])                                     # 4, 1 and 2 pages, and no token is appended
    side = PageBook(1, 40, "cpu", page=16, pages=10, of=book)
    PagedLayer(side, 4, 2, 8)
    side.room_for([40])
    book.adopt(side, [[0, 2]], 40)                                  # (the copy of the last page comes out of what rows 0 and 2 gave back)
    assert len(book.owned[0]) == len(book.owned[2]) == 3 and len(book.owned[1]) == 1
    used = set(book.owned[0]) | set(book.owned[1]) | set(book.owned[2])
    assert len(used) == 5 and used.isdisjoint(book.free) and len(book.free) == len(set(book.free)) == 5
    for r in range(3):
        assert book.table[r].tolist() == book.owned[r] + [-1] * (4 - len(book.owned[r]))
    layer.reset()
    assert sorted(book.free) == list(range(10)) and (book.table == -1).all()


@pytest.mark.parametrize("lengths", [[5, 4], [4, -1], [4], [4, 4, 4]])
def test_packed_prompts_that_are_no_counts_are_refused(lengths):
    """Before anything is read: a length above L would name the last ids of another row."""
    from mlx_parallm_b200.models._sequence import SequenceModel
    ids = torch.zeros((2, 4), dtype=torch.int64)
    for call in (SequenceModel.score, SequenceModel.__call__):
        with pytest.raises(ValueError, match="prompt_lengths"):
            call(object(), ids, prompt_lengths=lengths)


@pytest.mark.parametrize("want", [[[2], []], [[-1], []], [[0], [0]], [[0]]])
def test_wanted_positions_outside_their_entries_are_refused(want):
    from types import SimpleNamespace
    from mlx_parallm_b200.models._sequence import SequenceModel
    for sink in (None, lambda *a: None):
        with pytest.raises(ValueError, match="wanted position"):
            SequenceModel._forward_ragged_locked(SimpleNamespace(device="cpu"), [[1, 2], []], [SimpleNamespace(batch_size=2)], None, want, sink)


def test_token_logprobs_refuses_temperatures_at_which_masked_logits_would_weigh_something():
    f = _lib.lib().b200p_token_logprobs
    for T in (1.2e27, 1e28, 1e30, 3e38, 9e-31):
        assert f(256, 256, 256, 256, 256, 256, 4, 100, 100, 2, T, _lib.F32, 0) == -1, T

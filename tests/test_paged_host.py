"""Argument checks of the paged-cache entry points (no device: every refusal comes before a launch), the tile arithmetic of the window, and the
oracle of the GPU tests against itself."""
import math
import threading

import pytest
import torch

import paged_oracle as po
from mlx_parallm_b200 import _lib

OK = 1 << 20           # an aligned address that a refused call never touches
ARG, ALIGN = -1, -2


def L():
    return _lib.lib()


def append(**kw):
    a = dict(qkv=OK, ldq=12 * 64, q=OK, k=OK, v=OK, mass=0, table=OK, row=OK, slot=OK, pos=OK, qw=0, kw=0, rates=OK, n=32, pairs=0, eps=1e-6, M=2, H=8,
             G=2, D=64, P=9, page=16, rows=2, width=4, dtype=_lib.BF16, f32=0)
    a.update(kw)
    return L().b200p_paged_append(a["qkv"], a["ldq"], a["q"], a["k"], a["v"], a["mass"], a["table"], a["row"], a["slot"], a["pos"], a["qw"], a["kw"],
                                  a["rates"], a["n"], a["pairs"], a["eps"], a["M"], a["H"], a["G"], a["D"], a["P"], a["page"], a["rows"], a["width"],
                                  a["dtype"], a["f32"], 0)


def attn(**kw):
    a = dict(q=OK, k=OK, v=OK, mass=0, table=OK, row=OK, slot=OK, out=OK, M=2, H=8, G=2, D=64, P=9, page=16, rows=2, width=4, scale=1.0, first=0, window=0,
             dtype=_lib.BF16, flags=0, ws=OK, bytes=1 << 30)
    a.update(kw)
    return L().b200p_paged_attn(a["q"], a["k"], a["v"], a["mass"], a["table"], a["row"], a["slot"], a["out"], a["M"], a["H"], a["G"], a["D"], a["P"],
                                a["page"], a["rows"], a["width"], a["scale"], a["first"], a["window"], a["dtype"], a["flags"], a["ws"], a["bytes"], 0)


def select(**kw):
    a = dict(mass=OK, table=OK, lengths=OK, kept=OK, P=9, G=2, page=16, rows=2, width=4, keep=20, first=4, recent=8)
    a.update(kw)
    return L().b200p_paged_select(*[a[x] for x in ("mass", "table", "lengths", "kept", "P", "G", "page", "rows", "width", "keep", "first", "recent")], 0)


def compact(**kw):
    a = dict(k=OK, v=OK, mass=0, table=OK, lengths=OK, kept=OK, P=9, G=2, D=64, page=16, rows=2, width=4, keep=20, dtype=_lib.F16)
    a.update(kw)
    return L().b200p_paged_compact(*[a[x] for x in ("k", "v", "mass", "table", "lengths", "kept", "P", "G", "D", "page", "rows", "width", "keep", "dtype")], 0)


def gather(**kw):
    a = dict(k=OK, v=OK, table=OK, row_of=OK, lengths=OK, kc=OK, vc=OK, extra=0, count=2, G=2, D=64, P=9, page=16, rows=2, width=4, cap=64, dtype=_lib.F32)
    a.update(kw)
    return L().b200p_paged_gather(*[a[x] for x in ("k", "v", "table", "row_of", "lengths", "kc", "vc", "extra", "count", "G", "D", "P", "page", "rows", "width",
                                                   "cap", "dtype")], 0)


PAGES = [dict(page=8), dict(page=24), dict(page=0), dict(page=8192), dict(P=0), dict(P=1 << 31), dict(rows=0), dict(width=0), dict(width=1 << 27), dict(G=0),
         dict(table=0)]


@pytest.mark.parametrize("call", [append, attn, select, compact, gather])
@pytest.mark.parametrize("bad", PAGES, ids=str)
def test_pages_that_are_refused(call, bad):
    assert call(**bad) == ARG and _lib.last_error()


@pytest.mark.parametrize("call,bad,rc", [
    (append, dict(D=60), ARG), (append, dict(D=264), ARG), (append, dict(dtype=3), ARG), (append, dict(H=7), ARG), (append, dict(qkv=0), ARG),
    (append, dict(q=0), ARG), (append, dict(row=0), ARG), (append, dict(slot=0), ARG), (append, dict(pos=0), ARG), (append, dict(rates=0), ARG),
    (append, dict(n=33), ARG), (append, dict(n=-1), ARG), (append, dict(pairs=2), ARG), (append, dict(ldq=12 * 64 - 1), ARG), (append, dict(M=-1), ARG),
    (append, dict(f32=1, dtype=_lib.F32), ARG), (append, dict(k=OK + 8), ALIGN), (append, dict(v=OK + 2), ALIGN),
    (attn, dict(D=60), ARG), (attn, dict(D=0), ARG), (attn, dict(D=512), ARG), (attn, dict(dtype=-1), ARG), (attn, dict(H=9), ARG), (attn, dict(H=0), ARG),
    (attn, dict(q=0), ARG), (attn, dict(out=0), ARG), (attn, dict(k=0), ARG), (attn, dict(row=0), ARG), (attn, dict(slot=0), ARG), (attn, dict(M=-1), ARG),
    (attn, dict(M=65536), ARG), (attn, dict(first=-1), ARG), (attn, dict(window=-1), ARG), (attn, dict(flags=2), ARG), (attn, dict(q=OK + 2), ALIGN),
    (attn, dict(out=OK + 2), ALIGN), (attn, dict(k=OK + 2), ALIGN), (attn, dict(mass=OK, ws=0), ARG), (attn, dict(mass=OK, bytes=100), ARG),
    (select, dict(mass=0), ARG), (select, dict(lengths=0), ARG), (select, dict(kept=0), ARG), (select, dict(keep=0), ARG), (select, dict(keep=(1 << 30) + 1), ARG), (select, dict(first=-1), ARG),
    (select, dict(recent=-1), ARG), (select, dict(first=13), ARG), (select, dict(first=(1 << 31) - 1, recent=(1 << 31) - 1), ARG), (select, dict(rows=65536), ARG),
    (compact, dict(k=0), ARG), (compact, dict(kept=0), ARG), (compact, dict(keep=0), ARG), (compact, dict(keep=(1 << 30) + 1), ARG), (compact, dict(dtype=7), ARG), (compact, dict(v=OK + 8), ALIGN),
    (gather, dict(row_of=0), ARG), (gather, dict(kc=0), ARG), (gather, dict(cap=0), ARG), (gather, dict(count=-1), ARG), (gather, dict(vc=OK + 4), ALIGN),
], ids=lambda x: getattr(x, "__name__", str(x)))
def test_arguments_that_are_refused(call, bad, rc):
    assert call(**bad) == rc and _lib.last_error()


def test_nothing_to_do_needs_no_device():
    assert append(M=0) == 0 and attn(M=0) == 0 and gather(count=0) == 0


def test_workspace_grows_with_the_weights_only():
    f = L().b200p_paged_attn_workspace_bytes
    assert f(0, 8, 64, 0) == 0 and f(2, 8, 64, 1000) >= 4 * 2 * 8 * 1000 + f(2, 8, 64, 0)


def test_ops_refuse_cpu_tensors():
    from mlx_parallm_b200 import ops
    k = torch.zeros((2, 1, 16, 8))
    i = torch.zeros(1, dtype=torch.int32)
    t = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(_lib.B200PError):
        ops.paged_attn(torch.zeros((1, 8)), k, k, t, i, i, torch.zeros((1, 8)), 1.0)
    with pytest.raises(_lib.B200PError):
        ops.paged_append(torch.zeros((1, 24)), torch.zeros((1, 8)), k, k, t, i, i, i, 1)
    with pytest.raises(_lib.B200PError):
        ops.paged_evict(k, k, torch.zeros((2, 1, 16)), t, i, torch.zeros((1, 1, 4), dtype=torch.int32))
    with pytest.raises(_lib.B200PError):
        ops.paged_gather(k, k, t, i, i, k, k)


# ---------------------------------------------------------------- the oracle
def test_oracle_of_the_attention_is_a_softmax_over_the_visible_slots():
    g = torch.Generator().manual_seed(1)
    k, v = torch.randn((3, 1, 16, 8), generator=g), torch.randn((3, 1, 16, 8), generator=g)
    mass = torch.zeros((3, 1, 16))
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    q = torch.randn((1, 16), generator=g)
    out, tol, new, off = po.attn(q, k, v, mass, table, torch.tensor([0]), torch.tensor([19]), 2, 0.5, 2, 5, 0.0)
    keys, values = torch.cat([k[2], k[0]], 1)[0].double(), torch.cat([v[2], v[0]], 1)[0].double()
    seen = [0, 1, 15, 16, 17, 18, 19]
    assert po.visible(20, 2, 5) == seen
    for h in range(2):
        s = q[0, 8 * h:8 * h + 8].double() @ keys[seen].T * 0.5
        assert torch.allclose(out[0, h], torch.softmax(s, -1) @ values[seen], atol=1e-12)
    assert abs(float(new.sum()) - 2) < 1e-12 and float(new[1].abs().max()) == 0.0
    assert float(new[2, 0, 2:15].abs().max()) == 0.0 and float(new[0, 0, 4:].abs().max()) == 0.0


def test_oracle_of_the_eviction():
    mass = torch.tensor([[[5.0, 1, 1, math.nan, 0, 3, 1, 1, 0, 9, 9, 9, 9, 9, 9, 9]]])
    kept = po.select(mass, torch.zeros((1, 1), dtype=torch.int32), torch.tensor([10]), 5, 1, 1)
    assert kept[0, 0].tolist() == [0, 1, 2, 5, 9]
    k = torch.arange(16.0).reshape(1, 1, 16, 1)
    new, _, m = po.compact(k, k, mass, torch.zeros((1, 1), dtype=torch.int32), torch.tensor([10]), kept)
    assert new.flatten()[:6].tolist() == [0, 1, 2, 5, 9, 5] and m.flatten()[:5].tolist() == [5, 1, 1, 3, 9]


def test_oracle_of_the_append_turns_pairs():
    k = torch.zeros((1, 1, 16, 8))
    qkv = torch.zeros((1, 24))
    qkv[0, 0], qkv[0, 8 + 1] = 1.0, 1.0
    i = torch.tensor([0])
    rates = torch.tensor([1.0, 0.5])
    for pairs in (0, 1):
        q, kk, _, _, _ = po.append(qkv, k, k, None, torch.zeros((1, 1), dtype=torch.int32), i, i + 3, i + 2, 1, rates, pairs, None, None, 0.0)
        assert abs(float(q[0, 0, 0]) - math.cos(2.0)) < 1e-12 and abs(float(q[0, 0, 2 if pairs == 0 else 1]) - math.sin(2.0)) < 1e-12
        assert abs(float(kk[0, 0, 3, 1]) - math.cos(1.0 if pairs == 0 else 2.0)) < 1e-12


# ---------------------------------------------------------------- the book of pages
def book(**kw):
    from mlx_parallm_b200.models.paged import PageBook
    return PageBook(**{**dict(rows=3, max_tokens=100, device="cpu", page=16), **kw})


def test_book_gives_and_takes_pages():
    b = book(pages=9)
    assert b.width == 7 and b.max_tokens == 112
    b.room_for([17, 0, 16])
    assert [len(o) for o in b.owned] == [2, 0, 1] and len(b.free) == 6
    assert b.table[0, :2].tolist() == b.owned[0] and int(b.table[0, 2]) == -1 and int(b.table[1].max()) == -1
    b.room_for([17, 1, 32])                     # nothing new for row 0, a page each for the others
    assert [len(o) for o in b.owned] == [2, 1, 2]
    ids = [p for o in b.owned for p in o] + b.free
    assert sorted(ids) == list(range(9))
    before = [list(o) for o in b.owned]
    with pytest.raises(RuntimeError, match="exhausted"):
        b.room_for([100, 1, 32])
    assert b.owned == before, "all or nothing"
    with pytest.raises(RuntimeError, match="does not fit"):
        b.room_for([113, 0, 0])
    b.shrink([16, 0, 17])
    assert [len(o) for o in b.owned] == [1, 0, 2] and int(b.table[1].max()) == -1 and int(b.table[0, 1]) == -1
    assert sorted([p for o in b.owned for p in o] + b.free) == list(range(9))


@pytest.mark.parametrize("bad", [dict(page=8), dict(page=40), dict(rows=0), dict(max_tokens=0), dict(pages=0), dict(window=-1), dict(first=-1),
                                 dict(keep=112), dict(keep=10, first=8, recent=3), dict(keep=10, recent=-1)], ids=str)
def test_book_refuses(bad):
    with pytest.raises(ValueError):
        book(**bad)


def test_layers_share_the_book_and_keep_positions_of_the_text():
    from mlx_parallm_b200.models.paged import PagedLayer
    b = book()
    layers = [PagedLayer(b, 4, 2, 64) for _ in range(2)]
    assert layers[0].counters()[0] is b.lengths and layers[0].capacity == 112 and layers[1]._lengths is b.lengths
    for c in layers:
        c._offsets = [5, 20, 0]
    b.evicted = [0, 7, 0]
    b.room_for([5, 20, 0])
    layers[0]._sync_lengths()
    assert b.lengths.tolist() == [5, 20, 0] and b.positions.tolist() == [5, 27, 0]
    layers[0].release_rows_host([1])
    layers[0]._sync_lengths()
    assert b.positions.tolist() == [5, 0, 0] and b.owned[1] == []
    with pytest.raises(ValueError):
        layers[0].reset(4)
    for c in layers:
        c.reset(3)
    assert len(b.free) == b.pages and b.lengths.tolist() == [0, 0, 0] == b.positions.tolist() and layers[1].offsets == [0, 0, 0]
    with pytest.raises(RuntimeError, match="adds up"):
        b.cut(10, 0, 0)


# ---------------------------------------------------------------- generation up to the last place
class _Step:
    """A decode step that counts up and has room for ``room`` steps."""
    greedy = True

    def __init__(self, room):
        self.tok, self.probs, self.room, self.n = torch.zeros(1, dtype=torch.int32), torch.ones(1), room, 0

    def run(self):
        from mlx_parallm_b200.models.paged import PagesExhausted
        if self.n == self.room:
            raise PagesExhausted("full")
        self.n += 1
        self.tok += 1


class _Model:
    device, kernel_units, _lock = "cpu", (), threading.Lock()

    def __call__(self, ids, cache, last_only):
        return torch.zeros((1, 1, 4))

    def greedy_tokens(self, logits, tok, probs):
        tok.fill_(10)


def test_every_token_that_was_made_is_given_before_a_full_cache_raises(monkeypatch):
    """The step for the next token is launched before a token is handed out: that it finds no room is said when that token is asked for.  Prompt + n
    places give n + 1 tokens, so zip(generate_step(...), range(n)), which looks for one more, ends with all of its n."""
    from mlx_parallm_b200 import utils
    from mlx_parallm_b200.models.paged import PagesExhausted
    monkeypatch.setattr(utils.ops, "check_waits", lambda: None)
    cache = [type("C", (), {"_lengths": 1})()]
    for room in (1, 2, 5):
        step = _Step(room)
        monkeypatch.setattr(utils, "_decode_step_for", lambda *a: step)
        got = [int(y) for (y, _), _ in zip(utils.generate_step([[1, 2]], _Model(), cache=cache), range(room))]
        assert got == list(range(10, 10 + room))
        step.n = 0
        run, got = utils.generate_step([[1, 2]], _Model(), cache=cache), []
        with pytest.raises(PagesExhausted):
            for y, _ in run:
                got.append(int(y))
        assert got == list(range(10, 11 + room))


def test_a_cache_without_room_says_so_in_one_kind_of_error():
    from mlx_parallm_b200.models.paged import PagedLayer, PagesExhausted
    b = book(pages=9)
    with pytest.raises(PagesExhausted, match="does not fit"):
        b.room_for([113, 0, 0])
    with pytest.raises(PagesExhausted, match="exhausted"):
        b.room_for([100, 50, 0])
    b = book(keep=40, first=4)
    layer = PagedLayer(b, 4, 2, 64)
    layer._offsets = [60, 60, 60]
    layer.kpages = torch.empty(1)
    with pytest.raises(PagesExhausted, match="do not fit"):
        layer.ensure_capacity(60 + 110, torch.float32, "cpu")
    assert issubclass(PagesExhausted, RuntimeError)


# ---------------------------------------------------------------- scratch
@pytest.mark.parametrize("H,G,line", [(32, 8, 4), (32, 32, 1), (6, 3, 2), (9, 3, 4), (40, 8, 8), (16, 1, 16), (9, 1, 16), (17, 1, 32), (40, 1, 48)])
def test_workspace_of_known_key_heads(H, G, line):
    """fp32 scores of whole tiles, ``line`` of them per key head and slot, and never more than the call that does not know the key heads."""
    f, g = L().b200p_paged_attn_workspace_bytes_of, L().b200p_paged_attn_workspace_bytes
    assert f(3, H, G, 64, 1000) - f(3, H, G, 64, 200) == 3 * G * line * (1008 - 208) * 4
    assert f(3, H, G, 64, 0) == g(3, H, 64, 0) and f(3, H, G, 64, 1000) <= g(3, H, 64, 1000)
    need = f(2, H, G, 64, 64)
    assert attn(H=H, G=G, mass=OK, bytes=need - 1) == ARG
    assert f(2, 9, 2, 64, 10) == 0 == f(2, 8, 0, 64, 10) == f(0, 8, 2, 64, 10)


def observed_calls(monkeypatch, L, heads=32, kv=8, D=8, offset=0, behind=0, **kw):
    """The attention calls with weights that a portion of L tokens makes: (row, slot, workspace bytes) each."""
    from mlx_parallm_b200.models import paged
    calls = []
    b = book(**kw)
    layer = paged.PagedLayer(b, heads, kv, D)
    layer._offsets = [offset] * b.rows
    b.behind = behind
    layer.kpages = layer.vpages = torch.zeros(1, dtype=torch.float16)
    layer.mass = torch.zeros(1)
    for name in ("paged_append", "paged_gather", "attn"):
        monkeypatch.setattr(paged.ops, name, lambda *a, **k: None)
    monkeypatch.setattr(paged.ops, "paged_attn", lambda q, k, v, table, row, slot, out, scale, mass=None, workspace=None, **kw: calls.append(
        (row.tolist(), slot.tolist(), workspace.numel())) if mass is not None else None)
    row = torch.arange(b.rows, dtype=torch.int32).repeat_interleave(L)
    slot = torch.arange(L, dtype=torch.int32).repeat(b.rows) + offset
    q = torch.empty((b.rows * L, heads * D), dtype=torch.float16)
    layer.append_and_attend(None, q, torch.empty_like(q), (row, slot, slot), b.rows, L, heads, None, 1.0, None, None, 1e-6, None, False)
    return calls


@pytest.mark.parametrize("kw,L", [(dict(rows=64, max_tokens=16384, keep=1000), 100), (dict(rows=16, max_tokens=131072, keep=1000), 40),
                                  (dict(rows=64, max_tokens=16384, keep=1000, window=500, first=4), 100), (dict(rows=3, max_tokens=200, keep=100), 20)], ids=str)
def test_weights_of_a_prompt_take_a_bounded_workspace(monkeypatch, kw, L):
    """Every row's last tokens in order, once each, in calls whose scratch does not grow with the table and the batch (a single token per row, which
    a decode step has as well, is the least)."""
    from mlx_parallm_b200.models import paged
    from mlx_parallm_b200.ops import paged_attn_workspace_bytes
    calls = observed_calls(monkeypatch, L, **kw)
    keys = min(kw["max_tokens"], 536 if "window" in kw else 1 << 30)
    assert max(c[2] for c in calls) <= max(paged.OBSERVED_BYTES + (16 << 20), paged_attn_workspace_bytes(kw["rows"], 32, 8, keys, 8))
    seen = [[] for _ in range(kw["rows"])]
    for rows, slots, _ in calls:
        assert len(rows) < 65536
        for r, s in zip(rows, slots):
            seen[r].append(s)
    assert seen == [list(range(L - min(L, 32), L))] * kw["rows"]


def test_weights_of_more_tokens_than_a_call_takes(monkeypatch):
    calls = observed_calls(monkeypatch, 32, heads=1, kv=1, rows=3000, max_tokens=64, keep=40)
    assert sum(len(c[0]) for c in calls) == 3000 * 32 and max(len(c[0]) for c in calls) < 65536


# ---------------------------------------------------------------- rows that were given back
def test_a_row_that_was_given_back_takes_no_page_again():
    """Two rows over a pool that holds one and a bit: after row 1 is given back, row 0 has the pool to itself, step by step to its last place."""
    from mlx_parallm_b200.models._transformer import prepare_cache, release_rows
    from mlx_parallm_b200.models.paged import PagedLayer, PagesExhausted
    b = book(rows=2, max_tokens=64, pages=4)
    layers = [PagedLayer(b, 4, 2, 64) for _ in range(2)]

    def step(n):
        prepare_cache(layers, 2, n, torch.float32, "cpu")
        for c in layers:
            c.advance_host(n)

    step(20)
    assert [len(o) for o in b.owned] == [2, 2] and b.row_index.tolist() == [0, 1]
    release_rows(layers, [1])
    assert b.row_index.tolist() == [0, -1] and [len(o) for o in b.owned] == [2, 0] and len(b.free) == 2
    where = b.row_index.data_ptr()
    for n in range(21, 65):
        step(1)
        assert [len(o) for o in b.owned] == [-(-n // 16), 0] and all(c.offsets == [n, 0] for c in layers)
        assert int(b.table[1].max()) == -1
    with pytest.raises(PagesExhausted):
        step(1)
    release_rows(layers, [1, 0])
    step(3)
    assert b.row_index.tolist() == [-1, -1] and len(b.free) == 4 and layers[1].offsets == [0, 0]
    for c in layers:
        c.reset(2)
    assert b.row_index.tolist() == [0, 1] and b.row_index.data_ptr() == where
    step(5)
    assert [len(o) for o in b.owned] == [1, 1] and layers[0].offsets == [5, 5]


@pytest.mark.parametrize("rows", [[1, 3], [0, -1], [7]], ids=str)
def test_rows_that_do_not_exist_are_not_given_back(rows):
    """Refused before anything of the others is given back."""
    from mlx_parallm_b200.models._transformer import release_rows
    from mlx_parallm_b200.models.paged import PagedLayer
    b = book()
    layers = [PagedLayer(b, 4, 2, 64) for _ in range(2)]
    for c in layers:
        c._offsets = [5, 20, 9]
    b.room_for([5, 20, 9])
    layers[0]._sync_lengths()
    with pytest.raises(ValueError):
        release_rows(layers, rows)
    assert all(c.offsets == [5, 20, 9] for c in layers) and b.lengths.tolist() == [5, 20, 9] and b.row_index.tolist() == [0, 1, 2]
    assert [len(o) for o in b.owned] == [1, 2, 1]


def test_advance_refuses():
    f = L().b200p_paged_advance
    assert f(0, OK, OK, 4, 1, 0) == ARG and f(OK, 0, OK, 4, 1, 0) == ARG and f(OK, OK, 0, 4, 1, 0) == ARG and f(OK, OK, OK, -1, 1, 0) == ARG
    assert f(OK, OK, OK, 0, 1, 0) == 0
    from mlx_parallm_b200 import ops
    with pytest.raises(_lib.B200PError):
        ops.paged_advance(torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 1)


@pytest.mark.parametrize("window,first,offset,n,hides", [(40, 0, 0, 40, False), (40, 0, 0, 41, True), (40, 4, 10, 34, False), (40, 4, 10, 35, True),
                                                        (0, 5, 60, 30, False), (1, 0, 0, 2, True)])
def test_prompts_whose_window_hides_nothing_go_through_the_dense_view(monkeypatch, window, first, offset, n, hides):
    """A token at slot s sees all of its row while s < window + first: until then the window takes no prompt from the prompt kernels."""
    from mlx_parallm_b200.models import paged
    said = []
    real = {name: getattr(paged.ops, name) for name in ("paged_append", "paged_gather", "attn", "paged_attn")}
    b = book(window=window, first=first)
    layer = paged.PagedLayer(b, 4, 2, 8)
    layer._offsets = [offset, offset // 2, offset]
    layer.kpages = torch.zeros(1, dtype=torch.float16)
    for name in real:
        monkeypatch.setattr(paged.ops, name, lambda *a, _name=name, **k: said.append(_name))
    q = torch.empty((3 * n, 32), dtype=torch.float16)
    t = torch.zeros(3 * n, dtype=torch.int32)
    layer.append_and_attend(None, q, torch.empty_like(q), (t, t, t), 3, n, 4, None, 1.0, None, None, 1e-6, None, False)
    assert said == (["paged_append", "paged_attn"] if hides else ["paged_append", "paged_gather", "attn"])


@pytest.mark.parametrize("n", [1, 2, 6])
def test_front_ends_end_with_all_of_their_tokens(monkeypatch, n):
    """prompt + n - 1 places are enough for n tokens, through a front-end too: it looks for one token more (the step that runs ahead, whose random
    numbers later generations do not share) and misses nothing."""
    from fake_tokenizer import FakeTokenizer
    from mlx_parallm_b200 import utils
    from mlx_parallm_b200.models.paged import PagesExhausted
    monkeypatch.setattr(utils.ops, "check_waits", lambda: None)
    step = _Step(n - 1)
    monkeypatch.setattr(utils, "_decode_step_for", lambda *a: step)
    cache = [type("C", (), {"_lengths": 1})()]
    tok = utils.TokenizerWrapper(FakeTokenizer(1000))
    words = " ".join(f"w{i}" for i in range(10, 10 + n))
    kw = dict(max_tokens=n, cache=cache)

    def again():
        step.n = 0
        return step

    assert again() and utils.generate(_Model(), tok, "w1 w2", **kw) == words
    assert again() and "".join(utils.stream_generate(_Model(), tok, "w1 w2", **kw)).split() == words.split()
    assert again() and utils.batch_generate(_Model(), tok, ["w1 w2"], format_prompts=False, **kw) == [words]
    assert again() and len(list(utils.batch_stream_generate_text(_Model(), tok, [[1, 2]], **kw))) == n
    with pytest.raises(PagesExhausted):
        again() and utils.generate(_Model(), tok, "w1 w2", max_tokens=n + 1, cache=cache)
    # the step ahead of the last token is launched as ever
    for room, steps in ((50, n + 1), (n, n)):
        again().room = room
        utils.generate(_Model(), tok, "w1 w2", **kw)
        assert step.n == steps

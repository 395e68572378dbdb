"""Models over a cache in pages (DecoderModel.make_paged_cache) against the oracle and against the same model over dense caches."""
import numpy as np
import pytest
import torch

from helpers import greedy_report, make_pair, prompts_for, rel_err
from oracle.model import OracleModel, generate_step as oracle_generate_step

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-2          # per-step logits within 1e-2 relative, as for dense caches
MODELS = [("tiny-llama", "float16"), ("tiny-llama", "float32"), ("tiny-qwen3", "bfloat16"), ("small-llama", "float16"), ("small-phi3", "bfloat16")]


def tokens_of(gm, prompts, steps, cache):
    from mlx_parallm_b200.utils import generate_step
    return np.stack([y[:, 0].cpu().numpy() for _, (y, _) in zip(range(steps), generate_step(torch.from_numpy(prompts), gm, cache=cache))], 1)


@pytest.mark.parametrize("keep", [0, 30], ids=["plain", "weighed"])
@pytest.mark.parametrize("name,dtype", MODELS)
def test_logits_of_prompt_and_steps(name, dtype, keep):
    """A prompt, a portion behind it and single tokens: every position's logits against the oracle's whole forward."""
    cfg, om, gm = make_pair(name, dtype=dtype)
    ids = prompts_for(cfg, 3, 29)
    exp = om.forward(ids, om.make_cache(3))
    cache = gm.make_paged_cache(3, 40, page=16, keep=keep)
    t = torch.from_numpy(ids)
    got = [gm(t[:, :13], cache=cache), gm(t[:, 13:25], cache=cache)] + [gm(t[:, i:i + 1], cache=cache) for i in range(25, 29)]
    err = rel_err(torch.cat(got, 1).cpu().numpy(), exp)
    print(f"{name} {dtype}: logits rel err {err:.2e}")
    assert err < LOGIT_TOL
    assert cache[0].offsets == [29] * 3 and cache[0].book.lengths.tolist() == [29] * 3 == cache[0].book.positions.tolist()


@pytest.mark.parametrize("name,dtype", MODELS)
def test_greedy_generation(name, dtype):
    """generate_step over pages (captured decode step) keeps to the oracle's transcript but for near-ties."""
    cfg, om, gm = make_pair(name, dtype=dtype)
    ids = prompts_for(cfg, 4, 20, seed=3)
    got = tokens_of(gm, ids, 40, gm.make_paged_cache(4, 64, page=16))
    steps = [(y[:, 0], lg) for _, (y, lg) in zip(range(40), oracle_generate_step(ids, om))]
    frac, near, real = greedy_report(got, np.stack([y for y, _ in steps], 1), [lg for _, lg in steps], LOGIT_TOL)
    assert not real, real


def test_prompt_in_portions(monkeypatch):
    from mlx_parallm_b200.models import _transformer
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = prompts_for(cfg, 2, 150)
    whole = gm(torch.from_numpy(ids), cache=gm.make_paged_cache(2, 160, page=48), last_only=True)
    monkeypatch.setattr(_transformer, "MAX_TOKENS_PER_FORWARD", 100)
    parts = gm(torch.from_numpy(ids), cache=gm.make_paged_cache(2, 160, page=48), last_only=True)
    exp = om.forward(ids, om.make_cache(2), last_only=True)
    assert rel_err(whole.cpu().numpy(), exp) < LOGIT_TOL and rel_err(parts.cpu().numpy(), exp) < LOGIT_TOL


@pytest.mark.parametrize("observe", [0, 7, 60, 1000])
def test_weights_of_a_prompts_last_tokens(monkeypatch, observe):
    """The last ``observe`` tokens of a prompt give every head's weight of one each, and no others, in however many portions it is read."""
    from mlx_parallm_b200.models import _transformer
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 2, 150))
    seen = []
    for at_once in (8192, 100, 46):
        monkeypatch.setattr(_transformer, "MAX_TOKENS_PER_FORWARD", at_once)
        cache = gm.make_paged_cache(2, 200, page=48, keep=100, observe=observe)
        gm(ids, cache=cache, last_only=True)
        for c in cache:
            pages = c.book.table.cpu()
            mass = torch.stack([torch.cat([c.mass[p].cpu() for p in row if p >= 0], 1)[:, :150] for row in pages])
            # a row of 150 weights sums to 1 to about 150 roundings of 2^-24
            exp = min(observe, 150) * c.n_heads
            assert bool(((mass.sum((1, 2)) - exp).abs() <= 1e-4 * exp).all()), (at_once, mass.sum((1, 2)), exp)
            seen.append(mass)
        gm(ids[:, :1], cache=cache, last_only=True)             # and a step's token its own
        left = torch.stack([torch.cat([cache[0].mass[p].cpu() for p in row if p >= 0], 1)[:, :151] for row in cache[0].book.table.cpu()]).sum((1, 2))
        exp = (min(observe, 150) + 1) * cache[0].n_heads
        assert bool(((left - exp).abs() <= 1e-4 * exp).all())


def test_window_that_hides_nothing_and_one_that_does():
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = prompts_for(cfg, 2, 60)
    exp = om.forward(ids, om.make_cache(2), last_only=True)
    wide = gm(torch.from_numpy(ids), cache=gm.make_paged_cache(2, 64, page=16, window=64, first=3), last_only=True).cpu().numpy()
    assert rel_err(wide, exp) < LOGIT_TOL
    cache = gm.make_paged_cache(2, 64, page=16, window=16, first=2)
    narrow = gm(torch.from_numpy(ids), cache=cache, last_only=True).cpu().numpy()
    assert np.isfinite(narrow).all() and rel_err(narrow, exp) > 10 * LOGIT_TOL


@pytest.mark.parametrize("keep", [0, 24])
def test_captured_and_eager_steps_agree(keep):
    """The same tokens from a replayed and from a launched decode step, through growth of the rows and (keep) three cuts."""
    from mlx_parallm_b200.utils import DecodeSession
    cfg, _, gm = make_pair("small-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 3, 20, seed=5))
    out = []
    for graph in (False, True):
        cache = gm.make_paged_cache(3, 48 if keep else 128, page=16, keep=keep, first=2, recent=8)
        first = gm(ids, cache=cache, last_only=True)[:, -1].argmax(-1).to(torch.int32)
        session = DecodeSession(gm, cache, 3, True, use_graph=graph)
        session.tok.copy_(first)
        toks = []
        for _ in range(90):
            session.run()
            toks.append(session.tok.clone())
            assert bool(torch.isfinite(session.logits).all())
        out.append(torch.stack(toks, 1).cpu())
        book = cache[0].book
        assert book.positions.tolist() == [110] * 3 and book.lengths.tolist() == cache[0].offsets
        assert [n + e for n, e in zip(cache[0].offsets, book.evicted)] == [110] * 3
        if keep:
            assert max(cache[0].offsets) <= 48 and sum(len(o) for o in book.owned) + len(book.free) == book.pages
    assert torch.equal(out[0], out[1])


def test_long_generation_with_cuts_through_generate_step():
    cfg, _, gm = make_pair("tiny-qwen3", dtype="bfloat16")
    got = tokens_of(gm, prompts_for(cfg, 2, 30), 200, gm.make_paged_cache(2, 64, page=16, keep=40, first=4))
    assert got.shape == (2, 200) and (0 <= got).all() and (got < cfg["vocab_size"]).all()


def test_rows_are_given_back_and_taken_again():
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    cache = gm.make_paged_cache(2, 64, page=16, pages=4)
    book = cache[0].book
    ids = prompts_for(cfg, 2, 30)
    gm(torch.from_numpy(ids), cache=cache)
    assert len(book.free) == 0
    with pytest.raises(RuntimeError, match="exhausted"):
        gm(torch.from_numpy(ids[:, :9]), cache=cache)
    for c in cache:
        c.reset(2)
    assert len(book.free) == 4 and int(book.table.max()) == -1
    again = prompts_for(cfg, 2, 20, seed=9)
    got = gm(torch.from_numpy(again), cache=cache, last_only=True).cpu().numpy()
    assert rel_err(got, om.forward(again, om.make_cache(2), last_only=True)) < LOGIT_TOL


def test_a_prompt_that_does_not_fit_is_refused():
    cfg, _, gm = make_pair("tiny-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 1, 65))
    with pytest.raises(RuntimeError, match="does not fit"):
        gm(ids, cache=gm.make_paged_cache(1, 64, page=16))
    with pytest.raises(RuntimeError, match="do not fit"):
        gm(ids, cache=gm.make_paged_cache(1, 64, page=16, keep=32, first=2))


@pytest.mark.parametrize("pages", [None, 6], ids=["all pages", "pages that just suffice"])
def test_generations_that_just_fit(pages):
    """prompt + max_tokens places (a whole number of pages), through generate_step and the four text front-ends: all of the tokens, no error; one
    token more is refused once it is asked for."""
    from fake_tokenizer import FakeTokenizer
    from mlx_parallm_b200.models.paged import PagesExhausted
    from mlx_parallm_b200.tokenizer_utils import TokenizerWrapper
    from mlx_parallm_b200.utils import batch_generate, batch_stream_generate_text, generate, generate_step, stream_generate
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = prompts_for(cfg, 2, 28)
    width = 48 if pages is None else 64
    make = lambda rows: gm.make_paged_cache(rows, width, page=16, pages=None if pages is None else pages * rows // 2)
    steps = [(y[:, 0], lg) for _, (y, lg) in zip(range(21), oracle_generate_step(ids, om))]

    def check(got):
        got = np.stack(got, 1)
        n = got.shape[1]
        assert not greedy_report(got, np.stack([y for y, _ in steps[:n]], 1), [lg for _, lg in steps[:n]], LOGIT_TOL)[2]
        return n

    assert check([y[:, 0].cpu().numpy() for (y, _), _ in zip(generate_step(torch.from_numpy(ids), gm, cache=make(2)), range(20))]) == 20
    run = generate_step(torch.from_numpy(ids), gm, cache=make(2))
    assert check([next(run)[0][:, 0].cpu().numpy() for _ in range(21)]) == 21
    with pytest.raises(PagesExhausted):
        next(run)
    tok = TokenizerWrapper(FakeTokenizer(cfg["vocab_size"], eos_token_id=cfg["vocab_size"] + 1))      # (never said)
    texts = [" ".join(f"w{i}" for i in row) for row in ids]
    assert len(generate(gm, tok, texts[0], max_tokens=20, cache=make(1)).split()) == 20
    assert len("".join(stream_generate(gm, tok, texts[0], max_tokens=20, cache=make(1))).split()) == 20
    answers = batch_generate(gm, tok, texts, max_tokens=20, format_prompts=False, cache=make(2))
    assert check([np.array([int(t.split()[i][1:]) for t in answers]) for i in range(20)]) == 20
    said = list(batch_stream_generate_text(gm, tok, ids, 20, cache=make(2)))
    assert len(said) == 20 and all(reason == "length" for _, reason in said[-1])


@pytest.mark.parametrize("window", [0, 70])
def test_weights_of_a_prompts_last_tokens_in_small_calls(monkeypatch, window):
    """However many calls the workspace's bound makes of them: the same weights, to the roundings of a sum of 60 (fp32, and scores that came through
    logits of LOGIT_TOL in the layers before)."""
    from mlx_parallm_b200.models import paged
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 3, 90))
    out = []
    for size in (1 << 28, 1 << 20, 1):
        monkeypatch.setattr(paged, "OBSERVED_BYTES", size)
        cache = gm.make_paged_cache(3, 1000, page=48, keep=100, observe=60, window=window, first=3 if window else 0)
        gm(ids, cache=cache, last_only=True)
        out.append([c.mass.clone() for c in cache])
        assert all(abs(float(m.sum()) - 3 * 60 * c.n_heads) <= 1e-4 * 180 * c.n_heads for m, c in zip(out[-1], cache))
    for a, b, c in zip(*out):
        assert float((a - b).abs().max()) <= LOGIT_TOL * float(a.abs().max()) and float((a - c).abs().max()) <= LOGIT_TOL * float(a.abs().max())


@pytest.mark.parametrize("keep", [0, 24])
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "captured"])
def test_rows_given_back_stay_idle(graph, keep):
    """A row is given back between two replays of a step: its counters stay at nothing and it takes no page, the others' logits are the oracle's, and
    a portion of a prompt and (keep) a cut pass it by.  Nothing meets a place that does not exist."""
    from mlx_parallm_b200 import ops
    from mlx_parallm_b200.utils import DecodeSession
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = prompts_for(cfg, 3, 60, seed=11)
    ops.paged_fault_count(reset=True)
    cache = gm.make_paged_cache(3, 48, page=16, pages=8, keep=keep, first=2, recent=8)
    book = cache[0].book
    exp = om.forward(ids, om.make_cache(3))
    gm(torch.from_numpy(ids[:, :20]), cache=cache, last_only=True)
    session = DecodeSession(gm, cache, 3, True, use_graph=graph)

    def step(i, rows):
        session.tok.copy_(torch.from_numpy(ids[:, i]).to(torch.int32))
        session.run()
        assert bool(torch.isfinite(session.logits).all())
        if i < 48:                                                  # (cuts change what is seen)
            assert rel_err(session.logits[rows].cpu().numpy(), exp[rows, i]) < LOGIT_TOL

    for i in range(20, 30):
        step(i, [0, 1, 2])
    gm.release_rows(cache, [1])
    assert book.row_index.tolist() == [0, -1, 2] and book.owned[1] == [] and len(book.free) == 4
    for i in range(30, 34):
        step(i, [0, 2])
    got = gm(torch.from_numpy(ids[:, 34:40]), cache=cache).cpu().numpy()      # a portion
    assert rel_err(got[[0, 2]], exp[[0, 2], 34:40]) < LOGIT_TOL and np.isfinite(got).all()
    for i in range(40, 60 if keep else 48):
        step(i, [0, 2])
    n = 60 if keep else 48
    assert book.positions.tolist() == [n, 0, n] and book.lengths.tolist() == cache[0].offsets == [min(n, cache[0].offsets[0]), 0, cache[0].offsets[0]]
    assert book.owned[1] == [] and int(book.table[1].max()) == -1 and ops.paged_fault_count(reset=True) == 0
    for c in cache:
        c.reset(3)
    again = gm(torch.from_numpy(ids[:, :20]), cache=cache).cpu().numpy()
    assert rel_err(again, exp[:, :20]) < LOGIT_TOL


def test_dense_rows_are_not_given_back():
    cfg, _, gm = make_pair("tiny-llama", dtype="float16")
    with pytest.raises(NotImplementedError):
        gm.release_rows(gm.make_cache(2), [1])


def test_front_ends_use_the_last_place():
    """prompt + max_tokens - 1 places: the last token needs none."""
    from fake_tokenizer import FakeTokenizer
    from mlx_parallm_b200.tokenizer_utils import TokenizerWrapper
    from mlx_parallm_b200.utils import batch_generate, batch_stream_generate_text, generate, stream_generate
    cfg, _, gm = make_pair("tiny-llama", dtype="float16")
    ids = prompts_for(cfg, 2, 28)
    texts = [" ".join(f"w{i}" for i in row) for row in ids]
    tok = TokenizerWrapper(FakeTokenizer(cfg["vocab_size"], eos_token_id=cfg["vocab_size"] + 1))      # (never said)
    make = lambda rows: gm.make_paged_cache(rows, 48, page=16)
    assert len(generate(gm, tok, texts[0], max_tokens=21, cache=make(1)).split()) == 21
    assert len("".join(stream_generate(gm, tok, texts[0], max_tokens=21, cache=make(1))).split()) == 21
    assert [len(t.split()) for t in batch_generate(gm, tok, texts, max_tokens=21, format_prompts=False, cache=make(2))] == [21, 21]
    said = list(batch_stream_generate_text(gm, tok, ids, 21, cache=make(2)))
    assert len(said) == 21 and all(reason == "length" for _, reason in said[-1])


# ---------------------------------------------------------------- windows, cuts and dense caches, logit by logit
# Tolerance of the next tests: |engine - oracle| <= |engine - the oracle with the engine's rounding points| + |that - the oracle|.  LOGIT_TOL is for
# the first; the second is computed.  (bf16 needs it: half a step is 2^-8, and for tiny-qwen3's 61440 logits behind a window the rounding points alone,
# numerics="mirror", are 0.0053 from the oracle, whose own 16-bit projections are rounded before the norm, behind it and behind the rotation, where the
# engine rounds once.)
def mirror_of(om):
    return OracleModel(om.cfg, om.w, numerics="mirror")


def window_mask(L, offset, first, window):
    """bool [1, 1, L, offset + L]: token t at position offset + t sees j <= its own with j < first or j > its own - window."""
    s, j = offset + np.arange(L)[:, None], np.arange(offset + L)[None, :]
    return ((j <= s) & ((j < first) | (j > s - window)))[None, None]


@pytest.mark.parametrize("keep", [0, 60], ids=["plain", "weighed"])
@pytest.mark.parametrize("name,dtype", MODELS)
def test_logits_behind_a_window(name, dtype, keep):
    """Prompts that end where the window (16, and 2 first tokens) hides nothing yet, one token further, and long ones, in one piece, in portions and
    token by token: every position's logits against the oracle under the window's mask."""
    cfg, om, gm = make_pair(name, dtype=dtype)
    ids = prompts_for(cfg, 2, 60, seed=21)
    full = om.forward(ids, om.make_cache(2), visible=lambda layer: window_mask(60, 0, 2, 16))
    plain = om.forward(ids, om.make_cache(2))
    assert rel_err(full[:, :18], plain[:, :18]) < 1e-5 and rel_err(full[:, 18:], plain[:, 18:]) > 10 * LOGIT_TOL
    mi = mirror_of(om)
    tol = LOGIT_TOL + rel_err(mi.forward(ids, mi.make_cache(2), visible=lambda layer: window_mask(60, 0, 2, 16)), full)
    t = torch.from_numpy(ids)
    for cuts in ([18, 19, 20, 44, 45, 46, 60], [19, 60], [5, 18, 19, 60], [60]):
        cache = gm.make_paged_cache(2, 64, page=16, window=16, first=2, keep=keep)
        at = [0] + cuts
        got = torch.cat([gm(t[:, a:b], cache=cache) for a, b in zip(at, at[1:])], 1).cpu().numpy()
        assert rel_err(got, full) < tol, cuts


# What every slot receives, relative to the largest: weights move by twice what their scores do; q and k carry half a step of their type each, of products
# up to 8.3 in these models (|q| |k| scale), and the layers before them an error below LOGIT_TOL.
RECEIVED_TOL = {"float16": 3e-2, "float32": 3e-2, "bfloat16": 0.15}


@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("name,dtype", [("small-llama", "float16"), ("tiny-qwen3", "bfloat16"), ("tiny-llama", "float32")])
def test_logits_across_cuts(monkeypatch, name, dtype, window):
    """Steps through two cuts of full rows.  At each the cache has added up the weights that the oracle gives, keeps what the selection's definition
    says (the 2 first, the 8 newest, the most attended between, per layer and key head), and afterwards the logits are those of the oracle with everything
    else hidden and the tokens kept at their positions in the text."""
    import paged_oracle as po
    from mlx_parallm_b200 import ops
    cfg, om, gm = make_pair(name, dtype=dtype)
    B, prompt, total, keep, observe = 2, 30, 96, 24, 10
    ids = prompts_for(cfg, B, total, seed=31)
    cache, oc = gm.make_paged_cache(B, 48, page=16, keep=keep, first=2, recent=8, observe=observe, window=window), om.make_cache(B)
    mi = mirror_of(om)
    mc = mi.make_cache(B)
    G, layers = cache[0].n_kv_heads, len(cache)
    cut, evict = [], ops.paged_evict

    def spy(k, v, mass, table, lengths, kept, first=0, recent=0):
        before = [t.cpu().clone() for t in (mass, table, lengths)]
        evict(k, v, mass, table, lengths, kept, first=first, recent=recent)
        cut.append((*before, kept.cpu().clone(), first, recent))
        return kept

    monkeypatch.setattr(ops, "paged_evict", spy)
    alive = [[[list(range(prompt)) for _ in range(G)] for _ in range(B)] for _ in range(layers)]       # positions, by slot
    received = [np.zeros((B, G, total)) for _ in range(layers)]

    def seen(layer, n):
        """Of n tokens, which the token behind them sees."""
        m = np.zeros((B, G, 1, n + 1), bool)
        for b in range(B):
            for g in range(G):
                a = alive[layer][b][g] + [n]
                m[b, g, 0, [p for s, p in enumerate(a) if not window or s < 2 or s >= len(a) - window]] = True
        return m

    gm(torch.from_numpy(ids[:, :prompt]), cache=cache, last_only=True)
    w = []
    om.forward(ids[:, :prompt], oc, visible=lambda layer: window_mask(prompt, 0, 2, window or total), received=w)
    mi.forward(ids[:, :prompt], mc, visible=lambda layer: window_mask(prompt, 0, 2, window or total))
    for layer in range(layers):
        received[layer][:, :, :prompt] += w[layer][:, :, -observe:].sum(2)
    cuts = 0
    for n in range(prompt, total):
        got = gm(torch.from_numpy(ids[:, n:n + 1]), cache=cache).cpu().numpy()
        if cut:
            assert len(cut) == layers
            cuts += 1
            for layer, (mass, table, lengths, kept, first, recent) in enumerate(cut):
                assert (first, recent) == (2, 8) and lengths.tolist() == [48] * B and kept.shape == (B, G, keep)
                assert torch.equal(kept.long(), po.select(mass, table, lengths, keep, 2, 8))
                for b in range(B):
                    here = torch.cat([mass[p] for p in table[b] if p >= 0], 1)[:, :48].numpy()
                    for g in range(G):
                        exp = received[layer][b, g, alive[layer][b][g]]
                        assert np.abs(here[g] - exp).max() <= RECEIVED_TOL[dtype] * exp.max(), (n, layer, b, g)
                        assert kept[b, g, :2].tolist() == [0, 1] and kept[b, g, -8:].tolist() == list(range(40, 48))
                        alive[layer][b][g] = [alive[layer][b][g][s] for s in kept[b, g].tolist()]
            cut.clear()
        w = []
        exp = om.forward(ids[:, n:n + 1], oc, visible=lambda layer: seen(layer, n), received=w)
        rounded = mi.forward(ids[:, n:n + 1], mc, visible=lambda layer: seen(layer, n))
        assert rel_err(got, exp) < LOGIT_TOL + rel_err(rounded, exp), n
        for layer in range(layers):
            received[layer][:, :, :n + 1] += w[layer][:, :, 0]
            for b in range(B):
                for g in range(G):
                    alive[layer][b][g].append(n)
        assert cache[0].offsets == [len(alive[0][0][0])] * B and cache[0].book.positions.tolist() == [n + 1] * B
    assert cuts == 2                                                # at 48 tokens, and 24 further on


@pytest.mark.parametrize("name,dtype", MODELS)
def test_logits_of_dense_caches(name, dtype):
    """The same prompt, portion and steps over a dense cache and over pages: each within LOGIT_TOL of exact, so twice that of each other."""
    cfg, _, gm = make_pair(name, dtype=dtype)
    t = torch.from_numpy(prompts_for(cfg, 3, 40, seed=41))
    out = []
    for cache in (gm.make_cache(3), gm.make_paged_cache(3, 40, page=16), gm.make_paged_cache(3, 48, page=48, window=100, keep=40)):
        out.append(torch.cat([gm(t[:, a:b], cache=cache) for a, b in ((0, 25), (25, 37), (37, 38), (38, 39), (39, 40))], 1).cpu().numpy())
    print(f"{name} {dtype}: pages against dense {rel_err(out[1], out[0]):.2e} {rel_err(out[2], out[0]):.2e}")
    assert rel_err(out[1], out[0]) < 2 * LOGIT_TOL and rel_err(out[2], out[0]) < 2 * LOGIT_TOL


def test_logits_with_adapters():
    """LoRA on q and v of every layer, prompts and steps over pages, against the oracle with the same adapters."""
    from test_gpu_lora import _adapters
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ad = _adapters(cfg, 8, np.random.default_rng(5), layers=range(cfg["num_hidden_layers"]))
    for k in ad:
        if k.endswith("lora_a"):
            pre = k[:-len(".lora_a")]
            om.lora[pre] = (ad[k].float().numpy(), ad[pre + ".lora_b"].float().numpy(), 10.0)
    ids = prompts_for(cfg, 2, 24, seed=51)
    base = gm(torch.from_numpy(ids), cache=gm.make_paged_cache(2, 32, page=16)).cpu().numpy()
    gm.apply_lora(ad, 10.0)
    exp = om.forward(ids, om.make_cache(2))
    cache = gm.make_paged_cache(2, 32, page=16, keep=20)
    got = torch.cat([gm(torch.from_numpy(ids[:, a:b]), cache=cache) for a, b in ((0, 21), (21, 22), (22, 24))], 1).cpu().numpy()
    assert rel_err(got, exp) < LOGIT_TOL and rel_err(got, base) > 1e-3

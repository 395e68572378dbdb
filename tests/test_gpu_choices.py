"""Models that score texts, hold adapters for single rows and share prompts: DecoderModel.score, apply_loras / bind_adapters, share_prompt, generate_step's
log probabilities, generate_choices and score_text, alone and together."""
import math

import numpy as np
import pytest
import torch

from fake_tokenizer import FakeTokenizer
from helpers import make_pair, prompts_for, rel_err
from mlx_parallm_b200 import _lib
from mlx_parallm_b200.models import _transformer, paged
from mlx_parallm_b200.utils import generate_choices, generate_step, score_text

pytestmark = pytest.mark.gpu

LOGIT_TOL = 1e-2          # logits within 1e-2 of the largest, as everywhere: log probabilities differ by twice that at most
MODELS = [("tiny-llama", "float16"), ("tiny-llama", "float32"), ("tiny-qwen3", "bfloat16"), ("small-llama", "float16"), ("small-phi3", "bfloat16")]


def adapters_for(cfg, rank, seed, keys=("self_attn.q_proj", "self_attn.v_proj"), layers=None, size=0.3):
    g = torch.Generator().manual_seed(seed)
    D, h = cfg.get("head_dim") or cfg["hidden_size"] // cfg["num_attention_heads"], cfg["hidden_size"]
    width = {"q_proj": cfg["num_attention_heads"] * D, "k_proj": cfg["num_key_value_heads"] * D, "v_proj": cfg["num_key_value_heads"] * D}
    out = {}
    for i in layers if layers is not None else range(cfg["num_hidden_layers"]):
        for k in keys:
            out[f"model.layers.{i}.{k}.lora_a"] = torch.randn((h, rank), generator=g) / h ** 0.5
            out[f"model.layers.{i}.{k}.lora_b"] = torch.randn((rank, width[k.split(".")[-1]]), generator=g) * size
    return out


@pytest.fixture
def groups_always(monkeypatch):
    """Steps go by groups however little their rows share."""
    monkeypatch.setattr(paged, "SHARED_BYTES", 0)
    _lib.lib().b200p_paged_attn_shared_set_path(1)
    yield
    _lib.lib().b200p_paged_attn_shared_set_path(0)


# ---------------------------------------------------------------------------------------------------------------- scoring
@pytest.mark.parametrize("name,dtype", MODELS)
def test_score_against_the_oracle(name, dtype):
    cfg, om, gm = make_pair(name, dtype=dtype)
    ids = prompts_for(cfg, 3, 37)
    logits = torch.from_numpy(np.asarray(om.forward(ids, om.make_cache(3)), np.float64))
    lp = torch.log_softmax(logits, -1)
    tol = 2 * LOGIT_TOL * float(logits.abs().max())
    s = gm.score(torch.from_numpy(ids), top=4)
    assert s.logprob.shape == (3, 37) and s.top_ids.shape == (3, 37, 4)
    want = lp[:, :-1].gather(2, torch.from_numpy(ids)[:, 1:, None])[..., 0]
    assert (s.logprob[:, :-1].cpu() - want).abs().max() < tol and (s.logprob[:, -1] == 0).all()
    # an entropy moves by no more than the largest |log p| times what the probabilities move: (2 tol) here
    assert (s.entropy.cpu() - torch.special.entr(lp.exp()).sum(-1)).abs().max() < 2 * tol * float(lp.abs().max())
    assert (s.top_logprobs.cpu() - lp.gather(2, s.top_ids.long().cpu())).abs().max() < tol
    assert (s.top_logprobs.cpu() - lp.sort(-1, descending=True).values[..., :4]).abs().max() < tol


def test_score_in_portions_and_behind_a_cache(monkeypatch):
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 2, 300))
    whole = gm.score(ids, top=3)
    tol = 2 * LOGIT_TOL * float(np.abs(om.forward(ids.numpy(), om.make_cache(2))).max())
    monkeypatch.setattr(_transformer, "MAX_TOKENS_PER_FORWARD", 90)
    monkeypatch.setattr(_transformer, "SCORE_BYTES", 4 * cfg["vocab_size"] * 7)
    parts = gm.score(ids, top=3)
    assert (whole.logprob - parts.logprob).abs().max() < tol and (whole.entropy - parts.entropy).abs().max() < tol * 20
    cache = gm.make_cache(2)
    a, b = gm.score(ids[:, :100], cache=cache), gm.score(ids[:, 100:], cache=cache)
    assert (torch.cat([a.logprob[:, :-1], whole.logprob[:, 99:100], b.logprob], 1) - whole.logprob).abs().max() < tol
    hot = gm.score(ids, temperature=2.0)
    logits = gm(ids).double()
    want = torch.log_softmax(logits / 2, -1)[:, :-1].gather(2, ids[:, 1:, None].cuda())[..., 0]
    assert (hot.logprob[:, :-1] - want).abs().max() < tol
    one = gm.score(ids[:, :1], top=2)                                # a single token: nothing follows, but what may is known
    assert one.logprob.tolist() == [[0.0], [0.0]] and one.top_ids.shape == (2, 1, 2)


def test_score_of_a_model_with_packed_prompts():
    import negosun_oracle as O
    from mlx_parallm_b200.utils import _get_classes
    cfg = O.make_config([O.layer(4, 2, 8, 12, 0.35, v_mix=False, q_temp=(0.4, 6), mlp=O.moe_mlp(6, 2, 16, (3, 2), shared=20))])
    Model, Args = _get_classes(cfg)
    w = O.random_weights(cfg, 0)
    gm = Model(Args.from_dict(cfg)).load_weights(w, device="cuda", dtype=torch.float32)
    rng = np.random.default_rng(3)
    n = [9, 4, 1]
    rows = [rng.integers(0, cfg["vocab"], k).tolist() for k in n]
    ids = torch.tensor([[0] * (9 - k) + r for k, r in zip(n, rows)])
    s = gm.score(ids, top=2, prompt_lengths=n)
    for b, r in enumerate(rows):
        lp = torch.log_softmax(torch.as_tensor(O.forward(cfg, w, r)).double().cpu().view(len(r), -1), -1)
        at = 9 - n[b]
        assert (s.logprob[b, :at] == 0).all() and s.logprob[b, -1] == 0
        for l in range(n[b] - 1):
            assert abs(float(s.logprob[b, at + l]) - float(lp[l, r[l + 1]])) < 2e-3
        assert (s.top_logprobs[b, at:].cpu().double() - lp.sort(-1, descending=True).values[:, :2]).abs().max() < 2e-3
        assert (s.entropy[b, at:].cpu() - torch.special.entr(lp.exp()).sum(-1)).abs().max() < 5e-3


def test_scores_that_are_refused_leave_the_cache_as_it_was():
    import negosun_oracle as O
    from mlx_parallm_b200.utils import _get_classes
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ocfg = O.make_config([O.layer(4, 2, 8, 12, 0.35, v_mix=False, q_temp=(0.4, 6), mlp=O.moe_mlp(6, 2, 16, (3, 2), shared=20))])
    Model, Args = _get_classes(ocfg)
    packed = Model(Args.from_dict(ocfg)).load_weights(O.random_weights(ocfg, 0), device="cuda", dtype=torch.float32)
    for model, ids in ((gm, torch.from_numpy(prompts_for(cfg, 2, 9))), (packed, torch.randint(0, ocfg["vocab"], (2, 9)))):
        cache = model.make_cache(2)
        for kw in (dict(top=33), dict(top=-1), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=1e30)):
            with pytest.raises(ValueError):
                model.score(ids, cache=cache, **kw)
        for k in (33, -1):
            with pytest.raises(ValueError):
                next(generate_step(ids, model, cache=cache, logprobs=k))
        assert all(c.offsets == [0, 0] for c in cache)
        assert model.score(ids, cache=cache, top=1).top_ids.shape == (2, 9, 1) and cache[-1].offsets == [9, 9]


@pytest.mark.parametrize("paged_cache", [False, True])
@pytest.mark.parametrize("temp", [0.0, 0.8])
def test_log_probabilities_of_generated_tokens(temp, paged_cache):
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 3, 20))
    cache = gm.make_paged_cache(3, 64, page=16) if paged_cache else None
    tokens, said = [], []
    for _, (y, p, lp) in zip(range(12), generate_step(ids, gm, temp=temp, cache=cache, logprobs=5)):
        tokens.append(y)
        said.append(lp)
        if temp == 0:
            assert torch.equal(lp.top_ids[:, 0].long(), y[:, 0]) and torch.equal(lp.top_logprobs[:, 0], lp.logprob)
        assert (lp.logprob.exp() - p[:, 0]).abs().max() < 1e-5       # the probability that came before
    text = torch.cat([ids.cuda()] + tokens, 1)
    s = gm.score(text)
    tol = 2 * LOGIT_TOL * float(gm(text).abs().max())
    assert (torch.stack([v.logprob for v in said], 1) - s.logprob[:, 19:-1]).abs().max() < tol


# ---------------------------------------------------------------------------------------------------------------- adapters
@pytest.mark.parametrize("name,dtype", [("tiny-llama", "float16"), ("tiny-qwen3", "bfloat16"), ("small-llama", "float16")])
@pytest.mark.parametrize("paged_cache", [False, True])
def test_rows_under_their_own_adapters(name, dtype, paged_cache):
    """Prompt and steps of a mixed batch against the oracle's rows under their adapters (or none), and against apply_lora's."""
    cfg, om, gm = make_pair(name, dtype=dtype)
    td = getattr(torch, dtype)
    sets = [adapters_for(cfg, 8, 1), adapters_for(cfg, 16, 2), adapters_for(cfg, 3, 3, keys=("self_attn.v_proj",), layers=[1])]
    which = [0, -1, 1, 2, 0, 1]
    ids = torch.from_numpy(prompts_for(cfg, 6, 25))
    alone = []
    for r, w in enumerate(which):
        gm.apply_lora({} if w < 0 else sets[w], 2.0 + w)
        alone.append(gm(ids[r:r + 1]))
    gm.apply_lora({}, 1.0)
    plain = gm(ids)
    gm.apply_loras(sets, [2.0, 3.0, 4.0])
    # held, but no row is under one (decode-sized projections add their parts in the order they come: the same but for that)
    assert rel_err(gm(ids).cpu(), plain.cpu()) < LOGIT_TOL
    make = lambda: gm.make_paged_cache(6, 40, page=16) if paged_cache else gm.make_cache(6)
    cache = make()
    gm.bind_adapters(cache, which)
    got = torch.cat([gm(ids[:, :20], cache=cache)] + [gm(ids[:, i:i + 1], cache=cache) for i in range(20, 25)], 1)
    for r in range(6):
        om.lora = {} if which[r] < 0 else {k[:-len(".lora_a")]: (v.to(td).float().numpy(), sets[which[r]][k[:-1] + "b"].to(td).float().numpy(), 2.0 + which[r])
                                          for k, v in sets[which[r]].items() if k.endswith("lora_a")}
        exp = om.forward(ids[r:r + 1].numpy(), om.make_cache(1))[0]
        errs = rel_err(got[r].cpu(), exp), rel_err(alone[r][0].cpu(), exp)
        print(name, r, errs)
        # An update is x A of deviation 1 (x is normed, A's columns have length 1) times B of 0.3 over `rank` >= 8 sums times a scale >= 2: 1.7 or more of the
        # projection's own deviation of about 1.  Values and their 16-bit roundings are twice as large beside the same residual stream, so the tolerance
        # is that of two; the two ways, each that far from the oracle at most, are within the sum of both.
        tol = LOGIT_TOL * (2 if which[r] >= 0 else 1)
        assert max(errs) < tol, (r, errs)
        assert rel_err(got[r].cpu(), alone[r][0].cpu()) < 2 * tol, r
        if which[r] >= 0:
            assert rel_err(plain[r].cpu(), alone[r][0].cpu()) > 2 * LOGIT_TOL      # they matter
    cache[0].reset(6) if not paged_cache else [c.reset() for c in cache]
    assert cache[0].adapter_rows is None


def test_generation_under_adapters_that_change():
    """The captured step follows bind_adapters, and goes without them again."""
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    sets = [adapters_for(cfg, 16, 5), adapters_for(cfg, 32, 6, keys=("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj"))]
    ids = torch.from_numpy(prompts_for(cfg, 3, 10))
    for keys in (("self_attn.q_proj", "self_attn.v_proj"), ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj")):
        gm.apply_loras(sets, [1.0, 0.5], keys=keys)
        for which in ([0, 1, -1], [1, 1, 0], None, [-1, -1, -1]):
            said = [lp for _, (y, p, lp) in zip(range(6), generate_step(ids, gm, logprobs=1, adapters=which))]
            tokens = torch.stack([v.top_ids[:, 0] for v in said], 1).long()
            text = torch.cat([ids.cuda(), tokens], 1)
            s = gm.score(text, adapters=which)
            tol = 2 * LOGIT_TOL * float(gm(text).abs().max())
            assert (torch.stack([v.logprob for v in said], 1) - s.logprob[:, 9:-1]).abs().max() < tol, which
    plain = [y for _, (y, _) in zip(range(6), generate_step(ids, gm))]
    gm.apply_loras([], [])
    assert torch.equal(torch.cat(plain, 1), torch.cat([y for _, (y, _) in zip(range(6), generate_step(ids, gm))], 1))


def test_adapters_that_are_refused():
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ok = adapters_for(cfg, 8, 1)
    with pytest.raises(ValueError):
        gm.apply_loras([ok], [])
    with pytest.raises(NotImplementedError):
        gm.apply_loras([adapters_for(cfg, 65, 1)], [1.0])
    with pytest.raises(NotImplementedError):
        gm.apply_loras([ok], [1.0], keys=("self_attn.o_proj",))
    bad = dict(ok)
    bad["model.layers.0.self_attn.q_proj.lora_b"] = bad["model.layers.0.self_attn.q_proj.lora_b"][:, :-8]
    with pytest.raises(ValueError):
        gm.apply_loras([bad], [1.0])
    cache = gm.make_cache(2)
    with pytest.raises(ValueError):
        gm.bind_adapters(cache, [0, 0])                              # none are held
    gm.apply_loras([ok], [1.0])
    for rows in ([0], [0, 1], [0, -2], [0, 0, 0]):
        with pytest.raises(ValueError):
            gm.bind_adapters(cache, rows)
    with pytest.raises(RuntimeError):
        gm.apply_lora(ok, 1.0)
    gm.apply_loras([], [])
    gm.apply_lora(ok, 1.0)
    with pytest.raises(RuntimeError):
        gm.apply_loras([ok], [1.0])
    f32 = make_pair("tiny-llama", dtype="float32")[2]
    with pytest.raises(NotImplementedError):
        f32.apply_loras([ok], [1.0])


def test_adapters_on_a_tensor_parallel_shard_keep_their_output_columns():
    """A rank holds A whole and the columns of B that its rows of the projections have."""
    from mlx_parallm_b200 import synth, tp
    from mlx_parallm_b200.utils import _get_classes
    cfg = synth.get_config("small-llama", num_key_value_heads=2)
    w = synth.random_weights(cfg, seed=1234, dtype="float16")
    Model, Args = _get_classes(cfg)
    keys = ("self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj")
    sets = [adapters_for(cfg, 8, 1, keys), adapters_for(cfg, 20, 2, keys)]
    full = Model(Args.from_dict(cfg)).load_weights(w, device="cuda").apply_loras(sets, [1.0, 2.0], keys)
    for rank in range(2):
        part = Model(Args.from_dict(cfg)).load_weights(tp.shard_weights(w, cfg, rank, 2), device="cuda")
        part.set_tensor_parallel(rank, 2, None)
        part.apply_loras(sets, [1.0, 2.0], keys)
        for lf, lp in zip(full.layers, part.layers):
            (af, bf, sf, cf), (ap, bp, sp, cp) = lf.self_attn.loras, lp.self_attn.loras
            assert torch.equal(af, ap) and torch.equal(sf, sp)
            at = loc = 0
            for (_, width), (first, n) in zip(cf, cp):
                assert n == width // 2 and first == loc             # (the shard's fused block is its q, k and v rows)
                assert torch.equal(bp[:, loc:loc + n], bf[:, at + rank * n:at + (rank + 1) * n])
                at, loc = at + width, loc + n
        with pytest.raises(NotImplementedError):
            part.score(torch.zeros((1, 4), dtype=torch.int64))
        with pytest.raises(NotImplementedError):
            next(generate_step(torch.zeros((1, 4), dtype=torch.int64), part, logprobs=1))


# ---------------------------------------------------------------------------------------------------------------- shared prompts
@pytest.mark.parametrize("by_groups", [True, False])
@pytest.mark.parametrize("name,dtype", MODELS)
def test_rows_that_share_prompts(name, dtype, by_groups, request):
    """Steps, a portion and more steps of rows behind shared prompts against the oracle's whole texts."""
    if by_groups:
        request.getfixturevalue("groups_always")
    cfg, om, gm = make_pair(name, dtype=dtype)
    heads, tails = prompts_for(cfg, 2, 41), prompts_for(cfg, 6, 14, seed=9)
    groups = [[0, 3, 5], [1, 4]]                                    # row 2 is by itself
    texts = np.concatenate([heads[[0, 1, 1, 0, 1, 0]], tails], 1)
    exp = om.forward(texts, om.make_cache(6))
    cache = gm.make_paged_cache(6, 64, page=16, pages=2 * 3 + 6 * 2 + 3)
    book = cache[0].book
    head_logits = gm.share_prompt(cache, torch.from_numpy(heads), groups)
    assert head_logits.shape == (2, cfg["vocab_size"]) and rel_err(head_logits.cpu(), exp[[0, 1], 40]) < LOGIT_TOL
    assert book.by_groups == by_groups and book.lengths.tolist() == [41, 41, 0, 41, 41, 41]
    assert len(book.free) == book.pages - (2 * 2 + 5)               # two whole pages of each prompt, and everybody's third
    gm.share_prompt(cache, torch.from_numpy(heads[1:]), [[2]])
    t = torch.from_numpy(tails)
    got = [gm(t[:, :1], cache=cache), gm(t[:, 1:2], cache=cache), gm(t[:, 2:9], cache=cache)] + [gm(t[:, i:i + 1], cache=cache) for i in range(9, 14)]
    err = rel_err(torch.cat(got, 1).cpu().numpy(), exp[:, 41:])
    assert err < LOGIT_TOL, err
    gm.release_rows(cache, [0, 4])
    more = gm(t[:, :1], cache=cache)
    left = [1, 2, 3, 5]
    again = om.forward(np.concatenate([texts, tails[:, :1]], 1)[left], om.make_cache(4))[:, -1]
    assert rel_err(more[left, 0].cpu(), again) < LOGIT_TOL
    gm.release_rows(cache, [1, 2, 3, 5])
    assert len(book.free) == book.pages and not book.held
    for c in cache:
        c.reset()
    assert not book.by_groups and book.groups == []
    gm(torch.from_numpy(texts), cache=gm.make_paged_cache(6, 64, page=16))
    assert rel_err(gm(torch.from_numpy(texts[:, :20]), cache=cache).cpu(), exp[:, :20]) < LOGIT_TOL


def test_greedy_generation_behind_a_shared_prompt(monkeypatch, groups_always):
    """The captured step over groups gives what the step over pages without them gives, token for token but for near-ties."""
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    head = prompts_for(cfg, 1, 70)
    tails = torch.from_numpy(prompts_for(cfg, 5, 3, seed=2))
    runs = []
    for limit in (0, 1 << 60):
        monkeypatch.setattr(paged, "SHARED_BYTES", limit)
        cache = gm.make_paged_cache(5, 160, page=16)
        gm.share_prompt(cache, torch.from_numpy(head), [[0, 1, 2, 3, 4]])
        out = [(y[:, 0], lp) for _, (y, _, lp) in zip(range(40), generate_step(tails, gm, cache=cache, logprobs=2))]
        runs.append(out)
        assert cache[0].book.by_groups == (limit == 0)
    for r in range(5):
        for (a, la), (b, lb) in zip(*runs):
            if a[r] != b[r]:                                        # followed up to its first near-tie
                assert float(la.top_logprobs[r, 0] - la.top_logprobs[r, 1]) < 0.05
                break
            assert abs(float(la.logprob[r] - lb.logprob[r])) < 0.05


def test_a_prompt_of_rows_whose_adapter_is_gone():
    """Rows that were bound to an adapter that is no longer held have none, and share a prompt like any others."""
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 2, 20))
    gm.apply_loras([adapters_for(cfg, 8, 1), adapters_for(cfg, 8, 2)], [1.0, 1.0])
    cache = gm.make_paged_cache(4, 64, page=16)
    gm.bind_adapters(cache, [1, 0, 1, 0])
    gm.apply_loras([adapters_for(cfg, 8, 1)], [1.0])
    got = gm.share_prompt(cache, ids, [[0, 2], [1, 3]])
    plain = gm(ids, last_only=True)[:, -1]
    assert torch.equal(got[0], plain[0]) and not torch.equal(got[1], plain[1])
    gm.apply_loras([], [])
    cache = gm.make_paged_cache(4, 64, page=16)
    cache[0].adapter_rows, cache[0].adapter_index = [1, 0, 1, 0], torch.tensor([1, 0, 1, 0], dtype=torch.int32, device="cuda")
    assert torch.equal(gm.share_prompt(cache, ids, [[0, 2], [1, 3]]), plain)


def test_a_pool_that_is_too_small_for_a_shared_prompt():
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 1, 40))
    cache = gm.make_paged_cache(4, 64, page=16, pages=4)
    book = cache[0].book
    with pytest.raises(paged.PagesExhausted):
        gm.share_prompt(cache, ids, [[0, 1, 2, 3]])                  # 2 whole pages, and 4 of the rows
    assert len(book.free) == 4 and book.lengths.tolist() == [0] * 4 and (book.table == -1).all() and not book.held
    gm.share_prompt(cache, ids, [[0, 2]])
    with pytest.raises(paged.PagesExhausted):
        gm.share_prompt(cache, ids, [[1]])
    with pytest.raises(paged.PagesExhausted):
        gm.share_prompt(gm.make_paged_cache(2, 32, page=16), ids, [[0, 1]])
    assert book.lengths.tolist() == [40, 0, 40, 0] and len(book.free) == 0
    gm.release_rows(cache, [0])
    assert len(book.free) == 1


def test_a_prompt_finds_the_pages_that_a_failed_step_left_to_its_rows():
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 1, 40))
    cache = gm.make_paged_cache(2, 64, page=16, pages=4)             # the prompt's three and the copy of its last one
    book = cache[0].book
    book.room_for([40, 10])                                          # what a step takes before its kernels run
    gm.share_prompt(cache, ids, [[0, 1]])
    assert book.lengths.tolist() == [40, 40] and not book.free and len(set(book.owned[0]) | set(book.owned[1])) == 4
    for c in cache:
        c.reset()
    assert sorted(book.free) == [0, 1, 2, 3]


def test_prompts_that_cannot_be_shared():
    cfg, om, gm = make_pair("tiny-llama", dtype="float16")
    ids = torch.from_numpy(prompts_for(cfg, 2, 20))
    new = lambda **kw: gm.make_paged_cache(4, 64, page=16, **kw)
    for groups in ([[0]], [[0], []], [[0], [0]], [[0, 0], [1]], [[0], [4]], [[0], [-1]]):
        with pytest.raises(ValueError):
            gm.share_prompt(new(), ids, groups)
    with pytest.raises(ValueError):
        gm.share_prompt(new(), ids[:, :0], [[0], [1]])
    for kw in (dict(window=16, first=2), dict(keep=20)):
        with pytest.raises(NotImplementedError):
            gm.share_prompt(new(**kw), ids, [[0], [1]])
    with pytest.raises(NotImplementedError):
        gm.share_prompt(gm.make_cache(4), ids, [[0], [1]])
    cache = new()
    gm.share_prompt(cache, ids, [[0], [1]])
    with pytest.raises(ValueError):
        gm.share_prompt(cache, ids, [[1], [2]])                      # row 1 holds a prompt
    gm.release_rows(cache, [3])
    with pytest.raises(ValueError):
        gm.share_prompt(cache, ids, [[3], [2]])                      # given back
    gm.apply_loras([adapters_for(cfg, 8, 1)], [1.0])
    cache = new()
    gm.bind_adapters(cache, [0, 0, -1, -1])
    with pytest.raises(ValueError):
        gm.share_prompt(cache, ids, [[0, 2], [1]])


# ---------------------------------------------------------------------------------------------------------------- together
@pytest.mark.parametrize("name,dtype,prompt_tokens", [("small-llama", "float16", 90), ("tiny-qwen3", "bfloat16", 33), ("tiny-llama", "float16", 1)])
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_choices_under_adapters_and_their_scores(name, dtype, prompt_tokens, temp, groups_always):
    """Answers to one prompt under several adapters: shared pages, per-row updates and log probabilities in one captured step; scored anew as whole texts."""
    cfg, om, gm = make_pair(name, dtype=dtype)
    gm.apply_loras([adapters_for(cfg, 8, 1), adapters_for(cfg, 20, 2)], [1.0, 2.0])
    prompt = " ".join(f"w{i}" for i in prompts_for(cfg, 1, prompt_tokens)[0])
    tok = FakeTokenizer(cfg["vocab_size"], eos_token_id=0)
    which = [0, 1, -1, 0, 0, 1, -1]
    got = generate_choices(gm, tok, prompt, n=7, max_tokens=17, temp=temp, logprobs=3, adapters=which, page=16)
    assert len(got) == 7
    ids = tok.encode(prompt)
    for c, w in zip(got, which):
        assert c.finish_reason in ("stop", "length") and len(c.tokens) == len(c.logprobs) == len(c.top_logprobs) <= 17
        assert c.text == tok.decode(c.tokens) and (c.finish_reason == "stop" or len(c.tokens) == 17)
        text = torch.tensor([ids + c.tokens])
        s = gm.score(text, adapters=[w])
        cache = gm.make_cache(1)
        gm.bind_adapters(cache, [w])
        tol = 2 * LOGIT_TOL * float(gm(text, cache=cache).abs().max())
        if c.tokens:
            assert np.abs(np.array(c.logprobs) - s.logprob[0, len(ids) - 1:-1].cpu().numpy()).max() < tol
        if temp == 0:
            assert all(max(t.values()) <= lp + 1e-6 and len(t) == 3 for t, lp in zip(c.top_logprobs, c.logprobs))
    if temp == 0:                                                    # rows under one adapter say the same but for near-ties
        for a, b in ((0, 3), (3, 4), (1, 5), (2, 6)):
            for x, y, t in zip(got[a].tokens, got[b].tokens, got[a].top_logprobs):
                v = sorted(t.values())
                if v[-1] - v[-2] < 0.05:
                    break
                assert x == y


def test_choices_end_one_by_one():
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    prompt = " ".join(f"w{i}" for i in prompts_for(cfg, 1, 40)[0])
    free = generate_choices(gm, FakeTokenizer(cfg["vocab_size"], eos_token_id=cfg["vocab_size"] + 5), prompt, n=4, max_tokens=20, temp=1.5, page=16)
    assert all(c.finish_reason == "length" and len(c.tokens) == 20 and c.logprobs is None and c.top_logprobs is None for c in free)
    eos = free[0].tokens[5]
    tok = FakeTokenizer(cfg["vocab_size"], eos_token_id=eos)
    for c in generate_choices(gm, tok, prompt, n=4, max_tokens=20, temp=1.5, page=16, logprobs=0):
        assert eos not in c.tokens and (c.finish_reason == "stop" or len(c.tokens) == 20)
    assert [c.tokens for c in generate_choices(gm, tok, prompt, n=2, max_tokens=0)] == [[], []]
    for bad in (dict(n=0), dict(max_tokens=-1), dict(n=2, adapters=[0]), dict(n=1, adapters=[0]), dict(page=24)):
        with pytest.raises(ValueError):
            generate_choices(gm, tok, prompt, **bad)
    with pytest.raises(ValueError):
        generate_choices(gm, tok, "")


def test_score_text():
    cfg, om, gm = make_pair("small-llama", dtype="float16")
    tok = FakeTokenizer(cfg["vocab_size"], eos_token_id=0)
    texts = [" ".join(f"w{i}" for i in prompts_for(cfg, 1, n, seed=n)[0]) for n in (12, 1, 40)] + [""]
    out = score_text(gm, tok, texts, top=2)
    for text, o in zip(texts, out):
        ids = tok.encode(text)
        assert o["tokens"] == ids and len(o["token_logprobs"]) == len(ids) == len(o["top_logprobs"])
        if len(ids) < 2:
            assert math.isnan(o["perplexity"])
            continue
        lp = torch.log_softmax(gm(torch.tensor([ids]))[0].double(), -1)
        want = [float(lp[i, t]) for i, t in enumerate(ids[1:])]
        assert o["token_logprobs"][0] is None and np.abs(np.array(o["token_logprobs"][1:]) - want).max() < 0.05
        assert abs(math.log(o["perplexity"]) + np.mean(want)) < 0.05
        assert all(len(t) == 2 for t in o["top_logprobs"][1:])

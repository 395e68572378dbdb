"""b200p_token_logprobs against its definition in 64 bits: sizes, types, strides, ties, masks, special values, streams and graphs."""
import math

import pytest
import torch

from mlx_parallm_b200 import ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def reference(logits, tokens, top, temperature):
    x = logits.double().cpu()
    lp = torch.log_softmax(x / temperature, -1)
    entropy = torch.special.entr(lp.exp()).sum(-1)
    t = tokens.cpu().tolist()
    given = torch.stack([lp.new_zeros(()) if v < 0 else lp[i, v] if v < x.shape[1] else lp.new_tensor(math.nan) for i, v in enumerate(t)])
    order = torch.where(x.isnan(), -math.inf, x)
    ids = torch.sort(order, dim=-1, descending=True, stable=True).indices[:, :top]
    return given, entropy, ids, lp.gather(1, ids), lp


def tolerance(V, value):
    """A thread adds up to V / 512 weights one after the other, then come some 12 levels, each add half a step of 2^-23; the exponent's argument carries
    three roundings, which the weights scale by their share (u c e^-u c sums to no more than some 30 of the total), 2^x two steps.  So log s and t / s are off
    by less than (V / 512 + 128) 2^-24, and a log probability besides by 3 roundings of its own size."""
    return (V / 512 + 128) * 2.0 ** -24 * (2.0 + value.abs())


def same(got, want, V):
    got = got.double().cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
    fine = want.isfinite()
    assert (got[fine] - want[fine]).abs().le(tolerance(V, want[fine])).all(), float((got[fine] - want[fine]).abs().max())


def check(logits, tokens, top=0, temperature=1.0, **kw):
    r = ops.token_logprobs(logits, tokens, top=top, temperature=temperature, **kw)
    given, entropy, ids, alt, _ = reference(logits, tokens, top, temperature)
    V = logits.shape[1]
    same(r.logprob, given, V)
    same(r.entropy, entropy, V)
    assert r.top_ids.shape == (logits.shape[0], top) and r.top_ids.dtype is torch.int32
    assert torch.equal(r.top_ids.long().cpu(), ids)
    same(r.top_logprobs, alt, V)
    return r


def make(M, V, dtype, seed=0, spread=2.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((M, V), generator=g, device="cuda") * spread
    tokens = torch.randint(0, V, (M,), generator=g, device="cuda", dtype=torch.int32)
    return x.to(DT[dtype]), tokens


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 5, 8, 31, 300, 513, 4097, 32000, 50257])
@pytest.mark.parametrize("M", [1, 3, 33])
def test_sizes(M, V, dtype):
    x, t = make(M, V, dtype, seed=V + M)
    for top in sorted({0, 1, min(20, V), min(32, V)}):
        check(x, t, top)


@pytest.mark.parametrize("M", [1, 18, 19, 37, 38, 74, 75, 148, 149, 296, 297, 700])
def test_rows_at_the_borders_of_the_clusters(M):
    x, t = make(M, 6007, "f32", seed=M)
    check(x, t, 7)


def test_the_largest_vocabulary_and_tokens_at_its_ends():
    x, t = make(5, 151936, "f32")
    t[0], t[1], t[2], t[3] = 0, 151935, -1, 151936
    check(x, t, 20)
    t[:] = torch.tensor([-100, 2 ** 31 - 1, -2 ** 31, 7, 8], dtype=torch.int32)
    check(x, t, 0)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("offset", [0, 1, 2, 3, 5, 7])
def test_slices_of_wider_rows(dtype, offset):
    x, t = make(9, 1033, dtype)
    for V in (1, 3, 7, 9, 1000, 1020):
        check(x[:, offset:offset + V], t.clamp(max=V - 1), min(V, 5))
    check(x[2:3, offset:], t[:1].clamp(max=1000), 5)


@pytest.mark.parametrize("temperature", [1e-3, 0.1, 0.7, 1.9, 50.0])
def test_temperature(temperature):
    x, t = make(12, 3001, "f32")
    r = ops.token_logprobs(x, t, top=20, temperature=temperature)
    given, entropy, ids, alt, lp = reference(x, t, 20, temperature)
    assert torch.equal(r.top_ids.long().cpu(), ids)
    for got, want in ((r.logprob, given), (r.entropy, entropy), (r.top_logprobs, alt)):
        same(got, want, 3001)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 400])
def test_ties(M, dtype):
    V = 5003
    x, t = make(M, V, dtype)
    check(torch.round(x), t, 20)                                   # a few hundred of each
    check(torch.round(x / 8), t, 32)                               # some values, thousands of each
    check(torch.zeros_like(x), t, 32)
    check(torch.full_like(x, torch.finfo(DT[dtype]).min), t, 5)    # every logit the type's lowest
    signed = torch.zeros_like(x)
    signed[:, ::2] = -0.0
    check(signed, t, 9)
    up = torch.arange(V, device="cuda").expand(M, V).div(64).to(DT[dtype])
    check(up, t, 20)
    check(up.flip(1), t, 20)
    two = torch.full_like(x, -3.0)                                 # the second-best is everywhere
    two[:, V // 2] = 1.0
    check(two, t, 3)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("M", [1, 40, 400])
@pytest.mark.parametrize("left", [0, 1, 2, 7, 19, 20, 21, 600])
def test_masked_rows(M, left, dtype):
    V = 4001
    x, t = make(M, V, dtype)
    keep = torch.zeros((M, V), dtype=torch.bool, device="cuda")
    if left:
        keep.scatter_(1, torch.rand((M, V), device="cuda").argsort(1)[:, :left], True)
    check(x.masked_fill(~keep, -math.inf), t, 20)
    low = x.masked_fill(~keep, torch.finfo(DT[dtype]).min)
    check(low, t, 20)


@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_special_values_stay_in_their_row(value):
    x, t = make(6, 3000, "f32")
    x[1, 17], x[3, 2999], x[4, :] = value, value, value
    r = check(x, t, 10)
    assert r.entropy.cpu().isnan().tolist() == [False, True, False, True, True, False]
    x[3, 5] = -math.inf
    check(x, t, 10)


def test_one_certain_token():
    x = torch.full((3, 2048), -1e9, device="cuda")
    x[:, 77] = 1e9
    t = torch.tensor([77, 78, -1], dtype=torch.int32, device="cuda")
    r = ops.token_logprobs(x, t, top=2)
    assert r.logprob.tolist() == [0.0, -2e9, 0.0] and r.entropy.tolist() == [0.0] * 3
    assert r.top_ids.tolist() == [[77, 0]] * 3 and r.top_logprobs.tolist() == [[0.0, -2e9]] * 3


def test_without_tokens_and_into_given_outputs():
    x, t = make(7, 999, "f32")
    r = ops.token_logprobs(x, top=3)
    assert r.logprob is None
    full = check(x, t, 3)
    assert torch.equal(r.entropy, full.entropy) and torch.equal(r.top_ids, full.top_ids)
    out = ops.TokenLogprobs(*(torch.full_like(v, 5) for v in full))
    assert ops.token_logprobs(x, t, top=3, out=out) is out
    for a, b in zip(out, full):
        assert torch.equal(a, b)
    empty = ops.token_logprobs(x[:0], t[:0], top=3)
    assert empty.entropy.numel() == 0 and empty.top_ids.shape == (0, 3)


def test_same_bits_every_time():
    x, t = make(50, 32000, "f32")
    first = ops.token_logprobs(x, t, top=20)
    for _ in range(5):
        for a, b in zip(ops.token_logprobs(x, t, top=20), first):
            assert torch.equal(a, b)


def test_graph_and_streams():
    x, t = make(20, 9000, "f32")
    out = ops.token_logprobs(x, t, top=5)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.token_logprobs(x, t, top=5, out=out)
    y, u = make(20, 9000, "f32", seed=9)
    x.copy_(y), t.copy_(u)
    g.replay()
    other, side = make(20, 9000, "f32", seed=10), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        r = ops.token_logprobs(*other, top=5)
    torch.cuda.synchronize()
    for got, (a, b) in ((out, (y, u)), (r, other)):
        given, entropy, ids, alt, _ = reference(a, b, 5, 1.0)
        same(got.logprob, given, 9000), same(got.entropy, entropy, 9000), same(got.top_logprobs, alt, 9000)
        assert torch.equal(got.top_ids.long().cpu(), ids)


def test_rows_farther_apart_than_32_bits_reach():
    base = torch.empty((2 ** 31 + 5000,), dtype=torch.bfloat16, device="cuda")
    x = base.as_strided((2, 4001), (2 ** 31 + 8, 1), 3)
    y, t = make(2, 4001, "bf16")
    x.copy_(y)
    check(x, t, 20)


def test_refusals():
    x, t = make(4, 100, "f32")
    for bad in (dict(top=33), dict(top=-1), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(temperature=math.inf)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.token_logprobs(x, t, **bad)
    with pytest.raises((ValueError, RuntimeError)):
        ops.token_logprobs(x[:, :3], t, top=4)
    for logits, tokens in ((x.double(), t), (x, t.long()), (x, t[:3]), (x.t(), t), (x[0], t), (x, t.cpu()), (x.cpu(), t), (x[:, :0], t),
                           (x[:1].expand(4, 100), t)):
        with pytest.raises((ValueError, TypeError, RuntimeError)):
            ops.token_logprobs(logits, tokens)
    full = ops.token_logprobs(x, t, top=2)
    for bad in (full._replace(logprob=None), full._replace(entropy=full.entropy[:3]), full._replace(top_ids=full.top_ids.long())):
        with pytest.raises(ValueError):
            ops.token_logprobs(x, t, top=2, out=bad)


@pytest.mark.parametrize("temperature", [1e-30, 1e-20, 1e20, 1e27])
@pytest.mark.parametrize("V", [10, 1000, 4097, 32001])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_the_ends_of_the_temperatures(dtype, V, temperature):
    """What is masked by minus infinity weighs nothing at any temperature (by the type's lowest value what that leaves it), in rows that fill a thread's loads and
    in rows that do not."""
    for mask in (None, -math.inf, torch.finfo(DT[dtype]).min if temperature > 1 else None):      # (a lowest value over 1e-20 is no fp32 number)
        x, t = make(6, V, dtype, seed=V)
        if mask is not None:
            x[:, 3:V - 4] = mask
            t[0] = V // 2
        check(x, t, min(5, V), temperature)

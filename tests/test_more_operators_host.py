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

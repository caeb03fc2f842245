"""CPU: the sampler's definition on small rows, and what yapd_sample_tokens refuses (before any GPU call)."""

import math

import numpy as np
import pytest

from oracle import sample as OS
from yapd_amd import kernels

LN = [math.log(v) for v in (0.1, 0.4, 0.3, 0.2)]  # tokens in order: 1, 2, 3, 0


@pytest.mark.parametrize("u,T,k,p,m,want", [
    (0.0, 1, 0, 1.0, 0.0, 1), (0.39, 1, 0, 1.0, 0.0, 1), (0.41, 1, 0, 1.0, 0.0, 2), (0.71, 1, 0, 1.0, 0.0, 3),
    (0.95, 1, 0, 1.0, 0.0, 0), (0.95, 1, 2, 1.0, 0.0, 2), (0.56, 1, 2, 1.0, 0.0, 1), (0.58, 1, 2, 1.0, 0.0, 2),
    (0.99, 1, 0, 0.39, 0.0, 1), (0.99, 1, 0, 0.41, 0.0, 2), (0.99, 1, 0, 0.69, 0.0, 2), (0.99, 1, 0, 0.71, 0.0, 3),
    (0.99, 1, 2, 0.58, 0.0, 2), (0.99, 1, 2, 0.56, 0.0, 1),   # top-p of what top-k keeps
    (0.99, 1, 0, 1.0, 0.74, 2), (0.99, 1, 0, 1.0, 0.76, 1), (0.99, 1, 0, 0.71, 0.74, 2),
    (0.5, 0, 0, 1.0, 0.0, 1), (0.99, 1e9, 0, 1.0, 0.0, 0), (0.26, 1e9, 0, 1.0, 0.0, 2), (2.0, 1, 3, 1.0, 0.0, 3),
])
def test_definition(u, T, k, p, m, want):
    token, lp, _ = OS.sample_row(np.array(LN), u, T, k, p, m)
    assert token == want


def test_ties_and_masked_tokens():
    x = np.array([-np.inf, 2.0, 2.0, -np.inf, 2.0])
    assert [OS.sample_row(x, u, 1.0, 0, 1.0, 0.0)[0] for u in (0.0, 0.34, 0.67, 5.0)] == [1, 2, 4, 4]
    assert OS.sample_row(x, 0.99, 1.0, 2, 1.0, 0.0)[0] == 2
    assert OS.sample_row(np.full(3, -np.inf), 0.5, 1.0, 0, 1.0, 0.0)[0] == -1
    assert OS.sample_row(np.array([0.0, np.nan]), 0.5, 0.0, 0, 1.0, 0.0)[0] == -1


P = 4096
CALL = dict(logits=P, wide=0, seq=50, pos=0, rows=3, bl=1, vocab=50, u=P, t=None, t_all=1.0, k=None, k_all=0, p=None, p_all=1.0,
            m=None, m_all=0.0, token=P, logprob=P, stream=None)


@pytest.mark.parametrize("over,msg", [
    (dict(rows=-1), b"rows"), (dict(rows=1 << 22), b"2^22"), (dict(vocab=0), b"vocab"), (dict(vocab=(1 << 24) + 1), b"vocab"),
    (dict(t_all=-0.5), b"temperature"), (dict(t_all=math.nan), b"temperature"), (dict(p_all=math.nan), b"top_p"),
    (dict(m_all=math.nan), b"min_p"), (dict(logits=None), b"NULL"), (dict(u=None), b"NULL"), (dict(token=None), b"NULL"),
    (dict(logprob=None), b"NULL"), (dict(logits=P + 1), b"misaligned"), (dict(logits=P + 2, wide=1), b"misaligned"),
])
def test_refusals(over, msg):
    lib = kernels.load_library()
    assert lib.yapd_sample_tokens(*dict(CALL, **over).values()) == 1
    assert msg in lib.yapd_last_error()


def test_nothing_to_draw():
    assert kernels.load_library().yapd_sample_tokens(*dict(CALL, rows=0, logits=None).values()) == 0

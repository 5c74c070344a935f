"""Serving operators where they are easily wrong: weights far below the largest, values that are not finite, rows of next to equal logits,
very long rows, outputs at odd addresses. Against the definitions in 64 bits."""
import math

import pytest
import torch

import serving_cases as S
from test_gpu_serving import BF16, F16, F32, check_sample, cumulative, ops, pool, put, rnd  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- weights far below the largest ----------------------------------------------------------------------------------------

def one_ahead(n, at, gap, dtype, D=64):
    """q, k, v of one head, n keys: key `at` scores `gap`, all others 0 (scale 1). Its value is 0 in the first half of the dimensions,
    which show the others' share alone."""
    q, k = torch.zeros(n, 1, D, dtype=dtype, device="cuda"), torch.zeros(n, 1, D, dtype=dtype, device="cuda")
    q[:, 0, 3], k[at, 0, 3] = 1.0, gap
    v = rnd(7, n, 1, D, dtype=dtype).abs() + 1
    v[at, 0, :D // 2] = 0
    return q, k, v


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,batch", [(20000, 1), (4000, 500), (20001, 700)])
@pytest.mark.parametrize("gap", [12.0, 14.0, 16.0, 17.0, 18.0])
def test_paged_attention_of_weak_keys(ops, dtype, n, batch, gap):
    """What many keys far below one add up to, in front of it and behind it. (In a large batch few parts have the one key and many others.)"""
    for at in (0, n // 3):
        q, k, v = one_ahead(n, at, gap, dtype)
        k_pages, v_pages, table = pool([n], 16, 1, 64, dtype)
        put(k_pages, table, 0, 0, k), put(v_pages, table, 0, 0, v)
        got = ops.paged_attention(q[:1].expand(batch, 1, 64), k_pages, v_pages, table.expand(batch, -1),
                                  torch.full((batch,), n - 1, device="cuda"), 1.0)
        want, slack = S.attend(q[0], k[:, 0], v[:, 0], 1.0, weight_step=S.half_step(dtype) ** 2)
        # fp16 weights of less than 2^-18 of the largest: half of the smallest step, 2^-24, of numbers that go up to 2^15
        tiny = 2.0 ** -40 * v[:, 0].double().sum(0) if dtype is F16 else 0.0
        ok, why = S.within(got, want.expand(batch, 1, 64), slack + tiny, dtype)
        assert ok, (at, why)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("gap", [12.0, 14.0, 16.0, 18.0])
def test_packed_attention_of_weak_keys(ops, dtype, gap):
    n = 16001
    for at in (0, 700):
        q, k, v = one_ahead(n, at, gap, dtype)
        got = ops.packed_attention(q, k, v, cumulative([n]), 1.0)
        for r in (129, 699, 700, 2500, 8191, n - 1):
            want, slack = S.attend(q[r], k[:r + 1, 0], v[:r + 1, 0], 1.0, weight_step=S.half_step(dtype))
            # fp16 weights of less than 2^-21 of the largest: half of the smallest step, 2^-24, of numbers that go up to 2^7
            tiny = 2.0 ** -32 * v[:r + 1, 0].double().sum(0) if dtype is F16 else 0.0
            ok, why = S.within(got[r], want, slack + tiny, dtype)
            assert ok, (at, r, why)

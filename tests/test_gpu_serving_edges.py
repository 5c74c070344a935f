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


# ---- values that are not finite ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("n,D,page", [(150, 64, 16), (150, 128, 7), (4000, 64, 16), (4000, 128, 16), (1500, 256, 24)])
def test_paged_attention_of_values_that_are_not_finite(ops, dtype, n, D, page):
    """A value that is not finite makes its dimension so, of the heads that see it, and no other; infinities of both signs make NaN."""
    H, G = 6, 2
    k_pages, v_pages, table = pool([n, 40], page, G, D, dtype)
    k, v, q = rnd(1, n, G, D, dtype=dtype), rnd(2, n, G, D, dtype=dtype), rnd(3, 2, H, D, dtype=dtype)
    put(k_pages, table, 0, 0, k), put(v_pages, table, 0, 0, v)
    put(k_pages, table, 1, 0, k[:40]), put(v_pages, table, 1, 0, v[:40])
    pos = torch.tensor([n - 1, 39], device="cuda")
    want = ops.paged_attention(q, k_pages, v_pages, table, pos, 0.3)
    for t in (0, 17, n // 2, n - 1):
        w = v[t].clone()
        w[1, 5], w[1, 6], w[1, 7] = math.inf, -math.inf, math.nan
        put(v_pages, table, 0, t, w[None])
        got = ops.paged_attention(q, k_pages, v_pages, table, pos, 0.3)
        assert bool((got[0, 3:, 5] == math.inf).all()) and bool((got[0, 3:, 6] == -math.inf).all()) and bool(got[0, 3:, 7].isnan().all()), t
        got[0, 3:, 5:8] = want[0, 3:, 5:8]
        assert torch.equal(got, want), t
        put(v_pages, table, 0, t, v[t][None])
    w = v[10:12].clone()
    w[0, 0, 9], w[1, 0, 9] = math.inf, -math.inf
    put(v_pages, table, 0, 10, w)
    got = ops.paged_attention(q, k_pages, v_pages, table, pos, 0.3)
    assert bool(got[0, :3, 9].isnan().all())
    got[0, :3, 9] = want[0, :3, 9]
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype,gap", [(F16, 14.0), (F16, 30.0), (F16, 150.0), (BF16, 14.0), (BF16, 80.0), (F32, 14.0), (F32, 80.0)])
@pytest.mark.parametrize("n", [150, 4000])
def test_paged_attention_of_an_infinite_value_with_a_small_weight(ops, dtype, gap, n):
    """An infinite value that is seen is not lost and does not turn into NaN, as long as 32 bits hold its weight, in fp16 however small that is."""
    for at in (0, n // 2, n - 1):
        q, k, v = one_ahead(n, at, gap, dtype)
        for t in (1, n // 3, n - 2):
            w = v.clone()
            w[t, 0, 5] = -math.inf
            k_pages, v_pages, table = pool([n], 16, 1, 64, dtype)
            put(k_pages, table, 0, 0, k), put(v_pages, table, 0, 0, w)
            got = ops.paged_attention(q[:1], k_pages, v_pages, table, torch.tensor([n - 1], device="cuda"), 1.0)[0, 0]
            assert float(got[5]) == -math.inf and int(got.isfinite().sum()) == 63, (at, t)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 160])
@pytest.mark.parametrize("gap", [14.0, 30.0, 100.0])
def test_packed_attention_of_an_infinite_value_with_a_small_weight(ops, dtype, D, gap):
    n = 900
    for at in (0, 400):  # the key that has the weight, in front of the value and behind it
        q, k, v = one_ahead(n, at, gap, dtype, D)
        clean = ops.packed_attention(q, k, v, cumulative([n]), 1.0)
        for t in (3, 130, 300, 520):
            w = v.clone()
            w[t, 0, 5], w[t, 0, D - 1] = math.inf, math.nan
            got = ops.packed_attention(q, k, w, cumulative([n]), 1.0)
            assert bool((got[t:, 0, 5] == math.inf).all()) and bool(got[t:, 0, D - 1].isnan().all()), (at, t)
            got[t:, 0, 5], got[t:, 0, D - 1] = clean[t:, 0, 5], clean[t:, 0, D - 1]
            assert torch.equal(got, clean), (at, t)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 160])
def test_packed_attention_after_keys_that_weigh_nothing(ops, dtype, D):
    """Scores of -inf in a whole tile of keys, the first one, and scores far below 0 behind it."""
    n, H = 400, 2
    q, k, v = rnd(1, n, H, D, dtype=dtype).abs() + 1, rnd(2, n, H, D, dtype=dtype), rnd(3, n, H, D, dtype=dtype)
    k[:128, :, 0] = -math.inf
    k[128:, :, 1] = -300
    got = ops.packed_attention(q, k, v, cumulative([n]), 1.0)
    for r in (128, 129, 255, 256, 399):
        for h in range(H):
            want, slack = S.attend(q[r, h:h + 1], k[128:r + 1, h], v[128:r + 1, h], 1.0, weight_step=S.half_step(dtype))
            ok, why = S.within(got[r, h:h + 1], want, slack, dtype)
            assert ok, (r, h, why)


# ---- positions and addresses ------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("page,width", [(8176, (2 ** 31 - 16) // 8176), (49981, (2 ** 31 - 2) // 49981)])
def test_paged_attention_next_to_2_31_tokens(ops, page, width):
    """As many tokens as a table can have, all of one page: no position passes 32 bits, and nothing counts as refused."""
    k_pages, v_pages = torch.zeros(1, 1, page, 8, dtype=F16, device="cuda"), torch.ones(1, 1, page, 8, dtype=F16, device="cuda")
    table = torch.zeros(1, width, dtype=torch.int32, device="cuda")
    before = ops.paged_faults()
    got = ops.paged_attention(torch.ones(1, 1, 8, dtype=F16, device="cuda"), k_pages, v_pages, table,
                              torch.tensor([page * width - 1], device="cuda"), 1.0)
    # sums of 2^31 equal weights: 2^31 * 2^-24 would be the bound of a single running sum; parts of a 2^10th and their sum are off by 2^-3 at most
    assert ops.paged_faults() == before and float((got - 1).abs().max()) <= 2 ** -3


def test_paged_attention_behind_the_last_position(ops):
    """The largest position that there is: all tokens of the table are seen, and it is counted."""
    H, G, D, n = 2, 1, 64, 32
    k_pages, v_pages, table = pool([n], 16, G, D, F16)
    put(k_pages, table, 0, 0, rnd(1, n, G, D, dtype=F16)), put(v_pages, table, 0, 0, rnd(2, n, G, D, dtype=F16))
    q, before = rnd(3, 1, H, D, dtype=F16), ops.paged_faults()
    want = ops.paged_attention(q, k_pages, v_pages, table, torch.tensor([n - 1], device="cuda"), 0.125)
    assert ops.paged_faults() == before
    for p in (n, 2 ** 31, 2 ** 63 - 1):
        assert torch.equal(ops.paged_attention(q, k_pages, v_pages, table, torch.tensor([p], device="cuda"), 0.125), want), p
    assert ops.paged_faults() > before


def test_append_behind_the_last_position(ops):
    """Positions as large as there are: counted, not stored, and not taken for negative ones."""
    G, D = 2, 64
    k, v = rnd(1, 5, G, D, dtype=BF16), rnd(2, 5, G, D, dtype=BF16)
    k_pages, v_pages, table = pool([20, 20], 16, G, D, BF16)
    before = ops.paged_faults()
    _, k_out = ops.paged_append(None, k, v, k_pages, v_pages, table, torch.tensor([2 ** 63 - 1, 2 ** 63 - 2], device="cuda"),
                                cu_seqlens=cumulative([3, 2]), keys=True)
    assert torch.equal(k_out, k) and ops.paged_faults() - before == 5
    assert bool(k_pages.isnan().all()) and bool(v_pages.isnan().all())


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 72, 128, 200, 256])
def test_packed_attention_into_any_address(ops, dtype, D):
    """An output on any boundary holds the same bits, and rows of no sequence stay."""
    T, H, G = 300, 3, 1
    q, k, v = rnd(1, T, H, D, dtype=dtype), rnd(2, T, G, D, dtype=dtype), rnd(3, T, G, D, dtype=dtype)
    cu = cumulative([200, 90], first=4)
    want = ops.packed_attention(q, k, v, cu, 0.1)
    for at in (0, 16, 8, 3):
        room = torch.full((T * H * D + 16,), 7.0, dtype=dtype, device="cuda")
        out = room[at:at + T * H * D].view(T, H, D)
        assert ops.packed_attention(q, k, v, cu, 0.1, out=out) is out
        assert torch.equal(out[4:294], want[4:294]), at
        assert bool((out[:4] == 7).all()) and bool((out[294:] == 7).all()) and bool((room[:at] == 7).all()) and bool((room[at + T * H * D:] == 7).all())


# ---- sampling ------------------------------------------------------------------------------------------------------------------

NARROW = [{}, {"top_k": 3}, {"top_k": 700}, {"top_p": 0.7}, {"min_p": 0.5}, {"top_k": 900, "top_p": 0.5, "min_p": 0.9}]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("settings", NARROW, ids=str)
@pytest.mark.parametrize("unit", [1e-20, 1e-30, 1e-31, 3e-32, 1e-33, 1e-38])
def test_sample_tokens_of_next_to_equal_logits(ops, dtype, settings, unit):
    """Differences next to none: the entries weigh the same but keep their order."""
    logits, u = rnd(58, 6, 1500) * unit, torch.rand(6, device="cuda", generator=torch.Generator("cuda").manual_seed(10))
    check_sample(ops, logits.to(dtype), u, **settings)
    one = torch.zeros(6, 5003, device="cuda")
    one[:, 4000], one[3:, 17] = unit, -unit
    check_sample(ops, one.to(dtype), u, **settings)


def test_sample_tokens_of_many_small_weights(ops):
    """Entries 34 temperatures below the last one, which together make up 10^-7: a number that falls among them."""
    V = 2 ** 26
    logits = torch.zeros(1, V, device="cuda")
    logits[0, V - 1] = 34.0
    w = math.exp(-34.0)
    total = 1 + (V - 1) * w
    for part in (0.2, 0.9, 0.953, 0.9999, 1.0001, 2.0):
        u = torch.tensor([part * (V - 1) * w / total], device="cuda")
        at = float(u.double()) * total / w  # so many of them
        if not 1e-3 < at % 1 < 1 - 1e-3:
            continue
        assert int(ops.sample_tokens(logits, u)) == min(int(at), V - 1), part


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_sample_tokens_with_a_number_of_zero(ops, dtype):
    """The lowest index that is kept, however little it weighs."""
    V = 3001
    logits, u = rnd(59, 7, V).mul(2).to(dtype), torch.zeros(7, device="cuda")
    for b, below in enumerate((30, 44, 46, 60, 100, 700, 800)):
        logits[b, 0] = float(logits[b].float().max()) - below
    for settings in ({}, {"top_k": 50}, {"top_k": V - 1}, {"top_p": 0.9}, {"min_p": 0.1}, {"min_p": 1e-30}, {"top_k": V, "temperature": 2.0},
                     {"temperature": 0.5}):
        check_sample(ops, logits, u, **settings)


@pytest.mark.parametrize("number", [1e-9, 1e-12, 1e-19, 1e-21, 1e-30, 1e-38, 1e-44])
def test_sample_tokens_with_numbers_next_to_zero(ops, number):
    """Numbers that fall among entries of weights far below 32 bits."""
    V = 3001
    logits, u = rnd(62, 9, V).mul(2), torch.full((9,), number, device="cuda")
    for b in range(9):
        for i, below in enumerate((101, 95, 80, 60, 50, 47, 44, 30, 20)[b:]):
            logits[b, i] = float(logits[b].max()) - below
    for settings in ({}, {"top_k": V - 1}, {"min_p": 1e-25}):
        check_sample(ops, logits, u, **settings)


@pytest.mark.parametrize("dtype,low", [(BF16, -1e4), (F16, -1e4), (F32, -1e4), (F32, torch.finfo(F32).min), (F16, torch.finfo(F16).min)])
@pytest.mark.parametrize("spread", [0.5, 2.5])
def test_sample_tokens_with_finite_masks(ops, dtype, low, spread):
    """Ids that no token has, at a large negative number instead of -inf."""
    logits, u = rnd(60, 2, 151936).mul(spread), torch.rand(2, device="cuda", generator=torch.Generator("cuda").manual_seed(11))
    logits[:, 50000:50016] = low
    for settings in ({}, {"top_p": 0.5}, {"top_p": 0.9, "temperature": 0.8}, {"top_k": 50}, {"top_k": 3000, "min_p": 0.01}):
        check_sample(ops, logits.to(dtype), u, **settings)

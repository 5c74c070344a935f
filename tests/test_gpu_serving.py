"""Paged caches, attention over pages and packed prompts, sampling: against their definitions in 64 bits."""
import math

import pytest
import torch

import serving_cases as S

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops(cuda):
    from dejavu_b200 import _lib, ops

    yield ops
    assert _lib.load_serving().djv_serving_timeouts() == 0


def rnd(seed, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)


def cumulative(lengths, first=0):
    return torch.tensor([first] + lengths, device="cuda").cumsum(0).int()


def pool(lengths, page, G, D, dtype, seed=0, spare=2, layout="heads"):
    """Pages dealt out in random order for `lengths` tokens of each sequence: (k_pages, v_pages, table), filled with NaN."""
    need = [-(-n // page) for n in lengths]
    P = sum(need) + spare
    order = torch.randperm(P, generator=torch.Generator().manual_seed(seed)).int().tolist()
    table = torch.full((len(lengths), max(1, *need)), -7, dtype=torch.int32)
    for b, n in enumerate(need):
        table[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)

    def pages():
        if layout == "tokens":  # a page holds all heads of a token next to each other
            return torch.full((P, page, G, D), math.nan, dtype=dtype, device="cuda").transpose(1, 2)
        if layout == "gaps":
            return torch.full((P, G + 1, page + 1, D + 16), math.nan, dtype=dtype, device="cuda")[:, :G, :page, :D]
        return torch.full((P, G, page, D), math.nan, dtype=dtype, device="cuda")

    return pages(), pages(), table.cuda()


def put(pages, table, b, t, rows):
    """rows (n, G, D) become tokens t, t + 1, ... of sequence b."""
    page = pages.shape[2]
    at = torch.arange(t, t + rows.shape[0], device="cuda")
    pages[table[b, at // page].long(), :, at % page] = rows


# ---- append ---------------------------------------------------------------------------------------------------------------

def check_append(ops, q, k, v, pos, cu, lengths, page, freqs, amp, interleaved, layout="heads"):
    T, G, D = k.shape
    k_pages, v_pages, table = pool(lengths, page, G, D, k.dtype, layout=layout)
    q_out, k_out = ops.paged_append(q, k, v, k_pages, v_pages, table, pos, cu_seqlens=cu, freqs=freqs, amp=amp, interleaved=interleaved,
                                    keys=True)
    want_k, want_v = torch.full_like(k_pages, math.nan), torch.full_like(v_pages, math.nan)
    if cu is None:
        rows = [(b, b, p) for b, p in enumerate(pos.tolist())]
    else:
        c = cu.tolist()
        rows = [(r, b, p + r - c[b]) for b, p in enumerate(pos.tolist()) for r in range(c[b], c[b + 1])]
    rows = {r: (b, p) for r, b, p in rows if p >= 0}
    for r in range(T):
        if r not in rows:
            assert not bool(q_out[r].any()) and not bool(k_out[r].any())
            continue
        b, p = rows[r]
        for got, x in ((q_out[r], q[r]), (k_out[r], k[r])):
            y, slack = S.rotate(x, p, freqs, amp, interleaved)
            ok, why = S.within(got, y, slack, k.dtype)
            assert ok, (r, why)
        put(want_k, table, b, p, k_out[r][None])
        put(want_v, table, b, p, v[r][None])
    for got, want in ((k_pages, want_k), (v_pages, want_v)):  # what is not theirs is as it was
        assert torch.equal(got.nan_to_num(nan=77.0), want.nan_to_num(nan=77.0))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("H,G,D,half,interleaved,page", [(32, 8, 128, 64, False, 16), (4, 4, 64, 16, True, 24), (3, 1, 80, 20, False, 7),
                                                        (6, 2, 256, 128, True, 1), (2, 2, 32, 0, False, 64), (40, 40, 96, 48, False, 16),
                                                        (5, 5, 8, 4, False, 3), (5, 1, 16, 3, True, 5)])
def test_append_of_one_token_each(ops, dtype, H, G, D, half, interleaved, page):
    past = [0, 5, 31, 32, 100]
    qkv = rnd(1, 5, (H + 2 * G) * D, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, G * D, G * D), dim=1))
    freqs = (1000.0 ** (-torch.arange(half, device="cuda") / max(half, 1))).float() if half else None
    check_append(ops, q, k, v, torch.tensor(past, device="cuda"), None, [p + 1 for p in past], page, freqs, 1.25, interleaved)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lengths,past", [([1], [0]), ([7, 0, 33, 1], [0, 3, 15, 100]), ([0, 0, 5], [0, 0, 0]), ([70] * 3, [1, 2, 3]),
                                          ([1] * 40, list(range(40)))])
def test_append_of_prompts(ops, dtype, lengths, past):
    H, G, D, T = 6, 2, 64, sum(lengths)
    freqs = (10000.0 ** (-torch.arange(32, device="cuda") / 32)).float()
    q, k, v = rnd(2, T, H, D, dtype=dtype), rnd(3, T, G, D, dtype=dtype), rnd(4, T, G, D, dtype=dtype)
    check_append(ops, q, k, v, torch.tensor(past, device="cuda"), cumulative(lengths), [a + n for a, n in zip(past, lengths)], 16, freqs, 1.0,
                 False)


@pytest.mark.parametrize("form", ["odd_rows", "odd_address", "heads_last", "reversed_heads", "gaps", "tokens", "every_second"])
def test_append_takes_any_layout(ops, form):
    H, G, D, lengths = 4, 2, 64, [9, 5]
    T = sum(lengths)
    q, k, v = rnd(5, T, H, D, dtype=BF16), rnd(6, T, G, D, dtype=BF16), rnd(7, T, G, D, dtype=BF16)
    if form == "odd_rows":
        q, k, v = (torch.cat((x.flatten(1), x.flatten(1)[:, :3]), 1)[:, :x.shape[1] * D].unflatten(1, (-1, D)) for x in (q, k, v))
    if form == "odd_address":
        q, k, v = (torch.cat((x.flatten()[:1], x.flatten()))[1:].view(x.shape) for x in (q, k, v))
    if form == "heads_last":
        q, k, v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v))
    if form == "reversed_heads":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    if form == "every_second":
        q, k, v = (torch.stack((x, x), 1).flatten(0, 1)[::2] for x in (q, k, v))
    freqs = (100.0 ** (-torch.arange(32, device="cuda") / 32)).float()
    check_append(ops, q, k, v, torch.tensor([3, 0], device="cuda"), cumulative(lengths), [12, 5], 8, freqs, 1.0, False,
                 layout=form if form in ("gaps", "tokens") else "heads")


def test_append_rotates_far_positions_exactly(ops):
    """In 32 bits the angle of position 1000003 would be off by 2^-5."""
    H, G, D, page = 2, 1, 16, 1 << 16
    q, k, v = rnd(8, 2, H, D), rnd(9, 2, G, D), rnd(10, 2, G, D)
    freqs = torch.tensor([1.0, 0.7311, 0.1, 1e-3, 0.0, 3.1415927, 2.5, 1e-7], device="cuda")
    past = [1000003, 131071]
    check_append(ops, q, k, v, torch.tensor(past, device="cuda"), None, [p + 1 for p in past], page, freqs, 1.0, False)


def test_append_leaves_padding_alone(ops):
    """Rows in front of the first sequence and behind the last, rows at negative positions, a batch of nothing."""
    H, G, D = 4, 2, 64
    q, k, v = rnd(11, 12, H, D, dtype=F16), rnd(12, 12, G, D, dtype=F16), rnd(13, 12, G, D, dtype=F16)
    freqs = torch.rand(16, device="cuda")
    check_append(ops, q, k, v, torch.tensor([2, 0], device="cuda"), cumulative([4, 3], first=2), [6, 3], 4, freqs, 1.0, True)
    pos = torch.tensor([4, -1, 0, -5], device="cuda")
    check_append(ops, q[:4], k[:4], v[:4], pos, None, [5, 0, 1, 0], 4, freqs, 1.0, False)
    k_pages, v_pages, table = pool([1], 4, G, D, F16)
    a, b = ops.paged_append(q[:0], k[:0], v[:0], k_pages, v_pages, table, torch.zeros(1, dtype=torch.int64, device="cuda"),
                            cu_seqlens=cumulative([0]), keys=True)
    assert a.shape == (0, H, D) and b.shape == (0, G, D)


def test_append_counts_what_has_no_page(ops):
    """Entries that are no page, and positions behind the table, are not stored, only counted."""
    G, D, page = 2, 64, 4
    k, v = rnd(14, 5, G, D, dtype=BF16), rnd(15, 5, G, D, dtype=BF16)
    k_pages, v_pages, table = pool([8] * 5, page, G, D, BF16)
    table[1, 0], table[2, 1] = -1, k_pages.shape[0]
    before, good = ops.paged_faults(), table.clone()
    pos = torch.tensor([0, 0, 4, 8, 2 ** 40], device="cuda")
    q_out, k_out = ops.paged_append(None, k, v, k_pages, v_pages, table, pos, keys=True)
    assert q_out is None and torch.equal(k_out, k) and ops.paged_faults() - before == 4
    want = torch.full_like(k_pages, math.nan)
    put(want, good, 0, 0, k[:1])
    assert torch.equal(k_pages.nan_to_num(nan=77.0), want.nan_to_num(nan=77.0))


# ---- attention over pages ---------------------------------------------------------------------------------------------------

def check_decode(ops, dtype, H, G, D, page, lengths, scale=None, layout="heads", seed=20, amplify=1.0):
    k_pages, v_pages, table = pool(lengths, page, G, D, dtype, layout=layout)
    scale = D ** -0.5 if scale is None else scale
    q = rnd(seed, len(lengths), H, D, dtype=dtype)
    keys = [rnd(seed + 1 + b, 2, n, G, D, dtype=dtype) * amplify for b, n in enumerate(lengths)]
    for b, kv in enumerate(keys):
        if lengths[b]:
            put(k_pages, table, b, 0, kv[0])
            put(v_pages, table, b, 0, kv[1])
    pos = torch.tensor(lengths, device="cuda") - 1
    got = ops.paged_attention(q, k_pages, v_pages, table, pos, scale)
    assert got.shape == q.shape and got.dtype == dtype
    for b, kv in enumerate(keys):
        for g in range(G):
            heads = slice(g * (H // G), (g + 1) * (H // G))
            # (a kernel may hold weights as two terms of the cache's type: what is dropped is below half a step of the second)
            want, slack = S.attend(q[b, heads], kv[0][:, g], kv[1][:, g], scale, weight_step=S.half_step(dtype) ** 2)
            ok, why = S.within(got[b, heads], want, slack, dtype)
            assert ok, (b, g, lengths[b], why)
    again = ops.paged_attention(q, k_pages, v_pages, table, pos, scale)
    assert torch.equal(got, again)
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("H,G,D,page", [(32, 8, 128, 16), (12, 12, 64, 16), (8, 1, 128, 64), (40, 2, 80, 24), (6, 3, 256, 7), (5, 5, 32, 1),
                                        (64, 1, 96, 128), (3, 3, 8, 16), (17, 1, 136, 33)])
def test_paged_attention(ops, dtype, H, G, D, page):
    check_decode(ops, dtype, H, G, D, page, [1, 0, 2, 15, 16, 17, 63, 64, 65, 130, 333])


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lengths", [[5000], [1], [0], [1500, 3, 0, 2049], [257] * 30, [20000, 1, 1, 1, 40]])
def test_paged_attention_of_long_and_ragged_caches(ops, dtype, lengths):
    check_decode(ops, dtype, 8, 2, 64, 16, lengths)


def test_paged_attention_of_many_sequences(ops):
    lengths = [(37 * b) % 91 for b in range(1100)]
    check_decode(ops, F16, 2, 1, 32, 8, lengths)


@pytest.mark.parametrize("layout", ["gaps", "tokens"])
@pytest.mark.parametrize("dtype", [F16, F32])
def test_paged_attention_takes_any_layout(ops, layout, dtype):
    check_decode(ops, dtype, 8, 4, 64, 12, [100, 13, 700], layout=layout)


def test_paged_attention_takes_any_query_layout(ops):
    k_pages, v_pages, table = pool([50, 20], 16, 2, 64, BF16)
    put(k_pages, table, 0, 0, rnd(1, 50, 2, 64, dtype=BF16)), put(v_pages, table, 0, 0, rnd(2, 50, 2, 64, dtype=BF16))
    put(k_pages, table, 1, 0, rnd(3, 20, 2, 64, dtype=BF16)), put(v_pages, table, 1, 0, rnd(4, 20, 2, 64, dtype=BF16))
    pos, q = torch.tensor([49, 19], device="cuda"), rnd(5, 2, 4, 64, dtype=BF16)
    want = ops.paged_attention(q, k_pages, v_pages, table, pos, 0.1)
    wide = torch.full((2, 700), math.nan, dtype=BF16, device="cuda")
    for at in (0, 8, 3):
        wide[:, at:at + 256] = q.flatten(1)
        assert torch.equal(ops.paged_attention(wide[:, at:at + 256].unflatten(1, (4, 64)), k_pages, v_pages, table, pos, 0.1), want)
    assert torch.equal(ops.paged_attention(q.transpose(1, 2).contiguous().transpose(1, 2), k_pages, v_pages, table, pos, 0.1), want)
    wide_table = torch.full((2, 9), 10 ** 6, dtype=torch.int32, device="cuda")
    wide_table[:, :table.shape[1]] = table
    before = ops.paged_faults()
    assert torch.equal(ops.paged_attention(q, k_pages, v_pages, wide_table, pos, 0.1), want)
    assert torch.equal(ops.paged_attention(q, k_pages, v_pages, wide_table[:, :table.shape[1]], pos, 0.1), want)
    assert ops.paged_faults() == before


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.3, 4.0])
def test_paged_attention_scales(ops, dtype, scale):
    check_decode(ops, dtype, 4, 2, 64, 16, [1, 40, 300], scale=scale)


def test_paged_attention_of_large_scores(ops):
    """Scores of some thousands: one key has all the weight, and its value comes back."""
    H = G = 2
    D, n = 64, 1000
    k_pages, v_pages, table = pool([n], 16, G, D, BF16)
    k, v, q = rnd(1, n, G, D, dtype=BF16) * 30, rnd(2, n, G, D, dtype=BF16), rnd(3, 1, H, D, dtype=BF16) * 30
    put(k_pages, table, 0, 0, k), put(v_pages, table, 0, 0, v)
    got = ops.paged_attention(q, k_pages, v_pages, table, torch.tensor([n - 1], device="cuda"), 1.0)
    for h in range(H):
        score = k[:, h].double() @ q[0, h].double()
        top = score.topk(2).values
        assert float(top[0] - top[1]) > 20  # (the others weigh less than e^-20, below half a step of bf16)
        assert torch.equal(got[0, h], v[score.argmax(), h])


@pytest.mark.parametrize("dtype", [F16, F32])
def test_paged_attention_does_not_see_what_has_no_page(ops, dtype):
    """Entries that are no page hide their tokens; a sequence with no page at all gets zeros; shared pages are read by both."""
    H, G, D, page = 4, 2, 64, 16
    k_pages, v_pages, table = pool([48, 33, 20, 48], page, G, D, dtype)
    k, v = rnd(1, 48, G, D, dtype=dtype), rnd(2, 48, G, D, dtype=dtype)
    for b, n in enumerate((48, 33, 20, 48)):
        put(k_pages, table, b, 0, k[:n]), put(v_pages, table, b, 0, v[:n])
    q, before = rnd(3, 4, H, D, dtype=dtype), ops.paged_faults()
    table[1, 1], table[2, :2], table[3] = -1, 10 ** 9, table[0]
    got = ops.paged_attention(q, k_pages, v_pages, table, torch.tensor([47, 32, 19, 10 ** 12], device="cuda"), 0.125)
    assert ops.paged_faults() > before and not bool(got[2].any())
    keep = [list(range(48)), list(range(16)) + [32], [], list(range(48))]
    for b in (0, 1, 3):
        for h in range(H):
            want, slack = S.attend(q[b, h:h + 1], k[keep[b], h // 2], v[keep[b], h // 2], 0.125, S.half_step(dtype) ** 2)
            ok, why = S.within(got[b, h:h + 1], want, slack, dtype)
            assert ok, (b, h, why)


def test_paged_attention_far_into_a_large_pool(ops):
    """Pages whose offsets in the pool pass 32 bits."""
    G, D, page = 8, 256, 64
    P = 2 ** 31 // (G * D * page) + 40
    k_pages = torch.empty(P, G, page, D, dtype=BF16, device="cuda")
    v_pages = torch.empty_like(k_pages)
    table = torch.tensor([[P - 1, 3, P - 17]], dtype=torch.int32, device="cuda")
    k, v, q = rnd(1, 150, G, D, dtype=BF16), rnd(2, 150, G, D, dtype=BF16), rnd(3, 1, G, D, dtype=BF16)
    cu = cumulative([150])
    ops.paged_append(None, k, v, k_pages, v_pages, table, torch.zeros(1, dtype=torch.int64, device="cuda"), cu_seqlens=cu)
    assert torch.equal(k_pages[P - 17, :, 150 - 129], k[149])
    got = ops.paged_attention(q, k_pages, v_pages, table, torch.tensor([149], device="cuda"), 0.0625)
    for g in range(G):
        want, slack = S.attend(q[0, g:g + 1], k[:, g], v[:, g], 0.0625, S.half_step(BF16) ** 2)
        ok, why = S.within(got[0, g:g + 1], want, slack, BF16)
        assert ok, (g, why)


# ---- attention over packed prompts --------------------------------------------------------------------------------------------

def check_packed(ops, q, k, v, lengths, scale, first=0, weight_step=None, out=None):
    dtype, (T, H, D), G = q.dtype, q.shape, k.shape[1]
    got = ops.packed_attention(q, k, v, cumulative(lengths, first), scale, out=out)
    assert got.shape == q.shape and got.dtype == dtype
    # weights enter the second product in the inputs' type
    weight_step = S.half_step(dtype) if weight_step is None else weight_step
    start = first
    for n in lengths:
        for h in range(H):
            kk, vv = k[start:start + n, h // (H // G)].double(), v[start:start + n, h // (H // G)].double()
            qq = q[start:start + n, h].double()
            z = (qq @ kk.t()) * scale
            z.masked_fill_(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
            p = torch.softmax(z, 1)
            off = abs(scale) * (qq.abs() @ kk.abs().t()).amax(1, keepdim=True) * (D + 2) * 2.0 ** -24 if n else 0
            # as in serving_cases.attend
            slack = (p @ vv.abs()) * (2 * off + 2.0 ** -20 + n * 2.0 ** -24 + weight_step)
            ok, why = S.within(got[start:start + n, h], p @ vv, slack, dtype)
            assert ok, (start, n, h, why)
        start += n
    return got


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("H,G,D", [(8, 2, 128), (3, 3, 64), (4, 1, 80), (2, 1, 256), (5, 5, 32), (2, 2, 8), (6, 2, 96), (2, 2, 72), (1, 1, 200)])
def test_packed_attention(ops, dtype, H, G, D):
    lengths = [1, 127, 0, 128, 129, 2, 255, 256, 257, 0, 31, 400]
    T = sum(lengths)
    qkv = rnd(30, T, (H + 2 * G) * D, dtype=dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((H * D, G * D, G * D), dim=1))
    check_packed(ops, q, k, v, lengths, D ** -0.5)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("lengths", [[1], [2], [3000], [1] * 300, [513, 1023, 1, 1025], [64] * 9])
def test_packed_attention_lengths(ops, dtype, lengths):
    T, H, G, D = sum(lengths), 4, 2, 64
    check_packed(ops, rnd(31, T, H, D, dtype=dtype), rnd(32, T, G, D, dtype=dtype), rnd(33, T, G, D, dtype=dtype), lengths, 0.125)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("D", [64, 128, 144])
def test_packed_attention_is_not_touched_by_what_a_row_does_not_see(ops, dtype, D):
    """Infinities and NaN in later tokens and in other sequences, and in rows of none: earlier rows are what they are without."""
    lengths, H, G = [70, 200, 1, 130], 4, 2
    T = sum(lengths) + 9
    q, k, v = rnd(34, T, H, D, dtype=dtype), rnd(35, T, G, D, dtype=dtype), rnd(36, T, G, D, dtype=dtype)
    cu = cumulative(lengths, first=4)
    want = ops.packed_attention(q, k, v, cu, 0.1)
    assert bool(want.isfinite().all()) and not bool(want[:4].any()) and not bool(want[-5:].any())
    bad = (0, 1, 2, 3, 4 + 69, 4 + 70 + 150, 4 + 70 + 199, 4 + 270, 4 + 271 + 60, T - 5, T - 1)  # rows with something odd
    for i, r in enumerate(bad):
        for x in (k, v):
            x[r, :, i % D] = (math.nan, math.inf, -math.inf)[i % 3]
        v[r, :, (i + 1) % D] = (math.inf, math.nan, -math.inf)[i % 3]
    got = ops.packed_attention(q, k, v, cu, 0.1)
    start = 4
    for n in lengths:
        clean = min([r for r in bad if start <= r < start + n], default=start + n)
        assert torch.equal(got[start:clean], want[start:clean])
        for r in range(clean, start + n):
            assert not bool(got[r].isfinite().all())
        start += n
    assert not bool(got[:4].any()) and not bool(got[-5:].any())


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_attention_values_that_are_not_finite_reach_those_who_see_them(ops, dtype):
    """One infinite value: its dimension is infinite in every row that sees it, the others are as without it."""
    n, H, D = 150, 2, 64
    q, k, v = rnd(34, n, H, D, dtype=dtype), rnd(35, n, H, D, dtype=dtype), rnd(36, n, H, D, dtype=dtype)
    want = ops.packed_attention(q, k, v, cumulative([n]), 0.1)
    for r in (0, 60, 127, 128, 149):
        w = v.clone()
        w[r, 1, 5] = math.inf
        got = ops.packed_attention(q, k, w, cumulative([n]), 0.1)
        assert bool((got[r:, 1, 5] == math.inf).all())
        got[r:, 1, 5] = want[r:, 1, 5]
        assert torch.equal(got, want), r


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [136, 192, 256])
def test_packed_attention_of_wide_heads(ops, dtype, D):
    """Tiles of 64 keys, of which a sequence's last query tile sees one or two that not all its rows see."""
    lengths, H, G = [64, 65, 191, 192, 193, 1, 900, 63], 3, 1
    T = sum(lengths)
    check_packed(ops, rnd(51, T, H, D, dtype=dtype), rnd(52, T, G, D, dtype=dtype), rnd(53, T, G, D, dtype=dtype), lengths, D ** -0.5)
    up = torch.linspace(0, 300, 900, device="cuda")[:, None, None] / D  # scores that grow along the keys
    ones = torch.ones(900, 1, D, dtype=dtype, device="cuda")
    check_packed(ops, ones, (up * ones).to(dtype), rnd(54, 900, 1, D, dtype=dtype), [900], 1.0)


@pytest.mark.parametrize("dtype", [F16, BF16])
def test_packed_attention_of_wide_heads_with_values_that_are_not_finite(ops, dtype):
    n, H, D = 330, 2, 160
    q, k, v = rnd(34, n, H, D, dtype=dtype), rnd(35, n, H, D, dtype=dtype), rnd(36, n, H, D, dtype=dtype)
    want = ops.packed_attention(q, k, v, cumulative([n]), 0.1)
    for r in (0, 63, 64, 127, 128, 191, 192, 255, 256, 329):
        w = v.clone()
        w[r, 1, 150] = math.inf
        got = ops.packed_attention(q, k, w, cumulative([n]), 0.1)
        assert bool((got[r:, 1, 150] == math.inf).all())
        got[r:, 1, 150] = want[r:, 1, 150]
        assert torch.equal(got, want), r


@pytest.mark.parametrize("form", ["odd_rows", "odd_address", "heads_first", "every_second"])
def test_packed_attention_takes_any_layout(ops, form):
    lengths, H, G, D = [130, 7], 4, 2, 64
    T = sum(lengths)
    q, k, v = rnd(37, T, H, D, dtype=BF16), rnd(38, T, G, D, dtype=BF16), rnd(39, T, G, D, dtype=BF16)
    if form == "odd_rows":
        q, k, v = (torch.cat((x.flatten(1), x.flatten(1)[:, :3]), 1)[:, :x.shape[1] * D].unflatten(1, (-1, D)) for x in (q, k, v))
    if form == "odd_address":
        q, k, v = (torch.cat((x.flatten()[:1], x.flatten()))[1:].view(x.shape) for x in (q, k, v))
    if form == "heads_first":
        q, k, v = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v))
    if form == "every_second":
        q, k, v = (torch.stack((x, x), 3).flatten(2)[..., ::2] for x in (q, k, v))
    check_packed(ops, q, k, v, lengths, 0.125)


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("scale", [0.0, -0.4, 3.0])
def test_packed_attention_scales(ops, dtype, scale):
    q, k, v = rnd(40, 300, 2, 64, dtype=dtype), rnd(41, 300, 1, 64, dtype=dtype), rnd(42, 300, 1, 64, dtype=dtype)
    check_packed(ops, q, k, v, [300], scale)


def test_packed_attention_of_growing_scores(ops):
    """Scores that grow along the keys by some hundreds, so that sums are scaled again and again."""
    n, D = 900, 64
    q, k, v = rnd(43, n, 1, D, dtype=F16).abs(), rnd(44, n, 1, D, dtype=F16).abs(), rnd(45, n, 1, D, dtype=F16)
    k *= (torch.arange(n, device="cuda")[:, None, None] / 300).half()
    check_packed(ops, q, k, v, [n], 1.0)


def test_packed_attention_keeps_rows_of_no_sequence(ops):
    lengths, T, H, D = [60, 140], 230, 2, 64
    q, k, v = rnd(46, T, H, D, dtype=BF16), rnd(47, T, H, D, dtype=BF16), rnd(48, T, H, D, dtype=BF16)
    out = torch.full((T, H, D), 7.0, dtype=BF16, device="cuda")
    got = check_packed(ops, q, k, v, lengths, 0.125, first=11, out=out)
    assert got is out and bool((out[:11] == 7).all()) and bool((out[211:] == 7).all())
    for cu in ([0, 0, 0], [230, 230, 230]):
        got = ops.packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.125)
        assert not bool(got.any())


def test_packed_attention_stays_inside_with_odd_offsets(ops):
    """Offsets that are out of range or not ascending are cut to the rows there are."""
    q, k, v = rnd(46, 50, 2, 64, dtype=BF16), rnd(47, 50, 2, 64, dtype=BF16), rnd(48, 50, 2, 64, dtype=BF16)
    for cu in ([0, 1000], [-5, 30, 2 ** 31 - 1], [40, 10, 20]):
        ops.packed_attention(q, k, v, torch.tensor(cu, dtype=torch.int32, device="cuda"), 0.125)
    got = ops.packed_attention(q, k, v, torch.tensor([0, 1000], dtype=torch.int32, device="cuda"), 0.125)
    assert torch.equal(got, ops.packed_attention(q, k, v, cumulative([50]), 0.125))


# ---- sampling -------------------------------------------------------------------------------------------------------------------

def check_sample(ops, logits, u, **settings):
    B = logits.shape[0]
    got = ops.sample_tokens(logits, u, **settings).tolist()
    full = {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0, **settings}
    rows = [[float(x) for x in (v.tolist() if torch.is_tensor(v) else [v] * B)] for v in full.values()]
    for b, (row, r, t, k, p, m) in enumerate(zip(logits.cpu(), u.tolist(), *rows)):
        assert got[b] == S.sample(row, r, t, int(k), p, m), (b, t, k, p, m)


SETTINGS = [{}, {"temperature": 0.0}, {"temperature": 0.3}, {"top_k": 1}, {"top_k": 7}, {"top_k": 900}, {"top_k": 10 ** 6}, {"top_p": 0.0},
            {"top_p": 0.5}, {"top_p": 0.999}, {"min_p": 0.1}, {"min_p": 1.0}, {"top_k": 40, "top_p": 0.9, "min_p": 0.02, "temperature": 1.7},
            {"top_k": 600, "top_p": 0.7, "temperature": 5.0}]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("V", [1, 2, 33, 1000, 5003])
@pytest.mark.parametrize("settings", SETTINGS, ids=str)
def test_sample_tokens(ops, dtype, V, settings):
    logits = rnd(50 + V, 9, V, dtype=dtype) * 3
    u = torch.rand(9, device="cuda", generator=torch.Generator("cuda").manual_seed(V))
    u[0], u[1] = 0.0, 1 - 2.0 ** -24
    check_sample(ops, logits, u, **settings)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("spread", [0.0, 1e-3, 0.3, 20.0])
def test_sample_tokens_of_a_vocabulary(ops, dtype, spread):
    """Flat rows, rows of ties (a spread of 0 makes 50272 equal entries) and rows with one choice."""
    logits, u = rnd(51, 8, 50272, dtype=F32).mul(spread).to(dtype), torch.rand(8, device="cuda")
    for settings in ({}, {"top_k": 50}, {"top_p": 0.9}, {"top_k": 20000, "top_p": 0.8}, {"temperature": 0.01, "top_p": 0.9}, {"min_p": 0.5}):
        check_sample(ops, logits, u, **settings)


def test_sample_tokens_settings_by_row(ops):
    r = torch.Generator("cuda").manual_seed(3)
    B, V = 64, 3001
    logits, u = rnd(52, B, V) * 2, torch.rand(B, device="cuda", generator=r)
    pick = lambda *x: torch.tensor(x, device="cuda")[torch.randint(0, len(x), (B,), device="cuda", generator=r)]
    check_sample(ops, logits, u, temperature=pick(0.0, 0.5, 1.0, 2.0), top_k=pick(0, 1, 5, 300, 5000).int(), top_p=pick(0.0, 0.3, 0.9, 1.0, 1.5),
                 min_p=pick(0.0, 0.05, 0.9))


def test_sample_tokens_odd_entries(ops):
    """Entries of -inf, NaN, +inf and the type's lowest value; rows without any entry."""
    for dtype in (F16, BF16, F32):
        logits = rnd(53, 10, 777, dtype=dtype)
        low = torch.finfo(dtype).min
        logits[0], logits[1], logits[2] = -math.inf, math.nan, low
        logits[3, ::2], logits[4, 1:] = -math.inf, math.nan
        logits[5, ::3], logits[6, 100], logits[7, [3, 700]] = low, math.inf, math.inf
        logits[8, :776] = -math.inf
        logits[9] = -0.0
        logits[9, 100:] = 0.0
        u = torch.rand(10, device="cuda")
        for settings in ({}, {"top_k": 3}, {"top_p": 0.6}, {"min_p": 0.2}, {"temperature": 0.0}):
            got = ops.sample_tokens(logits, u, **settings).tolist()
            assert got[:2] == [-1, -1] and got[4] == 0 and got[6] == 100 and got[7] in (3, 700) and got[8] == 776
            if settings == {}:
                assert got[7] == (3 if float(u[7]) < 0.5 else 700)
            ordinary = [2, 3, 5, 8, 9]
            check_sample(ops, logits[ordinary], u[ordinary], **settings)


@pytest.mark.parametrize("settings", [{}, {"top_k": 30}, {"top_p": 0.7}, {"min_p": 0.5}], ids=str)
def test_sample_tokens_at_temperatures_far_from_one(ops, settings):
    """Next to none, of which one entry or its equals are left, and so large that all entries weigh the same."""
    t = [1e-45, 1e-40, 1e-35, 1e-28, 1e-10, 1e4, 1e15, 1e24, 1e28, 1e38]
    logits, u = rnd(57, len(t), 1500), torch.rand(len(t), device="cuda", generator=torch.Generator("cuda").manual_seed(9))
    logits[::2, 700] = logits[::2, 3] = 9.0
    check_sample(ops, logits, u, temperature=torch.tensor(t, device="cuda"), **settings)
    check_sample(ops, logits * 1e30, u, temperature=torch.tensor(t, device="cuda"), **settings)


def test_sample_tokens_takes_any_layout(ops):
    logits, u = rnd(54, 6, 1003), torch.rand(6, device="cuda")
    want = ops.sample_tokens(logits, u, top_p=0.9)
    wide = torch.full((6, 2100), math.inf, device="cuda")
    for at in (0, 4, 1):
        wide[:, at:at + 1003] = logits
        assert torch.equal(ops.sample_tokens(wide[:, at:at + 1003], u, top_p=0.9), want)
    wide[:, ::2][:, :1003] = logits
    assert torch.equal(ops.sample_tokens(wide[:, ::2][:, :1003], u, top_p=0.9), want)
    assert torch.equal(ops.sample_tokens(logits[:1].expand(6, -1), u[:1].expand(6).contiguous()),
                       ops.sample_tokens(logits[:1], u[:1]).expand(6))
    assert ops.sample_tokens(logits[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("dtype", [F16, F32])
def test_sample_tokens_of_millions(ops, dtype):
    """Rows too long for the blocks' memory, and for one sum of a thread: equal entries, so that the token is known."""
    V, first = 2 ** 25, 2 ** 22
    logits = torch.full((1, V), 1.5, dtype=dtype, device="cuda")
    for x in (0.0, 0.3, 0.77, 1 - 2.0 ** -24):
        u = torch.full((1,), x, device="cuda")
        assert int(ops.sample_tokens(logits, u)) == int(float(u) * V)
        logits[:, :first] = -math.inf
        assert int(ops.sample_tokens(logits, u, min_p=0.5)) == first + int(float(u) * (V - first))
        logits[:, :first] = 1.5


def test_sample_tokens_next_to_borders(ops):
    """Numbers next to the borders between tokens, where 32-bit weights cannot tell: the token of the 64-bit sums."""
    V, B = 4000, 256
    row = rnd(55, V)
    w = torch.exp(row.double() - row.double().max())
    run = w.cumsum(0) / w.sum()
    at = torch.randint(0, V - 1, (B,), generator=torch.Generator().manual_seed(1)).tolist()
    u = run[at].float()  # (rounded to 32 bits it lies on one side of the border or the other, as the sums in 64 bits do)
    check_sample(ops, row.expand(B, V).contiguous(), u)


def test_sample_tokens_follow_their_weights(ops):
    """Evenly spaced numbers: each token as often as its weight says, to within one."""
    row, n = rnd(56, 20), 4096
    u = (torch.arange(n, device="cuda") + 0.5) / n
    got = ops.sample_tokens(row.expand(n, 20).contiguous(), u).bincount(minlength=20)
    assert bool(((got - torch.softmax(row.double(), 0) * n).abs() <= 1.001).all())


# ---- together --------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_prompts_and_steps_together(ops, dtype):
    """Prompts of several requests, then steps of the batch: every step's row is what attention over the whole gives for it."""
    H, G, D, page, lengths, steps = 8, 2, 64, 16, [5, 33, 1, 100], 20
    B, scale = len(lengths), 0.125
    total = [n + steps for n in lengths]
    freqs = (10000.0 ** (-torch.arange(32, device="cuda") / 32)).float()
    q, k, v = rnd(60, sum(total), H, D, dtype=dtype), rnd(61, sum(total), G, D, dtype=dtype), rnd(62, sum(total), G, D, dtype=dtype)
    starts = [sum(total[:b]) for b in range(B)]
    zero = torch.zeros(B, dtype=torch.int64, device="cuda")
    k_all, v_all, table = pool(total, page, G, D, dtype)
    q_rot, k_rot = ops.paged_append(q, k, v, k_all, v_all, table, zero, cu_seqlens=cumulative(total), freqs=freqs, keys=True)
    whole = ops.packed_attention(q_rot, k_rot, v, cumulative(total), scale)

    k_pages, v_pages, _ = pool(total, page, G, D, dtype)
    rows = torch.tensor([starts[b] + i for b in range(B) for i in range(lengths[b])], device="cuda")
    q1, k1 = ops.paged_append(q[rows], k[rows], v[rows], k_pages, v_pages, table, zero, cu_seqlens=cumulative(lengths), freqs=freqs, keys=True)
    first = ops.packed_attention(q1, k1, v[rows], cumulative(lengths), scale)
    assert torch.equal(first, whole[rows])
    pos = torch.tensor(lengths, device="cuda")
    for i in range(steps):
        rows = torch.tensor([starts[b] + lengths[b] + i for b in range(B)], device="cuda")
        q1, none = ops.paged_append(q[rows], k[rows], v[rows], k_pages, v_pages, table, pos, freqs=freqs)
        assert none is None
        got = ops.paged_attention(q1, k_pages, v_pages, table, pos, scale)
        # both are off by their bounds (serving_cases.attend; |scores| here stay below 8): 3 roundings of weights or results
        bound = 3 * S.half_step(dtype) + 2.0 ** -15
        assert float((got.double() - whole[rows].double()).abs().max()) <= bound * float(v.abs().max())
        pos += 1
    assert torch.equal(k_pages.nan_to_num(nan=7.0), k_all.nan_to_num(nan=7.0))


def step_of(ops, s):
    q1, _ = ops.paged_append(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["pos"], freqs=s["freqs"])
    ctx = ops.paged_attention(q1, s["k_pages"], s["v_pages"], s["table"], s["pos"], 0.125)
    logits = ctx.flatten(1).float() @ s["head"]
    s["token"].copy_(ops.sample_tokens(logits, s["u"], temperature=0.9, top_k=40, top_p=0.95))
    s["pos"] += 1
    return ctx


def step_state(seed, B=3, H=8, G=2, D=64, room=4000):
    k_pages, v_pages, table = pool([room] * B, 16, G, D, BF16, seed=seed)
    k_pages.copy_(rnd(seed, *k_pages.shape, dtype=BF16)), v_pages.copy_(rnd(seed + 1, *v_pages.shape, dtype=BF16))
    return {"k_pages": k_pages, "v_pages": v_pages, "table": table, "pos": torch.tensor([1999, 37, -1], device="cuda"),
            "q": rnd(seed + 2, B, H, D, dtype=BF16), "k": rnd(seed + 3, B, G, D, dtype=BF16), "v": rnd(seed + 4, B, G, D, dtype=BF16),
            "freqs": torch.rand(32, device="cuda"), "head": rnd(seed + 5, H * D, 2000), "u": torch.rand(B, device="cuda"),
            "token": torch.zeros(B, dtype=torch.int64, device="cuda")}


def test_captured_steps_equal_eager_ones(ops):
    """Two captured steps, replayed at the same time on streams of their own beside eager calls, positions moving on."""
    states = [step_state(70), step_state(80)]
    copies = [{n: t.clone() for n, t in s.items()} for s in states]
    for s in states:
        step_of(ops, {n: t.clone() for n, t in s.items()})
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s, stream in zip(states, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(step_of(ops, s))
        graphs.append(g)
    third = step_state(90)
    third_copy = {n: t.clone() for n, t in third.items()}
    torch.cuda.synchronize()
    for _ in range(10):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
        step_of(ops, third)
    torch.cuda.synchronize()
    for s, c, o in zip(states + [third], copies + [third_copy], outs + [None]):
        for _ in range(10):
            want = step_of(ops, c)
        assert o is None or torch.equal(o, want)
        for n in ("pos", "token", "k_pages", "v_pages"):
            assert torch.equal(s[n], c[n]), n


def test_tensors_of_another_stream(ops):
    s, c = step_state(100), None
    c = {n: t.clone() for n, t in s.items()}
    want = step_of(ops, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step_of(ops, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(s["token"], c["token"])


def test_serving_operators_refuse_what_does_not_fit(ops):
    k_pages, v_pages, table = pool([20, 20], 16, 2, 64, BF16)
    q, k, v, pos = rnd(1, 2, 4, 64, dtype=BF16), rnd(2, 2, 2, 64, dtype=BF16), rnd(3, 2, 2, 64, dtype=BF16), torch.zeros(2, dtype=torch.int64, device="cuda")
    cu, wide = cumulative([1, 1]), rnd(4, 3, 4, 64, dtype=BF16)
    good = ops.paged_attention(q, k_pages, v_pages, table, pos - 1, 0.1)
    assert not bool(good.any())
    refused = [
        lambda: ops.paged_append(q, k, v.float(), k_pages, v_pages, table, pos),
        lambda: ops.paged_append(q, k[:1], v[:1], k_pages, v_pages, table, pos),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table.long(), pos),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table, pos.int()),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages.transpose(1, 2), table, pos),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table, pos, freqs=torch.rand(33, device="cuda")),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table, pos, freqs=torch.rand(8, device="cuda").half()),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table, pos, cu_seqlens=cu[:2]),
        lambda: ops.paged_append(q, k, v, k_pages, v_pages, table, pos, cu_seqlens=cu.long()),
        lambda: ops.paged_append(q, k, v, k_pages[..., :60], v_pages[..., :60], table, pos),
        lambda: ops.paged_append(q.cpu(), k.cpu(), v.cpu(), k_pages, v_pages, table, pos),
        lambda: ops.paged_attention(q[:, :3], k_pages, v_pages, table, pos, 0.1),
        lambda: ops.paged_attention(q, k_pages.half(), v_pages.half(), table, pos, 0.1),
        lambda: ops.paged_attention(q, k_pages, v_pages, table[:1], pos, 0.1),
        lambda: ops.paged_attention(q, k_pages, v_pages, table, pos, math.nan),
        lambda: ops.paged_attention(q, k_pages, v_pages, table, pos, math.inf),
        lambda: ops.paged_attention(q[..., :32], k_pages, v_pages, table, pos, 0.1),
        lambda: ops.packed_attention(q, k, v[:1], cu, 0.1),
        lambda: ops.packed_attention(q[:, :3], k, v, cu, 0.1),
        lambda: ops.packed_attention(q, k, v, cu.long(), 0.1),
        lambda: ops.packed_attention(q, k, v, cu[:1], 0.1),
        lambda: ops.packed_attention(q, k, v, cu, math.nan),
        lambda: ops.packed_attention(q, k, v, cu, 0.1, out=torch.empty(2, 4, 64, device="cuda")),
        lambda: ops.packed_attention(q.double(), k.double(), v.double(), cu, 0.1),
        lambda: ops.packed_attention(q, k, v, cu, 0.1, out=q),
        lambda: ops.packed_attention(wide[:2], k, v, cu, 0.1, out=wide[1:]),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(3, device="cuda")),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda").double()),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), temperature=-1.0),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), temperature=math.nan),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), top_k=-1),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), top_p=-0.1),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), min_p=1.1),
        lambda: ops.sample_tokens(q[:, 0], torch.rand(2, device="cuda"), top_k=torch.ones(2, device="cuda")),
        lambda: ops.sample_tokens(q[:, 0].long(), torch.rand(2, device="cuda")),
    ]
    for i, call in enumerate(refused):
        with pytest.raises((AssertionError, RuntimeError)):
            call()
            print("taken:", i)


# ---- in the generation loop --------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("cg", [False, True])
def test_generate_samples(ops, cg):
    """Every new token is the one that its logits, the settings and the generator's numbers give; top_k=1 stays greedy."""
    from dejavu_b200.gpt import GPTLMHeadModel, opt_config

    cfg = opt_config("opt-125m", n_layer=2, n_embd=256, hidden_size=256, n_head=4, n_inner=1024, vocab_size=512, max_position_embeddings=64,
                     mlp_sparse=False, att_sparse=False)
    model = GPTLMHeadModel(cfg, device="cuda", dtype=F16).eval().init_random(0, std=0.3)
    ids = torch.randint(0, 512, (3, 7), device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    settings = {"top_k": 20, "top_p": 0.9, "min_p": 0.01, "temperature": 1.5}
    kw = {"max_length": 20, "cg": cg, "vocab_size": 500, "return_dict_in_generate": True, "output_scores": True}
    out = model.generate(ids, generator=torch.Generator("cuda").manual_seed(5), **settings, **kw)
    g = torch.Generator("cuda").manual_seed(5)
    assert out.sequences.shape == (3, 20) and len(out.scores) == 13
    for i, scores in enumerate(out.scores):
        u = torch.rand(3, device="cuda", generator=g).tolist()
        for b in range(3):
            assert int(out.sequences[b, 7 + i]) == S.sample(scores[b].cpu(), u[b], 1.5, 20, 0.9, 0.01)
    again = model.generate(ids, generator=torch.Generator("cuda").manual_seed(5), **settings, **kw)
    assert torch.equal(out.sequences, again.sequences)
    greedy = model.generate(ids, **kw)
    assert torch.equal(greedy.sequences[:, 7:], torch.stack([s.argmax(-1) for s in greedy.scores], 1))
    cold = model.generate(ids, top_k=0, temperature=0.0, **kw)
    assert torch.equal(cold.sequences, greedy.sequences)
    for bad in ({"top_k": -1}, {"top_p": 1.5}, {"min_p": -0.1}, {"temperature": -1.0}, {"temperature": math.nan}):
        with pytest.raises(ValueError):
            model.generate(ids, **{"top_k": 0, **bad}, **kw)
    for p in model.transformer.ln_f.parameters():
        p.data.fill_(math.nan)
    none = model.generate(ids, top_k=0, **kw)  # no entry to choose from
    assert bool(none.scores[0].isnan().all()) and not bool(none.sequences[:, 7:].any())


def test_thousands_of_short_prompts(ops):
    """More sequences and more items than are put in order or searched in one go."""
    g = torch.Generator().manual_seed(3)
    lengths = torch.randint(0, 12, (5000,), generator=g).tolist()
    lengths[4000], lengths[77] = 700, 300
    T, H, G, D = sum(lengths), 16, 2, 64  # (some 500 items per block)
    q, k, v = rnd(1, T, H, D, dtype=BF16), rnd(2, T, G, D, dtype=BF16), rnd(3, T, G, D, dtype=BF16)
    got = ops.packed_attention(q, k, v, cumulative(lengths), 0.125)
    cu = cumulative(lengths).tolist()
    for b in [0, 1, 2, 76, 77, 78, 3999, 4000, 4001, 4998, 4999] + torch.randint(0, 5000, (40,), generator=g).tolist():
        rows = slice(cu[b], cu[b + 1])
        one = ops.packed_attention(q[rows], k[rows], v[rows], cumulative([lengths[b]]), 0.125)
        assert torch.equal(got[rows], one), b
    k_pages, v_pages, table = pool(lengths, 8, G, D, BF16)
    pos = torch.zeros(5000, dtype=torch.int64, device="cuda")
    ops.paged_append(None, k, v, k_pages, v_pages, table, pos, cu_seqlens=cumulative(lengths))
    want = torch.full_like(k_pages, math.nan)
    b = torch.repeat_interleave(torch.arange(5000, device="cuda"), torch.tensor(lengths, device="cuda"))
    at = torch.arange(T, device="cuda") - cumulative(lengths)[:-1].long()[b]
    want[table[b, at // 8].long(), :, at % 8] = k
    assert torch.equal(k_pages.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))

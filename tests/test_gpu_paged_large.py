"""Attention over the paged cache where scores are large or no numbers, and
in shapes at the ends of its forms.
Tolerances are derived per test, from constructions in which few roundings
take part."""
import numpy as np
import pytest

from test_gpu_paged import WIDE, Batch, Pool, attend, check

pytestmark = pytest.mark.gpu

FORMS = [(1, 0), (40, 0), (40, WIDE)]  # new tokens, spare pages: few rows, few of little work, many rows


@pytest.mark.parametrize("n,spare", FORMS)
@pytest.mark.parametrize("log2_score", [20.0, 24.7, 25.3, 26.2, 26.5, 26.9, 27.1, 27.5, 27.9, 28.4, 29.5, 40.0, 100.0])
def test_equal_scores_of_any_size_share_their_row(ctx, n, spare, log2_score):
    """One dimension of a query, and half of the positions with one key there
    (one score, in whatever way it is rounded), the others 0: the row is the
    mean of the first half's values. Off by the weights' two f16 terms (2^-22)
    and two f32 sums of `count` and 64 terms, half a step each."""
    rng = np.random.default_rng(61)
    heads, kv_heads, D, first = 4, 2, 128, 70
    batch = Batch(rng, 16, [n], [first], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()[0]
    pool.fill(0, owned)
    pool.scales[0][0, owned] = 2.0**-6
    pool.scales[1][0, owned] = 2.0**-4
    high = rng.random(len(owned)) < 0.5
    high[0] = True
    dim = 37
    for g in range(kv_heads):
        pool.codes[0][0, owned, g * D + dim] = np.where(high, 255, 128)
    query = np.zeros((n, heads, D), np.float32)
    query[:, :, dim] = 2.0**log2_score / (127 * 2.0**-6 * np.log2(np.e) / np.sqrt(D))
    got = attend(ctx, pool, 0, batch, query.reshape(n, heads * D), heads).reshape(n, heads, D)
    for t in range(n):
        seen = owned[:first + t + 1][high[:first + t + 1]]
        for h in range(heads):
            v = pool.values(1, 0, seen, h // 2)
            bound = np.abs(v).mean(0) * (2 * (len(owned) + 64) * 2.0**-24 + 2.0**-21) + 1e-30
            assert np.all(np.abs(got[t, h] - v.mean(0)) <= bound), (t, h, got[t, h, :4], v.mean(0)[:4])


@pytest.mark.parametrize("n,spare", [(1, 0), (50, 2), (50, WIDE)])
@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
def test_a_key_scale_that_is_no_number_reaches_its_head_s_rows_that_see_it(ctx, n, spare, scale):
    """Whatever sign the products with it have."""
    rng = np.random.default_rng(63)
    heads, kv_heads, D, f = 8, 2, 128, 61
    batch = Batch(rng, 16, [n], [f], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()[0]
    pool.fill(0, owned)
    query = rng.standard_normal((n, heads * D)).astype(np.float32)
    at = f - 5 if n == 1 else f + 19
    plain = attend(ctx, pool, 0, batch, query, heads).reshape(n, heads, D)
    pool.scales[0][0, owned[at], 3] = scale  # key/value head 1, dimensions 64 on
    got = attend(ctx, pool, 0, batch, query, heads).reshape(n, heads, D)
    reached = np.zeros(got.shape, bool)
    reached[max(0, at - f):, heads // kv_heads:] = True
    assert np.isnan(got[reached]).all()
    assert np.array_equal(got[~reached], plain[~reached])


@pytest.mark.parametrize("n,spare", FORMS)
@pytest.mark.parametrize("common", [50.0, 1000.0, 8000.0])
def test_large_scores_that_differ_by_little(ctx, n, spare, common):
    """Every score is about `common`, in one dimension, and differs by a few
    in another. A score is two products, each off by the query's two f16 terms
    (2^-22), and half a dozen f32 roundings: 2^-21 of its size with room for
    all of them, on both sides of the subtraction."""
    rng = np.random.default_rng(62)
    heads, kv_heads, D, first = 4, 2, 128, 150
    batch = Batch(rng, 16, [n], [first], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()[0]
    pool.fill(0, owned)
    pool.scales[0][0, owned] = 2.0**-6
    for g in range(kv_heads):
        pool.codes[0][0, owned, g * D + 5] = 228
    query = np.zeros((n, heads, D), np.float32)
    query[:, :, 5] = common * np.sqrt(D) / (100 * 2.0**-6)
    query[:, :, 99] = 2.0 * np.sqrt(D)
    got = attend(ctx, pool, 0, batch, query.reshape(n, heads * D), heads).reshape(n, heads, D)
    for t in range(n):
        seen = owned[:first + t + 1]
        for h in range(heads):
            k, v = pool.values(0, 0, seen, h // 2), pool.values(1, 0, seen, h // 2)
            q = query[t, h].astype(np.float64)
            s = k @ q / np.sqrt(D)
            w = np.exp(s - s.max())
            want = w @ v / w.sum()
            dw = np.expm1(2 * (np.abs(k) @ np.abs(q)).max() / np.sqrt(D) * 2.0**-21 + np.ptp(s) * 2.0**-23 + 2.0**-21)
            spread = w @ np.abs(v) / w.sum()
            bound = spread * (2 * dw + 2 * (len(seen) + 64) * 2.0**-24) + len(seen) * (w[:, None] * np.abs(v)).max() / w.sum() * 2.0**-21
            assert np.median(bound / spread) < 0.02  # (so that a wrong row shows)
            assert np.all(np.abs(got[t, h] - want) <= bound), (t, h)


@pytest.mark.parametrize("spare", [0, WIDE])
@pytest.mark.parametrize("ratio", [129, 256])
def test_more_heads_a_key_value_head_than_a_large_tile(ctx, ratio, spare):
    rng = np.random.default_rng(64)
    check(ctx, rng, (ratio, 1, 64), 16, [3, 1, 2], [200, 127, 128], spare=spare)
    check(ctx, rng, (ratio, 1, 64), 16, [1, 1, 1], [200, 127, 0], spare=spare, one_row=True)


def test_steps_of_many_heads_over_wide_tables(ctx):
    """The form for many rows, one row a sequence."""
    rng = np.random.default_rng(65)
    check(ctx, rng, (64, 1, 64), 16, [1] * 5, [300, 0, 127, 128, 64], spare=WIDE, one_row=True)
    check(ctx, rng, (80, 2, 128), 24, [1, 1], [3, 500], spare=WIDE, one_row=True, pad=3)


@pytest.mark.parametrize("first", [0, 130])
def test_a_chunk_of_more_than_64_tiles(ctx, first):
    rng = np.random.default_rng(66)
    check(ctx, rng, (16, 1, 64), 16, [7, 600, 5], [40, first, 3], pad=2)


@pytest.mark.parametrize("n,spare", FORMS)
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("log2_score", [12.0, 26.5, 27.5, 60.0])
def test_a_maximum_that_moves_over_a_long_context(ctx, n, spare, sign, log2_score):
    """Keys that rise, or fall, along a context that several workgroups take:
    a row is the mean of the values at the last key's positions (the next key's
    score is 32 and more away in base 2, or 2^-32 of the weights), with the
    same roundings as above."""
    rng = np.random.default_rng(67)
    heads, kv_heads, D, first = 4, 2, 128, 1500
    batch = Batch(rng, 16, [n], [first], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()[0]
    pool.fill(0, owned)
    pool.scales[0][0, owned] = 2.0**-6
    pool.scales[1][0, owned] = 2.0**-4
    step = np.arange(len(owned)) * 120 // len(owned)
    code = step if sign > 0 else -step - 1
    dim = 37
    for g in range(kv_heads):
        pool.codes[0][0, owned, g * D + dim] = 128 + code
    query = np.zeros((n, heads, D), np.float32)
    query[:, :, dim] = 2.0**log2_score / (127 * 2.0**-6 * np.log2(np.e) / np.sqrt(D))
    got = attend(ctx, pool, 0, batch, query.reshape(n, heads * D), heads).reshape(n, heads, D)
    for t in range(n):
        seen = owned[:first + t + 1]
        best = seen[code[:first + t + 1] == code[:first + t + 1].max()]
        for h in range(heads):
            v, others = pool.values(1, 0, best, h // 2), np.abs(pool.values(1, 0, seen, h // 2)).max()
            bound = np.abs(v).mean(0) * (2 * (len(owned) + 64) * 2.0**-24 + 2.0**-21) + len(owned) * 2.0**-32 * others
            assert np.all(np.abs(got[t, h] - v.mean(0)) <= bound), (t, h)

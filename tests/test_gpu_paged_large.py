"""Attention over the paged cache where scores are large or no numbers.
Tolerances are derived per test, from constructions in which few roundings
take part."""
import numpy as np
import pytest

from test_gpu_paged import WIDE, Batch, Pool, attend

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

"""The paged attention and sampling at the sizes that the header ends at."""
import numpy as np
import pytest

import qwenscriber_amd as qa
from test_gpu_paged import NONE, Pool, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("layout", [(1024, 1024, 64), (4096, 16, 64), (1024, 512, 128), (768, 256, 256)])
def test_many_heads(ctx, layout):
    rng = np.random.default_rng(81)
    check(ctx, rng, layout, 16, [1], [150], one_row=True)
    check(ctx, rng, layout, 16, [2, 1], [130, 0], pad=1)


@pytest.mark.parametrize("one_row", [True, False])
def test_65535_sequences(ctx, one_row):
    """A position each: a row is its value, off by the weight's two f16 terms
    (2^-22) and a handful of f32 roundings."""
    rng = np.random.default_rng(82)
    n, D = 65535, 64
    pool = Pool(ctx, rng, 1, n, 1, 1, D)
    pool.fill(0, np.arange(n))
    cache = pool.upload()
    order = rng.permutation(n).astype(np.uint32)
    query = rng.standard_normal((n, D)).astype(np.float32)
    bufs = [ctx.to_device(a) for a in (np.arange(n + 1, dtype=np.uint32), np.zeros(n, np.uint32), order, query)]
    out = ctx.buffer(query.nbytes)
    desc = qa.PagedBatch(n, n, 1, None if one_row else bufs[0].ptr, bufs[1].ptr, bufs[2].ptr)
    ctx.paged_attention(cache, 0, desc, out.ptr, bufs[3].ptr, D, 1)
    want = pool.values(1, 0, order, 0)
    assert np.all(np.abs(out.download(np.float32).reshape(n, D) - want) <= np.abs(want) * 2.0**-20)
    for b in bufs + [out]:
        b.free()
    pool.free()


@pytest.mark.parametrize("n", [1, 40])
def test_positions_next_to_the_tables_limit(ctx, n):
    """Tables of nearly 2^32 positions, all but three pages missing."""
    rng = np.random.default_rng(83)
    heads, kv_heads, D, page_size = 4, 2, 64, 4096
    table_pages = (2**32 - 2**16) // page_size - 1
    first = table_pages * page_size - n - 3
    pool = Pool(ctx, rng, 1, 3, page_size, kv_heads, D)
    pool.fill(0, np.arange(3 * page_size))
    table = np.full(table_pages, NONE, np.uint32)
    places = {0: 2, table_pages // 2: 0, table_pages - 1: 1}
    for at, page in places.items():
        table[at] = page
    width = heads * D
    query = rng.standard_normal((n, width)).astype(np.float32)
    bufs = [ctx.to_device(a) for a in (np.array([0, n], np.uint32), np.array([first], np.uint32), table, query)]
    out = ctx.buffer(query.nbytes)
    cache = pool.upload()
    desc = qa.PagedBatch(1, n, table_pages, *[b.ptr for b in bufs[:3]])
    ctx.paged_attention(cache, 0, desc, out.ptr, bufs[3].ptr, width, heads)
    got = out.download(np.float32).reshape(n, heads, D)
    where = np.concatenate([np.arange(page_size, dtype=np.int64) + at * page_size for at in sorted(places)])
    rows = np.concatenate([np.arange(page_size) + places[at] * page_size for at in sorted(places)])
    for h in range(heads):
        k, v = pool.values(0, 0, rows, h // 2), pool.values(1, 0, rows, h // 2)
        q = query[:, h * D:(h + 1) * D].astype(np.float64)
        s = q @ k.T / np.sqrt(D)
        s[where[None, :] > first + np.arange(n)[:, None]] = -np.inf
        w = np.exp(s - s.max(1, keepdims=True))
        total = w.sum(1, keepdims=True)
        spread = w @ np.abs(v) / total
        # As the chunks' bound: a score's two terms and D f32 products, then
        # sums of all positions.
        ds = (np.abs(q).max(1, keepdims=True) * 2.0**-22 + (D + 8) * 2.0**-24) * np.abs(k).sum(1).max() * np.abs(q).max() / np.sqrt(D)
        bound = spread * (2 * np.expm1(2 * ds + np.abs(s[np.isfinite(s)]).max() * 2.0**-22 + 2.0**-21) + 2 * (len(rows) + 64) * 2.0**-24)
        bound += len(rows) * (w / total).max(1, keepdims=True) * np.abs(v).max() * 2.0**-21
        assert np.all(np.abs(got[:, h] - w @ v / total) <= bound)
    for b in bufs + [out]:
        b.free()
    pool.free()


def test_a_row_of_2_to_the_26_logits(ctx):
    """Few tokens that count, the first and the last among them."""
    count = 2**26
    logits = np.full(count, -100.0, np.float32)
    at = np.array([0, 4095, 4096, 12345678, count - 4097, count - 1])
    logits[at] = [1.0, 2.0, 0.5, 3.0, 2.0, 2.5]
    order = at[np.lexsort((at, -logits[at]))]
    share = np.exp(logits[order].astype(np.float64))
    edge = np.cumsum(share) / share.sum()
    numbers = np.concatenate([[0.0], (edge[:-1] + edge[1:]) / 2, [0.999]]).astype(np.float32)
    buf, ids = ctx.to_device(logits), ctx.buffer(4)
    for rule in ((1.0, 0, 1.0, 0.0), (1.0, 6, 1.0, 0.0), (1.0, 0, 0.99999, 0.0), (1.0, 0, 1.0, 0.01)):
        params = ctx.to_device(np.frombuffer(bytes(qa.Sampling(*rule)), np.uint8))
        for u in numbers:
            number = ctx.to_device(np.array([u], np.float32))
            ctx.sample_rows(buf.ptr, 1, count, params.ptr, number.ptr, ids.ptr)
            assert ids.download(np.uint32)[0] == order[np.searchsorted(edge, np.float64(u), side="right")]
            number.free()
        params.free()
    buf.free()
    ids.free()

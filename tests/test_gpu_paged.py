"""The paged q8 key/value cache (qwh_paged_append, qwh_paged_attention,
qwh_paged_copy) against the same operations in 64 bits on the host.

Tolerances are worst-case bounds of the kernels' arithmetic, per output. The
attention's queries and its weights times value scales are sums of two f16
terms (off by at most 2^-22 of the largest of their group), products and sums
are f32 (half a step, 2^-24, for each of the terms that a sum adds), exponents
are exp2 of the hardware (2^-22). The append's norm and rotation are 64 bits
rounded once to f32 (2^-24), and its codes those of quantizeRow on that."""
import numpy as np
import pytest

import qwenscriber_amd as qa
from oracle import oracle as o

pytestmark = pytest.mark.gpu

NAN16 = np.uint16(0x7E00)
NONE = 0xFFFFFFFF


class Pool:
    """A pool on the host and on the device. Rows that no sequence owns hold
    NaN scales: a read of them that reaches a result shows."""

    def __init__(self, ctx, rng, layers, pages, page_size, kv_heads, head_dim):
        self.ctx, self.rng = ctx, rng
        self.layers, self.pages, self.page_size = layers, pages, page_size
        self.kv_heads, self.head_dim = kv_heads, head_dim
        self.width = kv_heads * head_dim
        rows = (layers, pages * page_size)
        self.codes = [np.full(rows + (self.width,), 255, np.uint8) for _ in range(2)]
        self.scales = [np.full(rows + (self.width // 64,), NAN16, np.uint16).view(np.float16) for _ in range(2)]
        self.buffers = []

    def fill(self, layer, rows, low=0.005, high=0.03):
        for k in range(2):
            normal = self.rng.standard_normal((len(rows), self.width)) * 50
            self.codes[k][layer, rows] = np.clip(np.rint(normal) + 128, 0, 255)
            self.scales[k][layer, rows] = self.rng.uniform(low, high, (len(rows), self.width // 64))

    def upload(self):
        self.buffers = [self.ctx.to_device(a.reshape(-1).view(np.uint8)) for a in
                        (self.scales[0], self.codes[0], self.scales[1], self.codes[1])]
        return qa.PagedCache(self.layers, self.pages, self.page_size, self.kv_heads, self.head_dim,
                             *[b.ptr for b in self.buffers])

    def download(self):
        got = [b.download(np.uint8) for b in self.buffers]
        return ([got[1].reshape(self.codes[0].shape), got[3].reshape(self.codes[1].shape)],
                [got[0].view(np.uint16).reshape(self.scales[0].shape), got[2].view(np.uint16).reshape(self.scales[1].shape)])

    def values(self, which, layer, rows, head):
        at = slice(head * self.head_dim, (head + 1) * self.head_dim)
        groups = slice(head * self.head_dim // 64, (head + 1) * self.head_dim // 64)
        scale = np.repeat(self.scales[which][layer, rows][:, groups].astype(np.float64), 64, axis=1)
        return (self.codes[which][layer, rows][:, at].astype(np.float64) - 128) * scale

    def free(self):
        for b in self.buffers:
            b.free()


class Batch:
    """New tokens per sequence, positions before them, and page tables."""

    def __init__(self, rng, page_size, new, first, spare=0, pad=0, one_row=False, holes=()):
        self.new, self.first, self.page_size = new, first, page_size
        self.one_row = one_row
        self.rows = sum(new) + pad
        need = [-(-(f + n) // page_size) for n, f in zip(new, first)]
        self.table_pages = max(need + [1]) + spare
        self.pages = sum(need) + 3
        order = rng.permutation(self.pages).astype(np.uint32)
        self.tables = np.full((len(new), self.table_pages), NONE, np.uint32)
        at = 0
        for b, n in enumerate(need):
            self.tables[b, :n] = order[at:at + n]
            at += n
        for b, page, entry in holes:
            self.tables[b, page] = entry
        self.starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        self.buffers = []

    def owned(self):
        """Every (sequence, position)'s pool row, or -1."""
        out = []
        for b, (n, f) in enumerate(zip(self.new, self.first)):
            p = np.arange(f + n)
            page = self.tables[b, p // self.page_size].astype(np.int64)
            out.append(np.where(page < self.pages, page * self.page_size + p % self.page_size, -1))
        return out

    def upload(self, ctx):
        arrays = [self.starts, np.asarray(self.first, np.uint32), self.tables]
        self.buffers = [ctx.to_device(a) for a in arrays]
        starts, first, tables = [b.ptr for b in self.buffers]
        return qa.PagedBatch(len(self.new), self.rows, self.table_pages, None if self.one_row else starts, first, tables)

    def free(self):
        for b in self.buffers:
            b.free()


def reference(pool, layer, batch, query, heads):
    """(out, bound) in 64 bits: rows [rows][heads * head_dim], and how far a
    kernel with the arithmetic above may be off."""
    D, ratio = pool.head_dim, heads // pool.kv_heads
    out = np.zeros((batch.rows, heads * D))
    bound = np.zeros_like(out)
    for b, owned in enumerate(batch.owned()):
        n, f = batch.new[b], batch.first[b]
        where = np.flatnonzero(owned >= 0)
        rows = owned[where]
        for g in range(pool.kv_heads):
            k, v = pool.values(0, layer, rows, g), pool.values(1, layer, rows, g)
            for t in range(n):
                row = int(batch.starts[b]) + t
                seen = where <= f + t
                if not seen.any():
                    continue
                ks, vs = k[seen], v[seen]
                for h in range(g * ratio, (g + 1) * ratio):
                    at = slice(h * D, (h + 1) * D)
                    q = query[row, at].astype(np.float64)
                    s = ks @ q / np.sqrt(D)
                    w = np.exp(s - s.max())
                    total = w.sum()
                    out[row, at] = w @ vs / total
                    # Scores: the query's two terms, and D products summed;
                    # in nats, on both sides of the subtraction.
                    top = np.abs(q).reshape(-1, 64).max(1).repeat(64)
                    ds = (np.abs(ks) @ (top * 2.0**-22 + np.abs(q) * (D + 8) * 2.0**-24)).max() / np.sqrt(D)
                    dw = np.expm1(2 * ds + np.abs(s - s.max()).max() * 2.0**-23 + 2.0**-21)
                    spread = (w @ np.abs(vs)) / total
                    count = len(ks)
                    largest = (w[:, None] * np.abs(vs)).max() / total
                    bound[row, at] = spread * (2 * dw + 2 * (count + 64) * 2.0**-24) + count * largest * 2.0**-21 + 1e-30
    return out, bound


def attend(ctx, pool, layer, batch, query, heads, stride=None):
    width = heads * pool.head_dim
    stride = stride or width
    held = np.full((batch.rows, stride), np.nan, np.float32)
    held[:, :width] = query
    cache, desc = pool.upload(), batch.upload(ctx)
    q = ctx.to_device(held)
    out = ctx.to_device(np.full((batch.rows, width), -77.0, np.float32))
    ctx.paged_attention(cache, layer, desc, out.ptr, q.ptr, stride, heads)
    got = out.download(np.float32).reshape(batch.rows, width)
    for x in (q, out):
        x.free()
    pool.free()
    batch.free()
    return got


def check(ctx, rng, layout, page_size, new, first, layers=1, layer=0, query_scale=2.0, stride_extra=0, change=None, **kw):
    heads, kv_heads, D = layout
    batch = Batch(rng, page_size, new, first, **kw)
    pool = Pool(ctx, rng, layers, batch.pages, page_size, kv_heads, D)
    owned = [r[r >= 0] for r in batch.owned()]
    pool.fill(layer, np.concatenate(owned) if owned else np.zeros(0, int))
    if change:
        change(pool, batch)
    query = (query_scale * rng.standard_normal((batch.rows, heads * D))).astype(np.float32)
    got = attend(ctx, pool, layer, batch, query, heads, heads * D + stride_extra)
    with np.errstate(all="ignore"):
        want, bound = reference(pool, layer, batch, query, heads)
    total = sum(new)
    assert np.all(got[total:] == -77.0), "rows behind the last sequence"
    err = np.abs(got[:total] - want[:total])
    bad = ~(err <= bound[:total])
    assert not bad.any(), (np.argwhere(bad)[:5].tolist(), err[bad][:5], bound[:total][bad][:5])
    return got[:total], want[:total]


LAYOUTS = [(16, 8, 128), (4, 4, 64), (8, 2, 64), (14, 2, 64), (6, 2, 128), (8, 1, 128), (4, 2, 256), (6, 2, 192), (40, 2, 64),
           (3, 1, 256), (5, 5, 192)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("page_size", [1, 16, 24])
def test_steps_of_one_token(ctx, layout, page_size):
    rng = np.random.default_rng(1)
    check(ctx, rng, layout, page_size, [1] * 7, [0, 1, 30, 31, 63, 64, 300], one_row=True)


@pytest.mark.parametrize("layout", LAYOUTS)
def test_chunks(ctx, layout):
    rng = np.random.default_rng(2)
    check(ctx, rng, layout, 16, [1, 5, 0, 33, 70], [0, 200, 9, 0, 77], pad=3)


@pytest.mark.parametrize("page_size", [1, 7, 16, 31, 64, 100, 500])
@pytest.mark.parametrize("n,first", [(1, 0), (2, 63), (16, 48), (31, 97), (64, 0), (65, 128), (130, 1)])
def test_pages_that_end_inside_a_tile(ctx, page_size, n, first):
    rng = np.random.default_rng(3)
    check(ctx, rng, (4, 2, 64), page_size, [n, 3], [first, 129], spare=2)


@pytest.mark.parametrize("batch", [1, 2, 63, 64, 65, 130])
def test_many_sequences(ctx, batch):
    rng = np.random.default_rng(4)
    new = [(3 * b + 1) % 4 for b in range(batch)]
    check(ctx, rng, (2, 1, 64), 16, new, [(37 * b) % 200 for b in range(batch)], pad=5)
    check(ctx, rng, (2, 1, 64), 16, [1] * batch, [(37 * b) % 200 for b in range(batch)], one_row=True)


@pytest.mark.parametrize("new,first", [([1], [4095]), ([1, 1], [8191, 5]), ([130], [3000]), ([515], [0])])
def test_long_contexts(ctx, new, first):
    rng = np.random.default_rng(5)
    check(ctx, rng, (4, 2, 128), 16, new, first, one_row=max(new) == 1)


# Tables far longer than the sequences: the kernel for many rows also takes
# chunks that would otherwise be little work.
WIDE = 70000


@pytest.mark.parametrize("layout", LAYOUTS)
def test_chunks_with_wide_tables(ctx, layout):
    rng = np.random.default_rng(31)
    check(ctx, rng, layout, 16, [1, 5, 0, 33, 70], [0, 200, 9, 0, 77], pad=3, spare=WIDE)


@pytest.mark.parametrize("page_size", [1, 7, 16, 31, 64, 100])
@pytest.mark.parametrize("n,first", [(31, 97), (64, 0), (65, 128), (130, 1)])
def test_pages_that_end_inside_a_tile_with_wide_tables(ctx, page_size, n, first):
    rng = np.random.default_rng(32)
    check(ctx, rng, (4, 2, 64), page_size, [n, 3], [first, 129], spare=1100000 // page_size)


@pytest.mark.parametrize("batch", [63, 64, 65, 130])
def test_many_sequences_of_many_rows(ctx, batch):
    rng = np.random.default_rng(33)
    new = [(7 * b + 1) % 50 for b in range(batch)]
    check(ctx, rng, (2, 1, 64), 16, new, [(37 * b) % 150 for b in range(batch)], pad=5)


@pytest.mark.parametrize("spare", [2, WIDE])
@pytest.mark.parametrize("scale", [np.inf, -np.inf, np.nan])
def test_a_value_scale_that_is_no_number_reaches_the_rows_that_see_it(ctx, spare, scale):
    """And of these only the 64 dimensions that it scales."""
    rng = np.random.default_rng(34)
    heads, kv_heads, D, n, f = 4, 2, 128, 50, 61
    batch = Batch(rng, 16, [n], [f], spare=spare)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()[0]
    pool.fill(0, owned)
    query = rng.standard_normal((n, heads * D)).astype(np.float32)
    want, bound = reference(pool, 0, batch, query, heads)
    at = 80  # seen by the tokens from 19 on
    pool.scales[1][0, owned[at], 3] = scale  # key/value head 1, dimensions 64 on
    got = attend(ctx, pool, 0, batch, query, heads).reshape(n, heads, 2, 64)
    reached = np.zeros(got.shape, bool)
    reached[at - f:, 2:, 1] = True
    assert not np.isfinite(got[reached]).any()
    assert np.all(np.abs(got - want.reshape(got.shape))[~reached] <= bound.reshape(got.shape)[~reached])


@pytest.mark.parametrize("n,spare", [(1, 0), (33, 0), (33, WIDE)])
def test_queries_whose_scaled_value_is_next_to_a_border_of_two_halves(ctx, n, spare):
    """The query's two terms have to be of one number: x times the scaling,
    rounded to f32 first or not, can round to two halves, a step apart (2^-11,
    where both terms hold 2^-22). One dimension a head, so that the bound has
    no sum of roundings to hide it in."""
    rng = np.random.default_rng(36)
    heads, kv_heads, D = 8, 2, 64
    x = rng.uniform(4, 8, 1 << 22).astype(np.float32)
    factor = np.float32(1.44269504088896340736) / np.sqrt(np.float32(D))
    exact = x.astype(np.float64) * np.float64(factor) * 32
    border = x[exact.astype(np.float16) != exact.astype(np.float32).astype(np.float16)]
    assert len(border) > 100
    batch = Batch(rng, 16, [n], [90], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    pool.fill(0, batch.owned()[0])
    query = np.zeros((n, heads, D), np.float32)
    at = rng.integers(0, D, (n, heads, 1))
    np.put_along_axis(query, at, border[rng.integers(0, len(border), at.shape)], 2)
    query = query.reshape(n, heads * D)
    got = attend(ctx, pool, 0, batch, query, heads)
    want, bound = reference(pool, 0, batch, query, heads)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("n", [3, 40])
def test_positions_without_a_page_with_wide_tables(ctx, n):
    rng = np.random.default_rng(35)
    check(ctx, rng, (4, 2, 128), 16, [n, n], [100, 37], spare=WIDE, holes=[(0, 0, NONE), (0, 5, NONE), (1, 1, NONE)])


def test_other_layers_strides_and_spare_rows(ctx):
    rng = np.random.default_rng(6)
    check(ctx, rng, (16, 8, 128), 16, [3, 20], [50, 7], layers=3, layer=2, stride_extra=2052, pad=9)
    # One row each with more rows than sequences: those behind stay.
    check(ctx, rng, (16, 8, 128), 16, [1, 1], [50, 7], layers=3, layer=1, pad=2, one_row=True)


def test_more_heads_than_a_tile_of_rows(ctx):
    rng = np.random.default_rng(7)
    check(ctx, rng, (64, 1, 64), 16, [1, 1], [99, 3], one_row=True)
    check(ctx, rng, (64, 1, 64), 16, [9, 2], [99, 3])


@pytest.mark.parametrize("n", [1, 40])
def test_positions_without_a_page(ctx, n):
    rng = np.random.default_rng(8)
    # Holes in the middle, at the first page, at the new tokens' own page; an
    # entry past the pool; and a sequence without any page: zeros.
    holes = [(0, 1, NONE), (0, 2, NONE), (1, 0, NONE), (2, 6, NONE), (2, 7, NONE), (3, 1, 10 ** 6), (3, 4, 2 ** 31)] + [
        (4, p, NONE) for p in range(8)]
    got, want = check(ctx, rng, (4, 2, 128), 16, [n] * 5, [100, 100, 100, 90, 80], holes=holes, spare=2)
    assert np.all(got[4 * n:] == 0.0)


def test_a_first_row_that_sees_nothing(ctx):
    # The first page has no entry: the tokens in it see nothing, later ones do.
    rng = np.random.default_rng(9)
    got, want = check(ctx, rng, (4, 2, 64), 16, [40], [0], holes=[(0, 0, NONE)])
    assert np.all(got[:16] == 0.0) and np.all(np.abs(got[16:]).max(1) > 0)


@pytest.mark.parametrize("scale", [np.inf, np.nan])
@pytest.mark.parametrize("n", [2, 40])
def test_a_later_position_s_infinities_do_not_reach_earlier_rows(ctx, scale, n):
    rng = np.random.default_rng(10)
    heads, kv_heads, D = 4, 2, 128
    batch = Batch(rng, 16, [n, n], [61, 200])
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    owned = batch.owned()
    pool.fill(0, np.concatenate(owned))
    query = rng.standard_normal((batch.rows, heads * D)).astype(np.float32)
    want, bound = reference(pool, 0, batch, query, heads)
    for k in range(2):  # the last token of sequence 0
        pool.scales[k][0, owned[0][-1]] = scale
    got = attend(ctx, pool, 0, batch, query, heads)
    keep = np.ones(batch.rows, bool)
    keep[n - 1] = False
    assert np.all(np.abs(got - want)[keep] <= bound[keep])
    assert not np.isfinite(got[n - 1]).all()


def test_scales_of_very_different_sizes(ctx):
    rng = np.random.default_rng(11)

    def change(pool, batch):
        rows = np.concatenate(batch.owned())
        s = pool.scales[1]
        s[0, rows] = 10.0 ** rng.uniform(-7, 3, s[0, rows].shape)  # f16's subnormals among them
        s[0, rows[::5]] = 0.0

    check(ctx, rng, (4, 2, 128), 16, [1, 40, 3], [300, 65, 0], change=change)
    check(ctx, rng, (4, 2, 128), 16, [1, 1, 1], [300, 65, 0], change=change, one_row=True)


@pytest.mark.parametrize("query_scale", [0.0, 1e-30, 1e-6, 100.0, 1e4])
def test_queries_of_any_size(ctx, query_scale):
    rng = np.random.default_rng(12)
    check(ctx, rng, (4, 2, 128), 16, [1, 20], [150, 60], query_scale=query_scale)


@pytest.mark.parametrize("n,spare", [(1, 0), (40, 0), (40, WIDE)])
def test_queries_next_to_the_largest_float(ctx, n, spare):
    rng = np.random.default_rng(47)
    heads, kv_heads, D = 4, 2, 128
    batch = Batch(rng, 16, [n], [70], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    pool.fill(0, batch.owned()[0], low=1e-4, high=5e-4)
    query = np.zeros((n, heads, D), np.float32)
    np.put_along_axis(query, rng.integers(0, D, (n, heads, 1)), np.float32(3.4e38), 2)
    query = query.reshape(n, heads * D)
    got = attend(ctx, pool, 0, batch, query, heads)
    with np.errstate(all="ignore"):
        want, _ = reference(pool, 0, batch, query, heads)
    # One position has all the weight, or several of one code share it.
    assert np.all(np.abs(got - want) <= 2.0**-20 * np.abs(want) + 1e-7)


@pytest.mark.parametrize("n,spare", [(1, 0), (40, 0), (40, WIDE)])
@pytest.mark.parametrize("value", [np.inf, -np.inf, np.nan])
def test_a_query_row_that_is_no_number_stays_alone(ctx, n, spare, value):
    rng = np.random.default_rng(48)
    heads, kv_heads, D = 8, 2, 128
    batch = Batch(rng, 16, [n] * 3, [70, 200, 5], spare=spare, one_row=n == 1)
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    pool.fill(0, np.concatenate(batch.owned()))
    query = rng.standard_normal((batch.rows, heads * D)).astype(np.float32)
    want, bound = reference(pool, 0, batch, query, heads)
    row, head = n + n // 2, 5
    query[row, head * D + 7] = value
    got = attend(ctx, pool, 0, batch, query, heads)
    keep = np.ones((batch.rows, heads, D), bool)
    keep[row, head] = False
    keep = keep.reshape(batch.rows, heads * D)
    assert np.all(np.abs(got - want)[keep] <= bound[keep])


def test_rows_of_zeros_in_the_cache(ctx):
    rng = np.random.default_rng(13)

    def change(pool, batch):
        for k in range(2):
            pool.codes[k][:] = 128

    got, _ = check(ctx, rng, (4, 2, 64), 16, [1, 20], [150, 60], change=change)
    assert np.all(got == 0.0)


def test_bad_starts_and_positions_stay_in_bounds(ctx):
    """Device values no host check sees: rows past the buffer, positions past
    the tables and falling starts touch nothing beyond the buffers (here: the
    rows they name stay, or hold some result); the context still works."""
    rng = np.random.default_rng(14)
    batch = Batch(rng, 16, [2, 2, 2], [10, 20, 30])
    pool = Pool(ctx, rng, 1, batch.pages, 16, 2, 64)
    pool.fill(0, np.concatenate(batch.owned()))
    query = rng.standard_normal((batch.rows, 4 * 64)).astype(np.float32)
    batch.starts = np.array([0, 2, 4, 4_000_000_000], np.uint32)
    batch.first = [10, 4_294_967_295, 30]
    got = attend(ctx, pool, 0, batch, query, 4)
    batch.starts, batch.first = np.array([0, 2, 4, 6], np.uint32), [10, 20, 30]
    want, bound = reference(pool, 0, batch, query, 4)
    assert np.all(np.abs(got - want)[[0, 1, 4, 5]] <= bound[[0, 1, 4, 5]])
    batch.starts = np.array([5, 1, 3, 2], np.uint32)
    attend(ctx, pool, 0, batch, query, 4)
    batch.starts = np.array([0, 2, 4, 6], np.uint32)
    got = attend(ctx, pool, 0, batch, query, 4)
    assert np.all(np.abs(got - want) <= bound)


def test_two_calls_give_the_same_bits(ctx):
    rng = np.random.default_rng(15)
    batch = Batch(rng, 16, [1, 60, 4], [4000, 900, 2000])
    pool = Pool(ctx, rng, 1, batch.pages, 16, 2, 128)
    pool.fill(0, np.concatenate(batch.owned()))
    query = rng.standard_normal((batch.rows, 4 * 128)).astype(np.float32)
    first = attend(ctx, pool, 0, batch, query, 4)
    assert np.array_equal(first, attend(ctx, pool, 0, batch, query, 4))


def test_a_pool_past_four_gibibytes(ctx):
    """Code planes of 5 GiB: rows whose byte offset passes 32 bits."""
    rng = np.random.default_rng(16)
    heads, kv_heads, D, page_size = 16, 8, 128, 64
    width, pages = kv_heads * D, 5 * 2 ** 30 // (page_size * 1024)
    sizes = [pages * page_size * width // 32, pages * page_size * width]
    planes = [ctx.buffer(sizes[i % 2]) for i in range(4)]
    cache = qa.PagedCache(1, pages, page_size, kv_heads, D, *[p.ptr for p in planes])
    small = Batch(rng, page_size, [1, 20], [150, 70])
    pool = Pool(ctx, rng, 1, small.pages, page_size, kv_heads, D)
    pool.fill(0, np.concatenate(small.owned()))
    # The same pages, far apart and the last ones of the pool.
    place = np.array([pages - 1 - 3000 * i for i in range(small.pages)], np.uint32)
    place[1] = 3
    for i, p in enumerate(place):
        rows = slice(i * page_size, (i + 1) * page_size)
        for k in range(2):
            planes[2 * k].upload(pool.scales[k][0, rows].view(np.uint16), int(p) * page_size * width // 32)
            planes[2 * k + 1].upload(pool.codes[k][0, rows], int(p) * page_size * width)
    query = rng.standard_normal((small.rows, heads * D)).astype(np.float32)
    want, bound = reference(pool, 0, small, query, heads)
    small.tables = np.where(small.tables < small.pages, place[np.minimum(small.tables, small.pages - 1)], small.tables)
    desc, q, out = small.upload(ctx), ctx.to_device(query), ctx.buffer(query.nbytes)
    ctx.paged_attention(cache, 0, desc, out.ptr, q.ptr, heads * D, heads)
    got = out.download(np.float32).reshape(want.shape)
    assert np.all(np.abs(got - want) <= bound)
    # And a copy from the last page to one near the start, and back.
    ctx.paged_copy(cache, [int(place[0])], [17])
    got = planes[1].download(np.uint8, page_size * width, 17 * page_size * width)
    assert np.array_equal(got.reshape(-1, width), pool.codes[0][0, :page_size])
    for b in planes + [q, out]:
        b.free()
    small.free()


# ---------------------------------------------------------------------------
def tables(ctx, D, positions, theta=1e6):
    cos, sin = ctx.buffer(positions * D * 2), ctx.buffer(positions * D * 2)
    ctx.rope_tables(D, positions, theta, cos.ptr, sin.ptr)
    return cos, sin


def test_rope_tables(ctx):
    # kernels.zig:534-564 in f32: angle = f32(p * f32(theta^(-2i/D))), so the
    # table is cos of an angle off by at most two steps of the angle.
    for D, positions in ((64, 1), (128, 777), (192, 50)):
        cos, sin = tables(ctx, D, positions)
        angle = np.arange(positions)[:, None] * 1e6 ** (-2.0 * np.arange(D // 2) / D)
        tol = angle * 4 * 2.0**-24 + 2.0**-23
        for buf, want in ((cos, np.cos(angle)), (sin, np.sin(angle))):
            assert np.all(np.abs(buf.download(np.float32).reshape(want.shape) - want) <= tol)
            buf.free()


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("one_row,in_place", [(True, False), (False, False), (False, True)])
def test_append(ctx, layout, one_row, in_place):
    heads, kv_heads, D = layout
    rng = np.random.default_rng(21)
    new, first = ([1] * 5, [0, 15, 16, 170, 3]) if one_row else ([1, 40, 0, 7], [0, 9, 4, 111])
    # (A hole under some of the new tokens, and rows behind the last sequence.)
    batch = Batch(rng, 16, new, first, pad=0 if one_row else 2, spare=1, one_row=one_row, holes=[(1, 0, NONE)])
    pool = Pool(ctx, rng, 2, batch.pages, 16, kv_heads, D)
    for layer in range(2):
        pool.fill(layer, np.concatenate([r[r >= 0] for r in batch.owned()]))
    width, row = heads * D, (heads + 2 * kv_heads) * D
    stride = row + 8
    qkv = np.full((batch.rows, stride), 5.0, np.float32)
    qkv[:, :row] = rng.standard_normal((batch.rows, row)) * 10.0 ** rng.uniform(-3, 3, (batch.rows, 1))
    norms = [(1 + 0.5 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)]
    eps = 1e-6
    cos, sin = tables(ctx, D, 512)
    c, s = (t.download(np.float32).reshape(512, D // 2).astype(np.float64) for t in (cos, sin))
    cache, desc = pool.upload(), batch.upload(ctx)
    x, nq, nk = ctx.to_device(qkv), ctx.to_device(norms[0]), ctx.to_device(norms[1])
    q = x if in_place else ctx.to_device(np.full((batch.rows, width), -77.0, np.float32))
    ctx.paged_append(cache, 1, desc, x.ptr, stride, heads, nq.ptr, nk.ptr, eps, cos.ptr, sin.ptr, 512, q.ptr,
                     stride if in_place else width)
    got_q = q.download(np.float32).reshape(batch.rows, -1)[:, :width]
    codes, scales = pool.download()
    want_codes = [p.copy() for p in pool.codes]
    want_scales = [p.view(np.uint16).copy() for p in pool.scales]
    want_q = qkv[:, :width].astype(np.float64) if in_place else np.full((batch.rows, width), -77.0)
    for b, owned in enumerate(batch.owned()):
        for t in range(new[b]):
            i, p = int(batch.starts[b]) + t, first[b] + t
            heads64 = qkv[i, :(heads + kv_heads) * D].astype(np.float64).reshape(-1, D)
            y = heads64 / np.sqrt((heads64 ** 2).mean(1, keepdims=True) + np.float64(np.float32(eps)))
            y = y * np.concatenate([np.tile(norms[0], (heads, 1)), np.tile(norms[1], (kv_heads, 1))]).astype(np.float64)
            low, high = y[:, :D // 2], y[:, D // 2:]
            y = np.concatenate([low * c[p] - high * s[p], high * c[p] + low * s[p]], 1)
            want_q[i] = y[:heads].reshape(-1)
            if owned[p] < 0:
                continue
            for k, values in enumerate((y[heads:].reshape(1, -1).astype(np.float32), qkv[i:i + 1, (heads + kv_heads) * D:row])):
                sc, da = o.quantize_rows(o.Q8, np.ascontiguousarray(values))
                want_codes[k][1, owned[p]] = np.frombuffer(da.tobytes(), np.uint8)
                want_scales[k][1, owned[p]] = np.frombuffer(sc.tobytes(), np.uint16)
    # One rounding to f32 of a value that 64 bits hold.
    assert np.all(np.abs(got_q - want_q) <= np.abs(want_q) * 2.0**-24 * (1 + 1e-6) + 1e-40)
    for k in range(2):
        assert np.array_equal(codes[k], want_codes[k]) and np.array_equal(scales[k], want_scales[k])
    for buf in [x, nq, nk, cos, sin] + ([] if in_place else [q]):
        buf.free()
    pool.free()
    batch.free()


def test_append_leaves_out_positions_past_the_tables(ctx):
    rng = np.random.default_rng(22)
    heads, kv_heads, D = 4, 2, 64
    batch = Batch(rng, 16, [3, 3, 3], [10, 14, 40])
    # Sequence 1 has one page (positions 14, 15 | 16), sequence 2's rotation
    # rows end at 41, sequence 0's first is far past everything.
    batch.tables[1, 1:] = NONE
    batch.first = [4_294_967_290, 14, 40]
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    qkv = rng.standard_normal((9, 8 * D)).astype(np.float32)
    cos, sin = tables(ctx, D, 41)
    ones = ctx.to_device(np.ones(D, np.float32))
    cache, desc = pool.upload(), batch.upload(ctx)
    x, q = ctx.to_device(qkv), ctx.to_device(np.full((9, heads * D), -77.0, np.float32))
    ctx.paged_append(cache, 0, desc, x.ptr, 8 * D, heads, ones.ptr, ones.ptr, 1e-6, cos.ptr, sin.ptr, 41, q.ptr, heads * D)
    got = q.download(np.float32).reshape(9, -1)
    written = (got != -77.0).all(1)
    assert written.tolist() == [False] * 3 + [True] * 3 + [True, False, False]
    codes, scales = pool.download()
    changed = np.flatnonzero((scales[0][0] != NAN16).any(1))
    want = sorted([batch.tables[1, 0] * 16 + 14, batch.tables[1, 0] * 16 + 15, batch.tables[2, 2] * 16 + 8])
    assert changed.tolist() == want
    for buf in (cos, sin, ones, x, q):
        buf.free()
    pool.free()
    batch.free()


def test_append_stores_what_the_flat_append_stores(ctx):
    """The value rows of qwh_kv_append_q8, also with infinities, NaN, zeros
    and values whose scale leaves f16."""
    rng = np.random.default_rng(23)
    heads, kv_heads, D = 2, 2, 128
    batch = Batch(rng, 16, [6], [0])
    pool = Pool(ctx, rng, 1, batch.pages, 16, kv_heads, D)
    qkv = rng.standard_normal((6, 6 * D)).astype(np.float32)
    v = qkv[:, 4 * D:]
    v[1] = 0.0
    v[2, 5], v[3, 70] = np.inf, np.nan
    v[4] *= np.float32(1e9)
    v[5] *= np.float32(1e-7)
    cos, sin = tables(ctx, D, 16)
    ones = ctx.to_device(np.ones(D, np.float32))
    cache, desc = pool.upload(), batch.upload(ctx)
    x, q = ctx.to_device(qkv), ctx.buffer(6 * heads * D * 4)
    ctx.paged_append(cache, 0, desc, x.ptr, 6 * D, heads, ones.ptr, ones.ptr, 1e-6, cos.ptr, sin.ptr, 16, q.ptr, heads * D)
    codes, scales = pool.download()
    width = kv_heads * D
    flat = [ctx.buffer(6 * width // 32), ctx.buffer(6 * width)] * 2
    flat = [ctx.buffer(n) for n in (6 * width // 32, 6 * width, 6 * width // 32, 6 * width)]
    for i in range(6):
        vp = x.ptr + (i * 6 * D + 4 * D) * 4
        ctx.kv_append_q8(vp, vp, width, i, *[f.ptr for f in flat])
    rows = batch.owned()[0]
    assert np.array_equal(codes[1][0, rows], flat[3].download(np.uint8).reshape(6, width))
    assert np.array_equal(scales[1][0, rows], flat[2].download(np.uint16).reshape(6, -1))
    for buf in flat + [cos, sin, ones, x, q]:
        buf.free()
    pool.free()
    batch.free()


# ---------------------------------------------------------------------------
@pytest.mark.parametrize("layers,page_size,kv_heads,D", [(28, 16, 8, 128), (1, 1, 1, 64), (3, 3, 1, 64), (2, 7, 3, 64), (1, 300, 8, 128),
                                                        (5, 64, 2, 192)])
def test_copies(ctx, layers, page_size, kv_heads, D):
    rng = np.random.default_rng(31)
    pages = 24
    pool = Pool(ctx, rng, layers, pages, page_size, kv_heads, D)
    for k in range(2):
        pool.codes[k][:] = rng.integers(0, 256, pool.codes[k].shape)
        pool.scales[k].view(np.uint16)[:] = rng.integers(0, 65536, pool.scales[k].shape)
    cache = pool.upload()
    sets = [([5], [6]), ([3, 3, 3, 3], [4, 5, 6, 7]), ([1, 2], [2, 1]), ([0, 1, 2, 3, 3], [1, 2, 3, 0, 9]),
            ([9, 8, 7], [8, 7, 6]), ([7, 8, 9], [8, 9, 10]), ([4, 4, 5], [4, 5, 6]), ([], [])]
    sets += [(rng.integers(0, pages, n), rng.permutation(pages)[:n]) for n in (5, 12, 24)] + [(np.arange(24), rng.permutation(24))]
    for src, dst in sets:
        ctx.paged_copy(cache, src, dst)
        for planes in (pool.codes, pool.scales):
            for k in range(2):
                whole = planes[k].reshape(layers, pages, -1)
                old = whole.copy()
                for a, b in zip(src, dst):
                    whole[:, b] = old[:, a]
        codes, scales = pool.download()
        for k in range(2):
            assert np.array_equal(codes[k], pool.codes[k]), (src, dst)
            assert np.array_equal(scales[k], pool.scales[k].view(np.uint16)), (src, dst)
    pool.free()


def test_copies_of_many_pages(ctx):
    rng = np.random.default_rng(32)
    pages = 1500
    pool = Pool(ctx, rng, 2, pages, 2, 1, 64)
    for k in range(2):
        pool.codes[k][:] = rng.integers(0, 256, pool.codes[k].shape)
        pool.scales[k].view(np.uint16)[:] = rng.integers(0, 65536, pool.scales[k].shape)
    cache = pool.upload()
    cycle = np.roll(np.arange(pages), 1)
    for src, dst in ((np.arange(pages), cycle), (rng.permutation(pages), rng.permutation(pages)), (np.full(900, 7), np.arange(500, 1400))):
        ctx.paged_copy(cache, src, dst)
        for k in range(2):
            for planes in (pool.codes, pool.scales):
                whole = planes[k].reshape(2, pages, -1)
                whole[:, dst] = whole[:, src]
    codes, scales = pool.download()
    for k in range(2):
        assert np.array_equal(codes[k], pool.codes[k]) and np.array_equal(scales[k], pool.scales[k].view(np.uint16))
    pool.free()


@pytest.mark.parametrize("pages", [65534, 65535, 65536, 70000])
def test_copies_in_pools_of_many_pages(ctx, pages):
    """Either side of the pools whose page numbers fit 16 bits."""
    rng = np.random.default_rng(49)
    pool = Pool(ctx, rng, 1, pages, 1, 1, 64)
    for k in range(2):
        pool.codes[k][:] = rng.integers(0, 256, pool.codes[k].shape)
        pool.scales[k].view(np.uint16)[:] = rng.integers(0, 65536, pool.scales[k].shape)
    cache = pool.upload()
    last = np.arange(pages - 5, pages)
    order = rng.permutation(pages)
    for src, dst in ((last, np.roll(last, 1)), (order[:2500], order[2500:5000]), (np.repeat(order[:300], 5), order[300:1800]),
                     (order[:1300], np.roll(order[:1300], 1))):
        ctx.paged_copy(cache, src, dst)
        for k in range(2):
            for planes in (pool.codes, pool.scales):
                whole = planes[k].reshape(1, pages, -1)
                whole[:, dst] = whole[:, src]
    codes, scales = pool.download()
    for k in range(2):
        assert np.array_equal(codes[k], pool.codes[k]) and np.array_equal(scales[k], pool.scales[k].view(np.uint16))
    pool.free()


def test_copies_from_scale_planes_on_four_bytes(ctx):
    rng = np.random.default_rng(33)
    pages, size = 6, 16 * 64 // 32
    scales = [ctx.to_device(rng.integers(0, 255, pages * size + 4, np.uint8)) for _ in range(2)]
    codes = [ctx.to_device(rng.integers(0, 255, pages * 16 * 64, np.uint8)) for _ in range(2)]
    cache = qa.PagedCache(1, pages, 16, 1, 64, scales[0].ptr + 4, codes[0].ptr, scales[1].ptr + 4, codes[1].ptr)
    before = [b.download(np.uint8) for b in scales]
    ctx.paged_copy(cache, [1, 2], [4, 5])
    for b, old in zip(scales, before):
        want = old.copy()
        want[4:].reshape(pages, -1)[[4, 5]] = want[4:].reshape(pages, -1)[[1, 2]]
        assert np.array_equal(b.download(np.uint8), want)
    for b in scales + codes:
        b.free()


# ---------------------------------------------------------------------------
def test_refusals(ctx):
    rng = np.random.default_rng(41)
    batch = Batch(rng, 16, [2, 1], [5, 6])
    pool = Pool(ctx, rng, 2, batch.pages, 16, 2, 64)
    cache, desc = pool.upload(), batch.upload(ctx)
    buf = ctx.buffer(1 << 16)

    def refused(status, call):
        with pytest.raises(qa.QwhError) as e:
            call()
        assert e.value.status == status, e.value

    def attention(c=cache, layer=0, d=desc, out=buf.ptr, q=buf.ptr + 8192, stride=256, heads=4):
        ctx.paged_attention(c, layer, d, out, q, stride, heads)

    def append(c=cache, layer=0, d=desc, x=buf.ptr, stride=512, heads=4, norm=buf.ptr, eps=1e-6, cos=buf.ptr, positions=64,
               q=buf.ptr + 8192, q_stride=256):
        ctx.paged_append(c, layer, d, x, stride, heads, norm, norm, eps, cos, cos, positions, q, q_stride)

    attention()
    append()
    for call in (attention, append):
        refused(-1, lambda: call(c=None))
        refused(-1, lambda: call(layer=2))
        refused(-1, lambda: call(d=None))
        refused(-7, lambda: call(heads=3))
        refused(-7, lambda: call(heads=0))
        refused(-1, lambda: call(q=None))
        refused(-1, lambda: call(q=buf.ptr + 8196))
        bad = qa.PagedCache(2, batch.pages, 16, 2, 96, *[b.ptr for b in pool.buffers])
        refused(-7, lambda: call(c=bad))
        wide = qa.PagedCache(2, batch.pages, 16, 2, 512, *[b.ptr for b in pool.buffers])
        refused(-3, lambda: call(c=wide))
    refused(-7, lambda: attention(stride=252))
    refused(-1, lambda: attention(stride=257))
    refused(-1, lambda: attention(out=None))
    refused(-1, lambda: attention(out=buf.ptr + 4))
    refused(-7, lambda: append(stride=508))
    refused(-7, lambda: append(q_stride=252))
    refused(-1, lambda: append(x=None))
    refused(-1, lambda: append(norm=None))
    refused(-1, lambda: append(cos=None))
    refused(-1, lambda: append(eps=float("nan")))
    refused(-1, lambda: append(eps=-1.0))
    refused(-1, lambda: append(q=buf.ptr))  # in place, with another stride than the rows'
    short = qa.PagedBatch(2, 1, 1, None, desc.first, desc.tables)
    refused(-7, lambda: attention(d=short))
    refused(-1, lambda: ctx.paged_copy(cache, [0, 1], [2, 2]))
    refused(-1, lambda: ctx.paged_copy(cache, [batch.pages], [0]))
    refused(-1, lambda: ctx.paged_copy(cache, [0], [batch.pages]))
    refused(-1, lambda: ctx.paged_copy(None, [0], [1]))
    with pytest.raises(ValueError):
        ctx.paged_copy(cache, [0, 1], [2])
    refused(-7, lambda: ctx.rope_tables(63, 4, 1e6, buf.ptr, buf.ptr))
    refused(-1, lambda: ctx.rope_tables(64, 4, 0.0, buf.ptr, buf.ptr))
    refused(-1, lambda: ctx.rope_tables(64, 4, 1e6, None, buf.ptr))
    # Nothing to do is no error, whatever else is missing.
    ctx.paged_attention(cache, 0, qa.PagedBatch(), 0, 0, 0, 4)
    ctx.paged_attention(cache, 0, qa.PagedBatch(2, 0, 0, desc.row_starts), 0, 0, 0, 4)
    ctx.paged_copy(cache, [], [])
    ctx.rope_tables(64, 0, 1e6, 0, 0)
    buf.free()
    pool.free()
    batch.free()


def test_two_contexts_at_once(ctx):
    """Their streams run side by side on one pool that both only read."""
    rng = np.random.default_rng(45)
    other = qa.Context(0)
    heads, kv_heads, D = 16, 8, 128
    batches = [Batch(rng, 16, [1] * 9, [37 * i for i in range(9)]), Batch(rng, 16, [300, 2, 1], [1000, 700, 0])]
    pools, query, out = [], [], []
    for c, batch in zip((ctx, other), batches):
        pool = Pool(c, rng, 1, batch.pages, 16, kv_heads, D)
        pool.fill(0, np.concatenate(batch.owned()))
        q = rng.standard_normal((batch.rows, heads * D)).astype(np.float32)
        pools.append((pool, pool.upload(), batch.upload(c)))
        query.append((q, c.to_device(q)))
        out.append(c.buffer(q.nbytes))
    for _ in range(20):
        for c, (_, cache, desc), (_, q), o_ in zip((ctx, other), pools, query, out):
            c.paged_attention(cache, 0, desc, o_.ptr, q.ptr, heads * D, heads)
    for (pool, _, _), batch, (q, qbuf), o_ in zip(pools, batches, query, out):
        want, bound = reference(pool, 0, batch, q, heads)
        assert np.all(np.abs(o_.download(np.float32).reshape(want.shape) - want) <= bound)
        for x in (qbuf, o_):
            x.free()
        pool.free()
        batch.free()
    other.close()


def test_a_pool_s_last_page_and_the_same_page_in_two_tables(ctx):
    """Sequences that share pages (a prompt's), the pool's last among them."""
    rng = np.random.default_rng(46)
    batch = Batch(rng, 16, [1, 4, 40], [50, 50, 50])
    shared = np.setdiff1d(np.arange(batch.pages), batch.tables.reshape(-1))[:1]
    for b in range(3):
        batch.tables[b, 1] = batch.pages - 1
        batch.tables[b, 0] = shared[0]
    pool = Pool(ctx, rng, 1, batch.pages, 16, 2, 128)
    pool.fill(0, np.unique(np.concatenate(batch.owned())))
    query = rng.standard_normal((batch.rows, 4 * 128)).astype(np.float32)
    got = attend(ctx, pool, 0, batch, query, 4)
    want, bound = reference(pool, 0, batch, query, 4)
    assert np.all(np.abs(got - want) <= bound)


# ---------------------------------------------------------------------------
def test_a_server_s_steps_with_a_fork(ctx):
    """A prompt appended and attended as one chunk, its pages shared by three
    branches (the last, half-filled one copied), then steps of one token for
    all branches: logits from the attention, tokens drawn from them, each
    token's rows appended. Against the same in 64 bits over flat caches."""
    rng = np.random.default_rng(51)
    heads, kv_heads, D, page_size, vocab, prompt, branches, steps = 4, 2, 64, 16, 300, 37, 3, 6
    width, kv, row = heads * D, kv_heads * D, (heads + 2 * kv_heads) * D
    pages, table_pages = 32, 4
    pool = Pool(ctx, rng, 2, pages, page_size, kv_heads, D)
    cache = pool.upload()
    embed = rng.standard_normal((vocab, row)).astype(np.float32)  # a token's projections
    head = (0.6 * rng.standard_normal((vocab, width))).astype(np.float32)
    head_matrix = ctx.matrix_upload(qa.FORMAT_F32, vocab, width, None, head)
    ones = ctx.to_device(np.ones(D, np.float32))
    cos, sin = tables(ctx, D, table_pages * page_size)
    c, s = (t.download(np.float32).reshape(-1, D // 2).astype(np.float64) for t in (cos, sin))
    rule = (0.9, 40, 0.95, 0.01)
    params = ctx.to_device(np.frombuffer(bytes(qa.Sampling(*rule)) * branches, np.uint8))

    def norm_rotate(x, p):
        y = x.reshape(-1, D).astype(np.float64)
        y = y / np.sqrt((y ** 2).mean(1, keepdims=True) + np.float64(np.float32(1e-6)))
        low, high = y[:, :D // 2], y[:, D // 2:]
        return np.concatenate([low * c[p] - high * s[p], high * c[p] + low * s[p]], 1)

    def stored(x):
        sc, da = o.quantize_rows(o.Q8, np.ascontiguousarray(x.reshape(1, -1), np.float32))
        sc = np.frombuffer(sc.tobytes(), np.float16).astype(np.float64)
        return ((np.frombuffer(da.tobytes(), np.uint8).astype(np.float64) - 128).reshape(-1, 64) * sc[:, None]).reshape(-1)

    class Flat:
        def __init__(self):
            self.k, self.v = np.zeros((0, kv)), np.zeros((0, kv))

        def token(self, token):
            p, x = len(self.k), embed[token]
            q = norm_rotate(x[:width], p).astype(np.float32).astype(np.float64)
            self.k = np.concatenate([self.k, stored(norm_rotate(x[width:width + kv], p))[None]])
            self.v = np.concatenate([self.v, stored(x[width + kv:])[None]])
            out = np.zeros(width)
            for h in range(heads):
                at = slice(h // 2 * D, (h // 2 + 1) * D)
                w = self.k[:, at] @ q[h] / 8.0
                w = np.exp(w - w.max())
                out[h * D:(h + 1) * D] = w @ self.v[:, at] / w.sum()
            return out

    def draw(logits, u):
        order = np.lexsort((np.arange(vocab), -logits))[:rule[1]]
        w = np.exp((logits[order] - logits[order[0]]) / np.float64(np.float32(rule[0])))
        w = w[:int(np.sum(np.cumsum(w) - w < np.float64(np.float32(rule[2])) * w.sum()))]
        w = w[w >= np.float64(np.float32(rule[3]))]
        return order[int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right"))]

    bufs = []

    def dev(a):
        bufs.append(ctx.to_device(np.ascontiguousarray(a)))
        return bufs[-1]

    # The prompt, through layer 1 of the pool.
    tokens = rng.integers(0, vocab, prompt)
    table = np.array([20, 3, 11, NONE], np.uint32)
    batch = qa.PagedBatch(1, prompt, table_pages, dev(np.array([0, prompt], np.uint32)).ptr, dev(np.zeros(1, np.uint32)).ptr,
                          dev(table).ptr)
    x, q, out = dev(embed[tokens]), ctx.buffer(prompt * width * 4), ctx.buffer(prompt * width * 4)
    bufs += [q, out]
    ctx.paged_append(cache, 1, batch, x.ptr, row, heads, ones.ptr, ones.ptr, 1e-6, cos.ptr, sin.ptr, 64, q.ptr, width)
    ctx.paged_attention(cache, 1, batch, out.ptr, q.ptr, width, heads)
    got = out.download(np.float32).reshape(prompt, width)
    flat = Flat()
    want = np.array([flat.token(t) for t in tokens])
    assert np.all(np.abs(got - want) <= 2e-5 * np.abs(want).max())
    # Three branches share the two full pages; the third page is copied.
    ctx.paged_copy(cache, [11, 11], [5, 6])
    branch_tables = np.array([[20, 3, own, NONE] for own in (11, 5, 6)], np.uint32)
    flats = [Flat() for _ in range(branches)]
    for f in flats:
        f.k, f.v = flat.k.copy(), flat.v.copy()
    current = np.array([7, 8, 9])
    q2, out2, logits, ids = (ctx.buffer(branches * n * 4) for n in (width, width, vocab, 1))
    bufs += [q2, out2, logits, ids]
    tables_dev = dev(branch_tables)
    for step in range(steps):
        u = rng.random(branches, np.float32)
        batch = qa.PagedBatch(branches, branches, table_pages, None, dev(np.full(branches, prompt + step, np.uint32)).ptr,
                              tables_dev.ptr)
        x = dev(embed[current])
        ctx.paged_append(cache, 1, batch, x.ptr, row, heads, ones.ptr, ones.ptr, 1e-6, cos.ptr, sin.ptr, 64, q2.ptr, width)
        ctx.paged_attention(cache, 1, batch, out2.ptr, q2.ptr, width, heads)
        ctx.linear(head_matrix, out2.ptr, width, branches, logits.ptr)
        ctx.sample_rows(logits.ptr, branches, vocab, params.ptr, dev(u).ptr, ids.ptr)
        drawn = ids.download(np.uint32)
        want = np.array([f.token(t) for f, t in zip(flats, current)])
        got = out2.download(np.float32).reshape(branches, width)
        assert np.all(np.abs(got - want) <= 2e-5 * np.abs(want).max())
        host = logits.download(np.float32).reshape(branches, vocab).astype(np.float64)
        assert np.all(np.abs(host - want @ head.T.astype(np.float64)) <= 1e-3)
        assert drawn.tolist() == [draw(host[b], np.float64(u[b])) for b in range(branches)]
        current = drawn
    for b in bufs + [ones, cos, sin, params]:
        b.free()
    ctx.matrix_release(head_matrix)
    pool.free()

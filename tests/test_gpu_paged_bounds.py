"""The paged attention stays within its buffers and its call's records, and
later calls are right, whatever earlier calls left in the context's scratch
memory."""
import numpy as np
import pytest

import qwenscriber_amd as qa
from test_gpu_paged import WIDE, Batch, Pool, reference

pytestmark = pytest.mark.gpu


def test_arrays_off_four_bytes_are_refused(ctx):
    """On the host: nothing is launched."""
    buf = ctx.buffer(1 << 16)
    cache = qa.PagedCache(1, 4, 16, 2, 64, *[buf.ptr] * 4)

    def refused(arrays=(0, 0, 0), floats=(0, 0, 0, 0), appends=True, attends=True):
        desc = qa.PagedBatch(1, 2, 4, *[buf.ptr + at for at in arrays])
        norms = [buf.ptr + at for at in floats]
        calls = []
        if appends:
            calls.append(lambda: ctx.paged_append(cache, 0, desc, buf.ptr, 512, 4, norms[0], norms[1], 1e-6, norms[2], norms[3], 64,
                                                  buf.ptr + 8192, 256))
        if attends:
            calls.append(lambda: ctx.paged_attention(cache, 0, desc, buf.ptr, buf.ptr + 8192, 256, 4))
        for call in calls:
            with pytest.raises(qa.QwhError) as e:
                call()
            assert e.value.status == -1 and "4-byte" in str(e.value)

    for k in range(3):
        refused(arrays=[2 * (i == k) for i in range(3)])
    for k in range(4):
        refused(floats=[(i == k) for i in range(4)], attends=False)
    buf.free()


class Call:
    """A batch over its own pool, its rows between guard rows."""

    def __init__(self, ctx, rng, new, first, spare, layout=(4, 2, 64)):
        self.ctx, (self.heads, kv_heads, D) = ctx, layout
        self.batch = Batch(rng, 16, new, first, spare=spare)
        self.pool = Pool(ctx, rng, 1, self.batch.pages, 16, kv_heads, D)
        self.pool.fill(0, np.concatenate(self.batch.owned()))
        self.width = self.heads * D
        self.query = rng.standard_normal((self.batch.rows, self.width)).astype(np.float32)
        self.want, self.bound = reference(self.pool, 0, self.batch, self.query, self.heads)
        self.cache = self.pool.upload()

    def run(self, starts):
        """The rows that a call with these starts leaves (guards checked)."""
        ctx, n = self.ctx, self.batch.rows
        good, self.batch.starts = self.batch.starts, np.asarray(starts, np.uint32)
        desc = self.batch.upload(ctx)
        self.batch.starts = good
        q, out = ctx.to_device(self.query), ctx.to_device(np.full((n + 2, self.width), -77.0, np.float32))
        ctx.paged_attention(self.cache, 0, desc, out.ptr + 4 * self.width, q.ptr, self.width, self.heads)
        got = out.download(np.float32).reshape(n + 2, self.width)
        assert np.all(got[[0, -1]] == -77.0)
        for x in (q, out):
            x.free()
        self.batch.free()
        return got[1:-1]

    def check(self):
        assert np.all(np.abs(self.run(self.batch.starts) - self.want) <= self.bound)

    def free(self):
        self.pool.free()


def test_falling_starts_after_calls_of_the_other_form():
    """In a fresh context, whose scratch memory is as small as its calls need:
    calls for few rows, for many rows and for both, each with well-formed and
    with falling starts, one after the other."""
    rng = np.random.default_rng(71)
    with qa.Context(0) as ctx:
        first = [200, 150, 300]
        few = Call(ctx, rng, [3, 2, 3], first, 0)
        both = Call(ctx, rng, [3, 40, 50], first, WIDE)
        many = Call(ctx, rng, [33, 40, 50], first, WIDE)
        falling = {few: ([0, 5, 2, 8], [5, 1, 3, 2], [8, 8, 8, 0]), both: ([0, 60, 20, 93], [93, 0, 93, 0], [7, 3, 93, 5]),
                   many: ([0, 100, 40, 123], [123, 0, 123, 0], [70, 60, 50, 40])}
        for call in (few, many, few, both, few, many, both):
            call.check()
            for starts in falling[call]:
                call.run(starts)
        for call in (both, many, few):
            call.check()
            call.free()

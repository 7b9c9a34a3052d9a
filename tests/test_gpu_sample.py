"""qwh_sample_rows and qwh_decoder_sample against the definition in 64 bits:
the drawn ids have to be equal."""
import numpy as np
import pytest

import qwenscriber_amd as qa
from util import random_norms, set_norms

pytestmark = pytest.mark.gpu
FLT_MAX = np.finfo(np.float32).max


def definition(logits, rule, u):
    """One row's token (include/qwhip.h qwh_sample_rows)."""
    heat, top_k, top_p, min_p = np.float64(np.float32(rule[0])), rule[1], np.float64(np.float32(rule[2])), np.float64(np.float32(rule[3]))
    l = np.where(np.isnan(logits), -np.inf, logits.astype(np.float64))
    order = np.lexsort((np.arange(len(l)), -l))
    top = l[order[0]]
    if top == -np.inf:
        return 0
    if not heat > 0:
        return order[0]
    with np.errstate(all="ignore"):
        w = np.exp(np.where(l[order] == top, 0.0, np.where(l[order] == -np.inf, -np.inf, (l[order] - top) / heat)))
    if top == np.inf:
        w = (l[order] == np.inf).astype(np.float64)
    if top_k > 0:
        w = w[:top_k]
    if top_p < 1:
        w = w[:max(1, int(np.sum(np.cumsum(w) - w < top_p * w.sum())))]
    if min_p > 0:
        w = w[w >= min(min_p, 1.0)]
    run = np.cumsum(w)
    u = 0.0 if not u > 0 else float(u)
    if u >= 1:
        return order[np.flatnonzero(w)[-1]]
    return order[int(np.searchsorted(run, u * run[-1], side="right"))]


def sample(ctx, logits, rules, u):
    rows, count = logits.shape
    params = np.frombuffer(b"".join(bytes(qa.Sampling(*r)) for r in rules), np.uint8)
    bufs = [ctx.to_device(a) for a in (np.ascontiguousarray(logits, np.float32), params, np.asarray(u, np.float32))]
    # (A guard word behind the ids.)
    ids = ctx.to_device(np.full(rows + 1, 12345678, np.uint32))
    ctx.sample_rows(bufs[0].ptr, rows, count, bufs[1].ptr, bufs[2].ptr, ids.ptr)
    got = ids.download(np.uint32)
    for b in bufs + [ids]:
        b.free()
    assert got[rows] == 12345678
    return got[:rows]


def check(ctx, logits, rules, u):
    got = sample(ctx, logits, rules, u)
    want = [definition(logits[r], rules[r], np.float32(u[r])) for r in range(len(rules))]
    assert got.tolist() == [int(w) for w in want]


OFF = (1.0, 0, 1.0, 0.0)
RULES = [OFF, (0.8, 50, 0.95, 0.02), (0.0, 0, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (1.3, 0, 1.0, 0.05), (0.7, 20, 1.0, 0.0),
         (2.0, 1000, 0.5, 0.0), (0.3, 5, 0.99, 0.5), (1.0, 1, 1.0, 0.0), (5.0, 0, 0.999, 1e-4), (1.0, 3, 0.0001, 0.0),
         (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 7.0), (0.05, 0, 1.0, 0.0), (100.0, 70, 1.0, 0.0)]


@pytest.mark.parametrize("count", [1, 2, 63, 64, 1000, 1025, 4096, 4099, 32000, 151936])
def test_rules(ctx, count):
    rng = np.random.default_rng(count)
    for spread in (0.3, 3.0):
        logits = (spread * rng.standard_normal((len(RULES), count))).astype(np.float32)
        for r in range(len(RULES)):
            logits[r, rng.integers(0, count, 8)] += rng.uniform(3, 9, 8).astype(np.float32)
        check(ctx, logits, RULES, rng.random(len(RULES), np.float32))


def test_many_rows_and_draws(ctx):
    rng = np.random.default_rng(1)
    rows = 300
    logits = (2.5 * rng.standard_normal((rows, 1500))).astype(np.float32)
    check(ctx, logits, [RULES[r % len(RULES)] for r in range(rows)], rng.random(rows, np.float32))


@pytest.mark.parametrize("count", [7, 5000, 20000])
def test_rows_of_equal_logits(ctx, count):
    """Ties go to the lower index, also where one step of the histogram holds
    more tokens than its list."""
    rng = np.random.default_rng(2)
    logits = np.full((len(RULES), count), 3.25, np.float32)
    check(ctx, logits, RULES, rng.random(len(RULES), np.float32))
    # Two levels, and levels a last bit apart.
    logits[:, ::3] = -1.0
    check(ctx, logits, RULES, rng.random(len(RULES), np.float32))
    logits[:, 1::3] = np.nextafter(np.float32(3.25), np.float32(0))
    check(ctx, logits, RULES, rng.random(len(RULES), np.float32))


def test_a_narrow_row(ctx):
    """Every logit within one step of the histogram, all different."""
    rng = np.random.default_rng(3)
    logits = (10.0 + 1e-3 * rng.standard_normal((len(RULES), 30000))).astype(np.float32)
    check(ctx, logits, RULES, rng.random(len(RULES), np.float32))


def test_masked_infinite_and_missing_logits(ctx):
    rng = np.random.default_rng(4)
    base = (2 * rng.standard_normal(3000)).astype(np.float32)
    rows, rules, u = [], [], []

    def add(change, rule=OFF, number=None):
        row = base.copy()
        change(row)
        rows.append(row)
        rules.append(rule)
        u.append(rng.random() if number is None else number)

    for rule in (OFF, RULES[1], RULES[2], RULES[3], RULES[4], (1.0, 2000, 0.99, 0.0)):
        add(lambda r: r.__setitem__(slice(5, None), -np.inf), rule)
        add(lambda r: r.__setitem__(slice(5, None), -FLT_MAX), rule)
        add(lambda r: r.__setitem__(slice(0, 2990), np.nan), rule)
        add(lambda r: r.__setitem__(0, np.nan), rule)
        add(lambda r: r.__setitem__([17, 900, 901], np.inf), rule)
        add(lambda r: r.__setitem__(slice(None), -np.inf), rule)
        add(lambda r: r.__setitem__(slice(None), np.nan), rule)
        add(lambda r: r.__setitem__(slice(None), -FLT_MAX), rule)
        add(lambda r: r.__setitem__(slice(None), FLT_MAX), rule)
        add(lambda r: r.__setitem__(slice(1, 400), FLT_MAX), rule)
        add(lambda r: r.__setitem__(slice(None), np.where(np.arange(3000) % 2, 0.0, -0.0)), rule)
        add(lambda r: r.__setitem__(slice(0, 2999), -np.inf), rule)
    check(ctx, np.array(rows), rules, u)


def test_numbers_at_the_ends(ctx):
    rng = np.random.default_rng(5)
    numbers = [0.0, -0.5, np.nan, 2.0**-149, 1 - 2.0**-24, 1.0, 3.0, np.inf, 0.5]
    for rule in (OFF, RULES[1], RULES[3], RULES[4], RULES[5], (1.0, 0, np.nan, np.nan), (np.nan, 0, 1.0, 0.0), (-1.0, 0, 1.0, 0.0),
                 (1e-40, 0, 1.0, 0.0), (np.inf, 0, 1.0, 0.0), (1.0, 2**32 - 1, 2.0, -1.0), (1.0, 200, 1.0, 0.0)):
        logits = (2 * rng.standard_normal((len(numbers), 200))).astype(np.float32)
        check(ctx, logits, [rule] * len(numbers), numbers)


def test_a_draw_follows_its_weights(ctx):
    """Numbers spread evenly over [0, 1) give each of a few tokens its share."""
    logits = np.log(np.array([0.5, 0.25, 0.125, 0.0625, 0.0625], np.float64)).astype(np.float32)
    rows = 4096
    u = (np.arange(rows) + 0.5) / rows
    got = sample(ctx, np.tile(logits, (rows, 1)), [OFF] * rows, u)
    share = np.bincount(got, minlength=5) / rows
    assert np.all(np.abs(share - [0.5, 0.25, 0.125, 0.0625, 0.0625]) <= 2 / rows)


def test_rows_of_many_parts(ctx):
    """More parts of a row than the second pass has threads."""
    rng = np.random.default_rng(8)
    rules = [OFF, (1.0, 0, 0.7, 0.0), (1.5, 100000, 1.0, 0.0)]
    logits = (2.0 * rng.standard_normal((3, 4300001))).astype(np.float32)
    logits[:, rng.integers(0, logits.shape[1], 5)] += 6
    check(ctx, logits, rules, rng.random(3, np.float32))


def test_more_parts_than_one_launch_holds(ctx):
    rng = np.random.default_rng(9)
    logits = rng.standard_normal((40000, 5)).astype(np.float32)
    check(ctx, logits, [RULES[r % len(RULES)] for r in range(40000)], rng.random(40000, np.float32))


def test_two_contexts_at_once(ctx):
    """Their streams run side by side; each has its own scratch memory."""
    rng = np.random.default_rng(10)
    other = qa.Context(0)
    logits = (2.5 * rng.standard_normal((len(RULES), 50000))).astype(np.float32)
    u = rng.random(len(RULES), np.float32)
    params = np.frombuffer(b"".join(bytes(qa.Sampling(*r)) for r in RULES), np.uint8)
    bufs = [[c.to_device(a) for a in (logits, params, u)] + [c.buffer(4 * len(RULES))] for c in (ctx, other)]
    for _ in range(20):
        for c, (l, p, n, ids) in zip((ctx, other), bufs):
            c.sample_rows(l.ptr, len(RULES), logits.shape[1], p.ptr, n.ptr, ids.ptr)
    want = [int(definition(logits[r], RULES[r], u[r])) for r in range(len(RULES))]
    for b in bufs:
        assert b[3].download(np.uint32).tolist() == want
        for x in b:
            x.free()
    other.close()


def test_a_decoder_s_steps_beside_larger_draws(ctx):
    """A decoder's captured step between calls that grow the context's
    scratch memory."""
    config = dict(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=1000, max_positions=32, eps=1e-6,
                  theta=1e6)

    def run(between):
        c = qa.Context(0)
        decoder = qa.Decoder(c, batch=3, **config)
        decoder.init_synthetic(9)
        set_norms(decoder, random_norms(config, 3), 2)
        tokens, out = np.array([5, 6, 7], np.uint32), []
        for step in range(6):
            decoder.forward(tokens, want_logits=True)
            if between:
                big = np.zeros((8 << step, 30000), np.float32)
                assert sample(c, big, [(0.0, 0, 1.0, 0.0)] * len(big), np.zeros(len(big))).tolist() == [0] * len(big)
            out.append([decoder.logits(b) for b in range(3)])
            tokens = decoder.sample(qa.Sampling(0.7, 40, 0.9, 0.0), [0.2, 0.5, 0.8])
        decoder.close()
        c.close()
        return np.array(out)

    assert np.array_equal(run(False), run(True))


def test_greedy_is_the_argmax(ctx):
    rng = np.random.default_rng(6)
    logits = np.round(3 * rng.standard_normal((20, 5000))).astype(np.float32)
    got = sample(ctx, logits, [(0.0, 0, 1.0, 0.0)] * 20, np.zeros(20))
    buf, ids = ctx.to_device(logits), ctx.buffer(80)
    ctx.argmax_rows(buf.ptr, 20, 5000, ids.ptr)
    assert np.array_equal(got, ids.download(np.uint32))
    buf.free()
    ids.free()


def test_refusals(ctx):
    buf = ctx.buffer(1024)

    def refused(status, *args):
        with pytest.raises(qa.QwhError) as e:
            ctx.sample_rows(*args)
        assert e.value.status == status

    p = buf.ptr
    refused(-1, None, 1, 4, p, p, p)
    refused(-1, p, 1, 4, None, p, p)
    refused(-1, p, 1, 4, p, None, p)
    refused(-1, p, 1, 4, p, p, None)
    refused(-1, p + 2, 1, 4, p, p, p)
    refused(-1, p, 1, 0, p, p, p)
    refused(-9, p, 65536, 4, p, p, p)
    refused(-9, p, 1, 2**26 + 1, p, p, p)
    ctx.sample_rows(0, 0, 4, 0, 0, 0)
    buf.free()


def test_decoder_sample(ctx):
    config = dict(hidden=256, layers=2, heads=4, kv_heads=2, head_dim=128, ffn=512, vocab=1000, max_positions=32, eps=1e-6,
                  theta=1e6)
    decoder = qa.Decoder(ctx, batch=3, **config)
    decoder.init_synthetic(9)
    set_norms(decoder, random_norms(config, 3), 2)
    rng = np.random.default_rng(7)
    tokens = np.array([5, 6, 7], np.uint32)
    rules = [(0.8, 50, 0.95, 0.0), (1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0)]
    for _ in range(4):
        decoder.forward(tokens, want_logits=True)
        u = rng.random(3, np.float32)
        got = decoder.sample([qa.Sampling(*r) for r in rules], u)
        logits = [decoder.logits(b) for b in range(3)]
        assert got.tolist() == [int(definition(logits[b], rules[b], u[b])) for b in range(3)]
        tokens = got
    # One record for all; after a prompt, the prompt's logits.
    decoder.reset()
    first = decoder.prefill(1, [1, 2, 3])
    assert decoder.sample(qa.Sampling(0.0, 0, 1.0, 0.0), [0.0] * 3)[1] == first
    with pytest.raises(ValueError):
        decoder.sample(qa.Sampling(1.0, 0, 1.0, 0.0), [0.5])
    decoder.close()


@pytest.mark.parametrize("batch,vocab", [(1, 2**26 + 64), (65536, 64)])
def test_decoder_sample_refuses_what_sample_rows_refuses(ctx, batch, vocab):
    config = dict(hidden=64, layers=1, heads=1, kv_heads=1, head_dim=64, ffn=64, vocab=vocab, max_positions=1, eps=1e-6, theta=1e6)
    decoder = qa.Decoder(ctx, batch=batch, **config)
    with pytest.raises(qa.QwhError) as e:
        decoder.sample(qa.Sampling(1.0, 0, 1.0, 0.0), np.zeros(batch))
    assert e.value.status == -9
    decoder.close()

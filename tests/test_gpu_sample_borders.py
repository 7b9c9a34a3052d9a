"""qwh_sample_rows where a rule or a number falls on a border of two tokens:
the weights that count are all equal, so every sum is a whole number of them
and the definition says which side it is."""
import numpy as np
import pytest

from test_gpu_sample import check

pytestmark = pytest.mark.gpu

NUMBERS = [0.0, 0.125, 0.25, 0.375, 0.5, 0.625, 0.75, 0.875, 1 - 2.0**-24]


def level(rng, count, kept):
    """A row of `count` equal logits, and all but `kept` of its places."""
    top = rng.choice([-3.0, 0.0, 0.7, 12.3, 800.1]) + rng.uniform(-1, 1)
    row = np.full(count, top, np.float32)
    low = rng.permutation(count)[kept:]
    return row, low


@pytest.mark.parametrize("count", [2, 4, 6, 14, 96, 256, 264, 4096, 5000, 20000, 60000, 151936])
@pytest.mark.parametrize("heat", [0.3, 0.8, 1.0, 2.5])
def test_equal_weights(ctx, count, heat):
    """All of a row, or those that top-k, min-p or a missing rest leave."""
    rng = np.random.default_rng(count)
    logits, rules, u = [], [], []
    for top_p in (0.125, 0.25, 0.5, 0.75, 1.0):
        for number in NUMBERS:
            kept = count if rng.random() < 0.3 else max(1, count // 2) // 8 * 8 or count
            row, low = level(rng, count, kept)
            way = rng.integers(0, 3)
            top_k, min_p = 0, 0.0
            if way == 0:
                row[low] = -np.inf
            elif way == 1:  # cut by top-k: of the equal ones the first
                row[low] -= np.float32(heat)
                top_k = kept
            else:
                row[low] = -np.inf
                min_p = 0.9
            logits.append(row)
            rules.append((heat, int(top_k), top_p, min_p))
            u.append(number)
    check(ctx, np.array(logits), rules, np.array(u, np.float32))


@pytest.mark.parametrize("count", [6, 300, 30000])
def test_min_p_leaves_equal_weights(ctx, count):
    """A lower level, which min-p drops."""
    rng = np.random.default_rng(count)
    logits, rules, u = [], [], []
    for number in NUMBERS:
        row, low = level(rng, count, count // 2)
        row[low] -= 1.0
        logits.append(row)
        rules.append((1.0, 0, 1.0, 0.5))
        u.append(number)
    check(ctx, np.array(logits), rules, np.array(u, np.float32))

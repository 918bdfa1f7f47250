"""The paged attention's splits along the keys and the three ways they are joined:
by the last block of a tile (up to 16 splits of few rows), by a launch of their own
(more of them, or those of the 128-row kernel). The plain forms and the bound are
those of test_gpu_paged.py; test_paged_plans.py checks on the CPU that each case
here is cut into as many as it says.
"""

import copy
import functools

import numpy as np
import pytest

from test_gpu_paged import Case, attend, check, ctx, store  # noqa: F401 (ctx: the fixture)

pytestmark = pytest.mark.gpu

# splits, storage, counts, lengths, kv, group, width: of the 128-row kernel
CUT_CHUNKS = [
    (2, "BF16", (80,), (4160,), 192, 1, 16),
    (3, "F16", (200, 70), (6200, 100), 64, 1, 64),
    (3, "E4M3", (100,), (6200,), 128, 1, 16),
    (3, "BF16", (66,), (6200,), 64, 2, 96),
    (5, "E4M3", (90, 1), (10300, 300), 48, 1, 16),
    (5, "F16", (70,), (10300,), 80, 1, 16),
    (13, "F16", (100,), (26700,), 32, 1, 16),
    (16, "BF16", (67,), (33000,), 32, 1, 16),
]
# splits, storage, counts, lengths, kv, group, width: of the kernels for few rows
CUT_ROWS = [
    (2, "E4M3", (1,), (300,), 2, 1, 64),
    (3, "F16", (1, 1), (700, 20), 2, 4, 64),
    (5, "F32", (5,), (1200,), 2, 1, 80),
    (13, "E4M3", (3,), (3300,), 1, 2, 128),
    (16, "BF16", (2,), (4000,), 1, 1, 64),
    (17, "F16", (1,), (4300,), 1, 1, 64),
    (33, "E4M3", (4,), (8400,), 1, 1, 128),
    (33, "F32", (1,), (8400,), 1, 2, 64),
]
PAGE = 64


@functools.lru_cache(maxsize=1)
def level(given):
    """The case with scores of one size everywhere, channel 0 of the keys ten times smaller
    and added to the scores as it is."""
    _, storage, counts, lengths, kv, group, width = given
    case = Case(storage, counts, lengths, kv, group, width, PAGE, seed=131)
    case.q[:, ::width] = 1.0 / case.scale
    case.key_rows[..., 0] *= np.float32(0.1)
    return case


def lifted(given, lifts, floor=0.0):
    """A case whose scores are lifted by lifts[i] in the i-th of its splits' spans, and by floor everywhere."""
    case = copy.copy(level(given))
    splits, longest = given[0], max(case.lengths)
    span = (longest // splits + 64) // 64 * 64
    case.key_rows = case.key_rows.copy()
    for s, n in enumerate(case.lengths):
        for block in range(-(-n // PAGE)):
            lift = lifts[min(block * PAGE // span, splits - 1) % len(lifts)] + floor
            case.key_rows[case.table[s, block], :, :, 0] += np.float32(lift)
    case.keys, case.key_exponents = store(case.key_rows, case.storage)
    return case


def named(given):
    return f"{given[0]}-{given[1]}"


@pytest.mark.parametrize("lifts", [(0.0, 2.0, 0.0), (0.0, 1.0, 2.0, 3.0), (3.0, -1.0, 0.0)], ids=str)
@pytest.mark.parametrize("given", CUT_CHUNKS + CUT_ROWS, ids=named)
def test_every_split_counts_once(ctx, given, lifts):  # noqa: F811
    # Every split holds a share of each row's weight that the others do not hide.
    check(ctx, lifted(given, lifts))


@pytest.mark.parametrize("floor", [-160.0, 160.0])
@pytest.mark.parametrize("given", CUT_CHUNKS[1::3] + CUT_ROWS, ids=named)
def test_scores_far_below_and_above_zero(ctx, given, floor):  # noqa: F811
    # exp2 of such a score is no fp32 number: only differences of scores may be taken.
    check(ctx, lifted(given, (0.0, 1.0, 0.5), floor))


@pytest.mark.parametrize("given", [g for g in CUT_CHUNKS + CUT_ROWS if g[0] in (3, 5, 17, 33)], ids=named)
def test_a_value_that_is_nan_in_a_faint_split(ctx, given):  # noqa: F811
    # A weight of 2^-290 times NaN is NaN, as within a split: the rows that see such a
    # value are not finite in its channel, and finite in the others.
    case = lifted(given, (-200.0,) + (0.0,) * (given[0] - 1))
    case.value_rows = case.value_rows.copy()
    case.value_rows[case.table[0, 0], :, 3, 5] = np.nan
    case.quantise()
    got = attend(ctx, case).reshape(case.rows, -1, case.width)[:case.counts[0]]
    assert np.isnan(got[:, :, 5]).all()
    assert np.isfinite(np.delete(got, 5, 2)).all()

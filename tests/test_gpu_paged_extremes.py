"""The paged attention at the ends of its numbers: E4M3 rows whose powers of two lie
far apart, every exponent byte, and operands whose product leaves fp32 (the plain
forms are those of test_gpu_paged.py).

Where all scores are equal the weights are 1/n exactly, and a row is a mean of
what its keys' value rows stand for: every channel of its own is off by no more
than the fp32 sum, Σ_j |v_jc|/n · (n + 16)·2^-24, whatever other channels and rows
hold. (The 16-bit parts of a weight lose nothing here: the largest weight of a
row is a power of two, and a smaller one is none of a row's.)
"""

import numpy as np
import pytest

from test_gpu_paged import Case, attend, check, ctx, e4m3_values  # noqa: F401 (ctx: the fixture)

pytestmark = pytest.mark.gpu

SHAPES = {
    # counts, lengths, kv, group, width
    "step": ([1, 1], [400, 50], 2, 2, 64),
    "step-wide": ([1, 2], [300, 129], 2, 4, 128),
    "few-narrow-tile": ([20, 3], [300, 200], 2, 1, 80),
    "few": ([40], [333], 2, 1, 64),                        # tiles of 32
    "many-splits": ([1], [4300], 1, 1, 64),                # joined by a launch
    "chunks": ([70, 1], [200, 90], 192, 1, 64),            # 128 rows a block
    "chunks-wide": ([129], [150], 192, 1, 96),
    "cut-chunks": ([90], [6200], 128, 1, 16),              # and joined
}
# The power of two of the value row at a position; None: a row of zeros.
POWERS = {
    "zeros, then 2^55": lambda p, n: None if p < 32 else 55,
    "zeros, one of 2^100 at the end": lambda p, n: 100 if p == n - 1 else None,
    "zeros and 2^70 in turn": lambda p, n: 70 if p % 2 else None,
    "2^60, then small": lambda p, n: 60 if p < 40 else -60,
    "small, then 2^100, then zeros": lambda p, n: -75 if p < n // 3 else 100 if p < n // 2 else None,
    "one of 2^40 in the middle": lambda p, n: 40 if p == n // 2 else 0,
    "every power": lambda p, n: (p * 13) % 190 - 70,
    "fp32's largest": lambda p, n: 125,
    "small": lambda p, n: -70,
}


def powered(shape, powers, seed=211):
    counts, lengths, kv, group, width = SHAPES[shape]
    case = Case("E4M3", counts, lengths, kv, group, width, 64, seed=seed, noise=0.0)
    np.clip(case.value_rows, -3, 3, out=case.value_rows)
    for s, n in enumerate(lengths):
        for p in range(n):
            power = POWERS[powers](p, n)
            case.value_rows[case.table[s, p // 64], :, p % 64] *= np.float32(0 if power is None else 2.0 ** power)
    return case


def means(case):
    """Causal rows of equal scores, and the bound of each value."""
    want = np.zeros((case.rows, case.kv * case.group * case.width))
    bound = np.zeros_like(want)
    for s, (count, length) in enumerate(zip(case.counts, case.lengths)):
        n = np.arange(length - count, length)[:, None] + 1.0
        rows = slice(case.starts[s], case.starts[s] + count)
        for h in range(case.kv):
            v = case.cached(s, h, 1)
            mean = np.cumsum(v, axis=0)[-count:] / n
            size = np.cumsum(np.abs(v), axis=0)[-count:] / n
            for g in range(case.group):
                columns = slice((h * case.group + g) * case.width, (h * case.group + g + 1) * case.width)
                want[rows, columns] = mean
                bound[rows, columns] = size * (n + 16) * 2.0 ** -24
    return want, bound


CASES = [(powers, shape) for powers in POWERS for shape in SHAPES
         if shape != "cut-chunks" or powers in ("zeros, then 2^55", "small, then 2^100, then zeros", "every power")]


@pytest.mark.parametrize("powers,shape", CASES)
def test_equal_scores_over_rows_of_far_powers(ctx, powers, shape):  # noqa: F811
    # A key weighs the same whatever its value row's power is.
    case = powered(shape, powers)
    case.q[:] = 0
    case.quantise()
    got = attend(ctx, case)
    want, bound = means(case)
    assert np.all(np.abs(got - want) <= bound), float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300)))


@pytest.mark.parametrize("shape", ["step", "few", "step-wide", "chunks"])
@pytest.mark.parametrize("powers", POWERS)
def test_scores_over_rows_of_far_powers(ctx, powers, shape):  # noqa: F811
    case = powered(shape, powers, seed=223)
    case.quantise()
    check(ctx, case)


@pytest.mark.parametrize("shape", SHAPES)
def test_channels_that_loud_rows_leave_alone(ctx, shape):  # noqa: F811
    # Loud rows hold zeros in the first half of the channels, where quiet ones are all there is.
    for loud, quiet in ((60, 0), (0, -60), (110, -70)):
        case = powered(shape, "one of 2^40 in the middle")
        for s, n in enumerate(case.lengths):
            for p in range(n):
                row = case.value_rows[case.table[s, p // 64], :, p % 64]
                row[:] = np.where(row >= 0, 1.0, -1.0) * np.float32(2.0 ** (loud if p % 5 == 2 else quiet))
                row[:, :(case.width // 2 if p % 5 == 2 else 0)] = 0
        case.q[:] = 0
        case.quantise()
        got = attend(ctx, case)
        want, bound = means(case)
        assert np.all(np.abs(got - want) <= bound), (loud, quiet)


@pytest.mark.parametrize("shape", ["step", "few", "step-wide", "chunks", "cut-chunks"])
def test_every_exponent_byte_of_values(ctx, shape):  # noqa: F811
    # Bytes that append never writes (below 47, past 247) mean 2^(byte - 127) too.
    case = powered(shape, "small")
    case.q[:] = 0
    case.quantise()
    case.values[:] = np.where(np.isfinite(e4m3_values()[case.values]), case.values, 0)
    for s, n in enumerate(case.lengths):
        for p in range(n):
            at = (case.table[s, p // 64], slice(None), p % 64)
            byte = (0, 255, 127, 46, 248, 90, 254, 1)[p % 8]
            case.value_exponents[at] = byte
            if byte > 240:  # (of at most 2^-6 in E4M3: what they stand for is an fp32 number)
                case.values[at] = case.values[at] & 0x88 | case.values[at] & 7
    got = attend(ctx, case)
    want, bound = means(case)
    assert np.all(np.abs(got - want) <= bound)


@pytest.mark.parametrize("shape", ["step", "few", "step-wide", "chunks"])
@pytest.mark.parametrize("byte", [0, 3, 250, 255])
def test_ends_of_the_exponent_bytes_of_keys(ctx, byte, shape):  # noqa: F811
    # All keys of one such byte, and the queries their inverse: ordinary scores.
    case = powered(shape, "one of 2^40 in the middle")
    case.value_rows[:] = np.random.default_rng(5).normal(0, 1, case.value_rows.shape)
    np.clip(case.key_rows, -3, 3, out=case.key_rows)
    case.quantise()
    # Signs and fractions as they came, of 2^-1 or (large bytes) below 2^-6: fp32 numbers all.
    kept = np.where(case.keys & 0x7F == 0x7F, 0, case.keys) & 0x87
    case.keys[:] = kept | (0x30 if byte < 127 else 0)
    case.key_exponents[:] = byte
    power = 120 if byte < 127 else 134 - byte
    case.q *= np.float32(2.0 ** power)
    case.scale = case.width ** -0.5 * (2.0 ** (7 - byte) if byte < 127 else 1.0)
    check(ctx, case)


@pytest.mark.parametrize("shape", ["step", "few", "step-wide", "chunks"])
def test_scores_of_zero_of_huge_operands(ctx, shape):  # noqa: F811
    # Keys and queries whose sizes multiply past fp32 but which share no channel.
    case = powered(shape, "one of 2^40 in the middle")
    case.q[:] = 0
    case.q[:, 1::case.width] = 2.0 ** 100
    case.key_rows[:] = 0
    case.key_rows[..., 0] = 2.0 ** 60
    case.quantise()
    got = attend(ctx, case)
    want, bound = means(case)
    assert np.all(np.abs(got - want) <= bound)


def test_a_bad_page_beside_rows_of_far_powers(ctx):  # noqa: F811
    # In a tile of keys whose value rows' powers lie far apart a page is none: rows that
    # see none of its keys are as they were, whatever the pool's first page holds.
    case = Case("E4M3", [70], [140], 384, 1, 64, 16, seed=227, noise=0.0, spare_pages=3)
    spare = int(np.setdiff1d(np.arange(case.pages), case.table)[-1])
    for rows in (case.key_rows, case.value_rows):
        rows[[0, spare]] = rows[[spare, 0]]
    case.table[case.table == 0] = spare
    case.value_rows *= np.float32(2.0 ** 12)       # the first row's power is large
    case.value_rows[case.table[0, 4], :, 1] = 0     # position 65
    case.quantise()
    case.value_exponents[0] = case.key_exponents[0] = 0
    clean = check(ctx, case)
    case.table[0, 7] = -1                           # positions 112 on
    got = attend(ctx, case)
    assert np.isnan(got[112 - 70:]).all()
    assert np.array_equal(got[:112 - 70], clean[:112 - 70])


@pytest.mark.parametrize("shape", ["few", "chunks"])
def test_a_nan_value_beside_rows_of_far_powers(ctx, shape):  # noqa: F811
    # Rows that see it are not finite in its channel, and as they were in the others;
    # rows before it are as they were, bit for bit.
    case = powered(shape, "zeros and 2^70 in turn")
    case.quantise()
    clean = check(ctx, case)
    count, length = case.counts[0], case.lengths[0]
    row = count // 2
    position = length - count + row | 1  # (one of those of 2^70)
    row = position - (length - count)
    page, place = case.table[0, position // 64], position % 64
    case.values[page, :, place, 5] = 127
    got = attend(ctx, case)
    assert np.array_equal(got[:row], clean[:row]) and np.array_equal(got[count:], clean[count:])
    hit = got[row:count].reshape(count - row, -1, case.width)
    assert not np.isfinite(hit[:, :, 5]).any()
    kept = clean[row:count].reshape(hit.shape)
    assert np.array_equal(np.delete(hit, 5, 2), np.delete(kept, 5, 2))


@pytest.mark.parametrize("storage", ["F16", "BF16"])
@pytest.mark.parametrize("count,kv", [(1, 2), (40, 2), (70, 192)])
def test_infinite_keys_of_16_bits(ctx, storage, count, kv):  # noqa: F811
    # Rows that see the key: NaN where fp32's score is +inf; where it is -inf, NaN or the row without it.
    for sign in (1.0, -1.0):
        case = Case(storage, [count], [120], kv, 1, 64, 16, seed=229)
        clean = check(ctx, case)
        seat = 120 - (count + 1) // 2
        at = (case.table[0, seat // 16], slice(None), seat % 16)
        case.key_rows[at + (5,)] = sign * np.inf
        case.quantise()
        got = attend(ctx, case)
        first = seat - (120 - count)
        assert np.array_equal(got[:first], clean[:first])
        assert first < count
        case.key_rows[at] = 0
        case.key_rows[at + (5,)] = sign * 1e4
        case.q[:, 5::64] += np.where(case.q[:, 5::64] < 0, -1, 1)  # (no query next to zero)
        case.quantise()
        without, bound = case.expected(True, np.full(got.shape, 7.25))
        case.key_rows[at + (5,)] = sign * np.inf
        case.quantise()
        got = attend(ctx, case).reshape(count, kv, 64)
        up = case.q[:, 5::64] * sign > 0
        assert np.isnan(got[first:][up[first:]]).all()
        down = got[first:][~up[first:]]
        near = np.abs(got - without.reshape(got.shape)) <= bound.reshape(got.shape)
        assert np.all(np.isnan(down) | near[first:][~up[first:]])


@pytest.mark.parametrize("count,kv", [(1, 2), (40, 2)])
def test_rows_whose_every_score_is_minus_infinity(ctx, count, kv):  # noqa: F811
    # In fp32 storage: no weight at all, through several waves and splits.
    for length in (120, 1500):
        case = Case("F32", [count], [length], kv, 1, 64, 16, seed=233)
        case.q[:, ::64] = 1.0
        case.key_rows[..., 0] = -np.inf
        case.quantise()
        assert np.all(attend(ctx, case) == 0)

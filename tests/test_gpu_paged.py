"""The paged cache's kernels through the C ABI (include/wsp_hip.h,
wsp_hip_paged_*) against plain forms in 64 bits.

Storing and reading back are exact: one rounding to the storage, which the plain
form makes from a table of every E4M3 value. Attention's bound, for a row that
sees n keys of width w, with A = max_j scale·Σ_c |q_c k_jc|:
  a score is off by at most A·((w + 8)·2^-24 + 2^-22 + 2^-23): w + 8 roundings
  of fp32 sums and products, the 16-bit parts of q (2^-22), the change to powers
  of two and exp2's own ulp;
  a weight by twice that, relative, and (n + 16)·2^-24 from the sums over keys
  and the weights' 16-bit parts, which also lose n·2^-30·max|v| below fp16's
  least numbers;
so |o - exact| <= Σ_j p_j |v_j|·(2·score bound + (n + 16)·2^-24) + n·2^-30·max|v|.
"""

import numpy as np
import pytest

from helpers import ensure_library
from whispereacp_amd import synthetic as S

pytestmark = pytest.mark.gpu

STORAGES = ["F32", "F16", "BF16", "E4M3"]


@pytest.fixture(scope="module")
def ctx():
    ensure_library()
    import torch
    from whispereacp_amd.decoder import KernelContext
    assert torch.cuda.is_available()
    return KernelContext(S.DecoderShape(64, 1, 1, 64, 64, 1, 1))


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------

def e4m3_values():
    """The value of each of the 256 bytes: 4 exponent bits biased by 7, 3 fraction
    bits, no infinities, NaN where all seven are set."""
    byte = np.arange(256)
    exponent, fraction = (byte >> 3) & 15, byte & 7
    magnitude = np.where(exponent == 0, fraction * 2.0 ** -9, (8 + fraction) * 2.0 ** (exponent - 10.0))
    magnitude[(byte & 127) == 127] = np.nan
    return np.where(byte < 128, magnitude, -magnitude)


E4M3 = e4m3_values()


def to_e4m3(x):
    """Bytes of the nearest E4M3 value of each |x| <= 448 (ties to the even byte); NaN and infinities 127."""
    table = E4M3[:127]
    a = np.where(np.isfinite(x), np.abs(x), 0.0)
    above = np.clip(np.searchsorted(table, a), 0, 126)
    below = np.maximum(above - 1, 0)
    up, down = table[above] - a, a - table[below]
    byte = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return np.where(np.isfinite(x), byte + 128 * np.signbit(x), 127).astype(np.uint8)


def row_exponents(rows):
    """The least k in [-80, 120] with the largest finite magnitude of each row [..., w] <= 448·2^k."""
    top = np.max(np.where(np.isfinite(rows), np.abs(rows), 0.0), axis=-1)
    k = np.full(top.shape, -80)
    for power in range(-80, 120):
        k[top > 448.0 * 2.0 ** power] = power + 1
    return k


def store(rows, storage):
    """(stored array, exponent bytes or None) of fp32 rows [..., w]."""
    if storage == "F32":
        return rows.copy(), None
    if storage == "F16":
        with np.errstate(over="ignore"):
            return rows.astype(np.float16), None
    if storage == "BF16":
        bits = rows.view(np.uint32).astype(np.uint64)
        rounded = ((bits + 0x7FFF + ((bits >> 16) & 1)) >> 16).astype(np.uint16)
        return np.where(np.isnan(rows), np.uint16(0x7FC0), rounded), None
    k = row_exponents(rows.astype(np.float64))
    return to_e4m3(rows.astype(np.float64) * 2.0 ** -k[..., None].astype(np.float64)), (k + 127).astype(np.uint8)


def widen(stored, exponents, storage):
    """What stored rows stand for, in 64 bits."""
    if storage == "BF16":
        return (stored.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if storage == "E4M3":
        return E4M3[stored] * 2.0 ** (exponents.astype(np.float64)[..., None] - 127)
    return stored.astype(np.float64)


def device_tensor(stored, storage):
    import torch
    if storage == "BF16":
        return torch.from_numpy(stored.view(np.int16)).cuda().view(torch.bfloat16)
    t = torch.from_numpy(stored).cuda()
    return t.view(torch.float8_e4m3fn) if storage == "E4M3" else t


def host_array(tensor, storage):
    import torch
    if storage == "BF16":
        return tensor.view(torch.int16).cpu().numpy().view(np.uint16)
    return (tensor.view(torch.uint8) if storage == "E4M3" else tensor).cpu().numpy()


class Case:
    """Sequences with new rows over a pool whose pages they own in a shuffled
    order; slots that no position takes hold NaN."""

    def __init__(self, storage, counts, lengths, kv=2, group=1, width=64, page=16, seed=1, spare_rows=0,
                 spare_pages=2, noise=1.0):
        self.storage, self.counts, self.lengths = storage, list(counts), list(lengths)
        self.kv, self.group, self.width, self.page = kv, group, width, page
        self.rng = np.random.default_rng(seed)
        blocks = [-(-max(n, 0) // page) for n in lengths]
        self.pages = sum(blocks) + spare_pages
        order, at = self.rng.permutation(self.pages), 0
        self.table = np.full((len(blocks), max(blocks + [1])), -1, np.int32)
        for s, n in enumerate(blocks):
            self.table[s, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.rows = int(self.starts[-1]) + spare_rows
        shape = (self.pages, kv, page, width)
        loud = np.exp(self.rng.normal(0, noise, shape[:3] + (1,)))
        self.key_rows = (self.rng.normal(0, 1, shape)).astype(np.float32)
        self.value_rows = (self.rng.normal(0, 1, shape) * loud).astype(np.float32)
        owned = np.zeros((self.pages, page), bool)
        for s, n in enumerate(self.lengths):
            for p in range(n):
                owned[self.table[s, p // page], p % page] = True
        for rows in (self.key_rows, self.value_rows):
            rows.transpose(0, 2, 1, 3)[~owned] = np.nan
        self.q = self.rng.normal(0, 1, (self.rows, kv * group * width)).astype(np.float32)
        self.scale = width ** -0.5
        self.quantise()

    def quantise(self):
        self.keys, self.key_exponents = store(self.key_rows, self.storage)
        self.values, self.value_exponents = store(self.value_rows, self.storage)

    def cached(self, s, h, which):
        """Sequence s's rows of head h, [length, width]."""
        pool, exponents = ((self.keys, self.key_exponents), (self.values, self.value_exponents))[which]
        places = np.arange(self.lengths[s])
        at = (self.table[s, places // self.page], h, places % self.page)
        return widen(pool[at], None if exponents is None else exponents[at], self.storage)

    def cache(self):
        import torch
        from whispereacp_amd.paged import PagedCache
        exponents = [torch.from_numpy(e).cuda() for e in (self.key_exponents, self.value_exponents) if e is not None]
        return PagedCache(device_tensor(self.keys, self.storage), device_tensor(self.values, self.storage), *exponents)

    def packed(self, **changes):
        import torch
        from whispereacp_amd.paged import PagedRows
        given = dict(rows=self.rows, max_count=max(self.counts + [0]), max_length=max(self.lengths + [0]))
        given.update(changes)
        return PagedRows(*(torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()
                           for a in (self.starts, np.array(self.lengths), self.table)), **given)

    def expected(self, causal, out):
        """out with the sequences' rows replaced, and the bound of each value."""
        bound = np.zeros_like(out)
        for s, (count, length) in enumerate(zip(self.counts, self.lengths)):
            if count == 0:
                continue
            rows = slice(self.starts[s], self.starts[s] + count)
            positions = np.arange(length - count, length)
            n = np.where(positions < 0, 0, positions + 1 if causal else length)[:, None]
            seen = np.arange(max(length, 0))[None, :] < n
            for h in range(self.kv):
                k, v = self.cached(s, h, 0), self.cached(s, h, 1)
                largest = np.maximum.accumulate(np.max(np.abs(v), axis=1)) if length > 0 else np.zeros(1)
                for g in range(self.group):
                    columns = slice((h * self.group + g) * self.width, (h * self.group + g + 1) * self.width)
                    q = self.q[rows, columns].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        scores = np.where(seen, q @ k.T * self.scale, -np.inf)
                        p = np.exp(scores - np.where(n > 0, scores.max(axis=1, keepdims=True, initial=-np.inf), 0))
                        p /= np.where(n > 0, p.sum(axis=1, keepdims=True), 1)
                    out[rows, columns] = p @ v
                    a = np.max(np.where(seen, np.abs(q) @ np.abs(k).T, 0), axis=1, initial=0)[:, None] * abs(self.scale)
                    score = a * ((self.width + 8) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23)
                    bound[rows, columns] = (p @ np.abs(v) * (2 * score + (n + 16) * 2.0 ** -24)
                                            + n * 2.0 ** -30 * largest[np.maximum(n - 1, 0)])
        return out, bound


def attend(ctx, case, causal=True, rows=None, cache=None, fill=7.25):
    import torch
    out = torch.full((case.rows, case.kv * case.group * case.width), fill, device="cuda")
    ctx.paged_attention(cache or case.cache(), rows or case.packed(), torch.from_numpy(case.q).cuda(),
                        case.kv * case.group, causal, case.scale, out)
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check(ctx, case, causal=True, **given):
    got = attend(ctx, case, causal, **given)
    want, bound = case.expected(causal, np.full(got.shape, 7.25))
    off = np.abs(got - want)
    assert np.all(off <= bound), (float(np.max(off)), float(np.max(off / np.maximum(bound, 1e-300))))
    return got


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------

def new_rows(case, seed, gap):
    """fp32 rows as columns of a wider tensor, `gap` floats between them, from an odd float on."""
    import torch
    width = case.kv * case.width
    wide = np.random.default_rng(seed).normal(0, 1, (case.rows, width + gap)).astype(np.float32)
    wide *= np.exp(np.random.default_rng(seed + 1).normal(0, 2, (case.rows, 1))).astype(np.float32)
    device = torch.from_numpy(np.concatenate([np.zeros(1, np.float32), wide.reshape(-1)])).cuda()
    return wide, device[1:].view(case.rows, width + gap)


def append(ctx, case, keys, values, cache=None, rows=None):
    import torch
    cache = cache or case.cache()
    ctx.paged_append(cache, rows or case.packed(), keys, values)
    torch.cuda.synchronize()
    return cache


def check_pool(case, cache, keys, values):
    """The pool against the case's with the new rows stored by the plain form."""
    for pool, exponents, start, powers, rows in (
            (cache.keys, cache.key_exponents, case.keys, case.key_exponents, keys),
            (cache.values, cache.value_exponents, case.values, case.value_exponents, values)):
        want, want_powers = start.copy(), None if powers is None else powers.copy()
        for s, (count, length) in enumerate(zip(case.counts, case.lengths)):
            for i in range(count):
                position = length - count + i
                if position < 0:
                    continue
                page = case.table[s, position // case.page]
                stored, k = store(rows[case.starts[s] + i].reshape(case.kv, case.width), case.storage)
                want[page, :, position % case.page] = stored
                if k is not None:
                    want_powers[page, :, position % case.page] = k
        got = host_array(pool, case.storage)
        if case.storage == "E4M3":
            assert np.array_equal(E4M3[got], E4M3[want], equal_nan=True)
            assert np.array_equal(exponents.cpu().numpy(), want_powers)
        elif case.storage == "BF16":
            assert np.array_equal(widen(got, None, "BF16"), widen(want, None, "BF16"), equal_nan=True)
        else:
            assert np.array_equal(got, want, equal_nan=True)


SHAPES = [
    # counts, lengths, kv, width, page, spare rows
    ([1], [1], 1, 64, 16, 0),                                # the first token
    ([1] * 5, [1, 16, 17, 40, 33], 3, 64, 16, 0),            # a step
    ([0, 4, 0, 1, 17, 0], [9, 4, 1, 130, 31, 0], 2, 128, 32, 3),
    ([70], [75], 20, 16, 64, 0),                             # narrow heads
    ([33, 2], [33, 300], 5, 80, 16, 2),                      # heads of no power of two
    ([300], [1100], 1, 112, 1024, 1),
]


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("counts,lengths,kv,width,page,spare", SHAPES)
def test_append_stores_and_read_gives_back(ctx, storage, counts, lengths, kv, width, page, spare):
    import torch
    case = Case(storage, counts, lengths, kv, 1, width, page, seed=3, spare_rows=spare)
    keys, device_keys = new_rows(case, 5, 3)
    values, device_values = new_rows(case, 9, 8)
    n = kv * width
    cache = append(ctx, case, device_keys[:, :n], device_values[:, :n])
    check_pool(case, cache, keys[:, :n], values[:, :n])
    back = [torch.full((case.rows, n + 5), 3.5, device="cuda") for _ in range(2)]
    ctx.paged_read(cache, case.packed(), back[0][:, :n], back[1][:, :n])
    torch.cuda.synchronize()
    for got, rows in zip(back, (keys, values)):
        want = np.full((case.rows, n + 5), 3.5)
        total = int(case.starts[-1])
        stored, k = store(rows[:total, :n].reshape(total, kv, width), storage)
        want[:total, :n] = widen(stored, k, storage).reshape(total, n)
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("storage", STORAGES)
def test_read_gives_whole_sequences(ctx, storage):
    import torch
    lengths = [40, 1, 0, 77]
    case = Case(storage, lengths, lengths, 3, 1, 96, 32, seed=8)
    back = [torch.zeros((case.rows, 3 * 96), device="cuda") for _ in range(2)]
    ctx.paged_read(case.cache(), case.packed(), *back)
    torch.cuda.synchronize()
    for which, got in enumerate(back):
        want = np.concatenate([np.stack([case.cached(s, h, which) for h in range(3)], 1).reshape(n, 3 * 96)
                               for s, n in enumerate(lengths)])
        assert np.array_equal(got.cpu().numpy(), want)


def odd_values(width):
    """Rows at the borders of the storages."""
    rows = np.zeros((12, width), np.float32)
    rng = np.random.default_rng(4)
    rows[1:] = rng.normal(0, 1, (11, width))
    rows[1, 0] = 448.0 * 2.0 ** 5                       # the largest of its power, exactly
    rows[2, 3] = np.nextafter(np.float32(448.0), np.float32(1000))  # one step past it
    rows[3, 5], rows[3, 6] = np.inf, -np.inf
    rows[4, 7] = np.nan
    rows[5] *= 1e-30                                     # below the least power
    rows[6] *= 2.0 ** -84                                # half in it
    rows[7, 1] = np.finfo(np.float32).max
    rows[8, 2] = 70000.0                                 # past fp16
    rows[9] = np.float32(1e-40)                          # fp32's denormals
    rows[10] = np.tile(np.float32([448, 432, 440, 416, 2.0 ** -6, 2.0 ** -10, 3 * 2.0 ** -10, -2.0 ** -9]),
                       width // 8)                        # ties, to even
    rows[11, :] = -0.0
    return rows


@pytest.mark.parametrize("storage", STORAGES)
def test_append_of_odd_values(ctx, storage):
    import torch
    rows = odd_values(64)
    case = Case(storage, [12], [21], 1, 1, 64, 16, seed=6)
    cache = append(ctx, case, torch.from_numpy(rows).cuda(), torch.from_numpy(rows[::-1].copy()).cuda())
    check_pool(case, cache, rows, rows[::-1])


def test_append_and_read_of_bad_pages(ctx):
    # A row whose page is not in the pool is dropped by append and reads as NaN;
    # one past the table too; one before its sequence is dropped and reads as zero.
    import torch
    case = Case("F16", [20, 3, 20], [40, 2, 40], 2, 1, 64, 16, seed=11)
    case.table = case.table[:, :2]           # positions 32 on are past the table
    case.table[2, 1] = case.pages            # one past the pool
    keys, device_keys = new_rows(case, 5, 0)
    values, device_values = new_rows(case, 7, 0)
    cache = append(ctx, case, device_keys, device_values)
    back = [torch.zeros((case.rows, 128), device="cuda") for _ in range(2)]
    ctx.paged_read(cache, case.packed(), *back)
    torch.cuda.synchronize()
    want_pool = case.keys.copy()
    want = np.zeros((case.rows, 128))
    for s, (count, length) in enumerate(zip(case.counts, case.lengths)):
        for i in range(count):
            row, position = case.starts[s] + i, length - count + i
            if position < 0:
                continue
            page = case.table[s, position // 16] if position < 32 else -1
            if 0 <= page < case.pages:
                want_pool[page, :, position % 16] = keys[row].astype(np.float16).reshape(2, 64)
                want[row] = keys[row].astype(np.float16)
            else:
                want[row] = np.nan
    assert np.array_equal(host_array(cache.keys, "F16"), want_pool, equal_nan=True)
    assert np.array_equal(back[0].cpu().numpy(), want, equal_nan=True)


# ---------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------

ATTENTION = [
    # counts, lengths, kv, group, width, page, spare rows
    ([1], [1], 1, 1, 64, 16, 0),                                    # one key
    ([1], [131], 6, 1, 64, 16, 0),                                  # a step of one stream
    ([1] * 4 + [0], [16, 1, 17, 100, 50], 3, 1, 64, 32, 2),         # a step of several, one at rest
    ([1, 1, 1], [700, 33, 64], 2, 4, 128, 64, 0),                   # shared heads
    ([1, 1], [200, 257], 1, 5, 80, 16, 0),                          # a group of five, heads 80 wide
    ([1], [300], 2, 17, 16, 16, 0),                                 # more query heads than a tile
    ([5, 1, 3], [90, 1, 3], 2, 3, 48, 16, 1),                       # a few new tokens
    ([16, 7], [16, 39], 2, 1, 64, 16, 0),                           # a prompt of one tile
    ([40, 0, 1, 9], [40, 7, 300, 120], 2, 2, 64, 32, 3),            # chunks
    ([150, 33], [150, 200], 1, 1, 128, 64, 0),
    ([70, 70], [333, 70], 1, 4, 96, 16, 0),
    ([257], [513], 1, 1, 64, 1024, 0),
    ([5, 2], [3, 2], 2, 2, 64, 16, 0),                              # rows before their sequence see nothing
    ([100], [64], 1, 1, 64, 16, 0),
]


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,lengths,kv,group,width,page,spare", ATTENTION)
def test_attention(ctx, storage, causal, counts, lengths, kv, group, width, page, spare):
    check(ctx, Case(storage, counts, lengths, kv, group, width, page, seed=13, spare_rows=spare), causal)


# Chunks of many heads, which take the kernel of 128 rows a block (from 384 blocks on).
CHUNKS = [
    # counts, lengths, kv, group, width, page, spare rows
    ([70, 0, 66], [70, 9, 300], 192, 1, 64, 16, 2),
    ([65, 3], [200, 3], 192, 1, 128, 32, 0),
    ([40, 129], [90, 130], 96, 3, 96, 64, 1),                       # shared heads, a ragged last tile
    ([33, 1], [64, 700], 200, 2, 48, 16, 0),                        # narrow heads
    ([90, 20], [500, 20], 200, 1, 112, 16, 0),
    ([100, 80], [64, 81], 200, 1, 80, 128, 0),                      # rows before their sequence
]


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("counts,lengths,kv,group,width,page,spare", CHUNKS)
def test_attention_of_chunks(ctx, storage, causal, counts, lengths, kv, group, width, page, spare):
    check(ctx, Case(storage, counts, lengths, kv, group, width, page, seed=83, spare_rows=spare), causal)


@pytest.mark.parametrize("storage", ["F16", "BF16", "E4M3"])
@pytest.mark.parametrize("kv,width", [(96, 64), (64, 80), (64, 128)])
def test_attention_of_chunks_over_long_sequences(ctx, storage, kv, width):
    # The 128-row kernel with its keys cut: the second sequence ends in the first cut,
    # rows of the first end on either side of it.
    check(ctx, Case(storage, [129, 70], [4160, 100], kv, 1, width, 64, seed=101))


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("count,length", [(1, 5000), (3, 9000), (20, 4100)])
def test_attention_over_long_sequences(ctx, storage, count, length):
    # Few rows over many keys: the keys are split and joined.
    check(ctx, Case(storage, [count, 1], [length, length // 3], 1, 2, 64, 64, seed=17))


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("width", [64, 128])
@pytest.mark.parametrize("kv", [1, 192])
def test_attention_of_large_scores(ctx, storage, width, kv):
    # Scores of some hundreds: one key takes nearly all, the running maximum
    # climbs along the keys, and late keys push early ones out.
    case = Case(storage, [1, 2, 40], [600, 90, 333], kv, 2, width, 32, seed=19)
    case.q *= 40
    for s, n in enumerate(case.lengths):
        for p in range(n):
            case.key_rows[case.table[s, p // 32], :, p % 32] *= 0.2 + 2.0 * p / n
    case.quantise()
    check(ctx, case)


@pytest.mark.parametrize("storage", ["F16", "BF16", "E4M3", "F32"])
@pytest.mark.parametrize("q_size,v_size", [(1e-6, 1e4), (1e5, 1e-4), (0.0, 1.0)])
@pytest.mark.parametrize("kv", [2, 192])
def test_attention_of_odd_magnitudes(ctx, storage, q_size, v_size, kv):
    # Queries far from one (their parts are scaled to fp16's range), values large
    # and small. Scores stay ordinary: scale undoes the queries' size.
    # (In fp16 the values stay below its 65504: ten times as many, not 10^4.)
    case = Case(storage, [1, 33, 5], [70, 100, 5], kv, 1 if kv == 2 else 2, 64, 16, seed=23)
    v_size = min(v_size, 10.0) if storage == "F16" else v_size
    case.q *= np.float32(q_size)
    case.scale = 0.125 / q_size if q_size else 0.125
    case.value_rows *= np.float32(v_size)
    case.quantise()
    check(ctx, case)


def test_attention_of_e4m3_rows_of_far_powers(ctx):
    # Rows whose powers of two lie far apart, rows of zeros among them: a
    # weight times its row's power spans more than fp16's range.
    for count, kv, width in ((1, 2, 64), (40, 2, 64), (70, 192, 64), (70, 192, 96)):
        case = Case("E4M3", [count, 1], [400, 50], kv, 1, width, 32, seed=29)
        powers = 2.0 ** case.rng.integers(-40, 30, case.value_rows.shape[:3] + (1,))
        case.value_rows *= powers.astype(np.float32)
        case.value_rows[:, :, ::5] *= 0
        case.key_rows[:, :, ::7] *= 2.0 ** -60
        case.quantise()
        check(ctx, case)


@pytest.mark.parametrize("kv", [2, 192])
@pytest.mark.parametrize("first,others", [(0, -15), (0, -22), (-80, -7), (-80, 100), (100, -30)])
def test_attention_of_e4m3_rows_far_from_the_first(ctx, kv, first, others):
    # The first key's and value's rows have power `first`, about, and the key nearly no
    # weight; all others' lie near `others`, among them fp16's least numbers as operands
    # and rows past its range. They keep an accuracy of their own: the bound is the one
    # above with A = 0.125·(4·60 + 63·16), the largest of |q| and |k| being four in
    # units of the others, and the others' values alone.
    case = Case("E4M3", [70, 1], [200, 90], kv, 1, 64, 32, seed=97, noise=0.0)
    unit = 2.0 ** (others + 7)
    for rows in (case.key_rows, case.value_rows):
        np.clip(rows, -4, 4, out=rows)
        rows *= np.float32(unit)
    np.clip(case.q, -4, 4, out=case.q)
    case.q[:, ::64] = 4
    case.scale = 0.125 / unit
    channel = case.key_rows[..., 0]
    channel[~np.isnan(channel)] = unit if first >= others else 60 * unit  # (scores of thirty)
    pages = case.table[:, 0]
    case.key_rows[pages, :, 0] = 0
    case.value_rows[pages, :, 0] = 0
    if first >= others:
        case.key_rows[pages, :, 0, 0] = -300 * 2.0 ** first  # (a score of -150·2^(first - others - 7) and less)
        case.value_rows[pages, :, 0] = 300 * 2.0 ** first
    case.quantise()
    got = attend(ctx, case)
    want, _ = case.expected(True, np.full(got.shape, 7.25))
    a = 0.125 * (4 * 60 + 63 * 16)
    bound = 4 * unit * (2 * a * (72 * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23) + 216 * 2.0 ** -24)
    assert np.max(np.abs(want)) > unit / 8
    assert np.max(np.abs(got - want)) <= bound


@pytest.mark.parametrize("storage", STORAGES)
@pytest.mark.parametrize("width", [64, 80, 128])
@pytest.mark.parametrize("counts,lengths,kv", [([40, 4, 1], [40, 20, 77], 2), ([200], [300], 2), ([70, 1], [110, 40], 192)])
def test_what_a_row_does_not_see_does_not_reach_it(ctx, storage, width, counts, lengths, kv):
    # Infinities and NaN in keys and values: rows before them are as without
    # them, bit for bit; rows that see them are not finite.
    case = Case(storage, counts, lengths, kv, 1, width, 16, seed=31)
    clean = check(ctx, case)
    s, head = 0, slice(width, 2 * width)
    for row, bad, in_keys in ((counts[0] - 9, np.nan, False), (counts[0] - 14, np.inf, False),
                              (counts[0] - 5, np.nan, True)):
        position = lengths[s] - counts[s] + row
        rows = case.key_rows if in_keys else case.value_rows
        kept = rows.copy()
        rows[case.table[s, position // 16], 1, position % 16, 5] = bad
        case.quantise()
        got = attend(ctx, case)
        first = case.starts[s] + row
        assert np.array_equal(got[:first], clean[:first])
        assert np.array_equal(got[:, :width], clean[:, :width])
        assert np.array_equal(got[:, 2 * width:], clean[:, 2 * width:])
        hit = got[first:case.starts[s + 1], head]
        assert not np.any(np.isfinite(hit if in_keys else hit[:, 5]))
        assert in_keys or np.array_equal(np.delete(hit, 5, 1),
                                         np.delete(clean[first:case.starts[s + 1], head], 5, 1)) \
            or storage == "E4M3"  # (the row's power is that of its finite values)
        assert np.array_equal(got[case.starts[s + 1]:], clean[case.starts[s + 1]:])
        rows[:] = kept


def test_keys_of_minus_infinity_weigh_nothing(ctx):
    # In fp32 a key whose score is -inf is a key with weight zero, the first one
    # too. (The 16-bit parts of a query hold zeros, and zero times inf is NaN.)
    case = Case("F32", [1, 20], [50, 40], 1, 1, 64, 16, seed=37)
    case.q[:, 0] = 1.0
    for s, p in ((0, 0), (0, 31), (1, 0), (1, 33)):
        case.key_rows[case.table[s, p // 16], 0, p % 16, 0] = -np.inf
    case.quantise()
    got = attend(ctx, case)
    with np.errstate(invalid="ignore"):
        want, _ = case.expected(True, np.full(got.shape, 7.25))
    assert np.isfinite(want).all()
    assert np.allclose(got, want, rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("count,kv", [(1, 2), (3, 2), (40, 2), (40, 128)])
@pytest.mark.parametrize("storage", ["F16", "E4M3"])
def test_attention_over_bad_pages(ctx, count, storage, kv):
    # A page outside the pool makes NaN of the rows that see one of its keys, and
    # of no others; so do a table that ends too early and a length past max_length.
    lengths = [150, 150, 150]
    case = Case(storage, [count] * 3, lengths, kv, 2, 64, 16, seed=41)
    clean = check(ctx, case)
    good = case.table.copy()
    block = (150 - count) // 16  # the new rows' first page
    case.table[1, block + 1 if count > 16 else 2] = 12345
    got = attend(ctx, case)
    rows = np.arange(case.starts[1], case.starts[2])
    first = (block + 1) * 16 - (150 - count) if count > 16 else 0
    assert np.isnan(got[rows[first:]]).all()
    keep = np.setdiff1d(np.arange(case.rows), rows[first:])
    assert np.array_equal(got[keep], clean[keep])
    case.table = good[:, :9]  # 144 positions
    got = attend(ctx, case)
    for s in range(3):
        for i in range(count):
            row = case.starts[s] + i
            if 150 - count + i >= 144:
                assert np.isnan(got[row]).all()
            else:
                assert np.array_equal(got[row], clean[row])
    case.table = good
    case.lengths = [150, 155, 150]
    got = attend(ctx, case, rows=case.packed(max_length=150))
    assert np.isnan(got[rows]).all() and np.array_equal(got[:rows[0]], clean[:rows[0]])


def test_rows_past_max_count_and_past_the_last_sequence_stay(ctx):
    # (A row's last bits may differ where another bound chooses another kernel.)
    for kv, counts, few in ((2, [3, 20], 4), (192, [3, 90], 70)):
        case = Case("F16", counts, [30, 100], kv, 1, 64, 16, seed=43, spare_rows=4)
        want, bound = case.expected(True, check(ctx, case).astype(np.float64))
        for rows, end in ((case.packed(max_count=few), 3 + few), (case.packed(rows=10), 10)):
            got = attend(ctx, case, rows=rows)
            assert np.all(np.abs(got - want)[:end] <= bound[:end]) and np.all(got[end:] == 7.25)


@pytest.mark.parametrize("storage", STORAGES)
def test_strided_tensors_at_odd_floats(ctx, storage):
    import torch
    for kv in (2, 192):
        strided(ctx, Case(storage, [1, 35], [200, 40], kv, 2, 64, 16, seed=47))


def strided(ctx, case):
    import torch
    clean = check(ctx, case)
    n = case.q.shape[1]
    wide = torch.zeros(case.rows * (n + 7) + 1, device="cuda")[1:].view(case.rows, n + 7)
    wide[:, 3:3 + n] = torch.from_numpy(case.q).cuda()
    out = torch.full((case.rows * (n + 5) + 3,), 7.25, device="cuda")[3:].view(case.rows, n + 5)
    ctx.paged_attention(case.cache(), case.packed(), wide[:, 3:3 + n], 2 * case.kv, True, case.scale, out[:, 1:1 + n])
    torch.cuda.synchronize()
    out = out.cpu().numpy()
    assert np.array_equal(out[:, 1:1 + n], clean)
    assert np.all(out[:, 0] == 7.25) and np.all(out[:, 1 + n:] == 7.25)


@pytest.mark.parametrize("storage", STORAGES)
def test_pools_past_32_bits(ctx, storage):
    # Slots whose element index passes 2^32 hold what was stored there.
    import torch
    from whispereacp_amd.paged import PagedCache
    heads, page, width = 16, 64, 128
    pages = 2 ** 32 // (heads * page * width) + 4
    cache = PagedCache.allocate(storage, pages, heads, page, width)
    small = Case(storage, [3, 40], [100, 50], heads, 1, width, page, seed=53, spare_pages=0)
    far = np.arange(pages - small.pages, pages)
    for pool, stored in ((cache.keys, small.keys), (cache.values, small.values)):
        pool[int(far[0]):] = device_tensor(stored, storage)
    for pool, powers in ((cache.key_exponents, small.key_exponents), (cache.value_exponents, small.value_exponents)):
        if pool is not None:
            pool[int(far[0]):] = torch.from_numpy(powers).cuda()
    near = small.table.copy()
    small.table = np.where(near >= 0, near + int(far[0]), near).astype(np.int32)
    rows = small.packed()
    keys, device_keys = new_rows(small, 5, 0)
    ctx.paged_append(cache, rows, device_keys, device_keys)
    back = [torch.zeros((small.rows, heads * width), device="cuda") for _ in range(2)]
    ctx.paged_read(cache, rows, *back)
    total = small.rows
    stored, k = store(keys.reshape(total, heads, width), storage)
    want = widen(stored, k, storage).reshape(total, -1)
    assert np.array_equal(back[0].cpu().numpy(), want) and np.array_equal(back[1].cpu().numpy(), want)
    # The attention over them is the attention over the same pages lower down.
    got = attend(ctx, small, cache=cache, rows=rows)
    low = PagedCache(*(t[int(far[0]):].clone() for t in (cache.keys, cache.values, cache.key_exponents,
                                                         cache.value_exponents) if t is not None))
    small.table = near
    assert np.array_equal(got, attend(ctx, small, cache=low)) and np.isfinite(got).all()


# ---------------------------------------------------------------------------
# together, streams, graphs, refusals
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("storage", STORAGES)
def test_a_prompt_and_steps_together(ctx, storage):
    # Prompts in chunks, then single tokens, a stream joining late: append and
    # attention as a decoder would call them, each step against the plain form.
    import torch
    case = Case(storage, [0, 0, 0], [90, 90, 90], 2, 2, 64, 16, seed=59)
    for rows in (case.key_rows, case.value_rows):
        rows[:] = np.nan
    case.quantise()
    cache = case.cache()
    lengths = [0, 0, 0]
    for counts in ([37, 5, 0], [30, 1, 0], [1, 1, 60], [1, 1, 1], [0, 1, 1], [1, 1, 1]):
        case.counts = counts
        lengths = [n + c for n, c in zip(lengths, counts)]
        case.lengths = lengths
        case.starts = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        case.rows = int(case.starts[-1])
        keys, device_keys = new_rows(case, 61 + sum(lengths), 0)
        values, device_values = new_rows(case, 67 + sum(lengths), 0)
        append(ctx, case, device_keys, device_values, cache)
        check_pool(case, cache, keys, values)
        case.keys, case.values = host_array(cache.keys, storage), host_array(cache.values, storage)
        if storage == "E4M3":
            case.key_exponents = cache.key_exponents.cpu().numpy()
            case.value_exponents = cache.value_exponents.cpu().numpy()
        case.q = case.rng.normal(0, 1, (case.rows, 4 * 64)).astype(np.float32)
        check(ctx, case, cache=cache)


def test_the_same_bits_every_time(ctx):
    for count, kv in ((1, 2), (7, 2), (64, 2), (64, 192)):
        case = Case("E4M3", [count, count], [2000, 700], kv, 2, 128, 64, seed=71)
        cache, rows = case.cache(), case.packed()
        first = attend(ctx, case, cache=cache, rows=rows)
        for _ in range(3):
            assert np.array_equal(attend(ctx, case, cache=cache, rows=rows), first)


def test_a_captured_step_follows_its_lengths():
    # Append and attention captured once; each replay takes the lengths, tables
    # and rows of its time. Replays are checked against eager calls between them.
    import torch
    from whispereacp_amd.decoder import KernelContext
    from whispereacp_amd.paged import PagedRows
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        context = KernelContext(S.DecoderShape(64, 1, 1, 64, 64, 1, 1))
        case = Case("E4M3", [1, 1, 1], [600, 600, 600], 2, 2, 64, 32, seed=73)
        cache, eager_cache = case.cache(), case.cache()
        rows = PagedRows(torch.tensor([0, 1, 2, 3], dtype=torch.int32, device="cuda"),
                         torch.ones(3, dtype=torch.int32, device="cuda"),
                         torch.from_numpy(case.table).cuda(), 3, 1, 600)
        lengths = rows._keep[1]
        x = torch.zeros((3, 128), device="cuda")
        q = torch.zeros((3, 256), device="cuda")
        out, eager = torch.zeros((3, 256), device="cuda"), torch.zeros((3, 256), device="cuda")

        def step(into, held):
            context.paged_append(held, rows, x, x)
            context.paged_attention(held, rows, q, 4, True, 0.125, into)

        step(out, cache)
        step(eager, eager_cache)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            step(out, cache)
        for step_lengths in ([1, 5, 599], [300, 6, 600], [301, 7, 33], [302, 500, 34]):
            lengths.copy_(torch.tensor(step_lengths, dtype=torch.int32))
            x.copy_(torch.randn(3, 128))
            q.copy_(torch.randn(3, 256))
            graph.replay()
            stream.synchronize()
            step(eager, eager_cache)
            stream.synchronize()
            assert torch.equal(out, eager) and bool(torch.isfinite(out).all())
            assert torch.equal(cache.keys.view(torch.uint8), eager_cache.keys.view(torch.uint8))


def test_empty_calls(ctx):
    import torch
    from whispereacp_amd.paged import PagedRows
    case = Case("F16", [1], [5], 2, 1, 64, 16)
    cache = case.cache()
    before = host_array(cache.keys, "F16").copy()
    none = torch.zeros((0, 128), device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    for rows in (PagedRows(torch.zeros(1, **i32), torch.zeros(0, **i32), torch.zeros((0, 4), **i32), 0, 0, 0),
                 PagedRows(torch.zeros(3, **i32), torch.zeros(2, **i32), torch.zeros((2, 4), **i32), 0, 0, 0)):
        ctx.paged_append(cache, rows, none, none)
        ctx.paged_read(cache, rows, none, none)
        ctx.paged_attention(cache, rows, none, 2, True, 0.125, none)
    # Rows that see nothing: no length at all, and no table.
    for lengths, table, longest in ((0, 4, 0), (0, 0, 9), (-5, 4, 9)):
        y = torch.full((2, 128), 7.25, device="cuda")
        nothing = PagedRows(torch.tensor([0, 1, 2], **i32), torch.full((2,), lengths, **i32),
                            torch.zeros((2, table), **i32), 2, 1, longest)
        ctx.paged_append(cache, nothing, y, y)
        ctx.paged_attention(cache, nothing, y, 2, True, 0.125, y.clone())
        out = torch.full((2, 128), 7.25, device="cuda")
        ctx.paged_attention(cache, nothing, y, 2, False, 0.125, out)
        torch.cuda.synchronize()
        assert bool((out == 0).all())
    idle = PagedRows(torch.zeros(3, **i32), torch.full((2,), 9, **i32), torch.zeros((2, 4), **i32), 2, 1, 9)
    x = torch.full((2, 128), 7.25, device="cuda")
    ctx.paged_append(cache, idle, x, x)
    ctx.paged_attention(cache, idle, x, 2, True, 0.125, x.clone())
    torch.cuda.synchronize()
    assert np.array_equal(host_array(cache.keys, "F16"), before, equal_nan=True)


def test_refusals(ctx):
    import torch
    from whispereacp_amd.decoder import LogicError
    from whispereacp_amd.paged import PagedCache, PagedRows
    case = Case("F16", [1], [5], 2, 1, 64, 16)
    cache, rows = case.cache(), case.packed()
    x = torch.zeros((1, 128), device="cuda")
    with pytest.raises(ValueError, match="query heads"):
        ctx.paged_attention(cache, rows, torch.zeros((1, 192), device="cuda"), 3, True, 0.125,
                            torch.zeros((1, 192), device="cuda"))
    with pytest.raises(ValueError, match="packed rows"):
        ctx.paged_append(cache, rows, x[:, :64], x)
    with pytest.raises(ValueError, match="packed rows"):
        ctx.paged_append(cache, rows, x.half(), x)
    with pytest.raises(ValueError, match="packed rows"):
        ctx.paged_read(cache, rows, x[:0], x)
    with pytest.raises(ValueError, match="context on device"):
        ctx.paged_append(cache, rows, x.cpu(), x)
    with pytest.raises(ValueError, match="floats apart"):
        ctx.paged_append(cache, case.packed(rows=2), torch.zeros(128, device="cuda").expand(2, 128),
                         torch.zeros((2, 128), device="cuda"))
    with pytest.raises(LogicError, match="heads up to"):
        ctx.paged_append(PagedCache.allocate("F16", 2, 2, 16, 72), rows, torch.zeros((1, 144), device="cuda"),
                         torch.zeros((1, 144), device="cuda"))
    with pytest.raises(LogicError, match="power of two"):
        ctx.paged_append(PagedCache.allocate("F16", 2, 2, 24, 64), rows, x, x)
    with pytest.raises(LogicError):
        PagedCache.allocate("I8", 2, 2, 16, 64)
    pool = torch.zeros((2, 2, 16, 64), device="cuda")
    with pytest.raises(ValueError, match="one type"):
        PagedCache(pool, pool.half())
    with pytest.raises(ValueError, match="exponents"):
        PagedCache(pool.to(torch.float8_e4m3fn), pool.to(torch.float8_e4m3fn))
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache(pool.transpose(0, 1), pool.transpose(0, 1))
    i32 = dict(dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="int32"):
        PagedRows(torch.zeros(2, device="cuda"), torch.zeros(1, **i32), torch.zeros((1, 1), **i32), 1, 1, 1)
    with pytest.raises(ValueError, match="positions a sequence"):
        PagedRows(torch.zeros(2, **i32), torch.zeros(1, **i32), torch.zeros((1, 1), **i32), 2 ** 32, 1, 1)
    with pytest.raises(ValueError, match="sequences"):
        PagedRows(torch.zeros(3, **i32), torch.zeros(1, **i32), torch.zeros((1, 1), **i32), 1, 1, 1)

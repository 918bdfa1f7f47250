"""The paged cache as programs use it beyond one call: every kernel and join captured
and replayed over other lengths, two contexts at once over one pool, pages that
sequences share, scales of zero and below (plain forms: test_gpu_paged.py).
"""

import numpy as np
import pytest

from helpers import ensure_library
from test_gpu_paged import Case, attend, check, ctx  # noqa: F401 (ctx: the fixture)
from whispereacp_amd import synthetic as S

pytestmark = pytest.mark.gpu


def context():
    ensure_library()
    from whispereacp_amd.decoder import KernelContext
    return KernelContext(S.DecoderShape(64, 1, 1, 64, 64, 1, 1))


CAPTURED = {
    # storage, counts, longest, kv, group, width, page, then the lengths of each replay
    "one-span": ("F16", [1, 1], 200, 2, 2, 64, 16, [[200, 1], [3, 150], [64, 65]]),
    "joined-in-place": ("E4M3", [1, 2], 2000, 2, 2, 128, 64, [[2000, 5], [700, 1999], [2, 300]]),
    "joined-after": ("BF16", [1], 9000, 1, 2, 64, 64, [[9000], [257], [5000], [1]]),
    "fp32": ("F32", [5, 1], 1500, 2, 1, 80, 16, [[1500, 30], [20, 900], [5, 1]]),
    "chunks": ("E4M3", [70, 66], 300, 192, 1, 64, 16, [[300, 66], [71, 299], [128, 130]]),
    "cut-chunks": ("F16", [70], 6200, 128, 1, 16, 64, [[6200], [100], [4300]]),
}


@pytest.mark.parametrize("name", CAPTURED)
def test_captured_attention_follows_its_lengths(name):
    import torch
    from whispereacp_amd.paged import PagedRows
    storage, counts, longest, kv, group, width, page, replays = CAPTURED[name]
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = context()
        case = Case(storage, counts, [longest] * len(counts), kv, group, width, page, seed=301)
        cache = case.cache()
        lengths = torch.tensor(replays[0], dtype=torch.int32, device="cuda")
        rows = PagedRows(torch.from_numpy(case.starts).cuda(), lengths, torch.from_numpy(case.table).cuda(), case.rows,
                         max(counts), longest)
        q = torch.from_numpy(case.q).cuda()
        out = torch.zeros_like(q)

        def attention():
            ctx.paged_attention(cache, rows, q, kv * group, True, case.scale, out)

        attention()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            attention()
        for at, now in enumerate(replays + replays[::-1]):
            lengths.copy_(torch.tensor(now, dtype=torch.int32))
            q.copy_(torch.from_numpy(case.rng.normal(0, 1, case.q.shape).astype(np.float32)))
            out.fill_(7.25)
            graph.replay()
            stream.synchronize()
            replayed = out.cpu().numpy()
            attention()
            stream.synchronize()
            assert np.array_equal(replayed, out.cpu().numpy()), at
            case.q, case.lengths = q.cpu().numpy(), list(now)
            want, bound = case.expected(True, np.full(replayed.shape, 7.25))
            assert np.all(np.abs(replayed - want) <= bound), at


def test_two_contexts_at_once_over_one_pool():
    # Each with its own stream, scratch and counters; the calls overlap on the GPU.
    import torch
    case = Case("E4M3", [1, 2], [4000, 3000], 2, 2, 128, 64, seed=307)
    cache, rows = case.cache(), case.packed()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    users = []
    for i, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            q = torch.from_numpy(case.q * np.float32(1 + i)).cuda()
            users.append((context(), q, [torch.zeros_like(q) for _ in range(20)]))
    torch.cuda.synchronize()
    for turn in range(20):
        for stream, (ctx, q, outs) in zip(streams, users):
            with torch.cuda.stream(stream):
                ctx.paged_attention(cache, rows, q, 4, True, case.scale, outs[turn])
    torch.cuda.synchronize()
    for i, (ctx, q, outs) in enumerate(users):
        case.q = q.cpu().numpy()
        want, bound = case.expected(True, np.zeros(case.q.shape))
        for out in outs:
            assert torch.equal(out, outs[0])
        assert np.all(np.abs(outs[0].cpu().numpy() - want) <= bound), i


@pytest.mark.parametrize("storage", ["F16", "E4M3"])
@pytest.mark.parametrize("count,kv", [(1, 2), (9, 2), (70, 192)])
def test_sequences_that_share_pages(ctx, storage, count, kv):  # noqa: F811
    # A common prompt: the first pages of both sequences are the same ones.
    case = Case(storage, [count, count], [200, 180], kv, 1, 64, 16, seed=311)
    case.table[1, :5] = case.table[0, :5]
    check(ctx, case)


@pytest.mark.parametrize("storage", ["F32", "F16", "BF16", "E4M3"])
@pytest.mark.parametrize("scale", [0.0, -0.125, 2.0 ** -20])
@pytest.mark.parametrize("count,kv", [(1, 2), (70, 192)])
def test_scales_of_zero_and_below(ctx, storage, scale, count, kv):  # noqa: F811
    case = Case(storage, [count], [300], kv, 1, 64, 16, seed=313)
    case.scale = scale
    check(ctx, case)


@pytest.mark.parametrize("storage", ["F32", "F16", "BF16", "E4M3"])
@pytest.mark.parametrize("count,kv", [(3, 2), (40, 2), (70, 192)])
def test_a_query_that_is_nan_stays_in_its_row(ctx, storage, count, kv):  # noqa: F811
    case = Case(storage, [count, 1], [300, 20], kv, 1, 64, 16, seed=317)
    clean = check(ctx, case)
    case.q[1, 5] = np.nan
    case.q[2, 64 + 7] = np.inf
    got = attend(ctx, case)
    assert np.isnan(got[1, :64]).all() and np.isnan(got[2, 64:128]).all()
    clean[1, :64] = got[1, :64] = clean[2, 64:128] = got[2, 64:128] = 0
    assert np.array_equal(got, clean)

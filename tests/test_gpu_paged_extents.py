"""The paged cache's calls that pass a launch's extents and go in several: more than
65535 sequences, more than 65535 row tiles, more than 2^24 packed rows. Attention
against softmax in 64 bits with test_gpu_paged.py's bound, on the GPU (the sizes);
storing and reading back exactly.
"""

import pytest

from test_gpu_paged import ctx  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu

WIDTH = 16


def attended(q, keys, values, seen, scale):
    """Rows q [n, w] over keys and values [n or 1, k, w], the first seen[n] of them, and the bound of each value."""
    import torch
    q, keys, values = q.double(), keys.double(), values.double()
    hidden = torch.arange(keys.shape[1], device="cuda")[None] >= seen[:, None]
    if keys.shape[0] == 1:
        scores = (q @ keys[0].T.contiguous()) * scale
        size = (q.abs() @ keys[0].abs().T.contiguous()) * scale
    else:
        scores = (q[:, None] * keys).sum(-1) * scale
        size = (q[:, None] * keys).abs().sum(-1) * scale
    p = torch.softmax(scores.masked_fill(hidden, -torch.inf), dim=1)
    score = size.masked_fill(hidden, 0).amax(dim=1, keepdim=True) * ((WIDTH + 8) * 2.0 ** -24 + 2.0 ** -22 + 2.0 ** -23)
    n = seen[:, None].double()
    if keys.shape[0] == 1:
        out, sizes = p @ values[0], p @ values[0].abs()
    else:
        out, sizes = (p[:, :, None] * values).sum(1), (p[:, :, None] * values.abs()).sum(1)
    return out, sizes * (2 * score + (n + 16) * 2.0 ** -24) + n * 2.0 ** -30 * values.abs().amax()


def randn(*shape, seed):
    import torch
    generator = torch.Generator(device="cuda")
    generator.manual_seed(seed)
    return torch.randn(shape, generator=generator, device="cuda")


@pytest.mark.parametrize("storage", ["F32", "F16"])
@pytest.mark.parametrize("group", [1, 65])  # (65 pairs a sequence take blocks of 128 in 16 bits)
def test_more_sequences_than_a_launch_takes(ctx, storage, group):  # noqa: F811
    import torch
    from whispereacp_amd.paged import PagedCache, PagedRows
    n = 70000
    pool = [randn(n, 1, 16, WIDTH, seed=7 + i).to({"F32": torch.float32, "F16": torch.float16}[storage]) for i in (0, 1)]
    table = torch.randperm(n, generator=torch.Generator().manual_seed(3)).int().cuda()
    lengths = torch.arange(n, device="cuda") % 3 + 1
    q = randn(n, group * WIDTH, seed=11)
    out = torch.full_like(q, 7.25)
    rows = PagedRows(torch.arange(n + 1, dtype=torch.int32, device="cuda"), lengths.int(), table[:, None].contiguous(), n, 1, 3)
    ctx.paged_attention(PagedCache(*pool), rows, q, group, True, 0.25, out)
    torch.cuda.synchronize()
    keys, values = (p[table.long(), 0, :3].float() for p in pool)
    for g in range(0, group, 13):
        part = slice(g * WIDTH, (g + 1) * WIDTH)
        want, bound = attended(q[:, part], keys, values, lengths, 0.25)
        assert bool(((out[:, part].double() - want).abs() <= bound).all()), g


@pytest.mark.parametrize("storage,tile_rows", [("F32", 32), ("F16", 128)])
def test_more_row_tiles_than_a_launch_takes(ctx, storage, tile_rows):  # noqa: F811
    import torch
    from whispereacp_amd.paged import PagedCache, PagedRows
    rows, length = 4, 70
    group = (65535 * tile_rows) // rows + 1000  # (tiles of a few hundred past the extent)
    dtype = {"F32": torch.float32, "F16": torch.float16}[storage]
    pool = [randn(5, 1, 16, WIDTH, seed=17 + i).to(dtype) for i in (0, 1)]
    table = torch.tensor([[3, 0, 4, 1, 2]], dtype=torch.int32, device="cuda")
    q = randn(rows, group * WIDTH, seed=23)
    out = torch.full_like(q, 7.25)
    i32 = dict(dtype=torch.int32, device="cuda")
    packed = PagedRows(torch.tensor([0, rows], **i32), torch.tensor([length], **i32), table, rows, rows, length)
    ctx.paged_attention(PagedCache(*pool), packed, q, group, True, 0.25, out)
    torch.cuda.synchronize()
    keys, values = (p[table[0].long(), 0].flatten(0, 1)[None, :length].float() for p in pool)
    for row in range(rows):
        got = out[row].view(group, WIDTH)
        seen = torch.full((group,), length - rows + row + 1, device="cuda")
        want, bound = attended(q[row].view(group, WIDTH), keys, values, seen, 0.25)
        assert bool(((got.double() - want).abs() <= bound).all()), row


def test_more_packed_rows_than_a_launch_takes(ctx):  # noqa: F811
    import torch
    from whispereacp_amd.paged import PagedCache, PagedRows
    counts = [2 ** 22 + 77, 2 ** 23, 1, 2 ** 22 + 1000]
    lengths = [counts[0], counts[1] + 5, 900, counts[3]]
    blocks = [-(-n // 1024) for n in lengths]
    pages, rows = sum(blocks) + 1, sum(counts) + 3
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(5)).int()
    table, at = torch.full((4, max(blocks)), -1, dtype=torch.int32), 0
    for s, n in enumerate(blocks):
        table[s, :n] = order[at:at + n]
        at += n
    starts = torch.tensor([0] + counts).cumsum(0).int().cuda()
    packed = PagedRows(starts, torch.tensor(lengths, dtype=torch.int32, device="cuda"), table.cuda(), rows, max(counts),
                       max(lengths))
    cache = PagedCache.allocate("F16", pages, 1, 1024, WIDTH)
    new = [randn(rows, WIDTH, seed=29 + i) for i in (0, 1)]
    back = [torch.full((rows, WIDTH), 3.5, device="cuda") for _ in (0, 1)]
    assert rows > 2 ** 24
    ctx.paged_append(cache, packed, *new)
    ctx.paged_read(cache, packed, *back)
    torch.cuda.synchronize()
    for x, y in zip(new, back):
        want = x.half().float()
        want[sum(counts):] = 3.5
        assert torch.equal(y, want)

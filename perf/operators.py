"""The calls of the paged key/value cache whose time this library is judged by:
appending new rows to the pages (in 8 bits where the cache holds E4M3), reading
cached rows back, and attention of new tokens over the pages.

A cache is a pool of pages [pages, heads, page, width] for keys and another for
values. Sequence s owns the pages its row of the table names, in the order of
its positions; its new rows lie one after another in the packed rows, sequence
after sequence, and are its last positions. E4M3 rows (one position of one
head) carry a power of two each, held as an exponent byte biased by 127.
"""

from __future__ import annotations

import math
import random

import torch

own = False  # False: the plain forms; True: the library's kernels

_TORCH = {"F32": torch.float32, "F16": torch.float16, "BF16": torch.bfloat16, "E4M3": torch.float8_e4m3fn}
_BYTES = {"F32": 4, "F16": 2, "BF16": 2, "E4M3": 1}


def listed():
    return [
        # A step of 32 transcription streams (large-v3's heads): each stream's
        # one new key and value row, straight out of the fused projection.
        dict(name="append-step-f16", op="append", storage="F16", sequences=32, kv=20, group=1, width=64, page=16,
             count=1, length=448, ragged=True, causal=True, fused=True, spare=0),
        # The prompts of eight new sequences entering a server's 8-bit cache.
        dict(name="append-prompts-e4m3", op="append", storage="E4M3", sequences=8, kv=8, group=4, width=128, page=64,
             count=4096, length=4096, ragged=True, causal=True, fused=True, spare=5),
        # One window's cross keys and values (base.en) back from their pages.
        dict(name="read-window-bf16", op="read", storage="BF16", sequences=1, kv=8, group=1, width=64, page=32,
             count=1500, length=1500, ragged=False, causal=False, fused=False, spare=0),
        # Four long sequences moved out of an 8-bit cache.
        dict(name="read-long-e4m3", op="read", storage="E4M3", sequences=4, kv=8, group=4, width=128, page=64,
             count=16384, length=16384, ragged=False, causal=False, fused=False, spare=0),
        # One token of one short stream (tiny.en's heads): latency alone.
        dict(name="step-1-f16", op="attention", storage="F16", sequences=1, kv=6, group=1, width=64, page=16,
             count=1, length=131, ragged=False, causal=True, fused=False, spare=0),
        # A step of 32 transcription streams (large-v3's heads) over their
        # self caches, of every length up to the longest.
        dict(name="step-32-e4m3", op="attention", storage="E4M3", sequences=32, kv=20, group=1, width=64, page=32,
             count=1, length=448, ragged=True, causal=True, fused=True, spare=3),
        # 16 streams' four prompt tokens over a window's cross keys (medium's
        # heads): every key is seen.
        dict(name="cross-16x4-bf16", op="attention", storage="BF16", sequences=16, kv=16, group=1, width=64, page=64,
             count=4, length=1500, ragged=False, causal=False, fused=False, spare=0),
        # Proposed tokens checked together, five a stream, in an fp32 cache of
        # heads 80 wide.
        dict(name="verify-8x5-f32", op="attention", storage="F32", sequences=8, kv=16, group=1, width=80, page=16,
             count=5, length=1500, ragged=True, causal=True, fused=False, spare=0),
        # A step of 64 sequences of a server, four query heads a cached head.
        dict(name="serve-64-e4m3", op="attention", storage="E4M3", sequences=64, kv=8, group=4, width=128, page=64,
             count=1, length=8192, ragged=True, causal=True, fused=True, spare=0),
        # One token of one very long sequence.
        dict(name="long-1-bf16", op="attention", storage="BF16", sequences=1, kv=8, group=4, width=128, page=128,
             count=1, length=131072, ragged=False, causal=True, fused=False, spare=0),
        # Chunks of prompts over what the cache holds of them (small's heads).
        dict(name="chunk-4x512-f16", op="attention", storage="F16", sequences=4, kv=12, group=1, width=64, page=32,
             count=512, length=2048, ragged=True, causal=True, fused=True, spare=7),
        # Two long prompts' next chunks, 2048 tokens over up to 16384.
        dict(name="prefill-2x2048-e4m3", op="attention", storage="E4M3", sequences=2, kv=8, group=4, width=128,
             page=64, count=2048, length=16384, ragged=False, causal=True, fused=False, spare=0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention", "attention"])
    storage = rng.choice(list(_BYTES))
    width = rng.choice([64, 64, 128, 128, 16 * rng.randint(1, 8)])
    kv = _log_int(rng, 1, 24)
    group = rng.choice([1, 1, 1, 2, 3, 4, 5, 8])
    page = 16 << rng.randint(0, 4)
    sequences = _log_int(rng, 1, 96)
    causal = op == "append" or rng.random() < 0.8
    length = _log_int(rng, 1, 131072)
    count = 1
    if op == "read":
        count = length if rng.random() < 0.5 else rng.randint(1, length)
    elif rng.random() < 0.6:
        count = _log_int(rng, 1, 4096)
    while sequences * length * kv * width > (2.5e8 if op == "attention" else 6e7):  # elements of each pool
        if sequences > 1:
            sequences = (sequences + 1) // 2
        else:
            length = length // 2 + 1
    count = min(count, length)
    while op == "attention" and sequences * kv * group * count * length > 1e9:  # scores
        count = count // 2 + 1
        if count <= 2:
            sequences = (sequences + 1) // 2
    return dict(op=op, storage=storage, sequences=sequences, kv=kv, group=group, width=width, page=page, count=count,
                length=length, ragged=rng.random() < 0.7, causal=causal, fused=rng.random() < 0.5,
                spare=rng.choice([0, 0, rng.randint(1, 9)]))


def _extents(case):
    """New rows and cached positions (the new ones among them) of each
    sequence. Ragged: the first is the longest, the others spread below it, and
    of four or more one rests (no new row)."""
    counts, lengths = [], []
    for i in range(case["sequences"]):
        part = 1.0 if i == 0 or not case["ragged"] else (0.6180339887 * i) % 1.0
        count = 1 + int((case["count"] - 1) * part)
        length = max(count, int(math.ceil(case["length"] * (0.1 + 0.9 * part))))
        if case["ragged"] and case["sequences"] >= 4 and i == case["sequences"] // 2:
            count = 0
        counts.append(count)
        lengths.append(length)
    return counts, lengths


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _quantise(rows):
    """E4M3 values and exponent bytes of fp32 rows [..., width]: the least power
    of two that brings a row's largest magnitude to 448 or below."""
    mantissa, exponent = torch.frexp(rows.abs().amax(dim=-1))
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8).clamp(-80, 120)
    return torch.ldexp(rows, -exponent[..., None]).to(torch.float8_e4m3fn), (exponent + 127).to(torch.uint8)


def _pool(case, pages, generator, spread):
    """A pool as steps before this one left it; every slot holds some row."""
    shape = (pages, case["kv"], case["page"], case["width"])
    rows = torch.randn(shape, generator=generator, device="cuda")
    rows *= spread
    if case["storage"] == "E4M3":
        return _quantise(rows)
    return rows.to(_TORCH[case["storage"]]), None


def prepare(case, seed):
    counts, lengths = _extents(case)
    kv, width, page, heads = case["kv"], case["width"], case["page"], case["kv"] * case["group"]
    generator = torch.Generator(device="cuda")
    generator.manual_seed(int(seed) * 7919 + 17)

    # The table: each sequence's pages in an order of their own, -1 past its end.
    blocks = [-(-n // page) for n in lengths]
    pages = sum(blocks) + 3
    order = list(range(pages))
    random.Random(int(seed)).shuffle(order)
    table_width, table, at = max(blocks), [], 0
    for n in blocks:
        table.append(order[at:at + n] + [-1] * (table_width - n))
        at += n
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    rows = starts[-1] + case["spare"]

    # Keys have channels louder than others, values rows louder than others.
    channels = torch.exp(0.5 * torch.randn((width,), generator=generator, device="cuda"))
    loud = torch.exp(0.5 * torch.randn((pages, kv, page, 1), generator=generator, device="cuda"))
    keys, key_exponents = _pool(case, pages, generator, channels)
    values, value_exponents = _pool(case, pages, generator, loud)

    state = dict(case=case, keys=keys, values=values, key_exponents=key_exponents, value_exponents=value_exponents,
                 table=torch.tensor(table, dtype=torch.int32, device="cuda"),
                 starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                 rows=rows, max_count=max(counts), max_length=max(lengths), scale=width ** -0.5)
    # The new rows: columns of the fused projection's output, or tensors of their own.
    fused = torch.randn((rows, (heads + 2 * kv) * width), generator=generator, device="cuda")
    q, k, v = fused.split([heads * width, kv * width, kv * width], dim=1)
    if not case["fused"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    if case["op"] == "append":
        state.update(new_keys=k, new_values=v)
    elif case["op"] == "read":
        state.update(out_keys=torch.zeros((rows, kv * width), device="cuda"),
                     out_values=torch.zeros((rows, kv * width), device="cuda"))
    else:
        state.update(q=q, out=torch.zeros((rows, heads * width), device="cuda"))
    if own:
        from whispereacp_amd import synthetic as S
        from whispereacp_amd.decoder import KernelContext
        from whispereacp_amd.paged import PagedCache, PagedRows
        state["context"] = KernelContext(S.DecoderShape(64, 1, 1, 64, 64, 1, 1))
        state["cache"] = PagedCache(keys, values, key_exponents, value_exponents)
        state["batch"] = PagedRows(state["starts"], state["lengths"], state["table"], rows, state["max_count"],
                                   state["max_length"])
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def _positions(s):
    """Packed rows of each sequence [sequences, max_count] (-1: none) and their positions."""
    first, counts = s["starts"][:-1, None].long(), (s["starts"][1:] - s["starts"][:-1])[:, None].long()
    index = torch.arange(s["max_count"], device="cuda")[None]
    return torch.where(index < counts, first + index, -1), s["lengths"][:, None].long() - counts + index


def _slots(s):
    """For the packed rows in order: the page and the place in it of each."""
    rows, positions = _positions(s)
    sequence = torch.arange(rows.shape[0], device="cuda")[:, None].expand_as(rows)
    taken = rows >= 0
    positions, sequence = positions[taken], sequence[taken]
    page = s["case"]["page"]
    return rows[taken], s["table"][sequence, positions // page].long(), positions % page


def _append(s):
    case = s["case"]
    rows, pages, places = _slots(s)
    for pool, exponents, new in ((s["keys"], s["key_exponents"], s["new_keys"]),
                                 (s["values"], s["value_exponents"], s["new_values"])):
        x = new[rows].view(-1, case["kv"], case["width"])
        if exponents is None:
            pool[pages, :, places] = x.to(pool.dtype)
        else:
            stored, powers = _quantise(x)
            pool.view(torch.uint8)[pages, :, places] = stored.view(torch.uint8)
            exponents[pages, :, places] = powers
    return _pools(s)


def _pools(s):
    return [t for t in (s["keys"], s["values"], s["key_exponents"], s["value_exponents"]) if t is not None]


def _widened(pool, exponents, pages, places=None):
    """Whole pages of a pool, or rows of them, in 32 bits."""
    def at(t):
        return t[pages] if places is None else t[pages, :, places]
    if exponents is None:
        return at(pool).float()
    values = at(pool.view(torch.uint8)).view(torch.float8_e4m3fn).float()
    return torch.ldexp(values, at(exponents).int()[..., None] - 127)


def _read(s):
    rows, pages, places = _slots(s)
    s["out_keys"][rows] = _widened(s["keys"], s["key_exponents"], pages, places).flatten(1)
    s["out_values"][rows] = _widened(s["values"], s["value_exponents"], pages, places).flatten(1)
    return s["out_keys"], s["out_values"]


def _attention(s):
    case = s["case"]
    kv, group, width = case["kv"], case["group"], case["width"]
    rows, positions = _positions(s)
    sequences, count = rows.shape
    table = s["table"].long().clamp(min=0)
    length = table.shape[1] * case["page"]

    def cached(pool, exponents):  # [sequences, kv, length, width]
        return _widened(pool, exponents, table).transpose(1, 2).reshape(sequences, kv, length, width)

    q = s["q"][rows.clamp(min=0)].view(sequences, count, kv, group, width).permute(0, 2, 1, 3, 4)
    q = (q * s["scale"]).reshape(sequences, kv, count * group, width)
    scores = torch.matmul(q, cached(s["keys"], s["key_exponents"]).transpose(2, 3).contiguous())
    scores = scores.view(sequences, kv, count, group, length)
    key = torch.arange(length, device="cuda")
    seen = (key < s["lengths"][:, None])[:, None]
    if case["causal"]:
        seen = seen & (key <= positions[:, :, None])
    scores = scores.masked_fill(~seen[:, None, :, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    scores = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = scores.sum(dim=-1, keepdim=True)
    values = cached(s["values"], s["value_exponents"])
    values = values.masked_fill(~(key < s["lengths"][:, None])[:, None, :, None], 0.0)
    out = torch.matmul(scores.view(sequences, kv, count * group, length), values)
    out = out.view(sequences, kv, count, group, width) / torch.where(total == 0, 1.0, total)
    out = out.permute(0, 2, 1, 3, 4).reshape(sequences, count, kv * group * width)
    s["out"][rows[rows >= 0]] = out[rows >= 0]
    return s["out"]


def run(s):
    case = s["case"]
    if own:
        context, cache, batch = s["context"], s["cache"], s["batch"]
        if case["op"] == "append":
            context.paged_append(cache, batch, s["new_keys"], s["new_values"])
            return _pools(s)
        if case["op"] == "read":
            context.paged_read(cache, batch, s["out_keys"], s["out_values"])
            return s["out_keys"], s["out_values"]
        context.paged_attention(cache, batch, s["q"], case["kv"] * case["group"], case["causal"], s["scale"], s["out"])
        return s["out"]
    return {"append": _append, "read": _read, "attention": _attention}[case["op"]](s)


def work(case):
    counts, lengths = _extents(case)
    row, heads = case["kv"] * case["width"], case["kv"] * case["group"]
    exponents = case["kv"] if case["storage"] == "E4M3" else 0
    stored = 2 * (row * _BYTES[case["storage"]] + exponents)  # a position's key and value
    fresh = sum(counts)
    if case["op"] != "attention":
        return {"bytes": fresh * (stored + 2 * 4 * row), "flops": 0}
    pairs = sum(n * m - (n * (n - 1) // 2 if case["causal"] else 0) for n, m in zip(counts, lengths))
    held = sum(m for n, m in zip(counts, lengths) if n > 0)
    return {"bytes": held * stored + fresh * 2 * 4 * heads * case["width"],
            "flops": 4 * heads * case["width"] * pairs}


# ---------------------------------------------------------------------------
# the definition in 64 bits, sequence by sequence
# ---------------------------------------------------------------------------

def _stored_rows(pool, exponents, pages, length):
    """A sequence's cached rows in order, [kv, length, width] in 64 bits."""
    if exponents is None:
        rows = pool[pages].double()
    else:
        rows = pool.view(torch.uint8)[pages].view(torch.float8_e4m3fn).double()
        rows = rows * torch.exp2(exponents[pages].double() - 127.0)[..., None]
    return torch.cat(list(rows), dim=1)[:, :length]


def exact(case, seed):
    s = prepare(case, seed)
    counts, lengths = _extents(case)
    page, kv, group, width = case["page"], case["kv"], case["group"], case["width"]
    table = s["table"].tolist()
    outs = None
    if case["op"] == "append":
        outs = [s["keys"].double(), s["values"].double()]
    elif case["op"] == "read":
        outs = [s["out_keys"].double(), s["out_values"].double()]
    else:
        outs = [s["out"].double()]
    first = 0
    for count, length, row in zip(counts, lengths, table):
        if count == 0:
            continue
        pages = torch.tensor(row[:-(-length // page)], device="cuda")
        span = slice(first, first + count)
        positions = torch.arange(length - count, length, device="cuda")
        if case["op"] == "append":
            at, place = pages[positions // page], positions % page
            for out, new in zip(outs, (s["new_keys"], s["new_values"])):
                x = new[span].double().view(count, kv, width)
                if case["storage"] == "E4M3":
                    power = torch.ceil(torch.log2(x.abs().amax(dim=-1, keepdim=True).clamp(min=1e-300) / 448.0))
                    x = x / torch.exp2(power.clamp(-80, 120))
                out[at, :, place] = x
        else:
            stored = [_stored_rows(s["keys"], s["key_exponents"], pages, length),
                      _stored_rows(s["values"], s["value_exponents"], pages, length)]
            if case["op"] == "read":
                for out, held in zip(outs, stored):
                    out[span] = held[:, length - count:].permute(1, 0, 2).reshape(count, kv * width)
            else:
                q = s["q"][span].double().view(count, kv, group, width)
                hidden = torch.arange(length, device="cuda")[None, :] > positions[:, None]
                result = outs[0][span].view(count, kv, group, width)
                for h in range(kv):
                    for g in range(group):
                        logits = torch.mm(q[:, h, g] * s["scale"], stored[0][h].t().contiguous())
                        if case["causal"]:
                            logits.masked_fill_(hidden, -math.inf)
                        result[:, h, g] = torch.mm(torch.softmax(logits, dim=1), stored[1][h])
        first += count
    if case["op"] == "append":
        return outs + ([None, None] if case["storage"] == "E4M3" else [])
    return tuple(outs) if case["op"] == "read" else outs[0]

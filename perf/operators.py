"""The work of the paged 8-bit key/value cache that its speed is measured on.

A server with many sessions of different ages keeps their keys and values in
pages of 16, 32 or 64 tokens, in 8 bits (int8 or e4m3) with one scale per page
and key/value head.  Each step does three things, each a `kind` here: it gives
out pages and makes the step's row map (`plan`), stores the step's keys and
values (`append`), and attends from the step's query rows over each sequence's
pages (`attention`).  Heads of 128; 16 query and 8 key/value heads are the
talker's, the others are what a user may bring.

Page layout, per key/value head a run of 2048-byte granules of 16 tokens:
  key   (token t, dimension d): (d / 64) * 1024 + t * 64 + d % 64
  value (token t, dimension d): (d / 64) * 1024 + (t / 4) * 256 + (d % 16) * 16 + (d / 16 % 4) * 4 + t % 4
"""
import math
import pathlib
import sys

import torch

DEVICE = "cuda"
HEAD = 128
GRANULE = 16  # tokens of a 2048-byte granule
SCALE = HEAD ** -0.5

own = False  # True: run() calls the framework's operators; False: their plain form
_library = None


def _hip():
    global _library
    if _library is None:
        package = str(pathlib.Path(__file__).resolve().parent.parent / "qwen3-tts-native_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        import qwen3_tts_hip

        _library = qwen3_tts_hip
    return _library


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------
def _plan(sequences, page, longest, prompt, prompts, ended, scarce=False):
    return {"kind": "plan", "sequences": sequences, "page": page, "longest": longest, "prompt": prompt,
            "prompts": prompts, "ended": ended, "scarce": scarce}


def _append(fmt, page, kv_heads, sequences, shortest, longest, held):
    return {"kind": "append", "format": fmt, "page": page, "kv_heads": kv_heads, "sequences": sequences,
            "shortest": shortest, "longest": longest, "held": held}


def _attention(fmt, page, heads, kv_heads, sequences, shortest, longest, few, many, window=0):
    return {"kind": "attention", "format": fmt, "page": page, "heads": heads, "kv_heads": kv_heads,
            "sequences": sequences, "shortest": shortest, "longest": longest, "few": few, "many": many,
            "window": window}


def listed():
    return [
        # the lockstep batch of eight sessions takes its next frame: the smallest call
        {"name": "plan_8", **_plan(8, 16, 1024, 1, 0, 0)},
        # a busy server's step: most sessions one frame on, some prompts let in, some sessions ended
        {"name": "plan_1000", **_plan(1000, 16, 2048, 401, 60, 25)},
        # eight sessions store one frame's key and value
        {"name": "append_8", **_append("int8", 16, 8, 8, 1, 1, 1023)},
        # a short prompt beside single tokens of other sessions
        {"name": "append_ragged", **_append("e4m3", 32, 8, 37, 1, 97, 333)},
        # the prompts of a full server's start: bandwidth
        {"name": "append_16k", **_append("int8", 16, 8, 40, 17, 801, 0)},
        # eight sessions' next frame over contexts of up to 1024
        {"name": "decode_8", **_attention("int8", 16, 16, 8, 8, 97, 1024, 1, 1)},
        # one listener of a long recording: one row, split over its context
        {"name": "decode_long", **_attention("e4m3", 64, 16, 8, 1, 65521, 65521, 1, 1)},
        # sixty-four sessions of every age
        {"name": "decode_64", **_attention("e4m3", 16, 16, 8, 64, 33, 4096, 1, 1)},
        # a full server: the cache's bytes from HBM
        {"name": "decode_256", **_attention("int8", 32, 16, 8, 256, 1111, 8192, 1, 1)},
        # one voice description longer than the matrix-product prefill's 512 rows
        {"name": "prompt_801", **_attention("int8", 16, 16, 8, 1, 801, 801, 801, 801)},
        # long prompts of different lengths together, more query heads to a key head
        {"name": "prompt_4096", **_attention("e4m3", 16, 32, 8, 4, 1777, 4096, 1777, 4096)},
        # a chunk of a long prompt beside single tokens, attention within a window
        {"name": "chunk_window", **_attention("int8", 64, 16, 4, 24, 700, 16384, 1, 512, 4000)},
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    limits = {}
    for case in listed():
        w = work(case)
        kept = limits.setdefault(case["kind"], {"bytes": 0, "flops": 0})
        for k in kept:
            kept[k] = max(kept[k], w[k])
    shapes = [{k: v for k, v in c.items() if k != "name"} for c in listed()]
    while True:
        case = _drawn(rng)
        w = work(case)
        if case not in shapes and all(w[k] <= limits[case["kind"]][k] for k in w):
            return case


def _drawn(rng):
    kind = rng.choice(["plan", "append", "append", "attention", "attention", "attention", "attention"])
    page, fmt = rng.choice([16, 32, 64]), rng.choice(["int8", "e4m3"])
    if kind == "plan":
        sequences = _log_int(rng, 1, 1000)
        prompts = rng.randint(0, max(0, sequences // 10))
        return _plan(sequences, page, _log_int(rng, 16, 2048), _log_int(rng, 1, 401), prompts,
                     rng.randint(0, (sequences - prompts) // 4), rng.choice([False, False, True]))
    if kind == "append":
        sequences, longest = _log_int(rng, 1, 256), _log_int(rng, 1, 801)
        return _append(fmt, page, rng.choice([1, 2, 4, 8]), sequences, rng.randint(1, longest), longest,
                       rng.choice([0, _log_int(rng, 1, 1023)]))
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (8, 8), (16, 4), (32, 8), (14, 2), (16, 2), (16, 1)])
    window = rng.choice([0, 0, 0, _log_int(rng, 64, 4096)])
    shape = rng.choice(["decode", "decode", "prompt", "mixed"])
    if shape == "decode":
        longest = _log_int(rng, 1, 16384)
        return _attention(fmt, page, heads, kv_heads, _log_int(rng, 1, 256), rng.randint(1, longest), longest, 1, 1,
                          window)
    if shape == "prompt":
        longest = _log_int(rng, 2, 4096)
        shortest = rng.randint(1, longest)
        return _attention(fmt, page, heads, kv_heads, _log_int(rng, 1, 16), shortest, longest, shortest, longest,
                          window)
    longest = _log_int(rng, 64, 8192)
    few = rng.randint(1, 3)
    return _attention(fmt, page, heads, kv_heads, _log_int(rng, 2, 32), rng.randint(few, longest), longest, few,
                      rng.randint(few, min(512, longest)), window)


# ---------------------------------------------------------------------------
# Sizes: they follow from the case alone
# ---------------------------------------------------------------------------
def _spread(low, high, count):
    """`count` whole numbers from high down to low, in an order that is neither rising nor falling."""
    if count == 1:
        return [high]
    step = next(s for s in range(count // 2 + 1, 2 * count) if math.gcd(s, count) == 1)
    return [high - (high - low) * (i * step % count) // (count - 1) for i in range(count)]


def _sizes(case):
    """(tokens held before the step, tokens of the step) of each sequence; -1: the sequence ends."""
    n = case["sequences"]
    if case["kind"] == "plan":
        held = _spread(1, case["longest"], n)
        new = [1] * n
        for i in range(case["prompts"]):  # a prompt for an empty place of the batch
            at = i * n // case["prompts"]
            held[at], new[at] = 0, case["prompt"] - i % max(1, case["prompt"] // 2)
        at = 0
        for _ in range(case["ended"]):
            while new[at % n] != 1 or held[at % n] == 0:
                at += 1
            new[at % n] = -1
            at += 3
        return held, new
    if case["kind"] == "append":
        held = [0] * n if case["held"] == 0 else _spread(0, case["held"], n)
        return held, _spread(case["shortest"], case["longest"], n)
    lengths = _spread(case["shortest"], case["longest"], n)
    if case["few"] == case["shortest"] and case["many"] == case["longest"] and case["many"] > 1:
        new = lengths  # whole prompts
    else:
        # one sequence in eight brings many rows, the others few
        new = [min(l, case["many"] if i % 8 == 0 else case["few"]) for i, l in enumerate(lengths)]
    return [l - m for l, m in zip(lengths, new)], new


def _pages(tokens, page):
    return -(-tokens // page)


def work(case):
    held, new = _sizes(case)
    rows = sum(m for m in new if m > 0)
    if case["kind"] == "plan":
        page = case["page"]
        taken = sum(_pages(h + m, page) - _pages(h, page) for h, m in zip(held, new) if m > 0)
        given = sum(_pages(h, page) for h, m in zip(held, new) if m < 0)
        # per sequence: tokens asked, length read and written, row start; per page
        # moved: read and written; per row: position and slot
        return {"bytes": 16 * len(held) + 8 * (taken + given) + 8 * rows, "flops": 0}
    width = case["kv_heads"] * HEAD
    if case["kind"] == "append":
        touched = sum(_pages(h + m, case["page"]) - h // case["page"] for h, m in zip(held, new))
        return {"bytes": rows * (4 + 2 * 2 * width + 2 * width) + 8 * touched * case["kv_heads"], "flops": 0}
    window = case["window"]
    keys = pairs = 0
    for h, m in zip(held, new):
        reach = [min(p + 1, window) if window else p + 1 for p in range(h, h + m)]
        keys += min(h + m, window + m - 1) if window else h + m
        pairs += sum(reach)
    size = 2 * keys * width + 8 * case["kv_heads"] * keys // case["page"] + 4 * rows * case["heads"] * HEAD
    return {"bytes": size, "flops": 4 * HEAD * case["heads"] * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _tables(generator, pages_each, pool):
    """A block table of distinct pages in random order (-1 where a sequence has none) and the pages left over."""
    order = torch.randperm(pool, generator=generator, device=DEVICE).int()
    counts = _ints(pages_each).long()
    table = torch.full((len(pages_each), max(1, max(pages_each))), -1, dtype=torch.int32, device=DEVICE)
    places = torch.arange(table.shape[1], device=DEVICE)[None] < counts[:, None]
    used = int(counts.sum())
    table[places] = order[:used]
    return table, order[used:]


def prepare(case, seed):
    generator = torch.Generator(DEVICE).manual_seed(seed)
    held, new = _sizes(case)
    page = case["page"]
    s = {"case": case, "sequences": len(held), "page": page, "rows": sum(m for m in new if m > 0)}
    if case["kind"] == "plan":
        stride = _pages(case["longest"] + case["prompt"], page)
        wanted = sum(_pages(h + m, page) - _pages(h, page) for h, m in zip(held, new) if m > 0)
        # a pool that runs short lets only some of them in
        pool = sum(_pages(h, page) for h in held) + (wanted // 2 if case["scarce"] else wanted + 7)
        table, rest = _tables(generator, [_pages(h, page) for h in held], pool)
        s["tables"] = torch.full((len(held), stride), -1, dtype=torch.int32, device=DEVICE)
        s["tables"][:, :table.shape[1]] = table
        s["free_pages"] = torch.full((pool,), -1, dtype=torch.int32, device=DEVICE)
        s["free_pages"][:rest.numel()] = rest
        s["free_count"] = _ints([rest.numel()])
        s["lengths"], s["new_tokens"] = _ints(held), _ints(new)
        s["pool"] = pool
        s["capacity"] = s["rows"] + 5  # a step's buffers are a little larger than the step
        s["new_lengths"], s["new_free_count"] = torch.empty_like(s["lengths"]), torch.empty_like(s["free_count"])
        s["row_starts"] = torch.empty(len(held) + 1, dtype=torch.int32, device=DEVICE)
        s["row_positions"] = torch.empty(s["capacity"], dtype=torch.int32, device=DEVICE)
        s["row_slots"] = torch.empty(s["capacity"], dtype=torch.int32, device=DEVICE)
        s["refused"] = torch.empty(1, dtype=torch.int32, device=DEVICE)
        return s
    kv_heads = case["kv_heads"]
    lengths = [h + m for h, m in zip(held, new)]
    pages_each = [_pages(l, page) for l in lengths]
    pool = sum(pages_each) + 3
    s["pool"], s["tables"] = pool, _tables(generator, pages_each, pool)[0]
    s["lengths"], s["row_starts"] = _ints(lengths), _ints([0] + new).cumsum(0, dtype=torch.int32)
    s["max_rows"], s["max_length"] = max(new), max(lengths)
    for name in ("key", "value"):
        shape = (pool, kv_heads, page // GRANULE, 2048)
        # normal values: a page's largest of 2048 and more lies near 3.5 deviations
        if case["format"] == "int8":
            held_bytes = torch.empty(shape, dtype=torch.int8, device=DEVICE)
        else:
            held_bytes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=DEVICE)
        for at in range(0, pool, 4096):
            part = torch.randn((min(4096, pool - at),) + shape[1:], generator=generator, device=DEVICE)
            part = (part * 36).round_().clamp_(-127, 127) if case["format"] == "int8" else (part * 80).clamp_(-448, 448)
            held_bytes[at:at + 4096] = part.to(held_bytes.dtype)
        s[name + "_pages"] = held_bytes
        if case["format"] == "int8":
            spread = torch.rand((pool, kv_heads), generator=generator, device=DEVICE)
            s[name + "_scales"] = (0.02 + 0.02 * spread) * (1.0 if name == "key" else 0.7)
        else:
            spread = torch.randint(-8, -5, (pool, kv_heads), generator=generator, device=DEVICE)
            s[name + "_scales"] = torch.exp2(spread.float())
    if case["kind"] == "append":
        for name in ("key", "value"):
            rows = torch.randn((s["rows"], kv_heads * HEAD), generator=generator, device=DEVICE)
            # heads and rows of different size, so that pages' scales grow now and then
            rows *= 0.3 + torch.rand((s["rows"], 1), generator=generator, device=DEVICE) * 1.7
            s[name] = rows.bfloat16()
        # the slots that the plan gives
        row = torch.arange(s["rows"], device=DEVICE)
        starts = s["row_starts"].long()
        sequence = torch.searchsorted(starts[1:], row, right=True)
        position = s["lengths"].long()[sequence] - starts[sequence + 1] + row
        s["row_slots"] = (s["tables"].long()[sequence, position // page] * page + position % page).int()
        return s
    s["query"] = torch.randn((s["rows"], case["heads"] * HEAD), generator=generator, device=DEVICE).bfloat16()
    s["out"] = torch.empty_like(s["query"])
    # scratch as a server keeps it, once for all its layers
    s["workspace"] = torch.empty(64 << 20, dtype=torch.uint8, device=DEVICE)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention}[kind](state)
    return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention}[kind](state)


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _plan_outputs(s):
    return [s[k] for k in ("tables", "free_pages", "new_free_count", "new_lengths", "row_starts", "row_positions",
                           "row_slots", "refused")]


def _append_outputs(s):
    return [s[k] for k in ("key_pages", "value_pages", "key_scales", "value_scales")]


def _cache(hip, s):
    case = s["case"]
    return hip.Kv8Cache(case["format"], s["page"], s["pool"], case["kv_heads"], s["key_pages"], s["value_pages"],
                        s["key_scales"], s["value_scales"])


def _own_plan(s):
    _hip().kv8_plan(s["sequences"], s["page"], s["pool"], s["tables"], s["tables"].shape[1], s["new_tokens"],
                    s["lengths"], s["new_lengths"], s["free_pages"], s["free_count"], s["new_free_count"],
                    s["row_starts"], s["row_positions"], s["row_slots"], s["capacity"], s["refused"],
                    stream=_stream())
    return _plan_outputs(s)


def _own_append(s):
    hip = _hip()
    hip.kv8_append(_cache(hip, s), s["key"], s["value"], s["row_slots"], s["rows"], stream=_stream())
    return _append_outputs(s)


def _own_attention(s):
    hip = _hip()
    hip.kv8_attention(_cache(hip, s), s["query"], s["out"], s["case"]["heads"], s["rows"], s["sequences"],
                      s["tables"], s["tables"].shape[1], s["lengths"], s["row_starts"], scale=SCALE,
                      window=s["case"]["window"], max_rows=s["max_rows"], max_length=s["max_length"],
                      workspace=s["workspace"], workspace_bytes=s["workspace"].numel(), stream=_stream())
    return s["out"]


def _plain_plan(s):
    page, table = s["page"], s["tables"]
    stride, capacity = table.shape[1], s["capacity"]
    length, asked = s["lengths"].long(), s["new_tokens"].long()
    column = torch.arange(stride, device=DEVICE)[None]
    row = torch.arange(capacity, device=DEVICE)
    # sequences that end give their pages back, in order
    held = (length + page - 1) // page
    ends = asked < 0
    back = torch.where(ends, held, 0)
    top = s["free_count"].long() + back.cumsum(0) - back
    place = top[:, None] + column
    given = ends[:, None] & (column < held[:, None])
    s["free_pages"][place[given]] = table[given]
    stack = s["free_count"].long() + back.sum()
    # who is let in: the table has room, then the row buffers, then the stack
    new = asked.clamp(min=0)
    fits = ~ends & (length + new <= stride * page)
    fits &= (new == 0) | (torch.where(fits, new, 0).cumsum(0) <= capacity)
    need = torch.where(fits, (length + new + page - 1) // page - held, 0)
    before = need.cumsum(0) - need
    fits &= (need == 0) | (before + need <= stack)
    need, new = torch.where(fits, need, 0), torch.where(fits, new, 0)
    fresh = (column >= held[:, None]) & (column < (held + need)[:, None])
    take = stack - 1 - (before[:, None] + column - held[:, None])
    table[fresh] = s["free_pages"][take[fresh]]
    s["new_free_count"].copy_(stack - need.sum())
    s["new_lengths"].copy_(torch.where(ends, 0, length + new))
    s["refused"].copy_((~ends & ~fits).sum())
    last = new.cumsum(0)
    s["row_starts"][0] = 0
    s["row_starts"][1:] = last
    # the row map
    sequence = torch.searchsorted(last, row, right=True).clamp(max=s["sequences"] - 1)
    position = length[sequence] + row - (last - new)[sequence]
    inside = row < last[-1]
    position = torch.where(inside, position, 0)
    slot = table[sequence, position // page].long() * page + position % page
    s["row_positions"].copy_(position)
    s["row_slots"].copy_(torch.where(inside, slot, -1))
    return _plan_outputs(s)


def _tokens_of(pages, is_key):
    """[..., granules, 2048] values as [..., granules * 16, 128]."""
    lead = pages.shape[:-2]
    if is_key:
        v = pages.unflatten(-1, (2, GRANULE, 64)).transpose(-3, -2)  # granule, token, half, dimension
        return v.reshape(*lead, -1, HEAD)
    v = pages.unflatten(-1, (2, 4, 16, 4, 4))  # half, token / 4, d % 16, d / 16 % 4, token % 4
    n = v.dim()
    v = v.permute(*range(n - 5), n - 4, n - 1, n - 5, n - 2, n - 3)
    return v.reshape(*lead, -1, HEAD)


def _pages_of(tokens, is_key):
    """The inverse of _tokens_of."""
    lead = tokens.shape[:-2]
    if is_key:
        return tokens.reshape(*lead, -1, GRANULE, 2, 64).transpose(-3, -2).reshape(*lead, -1, 2048)
    v = tokens.reshape(*lead, -1, 4, 4, 2, 4, 16)  # token / 4, token % 4, half, d / 16 % 4, d % 16
    n = v.dim()
    v = v.permute(*range(n - 5), n - 3, n - 5, n - 1, n - 2, n - 4)
    return v.reshape(*lead, -1, 2048)


def _scale_for(largest, fmt):
    """The scale of a page whose largest magnitude is `largest`."""
    if fmt == "int8":
        return (largest.double() / 127).float()
    part, exponent = torch.frexp(largest)
    power = torch.where(part <= 0.875, exponent - 9, exponent - 8)  # 448 = 0.875 * 2^9
    return torch.where(largest > 0, torch.ldexp(torch.ones_like(largest), power), 0.0)


def _held(x, dtype):
    """Values in units of their scale, as the cache holds them."""
    return x.round().clamp(-127, 127).to(dtype) if dtype == torch.int8 else x.float().clamp(-448, 448).to(dtype)


def _plain_append(s):
    page, kv_heads, fmt = s["page"], s["case"]["kv_heads"], s["case"]["format"]
    slots = s["row_slots"].long()
    at, offset = slots // page, slots % page
    # where the step's run of each page begins
    first = torch.full((s["pool"],), page, dtype=torch.long, device=DEVICE)
    first.scatter_reduce_(0, at, offset, "amin")
    touched = torch.nonzero(first < page).squeeze(1)
    first = first[touched]
    earlier = torch.arange(page, device=DEVICE)[None] < first[:, None]
    for name in ("key", "value"):
        pages, scales = s[name + "_pages"], s[name + "_scales"]
        x = s[name].float().unflatten(-1, (kv_heads, HEAD))
        largest = torch.zeros((s["pool"], kv_heads), device=DEVICE)
        largest.scatter_reduce_(0, at[:, None].expand(-1, kv_heads), x.abs().amax(-1), "amax")
        wanted = _scale_for(largest[touched], fmt)
        old = torch.where(first[:, None] > 0, scales[touched], 0.0)
        scale = torch.maximum(wanted, old)
        scales[touched] = scale
        # the page's earlier tokens in the new scale, then the new tokens
        ratio = torch.where(scale > 0, old.double() / scale.double(), 1.0)
        tokens = _tokens_of(pages.view(torch.uint8)[touched], name == "key").contiguous().view(pages.dtype)
        moved = _held(tokens.double() * ratio[..., None, None], pages.dtype)
        keep = earlier[:, None, :, None]
        tokens = torch.where(keep, moved.view(torch.uint8), tokens.view(torch.uint8))
        row_scale = scales[at].double()
        inverse = torch.where(row_scale > 0, 1 / row_scale, 0.0)
        new = _held(x.double() * inverse[..., None], pages.dtype).view(torch.uint8)
        place = torch.zeros(s["pool"], dtype=torch.long, device=DEVICE)
        place[touched] = torch.arange(touched.numel(), device=DEVICE)
        tokens[place[at], :, offset] = new
        # tokens behind the run in its last granule read as zero when the granule is new
        end = torch.zeros(s["pool"], dtype=torch.long, device=DEVICE).scatter_reduce_(0, at, offset + 1, "amax")[touched]
        token = torch.arange(page, device=DEVICE)[None]
        filled = (token >= end[:, None]) & (token < (end[:, None] + GRANULE - 1) // GRANULE * GRANULE)
        filled &= token // GRANULE * GRANULE >= first[:, None]
        tokens = torch.where(filled[:, None, :, None], 0, tokens)
        written = (token // GRANULE * GRANULE < end[:, None])[:, None, :, None]
        tokens = torch.where(written, tokens, _tokens_of(pages.view(torch.uint8)[touched], name == "key"))
        pages.view(torch.uint8)[touched] = _pages_of(tokens, name == "key")
    return _append_outputs(s)


def _plain_attention(s):
    case, page = s["case"], s["page"]
    kv_heads, heads = case["kv_heads"], case["heads"]
    sequences, group = s["sequences"], heads // kv_heads
    length, starts = s["lengths"].long(), s["row_starts"].long()
    rows, keys = s["max_rows"], s["tables"].shape[1] * page
    step = starts[1:] - starts[:-1]
    # the step's rows, sequence by sequence
    place = torch.arange(rows, device=DEVICE)[None].expand(sequences, -1)
    mine = place < step[:, None]
    index = torch.where(mine, starts[:-1, None] + place, 0)
    position = length[:, None] - step[:, None] + place
    query = s["query"][index].float().unflatten(-1, (kv_heads, group, HEAD))  # sequence, row, kv head, group, d
    query = query.permute(0, 2, 3, 1, 4).reshape(sequences, kv_heads, group * rows, HEAD)

    def cached(name):
        pages = s[name + "_pages"].view(torch.uint8)[s["tables"].clamp(min=0)]  # sequence, page, kv head, granule, byte
        tokens = _tokens_of(pages.transpose(1, 2), name == "key")  # sequence, kv head, page, token, d
        values = tokens.contiguous().view(s[name + "_pages"].dtype).float()
        scale = s[name + "_scales"][s["tables"].clamp(min=0)].transpose(1, 2)
        return (values * scale[..., None, None]).reshape(sequences, kv_heads, keys, HEAD)

    key_place = torch.arange(keys, device=DEVICE)
    reach = (key_place <= position[..., None]) & mine[..., None]
    if case["window"]:
        reach &= key_place > position[..., None] - case["window"]
    reach = reach[:, None, None]  # sequence, 1, 1, row, key
    scores = (query @ cached("key").transpose(-1, -2)).unflatten(2, (group, rows)) * SCALE
    scores = scores.masked_fill(~reach, -math.inf)
    top = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weight = torch.exp(scores - top)
    del scores
    total = weight.sum(-1, keepdim=True)
    value = cached("value").masked_fill((key_place >= length[:, None])[:, None, :, None], 0.0)
    out = (weight.flatten(2, 3) @ value).unflatten(2, (group, rows))
    out = torch.where(total > 0, out / total, 0.0)
    out = out.permute(0, 3, 1, 2, 4).reshape(sequences, rows, heads * HEAD).to(s["out"].dtype)
    s["out"][index[mine]] = out[mine]
    return s["out"]


# ---------------------------------------------------------------------------
# The definition in 64 bits, sequence by sequence, by the layout's formula
# ---------------------------------------------------------------------------
def _offsets(is_key):
    t = torch.arange(GRANULE, device=DEVICE)[:, None]
    d = torch.arange(HEAD, device=DEVICE)[None]
    if is_key:
        return d // 64 * 1024 + t * 64 + d % 64
    return d // 64 * 1024 + t // 4 * 256 + d % 16 * 16 + d // 16 % 4 * 4 + t % 4


def _read(s, name, sequence, length):
    """One sequence's keys or values [kv head][token][d] in 64 bits."""
    page = s["page"]
    token = torch.arange(length, device=DEVICE)
    pages = s["tables"][sequence].long()[token // page]
    granule = token % page // GRANULE
    raw = s[name + "_pages"][pages, :, granule]  # token, kv head, byte
    places = _offsets(name == "key")[token % GRANULE]
    raw = raw.double().gather(2, places[:, None].expand(-1, raw.shape[1], -1))
    return (raw * s[name + "_scales"][pages].double()[..., None]).transpose(0, 1)


def _exact_attention(s):
    case = s["case"]
    group, out = case["heads"] // case["kv_heads"], torch.zeros(s["query"].shape, dtype=torch.float64, device=DEVICE)
    starts = s["row_starts"].tolist()
    for i, length in enumerate(s["lengths"].tolist()):
        begin, end = starts[i], starts[i + 1]
        if end == begin:
            continue
        key, value = _read(s, "key", i, length), _read(s, "value", i, length)
        position = length - (end - begin) + torch.arange(end - begin, device=DEVICE)[:, None]
        token = torch.arange(length, device=DEVICE)[None]
        hidden = token > position
        if case["window"]:
            hidden |= token <= position - case["window"]
        for h in range(case["heads"]):
            q = s["query"][begin:end, h * HEAD:(h + 1) * HEAD].double()
            scores = (q @ key[h // group].T) / math.sqrt(HEAD)
            out[begin:end, h * HEAD:(h + 1) * HEAD] = scores.masked_fill(hidden, -math.inf).softmax(-1) @ value[h // group]
    return out


def _exact_scales(s):
    """The pages' scales after the step; what they scale is whole numbers or 8-bit values, compared as they are."""
    page, kv_heads, fmt = s["page"], s["case"]["kv_heads"], s["case"]["format"]
    slots = s["row_slots"].long()
    outputs = [None, None]
    for name in ("key", "value"):
        scales = s[name + "_scales"].double()
        x = s[name].double().reshape(-1, kv_heads, HEAD).abs().amax(-1)
        fresh = torch.unique((slots // page)[slots % page == 0])
        scales[fresh] = 0
        wanted = x / 127 if fmt == "int8" else torch.exp2(torch.ceil(torch.log2(x / 448)))
        outputs.append(scales.index_reduce(0, slots // page, wanted, "amax"))
    return outputs


def exact(case, seed):
    if case["kind"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    return _exact_attention(s) if case["kind"] == "attention" else _exact_scales(s)

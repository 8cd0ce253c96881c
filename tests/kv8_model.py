"""Plain restatements, in 64 bits, of the paged 8-bit key/value cache's three
operators (include/qwen3_tts_native.h, Qwen3TtsKv8*): the page plan as a walk
over the sequences, the quantising append run by run, and attention row by
row.  Values are held token by token here; `pack` and `unpack` are the pages'
byte layout, written from its formula."""
import numpy as np

D = 128
GRANULE = 16
NAN_BYTE = {"int8": 0x80, "e4m3": 0x7F}  # bytes that the cache never holds


def _e4m3_values():
    code = np.arange(256)
    exponent, mantissa = (code >> 3) & 15, code & 7
    magnitude = np.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * 2.0 ** (exponent - 10.0))
    value = np.where(code & 0x80, -magnitude, magnitude)
    value[(code & 0x7F) == 0x7F] = np.nan
    return value


E4M3 = _e4m3_values()
_POSITIVE = E4M3[:127]  # rising


def decode(fmt, codes):
    codes = np.asarray(codes, np.uint8)
    return codes.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3[codes]


def encode(fmt, x):
    """Nearest held value, ties to even, to the format's range; x finite."""
    x = np.asarray(x, np.float64)
    if fmt == "int8":
        return np.clip(np.rint(x), -127, 127).astype(np.int8).view(np.uint8)
    a = np.minimum(np.abs(x), 448.0)
    above = np.minimum(np.searchsorted(_POSITIVE, a), 126)
    below = np.maximum(above - 1, 0)
    up, down = _POSITIVE[above] - a, a - _POSITIVE[below]
    code = np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (code | np.where(np.signbit(x), 0x80, 0)).astype(np.uint8)


def scale_for(fmt, largest):
    largest = np.float64(largest)
    if largest == 0:
        return np.float32(0)
    if fmt == "int8":
        return np.float32(largest / 127)
    power = np.ceil(np.log2(largest / 448)) if largest else 0
    while 448 * 2.0 ** (power - 1) >= largest:
        power -= 1
    while 448 * 2.0 ** power < largest:
        power += 1
    return np.float32(2.0 ** power)


# ---------------------------------------------------------------------------
# Layout: codes [pages][heads][tokens][128] <-> bytes [pages][heads][granules][2048]
# ---------------------------------------------------------------------------
def _offsets(is_key):
    t, d = np.arange(GRANULE)[:, None], np.arange(D)[None]
    if is_key:
        return d // 64 * 1024 + t * 64 + d % 64
    return d // 64 * 1024 + t // 4 * 256 + d % 16 * 16 + d // 16 % 4 * 4 + t % 4


def pack(codes, is_key):
    pages, heads, tokens, _ = codes.shape
    out = np.empty((pages, heads, tokens // GRANULE, 2048), np.uint8)
    out[..., _offsets(is_key)] = codes.reshape(pages, heads, -1, GRANULE, D)
    return out


def unpack(raw, is_key):
    pages, heads, granules, _ = raw.shape
    return raw[..., _offsets(is_key)].reshape(pages, heads, granules * GRANULE, D)


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------
def plan(page, pages, tables, new_tokens, lengths, free_pages, free_count, capacity):
    """The step's arrays, from copies of the inputs."""
    tables, free = tables.copy(), list(free_pages[:free_count])
    stack = free_pages.copy()
    stride = tables.shape[1]
    count = lambda tokens: -(-tokens // page)  # noqa: E731
    for s, n in enumerate(new_tokens):
        if n < 0:
            free += list(tables[s, :count(lengths[s])])
    stack[:len(free)] = free
    rows_asked = pages_asked = taken = refused = 0
    new_lengths, starts, positions, slots = [], [0], [], []
    for s, (n, length) in enumerate(zip(new_tokens, lengths)):
        n, length = int(n), int(length)
        if n < 0:
            new_lengths.append(0)
            starts.append(len(positions))
            continue
        fits = length + n <= stride * page
        if fits:
            rows_asked += n
            fits = n == 0 or rows_asked <= capacity
        need = 0
        if fits:
            need = count(length + n) - count(length)
            pages_asked += need
            fits = need == 0 or pages_asked <= len(free)
        if not fits:
            refused += 1
            n = 0
        else:
            for j in range(need):
                tables[s, count(length) + j] = free[len(free) - 1 - (pages_asked - need + j)]
            taken += need
        for i in range(n):
            p = length + i
            positions.append(p)
            at = tables[s, p // page]
            slots.append(at * page + p % page if 0 <= at < pages else -1)
        new_lengths.append(length + n)
        starts.append(len(positions))
    pad = capacity - len(positions)
    as_int = lambda v: np.array(v, np.int32)  # noqa: E731
    return {"tables": tables, "free_pages": stack, "new_free_count": as_int([len(free) - taken]),
            "new_lengths": as_int(new_lengths), "row_starts": as_int(starts),
            "row_positions": as_int(positions + [0] * pad), "row_slots": as_int(slots + [-1] * pad),
            "refused": as_int([refused])}


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
def append(fmt, page, codes, scales, rows, slots):
    """Stores rows [rows][heads][128] (float32 values of bf16) in codes [pages][heads][page][128] and scales in
    place; returns a mask of the tokens whose bytes are defined afterwards among those touched."""
    pages, heads = scales.shape
    usable = np.array([s if 0 <= s < pages * page else -1 for s in slots])
    r = 0
    while r < len(usable):
        if usable[r] < 0:
            r += 1
            continue
        n = 1
        while r + n < len(usable) and usable[r + n] == usable[r] + n and usable[r + n] % page != 0:
            n += 1
        at, offset = divmod(int(usable[r]), page)
        x = rows[r:r + n].astype(np.float64)  # n, heads, d
        for h in range(heads):
            magnitude = np.abs(x[:, h])
            finite = magnitude[np.isfinite(magnitude)]
            wanted = scale_for(fmt, finite.max() if finite.size else 0.0)
            old = scales[at, h] if offset else np.float32(0)
            scale = max(wanted, old)
            if offset and scale != old:
                ratio = np.float64(old) / np.float64(scale)
                codes[at, h, :offset] = encode(fmt, decode(fmt, codes[at, h, :offset]) * ratio)
            with np.errstate(invalid="ignore"):
                inverse = 1 / np.float64(scale) if scale > 0 else 0.0
                q = x[:, h] * inverse
            q = np.where(np.isnan(q), 0.0, q)
            codes[at, h, offset:offset + n] = encode(fmt, np.clip(q, -1e6, 1e6))
            scales[at, h] = scale
        r += n


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attention(fmt, page, key_codes, value_codes, key_scales, value_scales, query, tables, lengths, row_starts, heads,
              scale, window, weight_error):
    """(out, tolerance) [rows][heads][128] in 64 bits, NaN where no sequence has the row.  `weight_error` is the
    relative rounding of a weight before its product with the value.

    The tolerance of one output: half a bf16 step of it, 2^-8, and with A the weighted mean of |v| the error of
    the weights, A * (weight_error + 2 * e): e bounds a score's error, 128 products and sums in fp32 (130 * 2^-24
    of the magnitudes' sum), the scales and the exponential's argument (6 * 2^-24 of the largest score) and
    the exponential itself, once in the weights and once in their sum; the sums over the tokens and the divisions
    are within (tokens / 4 + 64) * 2^-24, four lanes adding apart.  Where fp32 ends: a weight below 2^-126 may become
    0 (the sum of weights is at least 1), and so may its product with the value's scale, in front of the held value:
    2^-126 of |v| and of |held| a token."""
    rows, group = query.shape[0], heads // key_scales.shape[1]
    out = np.full((rows, heads, D), np.nan)
    tolerance = np.full((rows, heads, D), np.nan)
    q = query.reshape(rows, heads, D).astype(np.float64)
    for s, length in enumerate(lengths):
        begin, end = int(row_starts[s]), min(int(row_starts[s + 1]), rows)
        if end <= begin:
            continue
        token = np.arange(length)
        at = tables[s, token // page] if length else np.zeros(0, int)
        known = (at >= 0) & (at < key_scales.shape[0])
        at = np.where(known, at, 0)
        for kv in range(key_scales.shape[1]):
            def values(codes, scales):
                v = decode(fmt, codes[at, kv, token % page]) * scales[at, kv].astype(np.float64)[:, None]
                return np.where(known[:, None], v, 0.0)
            k, v = values(key_codes, key_scales), values(value_codes, value_scales)
            held = np.where(known[:, None], decode(fmt, value_codes[at, kv, token % page]), 0.0)
            for r in range(begin, end):
                position = length - (int(row_starts[s + 1]) - begin) + r - begin
                seen = known & (token <= position)
                if window:
                    seen &= token > position - window
                for h in range(kv * group, (kv + 1) * group):
                    if not seen.any():
                        out[r, h], tolerance[r, h] = 0.0, 0.0
                        continue
                    score = k[seen] @ q[r, h] * scale
                    w = np.exp(score - score.max())
                    w /= w.sum()
                    out[r, h] = w @ v[seen]
                    mean = w @ np.abs(v[seen])
                    e = 2.0 ** -24 * (130 * (np.abs(k[seen]) @ np.abs(q[r, h])).max() * abs(scale)
                                      + 6 * np.abs(score).max() + 4)
                    sums = 2.0 ** -24 * (seen.sum() / 4 + 64)
                    tolerance[r, h] = 2.0 ** -8 * np.abs(out[r, h]) + mean * (weight_error + 2 * e + sums) * (1 + 2.0 ** -8)
                    tolerance[r, h] += 2.0 ** -126 * (np.abs(v[seen]) + np.abs(held[seen])).sum(0)
    return out, tolerance

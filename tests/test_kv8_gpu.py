"""GPU checks of the paged 8-bit key/value cache (qwen3_tts_op_kv8_*) against
its 64-bit restatement (tests/kv8_model.py): the page plan's arrays and the
append's bytes and scales exactly, attention within bounds that follow from
its roundings (kv8_model.attention), the three together over many steps, and
captured into a HIP graph."""
import ctypes as C

import numpy as np
import pytest

import gen
import kv8_model as model
from test_zz_no_alloc import Runtime

pytestmark = pytest.mark.gpu

D = 128
# a weight's rounding in front of the value product: two bf16 that leave 2^-16
# of it where few rows share the products, one bf16 where many do
FEW_ROWS, MANY_ROWS = 2.0 ** -16, 2.0 ** -8


def dev(hip, a):
    return hip.DeviceArray.from_numpy(a)


# ---------------------------------------------------------------------------
# Plan
# ---------------------------------------------------------------------------
PLAN_NAMES = ("tables", "free_pages", "new_free_count", "new_lengths", "row_starts", "row_positions", "row_slots",
              "refused")


class Plan:
    """Device buffers of a plan; run() makes one call and compares every array with the model's."""

    def __init__(self, hip, page, pages, tables, lengths, free_pages, free_count, capacity, in_place=False):
        self.hip, self.page, self.pages, self.capacity = hip, page, pages, capacity
        self.sequences, self.stride = tables.shape
        self.tables, self.free_pages = dev(hip, tables.astype(np.int32)), dev(hip, free_pages.astype(np.int32))
        self.lengths, self.free_count = dev(hip, np.array(lengths, np.int32)), dev(hip, np.array([free_count], np.int32))
        new = lambda n: dev(hip, np.full(n, -77, np.int32))  # noqa: E731
        self.new_lengths = self.lengths if in_place else new(self.sequences)
        self.new_free_count = self.free_count if in_place else new(1)
        self.row_starts, self.refused = new(self.sequences + 1), new(1)
        self.row_positions, self.row_slots = new(max(capacity, 1)), new(max(capacity, 1))
        self.new_tokens = new(self.sequences)

    def launch(self, stream=None):
        self.hip.kv8_plan(self.sequences, self.page, self.pages, self.tables, self.stride, self.new_tokens,
                          self.lengths, self.new_lengths, self.free_pages, self.free_count, self.new_free_count,
                          self.row_starts, self.row_positions, self.row_slots, self.capacity, self.refused,
                          stream=stream)

    def expected(self, new_tokens):
        return model.plan(self.page, self.pages, self.tables.numpy(), new_tokens, self.lengths.numpy(),
                          self.free_pages.numpy(), int(self.free_count.numpy()[0]), self.capacity)

    def run(self, new_tokens, stream=None):
        want = self.expected(new_tokens)
        self.new_tokens.upload(np.array(new_tokens, np.int32))
        self.launch(stream)
        self.hip.synchronize()
        self.check(want)
        return want

    def check(self, want):
        for name in PLAN_NAMES:
            got = getattr(self, name).numpy()
            if name in ("row_positions", "row_slots"):
                got = got[:self.capacity]
            assert np.array_equal(got, want[name]), name


def batch(rng, page, sequences, longest, spare):
    """Lengths, tables of distinct pages in random order, and the stack of the pages left over."""
    lengths = rng.integers(0, longest + 1, sequences)
    count = -(-lengths // page)
    pages = int(count.sum()) + spare
    order = rng.permutation(pages)
    tables = np.full((sequences, -(-2 * longest // page) + 1), -1, np.int32)
    at = 0
    for s, n in enumerate(count):
        tables[s, :n] = order[at:at + n]
        at += n
    stack = np.full(pages, -1, np.int32)
    stack[:spare] = order[at:]
    return lengths, tables, stack, pages


@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("sequences,longest,prompt", [(1, 1, 1), (1, 500, 700), (8, 100, 3), (64, 40, 60), (65, 90, 5),
                                                     (257, 70, 40), (1025, 33, 20), (2300, 5, 2)])
def test_plan(hip, page, sequences, longest, prompt):
    rng = np.random.default_rng(page * 10007 + sequences * 31 + longest)
    lengths, tables, stack, pages = batch(rng, page, sequences, longest, spare := sequences + 20)
    new = rng.integers(0, prompt + 1, sequences)
    new[rng.random(sequences) < 0.15] = -1
    p = Plan(hip, page, pages, tables, lengths, stack, spare, int(np.maximum(new, 0).sum()) + 3)
    p.run(new)


@pytest.mark.parametrize("sequences", [5, 300, 1500])
@pytest.mark.parametrize("spare,share", [(0, 1.0), (7, 1.0), (50, 0.4), (10000, 0.6)])
def test_plan_refuses_what_does_not_fit(hip, sequences, spare, share):
    """Too few pages, too few row buffers and full tables, in all mixtures; refused sequences stay as they were."""
    rng = np.random.default_rng(sequences + spare)
    lengths, tables, stack, pages = batch(rng, 16, sequences, 60, spare)
    new = rng.integers(0, 45, sequences)
    new[rng.random(sequences) < 0.1] = -3
    new[rng.random(sequences) < 0.1] = 5000  # more than a table holds
    new[rng.random(sequences) < 0.1] = 0
    capacity = int(np.minimum(np.maximum(new, 0), 45).sum() * share)
    want = Plan(hip, 16, pages, tables, lengths, stack, spare, capacity).run(new)
    assert want["refused"][0] > 0


def test_plan_steps_in_place(hip):
    """Forty steps of one batch, lengths and stack updated in place: prompts come, grow and end, pages come round."""
    rng = np.random.default_rng(5)
    sequences, pages = 24, 90
    p = Plan(hip, 16, pages, np.full((sequences, 12), -1, np.int32), np.zeros(sequences, int),
             rng.permutation(pages), pages, 200, in_place=True)
    for _ in range(40):
        lengths = p.lengths.numpy()
        new = np.where(lengths > 0, 1, np.where(rng.random(sequences) < 0.3, rng.integers(1, 100, sequences), 0))
        new[(lengths > 0) & (rng.random(sequences) < 0.1)] = -1
        want = p.run(new)
        held = -(-want["new_lengths"] // 16)
        in_use = np.concatenate([want["tables"][s, :n] for s, n in enumerate(held)])
        free = want["free_pages"][:want["new_free_count"][0]]
        # every page is in one table or on the stack, once
        assert np.array_equal(np.sort(np.concatenate([in_use, free])), np.arange(pages))


def test_plan_without_row_buffers(hip):
    p = Plan(hip, 16, 4, np.full((2, 2), -1, np.int32), [0, 0], np.arange(4), 4, 0)
    p.run([0, 3])


def test_plan_of_odd_state(hip):
    """A stack count beyond the pool, a negative length and a table entry that is no page: clamped, slot -1."""
    tables = np.array([[9, -1, 2], [1, 7, 3], [-5, 0, 2]], np.int32)
    p = Plan(hip, 16, 4, tables, [3, -4, 20], np.array([0, 1, 2, 3]), 4, 9)
    p.free_count.upload(np.array([99], np.int32))
    p.new_tokens.upload(np.array([2, 1, 1], np.int32))
    p.launch()
    hip.synchronize()
    assert p.row_starts.numpy().tolist() == [0, 2, 3, 4]
    # sequence 0's page 9 does not exist; sequence 1 holds nothing and gets page 3; sequence 2's page 0 does
    assert p.row_slots.numpy()[:5].tolist() == [-1, -1, 3 * 16, 4, -1]
    assert p.new_lengths.numpy().tolist() == [5, 1, 21] and p.new_free_count.numpy()[0] == 3


# ---------------------------------------------------------------------------
# Append
# ---------------------------------------------------------------------------
class Store:
    """A cache on the device beside its model's codes and scales."""

    def __init__(self, hip, fmt, page, pages, heads, rng=None):
        self.hip, self.fmt, self.page, self.pages, self.heads = hip, fmt, page, pages, heads
        self.codes, self.scales, self.raw, self.device_scales = [], [], [], []
        for is_key in (True, False):
            if rng is None:  # a pool as it is after long use: stale bytes, stale scales
                codes = np.full((pages, heads, page, D), model.NAN_BYTE[fmt], np.uint8)
                scales = np.full((pages, heads), np.nan, np.float32)
            else:
                codes = model.encode(fmt, rng.standard_normal((pages, heads, page, D)) * (40 if fmt == "int8" else 90))
                scales = rng.uniform(0.01, 0.05, (pages, heads)).astype(np.float32)
            self.codes.append(codes)
            self.scales.append(scales)
            self.raw.append(dev(hip, model.pack(codes, is_key)))
            self.device_scales.append(dev(hip, scales))
        self.cache = hip.Kv8Cache(fmt, page, pages, heads, *self.raw, *self.device_scales)

    def append(self, key, value, slots):
        """The model's side of an append."""
        for i, rows in enumerate((key, value)):
            model.append(self.fmt, self.page, self.codes[i], self.scales[i],
                         gen.f32(rows).reshape(len(slots), self.heads, D), slots)

    def check(self, lengths_of_pages):
        """Bytes of the first lengths_of_pages[page] tokens, and the scales of pages that hold any."""
        for i, is_key in enumerate((True, False)):
            got = model.unpack(self.raw[i].numpy(), is_key)
            scales = self.device_scales[i].numpy()
            for at, n in enumerate(lengths_of_pages):
                if n:
                    assert np.array_equal(scales[at], self.scales[i][at]), (at, is_key)
                same = model.decode(self.fmt, got[at, :, :n]) == model.decode(self.fmt, self.codes[i][at, :, :n])
                assert same.all(), (at, is_key, np.argwhere(~same)[:4])


def kv_rows(rng, rows, heads, spread=True):
    x = rng.standard_normal((rows, heads * D)).astype(np.float32)
    if spread:  # rows of very different size: scales grow within a page
        x *= np.exp2(rng.uniform(-6, 4, (rows, 1))).astype(np.float32)
    return gen.bf16(x)


def fill_of(slots, page, pages, start=None):
    held = np.zeros(pages, int) if start is None else start.copy()
    for s in slots:
        if 0 <= s < page * pages:
            held[s // page] = s % page + 1
    return held


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads", [1, 3, 8])
def test_append_in_pieces(hip, fmt, page, heads):
    """One page's worth and more of tokens in pieces of every kind: alone, across granules, across pages, with the
    scale growing and not."""
    rng = np.random.default_rng(page + heads)
    store = Store(hip, fmt, page, 9, heads)
    table = rng.permutation(9)
    position = 0
    held = np.zeros(9, int)
    for n in (1, 1, 2, 13, 1, 5, 16, 31, 1, 70):
        p = np.arange(position, position + n)
        slots = (table[p // page] * page + p % page).astype(np.int32)
        position += n
        key, value = kv_rows(rng, n, heads), kv_rows(rng, n, heads)
        hip.kv8_append(store.cache, dev(hip, key), dev(hip, value), dev(hip, slots), n)
        hip.synchronize()
        store.append(key, value, slots)
        held = fill_of(slots, page, 9, held)
        store.check(held)
    assert position == 141


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page,rows,heads", [(16, 700, 8), (32, 1111, 5), (64, 900, 8), (16, 2900, 8), (64, 2500, 8)])
def test_append_many_rows(hip, fmt, page, rows, heads):
    """Many sequences' rows at once, runs that begin anywhere, rows left out between them."""
    rng = np.random.default_rng(rows)
    pages = rows // 2
    order, slots, at = list(rng.permutation(pages)), [], 0
    while len(slots) < rows:
        first = int(rng.integers(0, page)) if rng.random() < 0.5 else 0
        n = int(rng.integers(1, page - first + 1))
        slots += list(order[at] * page + first + np.arange(n))
        at += 1
        if rng.random() < 0.2:
            slots += [-1] if rng.random() < 0.5 else [pages * page, -9]
    slots = np.array(slots[:rows], np.int32)
    store = Store(hip, fmt, page, pages, heads, rng)
    key, value = kv_rows(rng, rows, heads), kv_rows(rng, rows, heads)
    before = [r.numpy() for r in store.raw]
    hip.kv8_append(store.cache, dev(hip, key), dev(hip, value), dev(hip, slots), rows)
    hip.synchronize()
    store.append(key, value, slots)
    held = fill_of(slots, page, pages)
    store.check(held)
    for raw, old in zip(store.raw, before):  # pages that no row meets
        assert np.array_equal(raw.numpy()[held == 0], old[held == 0])


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_append_of_odd_values(hip, fmt):
    """Zeros, infinities, NaN, subnormals and the largest magnitudes, in a page's first run and behind it."""
    rows = np.zeros((8, 2 * D), np.float32)
    rows[1, :] = np.linspace(-3, 3, 2 * D)
    rows[2, 5], rows[2, 9], rows[2, 130] = np.inf, -np.inf, np.nan
    rows[2, 6] = 2.5
    rows[4, :] = 1e-40
    rows[5, 0], rows[5, 200] = 3e38, -3.3e38
    rows[6, 3], rows[6, 131] = np.nan, np.inf  # nothing finite but zeros
    rows[7, :] = 1e-39
    bits = gen.bf16(rows)
    bits[np.isnan(rows)] = 0x7FC0
    for runs in ([[0], [1, 2], [3], [4], [5]], [[6], [7]], [[4, 7]], [[0, 3]], [[2]], [[5], [1]]):
        store = Store(hip, fmt, 16, 2, 2)
        position = 0
        for run in runs:
            x = np.ascontiguousarray(bits[run])
            slots = (16 + position + np.arange(len(run))).astype(np.int32)
            position += len(run)
            hip.kv8_append(store.cache, dev(hip, x), dev(hip, x), dev(hip, slots), len(run))
            hip.synchronize()
            store.append(x, x, slots)
            store.check([0, position])
            # what a granule holds is never a NaN
            for i, is_key in enumerate((True, False)):
                assert np.isfinite(model.decode(fmt, model.unpack(store.raw[i].numpy(), is_key)[1])).all()


def test_append_strided_rows(hip):
    """Keys and values as parts of fused q|k|v rows."""
    rng = np.random.default_rng(3)
    heads, rows, stride = 2, 5, 16 * D
    qkv = kv_rows(rng, rows, 16)
    store = Store(hip, "int8", 16, 2, heads)
    slots = np.arange(14, 19, dtype=np.int32)
    d = dev(hip, qkv)
    hip.kv8_append(store.cache, d.offset(4 * D), d.offset(8 * D), dev(hip, slots), rows, key_stride=stride,
                   value_stride=stride)
    hip.synchronize()
    store.scales = [np.where(np.arange(2)[:, None] == 0, np.float32(0), s) for s in store.scales]
    key, value = np.ascontiguousarray(qkv[:, 4 * D:6 * D]), np.ascontiguousarray(qkv[:, 8 * D:10 * D])
    # page 0's run begins at token 14 of a pool whose stale scale is no number: the new tokens' scale counts
    store.append(key, value, slots)
    for i, is_key in enumerate((True, False)):
        got = model.unpack(store.raw[i].numpy(), is_key)
        assert np.array_equal(got[0, :, 14:], store.codes[i][0, :, 14:])
        assert np.array_equal(got[1, :, :3], store.codes[i][1, :, :3])
        assert np.array_equal(store.device_scales[i].numpy(), store.scales[i])


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------
def attend(hip, store, lengths, new, heads, *, window=0, scale=D ** -0.5, seed=0, workspace=0, max_rows=None,
           max_length=None, spoil=None, tail_rows=3, query_pad=0, out_pad=0, sharp=1.0, few=None):
    """One attention over `lengths` tokens and `new` rows a sequence; compares all rows, and those behind the last.
    `few` says which products compute them, where a name of more rows than there are makes that other than it seems."""
    rng = np.random.default_rng(seed)
    page, sequences = store.page, len(lengths)
    count = [-(-l // page) for l in lengths]
    assert sum(count) <= store.pages
    order = rng.permutation(store.pages)
    tables = np.full((sequences, max(1, max(count))), -1, np.int32)
    at = 0
    for s, n in enumerate(count):
        tables[s, :n] = order[at:at + n]
        at += n
    # bytes that nothing may read: behind each length, and pages of no table
    for i, is_key in enumerate((True, False)):
        codes, scales = store.codes[i].copy(), store.scales[i].copy()
        for s, l in enumerate(lengths):
            if l % page:
                codes[tables[s, l // page], :, l % page:] = model.NAN_BYTE[store.fmt]
        unused = np.setdiff1d(np.arange(store.pages), order[:at])
        if spoil is None:
            codes[unused], scales[unused] = model.NAN_BYTE[store.fmt], np.nan
        store.raw[i].upload(model.pack(codes, is_key))
        store.device_scales[i].upload(scales)
    if spoil is not None:
        spoil(tables)
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    rows = int(starts[-1]) + tail_rows
    width = heads * D
    q = gen.bf16((rng.standard_normal((rows, width + query_pad)) * sharp).astype(np.float32))
    out = hip.DeviceArray((rows, width + out_pad), np.uint16)
    out.upload(np.full((rows, width + out_pad), 0x1234, np.uint16))
    scratch = hip.DeviceArray(max(workspace, 16), np.uint8)
    keep = [dev(hip, q), dev(hip, tables), dev(hip, np.array(lengths, np.int32)), dev(hip, starts)]
    hip.kv8_attention(store.cache, keep[0], out, heads, rows, sequences, keep[1], tables.shape[1], keep[2], keep[3],
                      scale=scale, window=window, max_rows=max_rows or max(max(new), 1),
                      max_length=max_length or max(max(lengths), 1), query_stride=width + query_pad,
                      out_stride=width + out_pad, workspace=scratch if workspace else None, workspace_bytes=workspace)
    hip.synchronize()
    got = out.numpy()
    group = heads // store.heads
    few = max(new) * group <= 16 if few is None else few
    want, tolerance = model.attention(store.fmt, page, *store.codes, *store.scales, gen.f32(q[:, :width]), tables,
                                      lengths, starts, heads, scale, window, FEW_ROWS if few else MANY_ROWS)
    live = int(starts[-1])
    assert np.all(got[live:] == 0x1234) and np.all(got[:, width:] == 0x1234)
    got = gen.f32(got[:live, :width]).reshape(live, heads, D).astype(np.float64)
    off = np.abs(got - want[:live])
    assert np.all(off <= tolerance[:live]), (np.argwhere(~(off <= tolerance[:live]))[:5],
                                             np.nanmax(off / np.maximum(tolerance[:live], 1e-30)))
    return got


HEADS = [(16, 8), (4, 4), (14, 2), (16, 1)]


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv_heads", HEADS)
def test_attention_single_tokens(hip, fmt, page, heads, kv_heads):
    rng = np.random.default_rng(heads * page)
    lengths = [1, 2, 15, 16, 17, 63, 64, 65, 129, 333, 0, 700]
    new = [1] * 10 + [0, 1]
    store = Store(hip, fmt, page, sum(-(-l // page) for l in lengths) + 2, kv_heads, rng)
    attend(hip, store, lengths, new, heads)


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (7, 1), (16, 1)])
@pytest.mark.parametrize("max_length", [100, 300, 4096])
def test_attention_prompts(hip, fmt, page, heads, kv_heads, max_length):
    """Whole prompts, chunks behind a context, single tokens and idle sequences together; the length that the caller
    names has the work dealt out in three ways."""
    rng = np.random.default_rng(heads * page + 1)
    lengths = [1, 40, 130, 300, 77, 0, 65, 200]
    new = [1, 40, 130, 33, 1, 0, 2, 17]
    store = Store(hip, fmt, page, sum(-(-l // page) for l in lengths) + 2, kv_heads, rng)
    attend(hip, store, lengths, new, heads, max_length=max_length)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("many", [False, True])
def test_attention_window(hip, window, many):
    rng = np.random.default_rng(window)
    lengths = [1, 64, 65, 300, 129]
    new = [1, 60, 65, 70, 1] if many else [1, 1, 3, 2, 1]
    store = Store(hip, "int8" if window % 2 else "e4m3", 32, 25, 2, rng)
    attend(hip, store, lengths, new, 4, window=window)


@pytest.mark.parametrize("fmt,page", [("e4m3", 16), ("int8", 16), ("e4m3", 64)])
@pytest.mark.parametrize("new", [[1, 1, 1], [1, 90, 60]])
def test_attention_window_over_stale_pages(hip, fmt, page, new):
    """Pages in front of every row's window were given away: their bytes and scales are no numbers, or their entries
    no pages."""
    rng = np.random.default_rng(page + 60)
    window, lengths = 45, [300, 299, 170]
    store = Store(hip, fmt, page, 60, 2, rng)

    def spoil(tables):
        stale = []
        for s, (length, n) in enumerate(zip(lengths, new)):
            low = max(length - n - window + 1, 0)
            for at in range(low // page):
                stale.append(int(tables[s, at]))
                if at % 3 == 0:
                    tables[s, at] = -7
        assert stale
        for i, is_key in enumerate((True, False)):
            raw, scales = store.raw[i].numpy(), store.device_scales[i].numpy()
            raw[stale], scales[stale] = model.NAN_BYTE[fmt], np.nan
            store.raw[i].upload(raw)
            store.device_scales[i].upload(scales)

    attend(hip, store, lengths, new, 4, window=window, spoil=spoil)


@pytest.mark.parametrize("fmt,page", [("int8", 16), ("e4m3", 32), ("int8", 64)])
def test_attention_many_short_sequences(hip, fmt, page):
    """A wave a workgroup: many sequences of contexts up to 110 tokens."""
    rng = np.random.default_rng(page + 50)
    lengths = [int(l) for l in rng.integers(0, 111, 140)]
    new = [int(l > 0 and rng.random() < 0.9) for l in lengths]
    store = Store(hip, fmt, page, sum(-(-l // page) for l in lengths) + 2, 8, rng)
    attend(hip, store, lengths, new, 16)


def test_attention_shared_prefix(hip):
    """Two sequences whose tables name the same pages."""
    rng = np.random.default_rng(51)
    store = Store(hip, "int8", 16, 26, 2, rng)

    def spoil(tables):
        tables[1, :10] = tables[0, :10]

    for new in ([1, 1], [70, 90]):
        attend(hip, store, [200, 175], new, 4, spoil=spoil)


@pytest.mark.parametrize("workspace", [0, 1 << 12, 1 << 16, 1 << 24])
@pytest.mark.parametrize("new", [[1, 1, 0], [2, 60, 1]])
def test_attention_long_context(hip, workspace, new):
    """Contexts that are shared among workgroups where the workspace allows it."""
    rng = np.random.default_rng(8)
    store = Store(hip, "e4m3", 16, 420, 1, rng)
    attend(hip, store, [5000, 900, 64], new, 2, workspace=workspace)


def test_attention_hints_only_choose_the_work(hip):
    """max_rows and max_length below the truth: the results stand."""
    rng = np.random.default_rng(9)
    store = Store(hip, "int8", 16, 120, 2, rng)
    for new in ([1, 1], [300, 20], [5, 130]):
        attend(hip, store, [1000, 400], new, 4, max_rows=1, max_length=1, workspace=1 << 20)
        attend(hip, store, [1000, 400], new, 4, max_rows=4096, max_length=1 << 20, workspace=1 << 20)


def test_attention_strides_and_scale(hip):
    rng = np.random.default_rng(10)
    store = Store(hip, "int8", 16, 60, 2, rng)
    for new in ([1, 1], [90, 3]):
        attend(hip, store, [400, 99], new, 4, query_pad=8 * D, out_pad=4, scale=-0.3)
        attend(hip, store, [400, 99], new, 4, scale=0.0, tail_rows=0)


def test_attention_sharp_rows(hip):
    """Scores far apart: nearly all weight on one token, maxima that keep growing along the context."""
    rng = np.random.default_rng(11)
    store = Store(hip, "int8", 16, 60, 2, rng)
    for new in ([1, 1], [90, 120]):
        attend(hip, store, [400, 120], new, 4, sharp=60.0)


def test_attention_values_of_unequal_pages(hip):
    """Scales of zero, tiny and huge ones beside ordinary ones."""
    rng = np.random.default_rng(12)
    for new in ([1, 1], [90, 120]):
        store = Store(hip, "int8", 16, 60, 2, rng)
        for i in (0, 1):
            for factor in (0.0, 1e-12, 30.0 if i == 0 else 1e9):
                store.scales[i][rng.random((60, 2)) < 0.15] *= np.float32(factor)
            store.codes[i][store.scales[i] == 0] = 0
        attend(hip, store, [400, 120], new, 4)


@pytest.mark.parametrize("new", [[2, 1, 1], [100, 40, 70]])
def test_attention_tables_without_pages(hip, new):
    """Entries that are no page count as nothing; a row that has nothing else becomes 0."""
    rng = np.random.default_rng(13)
    store = Store(hip, "e4m3", 32, 30, 2, rng)

    def spoil(tables):
        tables[0, 1], tables[0, 3] = -1, 30
        tables[1, :] = 1 << 30
        tables[2, 0] = -1

    got = attend(hip, store, [200, 64, 70], new, 4, spoil=spoil)
    assert np.all(got[new[0]:new[0] + new[1]] == 0)


def test_attention_in_place(hip):
    """out may be the query buffer."""
    rng = np.random.default_rng(14)
    store = Store(hip, "int8", 16, 40, 2, rng)
    tables, lengths = np.arange(40, dtype=np.int32).reshape(1, 40), np.array([600], np.int32)
    for rows in (1, 600):
        starts = np.array([0, rows], np.int32)
        q = gen.bf16(rng.standard_normal((rows, 4 * D)).astype(np.float32))
        keep = [dev(hip, tables), dev(hip, lengths), dev(hip, starts)]
        outs = []
        for same in (False, True):
            query = dev(hip, q)
            out = query if same else hip.DeviceArray(q.shape, np.uint16)
            scratch = hip.DeviceArray(1 << 22, np.uint8)
            hip.kv8_attention(store.cache, query, out, 4, rows, 1, keep[0], 40, keep[1], keep[2], max_rows=rows,
                              max_length=600, workspace=scratch, workspace_bytes=1 << 22)
            hip.synchronize()
            outs.append(out.numpy())
        assert np.array_equal(outs[0], outs[1])


# Few rows are dealt out in tiles of 16 pairs, many in blocks of 128 columns whose waves share the columns (wide), or
# the columns and the tokens (halved, quartered).  The rows that the buffers hold, used or not, and the sizes that the
# caller names choose among them: buffers of so many tiles of 16 pairs take each.
BLOCKS = {"wide": 2100, "halved": 1400, "quartered": 780}


def in_blocks(kind, heads):
    return {"tail_rows": BLOCKS[kind] * 16 // heads, "max_length": 4096}


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 3), (7, 1), (16, 1)])
@pytest.mark.parametrize("kind", BLOCKS)
def test_attention_prompts_in_blocks(hip, fmt, page, heads, kv_heads, kind):
    rng = np.random.default_rng(heads * page + 2)
    lengths = [1, 40, 130, 300, 77, 0, 65, 200]
    new = [1, 40, 130, 33, 1, 0, 2, 17]
    store = Store(hip, fmt, page, sum(-(-l // page) for l in lengths) + 2, kv_heads, rng)
    attend(hip, store, lengths, new, heads, **in_blocks(kind, heads))


@pytest.mark.parametrize("kind", BLOCKS)
@pytest.mark.parametrize("length,rows", [(1, 1), (33, 33), (1000, 700), (700, 129)])
def test_attention_one_prompt_in_blocks(hip, kind, length, rows):
    rng = np.random.default_rng(length)
    store = Store(hip, "int8", 16, 70, 2, rng)
    attend(hip, store, [length], [rows], 4, max_rows=700, few=False, **in_blocks(kind, 4))


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("kind", BLOCKS)
def test_attention_window_in_blocks(hip, window, kind):
    rng = np.random.default_rng(window + 1)
    lengths = [1, 64, 65, 300, 129]
    store = Store(hip, "int8" if window % 2 else "e4m3", 32, 25, 2, rng)
    attend(hip, store, lengths, [1, 60, 65, 70, 1], 4, window=window, max_rows=400, **in_blocks(kind, 4))


@pytest.mark.parametrize("fmt,page", [("e4m3", 16), ("int8", 16), ("e4m3", 64)])
@pytest.mark.parametrize("kind", BLOCKS)
def test_attention_window_over_stale_pages_in_blocks(hip, fmt, page, kind):
    rng = np.random.default_rng(page + 70)
    window, lengths, new = 200, [500, 499, 370], [1, 90, 60]
    store = Store(hip, fmt, page, 100, 2, rng)

    def spoil(tables):
        stale = []
        for s, (length, n) in enumerate(zip(lengths, new)):
            for at in range(max(length - n - window + 1, 0) // page):
                stale.append(int(tables[s, at]))
                if at % 3 == 0:
                    tables[s, at] = -7
        assert stale
        for i in (0, 1):
            raw, scales = store.raw[i].numpy(), store.device_scales[i].numpy()
            raw[stale], scales[stale] = model.NAN_BYTE[fmt], np.nan
            store.raw[i].upload(raw)
            store.device_scales[i].upload(scales)

    attend(hip, store, lengths, new, 4, window=window, spoil=spoil, max_rows=400, **in_blocks(kind, 4))


@pytest.mark.parametrize("workspace", [0, 1 << 12, 1 << 16, 1 << 24])
@pytest.mark.parametrize("new", [[31, 9, 1], [8, 32, 33], [500, 1, 20]])
@pytest.mark.parametrize("kind", [None, *BLOCKS])
def test_attention_long_context_of_some_rows(hip, workspace, new, kind):
    """Sequences of one to four tiles, alone or beside longer ones."""
    rng = np.random.default_rng(18)
    store = Store(hip, "e4m3", 16, 420, 1, rng)
    more = in_blocks(kind, 2) if kind else {}
    attend(hip, store, [5000, 900, 64], new, 2, workspace=workspace, **more)


@pytest.mark.parametrize("heads,kv_heads", [(4, 2), (3, 1), (7, 1), (16, 1), (2, 2)])
@pytest.mark.parametrize("new", [[1, 1, 1, 0], [1, 17, 3, 1], [40, 1, 9, 16], [60, 60, 2, 30]])
@pytest.mark.parametrize("workspace", [1 << 14, 1 << 25])
@pytest.mark.parametrize("window", [0, 700])
def test_attention_of_fewer_rows_than_named(hip, heads, kv_heads, new, workspace, window):
    """A captured step's sizes, of which each sequence uses some: what is left over shares the contexts."""
    rng = np.random.default_rng(heads)
    store = Store(hip, "int8", 32, 230, kv_heads, rng)
    attend(hip, store, [5000, 900, 300, 257], new, heads, window=window, workspace=workspace, max_rows=60, tail_rows=100)


@pytest.mark.parametrize("kind", BLOCKS)
def test_attention_of_odd_numbers_in_blocks(hip, kind):
    """Strides, scales, scores far apart, pages of unequal scales, tables that share pages or name none."""
    rng = np.random.default_rng(19)
    more = in_blocks(kind, 4)
    store = Store(hip, "int8", 16, 60, 2, rng)
    attend(hip, store, [400, 99], [90, 3], 4, query_pad=8 * D, out_pad=4, scale=-0.3, **more)
    attend(hip, store, [400, 99], [90, 3], 4, scale=0.0, **more)
    attend(hip, store, [400, 120], [90, 120], 4, sharp=60.0, **more)

    def share(tables):
        tables[1, :10] = tables[0, :10]

    attend(hip, store, [200, 175], [70, 90], 4, spoil=share, **more)
    store = Store(hip, "int8", 16, 60, 2, rng)
    for i in (0, 1):
        for factor in (0.0, 1e-12, 30.0 if i == 0 else 1e9):
            store.scales[i][rng.random((60, 2)) < 0.15] *= np.float32(factor)
        store.codes[i][store.scales[i] == 0] = 0
    attend(hip, store, [400, 120], [90, 120], 4, **more)
    store = Store(hip, "e4m3", 32, 30, 2, rng)

    def lose(tables):
        tables[0, 1], tables[0, 3] = -1, 30
        tables[1, :] = 1 << 30
        tables[2, 0] = -1

    got = attend(hip, store, [200, 64, 70], [100, 40, 70], 4, spoil=lose, **more)
    assert np.all(got[100:140] == 0)


@pytest.mark.parametrize("kind", BLOCKS)
def test_attention_in_place_in_blocks(hip, kind):
    rng = np.random.default_rng(20)
    store = Store(hip, "int8", 16, 40, 2, rng)
    rows = 600 + in_blocks(kind, 4)["tail_rows"]
    q = gen.bf16(rng.standard_normal((rows, 4 * D)).astype(np.float32))
    tables = dev(hip, np.tile(np.arange(40, dtype=np.int32), (3, 1)))
    keep = [dev(hip, np.array([600, 0, 9], np.int32)), dev(hip, np.array([0, 590, 590, 599], np.int32))]
    outs = []
    for same in (False, True):
        query = dev(hip, q)
        out = query if same else dev(hip, q)
        scratch = hip.DeviceArray(1 << 22, np.uint8)
        hip.kv8_attention(store.cache, query, out, 4, rows, 3, tables, 40, keep[0], keep[1], max_rows=590,
                          max_length=4096, workspace=scratch, workspace_bytes=1 << 22)
        hip.synchronize()
        outs.append(out.numpy())
    assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0][599:], q[599:])
    assert not np.array_equal(outs[0][:599], q[:599])


def test_attention_far_pages(hip):
    """Pages behind 2^32 bytes of the pool."""
    rng = np.random.default_rng(15)
    heads, page = 8, 16
    page_bytes = heads * 2048
    pages = (1 << 32) // page_bytes + 70
    raw = [hip.DeviceArray((pages, page_bytes), np.uint8) for _ in range(2)]
    scales = [hip.DeviceArray((pages, heads), np.float32) for _ in range(2)]
    cache = hip.Kv8Cache("int8", page, pages, heads, *raw, *scales)
    store = Store(hip, "int8", page, 64, heads, rng)  # the model's side, and the bytes that go to the far pages
    far = pages - 64
    for i, is_key in enumerate((True, False)):
        packed = model.pack(store.codes[i], is_key)
        hip.call("qwen3_tts_device_memcpy", raw[i].offset(far * page_bytes), packed.ctypes.data, packed.nbytes)
        hip.call("qwen3_tts_device_memcpy", scales[i].offset(far * heads), store.scales[i].ctypes.data,
                 store.scales[i].nbytes)
    tables = np.arange(64, dtype=np.int32).reshape(1, 64)
    for rows in (1, 70):
        starts, lengths = np.array([0, rows], np.int32), np.array([1000], np.int32)
        q = gen.bf16(rng.standard_normal((rows, 16 * D)).astype(np.float32))
        out = hip.DeviceArray(q.shape, np.uint16)
        keep = [dev(hip, q), dev(hip, tables + far), dev(hip, lengths), dev(hip, starts)]
        hip.kv8_attention(cache, keep[0], out, 16, rows, 1, keep[1], 64, keep[2], keep[3], max_rows=rows,
                          max_length=1000)
        # and a row stored there
        hip.synchronize()
        want, tolerance = model.attention("int8", page, *store.codes, *store.scales, gen.f32(q), tables, lengths,
                                          starts, 16, D ** -0.5, 0, FEW_ROWS if rows == 1 else MANY_ROWS)
        off = np.abs(gen.f32(out.numpy()).reshape(rows, 16, D) - want)
        assert np.all(off <= tolerance)
    key, value = kv_rows(rng, 2, heads), kv_rows(rng, 2, heads)
    slots = np.array([(pages - 1) * page, (pages - 1) * page + 1], np.int32)
    hip.kv8_append(cache, dev(hip, key), dev(hip, value), dev(hip, slots), 2)
    hip.synchronize()
    store.append(key, value, slots - far * page)
    for i, is_key in enumerate((True, False)):
        got = np.empty((1, heads, 1, 2048), np.uint8)
        hip.call("qwen3_tts_device_memcpy", got.ctypes.data, raw[i].offset((pages - 1) * page_bytes), got.nbytes)
        assert np.array_equal(model.unpack(got, is_key)[0, :, :2], store.codes[i][63, :, :2])


# ---------------------------------------------------------------------------
# The three together
# ---------------------------------------------------------------------------
class Server:
    """A small server's state: a plan in place, one layer's cache, buffers of fixed size."""

    def __init__(self, hip, rng, fmt, page, sequences, pages, capacity, heads, kv_heads):
        self.hip, self.fmt, self.heads, self.capacity = hip, fmt, heads, capacity
        self.plan = Plan(hip, page, pages, np.full((sequences, pages), -1, np.int32), np.zeros(sequences, int),
                         rng.permutation(pages), pages, capacity, in_place=True)
        self.store = Store(hip, fmt, page, pages, kv_heads)
        self.qkv = hip.DeviceArray((capacity, (heads + 2 * kv_heads) * D), np.uint16)
        self.out = hip.DeviceArray((capacity, heads * D), np.uint16)
        self.scratch = hip.DeviceArray(1 << 20, np.uint8)

    def launch(self, stream=None):
        p, width = self.plan, (self.heads + 2 * self.store.heads) * D
        p.launch(stream)
        self.hip.kv8_append(self.store.cache, self.qkv.offset(self.heads * D),
                            self.qkv.offset((self.heads + self.store.heads) * D), p.row_slots, self.capacity,
                            key_stride=width, value_stride=width, stream=stream)
        self.hip.kv8_attention(self.store.cache, self.qkv, self.out, self.heads, self.capacity, p.sequences, p.tables,
                               p.stride, p.new_lengths, p.row_starts, max_rows=self.capacity,
                               max_length=p.pages * p.page, query_stride=width, workspace=self.scratch,
                               workspace_bytes=1 << 20, stream=stream)

    def step(self, rng, new, launch):
        """Uploads a step's inputs, launches it and compares everything."""
        p, store = self.plan, self.store
        want = p.expected(new)
        qkv = kv_rows(rng, self.capacity, self.heads + 2 * store.heads, spread=False)
        qkv[int(want["row_starts"][-1]):] = 0x7FC0  # rows of no sequence: NaN
        self.qkv.upload(qkv)
        self.out.upload(np.full((self.capacity, self.heads * D), 0x1234, np.uint16))
        p.new_tokens.upload(np.array(new, np.int32))
        launch()
        self.hip.synchronize()
        p.check(want)
        q, k = self.heads * D, (self.heads + store.heads) * D
        store.append(np.ascontiguousarray(qkv[:, q:k]), np.ascontiguousarray(qkv[:, k:]), want["row_slots"])
        held = np.zeros(store.pages, int)
        for s, length in enumerate(want["new_lengths"]):
            for at in range(0, length, p.page):
                held[want["tables"][s, at // p.page]] = min(p.page, length - at)
        store.check(held)
        live = int(want["row_starts"][-1])
        ref, tolerance = model.attention(self.fmt, p.page, *store.codes, *store.scales, gen.f32(qkv[:, :q]),
                                         want["tables"], want["new_lengths"], want["row_starts"], self.heads,
                                         D ** -0.5, 0, MANY_ROWS)
        got = self.out.numpy()
        assert np.all(got[live:] == 0x1234)
        off = np.abs(gen.f32(got[:live]).reshape(live, self.heads, D) - ref[:live])
        assert np.all(off <= tolerance[:live])
        return want


def traffic(rng, lengths, prompt):
    new = np.where(lengths > 0, 1, np.where(rng.random(len(lengths)) < 0.5, rng.integers(1, prompt, len(lengths)), 0))
    new[(lengths > 0) & (rng.random(len(lengths)) < 0.12)] = -1
    return new


@pytest.mark.parametrize("fmt,page", [("int8", 16), ("e4m3", 32), ("int8", 64)])
def test_steps_of_a_server(hip, fmt, page):
    """Sequences come with prompts, grow by single tokens and end; pages come round with stale bytes in them."""
    rng = np.random.default_rng(page + 5)
    server = Server(hip, rng, fmt, page, 6, 26 if page == 16 else 16, 90, 4, 2)
    lengths, refused = np.zeros(6, int), 0
    for _ in range(14):
        want = server.step(rng, traffic(rng, lengths, 60), server.launch)
        lengths, refused = want["new_lengths"], refused + int(want["refused"][0])
    assert refused > 0 or page > 16


def test_steps_captured_into_a_graph(hip):
    """One graph of plan, append and attention, replayed for steps of different content, with eager steps of the
    same state between the replays."""
    rt = Runtime(hip)
    rng = np.random.default_rng(21)
    server = Server(hip, rng, "e4m3", 16, 5, 30, 64, 4, 2)
    s = rt.stream()
    lengths = np.zeros(5, int)
    # sized by the graph's buffers: nothing is launched while it is captured
    graph, exe = rt.capture(s, lambda: server.launch(s))
    try:
        for i in range(9):
            def replay():
                rt.launch(exe, s)
                rt.sync(s)
            want = server.step(rng, traffic(rng, lengths, 50), server.launch if i % 3 == 1 else replay)
            lengths = want["new_lengths"]
    finally:
        rt.destroy(graph, exe)
        hip.load().qwen3_tts_stream_destroy(s)


def test_steps_with_the_decode_primitives(hip):
    """A decode step as a model makes it: the plan's positions rotate the normalized query and key heads, which the
    append stores and the attention reads."""
    rng = np.random.default_rng(31)
    heads, kv_heads, sequences, pages = 4, 2, 5, 30
    plan = Plan(hip, 16, pages, np.full((sequences, 8), -1, np.int32), np.zeros(sequences, int), rng.permutation(pages),
                pages, 64, in_place=True)
    store = Store(hip, "int8", 16, pages, kv_heads)
    gains = [dev(hip, gen.gains(rng, D)) for _ in range(2)]
    lengths = np.zeros(sequences, int)
    for _ in range(6):
        new = traffic(rng, lengths, 14)
        want = plan.expected(new)
        q, k, v = (kv_rows(rng, 64, h, spread=False) for h in (heads, kv_heads, kv_heads))
        dq, dk, dv, out = dev(hip, q), dev(hip, k), dev(hip, v), dev(hip, np.zeros((64, heads * D), np.uint16))
        plan.new_tokens.upload(np.array(new, np.int32))
        plan.launch()
        for array, n, gain in ((dq, heads, gains[0]), (dk, kv_heads, gains[1])):
            hip.call("qwen3_tts_op_head_rms_norm_rows", array.ptr, gain.ptr, 64, n, D, C.c_float(1e-6), None)
            hip.call("qwen3_tts_op_rope_rows", array.ptr, 64, n, D, plan.row_positions.ptr, C.c_float(1e6), None)
        hip.kv8_append(store.cache, dk, dv, plan.row_slots, 64)
        hip.kv8_attention(store.cache, dq, out, heads, 64, sequences, plan.tables, plan.stride, plan.new_lengths,
                          plan.row_starts, max_rows=14, max_length=128)
        hip.synchronize()
        plan.check(want)
        live, lengths = int(want["row_starts"][-1]), want["new_lengths"]
        store.append(dk.numpy(), v, want["row_slots"])
        ref, tolerance = model.attention("int8", 16, *store.codes, *store.scales, gen.f32(dq.numpy()), want["tables"],
                                         lengths, want["row_starts"], heads, D ** -0.5, 0, MANY_ROWS)
        off = np.abs(gen.f32(out.numpy())[:live].reshape(live, heads, D) - ref[:live])
        assert np.all(off <= tolerance[:live])


FIRST_CALL = """
import sys
sys.path[:0] = {paths!r}
import numpy as np
import qwen3_tts_hip as hip
import test_kv8_gpu as t
from test_zz_no_alloc import Runtime
hip.load()
rt, rng = Runtime(hip), np.random.default_rng(3)
server = t.Server(hip, rng, "int8", 16, 4, 40, 300, 4, 2)
s = rt.stream()
graph, exe = rt.capture(s, lambda: server.launch(s))

def replay():
    rt.launch(exe, s)
    rt.sync(s)

lengths = np.zeros(4, int)
for new in ([200, 0, 30, 1], [1, 17, 1, 1], [-1, 1, 1, 1], [260, 1, 1, -1]):
    lengths = server.step(rng, new, replay)["new_lengths"]
print("same after capture as the first call")
"""


def test_first_calls_of_a_process_under_capture(hip):
    """A fresh process whose first launches of the three operators are captured; every replay is right."""
    import pathlib
    import subprocess
    import sys

    here = pathlib.Path(__file__).resolve().parent
    paths = [str(here), str(here.parent / "qwen3-tts-native_amd")]
    run = subprocess.run([sys.executable, "-c", FIRST_CALL.format(paths=paths)], capture_output=True, text=True, timeout=100)
    assert run.returncode == 0 and "same after capture" in run.stdout, run.stdout + run.stderr


def test_two_streams_with_workspaces_of_their_own(hip):
    """Attention of two servers on two streams, many calls in flight at once, each with its own workspace."""
    rt = Runtime(hip)
    rng = np.random.default_rng(22)
    streams = [rt.stream() for _ in range(2)]
    try:
        calls = []
        for st in streams:
            store = Store(hip, "int8", 16, 260, 2, rng)
            rows = 3
            q = gen.bf16(rng.standard_normal((rows, 4 * D)).astype(np.float32))
            lengths, starts = np.array([4000, 70, 30], np.int32), np.arange(4, dtype=np.int32)
            tables = np.full((3, 250), -1, np.int32)
            tables[0], tables[1, :5], tables[2, :2] = np.arange(250), np.arange(250, 255), np.arange(255, 257)
            keep = [dev(hip, a) for a in (q, tables, lengths, starts)]
            outs = [hip.DeviceArray(q.shape, np.uint16) for _ in range(6)]
            scratch = hip.DeviceArray(1 << 20, np.uint8)
            want, tolerance = model.attention("int8", 16, *store.codes, *store.scales, gen.f32(q), tables, lengths,
                                              starts, 4, D ** -0.5, 0, FEW_ROWS)
            calls.append((st, store, keep, outs, scratch, want, tolerance))
        for i in range(6):
            for st, store, keep, outs, scratch, _, _ in calls:
                hip.kv8_attention(store.cache, keep[0], outs[i], 4, 3, 3, keep[1], 250, keep[2], keep[3], max_rows=1,
                                  max_length=4000, workspace=scratch, workspace_bytes=1 << 20, stream=st)
        hip.synchronize()
        for _, _, _, outs, _, want, tolerance in calls:
            for out in outs:
                assert np.all(np.abs(gen.f32(out.numpy()).reshape(3, 4, D) - want) <= tolerance)
    finally:
        for st in streams:
            hip.load().qwen3_tts_stream_destroy(st)

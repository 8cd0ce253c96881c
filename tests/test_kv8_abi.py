"""CPU-side checks of the paged 8-bit cache's entry points: struct layouts,
refusals before any device is touched, empty calls, and the 64-bit model that
the GPU tests compare with."""
import ctypes as C

import numpy as np
import pytest

import kv8_model as model

FAKE = 4096  # an aligned address that is never dereferenced


def cache(hip, **changes):
    c = hip.Kv8CacheV1(C.sizeof(hip.Kv8CacheV1), hip.KV8_INT8, 16, 8, 2, 128, FAKE, FAKE, FAKE, FAKE)
    for k, v in changes.items():
        setattr(c, k, v)
    return c


def plan(hip, **changes):
    a = hip.Kv8PlanV1(C.sizeof(hip.Kv8PlanV1), 2, 16, 8, 4, 8, *[FAKE] * 11)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def append(hip, **changes):
    a = hip.Kv8AppendV1(C.sizeof(hip.Kv8AppendV1), 2, 256, 256, FAKE, FAKE, FAKE)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def attention(hip, **changes):
    a = hip.Kv8AttentionV1(C.sizeof(hip.Kv8AttentionV1), 4, 2, 512, 512, 2, 4, 1, 64, 0, 0.1, 0, FAKE, FAKE, FAKE, FAKE,
                           FAKE, None, 0)
    for k, v in changes.items():
        setattr(a, k, v)
    return a


def refused(hip, name, *args):
    with pytest.raises(hip.Qwen3TtsError) as e:
        hip.call(name, *args)
    assert e.value.status == hip.STATUS_INVALID_ARGUMENT
    return str(e.value)


def test_struct_layouts(hip):
    assert C.sizeof(hip.Kv8CacheV1) == 56
    assert C.sizeof(hip.Kv8PlanV1) == 112
    assert C.sizeof(hip.Kv8AppendV1) == 40
    assert C.sizeof(hip.Kv8AttentionV1) == 104


BAD_CACHE = [dict(struct_size=12), dict(format=2), dict(format=-1), dict(page_tokens=0), dict(page_tokens=24),
             dict(page_tokens=128), dict(pages=0), dict(pages=1 << 28), dict(key_value_heads=0),
             dict(key_value_heads=1 << 17), dict(head_dimension=64), dict(key_pages=None), dict(value_pages=FAKE + 8),
             dict(key_scales=FAKE + 2), dict(value_scales=None)]


@pytest.mark.parametrize("changes", BAD_CACHE)
def test_bad_caches_are_refused(hip, changes):
    c = cache(hip, **changes)
    refused(hip, "qwen3_tts_op_kv8_append_v1", C.byref(c), C.byref(append(hip)), None)
    refused(hip, "qwen3_tts_op_kv8_attention_v1", C.byref(c), C.byref(attention(hip)), None)


@pytest.mark.parametrize("changes", [
    dict(struct_size=0), dict(sequences=0), dict(sequences=-1), dict(page_tokens=17), dict(pages=0),
    dict(pages=1 << 28), dict(table_stride=0), dict(table_stride=1 << 28), dict(rows_capacity=-1), dict(rows_capacity=1 << 30), dict(lengths=None),
    dict(new_tokens=None), dict(new_lengths=None), dict(tables=None), dict(free_pages=None), dict(free_count=None),
    dict(new_free_count=None), dict(row_starts=None), dict(row_positions=None), dict(row_slots=None),
    dict(refused=None), dict(lengths=FAKE + 1)])
def test_plan_refusals(hip, changes):
    refused(hip, "qwen3_tts_op_kv8_plan_v1", C.byref(plan(hip, **changes)), None)


@pytest.mark.parametrize("changes", [
    dict(struct_size=8), dict(rows=-1), dict(key_stride=248), dict(value_stride=128), dict(key_stride=260),
    dict(key=None), dict(value=FAKE + 2), dict(row_slots=None), dict(row_slots=FAKE + 2)])
def test_append_refusals(hip, changes):
    refused(hip, "qwen3_tts_op_kv8_append_v1", C.byref(cache(hip)), C.byref(append(hip, **changes)), None)


@pytest.mark.parametrize("changes", [
    dict(struct_size=8), dict(query_heads=0), dict(query_heads=3), dict(query_heads=34), dict(rows=-1),
    dict(sequences=-1), dict(sequences=70000), dict(table_stride=0), dict(max_rows=0), dict(max_length=0),
    dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(reserved=1), dict(query=None),
    dict(query=FAKE + 8), dict(out=FAKE + 4), dict(tables=None), dict(lengths=FAKE + 2), dict(row_starts=None),
    dict(query_stride=504), dict(query_stride=516), dict(out_stride=514), dict(workspace_bytes=64),
    dict(workspace=FAKE + 4, workspace_bytes=64)])
def test_attention_refusals(hip, changes):
    refused(hip, "qwen3_tts_op_kv8_attention_v1", C.byref(cache(hip)), C.byref(attention(hip, **changes)), None)


def test_null_structs_are_refused(hip):
    assert "null" in refused(hip, "qwen3_tts_op_kv8_plan_v1", None, None)
    assert "null" in refused(hip, "qwen3_tts_op_kv8_append_v1", None, C.byref(append(hip)), None)
    assert "null" in refused(hip, "qwen3_tts_op_kv8_append_v1", C.byref(cache(hip)), None, None)
    assert "null" in refused(hip, "qwen3_tts_op_kv8_attention_v1", C.byref(cache(hip)), None, None)
    assert "null" in refused(hip, "qwen3_tts_op_kv8_attention_workspace_v1", C.byref(cache(hip)),
                             C.byref(attention(hip)), None)


def test_calls_without_rows_do_nothing(hip):
    hip.call("qwen3_tts_op_kv8_append_v1", C.byref(cache(hip)), C.byref(append(hip, rows=0, key=None)), None)
    hip.call("qwen3_tts_op_kv8_attention_v1", C.byref(cache(hip)), C.byref(attention(hip, rows=0, query=None)), None)
    hip.call("qwen3_tts_op_kv8_attention_v1", C.byref(cache(hip)), C.byref(attention(hip, sequences=0)), None)


def test_model_e4m3_values():
    """The format's published corners: largest 448, smallest normal 2^-6, smallest subnormal 2^-9, 0x7f no number."""
    assert model.E4M3[0x7E] == 448 and model.E4M3[0x08] == 2.0 ** -6 and model.E4M3[0x01] == 2.0 ** -9
    assert np.isnan(model.E4M3[[0x7F, 0xFF]]).all() and np.isfinite(np.delete(model.E4M3, [0x7F, 0xFF])).all()
    for code in range(256):
        if code & 0x7F != 0x7F:
            assert model.encode("e4m3", model.E4M3[code]) == code
    # ties go to the even code, beyond the range to its end
    assert model.encode("e4m3", 2.0 ** -10) == 0 and model.encode("e4m3", 3 * 2.0 ** -10) == 2
    assert model.encode("e4m3", 17.0) == model.encode("e4m3", 16.0) and model.encode("e4m3", 1e9) == 0x7E


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_model_rounds_by_half_a_step(fmt):
    rng = np.random.default_rng(1)
    x = rng.uniform(-1, 1, 4096) * (127 if fmt == "int8" else 448)
    off = np.abs(model.decode(fmt, model.encode(fmt, x)) - x)
    assert np.all(off <= (0.5 if fmt == "int8" else np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10)))


@pytest.mark.parametrize("is_key", [True, False])
def test_model_layout_is_one_to_one(is_key):
    codes = np.random.default_rng(2).integers(0, 256, (3, 2, 32, 128)).astype(np.uint8)
    raw = model.pack(codes, is_key)
    assert sorted(model._offsets(is_key).ravel()) == list(range(2048))
    assert np.array_equal(model.unpack(raw, is_key), codes)


def test_attention_workspace_is_bounded(hip):
    """Any sizes that a caller may name: an answer, and no more than a small part of the card's memory."""
    import random
    draw = random.Random(1)

    def size(bits):
        return round(2 ** draw.uniform(0, bits))

    for _ in range(20000):
        heads = draw.choice([1, 2, 4, 8, 16, 32])
        pages = hip.Kv8Cache("int8", 16, 100, heads, FAKE, FAKE, FAKE, FAKE)
        rows = size(20)
        bytes_ = hip.kv8_attention_workspace(pages, heads * draw.choice([1, 2, 3, 5, 8, 16]), rows, size(16) - 1,
                                             window=draw.choice([0, 0, size(20), 2 ** 31 - 1]),
                                             max_rows=draw.choice([1, size(12), rows, 2 ** 31 - 1]),
                                             max_length=draw.choice([size(20), 2 ** 31 - 1]))
        assert 0 <= bytes_ <= 1 << 28

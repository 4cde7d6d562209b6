"""CPU checks of the decoder operators' oracle (oracle/decoder.py) and of what the library refuses without a device."""
import ctypes

import numpy as np
import pytest

from oracle import decoder as D
from oracle import valu as V
from snntome_b200 import _lib
from snntome_b200.native import KV8Cache, NativeError, _int32, _sizes


def test_e4m3_numbers_are_those_of_the_type():
    import torch
    codes = torch.arange(256, dtype=torch.uint8)
    want = codes.view(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.array_equal(D.e4m3_values(), want, equal_nan=True)
    x = np.random.default_rng(1).normal(0, 50, 20000).clip(-448, 448)
    got = torch.from_numpy(x).to(torch.float8_e4m3fn).to(torch.float64).numpy()
    assert np.all(np.abs(got - x) <= D.e4m3_half_step(x) * (1 + 2.0 ** -20))


def test_window_and_sinks():
    see = D.visible(8, 0, 8, 3, 2)
    assert [list(np.flatnonzero(r)) for r in see] == [[0], [0, 1], [0, 1, 2], [0, 1, 2, 3], [0, 1, 2, 3, 4], [0, 1, 3, 4, 5], [0, 1, 4, 5, 6], [0, 1, 5, 6, 7]]
    assert np.array_equal(D.visible(5, 0, 5, 0, 3), np.tril(np.ones((5, 5), dtype=bool)))


def test_window_attention_without_a_window_is_the_causal_attention():
    h_q, h_kv, dim, seq, frames = 4, 2, 64, 32, 2
    pitch = seq * frames
    rng = np.random.default_rng(2)
    rq, rk = h_q * dim, h_kv * dim
    canvas = np.zeros((2 * rq + 2 * rk) * pitch, dtype=np.uint16)
    body = rng.normal(0, 1, ((rq + 2 * rk) * pitch)).astype(np.float16)
    canvas[: body.size] = body.view(np.uint16)
    x = body.astype(np.float64).reshape(-1, pitch)
    out, bound = D.window_attention(x[:rq], x[rq: rq + rk], x[rq + rk:], h_q, h_kv, seq, pitch, 0, 0, 10000.0)
    V.rope(canvas, 0, h_q, dim, pitch, seq)
    V.rope(canvas, rq * pitch, h_kv, dim, pitch, seq)
    o = (rq + 2 * rk) * pitch
    V.causal_attention(canvas, 0, rq * pitch, (rq + rk) * pitch, o, h_q, h_kv, dim, pitch, seq)
    assert np.all(np.abs(canvas[o:].view(np.float16).reshape(rq, pitch) - out) <= bound)


def test_probabilities():
    x = np.array([[1.0, -np.inf, np.nan], [1.0, -np.inf, 0.0], [0.0, -np.inf, 0.0]])
    lp, ent = D.logprobs(x)
    z = 2 * np.e + 1
    assert np.allclose(lp[:, 0], [1 - np.log(z), 1 - np.log(z), -np.log(z)])
    assert np.allclose(ent[0], np.log(z) - 2 * np.e / z)
    assert np.isnan(lp[:, 1:]).all() and np.isnan(ent[1:]).all()
    assert D.top_rows(x, 3).T.tolist() == [[0, 1, 2], [0, 1, 2], [1, 2, 0]]


def test_cache_sizes():
    f = KV8Cache.bytes_needed
    up = lambda n: (n + 255) // 256 * 256
    for c, h, d, n in [(1, 1, 64, 1), (3, 2, 128, 65), (64, 8, 64, 512)]:
        nb = (n + 63) // 64
        assert f(c, h, d, n) == up(c * h * nb * 128 * d) + up(c * h * nb * 8) + 2 * up(c * h * 64 * d * 2) + up(c * h * 4)
    assert f(0, 1, 64, 1) == 0 and f(1, 1, 96, 1) == 0 and f(1, 1, 64, 0) == 0 and f(1, 1, 64, 1 << 31) == 0
    for bad in [(0, 1, 64, 8), (1, 1, 80, 8), (1, -1, 64, 8), (1, 1, 64, 1 << 40)]:
        with pytest.raises(NativeError):
            KV8Cache(*bad)


@pytest.mark.parametrize("columns,h_kv,head_dim,max_seq", [(1 << 16, 1 << 16, 128, (1 << 31) - 1), (1 << 16, 1 << 15, 128, 1 << 24), (1 << 31, 1 << 31, 64, 1), ((1 << 32) - 1, (1 << 32) - 1, 64, 1)])
def test_caches_whose_sizes_would_wrap_have_none(columns, h_kv, head_dim, max_seq):
    lib = _lib.get_lib()
    assert lib.k44b_kv8_bytes(columns, h_kv, head_dim, max_seq) == 0
    desc = _lib.KV8CacheDesc(256, (1 << 64) - 1, columns, h_kv, head_dim, max_seq)      # never read: refused by its sizes
    assert lib.k44b_kv8_clear(ctypes.byref(desc), None) == -1


def test_calls_without_a_plan_or_a_cache_fail():
    lib = _lib.get_lib()
    desc = _lib.KV8CacheDesc(None, 0, 1, 1, 64, 8)
    assert lib.k44b_kv8_clear(None, None) == -1
    assert lib.k44b_kv8_clear(ctypes.byref(desc), None) == -1
    assert lib.k44b_plan_add_window_attn(None, b"", 0, 0, 0, 0, 1, 1, 64, 1, 0, 0, 1e4, 0) == -1
    assert lib.k44b_plan_add_kv8_fill(None, b"", ctypes.byref(desc), 0, 0, 1, 1e4, 0) == -1
    assert lib.k44b_plan_add_kv8_attn(None, b"", ctypes.byref(desc), 0, 0, 0, 0, 1, 0, 0, 1e4, 0) == -1
    assert lib.k44b_plan_add_logprobs(None, b"", 0, 1, None, None, None, 0, None, None) == -1
    assert lib.k44b_plan_set_positions(None, None, 0, None) == -1
    assert lib.k44b_plan_set_sequences(None, None, None, 0, None) == -1
    assert lib.k44b_plan_columns(None) == 0


def test_numbers_that_would_wrap_are_refused():
    for bad in (-1, 1 << 31, 1 << 40):
        with pytest.raises(NativeError):
            _sizes("size", bad)
    for bad in ([1.5], [1 << 31], [[1]], [-(1 << 31) - 1]):
        with pytest.raises(NativeError):
            _int32("list", bad)
    assert _int32("list", [3, -1]).dtype == np.int32 and _int32("list", []).size == 0

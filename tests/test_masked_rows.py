"""Rows that a decode attention does not see weigh nothing, whatever they hold: rows before a window that starts inside a
page, and rows behind the cursor in the last page (a rejected tail). Over every page type, without sinks, against the
plain 64-bit restatement in helpers/u4_reference.py."""
import numpy as np
import pytest

import saragossa_b200 as sg
from helpers import u4_reference as ref

DTYPES = [sg.KV_F32, sg.KV_BF16, sg.KV_U8G32, sg.KV_U4G32]
# u8: a weight and a scale are fp16 numbers (2^-12 each, the error of a product's factors), their product another (2^-12), and
# the query's second fp16 part leaves nothing of note: 3 * 2^-12 at most of any row's share, so of the result's largest terms
U8_REL = 2e-3


@pytest.fixture(scope="module")
def state():
    st = sg.DecodeResidentState(0)
    yield st
    assert st.device_status() == 0
    st.close()


def _bad_rows(n, kv_dim):
    """Rows of NaN, of infinities of either sign, and of a range that overflows."""
    x = np.empty((n, kv_dim), np.float32)
    x[0::4], x[1::4], x[2::4] = np.nan, np.inf, -np.inf
    x[3::4] = np.where(np.arange(kv_dim) % 2, np.float32(3.3e38), np.float32(-3.3e38))
    return x


def _close(got, want, dtype):
    if dtype != sg.KV_U8G32:
        return ref.close(got, want)[0]
    return np.linalg.norm(got.reshape(want[0].shape) - want[0]) <= U8_REL * np.linalg.norm(want[0])


def _cache(state, dtype, kv_heads, hd, q_heads, n, first, cap):
    """`cap` rows, of which [first, n) are finite and the others are not; and the finite ones as they read back, the others as
    zeros."""
    rng = np.random.default_rng(n + hd)
    k, v = rng.standard_normal((2, cap, kv_heads * hd)).astype(np.float32)
    kv = state.full_attention(cap, q_heads, kv_heads, hd, dtype, shuffled_seed=7)
    kv.seed(k, v, cap)
    held = [x.astype(np.float64) for x in kv.gather_rows_f32()]
    for x in (k, v):
        x[:first], x[n:] = _bad_rows(first, kv_heads * hd), _bad_rows(cap - n, kv_heads * hd)
    kv.seed(k, v, cap)
    for x in held:
        x[:first], x[n:] = 0.0, 0.0
    return kv, held


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(8, 2, 128), (16, 2, 128), (16, 2, 256), (4, 2, 64)])
@pytest.mark.parametrize("n,first", [(41, 0), (90, 60), (1003, 0), (1003, 509), (16, 15), (33, 32)])
def test_rows_out_of_sight(state, dtype, q_heads, kv_heads, hd, n, first):
    kv, (k, v) = _cache(state, dtype, kv_heads, hd, q_heads, n, first, n + 23)
    kv.truncate(n)
    q = np.random.default_rng(n).standard_normal((q_heads, hd)).astype(np.float32)
    want = ref.attention(q, k[:n], v[:n], kv_heads, first)
    assert _close(kv.attention_decode_windowed(q, first), want, dtype)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    kv.encode_attention_decode_noalloc(d_q, d_out, first)
    state.sync()
    assert _close(d_out.download(), want, dtype)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("n,window", [(41, 0), (41, 20), (47, 30), (700, 300)])
def test_a_step_behind_a_rejected_tail(state, dtype, hd, n, window):
    """The row of a fused append goes over the first row of the tail; the rest of the tail stays out of sight."""
    q_heads, kv_heads = 8, 2
    first = max(0, n + 1 - window) if window else 0
    kv, (k, v) = _cache(state, dtype, kv_heads, hd, q_heads, n, first, n + 23)
    rng = np.random.default_rng(n)
    new = rng.standard_normal((2, kv_heads * hd)).astype(np.float32)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    d_k, d_v, d_q, d_out = state.upload(new[0]), state.upload(new[1]), state.upload(q), state.alloc(q.nbytes)
    kv.encode_truncate(n)
    kv.encode_append_attention(d_k, d_v, d_q, d_out, window)
    state.sync()
    for held, row in zip((k, v), kv.gather_rows_f32(n, 1)):
        held[n] = row
    assert _close(d_out.download(), ref.attention(q, k[:n + 1], v[:n + 1], kv_heads, first), dtype)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(8, 2, 128), (16, 2, 256), (4, 2, 64), (2, 1, 96)])
def test_rows_that_nobody_wrote_are_zeros(state, dtype, q_heads, kv_heads, hd):
    """A cursor moved ahead of what was written: the rows between read back as zeros, and weigh as zeros do."""
    rng = np.random.default_rng(hd)
    kv = state.full_attention(90, q_heads, kv_heads, hd, dtype, shuffled_seed=3)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    kv.truncate(37)
    assert not kv.gather_rows_f32()[1].any()
    assert not kv.attention_decode(q).any()
    k, v = rng.standard_normal((2, 40, kv_heads * hd)).astype(np.float32)
    kv.append_batch(k, v)
    held = [x.astype(np.float64) for x in kv.gather_rows_f32()]
    for start in (0, 36, 37):
        assert _close(kv.attention_decode_windowed(q, start), ref.attention(q, *held, kv_heads, start), dtype), start
    kv.close()

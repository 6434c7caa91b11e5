"""Attention over 4-bit pages where a looser test would pass by chance: queries so large that one row takes all the weight, scores
that rise from page to page, and long caches in two launches at once."""
import numpy as np
import pytest

import saragossa_b200 as sg
from helpers import u4_reference as ref


@pytest.fixture(scope="module")
def state():
    st = sg.DecodeResidentState(0)
    yield st
    assert st.device_status() == 0
    st.close()


def _rows(n, kv_heads, hd, seed):
    return np.random.default_rng(seed).standard_normal((2, n, kv_heads * hd)).astype(np.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [3e3, 1e4, 1e6, 1e10])
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(8, 2, 64), (8, 2, 128), (16, 2, 128), (8, 1, 256), (4, 1, 256)])
def test_a_large_query_picks_its_row(state, q_heads, kv_heads, hd, scale):
    """Every head's query is a key of another row, scaled: the score of that row leads by some scale / 2, which is thousands of
    times what scores may be off (their bound in helpers/u4_reference.py, about scale * 1e-4), so the output is that row of
    V: weight 1, off by the two fp16 numbers of the weight (2^-21) and the sum of two parts (2^-23 of three times the row)."""
    n = 700
    k, v = _rows(n, kv_heads, hd, hd)
    kv = state.full_attention(n, q_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=4)
    kv.seed(k, v, n)
    kk, vv = (ref.stored(x, 0, hd, 3).reshape(n, kv_heads, hd) for x in (k, v))
    gqa = q_heads // kv_heads
    picks = [(97 * h + 5) % n for h in range(q_heads - 1)] + [n - 1]
    q = np.stack([kk[r, h // gqa] / np.linalg.norm(kk[r, h // gqa]) * scale for h, r in enumerate(picks)]).astype(np.float32)
    for h, r in enumerate(picks):      # the case is what it says it is
        s = kk[:, h // gqa] @ q[h].astype(np.float64) / np.sqrt(hd)
        lead = s[r] - np.delete(s, r).max()
        size = np.sum(np.abs(q[h])) * 3 * np.abs(kk[:, h // gqa]).max() / np.sqrt(hd)
        assert lead > 100 + 100 * (hd / 8 + 16) * size * 2.0 ** -23
    got = kv.attention_decode(q).reshape(q_heads, hd)
    for h, r in enumerate(picks):
        want = vv[r, h // gqa]
        assert np.abs(got[h] - want).max() <= 1e-5 * np.abs(want).max(), (h, r)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(8, 2, 64), (8, 2, 128), (16, 2, 128), (8, 1, 256)])
@pytest.mark.parametrize("rise", [0.02, 0.1, 0.5, -0.1])
def test_scores_that_rise_from_row_to_row(state, q_heads, kv_heads, hd, rise):
    """The largest score so far moves with nearly every page (or with none after the first, where they fall)."""
    n, gqa = 600, q_heads // kv_heads
    k, v = _rows(n, kv_heads, hd, 3 * hd)
    rng = np.random.default_rng(hd)
    toward = rng.standard_normal((kv_heads, hd))
    toward /= np.linalg.norm(toward, axis=1, keepdims=True)
    r = np.arange(n) * rise
    k = (k.reshape(n, kv_heads, hd) * 0.2 + (r[:, None, None] * np.sqrt(hd) * toward / 4)).astype(np.float32).reshape(n, -1)
    q = (4 * np.repeat(toward, gqa, 0) + 0.2 * rng.standard_normal((q_heads, hd))).astype(np.float32)
    kv = state.full_attention(n, q_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=4)
    kv.seed(k, v, n)
    kk, vv = (ref.stored(x, 0, hd, 3) for x in (k, v))
    # 1e-5 is for scores of normal rows and queries, whose products add up to 2 / pi sqrt(hd); the error goes with that sum
    sums = (np.abs(kk.reshape(n, kv_heads, 1, hd)) * np.abs(q.reshape(1, kv_heads, gqa, hd))).sum(-1).max() / np.sqrt(hd)
    ok, far = ref.close(kv.attention_decode(q), ref.attention(q, kk, vv, kv_heads), rel=1e-5 * max(1.0, sums / (2 / np.pi * np.sqrt(hd))))
    assert ok, far
    kv.close()


@pytest.mark.gpu
def test_long_caches_on_two_streams_at_once(state):
    """Launches whose blocks wait for one another (many splits that merge together), on two streams with nothing between them."""
    import torch
    n, q_heads, kv_heads, hd = 9000, 16, 2, 128
    state.set_concurrent_streams(True)
    cases = []
    for s in range(2):
        k, v = _rows(n, kv_heads, hd, 40 + s)
        kv = state.full_attention(n, q_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=s + 1)
        kv.seed(k, v, n)
        q = np.random.default_rng(s).standard_normal((q_heads, hd)).astype(np.float32)
        want = ref.attention(q, ref.stored(k, 0, hd, 3), ref.stored(v, 0, hd, 3), kv_heads)
        cases.append((kv, state.upload(q), state.alloc(q.nbytes), want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for kv, d_q, d_out, _, stream in cases:
            kv.encode_attention_decode_windowed(d_q, d_out, stream=stream.cuda_stream)
    torch.cuda.synchronize()
    assert state.device_status() == 0
    for kv, _, d_out, want, _ in cases:
        assert ref.close(d_out.download(), want)[0]
        kv.close()
    state.set_concurrent_streams(False)

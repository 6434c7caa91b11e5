"""Attention over 4-bit pages where the ranges of V differ from group to group of a head row and from row to row: every group of
32 output channels is held to its own size, not to the head's. Against the plain 64-bit restatement."""
import numpy as np
import pytest

import saragossa_b200 as sg
from helpers import u4_reference as ref

# How far a group of 32 output channels may be off, in the 2-norm. A row's share is its weight times (code * step + bias), the two
# parts summed on their own; B = the root of the sum over the rows of (weight * (|code * step| + |bias|))^2.
#  * A weight is off by what its score is off: 1e-5 for sums of the query's products as in helpers/u4_reference.py (the
#    roundings of different rows are independent: B, and the sum of all weights moves the result by as much of itself). Beside
#    that the row's power of two 2^e joins the score, which f32 then holds at the size of |e| + |score| < 128: three roundings or
#    truncations of 2^-18 each (half a step of 2^-17), times ln 2 of a weight: 3 * 2^-17 * 0.7 is twice that.
REL = 1e-5 + 3 * 2.0 ** -17 * 0.7
#  * A weight times a group's step goes to the products as two fp16 numbers, off by at most 2^-23 (half a unit of 2^-24 for the
#    lower number, as much for its remainder and 2^-24 for the weight's own lower number times a step below 2), with the
#    largest weight at 2^9 at least and a row's 2^e down to 2^-4 of what the weights are scaled for: 2^-23 / 2^(9-4) of 2^e and of
#    the largest weight, for every code.
CODES = 2.0 ** -28


@pytest.fixture(scope="module")
def state():
    st = sg.DecodeResidentState(0)
    yield st
    assert st.device_status() == 0
    st.close()


def by_group(got, q, k, raw_v, kv_heads, start=0, sinks=0):
    """The worst of every group's error in units of what it may be. raw_v: V as it was written, from row 0 on."""
    q_heads, hd = q.shape
    n, gqa, groups = len(k), q_heads // kv_heads, hd // 32
    code, step, bias = ref.quantize(raw_v, 0, hd)
    v = ref.stored(raw_v, 0, hd, 3)
    want, bound = ref.attention(q, k, v, kv_heads, start, sinks)
    got = got.reshape(want.shape).astype(np.float64)
    assert np.isfinite(got).all()
    rows = np.arange(n)
    seen = (rows < sinks) | (rows >= start)
    code = code.astype(np.float64).reshape(n, kv_heads, groups, 32)[seen]
    step, bias = (np.abs(x).reshape(n, kv_heads, groups, 1)[seen] for x in (step, bias))
    size = code * step + bias
    unit = code * np.exp2(np.floor(np.log2(step.max(2, keepdims=True))))       # 2^e is at most the widest group's step
    kk = k.reshape(n, kv_heads, hd)[seen]
    worst = 0.0
    for h in range(q_heads):
        s = kk[:, h // gqa] @ q[h].astype(np.float64) / np.sqrt(hd)
        p = np.exp(s - s.max())
        p /= p.sum()
        heads = size[:, h // gqa], unit[:, h // gqa]
        for g in range(groups):
            part = slice(32 * g, 32 * g + 32)
            err = got[h, part] - want[h, part]
            m, u = (x[:, g] for x in heads)
            may = REL * (np.sqrt(np.sum((p[:, None] * m) ** 2)) + np.linalg.norm(want[h, part])) + CODES * p.max() * np.sqrt(np.sum(u ** 2))
            most = bound[h, 0] * m.max() / size[:, h // gqa].max() + CODES * p.max() * u.sum(0).max()
            worst = max(worst, np.linalg.norm(err) / max(may, 1e-300), np.abs(err).max() / max(most, 1e-300))
    return worst


def _make(state, n, q_heads, kv_heads, hd, change, seed=1, cap=None):
    rng = np.random.default_rng(100 * hd + n + seed)
    k, v = rng.standard_normal((2, n, kv_heads, hd)).astype(np.float32)
    change(v)
    k, v = k.reshape(n, -1), v.reshape(n, -1)
    kv = state.full_attention(cap or n, q_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=9)
    kv.seed(k, v, n)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    return kv, q, ref.stored(k, 0, hd, 3), v


HEADS = [(8, 2), (16, 2)]           # four and eight query heads per KV head


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("size", [1e4, 1e6, 1e8, 1e10, 1e18, 1e-4, 1e-10])
@pytest.mark.parametrize("rows", ["one", "first page", "some", "half", "last"])
def test_rows_with_one_wide_or_narrow_group(state, hd, q_heads, kv_heads, size, rows):
    """A value of the first group (the whole group where it gets smaller) of some rows is scaled."""
    n = 600
    which = {"one": [3], "first page": range(16), "some": range(5, n, 37), "half": range(0, n, 2), "last": [n - 1]}[rows]

    def change(v):
        v[list(which), :, :32 if size < 1 else 1] *= np.float32(size)
    kv, q, k, v = _make(state, n, q_heads, kv_heads, hd, change)
    for start in (0, 4, 300):
        assert by_group(kv.attention_decode_windowed(q, start), q, k, v, kv_heads, start) <= 1.0, start
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("q_heads,kv_heads", HEADS)
@pytest.mark.parametrize("sizes", [[1e18, 1.0], [1e-12, 1.0], [1e12, 1e-8, 1.0], [1e6, 1e3, 1.0, 1e-3, 1e-6], [0.0, 1.0], [1.0] * 99 + [0.0]])
def test_rows_whose_other_groups_are_empty(state, hd, q_heads, kv_heads, sizes):
    """Row r has values of size sizes[r % m] in group r % m only, zeros elsewhere: in every group other rows count."""
    n, m = 500, len(sizes)

    def change(v):
        for r in range(n):
            keep = v[r, :, 32 * (r % m % (hd // 32)):][:, :32].copy()
            v[r] = 0.0
            v[r, :, 32 * (r % m % (hd // 32)):][:, :32] = keep * np.float32(sizes[r % m])
    kv, q, k, v = _make(state, n, q_heads, kv_heads, hd, change)
    assert by_group(kv.attention_decode(q), q, k, v, kv_heads) <= 1.0
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("narrow", [2.0 ** -8, 2.0 ** -12, 2.0 ** -15, 2.0 ** -17, 0.0])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_a_group_that_is_narrow_in_every_row(state, hd, narrow):
    def change(v):
        v[:, :, 32:64] *= np.float32(narrow)
    kv, q, k, v = _make(state, 900, 8, 2, hd, change)
    assert by_group(kv.attention_decode(q * np.float32(3.0)), q * np.float32(3.0), k, v, 2) <= 1.0
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [128, 256])
def test_wide_rows_in_sinks_windows_splits_and_steps(state, hd):
    """The wide row as a sink, just outside and inside a window, appended by the step, and in every merge."""
    n, q_heads, kv_heads = 3000, 16, 2

    def change(v):
        v[[2, 1000, 2990], :, 5] = np.float32(1e10)
    kv, q, k, v = _make(state, n, q_heads, kv_heads, hd, change, cap=n + 3)
    for sinks, start in ((0, 0), (4, 2000), (2, 999), (3, 1001), (0, 2991), (1, 2990)):
        kv.set_attention_sinks(sinks)
        assert by_group(kv.attention_decode_windowed(q, start), q, k, v, kv_heads, start, sinks) <= 1.0, (sinks, start)
    kv.set_attention_sinks(0)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    kv.encode_attention_decode_noalloc(d_q, d_out)
    state.sync()
    assert by_group(d_out.download(), q, k, v, kv_heads) <= 1.0
    rng = np.random.default_rng(6)
    for step in range(3):
        new = rng.standard_normal((2, kv_heads, hd)).astype(np.float32)
        if step == 1:
            new[1, :, 40] = np.float32(-1e14)
        d_k, d_v = state.upload(new[0]), state.upload(new[1])
        kv.encode_append_attention(d_k, d_v, d_q, d_out)
        state.sync()
        k = np.concatenate([k, ref.stored(new[0].reshape(1, -1), n + step, hd, 3)])
        v = np.concatenate([v, new[1].reshape(1, -1)])
        assert by_group(d_out.download(), q, k, v, kv_heads) <= 1.0, step
    batch = sg.Batch(state, [kv])
    for splits in (1, 2, 5, 8, 13, 40):
        batch.set_splits(splits)
        batch.enqueue_attention(d_q, d_out)
        state.sync()
        assert by_group(d_out.download(), q, k, v, kv_heads) <= 1.0, splits
    batch.close()
    kv.close()

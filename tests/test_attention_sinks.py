"""Windowed attention whose first rows stay visible (attention sinks), over every page type, and the release of the pages
between sinks and window. Against the plain 64-bit restatement in helpers/u4_reference.py."""
import numpy as np
import pytest

import saragossa_b200 as sg
from helpers import u4_reference as ref

U8_REL = 2e-3      # the u8 kernel weighs its codes with fp16 products: 2^-11 each, and f16 scales: 2^-11 again


# ---- the host's bookkeeping, without a device -------------------------------------------------------------
def _host_seq(rows, pages=16):
    pool = sg.PagePool(None, 1, 1, 32, sg.KV_F32, pages, 1, 16 * pages)
    seq = pool.sequence(16 * pages)
    seq.reserve(rows)
    return pool, seq


def _held(seq):
    return [i for i, p in enumerate(seq.block_table()) if p >= 0]


@pytest.mark.parametrize("calls,held", [
    ([(4, 100)], [0, 6, 7]),                       # sinks end inside page 0, the window starts inside page 6
    ([(16, 96)], [0, 6, 7]),
    ([(17, 96)], [0, 1, 6, 7]),
    ([(4, 100), (4, 120)], [0, 7]),                # the window moves on
    ([(40, 100), (4, 100)], [0, 6, 7]),            # fewer sinks
    ([(4, 100), (0, 100)], [6, 7]),                # none
    ([(0, 40), (4, 70)], [4, 5, 6, 7]),            # already gone
    ([(4, 15)], list(range(8))),                   # no page lies wholly inside
    ([(100, 20)], list(range(8))),
    ([(4, 100), (0, 0), (90, 10)], [0, 6, 7]),
    ([(0, 1000)], []),
    ([(2**63 - 1, 100), (0, 2**63 - 1)], []),      # the first names no page
])
def test_release_between(calls, held):
    pool, seq = _host_seq(128)
    free = pool.free_pages
    for c in calls:
        seq.release_between(*c)
    assert _held(seq) == held
    assert pool.free_pages == free + 8 - len(held)
    seq.reset()
    assert pool.free_pages == pool.num_pages
    seq.close()
    pool.close()


def test_release_refusals():
    pool, seq = _host_seq(128)
    for bad in ((-1, 20), (0, -5)):
        with pytest.raises(sg.InferError) as e:
            seq.release_between(*bad)
        assert e.value.kind == "Dimension"
    seq.release_between(32, 64)
    for bad in ((80, 120), (0, 16)):               # rows would stay between the two ranges
        with pytest.raises(sg.InferError) as e:
            seq.release_between(*bad)
        assert e.value.kind == "Dimension"
    assert _held(seq) == [0, 1, 4, 5, 6, 7]
    seq.release_before(64)
    assert _held(seq) == [4, 5, 6, 7]
    kv = seq.layer(0, 1)
    assert kv.attention_sinks() == 0
    kv.set_attention_sinks(5)
    assert kv.attention_sinks() == 5
    with pytest.raises(sg.InferError) as e:
        kv.set_attention_sinks(-1)
    assert e.value.kind == "Dimension" and kv.attention_sinks() == 5
    seq.close()
    pool.close()


# ---- GPU ------------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def state():
    st = sg.DecodeResidentState(0)
    yield st
    assert st.device_status() == 0
    st.close()


DTYPES = [sg.KV_F32, sg.KV_BF16, sg.KV_U8G32, sg.KV_U4G32]


def _fill(kv, n, kv_heads, hd, seed):
    rng = np.random.default_rng(seed)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    kv.seed(k, v, n)
    return k, v


def _held_rows(kv):
    return [x.astype(np.float64) for x in kv.gather_rows_f32()]


def _close(got, want, dtype):
    if dtype != sg.KV_U8G32:
        return ref.close(got, want)[0]
    return np.linalg.norm(got.reshape(want[0].shape) - want[0]) <= U8_REL * np.linalg.norm(want[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(32, 4, 128), (6, 2, 128), (16, 2, 256), (4, 2, 64), (12, 1, 128)])
@pytest.mark.parametrize("n", [1, 18, 33, 200, 1500])
def test_windows_with_sinks(state, dtype, q_heads, kv_heads, hd, n):
    kv = state.full_attention(n, q_heads, kv_heads, hd, dtype, shuffled_seed=2)
    _fill(kv, n, kv_heads, hd, n)
    k, v = _held_rows(kv)
    q = np.random.default_rng(n + 1).standard_normal((q_heads, hd)).astype(np.float32)
    for start in sorted({0, 1, 15, 16, 17, 40, n // 2, n - 16, n - 1}):
        if not 0 <= start < n:
            continue
        for sinks in (0, 1, 4, 16, 21, 10 ** 12):
            kv.set_attention_sinks(sinks)
            got = kv.attention_decode_windowed(q, start)
            assert _close(got, ref.attention(q, k, v, kv_heads, start, sinks), dtype), (start, sinks)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_both_kernels_and_no_allocations(state, dtype):
    n, q_heads, kv_heads, hd = 700, 16, 2, 128
    kv = state.full_attention(n, q_heads, kv_heads, hd, dtype, shuffled_seed=2)
    _fill(kv, n, kv_heads, hd, 5)
    k, v = _held_rows(kv)
    q = np.random.default_rng(6).standard_normal((q_heads, hd)).astype(np.float32)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    kv.set_attention_sinks(20)
    want = ref.attention(q, k, v, kv_heads, 403, 20)
    for which in (1, 2) if dtype != sg.KV_F32 else (1,):
        kv.set_attention_kernel(which)
        assert _close(kv.attention_decode_windowed(q, 403), want, dtype), which
    kv.encode_attention_decode_noalloc(d_q, d_out, 403)
    state.sync()
    assert _close(d_out.download(), want, dtype)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_masked_rows_may_hold_anything(state, dtype):
    """NaN and infinities between the sinks and the window, and behind the last row, inside pages that are read."""
    n, q_heads, kv_heads, hd, sinks, window = 90, 8, 2, 128, 5, 30
    rng = np.random.default_rng(8)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    kv = state.full_attention(112, q_heads, kv_heads, hd, dtype)
    kv.seed(k, v, n)
    clean = _held_rows(kv)
    for x in (k, v):
        x[sinks:n - window] = np.nan
        x[sinks + 1:n - window:2] = np.inf
    bad = np.full((22, kv_heads * hd), np.nan, np.float32)
    kv.seed(np.concatenate([k, bad]), np.concatenate([v, bad]), 112)
    kv.truncate(n)
    kv.set_attention_sinks(sinks)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    want = ref.attention(q, *clean, kv_heads, n - window, sinks)
    if dtype == sg.KV_U8G32:
        # (a u8 row of NaN is stored with codes of zero and a bias that is not a number only by chance: compare finite)
        assert np.isfinite(kv.attention_decode_windowed(q, n - window)).all()
    else:
        assert _close(kv.attention_decode_windowed(q, n - window), want, dtype)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [sg.KV_F32, sg.KV_BF16, sg.KV_U4G32])
@pytest.mark.parametrize("hd", [128, 256])
def test_streaming_with_released_pages(state, dtype, hd):
    """Two sequences decode far past their window as one batch; the pages between sinks and window go back to the pool, and
    the results are those of the rows that are left. Then a captured step does the same."""
    q_heads, kv_heads, sinks, window, tokens = 8, 2, 6, 50, 130
    kv_dim = kv_heads * hd
    pool = state.pool(1, kv_heads, hd, dtype, 16, 2, 512)
    pool.shuffle_free_list(3)
    seqs = [pool.sequence(512) for _ in range(2)]
    kvs = [s.layer(0, q_heads) for s in seqs]
    for kv in kvs:
        kv.set_attention_sinks(sinks)
    rng = np.random.default_rng(hd)
    rows = [rng.standard_normal((2, 400, kv_dim)).astype(np.float32) for _ in kvs]
    q = rng.standard_normal((tokens, 2, q_heads, hd)).astype(np.float32)
    lens = [3, 40]
    for kv, r, n in zip(kvs, rows, lens):
        kv.seed(r[0, :n], r[1, :n], n)
    batch = sg.Batch(state, kvs)
    d_k, d_v, d_q, d_out = (state.alloc(2 * 4 * m) for m in (kv_dim, kv_dim, q_heads * hd, q_heads * hd))
    most = 0
    for t in range(tokens):
        now = [n + t for n in lens]
        d_k.upload(np.stack([r[0, n] for r, n in zip(rows, now)]))
        d_v.upload(np.stack([r[1, n] for r, n in zip(rows, now)]))
        d_q.upload(q[t])
        batch.enqueue_step(d_k, d_v, d_q, d_out, sliding_window=window)
        state.sync()
        got = d_out.download().reshape(2, q_heads, hd)
        for i in range(2):
            n = now[i] + 1
            start = max(0, n - window)
            held = [ref.stored(x[:n], 0, hd, dtype) for x in rows[i]]
            assert ref.close(got[i], ref.attention(q[t, i], *held, kv_heads, start, sinks))[0], (t, i)
            seqs[i].release_between(sinks, max(0, n - window + 1))
        most = max(most, pool.num_pages - pool.free_pages)
    assert most <= 2 * 6                         # a page of sinks, and a window that may touch five
    with pytest.raises(sg.InferError):           # a wider window, or more sinks, reach rows that are gone
        batch.enqueue_attention(d_q, d_out, window + 40)
    for kv in kvs:
        kv.set_attention_sinks(17)
    with pytest.raises(sg.InferError) as e:
        batch.enqueue_attention(d_q, d_out, window)
    assert e.value.kind == "Dimension"
    with pytest.raises(sg.InferError):
        kvs[1].gather_rows_f32(0, 20)
    assert np.array_equal(kvs[1].gather_rows_f32(0, sinks)[0], ref.stored(rows[1][0, :sinks], 0, hd, dtype).astype(np.float32))
    kvs[0].set_attention_sinks(6)
    with pytest.raises(sg.InferError) as e:      # members differ
        batch.enqueue_attention(d_q, d_out, window)
    assert e.value.kind == "Config"
    for x in (batch, *seqs, pool):
        x.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_step_with_sinks(state, dtype):
    """A step of a windowed layer with sinks and a layer without a window, captured and replayed past the point where the
    window leaves the first page."""
    q_heads, kv_heads, hd, n, tokens = 8, 2, 128, 20, 40
    kv_dim = kv_heads * hd
    pool = state.pool(2, kv_heads, hd, dtype, 8, 1, 128)
    seq = pool.sequence(128)
    kvs = [seq.layer(layer, q_heads) for layer in range(2)]
    rng = np.random.default_rng(4)
    start = rng.standard_normal((2, 2, n, kv_dim)).astype(np.float32)
    for kv, r in zip(kvs, start):
        kv.set_attention_sinks(3)
        kv.seed(r[0], r[1], n)
    batches = [sg.Batch(state, [kv]) for kv in kvs]
    step = sg.Step(state, batches)
    d_k, d_v, d_q, d_out = (state.alloc(2 * 4 * m) for m in (kv_dim, kv_dim, q_heads * hd, q_heads * hd))
    step.capture(d_k, d_v, d_q, d_out, sliding_windows=[25, 0])
    for t in range(tokens):
        d_k.upload(rng.standard_normal((2, kv_dim)).astype(np.float32))
        d_v.upload(rng.standard_normal((2, kv_dim)).astype(np.float32))
        q = rng.standard_normal((2, q_heads, hd)).astype(np.float32)
        d_q.upload(q)
        step.replay()
        state.sync()
        got = d_out.download().reshape(2, q_heads, hd)
        for layer in range(2):
            k, v = _held_rows(kvs[layer])
            assert len(k) == n + t + 1
            first = max(0, len(k) - 25) if layer == 0 else 0
            assert _close(got[layer], ref.attention(q[layer], k, v, kv_heads, first, 3), dtype), (t, layer)
    step.close()
    for x in (*batches, seq, pool):
        x.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("splits", [0, 1, 2, 7, 14, 16])
def test_uneven_batch_with_sinks(state, dtype, splits):
    q_heads, kv_heads, hd, window, sinks = 16, 2, 128, 600, 37
    lens = [2500, 3, 601, 640, 36, 1200]
    pool = state.pool(1, kv_heads, hd, dtype, sum((n + 15) // 16 for n in lens), len(lens), max(lens))
    pool.shuffle_free_list(4)
    seqs = [pool.sequence(n) for n in lens]
    kvs = [s.layer(0, q_heads) for s in seqs]
    q = np.random.default_rng(2).standard_normal((len(lens), q_heads, hd)).astype(np.float32)
    want = []
    for i, (kv, n) in enumerate(zip(kvs, lens)):
        kv.set_attention_sinks(sinks)
        _fill(kv, n, kv_heads, hd, i)
        want.append(ref.attention(q[i], *_held_rows(kv), kv_heads, max(0, n - window), sinks))
    batch = sg.Batch(state, kvs)
    batch.set_splits(splits)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    d_out.upload(np.full(q.size, np.nan, np.float32))
    batch.enqueue_attention(d_q, d_out, sliding_window=window)
    state.sync()
    got = d_out.download().reshape(q.shape)
    for i in range(len(lens)):
        assert _close(got[i], want[i], dtype), (splits, i)
    for x in (batch, *seqs, pool):
        x.close()


class _At:
    """A device address that is not a multiple of 16."""

    def __init__(self, state, array):
        self.buf = state.alloc(array.nbytes + 16)
        self.ptr, self.shape, self.state = self.buf.ptr + 4, array.shape, state
        self.base = np.zeros(array.size + 4, np.float32)
        self.base[1:1 + array.size] = array.ravel()
        self.buf.upload(self.base)

    def download(self):
        return self.buf.download()[1:1 + int(np.prod(self.shape))].reshape(self.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [sg.KV_U4G32, sg.KV_BF16, sg.KV_U8G32])
def test_addresses_between_the_vector_boundaries(state, dtype):
    n, q_heads, kv_heads, hd, window, sinks = 90, 8, 2, 128, 40, 6
    rng = np.random.default_rng(3)
    k, v = rng.standard_normal((2, n + 1, kv_heads * hd)).astype(np.float32)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    twin = state.full_attention(n + 8, q_heads, kv_heads, hd, dtype)     # the same rows from aligned addresses
    twin.seed(k, v, n + 1)
    held = [x.reshape(n + 1, -1).astype(np.float64) for x in twin.gather_rows_f32(0, n + 1)]
    twin.close()
    kv = state.full_attention(n + 8, q_heads, kv_heads, hd, dtype, shuffled_seed=4)
    kv.set_attention_sinks(sinks)
    d_out = _At(state, np.zeros_like(q))
    kv.encode_append_rows(_At(state, k[:n]), _At(state, v[:n]), n)
    state.sync()
    assert np.array_equal(kv.gather_rows_f32(0, n)[0], held[0][:n].astype(np.float32))
    for call in (kv.encode_attention_decode_windowed, kv.encode_attention_decode_noalloc):
        call(_At(state, q), d_out, n - window)
        state.sync()
        assert ref.close(d_out.download(), ref.attention(q, held[0][:n], held[1][:n], kv_heads, n - window, sinks))[0]
    kv.encode_append_attention(_At(state, k[n:]), _At(state, v[n:]), _At(state, q), d_out, window)
    state.sync()
    assert ref.close(d_out.download(), ref.attention(q, *held, kv_heads, n + 1 - window, sinks))[0]
    assert np.array_equal(kv.gather_rows_f32(n, 1)[1], held[1][n:].astype(np.float32))
    kv.close()


@pytest.mark.gpu
def test_uneven_batch_with_the_widest_window(state):
    lens, hd = (600, 9), 64
    pool = state.pool(1, 1, hd, sg.KV_U4G32, 64, 2, 640)
    rng = np.random.default_rng(8)
    seqs = [pool.sequence(640) for _ in lens]
    kvs, want, q = [s.layer(0, 2) for s in seqs], [], rng.standard_normal((2, 2, hd)).astype(np.float32)
    for i, n in enumerate(lens):
        k, v = rng.standard_normal((2, n, hd)).astype(np.float32)
        kvs[i].seed(k, v, n)
        kvs[i].set_attention_sinks(2**63 - 1)
        want.append(ref.attention(q[i], *(ref.stored(x, 0, hd, sg.KV_U4G32) for x in (k, v)), 1))
    batch = sg.Batch(state, kvs)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    for window in (2**63 - 1, 1):                 # every row is in the window, or every row is a sink
        batch.enqueue_attention(d_q, d_out, window)
        state.sync()
        got = d_out.download().reshape(q.shape)
        assert all(ref.close(got[i], want[i])[0] for i in range(2))
    twice = sg.Batch(state, [kvs[0], kvs[0]])     # one sequence, two queries
    twice.enqueue_attention(d_q, d_out, 0)
    state.sync()
    assert ref.close(d_out.download().reshape(q.shape)[0], want[0])[0]
    with pytest.raises(sg.InferError) as e:       # but not two lengths
        twice.enqueue_truncate([20, 30])
    assert e.value.kind == "Dimension" and kvs[0].len() == 600
    twice.enqueue_truncate([20, 20])
    assert kvs[0].len() == 20
    for x in (twice, batch, *seqs, pool):
        x.close()

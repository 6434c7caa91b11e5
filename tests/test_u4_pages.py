"""Pages of 4-bit codes: the format on the CPU, and through the C ABI on the GPU the quantiser as rows are
written, the read-back and decode attention, against a plain 64-bit restatement (helpers/u4_reference.py)."""
import os
import subprocess
from fractions import Fraction

import numpy as np
import pytest

import saragossa_b200 as sg
from helpers import u4_reference as ref

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---- CPU: the restatement against exact fractions, the byte order, the host's bookkeeping ----------------
def _nearest_even(x: Fraction) -> int:
    low = x.numerator // x.denominator
    rest = x - low
    return low + (rest > Fraction(1, 2) or (rest == Fraction(1, 2) and low % 2 == 1))


def _bf16_fraction(x: Fraction) -> Fraction:
    if x == 0:
        return Fraction(0)
    sign, x = (-1 if x < 0 else 1), abs(x)
    e = 0
    while x >= 2 ** (e + 1):
        e += 1
    while x < Fraction(2) ** e:
        e -= 1
    unit = Fraction(2) ** (e - 7)
    return sign * _nearest_even(x / unit) * unit


def _quantize_fractions(group_rows, odd):
    """One head row (list of groups of floats) in exact arithmetic."""
    y = [[(-1 if odd else 1) * Fraction(float(x)) for x in g] for g in group_rows]
    bias = [_bf16_fraction(min(g)) for g in y]
    raw = [(max(g) - b) / 15 for g, b in zip(y, bias)]
    top, e = max([*raw, Fraction(1, 2 ** 40)]), -40
    while Fraction(2) ** (e + 1) <= top:
        e += 1
    step = [_bf16_fraction(max(r, Fraction(1, 2 ** 40), Fraction(2) ** (e - 16))) for r in raw]
    code = [[min(15, max(0, _nearest_even((x - b) / s))) for x in g] for g, b, s in zip(y, bias, step)]
    sign = -1 if odd else 1
    return code, [sign * s for s in step], [sign * b for b in bias]


def border_rows(n, kv_dim, seed):
    """Rows whose values sit on and next to the borders of the quantiser: halves of a step, powers of two, steps next to
    the middle of two bf16 values, constants, zeros, tiny and huge values, groups of very different ranges in a row."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((n, kv_dim)).astype(np.float32)
    steps = np.array([2.0 ** -7, 1.5 * 2.0 ** -7, 1.375 * 2.0 ** -3, 3.0, 0.0087890625, 1 + 2.0 ** -7], np.float32)
    eps = np.array([0, 2.0 ** -23, -2.0 ** -23, 2.0 ** -21, -2.0 ** -20, 1e-4, -1e-4], np.float32)
    for r in range(n):
        for g in range(kv_dim // 32):
            kind = rng.integers(0, 9)
            part = slice(g * 32, g * 32 + 32)
            if kind == 0:
                s = steps[rng.integers(len(steps))]
                c = rng.integers(0, 15, 32).astype(np.float32) + np.float32(0.5)
                row = (c * s * (1 + eps[rng.integers(0, len(eps), 32)])).astype(np.float32)
                row[0], row[1] = 0.0, 15 * s
                x[r, part] = row * (1 if r % 2 == 0 else -1)
            elif kind == 1:
                x[r, part] = np.float32(rng.standard_normal() * 10.0 ** rng.integers(-6, 6))
            elif kind == 2:
                x[r, part] = 0.0
            elif kind == 3:
                x[r, part] *= np.float32(2.0 ** int(rng.integers(-60, 60)))
            elif kind == 4:
                x[r, part] = np.float32(1000.0) + x[r, part] * np.float32(0.01)
            elif kind == 5:
                # the range is 15 times the middle between two bf16 values, a little above or below
                mid = np.float32((128 + rng.integers(0, 128) + 0.5) * 2.0 ** -8)
                x[r, part] = rng.random(32).astype(np.float32) * mid
                x[r, g * 32] = 0.0
                x[r, g * 32 + 1] = np.float32(15.0) * mid * (1 + eps[rng.integers(0, 3)])
                x[r, part] *= np.float32(1 if r % 2 == 0 else -1)
    return x


def test_reference_quantizer_is_exact():
    x = border_rows(24, 128, 3)
    code, scale, bias = ref.quantize(x, 0, 64)
    for r in range(len(x)):
        for head in range(2):
            want = _quantize_fractions(x[r, head * 64:head * 64 + 64].reshape(2, 32), r % 2)
            at = slice(head * 2, head * 2 + 2)
            assert code[r, head * 64:head * 64 + 64].reshape(2, 32).tolist() == want[0], r
            assert [Fraction(float(s)) for s in scale[r, at]] == want[1] and [Fraction(float(b)) for b in bias[r, at]] == want[2], r


def test_byte_order_of_a_tile_is_a_bijection(tmp_path):
    """Every (row, dim) has its own nibble, every (row, group) its own step and bias, all inside the tile."""
    src = tmp_path / "order.cpp"
    src.write_text(r'''
#include <cstdio>
#include <vector>
#include "layout.h"
using namespace sgk;
int main() {
  for (int hd = 32; hd <= 512; hd += 32) {
    const int bytes = (int)tile_bytes(KV_U4G32, hd), codes = PAGE_TOKENS * hd / 2;
    if (bytes % 16 || tile_code_bytes(KV_U4G32, hd) != codes) return 1;
    for (int v = 0; v < 2; ++v) {
      std::vector<int> nibble(2 * codes), byte(bytes);
      for (int r = 0; r < PAGE_TOKENS; ++r)
        for (int d = 0; d < hd; ++d) {
          const int at = v ? u4_v_byte(r, d, hd) : u4_k_byte(r, d, hd);
          if (at < 0 || at >= codes || nibble[2 * at + u4_nibble(d)]++) return 2;
        }
      for (int r = 0; r < PAGE_TOKENS; ++r)
        for (int g = 0; g < hd / QGROUP; ++g)
          for (int at : {u4_step_offset(v, r, g, hd), u4_bias_offset(r, g, hd)})
            if (at < codes || at + 2 > bytes || at % 2 || byte[at]++) return 3;
      for (int r = 8 * v; r < 8 * v + 8; ++r) {
        const int at = u4_pow_offset(r, hd);
        if (at < codes || at + 2 > bytes || byte[at]++) return 4;
      }
    }
  }
  return 0;
}
''')
    exe = tmp_path / "order"
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(ROOT, "saragossa_b200", "csrc"), "-o", str(exe), str(src)])
    assert subprocess.run([str(exe)]).returncode == 0


def test_u4_pool_sizes_and_refusals_without_a_device():
    pool = sg.PagePool(None, 2, 4, 128, sg.KV_U4G32, 8, 1, 64)
    assert pool.page_bytes == 2 * 4 * 2 * (128 * 10 + 16)
    pool.close()
    for hd, dtype in ((48, sg.KV_U4G32), (544, sg.KV_U4G32), (128, 4), (128, -1)):
        with pytest.raises(sg.InferError):
            sg.PagePool(None, 1, 1, hd, dtype, 8, 1, 64)
    with pytest.raises(sg.InferError) as e:
        sg.PagePool(None, 1, 1, 48, sg.KV_U4G32, 8, 1, 64)
    assert e.value.kind == "Config"


# ---- GPU ---------------------------------------------------------------------------------------------------
@pytest.fixture(scope="module")
def state():
    st = sg.DecodeResidentState(0)
    yield st
    assert st.device_status() == 0
    st.close()


def _check_codes(kv, x, y, hd, row0=0):
    got = kv.gather_rows_u4(row0, len(x))
    for (code, scale, bias), rows in ((got[:3], x), (got[3:], y)):
        want = ref.quantize(rows, row0, hd)
        assert np.array_equal(code, want[0])
        ok = np.isfinite(want[1])
        assert np.array_equal(scale[ok], ref.bf16_bits(want[1])[ok]) and np.array_equal(bias[ok], ref.bf16_bits(want[2])[ok])
    f32 = kv.gather_rows_f32(row0, len(x))
    for g, rows in zip(f32, (x, y)):
        assert np.array_equal(g, ref.read_back(rows, row0, hd), equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,hd", [(1, 32), (3, 64), (2, 96), (4, 128), (1, 160), (2, 256), (1, 384), (1, 512)])
def test_rows_are_quantised_as_they_are_written(state, kv_heads, hd):
    """Bit for bit, whichever append wrote a row: seed, several rows (from inside a page), one row."""
    n, kv_dim = 16 * 6 + 5, kv_heads * hd
    k, v = border_rows(n, kv_dim, hd), border_rows(n, kv_dim, hd + 1)
    kv = state.full_attention(n + 3, kv_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=3)
    kv.seed(k[:37], v[:37], 37)
    kv.append_batch(k[37:40], v[37:40])
    kv.append_row(k[40], v[40])
    kv.append_batch(k[41:], v[41:])
    _check_codes(kv, k, v, hd)
    _check_codes(kv, k[13:50], v[13:50], hd, 13)
    # a cursor moved back never clears memory, and the rows behind it are written over one by one
    kv.truncate(20)
    kv.append_row(k[0], v[1])
    assert np.array_equal(kv.gather_rows_f32(20, 1)[0], ref.read_back(k[:1], 20, hd))
    kv.truncate(n)
    assert np.array_equal(kv.gather_rows_f32(21, n - 21)[1], ref.read_back(v[21:], 21, hd), equal_nan=True)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n", [(128, 1), (128, 40), (64, 5), (256, 33)])
def test_groups_that_are_not_finite_read_back_as_nan(state, hd, n):
    rng = np.random.default_rng(n)
    k, v = rng.standard_normal((2, n, 2 * hd)).astype(np.float32)
    k[0, 3], v[0, hd + 5], v[n - 1, 0] = np.nan, np.inf, -np.inf
    k[n - 1, hd:hd + 32] = np.linspace(-3.3e38, 3.3e38, 32)      # the range overflows
    kv = state.full_attention(n, 2, 2, hd, sg.KV_U4G32)
    kv.seed(k, v, n)
    _check_codes(kv, k, v, hd)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n,interleaved", [(128, 1, False), (128, 70, False), (256, 21, True), (64, 17, False), (96, 6, False)])
def test_rope_append_quantises_the_rotated_rows(state, hd, n, interleaved):
    """The rows an f32 cache holds after the same call, quantised."""
    kv_heads, rng = 2, np.random.default_rng(hd + n)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    w = state.upload(rng.standard_normal(hd).astype(np.float32))
    d_k, d_v = state.upload(k), state.upload(v)
    rope = sg.make_rope(hd // 2, 1e6, interleaved=interleaved)
    kvs = [state.full_attention(n + 30, kv_heads, kv_heads, hd, dt) for dt in (sg.KV_F32, sg.KV_U4G32)]
    for kv in kvs:
        kv.seed(np.zeros((9, kv_heads * hd)), np.zeros((9, kv_heads * hd)), 9)
        if n == 1:
            kv.encode_rope_append(d_k, d_v, w, rope)
        else:
            kv.encode_rope_append_rows(d_k, d_v, n, w, rope)
    state.sync()
    fk, fv = kvs[0].gather_rows_f32(9, n)
    _check_codes(kvs[1], fk, fv, hd, 9)
    for kv in kvs:
        kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [sg.KV_F32, sg.KV_BF16, sg.KV_U8G32, sg.KV_U4G32])
def test_device_read_back_is_the_host_one(state, dtype):
    n, kv_dim = 83, 3 * 64
    k, v = np.random.default_rng(1).standard_normal((2, n, kv_dim)).astype(np.float32)
    kv = state.full_attention(n, 3, 3, 64, dtype, shuffled_seed=2)
    kv.seed(k, v, n)
    d_k, d_v = state.alloc(n * kv_dim * 4), state.alloc(n * kv_dim * 4)
    for row0, m in ((0, n), (17, 1), (5, 44), (n - 1, 1), (n, 0)):
        d_k.upload(np.full(n * kv_dim, 7.0, np.float32))
        d_v.upload(np.full(n * kv_dim, 7.0, np.float32))
        kv.encode_gather_rows_f32(d_k, d_v, row0, m)
        state.sync()
        want = kv.gather_rows_f32(row0, m) if m else (np.empty((0, kv_dim)),) * 2
        for d, w in zip((d_k, d_v), want):
            got = d.download().reshape(n, kv_dim)
            assert np.array_equal(got[:m], w) and np.all(got[m:] == 7.0)     # rows behind the last one as they were
    for row0, m in ((-1, 1), (0, n + 1), (n, 1), (2, -1)):
        with pytest.raises(sg.InferError) as e:
            kv.encode_gather_rows_f32(d_k, d_v, row0, m)
        assert e.value.kind == "Dimension"
    if dtype != sg.KV_U4G32:
        with pytest.raises(sg.InferError):
            kv.gather_rows_u4()
    else:
        with pytest.raises(sg.InferError):
            kv.gather_rows()
        with pytest.raises(sg.InferError):
            kv.gather_rows_u8()
    kv.close()


def filled(state, n, q_heads, kv_heads, hd, dtype=sg.KV_U4G32, seed=0, cap=None, outliers=True):
    """A KV state with n rows, and what it holds in f64."""
    rng = np.random.default_rng(1000 * seed + n + hd)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    k = k * (0.4 + rng.random(kv_heads * hd)).astype(np.float32) + (0.7 * rng.standard_normal(kv_heads * hd)).astype(np.float32)
    if outliers and n > 40:
        k[5] *= np.float32(4.0)
        v[n // 2] *= np.float32(300.0)        # ranges three orders of magnitude apart, in one row and across rows
        v[n // 3, :32] *= np.float32(1e-4)
        v[7] *= np.float32(1e-6)
    kv = state.full_attention(cap or n + 4, q_heads, kv_heads, hd, dtype, shuffled_seed=9)
    kv.seed(k, v, n)
    return kv, ref.stored(k, 0, hd, dtype), ref.stored(v, 0, hd, dtype)


SHAPES = [(1, 1, 128), (32, 4, 128), (8, 2, 128), (10, 2, 128), (7, 1, 256), (16, 2, 256), (8, 2, 64), (4, 4, 96), (24, 2, 128)]


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,hd", SHAPES)
@pytest.mark.parametrize("n", [1, 2, 16, 17, 31, 130, 700, 2500])
def test_attention_over_u4_pages(state, q_heads, kv_heads, hd, n):
    kv, k, v = filled(state, n, q_heads, kv_heads, hd)
    q = np.random.default_rng(n).standard_normal((q_heads, hd)).astype(np.float32)
    for start in sorted({0, n // 2, n - 1}):
        ok, far = ref.close(kv.attention_decode_windowed(q, start), ref.attention(q, k, v, kv_heads, start))
        assert ok, (start, far)
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-20, 1e-6, 30.0, 1e4])
@pytest.mark.parametrize("hd", [128, 256])
def test_attention_over_u4_pages_takes_any_size_of_query(state, hd, scale):
    kv, k, v = filled(state, 300, 8, 2, hd, outliers=False)
    q = (np.random.default_rng(5).standard_normal((8, hd)) * scale).astype(np.float32)
    q[3] = 0.0                                                     # all rows weigh the same
    want, bound = ref.attention(q, k, v, 2)
    got = kv.attention_decode(q).reshape(want.shape)
    if scale < 100:
        assert ref.close(got, (want, bound), rel=1e-5 * max(1.0, scale))[0]       # scores, and their errors, grow with q
    else:
        assert np.isfinite(got).all() and np.all(np.abs(got - want) <= np.minimum(bound, 2 * np.abs(v).max()))
    kv.close()


@pytest.mark.gpu
def test_generic_and_tensor_core_kernel_agree(state):
    kv, k, v = filled(state, 900, 16, 2, 128)
    q = np.random.default_rng(3).standard_normal((16, 128)).astype(np.float32)
    for which in (1, 2):
        kv.set_attention_kernel(which)
        assert ref.close(kv.attention_decode(q, attn_scalar=50.0), ref.attention(q, k, v, 2, scalar=50.0))[0], which
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_rows_behind_the_last_one_do_not_matter(state, hd):
    """A page of an earlier use may hold anything behind the cursor, NaN and infinities among it."""
    n, kv_heads = 41, 2
    kv, k, v = filled(state, n, 8, kv_heads, hd, cap=64)
    bad = np.full((23, kv_heads * hd), np.nan, np.float32)
    bad[::2] = np.inf
    kv.append_batch(bad, bad)
    q = np.random.default_rng(7).standard_normal((8, hd)).astype(np.float32)
    assert np.isnan(kv.attention_decode(q)).all()
    for m in (41, 33, 17):
        kv.truncate(m)
        assert ref.close(kv.attention_decode(q), ref.attention(q, k[:m], v[:m], kv_heads))[0], m
        start = max(0, m - 20)
        assert ref.close(kv.attention_decode_windowed(q, start), ref.attention(q, k[:m], v[:m], kv_heads, start))[0], m
    kv.close()


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,hd", [(32, 4, 128), (16, 2, 256), (8, 2, 64)])
def test_fused_append_and_graph_replay(state, q_heads, kv_heads, hd):
    """Step by step over several page borders: the appended row bit for bit, the attention over it; then the same tokens
    replayed as a captured step after a rollback in stream order."""
    n, tokens, kv_dim = 30, 21, kv_heads * hd
    pool = state.pool(2, kv_heads, hd, sg.KV_U4G32, 40, 4, 128)
    pool.shuffle_free_list(1)
    rng = np.random.default_rng(hd)
    lens = [n, n + 15, 1]
    hold = {}
    seqs, kvs = [pool.sequence(128) for _ in lens], []
    for layer in range(2):
        kvs.append([])
        for s, (seq, m) in enumerate(zip(seqs, lens)):
            k, v = rng.standard_normal((2, m, kv_dim)).astype(np.float32)
            kv = seq.layer(layer, q_heads)
            kv.seed(k, v, m)
            kvs[layer].append(kv)
            hold[layer, s] = [k, v]
    batches = [sg.Batch(state, kvs[layer]) for layer in range(2)]
    step = sg.Step(state, batches)
    B = len(lens)
    new_k, new_v = rng.standard_normal((2, tokens, 2, B, kv_dim)).astype(np.float32)
    q = rng.standard_normal((tokens, 2, B, q_heads, hd)).astype(np.float32)
    d_k, d_v = state.alloc(2 * B * kv_dim * 4), state.alloc(2 * B * kv_dim * 4)
    d_q, d_out = state.alloc(2 * B * q_heads * hd * 4), state.alloc(2 * B * q_heads * hd * 4)
    for replay in (False, True):     # (a captured step keeps the split count of its first token: held to the reference, not bit for bit)
        if replay:
            for layer in range(2):
                batches[layer].enqueue_truncate(lens)
            state.sync()
            assert [kv.len() for kv in kvs[1]] == lens
            step.capture(d_k, d_v, d_q, d_out)
        for t in range(tokens):
            d_k.upload(new_k[t]), d_v.upload(new_v[t]), d_q.upload(q[t])
            if replay:
                step.replay()
            else:
                step.enqueue(d_k, d_v, d_q, d_out)
            state.sync()
            got = d_out.download().reshape(2, B, q_heads, hd)
            for layer in range(2):
                for s in range(B):
                    rows = [np.concatenate([h, x[:t + 1, layer, s]]) for h, x in zip(hold[layer, s], (new_k, new_v))]
                    want = ref.attention(q[t, layer, s], *(ref.stored(x, 0, hd, sg.KV_U4G32) for x in rows), kv_heads)
                    assert ref.close(got[layer, s], want)[0], (t, layer, s)
                    assert kvs[layer][s].len() == len(rows[0])
        for layer in range(2):
            for s in range(B):
                rows = [np.concatenate([h, x[:, layer, s]]) for h, x in zip(hold[layer, s], (new_k, new_v))]
                _check_codes(kvs[layer][s], *rows, hd)
    step.close()
    for x in (*batches, *seqs, pool):
        x.close()


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[3000, 40, 1, 900, 17], [1200] * 6, [16]])
def test_batched_attention_over_u4_pages(state, lens):
    """Even and uneven batches, and every split count that a batch can be given, agree with each sequence alone."""
    q_heads, kv_heads, hd = 16, 2, 128
    pool = state.pool(1, kv_heads, hd, sg.KV_U4G32, sum((n + 15) // 16 for n in lens), len(lens), max(lens))
    pool.shuffle_free_list(4)
    seqs = [pool.sequence(n) for n in lens]
    rng = np.random.default_rng(len(lens))
    kvs, want = [], []
    q = rng.standard_normal((len(lens), q_heads, hd)).astype(np.float32)
    for seq, n, qi in zip(seqs, lens, q):
        k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
        kv = seq.layer(0, q_heads)
        kv.seed(k, v, n)
        kvs.append(kv)
        want.append(ref.attention(qi, ref.stored(k, 0, hd, 3), ref.stored(v, 0, hd, 3), kv_heads))
    batch = sg.Batch(state, kvs)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    for splits in (0, 1, 2, 3, 5, 13, 16):
        try:
            batch.set_splits(splits)
        except sg.InferError:
            continue
        d_out.upload(np.full(q.size, np.nan, np.float32))
        batch.enqueue_attention(d_q, d_out)
        state.sync()
        got = d_out.download().reshape(q.shape)
        for i in range(len(lens)):
            assert ref.close(got[i], want[i])[0], (splits, i)
    for x in (batch, *seqs, pool):
        x.close()


@pytest.mark.gpu
def test_a_long_cache_in_every_merge(state):
    """One long sequence (many splits that merge together), solo, in two streams at once, and in the form without allocations."""
    n, q_heads, kv_heads, hd = 9000, 16, 2, 128
    kv, k, v = filled(state, n, q_heads, kv_heads, hd)
    q = np.random.default_rng(3).standard_normal((q_heads, hd)).astype(np.float32)
    want = ref.attention(q, k, v, kv_heads)
    d_q, d_out = state.upload(q), state.alloc(q.nbytes)
    assert ref.close(kv.attention_decode(q), want)[0]
    state.set_concurrent_streams(True)
    assert ref.close(kv.attention_decode(q), want)[0]
    state.set_concurrent_streams(False)
    kv.encode_attention_decode_noalloc(d_q, d_out)
    state.sync()
    assert ref.close(d_out.download(), want)[0]
    kv.close()


@pytest.mark.gpu
def test_verify_rows_and_prefix_restore_over_u4_pages(state):
    """Draft rows are serial steps, a rejected tail is dropped in stream order; a restored prefix holds the same codes."""
    q_heads, kv_heads, hd, n = 8, 2, 128, 45
    kv_dim = kv_heads * hd
    rng = np.random.default_rng(11)
    k, v = rng.standard_normal((2, 64, kv_dim)).astype(np.float32)
    q = rng.standard_normal((6, q_heads, hd)).astype(np.float32)
    pool = state.pool(1, kv_heads, hd, sg.KV_U4G32, 24, 4, 96)
    seq = pool.sequence(96)
    kv = seq.layer(0, q_heads)
    kv.seed(k[:n], v[:n], n)
    d_k, d_v, d_q, d_out = state.upload(k[n:n + 6]), state.upload(v[n:n + 6]), state.upload(q), state.alloc(q.nbytes)
    kv.encode_verify_rows(d_k, d_v, d_q, d_out, 6)
    kv.encode_truncate(n + 2)                                # four rejected
    state.sync()
    assert kv.len() == n + 2
    got = d_out.download().reshape(q.shape)
    for r in range(6):
        rows = [ref.stored(x[:n + r + 1], 0, hd, 3) for x in (k, v)]
        assert ref.close(got[r], ref.attention(q[r], *rows, kv_heads))[0], r
    with pytest.raises(sg.InferError):
        kv.encode_truncate(97)
    cache = sg.BlockAwarePrefixCache(16, 64, pool=pool)
    tokens = list(range(32))
    root = sg.BlockHash.root()
    cache.insert_chain(root, tokens, seq)
    hit = cache.match_prefix(root, tokens)
    other = pool.sequence(96)
    cache.restore(hit, other)
    okv = other.layer(0, q_heads)
    assert okv.len() == 32
    _check_codes(okv, k[:32], v[:32], hd)
    okv.append_row(k[40], v[41])
    assert np.array_equal(okv.gather_rows_f32(32, 1)[0], ref.read_back(k[40:41], 32, hd))
    _check_codes(kv, k[:n + 2], v[:n + 2], hd)
    for x in (cache, seq, other, pool):
        x.close()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("spread", [[1e18, 1.0], [1e-12, 1.0], [1e12, 1e-12, 1.0], [1e-30], [1e15]])
def test_values_of_very_different_sizes(state, hd, spread):
    """V rows of very different ranges in one sequence, whatever their attention weights: every row keeps its share, and the
    sum of the weights loses none."""
    n, q_heads, kv_heads = 600, 8, 2
    rng = np.random.default_rng(17)
    k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
    v *= np.asarray(spread, np.float32)[np.arange(n) % len(spread)][:, None]
    k[::7] *= np.float32(3.0)
    kv = state.full_attention(n, q_heads, kv_heads, hd, sg.KV_U4G32, shuffled_seed=9)
    kv.seed(k, v, n)
    q = rng.standard_normal((q_heads, hd)).astype(np.float32)
    want = ref.attention(q, ref.stored(k, 0, hd, 3), ref.stored(v, 0, hd, 3), kv_heads)
    assert ref.close(kv.attention_decode(q), want)[0]
    kv.close()


@pytest.mark.gpu
def test_two_streams_and_a_pending_append(state):
    """Two KV states of one pool used on two streams of the caller, each with its own batch; then the append and the attention
    of one of them in stream order behind a long computation."""
    import torch
    q_heads, kv_heads, hd, n = 16, 2, 128, 1500
    rng = np.random.default_rng(23)
    state.set_concurrent_streams(True)
    kvs = [filled(state, n, q_heads, kv_heads, hd, seed=s, cap=n + 40) for s in (1, 2)]
    q = rng.standard_normal((2, q_heads, hd)).astype(np.float32)
    new = rng.standard_normal((2, 2, 20, kv_heads * hd)).astype(np.float32)
    streams = [torch.cuda.Stream() for _ in range(2)]
    busy = torch.randn(4096, 4096, device="cuda")
    bufs = [[state.upload(x) for x in (new[s, 0], new[s, 1], q[s])] + [state.alloc(q[s].nbytes)] for s in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for (kv, k, v), st, (d_k, d_v, d_q, d_out) in zip(kvs, streams, bufs):
            with torch.cuda.stream(st):
                busy @ busy
            h = st.cuda_stream
            kv.encode_truncate(n, stream=h)
            kv.encode_append_rows(d_k, d_v, 20, stream=h)
            kv.encode_attention_decode_windowed(d_q, d_out, stream=h)
    torch.cuda.synchronize()
    for s, (kv, k, v) in enumerate(kvs):
        rows = [np.concatenate([old, ref.stored(x, n, hd, 3)]) for old, x in ((k, new[s, 0]), (v, new[s, 1]))]
        assert kv.len() == n + 20
        assert ref.close(bufs[s][3].download(), ref.attention(q[s], *rows, kv_heads))[0], s
        kv.close()
    state.set_concurrent_streams(False)


@pytest.mark.gpu
def test_batched_truncate_moves_every_cursor(state):
    n_seq, cap = 600, 33                     # more members than one launch takes
    pool = state.pool(2, 1, 32, sg.KV_U4G32, n_seq * 3, n_seq, cap)
    seqs = [pool.sequence(cap) for _ in range(n_seq)]
    kvs = [s.layer(1, 1) for s in seqs]
    batch = sg.Batch(state, kvs)
    d = state.upload(np.ones((n_seq, 32), np.float32))
    for _ in range(20):
        batch.enqueue_append(d, d)
    lens = [(7 * i) % 21 for i in range(n_seq)]
    batch.enqueue_truncate(lens)
    batch.enqueue_append(d, d)               # the device's cursors are the ones that count here
    state.sync()
    assert [kv.len() for kv in kvs] == [n + 1 for n in lens]
    assert all(s.layer(0, 1).len() == 0 for s in seqs[:5])
    for i in (0, 1, 2, 511, 512, 599):
        kvs[i].gather_rows_f32(0, lens[i] + 1)
    bad = list(lens)
    bad[599] = cap + 1
    for wrong in (bad, lens[:-1]):
        with pytest.raises(sg.InferError) as e:
            batch.enqueue_truncate(wrong)
        assert e.value.kind == "Dimension"
    assert [kv.len() for kv in kvs] == [n + 1 for n in lens]
    for x in (batch, *seqs, pool):
        x.close()

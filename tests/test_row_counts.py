"""Row counts whose sum with a position passes the largest int64, or that an int does not hold, are refused like any other that
does not fit, and change nothing."""
import ctypes as C

import numpy as np
import pytest

import saragossa_b200 as sg

DIMENSION = 1


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gather", [(sg.KV_F32, "sgk_kv_gather_rows"), (sg.KV_BF16, "sgk_kv_gather_rows_f32"),
                                          (sg.KV_U8G32, "sgk_kv_gather_rows_u8"), (sg.KV_U4G32, "sgk_kv_gather_rows_u4")])
def test_counts_that_do_not_fit(dtype, gather):
    st = sg.DecodeResidentState(0)
    kv = st.full_attention(64, 2, 2, 32, dtype)
    rows = np.random.default_rng(1).standard_normal((2, 20, 64)).astype(np.float32)
    kv.seed(rows[0], rows[1], 20)
    before = kv.gather_rows_f32()
    bufs = [np.zeros(64 * 64, np.float32) for _ in range(6)]
    ptrs = [C.c_void_p(b.ctypes.data) for b in bufs]
    device = [st.upload(np.ones(64 * 64, np.float32)) for _ in range(2)]
    outs = ptrs if gather[-2:] in ("u8", "u4") else ptrs[:2]
    for row0, n in ((1, 2**63 - 1), (20, 2**63 - 1), (21, 0), (2**63 - 1, 1), (19, 2)):
        assert getattr(st.L, gather)(kv.h, C.c_int64(row0), C.c_int64(n), *outs) == DIMENSION, (row0, n)
        assert st.L.sgk_kv_enqueue_gather_rows_f32(kv.h, None, C.c_int64(row0), C.c_int64(n), C.c_void_p(device[0].ptr),
                                                   C.c_void_p(device[1].ptr)) == DIMENSION
    for n in (45, 2**31, 2**32 - 3, 2**32 + 1, 2**62, 2**63 - 1):
        with pytest.raises(sg.InferError) as e:
            kv.encode_append_rows(*device, n)
        assert e.value.kind == "Dimension" and kv.len() == 20, n
    assert st.L.sgk_kv_append_rows_f32(kv.h, ptrs[0], C.c_size_t(64), ptrs[1], C.c_size_t(64), C.c_int64(2**63 - 1)) == DIMENSION
    st.sync()
    assert kv.len() == 20 and all(np.array_equal(a, b) for a, b in zip(before, kv.gather_rows_f32()))
    kv.encode_append_rows(*device, 44)
    st.sync()
    assert kv.len() == 64 and st.device_status() == 0
    kv.close()
    st.close()

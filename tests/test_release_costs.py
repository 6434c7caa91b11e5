"""What a call on a long stream costs on the host does not grow with what the stream has behind it."""
import statistics
import time

import pytest

import saragossa_b200 as sg


def _time(call):
    t = time.perf_counter()
    call()
    return time.perf_counter() - t


@pytest.mark.parametrize("sinks", [0, 20])
def test_pages_returned_one_by_one(sinks):
    """A window moves over 40000 pages, one page a call: the last calls work on one page each, like the first."""
    pages = 40000
    pool = sg.PagePool(None, 1, 1, 32, sg.KV_F32, pages, 1, 16 * pages)
    seq = pool.sequence(16 * pages)
    seq.reserve(16 * pages)
    took = [_time(lambda: seq.release_between(sinks, 16 * i)) for i in range(4, pages)]
    assert pool.free_pages == pages - 1 - (2 if sinks else 0)
    # forty thousand pages looked at again in every call took 20 to 30 times the first calls' time
    assert statistics.median(took[-2000:]) < 6 * statistics.median(took[:2000])
    seq.close()
    pool.close()


def test_either_end_of_what_was_returned():
    pool = sg.PagePool(None, 1, 1, 32, sg.KV_F32, 16, 1, 256)
    seq = pool.sequence(256)
    seq.reserve(256)
    for call, held in (((96, 128), [0, 1, 2, 3, 4, 5, 8, 9, 10, 11, 12, 13, 14, 15]), ((100, 160), [0, 1, 2, 3, 4, 5, 10, 11, 12, 13, 14, 15]),
                       ((64, 112), [0, 1, 2, 3, 10, 11, 12, 13, 14, 15]), ((17, 210), [0, 1, 13, 14, 15]), ((40, 170), [0, 1, 13, 14, 15])):
        seq.release_between(*call)
        assert [i for i, p in enumerate(seq.block_table()) if p >= 0] == held
        assert pool.free_pages == 16 - len(held)
    seq.reset()
    assert pool.free_pages == 16
    seq.close()
    pool.close()


@pytest.mark.gpu
def test_truncating_a_large_batch():
    """The host's part of a batched truncation grows with the members, not with their pairs."""
    st = sg.DecodeResidentState(0)
    most, took = 6000, {}
    pool = st.pool(1, 1, 32, sg.KV_U4G32, most, most, 16)
    seqs = [pool.sequence(16) for _ in range(most)]
    kvs = [s.layer(0, 1) for s in seqs]
    for n in (600, most):
        batch = sg.Batch(st, kvs[:n])
        lens = [i % 16 for i in range(n)]
        batch.enqueue_truncate(lens)
        st.sync()
        times = []
        for _ in range(30):
            times.append(_time(lambda: batch.enqueue_truncate(lens)))
            st.sync()
        took[n] = min(times)
        batch.close()
    assert [kv.len() for kv in kvs] == lens
    # ten times the members, ten times the work (launches of 512 members among it); their pairs would be a hundred times as many
    assert took[most] < 30 * took[600], took
    both = sg.Batch(st, [kvs[3], kvs[5], kvs[3], kvs[7], kvs[3]])
    for bad in ([1, 2, 1, 3, 4], [1, 2, 4, 3, 1], [4, 2, 1, 3, 1]):
        with pytest.raises(sg.InferError) as e:
            both.enqueue_truncate(bad)
        assert e.value.kind == "Dimension"
    both.enqueue_truncate([9, 2, 9, 3, 9])
    st.sync()
    assert [kvs[i].len() for i in (3, 5, 7)] == [9, 2, 3]
    for x in (both, *seqs, pool, st):
        x.close()

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

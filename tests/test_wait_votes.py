"""A bounded wait of a whole warp has one answer: the page loops go on with votes, shuffles and matrix instructions of the whole
warp, so lanes whose own waits ended differently must not part there."""
import os
import re

import pytest

import saragossa_b200 as sg

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "saragossa_b200", "csrc")


@pytest.mark.parametrize("name", ["kernels_attn_mma.cu", "kernels_attn_u8.cu", "kernels_attn_u4.cu"])
def test_page_loops_wait_as_a_warp(name):
    """Wherever a page loop goes on by the answer of a wait, it is the warp's (a wait whose answer nobody takes may be a lane's)."""
    text = open(os.path.join(CSRC, name)).read()
    taken = [line for line in text.splitlines() if re.search(r"(=|&&|\|\||return|!|\() *mbar_wait\(", line)]
    assert not taken, taken
    assert "mbar_wait_warp(" in text


@pytest.mark.gpu
def test_lanes_with_different_answers_get_one():
    """Half of a warp waits on a barrier that is complete, the other half on one that nobody completes: no lane goes on."""
    st = sg.DecodeResidentState(0)
    for _ in range(2):
        with pytest.raises(sg.InferError) as e:
            st.selftest_wait_timeout()       # (the kernel reports another error where a lane does go on)
        assert e.value.kind == "Timeout"
        assert st.device_status() == 0
    st.close()

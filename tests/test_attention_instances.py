"""A batch asks the kernel instance that it is about to launch how many of its blocks fit at once: sinks set, changed and taken
away between the calls of one batch, with a short ring (which may let more blocks of one instance than of another onto an SM)
and split counts that make blocks wait for one another."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

CHILD = """
import sys
sys.path[:0] = [ROOT, ROOT + "/tests"]
import numpy as np
import saragossa_b200 as sg
from helpers import u4_reference as ref
st = sg.DecodeResidentState(0)
for dtype, rel in ((sg.KV_BF16, 1e-5), (sg.KV_U8G32, 2e-3), (sg.KV_U4G32, 1e-5)):
    for q_heads, kv_heads, hd in ((16, 2, 128), (8, 2, 256)):
        n = 4000
        rng = np.random.default_rng(hd)
        k, v = rng.standard_normal((2, n, kv_heads * hd)).astype(np.float32)
        kv = st.full_attention(n, q_heads, kv_heads, hd, dtype, shuffled_seed=5)
        kv.seed(k, v, n)
        k, v = (x.astype(np.float64) for x in kv.gather_rows_f32())
        q = rng.standard_normal((q_heads, hd)).astype(np.float32)
        batch = sg.Batch(st, [kv])
        d_q, d_out = st.upload(q), st.alloc(q.nbytes)
        for splits in (74, 148, 8, 16, 5):
            for sinks in (0, 20, 0, 5):
                try:
                    batch.set_splits(splits)
                except sg.InferError:
                    continue
                kv.set_attention_sinks(sinks)
                batch.enqueue_attention(d_q, d_out, 3000)
                st.sync()
                want = ref.attention(q, k, v, kv_heads, n - 3000, sinks)[0]
                err = np.linalg.norm(d_out.download().reshape(want.shape) - want) / np.linalg.norm(want)
                assert err <= rel, (dtype, hd, splits, sinks, err)
                assert st.device_status() == 0, (dtype, hd, splits, sinks)
        batch.close()
        kv.close()
st.close()
print("OK")
"""


@pytest.mark.gpu
@pytest.mark.parametrize("stages", ["", "4"])
def test_sinks_change_between_the_calls_of_a_batch(stages):
    env = dict(os.environ, SGK_ATTN_STAGES=stages) if stages else dict(os.environ)
    run = subprocess.run([sys.executable, "-c", f"ROOT = {ROOT!r}" + CHILD], env=env, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0 and "OK" in run.stdout, run.stderr[-2000:]

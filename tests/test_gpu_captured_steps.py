"""Captured steps of several sizes beside one another: they share the memory of their work areas, and give what the same steps give uncaptured."""
import numpy as np
import pytest
import torch

from test_gpu_drafts_evict_model import engine, models, prompt  # noqa: F401

pytestmark = pytest.mark.gpu


def pools():
    return {tuple(s["segment_pool_id"]) for s in torch.cuda.memory_snapshot()} - {(0, 0)}


@pytest.mark.parametrize("bits", [32, 4])
def test_captured_steps_share_their_work_areas(models, bits):
    m = models("Gemosun")
    out = []
    for graphs in (True, False):
        torch.cuda.empty_cache()
        before = pools()
        m.use_graphs = graphs
        try:
            eng = engine(m, kv_bits=bits, max_tokens=4096, max_keys=600)
            for i, n in enumerate((250, 500, 30)):
                eng.run_entries([{"id": str(i), "tokens": prompt(n, i), "want": []}])
            got = []
            for t in range(12):         # one, two and three requests in turn, over two ranges of keys each
                ids = ["0", "1", "2"][t % 3:] if t < 6 else ["2", "0", "1"][:1 + t % 3]
                got.append(eng.run_entries([{"id": i, "tokens": [5 + t], "want": [0]} for i in ids]))
            weights = [L["key_weight"].clone() for L in m.layers if "key_weight" in L]
            torch.cuda.synchronize()
            out.append((got, weights))
            assert len(pools() - before) <= 1 and (not graphs or len(m._graphs) >= 4)
        finally:
            m.use_graphs = True
    assert all(np.array_equal(a, b) for a, b in zip(out[0][0], out[1][0]))
    for a, b in zip(out[0][1], out[1][1]):
        for slot, n in ((0, 250), (1, 500), (2, 30)):
            assert torch.equal(a[slot, :, :n], b[slot, :, :n])

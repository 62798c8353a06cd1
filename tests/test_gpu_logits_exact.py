"""process_logits (csrc/seq/seq_logits.cu): a temperature and a repetition penalty are one f32 division each, rounded once, at every size of them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TINY, HUGE = float(np.finfo(np.float32).tiny), float(np.finfo(np.float32).max)


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    from blazr_b200 import seqops
    seqops.lib()
    seqops.error_flags()
    return seqops


@pytest.mark.parametrize("R,V", [(1, 1000), (3, 4099), (64, 128256)])
def test_temperatures_divide(ops, R, V):
    rng = np.random.default_rng(V)
    x = (rng.standard_normal((R, V)) * np.exp(rng.standard_normal((R, 1)))).astype(np.float32)
    x[:, ::7] *= np.float32(1e-30)
    for t in (0.7, 1.0, 1.3, 3.0, 1e-3, 1e3, TINY * 2.0 ** -20, TINY * 3, HUGE / 3, HUGE, -0.9):
        rules = np.tile(np.array([1, 0, 0, t], np.float32), (R, 1))
        out = torch.empty(R, V, device=DEV)
        ops.process_logits(torch.from_numpy(x).to(DEV), torch.from_numpy(rules).to(DEV), out)
        with np.errstate(over="ignore", under="ignore"):
            np.testing.assert_array_equal(out.cpu().numpy(), x / np.float32(t))


@pytest.mark.parametrize("rep", [0.3, 1.1, 7.0, 1e30, TINY])
def test_repetition_penalties_divide_or_multiply(ops, rep):
    rng = np.random.default_rng(3)
    R, V = 2, 4099
    x = rng.standard_normal((R, V)).astype(np.float32)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=DEV)
    rules = torch.from_numpy(np.tile(np.array([rep, 0, 0, 0], np.float32), (R, 1))).to(DEV)
    out = torch.empty(R, V, device=DEV)
    ops.process_logits(torch.from_numpy(x).to(DEV), rules, out, hist=i32([5, 9, 9, 4098, 0, 5]), hist_start=i32([0, 4, 6]), hist_prompt=i32([2, 0]))
    want, p = x.copy(), np.float32(rep)
    with np.errstate(over="ignore", under="ignore"):
        for r, ids in ((0, [5, 9, 4098]), (1, [0, 5])):
            want[r, ids] = np.where(x[r, ids] > 0, x[r, ids] / p, x[r, ids] * p)
    np.testing.assert_array_equal(out.cpu().numpy(), want)
    assert ops.error_flags() == 0

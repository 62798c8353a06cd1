"""Drafts verified, the weight of cached keys and eviction at places that test_gpu_between_steps.py does not reach (its docstring has the roundings that the bounds count)."""
import numpy as np
import pytest

from test_gpu_between_steps import evict, ops  # noqa: F401

pytestmark = pytest.mark.gpu


# ---- eviction in place -------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("kw", [dict(rows=[9000], keep=8000, L=1, G=4, D=128), dict(rows=[7000, 6500], keep=3000, L=2, G=2, D=80), dict(rows=[6000], keep=5990, L=1, G=1, D=600),
                                dict(rows=[5000] * 3, keep=4900, L=2, G=2, D=128, bits=4), dict(rows=[4000], keep=3999, L=1, G=3, D=7)], ids=str)
def test_long_sequences_are_cut_back_where_they_lie(ops, kw):
    """clusters of several blocks, many chunks each, rows that move by few places and by many"""
    kw = dict(kw)
    for seed in (1, 2):
        evict(ops, np.random.default_rng(seed), kw["rows"], kw["keep"], 4, 50, **{k: v for k, v in kw.items() if k not in ("rows", "keep")})

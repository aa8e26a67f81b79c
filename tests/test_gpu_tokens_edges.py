"""Ends of the ranges of the operators on columns of tokens.  Bounds and helpers of test_gpu_tokens.py."""
import numpy as np
import pytest

from test_gpu_tokens import F, check_log_probs

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ top lists

@pytest.mark.parametrize("h,w", [(1025, 40), (4096, 40), (5000, 40), (32000, 600), (131072, 2), (200001, 10)])
@pytest.mark.parametrize("lowest", [-1e9, float(np.finfo(np.float32).min), -np.inf])
def test_log_probs_of_a_mask_that_leaves_one_entry_fewer_than_asked_for(cm, h, w, lowest):
    """k - 1 entries are allowed, in as many lanes or in few, row 0 masked or not: the last of the list is the first masked row.  What
    is left unwritten stays NaN."""
    rng = np.random.default_rng(h + w)
    labels = F(rng.integers(0, h, (1, w)))
    for k in (2, 5, 20, 64):
        x = F(np.full((h, w), lowest))
        few = range(w) if w < 100 else list(range(24)) + list(range(w - 8, w))           # (columns that the oracle looks at)
        for c in range(w):
            n = k - 1 if c % 4 < 3 else int(rng.integers(0, k))
            step = 4 if c % 2 else 1                                  # (every row of a lane's group, or other groups)
            rows = 1 + step * rng.choice((h - 1) // step, n, replace=False)
            if c % 8 == 5 and n:
                rows[0] = 0
            x[rows, c] = rng.standard_normal(n)
        names = dict(logp=(1, w), entropy=(1, w), log_z=(1, w), top=(k, w), top_labels=(k, w))
        out = {name: cm.CUDAMatrix(F(np.full(shape, np.nan))) for name, shape in names.items()}
        cm.log_probs(cm.CUDAMatrix(x), cm.CUDAMatrix(labels), **out)
        few = list(few)
        got = {name: m.asarray()[:, few] for name, m in out.items()}
        assert not np.isnan(out['top_labels'].asarray()).any(), (h, w, k)
        check_log_probs(x[:, few], labels[:, few], k, got)

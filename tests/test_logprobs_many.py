"""Many long rows, where a warp or two work on a row, at bounds that count their longer sums.

With N threads to a row, a thread adds V / N values in two packed accumulators: n = V / (2 N) + 40 additions one
after another, so V / 64 + 40 for a warp and V / 128 + 40 for two. What follows is as for few rows."""
import numpy as np
import pytest

import test_logprobs


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,V,threads,n_top,pad", [(1200, 32000, 32, 1, 0), (1200, 50257, 32, 5, 3),
                                                   (800, 40001, 64, 8, 1)])
def test_many_long_rows(monkeypatch, dtype, T, V, threads, n_top, pad):
    n = V / (2 * threads) + 40
    monkeypatch.setattr(test_logprobs, "_rel", lambda V: (n + 45) * test_logprobs.U + 2.0 ** -21)
    tg = np.random.default_rng(T + V).integers(-1, V, (T, 1))
    test_logprobs._check(test_logprobs._logits(T, V, dtype, T + V, pad), tg, n_top)

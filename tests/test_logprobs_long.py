"""Rows of the largest length that ``token_logprobs`` takes, whose last indexes are next to 2^31."""
import numpy as np
import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "float32"])
@pytest.mark.parametrize("start,V", [(0, 2 ** 31 - 1), (1, 2 ** 31 - 1), (3, 2 ** 31 - 17)])
def test_last_values_of_the_longest_rows(dtype, start, V):
    """A mask leaves a few values, the last ones among them; starts that give a ragged head and tail. Five
    values: logp is off by the rounding of x - m, of log s and of their difference, and by s, whose
    five terms are within 2^-21 (the exponential) and 8 roundings of theirs."""
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs

    flat = torch.full((2 ** 31 + 8,), float("-inf"), dtype=getattr(torch, dtype), device="cuda")
    x = flat[start:start + V].unsqueeze(0)
    at = np.array([V - 1, 5, V - 2, V // 2, 0])
    val = np.array([3.0, 2.5, 2.0, 1.5, 1.0])
    for i, v in zip(at, val):
        x[0, int(i)] = v
    r = token_logprobs(x, targets=torch.from_numpy(np.append(at, V - 3)[None]).cuda(), n_top=8)
    torch.cuda.synchronize()
    lp = val - val.max() - np.log(np.exp(val - val.max()).sum())
    tol = 2.0 ** -21 + 20 * 2.0 ** -24 * (1 + np.abs(lp).max())
    assert r.top_ids[0].tolist() == at.tolist() + [-1] * 3
    assert np.abs(r.top_logp[0, :5].double().cpu().numpy() - lp).max() <= tol
    assert np.abs(r.logp[0, :5].double().cpu().numpy() - lp).max() <= tol
    assert torch.isneginf(r.logp[0, 5]) and torch.isneginf(r.top_logp[0, 5:]).all()
    assert abs(float(r.entropy[0]) + (np.exp(lp) * lp).sum()) <= 4 * tol

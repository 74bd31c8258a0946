"""The fused MoE layer where single activations stand far above their neighbours.

A weight of 0 beside an outlier leaves the sum to the other values, so what those lose shows. Bound of an
input's own rounding, from the kernel's rule: a value is kept in f32, or within 2^-22 of one that four
of its block of 32 reach a 32nd of, so within 2^-17 of the block's fourth largest magnitude. u =
2^-24: a block's dot takes 5 roundings and a sum over the lanes 14 (15 in a down row, as for
ordinary inputs); a value kept in f32 is one more term of a lane's sum, at most 32 of a lane here: 14 + 32
of the terms' absolute sum, in which an outlier with weight 0 has no part."""
import numpy as np
import pytest

from test_moe_few import U, _close, _layer, _make


def _fourth(v):
    return np.repeat(np.sort(np.abs(v).reshape(-1, 32), 1)[:, -4], 32) * 2.0 ** -17


def _sums(M, x, rounds):
    return M @ x, np.abs(M) @ _fourth(x) + rounds * U * (np.abs(M) @ np.abs(x))


def _expert(orc, gate, up, down, d, f, x):
    """(y, bound of its error), in 64 bits; every value of x is exact."""
    deq = lambda r, n, m: np.asarray(orc.dequantize(r, 2, n, m), np.float64).reshape(n, m)  # noqa: E731
    (g, dg), (u, du) = (_sums(deq(w, f, d), x, 46) for w in (gate, up))
    D = deq(down, d, f)
    s = g / (1 + np.exp(-g))
    h, dh = s * u, 1.1 * np.abs(u) * dg + np.abs(s) * du + 5 * U * np.abs(s * u)
    y, dy = _sums(D, h, 47)
    return y, dy + np.abs(D) @ (1.01 * dh)


def _reference(orc, w, x, d, f, E, k):
    r = orc.moe_route(x, w["router"], d, E, k, bias=None)
    out, tol = np.zeros(x.shape), np.zeros(x.shape)
    router = np.abs(w["router"].reshape(E, d)).astype(np.float64)
    cut = lambda a, e: a.reshape(E, -1)[e]  # noqa: E731
    for t in range(x.shape[0]):
        xt = x[t].astype(np.float64)
        moved = 2 * (d + d / 32 + 12) * U * (router[r["idx"][t]] @ np.abs(xt)).max()
        for e, g in zip(r["idx"][t], r["gates"][t]):
            y, dy = _expert(orc, cut(w["gate"], e), cut(w["up"], e), cut(w["down"], e), d, f, xt)
            out[t] += g * y
            tol[t] += g * dy + (g * (moved + (k + 8) * U) + (k + 4) * U * g) * np.abs(y)
    # an f32 operation that underflows is off by 2^-150 at most, whatever its value: fewer than 2^25 of
    # them lead to an output, and what follows them multiplies by less than 2^5
    return out, tol + 2.0 ** -120


def _zero(orc, w, which, rows, cols, at):
    """The weights of columns ``at`` of every row become 0."""
    a = np.asarray(orc.dequantize(w[which], 2, rows, cols), np.float32).reshape(rows, cols).copy()
    a[:, at] = 0.0
    w[which] = np.asarray(orc.quantize_q4_0(a.reshape(-1)))


@pytest.mark.gpu
@pytest.mark.parametrize("d,f,E,k,T", [(1024, 128, 8, 2, 1), (2048, 256, 6, 3, 5), (1024, 512, 4, 2, 16),
                                       (4096, 128, 4, 2, 13)])
@pytest.mark.parametrize("size", [20.0, 300.0, 3e4, 1e12])
def test_an_outlier_beside_a_weight_of_zero(orc, d, f, E, k, T, size):
    import torch

    rng = np.random.default_rng(d + f + T)
    w = _layer(orc, rng, d, f, E, k, None, False)
    at = np.arange(0, d, 32) + rng.integers(0, 32, d // 32)  # one a block
    for which in ("gate", "up"):
        _zero(orc, w, which, E * f, d, at)
    w["router"].reshape(E, d)[:, at] = 0.0
    x = rng.standard_normal((T, d)).astype(np.float32)
    x[:, at] = size * (1 + rng.random((T, at.size)))
    L = _make(w, d, f, E, k)
    y = L.forward(torch.from_numpy(x).cuda(), path="fused")
    L.ctx.sync_check()
    _close(y, *_reference(orc, w, x, d, f, E, k))


@pytest.mark.gpu
@pytest.mark.parametrize("f", [128, 512, 1024])
def test_an_outlier_in_the_hidden_row(orc, f):
    """Some up rows are a thousand times the others, and most of their down weights are 0."""
    import torch

    d, E, k, T = 1024, 4, 2, 6
    rng = np.random.default_rng(f)
    w = _layer(orc, rng, d, f, E, k, None, False)
    at = np.arange(0, f, 32) + rng.integers(0, 32, f // 32)
    up = np.asarray(orc.dequantize(w["up"], 2, E * f, d), np.float32).reshape(E, f, d).copy()
    up[:, at] *= 1000.0
    w["up"] = np.asarray(orc.quantize_q4_0(up.reshape(-1)))
    _zero(orc, w, "down", E * d, f, at)
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = _make(w, d, f, E, k)
    _close(L.forward(torch.from_numpy(x).cuda(), path="fused"), *_reference(orc, w, x, d, f, E, k))


@pytest.mark.gpu
def test_outliers_with_weights_and_every_spread(orc):
    """Outliers that count; blocks of few values, of values each a tenth of the one before, of zeros, of
    values near f32's smallest; an outlier that only one token of an item has."""
    import torch

    d, f, E, k, T = 1024, 256, 4, 2, 9
    rng = np.random.default_rng(3)
    w = _layer(orc, rng, d, f, E, k, None, False)
    x = rng.standard_normal((T, d)).astype(np.float32)
    x[0, rng.integers(0, d, 12)] *= 500.0
    x[1] = 0.0
    x[1, ::64] = 1.0
    x[2] = np.tile(10.0 ** -np.arange(32.0), d // 32) * rng.choice([-1, 1], d)
    x[3, 96:960] = 0.0
    x[4, :256] *= 1e-33
    x[5, 7] = 4000.0
    x[6] *= 1e-34
    x[7, 31::32] = 90.0
    L = _make(w, d, f, E, k)
    _close(L.forward(torch.from_numpy(x).cuda(), path="fused"), *_reference(orc, w, x, d, f, E, k))


@pytest.mark.gpu
def test_an_infinite_hidden_value_acts_as_in_f32(orc):
    """One up product overflows: infinities where its down weight is not 0, NaN where it is, as the
    path that keeps f32 gives them."""
    import torch

    d, f, E, k, T = 1024, 128, 2, 2, 3
    rng = np.random.default_rng(5)
    w = _layer(orc, rng, d, f, E, k, None, False)
    for which in ("gate", "up"):
        _zero(orc, w, which, E * f, d, [40])
    up = np.asarray(orc.dequantize(w["up"], 2, E * f, d), np.float32).reshape(E, f, d).copy()
    up[:, 17, 40] = 8000.0
    w["up"] = np.asarray(orc.quantize_q4_0(up.reshape(-1)))
    w["router"].reshape(E, d)[:, 40] = 0.0
    x = rng.standard_normal((T, d)).astype(np.float32)
    x[1, 40] = 3e38
    L, xd = _make(w, d, f, E, k), torch.from_numpy(x).cuda()
    y, want = L.forward(xd, path="fused"), L.forward(xd, path="gemv")
    assert not torch.isfinite(want[1]).any() and torch.isfinite(want[[0, 2]]).all()
    for test in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(test(y), test(want))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [5, 40, 300])
def test_outliers_of_other_tokens_change_nothing(orc, n):
    """The same bits alone and in a batch whose other tokens have outliers elsewhere, few or more than are
    listed."""
    import torch

    d, f, E, k, T = 1024, 128, 6, 2, 16
    rng = np.random.default_rng(n)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    x = rng.standard_normal((T, d)).astype(np.float32)
    for t in range(T):
        at = rng.integers(0, d, n)
        x[t, at] *= 10.0 ** rng.uniform(2.0, 4.0, n)
    x[3] = rng.standard_normal(d)
    xd = torch.from_numpy(x).cuda()
    y = L.forward(xd, path="fused")
    assert torch.equal(torch.cat([L.forward(xd[t:t + 1], path="fused") for t in range(T)]), y)
    assert torch.equal(L.forward(xd[4:11], path="fused"), y[4:11])

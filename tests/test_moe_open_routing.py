"""The fused MoE layer's tokens whose choice of experts the first kernel's bounds leave open: ties, logits
one unit apart, masked experts. The choice is the reference's, and finding it is no cliff."""
import numpy as np
import pytest

from test_moe_few import _close, _layer, _make, _reference


def _near_ties(w, E, d, rng, pairs):
    """Router rows that come in pairs: equal, or apart in single elements by one unit in the last place, so
    that sequential sums differ by a unit or not at all."""
    r = w["router"].reshape(E, d)
    for a, b in pairs:
        r[b] = r[a]
        for i in rng.integers(0, d, rng.integers(0, 4)):
            r[b, i] = np.nextafter(r[b, i], np.float32(rng.choice([-9.0, 9.0])))


@pytest.mark.gpu
@pytest.mark.parametrize("d,f,E,k,T,shared,bias,norm", [
    (1024, 128, 16, 3, 16, None, False, False), (1024, 128, 16, 5, 9, "gated", True, True),
    (2048, 128, 300, 7, 16, "gated", False, True), (2048, 128, 512, 31, 5, "plain", True, False),
    (4096, 128, 257, 4, 13, "gated", True, True), (4096, 128, 40, 32, 16, None, False, True),
    (1024, 256, 3, 2, 1, "gated", False, True), (2048, 256, 2, 1, 16, "gated", True, True)])
def test_logits_a_unit_apart(orc, d, f, E, k, T, shared, bias, norm):
    """Any wrong choice would show: the tied experts differ in all their weights."""
    import torch

    rng = np.random.default_rng(d + E + k)
    w = _layer(orc, rng, d, f, E, k, shared, False)
    at = rng.permutation(E)
    _near_ties(w, E, d, rng, list(zip(at[0::2], at[1::2])))
    if bias:
        w["bias"] = rng.choice(np.float32([0.0, 0.5, -0.25]), E)
        w["bias"][at[1::2]] = w["bias"][at[0::2][:E // 2]]
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = _make(w, d, f, E, k)
    y = L.forward(torch.from_numpy(x).cuda(), rmsnorm=norm, residual=True, path="fused")
    L.ctx.sync_check()
    _close(y, *_reference(orc, w, x, d, f, E, k, norm, True))


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_some_tokens_open(orc, norm):
    """Open and certain tokens in one batch, at every place; a token's output is the same alone, and in
    place."""
    import torch

    d, f, E, k = 1024, 128, 24, 4
    rng = np.random.default_rng(11)
    w = _layer(orc, rng, d, f, E, k, "gated", False)
    r = w["router"].reshape(E, d)
    r[1::2] = r[0::2]
    r[:, : d // 2] = rng.standard_normal((E, d // 2)).astype(np.float32) * 0.02
    x = rng.standard_normal((16, d)).astype(np.float32)
    x[[0, 3, 4, 9, 15], : d // 2] = 0.0  # here the pairs tie, elsewhere not
    L = _make(w, d, f, E, k - 1)
    xd = torch.from_numpy(x).cuda()
    y = L.forward(xd, rmsnorm=norm, residual=True, path="fused")
    _close(y, *_reference(orc, w, x, d, f, E, k - 1, norm, True))
    one = torch.cat([L.forward(xd[t:t + 1], rmsnorm=norm, residual=True, path="fused") for t in range(16)])
    assert torch.equal(one, y)
    L.forward(xd, out=xd, rmsnorm=norm, residual=True, path="fused")
    assert torch.equal(xd, y)


@pytest.mark.gpu
def test_open_tokens_in_graphs_on_two_streams(orc):
    import torch

    d, f, E, k = 1024, 128, 32, 3
    rng = np.random.default_rng(12)
    w = _layer(orc, rng, d, f, E, k, "gated", False)
    w["router"].reshape(E, d)[1::2] = w["router"].reshape(E, d)[0::2]
    L = _make(w, d, f, E, k)
    xs = [torch.randn(T, d, device="cuda") for T in (16, 3)]
    want = [L.forward(x, path="fused") for x in xs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(L.forward(x, path="fused"))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    L.ctx.sync_check()
    assert all(torch.equal(o, y) for o, y in zip(outs, want))


def _device_us(call):
    """Device time of a call in a captured graph, the best of five."""
    import torch

    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(20):
            call()
    best = float("inf")
    for _ in range(6):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        g.replay()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 50.0)
    return best


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
def test_open_tokens_cost_one_more_step(orc, norm):
    """Sixteen tokens whose experts all tie in pairs, against the same tokens and a router without ties: a
    barrier and one sequential chain more, not one for each token."""
    import torch

    d, f, E, k = 2048, 128, 64, 3
    rng = np.random.default_rng(13)
    w = _layer(orc, rng, d, f, E, k, None, False)
    x = torch.from_numpy(rng.standard_normal((16, d)).astype(np.float32)).cuda()
    plain = _make(w, d, f, E, k)
    w["router"].reshape(E, d)[1::2] = w["router"].reshape(E, d)[0::2]
    tied = _make(w, d, f, E, k)
    base, open_ = (_device_us(lambda: L.forward(x, rmsnorm=norm, path="fused")) for L in (plain, tied))
    assert open_ < 2.5 * base, (open_, base)

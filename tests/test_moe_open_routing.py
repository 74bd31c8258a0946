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


@pytest.mark.gpu
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("bias", [None, "steps", "masks", "few", "all", "mixed"])
def test_rows_of_zeros_and_masked_experts(orc, norm, bias):
    """A batch padded with zeros (every logit is its bias: they tie, or tie in steps), experts that a bias of
    -inf takes out, so that enough, fewer than k or none are left, and router rows of zeros."""
    import torch

    d, f, E, k = 1024, 128, 40, 6
    rng = np.random.default_rng(31)
    w = _layer(orc, rng, d, f, E, k, "gated", False)
    w["router"].reshape(E, d)[[3, 8, 30]] = 0.0
    b = np.zeros(E, np.float32)
    if bias == "steps":
        b[:] = rng.integers(0, 4, E)
    elif bias == "masks":
        b[rng.permutation(E)[:20]] = -np.inf
    elif bias == "few":
        b[rng.permutation(E)[: E - k + 2]] = -np.inf
    elif bias == "mixed":
        b[:] = rng.choice(np.float32([-np.inf, -0.0, 0.0, 1.0, 3e-4, -100.0, 2.0 ** -17]), E)
    elif bias == "all":
        b[:] = -np.inf
    w["bias"] = None if bias is None else b
    x = rng.standard_normal((16, d)).astype(np.float32)
    x[5:] = 0.0
    x[7, 3] = 1e-30
    L = _make(w, d, f, E, k)
    xd = torch.from_numpy(x).cuda()
    y = L.forward(xd, rmsnorm=norm, residual=True, path="fused")
    L.ctx.sync_check()
    if bias == "all":  # no probability anywhere: NaN, as the layer's other path gives
        want = L.forward(xd, rmsnorm=norm, residual=True, path="gemv")
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        return
    # an f32 operation that underflows is off by 2^-150 at most, whatever its value: fewer than 2^25 of
    # them lead to an output, and what follows them multiplies by less than 2^5
    want, tol = _reference(orc, w, x, d, f, E, k, norm, True)
    _close(y, want, tol + 2.0 ** -120)


@pytest.mark.gpu
@pytest.mark.parametrize("bias", [None, "steps", "mixed"])
def test_exact_ties_among_other_logits(orc, bias):
    """Router rows of zeros: their logits tie, exactly and at any place among the others, and which of them
    are chosen shows in the output."""
    import torch

    d, f, E, k, T = 1024, 128, 300, 9, 16
    rng = np.random.default_rng(33)
    w = _layer(orc, rng, d, f, E, k, None, False)
    w["router"].reshape(E, d)[rng.permutation(E)[: E - 12]] = 0.0
    if bias:
        w["bias"] = rng.choice(np.float32([0.0, 0.5, -0.25]) if bias == "steps" else
                               np.float32([-np.inf, -0.0, 0.0, 1e-6, 2.0 ** -17]), E)
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = _make(w, d, f, E, k)
    y = L.forward(torch.from_numpy(x).cuda(), path="fused")
    L.ctx.sync_check()
    _close(y, *_reference(orc, w, x, d, f, E, k, False, False))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["zeros", "masks"])
def test_padding_and_masks_are_certain(orc, what):
    """Neither a row of zeros nor a masked expert leaves a choice open: the time is that of other tokens."""
    import torch

    d, f, E, k = 2048, 128, 64, 4
    rng = np.random.default_rng(32)
    w = _layer(orc, rng, d, f, E, k, None, False)
    plain = _make(w, d, f, E, k)
    w["bias"] = np.zeros(E, np.float32)
    x = torch.from_numpy(rng.standard_normal((16, d)).astype(np.float32)).cuda()
    base = _device_us(lambda: plain.forward(x, rmsnorm=True, path="fused"))
    if what == "zeros":
        x[1:] = 0.0
    else:
        w["bias"][::5] = -np.inf
    L = _make(w, d, f, E, k)
    other = _device_us(lambda: L.forward(x, rmsnorm=True, path="fused"))
    assert other < 1.2 * base + 2.0, (other, base)


@pytest.mark.gpu
def test_a_token_more_than_fits_one_group(orc):
    """4096 wide, the inputs of 12 tokens fit a CTA; thirteen are worked on as seven and six, at hardly more than
    the price of twelve."""
    import torch

    d, f, E, k = 4096, 256, 32, 4
    rng = np.random.default_rng(41)
    w = _layer(orc, rng, d, f, E, k, None, False)
    w["bias"] = np.linspace(0.0, 30.0, E).astype(np.float32)[rng.permutation(E)]  # no choice is open
    L = _make(w, d, f, E, k)
    x = torch.from_numpy(rng.standard_normal((13, d)).astype(np.float32)).cuda()
    fits, more = (_device_us(lambda: L.forward(x[:T], path="fused")) for T in (12, 13))
    assert more < 1.2 * fits, (more, fits)

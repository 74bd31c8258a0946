"""The MoE layer of a few tokens in two kernels (``path="fused"``), against the definition in 64
bits over the reference's own routing, and against the layer's other path.

Tolerance, u = 2^-24, from the kernels' own sums. 32 inputs become integers of at least 2^21 for the
largest: each is within 2^-22 of the block's largest, F = 2^-22 max|block|. Block dots are exact
integers, turned into f32 with 3 roundings, scaled with 1 and added with 1; then a lane's blocks
(4 at most, 8 in a down row) and five (two) shuffles: at most 5 + 4 + 5 = 14 and 5 + 8 + 2 = 15
roundings of a block's absolute terms, which are at most (|x| + F) |w|. RMSNorm's input is the
reference's up to d / 8 + 64 roundings of one common factor (its sum of squares is sequential).
h = g s(g) u moves by 1.1 |u| dg + |g s(g)| du and rounds five times. Gates: logits are sums of 32
segments, within (d / 32 + 8) u sum|p| of exact ones, the reference's sequential ones within d u
sum|p|; a gate moves by twice the largest such change, relatively."""
import numpy as np
import pytest

U = 2.0 ** -24


def _layer(orc, rng, d, f, E, k, shared, bias):
    mk = lambda n: np.asarray(orc.quantize_q4_0((rng.standard_normal(n) * 0.02).astype(np.float32)))  # noqa: E731
    w = dict(router=(rng.standard_normal(E * d) * 0.02).astype(np.float32), gate=mk(E * f * d), up=mk(E * f * d),
             down=mk(E * d * f), shared=None, bias=None)
    if shared:
        w["shared"] = (mk(f * d), mk(f * d), mk(d * f),
                       (rng.standard_normal(d) * 0.02).astype(np.float32) if shared == "gated" else None)
    if bias:
        w["bias"] = (2.0 * np.log(1.0 / (rng.permutation(E) + 1.0))).astype(np.float32)
    return w


def _make(w, d, f, E, k):
    from powerinfer_x64_b200 import moe

    return moe.MoeLayer(w["router"], w["gate"], w["up"], w["down"], 2, d, f, E, k, shared=w["shared"],
                        router_bias=w["bias"])


def _fix(v):
    """What fixed point may move each value by: 2^-22 of its block's largest."""
    return np.repeat(np.abs(v).reshape(-1, 32).max(1), 32) * 2.0 ** -22


def _expert(orc, gate, up, down, d, f, x, dx):
    """(y, bound of its error) of one expert for one token, in 64 bits; dx: what is known of x."""
    deq = lambda r, n, m: np.asarray(orc.dequantize(r, 2, n, m), np.float64).reshape(n, m)  # noqa: E731
    G, Up, D = deq(gate, f, d), deq(up, f, d), deq(down, d, f)
    g, u = G @ x, Up @ x
    e = dx + _fix(x) + 14 * U * np.abs(x)
    dg, du = np.abs(G) @ e, np.abs(Up) @ e
    s = g / (1 + np.exp(-g))
    h, dh = s * u, 1.1 * np.abs(u) * dg + np.abs(s) * du + 5 * U * np.abs(s * u)
    return D @ h, np.abs(D) @ (1.01 * dh + 1.01 * _fix(h) + 15 * U * np.abs(h))


def _reference(orc, w, x, d, f, E, k, norm, residual):
    T = x.shape[0]
    xin = np.stack([orc.rms_norm(r, np.ones(d, np.float32)) for r in x]) if norm else x
    r = orc.moe_route(xin, w["router"], d, E, k, bias=w["bias"])
    out, tol = np.zeros((T, d)), np.zeros((T, d))
    cut = lambda a, e: a.reshape(E, -1)[e]  # noqa: E731
    router = np.abs(w["router"].reshape(E, d)).astype(np.float64)
    for t in range(T):
        xt = xin[t].astype(np.float64)
        dx = (d / 8 + 66) * U * np.abs(xt) if norm else np.zeros(d)
        moved = 2 * (d + d / 32 + 8 + (d / 8 + 66) * norm + 4) * U * (router[r["idx"][t]] @ np.abs(xt)).max()
        terms = []
        for e, g in zip(r["idx"][t], r["gates"][t]):
            y, dy = _expert(orc, cut(w["gate"], e), cut(w["up"], e), cut(w["down"], e), d, f, xt, dx)
            terms.append((float(g), float(g) * (moved + (k + 8) * U), y, dy))
        if w["shared"]:
            gate, up, down, sg = w["shared"]
            y, dy = _expert(orc, gate, up, down, d, f, xt, dx)
            z = 0.0 if sg is None else sg.astype(np.float64) @ xt
            dz = 0.0 if sg is None else (d / 32 + 8 + (d / 8 + 66) * norm) * U * (np.abs(sg) @ np.abs(xt))
            terms.append((1.0 if sg is None else 1 / (1 + np.exp(-z)), dz / 4 + 4 * U, y, dy))
        for g, dgate, y, dy in terms:
            out[t] += g * y
            tol[t] += g * dy + dgate * np.abs(y) + (k + 4) * U * g * np.abs(y)
        if residual:
            out[t] += x[t]
            tol[t] += 2 * U * (np.abs(x[t]) + np.abs(out[t]))
    return out, tol


def _close(got, want, tol):
    bad = np.abs(got.double().cpu().numpy() - want) - tol
    assert bad.max() <= 0, f"over the bound by {bad.max():.3e} at {np.unravel_index(bad.argmax(), bad.shape)}"


def test_refuses_without_a_gpu():
    import ctypes as C

    from powerinfer_x64_b200._lib import PI_ERR_ARG, lib

    assert lib().pi_moe_forward_fused(None, None, None, 1, None, 0, None, 0, None) == PI_ERR_ARG
    assert lib().pi_moe_fused_workspace(C.c_void_p(None), 4) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d,f,E,k,T,shared,bias,norm,residual", [
    (1024, 128, 8, 1, 1, None, False, False, False), (1024, 256, 64, 4, 16, None, False, False, False),
    (1024, 128, 9, 8, 3, "gated", True, True, True), (2048, 512, 16, 8, 1, "gated", False, True, True),
    (2048, 512, 32, 8, 5, "plain", True, False, False), (2048, 256, 300, 2, 16, "gated", False, True, False),
    (2048, 1024, 12, 3, 7, "gated", False, False, True), (4096, 128, 20, 5, 2, None, True, True, False),
    (4096, 512, 6, 2, 16, "gated", False, True, True), (4096, 1024, 4, 4, 9, "plain", False, False, False),
    (1024, 256, 512, 32, 16, "gated", False, True, True), (1024, 512, 1, 1, 4, None, False, False, True)])
def test_against_definition(orc, d, f, E, k, T, shared, bias, norm, residual):
    import torch

    rng = np.random.default_rng(d + f + E + k + T)
    w = _layer(orc, rng, d, f, E, k, shared, bias)
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = _make(w, d, f, E, k)
    xd = torch.from_numpy(x).cuda()
    y = L.forward(xd, rmsnorm=norm, residual=residual, path="fused")
    L.ctx.sync_check()
    _close(y, *_reference(orc, w, x, d, f, E, k, norm, residual))
    assert torch.equal(L.forward(xd, rmsnorm=norm, residual=residual, path="fused"), y)


@pytest.mark.gpu
def test_every_batch_size_equals_single_tokens(orc):
    """A token's output does not depend on the tokens beside it: the same bits alone and in a batch."""
    import torch

    d, f, E, k = 1024, 256, 16, 4
    rng = np.random.default_rng(1)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    x = torch.from_numpy(rng.standard_normal((16, d)).astype(np.float32)).cuda()
    one = torch.cat([L.forward(x[t:t + 1], path="fused") for t in range(16)])
    for T in range(1, 17):
        assert torch.equal(L.forward(x[:T], path="fused"), one[:T]), T


@pytest.mark.gpu
def test_ties_and_repeated_tokens(orc):
    """Equal router rows: the lowest index wins, as on the other paths; a token that stands twice."""
    import torch

    from test_gpu_parity import close

    d, f, E, k, T = 1024, 128, 32, 4, 8
    rng = np.random.default_rng(2)
    w = _layer(orc, rng, d, f, E, k, "gated", False)
    r = w["router"].reshape(E, d)
    r[1::2] = r[0::2]
    x = rng.standard_normal((T, d)).astype(np.float32)
    x[5] = x[2]
    x[7] = 0.0  # every logit ties at 0
    L = _make(w, d, f, E, k)
    y = L.forward(torch.from_numpy(x).cuda(), path="fused")
    _close(y, *_reference(orc, w, x, d, f, E, k, False, False))
    close(y.cpu().numpy(), L.forward(torch.from_numpy(x).cuda(), path="gemv").cpu().numpy())
    assert torch.equal(y[5], y[2])


@pytest.mark.gpu
def test_in_place_and_neighbours(orc):
    import torch

    d, f, E, k = 1024, 256, 8, 2
    rng = np.random.default_rng(3)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    x = torch.from_numpy(rng.standard_normal((6, d)).astype(np.float32)).cuda()
    want = L.forward(x, rmsnorm=True, residual=True, path="fused")
    buf = torch.full((10, d), 7.0, device="cuda")
    buf[2:8] = x
    L.forward(buf[2:8], out=buf[2:8], rmsnorm=True, residual=True, path="fused")
    assert torch.equal(buf[2:8], want) and (buf[:2] == 7).all() and (buf[8:] == 7).all()


@pytest.mark.gpu
def test_non_finite_tokens_stay_in_their_row(orc):
    import torch

    d, f, E, k = 1024, 128, 8, 2
    rng = np.random.default_rng(4)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    x = torch.from_numpy(rng.standard_normal((5, d)).astype(np.float32)).cuda()
    want = L.forward(x, path="fused")
    x[1, 3], x[3] = float("nan"), float("inf")
    y = L.forward(x, path="fused")
    L.ctx.sync_check()
    assert torch.equal(y[[0, 2, 4]], want[[0, 2, 4]])
    assert torch.isnan(y[1]).all() and not torch.isfinite(y[3]).any()


@pytest.mark.gpu
def test_errors(orc):
    import torch

    from powerinfer_x64_b200 import PiError, moe
    from powerinfer_x64_b200._lib import PI_ERR_ARG, PI_ERR_SHORT, lib, ptr, stream_ptr

    d, f, E, k = 1024, 128, 8, 2
    rng = np.random.default_rng(5)
    w = _layer(orc, rng, d, f, E, k, None, False)
    L = _make(w, d, f, E, k)
    x = torch.randn(17, d, device="cuda")

    def refused(code, fn, *a, **kw):
        with pytest.raises(PiError) as e:
            fn(*a, **kw)
        assert e.value.code == code

    fwd = lambda t, **kw: L.forward(t, path="fused", **kw)  # noqa: E731
    refused(PI_ERR_ARG, fwd, x)
    refused(PI_ERR_ARG, fwd, x[:2].double())
    refused(PI_ERR_ARG, fwd, x[:2, : d // 2])
    refused(PI_ERR_ARG, fwd, x[:2], out=torch.empty(3, d, device="cuda"))
    refused(PI_ERR_ARG, fwd, x[:2], fast=True)
    assert fwd(x[:0]).shape == (0, d)
    q8 = lambda n: orc.quantize_q8_0((rng.standard_normal(n) * 0.02).astype(np.float32))  # noqa: E731
    L8 = moe.MoeLayer(w["router"], q8(E * f * d), q8(E * f * d), q8(E * d * f), 8, d, f, E, k)
    refused(PI_ERR_ARG, L8.forward, x[:1], path="fused")
    out = torch.empty(4, d, device="cuda")
    ws = torch.empty(lib().pi_moe_fused_workspace(L.h, 4), dtype=torch.uint8, device="cuda")
    call = lambda flags, w_, n: lib().pi_moe_forward_fused(L.ctx.h, L.h, ptr(x), 4, ptr(out), flags, w_, n, stream_ptr())  # noqa: E731
    assert call(0, ptr(ws), ws.numel() - 1) == PI_ERR_SHORT
    assert call(4, ptr(ws), ws.numel()) == PI_ERR_ARG
    assert call(0, None, 0) == 0  # the stream's scratch arena
    torch.cuda.synchronize()
    assert torch.equal(out, fwd(x[:4]))


@pytest.mark.gpu
def test_streams_and_graphs(orc):
    """Two captured graphs on two streams at once and eager calls between them, on one layer: the
    cooperative kernels take turns, each call has its own workspace."""
    import torch

    d, f, E, k = 2048, 512, 16, 4
    rng = np.random.default_rng(6)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    xs = [torch.randn(T, d, device="cuda") for T in (1, 6)]
    eager = [L.forward(x, rmsnorm=True, residual=True, path="fused") for x in xs]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(L.forward(x, rmsnorm=True, residual=True, path="fused"))
        graphs.append(g)
    torch.cuda.synchronize()
    for i in range(40):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        if i % 10 == 0:
            assert torch.equal(L.forward(xs[0], rmsnorm=True, residual=True, path="fused"), eager[0])
    torch.cuda.synchronize()
    L.ctx.sync_check()
    assert all(torch.equal(o, e) for o, e in zip(outs, eager))
    side = torch.cuda.Stream()
    y = L.forward(xs[1], rmsnorm=True, residual=True, path="fused", stream=side)
    side.synchronize()
    assert torch.equal(y, eager[1])


@pytest.mark.gpu
def test_decode_step_of_all_three(orc):
    """A decode step's end as a server runs it: the last layer, the LM head with the requests'
    adapters, the scores; against the same chain in 64 bits on the layer's own output."""
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs
    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection
    from test_lora import _bank, _reference as project, _weights
    from test_logprobs import _reference as scores

    d, f, E, k, T, V, n, R = 1024, 256, 16, 4, 5, 5003, 3, 8
    rng = np.random.default_rng(7)
    w = _layer(orc, rng, d, f, E, k, "gated", False)
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = _make(w, d, f, E, k)
    y = L.forward(torch.from_numpy(x).cuda(), rmsnorm=True, residual=True, path="fused")
    _close(y, *_reference(orc, w, x, d, f, E, k, True, True))
    raw, head = _weights(orc, V, d, 8, rng)
    a, b, ranks, scales = _bank(rng, n, R, d, V, torch.bfloat16)
    ids = np.array([0, -1, 2, 1, 0], np.int32)
    bank = AdapterBank(a.cuda(), b.cuda(), ranks=torch.from_numpy(ranks).cuda(), scales=torch.from_numpy(scales).cuda())
    P = SharedProjection(raw, 8, V, d)
    logits = P.forward(y, bank, torch.from_numpy(ids).cuda())
    want, tol = project(orc, y.cpu().numpy(), head, 8, a, b, ranks, scales, ids)
    assert (np.abs(logits.double().cpu().numpy() - want) <= tol).all()
    best = logits.argmax(1)
    r = token_logprobs(logits, best, 3)
    lp, ent, top, _ = scores(logits.double().cpu().numpy(), best.cpu().numpy(), 3)
    assert np.abs(r.logp.cpu().numpy() - lp).max() <= (V / 256 + 90) * U + 2.0 ** -20
    assert np.array_equal(r.top_ids.cpu().numpy(), top)


@pytest.mark.gpu
def test_first_call_of_a_layer_under_capture(orc):
    import torch

    d, f, E, k = 1024, 256, 24, 5
    rng = np.random.default_rng(8)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", True), d, f, E, k)
    x = torch.randn(3, d, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = L.forward(x, rmsnorm=True, path="fused")
    for scale in (1.0, -0.5):
        x.mul_(scale)
        g.replay()
        assert torch.equal(y, L.forward(x, rmsnorm=True, path="fused"))
    L.ctx.sync_check()

"""A projection over GGUF weights beside many requests' low-rank adapters, against the
definition in 64 bits.

Tolerances, u = 2^-24, per output and with S the sum of the absolute values of its terms:
* base, Q8_0: block dots are exact; the product d_w d_x is exact in f32; each block's fused
  multiply-add rounds once, then the warps' sums: (blocks + 8) u S.
* base, Q4_0: x is held within 2^-22 of each value (or 2^-38 of the token's largest); 32
  products a block in f32 matrix instructions, 17 u for each of the four k-steps, then a
  rounding a block: (2^-22 + (blocks + 8 + 4 * 17) u) S + 2^-38 max|x| sum|w|.
* adapter: n_in / 256 + 8 + 5 roundings of h, then at most R + 2 of the outer sum."""
import numpy as np
import pytest

U = 2.0 ** -24


def _weights(orc, n_out, n_in, qtype, rng, std=0.05):
    w = (rng.standard_normal(n_out * n_in) * std).astype(np.float32)
    raw = np.asarray(orc.quantize_q8_0(w) if qtype == 8 else orc.quantize_q4_0(w))
    return raw, np.asarray(orc.dequantize(raw, qtype, n_out, n_in), np.float64).reshape(n_out, n_in)


def _bank(rng, n, R, n_in, n_out, dtype):
    import torch

    a = torch.from_numpy((rng.standard_normal((n, R, n_in)) / np.sqrt(n_in)).astype(np.float32)).to(dtype)
    b = torch.from_numpy((rng.standard_normal((n, n_out, R)) * 0.1).astype(np.float32)).to(dtype)
    ranks = rng.integers(0, R + 1, n).astype(np.int32)
    ranks[0] = R
    return a, b, ranks, rng.uniform(0.5, 2.0, n).astype(np.float32)


def _reference(orc, x, w, qtype, a=None, b=None, ranks=None, scales=None, ids=None):
    """(y, tolerance) float64 [T, n_out] from the definition."""
    n_in, nb = x.shape[1], x.shape[1] // 32
    if qtype == 8:
        base = np.asarray(orc.dequantize(orc.quantize_q8_0(x.reshape(-1)), 8, x.shape[0], n_in), np.float64).reshape(x.shape)
        rel, extra = (nb + 8) * U, 0.0
    else:
        base = x.astype(np.float64)
        rel = 2.0 ** -22 + (nb + 8 + 68) * U
        extra = 2.0 ** -38 * np.abs(base).max(1)[:, None] * np.abs(w).sum(1)[None, :]
    y = base @ w.T
    tol = rel * (np.abs(base) @ np.abs(w).T) + extra
    if a is not None:
        for t, i in enumerate(ids):
            if 0 <= i < len(ranks):
                r = ranks[i]
                A, B = a[i, :r].double().numpy(), b[i, :, :r].double().numpy()
                xt = x[t].astype(np.float64)
                y[t] += scales[i] * (B @ (A @ xt))
                tol[t] += (n_in / 256 * 8 + 13 + 1 + r + 2) * U * scales[i] * (np.abs(B) @ (np.abs(A) @ np.abs(xt)))
    return y, tol + 4 * U * np.abs(y)


def _close(got, y, tol):
    bad = np.abs(got.double().cpu().numpy() - y) - tol
    assert bad.max(initial=-1) <= 0, f"over the bound by {bad.max():.3e} at {np.unravel_index(bad.argmax(), bad.shape)}"


# ---------------------------------------------------------------------------
# without a GPU
# ---------------------------------------------------------------------------
def test_refuses_without_a_gpu():
    import ctypes as C

    import torch

    from powerinfer_x64_b200 import PiError
    from powerinfer_x64_b200._lib import PI_ERR_ARG, PiLoraBank, lib
    from powerinfer_x64_b200.lora import AdapterBank

    with pytest.raises(PiError) as e:
        AdapterBank(torch.zeros(1, 8, 32), torch.zeros(1, 16, 8))
    assert e.value.code == PI_ERR_ARG
    L, h = lib(), C.c_void_p(1)
    assert L.pi_proj_create(None, None, 0, 8, 32, 1, 0, C.byref(h)) == PI_ERR_ARG
    assert L.pi_proj_forward(None, None, None, 1, None, None, None, None, 0, None) == PI_ERR_ARG
    assert L.pi_proj_workspace(None, 4, C.byref(PiLoraBank())) == 0
    L.pi_proj_destroy(None)


# ---------------------------------------------------------------------------
# against the definition
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("qtype", [8, 2])
@pytest.mark.parametrize("T,n_in,n_out", [(1, 32, 1), (1, 2048, 2048), (3, 96, 17), (8, 288, 100), (9, 1024, 31),
                                          (16, 4096, 257), (17, 544, 3001), (33, 1024, 1000), (64, 256, 50),
                                          (65, 160, 333), (130, 512, 77), (5, 64, 40000), (40, 128, 40001),
                                          (18, 96, 80003), (61, 224, 76001), (20, 4096, 40)])
def test_projection_alone(orc, qtype, T, n_in, n_out):
    import torch

    from powerinfer_x64_b200.lora import SharedProjection

    rng = np.random.default_rng(T * 7 + n_in + n_out)
    raw, w = _weights(orc, n_out, n_in, qtype, rng)
    x = rng.standard_normal((T, n_in)).astype(np.float32)
    x[T // 2, : n_in // 2] *= 1e-3  # blocks of very different size
    want, tol = _reference(orc, x, w, qtype)
    xd = torch.from_numpy(x).cuda()
    for src in (raw, torch.from_numpy(raw.copy()).cuda()):  # weights on the host and on the device
        P = SharedProjection(src, qtype, n_out, n_in)
        y = P.forward(xd)
        _close(y, want, tol)
        assert torch.equal(P.forward(xd), y)


@pytest.mark.gpu
@pytest.mark.parametrize("qtype", [8, 2])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,n_in,n_out,n,R", [(1, 2048, 300, 1, 16), (7, 96, 33, 3, 1), (16, 512, 1000, 4, 12),
                                              (37, 1024, 3001, 5, 12), (70, 288, 129, 40, 5), (64, 256, 40000, 6, 8),
                                              (4, 4096, 64, 2, 64), (12, 320, 200, 3, 130), (50, 96, 76003, 7, 20)])
def test_adapters(orc, qtype, dtype, T, n_in, n_out, n, R):
    import torch

    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(T + n_in + n_out + R)
    raw, w = _weights(orc, n_out, n_in, qtype, rng)
    a, b, ranks, scales = _bank(rng, n, R, n_in, n_out, getattr(torch, dtype))
    # what lies past an adapter's rank is not used, whatever it is
    for i, r in enumerate(ranks):
        a[i, r:] = float("nan")
        b[i, :, r:] = float("inf")
    ids = rng.integers(-1, n, T).astype(np.int32)
    x = rng.standard_normal((T, n_in)).astype(np.float32)
    want, tol = _reference(orc, x, w, qtype, a, b, ranks, scales, ids)
    P = SharedProjection(raw, qtype, n_out, n_in)
    bank = AdapterBank(a.cuda(), b.cuda(), ranks=torch.from_numpy(ranks).cuda(), scales=torch.from_numpy(scales).cuda())
    y = P.forward(torch.from_numpy(x).cuda(), bank, torch.from_numpy(ids).cuda())
    _close(y, want, tol)


@pytest.mark.gpu
def test_defaults_of_a_bank_and_replaced_adapters(orc):
    """No ranks and scales: full rank, scale 1; a slot rewritten in place serves the next call."""
    import torch

    from powerinfer_x64_b200 import PiError
    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(3)
    T, n_in, n_out, n, R = 6, 256, 90, 2, 10
    raw, w = _weights(orc, n_out, n_in, 8, rng)
    a, b, _, _ = _bank(rng, n, R, n_in, n_out, torch.float32)
    x, ids = rng.standard_normal((T, n_in)).astype(np.float32), np.array([0, 1, -1, 1, 0, -7], np.int32)
    P, bank = SharedProjection(raw, 8, n_out, n_in), AdapterBank(a.cuda(), b.cuda())
    xd, idd = torch.from_numpy(x).cuda(), torch.from_numpy(ids).cuda()
    full, one = np.full(n, R, np.int32), np.ones(n, np.float32)
    _close(P.forward(xd, bank, idd), *_reference(orc, x, w, 8, a, b, full, one, ids))
    a2, b2 = torch.randn(4, n_in), torch.randn(n_out, 4)
    bank.set(1, a2.cuda(), b2.cuda(), 0.25)
    a[1, :4], b[1, :, :4] = a2, b2
    _close(P.forward(xd, bank, idd), *_reference(orc, x, w, 8, a, b, np.array([R, 4], np.int32),
                                                 np.array([1, 0.25], np.float32), ids))
    with pytest.raises(PiError):
        bank.set(2, a2.cuda(), b2.cuda())
    with pytest.raises(PiError):
        bank.set(0, torch.zeros(11, n_in).cuda(), torch.zeros(n_out, 11).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-30, 1e-3, 1e4, 1e30])
def test_4_bit_projection_at_any_scale(orc, scale):
    """Two f16 terms hold f32 inputs of any size; the largest and smallest token of a batch do not mix."""
    import torch

    from powerinfer_x64_b200.lora import SharedProjection

    rng = np.random.default_rng(8)
    raw, w = _weights(orc, 64, 512, 2, rng)
    x = rng.standard_normal((5, 512)).astype(np.float32) * np.float32(scale)
    x[1] *= np.float32(1e-5)
    x[3] = 0.0
    want, tol = _reference(orc, x, w, 2)
    _close(SharedProjection(raw, 2, 64, 512).forward(torch.from_numpy(x).cuda()), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("qtype", [8, 2])
def test_non_finite_inputs_stay_in_their_row(orc, qtype):
    import torch

    from powerinfer_x64_b200.lora import SharedProjection

    rng = np.random.default_rng(9)
    raw, w = _weights(orc, 40, 128, qtype, rng)
    x = rng.standard_normal((9, 128)).astype(np.float32)
    want, tol = _reference(orc, x, w, qtype)
    x[2, 5], x[8, 100] = np.nan, np.inf
    y = SharedProjection(raw, qtype, 40, 128).forward(torch.from_numpy(x).cuda())
    keep = [t for t in range(9) if t not in (2, 8)]
    _close(y[keep], want[keep], tol[keep])
    if qtype == 2:
        assert torch.isnan(y[[2, 8]]).all()


@pytest.mark.gpu
def test_rows_behind_the_batch_stay(orc):
    import torch

    from powerinfer_x64_b200.lora import SharedProjection

    rng = np.random.default_rng(10)
    raw, _ = _weights(orc, 50, 96, 8, rng)
    buf = torch.full((9, 50), 7.0, device="cuda")
    P = SharedProjection(raw, 8, 50, 96)
    P.forward(torch.randn(3, 96, device="cuda"), out=buf[2:5])
    assert (buf[:2] == 7).all() and (buf[5:] == 7).all() and not (buf[2:5] == 7).any()


@pytest.mark.gpu
def test_errors(orc):
    import torch

    from powerinfer_x64_b200 import PiError
    from powerinfer_x64_b200._lib import PI_ERR_ARG, PI_ERR_INDEX, PI_ERR_SHORT
    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(11)
    raw, w = _weights(orc, 20, 64, 8, rng)

    def refused(code, f, *a, **k):
        with pytest.raises(PiError) as e:
            f(*a, **k)
        assert e.value.code == code

    refused(PI_ERR_SHORT, SharedProjection, raw[:-1], 8, 20, 64)
    refused(PI_ERR_ARG, SharedProjection, raw, 0, 20, 64)
    refused(PI_ERR_ARG, SharedProjection, raw, 8, 20, 63)
    refused(PI_ERR_ARG, SharedProjection, raw, 8, 0, 64)
    P = SharedProjection(raw, 8, 20, 64)
    x = torch.randn(3, 64, device="cuda")
    ids = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    bank = AdapterBank(torch.randn(2, 8, 64, device="cuda"), torch.randn(2, 20, 8, device="cuda"))
    refused(PI_ERR_ARG, P.forward, x.double())
    refused(PI_ERR_ARG, P.forward, x.cpu())
    refused(PI_ERR_ARG, P.forward, x[:, :32])
    refused(PI_ERR_ARG, P.forward, torch.randn(64, 3, device="cuda").t())
    refused(PI_ERR_ARG, P.forward, x, bank)
    refused(PI_ERR_ARG, P.forward, x, None, ids)
    refused(PI_ERR_ARG, P.forward, x, bank, ids.long())
    refused(PI_ERR_ARG, P.forward, x, bank, ids[:2])
    refused(PI_ERR_ARG, P.forward, x, out=torch.empty(3, 21, device="cuda"))
    refused(PI_ERR_ARG, P.forward, x, AdapterBank(torch.zeros(1, 8, 32, device="cuda"),
                                                  torch.zeros(1, 20, 8, device="cuda")), ids)
    refused(PI_ERR_ARG, AdapterBank, torch.zeros(1, 8, 32, device="cuda"), torch.zeros(1, 20, 9, device="cuda"))
    refused(PI_ERR_ARG, AdapterBank, torch.zeros(1, 1025, 32, device="cuda"), torch.zeros(1, 20, 1025, device="cuda"))
    assert P.forward(x[:0]).shape == (0, 20)
    plain = P.forward(x)
    y = P.forward(x, bank, ids)  # token 2 names no adapter of the bank
    refused(PI_ERR_INDEX, P.ctx.sync_check)
    assert torch.equal(y[2], plain[2]) and not torch.equal(y[0], plain[0])
    P.ctx.sync_check()


@pytest.mark.gpu
def test_streams_and_graphs(orc):
    """Two captured graphs of one projection replayed at once on two streams, and eager calls
    between them: each has its own workspace."""
    import torch

    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(12)
    raw, _ = _weights(orc, 3001, 512, 8, rng)
    P = SharedProjection(raw, 8, 3001, 512)
    bank = AdapterBank(torch.randn(3, 16, 512, device="cuda"), torch.randn(3, 3001, 16, device="cuda"))
    xs = [torch.randn(T, 512, device="cuda") for T in (5, 40)]
    ids = [torch.randint(-1, 3, (x.shape[0],), device="cuda", dtype=torch.int32) for x in xs]
    eager = [P.forward(x, bank, i) for x, i in zip(xs, ids)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in xs], [], []
    for x, i, s in zip(xs, ids, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(P.forward(x, bank, i))
        graphs.append(g)
    torch.cuda.synchronize()
    for k in range(30):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        if k % 10 == 0:
            assert torch.equal(P.forward(xs[0], bank, ids[0]), eager[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, e) for o, e in zip(outs, eager))
    xs[0].mul_(2.0)
    ids[0].fill_(-1)
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], P.forward(xs[0]))


@pytest.mark.gpu
def test_scratch_arena_instead_of_a_workspace(orc):
    """The C entry point without a workspace uses the stream's arena; a short one is refused."""
    import ctypes as C

    import torch

    from powerinfer_x64_b200._lib import PI_ERR_ARG, PI_ERR_SHORT, PI_OK, lib, ptr, stream_ptr
    from powerinfer_x64_b200.lora import SharedProjection

    rng = np.random.default_rng(13)
    raw, _ = _weights(orc, 77, 160, 2, rng)
    P = SharedProjection(raw, 2, 77, 160)
    x, y = torch.randn(11, 160, device="cuda"), torch.empty(11, 77, device="cuda")
    args = (P.ctx.h, P.h, ptr(x), 11, None, None, ptr(y))
    assert lib().pi_proj_forward(*args, None, 0, stream_ptr()) == PI_OK
    torch.cuda.synchronize()
    assert torch.equal(y, P.forward(x))
    ws = torch.empty(lib().pi_proj_workspace(P.h, 11, None), dtype=torch.uint8, device="cuda")
    assert lib().pi_proj_forward(*args, ptr(ws), ws.numel() - 1, stream_ptr()) == PI_ERR_SHORT
    assert lib().pi_proj_forward(*args, C.c_void_p(ws.data_ptr() + 8), ws.numel(), stream_ptr()) == PI_ERR_ARG


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_one_adapter_for_a_long_batch_and_empty_ones(orc, dtype):
    """Groups of eight tokens over several chunks of 64, the same adapter everywhere; adapters of
    rank 0 add nothing."""
    import torch

    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(14)
    T, n_in, n_out, n, R = 201, 96, 47, 3, 20
    raw, w = _weights(orc, n_out, n_in, 8, rng)
    a, b, ranks, scales = _bank(rng, n, R, n_in, n_out, getattr(torch, dtype))
    ranks[:] = R, 0, 3
    x = rng.standard_normal((T, n_in)).astype(np.float32)
    P, xd = SharedProjection(raw, 8, n_out, n_in), torch.from_numpy(x).cuda()
    bank = AdapterBank(a.cuda(), b.cuda(), ranks=torch.from_numpy(ranks).cuda(), scales=torch.from_numpy(scales).cuda())
    for ids in (np.zeros(T, np.int32), np.ones(T, np.int32), np.arange(T, dtype=np.int32) % 3):
        y = P.forward(xd, bank, torch.from_numpy(ids).cuda())
        _close(y, *_reference(orc, x, w, 8, a, b, ranks, scales, ids))
    assert torch.equal(P.forward(xd, bank, torch.ones(T, dtype=torch.int32, device="cuda")), P.forward(xd))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["a", "b"])
def test_an_adapters_nan_stays_with_its_tokens(orc, which):
    import torch

    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(15)
    raw, _ = _weights(orc, 70, 64, 8, rng)
    a, b = torch.randn(4, 9, 64, device="cuda"), torch.randn(4, 70, 9, device="cuda")
    ids = torch.tensor([0, 1, 2, 3, -1, 2, 1, 0, 3, 3, 2], dtype=torch.int32, device="cuda")
    x = torch.randn(11, 64, device="cuda")
    P = SharedProjection(raw, 8, 70, 64)
    want = P.forward(x, AdapterBank(a, b), ids)
    (a if which == "a" else b)[2, 5 if which == "a" else slice(None), 4] = float("nan")
    y = P.forward(x, AdapterBank(a, b), ids)
    hit = ids == 2
    assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], want[~hit])


@pytest.mark.gpu
def test_first_call_of_a_shape_under_capture(orc):
    """What a shape's first call finds out (launch plan, workspace) it may find out while captured."""
    import torch

    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(16)
    raw, _ = _weights(orc, 900, 192, 2, rng)
    P = SharedProjection(raw, 2, 900, 192)
    bank = AdapterBank(torch.randn(2, 8, 192, device="cuda"), torch.randn(2, 900, 8, device="cuda"))
    x, ids = torch.randn(21, 192, device="cuda"), torch.arange(21, device="cuda").int() % 3 - 1
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = P.forward(x, bank, ids)
    g.replay()
    first = y.clone()
    bank.set(1, torch.randn(5, 192), torch.randn(900, 5), 2.0)  # the graph reads the bank as it is at each replay
    g.replay()
    assert torch.equal(y, P.forward(x, bank, ids)) and not torch.equal(y, first)


@pytest.mark.gpu
def test_projection_then_scores(orc):
    """A decode step's end: LM head with the requests' adapters, then the scores of its logits."""
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs
    from powerinfer_x64_b200.lora import AdapterBank, SharedProjection

    rng = np.random.default_rng(14)
    T, n_in, n_out, n, R = 5, 512, 4001, 3, 8
    raw, w = _weights(orc, n_out, n_in, 8, rng)
    a, b, ranks, scales = _bank(rng, n, R, n_in, n_out, torch.float16)
    ids = np.array([0, 1, 2, -1, 0], np.int32)
    x = rng.standard_normal((T, n_in)).astype(np.float32)
    want, tol = _reference(orc, x, w, 8, a, b, ranks, scales, ids)
    bank = AdapterBank(a.cuda(), b.cuda(), ranks=torch.from_numpy(ranks).cuda(), scales=torch.from_numpy(scales).cuda())
    logits = SharedProjection(raw, 8, n_out, n_in).forward(torch.from_numpy(x).cuda(), bank, torch.from_numpy(ids).cuda())
    best = torch.from_numpy(want.argmax(1)).cuda()
    r = token_logprobs(logits, best, 4)
    lp = want - want.max(1, keepdims=True)
    lp -= np.log(np.exp(lp).sum(1, keepdims=True))
    # a logit off by e moves a log probability by 2 e at most; then the scores' own f32 sums
    assert np.abs(r.logp.cpu().numpy() - lp.max(1)).max() <= 2 * tol.max() + (n_out / 256 + 90) * U + 2.0 ** -20
    assert torch.equal(r.top_ids[:, 0].long(), best)

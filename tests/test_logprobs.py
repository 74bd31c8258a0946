"""Log probabilities, entropy and alternatives from logits, against the definition in 64 bits.

Tolerances, with u = 2^-24. A thread adds at most n = V / 256 + 40 exponentials one after
another, then 5 + 8 + 16 partial sums; each exponential is within 2^-21 of its value
(ex2.approx within 2 ulp, and the rounded argument t log2(e) moves it by less than 2u |t|
with e^t |t| <= 1 / e), each addition and rescaling rounds once. So s is within
(n + 29 + 16) u + 2^-21 =: r of its value, relatively, and so is each of the two parts of the
entropy; log s carries r absolutely, and x - m one rounding more."""
import numpy as np
import pytest

U = 2.0 ** -24


def _rel(V):
    return (V / 256 + 40 + 45) * U + 2.0 ** -21


def _reference(x, targets=None, n_top=0):
    """x float64 [T, V] -> (logp, entropy, ids, top_logp), row by row from the definition."""
    T, V = x.shape
    lp = np.full((T, V), -np.inf)
    ent = np.zeros(T)
    for t in range(T):
        r = x[t]
        if np.isnan(r).any() or np.isposinf(r).any():
            lp[t], ent[t] = np.nan, np.nan
            continue
        live = np.isfinite(r)
        if live.any():
            m = r[live].max()
            # m is taken off first: beside a lowest value of -3e38, log s would vanish in m + log s
            lp[t][live] = (r[live] - m) - np.log(np.exp(r[live] - m).sum())
            ent[t] = -(np.exp(lp[t][live]) * lp[t][live]).sum()
    out = None
    if targets is not None:
        tg = targets.reshape(T, -1)
        out = np.where(tg < 0, 0.0, np.take_along_axis(lp, np.maximum(tg, 0), 1)).reshape(targets.shape)
    ids = tops = None
    if n_top:
        ids = np.full((T, n_top), -1, np.int64)
        tops = np.full((T, n_top), -np.inf)
        for t in range(T):
            if np.isnan(lp[t]).any():
                tops[t] = np.nan
                continue
            live = np.nonzero(np.isfinite(x[t]))[0]
            best = live[np.lexsort((live, -x[t][live]))][:n_top]  # by value, then by index
            ids[t, :best.size], tops[t, :best.size] = best, lp[t][best]
    return out, ent, ids, tops


def _close(got, ref, tol):
    got = got.cpu().numpy().astype(np.float64)
    assert got.shape == ref.shape
    # an f32 result beyond f32's range (-3e38 less 3e38) rounds to infinity
    ref = np.where(np.abs(ref) > np.finfo(np.float32).max, np.copysign(np.inf, ref), ref)
    fin = np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[~fin & ~np.isnan(ref)], ref[~fin & ~np.isnan(ref)])
    bad = np.abs(got[fin] - ref[fin]) - tol(np.abs(ref[fin]))
    assert bad.size == 0 or bad.max() <= 0, f"over the bound by {bad.max():.3e}"


def _check(x, targets=None, n_top=0, run=None):
    """x: CUDA logits [T, V]; everything against the definition on the same values."""
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs

    r = (run or token_logprobs)(x, targets=None if targets is None else torch.from_numpy(targets).cuda(), n_top=n_top)
    torch.cuda.synchronize()
    V = x.shape[1]
    lp, ent, ids, tops = _reference(x.double().cpu().numpy(), targets, n_top)
    # logp = t - log s: |t| <= |logp| + log s, log s <= log V
    ltol = lambda a: _rel(V) + 2 * U * (2 * a + 2 * np.log(V) + 1)  # noqa: E731
    _close(r.entropy, ent, lambda a: 2 * _rel(V) * (a + 1) + 4 * U * (np.log(V) + 1))
    if targets is None:
        assert r.logp is None
    else:
        _close(r.logp, lp, ltol)
    if n_top:
        assert np.array_equal(r.top_ids.cpu().numpy(), ids)
        _close(r.top_logp, tops, ltol)
    else:
        assert r.top_ids is None and r.top_logp is None
    return r


def _logits(T, V, dtype, seed, pad=0, std=2.5):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(T, V + pad, device="cuda", generator=g) * std
    return w.to(getattr(torch, dtype))[:, :V]


# ---------------------------------------------------------------------------
# refusals that need no GPU
# ---------------------------------------------------------------------------
def test_refuses_without_a_gpu():
    import torch

    from powerinfer_x64_b200 import PiError
    from powerinfer_x64_b200._lib import PI_ERR_ARG, lib
    from powerinfer_x64_b200.logprobs import token_logprobs

    for bad in (torch.zeros(2, 8), torch.zeros(8), torch.zeros(2, 8, dtype=torch.int32)):
        with pytest.raises(PiError) as e:
            token_logprobs(bad)
        assert e.value.code == PI_ERR_ARG
    assert lib().pi_token_logprobs(None, None, 0, 1, 8, 8, None, 0, 0, None, None, None, None, None) == PI_ERR_ARG


# ---------------------------------------------------------------------------
# against the definition
# ---------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("T,V,n_top,K,pad", [
    (1, 1, 1, 1, 0), (1, 2, 3, 2, 1), (3, 7, 32, 1, 0), (2, 31, 5, 0, 3), (5, 257, 32, 3, 2), (1, 1024, 1, 1, 0),
    (4, 4097, 20, 1, 5), (149, 1000, 4, 2, 0), (37, 32003, 8, 1, 1), (1, 151936, 20, 1, 0), (2, 151936, 32, 4, 0),
    (1, 262144, 32, 1, 7), (300, 5000, 0, 1, 0), (700, 3001, 2, 1, 0), (1200, 1, 1, 1, 0), (1300, 37, 32, 2, 1),
    (1184, 1031, 20, 1, 3), (1201, 9001, 1, 1, 0), (1500, 700, 0, 3, 0), (1190, 6000, 5, 0, 8)])
def test_against_definition(dtype, T, V, n_top, K, pad):
    x = _logits(T, V, dtype, 7 * T + V, pad)
    rng = np.random.default_rng(T + V)
    tg = rng.integers(0, V, (T, K))
    tg[rng.random((T, K)) < 0.2] = -1
    _check(x, tg if K else None, n_top)


@pytest.mark.gpu
def test_one_target_a_row_keeps_its_shape():
    r = _check(_logits(6, 300, "float32", 1), np.array([0, 299, -1, 5, -100, 17]), 2)
    assert tuple(r.logp.shape) == (6,) and float(r.logp[2]) == 0.0 and float(r.logp[4]) == 0.0


@pytest.mark.gpu
@pytest.mark.parametrize("V", [40, 3000, 50257, 151936])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_ties_take_the_lowest_index(dtype, V):
    """Few distinct values, constant rows, rising and falling rows, rows that repeat, zeros of both signs."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(V)
    i = torch.arange(V, device="cuda")
    rows = [torch.randint(0, 4, (V,), device="cuda", generator=g).float(), torch.zeros(V, device="cuda"), i / 64.0,
            -(i / 64.0), (i % 7).float(), torch.where(i % 2 == 0, -0.0, 0.0),
            torch.where(i == V - 1, 1.0, 0.0), torch.where(i % 1024 == 5, 3.0, 0.5)]
    _check(torch.stack(rows).to(getattr(torch, dtype)), None, 20)
    _check(torch.stack(rows).to(getattr(torch, dtype)), None, 1)
    if V <= 3000:  # as many rows as give each one warp
        many = torch.stack(rows).to(getattr(torch, dtype)).repeat(150, 1)
        _check(many, None, 20)
        _check(many, None, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("lowest", [False, True])
def test_masks(dtype, lowest):
    """Most, all but one, and all tokens masked, with -inf and with the type's lowest value."""
    import torch

    V = 20011
    x = _logits(8, V, dtype, 3)
    low = torch.finfo(x.dtype).min if lowest else float("-inf")
    keep = torch.rand(8, V, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.001
    keep[1] = False
    keep[2] = False
    keep[2, V - 1] = True
    keep[3] = False
    keep[3, :3] = True
    x = torch.where(keep, x, torch.full_like(x, low))
    tg = np.tile(np.array([0, 1, 2, V - 1]), (8, 1))
    few = x[:, :1500].repeat(150, 1)  # a warp a row
    few[3::8, :1497] = low
    _check(few, None, 20)
    r = _check(x, tg, 20)
    if not lowest:
        assert float(r.entropy[1]) == 0.0 and (r.top_ids[1] == -1).all() and torch.isneginf(r.logp[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [100, 70000])
def test_rows_without_a_distribution(V):
    """A NaN or +inf, wherever it stands, spoils its own row only."""
    import torch

    x = _logits(7, V, "float32", 5)
    x[1, 0] = float("nan")
    x[2, V - 1] = float("nan")
    x[3, V // 2] = float("inf")
    x[4] = float("-inf")
    x[4, 17] = float("nan")
    x[5] = torch.finfo(torch.float32).max  # the largest finite value is a value
    if V == 100:
        _check(x.repeat(180, 1), np.zeros((1260, 1), np.int64), 3)  # a warp a row
    r = _check(x, np.zeros((7, 1), np.int64), 3)
    assert torch.isnan(r.entropy[1:5]).all() and (r.top_ids[1:5] == -1).all()
    assert not torch.isnan(r.entropy[[0, 5, 6]]).any()


@pytest.mark.gpu
def test_extreme_spread_and_long_rows():
    import torch

    x = _logits(3, 200000, "float32", 9, std=300.0)
    x[1] *= 1e35
    x[2] = -3.0e38
    x[2, 77] = 3.0e38
    _check(x, np.array([[0], [5], [77]]), 8)


@pytest.mark.gpu
def test_strides_and_offsets():
    """Rows at odd strides and starts, a broadcast row, rows out of order."""
    import torch

    base = _logits(9, 1031, "float16", 2)
    big = torch.zeros(9, 1100, dtype=torch.float16, device="cuda")
    for start in range(0, 9):
        v = big[:, start:start + 1031]
        v.copy_(base)
        _check(v, np.full((9, 1), 1030), 6)
    _check(base[:1].expand(5, -1), np.zeros(5, np.int64), 3)
    _check(base[::2], np.zeros(5, np.int64), 3)


@pytest.mark.gpu
def test_row_offsets_beyond_32_bits():
    import torch

    flat = torch.zeros(2 ** 31 + 4096, dtype=torch.float16, device="cuda")
    x = flat.as_strided((2, 1000), (2 ** 31 + 2048, 1))
    x.copy_(_logits(2, 1000, "float16", 4))
    _check(x, np.array([[3], [999]]), 5)


@pytest.mark.gpu
def test_errors():
    import torch

    from powerinfer_x64_b200 import Context, PiError
    from powerinfer_x64_b200._lib import PI_ERR_ARG, PI_ERR_INDEX
    from powerinfer_x64_b200.logprobs import token_logprobs

    x = _logits(2, 64, "float32", 1)
    for kw in (dict(n_top=33), dict(n_top=-1), dict(targets=torch.zeros(2, dtype=torch.int32, device="cuda")),
               dict(targets=torch.zeros(3, dtype=torch.int64, device="cuda")),
               dict(targets=torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(PiError) as e:
            token_logprobs(x, **kw)
        assert e.value.code == PI_ERR_ARG
    for bad in (x.t(), x.double(), x[0], x[:, ::2], x[:, :0]):
        with pytest.raises(PiError):
            token_logprobs(bad)
    r = token_logprobs(x[:0], targets=torch.zeros((0, 2), dtype=torch.int64, device="cuda"), n_top=4)
    assert r.logp.shape == (0, 2) and r.top_ids.shape == (0, 4) and r.entropy.shape == (0,)
    r = token_logprobs(x, targets=torch.tensor([1, 64], device="cuda"))
    with pytest.raises(PiError) as e:
        Context.of(0).sync_check()
    assert e.value.code == PI_ERR_INDEX
    assert torch.isfinite(r.logp[0]) and torch.isnan(r.logp[1])
    Context.of(0).sync_check()  # reported once


@pytest.mark.gpu
def test_streams_graphs_and_repeats():
    """Two captured graphs replayed at once on two streams, inputs changed between replays;
    every run of the same input gives the same bits."""
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs

    xs = [_logits(3, 50000, "float32", s) for s in (1, 2)]
    tg = torch.zeros(3, 1, dtype=torch.int64, device="cuda")
    eager = [token_logprobs(x, tg, 7) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    graphs, outs = [], []
    for x, s in zip(xs, streams):
        s.wait_stream(torch.cuda.current_stream())
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(token_logprobs(x, tg, 7))
        graphs.append(g)
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert all(torch.equal(a, b) for a, b in zip(o, e))
    xs[0].copy_(xs[1])
    with torch.cuda.stream(streams[0]):
        streams[0].wait_stream(torch.cuda.current_stream())
        graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], eager[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("n_top", [1, 8, 32])
def test_rising_rows_and_many_rows(dtype, n_top):
    """Logits that rise along the row: every value is among the best so far, so that buffers fill
    again and again; few rows, more than eight and more than five for each SM."""
    import torch

    for T, V in ((3, 9001), (1300, 1500), (800, 2500)):
        up = torch.linspace(-3.0, 3.0, V, device="cuda").expand(T, V) + torch.arange(T, device="cuda")[:, None] % 5
        _check(up.to(getattr(torch, dtype)), np.full(T, V - 1), n_top)


@pytest.mark.gpu
def test_first_call_of_a_shape_under_capture():
    import torch

    from powerinfer_x64_b200.logprobs import token_logprobs

    x = torch.randn(2, 77777, device="cuda", dtype=torch.float16)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = token_logprobs(x, None, 11)
    g.replay()
    assert all(torch.equal(p, q) for p, q in zip(r, token_logprobs(x, None, 11)) if p is not None)


@pytest.mark.gpu
@pytest.mark.parametrize("qtype", [8, 0])
def test_lm_head_logprobs(orc, qtype):
    """The resident LM head and the scores of its logits, as a server chains them."""
    import torch

    from powerinfer_x64_b200.lmhead import LmHead

    rng = np.random.default_rng(6)
    n_in, n_out, T = 512, 3000, 4
    w = rng.normal(0, 0.05, (n_out, n_in)).astype(np.float32)
    raw = orc.quantize_q8_0(w.reshape(-1)) if qtype == 8 else w.tobytes()
    x = rng.normal(0, 1, (T, n_in)).astype(np.float32)
    logits = np.stack([orc.matvec_col_major(x[t], raw, qtype, n_in, n_out) for t in range(T)])
    head = LmHead(raw, qtype, n_out, n_in)
    xd = torch.from_numpy(x).cuda()
    _check(torch.from_numpy(logits).cuda(), np.arange(T), 5,
           run=lambda _, targets, n_top: head.logprobs(xd, targets, n_top))

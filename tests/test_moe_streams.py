"""MoE calls on a stream that is not the current one: memory comes from the pool of the stream that
works on it, whose order covers what was launched there before."""
import contextlib

import numpy as np
import pytest

from test_moe_few import _layer, _make


class _Stream:
    def __init__(self, handle):
        self.cuda_stream = handle


class _Tensor:
    """As much of a CUDA tensor as the calls look at; ``pool`` is the stream it was allocated on."""

    is_cuda, dtype, device = True, "f32", "cuda:0"

    def __init__(self, n, pool):
        self.n, self.pool, self.recorded = n, pool, []

    numel = lambda self: self.n  # noqa: E731
    get_device = lambda self: 0  # noqa: E731
    is_contiguous = lambda self: True  # noqa: E731
    data_ptr = lambda self: id(self)  # noqa: E731

    def record_stream(self, s):
        self.recorded.append(s.cuda_stream)


class _Torch:
    """torch's streams and allocations on the host: a tensor belongs to the stream that is current."""

    float32, uint8, int32 = "f32", "u8", "i32"

    def __init__(self):
        self.now, self.made, self.cuda = _Stream(0), [], self

    def current_stream(self, device=None):
        return self.now

    @contextlib.contextmanager
    def stream(self, s):
        before, self.now = self.now, s
        yield
        self.now = before

    def empty(self, *shape, **kw):
        shape = shape[0] if isinstance(shape[0], tuple) else shape
        self.made.append(_Tensor(int(np.prod(shape)), self.now.cuda_stream))
        return self.made[-1]

    zeros = empty


class _Lib:
    def __init__(self):
        self.calls = []

    def pi_moe_fused_workspace(self, layer, T):
        return 1000 * T

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, getattr(args[-1], "value", args[-1]) or 0))
            return 0

        return call


@pytest.mark.parametrize("call,path", [("forward", "fused"), ("forward", "auto"), ("forward_routed", "auto")])
@pytest.mark.parametrize("raw", [False, True])
def test_memory_comes_from_the_streams_pool(monkeypatch, call, path, raw):
    """Host-side: which stream each buffer is allocated on, against the one the kernels run on."""
    from powerinfer_x64_b200 import moe

    t, lib = _Torch(), _Lib()
    monkeypatch.setattr(moe, "_torch", lambda: t)
    monkeypatch.setattr(moe, "lib", lambda: lib)
    monkeypatch.setattr(moe, "ptr", lambda v: v)
    monkeypatch.setattr(moe, "stream_ptr", lambda s=None: (t.now if s is None else s).cuda_stream)
    monkeypatch.setattr(moe, "raw_stream", lambda device: t.now.cuda_stream)
    monkeypatch.setattr(moe, "torch_stream", lambda s, device: s if hasattr(s, "cuda_stream") else _Stream(s),
                        raising=False)
    L = moe.MoeLayer.__new__(moe.MoeLayer)
    L.ctx = type("Ctx", (), dict(device=0, h=None, check=staticmethod(lambda rc: None)))
    L.n_embd, L.n_expert, L.top_k, L.h, L._fused_ws = 64, 8, 2, None, {}
    x = _Tensor(3 * 64, 0)
    getattr(L, call)(x, path=path, stream=0x70 if raw else _Stream(0x70))
    assert lib.calls and all(s == 0x70 for _, s in lib.calls)
    assert t.made and all(m.pool == 0x70 for m in t.made)
    assert x.recorded == [0x70]
    out, t.made[:] = _Tensor(3 * 64, 0), []
    getattr(L, call)(x, out=out, path=path, stream=_Stream(0x70))
    assert out.recorded == [0x70] and all(m.pool == 0x70 for m in t.made)
    L.h = None


@pytest.mark.gpu
@pytest.mark.parametrize("raw", [False, True])
def test_calls_on_two_streams_without_a_wait(orc, raw):
    """Eager calls on the current stream and on another one, nothing waited for between them, batches of
    many sizes: what one frees the other does not get while it is in use."""
    import torch

    d, f, E, k = 1024, 256, 16, 4
    rng = np.random.default_rng(21)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    xs = torch.from_numpy(rng.standard_normal((16, d)).astype(np.float32)).cuda()
    want = {T: L.forward(xs[:T], rmsnorm=True, path="fused") for T in range(1, 17)}
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for i in range(200):
        T, U = 1 + i % 16, 1 + (7 * i) % 16
        got.append((T, L.forward(xs[:T], rmsnorm=True, path="fused")))
        got.append((U, L.forward(xs[:U], rmsnorm=True, path="fused", stream=side.cuda_stream if raw else side)))
    torch.cuda.synchronize()
    L.ctx.sync_check()
    assert all(torch.equal(y, want[T]) for T, y in got)


@pytest.mark.gpu
def test_host_tokens_and_routing_on_another_stream(orc):
    import torch

    d, f, E, k, T = 1024, 256, 16, 4, 9
    rng = np.random.default_rng(22)
    L = _make(_layer(orc, rng, d, f, E, k, "gated", False), d, f, E, k)
    x = rng.standard_normal((T, d)).astype(np.float32)
    want, routed = L.forward_routed(x)
    fused = L.forward(x, path="fused")
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        a, r = L.forward_routed(x, stream=side.cuda_stream)
        b, c = L.forward(x, stream=side), L.forward(x, path="fused", stream=side)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(a, want) and torch.equal(b, want) and torch.equal(c, fused)
        assert all(torch.equal(r[n], routed[n]) for n in routed)
    y = L.forward(x, path="fused", stream=0)  # the default stream's handle
    torch.cuda.synchronize()
    assert torch.equal(y, fused)

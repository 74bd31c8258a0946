"""Paths that a MoE call does not have are refused as its other arguments are."""
import pytest

from test_moe_streams import _Lib, _Tensor, _Torch


@pytest.mark.parametrize("call,path", [("forward", "fast"), ("forward_routed", "fused"), ("forward_routed", "")])
def test_unknown_paths_are_refused(monkeypatch, call, path):
    from powerinfer_x64_b200 import PiError, moe
    from powerinfer_x64_b200._lib import PI_ERR_ARG

    lib = _Lib()
    monkeypatch.setattr(moe, "_torch", _Torch)
    monkeypatch.setattr(moe, "lib", lambda: lib)
    L = moe.MoeLayer.__new__(moe.MoeLayer)
    L.ctx, L.n_embd, L.n_expert, L.top_k, L.h = None, 64, 8, 2, None
    with pytest.raises(PiError) as e:
        getattr(L, call)(_Tensor(64, 0), path=path)
    assert e.value.code == PI_ERR_ARG and not lib.calls


def test_a_stream_of_another_device_is_refused(monkeypatch):
    """The work would run on that device's idea of the current stream, in no order with the given one."""
    import types

    from powerinfer_x64_b200 import PiError, _lib

    there = types.SimpleNamespace(cuda_stream=0x70, device=types.SimpleNamespace(index=1))
    assert _lib.torch_stream(there, 1) is there
    with pytest.raises(PiError) as e:
        _lib.torch_stream(there, 0)
    assert e.value.code == _lib.PI_ERR_ARG

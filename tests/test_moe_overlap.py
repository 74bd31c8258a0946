"""The fused MoE layer's out may be x; a shifted overlap, which would be a race, is refused."""
import numpy as np
import pytest

from test_moe_few import _layer, _make


@pytest.mark.gpu
def test_shifted_overlap_is_refused(orc):
    import torch

    from powerinfer_x64_b200 import PiError
    from powerinfer_x64_b200._lib import PI_ERR_ARG

    d, f, E, k = 1024, 128, 4, 2
    L = _make(_layer(orc, np.random.default_rng(1), d, f, E, k, None, False), d, f, E, k)
    buf = torch.randn(9, d, device="cuda")
    for x, out in ((buf[0:4], buf[1:5]), (buf[3:7], buf[0:4]), (buf.view(-1)[4:4 + d], buf[0:1])):
        with pytest.raises(PiError) as e:
            L.forward(x, out=out, path="fused")
        assert e.value.code == PI_ERR_ARG
    want = L.forward(buf[0:4], path="fused")
    L.forward(buf[0:4], out=buf[4:8], path="fused")  # next to one another
    assert torch.equal(buf[4:8], want)
    L.forward(buf[0:4], out=buf[0:4], path="fused")
    assert torch.equal(buf[0:4], want)

"""Q4_0 layers of the narrowest documented expert width, against the oracle."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T", [3, 130])
def test_q4_0_layer_of_width_128(orc, T):
    """Width 128 has down rows of four block scales (8 bytes): no tensor map can stride them, so
    the layer must come without the prefill GEMM's maps and still run, decode and prefill."""
    import torch

    from powerinfer_x64_b200 import PiError, moe
    from powerinfer_x64_b200._lib import PI_ERR_ARG
    from test_gpu_parity import close

    d, f, E, k = 1024, 128, 8, 2
    rng = np.random.default_rng(f)
    mk = lambda n: orc.quantize_q4_0((rng.standard_normal(n) * 0.02).astype(np.float32))  # noqa: E731
    router = (rng.standard_normal(E * d) * 0.02).astype(np.float32)
    g, u, dn = mk(E * f * d), mk(E * f * d), mk(E * d * f)
    x = rng.standard_normal((T, d)).astype(np.float32)
    L = moe.MoeLayer(router, g, u, dn, 2, d, f, E, k)
    xd = torch.from_numpy(x).cuda()
    out = L.forward(xd).cpu().numpy()
    n = min(T, 6)
    close(out[:n], orc.moe_layer(x[:n], d, f, E, k, 2, router, g, u, dn, threads=4))
    with pytest.raises(PiError) as e:
        L.forward(xd, path="gemm")
    assert e.value.code == PI_ERR_ARG

"""An adapter bank made from parameters that are being trained."""
import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 5])
def test_a_bank_keeps_no_autograd_history(rank):
    import torch

    from powerinfer_x64_b200.lora import AdapterBank

    a = torch.randn(2, rank, 64, device="cuda", requires_grad=True)
    b = torch.randn(2, 20, rank, device="cuda", requires_grad=True)
    scales = torch.ones(2, device="cuda", requires_grad=True)
    bank = AdapterBank(a, b, scales=scales)
    for _ in range(3):
        bank.set(1, a[0] * 2.0, b[0], 0.5)
    assert not (bank.a.requires_grad or bank.b.requires_grad or bank.scales.requires_grad)
    assert torch.equal(bank.a[1, :rank], 2.0 * a[0]) and torch.equal(bank.b[0, :, :rank], b[0])

"""The gradient of experts that are closed to a row whose other values are no numbers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('experts', [4, 16, 30, 64, 100, 256, 300, 1000])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_a_closed_expert_has_no_gradient(cuda, experts, dtype):
    """d logits is 0 where the mask is off, in rows with an open NaN or infinity and with a gradient that is no number; open
    experts of such a row are NaN, rows beside it are what they are alone."""
    from odie_b200.experts import gate
    g = torch.Generator(device='cuda').manual_seed(experts)
    rows = 41
    logits = torch.randn((rows, experts), generator=g, device='cuda').to(dtype)
    mask = torch.rand((rows, experts), generator=g, device='cuda') < 0.6
    mask[:, 0], mask[:, 1], mask[:, 2] = True, False, True
    d_weights = torch.randn((rows, 2), generator=g, device='cuda')
    bad, bad_d = logits.clone(), d_weights.clone()
    bad[3, 0], bad[7, 2], bad_d[11, 0], bad_d[13, 1] = float('nan'), float('inf'), float('nan'), float('inf')
    bad[5, 1] = float('nan')  # closed: of no effect
    ill = torch.zeros(rows, dtype=torch.bool, device='cuda')
    ill[[3, 7, 11, 13]] = True
    for score, normalize in (('softmax', False), ('softmax', True), ('sigmoid', False), ('sigmoid', True)):
        leaf, clean = bad.clone().requires_grad_(), torch.where(mask, logits, 0.0).requires_grad_()
        (d,) = torch.autograd.grad(gate(leaf, 2, mask=mask, score=score, normalize=normalize).weights, leaf, bad_d)
        (want,) = torch.autograd.grad(gate(clean, 2, mask=mask, score=score, normalize=normalize).weights, clean, d_weights)
        assert (d[~mask] == 0).all(), (score, normalize, d[~mask].isnan().sum().item())
        assert torch.equal(d[~ill], want[~ill])
        if score == 'softmax' and not normalize:
            assert d[[3, 7, 11]][mask[[3, 7, 11]]].isnan().all()

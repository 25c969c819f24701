"""MelInversion in float16: its magnitudes, and gradients of a mean over the batch with the loss scaled as float16 needs it."""
import pytest
import torch

from tacotron2_amd import inversion as inv
from test_inversion import F16, F32, network64, randn, u

gpu = pytest.mark.gpu


def far(a, b):
    return float((a - b).norm() / b.norm())


@gpu
@pytest.mark.parametrize("scale", [2.0 ** 10, 2.0 ** 14])
def test_float16_network_and_its_gradients(scale):
    """About 14 roundings of the type between input and output, as many on the way back, of every gradient between the layers."""
    net = inv.MelInversion(n_mels=80, n_bins=33, channels=64, hidden=128, blocks=2, groups=8, dtype=F16, device="cuda")
    logmel = randn((3, 41, 80), F32, 1).cuda() - 2
    ends = [41, 17, 30]
    live = (torch.arange(41)[None, :] < torch.tensor(ends)[:, None])[:, :, None]
    mag = net(logmel, lengths=ends)
    assert mag.dtype == F32 and (mag > 0).all()
    ((mag.log() * live.cuda()).square().mean() * scale).backward()
    want, p = network64(net, logmel.to(F16), ends)
    ((want.log() * live).square().mean()).backward()
    assert far(mag.detach().double().cpu() * live, want.detach() * live) <= 14 * u(F16)
    for k, v in net.named_parameters():
        assert far(v.grad.double().cpu() / scale, p[k].grad) <= 3 * 14 * u(F16), k


@gpu
def test_float16_last_layer_learns_from_a_mean_over_a_batch():
    """Without a scaled loss: float16 itself would have three bits at most for any dz; the last layer's gradients are sums of them over
    frames and come out as float16 has those.  The layers before it get their gradient through float16."""
    B, T, C, N = 8, 700, 64, 513
    h = (randn((B, T, C), F32, 1).abs() + 0.5).to(F16).cuda()
    w = randn((N, C), F16, 2, 0.1 * C ** -0.5).cuda().requires_grad_()
    b = torch.full((N,), -3.0, dtype=F16, device="cuda").requires_grad_()
    mag = inv.dense(h, w, b, activation="exp", out_dtype=F32)
    (mag * 10).mean().backward()
    w64, b64 = (t.detach().double().cpu().requires_grad_() for t in (w, b))
    (torch.exp(h.double().cpu() @ w64.t() + b64) * 10).mean().backward()
    largest = float(10 * mag.detach().max()) / mag.numel()
    assert largest < 2.0 ** -21
    for got, want in ((w.grad, w64.grad), (b.grad, b64.grad)):
        # one rounding of the result (its smallest step), float32 sums of 5600 frames, exp of a float32 sum of 65 products
        tol = u(F16) * want.abs() + 2.0 ** -25 + ((B * T + 16) * 2.0 ** -23 + 81 * 2.0 ** -23 * 8 + 2.0 ** -20) * want.abs()
        assert ((got.double().cpu() - want).abs() <= tol).all()
        assert (got != 0).all()

"""Gradients of 16-bit dense layers whose dz = dy act'(z) does not fit the type: dy and z kept in float32, and float16's range.

Tolerances.  dz goes into the products in two planes of the type: bfloat16 within (2^-8)^2 |dz| (half a step of what half a step
left), float16 within (2^-11)^2 |dz| while 2^-14 <= |dz| < 128.  Below 2^-14 the higher plane leaves up to 2^-25, or all of dz, of
which the lower one, counting 2^-20, keeps 11 bits: min(2^-25 2^-12, 2^-11 |dz|), and 2^-45 (half its own smallest step, 2^-24)
where those run out.  act' is evaluated to 2^-20 of its scale, sums of n are off by (n + 16) 2^-23 of their magnitudes, and the
result is rounded once; nothing else is."""
import pytest
import torch

from tacotron2_amd import inversion as inv
from test_inversion import BF16, F16, F32, close, randn, scale64, slope64, tiny, u

gpu = pytest.mark.gpu


def gradients64(dy, x, w, z, name, dtype):
    """[(gradient, tolerance)] of dx, dweight, dbias on the device of the arguments."""
    dy, x, w = dy.double(), x.double(), w.double()
    dz = dy * slope64(z.double(), name)
    raw = dy.abs() * scale64(z.double(), name) * 2.0 ** -20 if name else torch.zeros_like(dz)
    off = raw + u(dtype) ** 2 * dz.abs()
    if dtype == F16:
        off = off + (2.0 ** -11 * dz.abs()).clamp(max=2.0 ** -37) + 2.0 ** -45
    M, N = dz.shape
    sums = ((dz @ w, off @ w.abs() + (N + 16) * 2.0 ** -23 * (dz.abs() @ w.abs())),
            (dz.t() @ x, off.t() @ x.abs() + (M + 16) * 2.0 ** -23 * (dz.abs().t() @ x.abs())),
            (dz.sum(0), raw.sum(0) + (M + 16) * 2.0 ** -23 * dz.abs().sum(0)))
    return [(v, t + u(dtype) * (v.abs() + t) + tiny(dtype)) for v, t in sums]


def check(dy, x, w, z, name, dtype, shift=lambda t: t):
    want = gradients64(dy, x, w, z, name, dtype)
    got = inv.dense_backward(shift(dy), shift(x), shift(w), shift(z) if name else None, activation=name)
    for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
        assert g.dtype == dtype
        close(g, v.cpu(), t.cpu(), what)
    return got


# one launch (few frames, odd widths), 64 and 128 tiles, the walking kernel's three layouts, contractions in parts
SIZES = [(1, 512, 1025), (7, 33, 70), (641, 80, 512), (300, 1001, 300), (2600, 136, 328), (2100, 512, 513), (9001, 130, 257),
         (16500, 512, 264), (33000, 256, 1024), (40000, 512, 96)]


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("name", [None, "silu", "exp"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_float32_dy_is_not_rounded_to_the_type(M, K, N, name, dtype):
    x, w = randn((M, K), dtype, 1).cuda(), randn((N, K), dtype, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), F32, 3).cuda(), randn((M, N), F32, 4, 0.1).cuda()
    got = check(dy, x, w, z, name, dtype)
    for k in range(3):                                       # one at a time, the same bits
        need = [j == k for j in range(3)]
        one = inv.dense_backward(dy, x, w, z if name else None, activation=name, needs=need)
        assert torch.equal(one[k], got[k])


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,N", [(70, 65, 30), (9000, 520, 600), (20000, 256, 512)])
def test_float32_dy_off_its_alignment(M, K, N, dtype):
    """Operands that start one element off: the kernel that reads the planes element by element."""
    def off(t):
        flat = torch.full((t.numel() + 1,), float("nan"), dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    x, w = randn((M, K), dtype, 1).cuda(), randn((N, K), dtype, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), F32, 3).cuda(), randn((M, N), F32, 4, 0.1).cuda()
    check(dy, x, w, z, "gelu", dtype, off)


@gpu
@pytest.mark.parametrize("name", ["relu", "silu", "gelu", "tanh", "exp"])
@pytest.mark.parametrize("M,K,N", [(641, 80, 512), (2600, 136, 328), (33000, 256, 512)])
def test_float16_layers_round_their_results_alone(M, K, N, name):
    x, w = randn((M, K), F16, 1).cuda(), randn((N, K), F16, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), F16, 3).cuda(), randn((M, N), F16, 4, 0.1).cuda()
    check(dy, x, w, z, name, F16)


@gpu
@pytest.mark.parametrize("dtype,od", [(F16, F16), (BF16, F32)])
@pytest.mark.parametrize("M", [32980, 32960, 33025])
def test_planes_change_inside_a_pair_of_steps(M, dtype, od):
    """The walking kernel takes steps of 32 frames in twos; the last part of these has an odd number of them a plane."""
    K, N = 512, 2048
    x, w = randn((M, K), dtype, 1).cuda(), randn((N, K), dtype, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), od, 3).cuda(), randn((M, N), od, 4, 0.1).cuda()
    check(dy, x, w, z, "silu", dtype)


@gpu
@pytest.mark.parametrize("dy_dtype,size", [(F32, 1.8e-8), (F16, 4e-6)])
@pytest.mark.parametrize("M,K,N", [(3000, 64, 64), (30000, 512, 513), (30000, 512, 512), (30000, 72, 256)])
def test_float16_gradients_below_its_range_reach_the_sums(M, K, N, dy_dtype, size):
    """A mean over a batch's magnitudes: most dz are below half of float16's smallest step, their sums over the frames are not."""
    x = (randn((M, K), F32, 1).abs() + 1).to(F16).cuda()
    w = randn((N, K), F16, 2, K ** -0.5).cuda()
    z = (randn((M, N), F32, 3, 0.5) - 7).to(dy_dtype).cuda()
    dy = ((randn((M, N), F32, 4).abs() + 0.5) * size).to(dy_dtype).cuda()
    up = dy if dy_dtype == F16 else dy * 64                  # frames for the smaller of the two
    assert float((up.double() * torch.exp(z.double())).median()) < 2.0 ** -25
    dw = check(up, x, w, z, "exp", F16)[1]
    assert (dw > 0).all()


@gpu
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("M,K,N", [(70, 65, 30), (16500, 512, 264), (2600, 136, 328)])
def test_values_that_are_not_finite_stay_in_their_rows(M, K, N, dtype):
    x, w = randn((M, K), dtype, 1).abs().cuda() + 0.1, randn((N, K), dtype, 2).abs().cuda() + 0.1
    dy = randn((M, N), F32, 3).cuda()
    want = gradients64(dy, x, w, torch.zeros_like(dy), None, dtype)
    dy[7, 3], dy[M - 9, N - 2] = float("inf"), float("nan")
    dx, dw, db = inv.dense_backward(dy, x, w)
    assert (dx[7] == float("inf")).all() and dx[M - 9].isnan().all()
    assert (dw[3] == float("inf")).all() and dw[N - 2].isnan().all()
    assert db[3] == float("inf") and db[N - 2].isnan()
    for got, (v, t), gone, what in ((dx, want[0], (7, M - 9), "dx"), (dw, want[1], (3, N - 2), "dweight")):
        rest = torch.ones(got.shape[0], dtype=torch.bool, device="cuda")
        rest[list(gone)] = False
        close(got[rest], v[rest].cpu(), t[rest].cpu(), what)

"""float32 products through 16-bit planes with their contraction in parts: sums that the planes do not give."""
import pytest
import torch

from tacotron2_amd import inversion as inv
from test_inversion import F32, close, dense64, randn

gpu = pytest.mark.gpu


def microseconds(f, n=5):
    f()
    best = float("inf")
    for _ in range(3):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        b.synchronize()
        best = min(best, a.elapsed_time(b) * 1000 / n)
    return best


@gpu
@pytest.mark.parametrize("K,N", [(512, 264), (130, 257), (512, 512)])
def test_one_infinite_gradient_costs_little_more_than_none(K, N):
    """A row of dweight is infinite then, over all frames: not a loop over them in one thread each."""
    M = 40000
    x, w, dy = randn((M, K), F32, 1).cuda(), randn((N, K), F32, 2).cuda(), randn((M, N), F32, 3).cuda()
    call = lambda: inv.dense_backward(dy, x, w, needs=(False, True, True))               # noqa: E731
    clean = call()[1].clone()
    before = microseconds(call)
    dy[7, 3], dy[M - 1, N - 1] = float("inf"), float("nan")
    dw = call()[1]
    assert torch.equal(dw[3], float("inf") * x[7]) and dw[N - 1].isnan().all()
    rest = [n for n in range(N) if n not in (3, N - 1)]
    size = dy[:, rest].abs().double().t() @ x.abs().double()                             # two ways of the same sums
    assert ((dw[rest] - clean[rest]).abs().double() <= 2 * (M + 16) * 2.0 ** -23 * size).all()
    assert torch.equal(dw.nan_to_num(9), call()[1].nan_to_num(9))
    after = microseconds(call)
    print(f"{before:.0f} us, with one infinity {after:.0f} us")
    assert after <= 8 * before


@gpu
@pytest.mark.parametrize("M,K,N", [(64, 16384, 2064), (64, 16384, 264), (300, 20001, 257)])
def test_blocks_below_their_rows_range_in_parts(M, K, N):
    """Rows of 60 powers of two: blocks of the result come from the operands, in parts; the residual is the result's own memory."""
    x, w, r = randn((M, K), F32, 1).cuda(), randn((N, K), F32, 2).cuda(), randn((M, N), F32, 4).cuda()
    w[:, 0] = 0.0
    x[::5, 0], x[::5, 1:] = 1e10, x[::5, 1:] * 1e-8
    x[M - 1, 5] = float("inf")
    w[:, 5] = w[:, 5].abs() + 0.1
    keep = r.clone()
    z = torch.empty_like(r)
    y = inv.dense(x, w, activation="tanh", residual=r, out=r, preactivation=z)
    assert (z[M - 1] == float("inf")).all() and torch.equal(y[M - 1], keep[M - 1] + 1)
    z64, z_tol, y64, y_tol = dense64(x[:M - 1], w, None, "tanh", keep[:M - 1], F32)
    close(z[:M - 1], z64.cpu(), z_tol.cpu(), "preactivation")
    close(y[:M - 1], y64.cpu(), y_tol.cpu(), "y")
    for _ in range(3):
        assert torch.equal(y, inv.dense(x, w, activation="tanh", residual=keep))


@gpu
def test_planes_hold_float32_to_a_step():
    """Values over all of a binade times one: 2^-23 of the planes, and 2^-23 of the sum, which a matrix instruction may cut off instead of
    rounding it.  Times each other: 2^-23 of either side's planes, twice 2^-23 for the product of the lower planes that is left out
    (2^-11 of a value each), 2^-23 of the sum: 5 of them (computed with exact planes and a cut-off sum on the CPU: 4.98)."""
    M, N = 2048, 1024
    steps = torch.arange(M * N, dtype=torch.float64).view(M, N) * 4 + 1
    x = ((1 + steps * 2.0 ** -23) * 2.0 ** (torch.arange(M) % 31 - 15)[:, None]).float()
    y = inv.dense(x.cuda(), torch.eye(N, device="cuda")).cpu()
    assert ((y.double() - x.double()).abs() <= 2 * 2.0 ** -23 * x.double()).all()
    both = (x.double() * x[0].double()[None, :])                                         # both factors rounded
    y = inv.dense(x.cuda(), torch.diag(x[0]).cuda()).cpu()
    assert ((y.double() - both).abs() <= 5 * 2.0 ** -23 * both).all()

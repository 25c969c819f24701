"""Dense layers and group norms of the learned mel inversion, their gradients and the network made of them, against
64-bit statements of the same formulas.

Tolerances.  u(t) = eps(t) / 2 is one rounding to type t.  A sum of n products in 32 bits is off by at most
(n + 16) 2^-23 times the sum of their magnitudes (twice the bound of a chain of correctly rounded additions: a matrix
instruction need not round every addition to nearest).  An activation or its derivative is evaluated to 2^-20 of the
larger of its value and its scale.  Every bound below is the sum of these along the formula; nothing is fitted."""
import ctypes
import math

import pytest
import torch

from tacotron2_amd import _lib
from tacotron2_amd import inversion as inv

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
ACTS = [None, "relu", "silu", "gelu", "tanh", "exp"]
gpu = pytest.mark.gpu


def u(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps      # one step of the subnormal range


def act64(z, name):
    return {None: lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * 0.5 * torch.special.erfc(-z / math.sqrt(2)), "tanh": lambda: torch.tanh(z),
            "exp": lambda: torch.exp(z)}[name]()


def slope64(z, name):
    if name is None:
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "tanh":
        return 1 - torch.tanh(z) ** 2
    return torch.exp(z)


def scale64(z, name):
    """What an error of the argument is multiplied by, and what the evaluation's 2^-20 is relative to."""
    if name == "exp":
        return torch.exp(z)
    return torch.full_like(z, 1.13)                       # the steepest of silu' (1.10), gelu' (1.13), tanh', relu'


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g, dtype=torch.float64) * scale).to(dtype)


def close(got, want, tol, what):
    got = got.detach().double().cpu()
    bad = ~((got - want).abs() <= tol)
    if bad.any():
        k = int(((got - want).abs() / tol.clamp_min(1e-300)).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; worst {got.flatten()[k]:.9g} against "
                             f"{want.flatten()[k]:.9g} (tolerance {tol.flatten()[k]:.3g})")


# -- dense -----------------------------------------------------------------------------------------------------
def dense64(x, w, b, name, r, out_dtype):
    """(z, its tolerance, y, its tolerance) in 64 bits; tolerances for results of out_dtype."""
    x, w = x.double(), w.double()
    b = torch.zeros(w.shape[0], dtype=torch.float64, device=w.device) if b is None else b.double()
    z = x @ w.t() + b
    size = x.abs() @ w.abs().t() + b.abs()
    off = (w.shape[1] + 16) * 2.0 ** -23 * size
    y = act64(z, name)
    y_off = scale64(z + off, name) * (off + 2.0 ** -20) if name else off
    if r is not None:
        y = y + r.double()
        y_off = y_off + 2.0 ** -24 * y.abs()
    return z, off + u(out_dtype) * z.abs() + tiny(out_dtype), y, y_off + u(out_dtype) * (y.abs() + y_off) + tiny(out_dtype)


DENSE_SIZES = [(1, 1, 1), (1, 512, 1025), (2, 80, 513), (3, 7, 33), (8, 1024, 1024), (16, 96, 250), (7, 828, 188), (4, 1910, 130), (3, 1911, 70), (8, 40, 33), (5, 64, 70), (6, 9, 20), (2, 8, 9), (17, 31, 65), (33, 64, 64),
               (64, 64, 64), (65, 128, 200), (128, 256, 256), (129, 513, 96), (257, 264, 520), (641, 80, 512), (300, 1024, 256),
               (1100, 72, 1025), (2600, 136, 328)]


@gpu
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("M,K,N", DENSE_SIZES)
def test_dense_sizes(M, K, N, dtype, out_dtype):
    name = ACTS[(M + K + N) % len(ACTS)]
    x, w, b = randn((M, K), dtype, 1), randn((N, K), dtype, 2, K ** -0.5), randn((N,), dtype, 3)
    r = randn((M, N), out_dtype, 4)
    z64, z_tol, y64, y_tol = dense64(x, w, b, name, r, out_dtype)
    z = torch.full((M, N), float("nan"), dtype=out_dtype, device="cuda")
    y = inv.dense(x.cuda(), w.cuda(), b.cuda(), activation=name, residual=r.cuda(), out_dtype=out_dtype, preactivation=z)
    assert y.dtype == out_dtype
    close(y, y64, y_tol, "y")
    close(z, z64, z_tol, "preactivation")
    plain = inv.dense(x.cuda(), w.cuda(), out_dtype=out_dtype)                       # no bias, activation, residual
    z64, z_tol, _, _ = dense64(x, w, None, None, None, out_dtype)
    close(plain, z64, z_tol, "product")
    assert torch.equal(plain, inv.dense(x.cuda(), w.cuda(), out_dtype=out_dtype))    # equal calls, equal bits


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("name", ACTS)
def test_dense_activations_over_their_range(name, dtype):
    # one input of weight 1: z runs over the range itself, the far ends included
    ends = torch.tensor([0.0, -0.0, 1e-6, -1e-6, 30.0, -30.0, 80.0, -80.0, 88.0, -100.0])
    z = torch.cat([torch.linspace(-12, 12, 1001), ends]).to(dtype)[:, None]
    one = torch.ones((1, 1), dtype=dtype)
    _, _, y64, y_tol = dense64(z, one, None, name, None, dtype)
    y64 = y64.to(dtype).double() if dtype == F16 else y64                            # exp past 65504 is inf in f16
    y = inv.dense(z.cuda(), one.cuda(), activation=name).double().cpu()
    both = torch.isinf(y) & torch.isinf(y64)
    close(torch.where(both, 0.0, y), torch.where(both, 0.0, y64), torch.where(both, 1.0, y_tol), "y")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(5, 80, 65), (130, 264, 192), (700, 136, 200)])
def test_dense_strides_and_offsets(M, K, N, dtype):
    """Rows inside wider buffers, odd offsets, transposed weights, broadcast residuals; what lies between rows stays."""
    x, w, b, r = randn((M, K), dtype, 1), randn((N, K), dtype, 2, K ** -0.5), randn((N,), dtype, 3), randn((M, N), dtype, 4)
    _, _, y64, y_tol = dense64(x, w, b, "silu", r, dtype)

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), dtype=dtype, device="cuda")
        wide[:, left:left + t.shape[1]] = t.cuda()
        return wide[:, left:left + t.shape[1]], wide

    for left, right in ((0, 8), (8, 0), (1, 2), (3, 0)):
        xs, _ = inside(x, left, right)
        ws, _ = inside(w, right, left)
        rs, _ = inside(r, left, left)
        ys, wide = inside(torch.zeros(M, N), left, right)
        bs = torch.cat([torch.zeros(left, dtype=dtype), b]).cuda()[left:]
        assert inv.dense(xs, ws, bs, activation="silu", residual=rs, out=ys).data_ptr() == ys.data_ptr()
        close(ys, y64, y_tol, f"y at {left}, {right}")
        assert wide[:, :left].isnan().all() and wide[:, left + N:].isnan().all()
    wt = w.cuda().t().contiguous().t()                                               # columns contiguous: copied first
    close(inv.dense(x.cuda(), wt, b.cuda(), activation="silu", residual=r.cuda()), y64, y_tol, "transposed weight")
    acc = r.cuda().clone()                                                           # the residual stream in place
    close(inv.dense(x.cuda(), w.cuda(), b.cuda(), activation="silu", residual=acc, out=acc), y64, y_tol, "in place")
    x3 = x.cuda().view(1, M, 1, K).expand(2, M, 1, K)                                # (..., K) with a broadcast batch
    y3 = inv.dense(x3, w.cuda(), b.cuda(), activation="silu", residual=r.cuda().view(1, M, 1, N).expand(2, M, 1, N))
    close(y3[1, :, 0], y64, y_tol, "leading dimensions")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_dense_far_rows(dtype):
    """Rows more than 2^32 bytes apart."""
    stride = (1 << 31) + 8 if dtype == BF16 else (1 << 30) + 8
    K, N = 64, 72
    if stride > 1 << 31:
        stride = 1 << 31
    x, w = randn((2, K), dtype, 1), randn((N, K), dtype, 2)
    big = torch.empty(stride + 128, dtype=dtype, device="cuda")
    xs = big.as_strided((2, K), (stride, 1))
    xs.copy_(x)
    z64, z_tol, _, _ = dense64(x, w, None, None, None, dtype)
    close(inv.dense(xs, w.cuda()), z64, z_tol, "far x")
    ys = big.as_strided((2, N), (stride, 1))
    inv.dense(x.cuda(), w.cuda(), out=ys)
    close(ys, z64, z_tol, "far y")
    for rows in (2, 40):                                     # weight rows as far apart, few rows and a tile of them
        ws = big.as_strided((2, K), (stride, 1))
        ws.copy_(w[:2])
        xr = randn((rows, K), dtype, 5)
        z64, z_tol, _, _ = dense64(xr, w[:2], None, None, None, dtype)
        close(inv.dense(xr.cuda(), ws), z64, z_tol, "far weight")
        close(inv.dense_backward(torch.ones(rows, 2, dtype=dtype, device="cuda"), xr.cuda(), ws)[0],
              w[:2].double().sum(0).expand(rows, K), 0.02 * w[:2].double().abs().sum(0).expand(rows, K) + 1e-6, "far dx")


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_dense_infinities_stay_in_their_rows(dtype):
    M, K, N = 70, 96, 80
    x, w = randn((M, K), dtype, 1), randn((N, K), dtype, 2).abs()
    x[3, 5], x[40, 0], x[66, 95] = float("inf"), float("nan"), -float("inf")
    y = inv.dense(x.cuda(), w.cuda()).cpu()
    assert torch.isinf(y[3]).all() and (y[3] > 0).all() and torch.isinf(y[66]).all() and (y[66] < 0).all()
    assert y[40].isnan().all()
    rest = [i for i in range(M) if i not in (3, 40, 66)]
    z64, z_tol, _, _ = dense64(x[rest], w, None, None, None, dtype)
    close(y[rest], z64, z_tol, "other rows")


def dense_back64(dy, x, w, z, name, dtype):
    dy, x, w = dy.double(), x.double(), w.double()
    dz = dy if name is None else dy * slope64(z.double(), name)
    raw = torch.zeros_like(dz) if name is None else dy.abs() * scale64(z.double(), name) * 2.0 ** -20
    off = raw + u(dtype) * dz.abs() + tiny(dtype)                             # dz is rounded to dtype for the products
    M, N = dz.shape
    dx, dx_tol = dz @ w, off @ w.abs() + (N + 16) * 2.0 ** -23 * (dz.abs() @ w.abs())
    dw, dw_tol = dz.t() @ x, off.t() @ x.abs() + (M + 16) * 2.0 ** -23 * (dz.abs().t() @ x.abs())
    db, db_tol = dz.sum(0), raw.sum(0) + (M + 16) * 2.0 ** -23 * dz.abs().sum(0)
    return [(v, t + u(dtype) * (v.abs() + t) + tiny(dtype)) for v, t in ((dx, dx_tol), (dw, dw_tol), (db, db_tol))]


@gpu
@pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)])
@pytest.mark.parametrize("M,K,N", DENSE_SIZES)
def test_dense_backward_sizes(M, K, N, dtype, out_dtype):
    name = ACTS[(M + K + N + 1) % len(ACTS)]
    x, w = randn((M, K), dtype, 1), randn((N, K), dtype, 2, K ** -0.5)
    z, dy = randn((M, N), out_dtype, 3), randn((M, N), out_dtype, 4)
    want = dense_back64(dy, x, w, z, name, dtype)
    got = inv.dense_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda() if name else None, activation=name)
    for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
        assert g.dtype == dtype
        close(g, v, t, what)
    again = inv.dense_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda() if name else None, activation=name)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    for k in range(3):                                                        # one at a time, the same bits
        need = [j == k for j in range(3)]
        one = inv.dense_backward(dy.cuda(), x.cuda(), w.cuda(), z.cuda() if name else None, activation=name, needs=need)
        assert torch.equal(one[k], got[k]) and all(one[j] is None for j in range(3) if j != k)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("name", [None, "gelu"])
@pytest.mark.parametrize("M,K,N", [(5, 80, 65), (130, 264, 192), (700, 136, 200)])
def test_dense_backward_strides(M, K, N, name, dtype):
    x, w = randn((M, K), dtype, 1), randn((N, K), dtype, 2, K ** -0.5)
    z, dy = randn((M, N), dtype, 3), randn((M, N), dtype, 4)
    want = dense_back64(dy, x, w, z, name, dtype)

    def inside(t, left, right):
        wide = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), dtype=dtype, device="cuda")
        wide[:, left:left + t.shape[1]] = t.cuda()
        return wide[:, left:left + t.shape[1]], wide

    for left, right in ((8, 0), (1, 2)):
        dx, dx_wide = inside(torch.zeros(M, K), left, right)
        dw, dw_wide = inside(torch.zeros(N, K), left, right)
        db = torch.zeros(N + left, dtype=dtype, device="cuda")[left:]
        got = inv.dense_backward(inside(dy, left, right)[0], inside(x, left, right)[0], inside(w, left, right)[0],
                                 inside(z, left, right)[0] if name else None, activation=name, dx=dx, dweight=dw, dbias=db)
        for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
            close(g, v, t, what)
        for wide, n in ((dx_wide, K), (dw_wide, K)):
            assert wide[:, :left].isnan().all() and wide[:, left + n:].isnan().all()


# sizes whose tiles fill the chip: the walking kernel (both sides' layouts), a rest of columns, odd and short contractions
LARGE_SIZES = [(4400, 512, 2048), (33000, 96, 257), (16500, 544, 512), (40000, 32, 256), (33001, 72, 256), (70000, 64, 264), (65500, 64, 256),
               (33000, 130, 600)]


@gpu
@pytest.mark.parametrize("dtype,out_dtype,name,extra", [(BF16, BF16, "gelu", False), (F16, F32, "exp", False), (F16, F16, "silu", True),
                                                        (BF16, F32, None, True), (F32, F32, "tanh", True)])
@pytest.mark.parametrize("M,K,N", LARGE_SIZES)
def test_dense_many_rows(M, K, N, dtype, out_dtype, name, extra):
    """The 64-bit side runs on the GPU here (plain float64 products)."""
    x, w, b = (t.cuda() for t in (randn((M, K), dtype, 1), randn((N, K), dtype, 2, K ** -0.5), randn((N,), dtype, 3)))
    r = randn((M, N), out_dtype, 4).cuda() if extra else None
    z = torch.full((M, N), float("nan"), dtype=out_dtype, device="cuda") if extra else None
    z64, z_tol, y64, y_tol = dense64(x, w, b, name, r, out_dtype)
    y = inv.dense(x, w, b, activation=name, residual=r, out_dtype=out_dtype, preactivation=z)
    close(y, y64.cpu(), y_tol.cpu(), "y")
    if extra:
        close(z, z64.cpu(), z_tol.cpu(), "preactivation")
        inv.dense(x, w, b, activation=name, residual=r, out_dtype=out_dtype, out=r)
        assert torch.equal(r, y)                                              # the residual stream in place


@gpu
@pytest.mark.parametrize("dtype,out_dtype,name", [(BF16, BF16, "gelu"), (F16, F32, "silu"), (BF16, BF16, None), (F32, F32, "gelu")])
@pytest.mark.parametrize("M,K,N", [(9001, 1024, 1024), (16500, 512, 264), (33000, 256, 1025), (16400, 264, 512)])
def test_dense_backward_many_rows(M, K, N, dtype, out_dtype, name):
    x, w = randn((M, K), dtype, 1).cuda(), randn((N, K), dtype, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), out_dtype, 3).cuda(), randn((M, N), out_dtype, 4).cuda()
    want = dense_back64(dy, x, w, z, name, dtype)
    got = inv.dense_backward(dy, x, w, z if name else None, activation=name)
    for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
        close(g, v.cpu(), t.cpu(), what)
    again = inv.dense_backward(dy, x, w, z if name else None, activation=name)
    assert all(torch.equal(a, c) for a, c in zip(got, again))


@gpu
def test_dense_full_precision_values_that_are_not_finite():
    """Large float32 products run on 16-bit planes: what those cannot hold has to come out as float32 has it."""
    M, K, N = 4400, 512, 2048
    x, w = randn((M, K), F32, 1).cuda(), randn((N, K), F32, 2, K ** -0.5).abs().cuda()
    z64, z_tol, _, _ = dense64(x, w, None, None, None, F32)
    x[3, 5], x[2000, 100], x[M - 1, K - 1] = float("inf"), float("nan"), -float("inf")
    y = inv.dense(x, w)
    assert (y[3] == float("inf")).all() and y[2000].isnan().all() and (y[M - 1] == -float("inf")).all()
    rest = torch.ones(M, dtype=torch.bool, device="cuda")
    rest[[3, 2000, M - 1]] = False
    close(y[rest], z64[rest].cpu(), z_tol[rest].cpu(), "the other rows")
    x = randn((M, K), F32, 1).cuda()
    x[50], x[51], x[4000] = 0.0, 0.0, 0.0
    x[50, 7], x[51, 8], x[4000, 9] = 3.4e38, -torch.finfo(F32).max, 1e-30        # the first two round up to infinity in 16 bits
    z64, z_tol, _, _ = dense64(x, w, None, None, None, F32)
    close(inv.dense(x, w), z64.cpu(), z_tol.cpu(), "product")


@gpu
@pytest.mark.parametrize("M,K,N", [(4400, 512, 2048), (64, 16384, 2064), (9000, 513, 600), (30000, 264, 1024)])
def test_dense_full_precision_over_wide_ranges(M, K, N):
    """Rows whose small values alone reach the result: a large one times zero, magnitudes over the range of float32."""
    x, w, b = randn((M, K), F32, 1).cuda(), randn((N, K), F32, 2).cuda(), randn((N,), F32, 3).cuda()
    r = randn((M, N), F32, 4).cuda()
    w[:, 0] = 0.0
    w[5] *= 2.0 ** torch.linspace(-80, 20, K, device="cuda").round()
    w[N - 1], w[7] = 0.0, 1e-38
    x[1] *= 1e-8
    x[1, 0] = 1e10                                        # 60 powers of two above the rest, times zero
    x[40] *= 2.0 ** torch.linspace(-60, 30, K, device="cuda").round()
    x[41], x[42] = 0.0, torch.finfo(F32).smallest_normal * torch.rand(K, device="cuda")
    x[M - 1] *= 1e30
    z64, z_tol, y64, y_tol = dense64(x, w, None, None, None, F32)
    # a product below the normal range is rounded (or flushed) there: one smallest normal number each at most
    low = K * torch.finfo(F32).smallest_normal
    close(inv.dense(x, w), z64.cpu(), z_tol.cpu() + low, "product")
    z64, z_tol, y64, y_tol = dense64(x, w, b, "silu", r, F32)
    keep = r.clone()
    z = torch.empty_like(r)
    got = inv.dense(x, w, b, activation="silu", residual=r, preactivation=z, out=r)
    close(z, z64.cpu(), z_tol.cpu() + low, "preactivation")
    close(got, y64.cpu(), y_tol.cpu() + 2 * low, "y")
    assert torch.equal(got, inv.dense(x, w, b, activation="silu", residual=keep))


@gpu
def test_dense_backward_full_precision_values_that_are_not_finite():
    M, K, N = 16500, 512, 264                                                  # dweight: parts of the frames, joined
    x, w, dy = randn((M, K), F32, 1).cuda(), randn((N, K), F32, 2).cuda(), randn((M, N), F32, 3).cuda()
    want = dense_back64(dy, x, w, None, None, F32)
    dy[7, 3], dy[16000, 200] = float("inf"), float("nan")
    dx, dw, db = inv.dense_backward(dy, x, w)
    assert torch.equal(dx[7], float("inf") * w[3]) and dx[16000].isnan().all()
    assert torch.equal(dw[3], float("inf") * x[7]) and dw[200].isnan().all()
    assert db[3] == float("inf") and db[200].isnan()
    for got, (v, t), gone, what in ((dx, want[0], (7, 16000), "dx"), (dw, want[1], (3, 200), "dweight"), (db, want[2], (3, 200), "dbias")):
        rest = torch.ones(got.shape[0], dtype=torch.bool, device="cuda")
        rest[list(gone)] = False
        close(got[rest], v[rest].cpu(), t[rest].cpu(), what)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(70, 1, 1), (70, 1, 3), (70, 5, 1), (1, 1, 9), (1, 9, 1), (200, 2, 130)])
@pytest.mark.parametrize("apart", [0, 4])
def test_dense_backward_narrow(M, K, N, apart, dtype):
    """One column, next to each other or a stride apart: which direction is contiguous does not show in the strides."""
    def view(t, more):
        wide = torch.full((t.shape[0], t.shape[1] + more), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, :t.shape[1]] = t.cuda()
        return wide[:, :t.shape[1]]

    x, w = randn((M, K), dtype, 1), randn((N, K), dtype, 2)
    z, dy = randn((M, N), dtype, 3), randn((M, N), dtype, 4)
    want = dense_back64(dy, x, w, z, "silu", dtype)
    for mix in ((0, apart), (apart, 0), (apart, apart)):
        got = inv.dense_backward(view(dy, mix[0]), view(x, mix[1]), view(w, mix[0]), view(z, mix[1]), activation="silu")
        for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
            close(g, v, t, what)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M,K,N", [(9000, 520, 600), (20000, 257, 512), (33000, 130, 257)])
def test_dense_many_rows_off_their_alignment(M, K, N, dtype):
    """Sizes of the large tiles whose operands start one element off: copied where a copy helps, else element by element."""
    def off(t):
        flat = torch.full((t.numel() + 1,), float("nan"), dtype=dtype, device="cuda")
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    x, w = randn((M, K), dtype, 1).cuda(), randn((N, K), dtype, 2, K ** -0.5).cuda()
    z, dy = randn((M, N), dtype, 3).cuda(), randn((M, N), dtype, 4).cuda()
    _, _, y64, y_tol = dense64(x, w, None, "silu", None, dtype)
    out = off(torch.zeros(M, N, dtype=dtype, device="cuda"))
    close(inv.dense(off(x), off(w), activation="silu", out=out), y64.cpu(), y_tol.cpu(), "y")
    want = dense_back64(dy, x, w, z, "silu", dtype)
    got = inv.dense_backward(off(dy), off(x), off(w), off(z), activation="silu")
    for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
        close(g, v.cpu(), t.cpu(), what)


@gpu
def test_dense_without_rows():
    w, b = torch.randn(6, 5, device="cuda"), torch.randn(6, device="cuda")
    x = torch.empty((2, 0, 5), device="cuda")
    assert inv.dense(x, w, b, activation="relu").shape == (2, 0, 6)
    dx, dw, db = inv.dense_backward(torch.empty((2, 0, 6), device="cuda"), x, w)
    assert dx.shape == (2, 0, 5) and not dw.any() and not db.any() and dw.shape == (6, 5) and db.shape == (6,)


# -- group norm ------------------------------------------------------------------------------------------------
def norm64(x, G, ga, be, eps, name, ends):
    """Forward in 64 bits: (y, tolerance before its rounding, xh, mean, rstd, (B, T, 1) mask)."""
    x = x.double()
    B, T, C = x.shape
    n = C // G
    mask = torch.arange(T)[None, :] < torch.tensor(ends)[:, None]
    mean, rstd = torch.zeros(B, G).double(), torch.zeros(B, G).double()
    size = torch.zeros(B, G).double()
    for b, e in enumerate(ends):
        if e > 0:
            rows = x[b, :e].reshape(e, G, n)
            mean[b] = rows.mean((0, 2))
            rstd[b] = 1 / torch.sqrt(rows.var((0, 2), unbiased=False) + eps)
            size[b] = rows.abs().mean((0, 2))
    wide = lambda v: v[:, None, :, None].expand(B, T, G, n).reshape(B, T, C)          # noqa: E731
    xl = torch.where(mask[:, :, None], x, 0.0)
    xh = (xl - wide(mean)) * wide(rstd)
    # mean and deviations in 32 bits, sums of pairs of partial sums: 64 roundings cover their depth at these sizes
    xh_off = wide(rstd) * 2.0 ** -24 * (64 * wide(size) + 2 * xl.abs()) + 2.0 ** -18 * xh.abs()
    ga = torch.ones(C).double() if ga is None else ga.double()
    be = torch.zeros(C).double() if be is None else be.double()
    z = xh * ga + be
    z_off = xh_off * ga.abs() + 2.0 ** -23 * ((xh * ga).abs() + be.abs())
    y = act64(z, name)
    y_off = scale64(z + z_off, name) * (z_off + 2.0 ** -20) if name else z_off
    m = mask[:, :, None].double()
    return y * m, y_off * m, xh, xh_off, mean, rstd, m


NORM_SIZES = [(1, 1, 1, 1), (1, 1, 32, 32), (1, 1, 512, 32), (2, 2, 6, 2), (3, 5, 35, 5), (1, 641, 512, 32), (4, 33, 96, 4),
              (2, 100, 80, 1), (3, 17, 1025, 1), (2, 300, 24, 8), (1, 2049, 16, 16), (5, 64, 256, 8), (2, 7, 2048, 2),
              (1, 9000, 40, 2), (8, 257, 512, 32), (1, 5000, 512, 1), (2, 900, 500, 5), (2, 70, 36, 4), (3, 50, 26, 2), (1, 3000, 250, 2),
              (3, 40, 4, 4), (2, 1200, 1022, 1), (2, 300, 2050, 2), (1, 90, 4098, 2049), (5, 40, 1027, 13)]


def ends_of(B, T, ragged):
    if not ragged:
        return [T] * B
    return [[T, 0, 1, (T + 1) // 2, max(T - 1, 0), min(T, 7), T, min(T, 2)][b % 8] for b in range(B)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,T,C,G", NORM_SIZES)
def test_group_norm_sizes(B, T, C, G, ragged, dtype):
    name = ACTS[(B + T + C + G) % len(ACTS)]
    ends = ends_of(B, T, ragged)
    x = (randn((B, T, C), F32, 1) + randn((1, 1, C), F32, 2)).to(dtype)
    ga, be = (randn((C,), F32, 3) * 0.2 + 1).to(dtype), randn((C,), dtype, 4, 0.3)
    y64, off, _, _, mean, rstd, m = norm64(x, G, ga, be, 1e-5, name, ends)
    xc = x.cuda()
    for b, e in enumerate(ends):
        xc[b, e:] = float("nan")                                      # what is masked is not read
    lengths = torch.tensor(ends, dtype=torch.int32, device="cuda") if ragged else None
    stats = torch.full((B, G, 2), float("nan"), device="cuda")
    y = inv.group_norm(xc, G, ga.cuda(), be.cuda(), activation=name, lengths=lengths, stats=stats)
    close(y, y64, off + u(dtype) * (y64.abs() + off) + tiny(dtype), "y")
    close(stats[..., 0], mean, 2.0 ** -18 * x.double().abs().max() + 0 * mean, "mean")
    close(stats[..., 1], rstd, 2.0 ** -17 * rstd, "rstd")
    assert torch.equal(y, inv.group_norm(xc, G, ga.cuda(), be.cuda(), activation=name, lengths=ends if ragged else None))
    assert inv.group_norm(xc, G, ga.cuda(), be.cuda(), activation=name, lengths=lengths, out=xc) is xc
    assert torch.equal(xc, y)                                         # in place


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_level_far_above_its_spread(dtype):
    """Mean 1000, deviation 1 (8 in bf16, whose steps are 4 there): no cancellation of squares."""
    B, T, C, G = 2, 700, 64, 4
    x = (randn((B, T, C), F32, 1, 1.0 if dtype == F32 else 8.0) + 1000).to(dtype)
    y64, off, _, _, _, _, _ = norm64(x, G, None, None, 1e-5, None, [T] * B)
    close(inv.group_norm(x.cuda(), G), y64, off + u(dtype) * (y64.abs() + off), "y")
    flat = torch.full((1, 50, 8), 3.25, dtype=dtype, device="cuda")   # no spread at all: (x - mean) is zero
    assert not inv.group_norm(flat, 2).any()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_group_norm_strides_and_lengths(dtype):
    B, T, C, G = 3, 40, 48, 6
    x, ga, be = randn((B, T, C), dtype, 1), randn((C,), dtype, 2), randn((C,), dtype, 3)
    for left, right, given, ends in ((0, 16, [40, -3, 400], [40, 0, 40]), (1, 2, [5, 40, 39], [5, 40, 39])):
        y64, off, _, _, _, _, _ = norm64(x, G, ga, be, 1e-3, "silu", ends)
        wide = torch.full((B, T, left + C + right), float("nan"), dtype=dtype, device="cuda")
        xs = wide[:, :, left:left + C]
        xs.copy_(x)
        out_wide = torch.full_like(wide, float("nan"))
        ys = out_wide[:, :, left:left + C]
        inv.group_norm(xs, G, ga.cuda(), be.cuda(), eps=1e-3, activation="silu", lengths=given, out=ys)
        close(ys, y64, off + u(dtype) * (y64.abs() + off) + tiny(dtype), "y")
        assert out_wide[:, :, :left].isnan().all() and out_wide[:, :, left + C:].isnan().all()
    xt = x.cuda().transpose(0, 1).contiguous().transpose(0, 1)       # frames of a batch at another stride: copied first
    y64, off, _, _, _, _, _ = norm64(x, G, ga, None, 1e-5, None, [T] * B)
    close(inv.group_norm(xt, G, ga.cuda()), y64, off + u(dtype) * (y64.abs() + off) + tiny(dtype), "y")
    close(inv.group_norm(x[0].cuda(), G, ga.cuda()), y64[0], (off + u(dtype) * (y64.abs() + off) + tiny(dtype))[0], "2-D")
    assert inv.group_norm(x[:, :0].cuda(), G).shape == (B, 0, C) and inv.group_norm(x[:0].cuda(), G).shape == (0, T, C)


def norm_back64(dy, x, G, ga, be, name, ends, stats, dtype):
    _, _, _, _, _, _, m = norm64(x, G, ga, be, 1e-5, None, ends)
    B, T, C = x.shape
    n = C // G
    x, dy = torch.where(m > 0, x.double(), 0.0), torch.where(m > 0, dy.double(), 0.0)
    ga = torch.ones(C).double() if ga is None else ga.double()
    be = torch.zeros(C).double() if be is None else be.double()
    wide = lambda v: v[:, None, :, None].expand(B, T, G, n).reshape(B, T, C)          # noqa: E731
    mean, rstd = wide(stats[..., 0].double()), wide(stats[..., 1].double())
    xh = (x - mean) * rstd
    xh_off = 2.0 ** -23 * (xh.abs() + rstd * x.abs())
    z = xh * ga + be
    z_off = xh_off * ga.abs() + 2.0 ** -23 * ((xh * ga).abs() + be.abs())
    du = dy * slope64(z, name)
    # the slope's own slope is at most 1 for silu', gelu', tanh'; exp is its own; a relu argument within z_off of zero may
    # fall on either side
    du_off = dy.abs() * scale64(z + z_off, name) * (2.0 ** -20 + z_off) if name else 0 * dy
    if name == "relu":
        du_off = du_off + dy.abs() * (z.abs() <= z_off)
    count = torch.tensor([max(e, 1) * n for e in ends]).double()[:, None]
    g = lambda v: v.reshape(B, T, G, n).sum((1, 3))                                   # noqa: E731
    v, v_off = du * ga, du_off * ga.abs() + 2.0 ** -23 * (du * ga).abs()
    vx_off = v_off * xh.abs() + v.abs() * (xh_off + 2.0 ** -23 * xh.abs())
    p, q = wide(g(v) / count), wide(g(v * xh) / count)
    # a group's sum: 64 roundings cover the depth of the partial sums (as above)
    p_off = wide((g(v_off) + 64 * 2.0 ** -24 * g(v.abs())) / count)
    q_off = wide((g(vx_off) + 64 * 2.0 ** -24 * g((v * xh).abs())) / count)
    dx = rstd * (v - p - xh * q)
    dx_off = rstd * (v_off + p_off + xh_off * q.abs() + xh.abs() * q_off
                     + 2.0 ** -22 * (v.abs() + p.abs() + (xh * q).abs()))
    dg, db = (du * xh * m).sum((0, 1)), (du * m).sum((0, 1))
    rows = 2.0 ** -24 * 256
    dg_off = ((du_off * xh.abs() + du.abs() * xh_off) * m).sum((0, 1)) + rows * (du * xh * m).abs().sum((0, 1))
    db_off = (du_off * m).sum((0, 1)) + rows * (du * m).abs().sum((0, 1))
    return [(v, t + u(dtype) * (v.abs() + t) + tiny(dtype)) for v, t in ((dx * m, dx_off * m), (dg, dg_off), (db, db_off))]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("B,T,C,G", NORM_SIZES)
def test_group_norm_backward_sizes(B, T, C, G, ragged, dtype):
    name = ACTS[(B + T + C + G + 1) % len(ACTS)]
    ends = ends_of(B, T, ragged)
    x = (randn((B, T, C), F32, 1) + randn((1, 1, C), F32, 2)).to(dtype)
    ga, be = (randn((C,), F32, 3) * 0.2 + 1).to(dtype), randn((C,), dtype, 4, 0.3)
    dy = randn((B, T, C), dtype, 5)
    lengths = torch.tensor(ends, dtype=torch.int32, device="cuda") if ragged else None
    xc, dyc = x.cuda(), dy.cuda()
    for b, e in enumerate(ends):
        xc[b, e:], dyc[b, e:] = float("nan"), float("inf")            # what is masked is not read
    stats = torch.empty((B, G, 2), device="cuda")
    inv.group_norm(xc, G, ga.cuda(), be.cuda(), activation=name, lengths=lengths, stats=stats)
    want = norm_back64(dy, x, G, ga, be, name, ends, stats.cpu(), dtype)
    args = (xc, G, stats, ga.cuda(), be.cuda())
    got = inv.group_norm_backward(dyc, *args, activation=name, lengths=lengths)
    for g, (v, t), what in zip(got, want, ("dx", "dweight", "dbias")):
        assert g.dtype == dtype
        close(g, v, t, what)
    again = inv.group_norm_backward(dyc, *args, activation=name, lengths=lengths)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    none = inv.group_norm_backward(dyc, xc, G, stats, ga.cuda(), be.cuda(), activation=name, lengths=lengths,
                                   needs=(False, True, False))
    assert none[0] is None and none[2] is None and torch.equal(none[1], got[1])
    inv.group_norm_backward(dyc, *args, activation=name, lengths=lengths, dx=dyc)                    # in place
    assert torch.equal(dyc, got[0])


# -- gradients against differences, autograd ---------------------------------------------------------------------
def slope_of(f, at, along, h):
    """d/ds f(at + s along) by central differences of 64-bit sums of float32 results."""
    return (f([a + h * d for a, d in zip(at, along)]) - f([a - h * d for a, d in zip(at, along)])) / (2 * h)


@gpu
@pytest.mark.parametrize("name", [None, "silu", "gelu", "tanh", "exp"])
def test_gradients_against_differences(name):
    """float32.  Central differences at h and 2 h differ by three times the h^2 term, which bounds the truncation; the
    results' roundings add 2^-22 sum|c y| / h."""
    B, T, C, N, G = 2, 9, 12, 10, 3
    ts = [randn(s, F32, k).cuda() for k, s in enumerate([(B, T, C), (C,), (C,), (N, C), (N,), (B, T, N)])]
    along = [randn(tuple(t.shape), F32, 20 + k).cuda() for k, t in enumerate(ts)]
    c = randn((B, T, N), F32, 50).cuda()
    lengths = [T, 6]
    c[1, 6:] = 0                                             # frames past the end: theirs are bias and residual only

    def net(v):
        h = inv.group_norm(v[0], G, v[1], v[2], activation=name, lengths=lengths)
        return inv.dense(h, v[3], v[4], activation=name, residual=v[5])

    def value(v):
        with torch.no_grad():
            return float((net(v).double() * c.double()).sum())

    leaves = [t.clone().requires_grad_() for t in ts]
    (net(leaves) * c).sum().backward()
    with torch.no_grad():
        size = float((net(ts).double() * c.double()).abs().sum())
    for k in range(len(ts)):                                 # each argument alone
        d = [a if j == k else torch.zeros_like(a) for j, a in enumerate(along)]
        h = 2.0 ** -7
        one, two = slope_of(value, ts, d, h), slope_of(value, ts, d, 2 * h)
        mine = float((leaves[k].grad.double() * d[k].double()).sum())
        tol = abs(one - two) + 2.0 ** -22 * size / h * 2 + 1e-4 * abs(one)
        assert abs(mine - one) <= tol, (k, mine, one, two, tol)


@gpu
def test_autograd_broadcast_and_shared_inputs():
    """One weight used twice, an expanded upstream gradient, a residual that is also the input."""
    w = randn((16, 16), F32, 1, 0.25).cuda().requires_grad_()
    x = randn((4, 16), F32, 2).cuda().requires_grad_()
    y = inv.dense(inv.dense(x, w, activation="tanh", residual=x), w)
    y.sum().backward()                                       # the gradient arrives as one expanded value
    x64, w64 = (t.detach().double().cpu().requires_grad_() for t in (x, w))
    ((torch.tanh(x64 @ w64.t()) + x64) @ w64.t()).sum().backward()
    close(x.grad, x64.grad, 1e-5 * (1 + x64.grad.abs()), "dx")        # sums of 16: (16 + 16) 2^-23 twice over, < 1e-5
    close(w.grad, w64.grad, 1e-5 * (1 + w64.grad.abs()), "dw")
    frozen = inv.dense(x.detach(), w.detach(), residual=x)   # only the residual requires one
    (g,) = torch.autograd.grad(frozen.sum(), x)
    assert torch.equal(g, torch.ones_like(g))


# -- streams and graphs ------------------------------------------------------------------------------------------
@gpu
def test_plain_calls_and_the_others_agree(monkeypatch):
    """The compiled way of the plain case and the way through Python: equal bits, and only the plain case is taken."""
    calls = inv._plain()
    assert calls is not None
    x, w, b, r = (randn(s, BF16, k).cuda() for k, s in enumerate(((2, 70, 64), (96, 64), (96,), (2, 70, 96))))
    z, dy = torch.empty(2, 70, 96, dtype=BF16, device="cuda"), randn((2, 70, 96), BF16, 9).cuda()
    ga, lens, stats = randn((64,), BF16, 5).cuda(), torch.tensor([70, 13], dtype=torch.int32, device="cuda"), torch.empty(2, 8, 2, device="cuda")

    def run():
        out = [inv.dense(x, w, b, activation="silu", residual=r, preactivation=z), z.clone(), inv.dense(x[0, 0], w, out_dtype=F32),
               *inv.dense_backward(dy, x, w, z, activation="silu"), *inv.dense_backward(dy, x, w, needs=(False, True, True)),
               inv.group_norm(x, 8, ga, activation="gelu", lengths=lens, stats=stats), stats.clone(), inv.group_norm(x[0], 4),
               *inv.group_norm_backward(x, x, 8, stats, ga, ga, lengths=lens), *inv.group_norm_backward(x, x, 8, stats, ga, lengths=[70, 13])]
        leaf = x.clone().requires_grad_()
        inv.group_norm(inv.dense(leaf, w, b, activation="tanh"), 8).float().square().sum().backward()
        return out + [leaf.grad]

    got = run()
    with monkeypatch.context() as m:
        m.setattr(inv, "_calls", None)
        want = run()
    assert len(got) == len(want)
    for a, c in zip(got, want):
        assert (a is None and c is None) or (a.dtype == c.dtype and a.shape == c.shape and torch.equal(a, c))
    assert torch.equal(calls.dense(x, w, b, None, None, None, 2), inv.dense(x, w, b, activation="silu"))
    bad = x.transpose(0, 1)
    for args in ((bad, w, None, None, None, None, 0), (x.cpu(), w, None, None, None, None, 0), (x, w.half(), None, None, None, None, 0),
                 (x, w, b[:5], None, None, None, 0), (x, w, b, None, r[0], None, 0), (x, w, b, r, r, None, 0),
                 (x, w, [1.0], None, None, None, 0), (x, w, b, None, None, F16, 0), (x, w, b, None, None, "f32", 0),
                 (None, w, b, None, None, None, 0), (x.clone().requires_grad_(), w, b, None, None, None, 0), (x[:0], w, b, None, None, None, 0),
                 (x, w, b, None, None, None, 9), (x, w[0], None, None, None, None, 0), (x, w, b)):
        assert calls.dense(*args) is None
    with pytest.raises(TypeError):
        calls.dense(x, w, b, None, None, None, "silu")
    for args in ((x, None, None, [1, 2], None, 8, 0, 1e-5), (x, None, None, None, stats[:1], 8, 0, 1e-5), (x, None, None, None, None, 7, 0, 1e-5),
                 (x, None, None, None, None, 8, 0, -1.0), (x, None, None, None, None, 8, 0, float("nan")), (x[0, 0], None, None, None, None, 8, 0, 1.0),
                 (x, None, None, lens.long(), None, 8, 0, 1e-5), (x, None, None, lens[:1], None, 8, 0, 1e-5)):
        assert calls.group_norm(*args) is None
    assert calls.dense_backward(dy, x, w, None, 2, True, True, True) is None                   # no preactivation
    assert calls.dense_backward(dy, x, w, None, 0, False, False, False) is None
    assert calls.group_norm_backward(x, x, stats[:, :4], None, None, None, 8, 0, True, True, True) is None


@gpu
def test_another_stream():
    x, w = torch.randn(700, 256, device="cuda"), torch.randn(192, 256, device="cuda")
    ga = torch.randn(192, device="cuda")
    want = inv.group_norm(inv.dense(x, w, activation="silu")[None], 8, ga)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = inv.group_norm(inv.dense(x, w, activation="silu")[None], 8, ga)
    side.synchronize()
    assert torch.equal(got, want)


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step_replays(dtype):
    """Forward and backward of norm + dense in one Plan.capture(), replayed on changing inputs between eager work."""
    from tacotron2_amd.plan import Plan
    plan = Plan(64, 16, 4, 4)
    B, T, C, N, G = 2, 300, 64, 96, 8
    M = B * T
    new = lambda *s, d=dtype: torch.zeros(s, dtype=d, device="cuda")                  # noqa: E731
    x, w, b, ga, be = new(B, T, C), new(N, C), new(N), new(C), new(C)
    lens = torch.tensor([T, 120], dtype=torch.int32, device="cuda")
    dy = new(B, T, N)
    h, stats, y, z = new(B, T, C), new(B, G, 2, d=F32), new(B, T, N), new(B, T, N)
    dh, dw, db, dx, dga, dbe = new(B, T, C), new(N, C), new(N), new(B, T, C), new(C), new(C)
    scratch = [torch.empty(max(1, n), dtype=torch.uint8, device="cuda") for n in (
        inv.group_norm_workspace(B, T, C, G, dtype), inv.dense_workspace(M, C, N, dtype),
        inv.dense_backward_workspace(M, C, N, dtype, None, "gelu"), inv.group_norm_backward_workspace(B, T, C, G, dtype))]

    def step():
        inv.group_norm(x, G, ga, be, activation="silu", lengths=lens, out=h, stats=stats, workspace=scratch[0])
        inv.dense(h, w, b, activation="gelu", out=y, preactivation=z, workspace=scratch[1])
        inv.dense_backward(dy, h, w, z, activation="gelu", dx=dh, dweight=dw, dbias=db, workspace=scratch[2])
        inv.group_norm_backward(dh, x, G, stats, ga, be, activation="silu", lengths=lens, dx=dx, dweight=dga, dbias=dbe,
                                workspace=scratch[3])

    outs = (h, stats, y, z, dh, dw, db, dx, dga, dbe)
    w_columns = new(C, N).t()
    with plan.capture() as g:
        step()
        with pytest.raises(RuntimeError, match="nothing may be allocated"):
            inv.dense(h, w, b)
        with pytest.raises(RuntimeError, match="nothing may be copied"):
            inv.dense(h, w_columns, out=y)
    for k in range(4):
        for j, t in enumerate((x, w, b, ga, be, dy)):
            t.copy_(randn(tuple(t.shape), dtype, 100 * k + j))
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        for t in outs:
            t.fill_(float("nan"))
        g.launch()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want)), f"replay {k}"
    g.close()
    plan.close()


@gpu
@pytest.mark.parametrize("M,K,N,T", [(600, 80, 96, 300), (4400, 512, 2048, 2200)])
def test_two_graphs_replay_side_by_side(M, K, N, T):
    """Each with its own workspaces, on two streams at once, the inputs changing in between."""
    from tacotron2_amd.plan import Plan
    plans = [Plan(64, 16, 4, 4) for _ in range(2)]
    sets, graphs = [], []
    for k, plan in enumerate(plans):
        x, w, dy, z = (t.cuda() for t in (randn((M, K), F32, k), randn((N, K), F32, 2 + k), randn((M, N), F32, 4 + k), randn((M, N), F32, 6 + k)))
        y, h, st = torch.zeros_like(dy), torch.zeros_like(dy).view(2, T, N), torch.zeros(2, 4, 2, device="cuda")
        dx, dw, db, dh = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(N, device="cuda"), torch.zeros_like(h)
        space = [torch.empty(max(1, n), dtype=torch.uint8, device="cuda") for n in (
            inv.dense_workspace(M, K, N), inv.dense_backward_workspace(M, K, N, F32, None, "silu"),
            inv.group_norm_workspace(2, T, N, 4), inv.group_norm_backward_workspace(2, T, N, 4))]

        def step(x=x, w=w, dy=dy, z=z, y=y, h=h, st=st, dx=dx, dw=dw, db=db, dh=dh, space=space):
            inv.dense(x, w, activation="silu", out=y, workspace=space[0])
            inv.dense_backward(dy, x, w, z, activation="silu", dx=dx, dweight=dw, dbias=db, workspace=space[1])
            inv.group_norm(y.view(2, T, N), 4, out=h, stats=st, workspace=space[2])
            inv.group_norm_backward(dy.view(2, T, N), y.view(2, T, N), 4, st, dx=dh, workspace=space[3])

        with plan.capture() as g:
            step()
        sets.append((step, (x, w, dy, z), (y, h, st, dx, dw, db, dh)))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        want = []
        for step, inputs, outs in sets:
            for t in inputs:
                t.mul_(0.5).add_(0.01 * turn)
            step()
            want.append([t.clone() for t in outs])
            for t in outs:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.launch()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(sets, want):
            assert all(torch.equal(a, b) for a, b in zip(outs, w)), f"turn {turn}"
    for g, plan in zip(graphs, plans):
        g.close()
        plan.close()


@gpu
def test_differentiable_form_refuses_capture():
    x, w = torch.randn(8, 16, device="cuda"), torch.randn(4, 16, device="cuda").requires_grad_()
    alive = inv.dense(x, w).sum()                            # an eager graph of the same leaf lives on
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    caught = []
    with torch.cuda.stream(side):
        graph.capture_begin()
        try:
            inv.dense(x, w)
        except RuntimeError as e:
            caught.append(str(e))
        try:
            inv.group_norm(x[None], 4, w[0])
        except RuntimeError as e:
            caught.append(str(e))
        with torch.no_grad():
            y = inv.dense(x, w)                              # without gradients it is recorded
        graph.capture_end()
    assert len(caught) == 2 and all("cannot be captured" in c for c in caught)
    for _ in range(3):
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, inv.dense(x, w.detach()))
    alive.backward()
    assert w.grad is not None


# -- the network ---------------------------------------------------------------------------------------------------
def network64(net, logmel, ends):
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in net.named_parameters()}
    x = logmel.double().cpu()
    B, T, _ = x.shape

    def norm(h, k):
        rows = []
        for b, e in enumerate(ends):
            live = h[b, :e].reshape(e, net.groups, -1)
            d = live - live.mean((0, 2), keepdim=True)
            d = (d / torch.sqrt((d * d).mean((0, 2), keepdim=True) + 1e-5)).reshape(e, -1)
            v = d * p[f"norm_w.{k}"] + p[f"norm_b.{k}"]
            rows.append(torch.cat([v * torch.sigmoid(v), torch.zeros(T - e, v.shape[-1], dtype=torch.float64)]))
        return torch.stack(rows)

    h = x @ p["w_in"].t() + p["b_in"]
    for k in range(len(net.w_up)):
        up = norm(h, k) @ p[f"w_up.{k}"].t() + p[f"b_up.{k}"]
        h = h + (up * 0.5 * torch.special.erfc(-up / math.sqrt(2))) @ p[f"w_down.{k}"].t() + p[f"b_down.{k}"]
    return torch.exp(norm(h, len(net.w_up)) @ p["w_out"].t() + p["b_out"]), p


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_network_runs_and_its_gradients(dtype):
    net = inv.MelInversion(n_mels=80, n_bins=33, channels=64, hidden=128, blocks=2, groups=8, dtype=dtype, device="cuda")
    logmel = randn((3, 41, 80), F32, 1).cuda() - 2
    ends = [41, 17, 30]
    mag = net(logmel, lengths=ends)
    assert mag.dtype == F32 and mag.shape == (3, 41, 33) and (mag > 0).all()
    live = (torch.arange(41)[None, :] < torch.tensor(ends)[:, None])[:, :, None]
    loss = (mag.log() * live.cuda()).square().mean()
    loss.backward()
    want, p = network64(net, logmel.to(dtype), ends)
    ((want.log() * live).square().mean()).backward()
    # a norm, two layers and a residual per block: about 14 roundings of the type between input and output
    far = lambda a, b: float((a - b).norm() / b.norm())                                # noqa: E731
    tol = 14 * u(dtype) if dtype == BF16 else 1e-5
    assert far((mag.detach().double().cpu() * live), want.detach() * live) <= tol
    for k, v in net.named_parameters():
        assert v.grad is not None and far(v.grad.double().cpu(), p[k].grad) <= 3 * tol, k


@gpu
def test_network_in_the_reconstruction_path(tmp_path):
    from tacotron2_amd import griffin_lim
    from tacotron2_amd.plan import get_plan
    net = inv.MelInversion(n_mels=80, n_bins=513, channels=64, hidden=64, blocks=1, groups=8, device="cuda")
    lm = randn((2, 30, 80), F32, 3) - 2
    kw = dict(n_fft=1024, hop=275, iterations=4, seed=5, normalize=None)
    x, mag = griffin_lim.logmel_to_audio(lm.cuda(), inversion=net, lengths=[30, 12], **kw)
    with torch.no_grad():
        want = net(lm.cuda(), lengths=[30, 12])
    want[1, 12:] = 0
    assert torch.equal(mag, want)
    plan = get_plan(1024, 275, 30, 2)
    x0 = griffin_lim.audio_utilities._start_signal(2, plan.signal_length(30), None, 5, "numpy", plan, plan.device)
    again = plan.run(mag, x0, 4)
    griffin_lim.audio_utilities._zero_past(again, [30, 12], 275, 1024)
    assert torch.equal(x, again)
    y, none = griffin_lim.logmel_to_audio(lm.numpy(), inversion=net, return_mag=False, lengths=[30, 12], **kw)
    assert none is None and torch.equal(x, y)
    one, _ = griffin_lim.logmel_to_audio(lm[1, :12].cuda(), inversion=net, **kw)      # an utterance alone
    assert torch.isfinite(one).all()
    for bad in (dict(basis="pinv"), dict(compression_factor=2.0)):
        with pytest.raises(ValueError, match="learned inversion"):
            griffin_lim.logmel_to_audio(lm.cuda(), inversion=net, **bad, **kw)
    with pytest.raises(ValueError, match="inversion maps"):
        griffin_lim.logmel_to_audio(lm.cuda(), inversion=net, n_fft=2048, hop=256, iterations=1)


# -- refusals ------------------------------------------------------------------------------------------------------
@gpu
def test_refusals_of_the_python_calls():
    x, w, b = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda"), torch.zeros(6, device="cuda")
    y = torch.zeros(4, 6, device="cuda")
    for bad in (dict(weight=w[:, :7]), dict(weight=w.half()), dict(bias=b[:5]), dict(weight=w.cpu()), dict(x=x.double()),
                dict(activation="swish"), dict(activation=["relu"]), dict(residual=y[:3]), dict(residual=y.half()),
                dict(out_dtype=F16), dict(out=y[:3]), dict(out=torch.zeros(6, 4, device="cuda").t()), dict(out=y.half()),
                dict(workspace=torch.zeros(4, device="cuda"), x=torch.zeros(16, 4096, device="cuda"),
                     weight=torch.zeros(6, 4096, device="cuda")),
                dict(preactivation=y, out=y), dict(weight=torch.zeros(0, 8, device="cuda"), bias=None), dict(weight=w[0])):
        with pytest.raises(ValueError):
            inv.dense(**{**dict(x=x, weight=w, bias=b), **bad})
    both = torch.zeros(64, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        inv.dense(both[:32].view(4, 8), w, out=both[20:44].view(4, 6))
    with pytest.raises(ValueError, match="overlaps"):
        inv.dense(x, w, residual=both[:24].view(4, 6), out=both[1:25].view(4, 6))
    space = torch.zeros(1 << 23, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="workspace overlaps"):
        inv.dense(torch.zeros(16, 4096, device="cuda"), torch.zeros(6, 4096, device="cuda"),
                  out=space[:384].view(torch.float32).view(16, 6), workspace=space)
    with pytest.raises(ValueError, match="workspace overlaps"):
        inv.dense_backward(torch.zeros(700, 512, device="cuda"), torch.zeros(700, 80, device="cuda"),
                           torch.zeros(512, 80, device="cuda"), dbias=space[-2048:].view(torch.float32),
                           workspace=space)
    with pytest.raises(ValueError, match="preactivation"):
        inv.dense_backward(y, x, w, activation="silu")
    with pytest.raises(ValueError):
        inv.dense_backward(y[:3], x, w)
    with pytest.raises(ValueError, match="overlaps"):
        inv.dense_backward(y, x, w, dx=x)
    with pytest.raises(ValueError, match="without gradients"):
        inv.dense(x, w.clone().requires_grad_(), out=y)
    h = torch.zeros(2, 5, 12, device="cuda")
    for bad in (dict(groups=5), dict(groups=0), dict(x=h[0, 0]), dict(weight=torch.ones(11, device="cuda")),
                dict(lengths=[1]), dict(eps=-1.0), dict(stats=torch.zeros(2, 3, device="cuda")), dict(out=h[:1]),
                dict(eps=float("nan")), dict(activation="softmax")):
        with pytest.raises(ValueError):
            inv.group_norm(**{**dict(x=h, groups=3), **bad})
    with pytest.raises(ValueError):
        inv.group_norm_backward(h, h.clone(), 3, torch.zeros(2, 4, 2, device="cuda"))


def test_python_calls_without_a_gpu():
    if torch.cuda.is_available():
        pytest.skip("has a GPU")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        inv.dense(torch.zeros(2, 3), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        inv.group_norm(torch.zeros(1, 2, 4), 2)
    with pytest.raises(ValueError, match="multiple of groups"):
        inv.MelInversion(channels=30, groups=4)


def test_refusals_of_the_c_calls():
    """The entry points check every argument before they touch the GPU: the pointers here are never followed."""
    lib = _lib.lib()
    p = ctypes.c_void_p(4096)
    good = dict(x=p, xs=8, w=p, ws=8, b=p, r=p, rs=6, y=p, ys=6, z=p, zs=6, rows=4, k=8, n=6, d=0, od=0, act=2, wk=p,
                wb=1 << 30, st=None)
    call = lambda **k: lib.gl_dense(*{**good, **k}.values())                           # noqa: E731
    for bad in (dict(x=None), dict(w=None), dict(y=None), dict(xs=7), dict(ws=7), dict(rs=5), dict(ys=5), dict(zs=5),
                dict(rows=-1), dict(rows=1 << 31), dict(k=0), dict(n=0), dict(n=(1 << 20) + 1), dict(d=3), dict(d=-1),
                dict(od=1), dict(d=1, od=2), dict(act=6), dict(act=-1), dict(xs=(1 << 31) + 1)):
        assert call(**bad) == -1, bad
        assert b"gl_dense" in lib.gl_last_error()
    assert call(rows=0) == 0
    need = lib.gl_dense_workspace(16, 4096, 6, 0, 0)
    assert need > 0 and lib.gl_dense_workspace(0, 4096, 6, 0, 0) == 0 and lib.gl_dense_workspace(1, 0, 6, 0, 0) == -1
    big = dict(rows=16, k=4096, xs=4096, ws=4096)
    assert call(**big, wb=need - 1) == -1 and b"workspace" in lib.gl_last_error()
    assert call(**big, wk=None) == -1 and call(**big, wk=ctypes.c_void_p(4104)) == -1
    back = dict(dy=p, dys=6, x=p, xs=8, w=p, ws=8, z=p, zs=6, dx=p, dxs=8, dw=p, dws=8, db=p, rows=4, k=8, n=6, d=0, od=0,
                act=2, wk=p, wb=1 << 30, st=None)
    call = lambda **k: lib.gl_dense_backward(*{**back, **k}.values())                  # noqa: E731
    for bad in (dict(dy=None), dict(x=None), dict(w=None), dict(z=None), dict(dys=5), dict(xs=7), dict(ws=7), dict(zs=5),
                dict(dxs=7), dict(dws=7), dict(rows=-2), dict(od=2), dict(act=9)):
        assert call(**bad) == -1, bad
    assert lib.gl_dense_backward_workspace(4, 8, 6, 0, 0, 2) == 0                       # one part each: nothing to join
    big = dict(rows=700, k=80, n=512, dys=512, xs=80, ws=80, zs=512, dxs=80, dws=80)
    need = lib.gl_dense_backward_workspace(700, 80, 512, 0, 0, 2)
    assert need > 0 and call(**big, wb=need - 1) == -1 and b"workspace" in lib.gl_last_error()
    assert call(**big, wk=None) == -1 and call(**big, wk=ctypes.c_void_p(4104)) == -1
    assert call(dx=None, dw=None, db=None) == 0
    norm = dict(x=p, xs=12, ga=p, be=p, f=p, y=p, ys=12, s=p, B=2, T=50000, C=12, G=3, d=0, act=0, eps=1e-5, wk=p, wb=1 << 30,
                st=None)
    call = lambda **k: lib.gl_group_norm(*{**norm, **k}.values())                      # noqa: E731
    for bad in (dict(x=None), dict(y=None), dict(xs=11), dict(ys=11), dict(B=-1), dict(B=65536), dict(T=-1), dict(C=0),
                dict(T=(1 << 30) + 1), dict(G=5), dict(G=0), dict(G=24), dict(d=4), dict(act=7), dict(eps=-1.0), dict(eps=float("nan")), dict(wb=1),
                dict(wk=None), dict(wk=ctypes.c_void_p(4100))):
        assert call(**bad) == -1, bad
    assert call(B=0) == 0 and call(T=0, s=None) == 0
    nback = dict(dy=p, dys=12, x=p, xs=12, s=p, ga=p, be=p, f=p, dx=p, dxs=12, dg=p, db=p, B=2, T=5, C=12, G=3, d=0, act=0,
                 wk=p, wb=1 << 30, st=None)
    call = lambda **k: lib.gl_group_norm_backward(*{**nback, **k}.values())            # noqa: E731
    for bad in (dict(dy=None), dict(x=None), dict(s=None), dict(dys=3), dict(xs=11), dict(dxs=11), dict(G=5), dict(wb=8),
                dict(wk=None), dict(act=-1), dict(d=9)):
        assert call(**bad) == -1, bad
    assert lib.gl_group_norm_workspace(2, 5, 12, 5, 0) == -1 and lib.gl_group_norm_workspace(2, 50000, 12, 3, 0) > 0


def test_row_strides_of_views():
    t = torch.zeros(4, 5, 6)
    assert inv._row_stride(t) == 6 and inv._row_stride(t[:, :, :3]) == 6 and inv._row_stride(t[0]) == 6
    assert inv._row_stride(t[:, :3]) is None and inv._row_stride(t[:, ::2, :]) is None and inv._row_stride(t[:, :, ::2]) is None
    assert inv._row_stride(t[1:, :, 1:]) == 6 and inv._row_stride(t[:, :1]) == 30 and inv._row_stride(t.transpose(0, 1)) is None
    assert inv._row_stride(torch.zeros(1, 3).expand(4, 3)) is None and inv._row_stride(torch.zeros(3)) == 3
    assert inv._row_stride(torch.zeros(7, 1)) == 1 and inv._row_stride(torch.zeros(1, 3).expand(1, 3)) == 3

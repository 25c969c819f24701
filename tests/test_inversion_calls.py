"""What the calls of the learned mel inversion refuse, raise and leave alone, whichever way they take (compiled or through Python)."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad

from tacotron2_amd import _lib
from tacotron2_amd import inversion as inv

gpu = pytest.mark.gpu
WAYS = ["compiled", "python"]


@pytest.fixture(params=WAYS)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(inv, "_calls", None)
    return request.param


@gpu
def test_a_result_past_the_memory_raises_torchs_own_error(way):
    """A terabyte of results: refused by the allocator, before anything runs."""
    x, w = torch.zeros(1 << 18, 1, device="cuda"), torch.zeros(1 << 20, 1, device="cuda")
    with pytest.raises(torch.OutOfMemoryError):
        inv.dense(x, w)
    assert torch.equal(inv.dense(x[:2], w[:3]), torch.zeros(2, 3, device="cuda"))


def arguments(device):
    """(call, its tensors) of the four operators."""
    x, w, b = (torch.randn(s, device=device) for s in ((3, 4), (6, 4), (6,)))
    y, st, g = torch.randn(3, 6, device=device), torch.ones(1, 2, 2, device=device), torch.ones(4, device=device)
    return [(lambda x, w, b, r: inv.dense(x, w, b, residual=r), [x, w, b, y]), (lambda x, w, b: inv.group_norm(x, 2, w, b), [x, g, g.clone()]),
            (lambda dy, x, w, z: inv.dense_backward(dy, x, w, z, activation="silu"), [y, x, w, y.clone()]),
            (lambda dy, x, st, w, b: inv.group_norm_backward(dy, x, 2, st, w, b), [x.clone(), x, st, g, g.clone()])]


def refuses_tangents(device):
    for call, tensors in arguments(device):
        for k, t in enumerate(tensors):
            with forward_ad.dual_level():
                dual = forward_ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(*tensors[:k], dual, *tensors[k + 1:])
                with torch.no_grad(), pytest.raises(RuntimeError, match="no forward-mode derivative"):
                    call(*tensors[:k], dual, *tensors[k + 1:])


def refuses_traces(device):
    for call, tensors in arguments(device):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(call, tuple(tensors), check_trace=False)


def test_tangents_and_traces_are_refused_without_a_gpu(way):
    refuses_tangents("cpu")
    refuses_traces("cpu")


@gpu
def test_tangents_and_traces_are_refused(way):
    refuses_tangents("cuda")
    refuses_traces("cuda")
    for call, tensors in arguments("cuda"):
        with forward_ad.dual_level():                        # a level alone, without a tangent, changes nothing
            inside = call(*tensors)
        outside = call(*tensors)
        for a, b in zip(inside if isinstance(inside, tuple) else (inside,), outside if isinstance(outside, tuple) else (outside,)):
            assert torch.equal(a, b)
    net = inv.MelInversion(n_mels=8, n_bins=9, channels=16, hidden=16, blocks=1, groups=4, device="cuda")
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(net, torch.zeros(1, 5, 8, device="cuda"), check_trace=False)


@gpu
def test_gradients_that_need_an_overwritten_tensor_are_refused(way):
    """What a call writes into the caller's tensor counts as a change of it."""
    x, w, y = torch.randn(3, 4, device="cuda"), torch.randn(6, 4, device="cuda"), torch.randn(3, 6, device="cuda")
    st, g, b = torch.ones(1, 2, 2, device="cuda"), torch.ones(4, device="cuda"), torch.zeros(6, device="cuda")
    other = torch.randn(3, 6, device="cuda")
    writes = [(lambda t: inv.dense(x, w, out=t), (3, 6)), (lambda t: inv.dense(x, w, preactivation=t, activation="silu"), (3, 6)),
              (lambda t: inv.group_norm(x, 2, out=t), (3, 4)), (lambda t: inv.group_norm(x, 2, stats=t), (1, 2, 2)),
              (lambda t: inv.dense_backward(y, x, w, dx=t), (3, 4)), (lambda t: inv.dense_backward(y, x, w, dweight=t), (6, 4)),
              (lambda t: inv.dense_backward(y, x, w, dbias=t), (6,)), (lambda t: inv.group_norm_backward(x, x.clone(), 2, st, g, g, dx=t), (3, 4)),
              (lambda t: inv.group_norm_backward(x, x.clone(), 2, st, g, g, dweight=t), (4,)),
              (lambda t: inv.group_norm_backward(x, x.clone(), 2, st, g, g, dbias=t), (4,))]
    for write, shape in writes:
        leaf = torch.randn(shape, device="cuda", requires_grad=True)
        square = leaf * leaf                                 # needs leaf's values
        with torch.no_grad():
            write(leaf.detach())
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            square.sum().backward()
    with torch.inference_mode():                             # tensors without a count of changes
        assert torch.equal(inv.dense(x, w, b, out=torch.empty(3, 6, device="cuda")), inv.dense(x, w, b))
        assert torch.equal(inv.dense(x, w, b, preactivation=torch.empty_like(other), activation="relu"), inv.dense(x, w, b, activation="relu"))
    z = torch.empty(3, 6, device="cuda")                     # and what a differentiable call keeps for itself is none
    xg = x.clone().requires_grad_()
    inv.group_norm(inv.dense(xg, w, b, activation="silu"), 2).sum().backward()
    assert xg.grad is not None and z._version == 0


def test_pointers_off_their_elements_are_refused():
    """Checked before anything runs: the pointers here are never followed.  Workspaces are large enough for all of them."""
    lib = _lib.lib()
    at = ctypes.c_void_p
    p = at(4096)
    dense = dict(x=p, xs=8, w=p, ws=8, b=p, r=p, rs=6, y=p, ys=6, z=p, zs=6, rows=4, k=8, n=6, d=1, od=0, act=2, wk=p, wb=1 << 30, st=None)
    back = dict(dy=p, dys=6, x=p, xs=8, w=p, ws=8, z=p, zs=6, dx=p, dxs=8, dw=p, dws=8, db=p, rows=4, k=8, n=6, d=1, od=0, act=2, wk=p,
                wb=1 << 30, st=None)
    norm = dict(x=p, xs=12, ga=p, be=p, f=p, y=p, ys=12, s=p, B=2, T=5, C=12, G=3, d=2, act=0, eps=1e-5, wk=p, wb=1 << 30, st=None)
    nback = dict(dy=p, dys=12, x=p, xs=12, s=p, ga=p, be=p, f=p, dx=p, dxs=12, dg=p, db=p, B=2, T=5, C=12, G=3, d=2, act=0, wk=p,
                 wb=1 << 30, st=None)
    for call, good, halves, words in ((lib.gl_dense, dense, "xwb", "ryz"), (lib.gl_dense_backward, back, ("x", "w", "dx", "dw", "db"), ("dy", "z")),
                                      (lib.gl_group_norm, norm, ("x", "ga", "be", "y"), "fs"),
                                      (lib.gl_group_norm_backward, nback, ("dy", "x", "ga", "be", "dx", "dg", "db"), "fs")):
        for names, off in ((halves, (1,)), (words, (1, 2))):
            for name in names:
                for k in off:
                    assert call(*{**good, name: at(4096 + k)}.values()) == -1, (call.__name__, name, k)
                    assert b"elements' size" in lib.gl_last_error()
        if "rows" in good:                                   # float32 throughout: two bytes off are refused for all of them
            for name in halves:
                assert call(*{**good, "d": 0, name: at(4098)}.values()) == -1, (call.__name__, name)

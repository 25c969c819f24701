"""What the calls of the learned mel inversion refuse, raise and leave alone, whichever way they take (compiled or through Python)."""
import ctypes

import pytest
import torch

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

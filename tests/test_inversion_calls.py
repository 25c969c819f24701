"""What the calls of the learned mel inversion refuse, raise and leave alone, whichever way they take (compiled or through Python)."""
import pytest
import torch

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

"""Products through planes in captured graphs: two planes of dz, and sums that float32's planes do not give, in some replays."""
import pytest
import torch

from tacotron2_amd import inversion as inv
from tacotron2_amd.plan import Plan
from test_inversion import BF16, F16, F32, randn

gpu = pytest.mark.gpu


def same(a, b):
    return torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(a.isnan(), b.isnan())


def rig(M, K, N, dtype, od, seed):
    """(step, its inputs, its outputs) of a forward and a backward call with their own workspaces."""
    x, w, dy = (torch.zeros(s, dtype=t, device="cuda") for s, t in (((M, K), dtype), ((N, K), dtype), ((M, N), od)))
    y, z = torch.zeros(M, N, dtype=od, device="cuda"), torch.zeros(M, N, dtype=od, device="cuda")
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(N, dtype=dtype, device="cuda")
    space = [torch.empty(max(1, n), dtype=torch.uint8, device="cuda") for n in (
        inv.dense_workspace(M, K, N, dtype, od), inv.dense_backward_workspace(M, K, N, dtype, od, "silu"))]

    def step():
        inv.dense(x, w, activation="silu", out_dtype=od, out=y, preactivation=z, workspace=space[0])
        inv.dense_backward(dy, x, w, z, activation="silu", dx=dx, dweight=dw, dbias=db, workspace=space[1])

    return step, (x, w, dy), (y, z, dx, dw, db)


def fill(inputs, seed, wild):
    for k, t in enumerate(inputs):
        t.copy_(randn(tuple(t.shape), F32, seed + k, 0.3).to(t.dtype))
    if wild:                                                 # some rows far apart in size, an infinite gradient
        inputs[0][:, 0] *= 2.0 ** 40 if inputs[0].dtype == F32 else 1.0
        inputs[1][:, 0] = 0
        inputs[2][5, 1] = float("inf")


@gpu
@pytest.mark.parametrize("M,K,N,dtype,od", [(641, 80, 96, BF16, F32), (9000, 512, 264, F16, F16), (9000, 136, 257, BF16, F32),
                                            (9001, 512, 264, F32, F32), (64, 16384, 264, F32, F32)])
def test_replays_with_and_without_wild_values(M, K, N, dtype, od):
    plan = Plan(64, 16, 4, 4)
    step, inputs, outs = rig(M, K, N, dtype, od, 0)
    fill(inputs, 1, False)
    step()
    with plan.capture() as g:
        step()
    for turn, wild in enumerate((False, True, True, False, True)):
        fill(inputs, 10 * turn, wild)
        step()
        torch.cuda.synchronize()
        want = [t.clone() for t in outs]
        assert wild == bool((~torch.isfinite(want[3])).any())
        for _ in range(2):
            for t in outs:
                t.fill_(3.0)
            g.launch()
            torch.cuda.synchronize()
            assert all(same(a, b) for a, b in zip(outs, want)), f"turn {turn}"
    g.close()
    plan.close()


@gpu
@pytest.mark.parametrize("M,K,N", [(9001, 512, 264), (20000, 130, 257)])
def test_two_graphs_repair_side_by_side(M, K, N):
    plans = [Plan(64, 16, 4, 4) for _ in range(2)]
    rigs = [rig(M, K, N, F32, F32, 50 * k) for k in range(2)]
    graphs = []
    for plan, (step, _, _) in zip(plans, rigs):
        with plan.capture() as g:
            step()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for turn in range(3):
        want = []
        for k, (step, inputs, outs) in enumerate(rigs):
            fill(inputs, 100 * k + 10 * turn, turn != 1)
            step()
            want.append([t.clone() for t in outs])
            for t in outs:
                t.fill_(3.0)
        torch.cuda.synchronize()
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.launch()
        torch.cuda.synchronize()
        for (_, _, outs), w in zip(rigs, want):
            assert all(same(a, b) for a, b in zip(outs, w)), f"turn {turn}"
    for g, plan in zip(graphs, plans):
        g.close()
        plan.close()

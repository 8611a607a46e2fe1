"""GPU: the FP8 path where its kernels change over - rows near FP32's ends, scores far below one, workspaces of other sizes, products whose
rows, tiles and K blocks end off every boundary."""
import pytest
import torch

from fp8_ref import route, rows_fp8, stack_fp8
from strixite_b200 import kernels as K
from test_gpu_fp8 import ACTS, DT, gen, group, rand, run_route, some_ids

pytestmark = pytest.mark.gpu


# ---- routing ---------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
def test_route_small_scores_beside_biases_of_their_size(score):
    """Two experts whose scores lie far below 1, one with a bias that brings its sum within a few steps of FP32 of the other's: the order of
    64 bits. As many picks as experts, so that none behind the last pick asks for 64 bits, and one such pair a token, so that no
    other pair does."""
    r = torch.Generator().manual_seed(7)
    wrong = []
    for _ in range(1000):
        u = torch.rand(3, generator=r, dtype=torch.float64)
        a = -(25 + 54 * u[0])
        l = torch.tensor([a, a - 6 * u[1], 0.0]).float().view(1, 3)[:, : 3 if score == "softmax" else 2]  # softmax: the scores are the exponentials
        E = l.shape[1]
        p = torch.sigmoid(l.double()) if score == "sigmoid" else torch.softmax(l.double(), 1)
        bias = torch.zeros(E)
        bias[1] = (p[0, 0] - p[0, 1] + (u[2] * 128 - 64) * 2.0**-24 * p[0, 0]).float()
        want, cw = route(l, E, score, bias, 1, 1, 1, True, 1.0)
        ids, coef, err = run_route(l.cuda(), E, score, bias.cuda(), 1, 1, 1, True, 1.0, K.Act.F32)
        if not torch.equal(ids.cpu(), want):
            wrong.append(float(a))
    assert not wrong, "%d of 1000 tokens in another order, scores e^%s" % (len(wrong), wrong[:8])


# ---- products --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,A,E,N", [(11, 1, 4, 128), (11, 1, 4, 130), (1200, 1, 4, 128), (4000, 2, 8, 1002)])
def test_combine_refuses_a_workspace_of_other_sizes(act, M, A, E, N):
    """Grouped for another number of slots: neither the partial sums nor y are written, and it is counted once."""
    g = gen(N)
    Kd = 128
    ws, n, _ = group(some_ids(g, M * A + 1, 1, E, ""), E)
    wq, wsc = stack_fp8(rand(g, E, N, Kd))
    hq, hs = rows_fp8(rand(g, M * A, Kd))
    ids, coef = some_ids(g, M, A, E, ""), torch.ones((M, A), device="cuda")
    partial, y = torch.full((M * A, N), 5.0, device="cuda"), torch.full((M, N), 7.0, dtype=DT[act], device="cuda")
    before = K.workspace_refusal_count()
    K.linear_fp8_experts_combine_grouped(hq, hs, K.Fp8Weight(wq, wsc, experts=E), E, ids, coef, ws, n, partial, M, A, y, act)
    assert K.workspace_refusal_count() == before + 1 and (partial == 5.0).all() and (y == 7.0).all()

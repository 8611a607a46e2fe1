"""GPU: the FP8 path where its kernels change over - rows near FP32's ends, scores far below one, workspaces of other sizes, products whose
rows, tiles and K blocks end off every boundary."""
import pytest
import torch

from fp8_ref import FP8, blocks, check_fp8_rows, route, rows_fp8, stack_fp8
from strixite_b200 import StrixError
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


# ---- norm and SwiGLU -------------------------------------------------------------------------------------------------

# Sum of squares, root and products as in the norm's own test, and eps scaled twice (two roundings of its share of the mean, halved by the root).
NORM_REL = (77 / 2 + 7) * 2.0**-24


def check_norm(x, eps, act, d):
    M = x.shape[0]
    w = rand(gen(d), d) * 0.1 + 1
    f = x.double()
    h64 = f / torch.sqrt(f.pow(2).mean(1, keepdim=True) + eps) * w.double()
    h, q, s = torch.empty_like(x), torch.empty((M, d), dtype=FP8, device="cuda"), torch.empty((M, blocks(d)), device="cuda")
    K.residual_rmsnorm_fp8(x, None, w, M, d, eps, None, h, q, s, act)
    tol = h64.abs() * (NORM_REL + (2.0**-8 if act == K.Act.BF16 else 0)) + 1e-37
    for m in range(M):
        assert ((h[m].double() - h64[m]).abs() <= tol[m]).all(), "row %d is off by up to %g of itself" % (m, ((h[m].double() - h64[m]).abs() / h64[m].abs()).max())
    check_fp8_rows(q, s, h64, NORM_REL)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("d", (16, 512, 2560, 8192))
def test_rmsnorm_fp8_rows_near_the_ends_of_fp32(act, d):
    """Rows whose squares leave FP32's range, or its normal range, on either side: their norm is an ordinary number."""
    g = gen(d)
    powers = (0, -45, -62, -64, -70, -90, -115, 45, 58, 62, 64, 90, 120)
    x = torch.stack([rand(g, d) * 2.0**p for p in powers]).to(DT[act])
    check_norm(x, 0.0, act, d)
    tiny = x[1:7].contiguous()
    for eps in (2.0**-90, 2.0**-128, 2.0**-140, 2.0**-149):  # above, near and below the squares' mean
        check_norm(tiny, eps, act, d)
    check_norm(x[6:].contiguous(), 1e-6, act, d)
    check_norm(x, 1e30, act, d)


@pytest.mark.parametrize("act", ACTS)
def test_rmsnorm_fp8_one_value_far_above_the_rest(act):
    d = 1024
    x = rand(gen(1), 4, d).to(DT[act])
    x[1, 700], x[2, 5] = 2.0**70, -(2.0**100)
    x[3] *= 2.0**-60
    x[3, 3] = 2.0**-20
    check_norm(x, 0.0, act, d)


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


# ---- errors ----------------------------------------------------------------------------------------------------------


def test_a_refused_launch_does_not_fail_the_next_call():
    """A launch that the runtime refuses (the legacy stream while a stream that synchronises with it is captured) is the error of its own call
    alone."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    M, A, E = 4, 2, 8
    ids = torch.zeros((M, A), dtype=torch.int32, device="cuda")
    n = K.moe_route_workspace_bytes(M, A, E)
    ws, err = torch.empty(n, dtype=torch.uint8, device="cuda"), K.new_err()
    gu, h = torch.ones((4, 512), device="cuda"), torch.empty((4, 256), device="cuda")
    q, s = torch.empty((4, 256), dtype=FP8, device="cuda"), torch.empty((4, 2), device="cuda")
    calls = (lambda: K.moe_group_routes(ids, M, A, E, ws, n, err), lambda: K.swiglu_fp8(gu, q, s, 4, 256, K.Act.F32), lambda: K.swiglu(gu, h, 4, 256, K.Act.F32))
    for call in calls:
        call()  # set up
    torch.cuda.synchronize()
    assert torch.cuda.current_stream().cuda_stream == 0
    for refused in calls:
        rc, stream = rt.cudaStreamCreate()
        assert int(rc) == 0
        rc, = rt.cudaStreamBeginCapture(stream, rt.cudaStreamCaptureMode.cudaStreamCaptureModeRelaxed)
        assert int(rc) == 0
        with pytest.raises(StrixError, match="cudaErrorStreamCapture"):
            refused()
        rt.cudaStreamEndCapture(stream)
        rt.cudaGetLastError()
        rt.cudaStreamDestroy(stream)
        for call in calls:
            call()
    torch.cuda.synchronize()

"""GPU: the FP8 path where its kernels change over - rows near FP32's ends, scores far below one, workspaces of other sizes, products whose
rows, tiles and K blocks end off every boundary."""
import pytest
import torch

from fp8_ref import FP8, blocks, check_fp8_rows, matrix_fp8, product_bound, route, rows_fp8, stack_fp8, wide_matrix, wide_rows
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


@pytest.mark.parametrize("act", ACTS)
def test_swiglu_fp8_blocks_near_the_floor_of_the_scale_and_far_above_one(act):
    """Blocks whose largest magnitude lies around 2^-99 and 2^-101 (where the scale stops at its floor), 2^-61 and 2^61 (where the form of the
    codes changes), and far beyond."""
    I = 128 * 10
    for rows in (1, 37):
        gu = rand(gen(rows), rows, 2 * I)
        for b, p in enumerate((-97, -99, -101, -104, -108, -61, -59, 59, 61, 100)):
            gu[:, I + b * 128 : I + (b + 1) * 128] *= 2.0**p
        gu = gu.to(DT[act])
        q, s = torch.empty((rows, I), dtype=FP8, device="cuda"), torch.empty((rows, blocks(I)), device="cuda")
        K.swiglu_fp8(gu, q, s, rows, I, act)
        gate, up = gu.double()[:, :I], gu.double()[:, I:]
        check_fp8_rows(q, s, gate * torch.sigmoid(gate) * up, 8 * 2.0**-24)  # as in the SwiGLU's own test


# ---- products --------------------------------------------------------------------------------------------------------


def dense(g, M, N, Kd):
    xq, xs = rows_fp8(rand(g, M, Kd))
    wq, ws = matrix_fp8(rand(g, N, Kd) * 0.02 * torch.exp(rand(g, N, 1)))
    x, w = wide_rows(xq, xs), wide_matrix(wq, ws)
    return xq, xs, K.Fp8Weight(wq, ws), x, w, x @ w.t()


@pytest.mark.parametrize("M,N,Kd", [(5000, 1100, 1040), (4097, 900, 2704), (30000, 100, 144), (20000, 300, 16), (6000, 1280, 400)])
def test_linear_fp8_many_rows_with_remainders(M, N, Kd):
    """Many rows: several tiles for a pair of CTAs, last tiles with one half of columns, K blocks that end early, also as the only one."""
    xq, xs, W, x, w, y64 = dense(gen(M + N), M, N, Kd)
    for act in ACTS:
        guard = torch.full((M * N + 64,), 7.0, dtype=DT[act], device="cuda")
        y = guard[: M * N].view(M, N)
        K.linear_fp8(xq, xs, W, y, M, act)
        assert ((y.double() - y64).abs() <= product_bound(x.abs(), w.abs(), Kd, y64, act == K.Act.BF16)).all()
        assert (guard[M * N :] == 7.0).all()
    assert K.umma_abort_count() == 0


@pytest.mark.parametrize("M,N,Kd,off", [(2293, 2115, 656, 8), (2293, 2116, 656, 1), (2293, 2114, 656, 2), (4097, 901, 2704, 3)])
def test_linear_fp8_many_rows_that_start_anywhere(M, N, Kd, off):
    """Rows of y that start at any element: stored in words or halves."""
    xq, xs, W, x, w, y64 = dense(gen(M + N), M, N, Kd)
    for act in ACTS:
        room = torch.full((M * N + 72,), 3.0, dtype=DT[act], device="cuda")
        y = room[off : off + M * N].view(M, N)
        K.linear_fp8(xq, xs, W, y, M, act)
        assert ((y.double() - y64).abs() <= product_bound(x.abs(), w.abs(), Kd, y64, act == K.Act.BF16)).all()
        assert (room[:off] == 3.0).all() and (room[off + M * N :] == 3.0).all()
    assert K.umma_abort_count() == 0


@pytest.mark.parametrize("M,A,E,N,Kd,kind", [(3000, 2, 40, 1001, 272, "steep"), (3000, 2, 40, 1002, 272, "bad"), (2500, 3, 24, 1100, 400, "steep"), (4000, 2, 16, 1153, 144, "one")])
def test_experts_many_slots_with_rows_that_start_anywhere(M, A, E, N, Kd, kind):
    g = gen(M + N)
    ids = some_ids(g, M, A, E, kind)
    wq, wsc = stack_fp8(rand(g, E, N, Kd) * 0.02)
    W = K.Fp8Weight(wq, wsc, experts=E)
    ws, n, _ = group(ids, E)
    flat = ids.view(-1).long()
    ok = (flat >= 0) & (flat < E)

    def exact(rows):
        y, tol = torch.zeros((M * A, N), dtype=torch.float64, device="cuda"), torch.zeros((M * A, N), dtype=torch.float64, device="cuda")
        for e in range(E):
            at, w = flat == e, wide_matrix(wq[e * N : (e + 1) * N], wsc[e * blocks(N) : (e + 1) * blocks(N)])
            y[at] = rows[at] @ w.t()
            tol[at] = product_bound(rows[at].abs(), w.abs(), Kd, y[at], False)
        return y, tol

    xq, xs = rows_fp8(rand(g, M, Kd))
    y64, tol = exact(wide_rows(xq, xs).repeat_interleave(A, 0))
    for act in ACTS:
        for off in (0, 1):
            room = torch.full((M * A * N + 72,), 3.0, dtype=DT[act], device="cuda")
            y = room[off : off + M * A * N].view(M * A, N)
            K.linear_fp8_experts_gather_grouped(xq, xs, W, E, ws, n, M, A, y, act)
            t = tol + (y64.abs() + tol) * 2.0**-8 if act == K.Act.BF16 else tol
            assert ((y.double() - y64).abs() <= t)[ok].all()
            assert (y[~ok] == 3.0).all() and (room[:off] == 3.0).all() and (room[off + M * A * N :] == 3.0).all()
    hq, hs = rows_fp8(rand(g, M * A, Kd))
    coef = torch.rand((M, A), generator=g, device="cuda")
    p64, tol = exact(wide_rows(hq, hs))
    c = coef.double()[:, :, None]
    s64, terms = (p64.view(M, A, N) * c).sum(1), (p64.view(M, A, N) * c).abs().sum(1)
    t32 = (tol.view(M, A, N) * c).sum(1) + terms * A * 2.0**-24
    failed = ~ok.view(M, A).all(1)
    for act in ACTS:
        room, partial = torch.full((M * N + 72,), 3.0, dtype=DT[act], device="cuda"), torch.empty((M * A, N), device="cuda")
        y = room[1 : 1 + M * N].view(M, N)
        K.linear_fp8_experts_combine_grouped(hq, hs, W, E, ids, coef, ws, n, partial, M, A, y, act)
        t = t32 + (s64.abs() + t32) * 2.0**-8 if act == K.Act.BF16 else t32
        assert ((y.double() - s64).abs() <= t)[~failed].all() and y[failed].isnan().all()
        assert room[0] == 3.0 and (room[1 + M * N :] == 3.0).all()
    assert K.umma_abort_count() == 0


def test_experts_with_a_stack_past_32_bit_offsets():
    """4.3 GB of codes in 256 matrices: the last ones are where they belong, with few slots and with many."""
    g = gen(21)
    E, N, Kd, A = 256, 4096, 4096, 4
    wq = torch.randint(0, 0x70, (E * N, Kd), generator=g, device="cuda", dtype=torch.uint8)  # e4m3 from 0 to 120, no NaN
    wsc = torch.rand((E * blocks(N), blocks(Kd)), generator=g, device="cuda") * 0.02
    W = K.Fp8Weight(wq, wsc, experts=E)
    for M in (3, 600):
        ids = torch.randint(E - 8, E, (M, A), generator=g, device="cuda").int()
        ids[0] = torch.tensor([0, 127, 128, E - 1])
        ws, n, _ = group(ids, E)
        xq, xs = rows_fp8(rand(g, M, Kd))
        y = torch.empty((M * A, N), device="cuda")
        K.linear_fp8_experts_gather_grouped(xq, xs, W, E, ws, n, M, A, y, K.Act.F32)
        x = wide_rows(xq, xs)
        for s in (0, 1, 2, 3, M * A // 2, M * A - 1):
            e, row = int(ids.view(-1)[s]), x[s // A : s // A + 1]
            w = wide_matrix(wq[e * N : (e + 1) * N].view(FP8), wsc[e * blocks(N) : (e + 1) * blocks(N)])
            y64 = row @ w.t()
            assert ((y[s : s + 1].double() - y64).abs() <= product_bound(row.abs(), w.abs(), Kd, y64, False)).all()
    assert K.umma_abort_count() == 0


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

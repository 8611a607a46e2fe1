"""GPU: the FP8 path - score-based routing, norm and SwiGLU with FP8 results, the dense and the grouped products - operator by operator
against plain 64-bit forms, and as the run of an FFN."""
import numpy as np
import pytest
import torch

import oracle
from fp8_ref import FP8, blocks, check_fp8_rows, product_bound, route, rows_fp8, stack_fp8, wide_matrix, wide_rows, matrix_fp8
from strixite_b200 import StrixError
from strixite_b200 import kernels as K

pytestmark = pytest.mark.gpu

ACTS = (K.Act.F32, K.Act.BF16)
DT = {K.Act.F32: torch.float32, K.Act.BF16: torch.bfloat16}


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def host_err(e):
    return e.cpu().numpy().view(np.uint32)[:3].tolist()


# ---- routing ---------------------------------------------------------------------------------------------------------


def run_route(logits, k, score, bias, G, tg, gt, renorm, scale, act, shared=None, ld=None, shared_ld=0, shared_id=0):
    M, E = logits.shape[0], (logits.shape[1] if ld is None else None) or logits.shape[1]
    A = k + (0 if shared is None else 1)
    ids = torch.full((M, A), -7, dtype=torch.int32, device="cuda")
    coef = torch.full((M, A), -7.0, device="cuda")
    err = K.new_err()
    K.moe_router_scored(logits, E if ld is None else ld, M, E, k, score, bias, G, tg, gt, renorm, scale, shared, shared_ld, shared_id, ids, coef, act, err)
    return ids, coef, err


# (E, k, groups, open groups, group_top): lanes with one expert and with many, groups that do not divide a warp, one expert per group
SHAPES = [(1, 1, 1, 1, 1), (31, 5, 1, 1, 1), (33, 32, 1, 1, 2), (64, 4, 8, 3, 2), (256, 8, 8, 4, 2), (512, 10, 8, 4, 2), (160, 6, 8, 3, 1), (1020, 17, 17, 5, 2),
          (96, 6, 3, 2, 2), (32, 3, 32, 7, 2), (1024, 32, 1, 1, 1), (992, 9, 31, 4, 2), (1024, 32, 32, 1, 2)]


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("E,k,G,tg,gt", SHAPES)
def test_route(act, score, E, k, G, tg, gt):
    g = gen(E * 100 + k)
    for M, with_bias, renorm, scale in ((1, True, True, 2.5), (67, False, True, 1.0), (130, True, False, 16.0)):
        logits = (rand(g, M, E) * 1.5 - 1.0).to(DT[act])
        bias = rand(g, E) * 0.05 if with_bias else None
        want, cw = route(logits, k, score, bias, G, tg, gt, renorm, scale)
        ids, coef, err = run_route(logits, k, score, bias, G, tg, gt, renorm, scale, act)
        assert host_err(err)[0] == 0
        assert torch.equal(ids.cpu(), want)
        # FP32 at most: the exponential and the score (4 steps of 2^-24), a sum of up to 1024 by lanes (32 + 5 steps), two divisions, a product
        assert ((coef.cpu().double() - cw).abs() <= cw.abs() * 44 * 2.0**-24).all()


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
def test_route_close_scores_and_ties(score):
    """Values that agree to the last bits of FP32 and beyond keep the order of 64 bits; equal ones go to the lower index."""
    g = gen(5)
    E, k, M = 64, 8, 200
    logits = torch.round(rand(g, M, E) * 2) / 2  # many equal logits
    for m in range(0, M, 3):  # neighbours one step of FP32 apart
        logits[m] = 1.0 + torch.randint(0, 4, (E,), generator=g, device="cuda") * 2.0**-23
    for bias in (None, torch.round(rand(g, E) * 8) * 2.0**-24):
        want, _ = route(logits, k, score, bias, 1, 1, 1, True, 1.0)
        ids, _, _ = run_route(logits, k, score, bias, 1, 1, 1, True, 1.0, K.Act.F32)
        assert torch.equal(ids.cpu(), want)
        want, _ = route(logits, k, score, bias, 8, 3, 2, True, 1.0)
        ids, _, _ = run_route(logits, k, score, bias, 8, 3, 2, True, 1.0, K.Act.F32)
        assert torch.equal(ids.cpu(), want)


@pytest.mark.parametrize("score", ("softmax", "sigmoid"))
@pytest.mark.parametrize("E,k,G,tg", ((1024, 16, 4, 1), (1024, 16, 2, 1), (1024, 32, 8, 7), (1008, 16, 16, 1), (1000, 12, 8, 2), (128, 12, 8, 3), (510, 30, 17, 1), (96, 32, 3, 1)))
def test_route_few_open_experts(score, E, k, G, tg):
    """About as many picks as lanes that hold open experts, or more; the same with many equal scores and with scores one step apart."""
    g = gen(E + k + G)
    M = 150
    logits = rand(g, M, E) * 1.5 - 1.0
    logits[50:100] = torch.round(logits[50:100] * 2) / 2
    logits[100:] = 1.0 + torch.randint(0, 3, (50, E), generator=g, device="cuda") * 2.0**-23
    for bias in (None, rand(g, E) * 0.05, torch.round(rand(g, E) * 4) * 2.0**-24):
        for gt in (1, 2):
            want, cw = route(logits, k, score, bias, G, tg, gt, True, 2.5)
            ids, coef, _ = run_route(logits, k, score, bias, G, tg, gt, True, 2.5, K.Act.F32)
            assert torch.equal(ids.cpu(), want)
            assert ((coef.cpu().double() - cw).abs() <= cw.abs() * 44 * 2.0**-24).all()


def test_route_extremes_shared_slot_and_failed_tokens():
    E, k = 48, 5
    logits = torch.zeros((9, E + 4), device="cuda")  # column E is the shared gate; rows E + 4 apart
    logits[0] = -3.0e38  # sigmoid 0 everywhere: weights stay 0
    logits[1, :E] = torch.arange(E, device="cuda") * 1.0e37  # from expert 35 on beyond FP32 (3.4028e38): infinite
    logits[2, 7] = float("nan")
    logits[3, 40], logits[3, 9] = float("inf"), float("-inf")
    logits[4, E] = float("-inf")
    logits[5, :E] = -200.0 - torch.arange(E, device="cuda")  # scores far below FP32's range
    logits[6, :E] = 30.0 + torch.arange(E, device="cuda") / 64  # scores next to 1
    logits[7, E] = 1.25
    ids, coef, err = torch.full((9, k + 1), -7, dtype=torch.int32, device="cuda"), torch.full((9, k + 1), -7.0, device="cuda"), K.new_err()
    K.moe_router_scored(logits, E + 4, 9, E, k, "sigmoid", None, 4, 2, 2, True, 1.0, logits[:, E:], E + 4, E, ids, coef, K.Act.F32, err)
    ids, coef = ids.cpu(), coef.cpu()
    e = host_err(err)
    assert e[0] == 1 and (e[1], e[2]) in ((1, 35), (2, 7), (3, 9), (4, E))
    for m in (1, 2, 3, 4):
        assert (ids[m] == -1).all() and coef[m].isnan().all()
    assert (coef[0, :k] == 0).all() and (ids[0] >= 0).all()
    for m in (5, 6, 7, 8):
        want, cw = route(logits[m : m + 1, :E], k, "sigmoid", None, 4, 2, 2, True, 1.0)
        assert torch.equal(ids[m : m + 1, :k], want)
        assert ((coef[m, :k].double() - cw[0]).abs() <= cw[0] * 44 * 2.0**-24).all()
        assert int(ids[m, k]) == E
        gate = 1 / (1 + np.exp(-float(logits[m, E])))
        assert abs(float(coef[m, k]) - gate) <= gate * 6 * 2.0**-24
    # a non-finite bias fails every token
    bias = torch.zeros(E, device="cuda")
    bias[3] = float("-inf")
    ids, coef, err = run_route(torch.zeros((5, E), device="cuda"), k, "softmax", bias, 1, 1, 1, True, 1.0, K.Act.F32)
    assert (ids == -1).all() and coef.isnan().all() and host_err(err)[2] == 3


def test_route_hundreds_of_candidates_and_odd_views():
    """Equal logits: every expert is a candidate and the lowest indices win. Logits that start and are spaced so that no vector load is
    aligned give the same as a copy."""
    for E, G, tg, k in ((1024, 1, 1, 32), (768, 3, 2, 20), (1023, 1, 1, 5)):
        for score in ("softmax", "sigmoid"):
            logits, bias = torch.full((5, E), 0.25, device="cuda"), torch.full((E,), 0.5, device="cuda")
            for b in (None, bias):
                ids, coef, _ = run_route(logits, k, score, b, G, tg, 2, True, 1.0, K.Act.F32)
                assert torch.equal(ids.cpu(), torch.arange(k, dtype=torch.int32).expand(5, k)) and (coef - 1 / k).abs().max() < 1e-6 / k
    g = gen(9)
    wide = (rand(g, 33, 261) * 1.5).bfloat16()
    bias = rand(g, 257)[1:] * 0.05  # 4 bytes past an aligned address
    for act, base in ((K.Act.BF16, wide), (K.Act.F32, wide.float())):
        view = base[:, 3:]  # 256 experts used, rows 261 apart
        ids = torch.empty((33, 8), dtype=torch.int32, device="cuda")
        coef, err = torch.empty((33, 8), device="cuda"), K.new_err()
        K.moe_router_scored(view, 261, 33, 256, 8, "sigmoid", bias, 8, 4, 2, True, 2.5, None, 0, 0, ids, coef, act, err)
        want, cw = route(base[:, 3:259].float(), 8, "sigmoid", bias, 8, 4, 2, True, 2.5)
        assert torch.equal(ids.cpu(), want) and ((coef.cpu().double() - cw).abs() <= cw * 44 * 2.0**-24).all()
        with pytest.raises(StrixError, match="ends before"):
            K.moe_router_scored(base[1:, 3:], 261, 33, 256, 8, "sigmoid", bias, 8, 4, 2, True, 2.5, None, 0, 0, ids, coef, act, err)


# ---- norm and SwiGLU -------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,d", [(1, 16), (3, 128), (7, 144), (5, 2048), (2, 2560), (3, 4112), (2, 8192), (2, 16384), (301, 512)])
def test_rmsnorm_fp8(act, M, d):
    g = gen(M * 7 + d)
    dt = DT[act]
    # the sum of squares: up to 64 values a thread in turn, 5 + 8 partial sums, halved by the root; the root, the quotient, two products
    rel = (77 / 2 + 6) * 2.0**-24
    for residual, centered, alias in ((True, False, None), (False, True, None), (True, True, "x"), (True, False, "y")):
        x, y, w = (rand(g, M, d) * 3).to(dt), rand(g, M, d).to(dt) if residual else None, rand(g, d) * 0.1 + (0 if centered else 1)
        if M > 2:
            x[1] = 0
            if residual:
                y[1] = 0
        xs = (x.float() + y.float()).to(dt) if residual else x
        f = xs.double()
        h64 = f / torch.sqrt(f.pow(2).mean(1, keepdim=True) + 1e-5) * (w.double() + (1 if centered else 0))
        x_out = None if not residual else x.clone() if alias == "x" else y.clone() if alias == "y" else torch.empty_like(x)
        xi, yi = (x_out if alias == "x" else x), (x_out if alias == "y" else y)
        h, q, s = torch.empty_like(x), torch.empty((M, d), dtype=FP8, device="cuda"), torch.empty((M, blocks(d)), device="cuda")
        K.residual_rmsnorm_fp8(xi, yi, w, M, d, 1e-5, x_out, h, q, s, act, centered=centered)
        if residual:
            assert torch.equal(x_out, xs)
        tol = h64.abs() * (rel + (2.0**-8 if act == K.Act.BF16 else 0)) + 1e-37
        assert ((h.double() - h64).abs() <= tol).all()
        check_fp8_rows(q, s, h64, rel)
        # one of the two outputs alone
        h2, q2, s2 = torch.empty_like(h), torch.empty_like(q), torch.empty_like(s)
        K.residual_rmsnorm_fp8(x, y, w, M, d, 1e-5, torch.empty_like(x) if residual else None, h2, None, None, act, centered=centered)
        K.residual_rmsnorm_fp8(x, y, w, M, d, 1e-5, torch.empty_like(x) if residual else None, None, q2, s2, act, centered=centered)
        assert torch.equal(h2, h) and torch.equal(q2.view(torch.uint8), q.view(torch.uint8)) and torch.equal(s2, s)


def test_rmsnorm_fp8_nonfinite_rows_stay_apart():
    M, d = 4, 256
    x = torch.ones((M, d), device="cuda")
    x[1, 5], x[2, 200] = float("nan"), float("inf")
    h, q, s = torch.empty_like(x), torch.empty((M, d), dtype=FP8, device="cuda"), torch.empty((M, 2), device="cuda")
    K.residual_rmsnorm_fp8(x, None, torch.ones(d, device="cuda"), M, d, 0.0, None, h, q, s, K.Act.F32)
    assert h[1].isnan().all() and q[1].float().isnan().all() and s[1].isnan().all()
    assert h[2, 200].isnan() and h[2].nan_to_num(0).eq(0).all()
    assert s[2, 1].isnan() and q[2, 128:].float().isnan().all() and q[2, :128].float().eq(0).all()
    for m in (0, 3):
        assert h[m].eq(1).all() and (q[m].float() * s[m].repeat_interleave(128)).sub(1).abs().max() < 1e-6


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("rows,I", [(1, 16), (1, 512), (60, 512), (7, 640), (3, 144), (333, 128), (2, 8208), (5000, 16)])
def test_swiglu_fp8(act, rows, I):
    g = gen(rows + I)
    gu = (rand(g, rows, 2 * I) * 2).to(DT[act])
    gu[0, 0], gu[0, I] = 90.0, 2.0  # expf(-gate) at the ends of its range
    gu[0, 1], gu[0, I + 1] = -100.0, 2.0
    if rows > 2:
        gu[1] = 0
    q, s = torch.empty((rows, I), dtype=FP8, device="cuda"), torch.empty((rows, blocks(I)), device="cuda")
    K.swiglu_fp8(gu, q, s, rows, I, act)
    gate, up = gu.double()[:, :I], gu.double()[:, I:]
    check_fp8_rows(q, s, gate * torch.sigmoid(gate) * up, 8 * 2.0**-24)  # the exponential (4), 1 + e, the quotient, the product


def test_swiglu_fp8_nan_stays_in_its_block():
    gu = torch.ones((2, 512), device="cuda")
    gu[1, 130] = float("nan")
    q, s = torch.empty((2, 256), dtype=FP8, device="cuda"), torch.empty((2, 2), device="cuda")
    K.swiglu_fp8(gu, q, s, 2, 256, K.Act.F32)
    assert q[1, 128:].float().isnan().all() and s[1, 1].isnan() and not q[1, :128].float().isnan().any() and not q[0].float().isnan().any()


# ---- the dense product -----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("M,N,Kd", [(600, 1000, 2704), (2400, 300, 2576), (384, 4096, 4096), (1025, 517, 2448), (1, 128, 128), (1, 1, 16), (1, 2048, 4096), (6, 1024, 2048), (16, 100, 144), (17, 129, 1040), (33, 640, 2560), (64, 4096, 512),
                                    (65, 257, 272), (128, 384, 8192), (129, 512, 640), (300, 1000, 1040), (1000, 136, 256), (513, 2048, 1024), (256, 4096, 128)])
def test_linear_fp8(M, N, Kd):
    g = gen(M + N + Kd)
    xq, xs = rows_fp8(rand(g, M, Kd))
    wq, ws = matrix_fp8(rand(g, N, Kd) * 0.02 * torch.exp(rand(g, N, 1)))
    x, w = wide_rows(xq, xs), wide_matrix(wq, ws)
    y64 = x @ w.t()
    W = K.Fp8Weight(wq, ws)
    for act in ACTS:
        guard = torch.full((M * N + 64,), 7.0, dtype=DT[act], device="cuda")
        y = guard[: M * N].view(M, N)
        K.linear_fp8(xq, xs, W, y, M, act)
        assert ((y.double() - y64).abs() <= product_bound(x.abs(), w.abs(), Kd, y64, act == K.Act.BF16)).all()
        assert (guard[M * N :] == 7.0).all()
        again = torch.empty_like(y)
        K.linear_fp8(xq, xs, W, again, M, act)
        assert torch.equal(again, y)
    assert K.umma_abort_count() == 0


def test_linear_fp8_nan_and_zero_rows_stay_apart():
    g = gen(3)
    M, N, Kd = 40, 300, 384
    x = rand(g, M, Kd)
    x[5] = 0
    xq, xs = rows_fp8(x)
    wq, ws = matrix_fp8(rand(g, N, Kd))
    xq.view(torch.uint8)[7, 200] = 0x7F
    wq.view(torch.uint8)[130, 3] = 0xFF
    xs[9, 2] = float("inf")
    y = torch.empty((M, N), device="cuda")
    K.linear_fp8(xq, xs, K.Fp8Weight(wq, ws), y, M, K.Act.F32)
    bad = ~y.isfinite()
    want = torch.zeros_like(bad)
    want[7], want[9], want[:, 130] = True, True, True
    assert torch.equal(bad, want)
    keep = torch.ones(N, dtype=torch.bool, device="cuda")
    keep[130] = False
    assert (y[5][keep] == 0).all()


def test_rows_and_outputs_past_32_bit_offsets():
    """More than 2^31 elements: the last rows are where they belong."""
    g = gen(11)
    M, d = 1100000, 2048
    x = torch.zeros((M, d), dtype=torch.bfloat16, device="cuda")
    x[0], x[-1] = rand(g, d), rand(g, d)
    q, s, w = torch.empty((M, d), dtype=FP8, device="cuda"), torch.empty((M, 16), device="cuda"), torch.ones(d, device="cuda")
    K.residual_rmsnorm_fp8(x, None, w, M, d, 1e-5, None, None, q, s, K.Act.BF16)
    for r in (0, M - 1):
        f = x[r : r + 1].double()
        check_fp8_rows(q[r : r + 1], s[r : r + 1], f / torch.sqrt(f.pow(2).mean(1, keepdim=True) + 1e-5), 45 * 2.0**-24)
    assert (q[M // 2].float() == 0).all()
    gu = x.view(M // 2, 2 * d)  # the same elements as merged rows of I = d
    q2, s2 = q.view(torch.uint8).view(-1)[: M // 2 * d].view(FP8).view(M // 2, d), s[: M // 2]
    K.swiglu_fp8(gu, q2, s2, M // 2, d, K.Act.BF16)
    last = gu[-1:].double()
    check_fp8_rows(q2[-1:], s2[-1:], last[:, :d] * torch.sigmoid(last[:, :d]) * last[:, d:], 8 * 2.0**-24)
    del x, gu, q, q2, s, s2
    M, N, Kd = 66000, 33000, 128
    xq, xs = rows_fp8(rand(g, M, Kd))
    wq, ws = matrix_fp8(rand(g, N, Kd))
    y = torch.empty((M, N), dtype=torch.bfloat16, device="cuda")
    K.linear_fp8(xq, xs, K.Fp8Weight(wq, ws), y, M, K.Act.BF16)
    for r in (0, 65070, M - 1):  # 65076 rows hold 2^31 elements
        a, b = wide_rows(xq[r : r + 1], xs[r : r + 1]), wide_matrix(wq, ws)
        y64 = a @ b.t()
        assert ((y[r : r + 1].double() - y64).abs() <= product_bound(a.abs(), b.abs(), Kd, y64, True)).all()


def test_linear_fp8_output_at_any_element():
    g = gen(12)
    for M, N, Kd in ((5, 130, 256), (600, 136, 384)):  # narrow and wide form, stores that are not aligned to vectors
        xq, xs = rows_fp8(rand(g, M, Kd))
        W = K.Fp8Weight(*matrix_fp8(rand(g, N, Kd)))
        for act in ACTS:
            want = torch.empty((M, N), dtype=DT[act], device="cuda")
            K.linear_fp8(xq, xs, W, want, M, act)
            room = torch.full((M * N + 9,), 3.0, dtype=DT[act], device="cuda")
            y = room[1 : 1 + M * N].view(M, N)
            K.linear_fp8(xq, xs, W, y, M, act)
            assert torch.equal(y, want) and room[0] == 3.0 and (room[1 + M * N :] == 3.0).all()


# ---- the experts' products -------------------------------------------------------------------------------------------


def group(ids, E):
    M, A = ids.shape
    n = K.moe_route_workspace_bytes(M, A, E)
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    err = K.new_err()
    K.moe_group_routes(ids, M, A, E, ws, n, err)
    return ws, n, err


def some_ids(g, M, A, E, kind):
    ids = torch.rand((M, E), generator=g, device="cuda").topk(A, dim=1).indices.int() if A <= E else torch.randint(0, E, (M, A), generator=g, device="cuda").int()
    if kind == "one":  # every token to the same expert first: one long list, some empty ones
        ids[:, 0] = E - 1
    if kind == "steep":  # lists of one slot next to lists of hundreds, several tiles of each for every block of threads
        share = torch.arange(1, E + 1, device="cuda").float() ** -1.5
        ids = torch.multinomial(share.expand(M, E), A, generator=g).int()
        ids = torch.randperm(E, generator=g, device="cuda").int()[ids.long()]
    if kind == "bad":
        ids[0, 0], ids[M - 1, A - 1] = -1, E
    if kind == "none":
        ids[:] = -1
    return ids.contiguous()


@pytest.mark.parametrize("M,A,E,N,Kd,kind", [(1, 1, 1, 128, 128, ""), (1, 8, 64, 1024, 512, ""), (6, 10, 64, 512, 640, "bad"), (1, 3, 5, 100, 144, "bad"), (40, 4, 16, 256, 256, "one"),
                                             (300, 2, 8, 136, 1040, "bad"), (700, 3, 6, 257, 272, "one"), (9, 2, 1023, 16, 16, ""), (33, 64, 7, 128, 128, ""), (5, 4, 8, 128, 256, "none"),
                                             (600, 8, 16, 640, 384, ""), (1000, 6, 300, 128, 128, "bad"), (4000, 4, 96, 1000, 640, "steep"), (700, 2, 64, 2048, 512, "steep"), (200, 4, 100, 2048, 512, "steep"),
                                             (6, 10, 512, 2048, 512, "steep")])
def test_experts(M, A, E, N, Kd, kind):
    g = gen(M * A + E + N)
    ids = some_ids(g, M, A, E, kind)
    wq, wsc = stack_fp8(rand(g, E, N, Kd) * 0.02)
    W = K.Fp8Weight(wq, wsc, experts=E)
    ws, n, _ = group(ids, E)
    w64 = torch.stack([wide_matrix(wq[e * N : (e + 1) * N], wsc[e * blocks(N) : (e + 1) * blocks(N)]) for e in range(E)])
    flat = ids.view(-1).long()
    ok = (flat >= 0) & (flat < E)

    def exact(rows):  # rows [M * A, Kd] in 64 bits
        y, tol = torch.zeros((M * A, N), dtype=torch.float64, device="cuda"), torch.zeros((M * A, N), dtype=torch.float64, device="cuda")
        for e in flat[ok].unique().tolist():
            at = flat == e
            y[at] = rows[at] @ w64[e].t()
            tol[at] = product_bound(rows[at].abs(), w64[e].abs(), Kd, y[at], False)
        return y, tol

    xq, xs = rows_fp8(rand(g, M, Kd))
    y64, tol = exact(wide_rows(xq, xs).repeat_interleave(A, 0))
    for act in ACTS:
        guard = torch.full((M * A * N + 64,), 7.0, dtype=DT[act], device="cuda")
        y = guard[: M * A * N].view(M * A, N)
        K.linear_fp8_experts_gather_grouped(xq, xs, W, E, ws, n, M, A, y, act)
        t = tol + (y64.abs() + tol) * 2.0**-8 if act == K.Act.BF16 else tol
        assert ((y.double() - y64).abs() <= t)[ok].all()
        assert (y[~ok] == 7.0).all() and (guard[M * A * N :] == 7.0).all()  # slots without an expert are left as they were

    hq, hs = rows_fp8(rand(g, M * A, Kd))
    coef = torch.rand((M, A), generator=g, device="cuda")
    p64, tol = exact(wide_rows(hq, hs))
    c = coef.double()[:, :, None]
    s64 = (p64.view(M, A, N) * c).sum(1)
    terms = (p64.view(M, A, N) * c).abs().sum(1)
    t32 = (tol.view(M, A, N) * c).sum(1) + terms * A * 2.0**-24
    failed = ~ok.view(M, A).all(1)
    for act in ACTS:
        partial, y = torch.empty((M * A, N), device="cuda"), torch.full((M, N), 7.0, dtype=DT[act], device="cuda")
        K.linear_fp8_experts_combine_grouped(hq, hs, W, E, ids, coef, ws, n, partial, M, A, y, act)
        t = t32 + (s64.abs() + t32) * 2.0**-8 if act == K.Act.BF16 else t32
        assert ((y.double() - s64).abs() <= t)[~failed].all()
        assert y[failed].isnan().all()
    assert K.umma_abort_count() == 0


def test_experts_refuse_a_workspace_of_other_sizes():
    """The same bytes, grouped for another split of the slots: nothing is stored, and it is counted."""
    E, N, Kd = 4, 128, 128
    g = gen(1)
    ws, n, _ = group(some_ids(g, 6, 2, E, ""), E)
    wq, wsc = stack_fp8(rand(g, E, N, Kd))
    xq, xs = rows_fp8(rand(g, 11, Kd))
    y = torch.full((11, N), 7.0, device="cuda")
    before = K.workspace_refusal_count()
    K.linear_fp8_experts_gather_grouped(xq, xs, K.Fp8Weight(wq, wsc, experts=E), E, ws, n, 11, 1, y, K.Act.F32)
    assert K.workspace_refusal_count() == before + 1 and (y == 7.0).all()


@pytest.mark.parametrize("M,A,E", [(2047, 1, 5), (2048, 1, 1023), (1, 64, 1), (700, 3, 512), (4097, 11, 513), (16384, 64, 1023), (65536, 10, 8)])
def test_grouping_by_one_block_and_by_a_cluster(M, A, E):
    """The workspace is a pure function of the ids, whichever form groups them (one block below 2048 slots, a cluster from there on)."""
    rng = np.random.default_rng(M + A)
    ids = rng.integers(0, E, (M, A)).astype(np.int32)
    ids[rng.random((M, A)) < 0.3] = E - 1
    if M > 1000:
        ids[M // 2, 0], ids[M - 1, A - 1] = -5, E
    ref, err_ref = oracle.group_routes(ids, E)
    t = torch.from_numpy(ids).cuda()
    n = K.moe_route_workspace_bytes(M, A, E)
    for _ in range(2):
        ws, err = torch.full((n // 4,), -99, dtype=torch.int32, device="cuda"), K.new_err()
        K.moe_group_routes(t, M, A, E, ws, n, err)
        got = ws.cpu().numpy()
        head = 4 + E + 2 + M * A
        assert np.array_equal(got[:head], ref[:head])
        Tmax, WTmax = M * A // 16 + E + 2, M * A // 64 + E + 2
        for at, size, count in ((head, Tmax, ref[0]), (head + 2 * Tmax, WTmax, ref[3])):
            for col in (at, at + size):
                assert np.array_equal(got[col : col + count], ref[col : col + count])
        assert host_err(err) == [int(v) for v in err_ref[:3]]


# ---- the run ---------------------------------------------------------------------------------------------------------


class Ffn:
    """A layer in FP8: norm -> routing -> experts' gate and up -> SwiGLU -> down and combine, plus a shared expert."""

    def __init__(self, seed, M, d, I, E, k, act):
        g = gen(seed)
        self.M, self.d, self.I, self.E, self.k, self.act, dt = M, d, I, E, k, act, DT[act]
        self.x, self.y = (rand(g, M, d) * 2).to(dt), rand(g, M, d).to(dt)
        self.gain, self.bias, self.router = rand(g, d) * 0.1 + 1, rand(g, E) * 0.02, (rand(g, E, d) * 0.02).bfloat16()
        self.gu = K.Fp8Weight(*stack_fp8(rand(g, E, 2 * I, d) * 0.02), experts=E)
        self.dn = K.Fp8Weight(*stack_fp8(rand(g, E, d, I) * 0.02), experts=E)
        self.sgu, self.sdn = K.Fp8Weight(*matrix_fp8(rand(g, 2 * I, d) * 0.02)), K.Fp8Weight(*matrix_fp8(rand(g, d, I) * 0.02))
        e = lambda *s, t=torch.float32: torch.zeros(s, dtype=t, device="cuda")  # noqa: E731
        S = M * k
        self.b = dict(x_out=e(M, d, t=dt), h=e(M, d, t=dt), q=e(M, d, t=FP8), s=e(M, blocks(d)), logits=e(M, E), ids=e(M, k, t=torch.int32), coef=e(M, k), err=e(4, t=torch.int32),
                      g1=e(S, 2 * I, t=dt), hq=e(S, I, t=FP8), hs=e(S, blocks(I)), partial=e(S, d), out=e(M, d, t=dt), sg=e(M, 2 * I, t=dt), sq=e(M, I, t=FP8), ss=e(M, blocks(I)),
                      sy=e(M, d, t=dt))
        self.n = K.moe_route_workspace_bytes(M, k, E)
        self.ws = torch.zeros(self.n, dtype=torch.uint8, device="cuda")

    def forward(self, stream=None):
        b, M, d, I, E, k, act = self.b, self.M, self.d, self.I, self.E, self.k, self.act
        K.residual_rmsnorm_fp8(self.x, self.y, self.gain, M, d, 1e-6, b["x_out"], b["h"], b["q"], b["s"], act, stream=stream)
        K.linear_bf16w(b["h"], self.router, b["logits"], M, E, d, act, K.Act.F32, stream=stream)
        K.moe_router_scored(b["logits"], E, M, E, k, "sigmoid", self.bias, 4, 2, 2, True, 2.5, None, 0, 0, b["ids"], b["coef"], K.Act.F32, b["err"], stream=stream)
        K.moe_group_routes(b["ids"], M, k, E, self.ws, self.n, b["err"], stream=stream)
        K.linear_fp8_experts_gather_grouped(b["q"], b["s"], self.gu, E, self.ws, self.n, M, k, b["g1"], act, stream=stream)
        K.swiglu_fp8(b["g1"], b["hq"], b["hs"], M * k, I, act, stream=stream)
        K.linear_fp8_experts_combine_grouped(b["hq"], b["hs"], self.dn, E, b["ids"], b["coef"], self.ws, self.n, b["partial"], M, k, b["out"], act, stream=stream)
        K.linear_fp8(b["q"], b["s"], self.sgu, b["sg"], M, act, stream=stream)
        K.swiglu_fp8(b["sg"], b["sq"], b["ss"], M, I, act, stream=stream)
        K.linear_fp8(b["sq"], b["ss"], self.sdn, b["sy"], M, act, stream=stream)
        K.residual_add(b["out"], b["sy"], M * d, act, stream=stream)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", (1, 6, 150))
def test_ffn_in_fp8(act, M):
    """Every step against the 64-bit form of the step before it (a code that lands on the other side of a rounding border at one step
    is an input of the next)."""
    f = Ffn(M, M, 512, 256, 16, 4, act)
    f.forward()
    b, E, k, I, d = f.b, f.E, f.k, f.I, f.d
    bf = act == K.Act.BF16
    assert host_err(b["err"])[0] == 0
    xo = b["x_out"].double()
    h64 = xo / torch.sqrt(xo.pow(2).mean(1, keepdim=True) + 1e-6) * f.gain.double()
    check_fp8_rows(b["q"], b["s"], h64, 45 * 2.0**-24)
    ids, coef = route(b["logits"], k, "sigmoid", f.bias, 4, 2, 2, True, 2.5)
    assert torch.equal(b["ids"].cpu(), ids) and ((b["coef"].cpu().double() - coef).abs() <= coef * 44 * 2.0**-24).all()
    x = wide_rows(b["q"], b["s"])
    flat = b["ids"].view(-1).long()

    def stack(w, n):
        return torch.stack([wide_matrix(w.q[e * n : (e + 1) * n], w.scale[e * blocks(n) : (e + 1) * blocks(n)]) for e in range(E)])

    gu, dn = stack(f.gu, 2 * I), stack(f.dn, d)
    for s in range(M * k):
        row = x[s // k : s // k + 1]
        y = row @ gu[flat[s]].t()
        assert ((b["g1"][s : s + 1].double() - y).abs() <= product_bound(row.abs(), gu[flat[s]].abs(), d, y, bf)).all()
    g1 = b["g1"].double()
    check_fp8_rows(b["hq"], b["hs"], g1[:, :I] * torch.sigmoid(g1[:, :I]) * g1[:, I:], 8 * 2.0**-24)
    hw = wide_rows(b["hq"], b["hs"])
    p = torch.stack([(hw[s : s + 1] @ dn[flat[s]].t())[0] for s in range(M * k)])
    tol = torch.stack([product_bound(hw[s : s + 1].abs(), dn[flat[s]].abs(), I, p[s : s + 1], False)[0] for s in range(M * k)])
    c = b["coef"].double()[:, :, None]
    routed, slack = (p.view(M, k, d) * c).sum(1), (tol.view(M, k, d) * c).sum(1) + (p.view(M, k, d) * c).abs().sum(1) * k * 2.0**-24
    sy = b["sy"].double()
    step = 2.0**-8 if bf else 2.0**-24
    assert ((b["out"].double() - (routed + sy)).abs() <= slack + (routed.abs() + slack) * step + (routed + sy).abs() * step + 1e-30).all()


def test_ffn_in_a_graph_on_streams_and_side_by_side():
    """Captured and replayed with other inputs, on a stream of its own, and two layers at once on two streams: the bits of the plain run."""
    f, o = Ffn(1, 40, 512, 256, 16, 4, K.Act.BF16), Ffn(2, 40, 512, 256, 16, 4, K.Act.BF16)
    keys = [k for k in f.b if k != "partial"]
    bits = lambda l: {k: l.b[k].clone().view(torch.uint8) for k in keys}  # noqa: E731
    f.forward(), o.forward()
    torch.cuda.synchronize()
    want_f, want_o = bits(f), bits(o)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        f.forward(stream=s1), o.forward(stream=s2)
    torch.cuda.synchronize()
    for l, want in ((f, want_f), (o, want_o)):
        assert all(torch.equal(v, bits(l)[k]) for k, v in want.items())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        f.forward()
    x = f.x.clone()
    f.x.copy_(o.x)
    graph.replay()
    torch.cuda.synchronize()
    other = bits(f)
    f.forward()
    torch.cuda.synchronize()
    assert all(torch.equal(v, bits(f)[k]) for k, v in other.items()) and not torch.equal(other["out"], want_f["out"])
    f.x.copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(v, bits(f)[k]) for k, v in want_f.items())


def test_ffn_with_the_shared_expert_on_a_second_stream():
    """The shared expert beside the routed ones, forked and joined by events, eager and captured: the bits of the run on one stream."""
    f = Ffn(3, 600, 512, 256, 16, 4, K.Act.BF16)
    f.forward()
    torch.cuda.synchronize()
    keys = [k for k in f.b if k != "partial"]
    want = {k: f.b[k].clone().view(torch.uint8) for k in keys}
    side = torch.cuda.Stream()

    def forked():
        b, M, d, I, E, k, act = f.b, f.M, f.d, f.I, f.E, f.k, f.act
        K.residual_rmsnorm_fp8(f.x, f.y, f.gain, M, d, 1e-6, b["x_out"], b["h"], b["q"], b["s"], act)
        side.wait_stream(torch.cuda.current_stream())
        K.linear_fp8(b["q"], b["s"], f.sgu, b["sg"], M, act, stream=side)
        K.swiglu_fp8(b["sg"], b["sq"], b["ss"], M, I, act, stream=side)
        K.linear_fp8(b["sq"], b["ss"], f.sdn, b["sy"], M, act, stream=side)
        K.linear_bf16w(b["h"], f.router, b["logits"], M, E, d, act, K.Act.F32)
        K.moe_router_scored(b["logits"], E, M, E, k, "sigmoid", f.bias, 4, 2, 2, True, 2.5, None, 0, 0, b["ids"], b["coef"], K.Act.F32, b["err"])
        K.moe_group_routes(b["ids"], M, k, E, f.ws, f.n, b["err"])
        K.linear_fp8_experts_gather_grouped(b["q"], b["s"], f.gu, E, f.ws, f.n, M, k, b["g1"], act)
        K.swiglu_fp8(b["g1"], b["hq"], b["hs"], M * k, I, act)
        K.linear_fp8_experts_combine_grouped(b["hq"], b["hs"], f.dn, E, b["ids"], b["coef"], f.ws, f.n, b["partial"], M, k, b["out"], act)
        torch.cuda.current_stream().wait_stream(side)
        K.residual_add(b["out"], b["sy"], M * d, act)

    def wipe():
        for k in keys:
            f.b[k].view(torch.uint8).zero_()

    wipe()
    forked()
    torch.cuda.synchronize()
    assert all(torch.equal(v, f.b[k].view(torch.uint8)) for k, v in want.items())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        forked()
    for _ in range(2):
        wipe()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(v, f.b[k].view(torch.uint8)) for k, v in want.items())


def test_wrappers_refuse_wrong_tensors():
    x = torch.zeros((4, 256), device="cuda")
    q, s = torch.zeros((4, 256), dtype=FP8, device="cuda"), torch.zeros((4, 2), device="cuda")
    w = torch.ones(256, device="cuda")
    for args, what in (((x.half(), None, w, 4, 256, 1e-6, None, None, q, s, 0), "float32"), ((x, None, w, 5, 256, 1e-6, None, None, q, s, 0), "1280"),
                       ((x.t(), None, w, 4, 256, 1e-6, None, None, q, s, 0), "contiguous"), ((x.cpu(), None, w, 4, 256, 1e-6, None, None, q, s, 0), "current device"),
                       ((x, None, w, 4, 256, 1e-6, None, None, q.half(), s, 0), "float8"), ((x, None, w, 4, 256, 1e-6, None, None, q, s, 7), "dtype 7"),
                       ((x, x, w, 4, 256, 1e-6, None, None, q, s, 0), "x_out"), ((x, None, w, 4, 256, 1e-6, None, None, None, None, 0), "neither")):
        with pytest.raises(StrixError, match=what):
            K.residual_rmsnorm_fp8(*args)
    W = K.Fp8Weight(torch.zeros((256, 256), dtype=FP8, device="cuda"), torch.ones((2, 2), device="cuda"))
    y = torch.zeros((4, 256), device="cuda")
    with pytest.raises(StrixError, match="1024"):
        K.linear_fp8(q, s, W, y[:2], 4, K.Act.F32)
    with pytest.raises(StrixError, match="holds 1 experts"):
        K.linear_fp8_experts_gather_grouped(q, s, W, 2, torch.zeros(4096, dtype=torch.uint8, device="cuda"), 4096, 4, 1, y, K.Act.F32)
    with pytest.raises(StrixError, match="score"):
        K.moe_router_scored(x, 256, 4, 256, 2, "top", None, 1, 1, 1, True, 1.0, None, 0, 0, torch.zeros(8, dtype=torch.int32, device="cuda"), torch.zeros(8, device="cuda"), 0, K.new_err())

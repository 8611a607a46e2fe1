"""CPU: what the FP8 entry points refuse, with a message and before anything reaches a device."""
import ctypes as C

import pytest
import torch

from strixite_b200 import Fp8Weight, StrixError
from strixite_b200._lib import Fp8View, last_error, lib


@pytest.fixture()
def mem():
    """Distinct aligned addresses, 1 MiB apart: nothing is read from them."""
    buf = (C.c_char * 64)()
    base = (C.addressof(buf) + (1 << 24)) // 256 * 256
    return lambda i: C.c_void_p(base + (i << 20))


def refused(rc, text):
    assert rc == 1 and text in last_error(), (rc, last_error())


def test_router_scored(mem):
    def call(M=4, E=64, k=8, ld=64, score=1, G=8, tg=4, gt=2, scale=1.0, shared=None, shared_ld=1, shared_id=0, act=0, ids=mem(1), coef=mem(2), logits=mem(0), err=mem(3), bias=None):
        return lib.strix_moe_router_scored(logits, ld, M, E, k, score, bias, G, tg, gt, 1, scale, shared, shared_ld, shared_id, ids, coef, act, err, None)

    refused(call(logits=None), "null pointer")
    refused(call(err=None), "null pointer")
    refused(call(M=0), "M = 0")
    refused(call(E=1025, ld=1025), "E = 1025")
    refused(call(score=2), "score 2")
    refused(call(G=7), "n_group = 7")
    refused(call(G=0), "n_group = 0")
    refused(call(E=66, ld=66, G=33), "n_group = 33")
    refused(call(tg=9), "topk_group = 9")
    refused(call(tg=0), "topk_group = 0")
    refused(call(gt=3), "group_top = 3")
    refused(call(k=0), "k = 0")
    refused(call(k=33), "k = 33")
    refused(call(tg=1, k=9), "k = 9")  # 8 experts in one open group
    refused(call(ld=63), "ld = 63")
    refused(call(scale=float("nan")), "route_scale")
    refused(call(scale=float("inf")), "route_scale")
    refused(call(act=2), "dtype 2")
    refused(call(shared=mem(4), shared_ld=0), "shared_ld")
    refused(call(shared=mem(4), shared_id=-1), "shared_id")
    refused(call(coef=mem(1)), "overlap")
    refused(call(ids=mem(0)), "overlaps the logits")
    refused(call(coef=mem(4), bias=mem(4)), "overlaps the bias")
    refused(call(coef=mem(4), shared=mem(4)), "overlaps the shared logits")
    refused(call(ld=1 << 40), "row strides")
    refused(call(shared=mem(4), shared_ld=1 << 40), "row strides")


def test_norm(mem):
    def call(x=mem(0), y=mem(1), w=mem(2), eps=1e-6, M=2, d=256, x_out=mem(3), h=mem(4), q=mem(5), s=mem(6), act=0):
        return lib.strix_residual_rmsnorm_fp8(x, y, w, 0, eps, M, d, x_out, h, q, s, act, None)

    refused(call(x=None), "null pointer")
    refused(call(w=None), "null pointer")
    refused(call(y=None), "x_out come together")
    refused(call(x_out=None), "x_out come together")
    refused(call(s=None), "scale come together")
    refused(call(h=None, q=None, s=None), "neither")
    refused(call(M=0), "M = 0")
    for d in (0, 8, 24, 16400):
        refused(call(d=d), "d = %d" % d)
    refused(call(eps=-1.0), "eps")
    refused(call(eps=float("nan")), "eps")
    refused(call(act=3), "dtype 3")
    refused(call(x=C.c_void_p(mem(0).value + 4)), "aligned")
    refused(call(s=C.c_void_p(mem(6).value + 2)), "aligned")
    refused(call(x_out=C.c_void_p(mem(0).value + 16)), "partly overlaps")
    refused(call(h=mem(0)), "overlaps input")
    refused(call(q=mem(4)), "overlap")
    refused(call(w=mem(4)), "overlaps input")


def test_swiglu(mem):
    def call(gu=mem(0), q=mem(1), s=mem(2), rows=2, I=256, act=0):
        return lib.strix_swiglu_fp8(gu, q, s, rows, I, act, None)

    refused(call(gu=None), "null pointer")
    refused(call(s=None), "null pointer")
    refused(call(rows=0), "rows = 0")
    for I in (0, 8, 100):
        refused(call(I=I), "I = %d" % I)
    refused(call(rows=1 << 34), "too large")
    refused(call(act=-1), "dtype -1")
    refused(call(gu=C.c_void_p(mem(0).value + 8)), "aligned")
    refused(call(q=mem(0)), "overlap")


def test_linear(mem):
    def call(xq=mem(0), xs=mem(1), q=mem(2), scale=mem(3), N=256, K=256, y=mem(4), M=4, act=0):
        v = Fp8View(q.value if q else None, scale.value if scale else None, N, K)
        return lib.strix_linear_fp8(xq, xs, C.byref(v), y, M, act, None)

    refused(lib.strix_linear_fp8(mem(0), mem(1), None, mem(4), 4, 0, None), "null weight")
    refused(call(q=None), "null weight")
    refused(call(xq=None), "null pointer")
    refused(call(y=None), "null pointer")
    refused(call(M=0), "M = 0")
    refused(call(N=0), "weight [0")
    for K in (0, 8, 120):
        refused(call(K=K), "weight [256, %d]" % K)
    refused(call(q=C.c_void_p(mem(2).value + 8)), "aligned")
    refused(call(xq=C.c_void_p(mem(0).value + 8)), "aligned")
    refused(call(y=C.c_void_p(mem(4).value + 2)), "aligned")
    refused(call(y=C.c_void_p(mem(4).value + 1), act=1), "aligned")
    refused(call(act=2), "dtype 2")
    refused(call(y=mem(0)), "overlaps")
    refused(call(y=mem(1)), "overlaps")
    refused(call(M=1 << 30, N=1 << 20, K=16, y=C.c_void_p(1 << 52)), "too many tiles")


def test_experts(mem):
    need = lib.strix_moe_route_workspace_bytes(4, 2, 8)

    def gather(xq=mem(0), E=8, ws=mem(2), n=need, M=4, A=2, y=mem(3), N=8 * 64, K=256, act=0):
        v = Fp8View(mem(4).value, mem(5).value, N, K)
        return lib.strix_linear_fp8_experts_gather_grouped(xq, mem(1), C.byref(v), E, ws, n, M, A, y, act, None)

    refused(gather(xq=None), "null pointer")
    refused(gather(E=7), "E = 7")
    refused(gather(E=0), "E = 0")
    refused(gather(E=1024, N=1024 * 64), "E = 1024")
    refused(gather(M=0), "M = 0")
    refused(gather(A=65), "A = 65")
    refused(gather(M=1 << 20, A=2), "A = 2")
    refused(gather(ws=None), "workspace")
    refused(gather(n=need - 4), "needs %d" % need)
    refused(gather(K=100), "100]")
    refused(gather(y=mem(0)), "overlaps")
    refused(gather(y=mem(2)), "overlaps the workspace")

    def combine(ids=mem(6), coef=mem(7), partial=mem(8), y=mem(3), E=8, n=need, act=0, hq=mem(0)):
        v = Fp8View(mem(4).value, mem(5).value, 8 * 64, 256)
        return lib.strix_linear_fp8_experts_combine_grouped(hq, mem(1), C.byref(v), E, ids, coef, mem(2), n, partial, 4, 2, y, act, None)

    refused(combine(ids=None), "null pointer")
    refused(combine(coef=None), "null pointer")
    refused(combine(partial=None), "partial")
    refused(combine(partial=mem(3)), "overlaps y")
    refused(combine(y=mem(6)), "overlaps ids")
    refused(combine(y=mem(0)), "overlaps the rows")
    refused(combine(y=mem(2)), "overlaps the workspace")
    refused(combine(act=5), "dtype 5")
    refused(combine(E=3), "E = 3")
    refused(combine(n=8), "needs %d" % need)
    refused(combine(hq=None), "null pointer")
    refused(combine(ids=C.c_void_p(mem(6).value + 2)), "4-byte aligned")
    refused(combine(coef=C.c_void_p(mem(7).value + 2)), "4-byte aligned")


def test_weight_object():
    q, s = torch.zeros((256, 144), dtype=torch.float8_e4m3fn), torch.ones((2, 2))
    assert Fp8Weight(q, s).nbytes() == 256 * 144 + 16
    assert Fp8Weight(q, torch.ones((4, 2)), experts=4).view().N == 256  # 64 rows an expert: a block row each
    for bad in (lambda: Fp8Weight(q.float(), s), lambda: Fp8Weight(q, s.double()), lambda: Fp8Weight(q, torch.ones((2, 1))), lambda: Fp8Weight(q.t(), s),
                lambda: Fp8Weight(q, s, experts=3), lambda: Fp8Weight(q, s, experts=0), lambda: Fp8Weight(q.view(-1), s)):
        with pytest.raises(StrixError):
            bad()


@pytest.mark.parametrize("act,off", ((0, 2), (0, 1), (1, 1)))
def test_combine_refuses_an_output_off_its_elements(mem, act, off):
    v = Fp8View(mem(4).value, mem(5).value, 8 * 64, 256)
    need = lib.strix_moe_route_workspace_bytes(4, 2, 8)
    y = C.c_void_p(mem(3).value + off)
    refused(lib.strix_linear_fp8_experts_combine_grouped(mem(0), mem(1), C.byref(v), 8, mem(6), mem(7), mem(2), need, mem(8), 4, 2, y, act, None), "aligned to its elements")


@pytest.mark.parametrize("act,which,off", ((0, "logits", 2), (1, "logits", 1), (0, "shared", 2), (1, "shared", 1), (0, "bias", 2), (0, "ids", 2), (1, "coef", 1), (1, "err", 2)))
def test_router_scored_refuses_pointers_off_their_elements(mem, act, which, off):
    p = {n: mem(i) for i, n in enumerate(("logits", "shared", "bias", "ids", "coef", "err"))}
    p[which] = C.c_void_p(p[which].value + off)
    refused(lib.strix_moe_router_scored(p["logits"], 64, 4, 64, 8, 1, p["bias"], 8, 4, 2, 1, 1.0, p["shared"], 1, 64, p["ids"], p["coef"], act, p["err"], None), "aligned to")


def test_the_package_imports_where_torch_has_no_cuda_calls():
    """A torch built without CUDA lacks these names; the quantizers, views and refusals work there."""
    import os
    import subprocess
    import sys

    code = ("import torch\n"
            "for n in ('_cuda_getCurrentRawStream', '_cuda_getDevice'):\n"
            "    if hasattr(torch._C, n): delattr(torch._C, n)\n"
            "from strixite_b200 import Fp8Weight, kernels as K\n"
            "w = Fp8Weight(torch.zeros((128, 128), dtype=torch.float8_e4m3fn), torch.ones((1, 1)))\n"
            "assert w.nbytes() == 128 * 128 + 4 and K.moe_route_workspace_bytes(4, 2, 8) > 0\n")
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

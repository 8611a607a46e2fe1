"""GPU: the FP8 path where its kernels change over - rows near FP32's ends, scores far below one, workspaces of other sizes, products whose
rows, tiles and K blocks end off every boundary."""
import pytest
import torch

from fp8_ref import rows_fp8, stack_fp8
from strixite_b200 import kernels as K
from test_gpu_fp8 import ACTS, DT, gen, group, rand, some_ids

pytestmark = pytest.mark.gpu


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

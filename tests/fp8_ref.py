"""Plain 64-bit forms of the FP8 operators for the tests, and inputs for them."""
import torch

FP8 = torch.float8_e4m3fn


def blocks(n):
    return -(-n // 128)


def rows_fp8(x):
    """FP32/64 rows [R, K] -> (q e4m3, scale f32 [R, blocks]) by the definition, in 64 bits."""
    R, K = x.shape
    pad = torch.zeros((R, blocks(K) * 128), dtype=torch.float64, device=x.device)
    pad[:, :K] = x.double()
    pad = pad.view(R, -1, 128)
    s = (pad.abs().amax(2).clamp_min(2.0**-100) / 448).float()
    q = (pad / s.double()[:, :, None]).clamp(-448, 448).view(R, -1)[:, :K].to(FP8).contiguous()
    return q, s


def matrix_fp8(w):
    """[N, K] -> (q e4m3, scale [blocks(N), blocks(K)])."""
    N, K = w.shape
    pad = torch.zeros((blocks(N) * 128, blocks(K) * 128), dtype=torch.float64, device=w.device)
    pad[:N, :K] = w.double()
    b = pad.view(blocks(N), 128, blocks(K), 128)
    s = (b.abs().amax((1, 3)).clamp_min(2.0**-100) / 448).float()
    q = (b / s.double()[:, None, :, None]).clamp(-448, 448).view(blocks(N) * 128, -1)[:N, :K].to(FP8).contiguous()
    return q, s


def stack_fp8(w):
    """[E, N, K] -> (q [E * N, K], scale [E * blocks(N), blocks(K)])."""
    parts = [matrix_fp8(m) for m in w]
    return torch.cat([p[0].view(torch.uint8) for p in parts]).view(FP8), torch.cat([p[1] for p in parts])


def wide_rows(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)[:, : q.shape[1]]


def wide_matrix(q, s):
    return q.double() * s.double().repeat_interleave(128, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def route(logits, k, score, bias, G, topk_group, group_top, renorm, scale):
    """ids, coef (float64) of finite logits [M, E], in 64 bits; ties to the lower index."""
    l = logits.double().cpu()
    M, E = l.shape
    p = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, 1)
    c = p + (0 if bias is None else bias.double().cpu())
    if G > 1:
        best = c.view(M, G, E // G).sort(dim=2, descending=True).values[:, :, :group_top].sum(2)
        order = best.sort(dim=1, descending=True, stable=True).indices[:, topk_group:]
        for m in range(M):
            for g in order[m].tolist():
                c[m, g * (E // G) : (g + 1) * (E // G)] = -float("inf")
    ids = c.sort(dim=1, descending=True, stable=True).indices[:, :k]
    w = p.gather(1, ids)
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return ids.int(), w * scale


def product_bound(xa, wa, K, y, bf16):
    """How far an FP32 evaluation of a block-scaled product may be from the exact one. xa, wa: |x|, |w| in 64 bits; y: the exact result.
    Each of the 128 terms of a block enters a sum whose every step loses at most 2^-23 (truncation) of the running magnitude, the
    block's scale is one product (2^-24), and the ceil(K / 128) FMAs lose 2^-24 each, up to three more for a sum over K parts:
    (128 * 2 + 1 + blocks + 3) * 2^-24 of sum |x||w|. A BF16 result adds half a BF16 step, 2^-8."""
    tol = (260 + blocks(K)) * 2.0**-24 * (xa @ wa.t()) + 1e-30
    return tol + (y.abs() + tol) * 2.0**-8 if bf16 else tol


def check_fp8_rows(q, s, h, rel):
    """q, s against the exact rows h [R, K] that they stand for; `rel`: how far the FP32 evaluation of h itself may be off. The scale is
    the block's largest magnitude / 448 (one more rounding); a value is off by half a step of e4m3: 2^-4 of itself, or half of
    the subnormal step 2^-9 in units of the scale."""
    R, K = h.shape
    pad = torch.zeros((R, blocks(K) * 128), dtype=torch.float64, device=h.device)
    pad[:, :K] = h
    want = pad.view(R, -1, 128).abs().amax(2).clamp_min(2.0**-100) / 448
    assert ((s.double() - want).abs() <= want * (rel + 2.0**-23)).all()
    sw = s.double().repeat_interleave(128, 1)[:, :K]
    tol = torch.maximum(h.abs() * 2.0**-4, sw * 2.0**-10) * (1 + 2.0**-20) + h.abs() * 2 * rel + sw * 448 * 2.0**-23
    bad = (q.double() * sw - h).abs() > tol
    assert not bad.any(), "%d of %d values are further off than half a step" % (int(bad.sum()), bad.numel())

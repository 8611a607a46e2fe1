"""The FP8 (e4m3, a scale per block of 128) mixture-of-experts FFN path, operator by operator: what is timed and what the results are.

    route   scores of the experts, a balance bias, expert groups, top-k, renormalised weights
    norm    residual add, RMS norm, and the result in FP8 with a scale per (row, 128 columns)
    swiglu  silu(gate) * up of merged rows, the result in FP8 the same way
    linear  rows in FP8 times a weight matrix in FP8 with a scale per 128 x 128 block
    experts the same product for every routed slot with its expert's matrix: `gather` (token rows -> slot rows) and
            `combine` (slot rows -> weighted sum per token)
"""
import math

import torch

own = False

FP8 = torch.float8_e4m3fn
E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100  # a block of zeros still has a scale that divides
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases -------------------------------------------------------------------------------------------------------


def listed():
    return [
        # one decoded token of a layer with 512 experts in 8 groups
        dict(name="route_decode", op="route", M=1, E=512, k=10, score="sigmoid", bias=True, groups=8, topk_group=4, group_top=2, renorm=True, scale=2.5, act="f32"),
        # an expert-parallel prefill batch
        dict(name="route_prefill", op="route", M=16384, E=512, k=10, score="sigmoid", bias=True, groups=8, topk_group=4, group_top=2, renorm=True, scale=2.5, act="f32"),
        # softmax scores, groups by their best expert, weights as they are, an odd batch, 16-bit logits
        dict(name="route_softmax_odd", op="route", M=4097, E=160, k=6, score="softmax", bias=False, groups=8, topk_group=3, group_top=1, renorm=False, scale=16.0, act="bf16"),
        # the verify step of speculative decoding: one accepted token and five drafts
        dict(name="norm_verify", op="norm", M=6, d=2048, act="bf16", residual=True, h=True, centered=False),
        # a prefill batch
        dict(name="norm_prefill", op="norm", M=16384, d=2048, act="bf16", residual=True, h=True, centered=False),
        # the 2560-wide model, FP32 activations, the first norm of a stack (no residual yet), an odd batch, gains stored around zero
        dict(name="norm_f32_odd", op="norm", M=1001, d=2560, act="f32", residual=False, h=False, centered=True),
        # the slots of a verify step: 6 tokens, 10 experts each
        dict(name="swiglu_verify", op="swiglu", rows=60, I=512, act="bf16"),
        # the slots of a prefill chunk of 4096 tokens
        dict(name="swiglu_prefill", op="swiglu", rows=40960, I=512, act="bf16"),
        # gate and up of the shared expert of a 4096-wide layer at a verify step, unrounded results
        dict(name="linear_verify", op="linear", M=6, N=2048, K=4096, act="f32"),
        # a dense projection of a 4096-wide model over a prefill batch
        dict(name="linear_prefill", op="linear", M=16384, N=4096, K=4096, act="bf16"),
        # down projection and combine of a verify step: about 60 experts, a row each
        dict(name="combine_verify", op="experts", M=6, A=10, E=512, N=2048, K=512, act="f32", combine=True),
        # gate and up of a prefill chunk: skewed loads, about 80 rows an expert
        dict(name="gather_prefill", op="experts", M=4096, A=10, E=512, N=1024, K=2048, act="bf16", combine=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["route", "norm", "swiglu", "linear", "experts"])
    act = rng.choice(["f32", "bf16"])
    if op == "route":
        groups = rng.choice([1, 2, 4, 8, 16])
        per = _log(rng, 4, 1024 // groups)
        topk_group = rng.randint(1, groups)
        return dict(op=op, M=_log(rng, 1, 16384), E=groups * per, k=rng.randint(1, min(16, topk_group * per)), score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6,
                    groups=groups, topk_group=topk_group, group_top=rng.randint(1, 2), renorm=rng.random() < 0.5, scale=rng.choice([1.0, 2.5]), act=act)
    if op == "norm":
        return dict(op=op, M=_log(rng, 1, 16384), d=16 * _log(rng, 8, 512), act=act, residual=rng.random() < 0.7, h=rng.random() < 0.5, centered=rng.random() < 0.5)
    if op == "swiglu":
        return dict(op=op, rows=_log(rng, 1, 40960), I=16 * _log(rng, 4, 128), act=act)
    if op == "linear":
        return dict(op=op, M=_log(rng, 1, 8192), N=_log(rng, 64, 4096), K=16 * _log(rng, 8, 256), act=act)
    E, A = _log(rng, 4, 256), rng.randint(1, 4)
    return dict(op=op, M=_log(rng, 1, 4096), A=A, E=E, N=_log(rng, 64, 2048), K=16 * _log(rng, 8, 128), act=act, combine=rng.random() < 0.5)


def work(c):
    es = 4 if c.get("act") == "f32" else 2
    if c["op"] == "route":
        return {"bytes": c["M"] * c["E"] * es + (4 * c["E"] if c["bias"] else 0) + c["M"] * c["k"] * 8, "flops": c["M"] * c["E"] * 4}
    if c["op"] == "norm":
        n = c["M"] * c["d"]
        return {"bytes": n * es * (1 + (2 if c["residual"] else 0) + (1 if c["h"] else 0)) + n + 4 * c["M"] * _blocks(c["d"]) + 4 * c["d"], "flops": 6 * n}
    if c["op"] == "swiglu":
        n = c["rows"] * c["I"]
        return {"bytes": 2 * n * es + n + 4 * c["rows"] * _blocks(c["I"]), "flops": 8 * n}
    N, K = c["N"], c["K"]
    per_matrix, per_row = N * K + 4 * _blocks(N) * _blocks(K), K + 4 * _blocks(K)
    if c["op"] == "linear":
        return {"bytes": per_matrix + c["M"] * (per_row + N * es), "flops": 2 * c["M"] * N * K}
    S = c["M"] * c["A"]
    used = c["E"] * (1 - (1 - c["A"] / c["E"]) ** c["M"]) if c["M"] * c["A"] < 8 * c["E"] else c["E"]  # experts that some token takes
    rows_in, rows_out = (S, c["M"]) if c["combine"] else (c["M"], S)
    return {"bytes": used * per_matrix + rows_in * per_row + rows_out * N * es + S * (8 if c["combine"] else 4), "flops": 2 * S * N * K}


# ---- inputs ----------------------------------------------------------------------------------------------------------


def _blocks(n):
    return -(-n // 128)


def _rows_fp8(x):
    """FP32 rows [R, K] as e4m3 with a scale per (row, 128 columns)."""
    R, K = x.shape
    pad = torch.nn.functional.pad(x, (0, _blocks(K) * 128 - K)).view(R, _blocks(K), 128)
    s = pad.abs().amax(2).clamp_min(AMAX_FLOOR) / E4M3_MAX
    q = (pad / s[:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).reshape(R, -1)[:, :K].contiguous().to(FP8)
    return q, s


def _matrix_fp8(g, N, K, n=1):
    """n matrices N(0, 0.02) [N, K] stacked [n * N, K] as e4m3, with a scale per 128 x 128 block [n * blocks(N), blocks(K)]."""
    NB, KB = _blocks(N), _blocks(K)
    q = torch.empty((n * N, K), dtype=FP8, device="cuda")
    s = torch.empty((n * NB, KB), dtype=torch.float32, device="cuda")
    step = max(1, (1 << 27) // (N * K))
    for i in range(0, n, step):
        m = min(step, n - i)
        w = torch.zeros((m, NB * 128, KB * 128), device="cuda")
        w[:, :N, :K] = torch.randn((m, N, K), generator=g, device="cuda") * 0.02
        b = w.view(m, NB, 128, KB, 128)
        t = b.abs().amax((2, 4)).clamp_min(AMAX_FLOOR) / E4M3_MAX
        b = (b / t[:, :, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX).view(m, NB * 128, KB * 128)[:, :N, :K]
        q[i * N:(i + m) * N] = b.reshape(m * N, K).to(FP8)
        s[i * NB:(i + m) * NB] = t.view(m * NB, KB)
    return q, s


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    empty = lambda shape, dtype: torch.empty(shape, dtype=dtype, device="cuda")  # noqa: E731
    dt = DTYPES[c["act"]]
    s = dict(c)
    if c["op"] == "route":
        s["logits"] = (rand(c["M"], c["E"]) * 1.5 - 1.0).to(dt)
        s["bias"] = rand(c["E"]) * 0.02 if c["bias"] else None
        s["ids"], s["coef"] = empty((c["M"], c["k"]), torch.int32), empty((c["M"], c["k"]), torch.float32)
        s["err"] = torch.zeros(4, dtype=torch.int32, device="cuda")
    elif c["op"] == "norm":
        M, d = c["M"], c["d"]
        s["x"] = (rand(M, d) * 2.0).to(dt)
        s["y"] = rand(M, d).to(dt) if c["residual"] else None
        s["w"] = rand(d) * 0.1 + (0.0 if c["centered"] else 1.0)
        s["x_out"] = empty((M, d), dt) if c["residual"] else None
        s["h_out"] = empty((M, d), dt) if c["h"] else None
        s["q"], s["s"] = empty((M, d), FP8), empty((M, _blocks(d)), torch.float32)
    elif c["op"] == "swiglu":
        s["gu"] = rand(c["rows"], 2 * c["I"]).to(dt)
        s["q"], s["s"] = empty((c["rows"], c["I"]), FP8), empty((c["rows"], _blocks(c["I"])), torch.float32)
    elif c["op"] == "linear":
        s["xq"], s["xs"] = _rows_fp8(rand(c["M"], c["K"]))
        s["wq"], s["ws"] = _matrix_fp8(g, c["N"], c["K"])
        s["out"] = empty((c["M"], c["N"]), dt)
    else:
        M, A, E, N, K = c["M"], c["A"], c["E"], c["N"], c["K"]
        # the routes of a skewed router: a popularity per expert and noise per token
        s["ids"] = (rand(E) * 0.5 + rand(M, E)).topk(A, dim=1).indices.to(torch.int32)
        s["wq"], s["ws"] = _matrix_fp8(g, N, K, E)
        s["xq"], s["xs"] = _rows_fp8(rand(M * A if c["combine"] else M, K))
        s["coef"] = torch.softmax(rand(M, A), 1) if c["combine"] else None
        s["out"] = empty((M, N) if c["combine"] else (M * A, N), dt)
        s["partial"] = empty((M * A, N), torch.float32) if c["combine"] else None
        s["err"] = torch.zeros(4, dtype=torch.int32, device="cuda")
        s["most"] = int(torch.bincount(s["ids"].view(-1), minlength=E).max())  # the longest list of an expert
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from strixite_b200 import kernels as K

    op = s["op"]
    if op == "route":
        K.moe_router_scored(s["logits"], s["E"], s["M"], s["E"], s["k"], s["score"], s["bias"], s["groups"], s["topk_group"], s["group_top"], s["renorm"], s["scale"],
                            None, 0, 0, s["ids"], s["coef"], K.act_of(s["logits"]), s["err"])
        return {"ids": s["ids"], "coef": s["coef"]}
    if op == "norm":
        K.residual_rmsnorm_fp8(s["x"], s["y"], s["w"], s["M"], s["d"], 1e-6, s["x_out"], s["h_out"], s["q"], s["s"], K.act_of(s["x"]), centered=s["centered"])
        return {"x": s["x_out"], "h": s["h_out"], "q": s["q"], "scale": s["s"]}
    if op == "swiglu":
        K.swiglu_fp8(s["gu"], s["q"], s["s"], s["rows"], s["I"], K.act_of(s["gu"]))
        return {"q": s["q"], "scale": s["s"]}
    act = K.act_of(s["out"])
    if op == "linear":
        if "w" not in s:
            s["w"] = K.Fp8Weight(s["wq"], s["ws"])
        K.linear_fp8(s["xq"], s["xs"], s["w"], s["out"], s["M"], act)
        return {"y": s["out"]}
    if "w" not in s:  # the views and the grouping workspace that a program keeps
        s["w"] = K.Fp8Weight(s["wq"], s["ws"], experts=s["E"])
        s["group_bytes"] = K.moe_route_workspace_bytes(s["M"], s["A"], s["E"])
        s["group"] = torch.empty(s["group_bytes"], dtype=torch.uint8, device="cuda")
    K.moe_group_routes(s["ids"], s["M"], s["A"], s["E"], s["group"], s["group_bytes"], s["err"])
    if s["combine"]:
        K.linear_fp8_experts_combine_grouped(s["xq"], s["xs"], s["w"], s["E"], s["ids"], s["coef"], s["group"], s["group_bytes"], s["partial"], s["M"], s["A"], s["out"], act)
    else:
        K.linear_fp8_experts_gather_grouped(s["xq"], s["xs"], s["w"], s["E"], s["group"], s["group_bytes"], s["M"], s["A"], s["out"], act)
    return {"y": s["out"]}


def _quant(h):
    q, scale = _rows_fp8(h)
    return {"q": q, "scale": scale}


def _wide(q, s, rows_per_scale):
    """e4m3 [R, K] with scales [ceil(R / rows_per_scale), blocks(K)] as FP32 values."""
    R, K = q.shape
    return q.float() * s.repeat_interleave(rows_per_scale, 0)[:R].repeat_interleave(128, 1)[:, :K]


def _run_plain(s):
    op, dt = s["op"], DTYPES[s["act"]]
    if op == "route":
        # in 64 bits: two experts whose scores agree to 32 bits still have an order
        M, E, G = s["M"], s["E"], s["groups"]
        l = s["logits"].double()
        if s["score"] == "sigmoid":
            p = 1.0 / (1.0 + torch.exp(-l))
        else:
            p = torch.exp(l - l.amax(1, keepdim=True))
            p = p / p.sum(1, keepdim=True)
        c = p if s["bias"] is None else p + s["bias"].double()
        if G > 1:
            best = c.view(M, G, E // G).sort(dim=2, descending=True).values[:, :, : s["group_top"]].sum(2)
            order = best.sort(dim=1, descending=True, stable=True).indices[:, : s["topk_group"]]
            open_ = torch.zeros((M, G), dtype=torch.bool, device=c.device).scatter_(1, order, True)
            c = torch.where(open_[:, :, None], c.view(M, G, E // G), -math.inf).reshape(M, E)
        ids = c.sort(dim=1, descending=True, stable=True).indices[:, : s["k"]]
        w = p.gather(1, ids)
        if s["renorm"]:
            w = w / w.sum(1, keepdim=True)
        return {"ids": ids.to(torch.int32), "coef": (w * s["scale"]).float()}
    if op == "norm":
        x = s["x"] if s["y"] is None else (s["x"].float() + s["y"].float()).to(dt)
        f = x.float()
        gain = 1.0 + s["w"] if s["centered"] else s["w"]
        h = f / torch.sqrt(f.square().mean(1, keepdim=True) + 1e-6) * gain
        return {"x": None if s["y"] is None else x, "h": h.to(dt) if s["h"] else None, **_quant(h)}
    if op == "swiglu":
        gate, up = s["gu"].float().view(s["rows"], 2, s["I"]).unbind(1)
        return _quant(gate / (1.0 + torch.exp(-gate)) * up)
    N, K = s["N"], s["K"]
    x = _wide(s["xq"], s["xs"], 1)
    if op == "linear":
        return {"y": (x @ _wide(s["wq"], s["ws"], 128).t()).to(dt)}
    M, A, E = s["M"], s["A"], s["E"]
    S, NB, KB = M * A, _blocks(N), _blocks(K)
    e = s["ids"].view(-1).long()
    rows = x if s["combine"] else x.repeat_interleave(A, 0)  # a row for every slot
    if S <= 128:  # few slots: each with its expert's matrix
        wq = s["wq"].view(torch.uint8).view(E, N, K)[e].view(FP8).float()
        w = wq * s["ws"].view(E, NB, KB)[e].repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K]
        y = torch.bmm(w, rows[:, :, None])[:, :, 0]
    else:  # every expert with its rows, filled up with zeros to the longest list
        w = s["wq"].view(E, N, K).float()
        w.view(E, N, K).mul_(s["ws"].view(E, NB, KB).repeat_interleave(128, 1)[:, :N].repeat_interleave(128, 2)[:, :, :K])
        by = e.sort(stable=True).indices
        first = torch.searchsorted(e[by], torch.arange(E, device=e.device))
        place = torch.empty_like(by)
        place[by] = torch.arange(S, device=e.device)
        place = place - first[e]
        wide = torch.zeros((E, s["most"], K), device=e.device)
        wide[e, place] = rows
        y = torch.bmm(wide, w.transpose(1, 2))[e, place]
    if s["combine"]:
        y = (y.view(M, A, N) * s["coef"][:, :, None]).sum(1)
    return {"y": y.to(dt)}


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------


def _exact_quant(h):
    R, K = h.shape
    q, scale = torch.empty((R, K), dtype=torch.float64, device=h.device), torch.empty((R, _blocks(K)), dtype=torch.float64, device=h.device)
    for b in range(_blocks(K)):
        part = h[:, b * 128:(b + 1) * 128]
        scale[:, b] = part.abs().max(1).values.clamp_min(AMAX_FLOOR) / 448
        q[:, b * 128:(b + 1) * 128] = (part / scale[:, b:b + 1]).clamp(-448, 448).to(FP8).double()
    return q, scale


def _exact_matrix(q, s, N, K):
    w = q.double()
    for i in range(_blocks(N)):
        for j in range(_blocks(K)):
            w[i * 128:(i + 1) * 128, j * 128:(j + 1) * 128] *= s[i, j].double()
    return w


def exact(c, seed):
    s = prepare(c, seed)
    op = c["op"]
    if op == "route":
        import numpy as np

        l = s["logits"].double().cpu().numpy()
        if c["score"] == "sigmoid":
            p = 1.0 / (1.0 + np.exp(-l))
        else:
            p = np.exp(l - l.max(1)[:, None])
            p /= p.sum(1)[:, None]
        choice = p + (0.0 if s["bias"] is None else s["bias"].double().cpu().numpy()[None, :])
        M, E, G = c["M"], c["E"], c["groups"]
        if G > 1:
            g = np.sort(choice.reshape(M, G, E // G), axis=2)[:, :, ::-1][:, :, : c["group_top"]].sum(2)
            shut = np.argsort(-g, axis=1, kind="stable")[:, c["topk_group"]:]
            closed = np.zeros((M, G), bool)
            np.put_along_axis(closed, shut, True, 1)
            choice = np.where(np.repeat(closed, E // G, axis=1), -np.inf, choice)
        ids = np.argsort(-choice, axis=1, kind="stable")[:, : c["k"]]
        w = np.take_along_axis(p, ids, 1)
        if c["renorm"]:
            w = w / w.sum(1)[:, None]
        return {"ids": ids.astype(np.int32), "coef": w * c["scale"]}
    if op == "norm":
        x = s["x"].double()
        if s["y"] is not None:
            x = (x + s["y"].double()).to(DTYPES[c["act"]]).double()
        h = x * (x.pow(2).sum(1, keepdim=True) / c["d"] + 1e-6).rsqrt() * (s["w"].double() + (1.0 if c["centered"] else 0.0))
        q, scale = _exact_quant(h)
        return {"x": x if c["residual"] else None, "h": h if c["h"] else None, "q": q, "scale": scale}
    if op == "swiglu":
        gu = s["gu"].double()
        gate = gu[:, : c["I"]]
        q, scale = _exact_quant(gate * torch.sigmoid(gate) * gu[:, c["I"]:])
        return {"q": q, "scale": scale}
    N, K = c["N"], c["K"]
    x = s["xq"].double()
    for j in range(_blocks(K)):
        x[:, j * 128:(j + 1) * 128] *= s["xs"][:, j:j + 1].double()
    if op == "linear":
        return {"y": torch.matmul(x, _exact_matrix(s["wq"], s["ws"], N, K).t())}
    ids, A, NB = s["ids"].long(), c["A"], _blocks(N)
    y = torch.zeros((c["M"] * A, N), dtype=torch.float64, device=x.device)
    for e in ids.unique().tolist():
        token, a = (ids == e).nonzero(as_tuple=True)
        slot = token * A + a
        w = _exact_matrix(s["wq"][e * N:(e + 1) * N], s["ws"][e * NB:(e + 1) * NB], N, K)
        y[slot] = torch.matmul(x[slot if c["combine"] else token], w.t())
    if c["combine"]:
        y = torch.einsum("man,ma->mn", y.view(c["M"], A, N), s["coef"].double())
    return {"y": y}

"""Measured cases of the matrix-model operators: orthogonalised updates of a
multi-target model, its 4-bit form, and prediction from that form.

Shapes are the library's: a model (and its gradient) is ``(ntasks, ntargets,
nfeatures)``, observations are ``(nobs, ntasks, nfeatures)``, predictions
``(nobs, ntasks, ntargets)``.

* ``orthogonalize``    five Newton-Schulz steps on every task's matrix G:
                       X = G/|G|_F, then X <- aX + (bA + cA^2)X with A = X X^T
* ``orthogonal_step``  momentum, its orthogonalised direction, the model update
* ``quantize_q4``      4-bit codes with one scale per target and group of features,
                       returned as the values they stand for
* ``predict_q4``       Yhat = X M^T from the codes and scales
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
LR, MU, WEIGHT_DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # 64 small models side by side, one gradient each: latency of the whole chain
        {"name": "ortho-64x16x256-f32", "op": "orthogonalize", "type": "f32", "ntasks": 64, "nt": 16, "nf": 256},
        # the wide dense model's gradient: few rows, long ones
        {"name": "ortho-256x4096-f32", "op": "orthogonalize", "type": "f32", "ntasks": 1, "nt": 256, "nf": 4096},
        # taller than wide, odd sizes, a few tasks
        {"name": "ortho-3x1021x333-f16", "op": "orthogonalize", "type": "f16", "ntasks": 3, "nt": 1021, "nf": 333},
        # a square projection of a large layer
        {"name": "ortho-4096x4096-bf16", "op": "orthogonalize", "type": "bf16", "ntasks": 1, "nt": 4096, "nf": 4096},
        # a training step of a mid-sized layer with ragged sizes
        {"name": "step-1000x777-bf16", "op": "orthogonal_step", "type": "bf16", "ntasks": 1, "nt": 1000, "nf": 777,
         "nesterov": True},
        # a training step of a large wide layer kept in float
        {"name": "step-2048x8192-f32", "op": "orthogonal_step", "type": "f32", "ntasks": 1, "nt": 2048, "nf": 8192,
         "nesterov": False},
        # 64 small models laid out for serving
        {"name": "quantize-64x16x256-f32", "op": "quantize_q4", "type": "f32", "ntasks": 64, "nt": 16, "nf": 256,
         "group": 64},
        # a large output layer laid out for serving
        {"name": "quantize-16384x4096-bf16", "op": "quantize_q4", "type": "bf16", "ntasks": 1, "nt": 16384,
         "nf": 4096, "group": 128},
        # one observation against 64 small models: latency
        {"name": "predict-1-64x16x256-f32", "op": "predict_q4", "type": "f32", "ntasks": 64, "nt": 16, "nf": 256,
         "nobs": 1, "group": 64},
        # one token against a large layer: the stream of the weights
        {"name": "predict-1-16384x4096-bf16", "op": "predict_q4", "type": "bf16", "ntasks": 1, "nt": 16384,
         "nf": 4096, "nobs": 1, "group": 128},
        # a few sequences' tokens together, odd sizes
        {"name": "predict-7-5003x2901-f16", "op": "predict_q4", "type": "f16", "ntasks": 1, "nt": 5003, "nf": 2901,
         "nobs": 7, "group": 128},
        # a prompt through a large layer
        {"name": "predict-2048-16384x4096-bf16", "op": "predict_q4", "type": "bf16", "ntasks": 1, "nt": 16384,
         "nf": 4096, "nobs": 2048, "group": 128},
    ]


def _log_int(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["orthogonalize", "orthogonalize", "orthogonal_step", "quantize_q4", "predict_q4", "predict_q4",
                     "predict_q4"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op in ("orthogonalize", "orthogonal_step"):
        while True:
            nt, nf, ntasks = _log_int(rng, 1, 8192), _log_int(rng, 8, 8192), _log_int(rng, 1, 64)
            m, n = min(nt, nf), max(nt, nf)
            if ntasks * m * n <= 4096 * 4096 and ntasks * m * m * n <= 4096 ** 3:
                break
        case = {"op": op, "type": kind, "ntasks": ntasks, "nt": nt, "nf": nf}
        if op == "orthogonal_step":
            case["nesterov"] = rng.random() < 0.5
        return case
    while True:
        nt, nf, ntasks = _log_int(rng, 1, 16384), _log_int(rng, 16, 8192), _log_int(rng, 1, 64)
        if ntasks * nt * nf <= 16384 * 4096:
            break
    case = {"op": op, "type": kind, "ntasks": ntasks, "nt": nt, "nf": nf, "group": rng.choice([64, 128])}
    if op == "predict_q4":
        top = min(4096, (2048 * 16384 * 4096) // (ntasks * nt * nf), (1 << 26) // (ntasks * max(nt, nf)))
        case["nobs"] = _log_int(rng, 1, max(1, top))
    return case


# ---- inputs -----------------------------------------------------------------

def _tensors(case, seed):
    """The case's inputs, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["type"]]
    ntasks, nt, nf = case["ntasks"], case["nt"], case["nf"]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    def gradient_like():
        # residuals times features: a few strong directions, features of unlike scale, and noise over all
        r = max(1, min(nt, nf, 32))
        decay = torch.exp(-torch.arange(r, device="cuda") / 6.0)
        strong = (randn(ntasks, nt, r) * decay) @ randn(ntasks, r, nf)
        feature = torch.exp(0.5 * randn(ntasks, 1, nf))
        return ((strong + 0.3 * randn(ntasks, nt, nf)) * feature * 0.05).to(dtype)

    if case["op"] == "orthogonalize":
        return {"G": gradient_like()}
    if case["op"] == "orthogonal_step":
        return {"M": (randn(ntasks, nt, nf) / math.sqrt(nf)).to(dtype), "grad": gradient_like(),
                "momentum": 4.0 * gradient_like().float() + 0.05 * randn(ntasks, nt, nf)}
    # weights whose rows differ in scale, with a few outlying features
    M = randn(ntasks, nt, nf) * torch.exp(0.3 * randn(ntasks, nt, 1)) / math.sqrt(nf)
    M = (M * torch.where(torch.rand(ntasks, 1, nf, device="cuda", generator=g) < 0.01, 8.0, 1.0)).to(dtype)
    if case["op"] == "quantize_q4":
        return {"M": M}
    return {"M": M, "X": randn(case["nobs"], ntasks, nf).to(dtype)}


def prepare(case, seed):
    state = _tensors(case, seed)
    state["case"] = case
    ntasks, nt, nf = case["ntasks"], case["nt"], case["nf"]
    if own:
        from gpu_algos_b200 import glm

        dtype = DTYPES[case["type"]]
        need = 0
        if case["op"] in ("orthogonalize", "orthogonal_step"):
            need = glm.orthogonal_workspace_bytes(dtype, nf, nt, ntasks)
        elif case["op"] == "predict_q4":
            state["model"] = glm.quantize_q4(state.pop("M"), case["group"])
            need = glm.predict_q4_workspace_bytes(dtype, nf, nt, ntasks, case["nobs"], case["group"])
        state["workspace"] = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
    elif case["op"] == "predict_q4":
        codes, scales = _plain_quantize(state.pop("M"), case["group"])
        codes = torch.nn.functional.pad(codes + 8, (0, codes.shape[2] % 2)).to(torch.uint8)
        state["codes"] = codes[..., 0::2] | (codes[..., 1::2] << 4)  # two to a byte, the first in the low half
        state["scales"] = scales
    return state


# ---- the plain forms --------------------------------------------------------

def _plain_orthogonalize(G):
    """float32 iterates of a float32 matrix, the norm in float64."""
    X = G
    tall = X.shape[1] > X.shape[2]
    if tall:
        X = X.transpose(1, 2)
    norm = X.double().square().sum((1, 2), keepdim=True).sqrt()
    X = torch.where(norm == 0, torch.zeros_like(X), (X.double() / norm).float())
    a, b, c = COEFFICIENTS
    for _ in range(STEPS):
        A = X @ X.transpose(1, 2)
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.transpose(1, 2) if tall else X


def _update_scale(nt, nf):
    return math.sqrt(max(1.0, nt / nf))


def _plain_step(M, grad, momentum, nesterov):
    g = grad.float()
    momentum.mul_(MU).add_(g)
    direction = _plain_orthogonalize(g + MU * momentum if nesterov else momentum)
    lr = LR * _update_scale(M.shape[1], M.shape[2])
    M.copy_(M.float() * (1.0 - LR * WEIGHT_DECAY) - lr * direction)
    return M, momentum


def _plain_quantize(M, group):
    """Codes in -7..7 and scales (of M's type), one per target and group of features."""
    ntasks, nt, nf = M.shape
    ngroups = -(-nf // group)
    W = torch.nn.functional.pad(M, (0, ngroups * group - nf)).reshape(ntasks, nt, ngroups, group)
    scales = (W.float().abs().amax(3) / 7.0).to(M.dtype)
    s = scales.double()[..., None]
    codes = torch.where(s == 0, 0.0, torch.round(W.double() / s)).clamp_(-7, 7).to(torch.int8)
    return codes.reshape(ntasks, nt, -1)[..., :nf], scales


def _plain_values(codes, scales, group):
    wide = scales.float().repeat_interleave(group, 2)[..., :codes.shape[2]]
    return codes.float() * wide


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        from gpu_algos_b200 import glm

        if op == "orthogonalize":
            return glm.orthogonalize(state["G"], workspace=state["workspace"])
        if op == "orthogonal_step":
            M = glm.orthogonal_step(state["M"], state["grad"], state["momentum"], LR, mu=MU,
                                    nesterov=case["nesterov"], weight_decay=WEIGHT_DECAY,
                                    workspace=state["workspace"])
            return M, state["momentum"]
        if op == "quantize_q4":
            return glm.dequantize_q4(glm.quantize_q4(state["M"], case["group"]))
        return glm.predict_q4(state["X"], state["model"], workspace=state["workspace"])
    if op == "orthogonalize":
        return _plain_orthogonalize(state["G"].float()).to(state["G"].dtype).contiguous()
    if op == "orthogonal_step":
        return _plain_step(state["M"], state["grad"], state["momentum"], case["nesterov"])
    if op == "quantize_q4":
        codes, scales = _plain_quantize(state["M"], case["group"])
        return _plain_values(codes, scales, case["group"]).to(scales.dtype)
    packed = state["codes"]
    codes = torch.stack((packed & 15, packed >> 4), dim=3).flatten(2)[..., :case["nf"]].float() - 8.0
    W = _plain_values(codes, state["scales"], case["group"])
    X = state["X"]
    return (X.float().transpose(0, 1) @ W.transpose(1, 2)).transpose(0, 1).to(X.dtype).contiguous()


# ---- what a pass cannot do without -------------------------------------------

def work(case):
    ntasks, nt, nf, width = case["ntasks"], case["nt"], case["nf"], BYTES[case["type"]]
    size = ntasks * nt * nf
    if case["op"] in ("orthogonalize", "orthogonal_step"):
        m, n = min(nt, nf), max(nt, nf)
        # symmetric products count half; either as the steps are written, or on the m x m side alone with one
        # product into X at the end
        direct = STEPS * (m * m * n + m ** 3 + 2 * m * m * n)
        inner = m * m * n + 2 * m * m * n + STEPS * 4 * m ** 3
        step = case["op"] == "orthogonal_step"
        return {"bytes": size * (3 * width + 8) if step else 2 * size * width, "flops": ntasks * min(direct, inner)}
    held = size / 2 + ntasks * nt * -(-nf // case["group"]) * width
    if case["op"] == "quantize_q4":
        return {"bytes": 2 * size * width + 2 * held, "flops": 3 * size}
    nobs = case["nobs"]
    return {"bytes": held + nobs * ntasks * (nt + nf) * width, "flops": 2 * nobs * size}


# ---- the definitions in 64 bits ----------------------------------------------

def _exact_direction(U):
    out = []
    for T in U.double():
        norm = torch.linalg.vector_norm(T)
        Z = T / norm if float(norm) > 0 else torch.zeros_like(T)
        flip = Z.shape[0] > Z.shape[1]
        Z = Z.T if flip else Z
        for _ in range(STEPS):
            gram = Z @ Z.T
            first = gram @ Z
            Z = COEFFICIENTS[0] * Z + COEFFICIENTS[1] * first + COEFFICIENTS[2] * (gram @ first)
        out.append(Z.T if flip else Z)
    return torch.stack(out)


def _exact_values(M, group):
    out = torch.zeros(M.shape, dtype=torch.float64, device=M.device)
    for lo in range(0, M.shape[2], group):
        W = M[:, :, lo:lo + group].double()
        s = (W.abs().amax(2, keepdim=True) / 7).to(M.dtype).double()
        q = torch.where(s > 0, (W / torch.where(s > 0, s, 1.0)).round(), torch.zeros_like(W))
        out[:, :, lo:lo + group] = q.clamp(-7, 7) * s
    return out


def exact(case, seed):
    t = _tensors(case, seed)
    if case["op"] == "orthogonalize":
        return _exact_direction(t["G"])
    if case["op"] == "orthogonal_step":
        g = t["grad"].double()
        momentum = MU * t["momentum"].double() + g
        U = g + MU * momentum if case["nesterov"] else momentum
        step = LR * _update_scale(case["nt"], case["nf"]) * _exact_direction(U)
        return t["M"].double() * (1 - LR * WEIGHT_DECAY) - step, momentum
    if case["op"] == "quantize_q4":
        return _exact_values(t["M"], case["group"])
    W = _exact_values(t["M"], case["group"])
    return torch.einsum("otf,tgf->otg", t["X"].double(), W)

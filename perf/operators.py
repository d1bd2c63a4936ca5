"""The operators of the backbone's feed-forward half with their gradients, as cases to be measured.

``run`` computes them in plain torch operations in 32 bits (``own`` false) or through ``iffnerf_amd.hip_block`` (``own`` true):

  norm     layer norm over the last axis                    y = (x - mean) / sqrt(var + eps) * w + b
  mlp      gated feed-forward block                         y = (act(x Wg^T + bg) * (x Wu^T + bu)) W3^T + b3,  [Wg; Wu] = w12
  dropout  dropout from a counter-based generator           y = residual + keep * x / (1 - p); the mask is never stored

"train" cases return the gradients of everything that is trained next to the output.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
DEV = "cuda:0"


def listed():
    return [
        # the class token of one query image through a norm at serving time: latency alone
        {"name": "norm_one_row", "op": "norm", "images": 1, "tokens": 1, "skip": 0, "dim": 384, "dtype": "bf16", "affine": True, "train": False},
        # one training step of a backbone norm: 32 images of 16 x 16 patches + class token, 384 wide, in the reference's fp32
        {"name": "norm_train_32x257x384", "op": "norm", "images": 32, "tokens": 257, "skip": 0, "dim": 384, "dtype": "fp32", "affine": True, "train": True},
        # the patch tokens behind the class token (a strided view) at an odd width, half precision
        {"name": "norm_train_patches_odd", "op": "norm", "images": 19, "tokens": 197, "skip": 1, "dim": 1001, "dtype": "fp16", "affine": True, "train": True},
        # a large training batch of a wide backbone
        {"name": "norm_train_256x257x1024", "op": "norm", "images": 256, "tokens": 257, "skip": 0, "dim": 1024, "dtype": "bf16", "affine": True, "train": True},
        # a single token through the block at serving time: the weights are read once
        {"name": "mlp_one_token", "op": "mlp", "rows": 1, "dim": 1536, "hidden": 4096, "out": 1536, "act": "silu", "bias": True, "dtype": "bf16", "train": False},
        # one query image at serving time, in the reference's fp32
        {"name": "mlp_257_fp32", "op": "mlp", "rows": 257, "dim": 384, "hidden": 1024, "out": 384, "act": "silu", "bias": True, "dtype": "fp32", "train": False},
        # one training step, 32 images, 384 wide, in mixed precision's type
        {"name": "mlp_train_8224_bf16", "op": "mlp", "rows": 8224, "dim": 384, "hidden": 1024, "out": 384, "act": "silu", "bias": True, "dtype": "bf16", "train": True},
        # sizes no tile divides, no biases, the other activation
        {"name": "mlp_train_odd", "op": "mlp", "rows": 1003, "dim": 387, "hidden": 1029, "out": 395, "act": "gelu", "bias": False, "dtype": "fp16", "train": True},
        # one training step of a wide backbone, 64 images: the matrix products alone
        {"name": "mlp_train_16448_bf16", "op": "mlp", "rows": 16448, "dim": 1536, "hidden": 4096, "out": 1536, "act": "silu", "bias": True, "dtype": "bf16", "train": True},
        # one image's tokens behind the block, with the residual stream added
        {"name": "dropout_257x384", "op": "dropout", "rows": 257, "dim": 384, "p": 0.1, "residual": True, "dtype": "bf16", "train": True},
        # an odd number of values, no residual
        {"name": "dropout_odd", "op": "dropout", "rows": 4099, "dim": 1001, "p": 0.5, "residual": False, "dtype": "fp16", "train": True},
        # a wide backbone's residual stream in fp32, 64 images
        {"name": "dropout_16448x1536", "op": "dropout", "rows": 16448, "dim": 1536, "p": 0.1, "residual": True, "dtype": "fp32", "train": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "mlp", "mlp", "dropout"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    width = 4 if dtype == "fp32" else 2
    odd = rng.random() < 0.4                                     # sizes of no alignment
    if op == "norm":
        tokens, dim = rng.randint(2, 289), _log(rng, 64, 2048)
        dim = dim | 1 if odd else -(-dim // 8) * 8
        most = 256 * 257 * 1024 * 2 // (tokens * dim * width)
        return {"op": op, "images": _log(rng, 1, max(1, most)), "tokens": tokens, "skip": rng.randint(0, 1), "dim": dim, "dtype": dtype,
                "affine": rng.random() < 0.8, "train": rng.random() < 0.7}
    if op == "mlp":
        dim, hidden = _log(rng, 64, 1536), _log(rng, 128, 4096)
        out = dim if rng.random() < 0.7 else _log(rng, 64, 1536)
        if odd:
            dim, hidden, out = dim | 1, hidden | 1, out | 1
        else:
            dim, hidden, out = -(-dim // 8) * 8, -(-hidden // 8) * 8, -(-out // 8) * 8
        # an fp32 pass is at most a sixth of the largest listed case's work
        rows = _log(rng, 1, 16448 if dtype != "fp32" else 4112)
        return {"op": op, "rows": rows, "dim": dim, "hidden": hidden, "out": out, "act": rng.choice(("silu", "gelu")),
                "bias": rng.random() < 0.7, "dtype": dtype, "train": rng.random() < 0.6}
    dim = _log(rng, 64, 2048)
    dim = dim | 1 if odd else -(-dim // 8) * 8
    return {"op": op, "rows": _log(rng, 16, 16448 * 1536 * 4 // (dim * width)), "dim": dim, "p": rng.choice((0.05, 0.1, 0.25, 0.5)),
            "residual": rng.random() < 0.6, "dtype": dtype, "train": rng.random() < 0.7}


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale + shift).to(dt)

    s = {"case": case}
    if case["op"] == "norm":
        # a residual stream: unit noise, a level per channel, a few channels far out
        level = torch.randn(case["dim"], generator=gen, device=DEV) * 0.5
        level[:: max(1, case["dim"] // 3)] *= 12.0
        stream = (torch.randn(case["images"], case["tokens"], case["dim"], generator=gen, device=DEV) + level).to(dt)
        s["x"] = stream[:, case["skip"]:].detach()
        s["dy"] = normal(*s["x"].shape, scale=1e-2)
        s["eps"] = 1e-6
        s["w"] = normal(case["dim"], scale=0.2, shift=1.0) if case["affine"] else None
        s["b"] = normal(case["dim"], scale=0.2) if case["affine"] else None
        leaves = ("x", "w", "b")
    elif case["op"] == "mlp":
        M, D, H, O = case["rows"], case["dim"], case["hidden"], case["out"]
        s["x"] = normal(M, D)
        s["w12"], s["w3"] = normal(2 * H, D, scale=D ** -0.5), normal(O, H, scale=H ** -0.5)
        s["b12"] = normal(2 * H, scale=0.1) if case["bias"] else None
        s["b3"] = normal(O, scale=0.1) if case["bias"] else None
        s["dy"] = normal(M, O, scale=1e-2)
        leaves = ("x", "w12", "b12", "w3", "b3")
    else:
        s["x"] = normal(case["rows"], case["dim"])
        s["residual"] = normal(case["rows"], case["dim"]) if case["residual"] else None
        s["dy"] = normal(case["rows"], case["dim"], scale=1e-2)
        s["seed"], s["offset"] = int(torch.randint(0, 2 ** 62, (1,), generator=gen, device=DEV)), seed * 7 + 3
        leaves = ("x", "residual")
    s["leaves"] = [n for n in leaves if s[n] is not None] if case["train"] else []
    for n in s["leaves"]:
        s[n].requires_grad_(True)
    return s


def run(state):
    with torch.set_grad_enabled(state["case"]["train"]):
        if own:
            from iffnerf_amd import hip_block
            c, s = state["case"], state
            if c["op"] == "norm":
                y = hip_block.layer_norm(s["x"], s["w"], s["b"], s["eps"])
            elif c["op"] == "mlp":
                y = hip_block.gated_mlp(s["x"], s["w12"], s["b12"], s["w3"], s["b3"], activation=c["act"])
            else:
                y = hip_block.dropout(s["x"], c["p"], s["seed"], s["offset"], residual=s["residual"])
            if not c["train"]:
                return {"y": y}
            grads = torch.autograd.grad(y, [s[n] for n in s["leaves"]], s["dy"])
            return {"y": y.detach(), **{"d" + n: g for n, g in zip(s["leaves"], grads)}}
        return _plain(state)


def _plain(s):
    c, dt = s["case"], DTYPES[s["case"]["dtype"]]
    f = {n: (s[n].detach().float() if s.get(n) is not None else None) for n in ("x", "w", "b", "w12", "b12", "w3", "b3", "residual", "dy")}
    for n in s["leaves"]:
        f[n] = f[n].detach().requires_grad_(True)
    if c["op"] == "norm":
        mean = f["x"].mean(-1, keepdim=True)
        d = f["x"] - mean
        y = d / torch.sqrt((d * d).mean(-1, keepdim=True) + s["eps"])
        if f["w"] is not None:
            y = y * f["w"] + f["b"]
    elif c["op"] == "mlp":
        gu = f["x"] @ f["w12"].t()
        if f["b12"] is not None:
            gu = gu + f["b12"]
        g, u = gu[:, :c["hidden"]], gu[:, c["hidden"]:]
        a = g * torch.sigmoid(g) if c["act"] == "silu" else 0.5 * g * (1.0 + torch.erf(g * (0.5 ** 0.5)))
        y = (a * u) @ f["w3"].t()
        if f["b3"] is not None:
            y = y + f["b3"]
    else:
        threshold = _threshold(c["p"])
        y = f["x"] * _keep(f["x"].numel(), s["seed"], s["offset"], threshold).reshape(f["x"].shape) * (65536.0 / (65536 - threshold))
        if f["residual"] is not None:
            y = y + f["residual"]
    if not s["leaves"]:
        return {"y": y.to(dt)}
    grads = torch.autograd.grad(y, [f[n] for n in s["leaves"]], f["dy"])
    return {"y": y.detach().to(dt), **{"d" + n: g.to(dt) for n, g in zip(s["leaves"], grads)}}


# ---------------------------------------------------------------------------------------- the generator
# Philox 4x32 with 10 rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011).  Value i of a tensor
# (in the order of its indices) takes 16 bits of block i // 8: counter (block, block >> 32, offset, offset >> 32), key (seed, seed >> 32);
# bits 16 (i % 2) .. 16 (i % 2) + 15 of word (i % 8) // 2.  It is kept where they are at least threshold = round(65536 p).
M0, M1, K0, K1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85


def _threshold(p):
    return int(math.floor(p * 65536 + 0.5))


def _keep(n, seed, offset, threshold):
    low = 0xFFFFFFFF
    block = torch.arange((n + 7) // 8, device=DEV, dtype=torch.int64)
    a, b = block & low, block >> 32
    c, d = torch.full_like(block, offset & low), torch.full_like(block, (offset >> 32) & low)
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(10):
        pa, pc = a * M0, c * M1                                   # (the 64 bits of a product, as a signed number)
        a, b, c, d = ((pc >> 32) & low) ^ b ^ k0, pc & low, ((pa >> 32) & low) ^ d ^ k1, pa & low
        k0, k1 = (k0 + K0) & low, (k1 + K1) & low
    words = torch.stack((a, b, c, d), dim=1)
    halves = torch.stack((words & 0xFFFF, words >> 16), dim=2).reshape(-1)[:n]
    return (halves >= threshold).float()


# ---------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    w = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        n, par = case["images"] * (case["tokens"] - case["skip"]) * case["dim"], 2 * case["dim"] if case["affine"] else 0
        # x in and y out; with gradients dy in, dx, dw and db out
        return {"bytes": w * (2 * n + par) * (2 if case["train"] else 1), "flops": n * (8 + (14 if case["train"] else 0))}
    if case["op"] == "mlp":
        M, D, H, O = case["rows"], case["dim"], case["hidden"], case["out"]
        par = 2 * H * D + O * H + (2 * H + O if case["bias"] else 0)
        return {"bytes": w * (M * D + M * O + par) * (2 if case["train"] else 1), "flops": 2 * M * H * (2 * D + O) * (3 if case["train"] else 1)}
    n = case["rows"] * case["dim"]
    # x (and the residual) in, y out; with gradients dy in and dx out (the residual's gradient is dy itself)
    return {"bytes": w * n * (2 + (1 if case["residual"] else 0) + (2 if case["train"] else 0)), "flops": 3 * n}


# ---------------------------------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        v = {n: t.detach().double() for n, t in s.items() if isinstance(t, torch.Tensor)}
        out = {"norm": _exact_norm, "mlp": _exact_mlp, "dropout": _exact_dropout}[case["op"]](case, s, v)
    keys = ["y"] + ["d" + n for n in s["leaves"]]
    return {k: out[k] for k in keys}


def _exact_norm(case, s, v):
    var, mean = torch.var_mean(v["x"], dim=-1, correction=0, keepdim=True)
    r = (var + s["eps"]).rsqrt()
    xh = (v["x"] - mean) * r
    e = v["dy"] * v["w"] if "w" in v else v["dy"]
    dx = r * (e - e.mean(-1, keepdim=True) - xh * (e * xh).mean(-1, keepdim=True))
    y = torch.addcmul(v["b"], xh, v["w"]) if "w" in v else xh
    return {"y": y, "dx": dx, "dw": (v["dy"] * xh).sum((0, 1)), "db": v["dy"].sum((0, 1))}


def _exact_mlp(case, s, v):
    H = case["hidden"]
    g, u = v["x"] @ v["w12"][:H].t(), v["x"] @ v["w12"][H:].t()
    if case["bias"]:
        g, u = g + v["b12"][:H], u + v["b12"][H:]
    if case["act"] == "silu":
        q = 1 / (1 + torch.exp(-g))
        act, slope = g * q, q * (1 + g * (1 - q))
    else:
        q = 0.5 * torch.erfc(-g / math.sqrt(2.0))
        act, slope = g * q, q + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    h = act * u
    y = h @ v["w3"].t()
    if case["bias"]:
        y = y + v["b3"]
    if not case["train"]:
        return {"y": y}
    dh = v["dy"] @ v["w3"]
    dg, du = dh * u * slope, dh * act
    return {"y": y, "dx": dg @ v["w12"][:H] + du @ v["w12"][H:], "dw12": torch.cat((dg.t() @ v["x"], du.t() @ v["x"])),
            "db12": torch.cat((dg.sum(0), du.sum(0))), "dw3": v["dy"].t() @ h, "db3": v["dy"].sum(0)}


def _exact_dropout(case, s, v):
    n = v["x"].numel()
    cut = int(case["p"] * 65536 + 0.5)
    ctr = np.zeros((4, (n + 7) // 8), np.uint64)
    ctr[0], ctr[2] = np.arange(ctr.shape[1], dtype=np.uint64), s["offset"] % 2 ** 32
    ctr[1], ctr[3] = ctr[0] >> np.uint64(32), s["offset"] >> 32
    ctr[0] &= np.uint64(2 ** 32 - 1)
    key = [s["seed"] % 2 ** 32, s["seed"] >> 32]
    for r in range(10):
        p, q = ctr[0] * np.uint64(M0), ctr[2] * np.uint64(M1)
        mask, up = np.uint64(2 ** 32 - 1), np.uint64(32)
        ctr = np.stack((q >> up ^ ctr[1] ^ np.uint64((key[0] + r * K0) % 2 ** 32), q & mask, p >> up ^ ctr[3] ^ np.uint64((key[1] + r * K1) % 2 ** 32), p & mask))
    bits = np.ascontiguousarray(ctr.T).astype("<u4").view("<u2").reshape(-1)[:n]
    gain = torch.from_numpy(np.where(bits >= cut, 65536.0 / (65536 - cut), 0.0)).to(DEV).reshape(v["x"].shape)
    out = {"y": v["x"] * gain + v.get("residual", 0), "dx": v["dy"] * gain, "dresidual": v["dy"]}
    return out

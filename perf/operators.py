"""What the normalisation over channels, the gradient norm with clipping and the clipped update are measured on.

A pass is one call as a training or inference program makes it: the normalisation of one layer (forward, backward, or
forward with its output in 8 bits), the clipping of a list of gradients by their global norm, or one clipped update of a
network's flat parameter vector. Sizes are those of this framework's networks.
"""
from __future__ import annotations

import math
import random

import torch

own = False

EPS = 1e-5
E4M3_MAX = 448.0
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # one 19 x 19 board through a layer of the Go network: nothing but latency
        {"name": "norm_board_361x128", "op": "norm", "rows": 361, "channels": 128, "valid": 128, "residual": False,
         "train": False, "relu": True},
        # a residual layer of the Go network at the Go tool's default batch, in training
        {"name": "norm_go_92416x128", "op": "norm", "rows": 92416, "channels": 128, "valid": 128, "residual": True,
         "train": True, "relu": True},
        # AlexNet's wide affine layers at the benchmark's batch: few rows, long ones
        {"name": "norm_affine_128x4096", "op": "norm", "rows": 128, "channels": 4096, "valid": 4096, "residual": False,
         "train": True, "relu": False},
        # the same Go layer backward
        {"name": "norm_back_go_92416x128", "op": "norm_back", "rows": 92416, "channels": 128, "valid": 128, "add": False,
         "relu": True},
        # CIFAR-10 ResNet's first stage, 128 images of 32 x 32 x 16 in padded channels, with the residual stream's delta
        {"name": "norm_back_cifar_131072x32", "op": "norm_back", "rows": 131072, "channels": 32, "valid": 16, "add": True,
         "relu": False},
        # one image's last feature map (8 x 8 x 512) in 8 bits
        {"name": "norm8_map_64x512", "op": "norm8", "rows": 64, "channels": 512, "valid": 512, "residual": False,
         "relu": True},
        # the first stage of ResNet-18 at 64 images, in 8 bits, with the residual
        {"name": "norm8_stage_262144x64", "op": "norm8", "rows": 262144, "channels": 64, "valid": 64, "residual": True,
         "relu": True},
        # LeNet's eight tensors, within the bound, as most steps are: launches
        {"name": "clip_lenet_8", "op": "clip", "tensors": 8, "numel": 431_080, "split": 1, "type": "float32", "over": False},
        # ResNet-18's 62 tensors, clipped
        {"name": "clip_resnet18_62", "op": "clip", "tensors": 62, "numel": 11_699_112, "split": 2, "type": "float32",
         "over": True},
        # AlexNet's 16 tensors as 16-bit gradients, clipped
        {"name": "clip_alexnet_bf16", "op": "clip", "tensors": 16, "numel": 62_378_344, "split": 3, "type": "bfloat16",
         "over": True},
        # a clipped step of the CIFAR-10 network's 85 thousand parameters
        {"name": "update_cifar", "op": "update", "numel": 85_098},
        # the largest: a clipped step of AlexNet's 62.4 million
        {"name": "update_alexnet", "op": "update", "numel": 62_378_344},
    ]


def _between(rng, least, most):
    return int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "norm_back", "norm_back", "norm8", "clip", "clip", "update"])
    if op == "update":
        return {"op": op, "numel": _between(rng, 1_000, 60_000_000)}
    if op == "clip":
        tensors = _between(rng, 1, 60)
        return {"op": op, "tensors": tensors, "numel": _between(rng, 1_000 * tensors, 60_000_000), "split": rng.randrange(1 << 30),
                "type": rng.choice(sorted(DTYPES)), "over": rng.random() < 0.5}
    # a layer: any number of channels, padded as the framework pads them, and any number of positions
    valid = _between(rng, 8, 8192)
    channels = valid if valid % 64 == 0 else (valid + 31) // 32 * 32
    case = {"op": op, "rows": _between(rng, 1, max(2, 16_000_000 // channels)), "channels": channels, "valid": valid,
            "relu": rng.random() < 0.5}
    if op == "norm_back":
        return case | {"add": rng.random() < 0.5}
    case["residual"] = rng.random() < 0.5
    return case | {"train": rng.random() < 0.5} if op == "norm" else case


def _sizes(case):
    """`tensors` sizes of four decades that add up to `numel`: a network's filters and its biases."""
    rng = random.Random(case["split"])
    shares = [10 ** rng.uniform(-4, 0) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["numel"] * s / sum(shares))) for s in shares]
    sizes[sizes.index(max(sizes))] += max(0, case["numel"] - sum(sizes))
    return sizes


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device="cuda") * std).to(dtype)

    state = {"case": case}
    if case["op"] == "update":
        n = (case["numel"] + 63) // 64 * 64
        state |= {"n": n, "w": normal(n, std=0.05), "g": normal(n, std=1e-3), "v": normal(n, std=1e-4)}
        state["w16"] = state["w"].bfloat16()
        # half of what the gradients' norm comes out as
        return state | {"max_norm": 0.5 * 1e-3 * math.sqrt(n), "out": torch.zeros(2, device="cuda")}
    if case["op"] == "clip":
        sizes = _sizes(case)
        state["grads"] = [normal(n, std=1e-3, dtype=DTYPES[case["type"]]) for n in sizes]
        norm = 1e-3 * math.sqrt(sum(sizes))
        # over: means over four devices' batches that are to be sums. The bound is one of two in turn, so that a pass has
        # something to clip where the one before it has clipped
        state |= {"bounds": (0.7 * norm, 1.6 * norm) if case["over"] else (16 * norm,) * 2, "scale": 4.0 if case["over"] else 1.0}
        return state | {"out": torch.zeros(2, device="cuda"), "at": 0}
    rows, c, valid = case["rows"], case["channels"], case["valid"]

    def activations(std):
        x = normal(rows, c, std=std)
        x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device="cuda"))     # positions differ in size
        x[:, valid:] = 0
        return x.bfloat16()

    gamma = 1.0 + normal(c, std=0.2)
    gamma[valid:] = 0
    state |= {"x": activations(1.0), "gamma": gamma}
    if case["op"] == "norm_back":
        x = state["x"].double()
        state["rstd"] = (x.square().sum(1) / valid + EPS).rsqrt().float()
        state |= {"dy": activations(1e-2), "dgamma": normal(c, std=1e-2), "dx": torch.empty_like(state["x"]),
                  "add": activations(1e-2) if case["add"] else None}
        state["dgamma"][valid:] = 0
        return state
    state["residual"] = activations(1.0) if case["residual"] else None
    state["h"] = torch.empty_like(state["x"]) if case["residual"] else None
    if case["op"] == "norm8":
        return state | {"q": torch.empty((rows, c), dtype=torch.float8_e4m3fn, device="cuda"),
                        "scales": torch.empty(rows, device="cuda")}
    state["y"] = torch.empty_like(state["x"])
    state["rstd"] = torch.empty(rows, device="cuda") if case["train"] else None
    return state


def _kernels():
    from rembrandt_b200.ops import native_ops as K
    return K


def _kept(state, name, make):
    """What a program makes once for its tensors and keeps."""
    if name not in state:
        state[name] = make()
    return state[name]


def run(state):
    return {"norm": _norm, "norm8": _norm8, "norm_back": _norm_back, "clip": _clip, "update": _update}[state["case"]["op"]](state)


def _layer(state):
    case = state["case"]
    return case["rows"], case["channels"], case["valid"]


def _plain_norm(state):
    """h, 1 / root mean square and the output in 32 bits."""
    case = state["case"]
    rows, c, valid = _layer(state)
    h = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).bfloat16()
    hf = h.float()
    rstd = ((hf * hf).sum(1) / valid + EPS).rsqrt()
    y = hf * rstd[:, None] * state["gamma"]
    return h, rstd, y.clamp_min(0.0) if case["relu"] else y


def _norm(state):
    case = state["case"]
    if own:
        _kernels().rms_norm_fwd(state["x"], *_layer(state), EPS, state["gamma"], state["y"], rstd=state["rstd"],
                                residual=state["residual"], h=state["h"], relu=case["relu"])
        return {"y": state["y"], "h": state["h"], "rstd": state["rstd"]}
    h, rstd, y = _plain_norm(state)
    return {"y": y.bfloat16(), "h": h if case["residual"] else None, "rstd": rstd if case["train"] else None}


def _norm8(state):
    case = state["case"]
    if own:
        _kernels().rms_norm_fwd_e4m3(state["x"], *_layer(state), EPS, state["gamma"], state["q"], state["scales"],
                                     residual=state["residual"], h=state["h"], relu=case["relu"])
        return {"q": state["q"], "scales": state["scales"], "h": state["h"]}
    h, _, y = _plain_norm(state)
    scales = y.abs().amax(1) / E4M3_MAX
    scales = torch.where(scales == 0, 1.0, scales)
    return {"q": (y / scales[:, None]).to(torch.float8_e4m3fn), "scales": scales, "h": h if case["residual"] else None}


def _norm_back(state):
    case = state["case"]
    rows, c, valid = _layer(state)
    if own:
        K = _kernels()
        ws = _kept(state, "ws", lambda: K.rms_norm_scratch(c, state["x"].device))
        K.rms_norm_bwd(state["x"], state["dy"], rows, c, valid, state["rstd"], state["gamma"], state["dgamma"], state["dx"], ws,
                       add=state["add"], relu=case["relu"])
        return {"dx": state["dx"], "dgamma": state["dgamma"]}
    xhat = state["x"].float() * state["rstd"][:, None]
    g = state["dy"].float()
    if case["relu"]:
        g = torch.where(xhat * state["gamma"] > 0, g, 0.0)
    state["dgamma"] += (g * xhat).sum(0)
    g = g * state["gamma"]
    dx = state["rstd"][:, None] * (g - xhat * ((g * xhat).sum(1, keepdim=True) / valid))
    if case["add"]:
        dx = dx + state["add"].float()
    return {"dx": dx.bfloat16(), "dgamma": state["dgamma"]}


def _plain_coefficient(norm, max_norm):
    return torch.where(norm.isfinite(), (max_norm / norm).clamp_max(1.0), 0.0)


def _clip(state):
    scale, max_norm, grads = state["scale"], state["bounds"][state["at"] % 2], state["grads"]
    state["at"] += 1
    if own:
        K = _kernels()
        many = _kept(state, "list", lambda: K.grad_list(grads))
        ws = _kept(state, "ws", lambda: K.grad_norm_scratch(grads[0].device))
        K.grad_norm(many, max_norm, state["out"], ws, scale=scale)
        K.clip_grads(many, state["out"], scale=scale)
        return {"out": state["out"], "grads": grads}
    # squares in 32 bits, their sum over millions in 64
    sums = torch.stack([(g.float() * g.float()).sum(dtype=torch.float64) for g in grads])
    norm = (scale * sums.sum().sqrt()).float()
    coefficient = _plain_coefficient(norm, max_norm)
    [g.copy_(g.float() * (scale * coefficient)) for g in grads]
    return {"out": torch.stack([norm, coefficient]), "grads": grads}


LR, MU, L2 = 0.01, 0.9, 5e-4


def _update(state):
    w, g, v, w16, max_norm = state["w"], state["g"], state["v"], state["w16"], state["max_norm"]
    if own:
        K = _kernels()
        many = _kept(state, "list", lambda: K.grad_list([g]))
        ws = _kept(state, "ws", lambda: K.grad_norm_scratch(g.device))
        K.grad_norm(many, max_norm, state["out"], ws)
        K.sgd_fused(w, g, v, w16, state["n"], LR, MU, L2, 1.0, 1, clip=state["out"])
        return {"w": w, "g": g, "v": v, "w16": w16, "out": state["out"]}
    norm = (g * g).sum(dtype=torch.float64).sqrt().float()
    coefficient = _plain_coefficient(norm, max_norm)
    v.mul_(MU).sub_(LR * (g * coefficient + L2 * w))
    w.add_(v)
    w16.copy_(w)
    g.zero_()
    return {"w": w, "g": g, "v": v, "w16": w16, "out": torch.stack([norm, coefficient])}


def work(case):
    if case["op"] == "update":
        n = (case["numel"] + 63) // 64 * 64
        return {"bytes": 26.0 * n + 8, "flops": 9.0 * n}
    if case["op"] == "clip":
        size = DTYPES[case["type"]].itemsize * float(sum(_sizes(case)))
        return {"bytes": size * (2 if case["over"] else 1) + 8, "flops": 3.0 * sum(_sizes(case))}
    rows, c = case["rows"], case["channels"]
    n = float(rows * c)
    if case["op"] == "norm_back":
        return {"bytes": n * (8 if case["add"] else 6) + 4 * rows + 12 * c, "flops": 9 * n}
    moved = n * (6 if case["residual"] else 2) + 4 * c
    if case["op"] == "norm8":
        return {"bytes": moved + n + 4 * rows, "flops": 6 * n}
    return {"bytes": moved + 2 * n + (4 * rows if case["train"] else 0), "flops": 5 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "update":
        w, g, v = (s[k].double() for k in "wgv")
        norm = torch.linalg.vector_norm(g)
        coefficient = torch.clamp(s["max_norm"] / norm, max=1.0)
        v = MU * v - LR * (coefficient * g + L2 * w)
        return {"w": w + v, "g": torch.zeros_like(g), "v": v, "w16": w + v, "out": torch.stack([norm, coefficient])}
    if case["op"] == "clip":
        norm = s["scale"] * torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g.double()) for g in s["grads"]]))
        coefficient = torch.clamp(s["bounds"][0] / norm, max=1.0)
        return {"out": torch.stack([norm, coefficient]), "grads": [g.double() * s["scale"] * coefficient for g in s["grads"]]}
    rows, c, valid = case["rows"], case["channels"], case["valid"]
    gamma, x = s["gamma"].double(), s["x"].double()
    if case["op"] == "norm_back":
        # by the chain rule from y = gamma * x * r, r = (mean of squares + eps) ^ -1/2, dr/dx = -r^3 x / valid
        r = s["rstd"].double()[:, None]
        dy = s["dy"].double() * ((gamma * x > 0) if case["relu"] else 1.0)
        through_r = (dy * gamma * x).sum(1, keepdim=True) * -(r ** 3) / valid
        dx = dy * gamma * r + through_r * x + (s["add"].double() if case["add"] else 0.0)
        return {"dx": dx, "dgamma": s["dgamma"].double() + torch.einsum("rc,rc,rk->c", dy, x, r)}
    h = x if s["residual"] is None else (x + s["residual"].double()).to(torch.bfloat16).double()
    mean = torch.einsum("rc,rc->r", h[:, :valid], h[:, :valid]) / valid
    y = gamma * h / torch.sqrt(mean + EPS)[:, None]
    y = torch.relu(y) if case["relu"] else y
    kept_h = h if case["residual"] else None
    if case["op"] == "norm8":
        scales = y.abs().max(1).values / E4M3_MAX
        scales[scales == 0] = 1.0
        return {"q": y / scales[:, None], "scales": scales, "h": kept_h}
    return {"y": y, "h": kept_h, "rstd": 1 / torch.sqrt(mean + EPS) if case["train"] else None}

"""Timing cases of the training operators: the AdamW step over all tensors of a network, and layer norm with its gradient.

`run` computes a case in its plain form, with elementary torch operations, or, with `own` set, through the framework's entry
points.  Sizes are those of the networks of this framework: boards of 3x3 to 19x19, 1 to 20 residual blocks, 128 to 512
channels, batches of one board up to the 3993 that self-play holds at once; rows of a few thousand values stand for wider
layers."""
import math

import torch

own = False

BLOCK = 256       # elements that share a scale where the AdamW state is held in 8 bits
PLANES = 17       # input planes of a board
LR, BETA1, BETA2, EPS, DECAY, STEP = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 1000
NORM_EPS = 1e-5
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    def adamw(name, board, blocks, channels, dtype, bits):
        return {"name": name, "op": "adamw", "board": board, "blocks": blocks, "channels": channels, "type": dtype, "bits": bits}

    def norm(name, rows, cols, dtype, train):
        return {"name": name, "op": "norm", "rows": rows, "cols": cols, "type": dtype, "train": train}

    return [
        # the smallest network that the tests train: 0.3 M parameters, latency counts
        adamw("adamw 6x6 1x128", 6, 1, 128, "float32", 32),
        # the headline network of Go 19x19: 24 M parameters, one optimizer step
        adamw("adamw 19x19 20x256", 19, 20, 256, "float32", 32),
        # a Reversi network whose weights are held in bfloat16
        adamw("adamw 8x8 10x256 bf16", 8, 10, 256, "bfloat16", 32),
        # the smallest and the headline network with their optimizer state in 8 bits
        adamw("adamw8 6x6 1x128", 6, 1, 128, "float32", 8),
        adamw("adamw8 19x19 20x256", 19, 20, 256, "float32", 8),
        # twice the width: 95 M bfloat16 parameters, what 8-bit state is for
        adamw("adamw8 9x9 20x512 bf16", 9, 20, 512, "bfloat16", 8),
        # one board of 19x19 through one layer of the trunk (a single position being played): latency
        norm("norm 1 board", 361, 256, "float32", False),
        # every game of a self-play round through one layer of the trunk
        norm("norm 3993 boards bf16", 3993 * 361, 256, "bfloat16", False),
        # a training batch of 256 boards, one layer of the trunk, forward and backward
        norm("norm train 256 boards", 256 * 361, 256, "float32", True),
        # the policy head's two planes, flattened, forward and backward: odd rows
        norm("norm train policy head", 512, 722, "float32", True),
        # the value head's plane, flattened, in bfloat16: odd rows that start on odd addresses
        norm("norm train value head bf16", 2048, 361, "bfloat16", True),
        # wide rows, forward and backward
        norm("norm train wide bf16", 4096, 8192, "bfloat16", True),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["float32", "bfloat16", "float16"])
    if rng.random() < 0.5:
        return {"op": "adamw", "board": rng.randint(3, 19), "blocks": rng.randint(1, 20), "channels": rng.choice([128, 192, 256, 320, 384]),
                "type": kind, "bits": rng.choice([32, 8])}
    train = rng.random() < 0.6
    cols = _spread(rng, 1, 8192)
    return {"op": "norm", "rows": _spread(rng, 1, min(1 << 20, (1 << 25) // cols)), "cols": cols, "type": kind, "train": train}


def _shapes(case):
    """The shapes of the network's parameters, in its order."""
    n, c, points = case["blocks"], case["channels"], case["board"] ** 2
    actions = points + 1
    return ([(c, PLANES, 3, 3), (c,)] + [(c, c, 3, 3)] * n + [(c,)] * n + [(c, c, 3, 3)] * n + [(c,)] * n
            + [(2, c, 1, 1), (2,), (actions, 2 * points), (actions,), (1, c, 1, 1), (1,), (256, points), (256,), (1, 256), (1,)])


def _padded(n):
    return -(-n // BLOCK) * BLOCK


def _random(case, seed):
    return torch.Generator(device="cuda").manual_seed(seed * 7919 + 11)


def _quantize(m, v):
    """8-bit codes and scales of a state in 64 bits, both laid out in blocks: m = s sgn(c) (c / 127)^2, v = s (c / 255)^4."""
    def scales(x):
        return x.abs().amax(1, keepdim=True).float()

    def companded(x, s, power, top):
        s = s.double()
        return torch.where(s > 0, (x.abs() / torch.where(s > 0, s, 1.0)).pow(1.0 / power) * top, torch.zeros_like(x)).round()

    sm, sv = scales(m), scales(v)
    cm = (companded(m, sm, 2, 127.0) * m.sign()).to(torch.int8)
    cv = companded(v, sv, 4, 255.0)
    cv = torch.where((v > 0) & (sv > 0), cv.clamp(min=1.0), cv).to(torch.uint8)
    return cm, sm.reshape(-1), cv, sv.reshape(-1)


def _dequantize(code, scale):
    c, s = code.double(), scale.double()[:, None]
    return s * c * c.abs() / 127.0 ** 2 if code.dtype == torch.int8 else s * c ** 4 / 255.0 ** 4


def prepare(case, seed):
    g = _random(case, seed)
    dtype = TYPES[case["type"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "norm":
        rows, cols = case["rows"], case["cols"]
        # a convolution's outputs: an offset and a spread for each channel, and rows of different size
        x = (normal(rows, cols) * (0.5 + torch.rand(cols, generator=g, device="cuda")) + normal(cols)) * (0.25 + torch.rand(rows, 1, generator=g, device="cuda"))
        state = {"case": case, "x": x.to(dtype), "weight": (1.0 + 0.1 * normal(cols)), "bias": 0.1 * normal(cols)}
        if case["train"]:
            state["dy"] = (normal(rows, cols) * 1e-2).to(dtype)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
        return state
    # all tensors of the network in one buffer each for weights, gradients and the two states, every tensor on a boundary of
    # 256 elements (what lies between two tensors is zero and stays so)
    sizes = [math.prod(s) for s in _shapes(case)]
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + _padded(n))
    total = starts[-1]
    inside = torch.zeros(total, device="cuda")
    for n, at in zip(sizes, starts):
        inside[at:at + n] = 1.0
    # gradients whose size changes from block to block over four decades, a hundredth of them exactly zero with no history
    size = torch.pow(10.0, -4.0 * torch.rand(total // BLOCK, generator=g, device="cuda")).repeat_interleave(BLOCK) * inside
    size = size * (torch.rand(total, generator=g, device="cuda") > 0.01)
    grad = normal(total) * size
    m, v = normal(total) * size * 0.3, size * size * (0.5 + torch.rand(total, generator=g, device="cuda"))
    state = {"case": case, "step": STEP, "param": (normal(total) * 0.05 * inside).to(dtype), "grad": grad.to(dtype)}
    if case["bits"] == 8:
        cm, sm, cv, sv = _quantize(m.double().view(-1, BLOCK), v.double().view(-1, BLOCK))
        state.update(m=cm.reshape(-1), m_scale=sm, v=cv.reshape(-1), v_scale=sv)
    else:
        state.update(m=m, v=v)
    for name in ("param", "grad", "m", "v"):
        state[name + "s"] = [state[name][at:at + n].view(s) for at, n, s in zip(starts, sizes, _shapes(case))]
    if case["bits"] == 8:
        for name in ("m_scale", "v_scale"):
            state[name + "s"] = [state[name][at // BLOCK:(at + _padded(n)) // BLOCK] for at, n in zip(starts, sizes)]
    return state


def _norm_plain(s):
    x, w, b = s["x"].float(), s["weight"], s["bias"]
    mean = x.mean(1, keepdim=True)
    centred = x - mean
    r = 1.0 / torch.sqrt((centred * centred).mean(1, keepdim=True) + NORM_EPS)
    h = centred * r
    y = (h * w + b).to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    wdy = dy * w
    dx = r * (wdy - wdy.mean(1, keepdim=True) - h * (wdy * h).mean(1, keepdim=True))
    return {"y": y, "dx": dx.to(s["x"].dtype), "dweight": (dy * h).sum(0), "dbias": dy.sum(0)}


def _adamw_plain(s):
    c1, c2 = 1.0 - BETA1 ** s["step"], 1.0 - BETA2 ** s["step"]
    if s["case"]["bits"] == 8:
        # in 64 bits: which code a value gets is decided at a border between two
        grad = s["grad"].double().view(-1, BLOCK)
        m = _dequantize(s["m"].view(-1, BLOCK), s["m_scale"]) * BETA1 + grad * (1.0 - BETA1)
        v = _dequantize(s["v"].view(-1, BLOCK), s["v_scale"]) * BETA2 + grad * grad * (1.0 - BETA2)
        cm, sm, cv, sv = _quantize(m, v)
        s["m"].copy_(cm.reshape(-1))
        s["m_scale"].copy_(sm)
        s["v"].copy_(cv.reshape(-1))
        s["v_scale"].copy_(sv)
        m, v = m.reshape(-1).float(), v.reshape(-1).float()
        held = [_dequantize(s[k].view(-1, BLOCK), s[k + "_scale"]).reshape(-1).float() for k in ("m", "v")]
    else:
        grad = s["grad"].float()
        m = s["m"].mul_(BETA1).add_(grad * (1.0 - BETA1))
        v = s["v"].mul_(BETA2).add_(grad * grad * (1.0 - BETA2))
        held = [m, v]
    p = s["param"].float()
    p = p - p * (LR * DECAY) - m / (torch.sqrt(v) * (1.0 / math.sqrt(c2)) + EPS) * (LR / c1)
    s["param"].copy_(p)
    return {"param": s["param"], "m": held[0], "v": held[1]}


def run(state):
    s = state
    if s["case"]["op"] == "norm":
        if not own:
            with torch.no_grad():
                return _norm_plain(s)
        from alphazero_amd.network.layer_norm import layer_norm
        y = layer_norm(s["x"], s["weight"], s["bias"], NORM_EPS)
        if not s["case"]["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y, "dx": dx, "dweight": dw, "dbias": db}
    s["step"] += 1
    if not own:
        return _adamw_plain(s)
    from alphazero_amd.network.adamw import adamw_step, dequantize_state
    adamw_step(s["params"], s["grads"], s["ms"], s["vs"], s["step"], lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY,
               exp_avg_scales=s.get("m_scales"), exp_avg_sq_scales=s.get("v_scales"))
    if s["case"]["bits"] == 8:
        return {"param": s["param"], "m": dequantize_state(s["m"], s["m_scale"]), "v": dequantize_state(s["v"], s["v_scale"])}
    return {"param": s["param"], "m": s["m"], "v": s["v"]}


def work(case):
    size = 4 if case["type"] == "float32" else 2
    if case["op"] == "norm":
        n, cols = case["rows"] * case["cols"], case["cols"]
        if case["train"]:
            return {"bytes": 4 * n * size + 4 * cols * 4, "flops": 20 * n}
        return {"bytes": 2 * n * size + 2 * cols * 4, "flops": 8 * n}
    n = sum(math.prod(s) for s in _shapes(case))
    # weights read and written, the gradient read; each state read and written; 8-bit states come back as 32-bit values too
    held = 2 * (1 + 1 + 4) + 16 / BLOCK if case["bits"] == 8 else 2 * (4 + 4)
    return {"bytes": n * (3 * size + held), "flops": 16 * n}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w, b = (s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "bias"))
        mean = x.sum(1, keepdim=True) / case["cols"]
        var = ((x - mean) ** 2).sum(1, keepdim=True) / case["cols"]
        y = (x - mean) / (var + NORM_EPS) ** 0.5 * w + b
        if not case["train"]:
            return {"y": y}
        dx, dw, db = torch.autograd.grad(y, (x, w, b), s["dy"].double())
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    t = STEP + 1
    held = {"m": s["m"].double(), "v": s["v"].double()}
    if case["bits"] == 8:
        held["m"] = held["m"].sign() * (held["m"] / 127.0) ** 2 * s["m_scale"].double().repeat_interleave(BLOCK)
        held["v"] = (held["v"] / 255.0) ** 4 * s["v_scale"].double().repeat_interleave(BLOCK)
    g, p = s["grad"].double(), s["param"].double()
    m = BETA1 * held["m"] + (1.0 - BETA1) * g
    v = BETA2 * held["v"] + (1.0 - BETA2) * g ** 2
    p = (1.0 - LR * DECAY) * p - LR * (m / (1.0 - BETA1 ** t)) / ((v / (1.0 - BETA2 ** t)) ** 0.5 + EPS)
    if case["bits"] == 8:
        # what the 8-bit codes of the new state stand for: the nearest of the values that a block can hold, measured in the
        # domain in which they are evenly spaced
        sm = m.view(-1, BLOCK).abs().max(1).values.float().double().repeat_interleave(BLOCK)
        sv = v.view(-1, BLOCK).max(1).values.float().double().repeat_interleave(BLOCK)
        root = torch.sqrt(m.abs() / sm.clamp(min=1e-300))
        m = torch.sign(m) * sm * (torch.floor(root * 127.0 + 0.5) / 127.0) ** 2
        root = torch.sqrt(torch.sqrt(v / sv.clamp(min=1e-300)))
        code = torch.floor(root * 255.0 + 0.5)
        v = sv * (torch.where(v > 0, code.clamp(min=1.0), code) / 255.0) ** 4
    return {"param": p, "m": m, "v": v}

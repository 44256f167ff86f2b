"""What the operators for fine-tuning and serving the dense ConvNeXt V2 cost, each next to its plain form.

Three operators, over the sizes of this repository's own configurations (`convnextv2_atto / nano / base / huge`) and odd ones beside them:

  adamw32  one AdamW step over many parameter tensors with fp32 moments, optionally behind a global gradient-norm clip
  adamw8   the same step with both moments held in 8 bits (256-element blocks with one fp32 scale each), and the moments' values read back
  int8     y = x W^T + b with x quantised to 8-bit integers per row (token) on the way, W quantised per output channel once

`own = False` runs the elementary torch form, `own = True` the calls a user makes of this package.

The 8-bit moments. A parameter's elements are cut into blocks of 256 in storage order; each tensor starts a block of its own. Per block
  exp_avg     m = s_m * k|k| / 127^2,  k in -127..127,  s_m = max|m| of the block,  k = sign(m) * round(127 * sqrt(|m| / s_m))
  exp_avg_sq  v = s_v * (k / 255)^4,   k in 0..255,     s_v = max v of the block,   k = round(255 * (v / s_v)^(1/4)), at least 1 where v > 0
rounded half up from the 64-bit value (a border is decided on more bits than 32), s_m and s_v rounded to fp32. The moments are formed in 64 bits, every
product and sum rounded on its own: (9 s + g) / 10 is often an exact tie between two fp32 scales. The parameter's own update uses the moments before
they are rounded to codes.
"""
import math
import random

import torch

own = False

BLOCK = 256
LR, BETA1, BETA2, EPS, DECAY, STEPS_DONE = 1.5e-4, 0.9, 0.95, 1e-8, 0.05, 40   # the pretraining recipe's AdamW, some way into a run
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}

# depths and widths of this repository's configurations (patch 8, 12 input bands, 1000 classes)
NETS = {
    "atto": ([2, 2, 6, 2], [40, 80, 160, 320]),
    "nano": ([2, 2, 8, 2], [80, 160, 320, 640]),
    "base": ([3, 3, 27, 3], [128, 256, 512, 1024]),
    "huge": ([3, 3, 27, 3], [352, 704, 1408, 2816]),
}


def listed():
    return [
        # the smallest network's whole parameter list, plain fp32 training: few bytes in many tensors, so latency counts
        {"name": "adamw32_atto_fp32", "op": "adamw32", "net": "atto", "dtype": "fp32", "clip": 0.0},
        # an ordinary fine-tuning step: base network, clipped gradients
        {"name": "adamw32_base_fp32_clip", "op": "adamw32", "net": "base", "dtype": "fp32", "clip": 1.0},
        # the largest network with bf16 parameters and gradients, fp32 moments
        {"name": "adamw32_huge_bf16", "op": "adamw32", "net": "huge", "dtype": "bf16", "clip": 0.0},
        # 8-bit moments, smallest network
        {"name": "adamw8_atto_fp32", "op": "adamw8", "net": "atto", "dtype": "fp32", "clip": 0.0},
        # 8-bit moments behind a clip, ordinary network in bf16
        {"name": "adamw8_base_bf16_clip", "op": "adamw8", "net": "base", "dtype": "bf16", "clip": 1.0},
        # 8-bit moments where they matter: the largest network with fp32 parameters
        {"name": "adamw8_huge_fp32", "op": "adamw8", "net": "huge", "dtype": "fp32", "clip": 0.0},
        # one pooled feature vector through a wide layer: bound by reading the weights
        {"name": "int8_one_row_bf16", "op": "int8", "dtype": "bf16", "m": 1, "k": 1024, "n": 4096, "bias": True},
        # eight images' pooled features through the classifier of the largest network
        {"name": "int8_head_8_fp16", "op": "int8", "dtype": "fp16", "m": 8, "k": 2816, "n": 1000, "bias": True},
        # one image's last stage (7 x 7 positions) in the largest network
        {"name": "int8_one_image_bf16", "op": "int8", "dtype": "bf16", "m": 49, "k": 2816, "n": 11264, "bias": True},
        # odd sizes in fp32, no bias: a small projection whose rows start at no vector boundary
        {"name": "int8_ragged_fp32", "op": "int8", "dtype": "fp32", "m": 1003, "k": 333, "n": 77, "bias": False},
        # 256 images of the third stage (14 x 14 positions) of the base network, widening layer
        {"name": "int8_base_batch_bf16", "op": "int8", "dtype": "bf16", "m": 50176, "k": 512, "n": 2048, "bias": True},
        # 256 images of the last stage of the largest network, narrowing layer
        {"name": "int8_huge_batch_bf16", "op": "int8", "dtype": "bf16", "m": 12544, "k": 11264, "n": 2816, "bias": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["adamw32", "adamw8", "int8", "int8"])
    if op != "int8":
        return {"op": op, "tensors": _log(rng, 1, 400), "total": _log(rng, 2_000, 400_000_000), "salt": rng.randrange(1 << 30),
                "dtype": rng.choice(["fp32", "bf16", "fp16"]), "clip": rng.choice([0.0, 0.25, 1.0, 4.0])}
    while True:
        c = {"op": op, "dtype": rng.choice(["fp32", "bf16", "bf16", "fp16"]), "m": _log(rng, 1, 50176), "k": _log(rng, 16, 11264),
             "n": _log(rng, 16, 11264), "bias": rng.random() < 0.5}
        if c["m"] * c["k"] * c["n"] <= 12544 * 11264 * 2816 and c["m"] * max(c["k"], c["n"]) <= 12544 * 11264:
            return c


# ---------------------------------------------------------------------------------------------------------------- inputs

def _block(c):
    return [((c, 1, 7, 7), 1), ((c,), 0), ((c,), 0), ((c,), 0), ((4 * c, c), 1), ((4 * c,), 0), ((1, 1, 1, 4 * c), 1), ((1, 1, 1, 4 * c), 0),
            ((c, 4 * c), 1), ((c,), 0)]


def _shapes(case):
    """(shape, decayed) of every parameter tensor: those of a network, or `tensors` odd-sized ones of about `total` elements."""
    if "net" in case:
        depths, d = NETS[case["net"]]
        front = [((d[0], 12, 3, 3), 1), ((d[0],), 0), ((d[0],), 0), ((d[0],), 0), ((d[0], 1, 1, 1), 1), ((d[0],), 0), ((d[0],), 0), ((d[0],), 0)]
        down = [x for a, b in zip(d, d[1:]) for x in (((a,), 0), ((a,), 0), ((b, a, 2, 2), 1), ((b,), 0))]
        blocks = [x for n, c in zip(depths, d) for _ in range(n) for x in _block(c)]
        return front + down + blocks + [((d[3],), 0), ((d[3],), 0), ((1000, d[3]), 1), ((1000,), 0)]
    r = random.Random(case["salt"])
    share = [math.exp(r.gauss(0.0, 2.0)) for _ in range(case["tensors"])]
    return [((max(1, int(case["total"] * x / sum(share))),), r.randrange(2)) for x in share]


def _layout(case):
    """Tensors without decay first, then those with it; each starts at a multiple of the block. -> [(offset, shape, numel)], where decay begins, size."""
    shapes = _shapes(case)
    out, at, cut = [], 0, 0
    for decayed in (0, 1):
        if decayed:
            cut = at
        for shape, d in shapes:
            if d == decayed:
                n = math.prod(shape)
                out.append((at, shape, n))
                at += -(-n // BLOCK) * BLOCK
    return out, cut, at


def _to_codes(m, v):
    """64-bit moments [blocks, 256] -> (codes of m, codes of v, scales of m, scales of v)."""
    sm, sv = m.abs().amax(1).float(), v.amax(1).float()
    dm, dv = sm.double().clamp(min=1e-300)[:, None], sv.double().clamp(min=1e-300)[:, None]
    km = torch.floor(127.0 * (m.abs() / dm).sqrt() + 0.5).clamp(max=127.0) * torch.sign(m)
    kv = torch.floor(255.0 * (v / dv).sqrt().sqrt() + 0.5).clamp(max=255.0)
    kv = torch.where(v > 0, kv.clamp(min=1.0), kv)
    return km.to(torch.int8), torch.where(dv > 1e-300, kv, torch.zeros_like(kv)).to(torch.uint8), sm, sv


def _from_codes(km, kv, sm, sv):
    k, l = km.double(), kv.double()
    return k * k.abs() * (sm.double() * (1.0 / 127.0 ** 2))[:, None], (l * l).square() * (sv.double() * (1.0 / 255.0 ** 4))[:, None]


def _adamw_inputs(case, seed):
    """Flat parameter, gradient and moment buffers (zero between the tensors): per-tensor gradient sizes over two decades, heavy tails."""
    places, cut, size = _layout(case)
    gen = torch.Generator("cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    inside = torch.zeros(size // BLOCK, device="cuda")
    starts = torch.tensor([o // BLOCK for o, _, _ in places], device="cuda")
    inside[starts] = torch.exp(1.5 * torch.randn(len(places), device="cuda", generator=gen) - 7.0)
    which = torch.zeros(size // BLOCK, dtype=torch.long, device="cuda")
    which[starts] = 1
    scale = inside[starts][which.cumsum(0) - 1]                                     # one gradient size per tensor, by block
    left = torch.tensor([n for _, _, n in places], device="cuda")[which.cumsum(0) - 1] - BLOCK * (
        torch.arange(size // BLOCK, device="cuda") - starts[which.cumsum(0) - 1])   # elements from a block's start to its tensor's end
    keep = torch.arange(BLOCK, device="cuda")[None, :] < left[:, None]
    make = lambda: torch.randn(size // BLOCK, BLOCK, device="cuda", generator=gen)  # noqa: E731
    g = make()
    g = torch.where(keep, g * g.abs() * scale[:, None], 0.0)
    m = torch.where(keep, 0.3 * make() * scale[:, None], 0.0)
    v = torch.where(keep, (m * m + torch.square(make() * scale[:, None])) * 0.7, 0.0)
    p = torch.where(keep, 0.02 * make(), 0.0)
    return {"p": p.reshape(-1).to(dt), "g": g.reshape(-1).to(dt), "m": m.reshape(-1), "v": v.reshape(-1), "cut": cut, "places": places}


def _int8_inputs(case, seed):
    """Activations with a few loud channels and rows of different size, weights as a layer initialises and trains them."""
    gen = torch.Generator("cuda").manual_seed(seed)
    m, k, n, dt = case["m"], case["k"], case["n"], DTYPES[case["dtype"]]
    loud = 1.0 + 6.0 * (torch.rand(k, device="cuda", generator=gen) < 0.01)
    x = torch.randn(m, k, device="cuda", generator=gen) * loud * (0.25 + torch.rand(m, 1, device="cuda", generator=gen))
    w = torch.randn(n, k, device="cuda", generator=gen) * (0.02 + 0.02 * torch.rand(n, 1, device="cuda", generator=gen))
    b = 0.1 * torch.randn(n, device="cuda", generator=gen) if case["bias"] else None
    return {"x": x.to(dt), "w": w, "b": b}


def _weight_codes(w):
    a = w.double().abs().amax(1)
    return torch.round(w.double() * 127.0 / a[:, None]).to(torch.int8), (a / 127.0).float()


def prepare(case, seed):
    if case["op"] == "int8":
        s = _int8_inputs(case, seed)
        if own:
            from mmearth_train_amd.int8 import quantize_weight
            return {"op": "int8", "x": s["x"], "w": quantize_weight(s["w"], s["b"])}
        q, sw = _weight_codes(s["w"])
        return {"op": "int8", "x": s["x"], "q": q, "sw": sw, "b": s["b"]}
    s = _adamw_inputs(case, seed)
    s |= {"op": case["op"], "clip": case["clip"], "t": STEPS_DONE}
    if own:
        # the parameters and gradients are a program's own tensors (views of two flat buffers, as the training engine of this package has
        # them); the moments come from a checkpoint in torch.optim.AdamW's layout
        from mmearth_train_amd.optim import AdamW
        params = [torch.nn.Parameter(s["p"][o:o + n].view(shape)) for o, shape, n in s["places"]]
        plain = [i for i, (o, _, _) in enumerate(s["places"]) if o < s["cut"]]
        decayed = [i for i, (o, _, _) in enumerate(s["places"]) if o >= s["cut"]]
        groups = [{"params": [params[i] for i in plain], "weight_decay": 0.0}, {"params": [params[i] for i in decayed], "weight_decay": DECAY}]
        groups = [q for q in groups if q["params"]]
        opt = AdamW(groups, lr=LR, betas=(BETA1, BETA2), eps=EPS, state_bits=32 if case["op"] == "adamw32" else 8, max_norm=case["clip"] or None)
        there = opt.state_dict()
        there["state"] = {i: {"step": torch.tensor(float(STEPS_DONE)), "exp_avg": s["m"][o:o + n].view(shape), "exp_avg_sq": s["v"][o:o + n].view(shape)}
                          for i, (o, shape, n) in enumerate(s["places"])}
        opt.load_state_dict(there)
        for p, (o, shape, n) in zip(params, s["places"]):
            p.grad = s["g"][o:o + n].view(shape)
        return {"op": case["op"], "clip": case["clip"], "opt": opt, "p": s["p"], "g": s["g"]}
    if case["op"] == "adamw8":
        s["km"], s["kv"], s["sm"], s["sv"] = _to_codes(s.pop("m").double().view(-1, BLOCK), s.pop("v").double().view(-1, BLOCK))
    return s


# ------------------------------------------------------------------------------------------------------------ plain forms

def _update(p, m, v, t, decay):
    """p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps), in the moments' type."""
    return p * (1.0 - LR * decay) - LR / (1.0 - BETA1 ** t) * m / (v.sqrt() / math.sqrt(1.0 - BETA2 ** t) + EPS)


def _clipped(g, clip):
    """The gradients times min(1, clip / (norm + 1e-6)); norm and factor from a 64-bit sum."""
    if not clip:
        return g, None
    norm = g.double().square().sum().sqrt()
    return g * (clip / (norm + 1e-6)).clamp(max=1.0).float(), norm.float()


def _adamw32_plain(s):
    s["t"] += 1
    g, norm = _clipped(s["g"].float(), s["clip"])
    s["m"].copy_(BETA1 * s["m"] + (1.0 - BETA1) * g)
    s["v"].copy_(BETA2 * s["v"] + (1.0 - BETA2) * g * g)
    c, p = s["cut"], s["p"].float()
    s["p"][:c] = _update(p[:c], s["m"][:c], s["v"][:c], s["t"], 0.0).to(s["p"].dtype)
    s["p"][c:] = _update(p[c:], s["m"][c:], s["v"][c:], s["t"], DECAY).to(s["p"].dtype)
    return {"p": s["p"], "exp_avg": s["m"], "exp_avg_sq": s["v"]} | ({} if norm is None else {"norm": norm})


def _adamw8_plain(s):
    # in 64 bits up to the codes: a code is decided by which side of a border its value lies on
    s["t"] += 1
    g, norm = _clipped(s["g"].double(), s["clip"])
    m, v = _from_codes(s["km"], s["kv"], s["sm"], s["sv"])
    g = g.view(-1, BLOCK)
    m = BETA1 * m + (1.0 - BETA1) * g
    v = BETA2 * v + (1.0 - BETA2) * g * g
    s["km"], s["kv"], s["sm"], s["sv"] = _to_codes(m, v)
    c, p, m, v = s["cut"], s["p"].float(), m.float().view(-1), v.float().view(-1)
    s["p"][:c] = _update(p[:c], m[:c], v[:c], s["t"], 0.0).to(s["p"].dtype)
    s["p"][c:] = _update(p[c:], m[c:], v[c:], s["t"], DECAY).to(s["p"].dtype)
    m, v = _from_codes(s["km"], s["kv"], s["sm"], s["sv"])
    return {"p": s["p"], "exp_avg": m.float().view(-1), "exp_avg_sq": v.float().view(-1)} | ({} if norm is None else {"norm": norm})


def _int8_plain(s):
    x = s["x"].double()                                   # 64 bits decide which side of a half a code's value lies on
    a = x.abs().amax(1, keepdim=True)
    q = torch.round(x * 127.0 / a.clamp(min=1e-300)).float()
    y = (q @ s["q"].float().t()) * (a / 127.0).float() * s["sw"]
    return (y if s["b"] is None else y + s["b"]).to(s["x"].dtype)


def run(s):
    if own:
        if s["op"] == "int8":
            from mmearth_train_amd.int8 import linear_int8
            return linear_int8(s["x"], s["w"])
        s["opt"].step()
        m, v = s["opt"].flat_moments()
        return {"p": s["p"], "exp_avg": m, "exp_avg_sq": v} | ({"norm": s["opt"].grad_norm} if s["clip"] else {})
    return {"adamw32": _adamw32_plain, "adamw8": _adamw8_plain, "int8": _int8_plain}[s["op"]](s)


# ---------------------------------------------------------------------------------------------------------- work and exact

def work(case):
    size = {"fp32": 4, "bf16": 2, "fp16": 2}[case["dtype"]]
    if case["op"] == "int8":
        m, k, n = case["m"], case["k"], case["n"]
        return {"bytes": m * k * size + n * k + 4 * n * (2 if case["bias"] else 1) + m * n * size, "flops": 2 * m * k * n}
    elements = sum(math.prod(shape) for shape, _ in _shapes(case))
    # parameters in and out, gradients in, moments in and out; the 8-bit form has one byte and a 256th of a scale each, and its values read back
    moments = 16 if case["op"] == "adamw32" else 4 + 16 / BLOCK + 8
    return {"bytes": int(elements * (3 * size + moments)), "flops": 15 * elements}


def _exact_adamw(case, seed):
    s = _adamw_inputs(case, seed)
    t, pad = STEPS_DONE + 1, torch.arange(s["p"].numel(), device="cuda") >= s["cut"]
    grad = s["g"].double()
    out = {}
    if case["clip"]:
        total = torch.linalg.vector_norm(grad)
        out["norm"] = total
        grad = grad * min(1.0, float(torch.tensor(case["clip"], dtype=torch.float64) / (total.cpu() + 1e-6)))
    m, v = s["m"].double(), s["v"].double()
    if case["op"] == "adamw8":
        m, v = _exact_rounded(m, v)
    m = torch.lerp(grad, m, BETA1)
    v = torch.lerp(grad.pow(2), v, BETA2)
    mhat, vhat = m / (1 - BETA1 ** t), v / (1 - BETA2 ** t)
    p = s["p"].double()
    p = p - LR * DECAY * p * pad - LR * mhat / (vhat.pow(0.5) + EPS)
    if case["op"] == "adamw8":
        m, v = _exact_rounded(m, v)
    return out | {"p": p, "exp_avg": m, "exp_avg_sq": v}


def _exact_rounded(m, v):
    """The values that the 8-bit codes of m and v stand for: m to the nearest border-separated square step of 127, v to the fourth-power step of 255."""
    top = m.view(-1, BLOCK).abs().amax(1).float().double().repeat_interleave(BLOCK)
    step = torch.nan_to_num(m.abs() / top).pow(0.5).mul(127.0).add(0.5).floor().clamp(0, 127)
    mr = torch.copysign((step / 127.0).pow(2) * top, m)
    top = v.view(-1, BLOCK).amax(1).float().double().repeat_interleave(BLOCK)
    step = torch.nan_to_num(v / top).pow(0.25).mul(255.0).add(0.5).floor().clamp(0, 255)
    step = torch.maximum(step, (v > 0).double())
    return mr, (step / 255.0).pow(4) * top


def _exact_int8(case, seed):
    s = _int8_inputs(case, seed)
    codes = lambda a: (torch.round(127.0 * a.double() / a.double().abs().amax(-1, keepdim=True)), a.double().abs().amax(-1) / 127.0)  # noqa: E731
    (qx, sx), (qw, sw) = codes(s["x"]), codes(s["w"])
    y = torch.matmul(qx, qw.transpose(0, 1).contiguous()) * torch.outer(sx, sw)
    return y if s["b"] is None else y + s["b"].double()


def exact(case, seed):
    return _exact_int8(case, seed) if case["op"] == "int8" else _exact_adamw(case, seed)

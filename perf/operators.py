"""Measured cases of the many-tensor optimizer operators.

``run`` makes one pass: an AdamW step over many tensors with 32-bit or 8-bit
moments (optionally clipping by the global gradient norm, optionally with
32-bit master copies of 16-bit parameters), the clipping of a set of gradients
on its own, or a checkpoint's moments taken into the 8-bit form and read back.
With ``own`` false the same is computed from elementary torch operations on the
flat buffers that the tensors are views of.
"""
import math
import random

import torch

own = False

BLOCK = 256           # elements that share an exponent in the 8-bit form
DITHER_I, DITHER_T = 0x9E3779B1, 0x6A09E667
M_TOP, V_TOP = 15, 31  # highest exponent field of the 4- and the 5-bit exponent
E_MIN = 64            # lowest block exponent (an fp32 exponent field)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
POOL_LR = {"means": 1.0, "scales": 2.0, "quats": 1.0, "opacities": 5.0, "sh0": 1.0, "shN": 0.05}
BETAS = (0.9, 0.999)


def listed():
    pool = {"op": "adamw", "kind": "pool", "p": "f32", "g": "f32", "master": False, "clip": False}
    net = {"op": "adamw", "kind": "net", "clip": True}
    return [
        # the six tensors of a 3,000-point scene: launch latency is all there is
        {"name": "step32 tiny scene", **pool, "bits": 32, "n": 3000, "degree": 0},
        # a 1M-Gaussian outdoor scene with degree-3 colours: 59M parameters
        {"name": "step32 outdoor scene", **pool, "bits": 32, "n": 1_000_000, "degree": 3},
        # an appearance network beside the scene: bf16 weights with 32-bit masters, clipped
        {"name": "step32 bf16 network", **net, "bits": 32, "p": "bf16", "g": "bf16", "master": True, "n": 96,
         "most": 1_500_000},
        # the same scenes with 8-bit moments
        {"name": "step8 tiny scene", **pool, "bits": 8, "n": 3000, "degree": 0},
        {"name": "step8 outdoor scene", **pool, "bits": 8, "n": 1_000_000, "degree": 3},
        # the whole 4M-slot pool of the densification workload, gradients summed over GPUs in bf16
        {"name": "step8 pool of 4M slots", **pool, "g": "bf16", "bits": 8, "n": 4_000_000, "degree": 3},
        # per-image embeddings, pose deltas and small layers in fp16: many ragged tensors, clipped
        {"name": "step8 ragged fp16", **net, "bits": 8, "p": "f16", "g": "f16", "master": False, "n": 160,
         "most": 70_000},
        # clipping on its own, before an optimizer that does not clip
        {"name": "clip tiny scene", "op": "clip", "kind": "pool", "g": "f32", "n": 3000, "degree": 0},
        {"name": "clip outdoor scene", "op": "clip", "kind": "pool", "g": "f32", "n": 1_000_000, "degree": 3},
        {"name": "clip ragged bf16", "op": "clip", "kind": "net", "g": "bf16", "n": 220, "most": 130_000},
        # a 32-bit checkpoint's moments resumed with 8-bit ones and read back
        {"name": "moments ragged", "op": "moments", "kind": "net", "n": 60, "most": 20_000},
        {"name": "moments outdoor scene", "op": "moments", "kind": "pool", "n": 1_000_000, "degree": 3},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    case = {"op": rng.choice(["adamw", "adamw", "adamw", "clip", "moments"]), "kind": rng.choice(["pool", "net"])}
    if case["kind"] == "pool":
        case.update(n=log(1, 2_000_000), degree=rng.choice([0, 1, 2, 3]))
    else:
        case.update(n=log(1, 240), most=log(1, 500_000))
    if case["op"] == "adamw":
        case["p"] = rng.choice(["f32", "f32", "bf16", "f16"])
        case["g"] = rng.choice(["f32", case["p"], "bf16"])
        case["master"] = case["p"] != "f32" and rng.random() < 0.5
        case["bits"] = rng.choice([8, 32])
        case["clip"] = rng.random() < 0.5
    elif case["op"] == "clip":
        case["g"] = rng.choice(["f32", "bf16", "f16"])
    return case


def shapes(case):
    """Name -> shape of the case's tensors."""
    n = case["n"]
    if case["kind"] == "pool":
        dims = {"means": 3, "scales": 3, "quats": 4, "opacities": 1, "sh0": 3, "shN": 3 * ((case["degree"] + 1) ** 2 - 1)}
        return {k: (n, d) for k, d in dims.items() if d}
    rng = random.Random(1000 * n + case["most"])
    sizes = [int(round(math.exp(rng.uniform(0.0, math.log(case["most"]))))) for _ in range(n)]
    sizes[rng.randrange(n)] = case["most"]
    return {"layer%03d" % i: (s,) for i, s in enumerate(sizes)}


def padded(case):
    """Per tensor its elements and the elements it takes in a flat buffer (whole blocks)."""
    sizes = [math.prod(s) for s in shapes(case).values()]
    return sizes, [-(-s // BLOCK) * BLOCK for s in sizes]


def hyper(case):
    """lr, eps, weight decay, and per tensor the factors of the first and the last."""
    names = list(shapes(case))
    if case["kind"] == "pool":
        return 1.6e-4, 1e-15, 0.01, {k: POOL_LR[k] for k in names}, {k: 0.0 if k == "opacities" else 1.0 for k in names}
    return 1e-3, 1e-8, 0.05, {k: 1.0 for k in names}, {k: float(i % 2) for i, k in enumerate(names)}


def views(flat, case):
    sizes, room = padded(case)
    starts = [sum(room[:i]) for i in range(len(room))]
    return {k: flat[a:a + n].view(s) for (k, s), n, a in zip(shapes(case).items(), sizes, starts)}


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(dev).manual_seed(seed)
    sizes, room = padded(case)
    total = sum(room)
    reps = torch.tensor(room, device=dev)
    local = torch.arange(total, device=dev) - (reps.cumsum(0) - reps).repeat_interleave(reps, output_size=total)
    live = local < torch.tensor(sizes, device=dev).repeat_interleave(reps, output_size=total)

    def normal():
        return torch.randn(total, generator=gen, device=dev)

    # gradient sizes spread over decades between elements; in a scene most rows are unseen in a view
    size = torch.exp(1.5 * normal() - 9.0)
    g = size * normal()
    if case["kind"] == "pool":
        g *= (torch.rand(total, generator=gen, device=dev) < 0.5)
    g = torch.where(live, g, 0.0).to(TYPES[case.get("g", "f32")])
    s = {"case": case, "g": g, "room": reps, "t": 100 + seed % 50}
    # a bound that clips
    s["max_norm"] = 0.37 * float(g.double().square().sum().sqrt()) if case["op"] == "clip" or case.get("clip") else None
    if case["op"] == "clip":
        s["out"] = torch.zeros_like(g)
        s["grads"], s["outs"] = views(g, case), views(s["out"], case)
        return s
    m = torch.where(live, 0.4 * size * normal(), 0.0)
    v = torch.where(live, (size * (0.6 + 0.8 * torch.rand(total, generator=gen, device=dev))).square(), 0.0)
    del size, g
    if case["op"] == "moments":
        s["m"], s["v"] = m, v
        s["local"] = local
        s["md"], s["vd"] = views(m, case), views(v, case)
        p = torch.zeros(total, device=dev)
        if own:
            from mlx_gsplat_b200 import FusedAdamW
            s["opt"] = FusedAdamW(views(p, case), state_bits=8)
        return s
    lr, eps, wd, lr_scales, decay_scales = hyper(case)
    p = torch.where(live, normal(), 0.0)
    s["p"] = p.to(TYPES[case["p"]])
    if case["master"]:
        s["master"] = s["p"].float()
    if case["bits"] == 8:
        s["local"] = local
        um, uv = dither(local, s["t"])
        s["mc"], s["me"] = encode(m, um, M_TOP, True)
        s["vc"], s["ve"] = encode(v, uv, V_TOP, False)
        m, v = decode(s["mc"], s["me"], M_TOP, True), decode(s["vc"], s["ve"], V_TOP, False)
    else:
        s["m"], s["v"] = m, v
    s["lr_scale"] = torch.tensor(list(lr_scales.values()), dtype=torch.float64, device=dev)
    s["decay_scale"] = torch.tensor(list(decay_scales.values()), dtype=torch.float64, device=dev)
    s["grads"] = views(s["g"], case)
    if own:
        from mlx_gsplat_b200 import FusedAdamW
        s["opt"] = FusedAdamW(views(s["p"], case), lr=lr, betas=BETAS, eps=eps, weight_decay=wd, lr_scales=lr_scales,
                              decay_scales=decay_scales, state_bits=case["bits"], master_weights=case["master"],
                              max_norm=s["max_norm"])
        s["opt"].load_moments(views(m, case), views(v, case), t=s["t"])
        for k in ("m", "v", "mc", "me", "vc", "ve", "local", "master"):
            s.pop(k, None)
    return s


# ---------------------------------------------------------------- the plain form
def dither(local, t):
    """20-bit offsets of the two moments' roundings, from the element's place in its tensor and the step."""
    w = (local * DITHER_I + t * DITHER_T) & 0xFFFFFFFF
    return w >> 12, (w ^ 0xFFFFFFFF) >> 12


def encode(x, u, top, signed):
    """8-bit codes (exponent field over 3 mantissa bits) and one exponent byte for 256 elements: the magnitude's
    fp32 bits plus the offset, cut to 3 mantissa bits; below the lowest exponent a fixed step."""
    a = x.abs().view(torch.int32).long()
    r = a + u
    e = (r.view(-1, BLOCK).amax(1) >> 23).clamp(E_MIN, 255)
    eb = e.repeat_interleave(BLOCK, output_size=x.numel())
    normal = (r >> 20) - ((eb - top) << 3)
    low = eb - (top - 1)  # exponent field of the lowest value with a whole mantissa
    fixed = torch.floor(x.abs().double() * torch.exp2((150 - low).double())).clamp(max=2.0 ** 40).long()
    code = torch.where(a >= (low << 23), normal, (fixed + u) >> 20)
    if signed:
        code = code | ((x < 0).long() << 7)
    else:
        code = torch.where((x > 0) & (code == 0), 1, code)
    return code.to(torch.uint8), e.to(torch.uint8)


def decode(code, e, top, signed):
    q = code.int()
    field = (q & 127 if signed else q) << 20
    x = field.view(torch.float32) * 2.0 ** (127 - top)
    x = x * (e.int() << 23).view(torch.float32).repeat_interleave(BLOCK, output_size=q.numel())
    return torch.where(q > 127, -x, x) if signed else x


def plain_adamw(s):
    case = s["case"]
    lr, eps, wd, _, _ = hyper(case)
    b1, b2 = BETAS
    total = s["g"].numel()
    out = {}
    scale = torch.ones((), dtype=torch.float64, device=s["g"].device)
    if case["clip"]:
        norm = s["g"].double().square().sum().sqrt()
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, scale)
        out["norm"] = norm.float()
    s["t"] += 1
    t = s["t"]
    bc1, bc2 = 1.0 - b1 ** t, 1.0 - b2 ** t
    step = ((lr / bc1) * s["lr_scale"]).float().repeat_interleave(s["room"], output_size=total)
    keep = (1.0 - lr * s["lr_scale"] * wd * s["decay_scale"]).float().repeat_interleave(s["room"], output_size=total)
    g = s["g"].float() * scale.float()
    if case["bits"] == 8:
        m, v = decode(s["mc"], s["me"], M_TOP, True), decode(s["vc"], s["ve"], V_TOP, False)
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    p = s["master"] if case["master"] else s["p"].float()
    p = p * keep - step * (m / (v.sqrt() * (1.0 / math.sqrt(bc2)) + eps))
    if case["master"]:
        s["master"] = out["master"] = p
    s["p"] = out["p"] = p.to(s["p"].dtype)
    if case["bits"] == 8:
        um, uv = dither(s["local"], t)
        s["mc"], s["me"] = encode(m, um, M_TOP, True)
        s["vc"], s["ve"] = encode(v, uv, V_TOP, False)
        m = decode(s["mc"], s["me"], M_TOP, True).bfloat16()
        v = decode(s["vc"], s["ve"], V_TOP, False).bfloat16()
    else:
        s["m"], s["v"] = m, v
    return {**out, "m": m, "v": v}


def run(s):
    case = s["case"]
    if own:
        from mlx_gsplat_b200 import clip_gradients
        if case["op"] == "clip":
            norm = clip_gradients(s["grads"], s["max_norm"], out=s["outs"])
            return {"norm": norm, "g": s["out"]}
        opt = s["opt"]
        if case["op"] == "moments":
            opt.load_moments(s["md"], s["vd"], t=s["t"])
            m, v = opt.moment_slabs(torch.bfloat16)
            return {"m": m, "v": v}
        norm = opt.step(s["grads"])
        # the 8-bit forms' values have at most 4 significant bits: bf16 holds them exactly
        m, v = opt.moment_slabs(torch.bfloat16 if case["bits"] == 8 else torch.float32)
        out = {"p": s["p"], "m": m, "v": v}
        if case["master"]:
            out["master"] = opt.master_slab
        if case["clip"]:
            out["norm"] = norm
        return out
    if case["op"] == "adamw":
        return plain_adamw(s)
    if case["op"] == "clip":
        norm = s["g"].double().square().sum().sqrt()
        scale = torch.where(norm > s["max_norm"], s["max_norm"] / norm, 1.0)
        return {"norm": norm.float(), "g": (s["g"].float() * scale.float()).to(s["g"].dtype)}
    um, uv = dither(s["local"], s["t"])
    mc, me = encode(s["m"], um, M_TOP, True)
    vc, ve = encode(s["v"], uv, V_TOP, False)
    return {"m": decode(mc, me, M_TOP, True).bfloat16(), "v": decode(vc, ve, V_TOP, False).bfloat16()}


def work(case):
    n = sum(math.prod(s) for s in shapes(case).values())
    width = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] == "clip":
        return {"bytes": 2 * width[case["g"]] * n, "flops": 3 * n}
    if case["op"] == "moments":
        return {"bytes": (8 + 2 + 2 / BLOCK + 4) * n, "flops": 20 * n}
    p = width[case["p"]] + 8 if case["master"] else 2 * width[case["p"]]
    state = 16 if case["bits"] == 32 else 4 + 4 / BLOCK + 4
    return {"bytes": (p + width[case["g"]] + state) * n, "flops": (20 if case["bits"] == 32 else 45) * n}


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    g = s["g"].double()
    norm = torch.linalg.vector_norm(g)
    if case["op"] == "clip":
        return {"norm": norm, "g": g * min(1.0, s["max_norm"] / float(norm))}
    if case["op"] == "moments":
        return {"m": nested(s["m"].double(), s["local"], s["t"], 18, False),
                "v": nested(s["v"].double(), s["local"], s["t"], 34, True)}
    lr, eps, wd, lr_scales, decay_scales = hyper(case)
    b1, b2 = BETAS
    t = s["t"] + 1
    if case["clip"]:
        g = g * min(1.0, s["max_norm"] / float(norm))
    if case["bits"] == 8:
        m, v = decode(s["mc"], s["me"], M_TOP, True).double(), decode(s["vc"], s["ve"], V_TOP, False).double()
    else:
        m, v = s["m"].double(), s["v"].double()
    m = torch.lerp(g, m, b1)
    v = torch.lerp(g ** 2, v, b2)
    p = s["p"].double()
    rate = torch.tensor([lr * x for x in lr_scales.values()], dtype=torch.float64, device=g.device)
    fade = torch.tensor([wd * x for x in decay_scales.values()], dtype=torch.float64, device=g.device)
    rate, fade = rate.repeat_interleave(s["room"]), fade.repeat_interleave(s["room"])
    direction = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    p = p - rate * (fade * p + direction)
    out = {"p": p, "master": p if case["master"] else None, "norm": norm if case["clip"] else None}
    if case["bits"] == 8:
        m, v = nested(m, s["local"], t, 18, False), nested(v, s["local"], t, 34, True)
    return {**{k: x for k, x in out.items() if x is not None}, "m": m, "v": v}


def nested(x, local, t, span, positive):
    """The values that the 8-bit form stands for: multiples of an eighth of x's binade, none finer than 2^-span times
    the binade of the block's top, reached from x by adding a fraction of the step and cutting."""
    w = (local * DITHER_I + t * DITHER_T) % 2 ** 32
    u = (w if not positive else 2 ** 32 - 1 - w).div(4096, rounding_mode="floor").double() / 2 ** 20
    a = x.abs()

    def cut(step):
        return step * torch.floor(a / step + u)

    own_step = torch.exp2(torch.frexp(a.clamp(min=1e-300)).exponent.double() - 4)
    top = torch.frexp(cut(own_step).view(-1, BLOCK).amax(1)).exponent.double() - 1
    top = top.clamp(min=E_MIN - 127).repeat_interleave(BLOCK)
    # the lowest whole binade lies `span` - 4 below the top's, and its step three more below it
    floor_step = torch.exp2(top - span + 1)
    step = torch.maximum(own_step, floor_step)
    y = cut(step)
    if positive:
        y = torch.where((a > 0) & (y == 0), step, y)
    return torch.copysign(y, x)

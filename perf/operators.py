"""The sequence operators and their plain forms: a gated linear recurrence (over whole sequences, with its gradients, and for one step) and an AdamW step over many tensors.

`own` chooses between the framework's kernels and elementary torch operations in 32 bits (64 for the squared norm of all gradients)."""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256              # elements that share a scale of 8-bit moments; every tensor starts at a multiple of it in the flat moments
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one step of every env of a recurrent rollout: 2048 envs, 128 units, some of them at an episode's start
        {"name": "step 2048x128 f32", "op": "step", "B": 2048, "H": 128, "type": "f32", "gate": True, "reset": True},
        # a step of a few robots that are evaluated at once, half-precision activations
        {"name": "step 64x256 bf16", "op": "step", "B": 64, "H": 256, "type": "bf16", "gate": False, "reset": False},
        # values over a stored rollout of whole episodes: no gradient wanted
        {"name": "scan 400x1024x128 f32", "op": "scan", "T": 400, "B": 1024, "H": 128, "type": "f32", "gate": False, "reset": True, "lens": False, "carry": False},
        # one very long recording of a few robots, read through once
        {"name": "scan 16384x4x256 bf16", "op": "scan", "T": 16384, "B": 4, "H": 256, "type": "bf16", "gate": True, "reset": False, "lens": False, "carry": True},
        # the padded minibatch of whole trajectories of the recurrent update: 1024 trajectories of up to 400 steps
        {"name": "train 400x1024x128 f32", "op": "train", "T": 400, "B": 1024, "H": 128, "type": "f32", "gate": True, "reset": False, "lens": True, "carry": False},
        # a short rollout of many envs with restarts inside and the state carried in
        {"name": "train 32x4096x256 bf16", "op": "train", "T": 32, "B": 4096, "H": 256, "type": "bf16", "gate": False, "reset": True, "lens": False, "carry": True},
        # backpropagation through one long trajectory
        {"name": "train 65536x1x128 f32", "op": "train", "T": 65536, "B": 1, "H": 128, "type": "f32", "gate": False, "reset": True, "lens": False, "carry": True},
        # odd sizes all over
        {"name": "train 333x37x100 f16", "op": "train", "T": 333, "B": 37, "H": 100, "type": "f16", "gate": True, "reset": True, "lens": True, "carry": True},
        # the recurrent actor and critic, two cells of 128 units each: an optimiser step of the PPO update
        {"name": "adamw recurrent nets 32", "op": "adamw", "net": "recurrent", "bits": 32, "grad": "f32", "clip": True},
        # many small tensors of odd sizes, moments in 8 bits
        {"name": "adamw 200 tensors 8", "op": "adamw", "net": "odd", "tensors": 200, "elements": 1500000, "bits": 8, "grad": "f32", "clip": False},
        # a large network: 15 layers of width 2048
        {"name": "adamw 15x2048^2 32", "op": "adamw", "net": "dense", "width": 2048, "layers": 15, "bits": 32, "grad": "f32", "clip": True},
        # the same with moments in 8 bits and gradients of a half-precision backward pass
        {"name": "adamw 15x2048^2 8", "op": "adamw", "net": "dense", "width": 2048, "layers": 15, "bits": 8, "grad": "bf16", "clip": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["step", "scan", "train", "train", "adamw", "adamw"])
    if op == "adamw":
        case = {"op": op, "bits": rng.choice([8, 32]), "grad": rng.choice(["f32", "f32", "bf16", "f16"]), "clip": rng.random() < 0.7}
        if rng.random() < 0.5:
            n = _log(rng, 1, 300)
            return {**case, "net": "odd", "tensors": n, "elements": _log(rng, 20000 + 100 * n, 3e7)}
        return {**case, "net": "dense", "width": _log(rng, 65, 2047), "layers": _log(rng, 1, 15)}
    case = {"op": op, "type": rng.choice(["f32", "f32", "bf16", "f16"]), "gate": rng.random() < 0.5, "reset": rng.random() < 0.5}
    case["H"] = _log(rng, 8, 1024) if rng.random() < 0.5 else 8 * _log(rng, 1, 128)
    if op == "step":
        return {**case, "B": _log(rng, 1, 8192)}
    case["T"] = _log(rng, 2, 65536)
    room = 4e7 / (case["T"] * case["H"])
    case["B"] = _log(rng, 1, max(1.0, min(4096.0, room)))
    if room < 1:
        case["T"] = int(4e7 / case["H"])
    return {**case, "lens": rng.random() < 0.4, "carry": rng.random() < 0.5}


def _shapes(case):
    """The tensors of a network, in the order of its flat parameter block, and the weight decay of each (none for what has one axis)."""
    if case["net"] == "recurrent":           # two LSTM cells of 128 on 50 inputs and a linear head: an actor with 10 outputs, a critic with 1
        shapes = []
        for out in (10, 1):
            for i in (50, 128):
                shapes += [(512, i), (512, 128), (512,), (512,)]
            shapes += [(out, 128), (out,)]
    elif case["net"] == "dense":
        w = case["width"]
        shapes = [s for _ in range(case["layers"]) for s in ((w, w), (w,))]
    else:                                    # sizes that spread over a factor of 100
        r = random.Random(case["elements"])
        part = [math.exp(r.uniform(0.0, math.log(100.0))) for _ in range(case["tensors"])]
        shapes = [(max(1, int(case["elements"] * p / sum(part))),) if k % 3 else (max(1, int(case["elements"] * p / sum(part) / 7)), 7) for k, p in enumerate(part)]
    return shapes, [0.01 if len(s) > 1 else 0.0 for s in shapes]


HYPER = {"lr": 1e-4, "betas": (0.9, 0.999), "eps": 1e-5}
MAX_NORM = 0.05                              # the PPO update's own
SEED = 7                                     # of the moments' rounding


# ---------------------------------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *s, dtype=torch.float32: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32).to(dtype)  # noqa: E731
    if case["op"] == "adamw":
        return _prepare_adamw(case, g)
    B, H, t = case["B"], case["H"], TYPES[case["type"]]
    lead = (B,) if case["op"] == "step" else (case["T"], B)
    # the gates' logits and the candidates come out of one product, side by side in its rows; forget gates of trained recurrences lean to keeping
    k = 3 if case["gate"] else 2
    proj = rand(*lead, k * H)
    proj[..., :H] = proj[..., :H] * 1.5 + 2.0
    proj = proj.to(t)
    s = {"case": case, "f": proj[..., :H], "x": proj[..., H:2 * H], "o": proj[..., 2 * H:] if case["gate"] else None, "reset": None, "lens": None, "h0": None}
    if case["op"] == "step":
        s["h"] = rand(B, H)
        if case["reset"]:
            s["reset"] = (torch.rand(B, generator=g, device=DEV) < 0.01).to(torch.uint8)
        return s
    T = case["T"]
    if case["carry"]:
        s["h0"] = rand(B, H)
    if case["reset"]:                        # an episode ends after 100 steps or so
        s["reset"] = (torch.rand(T, B, generator=g, device=DEV) < 0.01).to(torch.uint8)
    if case["lens"]:                         # trajectories of all lengths, the longest sets the padded length
        s["lens"] = torch.randint(1, T + 1, (B,), generator=g, device=DEV).to(torch.int32)
        s["lens"][seed % B] = T
    if case["op"] == "train":
        s["dy"] = rand(T, B, H, dtype=t)
        s["dh_last"] = rand(B, H) if case["carry"] else None
    return s


def _prepare_adamw(case, g):
    shapes, decay = _shapes(case)
    sizes = [math.prod(s) for s in shapes]
    total = sum(sizes)
    params = torch.randn(total, generator=g, device=DEV) * 0.05
    # gradients whose size differs from tensor to tensor, and some exact zeros (units that were never active)
    grads = torch.randn(total, generator=g, device=DEV) * 1e-2
    grads = torch.where(torch.rand(total, generator=g, device=DEV) < 0.02, torch.zeros_like(grads), grads)
    at, views, gviews = 0, [], []
    for k, (n, shape) in enumerate(zip(sizes, shapes)):
        grads[at:at + n] *= 10.0 ** (-(k % 4))
        views.append(params[at:at + n].view(shape))
        at += n
    grads = grads.to(TYPES[case["grad"]])
    at = 0
    for n, shape in zip(sizes, shapes):
        gviews.append(grads[at:at + n].view(shape))
        at += n
    s = {"case": case, "flat": params, "params": views, "grads": gviews, "decay": decay, "sizes": sizes}
    if own:                                  # the optimiser that a program keeps: it holds the moments
        from apex_amd import engine
        s["opt"] = engine.AdamW(views, weight_decay=decay, max_norm=MAX_NORM if case["clip"] else None, state_bits=case["bits"], seed=SEED, **HYPER)
    else:                                    # the same moments in the same places, and the step count
        padded = sum(-(-n // BLOCK) * BLOCK for n in sizes)
        at, rows = 0, []
        for n in sizes:
            rows.append(torch.arange(at, at + n, device=DEV))
            at += -(-n // BLOCK) * BLOCK
        z = lambda n, d: torch.zeros(n, dtype=d, device=DEV)  # noqa: E731
        s.update(t=0, where=torch.cat(rows), wd=torch.cat([torch.full((n,), w, device=DEV) for n, w in zip(sizes, decay)]))
        if case["bits"] == 32:
            s.update(m=z(padded, torch.float32), v=z(padded, torch.float32))
        else:
            s.update(mc=z(padded, torch.uint8), vc=z(padded, torch.uint8), ms=z(padded // BLOCK, torch.float32), vs=z(padded // BLOCK, torch.float32))
    return s


# ---------------------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        from apex_amd import engine
        if op == "step":
            y = engine.gated_scan_step(s["f"], s["x"], s["h"], o=s["o"], reset=s["reset"])
            return {"y": y, "h": s["h"]}
        opts = {"o": s.get("o"), "h0": s.get("h0"), "reset": s.get("reset"), "lens": s.get("lens")}
        if op == "scan":
            y, h = engine.gated_scan(s["f"], s["x"], **opts)
            return {"y": y, "h": h}
        if op == "train":
            y, h, save = engine.gated_scan(s["f"], s["x"], keep=True, **opts)
            df, dx, do, dh0 = engine.gated_scan_backward(s["f"], s["x"], s["dy"], save, dh_last=s["dh_last"], **opts)
            return _trained(s, y, h, df, dx, do, dh0)
        s["opt"].step(s["grads"])
        m, v = s["opt"].moments()
        return {"p": s["flat"], "m": m, "v": v}
    if op == "step":
        return _plain_step(s)
    if op == "adamw":
        return _plain_adamw(s)
    return _plain_scan(s, op == "train")


def _trained(s, y, h, df, dx, do, dh0):
    r = {"y": y, "h": h, "df": df, "dx": dx}
    if s["o"] is not None:
        r["do"] = do
    if s["h0"] is not None:
        r["dh0"] = dh0
    return r


def _plain_step(s):
    f, x, h = s["f"].float(), s["x"].float(), s["h"]
    p = h if s["reset"] is None else torch.where(s["reset"].bool()[:, None], 0.0, h)
    h.copy_(torch.sigmoid(f) * p + torch.sigmoid(-f) * x)
    y = h if s["o"] is None else h * torch.sigmoid(s["o"].float())
    return {"y": y.to(s["x"].dtype), "h": h}


def _doubling(a, b):
    """h_t = a_t h_{t-1} + b_t over the first axis, from zero: after k rounds a row holds the last 2^k steps."""
    d = 1
    while d < a.shape[0]:
        b = torch.cat([b[:d], torch.addcmul(b[d:], a[d:], b[:-d])])
        if 2 * d < a.shape[0]:
            a = torch.cat([a[:d], a[d:] * a[:-d]])
        d *= 2
    return b


def _plain_scan(s, train):
    t = s["x"].dtype
    f, x = s["f"].float(), s["x"].float()
    T, B, H = f.shape
    real = None
    if s["lens"] is not None:
        real = (torch.arange(T, device=f.device)[:, None] < s["lens"][None, :])[:, :, None]
    a, n = torch.sigmoid(f), torch.sigmoid(-f)
    keep = a if s["reset"] is None else torch.where(s["reset"].bool()[:, :, None], 0.0, a)      # what passes from a state to the next
    b = n * x
    if real is not None:
        keep, b = torch.where(real, keep, 1.0), torch.where(real, b, 0.0)
    start = torch.zeros(B, H, device=f.device) if s["h0"] is None else s["h0"]
    h = _doubling(keep, torch.cat([(b[0] + keep[0] * start)[None], b[1:]]))
    gate = None if s["o"] is None else torch.sigmoid(s["o"].float())
    y = h if gate is None else h * gate
    if real is not None:
        y = torch.where(real, y, 0.0)
    if not train:
        return {"y": y.to(t), "h": h[-1].clone()}
    dy = s["dy"].float()
    if real is not None:
        dy = torch.where(real, dy, 0.0)
    d = dy if gate is None else dy * gate
    if s["dh_last"] is not None:
        d = torch.cat([d[:-1], (d[-1] + s["dh_last"])[None]])
    # g_t = d_t + keep_{t+1} g_{t+1}: the same scan, from the end
    g = _doubling(torch.cat([torch.ones_like(keep[:1]), keep[1:].flip(0)]), d.flip(0)).flip(0)
    prev = torch.cat([start[None], h[:-1]])
    if s["reset"] is not None:
        prev = torch.where(s["reset"].bool()[:, :, None], 0.0, prev)
    df, dx = g * (prev - x) * a * n, g * n
    do = None if gate is None else dy * h * gate * torch.sigmoid(-s["o"].float())
    if real is not None:
        df, dx = torch.where(real, df, 0.0), torch.where(real, dx, 0.0)
    dh0 = keep[0] * g[0]
    return _trained(s, y.to(t), h[-1].clone(), df.to(t), dx.to(t), None if do is None else do.to(t), dh0)


def _mix(x):
    """32 mixed bits of 32 (in int64)."""
    x = x ^ (x >> 16)
    x = (x * 0x6A09E667) & M32
    x = x ^ (x >> 15)
    x = (x * 0xBB67AE85) & M32
    return x ^ (x >> 16)


def _noise(seed, t, at):
    """The 32 bits that round the moments of the elements `at` of the flat moments in step t."""
    one = lambda v: int(_mix(torch.tensor(v & M32, dtype=torch.int64)))  # noqa: E731
    key = one(one(seed) ^ one((seed >> 32) + 0x3C6EF373) ^ one(t + 0x54FF53A5))
    return _mix((at & M32) ^ key ^ (((at >> 32) * 0x3C6EF373) & M32))


def _decode(c, s, offset, signed):
    c = c.to(torch.int32)
    mag = c & 127 if signed else c
    v = torch.where(mag == 0, 0.0, ((mag + offset) << 20).view(torch.float32))
    v = (v.view(-1, BLOCK) * s[:, None]).view(-1)
    return torch.where(c > 127, -v, v) if signed else v


def _encode(w, bits, offset, signed):
    """8-bit codes and power-of-two scales of the values `w`; `bits` (16 of them) round each up or down so that its mean stays."""
    q = w.abs().view(-1, BLOCK)
    e = (q.max(1).values.view(torch.int32) >> 23).clamp(min=33)      # a scale of 2^-94 at least
    scale, inv = (e << 23).view(torch.float32), ((254 - e) << 23).view(torch.float32)
    q = (q * inv[:, None]).view(-1)
    least = (1 + 1 / 8) * 2.0 ** ((offset + 1) // 8 - 127)
    bits = bits << 4
    c = ((q.view(torch.int32) + bits) >> 20) - offset
    low = ((bits.to(torch.float32) * (least * 2.0 ** -20)) < q) if signed else q > 0      # v > 0 is never rounded to 0: it is divided by
    c = torch.where(q < least, low.to(torch.int32), c)
    if signed:
        c = torch.where((w < 0) & (c > 0), c + 128, c)
    return c.to(torch.uint8), scale


M_OFFSET, V_OFFSET = 904, 776                # codes (c + offset) << 20 are the bits of values up to 3.75, 1 + 3 / 8 bits of exponent and mantissa wide


def _plain_adamw(s):
    case = s["case"]
    (b1, b2), lr, eps = HYPER["betas"], HYPER["lr"], HYPER["eps"]
    g = torch.cat([x.reshape(-1) for x in s["grads"]]).float()
    if case["clip"]:
        total = g.double().square().sum().sqrt().float()
        g = g * torch.clamp(MAX_NORM / (total + 1e-6), max=1.0)
    s["t"] += 1
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m, v = _decode(s["mc"], s["ms"], M_OFFSET, True), _decode(s["vc"], s["vs"], V_OFFSET, False)
    full = torch.zeros_like(m)
    full[s["where"]] = g
    m = m * b1 + full * (1 - b1)
    v = v * b2 + (full * full) * (1 - b2)
    step = lr / (1 - b1 ** s["t"])
    denom = v.sqrt() * (1 / math.sqrt(1 - b2 ** s["t"])) + eps
    p = s["flat"]
    p.copy_(p * (1 - lr * s["wd"]) - step * (m / denom)[s["where"]])
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return {"p": p, "m": s["m"], "v": s["v"]}
    r = _noise(SEED, s["t"], torch.arange(m.numel(), device=m.device)).to(torch.int64)
    mc, ms = _encode(m, (r & 0xFFFF).to(torch.int32), M_OFFSET, True)
    vc, vs = _encode(v, (r >> 16).to(torch.int32), V_OFFSET, False)
    for k, x in (("mc", mc), ("vc", vc), ("ms", ms), ("vs", vs)):
        s[k].copy_(x)
    return {"p": p, "m": _decode(mc, ms, M_OFFSET, True).to(torch.bfloat16), "v": _decode(vc, vs, V_OFFSET, False).to(torch.bfloat16)}


# ---------------------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """The definitions step by step in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "adamw":
        return _exact_adamw(s)
    if case["op"] != "step" and case["T"] > 70000:
        return None
    f, x = s["f"].double(), s["x"].double()
    o = None if s["o"] is None else torch.sigmoid(s["o"].double())
    a, n = torch.sigmoid(f), torch.sigmoid(-f)
    if case["op"] == "step":
        p = s["h"].double()
        if s["reset"] is not None:
            p = p * (s["reset"] == 0)[:, None]
        h = a * p + n * x
        return {"y": h if o is None else h * o, "h": h}
    T, B, H = f.shape
    p = torch.zeros(B, H, dtype=torch.float64, device=DEV) if s["h0"] is None else s["h0"].double()
    go = torch.ones(T, B, 1, dtype=torch.bool, device=DEV) if s["reset"] is None else (s["reset"] == 0)[:, :, None]
    live = torch.ones(T, B, 1, dtype=torch.bool, device=DEV)
    if s["lens"] is not None:
        live = (torch.arange(T, device=DEV)[:, None] < s["lens"][None])[:, :, None]
    pa = torch.where(live, a * go, 1.0)      # what a step keeps of the state before it, and what it adds
    add = torch.where(live, n * x, 0.0)
    h = torch.empty(T, B, H, dtype=torch.float64, device=DEV)
    prev = torch.empty_like(h)
    for t in range(T):
        prev[t] = p
        p = torch.addcmul(add[t], pa[t], p, out=h[t])
    y = torch.where(live, h if o is None else h * o, 0.0)
    if case["op"] == "scan":
        return {"y": y, "h": h[-1]}
    dy = torch.where(live, s["dy"].double(), 0.0)
    c = torch.zeros(B, H, dtype=torch.float64, device=DEV) if s["dh_last"] is None else s["dh_last"].double()
    d = dy if o is None else dy * o
    g = torch.empty_like(h)
    for t in range(T - 1, -1, -1):
        torch.add(d[t], c, out=g[t])
        c = pa[t] * g[t]
    df = torch.where(live, g * (prev * go - x) * a * n, 0.0)
    dx = torch.where(live, g * n, 0.0)
    do = None if o is None else dy * h * o * (1 - o)
    return _trained(s, y, h[-1], df, dx, do, c)


def _exact_adamw(s):
    """The first step: moments start at zero.  Moments in 8 bits have no such value (they are rounded up or down by chance); the parameters have."""
    case = s["case"]
    (b1, b2), lr, eps = HYPER["betas"], HYPER["lr"], HYPER["eps"]
    g = torch.cat([x.reshape(-1) for x in s["grads"]]).double()
    if case["clip"]:
        g = g * min(1.0, MAX_NORM / (float(g.square().sum().sqrt()) + 1e-6))
    wd = torch.cat([torch.full((n,), w, device=DEV, dtype=torch.float64) for n, w in zip(s["sizes"], s["decay"])])
    m, v = (1 - b1) * g, (1 - b2) * g.square()
    p = s["flat"].double() * (1 - lr * wd) - lr * (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + eps)
    if case["bits"] == 8:
        return {"p": p, "m": None, "v": None}
    out, at, i = [torch.zeros(sum(-(-n // BLOCK) * BLOCK for n in s["sizes"]), dtype=torch.float64, device=DEV) for _ in range(2)], 0, 0
    for n in s["sizes"]:
        out[0][at:at + n], out[1][at:at + n] = m[i:i + n], v[i:i + n]
        at += -(-n // BLOCK) * BLOCK
        i += n
    return {"p": p, "m": out[0], "v": out[1]}


def work(case):
    if case["op"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case)[0])
        g = 4 if case["grad"] == "f32" else 2
        # gradient, parameter and both moments read, parameter and moments written; moments in 8 bits are read out as 16-bit values too
        return {"bytes": n * (g + 8 + (16 if case["bits"] == 32 else 4 + 4 + 16 / BLOCK)), "flops": n * 18}
    e, k = (4 if case["type"] == "f32" else 2), 3 if case["gate"] else 2
    if case["op"] == "step":
        n = case["B"] * case["H"]
        return {"bytes": n * (e * (k + 1) + 8), "flops": n * (8 + 4 * (k - 2))}
    n, rows = case["T"] * case["B"] * case["H"], case["T"] * case["B"]
    state = 4 * case["B"] * case["H"]
    bytes_ = n * e * (k + 1) + (rows if case["reset"] else 0) + state * (2 if case["carry"] else 1)
    if case["op"] == "scan":
        return {"bytes": bytes_, "flops": n * (8 + 4 * (k - 2))}
    # with the gradients: the outputs' gradient read, those of every input written; the inputs read once
    return {"bytes": bytes_ + n * e * (k + 1) + state * (2 if case["carry"] else 0), "flops": n * (24 + 10 * (k - 2))}

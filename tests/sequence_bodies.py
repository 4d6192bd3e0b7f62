"""Bodies of the sequence operators' tests: tests/test_gpu_sequence.py runs them on the GPU, tests/test_kernel_emulation_sequence.py on the kernels' sources compiled for the host.
The oracle is oracle/sequence.py in 64 bits.

Tolerances (u = 2^-24, half a step of f32 relative to the value; fast exponential and reciprocal: 2u each):
 * a gate's smaller half lo = e / (1 + e), e = 2^(-|f| log2 e): the argument's rounding moves e by |f| u, the exponential by 2u, the sum by u, the reciprocal by 2u, the product by u
   -> delta = (|f| + 6) u relative; the larger half is 1 - lo, u more.
 * h_t = a h + n x: the gates' error counts n delta (|h| + |x|) a step, sum and fma 2u |h| a step, and each fades with the memory: sum_k a^k n <= 1, sum_k a^k <= L =
   min(T, 1 / min n).  With M = max(|x|, |h0|): |error of h| <= M (2 delta + 4 u L).  Steps may be joined in chunks: the product of a chunk's a carries (chunk) u more, counted the
   same way: twice the bound.
 * g_t = d_t + a g: the same with G = max |g|: |error of g| <= 2 G (2 delta + 4 u L).
 * outputs: dx = n g, df = g (p - x) a n, do = d h s r with |a n|, |s r| <= 1/4, |p - x| <= 2 M; y = h s.  8 more roundings of u.  And half a step of the output's own type."""
import numpy as np
import torch

from oracle import sequence as Q

U = 2.0 ** -24
NP = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(t):
    return torch.finfo(NP[t]).eps / 2


def smallest(t):
    return 2.0 ** -25 if t == "f16" else 2.0 ** -134 if t == "bf16" else 0.0      # half a step of the numbers below the smallest normal one


def make(T, B, H, t, gate, reset, lens, carry, dev, seed, lean=1.0, layout="rows"):
    """inputs on the device, rounded to their type, and the same values in 64 bits"""
    r = np.random.RandomState(seed)
    k = 3 if gate else 2
    proj = r.randn(T, B, k * H) * 1.5
    proj[..., :H] = np.clip(proj[..., :H] + lean, -6, 6)
    proj = torch.tensor(proj, dtype=torch.float32).to(NP[t]).to(dev)
    parts = [proj[..., i * H:(i + 1) * H] for i in range(k)]
    if layout == "dense":
        parts = [p.contiguous() for p in parts]
    elif layout == "batch first":
        parts = [p.permute(1, 0, 2).contiguous().permute(1, 0, 2) for p in parts]
    elif layout == "shifted":      # rows that begin off every wide load's alignment
        parts = [torch.cat([p.new_zeros(T, B, 1), p], 2)[..., 1:] for p in parts]
    d = dict(f=parts[0], x=parts[1], o=parts[2] if gate else None,
             h0=torch.tensor(r.randn(B, H), dtype=torch.float32, device=dev) if carry else None,
             reset=torch.tensor((r.rand(T, B) < 0.15).astype(np.uint8), device=dev) if reset else None,
             lens=torch.tensor(r.randint(0, T + 1, B).astype(np.int32), device=dev) if lens else None)
    dy = torch.tensor(r.randn(T, B, H), dtype=torch.float32).to(NP[t]).to(dev)
    dh = torch.tensor(r.randn(B, H), dtype=torch.float32, device=dev) if carry else None
    return d, dy, dh


def f64(t):
    return None if t is None else t.detach().cpu().double().numpy() if t.is_floating_point() else t.detach().cpu().numpy()


def wide(d):
    return {k: f64(v) for k, v in d.items()}


def bounds(d, G=0.0, D=0.0):
    """(error of h, error of g, delta, M) of the derivation above; only what counts enters: padding may hold anything"""
    w = wide(d)
    T = w["f"].shape[0]
    live = np.ones(w["f"].shape[:2], bool) if w["lens"] is None else np.arange(T)[:, None] < w["lens"][None]
    f, x = w["f"][live], w["x"][live]
    if f.size == 0:
        return U, U, U, float(np.abs(w["h0"]).max()) if w["h0"] is not None and w["h0"].size else 0.0
    fin = np.abs(f[np.isfinite(f)])
    top = float(fin.max()) if fin.size else 0.0
    delta = (min(top, 100.0) + 6) * U
    L = min(T, 1 / max(float(Q.sigmoid(-f).min()), 1e-30))
    M = max(float(np.abs(x).max()), float(np.abs(w["h0"]).max()) if w["h0"] is not None else 0.0)
    return 2 * M * (2 * delta + 4 * U * L), 2 * G * (2 * delta + 4 * U * L), delta, M


def close(name, got, ref, tol, t):
    got = f64(got)
    assert np.isfinite(got).all(), (name, "not finite")
    err = np.abs(got - ref) - half_step(t) * np.abs(ref) * (1 + 1e-3) - smallest(t)
    assert got.shape == ref.shape and (got.size == 0 or err.max() <= tol), (name, float(err.max()), tol)


def check_scan(dev, T, B, H, t="f32", gate=False, reset=False, lens=False, carry=False, seed=0, lean=1.0, layout="rows", poison=False):
    from apex_amd import engine
    d, dy, dh = make(T, B, H, t, gate, reset, lens, carry, dev, seed, lean, layout)
    if poison:      # what must not count holds NaN and infinities: padding behind the ends, states in front of a reset
        assert lens and reset and carry
        n = d["lens"].cpu().numpy()
        for b in range(B):
            for k in ("f", "x", "o"):
                if d[k] is not None:
                    d[k][n[b]:, b] = [float("nan"), float("inf"), -float("inf"), torch.finfo(NP[t]).min][b % 4]
            dy[n[b]:, b] = float("nan")
            if n[b] > 0:
                d["reset"][0, b] = 1
                d["h0"][b] = float("nan") if b % 2 else float("inf")
    w = wide(d)
    keep_inputs = {k: v.clone() for k, v in d.items() if v is not None}
    y, hs, _, h = Q.gated_scan(**w)
    df, dx, do, dh0, G = Q.gated_scan_grad(dy=f64(dy), dh_last=f64(dh), **w)
    if poison:
        rows = n > 0
        d2 = dict(d, h0=torch.where(torch.tensor(rows, device=dev)[:, None], torch.zeros_like(d["h0"]), d["h0"]))
        eh, eg, delta, M = bounds(d2, G)
    else:
        eh, eg, delta, M = bounds(d, G)
    gy, gh, save = engine.gated_scan(**d, keep=True)
    y2, h2 = engine.gated_scan(**d)
    assert torch.equal(gy, y2) and torch.equal(gh, h2), "keep=True changes the outputs"
    close("y", gy, y, eh + 3 * U * M, t)
    close("h_last", gh, h, eh, "f32")
    out = engine.gated_scan_backward(d["f"], d["x"], dy, save, o=d["o"], h0=d["h0"], reset=d["reset"], lens=d["lens"], dh_last=dh)
    D = float(np.abs(f64(dy)[np.isfinite(f64(dy))]).max()) if dy.numel() else 0.0
    close("df", out[0], df, 0.25 * (2 * M * eg + G * 2 * eh) + 0.5 * M * G * (2 * delta + 8 * U), t)
    close("dx", out[1], dx, eg + G * (delta + 8 * U), t)
    if gate:
        close("do", out[2], do, 0.25 * D * eh + 0.25 * D * M * (2 * delta + 8 * U), t)
    else:
        assert out[2] is None
    if carry:
        fin = np.isfinite(dh0)
        assert fin.all()
        close("dh0", out[3], dh0, eg + 4 * U * max(G, 1.0), "f32")
    else:
        assert out[3] is None
    for k, v in keep_inputs.items():
        assert torch.equal(torch.nan_to_num(v.float()), torch.nan_to_num(d[k].float())), "input %s was written" % k
    return gy, gh, out


def check_step(dev, B, H, t="f32", gate=False, reset=False, seed=0, layout="rows", steps=3):
    """steps of gated_scan_step against one gated_scan over the same inputs in 64 bits"""
    from apex_amd import engine
    d, _, _ = make(steps, B, H, t, gate, reset, False, True, dev, seed, 1.0, layout)
    y, hs, _, _ = Q.gated_scan(**wide(d))
    eh, _, _, M = bounds(d)
    h = d["h0"].clone()
    for k in range(steps):
        got = engine.gated_scan_step(d["f"][k], d["x"][k], h, o=None if d["o"] is None else d["o"][k], reset=None if d["reset"] is None else d["reset"][k])
        close("y", got, y[k], eh + 3 * U * M, t)
        close("h", h, hs[k], eh, "f32")


# ------------------------------------------------------------------------------------------------ AdamW
def check_adamw(dev, shapes, bits=32, grad="f32", clip=None, steps=3, seed=0, wd=0.01, scale=1.0, flat=False, sizes=1.0):
    """steps of AdamW against the 64-bit oracle: 32-bit moments and the parameters to a few roundings, 8-bit moments code by code.
    Moments: g k (k: 4u), one product each and one sum -> (6 + 3 a step) u relative to the largest summand.  Parameters a step: 3u |p| for decay and difference, and of the
    update |step m / den| (m: (6 + 3 steps) u, square root of v, products, reciprocal: 12 u): (20 + 6 steps) u lr U with U the update's size, at most |m_hat| / eps."""
    from apex_amd import engine
    r = np.random.RandomState(seed)
    hyper = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-5)
    ns = [int(np.prod(s)) for s in shapes]
    if flat:
        block = torch.tensor(r.randn(sum(ns)) * 0.1, dtype=torch.float32).to(dev)
        ps, at = [], 0
        for s, n in zip(shapes, ns):
            ps.append(block[at:at + n].view(*s)); at += n
    else:
        ps = [torch.tensor(r.randn(*s) * 0.1, dtype=torch.float32).to(dev) for s in shapes]
    decay = [wd if k % 2 == 0 else 0.0 for k in range(len(shapes))]
    opt = engine.AdamW(ps, weight_decay=decay, max_norm=clip, state_bits=bits, seed=seed + (5 << 32), **hyper)
    where, total = Q.layout(ns)
    assert opt.elements == total
    P = [f64(p).reshape(-1) for p in ps]
    M, V = np.zeros(total), np.zeros(total)
    M32, V32 = np.zeros(total, np.float32), np.zeros(total, np.float32)
    spread = 0.0
    for t in range(1, steps + 1):
        g = [torch.tensor(r.randn(*s) * sizes * 10.0 ** (-(i % 4)) * (r.rand(*s) > 0.05), dtype=torch.float32).to(NP[grad]).to(dev) for i, s in enumerate(shapes)]
        opt.step(g, grad_scale=scale)
        g64 = [f64(x).reshape(-1) for x in g]
        norm, k = Q.clip_factor(g64, scale, clip)
        if clip:
            assert abs(float(opt.norm) - norm) <= 1e-12 * norm
        k32 = np.float32(scale) if not clip else np.float32(min(np.float32(1), np.float32(clip) / (np.float32(norm) + np.float32(1e-6)))) * np.float32(scale)
        full = np.zeros(total, np.float32)
        for i, n in enumerate(ns):
            full[where[i]:where[i] + n] = g64[i].astype(np.float32)
        if bits == 8:      # the moments before their rounding, from the codes that were there
            M, V = M32.astype(np.float64), V32.astype(np.float64)
        M32n, V32n = Q.moments_f32(full, M32, V32, hyper["betas"][0], hyper["betas"][1], k32)
        for i, n in enumerate(ns):
            s = slice(where[i], where[i] + n)
            p, M[s], V[s] = Q.adamw(P[i], g64[i], M[s], V[s], t, hyper["lr"], *hyper["betas"], hyper["eps"], decay[i], k)
            upd = np.abs(p - P[i]).max() if n else 0.0
            spread += 3 * U * (np.abs(P[i]).max() if n else 0.0) + (20 + 6 * t) * U * upd
            P[i] = p
            got = f64(ps[i]).reshape(-1)
            assert n == 0 or np.abs(got - p).max() <= spread, ("p", i, t, np.abs(got - p).max(), spread)
        if bits == 32:
            M32, V32 = M32n, V32n
            assert np.array_equal(opt.m.cpu().numpy(), M32) and np.array_equal(opt.v.cpu().numpy(), V32), "moments differ from separate f32 roundings"
            assert np.abs(M32 - M).max() <= (6 + 3 * t) * U * np.abs(M).max() and np.abs(V32 - V).max() <= (12 + 3 * t) * U * np.abs(V).max()
        else:
            rnd = Q.noise(seed + (5 << 32), t, np.arange(total))
            mc, ms = Q.encode(M32n, rnd & np.uint64(0xffff), Q.M_OFFSET, True)
            vc, vs = Q.encode(V32n, rnd >> np.uint64(16), Q.V_OFFSET, False)
            assert np.array_equal(opt.m_scale.cpu().numpy(), ms) and np.array_equal(opt.v_scale.cpu().numpy(), vs)
            assert np.array_equal(opt.m.cpu().numpy(), mc) and np.array_equal(opt.v.cpu().numpy(), vc)
            M32, V32 = Q.decode(mc, ms, Q.M_OFFSET, True).astype(np.float32), Q.decode(vc, vs, Q.V_OFFSET, False).astype(np.float32)
            # at most one step of the code (an eighth of the value's power of two) from the moment, below the range at most its smallest number
            sm, sv = np.repeat(ms, Q.BLOCK), np.repeat(vs, Q.BLOCK)
            assert (np.abs(M32 - M32n) <= np.maximum(np.abs(M32n) / 8, sm * 2.0 ** -13)).all() and (np.abs(V32 - V32n) <= np.maximum(V32n / 8, sv * 2.0 ** -29)).all()
            assert ((V32n > 0) == (V32 > 0)).all()
            got = opt.moments()
            assert np.array_equal(f64(got[0]), M32.astype(np.float64)) and np.array_equal(f64(got[1]), V32.astype(np.float64))
        assert int(opt.t) == t
    for v, p in zip(opt.views(opt.moments()[0]), ps):
        assert v.shape == p.shape
    return opt, ps


# ------------------------------------------------------------------------------------------------ what is not finite at steps that count
def check_not_finite(dev, T, B, H, t="f32", gate=False, lens=False, infinite=False, seed=0, at=None):
    """NaN (infinite: and infinities) in f, x, o and dy at steps that count, resets before and behind them: outputs are not finite exactly where the formulas' are, and right
    everywhere else.  An infinity may become a NaN between two resets (the steps are joined by products of gates), a NaN stays one.  at: the one sequence's (reset, step of a NaN gate)
    instead of places by chance.
    Tolerances are those of check_scan: M and L of the finite inputs; G with |dy|, without output gates and with every gate that is not a number open, which is no smaller than any
    finite |g|."""
    from apex_amd import engine
    d, dy, dh = make(T, B, H, t, gate, True, lens, True, dev, seed)
    r = np.random.RandomState(seed + 1)
    if at is not None:
        d["reset"].zero_(); d["reset"][at[0]] = 1
        d["f"][at[1]] = float("nan")
    else:
        bad = [float("nan")] + ([float("inf"), -float("inf")] if infinite else [])
        for x in (d["f"], d["x"], d["o"], dy):
            if x is None:
                continue
            for _ in range(max(2, T * B * H // 150)):
                x[r.randint(T), r.randint(B), r.randint(H)] = bad[r.randint(len(bad))]
    w, wy = wide(d), f64(dy)
    with np.errstate(invalid="ignore", over="ignore"):
        y, _, _, h = Q.gated_scan(**w)
        df, dx, do, dh0, _ = Q.gated_scan_grad(dy=wy, dh_last=f64(dh), **w)
    clean = {k: None if v is None else torch.tensor(np.where(np.isfinite(f64(v)), f64(v), {"f": 100.0}.get(k, 0.0)) if v.is_floating_point() else f64(v)) for k, v in d.items()}
    eh, _, delta, M = bounds(clean)
    size = np.abs(np.where(np.isfinite(wy), wy, 0.0))
    shut = dict(wide(clean), o=None, reset=None)
    G = Q.gated_scan_grad(dy=size, dh_last=np.abs(f64(dh)), **shut)[4]
    eg = bounds(clean, G)[1]
    D = float(size.max())
    gy, gh, save = engine.gated_scan(**d, keep=True)
    out = engine.gated_scan_backward(d["f"], d["x"], dy, save, o=d["o"], h0=d["h0"], reset=d["reset"], lens=d["lens"], dh_last=dh)
    seen = 0
    for name, got, ref, tol, kind in (("y", gy, y, eh + 3 * U * M, t), ("h_last", gh, h, eh, "f32"), ("df", out[0], df, 0.25 * (2 * M * eg + G * 2 * eh) + 0.5 * M * G * (2 * delta + 8 * U), t),
                                      ("dx", out[1], dx, eg + G * (delta + 8 * U), t), ("do", out[2], do, 0.25 * D * eh + 0.25 * D * M * (2 * delta + 8 * U), t), ("dh0", out[3], dh0, eg + 4 * U * max(G, 1.0), "f32")):
        if ref is None:
            assert got is None
            continue
        got, fine = f64(got), np.isfinite(ref)
        assert np.array_equal(np.isfinite(got), fine), (name, "not finite at", np.argwhere(np.isfinite(got) != fine)[:5].tolist())
        assert np.isnan(got[np.isnan(ref)]).all() or infinite, name
        err = np.abs(got[fine] - ref[fine]) - half_step(kind) * np.abs(ref[fine]) * (1 + 1e-3) - smallest(kind)
        assert err.size == 0 or err.max() <= tol, (name, float(err.max()), tol)
        seen += int((~fine).sum())
    assert seen > 0


def check_adamw_scaled_norm(dev):
    """norm is f64 throughout: |scale| sqrt(sum g^2) to 1e-12 whatever the scale (200 squares and their sum in f64: 200 x 2^-53)"""
    from apex_amd import engine
    g = torch.tensor(np.random.RandomState(0).randn(200), dtype=torch.float32).to(dev)
    for scale in (1.0 / 3, -0.1, 1e30, 7e-20):
        o = engine.AdamW([torch.zeros(200, device=dev)], max_norm=1.0)
        o.step([g], grad_scale=scale)
        N = Q.clip_factor([f64(g)], scale, 1.0)[0]
        assert abs(float(o.norm) - N) <= 1e-12 * N, (scale, float(o.norm), N)


def check_adamw_far_norms(dev):
    """Norms beyond f32's range and factors below its normal numbers: N is finite in 64 bits, so k = scale min(1, max_norm / (N + 1e-6)) counts as it stands.  Zero moments, one step.
    k: the norm, its sum with 1e-6, the division, scale and their product, each rounded to f32: 5u (where it is formed in f64: u).  k g: 6u.  m: (1 - beta1) and its product: 8u.
    v: the square 2 x 6 + 1, (1 - beta2) and its product: 15u.  Half a step of the smallest numbers twice: 2^-149.  The update: m 8u, half of v's 15u, square root 2u, ibc and its product
    2u, eps and its sum 2u, reciprocal 2u, its product u, lr / (1 - beta1) and its product 2u: 27u.  p: decay, its product and the difference: 3u of p (the decay's own roundings are
    1e-4 of that)."""
    from apex_amd import engine
    r = np.random.RandomState(4)
    for bits in (32, 8):
        for size, max_norm, scale, n in ((3e37, 1.0, 1.0, 1000), (1e37, 1e-3, 1.0, 2500), (3e37, 1e-6, -0.5, 2049), (1e25, 2.0, 1e30, 300), (1e30, 1e-3, 1e10, 5000), (2e37, 3e38, 1.0, 3000), (1e-25, 1e-3, 1e38, 700)):
            g = torch.tensor(r.randn(n) * size, dtype=torch.float32).clamp(-3.3e38, 3.3e38).to(dev)
            p = torch.tensor(r.randn(n) * 0.1, dtype=torch.float32).to(dev)
            p0, g64 = f64(p), f64(g)
            o = engine.AdamW([p], lr=1e-3, eps=1e-8, weight_decay=0.1, max_norm=max_norm, state_bits=bits)
            o.step([g], grad_scale=scale)
            N, k = Q.clip_factor([g64], scale, float(np.float32(max_norm)))
            assert np.isfinite(N) and abs(float(o.norm) - N) <= 1e-12 * N
            want, m, v = Q.adamw(p0, g64, np.zeros(n), np.zeros(n), 1, 1e-3, 0.9, 0.999, 1e-8, 0.1, k)
            what = (bits, size, max_norm, scale)
            if bits == 32:
                assert (np.abs(f64(o.m)[:n] - m) <= 8 * U * np.abs(m) + 2.0 ** -149).all(), what
            if v.max() > 3e38:      # (clipped to a norm of 3e38 the squares are no f32 numbers any more)
                continue
            if bits == 32:
                assert (np.abs(f64(o.v)[:n] - v) <= 15 * U * v + 2.0 ** -149).all(), what
            tol = 3.001 * U * np.abs(p0).max() + 27 * U * np.abs(want - p0).max()
            assert np.abs(f64(p) - want).max() <= tol, (what, np.abs(f64(p) - want).max(), tol)


def check_adamw_decays(dev, count, bits, clip, grad="f32", steps=3):
    """Tensors of a few sizes, more of them than one launch takes, each with a decay of its own between 0.1 and 1 at lr 1e-2: a step takes 1e-3 to 1e-2 of a parameter away, against a bound of
    some 1e-6 for EACH tensor, kept by itself over the steps.  Per step: 3u |p| (decay, its product, the difference; the decay's own roundings 2u of a hundredth: 0.02u more), and of the
    update 27u + 3u a step before (check_adamw_far_norms; m and v bring 3u more from every step)."""
    from apex_amd import engine
    r = np.random.RandomState(count)
    shapes = [(1 + k % 5, 1 + k % 3) for k in range(count)]
    ps = [torch.tensor(r.randn(*s), dtype=torch.float32).to(dev) for s in shapes]
    decay = [0.1 + 0.9 * ((7 * k) % count) / count for k in range(count)]
    hyper = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-5)
    opt = engine.AdamW(ps, weight_decay=decay, max_norm=clip, state_bits=bits, **hyper)
    P, M, V, spread = [f64(p) for p in ps], [np.zeros(s) for s in shapes], [np.zeros(s) for s in shapes], np.zeros(count)
    for t in range(1, steps + 1):
        g = [torch.tensor(r.randn(*s), dtype=torch.float32).to(NP[grad]).to(dev) for s in shapes]
        opt.step(g)
        k = Q.clip_factor([f64(x) for x in g], 1.0, clip)[1]
        moments = [(f64(a), f64(b)) for a, b in zip(opt.views(opt.moments()[0]), opt.views(opt.moments()[1]))]
        for i in range(count):
            p, M[i], V[i] = Q.adamw(P[i], f64(g[i]), M[i], V[i], t, hyper["lr"], *hyper["betas"], hyper["eps"], float(np.float32(decay[i])), k)
            if bits == 8:
                M[i], V[i] = moments[i]      # (what the next step begins with; this step's update uses the moments before their rounding)
            spread[i] += 3.02 * U * np.abs(P[i]).max() + (27 + 3 * t) * U * np.abs(p - P[i] * (1 - hyper["lr"] * decay[i])).max()
            err = np.abs(f64(ps[i]) - p).max()
            assert err <= spread[i], (i, t, err, spread[i])
            assert spread[i] < 0.01 * hyper["lr"] * 0.1 * np.abs(P[i]).max() or np.abs(P[i]).max() < 0.1, "the bound does not tell a decay from none"
            P[i] = p


def check_adamw_eight_bits_over_many_steps(dev, n, steps):
    """8-bit against 32-bit moments over the same gradients, N(1/2, 1) times 1e-2, steps of them.
    v: every rounding keeps the mean, so E v8 = v32.  With s = E g^2 and D = E (v8 - v32)^2: the rounding of what moved by d off the grid has a variance of at most |d| times the grid's step, at
    most v8 / 8, and d = (1 - b2) (g^2 - v8) with g independent of v8: D' <= b2^2 D + (1 - b2) / 8 (s v8 + v8^2) in the mean <= b2^2 D + (1 - b2) / 8 ((2 + e) s^2 + D), e = the variance of v32
    in s^2, below 0.01: D <= (2 + e) / 8 / (1 + b2 - 1 / 8) s^2 = 0.135 s^2 at every step.  The means of n elements: five standard deviations of 0.367 / sqrt(n) for v8 - v32, and 0.05 for its
    square (a fourth moment of 10 D^2 gives 5 x 3 x 0.135 / sqrt(1024) = 0.063 at the fewest elements used; taken as 0.07).
    p: m8's rounding is independent of v8's and keeps the mean; 1 / sqrt(v8) is above 1 / sqrt(v32) in the mean (convexity), to second order by 3/8 x 0.135 = 0.05; twice that is allowed above,
    and for the means of n displacements five of their own standard errors either way."""
    from apex_amd import engine
    r = np.random.RandomState(n)
    size, b2 = 1e-2, 0.999
    p8, p32 = (torch.zeros(n, device=dev) for _ in range(2))
    o8, o32 = engine.AdamW([p8], lr=1e-3, betas=(0.9, b2), eps=1e-8, state_bits=8, seed=3), engine.AdamW([p32], lr=1e-3, betas=(0.9, b2), eps=1e-8)
    for _ in range(steps):
        g = torch.tensor((0.5 + r.randn(n)) * size, dtype=torch.float32).to(dev)
        o8.step([g]); o32.step([g])
    s = 1.25 * size * size
    off = (f64(o8.moments()[1])[:n] - f64(o32.v)[:n]) / s
    assert abs(off.mean()) <= 5 * 0.367 / np.sqrt(n), off.mean()
    assert (off ** 2).mean() <= 0.135 + 0.07, (off ** 2).mean()
    a, b = -f64(p8), -f64(p32)
    room = 5 * np.sqrt(a.var() / n + b.var() / n)
    assert b.mean() > 0 and b.mean() - room <= a.mean() <= 1.1 * b.mean() + room, (a.mean(), b.mean(), room)
    return off, a, b

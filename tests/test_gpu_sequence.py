"""GPU: the gated linear recurrence and the AdamW step (apex_amd/engine.py gated_scan*, AdamW) against the 64-bit oracle, at the sizes, layouts and masks where they can go wrong;
their gradients against differences; captured, replayed and on streams; and both together as a training loop uses them.  Bodies and tolerances: tests/sequence_bodies.py."""
import numpy as np
import pytest
import torch

from oracle import sequence as Q
from tests import sequence_bodies as S

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a GPU")
    return torch.device("cuda:0")


SCANS = [
    dict(T=1, B=1, H=1), dict(T=1, B=3, H=5, gate=True, reset=True, lens=True, carry=True), dict(T=2, B=1, H=64), dict(T=7, B=2, H=3, carry=True), dict(T=16, B=1, H=64, gate=True),
    dict(T=17, B=3, H=21, reset=True, carry=True), dict(T=33, B=2, H=40, t="bf16", gate=True, lens=True, carry=True), dict(T=50, B=3, H=17, t="f16", reset=True, lens=True, carry=True),
    dict(T=400, B=64, H=128, gate=True, lens=True), dict(T=400, B=64, H=128, t="bf16", reset=True, carry=True), dict(T=32, B=512, H=256, t="f16", gate=True, reset=True, carry=True),
    dict(T=63, B=7, H=130, gate=True), dict(T=64, B=7, H=130, t="bf16"), dict(T=65, B=7, H=130, reset=True), dict(T=127, B=2, H=66, t="bf16", gate=True, carry=True), dict(T=129, B=2, H=72, carry=True),
    dict(T=255, B=1, H=256, reset=True), dict(T=257, B=1, H=256, t="bf16", gate=True, lens=True), dict(T=1000, B=1, H=128, carry=True), dict(T=1025, B=3, H=24, reset=True, gate=True, carry=True),
    dict(T=4099, B=1, H=128, reset=True, carry=True, lean=4.0), dict(T=5000, B=2, H=8, t="bf16", gate=True, lens=True, carry=True), dict(T=3001, B=1, H=5, t="f16", gate=True, reset=True),
    dict(T=2048, B=5, H=100, lens=True, carry=True), dict(T=12345, B=1, H=2, gate=True, lean=5.0), dict(T=70001, B=1, H=6, reset=True, carry=True, lean=5.0), dict(T=16448, B=2, H=33, t="bf16", gate=True, lens=True, carry=True),
    dict(T=512, B=1, H=4, carry=True), dict(T=513, B=1, H=4, carry=True), dict(T=575, B=60, H=130, gate=True, reset=True), dict(T=640, B=250, H=128, t="f16"), dict(T=511, B=1, H=4, lens=True),
    dict(T=70, B=33, H=16, gate=True, lens=True, layout="batch first"), dict(T=600, B=2, H=64, t="bf16", reset=True, carry=True, layout="batch first"),
    dict(T=90, B=9, H=64, gate=True, carry=True, layout="shifted"), dict(T=90, B=9, H=64, t="bf16", reset=True, layout="shifted"), dict(T=2100, B=1, H=64, t="f16", carry=True, layout="shifted"),
    dict(T=90, B=9, H=64, gate=True, carry=True, layout="dense"), dict(T=600, B=3, H=60, t="bf16", layout="dense"),
]


@pytest.mark.parametrize("case", SCANS, ids=lambda c: "-".join("%s%s" % kv for kv in c.items()))
def test_scan_against_64_bits(dev, case):
    S.check_scan(dev, **case)


@pytest.mark.parametrize("case", [dict(T=40, B=5, H=13, gate=True), dict(T=300, B=70, H=64, gate=True), dict(T=1500, B=6, H=32, t="bf16"), dict(T=4500, B=5, H=16, t="f16", gate=True)], ids=str)
def test_what_must_not_count_may_hold_anything(dev, case):
    """NaN, infinities and the type's lowest value behind the sequences' ends, and NaN and infinite states in front of a reset"""
    S.check_scan(dev, reset=True, lens=True, carry=True, poison=True, **case)


def test_gates_at_their_limits(dev):
    """f = +inf keeps the state to the bit, f = -inf takes the input to the bit, and very large finite f do the same"""
    from apex_amd import engine
    for T, B, H in ((9, 2, 8), (2000, 1, 8)):
        h0 = torch.randn(B, H, device=dev); x = torch.randn(T, B, H, device=dev)
        for big in (float("inf"), 3e38, 200.0):
            y, h = engine.gated_scan(torch.full_like(x, big), x, h0=h0)
            assert torch.equal(h, h0) and torch.equal(y, h0.expand(T, B, H))
            y, h = engine.gated_scan(torch.full_like(x, -big), x, h0=h0)
            assert torch.equal(y, x) and torch.equal(h, x[-1])


def test_nan_goes_no_further_than_its_channel(dev):
    from apex_amd import engine
    f = torch.randn(500, 3, 40, device=dev); x = torch.randn(500, 3, 40, device=dev)
    ref, _ = engine.gated_scan(f, x)
    x[100, 1, 7] = float("nan")
    y, h = engine.gated_scan(f, x)
    assert torch.isnan(y[100:, 1, 7]).all() and torch.isnan(h[1, 7])
    y[100:, 1, 7] = ref[100:, 1, 7]
    assert torch.equal(y, ref)


def test_scan_of_nothing(dev):
    from tests import test_kernel_emulation_sequence as E
    from apex_amd import engine
    h0 = torch.randn(3, 4, device=dev); z = torch.zeros(0, 3, 4, device=dev)
    y, h, save = engine.gated_scan(z, z, h0=h0, keep=True)
    assert y.shape == (0, 3, 4) and torch.equal(h, h0)
    assert torch.equal(engine.gated_scan_backward(z, z, z, save, h0=h0, dh_last=h0)[3], h0)
    for shape in ((5, 0, 4), (5, 3, 0)):
        assert engine.gated_scan(torch.zeros(*shape, device=dev), torch.zeros(*shape, device=dev))[0].shape == shape
    assert E.SCANS      # (the same with more cases on the CPU)


def test_gradients_against_differences(dev):
    """Central differences of sum(w y) + sum(u h_last) in 64 bits (the oracle's forward pass) along random directions: the third derivative's part is below 1e-6 at a step of 1e-3."""
    from apex_amd import engine
    d, dy, dh = S.make(37, 3, 9, "f32", True, True, True, True, dev, 5)
    _, _, save = engine.gated_scan(**d, keep=True)
    df, dx, do, dh0 = engine.gated_scan_backward(d["f"], d["x"], dy, save, o=d["o"], h0=d["h0"], reset=d["reset"], lens=d["lens"], dh_last=dh)
    w = S.wide(d)
    loss = lambda w: float((Q.gated_scan(**w)[0] * S.f64(dy)).sum() + (Q.gated_scan(**w)[3] * S.f64(dh)).sum())  # noqa: E731
    r = np.random.RandomState(1)
    for k, g in (("f", df), ("x", dx), ("o", do), ("h0", dh0)):
        for _ in range(3):
            v = r.randn(*w[k].shape)
            e = 1e-3
            diff = (loss({**w, k: w[k] + e * v}) - loss({**w, k: w[k] - e * v})) / (2 * e)
            assert abs(float((S.f64(g) * v).sum()) - diff) < 1e-4 * np.sqrt(v.size), k


@pytest.mark.parametrize("case", [dict(B=1, H=1), dict(B=5, H=13, gate=True, reset=True), dict(B=2048, H=128, gate=True, reset=True), dict(B=300, H=130, t="bf16", gate=True),
                                  dict(B=70, H=72, t="f16", reset=True), dict(B=9, H=64, gate=True, layout="shifted"), dict(B=9, H=64, t="bf16", gate=True, layout="shifted")], ids=str)
def test_step_against_64_bits(dev, case):
    S.check_step(dev, **case)


def test_steps_and_the_scan_agree(dev):
    from apex_amd import engine
    d, _, _ = S.make(20, 6, 48, "f32", True, True, False, True, dev, 3)
    y, h, = engine.gated_scan(**d)
    hs = d["h0"].clone()
    _, _, _, M = S.bounds(d)
    eh = S.bounds(d)[0]
    for t in range(20):
        yt = engine.gated_scan_step(d["f"][t], d["x"][t], hs, o=d["o"][t], reset=d["reset"][t])
        assert (yt - y[t]).abs().max() <= 2 * eh + 4 * S.U * M
    assert (hs - h).abs().max() <= 2 * eh


def test_results_do_not_depend_on_the_run(dev):
    """the same bits again, alone and with other work in flight on a second stream"""
    from apex_amd import engine
    d, dy, dh = S.make(3000, 2, 64, "bf16", True, True, True, True, dev, 9)
    def both():
        y, h, s = engine.gated_scan(**d, keep=True)
        return (y, h) + engine.gated_scan_backward(d["f"], d["x"], dy, s, o=d["o"], h0=d["h0"], reset=d["reset"], lens=d["lens"], dh_last=dh)
    ref = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = [both() for _ in range(4)]
    a = [both() for _ in range(4)]
    torch.cuda.synchronize()
    for r in a + b:
        assert all(torch.equal(p, q) for p, q in zip(r, ref))


def test_long_offsets(dev):
    """entries beyond 2^31 elements: the last rows of a [70000, 256, 128] scan and its gradients against a scan of the last rows alone"""
    from apex_amd import engine
    T, B, H, K = 70000, 256, 128, 50
    f = torch.empty(T, B, H, dtype=torch.bfloat16, device=dev).normal_(); x = torch.empty_like(f).normal_()
    reset = torch.zeros(T, B, dtype=torch.uint8, device=dev); reset[T - K] = 1
    y, h, save = engine.gated_scan(f, x, reset=reset, keep=True)
    ys, hs, ss = engine.gated_scan(f[T - K:], x[T - K:], keep=True)
    assert (y[T - K:].float() - ys.float()).abs().max() <= 2 ** -7 * ys.float().abs().max() and (h - hs).abs().max() <= 1e-5
    dy = y; y2 = torch.zeros_like(y[:1])
    df, dx, _, _ = engine.gated_scan_backward(f, x, dy, save, reset=reset)
    dfs, dxs, _, _ = engine.gated_scan_backward(f[T - K:], x[T - K:], dy[T - K:], ss)
    assert (df[T - K:].float() - dfs.float()).abs().max() <= 2 ** -7 * dfs.float().abs().max() and (dx[T - K:].float() - dxs.float()).abs().max() <= 2 ** -7 * dxs.float().abs().max()
    del y2


def test_long_offsets_batch_first(dev):
    """sequences of 1.1 x 10^9 elements each, one behind the other in memory: steps and sequences beyond 2^31 elements, against a scan of the last rows alone"""
    from apex_amd import engine
    T, B, H, K = 9000000, 3, 128, 70
    f = torch.empty(B, T, H, dtype=torch.bfloat16, device=dev).normal_().permute(1, 0, 2)
    out = torch.empty(B, T, H, dtype=torch.bfloat16, device=dev).permute(1, 0, 2)
    reset = torch.zeros(T, B, dtype=torch.uint8, device=dev); reset[T - K] = 1
    y, h = engine.gated_scan(f, f, reset=reset, out=out)
    ys, hs = engine.gated_scan(f[T - K:], f[T - K:])
    assert (y[T - K:].float() - ys.float()).abs().max() <= 2 ** -7 * ys.float().abs().max() and (h - hs).abs().max() <= 1e-5


def test_rows_outside_the_outputs_stay(dev):
    """outputs written into slices of larger buffers leave everything around them as it was"""
    from apex_amd import engine
    for T, t in ((30, torch.float32), (1500, torch.bfloat16)):
        B, H = 3, 40
        f = torch.randn(T, B, H, device=dev).to(t); x = torch.randn(T, B, H, device=dev).to(t); dy = torch.randn(T, B, H, device=dev).to(t)
        big = torch.full((T + 2, B + 1, 3 * H), 7.0, dtype=t, device=dev)
        out = big[1:-1, :B, H:2 * H]
        y, _, save = engine.gated_scan(f, x, keep=True, out=out)
        ref, _ = engine.gated_scan(f, x)
        assert torch.equal(out, ref)
        out.fill_(7.0)
        assert (big == 7).all()
        df, dx = engine.gated_scan_backward(f, x, dy, save, out=(big[1:-1, :B, :H], big[1:-1, :B, 2 * H:]))[:2]
        r = engine.gated_scan_backward(f, x, dy, save)
        assert torch.equal(df, r[0]) and torch.equal(dx, r[1])
        df.fill_(7.0); dx.fill_(7.0)
        assert (big == 7).all()


def test_repeated_and_overlapping_inputs(dev):
    """one row for all steps (stride 0), and the same tensor in several places"""
    from apex_amd import engine
    T, B, H = 300, 4, 32
    f = torch.randn(1, B, H, device=dev).expand(T, B, H); x = torch.randn(T, 1, H, device=dev).expand(T, B, H)
    a, b = engine.gated_scan(f, x, keep=True), engine.gated_scan(f.contiguous(), x.contiguous(), keep=True)
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    r, q = engine.gated_scan_backward(f, x, f, a[2]), engine.gated_scan_backward(f.contiguous(), x.contiguous(), f.contiguous(), b[2])
    assert torch.equal(r[0], q[0]) and torch.equal(r[1], q[1])
    y, _ = engine.gated_scan(x, x, o=x)
    z, _ = engine.gated_scan(x.clone(), x.clone(), o=x.clone())
    assert torch.equal(y, z)
    w = torch.randn(20, 3, 16, device=dev).permute(2, 1, 0)      # units far apart: copied
    y, _ = engine.gated_scan(w, w)
    assert torch.equal(y, engine.gated_scan(w.contiguous(), w.contiguous())[0])


ADAMW = [
    dict(shapes=[(1,)], clip=0.05), dict(shapes=[(5, 7), (3,), (257,), (16, 16)], clip=0.05, flat=True), dict(shapes=[(300,), (0,), (1,)], grad="bf16"), dict(shapes=[(2049, 3), (2048,), (4097,)], grad="f16", clip=1.0),
    dict(shapes=[(512, 50), (512, 128), (512,), (512,), (512, 128), (512, 128), (512,), (512,), (10, 128), (10,)], clip=0.05, flat=True), dict(shapes=[(1000, 999)], clip=0.05, scale=0.125),
    dict(shapes=[(k % 37 + 1, 3) for k in range(200)], clip=0.05, flat=True),
    dict(shapes=[(1,)], bits=8), dict(shapes=[(5, 7), (3,), (257,), (16, 16)], bits=8, clip=0.05, flat=True, scale=0.5), dict(shapes=[(2100,), (0,), (1,)], bits=8, grad="f16", clip=10.0),
    dict(shapes=[(k % 37 + 1, 3) for k in range(200)], bits=8, clip=0.01, flat=True), dict(shapes=[(1000, 999), (77,)], bits=8, grad="bf16"), dict(shapes=[(256, 64), (64,)], bits=8, sizes=1e-18),
    dict(shapes=[(40, 256)], bits=8, sizes=1e4, steps=6),
]


@pytest.mark.parametrize("case", ADAMW, ids=lambda c: "%d-%s-%s" % (len(c["shapes"]), c.get("bits", 32), c.get("grad", "f32")))
def test_adamw_against_64_bits(dev, case):
    S.check_adamw(dev, **case)


def test_adamw_a_tensor_beyond_32_bits(dev):
    """2^31 + 5000 elements in one tensor: around the 2^31st and at the end what a small optimiser makes of the same elements"""
    from apex_amd import engine
    n = 2 ** 31 + 5000
    p = torch.empty(n, device=dev).normal_(); g = torch.empty(n, dtype=torch.bfloat16, device=dev).normal_()
    cuts = [slice(0, 300), slice(2 ** 31 - 2500, 2 ** 31 + 2500), slice(n - 300, n)]
    small = [p[c].clone() for c in cuts]
    o, e = engine.AdamW([p, torch.zeros(3, device=dev)], weight_decay=0.1), engine.AdamW(small, weight_decay=0.1)
    for _ in range(2):
        o.step([g, torch.ones(3, dtype=torch.bfloat16, device=dev)])
        e.step([g[c].contiguous() for c in cuts])
    for c, q, m in zip(cuts, small, e.views(e.m)):
        assert torch.equal(p[c], q) and torch.equal(o.m[c], m)


def test_adamw_stands_for_clip_adam(dev):
    """without weight decay, one flat tensor: what the framework's flat step computes (both run the same formula, with roundings in other places)"""
    from apex_amd import engine, _lib
    n = 81418
    g = torch.Generator(device=dev); g.manual_seed(3)
    p = torch.randn(n, device=dev, generator=g) * 0.05; q = p.clone(); m = torch.zeros(n, device=dev); v = torch.zeros(n, device=dev); sc = torch.zeros(1, dtype=torch.float64, device=dev)
    o = engine.AdamW([p], lr=1e-4, eps=1e-5, max_norm=0.05)
    for t in range(1, 6):
        grad = torch.randn(n, device=dev, generator=g)
        _lib.check(_lib.load().apx_clip_adam(engine._p(q), engine._p(m), engine._p(v), engine._p(grad), n, 1.0, 0.05, 1e-4, 1e-5, t, engine._p(sc), engine._stream()))
        o.step([grad])
    # a step moves a parameter by about lr = 1e-4; its formula in f32 is good to 50 u of that, and p itself to u a step
    assert (p - q).abs().max() <= 5 * (50 * S.U * 1e-4 * 5 + 2 * S.U * 0.3)


def test_adamw_a_norm_that_is_not_finite_changes_nothing(dev):
    from apex_amd import engine
    for bits in (32, 8):
        p = [torch.ones(3000, device=dev), torch.ones(5, device=dev)]
        o = engine.AdamW(p, max_norm=1.0, state_bits=bits)
        o.step([torch.ones_like(x) for x in p])
        before = [x.clone() for x in (*p, o.m, o.v)]
        for bad in (float("nan"), float("inf")):
            g = [torch.ones_like(x) for x in p]; g[0][2999] = bad
            o.step(g)
            assert all(torch.equal(a, b) for a, b in zip(before, (*p, o.m, o.v))) and not np.isfinite(float(o.norm))
        assert int(o.t) == 3


def test_adamw_captured_and_replayed(dev):
    """a captured step counts at every replay and makes the same steps as an eager one, with other work between the replays"""
    from apex_amd import engine
    for bits in (32, 8):
        def fresh():
            g = torch.Generator(device=dev); g.manual_seed(1)
            p = [torch.randn(700, 3, device=dev, generator=g), torch.randn(11, device=dev, generator=g)]
            return p, engine.AdamW(p, max_norm=0.5, state_bits=bits, weight_decay=0.1), g
        p, o, g = fresh()
        grads = [torch.zeros_like(x) for x in p]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o.step(grads)
        q, e, _ = fresh()
        for k in range(5):
            new = [torch.randn(x.shape, device=dev, generator=g) * 10.0 ** (k - 2) for x in p]
            for a, b in zip(grads, new):
                a.copy_(b)
            graph.replay()
            (torch.randn(512, 512, device=dev) @ torch.randn(512, 512, device=dev)).sum().item()
            e.step(new)
            torch.cuda.synchronize()
            assert int(o.t) == k + 1 and all(torch.equal(a, b) for a, b in zip((*p, o.m, o.v, o.norm), (*q, e.m, e.v, e.norm)))


def test_scan_captured_and_replayed(dev):
    """two captured training passes of different lengths, replayed in turn with eager calls between: every replay gives the eager result on the inputs of the moment"""
    from apex_amd import engine
    def run(d, dy):
        y, h, s = engine.gated_scan(**d, keep=True)
        return (y, h) + tuple(g for g in engine.gated_scan_backward(d["f"], d["x"], dy, s, o=d["o"], h0=d["h0"], reset=d["reset"], lens=d["lens"]) if g is not None)
    sets = [S.make(3000, 1, 64, "f32", True, True, True, True, dev, 1, layout="dense"), S.make(100, 40, 64, "bf16", False, True, False, True, dev, 2, layout="dense"), S.make(5000, 1, 32, "f32", False, False, False, True, dev, 3, layout="dense")]
    graphs = []
    for d, dy, _ in sets:
        run(d, dy)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = run(d, dy)
        graphs.append((g, out))
    for k in range(4):
        for (d, dy, _), (g, out) in zip(sets, graphs):
            new = torch.randn_like(d["x"])
            d["x"].copy_(new)
            g.replay()
            ref = run(d, dy)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, ref)), k


def test_step_captured_and_replayed(dev):
    from apex_amd import engine
    f, x, h = torch.randn(50, 30, device=dev), torch.randn(50, 30, device=dev), torch.zeros(50, 30, device=dev)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = engine.gated_scan_step(f, x, h)
    h.zero_(); e = torch.zeros_like(h)
    for k in range(6):
        x.normal_()
        g.replay()
        r = engine.gated_scan_step(f, x, e)
        torch.cuda.synchronize()
        assert torch.equal(y, r) and torch.equal(h, e)


def test_a_recurrent_head_trained_with_both(dev):
    """A small recurrent core the way it would be used - one product for f | x | o, the scan, a head, masked squared error, gradients into slices of the product's gradient, AdamW on
    all tensors with decay on the matrices only -: its gradients against the same network in 64 bits (formulas by the chain rule on the oracle), then steps that run."""
    from apex_amd import engine
    T, B, D, H = 60, 10, 12, 32
    g = torch.Generator(device=dev); g.manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    obs, target = rnd(T, B, D), rnd(T, B)
    lens = torch.randint(1, T + 1, (B,), generator=g, device=dev).to(torch.int32)
    mask = (torch.arange(T, device=dev)[:, None] < lens).float()
    W, bias, out = rnd(3 * H, D) * 0.3, rnd(3 * H) * 0.1, rnd(H) * 0.3
    opt = engine.AdamW([W, bias, out], lr=1e-3, weight_decay=[0.01, 0.0, 0.01], max_norm=0.5, state_bits=8)
    for it in range(3):
        proj = (obs.view(-1, D) @ W.t() + bias).view(T, B, 3 * H)
        y, _, save = engine.gated_scan(proj[..., :H], proj[..., H:2 * H], o=proj[..., 2 * H:], lens=lens, keep=True)
        err = (y @ out - target) * mask
        dy = (2 * err / mask.sum())[..., None] * out
        dproj = torch.empty_like(proj)
        engine.gated_scan_backward(proj[..., :H], proj[..., H:2 * H], dy, save, o=proj[..., 2 * H:], lens=lens, out=(dproj[..., :H], dproj[..., H:2 * H], dproj[..., 2 * H:]))
        grads = [dproj.view(-1, 3 * H).t() @ obs.view(-1, D), dproj.sum((0, 1)), ((2 * err / mask.sum())[..., None] * y).sum((0, 1))]
        if it == 0:
            w64, o64, b64, out64 = S.f64(W), S.f64(obs), S.f64(bias), S.f64(out)
            p64 = o64.reshape(-1, D) @ w64.T + b64
            p64 = p64.reshape(T, B, 3 * H)
            n = lens.cpu().numpy()
            parts = dict(f=p64[..., :H], x=p64[..., H:2 * H], o=p64[..., 2 * H:], lens=n)
            y64 = Q.gated_scan(**parts)[0]
            e64 = (y64 @ out64 - S.f64(target)) * S.f64(mask)
            d64 = (2 * e64 / S.f64(mask).sum())[..., None] * out64
            df, dx, do, _, _ = Q.gated_scan_grad(dy=d64, **parts)
            dp = np.concatenate([df, dx, do], -1)
            refs = [dp.reshape(-1, 3 * H).T @ o64.reshape(-1, D), dp.sum((0, 1)), ((2 * e64 / S.f64(mask).sum())[..., None] * y64).sum((0, 1))]
            for got, ref in zip(grads, refs):      # f32 products over 600 rows: 600 u of the summands' size, far below 1e-4 of the result's norm
                assert np.linalg.norm(S.f64(got) - ref) <= 1e-4 * np.linalg.norm(ref)
        opt.step([x.contiguous() for x in grads])
    assert int(opt.t) == 3 and all(torch.isfinite(x).all() for x in (W, bias, out))


def test_refusals_on_the_device(dev):
    from apex_amd import engine
    f = torch.zeros(4, 2, 3, device=dev)
    for call in (lambda: engine.gated_scan(f, torch.zeros(4, 2, 3)), lambda: engine.gated_scan(f, f.clone(), out=f), lambda: engine.gated_scan(f, f, h0=torch.zeros(2, 3)),
                 lambda: engine.AdamW([f]).step([torch.zeros(4, 2, 3)]), lambda: engine.AdamW([f, torch.zeros(3)])):
        with pytest.raises((ValueError, RuntimeError)):
            call()


@pytest.mark.parametrize("case", [dict(T=24, B=1, H=2, at=(10, 12)), dict(T=300, B=1, H=2, at=(160, 165)), dict(T=300, B=1, H=2, at=(95, 97)), dict(T=400, B=9, H=64, gate=True, lens=True),
                                  dict(T=33, B=70, H=40, t="bf16", infinite=True), dict(T=5000, B=2, H=33, t="f16", gate=True, infinite=True), dict(T=1500, B=3, H=64, lens=True)],
                         ids=lambda c: "-".join("%s%s" % kv for kv in c.items()))
def test_what_is_not_finite_passes_no_reset(dev, case):
    S.check_not_finite(dev, **case)


def test_adamw_scaled_norm(dev):
    S.check_adamw_scaled_norm(dev)


def test_adamw_far_norms(dev):
    S.check_adamw_far_norms(dev)


def test_the_stream_is_torchs(dev):
    """the handle that the calls are launched on is that of torch.cuda.current_stream(), on the default stream, on another and inside a capture"""
    from apex_amd import engine
    same = lambda: (engine._stream().value or 0) == torch.cuda.current_stream().cuda_stream  # noqa: E731
    side = torch.cuda.Stream()
    assert same()
    with torch.cuda.stream(side):
        assert same() and engine._stream().value == side.cuda_stream
    graph, f = torch.cuda.CUDAGraph(), torch.zeros(2, 3, device=dev)
    with torch.cuda.graph(graph):
        assert same()
        f.add_(1)
    assert same()


@pytest.mark.parametrize("case", [dict(count=130, bits=32, clip=0.05), dict(count=250, bits=8, clip=None), dict(count=121, bits=32, clip=None, grad="bf16"), dict(count=500, bits=8, clip=1.0, grad="f16")], ids=str)
def test_adamw_every_tensor_has_its_decay(dev, case):
    S.check_adamw_decays(dev, **case)


@pytest.mark.parametrize("n,steps", [(1 << 16, 300), (5000, 3000)])
def test_adamw_eight_bits_over_many_steps(dev, n, steps):
    S.check_adamw_eight_bits_over_many_steps(dev, n, steps)

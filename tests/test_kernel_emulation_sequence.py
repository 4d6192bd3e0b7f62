"""CPU: the sequence operators' kernel SOURCES (apex_amd/csrc/gated_scan.hip, adamw.hip) compiled for the host under tools/hipemu, through the host code of apex_amd/engine.py and the
bodies of the GPU tests (tests/sequence_bodies.py), and the refusals of both layers (which end before anything is launched)."""
import ctypes as C

import numpy as np
import pytest
import torch

from oracle import sequence as Q
from tests import sequence_bodies as S
from tests.test_kernel_emulation_learner import dev  # noqa: F401  (the fixture that puts the emulated library in place)

SCANS = [
    dict(T=1, B=1, H=1), dict(T=1, B=3, H=5, gate=True, reset=True, lens=True, carry=True), dict(T=7, B=2, H=3, carry=True), dict(T=16, B=1, H=64, gate=True),
    dict(T=17, B=3, H=21, reset=True, carry=True), dict(T=33, B=2, H=40, t="bf16", gate=True, lens=True, carry=True), dict(T=50, B=3, H=17, t="f16", reset=True, lens=True, carry=True),
    dict(T=40, B=5, H=13, gate=True, reset=True, lens=True, carry=True, poison=True), dict(T=300, B=1, H=8, reset=True, carry=True, lean=4.0), dict(T=130, B=1, H=65, t="bf16", gate=True),
    dict(T=600, B=2, H=10, reset=True, carry=True), dict(T=1100, B=1, H=3, gate=True, lens=True, carry=True, t="bf16"), dict(T=17000, B=1, H=1, reset=True, carry=True, lean=4.0),
    dict(T=1030, B=3, H=44, gate=True, reset=True, lens=True, carry=True, poison=True, t="f16"), dict(T=70, B=2, H=16, gate=True, lens=True, layout="batch first"), dict(T=20, B=2, H=12, gate=True, carry=True, layout="shifted"), dict(T=21, B=2, H=12, t="bf16", layout="dense"),
]


@pytest.mark.parametrize("case", SCANS, ids=lambda c: "-".join("%s%s" % kv for kv in c.items()))
def test_emulated_scan(dev, case):  # noqa: F811
    S.check_scan(dev, **case)


def test_emulated_scan_of_nothing(dev):  # noqa: F811
    from apex_amd import engine
    h0 = torch.randn(3, 4)
    y, h, save = engine.gated_scan(torch.zeros(0, 3, 4), torch.zeros(0, 3, 4), h0=h0, keep=True)
    assert y.shape == (0, 3, 4) and torch.equal(h, h0) and save.numel() == 0
    dh = torch.randn(3, 4)
    df, dx, do, dh0 = engine.gated_scan_backward(torch.zeros(0, 3, 4), torch.zeros(0, 3, 4), torch.zeros(0, 3, 4), save, h0=h0, dh_last=dh)
    assert df.shape == (0, 3, 4) and torch.equal(dh0, dh)
    for shape in ((5, 0, 4), (5, 3, 0)):
        y, h = engine.gated_scan(torch.zeros(*shape), torch.zeros(*shape))
        assert y.shape == shape and h.shape == shape[1:]
    f = torch.randn(6, 2, 4)
    y, h = engine.gated_scan(f, f, h0=h0[:2].contiguous(), lens=torch.tensor([0, -5], dtype=torch.int32))
    assert torch.equal(h, h0[:2]) and not y.any()
    a, b = engine.gated_scan(f, f), engine.gated_scan(f, f, lens=torch.tensor([6, 2 ** 31 - 1], dtype=torch.int32))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_emulated_scan_reset_everywhere(dev):  # noqa: F811
    """a reset in front of every step: no step sees another one, whatever the start"""
    from apex_amd import engine
    for T in (5, 300):
        f, x, r = torch.randn(T, 2, 6), torch.randn(T, 2, 6), torch.ones(T, 2, dtype=torch.uint8)
        y, h, save = engine.gated_scan(f, x, h0=torch.full((2, 6), float("nan")), reset=r, keep=True)
        want = Q.sigmoid(-S.f64(f)) * S.f64(x)
        assert np.abs(S.f64(y) - want).max() < 1e-6 * np.abs(want).max() and torch.equal(h, y[-1])
        df, dx, _, dh0 = engine.gated_scan_backward(f, x, torch.ones(T, 2, 6), save, h0=torch.zeros(2, 6), reset=r, dh_last=torch.zeros(2, 6))
        a, n = Q.sigmoid(S.f64(f)), Q.sigmoid(-S.f64(f))
        assert np.abs(S.f64(dx) - n).max() < 1e-6 and np.abs(S.f64(df) + S.f64(x) * a * n).max() < 1e-6 * 4 and not dh0.any()


@pytest.mark.parametrize("case", [dict(B=1, H=1), dict(B=5, H=13, gate=True, reset=True), dict(B=3, H=64, t="bf16", gate=True), dict(B=4, H=8, t="f16", reset=True),
                                  dict(B=3, H=12, gate=True, layout="shifted")], ids=str)
def test_emulated_step(dev, case):  # noqa: F811
    S.check_step(dev, **case)


ADAMW = [
    dict(shapes=[(1,)], clip=0.05), dict(shapes=[(5, 7), (3,), (257,), (16, 16)], clip=0.05, flat=True), dict(shapes=[(300,), (0,), (1,)], grad="bf16"),
    dict(shapes=[(1,)], bits=8), dict(shapes=[(5, 7), (3,), (257,), (16, 16)], bits=8, clip=0.05, flat=True, scale=0.5), dict(shapes=[(2100,), (0,), (1,)], bits=8, grad="f16", clip=10.0),
    dict(shapes=[(256, 4), (64,)], bits=8, sizes=1e-18), dict(shapes=[(300,)], bits=8, sizes=1e-36),
    dict(shapes=[(k % 5 + 1,) for k in range(200)], bits=8, clip=0.01, steps=2), dict(shapes=[(k % 5 + 1,) for k in range(91)], clip=0.01, steps=2),
]


@pytest.mark.parametrize("case", ADAMW, ids=lambda c: "%d-%s" % (len(c["shapes"]), c.get("bits", 32)))
def test_emulated_adamw(dev, case):  # noqa: F811
    S.check_adamw(dev, **case)


def test_emulated_adamw_special_blocks(dev):  # noqa: F811
    """A norm that is not finite changes nothing but the count; without clipping an infinity or a NaN stays in its block; a block of zeros stays zero."""
    from apex_amd import engine
    p = [torch.ones(300), torch.ones(5)]
    o = engine.AdamW(p, max_norm=1.0, state_bits=8)
    o.step([torch.full((300,), float("inf")), torch.ones(5)])
    assert torch.equal(p[0], torch.ones(300)) and torch.equal(p[1], torch.ones(5)) and not o.m.any() and not o.v.any() and int(o.t) == 1 and float(o.norm) == float("inf")
    o = engine.AdamW(p, state_bits=8)
    g = torch.zeros(300); g[3] = float("nan")
    o.step([g, torch.zeros(5)])
    m, v = o.moments()
    assert torch.isnan(m[:256]).all() and not m[256:].any() and not v[256:].any() and torch.isnan(p[0][3]) and torch.isfinite(p[0][4:]).all() and torch.equal(p[1], torch.ones(5))


def test_emulated_adamw_of_nothing(dev):  # noqa: F811
    """empty tensors alone: the step counts, the norm is 0"""
    from apex_amd import engine
    for bits in (8, 32):
        o = engine.AdamW([torch.zeros(0), torch.zeros(3, 0)], max_norm=1.0, state_bits=bits)
        assert o._ws.numel() >= 64 + 8      # (room for the one partial sum of the launch that counts)
        o.norm.fill_(5.0)
        o.step([torch.zeros(0), torch.zeros(3, 0)])
        assert int(o.t) == 1 and float(o.norm) == 0.0 and o.moments()[0].numel() == 0


def test_emulated_adamw_rounding_keeps_the_mean(dev):  # noqa: F811
    """4096 elements that all hold the same moments: m = 0.1 g, v = 0.001 g^2 in the first step, rounded up or down to neighbours an eighth of a power of two apart.  The mean of n
    independent roundings is off by at most (step / 2) / sqrt(n) in the standard deviation: five of them here."""
    from apex_amd import engine
    n = 4096
    for g in (0.3, 1.234, 0.0777):
        o = engine.AdamW([torch.zeros(n)], state_bits=8, seed=11)
        o.step([torch.full((n,), g)])
        m, v = o.moments()
        for got, want in ((m.double(), 0.1 * g), (v.double(), 0.001 * g * g)):
            step = 2.0 ** np.floor(np.log2(want)) / 8
            assert abs(float(got.mean()) - want) < 5 * step / 2 / np.sqrt(n)
            assert len(torch.unique(got)) <= 2


# ------------------------------------------------------------------------------------------------ refusals (no device needed: they come before any launch)
def test_refusals_of_the_wrappers(dev):  # noqa: F811
    from apex_amd import engine
    f, x = torch.zeros(4, 2, 3), torch.zeros(4, 2, 3)
    bad = [
        lambda: engine.gated_scan(f[0], x[0]), lambda: engine.gated_scan(f.double(), x.double()), lambda: engine.gated_scan(f, x[:3]), lambda: engine.gated_scan(f, x.bfloat16()),
        lambda: engine.gated_scan(f, x, o=x[..., :2]), lambda: engine.gated_scan(f, x, h0=torch.zeros(2, 4)), lambda: engine.gated_scan(f, x, h0=torch.zeros(2, 3).bfloat16()),
        lambda: engine.gated_scan(f, x, reset=torch.zeros(4, 2)), lambda: engine.gated_scan(f, x, reset=torch.zeros(2, 4, dtype=torch.uint8)),
        lambda: engine.gated_scan(f, x, lens=torch.zeros(2, dtype=torch.int64)), lambda: engine.gated_scan(f, x, lens=torch.zeros(3, dtype=torch.int32)),
        lambda: engine.gated_scan(f, x, out=x), lambda: engine.gated_scan(f, x, out=torch.zeros(4, 2, 3, dtype=torch.float16)), lambda: engine.gated_scan(f, x, out=torch.zeros(1, 1, 3).expand(4, 2, 3)),
        lambda: engine.gated_scan(f, x, out=torch.zeros(4, 2, 6)[..., ::2]),
        lambda: engine.gated_scan_step(f, x, torch.zeros(2, 3)), lambda: engine.gated_scan_step(f[0], x[0], torch.zeros(2, 3).bfloat16()), lambda: engine.gated_scan_step(f[0], x[0], torch.zeros(3, 2).t()),
        lambda: engine.gated_scan_step(f[0], x[0], torch.zeros(2, 3), reset=torch.zeros(3, dtype=torch.uint8)),
    ]
    _, _, save = engine.gated_scan(f, x, keep=True)
    bad += [lambda: engine.gated_scan_backward(f, x, x[:3], save), lambda: engine.gated_scan_backward(f, x, x, save[:-1]), lambda: engine.gated_scan_backward(f, x, x, save.double()),
            lambda: engine.gated_scan_backward(f, x, x, save, out=(torch.zeros(4, 2, 3),)), lambda: engine.gated_scan_backward(f, x, x, save, dh_last=torch.zeros(3, 2))]
    t = torch.zeros(4, 2, 3)
    bad += [lambda: engine.gated_scan_backward(f, x, x, save, out=(t, t)), lambda: engine.gated_scan_backward(f, x, torch.ones(4, 2, 3), save, out=(t, f))]
    p, q = [torch.zeros(3), torch.zeros(4)], torch.zeros(9)
    bad += [lambda: engine.AdamW([]), lambda: engine.AdamW([torch.zeros(3).double()]), lambda: engine.AdamW([torch.zeros(3, 4).t()]), lambda: engine.AdamW(p, state_bits=16),
            lambda: engine.AdamW(p, weight_decay=[0.1]), lambda: engine.AdamW([p[0], p[0]]), lambda: engine.AdamW([q[:5], q[4:]])]
    o = engine.AdamW(p)
    bad += [lambda: o.step([torch.zeros(3)]), lambda: o.step([torch.zeros(3), torch.zeros(5)]), lambda: o.step([torch.zeros(3), torch.zeros(4).bfloat16()]),
            lambda: o.step([torch.zeros(3).double(), torch.zeros(4).double()]), lambda: o.step([torch.zeros(6)[::2], torch.zeros(4)]),
            lambda: engine.AdamW(p, eps=0.0).step([torch.zeros(3), torch.zeros(4)]), lambda: engine.AdamW(p, betas=(1.0, 0.9)).step([torch.zeros(3), torch.zeros(4)]),
            lambda: engine.AdamW(p, max_norm=0.0).step([torch.zeros(3), torch.zeros(4)]), lambda: engine.AdamW(p, max_norm=-1.0).step([torch.zeros(3), torch.zeros(4)]),
            lambda: o.step([p[0], torch.zeros(4)]), lambda: engine.AdamW(p, weight_decay=float("nan")).step([torch.zeros(3), torch.zeros(4)]),
            lambda: engine.AdamW(p, lr=float("nan")).step([torch.zeros(3), torch.zeros(4)])]
    for i, call in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            call()
            pytest.fail("call %d was taken" % i)
    assert not p[0].any() and int(o.t) == 0


def test_refusals_of_the_c_entry_points():
    """apx_* of the product library itself: every refusal returns APX_E_ARG with a message and launches nothing (there is no device here)."""
    from apex_amd import _lib
    lib = _lib.load()
    one = 16      # a pointer that is never followed: each call below is refused before

    def scan(fn, **change):
        a = _lib.GatedScanArgs(type=0, H=4, T=3, B=2, f=one, f_t=8, f_b=4, x=2 * one, x_t=8, x_b=4, y=3 * one, y_t=8, y_b=4, h_last=4 * one, dy=5 * one, dy_t=8, dy_b=4, df=6 * one, df_t=8, df_b=4,
                               dx=7 * one, dx_t=8, dx_b=4, save=8 * one)
        for k, v in change.items():
            setattr(a, k, v)
        return fn(C.byref(a), None)
    F, Bk = lib.apx_gated_scan_forward, lib.apx_gated_scan_backward
    calls = [scan(F, type=3), scan(F, type=-1), scan(F, T=-1), scan(F, B=-1), scan(F, H=-1), scan(F, f=None), scan(F, x=None), scan(F, y=None), scan(F, h_last=None),
             scan(F, f_t=-8), scan(F, y_b=3), scan(F, y_t=7), scan(F, y_t=0), scan(F, y=one), scan(F, h0=4 * one), scan(F, o=9 * one, o_t=-1), scan(F, T=1 << 58), scan(F, B=1 << 35),
             scan(F, f_t=1 << 60), scan(F, f_t=1 << 30), scan(F, x_b=1 << 30), scan(F, T=64, B=1 << 20, H=1 << 12, f_b=1 << 12, x_b=1 << 12, y_b=1 << 12, f_t=1 << 32, x_t=1 << 32, y_t=1 << 32), scan(Bk, dy_b=1 << 31), scan(Bk, save=None), scan(Bk, dy=None), scan(Bk, df=7 * one), scan(Bk, df=one), scan(Bk, o=9 * one, o_t=8, o_b=4), scan(Bk, dx_b=0),
             scan(Bk, dh0=11 * one, dh_last=11 * one)]
    s = _lib.GatedScanArgs(type=0, H=4, B=2, f=one, f_b=4, x=2 * one, x_b=4, y=3 * one, y_b=4)
    calls.append(lib.apx_gated_scan_step(C.byref(s), None, None))
    s.y_b = 2
    calls.append(lib.apx_gated_scan_step(C.byref(s), 4 * one, None))
    s.B, s.H, s.f_b, s.x_b, s.y_b = 1 << 20, 1 << 12, 1 << 12, 1 << 12, 1 << 12
    calls.append(lib.apx_gated_scan_step(C.byref(s), 4 * one, None))
    calls += [lib.apx_gated_scan_step(None, 4 * one, None), F(None, None), Bk(None, None), lib.apx_adamw(None, None)]

    def adam(**change):
        ptr, num, wd = (C.c_void_p * 1)(one), (C.c_int64 * 1)(5), None
        a = _lib.AdamwArgs(n_tensors=1, grad_type=0, state_bits=32, params=C.addressof(ptr), grads=C.addressof(ptr), numel=C.addressof(num), m=2 * one, v=3 * one, t=4 * one, lr=1e-3, beta1=0.9,
                           beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=0.0, workspace=5 * one, workspace_bytes=1 << 20)
        if "num" in change:
            num[0] = change.pop("num")
        if "null" in change:
            ptr[0] = change.pop("null")
        for k, v in change.items():
            setattr(a, k, v)
        return lib.apx_adamw(C.byref(a), None)
    nan, inf = float("nan"), float("inf")
    calls += [adam(n_tensors=-1), adam(params=None), adam(grads=None), adam(numel=None), adam(t=None), adam(grad_type=3), adam(state_bits=4), adam(beta1=1.0), adam(beta2=-0.1), adam(beta1=nan),
              adam(eps=0.0), adam(eps=-1.0), adam(eps=1e-46), adam(eps=nan), adam(lr=inf), adam(lr=1e39), adam(grad_scale=nan), adam(max_norm=nan), adam(num=-1), adam(num=1 << 41), adam(null=None),
              adam(m=None), adam(v=None), adam(state_bits=8), adam(workspace=None), adam(workspace=8), adam(workspace_bytes=64),
              lib.apx_adamw_moments(one, one, one, one, 255, one, one, None), lib.apx_adamw_moments(one, one, one, one, -256, one, one, None), lib.apx_adamw_moments(None, one, one, one, 256, one, one, None)]
    assert calls == [-1] * len(calls), [i for i, c in enumerate(calls) if c != -1]
    assert b"invalid argument" in lib.apx_last_error()
    assert lib.apx_gated_scan_save_floats(17, 2, 5) == 10 and lib.apx_gated_scan_save_floats(0, 2, 5) == 0
    assert lib.apx_adamw_state_elements(3, (C.c_int64 * 3)(1, 0, 257)) == 768


def test_refusals_of_misaligned_pointers():
    """a pointer that is not aligned to its own type is refused at every C entry"""
    from apex_amd import _lib
    lib = _lib.load()
    p = lambda k: 64 * k  # noqa: E731
    for kind, half in ((0, 2), (1, 1), (2, 1)):
        good = dict(type=kind, H=4, T=3, B=2, f=p(1), f_t=8, f_b=4, x=p(2), x_t=8, x_b=4, y=p(3), y_t=8, y_b=4, h_last=p(4), dy=p(5), dy_t=8, dy_b=4, df=p(6), df_t=8, df_b=4,
                    dx=p(7), dx_t=8, dx_b=4, save=p(8), o=p(9), o_t=8, o_b=4, do_=p(10), do_t=8, do_b=4, h0=p(11), dh0=p(12), dh_last=p(13), lens=p(14))
        call = lambda fn, k, by: fn(C.byref(_lib.GatedScanArgs(**{**good, k: good[k] + by})), None)  # noqa: E731
        assert [call(lib.apx_gated_scan_forward, k, half) for k in "fxoy"] == [-1] * 4
        assert [call(lib.apx_gated_scan_backward, k, half) for k in ("f", "x", "o", "dy", "df", "dx", "do_")] == [-1] * 7
        assert [call(lib.apx_gated_scan_forward, k, 2) for k in ("h0", "h_last", "lens", "save")] == [-1] * 4
        assert [call(lib.apx_gated_scan_backward, k, 2) for k in ("h0", "dh0", "dh_last", "lens", "save")] == [-1] * 5
        step = _lib.GatedScanArgs(**{**good, "h0": 0, "lens": 0})
        assert lib.apx_gated_scan_step(C.byref(step), p(15) + 2, None) == -1

    def adam(kind, at, gat, **change):
        ptr, grad, num = (C.c_void_p * 1)(at), (C.c_void_p * 1)(gat), (C.c_int64 * 1)(5)
        a = _lib.AdamwArgs(n_tensors=1, grad_type=kind, state_bits=32, params=C.addressof(ptr), grads=C.addressof(grad), numel=C.addressof(num), m=p(2), v=p(3), t=p(4), lr=1e-3, beta1=0.9,
                           beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=1.0, workspace=p(5), workspace_bytes=1 << 20, norm_out=p(6))
        for k, v in change.items():
            setattr(a, k, v)
        return lib.apx_adamw(C.byref(a), None)
    assert [adam(0, p(1) + 2, p(7)), adam(0, p(1), p(7) + 2), adam(1, p(1), p(7) + 1), adam(2, p(1), p(7) + 1), adam(0, p(1), p(7), t=p(4) + 4), adam(0, p(1), p(7), norm_out=p(6) + 4),
            adam(0, p(1), p(7), m=p(2) + 2)] == [-1] * 7
    assert [lib.apx_adamw_moments(*a, None) for a in ((p(1) + 4, p(2), p(3), p(4), 256, p(5), p(6)), (p(1), p(2), p(3) + 2, p(4), 256, p(5), p(6)), (p(1), p(2), p(3), p(4), 256, p(5) + 8, p(6)))] == [-1] * 3


def test_emulated_scan_of_two_far_steps(dev):  # noqa: F811
    """what has to lie within 4 GB are a call's own steps: two of them 2 GB apart are served, with three of them (4 GB) refused"""
    from apex_amd import _lib
    lib = _lib.load()
    a = dict(type=0, H=4, B=1, f=64, f_b=4, x=128, x_t=4, x_b=4, y=192, y_t=4, y_b=4, h_last=256)
    assert lib.apx_gated_scan_forward(C.byref(_lib.GatedScanArgs(T=3, f_t=1 << 29, **a)), None) == -1 and b"too far apart" in lib.apx_last_error()
    import mmap
    far = mmap.mmap(-1, (1 << 31) + 4096)      # (touched at its two ends alone)
    f = torch.frombuffer(far, dtype=torch.float32, count=(1 << 29) + 4).as_strided((2, 1, 4), (1 << 29, 4, 1))
    f.copy_(torch.randn(2, 1, 4))
    from apex_amd import engine
    x = torch.randn(2, 1, 4)
    y, h = engine.gated_scan(f, x)
    y2, h2 = engine.gated_scan(f.contiguous(), x)
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_wrappers_need_device_tensors():
    from apex_amd import _lib, engine
    f = torch.zeros(4, 2, 3)
    for call in (lambda: engine.gated_scan(f, f), lambda: engine.gated_scan_backward(f, f, f, f), lambda: engine.gated_scan_step(f[0], f[0], f[0].clone()), lambda: engine.AdamW([f])):
        with pytest.raises(_lib.ApxError):
            call()


def test_the_moments_noise_is_spread_evenly():
    """Each of the 32 bits that round the moments is set for half of the elements, and neighbours, steps and seeds do not go together: 2^16 samples, five standard deviations."""
    from oracle import sequence as Q
    n = 1 << 16
    a, b, c = Q.noise(7, 1, np.arange(n)), Q.noise(7, 2, np.arange(n)), Q.noise(8, 1, np.arange(n))
    bits = lambda r: (r[:, None] >> np.arange(32, dtype=np.uint64)) & np.uint64(1)  # noqa: E731
    lim = 5 * 0.5 / np.sqrt(n)
    for r in (a, a ^ b, a ^ c, a[1:] ^ a[:-1], a[256:] ^ a[:-256]):
        assert np.abs(bits(r).mean(0) - 0.5).max() < lim * 1.01


NOT_FINITE = [
    dict(T=24, B=1, H=2, at=(10, 12)), dict(T=24, B=1, H=2, at=(12, 10)), dict(T=24, B=1, H=2, at=(10, 10)), dict(T=40, B=1, H=3, at=(17, 22)), dict(T=40, B=1, H=3, at=(7, 8)),
    dict(T=300, B=1, H=2, at=(160, 165)), dict(T=300, B=1, H=2, at=(95, 97)), dict(T=300, B=1, H=2, gate=True, at=(159, 160)),
    dict(T=24, B=6, H=5, gate=True), dict(T=70, B=4, H=6, t="bf16"), dict(T=70, B=4, H=6, gate=True, lens=True, infinite=True), dict(T=300, B=3, H=6, gate=True, lens=True), dict(T=300, B=3, H=5, t="f16", infinite=True),
    dict(T=1100, B=2, H=4, infinite=True),
]


@pytest.mark.parametrize("case", NOT_FINITE, ids=lambda c: "-".join("%s%s" % kv for kv in c.items()))
def test_emulated_scan_what_is_not_finite_passes_no_reset(dev, case):  # noqa: F811
    S.check_not_finite(dev, **case)


def test_emulated_adamw_scaled_norm(dev):  # noqa: F811
    S.check_adamw_scaled_norm(dev)


def test_emulated_adamw_far_norms(dev):  # noqa: F811
    S.check_adamw_far_norms(dev)


def test_emulated_scan_leaves_unread_fields_alone(dev):  # noqa: F811
    """fields that a call does not read may hold anything: odd and huge strides, pointers to nowhere (never followed), in both directions, without o, without steps, and for one step"""
    from apex_amd import _lib, engine
    lib = _lib.load()
    T, B, H = 150, 3, 6
    odd, huge, low = 0x7ffffffffffffff1, (1 << 62) + 3, -(1 << 62)
    t = lambda *s: torch.randn(*s)  # noqa: E731
    f, x, dy, h0 = t(T, B, H), t(T, B, H), t(T, B, H), t(B, H)
    y, hl, df, dx = torch.zeros(T, B, H), torch.zeros(B, H), torch.zeros(T, B, H), torch.zeros(T, B, H)
    ry, rh, save = engine.gated_scan(f, x, h0=h0, keep=True)
    rdf, rdx, _, _ = engine.gated_scan_backward(f, x, dy, save, h0=h0)
    st = lambda k: {k + "_t": B * H, k + "_b": H}  # noqa: E731
    ws = torch.zeros(max(16, lib.apx_gated_scan_workspace_bytes(T, B, H)), dtype=torch.uint8)
    base = dict(type=0, H=H, T=T, B=B, f=f.data_ptr(), x=x.data_ptr(), **st("f"), **st("x"), workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    assert ws.data_ptr() % 16 == 0
    for a, b in ((odd, huge), (low, low), (huge, odd)):
        fwd = dict(base, y=y.data_ptr(), **st("y"), h0=h0.data_ptr(), h_last=hl.data_ptr(), o=0, o_t=a, o_b=b, dy=odd, dy_t=a, dy_b=b, df=odd, df_t=a, df_b=b, dx=odd, dx_t=a, dx_b=b, do_=odd, do_t=a,
                   do_b=b, dh_last=odd, dh0=odd)
        y.zero_(); hl.zero_()
        assert lib.apx_gated_scan_forward(C.byref(_lib.GatedScanArgs(**fwd)), None) == 0, lib.apx_last_error()
        assert torch.equal(y, ry) and torch.equal(hl, rh)
        bwd = dict(base, dy=dy.data_ptr(), **st("dy"), df=df.data_ptr(), **st("df"), dx=dx.data_ptr(), **st("dx"), save=save.data_ptr(), y=odd, y_t=a, y_b=b, h_last=odd, o=0, o_t=a, o_b=b, do_=odd, do_t=a, do_b=b)
        df.zero_(); dx.zero_()
        assert lib.apx_gated_scan_backward(C.byref(_lib.GatedScanArgs(**bwd)), None) == 0, lib.apx_last_error()
        assert torch.equal(df, rdf) and torch.equal(dx, rdx)
        none = dict(type=0, H=H, T=0, B=B, f=odd, f_t=a, f_b=b, x=odd, x_t=a, x_b=b, y=odd, y_t=a, y_b=b, o=odd, o_t=a, o_b=b, h0=h0.data_ptr(), h_last=hl.data_ptr())
        assert lib.apx_gated_scan_forward(C.byref(_lib.GatedScanArgs(**none)), None) == 0, lib.apx_last_error()
        assert torch.equal(hl, h0)
        h, y1 = h0.clone(), torch.zeros(B, H)
        one = dict(type=0, H=H, T=-7, B=B, f=f.data_ptr(), f_t=a, f_b=H, x=x.data_ptr(), x_t=b, x_b=H, y=y1.data_ptr(), y_t=a, y_b=H, h0=odd, lens=odd, h_last=odd, save=odd, dy=odd, dy_t=a, dy_b=b, dh_last=odd,
                   df=odd, dx=odd, do_=odd, dh0=odd, workspace=odd, workspace_bytes=3)
        assert lib.apx_gated_scan_step(C.byref(_lib.GatedScanArgs(**one)), h.data_ptr(), None) == 0, lib.apx_last_error()
        want = engine.gated_scan(f[:1], x[:1], h0=h0)
        assert torch.equal(y1, want[0][0]) and torch.equal(h, want[1])


def test_emulated_scan_refuses_operands_that_overlap(dev):  # noqa: F811
    """outputs shifted by one step, one sequence or one unit from an input or from each other are refused, slices of one buffer that keep apart are taken and give the same results"""
    from apex_amd import engine
    T, B, H = 6, 4, 5
    buf = lambda *s: torch.randn(*s)  # noqa: E731
    f, x, dy = buf(T, B, H), buf(T, B, H), buf(T, B, H)
    ry, _, save = engine.gated_scan(f, x, keep=True)
    rdf, rdx, _, _ = engine.gated_scan_backward(f, x, dy, save)

    def into(view, t):
        view.copy_(t)
        return view

    for make, cuts in ((lambda: buf(T + 1, B, H), (slice(0, T), slice(1, T + 1))), (lambda: buf(T, B + 1, H), ((slice(None), slice(0, B)), (slice(None), slice(1, B + 1)))),
                       (lambda: buf(T, B, H + 1), ((Ellipsis, slice(0, H)), (Ellipsis, slice(1, H + 1)))), (lambda: buf(T, B, 2 * H - 1), ((Ellipsis, slice(0, H)), (Ellipsis, slice(H - 1, 2 * H - 1))))):
        for a, b in (cuts, cuts[::-1]):
            big = make()
            for call in (lambda: engine.gated_scan(into(big[a], f), x, out=big[b]), lambda: engine.gated_scan(f, into(big[a], x), out=big[b]), lambda: engine.gated_scan(f, x, o=into(big[a], f), out=big[b]),
                         lambda: engine.gated_scan_backward(f, x, into(big[a], dy), save, out=(big[b], torch.empty(T, B, H))), lambda: engine.gated_scan_backward(f, x, dy, save, out=(big[a], big[b])),
                         lambda: engine.gated_scan(f, into(big[a], x), o=x, out=big[b])):
                with pytest.raises(RuntimeError, match="overlap"):
                    call()
    for make, cuts in ((lambda: buf(2 * T, B, H), (slice(0, T), slice(T, 2 * T))), (lambda: buf(2 * T, B, H), (slice(0, 2 * T, 2), slice(1, 2 * T, 2))), (lambda: buf(T, 2 * B, H), ((slice(None), slice(0, 2 * B, 2)), (slice(None), slice(1, 2 * B, 2)))),
                       (lambda: buf(T, B, 2 * H), ((Ellipsis, slice(0, H)), (Ellipsis, slice(H, 2 * H)))), (lambda: buf(B, T, 2 * H).permute(1, 0, 2), ((Ellipsis, slice(H, 2 * H)), (Ellipsis, slice(0, H))))):
        big = make()
        y, _ = engine.gated_scan(into(big[cuts[0]], f), x, out=big[cuts[1]])
        assert torch.equal(y, ry)
        df, dx, _, _ = engine.gated_scan_backward(f, x, dy, save, out=(big[cuts[0]], big[cuts[1]]))
        assert torch.equal(df, rdf) and torch.equal(dx, rdx)
    row = buf(T, B, 2 * H)      # one row for all steps, in columns of its own of the buffer that the output lies in
    one = row[0, 1, H:].expand(T, B, H)
    assert torch.equal(engine.gated_scan(f, one, out=row[..., :H])[0], engine.gated_scan(f, one.clone())[0])
    h = torch.randn(B, H); want = h.clone()      # h as an input of its own step
    y = engine.gated_scan_step(f[0], h, h)
    z = engine.gated_scan_step(f[0], want.clone(), want)
    assert torch.equal(h, want) and torch.equal(y, z)
    with pytest.raises(RuntimeError, match="overlap"):
        engine.gated_scan_step(f[0], x[0], h, out=h)


def test_emulated_scan_overlaps_by_chance(dev):  # noqa: F811
    """600 layouts in a small buffer: a call is refused exactly where its output shares a byte with an input (bytes counted one by one), else it gives what separate buffers give"""
    from apex_amd import _lib, engine
    lib = _lib.load()
    r = np.random.RandomState(0)
    refused = taken = 0
    while refused + taken < 600:
        T, B, H = r.randint(1, 5), r.randint(1, 5), r.randint(1, 5)
        near = H + r.randint(0, 9); far = (max(T, B) - 1) * near + H + r.randint(0, 9)
        ys = (far, near) if r.rand() < 0.5 else (near, far)
        fs = ys if r.rand() < 0.4 else tuple(int(r.choice([0, near, far, r.randint(0, 40)])) for _ in range(2))
        size = 3 * far * 5 + 64
        y0, f0, s0 = (int(r.randint(0, size // 3)) for _ in range(3))
        place = lambda at, st: {at + t * st[0] + b * st[1] + j for t in range(T) for b in range(B) for j in range(H)}  # noqa: E731
        mem = torch.randn(size)
        Y, F, S0 = place(y0, ys), place(f0, fs), set(range(s0, s0 + B * H))
        f = mem.as_strided((T, B, H), (*fs, 1), f0).clone(); h0 = mem[s0:s0 + B * H].view(B, H).clone()
        x, hl = torch.randn(T, B, H), torch.zeros(B, H)
        p = mem.data_ptr()
        args = dict(type=0, H=H, T=T, B=B, f=p + 4 * f0, f_t=fs[0], f_b=fs[1], x=x.data_ptr(), x_t=B * H, x_b=H, y=p + 4 * y0, y_t=ys[0], y_b=ys[1], h0=p + 4 * s0, h_last=hl.data_ptr())
        before = mem.clone()
        rc = lib.apx_gated_scan_forward(C.byref(_lib.GatedScanArgs(**args)), None)
        if Y & F or Y & S0:
            assert rc == -1 and b"overlap" in lib.apx_last_error() and torch.equal(mem, before), (T, B, H, ys, fs, y0, f0, s0)
            refused += 1
        else:
            assert rc == 0, (T, B, H, ys, fs, y0, f0, s0, lib.apx_last_error())
            ry, rh = engine.gated_scan(f, x, h0=h0)
            assert torch.equal(mem.as_strided((T, B, H), (*ys, 1), y0), ry) and torch.equal(hl, rh)
            taken += 1
    assert min(refused, taken) > 100


def test_emulated_adamw_refuses_memory_that_overlaps(dev):  # noqa: F811
    """a gradient that reaches into a parameter, a moment or another part of the state, and parameters or state that overlap, are refused and nothing changes; neighbours are taken"""
    from apex_amd import _lib, engine
    lib = _lib.load()
    n = 600
    block = torch.randn(4 * n)
    for order in (1, -1):
        for many in (1, 300):      # (more than the table on the stack holds, in ascending and descending order)
            ps = [torch.randn(3) for _ in range(many - 1)][::order] + [block[n:2 * n]]
            o = engine.AdamW(ps, state_bits=32)
            gs = [torch.randn(3) for _ in range(many - 1)]
            start = block.clone()
            for at in (1, n - 1, n + 1, 2 * n - 1):
                with pytest.raises(RuntimeError, match="gradient"):
                    o.step(gs + [block[at:at + n]])
            for bad in (o.m[:n], o.v[5:n + 5]):
                with pytest.raises(RuntimeError, match="gradient"):
                    o.step(gs + [bad])
            assert torch.equal(block, start) and int(o.t) == 0 and not o.m.any()
            o.step(gs + [block[:n]]); o.step(gs + [block[2 * n:3 * n]])
            assert int(o.t) == 2 and torch.equal(block[:n], start[:n]) and torch.equal(block[2 * n:], start[2 * n:])
    g, q = torch.randn(4), [torch.zeros(4), torch.zeros(4)]
    o = engine.AdamW(q)
    o.step([g, g])
    assert torch.equal(q[0], q[1]) and q[0].any()

    p, m, v, ws, t, norm = torch.randn(600), torch.zeros(1024), torch.zeros(1024), torch.zeros(20000, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64), torch.zeros(1, dtype=torch.float64)
    g = torch.randn(600)

    def step(**change):
        ptr, grad, num = (C.c_void_p * 2)(p.data_ptr(), p.data_ptr() + 4 * change.pop("second", 300)), (C.c_void_p * 2)(g.data_ptr(), g.data_ptr()), (C.c_int64 * 2)(300, 300)
        a = dict(n_tensors=2, grad_type=0, state_bits=32, params=C.addressof(ptr), grads=C.addressof(grad), numel=C.addressof(num), m=m.data_ptr(), v=v.data_ptr(), t=t.data_ptr(), lr=1e-3, beta1=0.9,
                 beta2=0.999, eps=1e-8, grad_scale=1.0, max_norm=1.0, workspace=ws.data_ptr(), workspace_bytes=ws.numel(), norm_out=norm.data_ptr())
        return lib.apx_adamw(C.byref(_lib.AdamwArgs(**{**a, **change})), None)
    before = p.clone()
    for change in (dict(second=299), dict(second=0), dict(m=v.data_ptr()), dict(v=m.data_ptr() + 4 * 1023), dict(t=norm.data_ptr()), dict(norm_out=ws.data_ptr() + 8), dict(t=m.data_ptr() + 8),
                   dict(m=p.data_ptr()), dict(v=g.data_ptr()), dict(norm_out=p.data_ptr() + 8)):
        assert step(**change) == -1 and any(w in lib.apx_last_error() for w in (b"overlap", b"lies on")), change
        assert torch.equal(p, before) and int(t[0]) == 0
    assert step() == 0 and int(t[0]) == 1 and not torch.equal(p, before)
    c, s, out = torch.zeros(1024, dtype=torch.uint8), torch.ones(8), torch.zeros(4096, dtype=torch.uint8)
    assert out.data_ptr() % 16 == 0 and c.data_ptr() % 16 == 0
    mom = lambda mo, vo: lib.apx_adamw_moments(c.data_ptr(), c.data_ptr() + 512, s.data_ptr(), s.data_ptr() + 8, 512, mo, vo, None)  # noqa: E731
    assert [mom(c.data_ptr(), out.data_ptr()), mom(out.data_ptr(), c.data_ptr() + 512), mom(out.data_ptr(), out.data_ptr() + 1008)] == [-1] * 3 and b"overlap" in lib.apx_last_error()
    assert mom(out.data_ptr(), out.data_ptr() + 1024) == 0


def test_adamw_sizes_of_no_tensors():
    """the two size functions follow no NULL and count nothing for sizes that a step refuses"""
    from apex_amd import _lib
    lib = _lib.load()
    none = lib.apx_adamw_workspace_bytes(0, None)
    assert none >= 64 + 8 and lib.apx_adamw_workspace_bytes(3, None) == none and lib.apx_adamw_state_elements(3, None) == 0 and lib.apx_adamw_state_elements(-1, None) == 0
    num = (C.c_int64 * 4)(-5, 1 << 39, (1 << 63) - 1, 3)
    assert lib.apx_adamw_state_elements(4, num) == 256 and lib.apx_adamw_workspace_bytes(4, num) == none


def test_the_stream_of_a_forked_process_is_refused(monkeypatch):
    """engine._stream() passes torch's own lazy initialisation: what torch.cuda.current_stream() refuses - a child forked from a process that uses the GPU - is refused with torch's message"""
    from apex_amd import engine
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)      # (what such a child would otherwise be told)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda k: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "_initialized", True)
    assert engine._stream().value is None      # the default stream's handle
    monkeypatch.setattr(torch.cuda, "_is_in_bad_fork", lambda: True)
    with pytest.raises(RuntimeError, match="fork"):
        engine._stream()


@pytest.mark.parametrize("case", [dict(count=130, bits=32, clip=0.05), dict(count=250, bits=8, clip=None), dict(count=121, bits=32, clip=None, grad="bf16"), dict(count=119, bits=8, clip=1.0)], ids=str)
def test_emulated_adamw_every_tensor_has_its_decay(dev, case):  # noqa: F811
    S.check_adamw_decays(dev, **case)


def test_emulated_adamw_eight_bits_over_many_steps(dev):  # noqa: F811
    S.check_adamw_eight_bits_over_many_steps(dev, 1024, 300)


def test_emulated_scan_dense_outputs_in_gaps(dev):  # noqa: F811
    """h_last between the steps of an f of many rows is taken, one element further into it refused; a step's h may be its own f or x and not its own o"""
    from apex_amd import _lib, engine
    lib = _lib.load()
    B, gap = 2500, 2600
    mem = torch.randn(2 * (2 * B + gap))
    f = mem.as_strided((2, B, 1), (2 * B + gap, 2, 1))
    x, y = torch.randn(2, B, 1), torch.zeros(2, B, 1)
    want, state = engine.gated_scan(f.clone(), x)
    for at, ok in ((2 * B, True), (2 * B + gap - B, True), (2 * B - 2, False), (2 * B + gap - B + 1, False), (2 * B - 1, True)):      # (the last row's element is followed by one of the gap)
        a = _lib.GatedScanArgs(type=0, H=1, T=2, B=B, f=f.data_ptr(), f_t=2 * B + gap, f_b=2, x=x.data_ptr(), x_t=B, x_b=1, y=y.data_ptr(), y_t=B, y_b=1, h_last=mem.data_ptr() + 4 * at)
        rc = lib.apx_gated_scan_forward(C.byref(a), None)
        assert rc == (0 if ok else -1), (at, lib.apx_last_error())
        if ok:
            assert torch.equal(y, want) and torch.equal(mem[at:at + B], state.view(-1))
    f, x, h = torch.randn(3, 8), torch.randn(3, 8), torch.randn(3, 8)
    for first in (True, False):
        a, b = h.clone(), h.clone()
        got = engine.gated_scan_step(a if first else f, x if first else a, a, o=x)
        ref = engine.gated_scan_step(b.clone() if first else f, x if first else b.clone(), b, o=x)
        assert torch.equal(got, ref) and torch.equal(a, b)
    with pytest.raises(RuntimeError, match="overlap"):
        engine.gated_scan_step(f, x, h, o=h)

"""The AdamW step over many tensors against its formula in 64 bits (needs a B200).

Tolerances: a few float32 roundings (u = 2^-24) of each term of the formula, the parameter type's one
rounding, and for 8-bit states e4m3's steps: half a step (2^-4 of the value, or 2^-10 of the block's scale
near zero) for m, a whole one for sqrt(v), which is rounded up or down at random.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}
SIZES = (1, 255, 256, 257, 1000, 31, 4096, 70_001, 8)
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-6, weight_decay=0.1)


def _dt(name):
    import torch

    return getattr(torch, name)


def _make(dtype, gdtype, seed, sizes=SIZES, misalign=0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(n, dt, scale):
        t = torch.zeros(n + misalign, dtype=_dt(dt), device="cuda")[misalign:]
        t.copy_(torch.randn(n, generator=g, device="cuda") * scale)
        return t

    return [one(n, dtype, 0.5) for n in sizes], [one(n, gdtype, 0.02) for n in sizes]


def _expect(p, g, m, v, t, gs=1.0, lr=None):
    """(p, m, v) of the formula in 64 bits, and their rounding errors in float32."""
    lr, (b1, b2), eps, wd = lr or HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    g = g.double() * gs
    m2 = b1 * m + (1 - b1) * g
    v2 = b2 * v + (1 - b2) * g * g
    em = 4 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + TINY["float32"]
    ev = 5 * U * v2 + TINY["float32"]
    denom = (v2 / (1 - b2 ** t)).sqrt() + eps
    upd = lr / (1 - b1 ** t) * m2 / denom
    p2 = p.double() * (1 - lr * wd) - upd
    # the update's relative error: m's, half of v's, and 8 roundings (the reciprocals and the quotient)
    ep = 3 * U * p.double().abs() + lr / (1 - b1 ** t) * em / denom + 16 * U * upd.abs()
    return (p2, ep), (m2, em), (v2, ev)


def _close(got, want, tol):
    d = (got.double() - want).abs()
    assert bool((d <= tol).all()), f"worst {float((d - tol).max())} over"


@pytest.mark.parametrize("dtype,gdtype,master,misalign", [
    ("float32", "float32", False, 0), ("float32", "float32", False, 1), ("bfloat16", "bfloat16", False, 0),
    ("bfloat16", "bfloat16", True, 0), ("bfloat16", "float32", True, 3), ("float16", "float16", True, 0),
    ("float16", "float32", False, 5),
])
def test_adamw_32_bit_states(dtype, gdtype, master, misalign):
    import torch

    from trident_b200 import AdamW

    params, _ = _make(dtype, gdtype, 1, misalign=misalign)
    opt = AdamW(params, master=master, **HYPER)
    scale = torch.tensor([0.25], device="cuda")
    for t in range(1, 4):
        grads = _make(dtype, gdtype, 10 + t)[1]
        src = [s.clone() for s in (opt.state["master"] if master else params)]
        m0, v0 = ([x.double() for x in opt.state[k]] for k in ("exp_avg", "exp_avg_sq"))
        opt.step(grads, grad_scale=scale if t == 2 else None, lr=0.03 if t == 3 else None)
        for i, g in enumerate(grads):
            (p, ep), (m, em), (v, ev) = _expect(src[i], g, m0[i], v0[i], t, 0.25 if t == 2 else 1.0, 0.03 if t == 3 else None)
            _close(opt.state["exp_avg"][i], m, em)
            _close(opt.state["exp_avg_sq"][i], v, ev)
            _close(params[i], p, ep + ROUND[dtype] * (p.abs() + ep) + TINY[dtype])
            if master:
                _close(opt.state["master"][i], p, ep)
                assert torch.equal(params[i], opt.state["master"][i].to(params[i].dtype))
    assert opt.step_count == 3


def _decode(opt, i):
    """(m, sqrt v, m's scales, the root's scales) of the 8-bit states, one scale a value."""
    n = opt.params[i].numel()
    ms, vs = (opt.state[k][i].double().repeat_interleave(256)[:n] for k in ("exp_avg_scale", "exp_avg_sq_root_scale"))
    return opt.state["exp_avg"][i].double() * ms, opt.state["exp_avg_sq_root"][i].double() * vs, ms, vs


@pytest.mark.parametrize("dtype,gdtype,master,misalign", [
    ("bfloat16", "bfloat16", False, 0), ("bfloat16", "bfloat16", True, 0), ("float32", "float32", False, 0),
    ("float32", "float32", False, 1), ("float16", "float32", False, 3),
])
def test_adamw_8_bit_states(dtype, gdtype, master, misalign):
    import torch

    from trident_b200 import AdamW

    params, _ = _make(dtype, gdtype, 2, misalign=misalign)
    opt = AdamW(params, master=master, state_bits=8, seed=7, **HYPER)
    for t in range(1, 5):
        grads = _make(dtype, gdtype, 20 + t)[1]
        src = [s.clone() for s in (opt.state["master"] if master else params)]
        old = [_decode(opt, i) for i in range(len(params))]
        opt.step(grads)
        for i, g in enumerate(grads):
            m0, r0 = old[i][:2]
            (p, ep), (m, em), (v, ev) = _expect(src[i], g, m0, r0 * r0, t)
            _close(params[i], p, 1.01 * ep + ROUND[dtype] * (p.abs() + ep) + TINY[dtype])
            gm, gr, ms, vs = _decode(opt, i)
            root = v.sqrt()
            _close(gm, m, 1.01 * (2.0 ** -4 * m.abs() + 2.0 ** -10 * ms) + em)
            _close(gr, root, 1.01 * (2.0 ** -3 * root + 2.0 ** -9 * vs) + 4 * U * root)
            assert bool(((gr > 0) == (v > 0)).all())  # a root is never rounded to 0
            pad = -len(m) % 256
            for x, key in ((m.abs(), "exp_avg_scale"), (root, "exp_avg_sq_root_scale")):
                top = torch.nn.functional.pad(x, (0, pad)).view(-1, 256).amax(1)
                _close(opt.state[key][i], top / 448, 1e-6 * top)


def test_adamw_8_bit_rounding_keeps_the_mean():
    """sqrt(v) between two e4m3 values is rounded to either so that the mean is kept: over 2^16 blocks whose
    largest value is 448 and whose others lie at a fraction of a step, within 6 standard errors."""
    import torch

    from trident_b200 import AdamW

    n = 256 * 4096
    p = torch.zeros(n, device="cuda")
    for k, frac in enumerate((0.03, 0.25, 0.5, 0.9)):
        g = torch.full((n,), 16.0 + 2.0 * frac, device="cuda")  # e4m3 has 16, 18, 20: steps of 2
        g[::256] = 448.0
        opt = AdamW([p], betas=(0.0, 0.0), eps=1.0, weight_decay=0.0, state_bits=8, seed=k)
        opt.step([g])
        root = opt.state["exp_avg_sq_root"][0].double().view(-1, 256)
        assert bool((root[:, 0] == 448).all())
        rest = root[:, 1:]
        assert bool(((rest == 16) | (rest == 18)).all())
        se = 2.0 * math.sqrt(frac * (1 - frac) / rest.numel())
        # 16 random bits: the chance is a multiple of 2^-16, and the root itself is off by a few u
        assert abs(float(rest.mean()) - (16 + 2 * frac)) <= 6 * se + 2.0 * 2.0 ** -16 + 64 * U


def test_adamw_8_bit_states_follow_a_change():
    """The states after gradients grow 16-fold: sqrt(v) gains 0.05% of itself in a typical step, which
    nearest rounding would never see. The blocks' largest values keep their size, so that the scales do not move."""
    import torch

    from trident_b200 import AdamW

    n = 256 * 64
    p = torch.zeros(n, device="cuda")
    opt = AdamW([p], lr=0.0, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8)
    v = 0.0
    for t in range(600):
        size = 0.01 if t < 100 else 0.16
        g = torch.full((n,), size, device="cuda")
        g[::256] = 5.0
        opt.step([g])
        v = 0.999 * v + 0.001 * size * size
    rest = _decode(opt, 0)[1].view(-1, 256)[:, 1:]
    # a value's random walk: at most sqrt(600) steps of 2^-3 with chance ~2^-8 each, averaged over 16,320 values;
    # v = E[root^2] exceeds E[root]^2 by the rounding's variance, some percent
    assert abs(float((rest * rest).mean()) / v - 1) < 0.1


def test_adamw_many_tensors_and_none():
    """More tensors than one launch takes, empty ones, and ones without a gradient."""
    import torch

    from trident_b200 import AdamW

    sizes = [(i * 37) % 300 for i in range(1000)]
    params, grads = _make("float32", "float32", 3, sizes=sizes)
    grads = [None if i % 11 == 5 else g for i, g in enumerate(grads)]
    before = [p.clone() for p in params]
    for bits in (32, 8):
        ps = [p.clone() for p in before]
        opt = AdamW(ps, state_bits=bits, **HYPER)
        opt.step(grads)
        for i, (p, g) in enumerate(zip(ps, grads)):
            if g is None:
                assert torch.equal(p, before[i]) and bool((opt.state["exp_avg"][i].float() == 0).all())
                continue
            z = torch.zeros_like(p).double()
            (want, ep), _, _ = _expect(before[i], g, z, z, 1)
            _close(p, want, ep)


def test_adamw_mixed_dtypes_resume_and_streams():
    """Parameters of two dtypes; a run that is stopped and resumed from its states gives the same bits, also
    on another stream."""
    import torch

    from trident_b200 import AdamW

    def start():
        return _make("bfloat16", "bfloat16", 4)[0] + _make("float32", "float32", 5)[0]

    def grads(t):
        return _make("bfloat16", "bfloat16", 30 + t)[1] + _make("float32", "float32", 40 + t)[1]

    for bits, master in ((32, True), (8, False)):
        a = start()
        opt = AdamW(a, state_bits=bits, master=master, seed=3, **HYPER)
        for t in range(4):
            opt.step(grads(t))
        torch.cuda.synchronize()
        b = start()
        first = AdamW(b, state_bits=bits, master=master, seed=3, **HYPER)
        for t in range(2):
            first.step(grads(t))
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            state = {k: [x.clone() for x in v] for k, v in first.state.items()}
            second = AdamW(b, state_bits=bits, master=master, seed=3, state=state, step=first.step_count, **HYPER)
            for t in range(2, 4):
                second.step(grads(t))
        side.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(a, b))
        for k in opt.state:
            assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(opt.state[k], second.state[k]))


def test_adamw_values_that_are_not_finite():
    """A NaN gradient stays with its value in 32 bits, and with its block of 256 in 8 bits."""
    import torch

    from trident_b200 import AdamW

    g = torch.full((1024,), 0.1, device="cuda")
    g[300] = float("nan")
    for bits in (32, 8):
        p = torch.ones(1024, device="cuda")
        opt = AdamW([p], state_bits=bits)
        opt.step([g])
        assert torch.isnan(p).nonzero().flatten().tolist() == [300]
        if bits == 8:
            m, r = _decode(opt, 0)[:2]
            for x in (m, r):
                bad = ~torch.isfinite(x)
                assert bool(bad[256:512].all()) and not bool(bad[:256].any()) and not bool(bad[512:].any())
    # zero gradients: states and scales of 0, no update beyond the decay
    p = torch.ones(300, device="cuda")
    opt = AdamW([p], state_bits=8, lr=0.5, weight_decay=0.5)
    opt.step([torch.zeros(300, device="cuda")])
    assert bool((p == 0.75).all())
    assert all(bool((x.float() == 0).all()) for v in opt.state.values() for x in v)


def test_adamw_in_a_graph():
    import torch

    from trident_b200 import AdamW

    params, grads = _make("float32", "float32", 6)
    other = [p.clone() for p in params]
    a, b = AdamW(params, **HYPER), AdamW(other, **HYPER)
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        a.step(grads)
    g.replay()
    b.step(grads)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(params, other))

"""Embedding lookup, layer norm and their gradients against their definitions in 64 bits (needs a B200).

Tolerances are the rounding errors that the operators may make, from their formulas: u = 2^-24 for each
float32 operation, the result type's unit roundoff for the one rounding at the end, and k u sum|terms| for
a float32 sum whose longest chain of additions has k links.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
ROUND = {"float32": 0.0, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}
TINY = {"float32": 2.0 ** -149, "bfloat16": 2.0 ** -133, "float16": 2.0 ** -24}  # half steps at zero, and more
DTYPES = ("float32", "bfloat16", "float16")


def _dt(name):
    import torch

    return getattr(torch, name)


def _randn(shape, dtype, seed, scale=1.0, shift=0.0):
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(shape, generator=g, device="cuda") * scale + shift).to(_dt(dtype))


def _strided(t, pad):
    """The same rows with `pad` extra elements between them."""
    import torch

    wide = torch.full((t.shape[0], t.shape[1] + pad), float("nan"), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _close(got, want, tol):
    import torch

    got = got.double()
    ok = (got - want).abs() <= tol
    assert bool(ok.all()), f"{int((~ok).sum())} of {ok.numel()} off, worst by {float(((got - want).abs() - tol).max())}"
    assert bool(torch.isfinite(got).all())


def _ids(T, V, seed, dtype="int64", kind="skewed"):
    import torch

    rng = np.random.default_rng(seed)
    if kind == "same":
        x = np.full(T, V - 1)
    elif kind == "none":
        x = np.full(T, -1)
    elif kind == "spread":
        x = rng.integers(0, V, T)
    else:
        x = np.minimum((V + 1) ** rng.random(T), V).astype(np.int64) - 1
        x[rng.random(T) < 0.1] = -1
    return torch.from_numpy(x.astype(dtype)).cuda()


# ---- lookup

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,V,D,pad,ids", [
    (1, 1, 1, 0, "int64"), (1, 5, 8, 0, "int32"), (33, 100, 7, 0, "int64"), (1000, 300, 96, 0, "int32"),
    (257, 5000, 960, 0, "int64"), (100, 40, 97, 3, "int32"), (64, 31, 128, 8, "int64"), (40, 9, 2050, 0, "int64"),
    (17, 9, 12, 1, "int64"), (9, 3, 4096, 0, "int32"),
])
def test_lookup(dtype, T, V, D, pad, ids):
    import torch

    import trident_b200 as tb

    table = _randn((V, D), dtype, 1)
    if pad:
        table = _strided(table, pad)
    x = _ids(T, V, 2, ids)
    scale = 1.7
    got = tb.embedding_lookup(table, x, scale=scale)
    assert got.shape == (T, D) and got.dtype == table.dtype
    want = torch.where((x >= 0)[:, None], table[x.clamp(min=0).long()].double() * float(np.float32(scale)), 0.0)
    _close(got, want, (ROUND[dtype] + 2 * U) * want.abs() + TINY[dtype])
    # a strided output, ids of more dims and another order of rows
    out = torch.full((T, D + 5), 7.0, dtype=table.dtype, device="cuda")
    tb.embedding_lookup(table, x, scale=scale, out=out[:, :D])
    assert torch.equal(out[:, :D], got) and bool((out[:, D:] == 7).all())
    two = x.repeat(2).view(2, T).t()
    assert torch.equal(tb.embedding_lookup(table, two, scale=scale), got[:, None].expand(T, 2, D))


def test_lookup_ids_outside_the_table():
    import torch

    import trident_b200 as tb
    from trident_b200 import _lib

    table = _randn((10, 24), "bfloat16", 1)
    for dt in (torch.int32, torch.int64):
        bad = 2 ** 40 if dt == torch.int64 else 2 ** 31 - 1
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = tb.embedding_lookup(table, torch.tensor([3, -1, 9], dtype=dt, device="cuda"), status=status)
        assert int(status) == 0 and bool((got[1] == 0).all()) and torch.equal(got[2], table[9])
        got = tb.embedding_lookup(table, torch.tensor([3, 10, -2, bad], dtype=dt, device="cuda"), status=status)
        assert int(status) == _lib.STATUS_BAD_ID and bool(torch.isnan(got[1:]).all()) and torch.equal(got[0], table[3])
        tb.embedding_lookup(table, torch.tensor([10], dtype=dt, device="cuda"))  # without a status
    empty = torch.empty(0, dtype=torch.int64, device="cuda")
    assert tb.embedding_lookup(table, empty).shape == (0, 24)
    assert bool(torch.isnan(tb.embedding_lookup(table[:0], torch.zeros(2, dtype=torch.int64, device="cuda"))).all())


def test_lookup_gathers_search_results():
    """The ids of a search, -1 where it found fewer than K rows, gather the rows themselves."""
    import torch

    import trident_b200 as tb
    from helpers import build_index, load_case

    f = load_case("g1_int_c1")
    idx = build_index(f)
    xq = torch.from_numpy(f["xq"]).cuda()
    _, ids, _ = idx.search(xq, int(f["nprobe"]), k=10)
    rows = torch.from_numpy(f["xb"]).cuda()
    assert torch.equal(tb.embedding_lookup(rows, ids), rows[ids])


# ---- the lookup's gradient

def _grad_reference(grad, ids, V, scale):
    """(sums, sums of magnitudes, counts) in 64 bits."""
    import torch

    ok = (ids >= 0) & (ids < V)
    i, g = ids[ok].long(), grad[ok].double() * float(np.float32(scale))
    z = lambda: torch.zeros((V, grad.shape[1]), dtype=torch.float64, device="cuda")  # noqa: E731
    return z().index_add_(0, i, g), z().index_add_(0, i, g.abs()), torch.bincount(i, minlength=V)[:, None].double()


def _grad_tol(want, mag, count, out_dtype, old=None):
    tol = (count + 4) * U * mag + ROUND[out_dtype] * want.abs() + TINY[out_dtype]
    if old is not None:
        tol = tol + 2 * U * (old.abs() + mag)
    return tol


GRAD_SHAPES = [
    # without a sort (T <= 1024)
    (1, 1, 1, "spread"), (1, 700, 33, "spread"), (37, 11, 8, "skewed"), (1024, 50, 96, "skewed"), (1000, 3, 960, "same"),
    (600, 5, 130, "none"), (1024, 4000, 2050, "spread"),
    # one, two and three passes of the sort, and the edges of its blocks and of the runs' pieces
    (1025, 1, 16, "spread"), (2048, 512, 32, "skewed"), (2049, 513, 31, "skewed"), (4096, 2000, 1, "skewed"),
    (6145, 262_144, 8, "spread"), (5000, 300_000, 12, "skewed"), (20_011, 70, 128, "skewed"), (1300, 40, 960, "none"),
    (40_000, 3, 64, "same"), (33_333, 2, 9, "spread"), (3000, 1500, 1032, "skewed"),
    # more ids than one cluster sorts, and more than fill the blocks of a pass once
    (140_001, 3000, 8, "skewed"), (131_073, 70_000, 16, "spread"), (1_100_000, 300_000, 4, "skewed"), (200_000, 1, 8, "same"),
    # zeros written beside the sort
    (5000, 20_000, 500, "skewed"),
]


@pytest.mark.parametrize("dtype,out_dtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float16", "float32")])
@pytest.mark.parametrize("T,V,D,kind", GRAD_SHAPES)
def test_lookup_gradient(dtype, out_dtype, T, V, D, kind):
    import torch

    import trident_b200 as tb

    grad, ids = _randn((T, D), dtype, 3), _ids(T, V, 4, kind=kind)
    want, mag, count = _grad_reference(grad, ids, V, 0.3)
    got = tb.embedding_grad(grad, ids, V, scale=0.3, dtype=_dt(out_dtype))
    assert got.dtype == _dt(out_dtype) and got.shape == (V, D)
    _close(got, want, _grad_tol(want, mag, count, out_dtype))
    assert bool((got[(count == 0)[:, 0]] == 0).all())
    assert torch.equal(got, tb.embedding_grad(grad, ids.int(), V, scale=0.3, dtype=_dt(out_dtype)))
    # added to what is there; rows that no id names keep their bits
    old = _randn((V, D), out_dtype, 5)
    out = old.clone()
    assert tb.embedding_grad(grad, ids, V, scale=0.3, out=out, accumulate=True) is out
    want = want + old.double()
    _close(out, want, _grad_tol(want, mag, count, out_dtype, old.double()))
    assert torch.equal(out[(count == 0)[:, 0]], old[(count == 0)[:, 0]])


@pytest.mark.parametrize("T", [300, 5000])
def test_lookup_gradient_strides_and_ids_outside(T):
    import torch

    import trident_b200 as tb
    from trident_b200 import _lib

    V, D = 90, 40
    grad, ids = _randn((T, D), "bfloat16", 6), _ids(T, V, 7)
    want = tb.embedding_grad(grad, ids, V)
    assert torch.equal(tb.embedding_grad(_strided(grad, 3), ids, V), want)       # rows at odd places
    assert torch.equal(tb.embedding_grad(grad.t().contiguous().t(), ids, V), want)  # columns first
    wide = torch.full((V, D + 7), 5.0, dtype=grad.dtype, device="cuda")
    tb.embedding_grad(grad, ids, V, out=wide[:, :D])
    assert torch.equal(wide[:, :D], want) and bool((wide[:, D:] == 5).all())
    # one row for every token (the gradient of a sum), as a broadcast tensor
    row = _randn((1, D), "bfloat16", 8)
    assert torch.equal(tb.embedding_grad(row.expand(T, D), ids, V), tb.embedding_grad(row.repeat(T, 1), ids, V))
    # bad ids give nothing, also where the gradient is not finite
    bad = ids.clone()
    bad[::7] = V + 5
    bad[3::7] = -9
    g = grad.clone()
    g[::7] = float("nan")
    g[3::7] = float("inf")
    g[ids == -1] = float("nan")
    keep = torch.where(((bad >= 0) & (bad < V)), bad, -1)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = tb.embedding_grad(g, bad, V, status=status)
    assert int(status) == _lib.STATUS_BAD_ID
    assert torch.equal(got, tb.embedding_grad(grad, keep, V))
    # a NaN stays in its own row
    g = grad.clone()
    at = int((ids == ids[ids >= 0][0]).nonzero()[0])
    g[at, 2] = float("nan")
    got = tb.embedding_grad(g, ids, V)
    assert int(torch.isnan(got).sum()) == 1 and bool(torch.isnan(got[ids[at], 2]))


def test_lookup_gradient_empty():
    import torch

    import trident_b200 as tb

    none = torch.empty(0, dtype=torch.int64, device="cuda")
    g = torch.empty((0, 6), device="cuda")
    assert bool((tb.embedding_grad(g, none, 4) == 0).all())
    out = torch.ones((4, 6), device="cuda")
    assert bool((tb.embedding_grad(g, none, 4, out=out, accumulate=True) == 1).all())
    assert tb.embedding_grad(g, none, 0).shape == (0, 6)


def test_lookup_gradient_is_the_derivative():
    """<grad, d lookup / d table . step> by central differences of the lookup's definition in 64 bits."""
    import torch

    import trident_b200 as tb

    T, V, D, scale = 1500, 40, 24, 2.5
    ids = _ids(T, V, 9)
    table, gout, step = (_randn(s, "float32", k).double() for s, k in (((V, D), 1), ((T, D), 2), ((V, D), 3)))
    f = lambda w: (torch.where((ids >= 0)[:, None], w[ids.clamp(min=0)], 0.0) * scale * gout).sum()  # noqa: E731
    h = 2.0 ** -10
    diff = (f(table + h * step) - f(table - h * step)) / (2 * h)
    got = tb.embedding_grad(gout.float(), ids, V, scale=scale).double()
    _, mag, count = _grad_reference(gout.float(), ids, V, scale)
    tol = (((count + 4) * U * mag) * step.abs()).sum() + 1e-9 * (mag * step.abs()).sum()  # f is linear: rounding alone
    assert abs((got * step).sum() - diff) <= tol


def test_embedding_offsets_beyond_32_bits():
    """A table of more than 2^32 elements: its last rows are read and their gradients added in their place."""
    import torch

    import trident_b200 as tb

    V, D = 4_200_000, 1032
    assert V * D > 2 ** 32
    table = torch.empty((V, D), dtype=torch.bfloat16, device="cuda")
    rows = torch.tensor([0, 1, 2 ** 32 // D + 1, V - 2, V - 1], device="cuda")
    vals = _randn((5, D), "bfloat16", 1)
    table[rows] = vals
    assert torch.equal(tb.embedding_lookup(table, rows), vals)
    ids = rows.repeat(500)
    grad = _randn((2500, D), "bfloat16", 2)
    want, mag, count = _grad_reference(grad, torch.arange(5, device="cuda").repeat(500), 5, 1.0)
    tb.embedding_grad(grad, ids, V, out=table, accumulate=True)
    want = want + vals.double()
    _close(table[rows], want, _grad_tol(want, mag, count, "bfloat16", vals.double()))


# ---- layer norm

def _norm_depth(D):
    return 64 + D / 1024  # a lane's 32 columns, the warp's 5 steps, 8 warps; a long row: D / 1024 columns


def _norm_reference(x, w, b, eps, dtype):
    x = x.double()
    D = x.shape[-1]
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    var = (d * d).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    w = 1.0 if w is None else w.double()
    b = 0.0 if b is None else b.double()
    y = d * rstd * w + b
    k = _norm_depth(D)
    e_mean = (k + 2) * U * x.abs().mean(-1, keepdim=True)
    e_rstd = (0.5 * ((k + 6) * U + e_mean ** 2 / (var + eps)) + 4 * U) * rstd
    aw = 1.0 if isinstance(w, float) else w.abs()
    tol = aw * (rstd * (e_mean + U * d.abs()) + d.abs() * e_rstd + 4 * U * d.abs() * rstd)
    tol = 1.01 * tol + (2 * U + ROUND[dtype]) * y.abs() + TINY[dtype]
    return (y, tol), (mean[..., 0], 1.01 * e_mean[..., 0] + TINY["float32"]), (rstd[..., 0], 1.01 * e_rstd[..., 0])


NORM_SHAPES = [(1, 1), (1, 8), (5, 7), (33, 96), (100, 128), (3, 960), (17, 961), (9, 1001), (4, 1024), (4, 1025),
               (3, 2050), (2, 4096), (2, 4097), (3, 8192), (2, 8200), (1, 20_001), (2000, 72)]


# as many rows as stay with resident warps: every number of columns a lane, several warps a row, rows that start
# anywhere (at 4-byte places where D is even)
MANY_ROWS = [(40_000, 24), (20_000, 64), (20_001, 128), (19_000, 200), (19_000, 500), (19_001, 960), (19_000, 1024), (10_000, 2048),
             (5000, 4096), (2500, 8192), (5001, 33), (5000, 98), (5000, 201), (5000, 350), (5001, 1001), (5000, 1022), (2600, 2050),
             (1300, 4099), (700, 8190)]


@pytest.mark.parametrize("dtype,param", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("rows,D", NORM_SHAPES + MANY_ROWS)
def test_layer_norm(dtype, param, rows, D):
    import torch

    import trident_b200 as tb

    x = _randn((rows, D), dtype, rows + D, 1.5, 0.7)
    w, b = _randn((D,), param, 1, 0.3, 1.0), _randn((D,), param, 2, 0.3)
    for ww, bb in ((w, b), (None, None), (w, None), (None, b)):
        outs = tb.layer_norm(x, ww, bb, eps=1e-5)
        for got, (want, tol) in zip(outs, _norm_reference(x, ww, bb, 1e-5, dtype)):
            _close(got, want, tol)
    y = tb.layer_norm(x, w, b)[0]
    assert torch.equal(tb.layer_norm(x, w, b, stats=False), y)
    _close(tb.layer_norm(_strided(x, 1), w, b, stats=False), *_norm_reference(x, w, b, 1e-5, dtype)[0])
    inplace = x.clone()
    assert tb.layer_norm(inplace, w, b, out=inplace, stats=False) is inplace and torch.equal(inplace, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,D,pad,skip", [(5000, 96, 8, 0), (5000, 100, 0, 1), (20_000, 64, 5, 3), (300, 97, 4, 1), (20_000, 960, 64, 0)])
def test_layer_norm_of_a_window(dtype, rows, D, pad, skip):
    """Rows inside wider rows, from a column on: strides and bases that allow wide loads and that do not. What lies
    around the window is NaN, and stays."""
    import torch

    import trident_b200 as tb

    wide = torch.full((rows + 1, D + pad + skip), float("nan"), dtype=_dt(dtype), device="cuda")
    x = wide[:rows, skip:skip + D]
    x.copy_(_randn((rows, D), dtype, 1, 1.5, 0.7))
    w, b = _randn((D,), dtype, 2, 0.3, 1.0), _randn((D,), dtype, 3)
    for got, (want, tol) in zip(tb.layer_norm(x, w, b), _norm_reference(x, w, b, 1e-5, dtype)):
        _close(got, want, tol)
    _, mean, rstd = tb.layer_norm(x)
    dy = torch.full_like(wide, float("nan"))[:rows, skip:skip + D]
    dy.copy_(_randn((rows, D), dtype, 4))
    before = wide.clone()
    out = wide[:rows, skip:skip + D]
    y = torch.empty_like(wide)
    y.fill_(7.0)
    tb.layer_norm(x, w, b, out=y[:rows, skip:skip + D], stats=False)
    _close(y[:rows, skip:skip + D], *_norm_reference(x, w, b, 1e-5, dtype)[0])
    assert bool((y[rows:] == 7).all()) and bool((y[:, :skip] == 7).all()) and bool((y[:, skip + D:] == 7).all())
    want = _norm_grad_reference(dy, x, w, mean, rstd, dtype, dtype)
    got = tb.layer_norm_grad(dy, x, w, mean, rstd, out=y[:rows, skip:skip + D])
    for g, (ref, tol) in zip(got, want):
        _close(g, ref, tol)
    assert bool((y[rows:] == 7).all()) and bool((y[:, :skip] == 7).all()) and bool((y[:, skip + D:] == 7).all())
    assert torch.equal(wide.nan_to_num(9.0), before.nan_to_num(9.0)) and out.shape == x.shape
    tb.layer_norm(x, w, b, out=x, stats=False)  # in place
    assert torch.equal(torch.isnan(wide), torch.isnan(before))


def test_layer_norm_values():
    """Constant rows, rows far from zero, and rows that are not finite next to rows that are."""
    import torch

    import trident_b200 as tb

    D = 512
    x = _randn((6, D), "float32", 1)
    x[0] = 0.0
    x[1] = 1e4 + x[1]     # the mean is 1e4 times the deviation: kept by the centred second pass
    x[2, 5] = float("nan")
    x[3, 6] = float("inf")
    x[4] = 3.0
    y, mean, rstd = tb.layer_norm(x, eps=1e-5)
    (wy, ty), (wm, tm), (wr, tr) = _norm_reference(x[[0, 1, 4, 5]], None, None, 1e-5, "float32")
    for got, want, tol in ((y, wy, ty), (mean, wm, tm), (rstd, wr, tr)):
        _close(got[[0, 1, 4, 5]], want, tol)
    assert bool(torch.isnan(y[2:4]).all())
    assert tb.layer_norm(x[:0])[0].shape == (0, D)
    z = x[None, :2].expand(3, 2, D)
    assert torch.equal(tb.layer_norm(z)[0], y[:2].expand(3, 2, D)) and tb.layer_norm(z)[1].shape == (3, 2)


def _norm_grad_reference(dy, x, w, mean, rstd, dtype, param):
    dy, x, m, r = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    rows, D = x.shape
    wd = 1.0 if w is None else w.double()
    xh = (x - m) * r
    exh = 2.01 * U * xh.abs() + TINY["float32"]
    g = dy * wd
    c1, c2 = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
    dx = r * (g - c1 - xh * c2)
    k = _norm_depth(D)
    e1 = (k + 4) * U * g.abs().mean(1, keepdim=True)
    e2 = (k + 8) * U * (g * xh).abs().mean(1, keepdim=True)
    t = r * (U * g.abs() + e1 + xh.abs() * e2 + exh * c2.abs() + 5 * U * (g.abs() + c1.abs() + (xh * c2).abs()))
    tx = 1.01 * t + ROUND[dtype] * dx.abs() + TINY[dtype]
    n = min(rows, rows / 64 + 90) + 10  # a group's rows, then the groups' partial sums
    dw, db = (dy * xh).sum(0), dy.sum(0)
    tw = n * U * (dy * xh).abs().sum(0) + ROUND[param] * dw.abs() + TINY[param]
    tb_ = n * U * dy.abs().sum(0) + ROUND[param] * db.abs() + TINY[param]
    return (dx, tx), (dw, 1.01 * tw), (db, 1.01 * tb_)


@pytest.mark.parametrize("dtype,param", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float32")])
@pytest.mark.parametrize("rows,D", NORM_SHAPES + [(6000, 96), (777, 1032), (130, 4100), (9000, 64), (9000, 128), (3000, 98), (3000, 1001)])
def test_layer_norm_gradient(dtype, param, rows, D):
    import torch

    import trident_b200 as tb

    x, dy = _randn((rows, D), dtype, rows + D, 1.5, 0.7), _randn((rows, D), dtype, 3)
    w = _randn((D,), param, 1, 0.3, 1.0)
    _, mean, rstd = tb.layer_norm(x, eps=1e-5)
    for ww in (w, None):
        outs = tb.layer_norm_grad(dy, x, ww, mean, rstd)
        for got, (want, tol) in zip(outs, _norm_grad_reference(dy, x, ww, mean, rstd, dtype, param if ww is not None else dtype)):
            _close(got, want, tol)
    dx, dw, db = tb.layer_norm_grad(dy, x, w, mean, rstd)
    again = tb.layer_norm_grad(dy, x, w, mean, rstd)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    only, none, none2 = tb.layer_norm_grad(dy, x, w, mean, rstd, param_grads=False)
    assert torch.equal(only, dx) and none is None and none2 is None
    inplace = dy.clone()
    tb.layer_norm_grad(inplace, x, w, mean, rstd, out=inplace)
    assert torch.equal(inplace, dx)


def test_layer_norm_gradient_strides_and_broadcast():
    import torch

    import trident_b200 as tb

    x, dy = _randn((50, 96), "bfloat16", 1), _randn((50, 96), "bfloat16", 2)
    w = _randn((96,), "bfloat16", 3)
    _, mean, rstd = tb.layer_norm(x)
    want = tb.layer_norm_grad(dy, x, w, mean, rstd)
    wide = torch.full((50, 100), 3.0, dtype=x.dtype, device="cuda")
    got = tb.layer_norm_grad(_strided(dy, 4), _strided(x, 8), w, mean, rstd, out=wide[:, :96])
    for a, (ref, tol) in zip(got, _norm_grad_reference(dy, x, w, mean, rstd, "bfloat16", "bfloat16")):
        _close(a, ref, tol)
    assert bool((wide[:, 96:] == 3).all())
    ones = torch.ones((), dtype=x.dtype, device="cuda").expand(50, 96)  # the gradient of a sum
    for a, b in zip(tb.layer_norm_grad(ones, x, w, mean, rstd), tb.layer_norm_grad(ones.contiguous(), x, w, mean, rstd)):
        assert torch.equal(a, b)
    dx, dw, db = tb.layer_norm_grad(dy[:0], x[:0], w, mean[:0], rstd[:0])
    assert dx.shape == (0, 96) and bool((dw == 0).all()) and bool((db == 0).all())


def test_layer_norm_gradient_is_the_derivative():
    """Against central differences of layer norm's definition in 64 bits, along a random direction of each
    input: the difference's own error is h^2 f'''/6, held far below the float32 rounding by h = 2^-12."""
    import torch

    import trident_b200 as tb

    rows, D, eps = 37, 50, 1e-3
    x, w, b, gout = (_randn(s, "float32", k).double() for s, k in (((rows, D), 1), ((D,), 2), ((D,), 3), ((rows, D), 4)))

    def f(x, w, b):
        d = x - x.mean(1, keepdim=True)
        return ((d / torch.sqrt((d * d).mean(1, keepdim=True) + eps) * w + b) * gout).sum()

    _, mean, rstd = tb.layer_norm(x.float(), w.float(), b.float(), eps=eps)
    grads = tb.layer_norm_grad(gout.float(), x.float(), w.float(), mean, rstd)
    h = 2.0 ** -12
    for k, got in enumerate(grads):
        args = [x, w, b]
        step = _randn(args[k].shape, "float32", 10 + k).double()
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * step, args[k] - h * step
        diff = (f(*up) - f(*down)) / (2 * h)
        assert abs((got.double() * step).sum() - diff) <= 1e-5 * (got.double() * step).abs().sum() + 1e-5


# ---- streams

def test_operators_on_another_stream():
    """Work queued on a side stream, with its inputs made there: results as on the default stream."""
    import torch

    import trident_b200 as tb

    def all_of(seed):
        table, ids = _randn((500, 128), "bfloat16", seed), _ids(3000, 500, seed)
        y = tb.embedding_lookup(table, ids, scale=2.0)
        z, mean, rstd = tb.layer_norm(y, table[0], table[1])
        dx, dw, db = tb.layer_norm_grad(z, y, table[0], mean, rstd)
        return [y, z, mean, rstd, dx, dw, db, tb.embedding_grad(dx, ids, 500)]

    want = all_of(1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = all_of(1)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_operators_in_a_graph():
    """A captured step replays on new contents of the same buffers."""
    import torch

    import trident_b200 as tb

    table, ids = _randn((500, 128), "float32", 1), _ids(3000, 500, 1)
    w, b = _randn((128,), "float32", 2), _randn((128,), "float32", 3)

    def step():
        y = tb.embedding_lookup(table, ids)
        z, mean, rstd = tb.layer_norm(y, w, b)
        dx, dw, db = tb.layer_norm_grad(z, y, w, mean, rstd)
        return dw, db, tb.embedding_grad(dx, ids, 500)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step()
    for seed in (5, 6):
        table.copy_(_randn((500, 128), "float32", seed))
        ids.copy_(_ids(3000, 500, seed))
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))


def test_zeros_beside_the_sort_on_streams_and_in_a_graph():
    """A gradient whose zeros are written on the library's second stream: on a side stream, with the output used at
    once after the call, and captured."""
    import torch

    import trident_b200 as tb

    V, D, T = 30_000, 256, 5000
    ids, grad = _ids(T, V, 1), _randn((T, D), "bfloat16", 2)
    want, mag, count = _grad_reference(grad, ids, V, 1.0)
    tol = _grad_tol(want, mag, count, "bfloat16")
    out = torch.full((V, D), 3.0, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(5):
            out.fill_(3.0)
            tb.embedding_grad(grad, ids, V, out=out)
            used = out * 1.0
    side.synchronize()
    _close(used, want, tol)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        tb.embedding_grad(grad, ids, V, out=out)
        used = out * 1.0
    for seed in (3, 4):
        grad.copy_(_randn((T, D), "bfloat16", seed))
        out.fill_(5.0)
        g.replay()
        torch.cuda.synchronize()
        want, mag, count = _grad_reference(grad, ids, V, 1.0)
        _close(used, want, _grad_tol(want, mag, count, "bfloat16"))

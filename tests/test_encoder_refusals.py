"""What the encoder operators refuse: at the C ABI (addresses that are never read) and in Python. No GPU needed."""
import ctypes

import pytest


@pytest.fixture(scope="module")
def L():
    from trident_b200 import _lib, build

    build.build()
    return _lib.lib()


INVALID, WORKSPACE, UNSUPPORTED = 1, 2, 4
A = 1 << 20  # a well-aligned address


def test_lookup_refusals(L):
    def call(table=A, dtype=0, V=10, D=8, ld=8, ids=A, bits=64, T=4, out=A, ld_out=8, status=None):
        return L.trident_embed_lookup(table, dtype, V, D, ld, ids, bits, T, 1.0, out, ld_out, status, None)

    assert call(T=0) == 0  # nothing to do
    for kw, code in (({"dtype": 3}, UNSUPPORTED), ({"dtype": -1}, UNSUPPORTED), ({"bits": 16}, UNSUPPORTED),
                     ({"T": -1}, UNSUPPORTED), ({"T": 1 << 31}, UNSUPPORTED), ({"V": 1 << 31}, UNSUPPORTED),
                     ({"V": -1}, UNSUPPORTED), ({"D": 0}, INVALID), ({"table": None}, INVALID), ({"ids": None}, INVALID),
                     ({"out": None}, INVALID), ({"ld": 7}, INVALID), ({"ld_out": 7}, INVALID), ({"table": A + 2}, INVALID),
                     ({"ids": A + 4}, INVALID), ({"ids": A + 2, "bits": 32}, INVALID), ({"out": A + 1, "dtype": 2}, INVALID),
                     ({"status": A + 2}, INVALID), ({"ld": 1 << 60}, UNSUPPORTED)):
        assert call(**kw) == code, kw


def test_lookup_gradient_refusals(L):
    n = ctypes.c_size_t(0)
    assert L.trident_embed_grad_workspace_size(5000, 100, 16, ctypes.byref(n)) == 0
    need = n.value

    def call(grad=A, dtype=2, ld=16, ids=A, bits=32, T=5000, V=100, D=16, acc=0, out=A, out_dtype=2, ld_out=16, ws=A, size=need):
        return L.trident_embed_grad(grad, dtype, ld, ids, bits, T, V, D, 1.0, acc, out, out_dtype, ld_out, ws, size, None, None)

    for kw, code in (({"dtype": 5}, UNSUPPORTED), ({"out_dtype": 1}, UNSUPPORTED), ({"acc": 2}, INVALID), ({"bits": 8}, UNSUPPORTED),
                     ({"grad": None}, INVALID), ({"out": None}, INVALID), ({"ids": None}, INVALID), ({"ld": 15}, INVALID),
                     ({"ld_out": 15}, INVALID), ({"size": need - 1}, WORKSPACE), ({"ws": None}, WORKSPACE), ({"ws": A + 16}, INVALID),
                     ({"T": -1}, UNSUPPORTED), ({"V": 1 << 31}, UNSUPPORTED), ({"D": 0}, INVALID), ({"out": A + 2, "out_dtype": 0}, INVALID)):
        assert call(**kw) == code, kw
    assert call(T=0, V=0) == 0
    assert L.trident_embed_grad_workspace_size(5000, 100, 0, ctypes.byref(n)) == INVALID
    assert L.trident_embed_grad_workspace_size(5000, 100, 16, None) == INVALID
    assert L.trident_embed_grad_workspace_size(-1, 100, 16, ctypes.byref(n)) == UNSUPPORTED


def test_layer_norm_refusals(L):
    def call(x=A, dtype=2, rows=4, D=8, ld=8, w=A, b=A, pd=0, eps=1e-5, y=A, ld_y=8, mean=A, rstd=A):
        return L.trident_layer_norm(x, dtype, rows, D, ld, w, b, pd, eps, y, ld_y, mean, rstd, None)

    assert call(rows=0) == 0
    for kw, code in (({"dtype": 3}, UNSUPPORTED), ({"pd": 1}, UNSUPPORTED), ({"rows": -1}, UNSUPPORTED), ({"rows": 1 << 31}, UNSUPPORTED),
                     ({"D": 0}, INVALID), ({"x": None}, INVALID), ({"y": None}, INVALID), ({"ld": 7}, INVALID), ({"ld_y": 0}, INVALID),
                     ({"eps": -1.0}, INVALID), ({"eps": float("nan")}, INVALID), ({"w": A + 2}, INVALID), ({"b": A + 1}, INVALID),
                     ({"mean": A + 2}, INVALID), ({"rstd": A + 2}, INVALID)):
        assert call(**kw) == code, kw


def test_layer_norm_gradient_refusals(L):
    n = ctypes.c_size_t(0)
    assert L.trident_layer_norm_grad_workspace_size(40, 16, ctypes.byref(n)) == 0
    need = n.value
    assert L.trident_layer_norm_grad_workspace_size(40, 16, None) == INVALID
    assert L.trident_layer_norm_grad_workspace_size(-1, 16, ctypes.byref(n)) == UNSUPPORTED

    def call(dy=A, ld_dy=16, x=A, ld_x=16, dtype=2, rows=40, D=16, w=A, pd=2, mean=A, rstd=A, dx=A, ld_dx=16, dw=A, db=A, ws=A, size=need):
        return L.trident_layer_norm_grad(dy, ld_dy, x, ld_x, dtype, rows, D, w, pd, mean, rstd, dx, ld_dx, dw, db, ws, size, None)

    for kw, code in (({"dtype": 3}, UNSUPPORTED), ({"pd": 1}, UNSUPPORTED), ({"rows": -1}, UNSUPPORTED), ({"D": 0}, INVALID),
                     ({"dy": None}, INVALID), ({"x": None}, INVALID), ({"dx": None}, INVALID), ({"mean": None}, INVALID),
                     ({"rstd": None}, INVALID), ({"ld_dy": 1}, INVALID), ({"ld_x": 1}, INVALID), ({"ld_dx": 1}, INVALID),
                     ({"size": need - 1}, WORKSPACE), ({"ws": None}, WORKSPACE), ({"ws": A + 128}, INVALID), ({"dw": A + 1}, INVALID),
                     ({"db": A + 1}, INVALID), ({"w": A + 1}, INVALID)):
        assert call(**kw) == code, kw


def test_adamw_refusals(L):
    from trident_b200 import _lib

    def call(count=1, tensor=None, config=None, tensors=True, conf=True):
        t = (_lib.AdamWTensor * 2)()
        for d in t:
            d.param = d.grad = d.m = d.v = A
            d.n = 5
            for k, v in (tensor or {}).items():
                setattr(d, k, v)
        c = _lib.AdamWConfig(param_dtype=2, grad_dtype=2, state_bits=32, step=1, lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8)
        for k, v in (config or {}).items():
            setattr(c, k, v)
        return L.trident_adamw_step(t if tensors else None, count, ctypes.byref(c) if conf else None, None)

    assert call(count=0) == 0
    for kw, code in (({"conf": False}, INVALID), ({"tensors": False}, INVALID), ({"count": -1}, INVALID),
                     ({"config": {"param_dtype": 7}}, UNSUPPORTED), ({"config": {"grad_dtype": 1}}, UNSUPPORTED),
                     ({"config": {"state_bits": 16}}, UNSUPPORTED), ({"config": {"step": 0}}, INVALID),
                     ({"config": {"beta1": 1.0}}, INVALID), ({"config": {"beta2": -0.1}}, INVALID), ({"config": {"eps": -1.0}}, INVALID),
                     ({"config": {"lr": float("nan")}}, INVALID), ({"config": {"weight_decay": -1.0}}, INVALID),
                     ({"config": {"grad_scale": A + 1}}, INVALID), ({"tensor": {"n": -1}}, INVALID), ({"tensor": {"param": None}}, INVALID),
                     ({"tensor": {"grad": None}}, INVALID), ({"tensor": {"m": None}}, INVALID), ({"tensor": {"v": A + 2}}, INVALID),
                     ({"tensor": {"param": A + 1}}, INVALID), ({"tensor": {"master": A + 2}}, INVALID),
                     ({"config": {"state_bits": 8}}, INVALID),  # no scales
                     ({"tensor": {"master": A}, "config": {"param_dtype": 0, "grad_dtype": 0}}, INVALID),
                     ({"tensor": {"n": 1 << 50}}, UNSUPPORTED)):
        assert call(**kw) == code, kw
    assert "2^31" in _lib.last_error()


def test_python_refuses_host_tensors_and_other_types():
    import torch

    import trident_b200 as tb

    table, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        tb.embedding_lookup(table, ids)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        tb.embedding_lookup(table.double(), ids)
    with pytest.raises(ValueError, match="CUDA"):
        tb.embedding_grad(torch.zeros(3, 8), ids, 4)
    with pytest.raises(ValueError, match="CUDA"):
        tb.layer_norm(table)
    with pytest.raises(ValueError, match="CUDA"):
        tb.layer_norm_grad(table, table, None, ids, ids)
    with pytest.raises(ValueError, match="CUDA"):
        tb.AdamW([table])
    with pytest.raises(ValueError, match="state_bits"):
        tb.AdamW([table], state_bits=4)
    with pytest.raises(ValueError, match="empty"):
        tb.AdamW([])


@pytest.mark.gpu
def test_python_refusals_on_the_device():
    import torch

    import trident_b200 as tb

    table, ids = torch.zeros(4, 8, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (lambda: tb.embedding_lookup(table[0], ids), lambda: tb.embedding_lookup(table, ids.float()),
                lambda: tb.embedding_lookup(table, ids.cpu()), lambda: tb.embedding_lookup(table, ids, out=table),
                lambda: tb.embedding_lookup(table, ids, status=ids),
                lambda: tb.embedding_lookup(table, ids, out=torch.empty(8, 3, device="cuda").t()),
                lambda: tb.embedding_grad(table, ids, 4), lambda: tb.embedding_grad(table[:3], ids, 4, accumulate=True),
                lambda: tb.embedding_grad(table[:3], ids, 4, out=table[:3]),
                lambda: tb.layer_norm(table, ids), lambda: tb.layer_norm(table, table[0], table[0].half()),
                lambda: tb.layer_norm(table, out=table[:2]), lambda: tb.layer_norm_grad(table, table[:2], None, table[0], table[0]),
                lambda: tb.layer_norm_grad(table, table, None, ids, ids), lambda: tb.AdamW([table.t()]),
                lambda: tb.AdamW([table], state={"exp_avg": [table]}), lambda: tb.AdamW([table], step=-1),
                lambda: tb.AdamW([table]).step([]), lambda: tb.AdamW([table]).step([table[:2]]),
                lambda: tb.AdamW([table]).step([table.half()]), lambda: tb.AdamW([table]).step([table], grad_scale=ids)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(tb._lib.TridentError, match="eps"):
        tb.layer_norm(table, eps=-1.0)

"""The query-encoder operators: embedding lookup and its gradient, layer norm and its gradient, AdamW.

Each case is one call of one operator at sizes of an encoder in front of an index: queries of 32
tokens, batches of 1,000 and 10,000 queries, vectors of 96, 128 and 960 dims, tables of 65,536 and
262,144 rows (the list counts of the search benchmark, also used as vocabulary sizes here).
"""
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 256                      # elements of a tensor that share the scales of an 8-bit state
G32, R32, M32 = 0x9E3779B9, 0x6A09E667, 0xFFFFFFFF
LR, B1, B2, ADAM_EPS, DECAY, SEED = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 12345
LN_EPS = 1e-5


def listed():
    return [
        # one query's 32 tokens: serving, where latency counts
        {"name": "lookup_query", "op": "lookup", "dtype": "bf16", "ids": "i64", "T": 32, "V": 65536, "D": 960, "pad": 0.0},
        # a batch of 10,000 queries padded to 32 tokens: encoding for a search of that batch
        {"name": "lookup_batch", "op": "lookup", "dtype": "bf16", "ids": "i64", "T": 320000, "V": 65536, "D": 960, "pad": 0.2},
        # an odd width and table, whose rows start at no 16-byte boundary, 32-bit ids
        {"name": "lookup_odd", "op": "lookup", "dtype": "f32", "ids": "i32", "T": 33333, "V": 30011, "D": 97, "pad": 0.1},
        # the table's gradient for a training batch of 1,000 queries, the whole table written
        {"name": "table_grad", "op": "table_grad", "dtype": "bf16", "out": "bf16", "ids": "i64", "T": 32000, "V": 65536, "D": 960,
         "pad": 0.1, "accumulate": False},
        # gradient accumulation of 10,000 queries into a large table's 32-bit gradient
        {"name": "table_grad_add", "op": "table_grad", "dtype": "bf16", "out": "f32", "ids": "i64", "T": 320000, "V": 262144, "D": 128,
         "pad": 0.2, "accumulate": True},
        # layer norm of one query's tokens
        {"name": "norm_query", "op": "norm", "dtype": "bf16", "param": "bf16", "rows": 32, "D": 960},
        # of the tokens of 10,000 queries
        {"name": "norm_batch", "op": "norm", "dtype": "bf16", "param": "bf16", "rows": 320000, "D": 960},
        # backward, 32-bit training at an odd width and row count
        {"name": "norm_grad_odd", "op": "norm_grad", "dtype": "f32", "param": "f32", "rows": 10007, "D": 1001},
        # backward for the tokens of 10,000 queries, 32-bit weights
        {"name": "norm_grad_batch", "op": "norm_grad", "dtype": "bf16", "param": "f32", "rows": 320000, "D": 960},
        # the step of a small encoder (a few small tensors): launch latency
        {"name": "adamw_small", "op": "adamw", "dtype": "f32", "master": False, "bits": 32, "tensors": 6, "values": 100000, "clip": False},
        # 16-bit parameters with 32-bit master copies and states, ragged tensors, clipped gradients
        {"name": "adamw_master", "op": "adamw", "dtype": "bf16", "master": True, "bits": 32, "tensors": 40, "values": 40000000, "clip": True},
        # the large tables' step with 8-bit states
        {"name": "adamw_8bit", "op": "adamw", "dtype": "bf16", "master": False, "bits": 8, "tensors": 12, "values": 100000000, "clip": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["lookup", "table_grad", "norm", "norm_grad", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "adamw":
        bits = rng.choice([8, 32])
        values = _log(rng, 1000, 40000000)
        return {"op": op, "dtype": dtype, "master": dtype != "f32" and rng.random() < 0.5, "bits": bits,
                "tensors": min(_log(rng, 1, 60), values // 100), "values": values, "clip": rng.random() < 0.5}
    D = _log(rng, 8, 2048)
    if rng.random() < 0.5:
        D = max(8, D // 8 * 8)  # half of the widths allow wide loads
    if op in ("norm", "norm_grad"):
        rows = _log(rng, 1, min(320000, 150000000 // D))
        return {"op": op, "dtype": dtype, "param": rng.choice([dtype, "f32"]), "rows": rows, "D": D}
    V = _log(rng, 100, min(262144, 80000000 // D))
    T = _log(rng, 1, min(320000, 80000000 // D))
    case = {"op": op, "dtype": dtype, "ids": rng.choice(["i32", "i64"]), "T": T, "V": V, "D": D, "pad": rng.choice([0.0, 0.1, 0.5])}
    if op == "table_grad":
        case.update(out=rng.choice([dtype, "f32"]), accumulate=rng.random() < 0.5)
    return case


# ---- inputs

def _gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(int(seed))


def _randn(gen, shape, dtype, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dtype)


def _stride(V):
    """Spreads the frequent tokens over the table: multiplication by a number prime to V."""
    a = max(1, int(V * 0.6180339887) | 1)
    while math.gcd(a, V) != 1:
        a += 2
    return a


def _ids(gen, case):
    """Token ids whose frequency falls as one over their rank, and -1 where a query is padded."""
    T, V = case["T"], case["V"]
    u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
    rank = torch.clamp(torch.exp(u * math.log(V + 1)).floor().long() - 1, 0, V - 1)
    ids = rank * _stride(V) % V
    pad = torch.rand(T, generator=gen, device="cuda") < case["pad"]
    return torch.where(pad, -1, ids).to(torch.int32 if case["ids"] == "i32" else torch.int64)


def _distinct(case):
    """The expected number of table rows that the ids name."""
    r = np.arange(case["V"], dtype=np.float64)
    p = np.log((r + 2) / (r + 1)) / math.log(case["V"] + 1) * (1 - case["pad"])
    return float(-np.expm1(case["T"] * np.log1p(-np.minimum(p, 1 - 1e-12))).sum())


def _sizes(case):
    """Ragged tensor sizes (the same for every seed), and where each starts in the padded buffer."""
    rng = random.Random(case["values"] * 64 + case["tensors"])
    share = [math.exp(rng.uniform(0, 4)) for _ in range(case["tensors"])]
    sizes = [max(1, int(case["values"] * s / sum(share))) for s in share]
    starts, at = [], 0
    for n in sizes:
        starts.append(at)
        at += -(-n // BLOCK) * BLOCK
    return sizes, starts, at


def prepare(case, seed):
    gen = _gen(seed)
    dt = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "lookup":
        s["table"] = _randn(gen, (case["V"], case["D"]), dt, 0.05)
        s["ids"] = _ids(gen, case)
        s["scale"] = math.sqrt(case["D"])
    elif case["op"] == "table_grad":
        s["ids"] = _ids(gen, case)
        s["grad"] = _randn(gen, (case["T"], case["D"]), dt, 0.01)
        s["scale"] = math.sqrt(case["D"])
        if case["accumulate"]:
            s["total"] = _randn(gen, (case["V"], case["D"]), DTYPES[case["out"]], 0.1)
    elif case["op"] in ("norm", "norm_grad"):
        R, D = case["rows"], case["D"]
        row = torch.randn(R, 1, generator=gen, device="cuda")
        x = torch.randn(R, D, generator=gen, device="cuda").mul_(1.5).add_(row)
        s["x"] = x.to(dt)
        s["w"] = _randn(gen, (D,), torch.float32, 0.2).add_(1).to(DTYPES[case["param"]])
        s["b"] = _randn(gen, (D,), torch.float32, 0.2).to(DTYPES[case["param"]])
        if case["op"] == "norm_grad":
            x = s["x"].float()
            s["mean"] = x.mean(1)
            s["rstd"] = 1 / torch.sqrt((x - s["mean"][:, None]).square_().mean(1) + LN_EPS)
            s["dy"] = _randn(gen, (R, D), dt, 0.1)
    else:
        sizes, starts, total = _sizes(case)
        live = torch.zeros(total, dtype=torch.bool, device="cuda")
        for n, at in zip(sizes, starts):
            live[at:at + n] = True
        # gradients whose size differs from value to value over some orders of magnitude
        size = torch.exp(torch.randn(total, generator=gen, device="cuda") * 1.5 - 6) * live
        p = torch.randn(total, generator=gen, device="cuda").mul_(0.05) * live
        g = size * torch.randn(total, generator=gen, device="cuda")
        m = size * torch.randn(total, generator=gen, device="cuda").mul_(0.3)
        root = size * (0.7 + 0.6 * torch.rand(total, generator=gen, device="cuda"))
        s["step"] = 1 + int(seed) % 1000
        s["g"] = g.to(dt)
        s["p"] = p.to(dt)
        if case["master"]:
            s["master"] = p
        if case["clip"]:
            s["clip"] = torch.rand(1, generator=gen, device="cuda").mul_(0.5).add_(0.5)
        if case["bits"] == 32:
            s["m"], s["v"] = m, root * root
        else:
            for name, x in (("m", m), ("s", root)):
                x = x.view(-1, BLOCK)
                top = x.abs().amax(1, keepdim=True)
                s[name + "_scale"] = (top / torch.full_like(top, 448.0)).view(-1)
                inv = torch.where(top > 0, 448.0 / top, torch.zeros_like(top))
                s[name + "8"] = (x * inv).clamp_(-448, 448).to(torch.float8_e4m3fn).view(-1)
        if own:
            from trident_b200 import AdamW

            cut = lambda t: [t[at:at + n] for n, at in zip(sizes, starts)]  # noqa: E731
            blocks = lambda t: [t[at // BLOCK:(at + n + BLOCK - 1) // BLOCK] for n, at in zip(sizes, starts)]  # noqa: E731
            if case["bits"] == 32:
                state = {"exp_avg": cut(s["m"]), "exp_avg_sq": cut(s["v"])}
            else:
                state = {"exp_avg": cut(s["m8"]), "exp_avg_scale": blocks(s["m_scale"]),
                         "exp_avg_sq_root": cut(s["s8"]), "exp_avg_sq_root_scale": blocks(s["s_scale"])}
            if case["master"]:
                state["master"] = cut(s["master"])
            s["opt"] = AdamW(cut(s["p"]), lr=LR, betas=(B1, B2), eps=ADAM_EPS, weight_decay=DECAY, state_bits=case["bits"],
                             master=case["master"], seed=SEED, state=state, step=s["step"] - 1)
            s["grads"] = cut(s["g"])
    return s


# ---- one pass

def run(state):
    return (_run_own if own else _run_plain)(state, state["case"])


def _adam_outputs(s, case):
    names = ["p", "m", "v"] if case["bits"] == 32 else ["p", "m8", "m_scale", "s8", "s_scale"]
    return {n: s[n] for n in names + (["master"] if case["master"] else [])}


def _run_own(s, case):
    import trident_b200 as tb

    if case["op"] == "lookup":
        return tb.embedding_lookup(s["table"], s["ids"], scale=s["scale"])
    if case["op"] == "table_grad":
        if case["accumulate"]:
            return tb.embedding_grad(s["grad"], s["ids"], case["V"], scale=s["scale"], out=s["total"], accumulate=True)
        return tb.embedding_grad(s["grad"], s["ids"], case["V"], scale=s["scale"], dtype=DTYPES[case["out"]])
    if case["op"] == "norm":
        return tb.layer_norm(s["x"], s["w"], s["b"], eps=LN_EPS)
    if case["op"] == "norm_grad":
        return tb.layer_norm_grad(s["dy"], s["x"], s["w"], s["mean"], s["rstd"])
    s["opt"].step(s["grads"], grad_scale=s.get("clip"))
    return _adam_outputs(s, case)


def _run_plain(s, case):
    if case["op"] == "lookup":
        ids, table = s["ids"], s["table"]
        rows = table[ids.clamp(min=0)].float() * s["scale"]
        return torch.where((ids >= 0)[:, None], rows, 0.0).to(table.dtype)
    if case["op"] == "table_grad":
        ids, out = s["ids"].long(), DTYPES[case["out"]]
        rows = torch.where((ids >= 0)[:, None], s["grad"].float() * s["scale"], 0.0)
        if not case["accumulate"]:
            return torch.zeros((case["V"], case["D"]), device="cuda").index_add_(0, ids.clamp(min=0), rows).to(out)
        if out == torch.float32:
            return s["total"].index_add_(0, ids.clamp(min=0), rows)
        return s["total"].copy_(s["total"].float().index_add_(0, ids.clamp(min=0), rows))
    if case["op"] == "norm":
        x = s["x"].float()
        mean = x.sum(1) / case["D"]
        x = x - mean[:, None]
        rstd = 1 / torch.sqrt((x * x).sum(1) / case["D"] + LN_EPS)
        return (x * rstd[:, None] * s["w"].float() + s["b"].float()).to(s["x"].dtype), mean, rstd
    if case["op"] == "norm_grad":
        dy, rstd = s["dy"].float(), s["rstd"][:, None]
        xh = (s["x"].float() - s["mean"][:, None]) * rstd
        g = dy * s["w"].float()
        dx = rstd * (g - g.sum(1, keepdim=True) / case["D"] - xh * ((g * xh).sum(1, keepdim=True) / case["D"]))
        return dx.to(s["x"].dtype), (dy * xh).sum(0).to(s["w"].dtype), dy.sum(0).to(s["w"].dtype)
    return _adamw_plain(s, case)


def _adamw_plain(s, case):
    t = s["step"]
    s["step"] = t + 1
    g = s["g"].float()
    if case["clip"]:
        g = g * s["clip"]
    if case["bits"] == 32:
        m, v = s["m"], s["v"]
    else:
        m = (s["m8"].float().view(-1, BLOCK) * s["m_scale"][:, None]).view(-1)
        root = (s["s8"].float().view(-1, BLOCK) * s["s_scale"][:, None]).view(-1)
        v = root * root
    m = m * B1 + g * (1 - B1)
    v = v * B2 + (g * g) * (1 - B2)
    root = torch.sqrt(v)
    p = s["master"] if case["master"] else s["p"].float()
    p = p * (1 - LR * DECAY) - m * (LR / (1 - B1 ** t)) / (root * (1 / math.sqrt(1 - B2 ** t)) + ADAM_EPS)
    s["p"].copy_(p)
    if case["master"]:
        s["master"].copy_(p)
    if case["bits"] == 32:
        s["m"].copy_(m)
        s["v"].copy_(v)
        return _adam_outputs(s, case)
    # m to the nearest value; sqrt(v) up or down at random, with the chance that keeps its mean,
    # by 16 random bits for each value (a hash of the step and the value's place)
    top = m.view(-1, BLOCK).abs().amax(1, keepdim=True)
    live = top >= 1e-30
    inv = torch.where(live, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    s["m8"].copy_((m.view(-1, BLOCK) * inv).clamp(-448, 448).view(-1))
    s["m_scale"].copy_(torch.where(live, top / torch.full_like(top, 448.0), torch.zeros_like(top)).view(-1))
    top = root.view(-1, BLOCK).amax(1, keepdim=True)
    live = top >= 1e-30
    inv = torch.where(live, torch.full_like(top, 448.0) / top, torch.zeros_like(top))
    u = (root.view(-1, BLOCK) * inv).clamp(max=448).view(-1)
    at = torch.arange(u.numel() // 2, device="cuda")
    h = (at * G32 + ((SEED + t * R32) & M32)) & M32
    h = ((h ^ (h >> 16)) * R32) & M32
    h = ((h ^ (h >> 15)) * G32) & M32
    r = torch.stack([h & 0xFFFF, h >> 16], 1).view(-1).to(torch.int32) * 16
    q = ((u.view(torch.int32) + r) & ~0xFFFFF).view(torch.float32)
    s["s8"].copy_(torch.where(u > 0, q.clamp(2.0 ** -9, 448.0), 0.0))
    s["s_scale"].copy_(torch.where(live, top / torch.full_like(top, 448.0), torch.zeros_like(top)).view(-1))
    return _adam_outputs(s, case)


# ---- what a pass cannot do without

def work(case):
    op, e = case["op"], SIZE[case["dtype"]]
    if op in ("lookup", "table_grad"):
        T, D = case["T"], case["D"]
        n, ids = _distinct(case), T * (4 if case["ids"] == "i32" else 8)
        if op == "lookup":
            return {"bytes": T * D * e + n * D * e + ids, "flops": T * D}
        o = SIZE[case["out"]]
        table = 2 * n * D * o if case["accumulate"] else case["V"] * D * o
        return {"bytes": T * (1 - case["pad"]) * D * e + ids + table, "flops": T * D}
    if op in ("norm", "norm_grad"):
        n, par = case["rows"] * case["D"], case["D"] * SIZE[case["param"]]
        if op == "norm":
            return {"bytes": 2 * n * e + 2 * par + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * e + 3 * par + 8 * case["rows"], "flops": 14 * n}
    n = sum(_sizes(case)[0])
    each = 3 * e + (8 if case["master"] else 0) - (e if case["master"] else 0)  # a master copy is read in the parameter's place
    each += 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * each, "flops": 16 * n}


# ---- the definitions in 64 bits

def exact(case, seed):
    s = prepare({**case}, seed)
    d = lambda name: s[name].to(torch.float64)  # noqa: E731
    if case["op"] == "lookup":
        table = torch.cat([d("table"), torch.zeros(1, case["D"], dtype=torch.float64, device="cuda")])  # row V: a padded token's
        ids = s["ids"].long()
        return torch.index_select(table, 0, torch.where(ids < 0, case["V"], ids)).mul_(s["scale"])
    if case["op"] == "table_grad":
        order = torch.sort(s["ids"].long(), stable=True).indices
        ids = s["ids"].long()[order]
        order, ids = order[ids >= 0], ids[ids >= 0]
        out = d("total") if case["accumulate"] else torch.zeros((case["V"], case["D"]), dtype=torch.float64, device="cuda")
        return out.index_add_(0, ids, d("grad")[order] * s["scale"])
    if case["op"] == "norm":
        x = d("x")
        mean = x.mean(1)
        var = torch.var(x, 1, correction=0)
        rstd = (var + LN_EPS) ** -0.5
        return (x - mean[:, None]) * rstd[:, None] * d("w") + d("b"), mean, rstd
    if case["op"] == "norm_grad":
        # dx = J^T (w dy) with J = r (I - 1 1^T / D - xh xh^T / D)
        r = d("rstd")[:, None]
        xh = (d("x") - d("mean")[:, None]) * r
        dy = d("dy")
        dw, db = torch.einsum("rd,rd->d", dy, xh), dy.sum(0)
        dy = dy * d("w")
        along = torch.einsum("rd,rd->r", dy, xh)[:, None]
        return r * (dy - (dy.mean(1, keepdim=True) + xh * along / case["D"])), dw, db
    t = s["step"]
    g = d("g") * (float(s["clip"]) if case["clip"] else 1.0)
    if case["bits"] == 32:
        m, v = d("m"), d("v")
    else:
        m = d("m8") * d("m_scale").repeat_interleave(BLOCK)
        v = (d("s8") * d("s_scale").repeat_interleave(BLOCK)) ** 2
    m = B1 * m + (1 - B1) * g
    v = B2 * v + (1 - B2) * g ** 2
    p = d("master") if case["master"] else d("p")
    p = p - LR * DECAY * p - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)) ** 0.5 + ADAM_EPS)
    out = {"p": p}
    if case["master"]:
        out["master"] = p
    if case["bits"] == 32:
        out.update(m=m, v=v)
    else:  # the 8-bit values depend on how they are rounded, their scales do not
        out.update(m8=None, s8=None, m_scale=m.view(-1, BLOCK).abs().amax(1) / 448, s_scale=v.view(-1, BLOCK).amax(1) ** 0.5 / 448)
    return out

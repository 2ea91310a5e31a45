"""Cases of the learned head's operators: the softmax cross entropy over a whole catalogue with its gradients, the root-mean-square norm with the
residual's addition (with its gradients, and with an output in 8 bits), and the product of 8-bit rows with a scale for each row of both sides.

`run` computes a case in its plain form (elementary torch operations in 32 bits), or with `own` set by the calls that a user makes of `hwer`."""
import os
import sys

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LOGIT_SCALE = 20.0      # 1 / temperature: cosine similarities in [-1, 1] become logits in [-20, 20]
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one training pass over the MovieLens-100K shape: every user against every item, float32 rows as the index holds them
        dict(name="ce_ml100k_f32", op="ce", rows=943, classes=1682, d=64, type="f32", bias=False),
        # a batch of users against the MovieLens-20M catalogue, float32 rows
        dict(name="ce_ml20m_batch_f32", op="ce", rows=4096, classes=26744, d=128, type="f32", bias=False),
        # a ragged batch, an odd catalogue and width, half precision, with an offset for each item (log-popularity; retired items at -inf)
        dict(name="ce_odd_bias_f16", op="ce", rows=1037, classes=50021, d=250, type="f16", bias=True),
        # a batch of 4 096 queries against one 1.25 M-item shard of a large catalogue
        dict(name="ce_shard_bf16", op="ce", rows=4096, classes=1250000, d=128, type="bf16", bias=False),
        # a tower's norm in a training step: norm and residual forward, then their gradients
        dict(name="norm_train_bf16", op="norm", rows=16384, d=1024, type="bf16", weight="bf16"),
        # the same over an odd number of narrow float32 rows
        dict(name="norm_train_odd_f32", op="norm", rows=9743, d=250, type="f32", weight="f32"),
        # one query while serving: norm, residual and 8-bit codes of a single row
        dict(name="norm_q8_one_row_bf16", op="norm_q8", rows=1, d=4096, type="bf16", weight="bf16", residual=True),
        # a large batch on its way into an 8-bit layer
        dict(name="norm_q8_batch_bf16", op="norm_q8", rows=32768, d=2048, type="bf16", weight="f32", residual=True),
        # an 8-bit layer for one query: every weight is read once for a single row
        dict(name="matmul_q8_one_row", op="matmul_q8", m=1, n=8192, k=8192, type="bf16", bias=False),
        # scores of a ragged handful of queries against the MovieLens-1M catalogue
        dict(name="matmul_q8_odd_f32", op="matmul_q8", m=37, n=3706, k=250, type="f32", bias=True),
        # all scores of 4 096 queries against the MovieLens-20M catalogue
        dict(name="matmul_q8_catalogue", op="matmul_q8", m=4096, n=26744, k=128, type="bf16", bias=False),
        # an 8-bit layer over a large batch
        dict(name="matmul_q8_layer", op="matmul_q8", m=8192, n=8192, k=4096, type="bf16", bias=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    op = rng.choice(["ce", "ce", "norm", "norm_q8", "matmul_q8", "matmul_q8"])
    kind = rng.choice(["f32", "f16", "bf16"])
    if op == "ce":
        rows, classes = _log(rng, 1, 8192), _log(rng, 2, 1250000)
        d = rng.choice([64, 128, 256, rng.randint(1, 256), rng.randint(1, 256)])
        while rows * classes > 4096 * 1250000 // 4:
            rows = (rows + 1) // 2
        return dict(op="ce", rows=rows, classes=classes, d=d, type=kind, bias=rng.random() < 0.4)
    if op == "matmul_q8":
        m, n, k = _log(rng, 1, 8192), _log(rng, 1, 65536), _log(rng, 8, 8192)
        while m * n > 8192 * 8192 or m * n * k > 8192 * 8192 * 4096:
            m = (m + 1) // 2
        return dict(op="matmul_q8", m=m, n=n, k=k, type=kind, bias=rng.random() < 0.5)
    rows, d = _log(rng, 1, 65536), _log(rng, 8, 16384)
    while rows * d > 32768 * 2048:
        rows = (rows + 1) // 2
    case = dict(op=op, rows=rows, d=d, type=kind, weight=rng.choice(["f32", kind]))
    if op == "norm_q8":
        case["residual"] = rng.random() < 0.6
    return case


def work(case):
    s = SIZE[case["type"]]
    if case["op"] == "ce":
        n, v, d = case["rows"], case["classes"], case["d"]
        extra = 8 * v if case["bias"] else 0                       # the offsets and their gradient
        return {"bytes": 2 * s * (n + v) * d + 8 * n + 4 + extra,     # rows in, gradients out, targets, the loss
                "flops": 6 * n * v * d + 5 * n * v}                # logits, two gradients; maximum, exponential, sums
    if case["op"] == "matmul_q8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + (4 * n if case["bias"] else 0) + s * m * n, "flops": 2 * m * n * k}
    n, d, w = case["rows"], case["d"], SIZE[case["weight"]]
    if case["op"] == "norm":
        # forward: x, residual -> y, h; backward: dy, dh (h is there from the forward, and is read again) -> dx, dweight
        return {"bytes": 8 * s * n * d + 2 * w * d, "flops": 16 * n * d}
    return {"bytes": n * d * ((3 if case["residual"] else 1) * s + 4) + w * d, "flops": 8 * n * d}


# ---------------------------------------------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _ce_inputs(case, seed):
    g = _generator(seed)
    n, v, d, t = case["rows"], case["classes"], case["d"], TYPES[case["type"]]
    table = _normal(g, v, d)
    table /= table.norm(dim=1, keepdim=True).clamp_min(1e-6)
    # popularity falls off along the catalogue, and a query leans towards the item that was chosen next
    target = (v * torch.rand(n, generator=g, device="cuda") ** 3).long().clamp_max(v - 1)
    queries = 0.5 * table[target] + 0.9 * _normal(g, n, d) / d ** 0.5
    queries /= queries.norm(dim=1, keepdim=True).clamp_min(1e-6)
    bias = None
    if case["bias"]:
        bias = -torch.log1p(torch.arange(v, device="cuda").float()) * 0.3 + 0.1 * _normal(g, v)
        retired = torch.arange(v, device="cuda") % 97 == 5
        bias[retired] = -float("inf")
        target = torch.where(retired[target], -1, target)
    if n > 8:
        target[torch.rand(n, generator=g, device="cuda") < 0.02] = -1          # rows without a known next item
    return queries.to(t), table.to(t), target, bias


def _norm_inputs(case, seed):
    g = _generator(seed)
    n, d, t = case["rows"], case["d"], TYPES[case["type"]]
    s = dict(x=_normal(g, n, d).to(t), weight=(1 + 0.2 * _normal(g, d)).to(TYPES[case["weight"]]), residual=None)
    if case["op"] == "norm" or case["residual"]:
        stream = 2 * _normal(g, n, d)
        stream[:, :: max(1, d // 3)] *= 6                          # a residual stream has a few strong columns
        s["residual"] = stream.to(t)
    if case["op"] == "norm":
        s["dy"], s["dh"] = _normal(g, n, d).to(t), (0.5 * _normal(g, n, d)).to(t)
    return s


def _q8(g, rows, k):
    x = _normal(g, rows, k)
    top = x.abs().amax(dim=1, keepdim=True).clamp_min(1e-6)
    return (x * (127 / top)).round().to(torch.int8), (top / 127).reshape(-1)


def _matmul_inputs(case, seed):
    g = _generator(seed)
    a, a_scale = _q8(g, case["m"], case["k"])
    b, b_scale = _q8(g, case["n"], case["k"])
    return dict(a=a, a_scale=a_scale, b=b, b_scale=b_scale, bias=_normal(g, case["n"]) if case["bias"] else None)


def _inputs(case, seed):
    if case["op"] == "ce":
        return dict(zip(("queries", "table", "target", "bias"), _ce_inputs(case, seed)))
    return _matmul_inputs(case, seed) if case["op"] == "matmul_q8" else _norm_inputs(case, seed)


def prepare(case, seed):
    return dict(case=dict(case), **_inputs(case, seed))


# ---------------------------------------------------------------------------------------------------------------- one pass
def _plain_ce(s):
    x, e, t = s["queries"].float(), s["table"].float(), s["target"]
    z = (x * LOGIT_SCALE) @ e.t()
    if s["bias"] is not None:
        z += s["bias"]
    counted = t >= 0
    at = t.clamp_min(0)[:, None]
    z_t = z.gather(1, at)[:, 0]
    top = z.amax(dim=1, keepdim=True)
    p = z.sub_(top).exp_()
    total = p.sum(dim=1, keepdim=True)
    loss_rows = total.log()[:, 0] + top[:, 0] - z_t
    n = counted.sum().clamp_min(1).float()
    loss = torch.where(counted, loss_rows, 0).sum() / n
    p /= total
    p.scatter_add_(1, at, torch.full_like(z_t, -1)[:, None])
    p *= (counted.float() / n)[:, None]
    out = (loss, ((p @ e) * LOGIT_SCALE).to(s["queries"].dtype), ((p.t() @ x) * LOGIT_SCALE).to(s["table"].dtype))
    return out if s["bias"] is None else out + (p.sum(dim=0),)


def _plain_norm(s):
    w = s["weight"].float()
    h = (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = h.float()
    rstd = (f.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    y = f * rstd * w
    dy = s["dy"].float()
    dw = (dy * f * rstd).sum(dim=0)
    gy = dy * w
    dx = rstd * (gy - f * (rstd.square() * (gy * f).mean(dim=1, keepdim=True))) + s["dh"].float()
    return y.to(h.dtype), h, dx.to(h.dtype), dw.to(s["weight"].dtype)


def _plain_norm_q8(s):
    # codes next to a border between two of them need the quotient in 64 bits
    h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["x"].dtype)
    f = h.float()
    rstd = (f.square().mean(dim=1, keepdim=True) + EPS).rsqrt()
    v = h.double() * s["weight"].double()
    top = v.abs().amax(dim=1, keepdim=True)
    codes = torch.where(top > 0, 127 * v / top, 0).round()
    y = codes.float() * (top.float() * rstd / 127)
    return (y,) if s["residual"] is None else (y, h)


def _plain_matmul_q8(s):
    out = (s["a"].float() @ s["b"].float().t()) * s["a_scale"][:, None] * s["b_scale"]
    if s["bias"] is not None:
        out += s["bias"]
    return out.to(TYPES[s["case"]["type"]])


def _own(s):
    path = os.path.join(os.getcwd(), "hybrid-weighted-embedding-recommender_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import hwer
    op = s["case"]["op"]
    if op == "ce":
        return hwer.catalogue_cross_entropy_grads(s["queries"], s["table"], s["target"], scale=LOGIT_SCALE, bias=s["bias"])
    if op == "norm":
        y, h = hwer.rms_norm(s["x"], s["weight"], s["residual"], eps=EPS)
        dx, dw = hwer.rms_norm_grads(s["dy"], h, s["weight"], eps=EPS, dh=s["dh"])
        return y, h, dx, dw
    if op == "norm_q8":
        out = hwer.rms_norm_q8(s["x"], s["weight"], s["residual"], eps=EPS)
        return (out[0] * out[1][:, None],) + tuple(out[2:])
    return hwer.matmul_q8(s["a"], s["a_scale"], s["b"], s["b_scale"], bias=s["bias"], out_dtype=TYPES[s["case"]["type"]])


def run(state):
    if own:
        return _own(state)
    return {"ce": _plain_ce, "norm": _plain_norm, "norm_q8": _plain_norm_q8, "matmul_q8": _plain_matmul_q8}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_ce(case, s):
    x, e, t, bias = s["queries"].double(), s["table"].double(), s["target"], s["bias"]
    n_counted = max(1, int((t >= 0).sum()))
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    dx, de = torch.zeros_like(x), torch.zeros_like(e)
    db = torch.zeros(len(e), dtype=torch.float64, device="cuda")
    step = max(1, (1 << 29) // len(e))
    for r in range(0, len(x), step):
        keep = t[r:r + step] >= 0
        xs, ts = x[r:r + step][keep], t[r:r + step][keep]
        if not len(xs):
            continue
        z = LOGIT_SCALE * (xs @ e.t())
        if bias is not None:
            z += bias.double()
        lse = torch.logsumexp(z, dim=1)
        at = torch.arange(len(xs), device="cuda")
        loss += (lse - z[at, ts]).sum()
        z.sub_(lse[:, None]).exp_()
        z[at, ts] -= 1
        g = torch.zeros((len(keep), x.shape[1]), dtype=torch.float64, device="cuda")
        g[keep] = z @ e
        dx[r:r + step] = g
        de += z.t() @ xs
        db += z.sum(dim=0)
    out = (loss / n_counted, dx * (LOGIT_SCALE / n_counted), de * (LOGIT_SCALE / n_counted))
    return out if bias is None else out + (db / n_counted,)


def _exact_norm(case, s):
    h = s["x"] if s["residual"] is None else (s["x"].double() + s["residual"].double()).to(s["x"].dtype)
    f, w = h.double(), s["weight"].double()
    size = (f * f).mean(dim=1, keepdim=True) + EPS
    if case["op"] == "norm_q8":
        v = f * w
        top = v.abs().amax(dim=1, keepdim=True)
        y = torch.where(top > 0, torch.round(v * 127 / top), 0) * top / (127 * size.sqrt())
        return (y,) if s["residual"] is None else (y, h.double())
    unit = f / size.sqrt()
    dunit = s["dy"].double() * w
    dx = (dunit - unit * (dunit * unit).mean(dim=1, keepdim=True)) / size.sqrt() + s["dh"].double()
    return unit * w, h.double(), dx, (s["dy"].double() * unit).sum(dim=0)


def _exact_matmul(case, s):
    out = torch.mm(s["a"].double(), s["b"].double().t())
    out = out * torch.outer(s["a_scale"].double(), s["b_scale"].double())
    return out if s["bias"] is None else out + s["bias"].double()


def exact(case, seed):
    s = _inputs(case, seed)
    return {"ce": _exact_ce, "norm": _exact_norm, "norm_q8": _exact_norm, "matmul_q8": _exact_matmul}[case["op"]](case, s)

"""What is measured of the head's low-precision dense layer and of the distillation loss.

`dense`    out = act(x W + bias) + residual on 16-bit inputs, and its gradients
           d_x = dz W^T, d_weight = x^T dz, d_bias = sum dz  with  dz = d_out * act'(pre)
`distill`  row r:  w_r T^2 KL(p || q),  p = softmax(t / T) over the teacher's k stored logits t,
           q = softmax(z / T) over all V logits z of the student, and its gradient in z

Sizes are those of this framework's detection head (pooled rows of 7 * 7 * 512 = 25,088, hidden
width 4,096, 21 classes, 84 box deltas, 128 sampled or 1,500 / 2,000 proposed RoIs per image, 8
images per training step) and generic ones for wide label sets and odd shapes.

With `own` False the passes are elementary torch operations in 32 bits; with `own` True they are
the calls of the framework's own operators.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
SIZES = {"bf16": 2, "f16": 2, "f32": 4}


# ---- cases ------------------------------------------------------------------------------------
def _dense(op, m, k, n, dtype, act, layout, bias=True, residual=False, pre=False, **name):
    return {**name, "op": op, "m": m, "k": k, "n": n, "dtype": dtype, "act": act, "layout": layout,
            "bias": bias, "residual": residual, "pre": pre}


def _distill(op, rows, v, k, dtype, temperature, ragged, **name):
    return {**name, "op": op, "rows": rows, "v": v, "k": k, "dtype": dtype,
            "temperature": temperature, "ragged": ragged}


def listed():
    return [
        # one RoI's hidden row through the second layer: a single-row call, where latency counts
        _dense("dense_fwd", 1, 4096, 4096, "bf16", "silu", "nk", name="dense one row"),
        # the 128 sampled RoIs of one image through the first layer: bound by its 205 MB of weights
        _dense("dense_fwd", 128, 25088, 4096, "bf16", "relu", "kn", name="dense 128 sampled rois"),
        # odd sizes in every dimension, rows that are not 16-byte aligned
        _dense("dense_fwd", 777, 1003, 531, "f16", "gelu", "kn", residual=True, name="dense odd sizes"),
        # one image's 2,000 proposals through the first layer, serving
        _dense("dense_fwd", 2000, 25088, 4096, "bf16", "relu", "kn", name="dense one image fc1"),
        # a training step's 8 x 2,000 proposals through a residual hidden layer, pre-activations kept
        _dense("dense_fwd", 16000, 4096, 4096, "bf16", "gelu", "nk", residual=True, pre=True,
               name="dense hidden layer training"),
        # gradients of the box-delta layer: a narrow output, sums over 16,000 rows
        _dense("dense_bwd", 16000, 4096, 84, "bf16", "none", "nk", name="dense backward box deltas"),
        # gradients with odd sizes
        _dense("dense_bwd", 1111, 779, 333, "f16", "silu", "kn", name="dense backward odd sizes"),
        # gradients of the first layer in a training step: the largest products of the head
        _dense("dense_bwd", 16000, 25088, 4096, "bf16", "relu", "kn", name="dense backward fc1"),
        # class logits of a training step's proposals against 8 stored teacher logits each
        _distill("distill_loss", 16000, 21, 8, "f32", 2.0, False, name="distill 21 classes"),
        # one row of a wide label set: a single-row call
        _distill("distill_loss", 1, 131072, 64, "f32", 1.0, False, name="distill one wide row"),
        # a training batch over a wide label set
        _distill("distill_loss", 4096, 65536, 64, "bf16", 2.0, False, name="distill wide batch"),
        # the separate backward with upstream gradients, short teacher lists and masked rows
        _distill("distill_bwd", 1027, 32003, 33, "f16", 1.5, True, name="distill backward ragged"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["dense_fwd", "dense_fwd", "dense_bwd", "distill_loss", "distill_bwd"])
    if op.startswith("dense"):
        m, k, n = _log_int(rng, 1, 16000), _log_int(rng, 16, 25088), _log_int(rng, 8, 4096)
        if rng.random() < 0.5:      # half of the layers have widths in whole vectors
            k, n = max(16, k // 8 * 8), max(8, n // 8 * 8)
        act = rng.choice(["none", "relu", "gelu", "silu"])
        fwd = op == "dense_fwd"
        return _dense(op, m, k, n, rng.choice(["bf16", "f16"]), act, rng.choice(["kn", "nk"]),
                      bias=rng.random() < 0.75, residual=fwd and rng.random() < 0.5,
                      pre=fwd and rng.random() < 0.3)
    v = _log_int(rng, 16, 131072)
    rows = _log_int(rng, 1, max(1, min(16000, (4096 * 65536) // v)))
    k = _log_int(rng, 1, min(128, v))
    return _distill(op, rows, v, k, rng.choice(["bf16", "f16", "f32"]), rng.choice([1.0, 1.5, 2.0, 4.0]),
                    rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    if case["op"].startswith("dense"):
        m, k, n = case["m"], case["k"], case["n"]
        x = torch.relu(normal(m, k)).to(dt)                     # pooled or hidden rows: after a ReLU
        if case["layout"] == "kn":
            w = (normal(k, n) * k ** -0.5).to(dt)
        else:
            w = (normal(n, k) * k ** -0.5).to(dt).t()           # a Linear module's weight, as [K, N]
        s = dict(case=case, x=x, w=w, b=(0.1 * normal(n)).to(dt) if case["bias"] else None)
        s["residual"] = normal(m, n).to(dt) if case["residual"] else None
        if case["op"] == "dense_bwd":
            s["pre"] = None if case["act"] == "none" else normal(m, n).to(dt)
            s["d_out"] = normal(m, n).to(dt)
        return s
    rows, v, k = case["rows"], case["v"], case["k"]
    z = 2.0 * normal(rows, v)
    # k distinct labels per row, the teacher's logits there falling from the top, the student's raised
    step = torch.randint(1, v // k + 1, (rows, 1), generator=g, device="cuda")
    idx = (torch.randint(0, v, (rows, 1), generator=g, device="cuda")
           + step * torch.arange(k, device="cuda")) % v
    fall = torch.cumsum(torch.rand((rows, k), generator=g, device="cuda"), 1)
    t = (10.0 - fall).to(dt)
    z.scatter_add_(1, idx, 8.0 - fall + normal(rows, k))
    weight = None
    if case["ragged"]:
        kept = torch.randint(0, k + 1, (rows, 1), generator=g, device="cuda")   # 0: an empty list
        kept[0] = k
        idx = torch.where(torch.arange(k, device="cuda") < kept, idx, torch.full_like(idx, -1))
        weight = torch.rand(rows, generator=g, device="cuda") + 0.5
        masked = torch.rand(rows, generator=g, device="cuda") < 0.2
        masked[0] = False
        weight = weight * ~masked                                               # masked rows: 0
    z = z.to(dt)
    s = dict(case=case, z=z, t=t, idx=idx, weight=weight)
    if case["op"] == "distill_bwd":
        s["d_loss"] = 1.0 + 0.1 * normal(rows)
        s["lse"] = torch.logsumexp(z.float() / case["temperature"], 1)          # the forward's
    return s


# ---- one pass ---------------------------------------------------------------------------------
def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z * 0.5 ** 0.5)) + z * torch.exp(-0.5 * z * z) * (2.0 * math.pi) ** -0.5
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain_dense_fwd(s):
    c, dt = s["case"], s["x"].dtype
    z = s["x"].float() @ s["w"].float()
    if s["b"] is not None:
        z = z + s["b"].float()
    out = _act(z, c["act"])
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return {"out": out.to(dt), "pre": z.to(dt) if c["pre"] else None}


def _plain_dense_bwd(s):
    c, dt = s["case"], s["x"].dtype
    dz = s["d_out"].float()
    if c["act"] != "none":
        dz = dz * _act_grad(s["pre"].float(), c["act"])
    return {"d_x": (dz @ s["w"].float().t()).to(dt), "d_weight": (s["x"].float().t() @ dz).to(dt),
            "d_bias": dz.sum(0).to(dt) if c["bias"] else None}


def _plain_teacher(s, inv_t):
    """The teacher's probabilities over its stored labels: 0 at padding and in empty lists."""
    there = s["idx"] >= 0
    t = torch.where(there, s["t"].float() * inv_t, torch.full_like(s["t"], -math.inf, dtype=torch.float32))
    top = t.amax(1, keepdim=True)
    e = torch.where(there, torch.exp(t - top), torch.zeros_like(t))
    total = e.sum(1, keepdim=True)
    some = total > 0
    total = torch.where(some, total, torch.ones_like(total))
    log_p = torch.where(there, t - top, torch.zeros_like(t)) - torch.log(total)
    return e / total, log_p, some


def _plain_distill(s):
    c = s["case"]
    T = c["temperature"]
    z = s["z"].float() * (1.0 / T)
    p, log_p, some = _plain_teacher(s, 1.0 / T)
    at = s["idx"].clamp(min=0)
    weight = some[:, 0].float() if s["weight"] is None else s["weight"] * some[:, 0]
    if c["op"] == "distill_loss":
        top = z.amax(1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(1, keepdim=True)
        log_total = torch.log(total)
        log_q = (z.gather(1, at) - top) - log_total
        loss = weight * (T * T) * torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
        q = e / total
        scale = weight
    else:
        q = torch.exp(z - s["lse"][:, None])
        scale = weight * s["d_loss"]
    grad = q.scatter_add(1, at, -p) * (scale * T)[:, None]
    if c["op"] == "distill_loss":
        lse = torch.where(weight != 0, (top + log_total)[:, 0], torch.zeros_like(weight))
        return {"loss": loss, "lse": lse, "d_logits": grad.to(s["z"].dtype)}
    return {"d_logits": grad.to(s["z"].dtype)}


def _own_pass(s):
    from objectdetection_amd import ops
    c = s["case"]
    if c["op"] == "dense_fwd":
        got = ops.dense_fwd(s["x"], s["w"], s["b"], act=c["act"], residual=s["residual"], want_pre=c["pre"])
        return {"out": got[0], "pre": got[1]} if c["pre"] else {"out": got, "pre": None}
    if c["op"] == "dense_bwd":
        return ops.dense_bwd(s["d_out"], s["x"], s["w"], pre=s["pre"], act=c["act"], want_db=c["bias"])
    if c["op"] == "distill_loss":
        return ops.distill_loss(s["z"], s["t"], s["idx"], weight=s["weight"], temperature=c["temperature"])
    return {"d_logits": ops.distill_bwd(s["d_loss"], s["z"], s["t"], s["idx"], s["lse"], weight=s["weight"],
                                        temperature=c["temperature"])}


def run(state):
    if own:
        return _own_pass(state)
    op = state["case"]["op"]
    if op == "dense_fwd":
        return _plain_dense_fwd(state)
    if op == "dense_bwd":
        return _plain_dense_bwd(state)
    return _plain_distill(state)


# ---- what a pass cannot do without ------------------------------------------------------------
def work(case):
    es = SIZES[case["dtype"]]
    if case["op"].startswith("dense"):
        m, k, n = case["m"], case["k"], case["n"]
        if case["op"] == "dense_fwd":
            values = m * k + k * n + m * n * (1 + case["residual"] + case["pre"]) + n * case["bias"]
            return {"bytes": es * values, "flops": 2 * m * k * n}
        # d_out, the pre-activations, x and W read; d_x, d_weight and d_bias written
        values = m * n * (1 + (case["act"] != "none")) + 2 * m * k + 2 * k * n + n * case["bias"]
        return {"bytes": es * values, "flops": 4 * m * k * n}
    rows, v, k = case["rows"], case["v"], case["k"]
    # logits read (a fifth of the ragged rows is masked, one in k + 1 has no label: those are not)
    # and their gradients written; the stored logits and labels; row scalars
    read = 0.8 * k / (k + 1) if case["ragged"] else 1.0
    return {"bytes": int((1 + read) * es * rows * v) + rows * k * (es + 8) + 8 * rows, "flops": int(6 * read * rows * v)}


# ---- the definition in 64 bits ----------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("dense"):
        x, w = s["x"].double(), s["w"].double()
        if case["op"] == "dense_fwd":
            z = torch.matmul(x, w)
            if s["b"] is not None:
                z += s["b"].double()
            a = {"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)),
                 "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
            if s["residual"] is not None:
                a = a + s["residual"].double()
            return {"out": a, "pre": z if case["pre"] else None}
        d = s["d_out"].double()
        if case["act"] != "none":
            z = s["pre"].double().requires_grad_(True)
            with torch.enable_grad():
                a = {"relu": lambda: z * (z > 0), "gelu": lambda: z * torch.special.ndtr(z),
                     "silu": lambda: z * torch.sigmoid(z)}[case["act"]]()
                d, = torch.autograd.grad(a, z, d)
        return {"d_x": torch.matmul(d, w.transpose(0, 1)), "d_weight": torch.matmul(x.transpose(0, 1), d),
                "d_bias": torch.sum(d, 0) if case["bias"] else None}
    T, v = case["temperature"], case["v"]
    z, idx = s["z"].double() / T, s["idx"]
    # padded entries go to a class V that is dropped again
    at = torch.where(idx < 0, torch.full_like(idx, v), idx)
    t = torch.full((case["rows"], v + 1), -math.inf, dtype=torch.float64, device=z.device)
    t.scatter_(1, at, s["t"].double() / T)
    t = t[:, :v]
    listed_any = (idx >= 0).any(1)
    p = torch.where(listed_any[:, None], torch.softmax(t, 1), torch.zeros_like(t)).nan_to_num(nan=0.0)
    weight = torch.ones(case["rows"], dtype=torch.float64, device=z.device) if s["weight"] is None else s["weight"].double()
    if case["op"] == "distill_loss":
        log_q = torch.log_softmax(z, 1)
        terms = torch.special.xlogy(p, p) - torch.where(p > 0, p * log_q, torch.zeros_like(p))
        loss = weight * T * T * terms.sum(1)
        grad = (torch.exp(log_q) * listed_any[:, None] - p) * (weight * T)[:, None]
        takes_part = listed_any & (weight != 0)      # the other rows have no loss, gradient or lse
        return {"loss": loss, "lse": torch.logsumexp(z, 1) * takes_part, "d_logits": grad}
    q = torch.exp(z - s["lse"].double()[:, None]) * listed_any[:, None]
    return {"d_logits": (q - p) * (weight * s["d_loss"].double() * T)[:, None]}

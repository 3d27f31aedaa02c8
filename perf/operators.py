"""Cases and plain forms of the row operators: the root-mean-square norm (with the residual's addition and an 8-bit
output), the matrix product with its epilogue in 16 and in 8 bits, and the balance loss of the priors' competition.

With `own` false every operator is computed from elementary torch operations in 32 bits; with `own` true by this
package's entry points (compression_amd.ops)."""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
E4M3_MAX = 448.0
ACTS = ("none", "relu", "gelu", "silu")
LN2 = math.log(2.0)

# The sizes a drawn case stays within: those of the largest listed cases.
MOST_NORM = 32768 * 4096
MOST_FLOPS = 2 * 8192 * 8192 * 4096
MOST_SCORES = (1 << 20) * 64


def listed():
    return [
        # one location's residual stream in front of an 8-bit product: latency
        dict(name="norm_one_8bit", op="norm", rows=1, channels=4096, type="bf16", residual=True, eight=True),
        # the latent of 24 images of 768 x 512 (32 x 48 locations each), 192 channels, plain 16-bit output
        dict(name="norm_locations", op="norm", rows=36864, channels=192, type="f16", residual=False, eight=False),
        # a long run of rows, with the residual's addition and an 8-bit output
        dict(name="norm_rows_8bit", op="norm", rows=32768, channels=4096, type="bf16", residual=True, eight=True),
        # one row through a wide layer: the weights are read once, nothing else counts
        dict(name="linear_one", op="linear", rows=1, outputs=4096, inputs=4096, type="bf16", act="gelu", bias=True, residual=False),
        # the locations of one 768 x 512 image through an odd-sized hidden layer and back onto the residual stream
        dict(name="linear_ragged", op="linear", rows=1537, outputs=1000, inputs=1111, type="bf16", act="silu", bias=True, residual=True),
        # 24 images' locations, 256 latent channels to a hidden layer of four times that
        dict(name="linear_locations", op="linear", rows=36864, outputs=1024, inputs=256, type="f16", act="gelu", bias=True, residual=False),
        # a large layer with everything in its epilogue
        dict(name="linear_large", op="linear", rows=8192, outputs=8192, inputs=4096, type="bf16", act="silu", bias=True, residual=True),
        # a few rows of 8-bit operands: the weights' bytes
        dict(name="linear8_few", op="linear8", rows=7, outputs=4096, inputs=4096, type="bf16", act="relu", bias=True, residual=False),
        # the hidden layer back onto the residual stream, 8-bit operands
        dict(name="linear8_locations", op="linear8", rows=36864, outputs=256, inputs=1024, type="f16", act="none", bias=True, residual=True),
        # the large layer in 8 bits
        dict(name="linear8_large", op="linear8", rows=8192, outputs=8192, inputs=4096, type="bf16", act="gelu", bias=True, residual=True),
        # one image's competition, its costs in bits laid out prior by prior as the competition writes them
        dict(name="balance_image", op="balance", rows=1536, experts=64, type="f32", top_k=1, by_expert=True, bits=True, mask=False),
        # a large batch of 16-bit scores with two choices a row and padding rows
        dict(name="balance_large", op="balance", rows=1 << 20, experts=64, type="bf16", top_k=2, by_expert=False, bits=False, mask=True),
    ]


def _spread(rng, lo, hi):
    """A whole number of lo..hi, even over the logarithm; one in three is made a multiple of 16 where that stays in range."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.33 and v >= 16:
        v = v // 16 * 16
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("norm", "linear", "linear8", "balance"))
    if op == "norm":
        channels = _spread(rng, 1, 8192)
        rows = _spread(rng, 1, min(65536, MOST_NORM // channels))
        return dict(op=op, rows=rows, channels=channels, type=rng.choice(("f32", "f16", "bf16")), residual=rng.random() < 0.5,
                    eight=rng.random() < 0.5)
    if op in ("linear", "linear8"):
        outputs, inputs = _spread(rng, 1, 8192), _spread(rng, 1, 8192)
        rows = _spread(rng, 1, max(1, min(40000, MOST_FLOPS // (2 * outputs * inputs))))
        return dict(op=op, rows=rows, outputs=outputs, inputs=inputs, type=rng.choice(("f16", "bf16")), act=rng.choice(ACTS),
                    bias=rng.random() < 0.7, residual=rng.random() < 0.5)
    experts = _spread(rng, 2, 256)
    rows = _spread(rng, 1, min(1 << 20, MOST_SCORES // experts))
    return dict(op=op, rows=rows, experts=experts, type=rng.choice(("f32", "f16", "bf16")), top_k=rng.randint(1, min(8, experts)),
                by_expert=rng.random() < 0.4, bits=rng.random() < 0.4, mask=rng.random() < 0.5)


def _to_e4m3(v):
    """Rows of v as e4m3 values and the scale that each row's largest value sets."""
    s = v.abs().amax(1) / E4M3_MAX
    s = torch.where(s > 0, s, torch.ones_like(s))
    return (v / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case)
    t = TYPES[case["type"]]
    if case["op"] == "norm":
        rows, ch = case["rows"], case["channels"]
        # channels of a residual stream differ in their spread
        spread = torch.exp(0.5 * normal(ch))
        s["x"] = (normal(rows, ch) * spread).to(t)
        s["r"] = (normal(rows, ch) * 2.0).to(t) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * normal(ch)
    elif case["op"] in ("linear", "linear8"):
        rows, n, k = case["rows"], case["outputs"], case["inputs"]
        x, w = normal(rows, k), normal(n, k) / math.sqrt(k)
        if case["op"] == "linear":
            s["x"], s["w"], s["sx"], s["sw"] = x.to(t), w.to(t), None, None
        else:
            (s["x"], s["sx"]), (s["w"], s["sw"]) = _to_e4m3(x), _to_e4m3(w)
        s["b"] = 0.5 * normal(n) if case["bias"] else None
        s["r"] = normal(rows, n).to(t) if case["residual"] else None
    else:
        rows, e = case["rows"], case["experts"]
        # some priors are cheap nearly everywhere: use is far from even
        v = normal(rows, e) * 1.5 + normal(e)
        if case["bits"]:                                  # total bits of a location under every prior
            v = 40.0 - 4.0 * v
        v = v.to(t)
        s["scores"] = v.t().contiguous().t() if case["by_expert"] else v
        s["scale"] = -0.25 * LN2 if case["bits"] else 1.0
        s["mask"] = (torch.rand(rows, generator=g, device=DEV) < 0.9) if case["mask"] else None
        s["grad_out"] = torch.full((1,), 0.01, device=DEV)
    return s


def _norm_plain(s):
    h = s["x"].float()
    if s["r"] is not None:
        h = h + s["r"].float()
    y = h * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6) * s["weight"]
    out = {"h": h.to(s["x"].dtype)} if s["r"] is not None else {}
    if s["eight"]:
        out["q"], out["scale"] = _to_e4m3(y)
    else:
        out["y"] = y.to(s["x"].dtype)
    return out


def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    return v


def _linear_plain(s):
    y = s["x"].float() @ s["w"].float().t()
    if s["sx"] is not None:
        y = y * s["sx"][:, None] * s["sw"]
    if s["b"] is not None:
        y = y + s["b"]
    y = _act(y, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return {"y": y.to(TYPES[s["type"]])}


def _chosen(v, k):
    """The k largest of every row as truth values; among equal ones the lowest index."""
    edge = v.topk(k, 1).values[:, -1:]
    above, equal = v > edge, v == edge
    return above | (equal & (equal.to(torch.int32).cumsum(1) <= k - above.sum(1, keepdim=True)))


def _balance_plain(s):
    v, k = s["scores"].float(), s["top_k"]
    rows, e = v.shape
    keep = s["mask"] if s["mask"] is not None else torch.ones(rows, dtype=torch.bool, device=v.device)
    z = v * s["scale"]
    p = torch.exp(z - z.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True) * keep[:, None]
    chosen = _chosen(v if s["scale"] > 0 else -v, k) & keep[:, None]
    n = keep.sum()
    counts = chosen.sum(0)
    f = counts.double() / (k * n).clamp(min=1)
    loss = e * (f * p.double().sum(0)).sum() / n.clamp(min=1)
    f = f.float()
    grad = p * (f - (p * f).sum(1, keepdim=True)) * (s["grad_out"] * (s["scale"] * e) / n.clamp(min=1))
    return {"loss": loss.float(), "counts": counts.to(torch.int32), "grad": grad.to(s["scores"].dtype)}


def _own_run(s):
    from compression_amd import _lib, ops
    if s["op"] == "norm":
        got = ops.rms_norm(s["x"], s["weight"], eps=1e-6, residual=s["r"], quantize=s["eight"])
        got = got if isinstance(got, tuple) else (got,)
        names = (["q", "scale"] if s["eight"] else ["y"]) + (["h"] if s["r"] is not None else [])
        return dict(zip(names, got))
    if s["op"] in ("linear", "linear8"):
        act = {"none": _lib.MPC_ACT_NONE, "relu": _lib.MPC_ACT_RELU, "gelu": _lib.MPC_ACT_GELU, "silu": _lib.MPC_ACT_SILU}[s["act"]]
        return {"y": ops.linear(s["x"], s["w"], bias=s["b"], act=act, residual=s["r"], x_scale=s["sx"], weight_scale=s["sw"],
                                out_dtype=TYPES[s["type"]])}
    loss, counts, n = ops.prior_balance(s["scores"], scale=s["scale"], top_k=s["top_k"], mask=s["mask"])
    grad = ops.prior_balance_grad(s["scores"], counts, n, s["grad_out"], scale=s["scale"], top_k=s["top_k"], mask=s["mask"])
    return {"loss": loss, "counts": counts, "grad": grad}


def run(state):
    if own:
        return _own_run(state)
    if state["op"] == "norm":
        return _norm_plain(state)
    if state["op"] in ("linear", "linear8"):
        return _linear_plain(state)
    return _balance_plain(state)


def work(case):
    if case["op"] == "norm":
        n, b = case["rows"] * case["channels"], TYPES[case["type"]].itemsize
        moved = n * b * (3 if case["residual"] else 1) + n * (1 if case["eight"] else b) + 4 * case["channels"]
        return {"bytes": moved + (4 * case["rows"] if case["eight"] else 0), "flops": 6 * n}
    if case["op"] in ("linear", "linear8"):
        m, n, k = case["rows"], case["outputs"], case["inputs"]
        b = 1 if case["op"] == "linear8" else 2
        moved = b * (m * k + n * k) + 2 * m * n * (2 if case["residual"] else 1) + (4 * n if case["bias"] else 0)
        return {"bytes": moved + (4 * (m + n) if b == 1 else 0), "flops": 2 * m * n * k}
    n = case["rows"] * case["experts"]
    return {"bytes": 3 * n * TYPES[case["type"]].itemsize + (2 * case["rows"] if case["mask"] else 0), "flops": 12 * n}


def exact(case, seed):
    """The same outputs from the definitions in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        h = h if s["r"] is None else h + s["r"].double()
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / h.shape[1] + 1e-6) * s["weight"].double()
        out = {} if s["r"] is None else {"h": h}
        if not case["eight"]:
            return {**out, "y": y}
        top = y.abs().max(1).values
        scale = torch.where(top > 0, top / E4M3_MAX, torch.ones_like(top))
        return {**out, "q": y / scale[:, None], "scale": scale}
    if case["op"] in ("linear", "linear8"):
        x, w = s["x"].double(), s["w"].double()
        if s["sx"] is not None:
            x, w = x * s["sx"].double()[:, None], w * s["sw"].double()[:, None]
        y = torch.mm(x, w.t().contiguous())
        if s["b"] is not None:
            y += s["b"].double()
        if case["act"] == "relu":
            y = y.clamp(min=0.0)
        elif case["act"] == "gelu":
            y = 0.5 * y * torch.special.erfc(-y / math.sqrt(2.0))
        elif case["act"] == "silu":
            y = y * torch.sigmoid(y)
        return {"y": y if s["r"] is None else y + s["r"].double()}
    v, k, e = s["scores"].double(), case["top_k"], case["experts"]
    keep = torch.ones(case["rows"], dtype=torch.bool, device=v.device) if s["mask"] is None else s["mask"]
    p = torch.softmax(v * s["scale"], 1)[keep]
    order = torch.sort(v[keep] if s["scale"] > 0 else -v[keep], dim=1, descending=True, stable=True).indices[:, :k]
    counts = torch.bincount(order.reshape(-1), minlength=e)
    n = p.shape[0]
    grad = torch.zeros_like(v)
    if n == 0:
        return {"loss": torch.zeros((), dtype=torch.float64), "counts": counts.to(torch.int32), "grad": grad}
    f = counts.double() / (k * n)
    loss = e * (f * p.mean(0)).sum()
    grad[keep] = p * (f - p @ f[:, None]) * (s["grad_out"].double() * s["scale"] * e / n)
    return {"loss": loss, "counts": counts.to(torch.int32), "grad": grad}

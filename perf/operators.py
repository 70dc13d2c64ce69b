"""Performance cases of the operators that fine-tune a head over the encoder: the layer norm with its
gradients, the linear layer with bias, activation and residual with its gradients, the loss over a
request's choices with its gradient, and the AdamW step over many tensors.

Each case runs either in plain torch operations (`own` false: f32 whatever the inputs' type, rounded
once at the end) or through the library's entry points (`own` true). `exact` is the same result in
64 bits. Sizes come from the library's default model (hidden 768, GeGLU 1152, 22 layers, vocabulary
50368, head feed-forward 2048, scorer 384, packs of 12288 rows).
"""
import importlib
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4}
EPS = 1e-5                              # layer norm
BETA1, BETA2, ADAM_EPS = 0.9, 0.999, 1e-8
LR, DECAY, STEP, GRAD_SCALE = 1e-3, 0.01, 20, 0.5
BLOCK = 256                             # elements that share a scale of an 8-bit state
FP8_MAX, FP8_MIN = 448.0, 2.0 ** -9     # e4m3: the largest and the smallest value above zero


def _jc():
    return importlib.import_module("julia-cuda_b200")


# ------------------------------------------------------------------------------------------------
# the cases

def listed():
    return [
        # The scorer's norm on the markers of one request: all launch latency.
        {"name": "norm_12x768_f16", "op": "norm", "rows": 12, "d": 768, "type": "f16"},
        # Features of many packs normed at an odd width: rows that start on no vector boundary.
        {"name": "norm_65537x1001_f16", "op": "norm", "rows": 65537, "d": 1001, "type": "f16"},
        # The norm before a head's feed-forward, backward over one full pack, with the gradient that
        # comes past the block on the residual path.
        {"name": "norm_bwd_12288x768_bf16", "op": "norm_bwd", "rows": 12288, "d": 768,
         "type": "bf16", "add": True},
        # The scorer's first layer on the markers of one request.
        {"name": "linear_12x768x384_f16", "op": "linear", "m": 12, "k": 768, "n": 384,
         "type": "f16", "act": "gelu", "bias": True, "res": False, "keep": True},
        # A head's second feed-forward layer over a full pack: bias and residual in the epilogue.
        {"name": "linear_12288x2048x768_bf16", "op": "linear", "m": 12288, "k": 2048, "n": 768,
         "type": "bf16", "act": "none", "bias": True, "res": True, "keep": False},
        # A head's first feed-forward layer over a full pack, backward.
        {"name": "linear_bwd_12288x768x2048_f16", "op": "linear_bwd", "m": 12288, "k": 768,
         "n": 2048, "type": "f16", "act": "relu"},
        # A scorer's last layer, one output column, backward over the markers of a batch: nothing
        # in it has the alignment of a matrix tile.
        {"name": "linear_bwd_1531x384x1_bf16", "op": "linear_bwd", "m": 1531, "k": 384, "n": 1,
         "type": "bf16", "act": "none"},
        # A small batch of questions.
        {"name": "loss_16x6", "op": "loss", "requests": 16, "most": 12},
        # A whole evaluation set at once, from one to twelve choices each.
        {"name": "loss_1000003x6", "op": "loss", "requests": 1000003, "most": 12},
        # The scorer alone is trained.
        {"name": "adamw_scorer", "op": "adamw", "bits": 32, "d": 768, "inter": 1152, "vocab": 0,
         "layers": 0, "head_layers": 0, "head_ff": 2048, "scorer": 384, "grad": "f32",
         "copy": "f16"},
        # Everything is trained, with 16-bit gradients and a 16-bit working copy of the weights.
        {"name": "adamw_model", "op": "adamw", "bits": 32, "d": 768, "inter": 1152, "vocab": 50368,
         "layers": 22, "head_layers": 2, "head_ff": 2048, "scorer": 384, "grad": "bf16",
         "copy": "bf16"},
        # The same with the optimizer's states in 8 bits.
        {"name": "adamw_model_8bit", "op": "adamw", "bits": 8, "d": 768, "inter": 1152,
         "vocab": 50368, "layers": 22, "head_layers": 2, "head_ff": 2048, "scorer": 384,
         "grad": "bf16", "copy": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm_bwd", "linear", "linear_bwd", "loss", "adamw"])
    if op in ("norm", "norm_bwd"):
        d = _log(rng, 48, 4096)
        if rng.random() < 0.6:
            d = -(-d // 8) * 8
        c = {"op": op, "rows": _log(rng, 1, min(98304, 50_000_000 // d)), "d": d,
             "type": rng.choice(["f16", "bf16", "f32"])}
        if op == "norm_bwd":
            c["add"] = rng.random() < 0.5
        return c
    if op in ("linear", "linear_bwd"):
        n, k = _log(rng, 1, 2304), _log(rng, 8, 2304)
        if rng.random() < 0.7:
            n, k = -(-n // 8) * 8, -(-k // 8) * 8
        c = {"op": op, "m": _log(rng, 1, 12288), "k": k, "n": n,
             "type": rng.choice(["f16", "bf16"]), "act": rng.choice(["none", "relu", "gelu"])}
        if op == "linear":
            c.update(bias=rng.random() < 0.7, res=rng.random() < 0.5, keep=rng.random() < 0.5)
        return c
    if op == "loss":
        return {"op": op, "requests": _log(rng, 1, 500000), "most": _log(rng, 2, 12) + (
            rng.randrange(500) if rng.random() < 0.1 else 0)} if rng.random() < 0.8 else {
            "op": op, "requests": _log(rng, 1, 2000), "most": _log(rng, 64, 1500)}
    return {"op": op, "bits": rng.choice([32, 8]), "d": 64 * rng.randint(1, 12),
            "inter": 64 * rng.randint(1, 18), "vocab": _log(rng, 1, 50368),
            "layers": rng.randint(0, 21), "head_layers": rng.randint(0, 2),
            "head_ff": 64 * rng.randint(1, 32), "scorer": _log(rng, 16, 384),
            "grad": rng.choice(["f32", "f16", "bf16"]), "copy": rng.choice(["", "f16", "bf16"])}


def _shapes(c):
    """The tensors of a model of this shape, matrices as (rows, columns), vectors as (n,)."""
    d, i, f, s = c["d"], c["inter"], c["head_ff"], c["scorer"]
    got = [(c["vocab"], d), (d,)] if c["vocab"] else []
    got += [(d,), (3 * d, d), (d, d), (d,), (2 * i, d), (d, i)] * c["layers"]
    got += [(d,), (d,), (3 * d, d), (3 * d,), (d, d), (d,), (d,), (d,), (f, d), (f,), (d, f),
            (d,)] * c["head_layers"]
    return got + [(d,), (d,), (s, d), (s,), (1, s), (1,)]


# ------------------------------------------------------------------------------------------------
# the inputs

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=gen, device="cuda") * std + mean


def _choices(c, gen):
    """How many choices each request has, 1 to `most`, and where they begin: as many in all
    whatever the seed, which gives their order."""
    n = c["most"] - torch.arange(c["requests"], device="cuda") % c["most"]
    n = n[torch.randperm(c["requests"], generator=gen, device="cuda")]
    at = torch.zeros(c["requests"] + 1, dtype=torch.int32, device="cuda")
    at[1:] = n.cumsum(0)
    return n, at


def _to_fp8(x, floor):
    """x [blocks, BLOCK] in e4m3 with a scale a block; `floor`: what is above zero stays there."""
    scale = x.abs().amax(1) / FP8_MAX
    y = x / torch.where(scale > 0, scale, 1.0)[:, None]
    if floor:
        y = torch.where(x > 0, y.clamp_min(FP8_MIN), y)
    return y.clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn), scale


def _inputs(c, seed):
    gen, op = _gen(seed), c["op"]
    s = {"c": c}
    if op in ("norm", "norm_bwd"):
        t = TYPES[c["type"]]
        s["x"] = _normal(gen, c["rows"], c["d"], std=1.5, mean=0.2).to(t)
        s["gamma"] = _normal(gen, c["d"], std=0.05, mean=1.0)
        s["beta"] = _normal(gen, c["d"], std=0.02)
        if op == "norm_bwd":
            s["dy"] = _normal(gen, c["rows"], c["d"], std=0.1).to(t)
            s["add"] = _normal(gen, c["rows"], c["d"], std=0.1).to(t) if c["add"] else None
            x = s["x"].float()
            mean = x.mean(1)
            var = (x - mean[:, None]).square().mean(1)
            s["stats"] = torch.stack([mean, (var + EPS).rsqrt()], 1).contiguous()
    elif op in ("linear", "linear_bwd"):
        t, m, n, k = TYPES[c["type"]], c["m"], c["n"], c["k"]
        s["x"] = _normal(gen, m, k).to(t)
        s["w"] = _normal(gen, n, k, std=1 / math.sqrt(k)).to(t)
        if op == "linear":
            s["bias"] = _normal(gen, n, std=0.1) if c["bias"] else None
            s["res"] = _normal(gen, m, n).to(t) if c["res"] else None
        else:
            s["dy"] = _normal(gen, m, n, std=0.1).to(t)
            s["z"] = _normal(gen, m, n).to(t) if c["act"] != "none" else None
    elif op == "loss":
        n, s["at"] = _choices(c, gen)
        s["logits"] = _normal(gen, int(s["at"][-1]), std=3.0)
        s["gold"] = (torch.rand(c["requests"], generator=gen, device="cuda") * n).to(torch.int32)
        s["gold"] = torch.minimum(s["gold"], n.to(torch.int32) - 1)
        # A request in eleven has no answer and counts for nothing.
        s["gold"][torch.arange(c["requests"], device="cuda") % 11 == 7] = -1
        s["weight"] = torch.rand(c["requests"], generator=gen, device="cuda") + 0.5
    else:
        shapes = _shapes(c)
        sizes = [math.prod(x) for x in shapes]
        blocks = [-(-x // BLOCK) for x in sizes]
        s["shapes"], s["sizes"], s["blocks"] = shapes, sizes, blocks
        # One buffer for all tensors, each on a block boundary with zeros up to the next.
        per_block = torch.tensor(blocks, device="cuda")
        left = torch.tensor(sizes, device="cuda").repeat_interleave(per_block)
        first = (per_block.cumsum(0) - per_block).repeat_interleave(per_block)
        left = left - (torch.arange(sum(blocks), device="cuda") - first) * BLOCK
        real = torch.arange(BLOCK, device="cuda")[None, :] < left[:, None]
        s["p"] = _normal(gen, sum(blocks), BLOCK, std=0.02) * real
        s["g"] = (_normal(gen, sum(blocks), BLOCK, std=2e-3) * real).to(TYPES[c["grad"]])
        m = _normal(gen, sum(blocks), BLOCK, std=4e-4) * real
        v = _normal(gen, sum(blocks), BLOCK, std=1e-4).square() * real
        if c["bits"] == 8:
            s["m"], s["m_scale"] = _to_fp8(m, False)
            s["v"], s["v_scale"] = _to_fp8(v, True)
        else:
            s["m"], s["v"] = m, v
        decay = torch.tensor([DECAY if len(x) > 1 else 0.0 for x in shapes], device="cuda")
        s["decay"] = decay.repeat_interleave(per_block)
        s["grad_scale"] = torch.full((1,), GRAD_SCALE, device="cuda")
        s["copy"] = s["p"].to(TYPES[c["copy"]]) if c["copy"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    op, new = case["op"], torch.empty_like
    f32 = lambda *n: torch.empty(*n, dtype=torch.float32, device="cuda")  # noqa: E731
    if op == "norm":
        s["y"], s["stats"] = new(s["x"]), f32(case["rows"], 2)
    elif op == "norm_bwd":
        s["dx"], s["dgamma"], s["dbeta"] = new(s["x"]), f32(case["d"]), f32(case["d"])
    elif op == "linear":
        s["y"] = torch.empty(case["m"], case["n"], dtype=s["x"].dtype, device="cuda")
        s["z"] = new(s["y"]) if case["keep"] else None
    elif op == "linear_bwd":
        s["dx"], s["dw"], s["dbias"] = new(s["x"]), new(s["w"]), f32(case["n"])
    elif op == "loss":
        s["loss"], s["dlogits"] = f32(case["requests"]), new(s["logits"])
    elif own:
        # The optimizer is a handle that a training program keeps over all its steps.
        cut = lambda t: [x.reshape(-1)[:n] for x, n in zip(t.split(s["blocks"]), s["sizes"])]  # noqa: E731
        scales = {}
        if case["bits"] == 8:
            scales = {"exp_avg_scale": s["m_scale"].split(s["blocks"]),
                      "exp_avg_sq_scale": s["v_scale"].split(s["blocks"])}
        s["opt"] = _jc().AdamW(cut(s["p"]), cut(s["g"]), bits=case["bits"],
                               weight_decay=[DECAY if len(x) > 1 else 0.0 for x in s["shapes"]],
                               copies=cut(s["copy"]) if case["copy"] else None,
                               exp_avg=cut(s["m"]), exp_avg_sq=cut(s["v"]), **scales)
    return s


# ------------------------------------------------------------------------------------------------
# one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _adamw_outputs(s):
    out = {k: s[k] for k in ("p", "m", "v")}
    if s["c"]["bits"] == 8:
        out.update(m_scale=s["m_scale"], v_scale=s["v_scale"])
    if s["copy"] is not None:
        out["copy"] = s["copy"]
    return out


def _run_own(s):
    jc, c = _jc(), s["c"]
    op = c["op"]
    if op == "norm":
        jc.layer_norm(s["x"], s["gamma"], s["beta"], s["y"], stats=s["stats"], eps=EPS)
        return {"y": s["y"], "stats": s["stats"]}
    if op == "norm_bwd":
        jc.layer_norm_backward(s["dy"], s["x"], s["gamma"], s["stats"], s["dx"], s["dgamma"],
                               s["dbeta"], add=s["add"])
        return {"dx": s["dx"], "dgamma": s["dgamma"], "dbeta": s["dbeta"]}
    if op == "linear":
        jc.linear(s["x"], s["w"], s["y"], bias=s["bias"], act=c["act"], res=s["res"], z=s["z"])
        return {"y": s["y"], "z": s["z"]}
    if op == "linear_bwd":
        jc.linear_backward(s["dy"], s["x"], s["w"], z=s["z"], act=c["act"], dx=s["dx"], dw=s["dw"],
                           dbias=s["dbias"])
        return {"dx": s["dx"], "dw": s["dw"], "dbias": s["dbias"]}
    if op == "loss":
        jc.choice_loss(s["logits"], s["at"], s["gold"], s["loss"], dlogits=s["dlogits"],
                       weight=s["weight"])
        return {"loss": s["loss"], "dlogits": s["dlogits"]}
    s["opt"].step(STEP, lr=LR, betas=(BETA1, BETA2), eps=ADAM_EPS, grad_scale=s["grad_scale"])
    return _adamw_outputs(s)


def _run_plain(s):
    c = s["c"]
    op = c["op"]
    if op == "norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        xc = x - mean
        rstd = (xc.square().mean(1, keepdim=True) + EPS).rsqrt()
        return {"y": (xc * rstd * s["gamma"] + s["beta"]).to(s["x"].dtype),
                "stats": torch.cat([mean, rstd], 1)}
    if op == "norm_bwd":
        dy, d = s["dy"].float(), c["d"]
        rstd = s["stats"][:, 1:]
        xhat = (s["x"].float() - s["stats"][:, :1]) * rstd
        dxhat = dy * s["gamma"]
        dx = rstd * (dxhat - dxhat.sum(1, keepdim=True) / d
                     - xhat * ((dxhat * xhat).sum(1, keepdim=True) / d))
        if s["add"] is not None:
            dx = dx + s["add"].float()
        return {"dx": dx.to(s["x"].dtype), "dgamma": (dy * xhat).sum(0), "dbeta": dy.sum(0)}
    if op == "linear":
        t = s["x"].dtype
        z = s["x"].float() @ s["w"].float().t()
        if s["bias"] is not None:
            z = z + s["bias"]
        y = z
        if c["act"] == "relu":
            y = z.clamp_min(0)
        elif c["act"] == "gelu":
            y = 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
        if s["res"] is not None:
            y = y + s["res"].float()
        return {"y": y.to(t), "z": z.to(t) if c["keep"] else None}
    if op == "linear_bwd":
        t = s["x"].dtype
        dz = s["dy"].float()
        if c["act"] == "relu":
            dz = dz * (s["z"] > 0)
        elif c["act"] == "gelu":
            z = s["z"].float()
            cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
            dz = dz * (cdf + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi)))
        return {"dx": (dz @ s["w"].float()).to(t), "dw": (dz.t() @ s["x"].float()).to(t),
                "dbias": dz.sum(0)}
    if op == "loss":
        # Every request has one choice at least here.
        at, gold, lg = s["at"].long(), s["gold"].long(), s["logits"]
        r, n = c["requests"], lg.numel()
        seg = torch.repeat_interleave(torch.arange(r, device="cuda"), at[1:] - at[:-1],
                                      output_size=n)
        most = torch.full((r,), -math.inf, device="cuda").scatter_reduce(0, seg, lg, "amax")
        e = torch.exp(lg - most[seg])
        total = torch.zeros(r, device="cuda").index_add(0, seg, e)
        counts = gold >= 0
        w = torch.where(counts, s["weight"], 0.0)
        right = at[:-1] + gold.clamp_min(0)
        loss = torch.where(counts, w * (most + torch.log(total) - lg[right]), 0.0)
        hot = (torch.arange(n, device="cuda") == right[seg]).float()
        return {"loss": loss, "dlogits": w[seg] * (e / total[seg] - hot)}
    g = s["g"].float() * s["grad_scale"]
    m, v = s["m"].float(), s["v"].float()
    if c["bits"] == 8:
        m, v = m * s["m_scale"][:, None], v * s["v_scale"][:, None]
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    up = (m / (1 - BETA1 ** STEP)) / ((v / (1 - BETA2 ** STEP)).sqrt() + ADAM_EPS)
    s["p"].copy_(s["p"] * (1 - LR * s["decay"])[:, None] - LR * up)
    if c["bits"] == 8:
        s["m"], s["m_scale"] = _to_fp8(m, False)
        s["v"], s["v_scale"] = _to_fp8(v, True)
    else:
        s["m"], s["v"] = m, v
    if s["copy"] is not None:
        s["copy"].copy_(s["p"])
    return _adamw_outputs(s)


# ------------------------------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits

def work(case):
    c, op = case, case["op"]
    if op in ("norm", "norm_bwd"):
        e, b = c["rows"] * c["d"], BYTES[c["type"]]
        if op == "norm":
            return {"bytes": 2 * e * b + 8 * c["d"] + 8 * c["rows"], "flops": 8 * e}
        return {"bytes": (3 + c["add"]) * e * b + 12 * c["d"] + 8 * c["rows"], "flops": 14 * e}
    if op in ("linear", "linear_bwd"):
        m, n, k, b = c["m"], c["n"], c["k"], BYTES[c["type"]]
        if op == "linear":
            out = 1 + c["res"] + c["keep"]
            return {"bytes": (m * k + n * k + out * m * n) * b + 4 * n * c["bias"],
                    "flops": 2 * m * n * k}
        inp = 2 if c["act"] != "none" else 1
        return {"bytes": (2 * m * k + 2 * n * k + inp * m * n) * b + 4 * n,
                "flops": 4 * m * n * k}
    if op == "loss":
        full, rest = divmod(c["requests"], c["most"])
        n = full * c["most"] * (c["most"] + 1) // 2 + rest * c["most"] - rest * (rest - 1) // 2
        return {"bytes": 8 * n + 16 * c["requests"], "flops": 8 * n}
    n = sum(math.prod(x) for x in _shapes(c))
    state = 16 if c["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": n * (8 + state + BYTES[c["grad"]] + (2 if c["copy"] else 0)), "flops": 15 * n}


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    op, f = c["op"], torch.float64
    if op == "norm":
        x = s["x"].to(f)
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        rstd = 1 / torch.sqrt(var + EPS)
        return {"y": torch.addcmul(s["beta"].to(f), (x - mean) * rstd, s["gamma"].to(f)),
                "stats": torch.cat([mean, rstd], 1)}
    if op == "norm_bwd":
        x, dy, gamma = s["x"].to(f), s["dy"].to(f), s["gamma"].to(f)
        var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
        sd = torch.sqrt(var + EPS)
        n = (x - mean) / sd
        u = dy * gamma
        dx = (u - u.mean(1, keepdim=True) - n * (u * n).mean(1, keepdim=True)) / sd
        return {"dx": dx if s["add"] is None else dx + s["add"].to(f),
                "dgamma": torch.einsum("rd,rd->d", dy, n), "dbeta": dy.sum(0)}
    if op == "linear":
        z = torch.einsum("mk,nk->mn", s["x"].to(f), s["w"].to(f))
        z = z if s["bias"] is None else z + s["bias"].to(f)
        y = {"none": z, "relu": torch.where(z > 0, z, torch.zeros_like(z)),
             "gelu": z * torch.special.ndtr(z)}[c["act"]]
        return {"y": y if s["res"] is None else y + s["res"].to(f), "z": z if c["keep"] else None}
    if op == "linear_bwd":
        dz = s["dy"].to(f)
        if c["act"] != "none":
            z = s["z"].to(f)
            dz = dz * ((z > 0).to(f) if c["act"] == "relu" else torch.special.ndtr(z)
                       + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi))
        return {"dx": torch.einsum("mn,nk->mk", dz, s["w"].to(f)),
                "dw": torch.einsum("mn,mk->nk", dz, s["x"].to(f)), "dbias": dz.sum(0)}
    if op == "loss":
        at = s["at"].long()
        n = at[1:] - at[:-1]
        lg = s["logits"].to(f)
        if c["requests"] * c["most"] > 200_000_000:
            return None
        # One row a request, the places past its choices at minus infinity.
        col = torch.arange(c["most"], device="cuda")[None, :]
        there = col < n[:, None]
        wide = torch.full((c["requests"], c["most"]), -math.inf, dtype=f, device="cuda")
        wide[there] = lg
        logp = wide - torch.logsumexp(wide, 1, keepdim=True)
        gold = s["gold"].long()
        w = torch.where(gold >= 0, s["weight"].to(f), torch.zeros((), dtype=f, device="cuda"))
        picked = logp.gather(1, gold.clamp_min(0)[:, None])[:, 0]
        dl = w[:, None] * (logp.exp() - (col == gold[:, None]).to(f))
        return {"loss": -(w * picked), "dlogits": dl[there]}
    g = s["g"].to(f) * GRAD_SCALE
    m, v, p = s["m"].to(f), s["v"].to(f), s["p"].to(f)
    if c["bits"] == 8:
        m, v = m * s["m_scale"].to(f)[:, None], v * s["v_scale"].to(f)[:, None]
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    p -= LR * s["decay"].to(f)[:, None] * p
    p -= LR / (1 - BETA1 ** STEP) * m / (torch.sqrt(v / (1 - BETA2 ** STEP)) + ADAM_EPS)
    out = {"p": p, "m": m, "v": v}
    if c["bits"] == 8:
        # The states in units of their blocks' scales, before they are rounded to 8 bits.
        ms, vs = m.abs().amax(1) / FP8_MAX, v.amax(1) / FP8_MAX
        out.update(m=m / ms.clamp_min(1e-300)[:, None], v=v / vs.clamp_min(1e-300)[:, None],
                   m_scale=ms, v_scale=vs)
    if s["copy"] is not None:
        out["copy"] = p
    return out

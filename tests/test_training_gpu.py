"""The fine-tuning operators on the GPU against plain implementations in 64 bits.

Tolerances, all derived before the first run. u is a type's unit roundoff: 2^-11 (f16), 2^-8 (bf16),
2^-24 (f32).
  - A value rounded once is within u of itself; f32 work before that adds a few f32 roundoffs.
  - A sum in f32 is within (chain) x 2^-24 of the sum of its terms' magnitudes, chain being the
    longest run of additions any term passes through. No kernel here chains more than 400 in a row
    at these sizes (CHAIN), so SUM = 400 x 2^-24 = 2.4e-5 of the summed magnitudes bounds it.
  - dx and dw of a linear layer also read dz rounded to the type: another u of the summed magnitudes
    at worst; their 2-norms, where roundings average out, stay within 2 u (the rounding of dz and
    that of the result: u each).
Gradients are also tested against central differences of the 64-bit function along random
directions: those agree to 1e-6 of the magnitudes, so the kernels' own bound decides."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SUM = 400 * 2.0 ** -24
HALVES = [torch.float16, torch.bfloat16]
TYPES = HALVES + [torch.float32]


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


def rows_of(t, layout):
    """A copy of matrix t: "dense", "strided" (rows further apart, still on 16-byte boundaries),
    "odd" (rows one element further apart) or "shifted" (starting one element in)."""
    r, c = t.shape
    if layout == "dense":
        return t.clone()
    pad, at = {"strided": (16, 0), "odd": (1, 0), "shifted": (8, 1)}[layout]
    base = torch.full((r * (c + pad) + 1,), math.nan, dtype=t.dtype, device=t.device)
    v = base[at:at + r * (c + pad)].view(r, c + pad)[:, :c]
    v.copy_(t)
    return v


def near(got, want, tol, what=""):
    d = (got.double() - want).abs()
    assert torch.isfinite(got.double()).all(), what
    bad = d > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {float((d / tol.clamp_min(1e-300)).max()):.3g} of the bound"


def norm_near(got, want, tol, what=""):
    n = float(want.norm())
    e = float((got.double() - want).norm()) / n if n else float(got.double().norm())
    assert e <= tol, f"{what}: {e:.3e} > {tol:.3e}"


# ------------------------------------------------------------------------------------------------
# layer norm

WIDTHS = [1, 2, 7, 8, 64, 96, 255, 256, 257, 384, 511, 512, 520, 640, 768, 771, 1000, 1001, 1024,
          1025, 1032, 2048, 2050, 3000, 4096, 4100, 5003, 8192, 16384]


def norm64(x, gamma, beta, eps):
    x = x.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    y = xh * gamma.double()
    return (y if beta is None else y + beta.double()), mean, rstd, xh


def norm_tol(want, xh, gamma, beta, x, rstd, t):
    """u of the result, and f32's error in x - mean: a few roundoffs of |x| (and of the mean) scaled
    by rstd, a few of the product."""
    scale = (x.double().abs() + x.double().abs().mean(1, keepdim=True)) * rstd + xh.abs()
    b = 0 if beta is None else beta.double().abs()
    return U[t] * want.abs() + SUM * (scale * gamma.double().abs() + b) + 2.0 ** -25 * (t is torch.float16)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("d", WIDTHS)
def test_layer_norm_widths(jc, t, d):
    g = gen(d)
    rows = 37 if d < 4000 else 9
    x = normal(g, rows, d, std=1.5, mean=0.3, dtype=t)
    gamma, beta = normal(g, d, std=0.1, mean=1.0), normal(g, d, std=0.1)
    y, st = torch.full_like(x, math.nan), torch.full((rows, 2), math.nan, device="cuda")
    jc.layer_norm(x, gamma, beta, y, stats=st, eps=1e-5)
    want, mean, rstd, xh = norm64(x, gamma, beta, 1e-5)
    near(y, want, norm_tol(want, xh, gamma, beta, x, rstd, t), "y")
    near(st[:, :1], mean, SUM * x.double().abs().mean(1, keepdim=True), "mean")
    near(st[:, 1:], rstd, SUM * rstd * (1 + rstd * rstd * x.double().square().mean(1, keepdim=True)), "rstd")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layout", ["strided", "odd", "shifted"])
@pytest.mark.parametrize("rows,d", [(1, 768), (5, 1001), (131, 264), (3, 2056), (0, 64)])
def test_layer_norm_layouts(jc, t, layout, rows, d):
    g = gen(7)
    x = rows_of(normal(g, rows, d, dtype=t), layout)
    gamma = normal(g, d, mean=1.0)
    y = rows_of(torch.zeros(rows, d, dtype=t, device="cuda"), layout)
    jc.layer_norm(x, gamma, None, y)
    want, _, rstd, xh = norm64(x, gamma, None, 1e-5)
    near(y, want, norm_tol(want, xh, gamma, None, x, rstd, t), "y")
    if rows:
        jc.layer_norm(x, gamma, None, x)   # in place
        assert torch.equal(x, y)


def test_layer_norm_large_mean_and_constant_rows(jc):
    """Rows whose deviations are small beside their mean, and rows with none at all (y = beta)."""
    g = gen(3)
    x = normal(g, 64, 768, std=1e-2, mean=100.0)
    x[5] = 7.25
    gamma, beta = normal(g, 768, mean=1.0), normal(g, 768)
    y = torch.empty_like(x)
    jc.layer_norm(x, gamma, beta, y)
    want, _, rstd, xh = norm64(x, gamma, beta, 1e-5)
    near(y, want, norm_tol(want, xh, gamma, beta, x, rstd, torch.float32), "y")
    assert torch.equal(y[5], beta)


def test_layer_norm_nonfinite_rows_stay_alone(jc):
    g = gen(4)
    x = normal(g, 16, 768, dtype=torch.bfloat16)
    y = torch.empty_like(x)
    gamma = torch.ones(768, device="cuda")
    jc.layer_norm(x, gamma, None, y)
    x2, y2 = x.clone(), torch.empty_like(x)
    x2[3, 100], x2[9, 5] = math.nan, math.inf
    jc.layer_norm(x2, gamma, None, y2)
    ok = torch.ones(16, dtype=torch.bool)
    ok[3] = ok[9] = False
    assert torch.equal(y[ok], y2[ok]) and y2[3].isnan().all() and y2[9].isnan().all()


def norm_grads64(dy, x, gamma, eps):
    _, _, rstd, xh = norm64(x, gamma, None, eps)
    dy = dy.double()
    u = dy * gamma.double()
    dx = rstd * (u - u.mean(1, keepdim=True) - xh * (u * xh).mean(1, keepdim=True))
    mag = rstd * (u.abs() + u.abs().mean(1, keepdim=True) + xh.abs() * (u * xh).abs().mean(1, keepdim=True))
    return dx, (dy * xh).sum(0), dy.sum(0), mag, (dy * xh).abs().sum(0), dy.abs().sum(0)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,d,layout", [
    (1, 768, "dense"), (2, 1, "dense"), (5, 8, "dense"), (37, 255, "dense"), (1000, 256, "dense"),
    (4001, 384, "dense"), (3000, 768, "dense"), (3, 1001, "odd"), (700, 1000, "strided"),
    (600, 1024, "dense"), (33, 771, "shifted"), (90, 2048, "dense"), (650, 1025, "dense"),
    (17, 4096, "strided"), (29, 4100, "dense"), (7, 16384, "dense"), (9000, 64, "dense"),
    (4, 5003, "shifted")])
@pytest.mark.parametrize("add", [False, True])
def test_layer_norm_backward(jc, t, rows, d, layout, add):
    g = gen(rows + d)
    x = rows_of(normal(g, rows, d, std=1.5, mean=0.3, dtype=t), layout)
    dy = rows_of(normal(g, rows, d, std=0.1, dtype=t), layout)
    res = rows_of(normal(g, rows, d, std=0.1, dtype=t), layout) if add else None
    gamma = normal(g, d, std=0.1, mean=1.0)
    y, st = torch.empty(rows, d, dtype=t, device="cuda"), torch.empty(rows, 2, device="cuda")
    jc.layer_norm(x, gamma, None, y, stats=st)
    dx = rows_of(torch.zeros(rows, d, dtype=t, device="cuda"), layout)
    dg, db = (torch.full((d,), math.nan, device="cuda") for _ in range(2))
    jc.layer_norm_backward(dy, x, gamma, st, dx, dg, db, add=res)
    wx, wg, wb, mag, mg, mb = norm_grads64(dy, x, gamma, 1e-5)
    # The saved statistics are f32: an error of SUM in them moves xh by as much of |x| rstd.
    _, _, rstd, xh = norm64(x, gamma, None, 1e-5)
    off = SUM * (x.double().abs() + x.double().abs().mean(1, keepdim=True)) * rstd
    u = dy.double().abs() * gamma.double().abs()
    tx = SUM * mag + rstd * (off * (u * xh.abs()).mean(1, keepdim=True) + xh.abs() * (u * off).mean(1, keepdim=True))
    if add:
        wx = wx + res.double()
        tx = tx + SUM * res.double().abs()
    near(dx, wx, U[t] * wx.abs() + 2 * tx + 2.0 ** -25 * (t is torch.float16), "dx")
    near(dg, wg, SUM * mg + (dy.double().abs() * off).sum(0) + 1e-30, "dgamma")
    near(db, wb, SUM * mb + 1e-30, "dbeta")
    # The same again, into dy's own storage, without the parameters' gradients: the same bits.
    first = dx.clone()
    jc.layer_norm_backward(dy, x, gamma, st, dy, add=res)
    assert torch.equal(dy, first)


def test_layer_norm_backward_no_rows(jc):
    dg, db = (torch.full((96,), math.nan, device="cuda") for _ in range(2))
    e = torch.empty(0, 96, device="cuda", dtype=torch.float16)
    jc.layer_norm_backward(e, e, torch.ones(96, device="cuda"), torch.empty(0, 2, device="cuda"), e,
                           dg, db)
    assert (dg == 0).all() and (db == 0).all()


def test_layer_norm_gradients_against_differences(jc):
    g = gen(11)
    rows, d, h = 7, 96, 1e-5
    x, dy = normal(g, rows, d), normal(g, rows, d)
    gamma, beta = normal(g, d, mean=1.0), normal(g, d)
    y, st, dx = torch.empty_like(x), torch.empty(rows, 2, device="cuda"), torch.empty_like(x)
    dg, db = torch.empty_like(gamma), torch.empty_like(beta)
    jc.layer_norm(x, gamma, beta, y, stats=st)
    jc.layer_norm_backward(dy, x, gamma, st, dx, dg, db)

    def f(x, gamma, beta):
        return float((norm64(x, gamma, beta, 1e-5)[0] * dy.double()).sum())
    for i, (grad, at) in enumerate([(dx, 0), (dg, 1), (db, 2)]):
        v = [x.double(), gamma.double(), beta.double()]
        way = torch.randn(v[at].shape, generator=gen(50 + i), device="cuda").double()
        up, dn = list(v), list(v)
        up[at], dn[at] = v[at] + h * way, v[at] - h * way
        want = (f(*up) - f(*dn)) / (2 * h)
        got = float((grad.double() * way).sum())
        # SUM's error of every gradient element, plus the differences' own.
        assert abs(got - want) <= (SUM * 4 + 1e-6) * float((dy.double().abs().sum() * 8)), (i, got, want)


def test_layer_norm_same_bits_every_time(jc):
    g = gen(5)
    x, dy = normal(g, 5000, 768, dtype=torch.float16), normal(g, 5000, 768, dtype=torch.float16)
    gamma = normal(g, 768, mean=1.0)
    st = torch.empty(5000, 2, device="cuda")
    jc.layer_norm(x, gamma, None, torch.empty_like(x), stats=st)
    outs = []
    for _ in range(3):
        dx, dg, db = torch.empty_like(x), torch.empty_like(gamma), torch.empty_like(gamma)
        jc.layer_norm_backward(dy, x, gamma, st, dx, dg, db)
        outs.append((dx, dg, db))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


# ------------------------------------------------------------------------------------------------
# linear

def gelu64(z):
    return z * torch.special.ndtr(z)


def act64(z, act):
    return {"none": z, "relu": z.clamp_min(0), "gelu": gelu64(z)}[act]


def dact64(z, act):
    if act == "none":
        return torch.ones_like(z)
    if act == "relu":
        return (z > 0).double()
    return torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


SHAPES = [(1, 1, 1), (1, 384, 768), (12, 384, 768), (3, 1, 384), (129, 1, 96), (64, 64, 64),
          (128, 256, 64), (127, 136, 72), (130, 257, 65), (293, 768, 768), (300, 2048, 768),
          (513, 768, 2048), (257, 100, 50), (1000, 7, 1001), (33, 1001, 8), (700, 384, 1536),
          (5, 2304, 768), (2100, 264, 200), (901, 999, 1001), (1300, 777, 770), (640, 1001, 1000), (1500, 1000, 333)]


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("act,bias,res,keep", [("none", False, False, False), ("relu", True, True, True),
                                               ("gelu", True, False, True), ("gelu", False, True, False)])
def test_linear(jc, t, m, n, k, act, bias, res, keep):
    g = gen(m + 3 * n + 7 * k)
    x, w = normal(g, m, k, dtype=t), normal(g, n, k, std=1 / math.sqrt(k), dtype=t)
    b = normal(g, n, std=0.2) if bias else None
    r = normal(g, m, n, dtype=t) if res else None
    y = torch.full((m, n), math.nan, dtype=t, device="cuda")
    z = torch.full_like(y, math.nan) if keep else None
    jc.linear(x, w, y, bias=b, act=act, res=r, z=z)
    z64 = x.double() @ w.double().t()
    mag = x.double().abs() @ w.double().abs().t()
    if bias:
        z64, mag = z64 + b.double(), mag + b.double().abs()
    y64 = act64(z64, act)
    if res:
        y64, mag = y64 + r.double(), mag + r.double().abs()
    tiny = 2.0 ** -25
    # |act'| is at most 1.13, so an error of z passes on as 1.13 of itself.
    near(y, y64, U[t] * y64.abs() + 1.13 * SUM * mag + tiny, "y")
    if keep:
        near(z, z64, U[t] * z64.abs() + SUM * mag + tiny, "z")
    assert jc.device_error() == 0


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("layout", ["strided", "odd", "shifted"])
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (200, 136, 264), (65, 33, 70), (0, 16, 16)])
def test_linear_layouts(jc, t, layout, m, n, k):
    g = gen(9)
    x, w = rows_of(normal(g, m, k, dtype=t), layout), rows_of(normal(g, n, k, std=0.1, dtype=t), layout)
    r = rows_of(normal(g, m, n, dtype=t), layout)
    blank = torch.zeros(m, n, dtype=t, device="cuda")
    y, z = rows_of(blank, layout), rows_of(blank, layout)
    bias = normal(g, n)
    jc.linear(x, w, y, bias=bias, act="relu", res=r, z=z)
    z64 = x.double() @ w.double().t() + bias.double()
    mag = x.double().abs() @ w.double().abs().t() + bias.double().abs() + r.double().abs()
    y64 = z64.clamp_min(0) + r.double()
    near(y, y64, U[t] * y64.abs() + SUM * mag, "y")
    near(z, z64, U[t] * z64.abs() + SUM * mag, "z")
    jc.linear(x, w, r, bias=bias, act="relu", res=r)   # the residual's storage updated in place
    assert torch.equal(r, y)
    dy = rows_of(normal(g, m, n, dtype=t), layout)
    dx = rows_of(torch.zeros(m, k, dtype=t, device="cuda"), layout)
    dw = rows_of(torch.zeros(n, k, dtype=t, device="cuda"), layout)
    db = torch.full((n,), math.nan, device="cuda")
    jc.linear_backward(dy, x, w, z=z, act="relu", dx=dx, dw=dw, dbias=db)
    check_linear_grads(t, dy, x, w, z, "relu", dx, dw, db)


def check_linear_grads(t, dy, x, w, z, act, dx, dw, db):
    dz = dy.double() * (dact64(z.double(), act) if act != "none" else 1.0)
    off = 0.0 if act == "none" else U[t]
    # f16 cannot hold a dz below 2^-25 apart: that much of each operand's magnitude at most.
    tiny = 2.0 ** -25 if t is torch.float16 else 0.0
    act_err = 4e-7 * dy.double().abs()   # the approximation of GELU', absolute
    wx, mx = dz @ w.double(), dz.abs() @ w.double().abs()
    near(dx, wx, U[t] * wx.abs() + (SUM + off) * mx + (act_err + tiny) @ w.double().abs() + tiny, "dx")
    norm_near(dx, wx, 2 * U[t] + SUM, "dx")
    ww, mw = dz.t() @ x.double(), dz.abs().t() @ x.double().abs()
    near(dw, ww, U[t] * ww.abs() + (SUM + off) * mw + (act_err + tiny).t() @ x.double().abs() + tiny, "dw")
    norm_near(dw, ww, 2 * U[t] + SUM, "dw")
    near(db, dz.sum(0), SUM * dz.abs().sum(0) + act_err.sum(0) + 1e-30, "dbias")


@pytest.mark.parametrize("t", HALVES)
@pytest.mark.parametrize("m,n,k", SHAPES + [(5000, 384, 768), (4097, 40, 24)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
def test_linear_backward(jc, t, m, n, k, act):
    g = gen(m + n + k)
    x, w = normal(g, m, k, dtype=t), normal(g, n, k, std=1 / math.sqrt(k), dtype=t)
    dy, z = normal(g, m, n, std=0.5, dtype=t), normal(g, m, n, dtype=t)
    dx, dw = torch.full_like(x, math.nan), torch.full_like(w, math.nan)
    db = torch.full((n,), math.nan, device="cuda")
    jc.linear_backward(dy, x, w, z=z if act != "none" else None, act=act, dx=dx, dw=dw, dbias=db)
    check_linear_grads(t, dy, x, w, z, act, dx, dw, db)
    # Each gradient alone has the same bits as all together, and twice gives the same bits.
    for kw in (dict(dx=torch.empty_like(dx)), dict(dw=torch.empty_like(dw)), dict(dbias=torch.empty_like(db))):
        jc.linear_backward(dy, x, w, z=z if act != "none" else None, act=act, **kw)
        (name, got), = kw.items()
        assert torch.equal(got, {"dx": dx, "dw": dw, "dbias": db}[name]), name
    assert jc.device_error() == 0


def test_linear_relu_at_zero_and_nan(jc):
    """ReLU's gradient is 0 at 0 (and at -0); NaN goes through the forward pass."""
    t = torch.float16
    z = torch.tensor([[0.0, -0.0, 1.0, -1.0, 2.0 ** -24, -2.0 ** -24, 5.0, math.inf]], device="cuda", dtype=t)
    eye = torch.eye(8, device="cuda", dtype=t)
    dx = torch.empty_like(z)
    jc.linear_backward(torch.ones_like(z), z, eye, z=z, act="relu", dx=dx)
    assert dx.tolist() == [[0, 0, 1, 0, 1, 0, 1, 1]]
    x = torch.zeros(2, 8, device="cuda", dtype=t)
    x[1, 3] = math.nan
    for act in ("none", "relu", "gelu"):
        y = torch.empty(2, 8, device="cuda", dtype=t)
        jc.linear(x, eye, y, act=act)
        assert (y[0] == 0).all() and y[1].isnan().all(), act


def test_linear_gradients_against_differences(jc):
    g = gen(21)
    t, h = torch.bfloat16, 1e-5
    m, n, k = 9, 24, 40
    for act in ("none", "relu", "gelu"):
        x, w = normal(g, m, k, dtype=t), normal(g, n, k, std=0.3, dtype=t)
        b, dy = normal(g, n), normal(g, m, n, dtype=t)
        z = (x.double() @ w.double().t() + b.double())
        z16 = z.to(t)
        b = b + 0  # z as saved is rounded: differences are taken about the rounded point
        shift = z16.double() - z
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        jc.linear_backward(dy, x, w, z=z16, act=act, dx=dx, dw=dw, dbias=db)

        def f(x, w, b):
            return float((act64(x @ w.t() + b + shift, act) * dy.double()).sum())
        for i, (grad, at) in enumerate([(dx, 0), (dw, 1), (db, 2)]):
            v = [x.double(), w.double(), b.double()]
            way = torch.randn(v[at].shape, generator=gen(60 + i), device="cuda").double()
            up, dn = list(v), list(v)
            up[at], dn[at] = v[at] + h * way, v[at] - h * way
            want = (f(*up) - f(*dn)) / (2 * h)
            got = float((grad.double() * way).sum())
            # Two roundings of the type for each element, 1e-4 for the differences at ReLU's kink.
            tol = 2 * U[t] * float((grad.double() * way).abs().sum()) * 1.5 + 1e-4
            assert abs(got - want) <= tol, (act, i, got, want)


# ------------------------------------------------------------------------------------------------
# the loss

def loss64(logits, offsets, gold, weight):
    lg, off = logits.double().cpu(), offsets.tolist()
    loss, dl = torch.zeros(len(off) - 1, dtype=torch.float64), torch.zeros_like(lg)
    for r, (a, b) in enumerate(zip(off[:-1], off[1:])):
        w = 1.0 if weight is None else float(weight[r])
        l = lg[a:b]
        if int(gold[r]) < 0 or w == 0 or not (l != -math.inf).any():
            continue
        lse = torch.logsumexp(l, 0)
        loss[r] = w * (lse - l[int(gold[r])])
        p = torch.exp(l - lse)
        p[int(gold[r])] -= 1
        dl[a:b] = w * p
    return loss.cuda(), dl.cuda()


def run_loss(jc, logits, offsets, gold, weight=None):
    loss = torch.full((gold.numel(),), math.nan, device="cuda")
    dl = torch.full_like(logits, math.nan)
    jc.choice_loss(logits, offsets, gold, loss, dlogits=dl, weight=weight)
    return loss, dl


@pytest.mark.parametrize("requests,lo,hi", [(1, 1, 1), (1, 5, 5), (3, 0, 3), (16, 1, 12), (777, 0, 9), (100, 1, 70),
                                            (40, 33, 200), (9, 900, 3000), (2, 50000, 50368), (20000, 2, 4)])
@pytest.mark.parametrize("weighted", [False, True])
def test_choice_loss(jc, requests, lo, hi, weighted):
    rng = np.random.default_rng(requests + hi)
    n = rng.integers(lo, hi + 1, requests)
    off = torch.from_numpy(np.concatenate([[0], n.cumsum()]).astype(np.int32)).cuda()
    logits = torch.from_numpy(rng.normal(0, 4, int(n.sum())).astype(np.float32)).cuda()
    gold = torch.from_numpy(np.where(rng.random(requests) < 0.1, -1, (rng.random(requests) * n).astype(np.int64))
                            .astype(np.int32)).cuda()
    gold[torch.from_numpy(n == 0).cuda()] = -1
    w = torch.from_numpy(rng.random(requests).astype(np.float32)).cuda() if weighted else None
    loss, dl = run_loss(jc, logits, off, gold, w)
    wl, wd = loss64(logits, off, gold, w)
    # exp and log are good to 2 ulp; the logits' differences are rounded at their own size (20 here),
    # which moves a probability by as much: 64 x 2^-24 of a weight, beside the sums' bound.
    top = float(logits.abs().max()) if logits.numel() else 1.0
    near(loss, wl, (SUM + 4 * top * 2.0 ** -24) * (1 + wl.abs()), "loss")
    near(dl, wd, (SUM + 4 * top * 2.0 ** -24) * torch.ones_like(wd), "dlogits")
    assert jc.device_error() == 0


def test_choice_loss_infinities(jc):
    """Logits of -infinity are choices that cannot be; of a request with only such, nothing counts."""
    inf = math.inf
    lg = torch.tensor([1.0, -inf, 2.0, -inf, -inf, 0.5, -3.4e38, -3.4e38, 88.0, -100.0, math.nan, 1.0, -inf, 4.0],
                      device="cuda")
    off = torch.tensor([0, 3, 5, 8, 10, 12, 14], dtype=torch.int32, device="cuda")
    gold = torch.tensor([2, 0, 1, 0, 1, 0], dtype=torch.int32, device="cuda")
    loss, dl = run_loss(jc, lg, off, gold)
    p = 1 / (1 + math.e)
    assert loss[0].item() == pytest.approx(math.log(1 + math.exp(-1)), abs=1e-6)
    assert dl[:3].tolist() == pytest.approx([p, 0, -p], abs=1e-6)
    assert loss[1] == 0 and (dl[3:5] == 0).all()
    assert loss[2].item() == pytest.approx(3.4e38, rel=1e-6) and dl[5:8].tolist() == [1, -1, 0]
    assert loss[3] == 0 and (dl[8:10] == 0).all()
    assert loss[4].isnan() and dl[10:12].isnan().all()
    assert loss[5] == inf and dl[12:14].tolist() == [-1, 1]


def test_choice_loss_gradient_against_differences(jc):
    rng = np.random.default_rng(1)
    off = torch.tensor([0, 4, 5, 12], dtype=torch.int32, device="cuda")
    gold = torch.tensor([3, 0, 2], dtype=torch.int32, device="cuda")
    lg = torch.from_numpy(rng.normal(0, 2, 12).astype(np.float32)).cuda()
    w = torch.tensor([1.0, 2.0, 0.5], device="cuda")
    _, dl = run_loss(jc, lg, off, gold, w)
    for i in range(12):
        e = torch.zeros(12, device="cuda", dtype=torch.float64)
        e[i] = 1e-5
        d = (loss64(lg.double() + e, off, gold, w)[0].sum() - loss64(lg.double() - e, off, gold, w)[0].sum()) / 2e-5
        assert abs(float(d) - float(dl[i])) < 1e-6


def test_choice_loss_out_of_range_is_recorded(jc):
    """A right marker past its request's markers: device error 6, loss 0, its gradients untouched."""
    lg = torch.zeros(6, device="cuda")
    off = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    loss, dl = run_loss(jc, lg, off, torch.tensor([3, 1], dtype=torch.int32, device="cuda"))
    assert jc.device_error() == 6 and jc.device_error() == 0
    assert loss[0] == 0 and dl[:3].isnan().all()
    assert loss[1].item() == pytest.approx(math.log(3), abs=1e-6) and dl[3:].isfinite().all()
    bad = torch.tensor([0, 7, 6], dtype=torch.int32, device="cuda")
    loss, _ = run_loss(jc, lg, bad, torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    assert jc.device_error() == 6 and loss.tolist() == [0, 0]


# ------------------------------------------------------------------------------------------------
# AdamW

SIZES = [1, 7, 255, 256, 257, 2048, 2049, 5000, 384 * 768, 384, 0]


def adam64(p, g, m, v, t, lr, b1, b2, eps, decay, scale):
    g = g.double() * scale
    m = b1 * m.double() + (1 - b1) * g
    v = b2 * v.double() + (1 - b2) * g * g
    up = (m / (1 - b1 ** t)) / (torch.sqrt(v / (1 - b2 ** t)) + eps)
    return p.double() * (1 - lr * decay) - lr * up, m, v, up


def blocks(x):
    n = -(-x.numel() // 256)
    out = torch.zeros(n * 256, dtype=torch.float64, device="cuda")
    out[:x.numel()] = x.double()
    return out.view(n, 256)


def make(t, shift, n, g, std):
    base = torch.zeros(n + 8, dtype=t, device="cuda")
    v = base[shift:shift + n]
    v.copy_(normal(g, n, std=std))
    return v


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", TYPES)
@pytest.mark.parametrize("copy", [None, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shift", [0, 1])
def test_adamw(jc, bits, grad, copy, shift):
    """Three steps; each compared with the 64-bit step from the state the kernel left before."""
    g = gen(bits + shift)
    ps = [make(torch.float32, shift, n, g, 0.02) for n in SIZES]
    gs = [make(grad, shift, n, g, 1e-3) for n in SIZES]
    cs = None if copy is None else [make(copy, shift, n, g, 1.0) for n in SIZES]
    decay = [0.01 * (i % 3) for i in range(len(SIZES))]
    opt = jc.AdamW(ps, gs, bits=bits, weight_decay=decay, copies=cs)
    scale = torch.full((1,), 0.5, device="cuda")

    def state(i):
        m, v = opt.exp_avg[i], opt.exp_avg_sq[i]
        if bits == 32:
            return m.double(), v.double()
        n = m.numel()
        return ((blocks(m.float()) * opt.exp_avg_scale[i].double()[:, None]).view(-1)[:n],
                (blocks(v.float()) * opt.exp_avg_sq_scale[i].double()[:, None]).view(-1)[:n])
    u = 2.0 ** -24
    for t in (1, 2, 3):
        before = [(p.clone(), *state(i)) for i, p in enumerate(ps)]
        opt.step(t, lr=1e-2, betas=(0.9, 0.99), eps=1e-8, grad_scale=scale if t > 1 else None)
        for i, p in enumerate(ps):
            if not p.numel():
                continue
            p0, m0, v0 = before[i]
            wp, wm, wv, up = adam64(p0, gs[i], m0, v0, t, 1e-2, 0.9, 0.99, 1e-8, decay[i], 0.5 if t > 1 else 1.0)
            # m's terms can cancel: its error is of the terms' size, and up's with it.
            mag = m0.abs() * 0.9 + gs[i].double().abs() * 0.1
            den = (mag / wm.abs().clamp_min(1e-30)).clamp_max(1e6)
            near(p, wp, 4 * u * p0.double().abs() + 1e-2 * up.abs() * u * (16 + 8 * den) + 1e-30, f"p {t} {i}")
            if copy is not None:
                assert torch.equal(cs[i], p.to(copy))
            m, v = state(i)
            if bits == 32:
                near(m, wm, 4 * u * mag + 1e-30, "m")
                near(v, wv, 4 * u * wv + 1e-37, "v")
            else:
                # e4m3: half a step of 2^-3 (normal) or of 2^-9 of the scale, which is f32.
                for got, want, sc in ((m, wm, opt.exp_avg_scale[i]), (v, wv, opt.exp_avg_sq_scale[i])):
                    top = blocks(want).abs().amax(1) / 448
                    near(sc, top, 8 * u * top * 8 + 1e-37, "scale")
                    unit = top.repeat_interleave(256)[:want.numel()]
                    least = 2.0 ** -9 if got is v else 2.0 ** -10   # v above 0 is held at 2^-9 at least
                    near(got, want, (2.0 ** -4 + 1e-5) * want.abs() + (least + 1e-6) * unit + 1e-37, "state")
                assert ((v > 0) == (wv > 0)).all()
    opt.close()


@pytest.mark.parametrize("grad", TYPES)
def test_adamw_8bit_codes_are_exact(jc, grad):
    """Codes and scales are those of the formula's operations rounded one by one in f32 (torch's own
    multiplications, additions and divisions), bit for bit, over several steps."""
    g = gen(77)
    n = 300 * 256
    p, grads = normal(g, n, std=0.02), normal(g, n, std=1e-3, dtype=grad)
    grads[5 * 256:6 * 256] = 0   # a block without gradients
    grads[7 * 256 + 3] = 1.0     # and one with a single large one
    scale = torch.full((1,), 0.37, device="cuda")
    opt = jc.AdamW([p], [grads], bits=8)
    m = v = torch.zeros(300, 256, device="cuda")
    for t in range(1, 6):
        grads.copy_(grads.float() * (1 + 0.1 * t))
        opt.step(t, lr=1e-3, betas=(0.9, 0.999), grad_scale=scale)
        gf = grads.float().view(300, 256) * scale
        m = (m * 0.9) + (gf * (1 - 0.9))
        v = (v * 0.999) + (gf * (1 - 0.999)) * gf
        out = []
        for x, floor in ((m, False), (v, True)):
            sc = x.abs().amax(1) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device="cuda")
            y = x / torch.where(sc > 0, sc, 1.0)[:, None]
            y = torch.where(x > 0, y.clamp_min(2.0 ** -9), y) if floor else y
            out.append((y.clamp(-448, 448).to(torch.float8_e4m3fn), sc))
        (mc, ms), (vc, vs) = out
        assert torch.equal(opt.exp_avg_scale[0], ms) and torch.equal(opt.exp_avg_sq_scale[0], vs), t
        assert torch.equal(opt.exp_avg[0].view(torch.uint8), mc.view(-1).view(torch.uint8)), t
        assert torch.equal(opt.exp_avg_sq[0].view(torch.uint8), vc.view(-1).view(torch.uint8)), t
        m, v = mc.float() * ms[:, None], vc.float() * vs[:, None]


def test_adamw_does_not_touch_its_neighbours(jc):
    base = torch.full((3000,), 5.0, device="cuda")
    grads = torch.ones(3000, device="cuda")
    m, v = torch.zeros(3000, device="cuda"), torch.zeros(3000, device="cuda")
    cut = lambda t: [t[3:3 + 1001], t[1500:1500 + 300]]  # noqa: E731
    jc.AdamW(cut(base), cut(grads), exp_avg=cut(m), exp_avg_sq=cut(v)).step(1, lr=0.1)
    inside = torch.zeros(3000, dtype=torch.bool, device="cuda")
    inside[3:1004] = inside[1500:1800] = True
    assert (base[~inside] == 5).all() and (m[~inside] == 0).all() and (v[~inside] == 0).all()
    assert (base[inside] - 4.9).abs().max() < 1e-5


def test_adamw_zero_gradients_and_eps(jc):
    """No gradient yet: 0 / (0 + eps), the weights only decay; states stay 0 in 8 bits too."""
    for bits in (32, 8):
        p = torch.ones(1000, device="cuda")
        opt = jc.AdamW([p], [torch.zeros(1000, device="cuda")], bits=bits, weight_decay=0.5)
        opt.step(1, lr=0.1)
        assert (p - 0.95).abs().max() < 1e-6
        assert (opt.exp_avg[0].float() == 0).all() and (opt.exp_avg_sq[0].float() == 0).all()


def test_adamw_8bit_follows_32bit(jc):
    """Both descend the same noisy quadratic, the 8-bit run within a tenth of the way of the other."""
    g = gen(8)
    target = normal(g, 4096)
    runs = {}
    for bits in (32, 8):
        p, grad = torch.zeros(4096, device="cuda"), torch.empty(4096, device="cuda")
        opt = jc.AdamW([p], [grad], bits=bits)
        noise = gen(9)
        for t in range(1, 301):
            grad.copy_(p - target + 0.1 * torch.randn(4096, generator=noise, device="cuda"))
            opt.step(t, lr=2e-2)
        runs[bits] = float((p - target).norm() / target.norm())
    assert runs[32] < 0.1 and runs[8] < runs[32] + 0.1


# ------------------------------------------------------------------------------------------------
# streams, graphs, refusals

def test_other_stream_and_graph(jc):
    """Every operator queued on a stream of its own, and captured into a CUDA graph and replayed."""
    g = gen(2)
    t = torch.float16
    x, w = normal(g, 300, 256, dtype=t), normal(g, 128, 256, std=0.1, dtype=t)
    y, z, dy = (torch.zeros(300, 128, dtype=t, device="cuda") for _ in range(3))
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros(128, device="cuda")
    gamma, n, st = torch.ones(256, device="cuda"), torch.zeros_like(x), torch.zeros(300, 2, device="cuda")
    dn, dg = torch.zeros_like(x), torch.zeros(256, device="cuda")
    off = torch.arange(0, 301, 3, dtype=torch.int32, device="cuda")
    gold = torch.ones(100, dtype=torch.int32, device="cuda")
    lg, loss, dl = normal(g, 300), torch.zeros(100, device="cuda"), torch.zeros(300, device="cuda")
    p, grad = torch.ones(1000, device="cuda"), torch.ones(1000, device="cuda")
    opt = jc.AdamW([p], [grad])

    def go(stream=None):
        jc.layer_norm(x, gamma, None, n, stats=st, stream=stream)
        jc.linear(n, w, y, act="gelu", z=z, stream=stream)
        jc.choice_loss(lg, off, gold, loss, dlogits=dl, stream=stream)
        jc.linear_backward(y, n, w, z=z, act="gelu", dx=dx, dw=dw, dbias=db, stream=stream)
        jc.layer_norm_backward(dx, x, gamma, st, dn, dg, stream=stream)
        opt.step(1, lr=0.1, stream=stream)
    outs = (n, y, z, loss, dl, dx, dw, db, dn, dg)
    go()
    torch.cuda.synchronize()
    want = [o.clone() for o in outs]
    side = torch.cuda.Stream()
    for o in outs:
        o.zero_()
    side.wait_stream(torch.cuda.current_stream())
    go(side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    for o in outs:
        o.zero_()
    p.fill_(1.0)
    for s in (opt.exp_avg[0], opt.exp_avg_sq[0]):
        s.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want)) and (p - 0.9).abs().max() < 1e-6
    assert jc.device_error() == 0


def test_python_refusals(jc):
    f16 = dict(dtype=torch.float16, device="cuda")
    x, w, y = torch.zeros(4, 8, **f16), torch.zeros(6, 8, **f16), torch.zeros(4, 6, **f16)
    gamma = torch.ones(8, device="cuda")
    E = jc.JuliaCudaError
    for bad in (lambda: jc.layer_norm(x, gamma[:7], None, x), lambda: jc.layer_norm(x, gamma, None, y),
                lambda: jc.layer_norm(x.double(), gamma, None, x), lambda: jc.layer_norm(x, gamma.half(), None, x),
                lambda: jc.layer_norm(x.t(), torch.ones(4, device="cuda"), None, x.t()),
                lambda: jc.layer_norm(x, gamma, None, x, eps=-1.0),
                lambda: jc.layer_norm(x.cpu(), gamma, None, x),
                lambda: jc.linear(x, w, y, act="tanh"), lambda: jc.linear(x, w.bfloat16(), y),
                lambda: jc.linear(x.float(), w.float(), y.float()), lambda: jc.linear(x, w, y.t()),
                lambda: jc.linear(x, w, y, bias=gamma), lambda: jc.linear(x, w[:, :7], y),
                lambda: jc.linear_backward(y, x, w, act="relu", dx=x),
                lambda: jc.linear_backward(y, x, w, dw=w, ws=torch.empty(1, device="cuda")),
                lambda: jc.choice_loss(torch.zeros(4, device="cuda"), torch.zeros(2, device="cuda"),
                                       torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(1, device="cuda")),
                lambda: jc.AdamW([gamma], [gamma[:4]]), lambda: jc.AdamW([x], [x]),
                lambda: jc.AdamW([gamma], [gamma], bits=16), lambda: jc.AdamW([gamma], []),
                lambda: jc.AdamW([gamma], [gamma], copies=[gamma])):
        with pytest.raises(E):
            bad()
    opt = jc.AdamW([gamma], [gamma.clone()])
    for kw in (dict(t=0, lr=1.0), dict(t=1, lr=math.nan), dict(t=1, lr=1.0, betas=(1.0, 0.9)),
               dict(t=1, lr=1.0, eps=-1.0)):
        with pytest.raises(E):
            opt.step(**kw)
    assert (gamma == 1).all()

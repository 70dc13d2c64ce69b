"""The fine-tuning operators where their ranges end: states that fade away, logits far from 0, empty
batches, scratch of other streams, very many rows."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def normal(g, *shape, std=1.0, mean=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(dtype)


def test_adamw_8bit_blocks_that_lose_their_gradients(jc):
    """Three steps with gradients and 1300 without: the moments shrink with their blocks' scales, through
    the subnormal numbers. Nothing becomes NaN, and codes and scales stay those of the formula's
    operations rounded one by one in f32 (torch's own), bit for bit."""
    g = gen(41)
    n, size = 4, 3 * 256 + 100
    pad = n * 256 - size
    p, grad = normal(g, size, std=0.02), normal(g, size, std=1e-3)
    grad[256:512:3] = 0                              # elements that never had a gradient
    grad[512:768] *= 10.0 ** torch.linspace(-6, 0, 256, device="cuda")
    before = p.clone()
    opt = jc.AdamW([p], [grad], bits=8)
    m = v = torch.zeros(n, 256, device="cuda")
    lowest = math.inf
    for t in range(1, 1304):
        if t == 4:
            grad.zero_()
        opt.step(t, lr=1e-4, betas=(0.9, 0.9))
        gf = torch.nn.functional.pad(grad, (0, pad)).view(n, 256)
        m = (m * 0.9) + (gf * (1 - 0.9))
        v = (v * 0.9) + (gf * (1 - 0.9)) * gf
        out = []
        for x, floor in ((m, False), (v, True)):
            sc = x.abs().amax(1) * torch.tensor(1.0 / 448.0, dtype=torch.float32, device="cuda")
            y = x / torch.where(sc > 0, sc, 1.0)[:, None]
            y = torch.where(x > 0, y.clamp_min(2.0 ** -9), y) if floor else y
            out.append((y.clamp(-448, 448).to(torch.float8_e4m3fn), sc))
        (mc, ms), (vc, vs) = out
        assert torch.equal(opt.exp_avg_scale[0], ms) and torch.equal(opt.exp_avg_sq_scale[0], vs), t
        assert torch.equal(opt.exp_avg[0].view(torch.uint8), mc.view(-1)[:size].view(torch.uint8)), t
        assert torch.equal(opt.exp_avg_sq[0].view(torch.uint8), vc.view(-1)[:size].view(torch.uint8)), t
        m, v = mc.float() * ms[:, None], vc.float() * vs[:, None]
        lowest = min(lowest, float(ms.max()))
    assert lowest < 1e-43                            # the scales did go through the subnormals
    # Three steps of lr at most each way, then a tail of beta1's powers: 1 / (1 - 0.9) more of them.
    assert p.isfinite().all() and float((p - before).abs().max()) < 1e-4 * (3 + 10) * 10


def test_scratch_comes_from_the_pool_of_the_stream_that_uses_it(jc):
    """Backward calls queued on two streams side by side, none waiting for the other, have scratch of their
    own: the bits of calls one after the other."""
    g = gen(12)
    m, n, k, t = 4096, 768, 512, torch.float16
    x, w = normal(g, m, k + 1, dtype=t)[:, 1:], normal(g, n, k, std=0.05, dtype=t)  # x: copied into scratch
    gamma, xd = torch.ones(k, device="cuda"), normal(g, m, k, dtype=t)
    stats = torch.empty(m, 2, device="cuda")
    y = torch.empty_like(xd)
    jc.layer_norm(xd, gamma, None, y, stats=stats)

    def calls(dy, dn, stream):
        out = dict(dx=torch.empty(m, k, dtype=t, device="cuda"), dw=torch.empty_like(w),
                   dbias=torch.empty(n, device="cuda"))
        norm = torch.empty_like(xd), torch.empty_like(gamma), torch.empty_like(gamma)
        forward = torch.empty(m, n, dtype=t, device="cuda")
        yield (*out.values(), *norm, forward)
        jc.linear_backward(dy, x, w, z=dy, act="relu", stream=stream, **out)
        jc.layer_norm_backward(dn, xd, gamma, stats, *norm, stream=stream)
        jc.linear(x, w, forward, stream=stream)
        yield None
    data = [(normal(g, m, n, dtype=t), normal(g, m, k, dtype=t)) for _ in range(2)]
    want = []
    for dy, dn in data:
        c = calls(dy, dn, None)
        outs = next(c)
        next(c)
        torch.cuda.synchronize()
        want.append([o.clone() for o in outs])
    torch.cuda.empty_cache()
    side = torch.cuda.Stream()
    of_side = lambda: sum(s["total_size"] for s in torch.cuda.memory_snapshot() if s["stream"] == side.cuda_stream)  # noqa: E731
    assert of_side() == 0
    for stream in (side, side.cuda_stream):
        cs = [calls(*data[i % 2], stream if i % 2 else None) for i in range(12)]
        outs = [next(c) for c in cs]
        torch.cuda.synchronize()     # the outputs' storage is free on every stream
        for c in cs:
            next(c)
        torch.cuda.synchronize()
        for i, got in enumerate(outs):
            assert all(torch.equal(a, b) for a, b in zip(got, want[i % 2])), i
    assert of_side() >= m * n * 2    # dz at least
    assert jc.device_error() == 0


def test_adamw_first_step_on_a_stream_of_its_own(jc):
    """The table of a few thousand tensors is on the device when AdamW returns: a step at once, on a stream
    that is ordered behind no other, moves every parameter."""
    side = torch.cuda.Stream()
    for _ in range(5):
        base = torch.zeros(6000 * 300, device="cuda")
        p, grad = list(base.view(6000, 300)), list(torch.ones_like(base).view(6000, 300))
        m, v = (list(torch.zeros_like(base).view(6000, 300)) for _ in range(2))
        torch.cuda.synchronize()
        opt = jc.AdamW(p, grad, exp_avg=m, exp_avg_sq=v)
        opt.step(1, lr=0.5, stream=side)
        side.synchronize()
        assert (base + 0.5).abs().max() < 1e-6
        opt.close()


def test_adamw_states_are_zero_before_any_step(jc):
    """The states made by AdamW are there when it returns, for steps on any stream."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        p = torch.ones(1000, device="cuda")
        side.synchronize()
        torch.cuda._sleep(int(2e8))   # about 0.1 s
        opt = jc.AdamW([p], [torch.ones_like(p)], bits=8)
        assert side.query()
    opt.close()


@pytest.mark.parametrize("lo,hi", [(2, 8), (17, 24), (60, 120), (700, 900)])
@pytest.mark.parametrize("offset", [0.0, 1000.0, -1000.0, 30000.0])
def test_choice_loss_far_from_zero(jc, lo, hi, offset):
    """The loss depends on the logits' differences alone: logits far from 0 cost it nothing. Half of the
    requests are confident (the right logit leads by about 8). Bound: differences from the largest logit
    are rounded once, their exponentials off by |x| 2^-23 and 2^-22 of themselves (x e^-x is 0.37 at most)
    and the sum by its longest chain, 25: 64 x 2^-24 of 1 + the loss in all, whatever the offset."""
    g = gen(lo)
    requests = 200
    n = torch.randint(lo, hi + 1, (requests,), generator=g, device="cuda")
    off = torch.zeros(requests + 1, dtype=torch.int32, device="cuda")
    off[1:] = n.cumsum(0)
    gold = (torch.rand(requests, generator=g, device="cuda") * n).to(torch.int32)
    gold = torch.minimum(gold, n.to(torch.int32) - 1)
    lg = normal(g, int(off[-1]))
    lg[(off[:-1] + gold).long()[::2]] += 8 + math.log(hi)
    lg += offset
    loss, dl = torch.full((requests,), math.nan, device="cuda"), torch.full_like(lg, math.nan)
    jc.choice_loss(lg, off, gold, loss, dlogits=dl)
    rows = lg.double().split(n.tolist())
    want = torch.stack([torch.log(torch.exp(l - l.max()).sum()) + (l.max() - l[w]) for l, w in zip(rows, gold.tolist())])
    assert ((loss.double() - want).abs() <= 64 * 2.0 ** -24 * (1 + want)).all()


@pytest.mark.parametrize("n", [1, 3, 8, 9])
def test_linear_backward_of_no_rows_without_scratch(jc, n):
    """No rows: the gradients of the parameters are 0, and no scratch is asked for."""
    L, k = jc.lib(), 40
    w, dw = torch.ones(n, k, device="cuda", dtype=torch.float16), torch.full((n, k), math.nan, device="cuda", dtype=torch.float16)
    db = torch.full((n,), math.nan, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    args = (0, 0, None, n, None, k, w.data_ptr(), k, None, n, 0, n, k, None, k)
    assert L.jc_linear_backward(*args, dw.data_ptr(), k, db.data_ptr(), None, stream) == 0, jc.last_error()
    assert (dw == 0).all() and (db == 0).all()
    dw.fill_(math.nan)
    assert L.jc_linear_backward(*args, dw.data_ptr(), k, None, None, stream) == 0, jc.last_error()
    assert (dw == 0).all()
    db.fill_(math.nan)
    assert L.jc_linear_backward(*args, None, k, db.data_ptr(), None, stream) == 0, jc.last_error()
    assert (db == 0).all()


@pytest.mark.parametrize("d,t", [(771, torch.float16), (1001, torch.bfloat16), (2051, torch.float16), (509, torch.float32)])
def test_layer_norm_rows_after_the_tensors_first(jc, d, t):
    """Rows off 16-byte boundaries, many for each block: the first and last rows are copied by the threads,
    and the bulk copies that follow take their place. Every row is within u of 64 bits, and f32's error
    of sums (400 x 2^-24 of the magnitudes)."""
    g = gen(d)
    rows = 30011
    x, dy, add = (normal(g, rows, d, dtype=t) for _ in range(3))
    gamma, y, stats = torch.ones(d, device="cuda"), torch.full_like(x, math.nan), torch.empty(rows, 2, device="cuda")
    dx, dg, db = torch.full_like(x, math.nan), torch.empty_like(gamma), torch.empty_like(gamma)
    jc.layer_norm(x, gamma, None, y, stats=stats)
    jc.layer_norm_backward(dy, x, gamma, stats, dx, dg, db, add=add)
    assert jc.device_error() == 0
    u, f32 = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}[t], 400 * 2.0 ** -24
    x, dy, add = x.double(), dy.double(), add.double()
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + 1e-5)
    xh = (x - mean) * rstd
    mag = (x.abs() + x.abs().mean(1, keepdim=True)) * rstd
    assert ((y.double() - xh).abs() <= u * xh.abs() + f32 * mag + 2.0 ** -25).all()
    want = rstd * (dy - dy.mean(1, keepdim=True) - xh * (dy * xh).mean(1, keepdim=True)) + add
    tol = f32 * (rstd * (dy.abs() + 1 + mag * (1 + (dy * xh).abs().mean(1, keepdim=True))) + add.abs())
    assert ((dx.double() - want).abs() <= u * want.abs() + 2 * tol + 2.0 ** -25).all()
    assert ((dg.double() - (dy * xh).sum(0)).abs() <= f32 * (dy.abs() * mag).sum(0)).all()
    assert ((db.double() - dy.sum(0)).abs() <= f32 * dy.abs().sum(0)).all()


def test_linear_backward_of_millions_of_rows(jc):
    """More rows than 65535 blocks of 64. Sums of m values of variance 1 stay below 6 sqrt(m) on their way;
    the longest chain of additions is an eighth of 65535 partial sums (dbias) and the 16-row steps of one of
    32 splits (dw), 8300 either way, each addition within 2^-23 of what it adds to."""
    g = gen(6)
    m, n, k = 65535 * 64 + 77, 9, 8
    t = torch.bfloat16
    dy, x, w = normal(g, m, n, dtype=t), normal(g, m, k, dtype=t), normal(g, n, k, dtype=t)
    dx, dw, db = torch.full_like(x, math.nan), torch.full_like(w, math.nan), torch.full((n,), math.nan, device="cuda")
    jc.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db)
    assert jc.device_error() == 0
    u, d64, x64 = 2.0 ** -8, dy.double(), x.double()
    off = 8300 * 2.0 ** -23 * 6 * math.sqrt(m)
    assert ((db.double() - d64.sum(0)).abs() <= off).all()
    want = d64.t() @ x64
    assert ((dw.double() - want).abs() <= u * want.abs() + off).all()
    for a in (0, m // 2, m - 1000):
        d = d64[a:a + 1000]
        want = d @ w.double()
        assert ((dx[a:a + 1000].double() - want).abs() <= u * want.abs() + 32 * 2.0 ** -24 * (d.abs() @ w.double().abs())).all()


@pytest.mark.parametrize("rows,n", [(3, 1), (0, 8)])
def test_linear_backward_of_few_columns_and_a_long_contraction(jc, rows, n):
    """More contracted elements than the grid of the kernel for few columns has: each gradient within two
    roundings of the type (dz is exact here), dw 0 where there are no rows."""
    g = gen(n)
    k, t = 65535 * 256 + 8, torch.float16
    dy, x, w = normal(g, rows, n, dtype=t), normal(g, rows, k, dtype=t), normal(g, n, k, dtype=t)
    dx, dw, db = torch.full_like(x, math.nan), torch.full_like(w, math.nan), torch.full((n,), math.nan, device="cuda")
    jc.linear_backward(dy, x, w, dx=dx, dw=dw, dbias=db)
    assert jc.device_error() == 0
    tol = lambda a, b: 2.0 ** -10 * (a.double().abs() @ b.double().abs()) + 2.0 ** -25  # noqa: E731
    assert ((dx.double() - dy.double() @ w.double()).abs() <= tol(dy, w)).all()
    assert ((dw.double() - dy.double().t() @ x.double()).abs() <= tol(dy.t(), x)).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= 2.0 ** -22 * dy.double().abs().sum(0)).all()

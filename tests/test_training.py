"""The fine-tuning operators' C entry points on CPU: what they refuse, found on the host before any
launch, and their scratch sizes."""
import ctypes

import pytest

RELU, GELU = 64, 128


@pytest.fixture(scope="module")
def buf():
    raw = (ctypes.c_uint8 * 4096)()
    at = ctypes.addressof(raw)
    return raw, (at + 255) // 256 * 256


def test_layer_norm_refusals(jc, buf):
    L, p = jc.lib(), buf[1]

    def call(type=0, x=p, ldx=8, gamma=p, beta=p, eps=1e-5, rows=2, d=8, y=p, ldy=8, stats=p):
        return L.jc_layer_norm(type, x, ldx, gamma, beta, eps, rows, d, y, ldy, stats, None)
    for kw, why in ((dict(type=3), "element type"), (dict(d=0), "1 to 16384"), (dict(d=16385), "1 to 16384"),
                    (dict(x=None), "x is null"), (dict(y=None), "y is null"), (dict(gamma=None), "gamma is null"),
                    (dict(ldx=7), "rows overlap"), (dict(ldy=7), "rows overlap"), (dict(x=p + 1), "aligned"),
                    (dict(type=2, x=p + 2), "aligned"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                    (dict(eps=float("inf")), "eps"), (dict(beta=p + 2), "beta"), (dict(stats=p + 4), "stats")):
        assert call(**kw) == -1 and why in jc.last_error(), (kw, jc.last_error())
    assert call(rows=0, x=None, y=None) == 0   # nothing to do


def test_layer_norm_backward_refusals(jc, buf):
    L, p = jc.lib(), buf[1]

    def call(type=1, dy=p, x=p, gamma=p, stats=p, add=None, ldadd=8, rows=2, d=8, dx=p, lddx=8, dg=p, db=p, ws=p):
        return L.jc_layer_norm_backward(type, dy, 8, x, 8, gamma, stats, add, ldadd, rows, d, dx, lddx, dg, db, ws,
                                        None)
    for kw, why in ((dict(type=9), "element type"), (dict(dy=None), "dy is null"), (dict(x=None), "x is null"),
                    (dict(stats=None), "stats is null"), (dict(dx=None), "dx is null"), (dict(lddx=4), "overlap"),
                    (dict(add=p, ldadd=3), "add"), (dict(ws=None, rows=100), "ws is null"), (dict(dg=p + 1), "dgamma")):
        assert call(**kw) == -1 and why in jc.last_error(), (kw, jc.last_error())
    assert L.jc_layer_norm_ws_floats(100000, 768) >= 2 * 768


def test_linear_refusals(jc, buf):
    L, p = jc.lib(), buf[1]

    def fwd(type=0, act=0, x=p, ldx=8, w=p, ldw=8, bias=None, res=None, ldres=8, y=p, ldy=8, z=None, ldz=8, m=2,
            n=8, k=8, ws=None):
        return L.jc_linear(type, act, x, ldx, w, ldw, bias, res, ldres, y, ldy, z, ldz, m, n, k, ws, None)
    for kw, why in ((dict(type=2), "JC_F16 or JC_BF16"), (dict(act=1), "act"), (dict(act=RELU | GELU), "act"),
                    (dict(n=0), "must not be 0"), (dict(k=0), "must not be 0"), (dict(x=None), "x is null"),
                    (dict(w=None), "w is null"), (dict(y=None), "y is null"), (dict(ldw=7), "w's rows"),
                    (dict(res=p, ldres=2), "res's rows"), (dict(z=p + 1), "z is not aligned"),
                    (dict(bias=p + 2), "bias"), (dict(m=9000, n=600, k=700, ldx=701, ldw=700, ldy=600), "ws is null"),
                    (dict(m=9000, n=600, k=700, ldx=701, ldw=700, ldy=600, ws=p + 8), "ws is misaligned")):
        assert fwd(**kw) == -1 and why in jc.last_error(), (kw, jc.last_error())
    assert fwd(m=0, x=None, y=None) == 0

    def bwd(type=0, act=0, dy=p, x=p, w=p, z=None, m=2, n=8, k=8, dx=p, dw=p, db=p, ws=p, lddw=8):
        return L.jc_linear_backward(type, act, dy, 8, x, 8, w, 8, z, 8, m, n, k, dx, 8, dw, lddw, db, ws, None)
    for kw, why in ((dict(type=7), "JC_F16"), (dict(act=2), "act"), (dict(k=0), "must not be 0"),
                    (dict(dy=None), "dy is null"), (dict(x=None), "x is null"), (dict(w=None), "w is null"),
                    (dict(act=RELU), "z is null"), (dict(lddw=1), "dw's rows"), (dict(ws=None), "ws is null"),
                    (dict(ws=p + 16), "ws is misaligned")):
        assert bwd(**kw) == -1 and why in jc.last_error(), (kw, jc.last_error())
    size = L.jc_linear_backward_ws_bytes
    assert size(p, 768, p, 768, 4096, 2048, 768) >= 4096 * 2048 * 2   # dz
    assert size(p, 768, p, 768, 10, 0, 5) == 0
    assert L.jc_linear_ws_bytes(p, 768, p, 768, 4096, 2048, 768) == 0
    # A copy of x, of w, or of both, their rows on 16-byte boundaries.
    m, n = 9000, 600
    assert L.jc_linear_ws_bytes(p, 769, p, 768, m, n, 768) == m * 768 * 2
    assert L.jc_linear_ws_bytes(p, 768, p + 2, 768, m, n, 768) == n * 768 * 2
    assert L.jc_linear_ws_bytes(p, 767, p, 767, m, n, 767) == (m + n) * 768 * 2


def test_choice_loss_refusals(jc, buf):
    L, p = jc.lib(), buf[1]

    def call(logits=p, n=4, off=p, gold=p, weight=None, r=2, loss=p, dl=p):
        return L.jc_choice_loss(logits, n, off, gold, weight, r, loss, dl, None)
    for kw, why in ((dict(logits=None), "logits is null"), (dict(off=None), "offsets is null"),
                    (dict(gold=None), "gold is null"), (dict(loss=None), "loss is null"),
                    (dict(weight=p + 1), "weight"), (dict(dl=p + 2), "dlogits"), (dict(n=2 ** 31), "2^31")):
        assert call(**kw) == -1 and why in jc.last_error(), (kw, jc.last_error())
    assert call(r=0, off=None, gold=None, loss=None) == 0


def test_adamw_refusals(jc, buf):
    from importlib import import_module
    T = import_module("julia-cuda_b200.training").AdamwTensor
    L, p = jc.lib(), buf[1]

    def call(bits=32, count=1, **kw):
        f = dict(p=p, g=p, m=p, v=p, m_scale=p, v_scale=p, copy=None, n=8, weight_decay=0.0, grad_type=2, copy_type=0)
        f.update(kw)
        t = T(*[f[name] for name, _ in T._fields_])
        return L.jc_adamw_create(ctypes.byref(t), count, bits)
    for kw, why in ((dict(bits=16), "32 or 8"), (dict(p=None), "null"), (dict(g=None), "null"), (dict(v=None), "null"),
                    (dict(bits=8, m_scale=None), "scales"), (dict(grad_type=3), "gradient type"),
                    (dict(copy=p, copy_type=2), "copy_type"), (dict(weight_decay=float("nan")), "weight_decay"),
                    (dict(p=p + 2), "aligned"), (dict(copy=p + 1), "aligned"), (dict(n=2 ** 62), "too many")):
        assert not call(**kw) and why in jc.last_error(), (kw, jc.last_error())
    assert L.jc_adamw_step(None, 1, 0.1, 0.9, 0.999, 1e-8, None, None) == -1 and "no optimizer" in jc.last_error()
    L.jc_adamw_free(None)

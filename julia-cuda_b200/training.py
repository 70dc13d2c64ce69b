"""The fine-tuning operators on torch device tensors: layer norm, linear layers, the loss over a
request's choices and the AdamW step, with their gradients (include/julia_cuda.h, "fine-tuning
operators"). As with the inference kernels, outputs are the caller's tensors and everything is
queued on the current stream (or `stream`). Also available from the package itself.
"""
from __future__ import annotations

import ctypes
import importlib.util
import os

import torch

from . import HERE, JuliaCudaError, last_error, lib

F16, BF16, F32 = 0, 1, 2
_TYPES = {torch.float16: F16, torch.bfloat16: BF16, torch.float32: F32}


def _load_binding():
    """The compiled checks and calls (csrc/torch_binding.cpp)."""
    path = os.path.join(HERE, "_binding.so")
    if not os.path.exists(path):
        raise JuliaCudaError(f"{path} is not built (run build() / make -C julia-cuda_b200)")
    lib()
    spec = importlib.util.spec_from_file_location("_binding", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_error(JuliaCudaError)
    return module


_b = _load_binding()


def _fail(what: str):
    raise JuliaCudaError(what)


def _vector(op: str, name: str, t, n: int, dev: int, dtype=torch.float32):
    if t is None:
        return None
    if (t.dtype is not dtype or t.numel() != n or not t.is_cuda or t.get_device() != dev
            or not t.is_contiguous()):
        _fail(f"{op}: {name} must be a contiguous tensor on the current device of {n} elements of {dtype}")
    return t.data_ptr()


def layer_norm(x, gamma, beta, y, stats=None, eps: float = 1e-5, stream=None) -> None:
    """y = (x - mean) rstd gamma + beta per row (jc_layer_norm). x, y [rows, d] of one type (f16, bf16
    or f32), gamma and beta [d] f32 (beta may be None); stats, if given, [rows, 2] f32 receives mean
    and rstd for the backward pass."""
    _b.layer_norm(x, gamma, beta, y, stats, eps, stream)


def layer_norm_backward(dy, x, gamma, stats, dx, dgamma=None, dbeta=None, add=None, ws=None,
                        stream=None) -> None:
    """The gradients of layer_norm (jc_layer_norm_backward): dx (plus `add`, the gradient that
    reaches x past the norm), dgamma and dbeta [d] f32. ws: jc_layer_norm_ws_floats(rows, d) floats
    (allocated here when not given)."""
    _b.layer_norm_backward(dy, x, gamma, stats, dx, dgamma, dbeta, add, ws, stream)


def linear(x, w, y, *, bias=None, act: str = "none", res=None, z=None, ws=None, stream=None) -> None:
    """y = act(x w^T + bias) + res (jc_linear): x [m, k], w [n, k], y, res [m, n] of one 16-bit type,
    bias [n] f32. z, if given, keeps the values before the activation for the backward pass. ws:
    jc_linear_ws_bytes(...) bytes, needed where rows of x or w start off 16-byte boundaries (allocated
    here when not given)."""
    _b.linear(x, w, y, bias, act, res, z, ws, stream)


def linear_backward(dy, x, w, *, z=None, act: str = "none", dx=None, dw=None, dbias=None, ws=None,
                    stream=None) -> None:
    """The gradients of linear (jc_linear_backward), each written if its tensor is given: dx [m, k],
    dw [n, k] of x's type, dbias [n] f32. z (linear's) is read unless act is "none". ws:
    jc_linear_backward_ws_bytes(...) bytes (allocated here when not given)."""
    _b.linear_backward(dy, x, w, z, act, dx, dw, dbias, ws, stream)


def choice_loss(logits, offsets, gold, loss, dlogits=None, weight=None, stream=None) -> None:
    """Each request's loss over its own markers and its gradient (jc_choice_loss): logits f32,
    offsets int32 [requests + 1], gold int32 [requests] (the right marker of each request, below 0:
    none), weight f32 [requests]; writes loss [requests] and dlogits (as logits; those of logits that no
    request has are left alone)."""
    _b.choice_loss(logits, offsets, gold, loss, dlogits, weight, stream)


class AdamwTensor(ctypes.Structure):
    """jc_adamw_tensor."""

    _fields_ = [("p", ctypes.c_void_p), ("g", ctypes.c_void_p), ("m", ctypes.c_void_p),
                ("v", ctypes.c_void_p), ("m_scale", ctypes.c_void_p), ("v_scale", ctypes.c_void_p),
                ("copy", ctypes.c_void_p), ("n", ctypes.c_uint64), ("weight_decay", ctypes.c_float),
                ("grad_type", ctypes.c_uint32), ("copy_type", ctypes.c_uint32)]


class AdamW:
    """AdamW over many tensors, one launch a step (jc_adamw_create / jc_adamw_step).

    params: contiguous f32 device tensors; grads: a tensor of as many elements for each (f16, bf16 or
    f32), whose storage every step reads, so gradients are written in place; copies: optional f16 or
    bf16 tensors (or None) that receive the updated parameters. weight_decay: one number, or one for
    each tensor. bits: 32 or 8, the width of the states exp_avg and exp_avg_sq (f32, or float8_e4m3fn
    with a scale for each 256 elements in exp_avg_scale and exp_avg_sq_scale), made here as zeros
    unless given."""

    BLOCK = 256

    def __init__(self, params, grads, *, bits: int = 32, weight_decay=0.0, copies=None, exp_avg=None,
                 exp_avg_sq=None, exp_avg_scale=None, exp_avg_sq_scale=None):
        self._h = None
        self._dev = dev = torch.cuda.current_device()
        n = len(params)
        if bits not in (8, 32):
            _fail("AdamW: states of 32 or 8 bits")
        state = torch.float32 if bits == 32 else torch.float8_e4m3fn
        blocks = [-(-p.numel() // self.BLOCK) for p in params]
        new = lambda dt, sizes: [torch.zeros(k, dtype=dt, device=p.device)  # noqa: E731
                                 for p, k in zip(params, sizes)]
        sizes = [p.numel() for p in params]
        self.params, self.grads, self.bits = list(params), list(grads), bits
        self.copies = list(copies) if copies is not None else [None] * n
        self.exp_avg = list(exp_avg) if exp_avg is not None else new(state, sizes)
        self.exp_avg_sq = list(exp_avg_sq) if exp_avg_sq is not None else new(state, sizes)
        scaled = bits == 8
        self.exp_avg_scale = (list(exp_avg_scale) if exp_avg_scale is not None
                              else new(torch.float32, blocks) if scaled else [None] * n)
        self.exp_avg_sq_scale = (list(exp_avg_sq_scale) if exp_avg_sq_scale is not None
                                 else new(torch.float32, blocks) if scaled else [None] * n)
        decay = list(weight_decay) if hasattr(weight_decay, "__len__") else [weight_decay] * n
        if any(len(x) != n for x in (self.grads, self.copies, self.exp_avg, self.exp_avg_sq, decay,
                                     self.exp_avg_scale, self.exp_avg_sq_scale)):
            _fail("AdamW: as many gradients, states, copies and decays as parameters")
        table = (AdamwTensor * max(n, 1))()
        for i, p in enumerate(self.params):
            k, g, c, at = p.numel(), self.grads[i], self.copies[i], f"of tensor {i}"
            if p.get_device() != self._dev:
                _fail("AdamW: the tensors are not on the current device")
            if g.dtype not in _TYPES:
                _fail(f"AdamW: the gradient {at} must be float16, bfloat16 or float32")
            if c is not None and c.dtype not in (torch.float16, torch.bfloat16):
                _fail(f"AdamW: the copy {at} must be float16 or bfloat16")
            sc = blocks[i] if scaled else 0
            table[i] = AdamwTensor(
                _vector("AdamW", f"the parameter {at}", p, k, dev),
                _vector("AdamW", f"the gradient {at}", g, k, dev, g.dtype),
                _vector("AdamW", f"exp_avg {at}", self.exp_avg[i], k, dev, state),
                _vector("AdamW", f"exp_avg_sq {at}", self.exp_avg_sq[i], k, dev, state),
                _vector("AdamW", f"exp_avg_scale {at}", self.exp_avg_scale[i], sc, dev),
                _vector("AdamW", f"exp_avg_sq_scale {at}", self.exp_avg_sq_scale[i], sc, dev),
                None if c is None else _vector("AdamW", f"the copy {at}", c, k, dev, c.dtype), k,
                float(decay[i]), _TYPES[g.dtype], F32 if c is None else _TYPES[c.dtype])
        # The zeros made above are there before a step on whatever stream.
        torch.cuda.current_stream().synchronize()
        self._h = lib().jc_adamw_create(table, n, bits)
        if not self._h:
            raise JuliaCudaError(last_error())

    def step(self, t: int, *, lr: float, betas=(0.9, 0.999), eps: float = 1e-8, grad_scale=None,
             stream=None) -> None:
        """Step t (from 1). grad_scale: one f32 on the device that every gradient is multiplied by."""
        if not self._h:
            _fail("AdamW: closed")
        _b.adamw_step(self._h, self._dev, t, lr, betas[0], betas[1], eps, grad_scale, stream)

    def close(self) -> None:
        if self._h:
            lib().jc_adamw_free(self._h)
            self._h = None

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

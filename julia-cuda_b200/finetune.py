"""Fine-tunes the scorer (LayerNorm, lin1, GELU, lin2) of a checkpoint on labelled requests: the encoder
and the head stay as they are and run on the inference engine, the scorer trains on their outputs at
the marker rows with the operators of training.py.

    python -m julia-cuda_b200.finetune MODEL_DIR requests.jsonl labels.jsonl OUT_DIR
        [--epochs N] [--batch N] [--lr X] [--weight-decay X] [--bits 32|8] [--max-length N] [--seed N]

reads the requests as the julia-cuda executable does ({"ids", "markers", "qtype"}, one a line) and the
labels as scoring.py does ({"keys": one per marker, "gold": the right key}), prints each epoch's mean
loss and accuracy, and writes OUT_DIR as a checkpoint of the same model with the new scorer.
"""
from __future__ import annotations

import argparse
import json
import math
import sys

import numpy as np
import torch

from . import (AdamW, Engine, JuliaCudaError, choice_loss, layer_norm, layer_norm_backward, linear,
               linear_backward, raw_offsets, read_checkpoint, save_checkpoint)

QTYPES = {"choice": 0, "score": 1, "noul": 2}


def _head_rows(engine: Engine, n: int) -> int:
    """How many of a request's n rows the head runs on (Engine.set_head_length)."""
    return min(engine.head_length or n, n)


def _checked(engine: Engine, seqs):
    """The requests as arrays. Like julia_cuda_run, all are looked over before any is queued: the device
    calls follow the token ids and markers that they are given."""
    out = []
    for i, (ids, markers, qtype) in enumerate(seqs):
        ids, markers, qtype = np.asarray(ids, np.int64), np.asarray(markers, np.int64), int(qtype)
        past = ids[(ids < 0) | (ids >= engine.cfg.vocab)]
        head = _head_rows(engine, ids.size)
        why = ""
        if not ids.size:
            why = "no tokens"
        elif past.size:
            why = f"token id {past[0]} is past the vocabulary"
        elif ((markers < 0) | (markers >= head)).any():
            why = f"a marker is past the {'sequence' if head == ids.size else 'head rows'}"
        elif not 0 <= qtype < engine.cfg.n_qtypes:
            why = f"no question type {qtype}"
        if why:
            raise JuliaCudaError(f"features: sequence {i}: {why}")
        out.append((ids, markers, qtype))
    return out


def features(engine: Engine, seqs):
    """The scorer's inputs, the head's outputs at the marker rows: ([markers, D] f16, offsets int32
    [requests + 1]) of requests (ids, markers, qtype), on the engine's device."""
    rows, at = [], [0]
    layers = engine.cfg.n_head_layers + 1
    for ids, markers, qtype in _checked(engine, seqs):
        ids = torch.as_tensor(ids.astype(np.int32), device="cuda")
        mk = torch.as_tensor(markers.astype(np.int32), device="cuda")
        trace = torch.empty(layers, _head_rows(engine, ids.numel()), engine.cfg.d_model,
                            dtype=torch.float16, device="cuda")
        logits = torch.empty(max(mk.numel(), 1), device="cuda")
        engine.forward_trace(ids, mk, qtype, logits, head_trace=trace)
        rows.append(trace[-1][mk.long()])
        at.append(at[-1] + mk.numel())
    if engine.device_error():
        raise JuliaCudaError("features: the engine recorded a device error")
    x = torch.cat(rows) if rows else torch.empty(0, engine.cfg.d_model, dtype=torch.float16,
                                                 device="cuda")
    return x, torch.tensor(at, dtype=torch.int32, device="cuda")


class ScorerTrainer:
    """The scorer of a raw model (include/julia_cuda.h's raw format) in training: f32 parameters, 16-bit
    working copies of the two matrices, gradients and AdamW states of `bits` bits."""

    NAMES = ("norm.weight", "norm.bias", "lin1.weight", "lin1.bias", "lin2.weight", "lin2.bias")

    def __init__(self, cfg, raw: np.ndarray, *, lr: float = 1e-3, weight_decay: float = 0.01,
                 bits: int = 32, dtype=torch.float16, loss_scale: float = 1024.0):
        self.cfg, self.lr, self.dtype, self.loss_scale, self.t = cfg, lr, dtype, loss_scale, 0
        d, s = cfg.d_model, cfg.scorer_hidden
        shapes = ((d,), (d,), (s, d), (s,), (1, s), (1,))
        self._at = [int(o) for o in raw_offsets(cfg)[-len(shapes):]]
        self.params = [torch.from_numpy(np.array(raw[o:o + int(np.prod(n))], np.float32)).cuda().view(n)
                       for o, n in zip(self._at, shapes)]
        matrix = [len(n) == 2 for n in shapes]
        self.copies = [p.to(dtype) if m else None for p, m in zip(self.params, matrix)]
        # One buffer a type, so that a step looks two tensors over for infinities.
        sizes = [int(np.prod(n)) for n in shapes]
        flat = {m: torch.zeros(sum(k for k, o in zip(sizes, matrix) if o == m), device="cuda",
                               dtype=dtype if m else torch.float32) for m in (True, False)}
        cut = {m: iter(flat[m].split([k for k, o in zip(sizes, matrix) if o == m])) for m in flat}
        self.grads = [next(cut[m]).view(n) for n, m in zip(shapes, matrix)]
        self._flat_grads = list(flat.values())
        self.opt = AdamW(self.params, self.grads, bits=bits, copies=self.copies,
                         weight_decay=[weight_decay if m else 0.0 for m in matrix])

    def forward(self, x):
        """The logits [rows] f32 of features x [rows, D], and what the backward pass reads."""
        gamma, beta, _, b1, _, b2 = self.params
        w1, w2 = self.copies[2], self.copies[4]
        rows, new = x.shape[0], lambda n: torch.empty(x.shape[0], n, dtype=self.dtype, device=x.device)  # noqa: E731
        xn, z, h, y = new(x.shape[1]), new(w1.shape[0]), new(w1.shape[0]), new(1)
        stats = torch.empty(rows, 2, device=x.device)
        layer_norm(x, gamma, beta, xn, stats=stats, eps=self.cfg.head_eps)
        linear(xn, w1, h, bias=b1, act="gelu", z=z)
        linear(h, w2, y, bias=b2)
        return y[:, 0].float(), (x, xn, stats, z, h)

    def step(self, x, offsets, gold, weight=None):
        """One training step on features x (features()) of requests whose right markers are `gold` (int32,
        counted from the request's first; below 0: none). Returns (each request's loss, the logits before
        the step), on the device. Where a gradient is past what its type holds, nothing is updated and
        loss_scale is halved for the next step."""
        x = x.to(self.dtype)
        logits, (x, xn, stats, z, h) = self.forward(x)
        loss, dlogits = torch.empty(gold.numel(), device=x.device), torch.empty_like(logits)
        choice_loss(logits, offsets, gold, loss, dlogits=dlogits, weight=weight)
        # 16-bit gradients hold the loss times loss_scale; the optimizer divides by it, and by the
        # requests that count, without the host.
        counted = (gold >= 0).sum().clamp_min(1).float().reshape(1)
        dy = (dlogits * self.loss_scale).to(self.dtype)[:, None]
        w1, w2 = self.copies[2], self.copies[4]
        dgamma, dbeta, dw1, db1, dw2, db2 = self.grads
        dh, dxn, dx = torch.empty_like(h), torch.empty_like(xn), torch.empty_like(x)
        linear_backward(dy, h, w2, dx=dh, dw=dw2, dbias=db2)
        linear_backward(dh, xn, w1, z=z, act="gelu", dx=dxn, dw=dw1, dbias=db1)
        layer_norm_backward(dxn, x, self.params[0], stats, dx, dgamma, dbeta)
        # The largest magnitudes: infinite or NaN where any gradient is.
        matrices, vectors = (torch.linalg.vector_norm(g, math.inf) for g in self._flat_grads)
        if not math.isfinite(matrices + vectors):
            if self.loss_scale < 2.0 ** -10:
                raise JuliaCudaError("step: the gradients are not finite at any loss scale")
            self.loss_scale /= 2
            return loss, logits
        self.t += 1
        self.opt.step(self.t, lr=self.lr, grad_scale=1.0 / (self.loss_scale * counted))
        return loss, logits

    def write(self, raw: np.ndarray) -> np.ndarray:
        """A copy of the raw model with the trained scorer, for Engine.load_raw or save_checkpoint."""
        out = np.array(raw, np.float32)
        for o, p in zip(self._at, self.params):
            out[o:o + p.numel()] = p.detach().cpu().numpy().reshape(-1)
        return out


def read_requests(path: str):
    """(ids, markers, qtype) of each line, as the julia-cuda executable reads them."""
    with open(path) as f:
        lines = [json.loads(line) for line in f if line.strip()]
    return [(r["ids"], r.get("markers", []), QTYPES.get(r.get("qtype", 0), r.get("qtype", 0)))
            for r in lines]


def read_gold(path: str):
    """The right marker of each label line: the place of `gold` in `keys`, -1 if it is not there."""
    with open(path) as f:
        labels = [json.loads(line) for line in f if line.strip()]
    return [r["keys"].index(r["gold"]) if r["gold"] in r["keys"] else -1 for r in labels]


def train(engine: Engine, raw: np.ndarray, seqs, gold, *, epochs: int = 10, batch: int = 64,
          seed: int = 0, log=print, **kw) -> np.ndarray:
    """Trains the scorer on the requests and returns the new raw model. kw: ScorerTrainer's."""
    if len(seqs) != len(gold) or any(g >= len(s[1]) for s, g in zip(seqs, gold)):
        raise JuliaCudaError("train: one right marker for each request, among its markers")
    if not seqs:
        raise JuliaCudaError("train: no requests")
    x, offsets = features(engine, seqs)
    at = offsets.tolist()
    trainer = ScorerTrainer(engine.cfg, raw, **kw)
    rng = np.random.default_rng(seed)
    for epoch in range(epochs):
        order, losses, right, counted = rng.permutation(len(seqs)), [], 0, 0
        for b in range(0, len(order), batch):
            part = order[b:b + batch]
            n = [at[i + 1] - at[i] for i in part]
            rows = torch.as_tensor(np.concatenate([np.arange(at[i], at[i + 1]) for i in part]),
                                   device="cuda")
            off = torch.tensor(np.concatenate([[0], np.cumsum(n)]), dtype=torch.int32, device="cuda")
            g = torch.tensor([gold[i] for i in part], dtype=torch.int32, device="cuda")
            loss, logits = trainer.step(x[rows], off, g)
            losses.append(loss)
            for r, (l, want) in enumerate(zip(logits.split(n), g.tolist())):
                if want >= 0:
                    right, counted = right + int(int(l.argmax()) == want), counted + 1
        mean = float(torch.cat(losses).sum()) / max(counted, 1)
        log(f"epoch {epoch + 1}: mean loss {mean:.4f}, {right}/{counted} right")
    return trainer.write(raw)


def main(argv=None) -> int:
    p = argparse.ArgumentParser(prog="julia-cuda_b200.finetune", description=__doc__,
                                formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("model_dir")
    p.add_argument("requests")
    p.add_argument("labels")
    p.add_argument("out_dir")
    p.add_argument("--epochs", type=int, default=10)
    p.add_argument("--batch", type=int, default=64)
    p.add_argument("--lr", type=float, default=1e-3)
    p.add_argument("--weight-decay", type=float, default=0.01)
    p.add_argument("--bits", type=int, choices=(32, 8), default=32)
    p.add_argument("--max-length", type=int, default=0)
    p.add_argument("--seed", type=int, default=0)
    a = p.parse_args(argv)
    try:
        seqs, gold = read_requests(a.requests), read_gold(a.labels)
        cfg, raw = read_checkpoint(a.model_dir)
        longest = a.max_length or max([len(s[0]) for s in seqs], default=1)
        engine = Engine.load_raw(cfg, raw, max_length=longest)
        new = train(engine, raw, seqs, gold, epochs=a.epochs, batch=a.batch, seed=a.seed, lr=a.lr,
                    weight_decay=a.weight_decay, bits=a.bits)
        save_checkpoint(a.out_dir, cfg, new)
    except (JuliaCudaError, OSError, KeyError, ValueError) as e:
        print(f"finetune: {e}", file=sys.stderr)
        return 1
    return 0


if __name__ == "__main__":
    sys.exit(main())

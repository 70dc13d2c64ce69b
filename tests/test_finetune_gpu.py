"""Fine-tuning the scorer end to end: features from the engine, a training step against 64-bit autograd
of the same scorer, training to convergence, the new weights served by a new engine, and the command."""
import json

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup(jc):
    from importlib import import_module
    ft = import_module("julia-cuda_b200.finetune")
    cfg = jc.default_config(d_model=128, inter=128, n_layers=3, vocab=500, head_ff=128, scorer_hidden=64,
                            max_positions=128)
    raw = jc.init_random(cfg, 5)
    eng = jc.Engine.load_raw(cfg, raw, max_length=128)
    rng = np.random.default_rng(0)
    seqs = []
    for _ in range(60):
        n = int(rng.integers(20, 90))
        k = int(rng.integers(2, 7))
        seqs.append((rng.integers(0, 500, n).tolist(), sorted(rng.choice(n, k, replace=False).tolist()), 0))
    gold = [int(rng.integers(0, len(s[1]))) for s in seqs]
    return ft, cfg, raw, eng, seqs, gold


def test_features_give_the_engines_logits(jc, setup):
    """The scorer's forward pass over the features is the engine's own scorer (both in f16)."""
    ft, cfg, raw, eng, seqs, _ = setup
    x, off = ft.features(eng, seqs)
    logits, _ = ft.ScorerTrainer(cfg, raw).forward(x)
    want = torch.from_numpy(np.concatenate(eng.run(seqs)[0])).cuda()
    assert off.tolist()[-1] == x.shape[0] == want.numel()
    # f16 rounds the scorer's two layers and the logits once each: a few 2^-11 of the logits' size, and
    # the engine folds the norm into lin1's weights, rounded once more.
    assert (logits - want).abs().max() < 8 * 2.0 ** -11 * max(1.0, float(want.abs().max()))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_step_gradients_match_autograd(jc, setup, dtype):
    ft, cfg, raw, eng, seqs, gold = setup
    x, off = ft.features(eng, seqs)
    x = x.to(dtype)
    tr = ft.ScorerTrainer(cfg, raw, dtype=dtype, lr=0.0, weight_decay=0.0)
    g = torch.tensor(gold, dtype=torch.int32, device="cuda")
    g[3] = -1
    ps = [(c if c is not None else p).double().clone().requires_grad_() for p, c in zip(tr.params, tr.copies)]
    loss, _ = tr.step(x, off, g)
    xn = torch.nn.functional.layer_norm(x.double(), (cfg.d_model,), ps[0], ps[1], cfg.head_eps)
    lg = (torch.nn.functional.gelu(xn @ ps[2].t() + ps[3]) @ ps[4].t() + ps[5])[:, 0]
    total = [torch.logsumexp(l, 0) - l[int(w)] for l, w in zip(lg.split((off[1:] - off[:-1]).tolist()), g)
             if int(w) >= 0]
    want = torch.stack(total)
    u = 2.0 ** (-11 if dtype is torch.float16 else -8)
    assert (loss[g >= 0].double() - want).abs().max() < 16 * u
    assert loss[3] == 0
    grads = torch.autograd.grad(want.sum(), ps)
    # Each gradient passes up to six roundings of the type (dy, w2, dh's dz, dxn, the activations, itself).
    for name, a, b in zip(tr.NAMES[:-1], tr.grads, grads):
        e = float((a.double() / tr.loss_scale - b).norm() / b.norm())
        assert e < 8 * u, (name, e)
    # A shift of all logits changes no loss: lin2.bias's gradient is 0 but for dy's roundings, u of each
    # logit's gradient, of which a request's magnitudes sum to 2 at most.
    assert float((tr.grads[-1].double() / tr.loss_scale - grads[-1]).abs()) <= 2 * u * len(seqs)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_fits_the_labels(jc, setup, bits):
    """The labels are random, so only a trained scorer can hold them: it does, and an engine loaded
    with the new weights answers as the trainer does."""
    ft, cfg, raw, eng, seqs, gold = setup
    said = []
    new = ft.train(eng, raw, seqs, gold, epochs=60, batch=20, lr=5e-3, weight_decay=0.0, bits=bits,
                   log=said.append)
    eng2 = jc.Engine.load_raw(cfg, new, max_length=128)
    out, _ = eng2.run(seqs)
    right = sum(int(np.argmax(o)) == g for o, g in zip(out, gold))
    assert right >= 0.9 * len(gold), (right, said[0], said[-1])
    before = sum(int(np.argmax(o)) == g for o, g in zip(eng.run(seqs)[0], gold))
    assert before < 0.6 * len(gold)
    keep = jc.raw_offsets(cfg)[-6]
    assert np.array_equal(new[:keep], raw[:keep])   # nothing but the scorer moved
    eng2.close()


def test_train_refuses_a_marker_that_is_not_there(jc, setup):
    ft, cfg, raw, eng, seqs, gold = setup
    with pytest.raises(jc.JuliaCudaError):
        ft.train(eng, raw, seqs, [99] * len(seqs), epochs=1)


def test_command(jc, setup, tmp_path):
    ft, cfg, raw, eng, seqs, gold = setup
    src, out = tmp_path / "model", tmp_path / "out"
    src.mkdir()
    out.mkdir()
    jc.save_checkpoint(str(src), cfg, raw)
    (tmp_path / "req.jsonl").write_text("".join(json.dumps({"ids": s[0], "markers": s[1], "qtype": "choice"}) + "\n"
                                                for s in seqs))
    (tmp_path / "lab.jsonl").write_text("".join(
        json.dumps({"keys": [f"k{j}" for j in range(len(s[1]))], "gold": f"k{g}"}) + "\n" for s, g in zip(seqs, gold)))
    args = [str(src), str(tmp_path / "req.jsonl"), str(tmp_path / "lab.jsonl"), str(out), "--epochs", "3", "--lr", "5e-3"]
    assert ft.main(args) == 0
    cfg2, raw2 = jc.read_checkpoint(str(out))
    assert cfg2.scorer_hidden == cfg.scorer_hidden and not np.array_equal(raw2, raw)
    assert ft.main([str(tmp_path / "absent")] + args[1:]) == 1

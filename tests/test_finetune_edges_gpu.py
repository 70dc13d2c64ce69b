"""Fine-tuning the scorer where things go wrong: gradients past their type, nothing to train on."""
import importlib
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def setup(jc):
    """The module, a model, and features of requests as the engine would give them."""
    ft = importlib.import_module("julia-cuda_b200.finetune")
    cfg = jc.default_config(d_model=128, inter=128, n_layers=3, vocab=500, head_ff=128, scorer_hidden=64,
                            max_positions=128)
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(240, cfg.d_model, generator=g, device="cuda").half()
    off = torch.arange(0, 241, 4, dtype=torch.int32, device="cuda")
    gold = torch.randint(0, 4, (60,), generator=g, device="cuda").int()
    return ft, cfg, jc.init_random(cfg, 5), x, off, gold


def test_gradients_past_f16_skip_the_step(setup):
    """A loss scale that overflows f16 leaves the scorer and the optimizer as they were, and is halved until
    steps go through."""
    ft, cfg, raw, x, off, gold = setup
    tr = ft.ScorerTrainer(cfg, raw, loss_scale=2.0 ** 19)
    before = [p.clone() for p in tr.params]
    tr.step(x, off, gold)
    assert tr.t == 0 and tr.loss_scale == 2.0 ** 18
    assert all(torch.equal(a, b) for a, b in zip(before, tr.params))
    assert all((s == 0).all() for s in tr.opt.exp_avg)
    for _ in range(20):
        tr.step(x, off, gold)
    assert tr.t > 0 and all(p.isfinite().all() for p in tr.params)
    assert not torch.equal(before[2], tr.params[2])


def test_features_that_are_not_finite_end_in_an_error(jc, setup):
    ft, cfg, raw, x, off, gold = setup
    tr = ft.ScorerTrainer(cfg, raw)
    before = [p.clone() for p in tr.params]
    bad = x.clone()
    bad[7, 5] = math.nan
    with pytest.raises(jc.JuliaCudaError, match="not finite"):
        for _ in range(60):
            tr.step(bad, off, gold)
    assert tr.t == 0 and all(torch.equal(a, b) for a, b in zip(before, tr.params))


def test_nothing_to_train_on(jc, setup, tmp_path, capsys):
    """No requests is an error of the call and of the command; requests without markers train nothing."""
    ft, cfg, raw = setup[:3]
    eng = jc.Engine.load_raw(cfg, raw, max_length=64)
    with pytest.raises(jc.JuliaCudaError, match="no requests"):
        ft.train(eng, raw, [], [], epochs=1)
    new = ft.train(eng, raw, [(list(range(9)), [], 0)] * 3, [-1] * 3, epochs=2, weight_decay=0.0)
    assert np.array_equal(new, raw)
    eng.close()
    (tmp_path / "model").mkdir()
    (tmp_path / "out").mkdir()
    jc.save_checkpoint(str(tmp_path / "model"), cfg, raw)
    (tmp_path / "empty.jsonl").write_text("\n")
    args = [str(tmp_path / n) for n in ("model", "empty.jsonl", "empty.jsonl", "out")]
    assert ft.main(args) == 1 and "no requests" in capsys.readouterr().err


def test_features_under_a_head_length(jc, setup):
    """An engine whose head runs on the first rows of a request only: the scorer over its features gives the
    engine's own logits, and markers past those rows are refused."""
    ft, cfg, raw = setup[:3]
    eng = jc.Engine.load_raw(cfg, raw, max_length=128)
    rng = np.random.default_rng(4)
    seqs = [(rng.integers(0, 500, n).tolist(), sorted(rng.choice(min(n, 20), 4, replace=False).tolist()), 0)
            for n in (90, 12, 33, 20, 64)]
    eng.set_head_length(20)
    x, off = ft.features(eng, seqs)
    logits, _ = ft.ScorerTrainer(cfg, raw).forward(x)
    want = torch.from_numpy(np.concatenate(eng.run(seqs)[0])).cuda()
    # f16 rounds the scorer's two layers and the logits once each, and the engine lin1's folded weights.
    assert (logits - want).abs().max() < 8 * 2.0 ** -11 * max(1.0, float(want.abs().max()))
    with pytest.raises(jc.JuliaCudaError, match="sequence 1: a marker is past the head rows"):
        ft.features(eng, [seqs[0], (list(range(40)), [20], 0)])
    eng.set_head_length(0)
    assert ft.features(eng, [(list(range(40)), [20], 0)])[0].shape == (1, cfg.d_model)
    eng.close()

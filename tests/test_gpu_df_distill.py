"""GPU: the DF observer's trainer learning from another observer's top logits (wfd_distill in the step's launch plan), its quality
read-out (wfd_label_scores) and the command line around both."""
import os

import numpy as np
import pytest
import torch

from oracle import wfdgan_oracle as O
from tests import heads_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _engine(L, C, B, **kw):
    from wfd_gan_amd.df_engine import DFTrainEngine
    torch.manual_seed(3)
    return DFTrainEngine(L, C, B, O.make_df_state(L, C), device=DEV, seed=5, **kw)


@pytest.mark.parametrize("shape", [(72, 7, 16, 5), (200, 100, 33, 10), (96, 300, 8, 64)])
def test_step_uses_the_teachers_entries(shape):
    """Loss and logit gradient of a training step against the definition on the step's own logits; the classifier's weight
    gradient is their product with the head's input."""
    from wfd_gan_amd.df_engine import Distill
    L, C, B, k = shape
    d = Distill(k, 2.0, 0.6)
    eng = _engine(L, C, B, distill=d)
    g = torch.Generator().manual_seed(9)
    x, y = torch.rand(B, L, generator=g), torch.randint(0, C, (B,), generator=g)
    ti = torch.stack([torch.randperm(C, generator=g)[:k] for _ in range(B)]).to(torch.int32)
    tv = torch.randn(B, k, generator=g)
    ti[1, k // 2:] = -1
    eng.set_batch(x, y)
    eng.set_teacher(ti, tv)
    eng.draw_masks()
    eng.train_step()
    torch.cuda.synchronize()
    logits = eng.buf["LOG"][:, :C].cpu()
    loss, bl, grad, bd = R.distill(logits, ti, tv, y.to(torch.int32), d.temperature, d.weight, 1.0 - d.weight,
                                   torch.full((B,), 1.0 / B))
    R.check(eng.buf["CE"], loss, bl, torch.float32, "loss")
    R.check(eng.buf["DLOG"][:, :C], grad, bd, torch.float32, "dlogits")
    assert abs(eng.loss() - float(loss.mean())) <= 1e-5 * float(loss.abs().mean())      # B <= 33 additions: 33 U of the sum
    want = eng.buf["DLOG"][:, :C].double().cpu().T @ eng.buf["Hd2"].double().cpu()
    got = eng.P.g["fc.weight"].double().cpu()
    assert float((got - want).abs().max()) <= 1e-5 * float(want.abs().max())            # B products per entry


def test_without_a_teacher_nothing_changes():
    """weight 0 is the labels' cross entropy: the loss of the plain step on the same batch and masks."""
    from wfd_gan_amd.df_engine import Distill
    a, b = _engine(200, 10, 16), _engine(200, 10, 16, distill=Distill(4, 2.0, 0.0))
    g = torch.Generator().manual_seed(2)
    x, y = torch.rand(16, 200, generator=g), torch.randint(0, 10, (16,), generator=g)
    for e in (a, b):
        e.set_batch(x, y)
        e.draw_masks()
        e.train_step()
    assert abs(a.loss() - b.loss()) <= 1e-6 * abs(a.loss()) + 1e-6      # log-sum-exp of 10 values twice: some U each
    with pytest.raises(RuntimeError, match="without distill"):
        a.set_teacher(torch.zeros(16, 4, dtype=torch.int32), torch.zeros(16, 4))
    for bad in (Distill(0), Distill(11), Distill(4, 0.0), Distill(4, 1.0, 1.5)):
        with pytest.raises(ValueError, match="distill"):
            _engine(200, 10, 16, distill=bad)


def test_refusals_of_a_teachers_rows_and_of_k():
    """A teacher's row for all traces would be spread over the batch without a word; the best alternative is what top1 counts."""
    from wfd_gan_amd.df_engine import Distill
    e = _engine(96, 9, 6, distill=Distill(4))
    for bad in ((1, 4), (4,), (6, 3), (7, 4)):
        with pytest.raises(ValueError, match="set_teacher"):
            e.set_teacher(torch.zeros(bad, dtype=torch.int32), torch.zeros(bad))
    with pytest.raises(ValueError, match="set_teacher"):
        e.set_teacher(torch.zeros(6, 4, dtype=torch.int32), torch.zeros(1, 4))
    X, y = torch.rand(5, 96, device=DEV), torch.zeros(5, dtype=torch.int32, device=DEV)
    for k in (0, -1, 65):
        with pytest.raises(ValueError, match="evaluate: k"):
            e.evaluate(X, y, k)
    assert e.evaluate(X, y, 64).keys() == {"top1", "top_k", "logprob", "entropy"}


@pytest.mark.parametrize("C,k", [(7, 3), (100, 5), (3, 5)])
def test_evaluate_and_teacher_alternatives(C, k):
    from wfd_gan_amd.df_engine import teacher_alternatives
    L, N = 120, 150
    eng = _engine(L, C, 8)
    g = torch.Generator().manual_seed(7)
    X = torch.rand(N, L, generator=g)
    y = torch.randint(0, C, (N,), generator=g)
    sd = {n: v.cpu() for n, v in eng.state_dict().items()}
    logits = O.df_forward({n: (v.double() if v.is_floating_point() else v) for n, v in sd.items()}, X.double()[:, None, :])
    lp = logits.log_softmax(1)
    got = eng.evaluate(X.to(DEV), y.to(DEV), k, bs=64)
    kk = min(k, C)
    hit = logits.topk(kk, dim=1).indices == y[:, None]
    assert abs(got["top1"] - float(hit[:, 0].double().mean())) <= 1.0 / N + 1e-9           # a tie of rounding may swap one row
    assert abs(got["top_k"] - float(hit.any(1).double().mean())) <= 1.0 / N + 1e-9
    # the observer's fp32 forward is within 1e-4 of the 64-bit one on these inputs (its own tests: 1e-3)
    assert abs(got["logprob"] - float(lp.gather(1, y[:, None]).mean())) <= 1e-3
    assert abs(got["entropy"] - float(-(lp.exp() * lp).sum(1).mean())) <= 1e-3
    assert got["top1"] == eng.accuracy(X.to(DEV), y.to(DEV), bs=64)
    ti, tv = teacher_alternatives(eng.state_dict(), L, C, X.to(DEV), kk, bs=64)
    assert ti.shape == (N, kk) and bool((tv[:, :-1] >= tv[:, 1:]).all())
    assert float((tv.cpu().double() - lp.gather(1, ti.cpu().long())).abs().max()) <= 1e-3


def test_train_df_cli_learns_from_a_teacher(tmp_path, capsys):
    """The command runs from dataset to checkpoint with a teacher, and refuses one that does not fit."""
    from wfd_gan_amd import train_df
    from wfd_gan_amd.model import DF
    n_cls, n_inst, L = 4, 30, 96
    rng = np.random.default_rng(0)
    X = np.zeros((n_cls * n_inst, L + 1))
    y = np.repeat(np.arange(n_cls), n_inst)
    for r in range(X.shape[0]):
        n = rng.integers(40, L)
        X[r, 0] = n
        X[r, 1:1 + n] = rng.integers(1, 6, n) + (np.arange(n) % (r // n_inst + 2) == 0) * 20
    npz = str(tmp_path / "raw_feature_x.npz")
    np.savez(npz, features=X, labels=y)
    teacher, student = str(tmp_path / "teacher.ckpt"), str(tmp_path / "student.ckpt")
    base = [npz, "--num_epochs", "1", "--batch_size", "32", "--seed", "1"]
    train_df.main(base + ["--out", teacher])
    path, losses, _ = train_df.main(base + ["--out", student, "--teacher", teacher, "--teacher_k", "3", "--top_k", "2"])
    assert path == student and os.path.isfile(student) and np.isfinite(losses).all()
    DF(L, n_cls).load_state_dict(torch.load(student, weights_only=True), strict=True)
    other = str(tmp_path / "other.ckpt")
    torch.save(DF(L, n_cls + 1).state_dict(), other)
    with pytest.raises(RuntimeError, match="size mismatch"):
        train_df.main(base + ["--out", student, "--teacher", other])

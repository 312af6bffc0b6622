"""GPU: the DF observer's read-outs over rows that are on the host, on the GPU, or in another layout."""
import pytest
import torch

from oracle import wfdgan_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_read_outs_of_rows_on_the_host():
    """accuracy() and evaluate() copy each batch to the GPU; the numbers are those of rows that are there already."""
    from wfd_gan_amd.df_engine import DFTrainEngine
    L, C, N = 120, 7, 150
    torch.manual_seed(3)
    eng = DFTrainEngine(L, C, 8, O.make_df_state(L, C), device=DEV)
    g = torch.Generator().manual_seed(7)
    X, y = torch.rand(N, L, generator=g), torch.randint(0, C, (N,), generator=g)
    there = eng.accuracy(X.to(DEV), y.to(DEV), bs=64), eng.evaluate(X.to(DEV), y.to(DEV), 3, bs=64)
    assert (eng.accuracy(X, y, bs=64), eng.evaluate(X, y, 3, bs=64)) == there
    assert (eng.accuracy(X[:, None], y, bs=64), eng.evaluate(X.double(), y.to(DEV), 3, bs=64)) == there


def test_read_outs_run_on_their_own_device(monkeypatch):
    """Launch plans take the current device's stream: the read-outs make theirs the current one, so that the plans' work is ordered
    with what the tensors' own device does."""
    from wfd_gan_amd import df_engine
    entered = []

    class Device(torch.cuda.device):
        def __init__(self, device):
            entered.append(torch.device(device))
            super().__init__(device)
    torch.manual_seed(3)
    eng = df_engine.DFTrainEngine(96, 5, 4, O.make_df_state(96, 5), device=DEV)
    X, y = torch.rand(9, 96, device=DEV), torch.zeros(9, dtype=torch.int64, device=DEV)
    monkeypatch.setattr(torch.cuda, "device", Device)
    for call in (lambda: eng.accuracy(X, y), lambda: eng.evaluate(X, y, 2),
                 lambda: df_engine.teacher_alternatives(eng.state_dict(), 96, 5, X, 2)):
        entered.clear()
        call()
        assert torch.device(DEV) in entered


def test_labels_of_the_read_outs():
    """A column of labels counts as labels; fewer than there are rows are refused before anything reads them."""
    from wfd_gan_amd.df_engine import DFTrainEngine
    torch.manual_seed(3)
    eng = DFTrainEngine(96, 5, 4, O.make_df_state(96, 5), device=DEV)
    g = torch.Generator().manual_seed(4)
    X, y = torch.rand(40, 96, generator=g).to(DEV), torch.randint(0, 5, (40,), generator=g)
    assert eng.evaluate(X, y[:, None], 2) == eng.evaluate(X, y, 2) and eng.accuracy(X, y[:, None]) == eng.accuracy(X, y)
    for who in ("accuracy", "evaluate"):
        with pytest.raises(ValueError, match=f"{who}: 40 rows"):
            getattr(eng, who)(X, y[:39])


def test_a_step_that_learns_from_a_teacher_needs_the_batchs_entries():
    """Without them it would train on the labels' share of the loss alone, or on the entries of the batch before, without a word."""
    from wfd_gan_amd.df_engine import DFTrainEngine, Distill
    torch.manual_seed(3)
    state = O.make_df_state(96, 5)
    eng = DFTrainEngine(96, 5, 4, state, device=DEV, distill=Distill(3))
    g = torch.Generator().manual_seed(4)
    x, y = torch.rand(4, 96, generator=g), torch.randint(0, 5, (4,), generator=g)
    ti, tv = torch.tensor([[0, 1, 2]] * 4, dtype=torch.int32), torch.randn(4, 3, generator=g)
    eng.draw_masks()
    with pytest.raises(RuntimeError, match="set_teacher was not called"):
        eng.train_step()
    for _ in range(2):
        eng.set_batch(x, y)
        with pytest.raises(RuntimeError, match="set_teacher was not called"):
            eng.train_step()
        eng.set_teacher(ti, tv)
        for _ in range(2):                                # several steps on one batch
            eng.train_step()
    eng.set_teacher(ti, tv)                               # the other way round
    eng.set_batch(x, y)
    eng.train_step()
    assert int(eng.step.item()) == 5
    eng.forward_train()                                   # the forward pass alone needs no teacher
    plain = DFTrainEngine(96, 5, 4, state, device=DEV, distill=Distill(3, 2.0, 0.0))
    plain.set_batch(x, y)
    plain.draw_masks()
    plain.train_step()                                    # nor does a share of 0

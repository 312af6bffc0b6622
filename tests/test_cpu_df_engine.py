"""CPU: host-side decisions of the DF observer's engine around the classifier-head operators; nothing here reaches a GPU."""
from types import SimpleNamespace

import pytest
import torch

from wfd_gan_amd import df_engine


def test_observer_batches_are_on_the_observers_device_wherever_the_rows_are(monkeypatch):
    """Kernels get the addresses of these buffers: rows on the host must not put them there ("meta" stands for the GPU)."""
    seen = []
    buffers = dict(Y=None, PO=None, F1=None, F2=None, LOG=torch.zeros(3, 4), ldc=4)
    monkeypatch.setattr(df_engine, "observer_buffers", lambda df, n, dev: (seen.append(torch.device(dev)), buffers)[1])
    monkeypatch.setattr(df_engine, "observer_forward", lambda pl, df, xin, *a: seen.append(xin.device))
    monkeypatch.setattr(df_engine, "Plan", lambda ws: SimpleNamespace(run=lambda: None))
    df = SimpleNamespace(L=5, C=2, fc_w=torch.empty(2, 512, device="meta"))
    got = [(a, tuple(l.shape)) for a, l in df_engine.observer_logits(df, torch.zeros(7, 5), None, 3)]
    assert [a for a, _ in got] == [0, 3, 6] and got[0][1] == (3, 2)
    assert len(seen) == 4 and all(d.type == "meta" for d in seen)


def test_teacher_alternatives_refuses_rows_on_the_host():
    with pytest.raises(ValueError, match="must be on the GPU"):
        df_engine.teacher_alternatives({}, 5, 2, torch.zeros(7, 5), 1)


def test_read_outs_refuse_fewer_labels_than_rows():
    """Kernels read a label per row; the engine here is a shell that was never built."""
    eng = object.__new__(df_engine.DFTrainEngine)
    eng.dev = torch.device("cpu")
    X = torch.zeros(7, 5)
    for shape in ((6,), (0,), (7, 2), (3, 3), ()):
        with pytest.raises(ValueError, match="accuracy: 7 rows"):
            eng._labels(X, torch.zeros(shape, dtype=torch.int64), "accuracy")
    for shape in ((7,), (7, 1), (9,)):
        assert eng._labels(X, torch.arange(9)[:shape[0]].reshape(shape), "accuracy").tolist()[:7] == list(range(7))


@pytest.mark.parametrize("k", [0, -1, 6, 65])
def test_teacher_alternatives_refuses_a_k_that_an_engine_does_not_take(k):
    with pytest.raises(ValueError, match="k must be 1 .. 5"):
        df_engine.teacher_alternatives({}, 5, 5, torch.zeros(7, 5), k)

"""The scratch of the table's gradient is asked for on the tensors' device, without a GPU."""
import contextlib

import torch

from equitorch_b200 import _lib
from equitorch_b200.ops import embedding_op


def test_scratch_is_of_the_tensors_device(monkeypatch):
    inside, asked = [], []

    @contextlib.contextmanager
    def on_device(dev):
        inside.append(dev)
        yield
        inside.pop()

    class Library:
        def eqt_embedding_grad_scratch(self, *_):
            asked.append(list(inside))
            return 512

        def eqt_embedding_grad(self, *args):
            assert inside and args[9] == 512
            return 0
    monkeypatch.setattr(_lib, "on_device", on_device)
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: t[0].device)
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: None)
    monkeypatch.setattr(_lib, "lib", lambda: Library())
    embedding_op.embedding_grad(torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4), 5, 1.0)
    assert asked == [[torch.device("cpu")]]

"""Which device the library is bound to."""
import torch

from kvhip import _lib as L


def test_first_use_binds_the_current_device(monkeypatch):
    """`kvhip_init` makes its device the current one: a first call on another device than the first stays there."""
    bound = []

    class Library:
        @staticmethod
        def kvhip_init(device):
            bound.append(device)
            return 0

    monkeypatch.setattr(L, "load", lambda: Library)
    for available, given, want in ((True, (), 3), (False, (), 0), (True, (5,), 5)):
        monkeypatch.setattr(L, "_inited", False)
        monkeypatch.setattr(torch.cuda, "is_available", lambda: available)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: 3)
        L.init(*given)
        L.init()
        assert bound.pop() == want and not bound

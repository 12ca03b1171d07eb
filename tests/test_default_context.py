"""The process-wide contexts: one for each device, kept."""
import pytest

torch = pytest.importorskip("torch")
import shoehorn_b200 as sh  # noqa: E402


def test_a_device_keeps_its_context_while_others_are_used(monkeypatch):
    """A captured graph holds its context's status word, and work may be under
    way: a call for another device must not free the first one's context."""
    made, freed, now = [], [], [0]

    class Fake:
        def __init__(self, device):
            self.torch, self.device = torch, device
            made.append(device)

        def __del__(self):
            freed.append(self.device)

    monkeypatch.setattr(sh, "Context", Fake)
    monkeypatch.setattr(sh, "_default_ctxs", {}, raising=False)
    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    first = id(sh.default_context())
    assert sh.default_context(device=1).device == 1
    now[0] = 1
    assert sh.default_context().device == 1
    assert not freed and id(sh.default_context(0)) == first
    assert made == [0, 1]

"""smoke()'s check of the 8-bit product, on the CPU: a context that answers as
the device should passes, one whose product or numbers are NaN does not."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import __graft_entry__ as entry  # noqa: E402
import shoehorn_b200 as sh  # noqa: E402
from oracle import oracle as O  # noqa: E402


class Answers:
    """The calls that smoke() makes; codes are the numbers themselves."""
    spoil = None

    def __init__(self, device):
        self.bits = self.im = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        pass

    def encode_rows(self, ty, src, im, sync):
        self.bits, self.im = src.numpy().view(np.uint16), im.numpy()
        return torch.from_numpy(O.encode_tensor_bf16(int(ty), self.bits, self.im, n_threads=1))

    def row_errors(self, types, src, im):
        return torch.from_numpy(np.stack([O.row_errors_bf16(int(t), self.bits, self.im, n_threads=1) for t in types]))

    def encode_f8(self, x, block_rows=1):
        return x, None

    def matmul_f8(self, a, sa, w, sw, dtype):
        return self.given("product", a @ w.t())

    def decode_f8(self, codes, scales, block_rows=1, sync=False):
        return self.given("rows" if block_rows == 1 else "weight", codes.clone())

    def given(self, what, t):
        if self.spoil == what:
            t.view(-1)[-1] = float("nan")
        return t


@pytest.fixture
def smoke(monkeypatch):
    monkeypatch.setattr(sh, "Context", Answers)
    monkeypatch.setattr(torch.Tensor, "cuda", lambda self: self)
    return entry.smoke


def test_right_answers_pass(smoke):
    smoke()


@pytest.mark.parametrize("what", ["product", "rows", "weight"])
def test_nan_does_not(smoke, monkeypatch, what):
    monkeypatch.setattr(Answers, "spoil", what)
    with pytest.raises(AssertionError, match="8-bit product"):
        smoke()

"""What needs no GPU of the 8-bit blocks: refusals of the C entry points, and
the pointers, sizes and strides that the Python calls hand them."""
import pytest

torch = pytest.importorskip("torch")
import shoehorn_b200 as sh  # noqa: E402


class Recorder:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


class CpuContext(sh.Context):
    """Takes CPU tensors for the device's, and launches nothing."""

    def __init__(self):
        self.torch, self.device, self.handle = torch, 0, None

    def _f8_here(self, t, what):
        pass

    def _f8_stream(self):
        return None


@pytest.fixture
def rec(monkeypatch):
    r = Recorder()
    monkeypatch.setattr(sh, "lib", lambda: r)
    return r


def test_c_entry_points_refuse_without_a_context():
    L = sh.lib()
    assert L.shc_encode_f8(None, 30, None, 1, 1, 128, 128, 0, 1, None, 128, 0, None, None) == -1
    assert L.shc_decode_f8(None, 30, None, 1, 1, 128, 128, 0, 1, None, None, None) == -1
    assert L.shc_matmul_f8(None, None, 128, None, 1, 0, None, 128, None, 1, 128, 0, 30, None, 1, None) == -1
    assert L.shc_matmul_f8_grouped(None, None, 128, None, 1, 0, None, 128, 128, None, 1, 1, 128, None, 0, 0, 30, None, 1,
                                   None) == -1


def test_tensors_of_another_device_are_refused():
    ctx = CpuContext()
    del CpuContext._f8_here  # the real check
    try:
        with pytest.raises(ValueError, match="cuda:0"):
            ctx.encode_f8(torch.zeros(2, 128))
    finally:
        CpuContext._f8_here = lambda self, t, what: None


@pytest.mark.parametrize("cols,pitch", [(1, 16), (16, 16), (17, 32), (128, 128), (1030, 1040)])
def test_encode_lays_rows_on_16_byte_boundaries(rec, cols, pitch):
    codes, scales = CpuContext().encode_f8(torch.zeros(3, cols), 1)
    assert codes.stride() == (pitch, 1) and codes.shape == (3, cols)
    assert scales.shape == (3, -(-cols // 128))
    (name, args), = rec.calls
    assert name == "shc_encode_f8" and args[3:9] == (1, 3, cols, cols, 0, 1) and args[10] == pitch
    codes, scales = CpuContext().encode_f8(torch.zeros(2, 130, cols), 128)
    assert codes.stride() == (130 * pitch, pitch, 1) and scales.shape == (2, 2, -(-cols // 128))
    assert rec.calls[1][1][3:9] == (2, 130, cols, cols, 130 * cols, 128)


def test_products_pass_strides_on(rec):
    ctx = CpuContext()
    a, sa = ctx.encode_f8(torch.zeros(10, 300))
    w, sw = ctx.encode_f8(torch.zeros(4, 200, 300), 128)
    off = torch.zeros(5, dtype=torch.int64)
    rec.calls.clear()
    out = torch.zeros(10, 256)[:, 3:203]
    ctx.matmul_f8_grouped(a, sa, w, sw, off, out=out)
    name, v = rec.calls[0]
    assert name == "shc_matmul_f8_grouped"
    assert (v[2], v[4], v[5], v[7], v[8]) == (304, 3, 10, 304, 200 * 304)
    assert v[10:13] == (4, 200, 300) and v[14:17] == (True, False, 0) and v[18] == 256
    g, sg = ctx.encode_f8(torch.zeros(1, 200))
    rec.calls.clear()
    d = ctx.matmul_f8(g, sg, w[2], sw[2], transposed=True)
    name, v = rec.calls[0]
    assert d.shape == (1, 300) and d.dtype == torch.bfloat16
    assert (v[2], v[4], v[5], v[7], v[9], v[10], v[11], v[12], v[14]) == (208, 2, 1, 304, 200, 300, True, 30, 300)


def test_shapes_and_layouts_that_are_refused(rec):
    ctx = CpuContext()
    a, sa = ctx.encode_f8(torch.zeros(4, 256))
    w, sw = ctx.encode_f8(torch.zeros(128, 256), 128)
    off = torch.zeros(2, dtype=torch.int32)
    rec.calls.clear()
    for call, kind in [
        (lambda: ctx.encode_f8(torch.zeros(4)), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 0)), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8).t()), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8, dtype=torch.float64)), TypeError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8), block_rows=2), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8), out=torch.zeros(4, 8, dtype=torch.uint8)), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8), scales=torch.zeros(4, 2)), ValueError),
        (lambda: ctx.decode_f8(a, sa[:, :1]), ValueError),
        (lambda: ctx.decode_f8(a, sa, out=torch.zeros(4, 300)[:, :256]), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, transposed=True), ValueError),
        (lambda: ctx.matmul_f8(a[:, 8:136], sa[:, :1], w[:, :128], sw[:, :1].contiguous()), ValueError),
        (lambda: ctx.matmul_f8(a, sa.t().contiguous().t(), w, sw), ValueError),
        (lambda: ctx.matmul_f8(a, sa[:1].expand(4, 2), w, sw), ValueError),
        (lambda: ctx.matmul_f8(a[:1].expand(4, 256), sa, w, sw), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, out=torch.zeros(4, 129)), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, out=torch.zeros(4, 128), dtype=torch.float16), ValueError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w[None], sw[None], off.repeat(2)), ValueError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w[None], sw[None], off.short()), TypeError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w, sw, off), ValueError),
    ]:
        with pytest.raises(kind):
            call()
    assert not rec.calls


def test_given_outputs_are_checked_before_a_stream_is_asked_to_keep_them(rec, monkeypatch):
    ctx = CpuContext()
    asked = []
    monkeypatch.setattr(ctx, "_f8_on", lambda *a: asked.append(a), raising=False)
    for kw in ({"out": torch.zeros(4, 8, dtype=torch.uint8)}, {"scales": torch.zeros(4, 2)}):
        with pytest.raises(ValueError):
            ctx.encode_f8(torch.zeros(4, 8), **kw)
    assert not asked and not rec.calls

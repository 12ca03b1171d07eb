"""BF16 rows given as their bits, as encode_rows takes them."""
import pytest

torch = pytest.importorskip("torch")
import shoehorn_b200 as sh  # noqa: E402
from test_f8_host import CpuContext, rec  # noqa: E402,F401

BITS = [torch.int16, torch.uint16]


@pytest.mark.parametrize("dtype", BITS, ids=str)
def test_bits_are_passed_on_as_bf16(rec, dtype):  # noqa: F811
    codes, scales = CpuContext().encode_f8(torch.zeros(3, 200, dtype=torch.bfloat16).view(dtype))
    (name, args), = rec.calls
    assert name == "shc_encode_f8" and args[1] == sh.SRC_BF16 and args[3:9] == (1, 3, 200, 200, 0, 1)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (3, 200) and scales.shape == (3, 2) and scales.dtype == torch.float32


def test_bits_are_no_type_of_results(rec):  # noqa: F811
    ctx = CpuContext()
    a, sa = ctx.encode_f8(torch.zeros(3, 256))
    w, sw = ctx.encode_f8(torch.zeros(128, 256), 128)
    rec.calls.clear()
    for dtype in BITS + [torch.int8]:
        with pytest.raises(TypeError):
            ctx.decode_f8(a, sa, dtype=dtype)
        with pytest.raises(TypeError):
            ctx.matmul_f8(a, sa, w, sw, dtype=dtype)
    with pytest.raises(TypeError):
        ctx.encode_f8(torch.zeros(3, 256, dtype=torch.int32))
    assert not rec.calls


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", BITS, ids=str)
@pytest.mark.parametrize("block_rows", [1, 128])
def test_bits_give_the_codes_of_their_numbers(ctx, block_rows, dtype):
    x = torch.randn(130, 333, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16)
    want, ws = ctx.encode_f8(x, block_rows)
    codes, scales = ctx.encode_f8(x.view(dtype), block_rows, sync=True)
    assert torch.equal(codes.view(torch.uint8), want.view(torch.uint8)) and torch.equal(scales, ws)

"""Products of 8-bit blocks whose two scales multiply to a number outside f32's
normal range while the result lies inside f32's.

Tolerance: as in test_f8.py ((128 * 2^-23 + (blocks + 2) * 2^-24) * S + eps / 2
* |exact|), and half a step of f32's subnormals, 2^-150, for each block's
addition and the final conversion, since those may fall among them."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

BF16, F32 = torch.bfloat16, torch.float32


def codes(g, *shape, of):
    """Codes drawn from the numbers `of`, in rows on 16-byte boundaries."""
    v = torch.tensor(of, device="cuda")[torch.randint(len(of), shape, generator=g, device="cuda")]
    held = torch.zeros(*shape[:-1], -(-shape[-1] // 16) * 16, device="cuda").to(torch.float8_e4m3fn)[..., :shape[-1]]
    held.copy_(v.to(torch.float8_e4m3fn))
    return held


def scales(g, *shape, lo, hi):
    """2^lo to 2^hi, mantissas and all."""
    return torch.exp2(torch.rand(*shape, generator=g, device="cuda", dtype=torch.float64) * (hi - lo) + lo).float()


def numbers(c, s, block_rows):
    s = s.double().repeat_interleave(128, -1)[..., :c.shape[-1]]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, -2)[..., :c.shape[-2], :]
    return c.float().double() * s


def check(got, a, sa, w, sw, transposed):
    x, y = numbers(a, sa, 1), numbers(w, sw, 128)
    y = y if transposed else y.t()
    want, mags, blocks = x @ y, x.abs() @ y.abs(), sa.shape[1]
    tol = (128 * 2.0**-23 + (blocks + 2) * 2.0**-24) * mags + torch.finfo(got.dtype).eps / 2 * want.abs() + (blocks + 1) * 2.0**-150
    if got.dtype == BF16:
        tol = tol + 2.0**-134  # half a step of bf16's subnormals
    assert torch.isfinite(want).all() and want.abs().max() < torch.finfo(BF16).max
    bad = ~((got.double() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first {got[bad][0]} for {want[bad][0]}"


SIZES = [  # rows, outputs, contraction, experts: one for each tile shape
    (3, 700, 2100, 0), (40, 5000, 2500, 0), (300, 2500, 3800, 0), (2000, 2049, 600, 0), (2047, 4100, 4090, 0), (300, 1000, 1100, 4),
]
RANGES = {  # exponents of the rows' scales and of the weight's; the codes; what the product of two scales does
    "subnormal": ((-110, -80), (-45, -38), [-448.0, -17.0, -0.5, 0.0, 1.0, 30.0, 320.0]),
    "zero": ((-126, -116), (-40, -34), [-448.0, -288.0, 0.0, 352.0, 416.0]),
    "gradients": ((-116, -100), (-14, -12), [-448.0, -2.0**-9, 0.0, 2.0**-9, 1.5, 240.0]),
    "infinite": ((97, 109), (19, 31), [0.0] * 30 + [2.0**-9, -(2.0**-9)]),
    "both ends": ((-119, 119), (-2, 2), [0.0] * 60 + [2.0**-9, -(2.0**-9)]),
    "far beyond": ((118, 119), (118, 119), [0.0]),
}


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("name", RANGES)
@pytest.mark.parametrize("rows,out,inner,experts", SIZES)
def test_results_do_not_depend_on_the_product_of_two_scales(ctx, rows, out, inner, experts, name, transposed):
    (alo, ahi), (wlo, whi), of = RANGES[name]
    g = torch.Generator(device="cuda").manual_seed(rows + out)
    n, k = (inner, out) if transposed else (out, inner)
    lead = (experts,) if experts else ()
    a, sa = codes(g, rows, inner, of=of), scales(g, rows, -(-inner // 128), lo=alo, hi=ahi)
    w, sw = codes(g, *lead, n, k, of=of), scales(g, *lead, -(-n // 128), -(-k // 128), lo=wlo, hi=whi)
    sa[rows // 3] = 1.0  # a row whose products stay in range, beside the others
    if name in ("infinite", "both ends"):
        a[rows // 3] = 0
    for dtype in (F32, BF16):
        if experts:
            at = torch.arange(experts + 1, device="cuda") * rows // experts
            got = ctx.matmul_f8_grouped(a, sa, w, sw, at, transposed=transposed, dtype=dtype, sync=True)
            for e in range(experts):
                lo, hi = int(at[e]), int(at[e + 1])
                check(got[lo:hi], a[lo:hi], sa[lo:hi], w[e], sw[e], transposed)
        else:
            got = ctx.matmul_f8(a, sa, w, sw, transposed=transposed, dtype=dtype, sync=True)
            check(got, a, sa, w, sw, transposed)


def test_scales_that_are_no_numbers_stay_so(ctx):
    """A scale that is infinite or NaN, or zero, is multiplied as it stands."""
    g = torch.Generator(device="cuda").manual_seed(5)
    a, w = codes(g, 4, 256, of=[1.0, 2.0]), codes(g, 130, 256, of=[1.0, 3.0])
    sa, sw = torch.ones(4, 2, device="cuda"), torch.ones(2, 2, device="cuda")
    sa[1, 0], sa[2, 1], sa[3] = float("inf"), float("nan"), 0.0
    got = ctx.matmul_f8(a, sa, w, sw, dtype=F32, sync=True)
    assert torch.isfinite(got[0]).all() and (got[1] == float("inf")).all() and torch.isnan(got[2]).all() and (got[3] == 0).all()

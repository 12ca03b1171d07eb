"""Block-scaled 8-bit codes and products on the GPU, against plain 64-bit
implementations of the format's rules.

Tolerances.  A code is e4m3(fl(x * fl(448 / top))): two f32 roundings, then
half an E4M3 step.  A product sums 128 products in f32 (the order is the
tensor core's, so each of at most 128 additions is allowed one f32 step,
2^-23, of the sum of magnitudes S), scales it by the f32 product of two scales
(2^-24) and adds it in a fused multiply-add (2^-24 a block), and is rounded
once to the output type (eps / 2): |D - exact| <= (128 * 2^-23 + (blocks + 2)
* 2^-24) * S + eps / 2 * |exact| (+ half a subnormal step of f16)."""
import math
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import shoehorn_b200 as sh  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TOP, LEAST = 448.0, 448.0 * 2.0**-126
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def up(n, to):
    return -(-n // to)


def blocks_of(x, block_rows):
    """[.., row blocks, block_rows, column blocks, 128] of x, zeros where a block is part empty."""
    *lead, rows, cols = x.shape
    rb, cb = up(rows, block_rows), up(cols, 128)
    p = torch.zeros(*lead, rb * block_rows, cb * 128, dtype=x.dtype, device=x.device)
    p[..., :rows, :cols] = x
    return p.view(*lead, rb, block_rows, cb, 128)


def plain_encode(x, block_rows):
    """(code bytes, scales) by the documented rule, in f32 as it is written."""
    x = x.to(F32)
    rows, cols = x.shape[-2:]
    p = blocks_of(x, block_rows)
    fin = torch.isfinite(p)
    top = torch.where(fin, p.abs(), torch.zeros_like(p)).amax((-3, -1), keepdim=True)
    top = torch.maximum(top, torch.tensor(LEAST, dtype=F32, device=x.device))
    v = (p * (torch.tensor(TOP, dtype=F32, device=x.device) / top)).clamp(-TOP, TOP)
    v = torch.where(fin, v, torch.full_like(v, math.nan))
    codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(fin, codes, torch.full_like(codes, 0x7F))
    codes = codes.reshape(*x.shape[:-2], p.shape[-4] * block_rows, -1)[..., :rows, :cols]
    return codes, (top / torch.tensor(TOP, dtype=F32, device=x.device))[..., 0, :, 0]


def numbers(codes, scales, block_rows):
    """code * scale in 64 bits."""
    s = scales.double().repeat_interleave(128, -1)[..., :codes.shape[-1]]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, -2)[..., :codes.shape[-2], :]
    return codes.float().double() * s


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def within(got, want, mags, blocks):
    """The tolerance of the module's docstring; got and want agree on NaN."""
    fi = torch.finfo(got.dtype)
    tol = (128 * 2.0**-23 + (blocks + 2) * 2.0**-24) * mags + fi.eps / 2 * want.abs() + fi.smallest_normal * fi.eps / 2
    d = got.double()
    assert torch.equal(torch.isnan(d), torch.isnan(want))
    bad = ~((d - want).abs() <= tol) & ~torch.isnan(want)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, " \
                          f"largest excess {float(((d - want).abs() / tol)[bad].max())} x"


def check_product(got, a, sa, w, sw, transposed):
    x, y = numbers(a, sa, 1), numbers(w, sw, 128)
    y = y if transposed else y.t()
    within(got, x @ y, x.abs() @ y.abs(), sa.shape[1])


# ---------------------------------------------------------------- encode, decode

SHAPES = [(1, 1), (1, 128), (2, 16), (3, 129), (5, 7), (130, 127), (128, 256), (257, 1030), (40, 4096)]


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_encode_follows_the_rule(ctx, shape, dtype, block_rows):
    x = (rand(gen(shape[0] * 7 + shape[1]), *shape) * torch.exp(rand(gen(3), shape[1]))).to(dtype)
    codes, scales = ctx.encode_f8(x, block_rows, sync=True)
    want, ws = plain_encode(x, block_rows)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and codes.stride(0) % 16 == 0
    assert torch.equal(codes.view(torch.uint8), want)
    assert torch.equal(scales, ws)
    # 64 bits: half an E4M3 step (2^-4 of the value, 2^-10 among its subnormals) and three f32 roundings
    x64, scale = x.double(), numbers(torch.ones_like(want).to(torch.float8_e4m3fn), scales, block_rows)
    off = (numbers(codes, scales, block_rows) - x64).abs()
    assert (off <= x64.abs() * (2.0**-4 + 3 * 2.0**-24) + scale * 2.0**-10).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_encode_unusual_values(ctx, block_rows):
    """Zeros, subnormals, the largest numbers, ties, NaN and infinities."""
    x = torch.zeros(9, 384, device="cuda")
    g = gen(5)
    x[0, 128:256] = rand(g, 128) * 1e-41
    x[1] = rand(g, 384) * 1e38
    x[1, 5] = torch.finfo(F32).max
    x[2] = rand(g, 384)
    x[2, 3], x[2, 200], x[2, 201] = math.nan, math.inf, -math.inf
    x[3, :128] = math.inf
    x[4, :128] = math.nan
    x[5] = torch.arange(384, device="cuda") / 16  # many values half way between two codes
    x[6, 7] = -1e-30
    x[7] = -0.0
    x[8, 383] = 2.0**-126
    codes, scales = ctx.encode_f8(x, block_rows, sync=True)
    want, ws = plain_encode(x, block_rows)
    assert torch.equal(codes.view(torch.uint8), want)
    assert torch.equal(scales, ws)
    assert torch.isfinite(scales).all() and (scales > 0).all()


@pytest.mark.parametrize("block_rows", [1, 128])
def test_encode_strided_sources_and_given_outputs(ctx, block_rows):
    g = gen(11)
    big = rand(g, 3, 150, 700).to(BF16)
    for x in (big[1:, 3:140, 5:600], big[:, ::2, 8:330], big[0].expand(2, -1, -1), big[:, 1:2], big[1, :, 16:17]):
        codes, scales = ctx.encode_f8(x, block_rows, sync=True)
        want, ws = plain_encode(x, block_rows)
        assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, ws)
    # a view of a larger buffer: nothing beside the codes is written
    buf = torch.full((2, 160, 640), 0xA5, dtype=torch.uint8, device="cuda")
    x = big[:2, :130, :333]
    out = buf[:, 16:146, 32:365]
    scales = torch.empty(2, up(130, block_rows), 3, device="cuda")
    ctx.encode_f8(x, block_rows, out=out, scales=scales, sync=True)
    want, ws = plain_encode(x, block_rows)
    assert torch.equal(out, want) and torch.equal(scales, ws)
    out.fill_(0xA5)
    assert (buf == 0xA5).all()


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 129), (2, 130, 120), (257, 1030), (64, 512)], ids=str)
def test_decode_is_code_times_scale(ctx, shape, dtype, block_rows):
    codes, scales = ctx.encode_f8(rand(gen(2), *shape) * 0.1, block_rows)
    got = ctx.decode_f8(codes, scales, block_rows, dtype=dtype, sync=True)
    # one f32 rounding and the output's: the f32 product, rounded
    s = scales.repeat_interleave(128, -1)[..., :shape[-1]]
    if block_rows > 1:
        s = s.repeat_interleave(128, -2)[..., :shape[-2], :]
    assert got.is_contiguous() and torch.equal(got, (codes.float() * s).to(dtype))


@pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=str)
@pytest.mark.parametrize("cols", [1, 3, 9, 127, 129, 1023, 1030, 2051])
def test_decode_and_encode_at_every_alignment(ctx, dtype, cols):
    """Outputs and sources that start at any element: no row on a 16-byte boundary but by chance."""
    g = gen(cols)
    codes, scales = ctx.encode_f8(rand(g, 5, cols))
    s = scales.repeat_interleave(128, -1)[:, :cols]
    for left in range(9):
        buf = torch.full((5 * cols + 32,), 3.0, dtype=dtype, device="cuda")
        out = buf[left:left + 5 * cols].view(5, cols)
        ctx.decode_f8(codes, scales, dtype=dtype, out=out, sync=True)
        assert torch.equal(out, (codes.float() * s).to(dtype))
        x = out.clone()
        out.copy_(rand(g, 5, cols))
        for block_rows in (1, 128):
            want, ws = plain_encode(out, block_rows)
            got, gs = ctx.encode_f8(out, block_rows, sync=True)
            assert torch.equal(got.view(torch.uint8), want) and torch.equal(gs, ws)
        out.fill_(3.0)
        assert (buf == 3.0).all() and x.shape == out.shape


def test_decode_every_code(ctx):
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").view(2, 128)
    got = ctx.decode_f8(codes, torch.ones(2, 1, device="cuda"), sync=True)
    want = codes.view(torch.float8_e4m3fn).float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(7e9), want.nan_to_num(7e9))


# ---------------------------------------------------------------- products

def encoded(ctx, g, rows, cols, block_rows, size=1.0):
    return ctx.encode_f8(rand(g, rows, cols) * size * torch.exp(0.5 * rand(g, cols)), block_rows)


PRODUCTS = [  # rows, n, k
    (1, 1, 1), (1, 128, 128), (2, 16, 16), (1, 4096, 4096), (3, 127, 129), (5, 130, 1), (7, 1, 300), (31, 1000, 127),
    (33, 256, 640), (64, 2048, 1024), (127, 129, 1030), (128, 128, 256), (129, 384, 2048), (256, 512, 512),
    (300, 1000, 385), (513, 777, 1290), (1500, 2049, 1024), (2048, 4096, 512),
]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_product(ctx, m, n, k, transposed):
    g = gen(m + n + k)
    a, sa = encoded(ctx, g, m, n if transposed else k, 1)
    w, sw = encoded(ctx, g, n, k, 128, 0.02)
    for dtype in (F32, BF16, F16):
        got = ctx.matmul_f8(a, sa, w, sw, transposed=transposed, dtype=dtype, sync=True)
        assert got.dtype == dtype and got.shape == (m, k if transposed else n)
        check_product(got, a, sa, w, sw, transposed)


SHAPES_OF_TILES = [  # rows, outputs, contraction, experts: sizes that the kernel's tile shapes are chosen for
    (1, 1030, 1100, 0), (3, 700, 2100, 0), (130, 1000, 4200, 0),  # contraction shared by four and eight CTAs
    (40, 5000, 2500, 0), (1, 9000, 5100, 0),  # by two
    (300, 2500, 3800, 0), (2000, 2049, 600, 0), (2047, 4100, 4090, 0),  # 128 x 128, 128 x 256, pairs
    (300, 200, 2500, 3), (20, 300, 4200, 2), (5000, 1000, 1100, 8), (2000, 1000, 1100, 8), (9000, 4100, 4090, 4),
]


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,out,inner,experts", SHAPES_OF_TILES)
def test_every_tile_shape(ctx, rows, out, inner, experts, transposed):
    g = gen(rows + out)
    n, k = (inner, out) if transposed else (out, inner)
    a, sa = encoded(ctx, g, rows, inner, 1)
    for dtype, pad in ((F32, 0), (BF16, 3), (F16, 16)):
        buf = torch.full((rows, out + pad), 3.0, dtype=dtype, device="cuda")
        got = buf[:, :out]
        if experts:
            w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
            at = torch.sort(torch.randint(rows + 1, (experts + 1,), generator=g, device="cuda"))[0]
            before = got.clone()
            ctx.matmul_f8_grouped(a, sa, w, sw, at, transposed=transposed, out=got, sync=True)
            check_grouped(got, before, a, sa, w, sw, at, transposed)
        else:
            w, sw = encoded(ctx, g, n, k, 128, 0.05)
            ctx.matmul_f8(a, sa, w, sw, transposed=transposed, out=got, sync=True)
            check_product(got, a, sa, w, sw, transposed)
        assert (buf[:, out:] == 3.0).all()


def test_no_rows(ctx):
    w, sw = encoded(ctx, gen(1), 64, 96, 128)
    a = torch.empty(0, 96, dtype=torch.float8_e4m3fn, device="cuda")
    assert ctx.matmul_f8(a, torch.empty(0, 1, device="cuda"), w, sw, sync=True).shape == (0, 64)
    codes, scales = ctx.encode_f8(torch.empty(0, 96, device="cuda"), sync=True)
    assert codes.shape == (0, 96) and scales.shape == (0, 1)
    assert ctx.decode_f8(codes, scales, sync=True).shape == (0, 96)
    w3, sw3 = w[None], sw[None]
    off = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert ctx.matmul_f8_grouped(a, torch.empty(0, 1, device="cuda"), w3, sw3, off, sync=True).shape == (0, 64)


@pytest.mark.parametrize("transposed", [False, True])
def test_product_of_views_into_larger_buffers(ctx, transposed):
    """Rows of codes, of scales and of the result that are slices; nothing
    beside the result is written."""
    g = gen(21)
    a, sa = encoded(ctx, g, 200, 1152, 1)
    w, sw = encoded(ctx, g, 640, 1152, 128, 0.02)
    if transposed:
        a, sa = encoded(ctx, g, 200, 1152, 1)
        w, sw = encoded(ctx, g, 640, 1000, 128, 0.02)
        a1, s1, w1, s1w = a[7:190, 256:896], sa[7:190, 2:7], w, sw
    else:
        a1, s1, w1, s1w = a[7:190, 256:768], sa[7:190, 2:6], w[128:513, 384:896], sw[1:5, 3:7].contiguous()
    cols = w1.shape[1] if transposed else w1.shape[0]
    for dtype, left in ((BF16, 3), (F32, 8), (F16, 16)):
        buf = torch.full((200, cols + 50), 7.0, dtype=dtype, device="cuda")
        out = buf[9:192, left:left + cols]
        assert ctx.matmul_f8(a1, s1, w1, s1w, transposed=transposed, out=out, sync=True) is out
        check_product(out, a1, s1, w1, s1w, transposed)
        out.fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("transposed", [False, True])
def test_nan_codes_stay_in_their_row_and_column(ctx, transposed):
    g = gen(31)
    a, sa = encoded(ctx, g, 70, 256, 1)
    w, sw = encoded(ctx, g, 256, 256, 128)
    a.view(torch.uint8)[13, 200] = 0x7F
    w.view(torch.uint8)[(77, 5) if not transposed else (5, 77)] = 0xFF
    got = ctx.matmul_f8(a, sa, w, sw, transposed=transposed, dtype=F32, sync=True)
    nan = torch.isnan(got)
    assert nan[13].all() and nan[:, 77].all() and int(nan.sum()) == 70 + 256 - 1
    check_product(got, a, sa, w, sw, transposed)


def test_scales_of_every_size(ctx):
    """Blocks whose scales differ by many orders; zeros times anything is zero."""
    g = gen(41)
    x = rand(g, 40, 512) * torch.exp2(torch.randint(-60, 60, (40, 512), generator=g, device="cuda").float())
    x[3] = 0
    y = rand(g, 200, 512) * torch.exp2(torch.randint(-8, 8, (200, 512), generator=g, device="cuda").float())
    a, sa = ctx.encode_f8(x, 1)
    w, sw = ctx.encode_f8(y, 128)
    got = ctx.matmul_f8(a, sa, w, sw, dtype=F32, sync=True)
    check_product(got, a, sa, w, sw, False)
    assert (got[3] == 0).all()


def whole(g, rows, cols, block_rows):
    """Codes that are small whole numbers, with scales of one: sums are exact in f32."""
    v = torch.randint(-4, 5, (rows, cols), generator=g, device="cuda").float()
    pitch = up(cols, 16) * 16
    codes = torch.zeros(rows, pitch, device="cuda").to(torch.float8_e4m3fn)[:, :cols]
    codes.copy_(v.to(torch.float8_e4m3fn))
    return codes, torch.ones(up(rows, block_rows), up(cols, 128), device="cuda")


@pytest.mark.parametrize("m,n,k", [(3, 200, 150), (140, 260, 129)])
def test_gradient_of_the_rows(ctx, m, n, k):
    """L = <G, A W^T>: dL/dA is G W by the formula, and by differences of L
    (whole numbers, so both are exact)."""
    g = gen(m)
    a, one_a = whole(g, m, k, 1)
    w, one_w = whole(g, n, k, 128)
    G, one_g = whole(g, m, n, 1)
    grad = ctx.matmul_f8(G, one_g, w, one_w, transposed=True, dtype=F32, sync=True)
    assert torch.equal(grad.double(), G.double() @ w.double())
    for i, j in ((0, 0), (m - 1, k - 1), (m // 2, k // 3)):
        L = []
        for h in (1, -1):
            moved = a.clone()
            moved[i, j] = (a[i, j].float() + h).to(torch.float8_e4m3fn)
            held = torch.zeros(m, up(k, 16) * 16, device="cuda").to(torch.float8_e4m3fn)[:, :k]
            held.copy_(moved)
            d = ctx.matmul_f8(held, one_a, w, one_w, dtype=F32, sync=True)
            L.append(float((G.double() * d.double()).sum()))
        assert float(grad[i, j]) == (L[0] - L[1]) / 2


# ---------------------------------------------------------------- grouped by expert

def check_grouped(got, before, a, sa, w, sw, offsets, transposed):
    """Each expert's rows against 64 bits; rows of no expert as they were."""
    rows = a.shape[0]
    at = [min(max(int(v), 0), rows) for v in offsets.tolist()]
    mine = torch.zeros(rows, dtype=torch.bool, device="cuda")
    for e in range(w.shape[0]):
        lo, hi = at[e], at[e + 1]
        if hi > lo:
            check_product(got[lo:hi], a[lo:hi], sa[lo:hi], w[e], sw[e], transposed)
            mine[lo:hi] = True
    assert torch.equal(got[~mine], before[~mine])


OFFSETS = {
    "one": [0, 300],
    "empty_first": [0, 0, 300],
    "uneven": [0, 1, 1, 129, 130, 257, 257, 300, 300],
    "ends_early": [5, 40, 40, 200],
    "all_in_the_last": [0, 0, 0, 0, 300],
    "none": [7, 7, 7],
    "out_of_range": [-50, 10, 100, 10**6],
    "decreasing": [0, 100, 40, 40],
}


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("name", OFFSETS)
def test_grouped(ctx, name, transposed):
    at = OFFSETS[name]
    g = gen(len(name))
    rows, n, k, experts = 300, 200, 330, len(at) - 1
    a, sa = encoded(ctx, g, rows, n if transposed else k, 1)
    w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
    for dtype, ot in ((F32, torch.int32), (BF16, torch.int64), (F16, torch.int32)):
        offsets = torch.tensor(at, dtype=ot, device="cuda")
        before = torch.full((rows, k if transposed else n), 3.0, dtype=dtype, device="cuda")
        out = before.clone()
        ctx.matmul_f8_grouped(a, sa, w, sw, offsets, transposed=transposed, out=out, sync=True)
        check_grouped(out, before, a, sa, w, sw, offsets, transposed)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("experts,rows,n,k", [(64, 96, 256, 128), (70, 500, 130, 257), (33, 33, 64, 64), (3, 2000, 384, 512),
                                              (200, 64, 128, 384), (8, 1100, 1000, 520)])
def test_grouped_many_experts(ctx, experts, rows, n, k, transposed):
    g = gen(experts)
    a, sa = encoded(ctx, g, rows, n if transposed else k, 1)
    w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
    counts = torch.bincount(torch.randint(experts, (rows,), generator=g, device="cuda") ** 2 // experts, minlength=experts)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    got = ctx.matmul_f8_grouped(a, sa, w, sw, offsets, transposed=transposed, dtype=F32, sync=True)
    check_grouped(got, got, a, sa, w, sw, offsets, transposed)


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("rows,n,k,experts,at", [
    (100, 1000, 2500, 8, [0, 60, 10, 70, 10, 80, 10, 90, 10]),  # contraction shared by a cluster,
    (100, 2500, 1000, 8, [0, 60, 10, 70, 10, 80, 10, 90, 10]),  # transposed too
    (300, 256, 200, 5, [0, 200, 50, 250, 0, 300]),
    (500, 130, 257, 70, None),  # more experts than are looked up at once
    (3000, 1024, 1100, 6, [0, 2000, 100, 2500, 100, 2700, 3000]),
])
def test_grouped_offsets_that_fall_and_rise(ctx, rows, n, k, experts, at, transposed):
    """An offset below an earlier one is read as the largest before it: no row has two experts."""
    g = gen(rows + experts)
    a, sa = encoded(ctx, g, rows, n if transposed else k, 1)
    w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
    if at is None:
        offsets = torch.randint(rows + 1, (experts + 1,), generator=g, device="cuda") * torch.arange(experts + 1, device="cuda") // experts
    else:
        offsets = torch.tensor(at, dtype=torch.int32, device="cuda")
    before = torch.full((rows, k if transposed else n), 3.0, device="cuda")
    out = before.clone()
    ctx.matmul_f8_grouped(a, sa, w, sw, offsets, transposed=transposed, out=out, sync=True)
    check_grouped(out, before, a, sa, w, sw, torch.cummax(offsets, 0)[0], transposed)


@pytest.mark.parametrize("transposed", [False, True])
def test_grouped_weights_a_part_row_apart(ctx, transposed):
    """Matrices whose distance is neither a multiple of the row pitch nor whole rows."""
    g = gen(9)
    experts, n, k, rows, pitch = 3, 30, 100, 90, 256
    step = (n - 1) * pitch + 112
    a, sa = encoded(ctx, g, rows, n if transposed else k, 1)
    w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
    apart = torch.zeros(experts * step + pitch, dtype=torch.uint8, device="cuda").as_strided((experts, n, k), (step, pitch, 1))
    apart.copy_(w.view(torch.uint8))
    offsets = torch.tensor([0, 20, 60, 90], device="cuda")
    got = ctx.matmul_f8_grouped(a, sa, apart, sw, offsets, transposed=transposed, dtype=F32, sync=True)
    check_grouped(got, got, a, sa, w, sw, offsets, transposed)


def test_grouped_weights_apart(ctx):
    """Experts' weights some distance from one another, and only some of them."""
    g = gen(9)
    w, sw = ctx.encode_f8(rand(g, 6, 140, 300) * 0.05, 128)
    a, sa = encoded(ctx, g, 90, 300, 1)
    offsets = torch.tensor([0, 20, 90], dtype=torch.int32, device="cuda")
    w2, s2 = w[1::4, :130], sw[1::4].contiguous()
    got = ctx.matmul_f8_grouped(a, sa, w2, s2, offsets, dtype=F32, sync=True)
    check_grouped(got, got, a, sa, w2, s2, offsets, False)


# ---------------------------------------------------------------- as programs use them

def test_same_calls_give_the_same_bits(ctx):
    g = gen(17)
    for m, n, k in ((1, 2048, 4096), (40, 512, 2048), (700, 1000, 1030)):
        a, sa = encoded(ctx, g, m, k, 1)
        w, sw = encoded(ctx, g, n, k, 128)
        first = ctx.matmul_f8(a, sa, w, sw, dtype=F32, sync=True)
        for _ in range(3):
            assert torch.equal(ctx.matmul_f8(a, sa, w, sw, dtype=F32, sync=True), first)


def test_rows_do_not_depend_on_their_neighbours(ctx):
    """A row's result is its own, whatever else is in its tile."""
    g = gen(19)
    a, sa = encoded(ctx, g, 128, 512, 1)
    w, sw = encoded(ctx, g, 256, 512, 128)
    allof = ctx.matmul_f8(a, sa, w, sw, dtype=F32, sync=True)
    garbage = a.clone()
    garbage.view(torch.uint8)[1:] = 0x7F
    got = ctx.matmul_f8(garbage, sa, w, sw, dtype=F32, sync=True)
    assert torch.equal(got[0], allof[0])


def test_another_stream_and_two_at_once(ctx):
    g = gen(23)
    sets = []
    for i in range(2):
        a, sa = encoded(ctx, g, 300 + i, 1024, 1)
        w, sw = encoded(ctx, g, 512, 1024, 128)
        sets.append((a, sa, w, sw))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            got[i].append(ctx.matmul_f8(*sets[i], dtype=F32, stream=streams[i]))
    x = rand(g, 64, 300)
    torch.cuda.synchronize()
    codes, scales = ctx.encode_f8(x, stream=streams[0])
    back = ctx.decode_f8(codes, scales, stream=streams[0])
    for s in streams:
        ctx.sync(s)
    for i in range(2):
        for d in got[i]:
            assert torch.equal(d, got[i][0])
        check_product(got[i][0], *sets[i], False)
    assert torch.equal(back.double(), numbers(codes, scales, 1).float().double())


def test_captured_and_replayed(ctx):
    """Encode and grouped product in a graph: replays follow new inputs and
    new offsets, and two graphs replayed at once do not meet."""
    g = gen(29)
    experts, rows, n, k = 4, 200, 384, 512
    w, sw = ctx.encode_f8(rand(g, experts, n, k) * 0.05, 128)
    graphs = []
    for i in range(2):
        x = rand(g, rows, k).to(BF16)
        offsets = torch.tensor([0, 50, 50, 120, rows], dtype=torch.int32, device="cuda")
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            a, sa = ctx.encode_f8(x)
            ctx.matmul_f8_grouped(a, sa, w, sw, offsets, dtype=F32)
            ctx.matmul_f8(a[:1], sa[:1], w[0], sw[0], dtype=F32)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            a, sa = ctx.encode_f8(x)
            d = ctx.matmul_f8_grouped(a, sa, w, sw, offsets, dtype=F32)
            one = ctx.matmul_f8(a[:1], sa[:1], w[0], sw[0], dtype=F32)
        graphs.append((graph, x, offsets, a, sa, d, one))
    for turn in range(3):
        at = [[0, 50, 50, 120, rows], [0, 0, 1, 2, rows], [0, 200, 200, 200, rows]][turn]
        torch.cuda.synchronize()
        for graph, x, offsets, *_ in graphs:
            x.copy_(rand(g, rows, k))
            offsets.copy_(torch.tensor(at))
        torch.cuda.synchronize()
        for (graph, *_), s in zip(graphs, (torch.cuda.Stream(), torch.cuda.Stream())):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for graph, x, offsets, a, sa, d, one in graphs:
            want, ws = plain_encode(x, 1)
            assert torch.equal(a.view(torch.uint8), want) and torch.equal(sa, ws)
            check_grouped(d, d, a, sa, w, sw, offsets, False)
            check_product(one, a[:1], sa[:1], w[0], sw[0], False)


def test_the_first_call_of_a_process_may_be_captured():
    """Nothing that a first call sets up keeps it out of a graph."""
    code = """
import torch, shoehorn_b200 as sh
ctx = sh.Context(0)
x = torch.randn(200, 384, device="cuda")
w = torch.randn(256, 384, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    a, sa = ctx.encode_f8(x)
    b, sb = ctx.encode_f8(w, 128)
    d = ctx.matmul_f8(a, sa, b, sb, dtype=torch.float32)
    e = ctx.matmul_f8(a[:1], sa[:1], b, sb, dtype=torch.float32)
graph.replay()
torch.cuda.synchronize()
ctx.sync()
want = ctx.decode_f8(a, sa).double() @ ctx.decode_f8(b, sb, 128).double().t()
assert (d - want).abs().max() < 1e-4 * want.abs().max(), (d - want).abs().max()
assert torch.equal(d[:1], e) or (d[:1] - e).abs().max() < 1e-4 * want.abs().max()
print("captured")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "captured" in r.stdout, r.stdout + r.stderr


def test_experts_from_quantised_tensors(ctx):
    """The framework's own blocks (Q6_K, Q8_0 experts) unpacked, encoded to
    8-bit blocks and run as an expert feed-forward, forward and back to the
    gradient of its input, each stage against 64 bits of what went into it."""
    g = gen(37)
    experts, rows, hidden, ffn = 5, 150, 512, 768
    counts = torch.tensor([40, 0, 1, 90, 19], device="cuda")
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])

    def weights(ty, n, k):
        src = (rand(g, experts * n, k) * 0.02).to(BF16)
        back = ctx.decode_rows(ty, ctx.encode_rows(ty, src), k).view(experts, n, k)
        codes, scales = ctx.encode_f8(back, 128)
        want, ws = plain_encode(back, 128)
        assert torch.equal(codes.view(torch.uint8), want) and torch.equal(scales, ws)
        return codes, scales

    up_w, up_s = weights(sh.GgmlType.Q6_K, ffn, hidden)
    down_w, down_s = weights(sh.GgmlType.Q8_0, hidden, ffn)
    x, sx = ctx.encode_f8(rand(g, rows, hidden).to(BF16))
    h = ctx.matmul_f8_grouped(x, sx, up_w, up_s, offsets)
    check_grouped(h, h, x, sx, up_w, up_s, offsets, False)
    q, sq = ctx.encode_f8(torch.nn.functional.silu(h))
    y = ctx.matmul_f8_grouped(q, sq, down_w, down_s, offsets)
    check_grouped(y, y, q, sq, down_w, down_s, offsets, False)
    gy, sgy = ctx.encode_f8(rand(g, rows, hidden))
    gq = ctx.matmul_f8_grouped(gy, sgy, down_w, down_s, offsets, transposed=True)
    check_grouped(gq, gq, gy, sgy, down_w, down_s, offsets, True)
    gh = gq.float() * torch.autograd.functional.vjp(torch.nn.functional.silu, h.float(), torch.ones_like(h.float()))[1]
    e, se = ctx.encode_f8(gh)
    gx = ctx.matmul_f8_grouped(e, se, up_w, up_s, offsets, transposed=True)
    check_grouped(gx, gx, e, se, up_w, up_s, offsets, True)
    ctx.sync()


# ---------------------------------------------------------------- refusals

def test_refusals_before_any_launch(ctx):
    g = gen(1)
    a, sa = encoded(ctx, g, 4, 256, 1)
    w, sw = encoded(ctx, g, 128, 256, 128)
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    launches = ctx.launch_count()
    for call, kind in [
        (lambda: ctx.encode_f8(torch.zeros(4, 128)), ValueError),
        (lambda: ctx.encode_f8(a.view(torch.uint8)), TypeError),
        (lambda: ctx.encode_f8(torch.zeros(4, device="cuda")), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 0, device="cuda")), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8, device="cuda").t()), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8, device="cuda"), block_rows=64), ValueError),
        (lambda: ctx.encode_f8(torch.zeros(4, 8, device="cuda"), out=torch.zeros(4, 8, dtype=torch.uint8, device="cuda")), ValueError),
        (lambda: ctx.decode_f8(a, sw), ValueError),
        (lambda: ctx.decode_f8(a, sa, dtype=torch.float64), TypeError),
        (lambda: ctx.decode_f8(a, sa.double()), TypeError),
        (lambda: ctx.matmul_f8(a[:, 1:129], sa[:, :1], w[:, :128], sw[:, :1].contiguous()), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w[:, :128], sw[:, :1].contiguous()), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, transposed=True), ValueError),
        (lambda: ctx.matmul_f8(a, sa[:3], w, sw), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w.cpu(), sw), ValueError),
        (lambda: ctx.matmul_f8(a.to(torch.float8_e5m2), sa, w, sw), TypeError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, dtype=torch.int8), TypeError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, out=torch.zeros(4, 127, device="cuda")), ValueError),
        (lambda: ctx.matmul_f8(a, sa, w, sw, out=torch.zeros(1, 128, device="cuda").expand(4, 128)), ValueError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w, sw, off), ValueError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w[None], sw[None], off[:1]), ValueError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w[None], sw[None], off.float()), TypeError),
        (lambda: ctx.matmul_f8_grouped(a, sa, w[None], sw[None], off.cpu()), ValueError),
    ]:
        with pytest.raises(kind):
            call()
    assert ctx.launch_count() == launches


def test_the_c_entry_points_refuse_what_the_kernels_cannot_take(ctx):
    L, h = sh.lib(), ctx.handle
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = buf.data_ptr()
    good = dict(a=p, lda=128, sa=p, ssa=1, rows=2, w=p, ldw=128, sw=p, n=4, k=128, t=0, dt=30, d=p, ldd=4)

    def mm(**over):
        v = {**good, **over}
        return L.shc_matmul_f8(h, v["a"], v["lda"], v["sa"], v["ssa"], v["rows"], v["w"], v["ldw"], v["sw"], v["n"], v["k"],
                               v["t"], v["dt"], v["d"], v["ldd"], None)

    launches = ctx.launch_count()
    for over in (dict(a=None), dict(a=p + 1), dict(a=p + 8), dict(lda=120), dict(lda=64), dict(ssa=0), dict(rows=-1), dict(rows=1 << 31),
                 dict(w=None), dict(w=p + 4), dict(ldw=100), dict(sw=None), dict(sw=p + 2), dict(n=0), dict(k=0), dict(dt=8),
                 dict(d=None), dict(d=p + 1), dict(ldd=3), dict(lda=1 << 40), dict(sa=p + 1)):
        assert mm(**over) == -1, over
    assert mm(rows=0) == 0
    f = L.shc_matmul_f8_grouped
    assert f(h, p, 128, p, 1, 2, p, 128, 512, p, 2, 4, 128, None, 0, 0, 30, p, 4, None) == -1  # no offsets
    assert f(h, p, 128, p, 1, 2, p, 128, 500, p, 2, 4, 128, p, 0, 0, 30, p, 4, None) == -1  # experts off 16 bytes
    assert f(h, p, 128, p, 1, 2, p, 128, 256, p, 2, 4, 128, p, 0, 0, 30, p, 4, None) == -1  # experts overlap
    assert f(h, p, 128, p, 1, 2, p, 128, 512, p, 2, 4, 128, p + 4, 1, 0, 30, p, 4, None) == -1  # int64 off 8 bytes
    assert f(h, p, 128, p, 1, 2, p, 128, 512, p, -1, 4, 128, p, 0, 0, 30, p, 4, None) == -1
    assert f(h, p, 128, p, 1, 2, p, 128, 512, p, 0, 4, 128, p, 0, 0, 30, p, 4, None) == 0  # no experts
    e = L.shc_encode_f8
    assert e(h, 30, p, 1, 2, 128, 128, 0, 2, p, 128, 0, p, None) == -1
    assert e(h, 30, p + 1, 1, 2, 128, 128, 0, 1, p, 128, 0, p, None) == -1
    assert e(h, 7, p, 1, 2, 128, 128, 0, 1, p, 128, 0, p, None) == -1
    assert e(h, 30, p, 1, 2, 0, 128, 0, 1, p, 128, 0, p, None) == -1
    assert e(h, 30, p, 1, 2, 128, -1, 0, 1, p, 128, 0, p, None) == -1
    assert e(h, 30, p, 2, 2, 128, 128, 256, 1, p, 128, 128, p, None) == -1  # matrices of codes overlap
    assert e(h, 30, None, 1, 2, 128, 128, 0, 1, p, 128, 0, p, None) == -1
    d = L.shc_decode_f8
    assert d(h, 30, p, 1, 2, 128, 128, 0, 3, p, p, None) == -1
    assert d(h, 0, p, 1, 2, 128, 128, 0, 1, p, p + 2, None) == -1
    assert d(h, 0, p + 3, 1, 2, 128, 128, 0, 1, p, p, None) == -1
    assert ctx.launch_count() == launches

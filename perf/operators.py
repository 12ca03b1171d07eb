"""The block-scaled 8-bit operators, as they are measured: real work over the
range of sizes they serve, in plain torch operations and through the
framework's own calls.

  encode    rows to E4M3 codes with one scale for each block of 128 columns
            (activations) or of 128 x 128 elements (weights)
  decode    codes and scales back to numbers
  matmul    D = A W^T of encoded rows and an encoded weight, or with
            `transposed` D = A W, the gradient that passes back through W
  grouped   the same where the rows, sorted by expert, each meet their own
            expert's weight; experts have ragged numbers of rows, some none

A scale is the block's largest magnitude / 448 and a code is the value's
multiple of that scale rounded to E4M3, so a code times its scale is the value
that is held.  Codes lie in rows whose pitch is a multiple of 16 bytes.
"""
import math

import torch

own = False

BLOCK = 128
TOP = 448.0            # largest E4M3 magnitude
LEAST = TOP * 2.0**-126  # keeps a scale and its inverse normal f32 numbers
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token's hidden state on its way into a projection: latency
        {"name": "encode_token", "op": "encode", "rows": 1, "cols": 4096, "block_rows": 1, "src": "bf16"},
        # a long prompt's activations behind the feed-forward's up projection
        {"name": "encode_prompt", "op": "encode", "rows": 8192, "cols": 14336, "block_rows": 1, "src": "bf16"},
        # a weight of no round size, as decoded from a quantised file
        {"name": "encode_weight_odd", "op": "encode", "rows": 1000, "cols": 1031, "block_rows": 128, "src": "f32"},
        # a feed-forward weight unpacked for a consumer that takes bf16
        {"name": "decode_weight", "op": "decode", "rows": 14336, "cols": 4096, "block_rows": 128, "out": "bf16"},
        # a few rows of activations of odd width read back for their error
        {"name": "decode_rows_odd", "op": "decode", "rows": 515, "cols": 1030, "block_rows": 1, "out": "f32"},
        # generating: one token through a square projection
        {"name": "matmul_token", "op": "matmul", "m": 1, "n": 4096, "k": 4096, "transposed": False, "out": "bf16"},
        # a prompt through the feed-forward's up projection
        {"name": "matmul_prompt", "op": "matmul", "m": 4096, "n": 14336, "k": 4096, "transposed": False, "out": "bf16"},
        # ragged in every dimension, kept in f32
        {"name": "matmul_odd", "op": "matmul", "m": 1037, "n": 2008, "k": 1030, "transposed": False, "out": "f32"},
        # the gradient of a projection's input, passed back through the frozen weight
        {"name": "matmul_gradient", "op": "matmul", "m": 2048, "n": 8192, "k": 4096, "transposed": True, "out": "bf16"},
        # a dozen tokens generating, eight of 64 experts each: most experts have one row or two
        {"name": "experts_generate", "op": "grouped", "experts": 64, "m": 96, "n": 2048, "k": 1024, "transposed": False, "out": "bf16"},
        # a prompt's rows over eight large experts, unevenly, one without any
        {"name": "experts_prompt", "op": "grouped", "experts": 8, "m": 4096, "n": 14336, "k": 4096, "transposed": False, "out": "bf16"},
        # gradients of the inputs of sixteen experts of odd size
        {"name": "experts_gradient_odd", "op": "grouped", "experts": 16, "m": 3001, "n": 1000, "k": 2050, "transposed": True, "out": "f32"},
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _width(rng, lo, hi):
    """A row length: half of them multiples of 128, the others anything."""
    v = _spread(rng, lo, hi)
    return max(lo, v // BLOCK * BLOCK) if v >= BLOCK and rng.random() < 0.5 else v


def draw(rng):
    op = rng.choice(["encode", "decode", "matmul", "grouped"])
    if op in ("encode", "decode"):
        c = {"op": op, "rows": _spread(rng, 1, 8192), "cols": _width(rng, 16, 14336), "block_rows": rng.choice([1, 128])}
        c["src" if op == "encode" else "out"] = rng.choice(["bf16", "f16", "f32"])
        if op == "decode":
            c["rows"] = min(c["rows"], 14336 * 4096 // c["cols"])
        return c
    c = {"op": op, "m": _spread(rng, 1, 4096), "n": _width(rng, 64, 14336), "k": _width(rng, 64, 8192),
         "transposed": rng.random() < 0.4, "out": rng.choice(["bf16", "f16", "f32"])}
    if op == "grouped":
        c["experts"] = _spread(rng, 2, 64)
        room = 8 * 14336 * 4096 // (c["experts"] * c["k"])  # no more weight than the largest listed case
        c["n"] = max(1, min(c["n"], room))
    c["m"] = max(1, min(c["m"], 4096 * 14336 * 4096 // (c["n"] * c["k"])))
    return c


# ---------------------------------------------------------------- inputs

def _up(n, to):
    return -(-n // to) * to


def _pitched(codes):
    """The same codes in rows whose pitch is a multiple of 16 bytes."""
    *lead, cols = codes.shape
    held = torch.zeros(*lead, _up(cols, 16), dtype=torch.uint8, device=codes.device)
    held[..., :cols] = codes.view(torch.uint8)
    return held.view(torch.float8_e4m3fn)[..., :cols]


def _activations(g, rows, cols):
    """Rows of unit size whose channels differ, as hidden states do."""
    by_channel = torch.exp(torch.randn(cols, generator=g, device="cuda") * 0.5)
    return torch.randn(rows, cols, generator=g, device="cuda") * by_channel


def _weights(g, rows, cols):
    """N(0, 0.02) with one element in a thousand at +-8 sigma."""
    w = torch.randn(rows, cols, generator=g, device="cuda") * 0.02
    far = torch.rand(rows, cols, generator=g, device="cuda") < 0.001
    return torch.where(far, torch.sign(w) * 0.16, w)


def _rows_of_experts(g, experts, rows):
    """Where each expert's rows start: uneven shares, and one expert without any."""
    share = torch.exp(torch.randn(experts, generator=g, device="cuda"))
    if experts > 2:
        share[int(torch.randint(experts, (1,), generator=g, device="cuda"))] = 0.0
    chosen = torch.multinomial(share, rows, replacement=True, generator=g)
    counts = torch.bincount(chosen, minlength=experts)
    return torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32), int(counts.max())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    if op in ("encode", "decode"):
        make = _activations if case["block_rows"] == 1 else _weights
        x = make(g, case["rows"], case["cols"])
        if op == "encode":
            return {**case, "x": x.to(DTYPES[case["src"]])}
        codes, scales = _encode(x, case["block_rows"])
        return {**case, "codes": _pitched(codes), "scales": scales}
    m, n, k = case["m"], case["n"], case["k"]
    a, a_scales = _encode(_activations(g, m, n if case["transposed"] else k), 1)
    state = {**case, "a": _pitched(a), "a_scales": a_scales}
    if op == "matmul":
        w, w_scales = _encode(_weights(g, n, k), BLOCK)
        return {**state, "w": _pitched(w), "w_scales": w_scales}
    parts = [_encode(_weights(g, n, k), BLOCK) for _ in range(case["experts"])]
    state["w"] = _pitched(torch.stack([p[0].view(torch.uint8) for p in parts]).view(torch.float8_e4m3fn))
    state["w_scales"] = torch.stack([p[1] for p in parts])
    state["offsets"], state["longest"] = _rows_of_experts(g, case["experts"], m)
    return state


# ---------------------------------------------------------------- plain forms

def _encode(x, block_rows):
    rows, cols = x.shape
    x = x.float()
    rb, cb = -(-rows // block_rows), -(-cols // BLOCK)
    p = torch.zeros(rb * block_rows, cb * BLOCK, device=x.device)
    p[:rows, :cols] = x
    p = p.view(rb, block_rows, cb, BLOCK)
    top = torch.where(torch.isfinite(p), p.abs(), 0.0).amax(dim=(1, 3), keepdim=True).clamp_min(LEAST)
    v = p * (TOP / top)
    codes = torch.where(torch.isfinite(p), v.clamp(-TOP, TOP), math.nan).to(torch.float8_e4m3fn)
    codes = codes.view(rb * block_rows, cb * BLOCK)[:rows, :cols]
    return codes, (top / TOP).view(rb, cb)


def _decode(codes, scales, block_rows):
    rows, cols = codes.shape[-2:]
    s = scales.repeat_interleave(BLOCK, -1)[..., :cols]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, -2)[..., :rows, :]
    return codes.float() * s


def _plain(s):
    op = s["op"]
    if op == "encode":
        return _encode(s["x"], s["block_rows"])
    if op == "decode":
        return _decode(s["codes"], s["scales"], s["block_rows"]).to(DTYPES[s["out"]])
    a = _decode(s["a"], s["a_scales"], 1)
    w = _decode(s["w"], s["w_scales"], BLOCK)
    if not s["transposed"]:
        w = w.transpose(-1, -2)
    if op == "matmul":
        return torch.matmul(a, w).to(DTYPES[s["out"]])
    # every expert's rows in a batch as long as the longest, then back in order
    at = torch.arange(s["longest"], device=a.device)
    start, stop = s["offsets"][:-1, None].long(), s["offsets"][1:, None].long()
    there = start + at < stop
    place = torch.where(there, start + at, 0)
    d = torch.bmm(a[place] * there[..., None], w).to(DTYPES[s["out"]])
    row = torch.arange(s["m"], device=a.device)
    expert = (row[:, None] >= stop[:, 0]).sum(1)
    return d[expert, row - start[expert, 0]]


def run(state):
    s = state
    if not own:
        return _plain(s)
    import shoehorn_b200 as sh
    ctx = sh.default_context()
    op = s["op"]
    if op == "encode":
        return ctx.encode_f8(s["x"], block_rows=s["block_rows"])
    if op == "decode":
        return ctx.decode_f8(s["codes"], s["scales"], block_rows=s["block_rows"], dtype=DTYPES[s["out"]])
    if op == "matmul":
        return ctx.matmul_f8(s["a"], s["a_scales"], s["w"], s["w_scales"], transposed=s["transposed"], dtype=DTYPES[s["out"]])
    return ctx.matmul_f8_grouped(s["a"], s["a_scales"], s["w"], s["w_scales"], s["offsets"], transposed=s["transposed"],
                                 dtype=DTYPES[s["out"]])


# ---------------------------------------------------------------- work and 64-bit values

SIZE = {"bf16": 2, "f16": 2, "f32": 4}


def work(case):
    def held(rows, cols, block_rows):  # codes and scales
        return rows * cols + 4 * -(-rows // block_rows) * -(-cols // BLOCK)

    if case["op"] in ("encode", "decode"):
        e = case["rows"] * case["cols"]
        wide = SIZE[case.get("src") or case["out"]]
        # a magnitude, a maximum and a multiplication for each element; one multiplication
        return {"bytes": e * wide + held(case["rows"], case["cols"], case["block_rows"]),
                "flops": e * (3 if case["op"] == "encode" else 1)}
    m, n, k = case["m"], case["n"], case["k"]
    inner, outer = (n, k) if case["transposed"] else (k, n)
    weights = min(case.get("experts", 1), m)  # no more experts than rows need be read
    bytes_ = held(m, inner, 1) + weights * held(n, k, BLOCK) + m * outer * SIZE[case["out"]]
    return {"bytes": bytes_ + 4 * (case.get("experts", 0) + 1), "flops": 2 * m * n * k}


def _e4m3(v):
    """The E4M3 number nearest each f64 value, ties to the even one."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    return torch.round(v / step) * step


def _exact_numbers(codes, scales, block_rows):
    i = torch.arange(codes.shape[0], device=codes.device)[:, None] // block_rows
    j = torch.arange(codes.shape[1], device=codes.device)[None, :] // BLOCK
    return codes.float().double() * scales.double()[i, j]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "encode":
        x = s["x"].double()
        i = torch.arange(x.shape[0], device=x.device)[:, None] // s["block_rows"]
        j = torch.arange(x.shape[1], device=x.device)[None, :] // BLOCK
        blocks = int(j.max()) + 1
        top = torch.zeros((int(i.max()) + 1) * blocks, dtype=torch.float64, device=x.device)
        which = (i * blocks + j)
        top.scatter_reduce_(0, which.reshape(-1), x.abs().reshape(-1), "amax")
        top = top.clamp_min(LEAST)
        return _e4m3(x * TOP / top[which]), (top / TOP).view(-1, blocks)
    if case["op"] == "decode":
        return _exact_numbers(s["codes"], s["scales"], s["block_rows"])
    a = _exact_numbers(s["a"], s["a_scales"], 1)
    if case["op"] == "matmul":
        w = _exact_numbers(s["w"], s["w_scales"], BLOCK)
        return a @ (w if s["transposed"] else w.t())
    rows, at = [], s["offsets"].tolist()
    for e in range(s["experts"]):
        if at[e + 1] > at[e]:
            w = _exact_numbers(s["w"][e], s["w_scales"][e], BLOCK)
            rows.append(a[at[e]:at[e + 1]] @ (w if s["transposed"] else w.t()))
    return torch.cat(rows)

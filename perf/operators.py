"""Cases of the four-bit weights: rows quantised into blocks of 32 numbers with one power-of-two scale (microscaled E2M1),
the product of bfloat16 rows with such weights, and the same product for routed experts.

    own = False     the plain form: elementary torch operations in float32
    own = True      the framework's calls
"""
from __future__ import annotations

import math

import torch

own = False

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)      # magnitudes of the eight codes without a sign
BLOCK = 32


# --------------------------------------------------------------------------- cases

def _rows(rows, columns, dtype):
    return dict(kind="rows", rows=rows, columns=columns, dtype=dtype)


def _linear(rows, inputs, outputs, out, gated=False):
    return dict(kind="linear", rows=rows, inputs=inputs, outputs=outputs, out=out, gated=gated)


def _experts(tokens, top, experts, inputs, outputs, first):
    """first: the product that gathers the tokens' rows and gates (outputs: twice the inner size); else the second one."""
    return dict(kind="experts", tokens=tokens, top=top, experts=experts, inputs=inputs, outputs=outputs, first=first)


def listed():
    return [
        # a small map (the router-sized end of a model) put into four bits when a model is loaded
        dict(_rows(64, 2048, "bfloat16"), name="rows_64x2048"),
        # a checkpoint kept in 32 bits, a width that ends inside a block
        dict(_rows(1537, 1000, "float32"), name="rows_1537x1000_f32"),
        # the largest single matrix of the 7B shape: gate and up rows of a feed-forward
        dict(_rows(28672, 4096, "bfloat16"), name="rows_28672x4096"),
        # one user alone, keys' and values' map of a small model: latency
        dict(_linear(1, 2048, 1024, "bfloat16"), name="linear_1_row"),
        # eight users decoding, 7B shape: gate and up with the activation, and the way down in float32
        dict(_linear(8, 4096, 28672, "bfloat16", gated=True), name="gated_8_rows"),
        dict(_linear(8, 14336, 4096, "float32"), name="linear_8_rows_down"),
        # sixty-odd decoded rows of the 12B shape, projection of queries, keys and values
        dict(_linear(67, 5120, 6144, "float32"), name="linear_67_rows"),
        # a portion with odd everything: no size a multiple of a tile, a block or a copy
        dict(_linear(301, 1001, 1543, "bfloat16"), name="linear_odd_301"),
        # the benchmark's prompt: 2,048 rows through gate and up
        dict(_linear(2048, 4096, 28672, "bfloat16", gated=True), name="gated_2048_rows"),
        # routed experts, eight decoding users: few rows for each of many experts
        dict(_experts(8, 6, 64, 4096, 3584, True), name="experts_8_up"),
        dict(_experts(8, 6, 64, 1792, 4096, False), name="experts_8_down"),
        # routed experts over a prompt
        dict(_experts(2048, 6, 64, 4096, 3584, True), name="experts_2048_up"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rows", "linear", "linear", "experts"])
    if kind == "rows":
        rows, columns = _log(rng, 1, 28672), _log(rng, 31, 16384)
        while rows * columns > 28672 * 4096:
            rows = rows // 2 + 1
        return _rows(rows, columns, rng.choice(["bfloat16", "float32"]))
    if kind == "linear":
        rows, inputs, outputs = _log(rng, 1, 2048), _log(rng, 128, 14336), _log(rng, 64, 28672)
        if rng.random() < 0.6:                           # sizes of most models are multiples of something
            inputs, outputs = inputs // 64 * 64, outputs // 64 * 64
        gated = rng.random() < 0.4
        outputs -= outputs % 2 if gated else 0
        while rows * inputs * outputs > 2048 * 4096 * 28672:
            rows = rows // 2 + 1
        # (float32 goes to the norm behind a product of decoded rows; a portion's products leave in bfloat16)
        return _linear(rows, inputs, outputs, rng.choice(["bfloat16", "float32"]) if rows <= 128 else "bfloat16", gated)
    experts = rng.choice([4, 8, 16, 32, 64])
    top = rng.randint(1, min(8, experts))
    inputs, outputs = 8 * _log(rng, 16, 512), 8 * _log(rng, 16, 448)
    return _experts(_log(rng, 1, 2048), top, experts, inputs, outputs, rng.random() < 0.5)


def work(case):
    k = case["columns"] if case["kind"] == "rows" else case["inputs"]
    packed = 17 * -(-k // BLOCK)                         # bytes of a row: 16 of codes and one scale a block
    if case["kind"] == "rows":
        # into four bits and back: what a block holds is compared as the values it stands for
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": case["rows"] * (k * size + 2 * packed + 2 * k), "flops": 3 * case["rows"] * k}
    n = case["outputs"]
    if case["kind"] == "linear":
        m, wide = case["rows"], 4 if case["out"] == "float32" else 2
        return {"bytes": n * packed + m * k * 2 + m * (n // 2 if case["gated"] else n) * wide, "flops": 2 * m * n * k}
    pairs = case["tokens"] * case["top"]
    used = case["experts"] * (1.0 - (1.0 - case["top"] / case["experts"]) ** case["tokens"])      # experts that anyone chose
    read, wide = (case["tokens"] * k * 2, n) if case["first"] else (pairs * k * 2, 4 * n)
    return {"bytes": int(used * n * packed + read + pairs * wide), "flops": 2 * pairs * n * k}


# --------------------------------------------------------------------------- inputs

def _quantize(x):
    """(codes uint8 [rows, 16 blocks], scales uint8 [rows, blocks]) of x [rows, columns]; column 2 i in the low half of
    byte i."""
    rows, columns = x.shape
    blocks = -(-columns // BLOCK)
    x = torch.nn.functional.pad(x.float(), (0, blocks * BLOCK - columns)).view(rows, blocks, BLOCK)
    largest = x.abs().amax(-1)
    mantissa, exponent = torch.frexp(largest)                                  # mantissa in [1/2, 1)
    scale = exponent + 124 + (mantissa >= 0.875).int()
    scale = torch.where(largest == 0, 0, scale.clamp(0, 254))
    y = torch.ldexp(x, (127 - scale).unsqueeze(-1))
    m = y.abs()
    code = (m > 0.25).int() + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5)      # ties to even codes
    code = (code + 8 * torch.signbit(x).int()).view(rows, blocks * BLOCK)
    return (code[:, 0::2] + 16 * code[:, 1::2]).to(torch.uint8), scale.to(torch.uint8)


def _values(codes, scales, columns):
    """float32 [rows, columns] of codes and scales."""
    rows, blocks = scales.shape
    grid = torch.tensor(GRID + tuple(-v for v in GRID), device=codes.device)
    v = torch.stack([grid[(codes & 15).long()], grid[(codes >> 4).long()]], -1).view(rows, blocks, BLOCK)
    v = v * torch.exp2(scales.float() - 127.0).unsqueeze(-1)
    return v.view(rows, blocks * BLOCK)[:, :columns]


def _stretches(case, g):
    """Which expert every (token, choice) goes to, sorted by expert with every expert's stretch padded to whole tiles:
    (tile, place_token, tile_expert, [(expert, first place, places)])."""
    tokens, top, experts = case["tokens"], case["top"], case["experts"]
    chosen = torch.rand(tokens, experts, generator=g).argsort(1)[:, :top]
    pairs = tokens * top
    tile = 16 if pairs <= 16 * experts else 32
    tiles = pairs // tile + min(experts, pairs)
    place_token = torch.full((tiles * tile,), -1, dtype=torch.int32)
    tile_expert = torch.full((tiles,), -1, dtype=torch.int32)
    stretches, at = [], 0
    for e in range(experts):
        who = (chosen == e).any(1).nonzero().flatten()
        n = len(who)
        if n == 0:
            continue
        place_token[at:at + n] = who.int()
        wide = -(-n // tile) * tile
        tile_expert[at // tile:(at + wide) // tile] = e
        stretches.append((e, at, n))
        at += wide
    return tile, place_token.cuda(), tile_expert.cuda(), stretches


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    if case["kind"] == "rows":
        # rows of different sizes, as trained weights have them
        x = normal(case["rows"], case["columns"]) * (0.02 * torch.exp2(normal(case["rows"], 1)))
        return dict(x=x.to(getattr(torch, case["dtype"])))
    k, n = case["inputs"], case["outputs"]
    if case["kind"] == "linear":
        codes, scales = _quantize(normal(n, k) * k ** -0.5)
        a = normal(case["rows"], k).bfloat16()
        return dict(a=a, codes=codes, scales=scales)
    s = dict(zip(("tile", "place_token", "tile_expert", "stretches"),
                 _stretches(case, torch.Generator().manual_seed(seed))))
    parts = [_quantize(normal(n, k) * k ** -0.5) for _ in range(case["experts"])]
    s["codes"], s["scales"] = (torch.stack([p[i] for p in parts]) for i in range(2))
    if case["first"]:
        s["a"] = normal(case["tokens"], k).bfloat16()
    else:                                                # what the first product left: rows by place, zeros where nobody is
        a = normal(len(s["place_token"]), k) * (s["place_token"] >= 0).unsqueeze(1)
        s["a"] = (a * a.abs()).bfloat16()
    return s


def prepare(case, seed):
    s = dict(_inputs(case, seed), case=case)
    if case["kind"] == "linear":
        wide = case["outputs"] // 2 if case["gated"] else case["outputs"]
        s["out"] = torch.zeros(case["rows"], wide, dtype=getattr(torch, case["out"]), device="cuda")
    elif case["kind"] == "experts":
        # (places of tiles without an expert are left as they are: zeros from here on)
        wide, dtype = (case["outputs"] // 2, torch.bfloat16) if case["first"] else (case["outputs"], torch.float32)
        s["out"] = torch.zeros(len(s["place_token"]), wide, dtype=dtype, device="cuda")
    if own and case["kind"] != "rows":
        from types import SimpleNamespace

        from flambeau_b200.engine.runtime import Runtime
        from flambeau_b200.kernels import ops
        runtime = Runtime("cuda:0", "bfloat16")
        s["ctx"] = SimpleNamespace(runtime=runtime, ws=runtime.ws)
        s["w"] = ops.Mxfp4Weight(s["codes"], s["scales"], case["inputs"])
    return s


# --------------------------------------------------------------------------- one pass

def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from flambeau_b200.kernels import ops
    case = s["case"]
    if case["kind"] == "rows":
        codes, scales = ops.quantize_mxfp4(s["x"])
        return ops.dequantize_mxfp4(codes, scales, case["columns"], torch.bfloat16)
    if case["kind"] == "linear":
        if case["gated"]:
            ops.gated_linear(s["a"], s["w"], s["out"], "silu", s["ctx"])
        else:
            ops.linear(s["a"], s["w"], s["out"], s["ctx"])
    elif case["first"]:
        ops.grouped_gated_linear(s["a"], s["place_token"], s["w"], s["tile_expert"], s["tile"], s["out"], "silu", s["ctx"])
    else:
        ops.grouped_linear(s["a"], None, s["w"], s["tile_expert"], s["tile"], s["out"], None, s["ctx"])
    return s["out"]


def _silu_gated(z):
    """Rows alternate: a gate, then what it multiplies."""
    g, u = z[:, 0::2], z[:, 1::2]
    return g / (1.0 + torch.exp(-g)) * u


def _run_plain(s):
    case = s["case"]
    if case["kind"] == "rows":
        codes, scales = _quantize(s["x"])
        return _values(codes, scales, case["columns"]).bfloat16()
    k = case["inputs"]
    if case["kind"] == "linear":
        z = s["a"].float() @ _values(s["codes"], s["scales"], k).T
        return (_silu_gated(z) if case["gated"] else z).to(s["out"].dtype)
    out = torch.zeros_like(s["out"])
    for e, at, n in s["stretches"]:
        rows = s["a"][s["place_token"][at:at + n].long()] if case["first"] else s["a"][at:at + n]
        z = rows.float() @ _values(s["codes"][e], s["scales"][e], k).T
        out[at:at + n] = _silu_gated(z) if case["first"] else z
    return out


# --------------------------------------------------------------------------- the definition in 64 bits

def _nearest(x):
    """Every number of x [rows, columns] put on its block's grid, in float64: the scale is the smallest power of two (not
    below 2^-127) under which the block's largest magnitude lies below 7, where rounding still ends at 6; of two grid
    points that are equally near, the one with the even code."""
    rows, columns = x.shape
    x = x.double()
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    out = torch.empty_like(x)
    for c in range(0, columns, BLOCK):
        part = x[:, c:c + BLOCK]
        largest = part.abs().amax(1, keepdim=True)
        e = torch.ceil(torch.log2(torch.where(largest > 0, largest, 1.0) / 7.0)).clamp(min=-127.0)
        e = torch.where(largest < 7.0 * torch.exp2(e), e, e + 1)               # (the logarithm's last bit does not decide)
        e = torch.where(largest < 7.0 * torch.exp2(e - 1), e - 1, e).clamp(min=-127.0)
        y = part.abs() / torch.exp2(e)
        up = torch.bucketize(y, grid).clamp(max=7)                             # first point not below y
        lo, hi = grid[(up - 1).clamp(min=0)], grid[up]
        take = (hi - y < y - lo) | ((hi - y == y - lo) & (up % 2 == 0))
        out[:, c:c + BLOCK] = torch.where(take, hi, lo) * torch.sign(part) * torch.exp2(e)
    return out


def _decoded(codes, scales, columns):
    """float64 [rows, columns]: sign bit, two bits of exponent, one of mantissa."""
    c = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.int64, device=codes.device)
    c[:, 0::2], c[:, 1::2] = (codes % 16).long(), torch.div(codes, 16, rounding_mode="floor").long()
    e, m = (c >> 1) & 3, (c & 1).double()
    v = torch.where(e == 0, m / 2, (1 + m / 2) * (2.0 ** (e - 1).double()))
    v = torch.where(c >= 8, -v, v) * (2.0 ** (scales.double() - 127)).repeat_interleave(BLOCK, 1)
    return v[:, :columns]


def exact(case, seed):
    s = _inputs(case, seed)
    if case["kind"] == "rows":
        return _nearest(s["x"])

    def product(rows, codes, scales, gated):
        z = rows.double() @ _decoded(codes, scales, case["inputs"]).T
        if gated:
            z = z.view(len(z), -1, 2)
            z = z[..., 0] * torch.sigmoid(z[..., 0]) * z[..., 1]
        return z
    if case["kind"] == "linear":
        return product(s["a"], s["codes"], s["scales"], case["gated"])
    wide = case["outputs"] // 2 if case["first"] else case["outputs"]
    out = torch.zeros(len(s["place_token"]), wide, dtype=torch.float64, device="cuda")
    place = s["place_token"].cpu()
    for e in range(case["experts"]):
        mine = (s["tile_expert"].cpu() == e).repeat_interleave(s["tile"]) & (place >= 0)
        where = mine.nonzero().flatten().cuda()
        if len(where):
            rows = s["a"][s["place_token"][where].long()] if case["first"] else s["a"][where]
            out[where] = product(rows, s["codes"][e], s["scales"][e], case["first"])
    return out

"""The MXFP4 operators' measured cases: what a serving program calls, over the range it calls it at.

MXFP4: 32 consecutive values of a row share a power-of-two scale (an E8M0 byte, the
exponent biased by 127), and each is a 4-bit e2m1 code (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives; the even column in a byte's low half).  The scale is the smallest at
which the block's largest value rounds to 6 or less; a block with a value that is not
finite has exponent 255 and is NaN.

A case is a dict of plain values.  ``kind`` names what is called:

* ``roundtrip``   rows quantised and read back: ``quantize_rows_mxfp4`` and
  ``dequantize_rows_mxfp4``.
* ``dequantise``  a quantised matrix read back alone.
* ``pack``        expert masters made into the packed operands (quantised along the
  reduction), and those widened to the bfloat16 operands that hold the same weights.
* ``ffn``         the routed experts as the layer runs them: tokens quantised, the
  gathering gate/up product with the SwiGLU and h's quantisation, the down product.
* ``down``        the down product alone, on rows in the experts' order.

Layouts that the calls share: the packed gate/up operand has 2F rows an expert, blocks
of 32 gate and 32 up columns alternating, D values each; the down operand D rows of F
values.  A packed operand keeps its codes as the matrix instruction reads them, ``[N,
rows / 32, K / 64, 64, 16]``: lane 32 h + r of a block has the 32 codes of row r from
column 32 h on.  Its exponents are ``[N, K / 128, rows, 4]``.
"""
import math

import torch

own = False

BLOCK = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _rows(kind, rows, cols, dtype, **more):
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, **more)


def _experts(kind, tokens, experts, active, d_model, d_ff, **more):
    return dict(kind=kind, tokens=tokens, experts=experts, active=active, d_model=d_model, d_ff=d_ff, **more)


def _pack(experts, d_model, d_ff, dtype, **more):
    return dict(kind="pack", experts=experts, d_model=d_model, d_ff=d_ff, dtype=dtype, **more)


def listed():
    return [
        # the tokens of a small decode batch in float32, an odd number of blocks a row
        _rows("roundtrip", 7, 1056, "f32", name="roundtrip_7_f32"),
        # a long prefill's tokens on their way into the experts
        _rows("roundtrip", 16384, 2048, "bf16", name="roundtrip_16384"),
        # a decode batch's h looked at in float32
        _rows("dequantise", 385, 1024, "f32", name="dequantise_385_f32"),
        # a prefill's h, or a whole operand, widened to bfloat16
        _rows("dequantise", 131072, 1024, "bf16", name="dequantise_131072"),
        # a small layer's masters packed when it is loaded
        _pack(8, 256, 512, "f32", name="pack_8"),
        # the benchmark layer's masters packed
        _pack(64, 2048, 1024, "f32", name="pack_64"),
        # one sequence's decode step: one token, eight experts
        _experts("ffn", 1, 64, 8, 2048, 1024, name="ffn_1"),
        # a serving batch's decode step on the layer with wide experts
        _experts("ffn", 48, 32, 4, 4096, 2048, name="ffn_48"),
        # a short prompt of odd length on a layer whose sizes are odd multiples of 128
        _experts("ffn", 333, 24, 3, 1152, 640, name="ffn_333"),
        # the benchmark's layer, the largest prefill
        _experts("ffn", 16384, 64, 8, 2048, 1024, name="ffn_16384"),
        # the down product of a decode batch and of a prefill
        _experts("down", 100, 64, 8, 2048, 1024, name="down_100"),
        _experts("down", 8192, 32, 4, 4096, 2048, name="down_8192"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["roundtrip", "dequantise", "pack", "ffn", "ffn", "ffn", "ffn", "down", "down"])
    if kind in ("roundtrip", "dequantise"):
        cols = BLOCK * _log_int(rng, 4, 128)
        return _rows(kind, _log_int(rng, 1, (1 << 25) // cols), cols, rng.choice(["bf16", "f32"]))
    while True:
        d_model, d_ff = 128 * rng.randint(2, 32), 128 * rng.randint(1, 16)
        experts = _log_int(rng, 1, 128)
        if experts * d_model * d_ff <= (1 << 27):
            break
    if kind == "pack":
        return _pack(experts, d_model, d_ff, rng.choice(["bf16", "f32"]))
    active = rng.randint(1, min(8, experts))
    most = (16384 * 8 * 2048 * 1024) // (active * d_model * d_ff)
    return _experts(kind, _log_int(rng, 1, min(16384, most)), experts, active, d_model, d_ff)


# --------------------------------------------------------------- quantising --

def _scales(biased):
    """2^(biased - 127) in float32, NaN at 255."""
    biased = biased.to(torch.int32)
    bits = torch.where(biased > 0, biased << 23, torch.full_like(biased, 0x00400000))
    bits = torch.where(biased == 255, torch.full_like(biased, 0x7FC00000), bits)
    return bits.view(torch.float32)


def _quantise(v):
    """e2m1 codes (one a value) and biased exponents (one a block) of float32 rows."""
    blocks = v.reshape(*v.shape[:-1], v.shape[-1] // BLOCK, BLOCK)
    amax = blocks.abs().amax(-1)
    biased = (((amax.view(torch.int32) + 0x200000) >> 23) - 2).clamp_(min=0)
    biased = torch.where(torch.isfinite(amax), biased, torch.full_like(biased, 255))
    inverse = torch.where(biased < 255, (254 - biased) << 23, torch.zeros_like(biased)).view(torch.float32)
    a = (blocks * inverse.unsqueeze(-1)).nan_to_num(0.0)
    # halfway cases go to the code whose last bit is 0
    m = a.abs()
    code = ((m > 0.25).to(torch.uint8) + (m >= 0.75) + (m > 1.25) + (m >= 1.75) + (m > 2.5) + (m >= 3.5) + (m > 5.0))
    code = code + (torch.signbit(a).to(torch.uint8) << 3)
    return code.reshape(v.shape), biased.to(torch.uint8)


def _halves(code):
    """Two codes a byte, the even column in the low half."""
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _values(packed, biased):
    """float32 values of packed codes [..., C / 2] and exponents [..., C / 32]."""
    code = torch.stack((packed & 15, packed >> 4), -1).reshape(*packed.shape[:-1], packed.shape[-1] * 2)
    table = torch.tensor(E2M1 + tuple(-x for x in E2M1), dtype=torch.float32, device=packed.device)
    v = table[code.int()].reshape(*biased.shape, BLOCK)
    return (v * _scales(biased).unsqueeze(-1)).reshape(code.shape)


def _operand_codes(rows):
    """[N, rows, K / 2] as a packed operand keeps them: [N, rows / 32, K / 64, 64, 16]."""
    n, r, half = rows.shape
    blocks = rows.reshape(n, r // 32, 32, half // 32, 2, 16).permute(0, 1, 3, 4, 2, 5)
    return blocks.reshape(n, r // 32, half // 32, 64, 16)


def _row_codes(packed):
    """The other way: [N, rows / 32, K / 64, 64, 16] -> [N, rows, K / 2]."""
    n, r, c = packed.shape[:3]
    return packed.reshape(n, r, c, 2, 32, 16).permute(0, 1, 4, 2, 3, 5).reshape(n, r * 32, c * 32)


def _operand_exponents(biased):
    """[N, rows, K / 32] as a packed operand keeps them: [N, K / 128, rows, 4]."""
    n, rows, blocks = biased.shape
    return biased.reshape(n, rows, blocks // 4, 4).transpose(1, 2).contiguous()


def _row_exponents(packed):
    """The other way: [N, K / 128, rows, 4] -> [N, rows, K / 32]."""
    n, groups, rows, _ = packed.shape
    return packed.transpose(1, 2).reshape(n, rows, groups * 4)


def _gate_up_rows(gate, up):
    """[N, F, D] gate and up rows in the packed order: 32 of one, 32 of the other."""
    n, f, d = gate.shape
    return torch.stack((gate.reshape(n, f // BLOCK, BLOCK, d), up.reshape(n, f // BLOCK, BLOCK, d)),
                       2).reshape(n, 2 * f, d)


# ------------------------------------------------------------------- states --

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _tokens(g, rows, cols):
    """Activations: each row at a level of its own, a few columns far above the rest."""
    v = _normal(g, (rows, cols)) * torch.exp(_normal(g, (rows, 1), 0.5))
    return v * torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)


def _operand(g, experts, rows, k):
    """A packed operand of random weights, expert by expert."""
    codes = torch.empty((experts, rows, k // 2), dtype=torch.uint8, device="cuda")
    biased = torch.empty((experts, rows, k // BLOCK), dtype=torch.uint8, device="cuda")
    for e in range(experts):
        code, biased[e] = _quantise(_normal(g, (rows, k), 0.02))
        codes[e] = _halves(code)
    return _operand_codes(codes), _operand_exponents(biased)


def _plan(g, case):
    """Who goes where, as the layer's dispatch plan says it: no token is dropped."""
    t, n, k = case["tokens"], case["experts"], case["active"]
    popular = _normal(g, (n,), 0.5)
    top = (_normal(g, (t, n)) + popular).topk(k, dim=1).indices.reshape(-1)
    order = torch.argsort(top, stable=True)
    counts = torch.bincount(top, minlength=n)
    offsets = torch.zeros(n + 1, dtype=torch.int64, device="cuda")
    offsets[1:] = counts.cumsum(0)
    place = torch.empty_like(order)
    place[order] = torch.arange(t * k, device="cuda")
    live = counts.nonzero().reshape(-1)
    expert = torch.searchsorted(live, top[order])       # of each row, among the live ones
    return dict(counts=counts.int(), offsets=offsets.int(), slot_pos=place.int(), perm_src=order.int(),
                keep=torch.ones(t * k, dtype=torch.uint8, device="cuda"), live=live, most=int(counts.max()),
                expert=expert, within=torch.arange(t * k, device="cuda") - offsets[top[order]])


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    s = dict(kind=kind, case=case)
    if kind in ("roundtrip", "dequantise"):
        x = _tokens(g, case["rows"], case["cols"])
        if kind == "roundtrip":
            s["x"] = x.to(TYPES[case["dtype"]])
        else:
            code, s["exp"] = _quantise(x)
            s["q"] = _halves(code)
        return s
    n, d, f = case["experts"], case["d_model"], case["d_ff"]
    if kind == "pack":
        for name, shape in (("gate", (n, d, f)), ("up", (n, d, f)), ("down", (n, f, d))):
            s[name] = _normal(g, shape, 0.02).to(TYPES[case["dtype"]])
        return s
    s["plan"] = _plan(g, case)
    s["down"], s["down_exp"] = _operand(g, n, d, f)
    if kind == "ffn":
        s["x"] = _tokens(g, case["tokens"], d).to(torch.bfloat16)
        s["gate_up"], s["gate_up_exp"] = _operand(g, n, 2 * f, d)
    else:
        code, s["h_exp"] = _quantise(_tokens(g, case["tokens"] * case["active"], f))
        s["h_q"] = _halves(code)
    return s


# ------------------------------------------------------------- plain forms --

def _product(rows, plan, codes, exponents):
    """rows [R, K] in the experts' order times each one's operand: the experts as a batch,
    each padded to the fullest one's rows."""
    live = plan["live"]
    if live.numel() < codes.shape[0]:
        codes, exponents = codes[live], exponents[live]
    w = _values(_row_codes(codes), _row_exponents(exponents))
    batch = torch.zeros((w.shape[0], plan["most"], w.shape[2]), dtype=torch.float32, device="cuda")
    batch[plan["expert"], plan["within"]] = rows
    return torch.bmm(batch, w.transpose(1, 2).contiguous())[plan["expert"], plan["within"]]


def _plain_packed(rows):
    code, biased = _quantise(rows)
    return _values(_halves(code), biased).to(torch.bfloat16)


def _plain_down(s, h):
    return _product(h, s["plan"], s["down"], s["down_exp"]).to(torch.bfloat16)


def _plain(s):
    kind = s["kind"]
    if kind == "roundtrip":
        code, biased = _quantise(s["x"].float())
        return _values(_halves(code), biased).to(s["x"].dtype)
    if kind == "dequantise":
        return _values(s["q"], s["exp"]).to(TYPES[s["case"]["dtype"]])
    if kind == "pack":
        gate, up, down = (s[name].float().transpose(1, 2).contiguous() for name in ("gate", "up", "down"))
        return [_plain_packed(_gate_up_rows(gate, up)), _plain_packed(down)]
    if kind == "down":
        return _plain_down(s, _values(s["h_q"], s["h_exp"]))
    code, biased = _quantise(s["x"].float())
    x = _values(_halves(code), biased)
    gu = _product(x[s["plan"]["perm_src"].long() // s["case"]["active"]], s["plan"], s["gate_up"], s["gate_up_exp"])
    g, u = gu.reshape(gu.shape[0], -1, 2, BLOCK).unbind(2)
    h = (g / (1.0 + torch.exp(-g)) * u).reshape(gu.shape[0], -1)
    code, biased = _quantise(h)
    return _plain_down(s, _values(_halves(code), biased))


# ------------------------------------------------------------ the framework --

def _own(s):
    from hanuman_amd import kernels as K
    kind = s["kind"]
    if kind == "roundtrip":
        q, exp = K.quantize_rows_mxfp4(s["x"])
        return K.dequantize_rows_mxfp4(q, exp, s["x"].dtype)
    if kind == "dequantise":
        return K.dequantize_rows_mxfp4(s["q"], s["exp"], TYPES[s["case"]["dtype"]])
    if kind == "pack":
        return [K.unpack_mxfp4(*K.pack_mxfp4_gate_up(s["gate"], s["up"])),
                K.unpack_mxfp4(*K.pack_mxfp4_down(s["down"]))]
    p, c = s["plan"], s["case"]
    if kind == "down":
        return K.grouped_down_mxfp4(s["h_q"], s["h_exp"], p["offsets"], s["down"], s["down_exp"])
    rows = c["tokens"] * c["active"]
    plan = K.Plan(p["counts"], p["offsets"], p["slot_pos"], p["perm_src"], p["keep"], rows, rows, c["experts"],
                  c["active"])
    x_q, x_exp = K.quantize_rows_mxfp4(s["x"])
    h_q, h_exp = K.grouped_gate_up_mxfp4_gather(x_q, x_exp, plan, s["gate_up"], s["gate_up_exp"])
    return K.grouped_down_mxfp4(h_q, h_exp, p["offsets"], s["down"], s["down_exp"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------ what is right --

def _power_of_two(e):
    """2^e in float64, from its bits: a power function may be off in the last one."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_rows(v):
    """The values that float64 rows stand for in MXFP4: the scale from the largest value's
    logarithm, each value to the nearest multiple of its step, ties to the even multiple."""
    b = v.reshape(*v.shape[:-1], -1, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    mantissa, exponent = torch.frexp(amax)              # amax = mantissa * 2^exponent, mantissa in [0.5, 1)
    e = exponent - 3 + (mantissa >= 0.875).int()        # 7 and more of a scale's units take the next scale
    e = torch.where(amax > 0, e, torch.full_like(e, -127)).clamp(min=-127)
    scale = _power_of_two(e)
    m = b / scale
    octave = torch.frexp(m.abs())[1] - 1                # floor(log2 |m|)
    step = _power_of_two(octave.clamp(min=0) - 1)
    return ((torch.round(m / step) * step).clamp(-6.0, 6.0) * scale).reshape(v.shape)


def _exact_operand(codes, exponents):
    """float64 weights [rows, K] of one expert's packed operand."""
    lanes = codes.reshape(codes.shape[0], -1, 2, 32, 16).transpose(1, 3).transpose(2, 3)
    return _exact_codes(lanes.reshape(codes.shape[0] * 32, -1), exponents.permute(1, 0, 2))


def _exact_codes(codes, exponents):
    """float64 values [rows, K] of codes [rows, K / 2] and exponents whose first index is the row."""
    bits = torch.stack((codes % 16, codes // 16), -1).reshape(codes.shape[0], -1)
    fraction, power = (bits % 2).double(), (bits // 2 % 4).long()
    size = torch.where(power > 0, (1 + fraction / 2) * _power_of_two(power - 1), fraction / 2)
    size = torch.where(bits >= 8, -size, size)
    e = exponents.reshape(codes.shape[0], -1).long() - 127
    return size * _power_of_two(e).repeat_interleave(BLOCK, 1)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "roundtrip":
        return _exact_rows(s["x"].double())
    if kind == "dequantise":
        return _exact_codes(s["q"], s["exp"])
    if kind == "pack":
        n, f = case["experts"], case["d_ff"]
        column = torch.arange(2 * f, device="cuda")
        column = torch.where(column // 32 % 2 == 0, 0, f) + column // 64 * 32 + column % 32
        gate_up, down = [], []
        for e in range(n):
            both = torch.cat((s["gate"][e], s["up"][e]), 1)[:, column]
            gate_up.append(_exact_rows(both.double().t().contiguous()).to(torch.float32))
            down.append(_exact_rows(s["down"][e].double().t().contiguous()).to(torch.float32))
        return [torch.stack(gate_up), torch.stack(down)]
    p = s["plan"]
    out = torch.empty((case["tokens"] * case["active"], case["d_model"]), dtype=torch.float64, device="cuda")
    x = _exact_rows(s["x"].double()) if kind == "ffn" else None
    edges = p["offsets"].tolist()
    for e in range(case["experts"]):
        lo, hi = edges[e], edges[e + 1]
        if lo == hi:
            continue
        if kind == "ffn":
            w = _exact_operand(s["gate_up"][e], s["gate_up_exp"][e])
            gu = x[p["perm_src"][lo:hi].long() // case["active"]] @ w.t()
            gu = gu.reshape(hi - lo, -1, 2, BLOCK)
            h = _exact_rows((gu[:, :, 0] * torch.sigmoid(gu[:, :, 0]) * gu[:, :, 1]).reshape(hi - lo, -1))
        else:
            h = _exact_codes(s["h_q"][lo:hi], s["h_exp"][lo:hi])
        out[lo:hi] = h @ _exact_operand(s["down"][e], s["down_exp"][e]).t()
    return out


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once; a code and
    its share of a scale are 17 / 32 of a byte.  Only the experts with rows are read."""
    kind = case["kind"]
    size = {"bf16": 2, "f32": 4}
    code = 17 / 32
    if kind in ("roundtrip", "dequantise"):
        values = case["rows"] * case["cols"]
        wide = size[case["dtype"]]
        # the codes are quantise's output and dequantise's input
        return dict(bytes=values * (2 * wide + 2 * code) if kind == "roundtrip" else values * (wide + code), flops=0)
    d, f = case["d_model"], case["d_ff"]
    if kind == "pack":
        values = 3 * case["experts"] * d * f
        return dict(bytes=values * (size[case["dtype"]] + 2 * code + 2), flops=0)
    rows = case["tokens"] * case["active"]
    live = min(case["experts"], rows)
    if kind == "down":
        return dict(bytes=(rows * f + live * d * f) * code + rows * d * 2, flops=2 * rows * d * f)
    return dict(bytes=case["tokens"] * d * 2 + live * 3 * d * f * code + rows * d * 2, flops=6 * rows * d * f)

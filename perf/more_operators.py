"""The half block around the experts, measured: norm, routing by groups, int8 experts.

A case is a dict of plain values.  ``kind`` names what is called:

* ``norm``        ``add_rms_norm``: the residual's addition, the root-mean-square norm and
  the normed rows' 8-bit codes in one call; the codes are read back.
* ``norm_bwd``    its gradients, from the saved sum and reciprocal root.
* ``route``       ``router`` with groups: logits, and the experts of the best groups.
* ``logits``      ``router_from_logits`` with groups.
* ``route_train`` that and the gates' gradient with respect to the logits.
* ``ffn``         the routed experts as the layer runs them in int8: tokens quantised, the
  gathering gate/up product with the SwiGLU, h quantised, the down product.

8-bit rows: a row's scale is its largest value over 127 (int8) or 448 (e4m3), a code the
value times the largest code over the largest value, rounded to nearest even; a row of
zeros has scale 1.

Routing by groups: an expert's key is its logit (softmax), or its logit's sigmoid plus its
bias, in float32; a group's score is its largest key (softmax) or the sum of its two
largest.  The experts with the largest keys among those of the groups with the largest
scores are taken, the lower index first where equal.  Sigmoid and exponential are the
framework's float32 sequence of single operations (range reduction by ln 2 in two parts, a
polynomial of degree 7), so that which expert is taken does not hang on a last bit.

Layout that the int8 products share: codes of a packed operand are kept as the matrix
instruction reads them, ``[N, rows / 32, K / 32, 64, 16]``: lane 32 h + r of a block has
the 16 codes of row r from column 16 h on.  The gate/up operand's rows are blocks of 32
gate and 32 up columns alternating.  Scales are ``[N, rows]`` in the operand's row order.
"""
import math

import torch

own = False

EPS = 1e-6
RSF = 2.5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LARGEST = {"int8": 127.0, "e4m3": 448.0}
BLOCK = 32


def _norm(kind, rows, cols, dtype, **more):
    return dict(kind=kind, rows=rows, cols=cols, dtype=dtype, **more)


def _route(kind, tokens, experts, groups, top_groups, active, routing, **more):
    return dict(kind=kind, tokens=tokens, experts=experts, groups=groups, top_groups=top_groups, active=active,
                routing=routing, **more)


def _ffn(tokens, experts, active, d_model, d_ff, **more):
    return dict(kind="ffn", tokens=tokens, experts=experts, active=active, d_model=d_model, d_ff=d_ff, **more)


def listed():
    return [
        # one sequence's decode step ahead of int8 experts
        _norm("norm", 1, 2048, "bf16", quant="int8", residual=True, name="norm_1"),
        # a ragged batch of prompts in float32, the first norm of a block (nothing to add)
        _norm("norm", 385, 1056, "f32", quant="int8", residual=False, name="norm_385_f32"),
        # a long prefill ahead of e4m3 experts
        _norm("norm", 16384, 2048, "bf16", quant="e4m3", residual=True, name="norm_16384"),
        # a training step's batch on the published layer's width, and a wide layer's
        _norm("norm_bwd", 2048, 1536, "f32", name="norm_bwd_2048_f32"),
        _norm("norm_bwd", 16384, 4096, "bf16", name="norm_bwd_16384"),
        # one token on the benchmark layer's experts in groups of eight
        _route("route", 1, 64, 8, 4, 8, "sigmoid", d_model=2048, name="route_1"),
        # a prefill on the widest layer that the router takes
        _route("logits", 16384, 256, 8, 4, 8, "sigmoid", name="logits_16384"),
        # a training batch on the published layer's experts, in groups of twenty
        _route("route_train", 4096, 80, 4, 2, 8, "softmax", name="route_train_4096"),
        # one sequence's decode step: one token, eight experts
        _ffn(1, 64, 8, 2048, 1024, name="ffn_1"),
        # a serving batch's decode step on the layer with wide experts
        _ffn(48, 32, 4, 4096, 2048, name="ffn_48"),
        # a short prompt of odd length on a layer whose sizes are odd multiples of 128
        _ffn(333, 24, 3, 1152, 640, name="ffn_333"),
        # the benchmark's layer, the largest prefill
        _ffn(16384, 64, 8, 2048, 1024, name="ffn_16384"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm", "norm", "norm_bwd", "route", "logits", "route_train", "ffn", "ffn", "ffn"])
    if kind in ("norm", "norm_bwd"):
        cols = 8 * _log_int(rng, 16, 1024)
        rows = _log_int(rng, 1, (1 << 25) // cols)
        case = _norm(kind, rows, cols, rng.choice(["bf16", "f32"]))
        if kind == "norm":
            case.update(quant=rng.choice(["int8", "e4m3"]), residual=rng.choice([True, True, False]))
        return case
    if kind == "ffn":
        while True:
            d_model, d_ff = 128 * rng.randint(2, 32), 128 * rng.randint(1, 16)
            experts = _log_int(rng, 1, 128)
            if experts * d_model * d_ff <= (1 << 27):
                break
        active = rng.randint(1, min(8, experts))
        most = (16384 * 8 * 2048 * 1024) // (active * d_model * d_ff)
        return _ffn(_log_int(rng, 1, min(16384, most)), experts, active, d_model, d_ff)
    groups = rng.choice([2, 4, 4, 5, 8, 8, 16])
    experts = groups * rng.randint(2, 256 // groups)
    top_groups = rng.randint(1, groups - 1)
    active = rng.randint(1, min(12, top_groups * (experts // groups)))
    case = _route(kind, _log_int(rng, 1, 4096 if kind == "route" else 16384), experts, groups, top_groups, active,
                  rng.choice(["sigmoid", "softmax"]))
    if kind == "route":
        case["d_model"] = 128 * rng.randint(2, 32)
    return case


# ------------------------------------------------------------------- states --

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).mul_(std)


def _tokens(g, rows, cols):
    """Activations: each row at a level of its own, a few columns far above the rest."""
    v = _normal(g, (rows, cols)) * torch.exp(_normal(g, (rows, 1), 0.5))
    return v * torch.where(torch.rand(cols, generator=g, device="cuda") < 0.01, 8.0, 1.0)


def _operand_codes(rows):
    """int8 codes [rows, K] of an expert as a packed operand keeps them."""
    r, k = rows.shape
    return rows.reshape(r // 32, 32, k // 32, 2, 16).permute(0, 2, 3, 1, 4).reshape(r // 32, k // 32, 64, 16)


def _operand(g, experts, rows, k):
    """A packed operand of random weights, expert by expert, and its scales."""
    codes = torch.empty((experts, rows // 32, k // 32, 64, 16), dtype=torch.int8, device="cuda")
    scales = torch.empty((experts, rows), dtype=torch.float32, device="cuda")
    for e in range(experts):
        code, scales[e] = _codes8(_normal(g, (rows, k), 0.02), "int8")
        codes[e] = _operand_codes(code.to(torch.int8))
    return codes, scales


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
    if kind in ("norm", "norm_bwd"):
        shape, dtype = (case["rows"], case["cols"]), TYPES[case["dtype"]]
        s["weight"] = 1.0 + _normal(g, (case["cols"],), 0.1)
        if kind == "norm":
            s["x"] = _tokens(g, *shape).to(dtype)
            s["residual"] = _tokens(g, *shape).to(dtype) if case["residual"] else None
            return s
        s["sum"] = _tokens(g, *shape).to(dtype)
        s["rstd"] = torch.rsqrt(s["sum"].float().pow(2).mean(1) + EPS)
        s["dy"] = _normal(g, shape, 1e-2).to(dtype)
        s["d_sum"] = _normal(g, shape, 1e-2).to(dtype)
        return s
    if kind == "ffn":
        n, d, f = case["experts"], case["d_model"], case["d_ff"]
        s["plan"] = _plan(g, case)
        s["x"] = _tokens(g, case["tokens"], d).to(torch.bfloat16)
        s["gate_up"], s["gate_up_scale"] = _operand(g, n, 2 * f, d)
        s["down"], s["down_scale"] = _operand(g, n, d, f)
        return s
    t, n = case["tokens"], case["experts"]
    # a trained layer's balancing bias is small and not zero
    s["bias"] = _normal(g, (n,), 0.02) if case["routing"] == "sigmoid" else None
    if kind == "route":
        s["x"] = _normal(g, (t, case["d_model"])).to(torch.bfloat16)
        s["router"] = _normal(g, (case["d_model"], n), 0.02)
        return s
    s["logits"] = _normal(g, (t, n))
    if kind == "route_train":
        s["d_gates"] = _normal(g, (t, case["active"]), 1e-2)
    return s


# ------------------------------------------------------------- plain forms --

def _codes8(v, to):
    """8-bit codes (as the values of their type, in float32) of float32 rows and the rows' scales."""
    most = LARGEST[to]
    amax = v.abs().amax(-1)
    zero = amax == 0
    scale = torch.where(zero, torch.ones_like(amax), amax / most)
    inverse = torch.where(zero, torch.ones_like(amax), most / amax)
    code = (v * inverse.unsqueeze(-1)).clamp(-most, most)
    return torch.round(code) if to == "int8" else code.to(torch.float8_e4m3fn).float(), scale


def _plain_norm(s):
    case, x = s["case"], s["x"]
    total = x
    if s["residual"] is not None:
        total = (x.float() + s["residual"].float()).to(x.dtype)
    v = total.float()
    rstd = 1.0 / torch.sqrt((v * v).mean(1) + EPS)
    y = (v * rstd.unsqueeze(1) * s["weight"]).to(x.dtype)
    code, scale = _codes8(y.float(), case["quant"])
    return [total, y, rstd, (code * scale.unsqueeze(1)).to(torch.bfloat16)]


def _plain_norm_bwd(s):
    v, dy, rstd = s["sum"].float(), s["dy"].float(), s["rstd"].unsqueeze(1)
    xhat = v * rstd
    dn = dy * s["weight"]
    dx = s["d_sum"].float() + rstd * (dn - xhat * (dn * xhat).mean(1, keepdim=True))
    return [dx.to(s["sum"].dtype), (dy * xhat).sum(0)]


def _bits(pattern):
    return torch.tensor(pattern, dtype=torch.int32, device="cuda").view(torch.float32)


def _exp32(x):
    """The framework's float32 exponential, one rounded operation after another."""
    n = torch.round(x * _bits(0x3FB8AA3B))
    r = x - n * _bits(0x3F317200)
    r = r - n * _bits(0x35BFBE8E)
    p = _bits(0x39500D01).expand_as(x)
    for c in (0x3AB60B61, 0x3C088889, 0x3D2AAAAB, 0x3E2AAAAB, 0x3F000000, 0x3F800000, 0x3F800000):
        p = p * r
        p = p + _bits(c)
    # 2^n as two factors, each of which float32 holds
    half = torch.floor(n * 0.5)
    power = [((h.int().clamp(-126, 127) + 127) << 23).view(torch.float32) for h in (half, n - half)]
    e = p * power[0] * power[1]
    e = torch.where(x > 88.5, torch.full_like(x, math.inf), e)
    return torch.where(x < -87.0, torch.zeros_like(x), e)


def _divide32(a, b):
    """Correctly rounded float32 quotient."""
    return (a.double() / b.double()).float()


def _sigmoid32(x):
    return _divide32(torch.ones_like(x), 1.0 + _exp32(-x))


def _first_largest(key, k):
    """Indices of the k largest of each row, largest first, the lower index first on ties."""
    return torch.sort(key, dim=1, descending=True, stable=True).indices[:, :k]


def _plain_select(logits, bias, case):
    t, n = logits.shape
    groups = case["groups"]
    sigmoid = case["routing"] == "sigmoid"
    value = _sigmoid32(logits) if sigmoid else logits
    key = value + bias if sigmoid else logits
    by_group = key.reshape(t, groups, n // groups)
    if sigmoid:
        best = torch.sort(by_group, dim=2, descending=True).values
        score = best[:, :, 0] + best[:, :, 1]
    else:
        score = by_group.amax(2)
    taken = torch.zeros((t, groups), dtype=torch.bool, device="cuda")
    taken.scatter_(1, _first_largest(score, case["top_groups"]), True)
    key = torch.where(taken.unsqueeze(2), by_group, torch.full_like(by_group, -math.inf)).reshape(t, n)
    idx = _first_largest(key, case["active"])
    picked = torch.gather(value, 1, idx)
    if not sigmoid:
        picked = _exp32(picked - picked[:, :1])
        return idx.int(), picked / picked.sum(1, keepdim=True)
    return idx.int(), picked / (picked.sum(1, keepdim=True) + 1e-9) * RSF


def _plain_route(s):
    kind, case = s["kind"], s["case"]
    if kind == "route":
        logits = (s["x"].double() @ s["router"].double()).float()
        return [logits, *_plain_select(logits, s["bias"], case)]
    idx, gates = _plain_select(s["logits"], s["bias"], case)
    if kind == "logits":
        return [idx, gates]
    dg = s["d_gates"]
    if case["routing"] == "softmax":
        dl = gates * (dg - (gates * dg).sum(1, keepdim=True))
    else:
        sg = _sigmoid32(torch.gather(s["logits"], 1, idx.long()))
        z = sg.sum(1, keepdim=True) + 1e-9
        dl = RSF * (dg / z - (dg * sg).sum(1, keepdim=True) / (z * z)) * sg * (1.0 - sg)
    return [idx, gates, torch.zeros_like(s["logits"]).scatter_(1, idx.long(), dl)]


def _weights(codes, scales):
    """float32 [N, rows, K] of a packed operand."""
    n, r, k = codes.shape[:3]
    rows = codes.reshape(n, r, k, 2, 32, 16).permute(0, 1, 4, 2, 3, 5).reshape(n, r * 32, k * 32)
    return rows.float() * scales.unsqueeze(2)


def _product(rows, plan, codes, scales):
    """rows [R, K] in the experts' order times each one's operand: the experts as a batch,
    each padded to the fullest one's rows."""
    live = plan["live"]
    if live.numel() < codes.shape[0]:
        codes, scales = codes[live], scales[live]
    w = _weights(codes, scales)
    batch = torch.zeros((w.shape[0], plan["most"], w.shape[2]), dtype=torch.float32, device="cuda")
    batch[plan["expert"], plan["within"]] = rows
    return torch.bmm(batch, w.transpose(1, 2).contiguous())[plan["expert"], plan["within"]]


def _plain_ffn(s):
    code, scale = _codes8(s["x"].float(), "int8")
    x = (code * scale.unsqueeze(1))[s["plan"]["perm_src"].long() // s["case"]["active"]]
    gu = _product(x, s["plan"], s["gate_up"], s["gate_up_scale"])
    g, u = gu.reshape(gu.shape[0], -1, 2, BLOCK).unbind(2)
    # h is a product's result of its own, and in bfloat16 as such
    h = (g / (1.0 + torch.exp(-g)) * u).reshape(gu.shape[0], -1).to(torch.bfloat16)
    code, scale = _codes8(h.float(), "int8")
    return _product(code * scale.unsqueeze(1), s["plan"], s["down"], s["down_scale"]).to(torch.bfloat16)


def _plain(s):
    if s["kind"] == "norm":
        return _plain_norm(s)
    if s["kind"] == "norm_bwd":
        return _plain_norm_bwd(s)
    return _plain_ffn(s) if s["kind"] == "ffn" else _plain_route(s)


# ------------------------------------------------------------ the framework --

def _own_route(s):
    from hanuman_amd import _lib
    from hanuman_amd import kernels as K
    kind, c = s["kind"], s["case"]
    sigmoid = c["routing"] == "sigmoid"
    mode = _lib.ROUTE_SIGMOID_BIAS if sigmoid else _lib.ROUTE_SOFTMAX
    rsf = RSF if sigmoid else 1.0
    limit = dict(n_groups=c["groups"], top_groups=c["top_groups"])
    if kind == "route":
        return list(K.router(s["x"], s["router"], s["bias"], c["active"], mode, rsf, **limit))
    idx, gates = K.router_from_logits(s["logits"], s["bias"], c["active"], mode, rsf, **limit)
    if kind == "logits":
        return [idx, gates]
    return [idx, gates, K.router_bwd(s["logits"], idx, gates, s["d_gates"], c["experts"], mode, rsf)]


def _own(s):
    from hanuman_amd import kernels as K
    kind, c = s["kind"], s["case"]
    if kind == "norm":
        r = K.add_rms_norm(s["x"], s["weight"], s["residual"], EPS, quant=c["quant"])
        read_back = K.dequantize_rows_i8 if c["quant"] == "int8" else K.dequantize_rows_fp8
        return [r.sum, r.y, r.rstd, read_back(r.q, r.scale, torch.bfloat16)]
    if kind == "norm_bwd":
        return list(K.add_rms_norm_bwd(s["dy"], s["sum"], s["weight"], s["rstd"], s["d_sum"]))
    if kind != "ffn":
        return _own_route(s)
    p = s["plan"]
    rows = c["tokens"] * c["active"]
    plan = K.Plan(p["counts"], p["offsets"], p["slot_pos"], p["perm_src"], p["keep"], rows, rows, c["experts"],
                  c["active"])
    x_q, x_scale = K.quantize_rows_i8(s["x"])
    h = K.grouped_gate_up_i8_gather(x_q, x_scale, plan, s["gate_up"], s["gate_up_scale"])
    h_q, h_scale = K.quantize_rows_i8(h, p["offsets"])
    return K.grouped_down_i8(h_q, h_scale, p["offsets"], s["down"], s["down_scale"])


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ------------------------------------------------------------ what is right --

def _exact_rows(v, to):
    """The values that 8-bit codes of float64 rows stand for."""
    amax = v.abs().amax(-1, keepdim=True)
    step = torch.where(amax > 0, amax / LARGEST[to], torch.ones_like(amax))
    m = v / step
    if to == "int8":
        return torch.round(m) * step
    octave = (torch.frexp(m.abs())[1] - 1).clamp(min=-6)    # floor(log2 |m|), subnormals below 2^-6
    unit = _power_of_two(octave - 3)
    return (torch.round(m / unit) * unit).clamp(-448.0, 448.0) * step


def _power_of_two(e):
    """2^e in float64, from its bits: a power function may be off in the last one."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _single(v):
    """float64 values to the nearest float32, in float64."""
    return v.float().double()


def _exact_exp32(x):
    """The float32 exponential's definition, each of its operations in float64 and rounded to
    float32 (which is that operation's float32 result: 53 bits are more than twice 24)."""
    def f(bits):
        fraction, exponent = bits & 0x7FFFFF, bits >> 23
        return math.ldexp(0x800000 + fraction, exponent - 150)
    n = torch.round(_single(x * f(0x3FB8AA3B)))
    r = _single(x - _single(n * f(0x3F317200)))
    r = _single(r - _single(n * f(0x35BFBE8E)))
    p = torch.full_like(x, f(0x39500D01))
    for c in (0x3AB60B61, 0x3C088889, 0x3D2AAAAB, 0x3E2AAAAB, 0x3F000000, 0x3F800000, 0x3F800000):
        p = _single(_single(p * r) + f(c))
    return _single(p * _power_of_two(n.clamp(-200, 200)))


def _exact_select(logits, bias, case):
    """(indices, gates): the selection on the keys that the definition gives, the gates from
    the true sigmoid or exponential."""
    t, n = logits.shape
    groups, sigmoid = case["groups"], case["routing"] == "sigmoid"
    key = logits
    if sigmoid:
        key = _single(1.0 / _single(1.0 + _exact_exp32(-logits)))
        key = _single(key + bias.double())
    members = key.reshape(t, groups, n // groups)
    top = members.topk(2, dim=2).values
    score = _single(top[:, :, 0] + top[:, :, 1]) if sigmoid else top[:, :, 0]
    # a group's rank: how many others are above it, or as high with a lower index
    lower = torch.ones((groups, groups), dtype=torch.bool, device="cuda").tril(-1)
    rank = ((score.unsqueeze(1) > score.unsqueeze(2)) | ((score.unsqueeze(1) == score.unsqueeze(2)) & lower)).sum(2)
    key = members.masked_fill((rank >= case["top_groups"]).unsqueeze(2), -math.inf).reshape(t, n)
    idx = torch.empty((t, case["active"]), dtype=torch.long, device="cuda")
    column = torch.arange(n, device="cuda")
    for k in range(case["active"]):
        first = torch.where(key == key.amax(1, keepdim=True), column, n).amin(1)
        idx[:, k] = first
        key = key.scatter(1, first.unsqueeze(1), -math.inf)
    picked = torch.gather(logits, 1, idx)
    if not sigmoid:
        return idx, torch.softmax(picked, 1)
    sg = torch.sigmoid(picked)
    return idx, sg / (sg.sum(1, keepdim=True) + 1e-9) * RSF


def _exact_route(s):
    kind, case = s["kind"], s["case"]
    if kind == "route":
        x, w = s["x"].double(), s["router"].double()
        logits = sum(x[:, d:d + 256] @ w[d:d + 256] for d in range(0, case["d_model"], 256))
        return [logits, *_exact_select(_single(logits), s["bias"], case)]
    logits = s["logits"].double()
    idx, gates = _exact_select(logits, s["bias"], case)
    if kind == "logits":
        return [idx, gates]
    picked = torch.gather(logits, 1, idx).requires_grad_(True)
    with torch.enable_grad():
        if case["routing"] == "softmax":
            again = torch.softmax(picked, 1)
        else:
            sg = torch.sigmoid(picked)
            again = sg / (sg.sum(1, keepdim=True) + 1e-9) * RSF
        d, = torch.autograd.grad(again, picked, s["d_gates"].double())
    return [idx, gates, torch.zeros_like(logits).scatter_(1, idx, d)]


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "norm":
        dtype = s["x"].dtype
        total = s["x"].double()
        if s["residual"] is not None:
            # the sum is a result of its own, and the norm is the rounded sum's
            total = total + s["residual"].double()
        v = total.to(dtype).double()
        rstd = (v.square().sum(1) / case["cols"] + EPS).pow(-0.5)
        y = s["weight"].double() * (v * rstd.unsqueeze(1))
        return [total, y, rstd, _exact_rows(y.to(dtype).double(), case["quant"])]
    if kind == "norm_bwd":
        # the gradient of the weighted sum of both outputs, as autograd takes it
        v = s["sum"].double().requires_grad_(True)
        w = s["weight"].double().requires_grad_(True)
        with torch.enable_grad():
            y = v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * w
            out = torch.autograd.grad((y, v * 1.0), (v, w), (s["dy"].double(), s["d_sum"].double()))
        return list(out)
    if kind != "ffn":
        return _exact_route(s)
    p = s["plan"]
    out = torch.empty((case["tokens"] * case["active"], case["d_model"]), dtype=torch.float64, device="cuda")
    x = _exact_rows(s["x"].double(), "int8")
    edges = p["offsets"].tolist()

    def weights(codes, scales):
        lanes = codes.reshape(codes.shape[0], -1, 2, 32, 16).transpose(1, 3).transpose(2, 3)
        return lanes.reshape(codes.shape[0] * 32, -1).double() * scales.double().unsqueeze(1)

    for e in range(case["experts"]):
        lo, hi = edges[e], edges[e + 1]
        if lo == hi:
            continue
        gu = x[p["perm_src"][lo:hi].long() // case["active"]] @ weights(s["gate_up"][e], s["gate_up_scale"][e]).t()
        gu = gu.reshape(hi - lo, -1, 2, BLOCK)
        h = (gu[:, :, 0] * torch.sigmoid(gu[:, :, 0]) * gu[:, :, 1]).reshape(hi - lo, -1)
        h = _exact_rows(h.to(torch.bfloat16).double(), "int8")
        out[lo:hi] = h @ weights(s["down"][e], s["down_scale"][e]).t()
    return out


def work(case):
    """Bytes and operations of one pass: inputs read once, outputs written once.  Only the
    experts with rows are read."""
    kind = case["kind"]
    if kind in ("norm", "norm_bwd"):
        values, size = case["rows"] * case["cols"], {"bf16": 2, "f32": 4}[case["dtype"]]
        if kind == "norm_bwd":
            return dict(bytes=values * 4 * size + 8 * case["cols"] + 4 * case["rows"], flops=10 * values)
        # the sum and the normed rows written; codes written, read and read back in bfloat16
        moved = size * (4 if case["residual"] else 2) + 1 + 1 + 2
        return dict(bytes=values * moved + 4 * case["cols"] + 8 * case["rows"], flops=6 * values)
    if kind == "ffn":
        d, f = case["d_model"], case["d_ff"]
        rows = case["tokens"] * case["active"]
        live = min(case["experts"], rows)
        return dict(bytes=case["tokens"] * d * 2 + live * (3 * d * f + (2 * f + d) * 4) + rows * d * 2,
                    flops=6 * rows * d * f)
    t, n, k = case["tokens"], case["experts"], case["active"]
    if kind == "route":
        d = case["d_model"]
        return dict(bytes=t * d * 2 + d * n * 4 + t * n * 4 + t * k * 8, flops=2 * t * d * n)
    # a training step's gradients of the logits, dense
    return dict(bytes=t * n * 4 + t * k * 8 + (t * n * 4 + t * k * 4 if kind == "route_train" else 0), flops=8 * t * n)

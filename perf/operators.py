"""Performance cases of the element-wise optimizer operators: the AdamW step over many tensors with 32-bit and with
8-bit states, the global gradient norm with clipping, and the block quantiser of the 8-bit states.

``run`` computes a case in plain torch operations, or, with ``own``, by the calls a user makes.  Every tensor of a
case is a view into one flat buffer per role (parameters, gradients, ...), each starting at a multiple of 256
elements, so that ``run`` can return whole roles as single tensors.
"""

import math

import torch


own = False

BLOCK = 256  # elements that share the exponent byte of an 8-bit state
BETAS, EPS, LR, WD = (0.9, 0.95), 1e-8, 3e-4, 0.1
_DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# sizes of the tensors of a set relative to one another: projections, key/value blocks, MLP matrices, biases, norms
_PATTERN = (16, 4, 56, 16, 1, 3, 2)


def listed():
    return [
        # one norm weight: nothing but the latency of the call
        {"name": "adamw32 one norm weight", "op": "adamw32", "tensors": 1, "numel": 4096, "p": "f32", "g": "f32",
         "remainder": False, "scaled": False, "method": "decoupled"},
        # all norm weights and biases of a model beside its Muon matrices: many small tensors, one launch's worth of work
        {"name": "adamw32 129 small tensors", "op": "adamw32", "tensors": 129, "numel": 600_001, "p": "f32", "g": "f32",
         "remainder": False, "scaled": True, "method": "decoupled"},
        # bf16 weights with the low half of their fp32 masters, two layers' worth of matrices
        {"name": "adamw32 bf16 + remainder", "op": "adamw32", "tensors": 14, "numel": 436_207_616, "p": "bf16",
         "g": "bf16", "remainder": True, "scaled": True, "method": "decoupled"},
        # embedding and output layer in fp32, the usual companions of Muon
        {"name": "adamw32 embedding and head", "op": "adamw32", "tensors": 2, "numel": 537_001_984, "p": "f32", "g": "f32",
         "remainder": False, "scaled": False, "method": "decoupled"},
        # a single odd bias with 8-bit states
        {"name": "adamw8 one odd bias", "op": "adamw8", "tensors": 1, "numel": 4097, "p": "f32", "g": "f32",
         "remainder": False, "scaled": False, "method": "decoupled"},
        # one layer of bf16 weights with remainders and 8-bit states: a large model on few GPUs
        {"name": "adamw8 bf16 layer", "op": "adamw8", "tensors": 7, "numel": 218_103_809, "p": "bf16", "g": "bf16",
         "remainder": True, "scaled": True, "method": "decoupled"},
        # the embedding in fp32 with 8-bit states
        {"name": "adamw8 embedding", "op": "adamw8", "tensors": 1, "numel": 268_435_456, "p": "f32", "g": "f32",
         "remainder": False, "scaled": False, "method": "decoupled"},
        # norm of the small parameters' gradients
        {"name": "norm 129 small tensors", "op": "norm", "tensors": 129, "numel": 600_001, "g": "f32"},
        # norm and clipping coefficient of two layers' bf16 gradients, read once
        {"name": "norm bf16 layers", "op": "norm", "tensors": 14, "numel": 436_207_616, "g": "bf16"},
        # fp32 gradients of one layer scaled in place
        {"name": "clip one layer in place", "op": "clip", "tensors": 7, "numel": 218_103_809, "g": "f32"},
        # a checkpointed state into 8 bits and back: a small odd one, and the embedding's
        {"name": "quantize odd bias", "op": "quantize", "tensors": 1, "numel": 14_337, "g": "f32", "signed": True},
        {"name": "quantize embedding", "op": "quantize", "tensors": 1, "numel": 268_435_456, "g": "f32", "signed": False},
    ]  # fmt: skip


def draw(rng):
    op = rng.choice(("adamw32", "adamw32", "adamw8", "adamw8", "norm", "clip", "quantize"))
    tensors = 1 if op == "quantize" else rng.choice((1, 2, 3, 7, 14, 40, 129, 200))
    numel = max(tensors, int(2 ** rng.uniform(0 if tensors == 1 else 8, 28)) + rng.randrange(7))
    case = {"op": op, "tensors": tensors, "numel": numel, "g": rng.choice(("f32", "bf16"))}
    if op == "quantize":
        case["signed"] = rng.choice((True, False))
    if op.startswith("adamw"):
        case["p"] = rng.choice(("f32", "bf16"))
        case["remainder"] = case["p"] == "bf16" and rng.choice((True, False))
        case["scaled"] = rng.choice((True, False))
        case["method"] = rng.choice(("decoupled", "independent", "l2", "palm"))
    return case


def _sizes(case):
    k, n = case["tensors"], case["numel"]
    weights = [_PATTERN[i % len(_PATTERN)] for i in range(k)]
    sizes = [max(1, n * w // sum(weights)) for w in weights]
    sizes[0] = max(1, sizes[0] + n - sum(sizes))
    return sizes


def work(case):
    n, g = sum(_sizes(case)), {"f32": 4, "bf16": 2}[case["g"]]
    if case["op"] == "norm":
        return {"bytes": n * g, "flops": 2 * n}
    if case["op"] == "clip":
        return {"bytes": 2 * n * g, "flops": 3 * n}  # read and written once
    if case["op"] == "quantize":
        return {"bytes": n * (g + 1 + 4) + 2 * n // BLOCK, "flops": 10 * n}  # values in, codes in between, fp32 out
    p = {"f32": 4, "bf16": 2}[case["p"]] + (2 if case["remainder"] else 0)
    if case["op"] == "adamw32":
        return {"bytes": n * (g + 2 * p + 16), "flops": 15 * n}
    # codes and exponents read and written, and the two states read back as bf16 values
    return {"bytes": n * (g + 2 * p + 4 + 4) + 4 * n // BLOCK, "flops": 40 * n}


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _views(flat, sizes, starts):
    return [flat[a : a + n] for a, n in zip(starts, sizes)]


def prepare(case, seed):
    dev = "cuda"
    gen = torch.Generator(device=dev).manual_seed(seed)
    sizes = _sizes(case)
    starts, total = [], 0
    for n in sizes:
        starts.append(total)
        total += (n + BLOCK - 1) // BLOCK * BLOCK
    keep = torch.zeros(total, dtype=torch.bool, device=dev)
    for a, n in zip(starts, sizes):
        keep[a : a + n] = True

    def rand():
        return torch.randn(total, generator=gen, device=dev)

    # every run of 64 elements has a scale of its own, and one run in eight has no gradient yet (rows nobody used)
    runs = (total + 63) // 64
    scale = 1e-3 * torch.exp(torch.randn(runs, generator=gen, device=dev))
    scale *= torch.rand(runs, generator=gen, device=dev) > 0.125
    scale = scale.repeat_interleave(64)[:total] * keep
    s = {"case": case, "sizes": sizes, "starts": starts}
    s["G"] = (rand() * scale).to(_DTYPES[case["g"]])
    s["grads"] = _views(s["G"], sizes, starts)
    if case["op"] in ("norm", "clip"):
        s["max_norm"] = 0.5 * float(torch.linalg.vector_norm(s["G"].double()))
        return s
    if case["op"] == "quantize":
        s["seed"] = seed % (1 << 31)
        x = s["G"].float()
        s["x"] = (x if case["signed"] else x * x).to(_DTYPES[case["g"]])[: sizes[0]].clone()
        return s
    p32 = rand() * 0.02 * keep
    s["P"] = p32.to(_DTYPES[case["p"]])
    s["params"] = _views(s["P"], sizes, starts)
    if case["remainder"]:
        bits = p32.view(torch.int32).long()
        hi = (bits + 0x8000) >> 16
        s["R"] = (bits - (hi << 16)).to(torch.int16)
        s["P"].copy_((hi << 16).to(torch.int32).view(torch.float32))
        s["remainders"] = _views(s["R"], sizes, starts)
    else:
        s["remainders"] = None
    m, v = rand() * scale * 0.3, scale * scale * (0.25 + rand().square())
    if case["op"] == "adamw32":
        s["M"], s["V"] = m, v
    else:
        for key, x, bits in (("M", m, 4), ("V", v, 5)):
            s[key], s[key + "e"] = _start_codes(x, bits)
            s[key + "es"] = _views(s[key + "e"], [(n + BLOCK - 1) // BLOCK for n in sizes], [a // BLOCK for a in starts])
        s["seed"] = seed % (1 << 31)
    s["Ms"], s["Vs"] = _views(s["M"], sizes, starts), _views(s["V"], sizes, starts)
    s["scale"] = torch.full((), 0.75, device=dev) if case["scaled"] else None
    s["step"] = 1000
    return s


def _start_codes(x, exponent_bits):
    """Codes to the nearest of the given values, as the state of an earlier step would hold them."""
    k = {4: 113, 5: 97}[exponent_bits]
    field = (x.abs().view(-1, BLOCK).amax(1).view(torch.int32) >> 23).clamp(min=1)
    y = x.abs().view(-1, BLOCK) * ((254 - field) << 23).view(torch.float32)[:, None] * 2.0**-k
    code = ((y.view(torch.int32) + 0x80000) >> 20).view(-1)
    code = torch.where(x < 0, code + 128, code) if exponent_bits == 4 else torch.where(x > 0, code.clamp(min=1), code)
    return code.to(torch.uint8), field.to(torch.uint8)


# ---- plain forms ----------------------------------------------------------------------------------------------------


def _factors(method, step):
    decay = {"decoupled": 1 - LR * WD, "independent": 1 - WD, "palm": 1 - LR * LR * WD, "l2": 1.0}[method]
    return decay, (WD if method == "l2" else 0.0), LR / (1 - BETAS[0] ** step), 1 / math.sqrt(1 - BETAS[1] ** step)


def _adam(p, g, m, v, scale, method, step):
    """One step on fp32 values, every operation rounded once: the new (p, m, v)."""
    decay, l2, size, inv = _factors(method, step)
    if scale is not None:
        g = g * scale
    if l2:
        g = g + p * l2
    p = p * decay
    m = m * BETAS[0] + g * (1 - BETAS[0])
    v = v * BETAS[1] + (g * g) * (1 - BETAS[1])
    return p - (m / (v.sqrt() * inv + EPS)) * size, m, v


def _adam_lists(ps, gs, ms, vs, scale, method, step):
    """The same over lists of tensors; m and v change in place, the new fp32 parameters are returned."""
    decay, l2, size, inv = _factors(method, step)
    if scale is not None:
        gs = torch._foreach_mul(gs, scale)
    if l2:
        gs = torch._foreach_add(gs, torch._foreach_mul(ps, l2))
    ps = torch._foreach_mul(ps, decay)
    torch._foreach_mul_(ms, BETAS[0])
    torch._foreach_add_(ms, torch._foreach_mul(gs, 1 - BETAS[0]))
    torch._foreach_mul_(vs, BETAS[1])
    squares = torch._foreach_mul(gs, gs)
    torch._foreach_mul_(squares, 1 - BETAS[1])
    torch._foreach_add_(vs, squares)
    denom = torch._foreach_sqrt(vs)
    torch._foreach_mul_(denom, inv)
    torch._foreach_add_(denom, EPS)
    update = torch._foreach_div(ms, denom)
    torch._foreach_mul_(update, size)
    return torch._foreach_sub(ps, update)


def _join(p, r):
    return ((p.view(torch.int16).to(torch.int32) << 16) + r.to(torch.int32)).view(torch.float32)


def _split_into(p, r, x):
    bits = x.view(torch.int32)
    hi = (bits + 0x8000) >> 16
    r.copy_(bits - (hi << 16))
    p.view(torch.int16).copy_(hi)


def _mix(x):
    """A mixer of 32-bit integers (the finaliser of MurmurHash3), on non-negative int64 values."""
    x = ((x ^ (x >> 16)) * 0x85EBCA6B) & 0xFFFFFFFF
    x = ((x ^ (x >> 13)) * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _noise(s, step):
    """The 32 random bits of every element: from the seed, the tensor's place in the list, the step and the element."""
    first = torch.zeros(s["G"].numel(), dtype=torch.int64, device=s["G"].device)
    first[torch.tensor(s["starts"], device=first.device)] = 1
    tensor = first.cumsum(0) - 1
    index = torch.arange(first.numel(), device=first.device) - torch.tensor(s["starts"], device=first.device)[tensor]
    key = _mix(_mix(_mix(torch.full_like(tensor, s["seed"])) ^ tensor) ^ step)
    return _mix(key ^ (index & 0xFFFFFFFF))


def _decode(code, field, exponent_bits):
    k = {4: 113, 5: 97}[exponent_bits]
    c = code.to(torch.int32)
    mag = (c & 0x7F) if exponent_bits == 4 else c
    x = (mag << 20).view(torch.float32).view(-1, BLOCK) * 2.0**k * (field.to(torch.int32) << 23).view(torch.float32)[:, None]
    x = x.view(-1)
    return torch.where(c >= 128, -x, x) if exponent_bits == 4 else x


def _encode(x, bits16, exponent_bits):
    k = {4: 113, 5: 97}[exponent_bits]
    mag = x.abs().view(-1, BLOCK)
    field = (mag.amax(1).view(torch.int32) >> 23).clamp(min=1)
    y = mag * ((254 - field) << 23).view(torch.float32)[:, None] * 2.0**-k
    code = ((y.view(torch.int32) + ((bits16.to(torch.int32) << 4) + 8).view(-1, BLOCK)) >> 20).view(-1)
    code = torch.where(x < 0, code + 128, code) if exponent_bits == 4 else torch.where(x > 0, code.clamp(min=1), code)
    return code.to(torch.uint8), field.to(torch.uint8)


def _coefficient(norm, max_norm):
    return (max_norm / (norm + 1e-6)).clamp(max=1.0)


def run(s):
    case, op = s["case"], s["case"]["op"]
    if op in ("norm", "clip"):
        return _run_norm(s, op == "clip")
    if op == "quantize":
        return _run_quantize(s)
    s["step"] += 1
    return _run_adamw32(s) if op == "adamw32" else _run_adamw8(s)


def _run_norm(s, in_place):
    if in_place:
        s["max_norm"] *= 0.999  # below the norm that the previous pass left: every pass scales
    if own:
        from emerging_optimizers_b200.utils import clip_coefficient, clip_grads_

        if in_place:
            return {"norm": clip_grads_(s["grads"], s["max_norm"]), "g": s["G"]}
        norm, coef = clip_coefficient(s["grads"], s["max_norm"])
        return {"norm": norm, "coef": coef}
    x = s["G"].double()
    norm = (x * x).sum().sqrt().float()
    coef = _coefficient(norm, s["max_norm"])
    if in_place:
        s["G"].copy_(s["G"].float() * coef)
        return {"norm": norm, "g": s["G"]}
    return {"norm": norm, "coef": coef}


def _run_quantize(s):
    signed = s["case"]["signed"]
    if own:
        from emerging_optimizers_b200.scalar_optimizers import dequantize_blockwise, quantize_blockwise

        codes, exponents = quantize_blockwise(s["x"], signed=signed, seed=s["seed"])
        return dequantize_blockwise(codes, exponents, signed=signed, dtype=torch.bfloat16)
    n = s["x"].numel()
    x = torch.nn.functional.pad(s["x"].float(), (0, -n % BLOCK))
    key = _mix(_mix(_mix(torch.full((1,), s["seed"], device=x.device)) ^ 0) ^ 0)
    bits = _mix(key ^ (torch.arange(x.numel(), device=x.device) & 0xFFFFFFFF))
    bits = (bits & 0xFFFF) if signed else (bits >> 16)
    kind = 4 if signed else 5
    codes, exponents = _encode(x, bits, kind)
    return _decode(codes, exponents, kind)[:n].to(torch.bfloat16)


def _run_adamw32(s):
    case = s["case"]
    if own:
        from emerging_optimizers_b200.scalar_optimizers import adamw_step

        adamw_step(s["params"], s["grads"], s["Ms"], s["Vs"], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, step=s["step"],
                   weight_decay_method=case["method"], grad_scale=s["scale"], remainders=s["remainders"])  # fmt: skip
    elif case["remainder"]:
        p, s["M"][:], s["V"][:] = _adam(_join(s["P"], s["R"]), s["G"].float(), s["M"], s["V"], s["scale"], case["method"], s["step"])
        _split_into(s["P"], s["R"], p)
    elif case["p"] == "f32" and case["g"] == "f32":
        new = _adam_lists(s["params"], s["grads"], s["Ms"], s["Vs"], s["scale"], case["method"], s["step"])
        torch._foreach_copy_(s["params"], new)
    else:
        wide = [p.float() for p in s["params"]], [g.float() for g in s["grads"]]
        new = _adam_lists(*wide, s["Ms"], s["Vs"], s["scale"], case["method"], s["step"])
        torch._foreach_copy_(s["params"], new)
    out = {"p": s["P"], "m": s["M"], "v": s["V"]}
    return {**out, "remainder": s["R"]} if case["remainder"] else out


def _run_adamw8(s):
    case = s["case"]
    if own:
        from emerging_optimizers_b200.scalar_optimizers import adamw_step_8bit, dequantize_blockwise

        adamw_step_8bit(s["params"], s["grads"], s["Ms"], s["Mes"], s["Vs"], s["Ves"], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD,
                        step=s["step"], seed=s["seed"], weight_decay_method=case["method"], grad_scale=s["scale"],
                        remainders=s["remainders"])  # fmt: skip
        m = dequantize_blockwise(s["M"], s["Me"], signed=True, dtype=torch.bfloat16)
        v = dequantize_blockwise(s["V"], s["Ve"], signed=False, dtype=torch.bfloat16)
    else:
        p = _join(s["P"], s["R"]) if case["remainder"] else s["P"].float()
        m, v = _decode(s["M"], s["Me"], 4), _decode(s["V"], s["Ve"], 5)
        p, m, v = _adam(p, s["G"].float(), m, v, s["scale"], case["method"], s["step"])
        bits = _noise(s, s["step"])
        s["M"][:], s["Me"][:] = _encode(m, bits & 0xFFFF, 4)
        s["V"][:], s["Ve"][:] = _encode(v, bits >> 16, 5)
        if case["remainder"]:
            _split_into(s["P"], s["R"], p)
        else:
            s["P"].copy_(p)
        m, v = _decode(s["M"], s["Me"], 4).to(torch.bfloat16), _decode(s["V"], s["Ve"], 5).to(torch.bfloat16)
    # the states are given as the values that their codes stand for (four significant bits: exact in bf16)
    out = {"p": s["P"], "m": m, "v": v}
    return {**out, "remainder": s["R"]} if case["remainder"] else out


# ---- 64-bit definitions ---------------------------------------------------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    g = s["x" if case["op"] == "quantize" else "G"].double()
    if case["op"] in ("norm", "clip"):
        norm = float(torch.sqrt(torch.sum(g**2)))
        limit = s["max_norm"] * (0.999 if case["op"] == "clip" else 1.0)
        coef = min(1.0, limit / (norm + 1e-6))
        return {"norm": norm, "g": g * coef} if case["op"] == "clip" else {"norm": norm, "coef": coef}
    if case["op"] == "quantize":
        pad = torch.cat([g, g.new_zeros(-g.numel() % BLOCK)])
        return _exact_rounded(pad, _exact_random(s, [pad.numel()], 0, case["signed"]), case["signed"])[: g.numel()]
    t = s["step"] + 1
    p = s["P"].double()
    if case["remainder"]:
        # the fp32 master lies `remainder` units in its last place beyond the bf16 value, counted on the bit patterns
        p = (s["P"].float().view(torch.int32) + s["R"].to(torch.int32)).view(torch.float32).double()
    if case["op"] == "adamw32":
        m, v = s["M"].double(), s["V"].double()
    else:
        m, v = _exact_values(s["M"], s["Me"], True), _exact_values(s["V"], s["Ve"], False)
    if s["scale"] is not None:
        g = g * 0.75
    if case["method"] == "l2":
        g = g + WD * p
    shrink = {"decoupled": LR * WD, "independent": WD, "palm": LR**2 * WD, "l2": 0.0}[case["method"]]
    m += (1 - BETAS[0]) * (g - m)
    v += (1 - BETAS[1]) * (g**2 - v)
    p -= shrink * p
    p -= LR * (m / (1 - BETAS[0] ** t)) / (torch.sqrt(v / (1 - BETAS[1] ** t)) + EPS)
    if case["op"] == "adamw8":
        spans = [b - a for a, b in zip(s["starts"], s["starts"][1:] + [g.numel()])]
        m = _exact_rounded(m, _exact_random(s, spans, t, True), True)
        v = _exact_rounded(v, _exact_random(s, spans, t, False), False)
    return {"p": p, "m": m, "v": v, "remainder": None}


def _exact_values(code, field, signed):
    """What a code stands for: 1.mmm * 2^(e - top), or 0.mmm at the lowest e, times the block's power of two."""
    c = code.double()
    sign = torch.where(c >= 128, -1.0, 1.0) if signed else 1.0
    if signed:
        c = torch.remainder(c, 128)
    e, mant = torch.floor(c / 8), torch.remainder(c, 8)
    top = 14 if signed else 30
    value = torch.where(e > 0, (1 + mant / 8) * torch.exp2(e - top), mant / 8 * 2.0 ** (1 - top))
    return sign * value * torch.exp2(field.double() - 127).repeat_interleave(BLOCK)


def _exact_random(s, spans, step, signed):
    """Uniform numbers (r + 1/2) / 65536 with r from the mixer of (seed, tensor, step, element)."""

    def mixer(x):
        for shift, factor in ((16, 0x85EBCA6B), (13, 0xC2B2AE35)):
            x = x ^ (x >> shift)
            x = (x * factor) % (1 << 32)
        return x ^ (x >> 16)

    dev, parts = s["G"].device, []
    for i, n in enumerate(spans):
        key = mixer(mixer(mixer(s["seed"]) ^ i) ^ step)
        r = mixer(torch.arange(n, device=dev) % (1 << 32) ^ key)
        parts.append(r % 65536 if signed else r // 65536)
    return (torch.cat(parts).double() + 0.5) / 65536


def _power_below(x):
    """The largest power of two that is at most x."""
    return torch.exp2(torch.frexp(x).exponent.double() - 1)


def _exact_rounded(x, u, signed):
    """Stochastic rounding to four significant bits within the exponent range below the block's power of two."""
    mag = x.abs()
    scale = _power_below(mag.view(-1, BLOCK).amax(1).clamp(min=2.0**-126)).repeat_interleave(BLOCK)
    t = mag / scale
    lowest = -13 if signed else -29
    grid = _power_below(t.clamp(min=2.0**lowest)) / 8
    q = torch.floor(t / grid + u) * grid
    if not signed:
        q = torch.where(t > 0, q.clamp(min=2.0 ** (lowest - 3)), q)
    return torch.where(x < 0, -q, q) * scale

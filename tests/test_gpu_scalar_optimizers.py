"""AdamW with 32- and 8-bit moments, gradient norm and clipping, and the block quantiser on the GPU, against their
float64 statements."""

import os

import numpy as np
import pytest
import torch

from emerging_optimizers_b200 import build as eo_build
from emerging_optimizers_b200 import utils
from emerging_optimizers_b200.orthogonalized_optimizers import Muon
from emerging_optimizers_b200.scalar_optimizers import (
    AdamW,
    adamw_step,
    adamw_step_8bit,
    dequantize_blockwise,
    quantize_blockwise,
)
from tests import _scalar_ref as ref


pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
ULP = 2.0**-24  # one fp32 rounding, relative
SIZES = [1, 255, 256, 257, 0, 2048, 2049, 12345]
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
REF = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, wd=0.1)


@pytest.fixture(scope="module", autouse=True)
def host_module():
    if not os.path.exists(eo_build.HOST_OUT):
        eo_build.build_host()


def _randn(n, seed, scale=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(n) * scale).astype(np.float32)).cuda()


def _np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _inputs(sizes, p_dtype=F32, g_dtype=F32, seed=0):
    ps = [_randn(n, seed + 4 * i, 0.02).to(p_dtype) for i, n in enumerate(sizes)]
    gs = [_randn(n, seed + 4 * i + 1, 1e-3).to(g_dtype) for i, n in enumerate(sizes)]
    ms = [_randn(n, seed + 4 * i + 2, 3e-4) for i, n in enumerate(sizes)]
    vs = [_randn(n, seed + 4 * i + 3, 1e-3).square() for i, n in enumerate(sizes)]
    for i, n in enumerate(sizes):  # some elements nobody touched
        gs[i][n // 2 : n // 2 + n // 8], ms[i][n // 2 : n // 2 + n // 8], vs[i][n // 2 : n // 2 + n // 8] = 0, 0, 0
    return ps, gs, ms, vs


def _clone(lists):
    return [[t.clone() for t in ts] for ts in lists]


def _quantized(ts, signed):
    pairs = [quantize_blockwise(t, signed=signed) for t in ts]
    return [c for c, _ in pairs], [e for _, e in pairs]


def _bits(t):
    return t.view(torch.int16 if t.dtype == BF16 else torch.int32 if t.dtype == F32 else t.dtype)


def _same(a, b):
    """The same bits, NaN included."""
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(_bits(a), _bits(b))


# ---- AdamW, 32-bit moments ------------------------------------------------------------------------------------------


@pytest.mark.parametrize("method", ["decoupled", "independent", "palm", "l2"])
@pytest.mark.parametrize("p_dtype,g_dtype", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("scaled", [False, True])
def test_adamw_step_against_float64(method, p_dtype, g_dtype, scaled):
    ps, gs, ms, vs = _inputs(SIZES, p_dtype, g_dtype)
    before = _clone((ps, gs, ms, vs))
    scale = torch.tensor(0.37, device="cuda") if scaled else None
    adamw_step(ps, gs, ms, vs, **HYPER, step=7, weight_decay_method=method, grad_scale=scale)
    for p, g, m, v, p0, g0, m0, v0 in zip(ps, gs, ms, vs, *before):
        (p64, m64, v64), (pm, mm, vm) = ref.adamw(
            _np64(p0), _np64(g0), _np64(m0), _np64(v0), **REF, step=7, method=method, scale=float(scale) if scaled else 1.0
        )
        assert torch.equal(g, g0)
        # m: up to four roundings of each term and of beta, one of the sum; v: three more; p adds the root (half of v's),
        # the factors and the quotient.  The bf16 parameter is rounded once more, by at most 2^-8.
        assert np.all(np.abs(_np64(m) - m64) <= 8 * ULP * mm)
        assert np.all(np.abs(_np64(v) - v64) <= 12 * ULP * vm)
        last = 2.0**-8 * np.abs(p64) if p_dtype == BF16 else 0.0
        assert np.all(np.abs(_np64(p) - p64) <= (16 * ULP * pm) * (1 + 2.0**-8) + last)


@pytest.mark.parametrize("method", ["decoupled", "l2"])
@pytest.mark.parametrize("steps", [(1, 2, 3), (1000, 100000)])
def test_adamw_step_gives_the_bits_of_single_operations(method, steps):
    """Parameters and moments are bit for bit what torch's elementary fp32 operations leave, each rounded once: no
    contraction, the root and the quotient to nearest.  2^23 elements: about every mantissa under the root."""
    (p,), (g,), (m,), (v,) = _inputs([1 << 23])
    m *= torch.exp(4 * _randn(1 << 23, 91))
    v *= torch.exp(8 * _randn(1 << 23, 92))
    p0, m0, v0 = p.clone(), m.clone(), v.clone()
    lr, (b1, b2), eps, wd = HYPER["lr"], HYPER["betas"], HYPER["eps"], HYPER["weight_decay"]
    for step in steps:
        scale = torch.tensor(0.7, device="cuda")
        adamw_step([p], [g], [m], [v], **HYPER, step=step, weight_decay_method=method, grad_scale=scale)
        x = g * scale
        if method == "l2":
            x = x + p0 * wd
        p0 = p0 * ref.decay_factor(method, lr, wd)
        m0 = m0 * b1 + x * (1 - b1)
        v0 = v0 * b2 + (x * x) * (1 - b2)
        p0 = p0 - (m0 / (v0.sqrt() * (1 / (1 - b2**step) ** 0.5) + eps)) * (lr / (1 - b1**step))
        assert _same(m, m0) and _same(v, v0) and _same(p, p0)


@pytest.mark.parametrize("off", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 3, 0), (0, 0, 0, 5), (1, 2, 3, 4)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_adamw_step_at_any_alignment_gives_the_same_bits(off, dtype):
    n = 5000
    (p,), (g,), (m,), (v,) = _inputs([n], dtype, dtype)
    moved = []
    for t, o in zip((p, g, m, v), off):
        room = torch.full((n + 16,), 9.0, dtype=t.dtype, device="cuda")
        room[o : o + n] = t
        moved.append((room, room[o : o + n], o))
    adamw_step([p], [g], [m], [v], **HYPER, step=3)
    adamw_step(*[[view] for _, view, _ in moved], **HYPER, step=3)
    for t, (room, view, o) in zip((p, g, m, v), moved):
        assert _same(t, view)
        assert bool((room[:o] == 9).all()) and bool((room[o + n :] == 9).all())  # nothing beside it was written


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("size,eps", [(1e18, 1e-8), (1e12, 1e-8), (1e-15, 1e-8), (1e-15, 0.0), (1e-18, 1e-30), (3e-21, 0.0)])
def test_gradients_of_any_size(size, eps, bits):
    """First steps on gradients whose squares reach the ends of the fp32 range: against float64 from the moments that the
    fp32 step leaves (their own rounding, of subnormal numbers among them, is not in question here)."""
    n = 2000
    g = _randn(n, 3, size)
    p = torch.zeros(n, device="cuda")
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), eps=eps, weight_decay=0.0)
    adamw_step([p], [g], [m], [v], **hyper, step=1)
    if bits == 8:
        q = torch.zeros(n, device="cuda")
        state = [[torch.zeros(k, dtype=torch.uint8, device="cuda")] for k in (n, 8, n, 8)]
        adamw_step_8bit([q], [g], *state, **hyper, step=1, seed=0)
        assert _same(q, p)
    m64, v64 = _np64(m), _np64(v)
    some = (v64 > 0) & np.isfinite(v64)
    assert some.mean() > 0.5
    want = -(1e-2 / (1 - 0.9)) * m64[some] / (np.sqrt(v64[some] / (1 - 0.95)) + eps)
    # the root, three products, a sum, the quotient, two factors: at most ten roundings; 3e-7 (five roundings) for a root below
    # 2^-102, and the rounding of a parameter that may itself be subnormal
    assert np.all(np.abs(_np64(p)[some] - want) <= 15 * ULP * np.abs(want) + 2.0**-149)


def test_adamw_first_step_and_empty_lists():
    p, g = _randn(300, 1), _randn(300, 2)
    m, v = torch.zeros_like(p), torch.zeros_like(p)
    (want, _, _), (mag, _, _) = ref.adamw(_np64(p), _np64(g), 0 * _np64(p), 0 * _np64(p), **REF, step=1)
    adamw_step([p], [g], [m], [v], **HYPER, step=1)
    assert np.all(np.abs(_np64(p) - want) <= 16 * ULP * mag)
    empty = torch.empty(0, device="cuda")
    adamw_step([empty], [empty], [empty], [empty], **HYPER, step=1)


@pytest.mark.parametrize("count", [24, 25, 384, 385, 800])
def test_adamw_step_over_many_tensors_equals_one_by_one(count):
    sizes = [1 + (37 * i) % 700 for i in range(count)]
    lists = _inputs(sizes)
    alone = _clone(lists)
    adamw_step(*lists, **HYPER, step=2)
    for k in range(count):
        adamw_step(*[[ts[k]] for ts in alone], **HYPER, step=2)
    for a, b in zip(lists, alone):
        assert all(_same(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("bits", [32, 8])
def test_remainders_hold_the_fp32_master(bits):
    """bf16 weights with remainders take the path of fp32 weights, bit for bit, over several steps."""
    sizes = [1, 300, 4096]
    ps, gs, ms, vs = _inputs(sizes, F32, F32)
    wide = [p.bfloat16().float() for p in ps]
    narrow = [p.bfloat16() for p in ps]
    rs = [torch.zeros_like(p, dtype=torch.int16) for p in narrow]
    (m_codes, me), (v_codes, ve) = _quantized(ms, True), _quantized(vs, False)
    for params, rem in ((wide, None), (narrow, rs)):
        if bits == 32:
            state = [[t.clone() for t in ts] for ts in (ms, vs)]
        else:
            state = [[t.clone() for t in ts] for ts in (m_codes, me, v_codes, ve)]
        for step in range(1, 6):
            if bits == 32:
                adamw_step(params, gs, *state, **HYPER, step=step, remainders=rem)
            else:
                adamw_step_8bit(params, gs, *state, **HYPER, step=step, seed=4, remainders=rem)
    for p, r, w in zip(narrow, rs, wide):
        joined = ref.join(p.view(torch.int16).cpu().numpy(), r.cpu().numpy())
        assert np.array_equal(joined, w.cpu().numpy())
        # and the bf16 part is the nearest to it
        assert np.all(np.abs(_np64(p) - joined.astype(np.float64)) <= 2.0**-8 * np.abs(joined))
    assert any(bool((r != 0).any()) for r in rs)


def test_remainders_of_special_values():
    p = torch.tensor([float("inf"), -float("inf"), float("nan"), 0.0, -0.0, 3.38e38], device="cuda").bfloat16()
    r = torch.zeros_like(p, dtype=torch.int16)
    z = torch.zeros(6, device="cuda")
    adamw_step([p], [z], [z.clone()], [z.clone()], **{**HYPER, "weight_decay": 0.0}, step=1, remainders=[r])
    out = p.float().cpu()
    assert out[0] == float("inf") and out[1] == -float("inf") and torch.isnan(out[2])
    assert out[3] == 0 and out[4] == 0 and torch.isfinite(out[5])
    assert bool((r == 0).all())


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [5, 2048])
def test_weights_set_to_zero_with_stale_remainders(bits, n):
    """A mask or a padding row zeroes bf16 weights and leaves their remainders: they count as zeros (a remainder that is not
    negative as the subnormal number that it stands for)."""
    (p,), (g,), (m,), (v,) = _inputs([n], BF16, BF16)
    r = torch.arange(n, device="cuda").sub(n // 2).to(torch.int16)
    p[::2] = torch.where(torch.arange(0, n, 2, device="cuda") % 4 == 0, 0.0, -0.0).bfloat16()
    fresh, r_fresh = p.clone(), r.clone()
    r_fresh[(p == 0) & (r < 0)] = 0
    for q, rem in ((p, r), (fresh, r_fresh)):
        if bits == 32:
            adamw_step([q], [g], [m.clone()], [v.clone()], **HYPER, step=3, remainders=[rem])
        else:
            state = [[t] for t in (*quantize_blockwise(m, signed=True), *quantize_blockwise(v, signed=False))]
            adamw_step_8bit([q], [g], *state, **HYPER, step=3, seed=1, remainders=[rem])
    assert bool(torch.isfinite(p).all()) and _same(p, fresh) and torch.equal(r, r_fresh)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite_stay_where_they_are(bits):
    n = 1000
    (p,), (g,), (m,), (v,) = _inputs([n])
    g2 = g.clone()
    bad = [0, 255, 256, 700]
    g2[bad[0]], g2[bad[1]], g2[bad[2]], g2[bad[3]] = float("nan"), float("inf"), -float("inf"), 2e19  # squared: infinite
    outs = []
    for grad in (g, g2):
        q = p.clone()
        if bits == 32:
            mm, vv = m.clone(), v.clone()
            adamw_step([q], [grad], [mm], [vv], **HYPER, step=5)
        else:
            (mc,), (me,) = _quantized([m], True)
            (vc,), (ve,) = _quantized([v], False)
            adamw_step_8bit([q], [grad], [mc], [me], [vc], [ve], **HYPER, step=5, seed=1)
            mm, vv = dequantize_blockwise(mc, me, signed=True), dequantize_blockwise(vc, ve, signed=False)
        outs.append((q, mm, vv))
    clean = torch.ones(n, dtype=torch.bool, device="cuda")
    clean[bad] = False
    (q0, m0, v0), (q1, m1, v1) = outs
    assert _same(q0[clean], q1[clean]) and _same(v0[clean], v1[clean])
    assert bool(torch.isfinite(m1[clean]).all())
    if bits == 32:
        assert _same(m0[clean], m1[clean])
    else:  # 2e19 is finite in m: it sets its block's exponent, and what is 2^-17 smaller rounds to zero
        same = clean.clone()
        same[512:768] = False
        assert _same(m0[same], m1[same])
    assert bool(torch.isnan(m1[0])) and not bool(torch.isfinite(m1[255])) and not bool(torch.isfinite(m1[256]))
    assert not bool(torch.isfinite(v1[bad]).any())


# ---- 8-bit moments ----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("p_dtype,g_dtype", [(F32, F32), (F32, BF16), (BF16, F32), (BF16, BF16)])
@pytest.mark.parametrize("method", ["decoupled", "l2"])
def test_adamw_8bit_is_the_32bit_step_between_decoding_and_rounding(p_dtype, g_dtype, method):
    """Parameters: the bits of the fp32 step on the decoded moments.  New codes: the float64 statement of the rounding
    applied to that step's moments, code for code."""
    ps, gs, ms, vs = _inputs(SIZES, p_dtype, g_dtype)
    (mc, me), (vc, ve) = _quantized(ms, True), _quantized(vs, False)
    m32 = [dequantize_blockwise(c, e, signed=True) for c, e in zip(mc, me)]
    v32 = [dequantize_blockwise(c, e, signed=False) for c, e in zip(vc, ve)]
    p32 = [p.clone() for p in ps]
    scale = torch.tensor(0.5, device="cuda")
    adamw_step(p32, gs, m32, v32, **HYPER, step=11, weight_decay_method=method, grad_scale=scale)
    adamw_step_8bit(ps, gs, mc, me, vc, ve, **HYPER, step=11, seed=77, weight_decay_method=method, grad_scale=scale)
    for i, n in enumerate(SIZES):
        assert _same(ps[i], p32[i])
        if n == 0:
            continue
        for codes, exponents, wide, signed in ((mc[i], me[i], m32[i], True), (vc[i], ve[i], v32[i], False)):
            want, want_e = ref.quantize(wide.cpu().numpy(), signed, ref.random_bits(n, 77, i, 11, signed))
            assert np.array_equal(exponents.cpu().numpy(), want_e)
            assert np.array_equal(codes.cpu().numpy(), want)


@pytest.mark.parametrize("n", [3001, 70_000])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("off,off_codes", [(1, 1), (4, 4), (4, 0), (8, 8), (0, 1)])
def test_adamw_8bit_at_any_alignment_gives_the_same_bits(off, off_codes, dtype, n):
    (p,), (g,), (m,), (v,) = _inputs([n], dtype, dtype)
    (mc,), (me,) = _quantized([m], True)
    (vc,), (ve,) = _quantized([v], False)
    moved = []
    for t in (p, g, mc, me, vc, ve):
        o = off_codes if t.dtype == torch.uint8 else off
        room = torch.full((t.numel() + 16,), 9, dtype=t.dtype, device="cuda")
        room[o : o + t.numel()] = t
        moved.append((room, room[o : o + t.numel()], o))
    adamw_step_8bit([p], [g], [mc], [me], [vc], [ve], **HYPER, step=3, seed=2)
    adamw_step_8bit(*[[view] for _, view, _ in moved], **HYPER, step=3, seed=2)
    for t, (room, view, o) in zip((p, g, mc, me, vc, ve), moved):
        assert _same(t, view)
        assert bool((room[:o] == 9).all()) and bool((room[o + t.numel() :] == 9).all())


def test_random_bits_depend_on_seed_step_and_place():
    n = 4096
    lists = _inputs([n, n])
    for k in (0, 2, 3):  # the same tensor twice
        lists[k][1].copy_(lists[k][0])
    lists[1][1].copy_(lists[1][0])

    def run(step, seed):
        (mc, me), (vc, ve) = _quantized(lists[2], True), _quantized(lists[3], False)
        adamw_step_8bit([p.clone() for p in lists[0]], lists[1], mc, me, vc, ve, **HYPER, step=step, seed=seed)
        return mc + vc

    base = run(1000, 5)
    assert all(_same(a, b) for a, b in zip(base, run(1000, 5)))
    for other in (run(1001, 5), run(1000, 6), [base[1], base[0], base[3], base[2]]):
        assert all(0.05 < float((a != b).float().mean()) for a, b in zip(base, other))


@pytest.mark.parametrize("beta2", [0.95, 0.999])
def test_8bit_moments_follow_gradients_that_shrink(beta2):
    """After gradients fall tenfold the 8-bit second moments fall with the fp32 ones.  Rounded to nearest they would stand
    still.  One step moves a moment by a random part of at most (1 - beta2) + one unit (1/8), so their mean over n
    independent elements is off by less than a hundredth; 5 % is allowed."""
    n, steps = 1 << 16, int(5 / (1 - beta2))
    p = torch.zeros(n, device="cuda")
    (mc, vc), (me, ve) = [[torch.zeros(k, dtype=torch.uint8, device="cuda") for _ in range(2)] for k in (n, n // 256)]
    m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    hyper = {**HYPER, "betas": (0.9, beta2), "weight_decay": 0.0}
    for phase in range(2):
        for t in range(steps):
            g = torch.randn(n, generator=gen, device="cuda") * (1e-3 if phase == 0 else 1e-4)
            adamw_step([p], [g], [m], [v], **hyper, step=phase * steps + t + 1)
            adamw_step_8bit([p], [g], [mc], [me], [vc], [ve], **hyper, step=phase * steps + t + 1, seed=1)
        got = dequantize_blockwise(vc, ve, signed=False).double().mean()
        assert abs(float(got / v.double().mean()) - 1) < 0.05


def test_offsets_past_32_bits():
    """A tensor of more than 2^32 elements: its last ones are updated as a tensor of their own is, and rounded by the bits
    of their own place."""
    n, tail = (1 << 32) + 777, 777 + 256
    p = torch.zeros(n, dtype=BF16, device="cuda")
    g = torch.zeros(n, dtype=BF16, device="cuda")
    mc, vc = torch.zeros(n, dtype=torch.uint8, device="cuda"), torch.zeros(n, dtype=torch.uint8, device="cuda")
    me = torch.zeros(-(-n // 256), dtype=torch.uint8, device="cuda")
    ve = torch.zeros_like(me)
    p_tail, g_tail = _randn(tail, 1, 0.02).bfloat16(), _randn(tail, 2, 1e-3).bfloat16()
    p[-tail:], g[-tail:] = p_tail, g_tail
    m, v = torch.zeros(tail, device="cuda"), torch.zeros(tail, device="cuda")
    adamw_step([p_tail], [g_tail], [m], [v], **HYPER, step=1)
    norm = utils.global_grad_norm([g])
    assert abs(float(norm) / float(torch.linalg.vector_norm(g_tail.double())) - 1) <= 2 * ULP
    adamw_step_8bit([p], [g], [mc], [me], [vc], [ve], **HYPER, step=1, seed=3)
    assert _same(p[-tail:], p_tail)
    for codes, exponents, wide, signed in ((mc, me, m, True), (vc, ve, v, False)):
        want, want_e = ref.quantize(wide.cpu().numpy(), signed, ref.random_bits(tail, 3, 0, 1, signed, first=n - tail))
        assert np.array_equal(codes[-tail:].cpu().numpy(), want)
        assert np.array_equal(exponents[-len(want_e) :].cpu().numpy(), want_e)
        assert not bool(codes[: 1 << 20].any())


# ---- quantiser --------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 255, 256, 257, 8192, 10001])
@pytest.mark.parametrize("seed", [None, 12345])
def test_quantizer_gives_the_codes_of_its_statement(signed, dtype, n, seed):
    x = _randn(n, n) * torch.exp(3 * _randn(n, n + 1))
    x = (x if signed else x * x).to(dtype)
    codes, exponents = quantize_blockwise(x, signed=signed, seed=seed)
    bits = None if seed is None else ref.random_bits(n, seed, 0, 0, signed)
    want, want_e = ref.quantize(x.float().cpu().numpy(), signed, bits)
    assert np.array_equal(codes.cpu().numpy(), want) and np.array_equal(exponents.cpu().numpy(), want_e)
    for out in (F32, BF16):
        y = dequantize_blockwise(codes, exponents, signed=signed, dtype=out)
        assert y.dtype == out and np.array_equal(_np64(y), ref.dequantize(want, want_e, signed))


@pytest.mark.parametrize("signed", [True, False])
@pytest.mark.parametrize("seed", [None, 7])
def test_quantizer_at_every_block_exponent(signed, seed):
    """One block for every power of two of the fp32 range, values down to 2^-35 of it."""
    rng = np.random.default_rng(5)
    rows = [np.ldexp(rng.uniform(1, 2, 256) * np.ldexp(1.0, -rng.integers(0, 36, 256)), e) for e in range(-130, 128)]
    x = np.concatenate(rows).astype(np.float32)
    x = np.where(rng.random(x.size) < 0.5, -x, x) if signed else x
    codes, exponents = quantize_blockwise(torch.from_numpy(x).cuda(), signed=signed, seed=seed)
    bits = None if seed is None else ref.random_bits(x.size, seed, 0, 0, signed)
    want, want_e = ref.quantize(x, signed, bits)
    assert np.array_equal(exponents.cpu().numpy(), want_e)
    assert np.array_equal(codes.cpu().numpy(), want)
    y = dequantize_blockwise(codes, exponents, signed=signed)
    assert np.array_equal(_np64(y), ref.dequantize(want, want_e, signed).astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("signed", [True, False])
def test_quantizer_at_the_ends_of_the_fp32_range(signed):
    tiny, huge = 2.0**-126, 3.4e38
    rows = [
        [0.0] * 256,
        [huge] + [1.0] * 255,
        [tiny] * 256,
        [2.0**-140] * 256,  # subnormal: below the lowest block power, yet not zero (unsigned)
        [float("nan"), float("inf"), -float("inf")] + [1.0] * 253,
        [float("nan")] * 256,
        [1.0, 1e-30] + [1.99] * 254,
        [-1.0, -0.0, 0.5] + [0.25] * 253,
    ]
    x = torch.tensor(rows, dtype=F32).reshape(-1)
    codes, exponents = quantize_blockwise(x.cuda(), signed=signed)
    y = dequantize_blockwise(codes, exponents, signed=signed).cpu().reshape(len(rows), 256)
    assert bool((y[0] == 0).all())
    assert abs(float(y[1, 0]) / huge - 1) <= 1 / 16 and (float(y[1, 1]) > 0) != signed
    assert bool((y[2] == tiny).all())
    if signed:
        assert bool((y[3] == 2.0**-140).all())  # 2^-14 of the lowest block power, 2^-126
    else:
        assert bool((y[3] == 2.0**-140).all())
    assert torch.isnan(y[4, 0]) and torch.isnan(y[4, 1]) and torch.isnan(y[4, 2]) and bool((y[4, 3:] == 1).all())
    assert bool(torch.isnan(y[5]).all())
    assert (float(y[6, 1]) > 0) != signed  # an unsigned value above zero stays above zero
    if signed:
        assert float(y[7, 0]) == -1 and float(y[7, 1]) == 0
    else:
        assert torch.isnan(y[7, 0]) and float(y[7, 1]) == 0 and float(y[7, 2]) == 0.5
    empty_codes, empty_exponents = quantize_blockwise(torch.empty(0, device="cuda"), signed=signed)
    assert empty_codes.numel() == 0 and empty_exponents.numel() == 0
    assert dequantize_blockwise(empty_codes, empty_exponents, signed=signed).numel() == 0


# ---- norm and clipping ------------------------------------------------------------------------------------------------


def _norm64(gs):
    return float(np.sqrt(sum((_np64(g) ** 2).sum() for g in gs)))


@pytest.mark.parametrize("count", [1, 5, 24, 25, 400])
@pytest.mark.parametrize("mix", ["fp32", "bf16", "both"])
def test_clipping_against_float64(count, mix):
    sizes = [(1 + 997 * i) % 5000 for i in range(count)]
    gs = [_randn(n, i, 0.1).to(BF16 if mix == "bf16" or (mix == "both" and i % 2) else F32) for i, n in enumerate(sizes)]
    norm = _norm64(gs)
    before = [g.clone() for g in gs]
    assert abs(float(utils.global_grad_norm(gs)) - norm) <= 2 * ULP * norm
    got, coef = utils.clip_coefficient(gs, 0.5 * norm)
    want = 0.5 * norm / (norm + 1e-6)
    assert abs(float(got) - norm) <= 2 * ULP * norm and abs(float(coef) - want) <= 6 * ULP * want
    assert all(_same(a, b) for a, b in zip(gs, before))
    again = utils.clip_grads_(gs, 0.5 * norm)
    assert _same(again, got)  # the same sums in the same order
    for a, b in zip(gs, before):
        want_g = _np64(b) * want
        # the coefficient is at most 6 roundings off, the product one; bf16 results are rounded by 2^-8 at most
        assert np.all(np.abs(_np64(a) - want_g) <= (8 * ULP + (2.0**-8 * 1.01 if a.dtype == BF16 else 0)) * np.abs(want_g))
    kept = [g.clone() for g in gs]
    utils.clip_grads_(gs, 10 * norm)  # nothing to clip
    assert all(_same(a, b) for a, b in zip(gs, kept))


def test_norm_of_values_whose_squares_leave_fp32():
    for scale in (1e-30, 1e25):
        g = _randn(10000, 3, scale)
        assert abs(float(utils.global_grad_norm([g])) / _norm64([g]) - 1) <= 2 * ULP
    assert float(utils.global_grad_norm([torch.empty(0, device="cuda")])) == 0.0
    norm, coef = utils.clip_coefficient([torch.zeros(5, device="cuda")], 1.0)
    assert float(norm) == 0.0 and float(coef) == 1.0


def test_norms_that_are_not_finite():
    g = torch.ones(300, device="cuda")
    p = torch.nn.Parameter(torch.zeros(300, device="cuda"))
    p.grad = g
    g[7] = float("inf")
    assert float(utils.global_grad_norm([g])) == float("inf")
    with pytest.raises(RuntimeError, match="not finite"):
        utils.clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert bool((g[:7] == 1).all())  # nothing was scaled
    g[8] = float("nan")
    norm, coef = utils.clip_coefficient([g], 1.0)
    assert torch.isnan(norm) and torch.isnan(coef)
    utils.clip_grad_norm_([p], 1.0)
    assert bool(torch.isnan(g).all())


def test_clip_grad_norm_matches_torch():
    params = [torch.nn.Parameter(torch.zeros(n, device="cuda")) for n in (10, 1000, 33, 4)]
    other = [torch.nn.Parameter(torch.zeros_like(p)) for p in params]
    for i, (p, q) in enumerate(zip(params[:3], other)):
        p.grad, q.grad = _randn(p.numel(), i), _randn(p.numel(), i)
    a, b = utils.clip_grad_norm_(params, 1.0), torch.nn.utils.clip_grad_norm_(other, 1.0)
    assert abs(float(a) / float(b) - 1) <= 1e-6  # torch sums in fp32: 1043 terms, pairwise
    for p, q in zip(params[:3], other):
        assert torch.allclose(p.grad, q.grad, rtol=2e-6, atol=0)
    assert params[3].grad is None


# ---- the optimizer ------------------------------------------------------------------------------------------------------


def _model_params(dtype=F32):
    shapes = [(50, 16), (16,), (7, 3, 5), (33,)]
    return [torch.nn.Parameter(_randn(int(np.prod(s)), i, 0.02).reshape(s).to(dtype)) for i, s in enumerate(shapes)]


def _set_grads(params, step, dtype=None):
    for i, p in enumerate(params):
        p.grad = _randn(p.numel(), 100 * step + i, 1e-3).reshape(p.shape).to(p.dtype)


def test_optimizer_matches_torch_adamw():
    a, b = _model_params(), _model_params()
    ours, theirs = [
        cls([{"params": x[:2], "lr": 1e-2}, {"params": x[2:], "weight_decay": 0.0}], lr=3e-3, betas=(0.9, 0.99), weight_decay=0.1)
        for cls, x in ((AdamW, a), (torch.optim.AdamW, b))
    ]  # fmt: skip
    schedules = [torch.optim.lr_scheduler.ExponentialLR(o, 0.9) for o in (ours, theirs)]
    for step in range(6):
        _set_grads(a, step)
        _set_grads(b, step)
        if step == 2:  # a parameter without a gradient keeps its state and its own count
            a[1].grad = b[1].grad = None
        ours.step()
        theirs.step()
        for s in schedules:
            s.step()
    for p, q in zip(a, b):
        # an update is at most lr (0.01) times a few; both sides are within some 20 roundings of the exact one
        assert torch.allclose(p, q, rtol=0, atol=6 * 1e-2 * 3 * 20 * ULP + 6 * 2 * ULP * float(q.detach().abs().max()))
        assert ours.state[p]["step"] == int(theirs.state[q]["step"])
    c = _model_params()
    third = AdamW([{"params": c[:2]}, {"params": c[2:]}])
    third.load_state_dict(theirs.state_dict())  # a checkpoint of torch's class
    assert third.state[c[1]]["step"] == 5 and torch.equal(third.state[c[0]]["exp_avg"], theirs.state[b[0]]["exp_avg"])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_checkpoint_resumes_bit_for_bit(bits, dtype):
    kw = dict(lr=1e-2, state_bits=bits, master_remainder=True, seed=9)
    a = _model_params(dtype)
    whole = AdamW(a, **kw)
    for step in range(4):
        if step == 2:
            b = [torch.nn.Parameter(p.detach().clone()) for p in a]
            saved = whole.state_dict()
            for i, state in saved["state"].items():  # as it comes back from a file
                saved["state"][i] = {k: v.cpu() if torch.is_tensor(v) else v for k, v in state.items()}
            rest = AdamW(b, **kw)
            rest.load_state_dict(saved)
        for params, opt in ((a, whole),) + (((b, rest),) if step >= 2 else ()):
            _set_grads(params, step)
            opt.step()
    for p, q in zip(a, b):
        assert _same(p.detach(), q.detach())
        for key, value in whole.state[p].items():
            other = rest.state[q][key]
            assert _same(value, other) if torch.is_tensor(value) else value == other


@pytest.mark.parametrize("source,target", [(True, False), (False, True)])
def test_checkpoint_between_host_and_device_counters(source, target):
    a = _model_params()
    first = AdamW(a, lr=1e-2, capturable=source)
    for step in range(3):
        _set_grads(a, step)
        first.step()
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    second = AdamW(b, lr=1e-2, capturable=target)
    second.load_state_dict(first.state_dict())
    for params, opt in ((a, first), (b, second)):
        _set_grads(params, 9)
        opt.step()
    for p, q in zip(a, b):
        assert int(first.state[p]["step"]) == int(second.state[q]["step"]) == 4
        for x, y in zip(first.moments(p), second.moments(q)):
            assert _same(x, y)
        # the factors may differ in their last place (see the test of device counters)
        assert torch.allclose(p.detach(), q.detach(), rtol=4 * ULP, atol=4 * 3 * ULP * 1e-2)


def test_checkpoints_move_between_widths():
    a = _model_params(BF16)
    wide = AdamW(a, lr=1e-2, master_remainder=True)
    _set_grads(a, 0)
    wide.step()
    narrow = AdamW([torch.nn.Parameter(p.detach().clone()) for p in a], state_bits=8)
    narrow.load_state_dict(wide.state_dict())
    back = AdamW([torch.nn.Parameter(p.detach().clone()) for p in a])
    back.load_state_dict(narrow.state_dict())
    for p, q, r in zip(a, narrow.param_groups[0]["params"], back.param_groups[0]["params"]):
        assert narrow.state[q]["step"] == 1 and "remainder" not in narrow.state[q]
        for name, signed, moment in (("exp_avg", True, 0), ("exp_avg_sq", False, 1)):
            x = wide.state[p][name]
            codes, exponents = ref.quantize(x.cpu().numpy().reshape(-1), signed)
            want = ref.dequantize(codes, exponents, signed).reshape(x.shape)
            assert np.array_equal(_np64(narrow.moments(q)[moment]), want)
            assert back.state[r][name].dtype == F32 and np.array_equal(_np64(back.state[r][name]), want)


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_in_other_memory_orders(bits):
    """A transposed and a channels-last parameter, gradients in their order and in another one."""
    base, conv = _randn(48 * 20, 1, 0.02).reshape(48, 20), _randn(4 * 6 * 5 * 5, 2, 0.02).reshape(4, 6, 5, 5)
    laid = [torch.nn.Parameter(base.t()), torch.nn.Parameter(conv.to(memory_format=torch.channels_last))]
    # the same elements in memory order, as contiguous parameters
    flat = [torch.nn.Parameter(base.clone()), torch.nn.Parameter(conv.permute(0, 2, 3, 1).contiguous())]
    assert not laid[0].is_contiguous() and not laid[1].is_contiguous()
    opts = [AdamW(laid, lr=1e-2, state_bits=bits), AdamW(flat, lr=1e-2, state_bits=bits)]
    for step in range(3):
        for p in laid:
            p.grad = torch.empty_like(p).copy_(_randn(p.numel(), 10 * step + p.dim(), 1e-3).reshape(p.shape))
            if step == 1:
                p.grad = p.grad.contiguous()
        flat[0].grad = laid[0].grad.t().contiguous()
        flat[1].grad = laid[1].grad.permute(0, 2, 3, 1).contiguous()
        for o in opts:
            o.step()
    assert torch.equal(laid[0].t(), flat[0]) and torch.equal(laid[1].permute(0, 2, 3, 1), flat[1])
    for k in range(2):
        assert torch.equal(opts[0].moments(laid[0])[k].t(), opts[1].moments(flat[0])[k])
    again = AdamW([torch.nn.Parameter(p.detach().contiguous()) for p in laid], state_bits=bits)
    again.load_state_dict(opts[0].state_dict())  # into contiguous parameters
    assert again.moments(again.param_groups[0]["params"][0])[0].shape == laid[0].shape
    gap = torch.nn.Parameter(torch.zeros(6, 8, device="cuda")[:, :4])
    gap.grad = torch.zeros(6, 4, device="cuda")
    with pytest.raises(ValueError, match="dense"):
        AdamW([gap]).step()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_captured_step_replays_as_eager_steps(bits, dtype):
    kw = dict(betas=(0.9, 0.99), weight_decay=0.1, state_bits=bits, capturable=True, seed=3)
    a, b = _model_params(dtype), _model_params(dtype)
    lrs = [torch.tensor(1e-2, device="cuda") for _ in range(2)]
    eager, graphed = AdamW(a, lr=lrs[0], **kw), AdamW(b, lr=lrs[1], **kw)
    _set_grads(a, 0)
    _set_grads(b, 0)
    scale = torch.tensor(1.0, device="cuda")
    eager.step(grad_scale=scale)
    graphed.step(grad_scale=scale)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        utils.clip_grads_([p.grad for p in b], 1.0)
        graphed.step(grad_scale=scale)
    for step in range(1, 5):
        lr = 1e-2 / (step + 1)
        for params, opt in ((a, eager), (b, graphed)):
            for i, p in enumerate(params):
                p.grad.copy_(_randn(p.numel(), 100 * step + i, 1e-1).reshape(p.shape))
        for t in lrs:
            t.fill_(lr)
        scale.fill_(1.0 / step)
        utils.clip_grads_([p.grad for p in a], 1.0)
        eager.step(grad_scale=scale)
        graph.replay()
        for p, q in zip(a, b):
            assert _same(p.detach(), q.detach())
            assert int(eager.state[p]["step"]) == int(graphed.state[q]["step"]) == step + 1
            for x, y in zip(eager.moments(p), graphed.moments(q)):
                assert _same(x, y)


def test_device_counters_give_the_bits_of_host_counters():
    """The factors are computed in float64 on either side; the two pow functions agree to far below one fp32 rounding, so
    at most one unit in the last place of the two factors, hence of the update, can differ."""
    lists = _inputs([3000])
    other = _clone(lists)
    for step in (1, 2, 1000, 100000):
        adamw_step(*lists, **HYPER, step=step)
        adamw_step(*other, **{**HYPER, "lr": HYPER["lr"]}, step=torch.tensor(step, device="cuda"))
        assert _same(lists[2][0], other[2][0]) and _same(lists[3][0], other[3][0])
        assert torch.allclose(lists[0][0], other[0][0], rtol=4 * ULP, atol=4 * 3 * ULP * HYPER["lr"])


def test_capture_refuses_what_it_would_freeze():
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    p.grad = torch.ones(8, device="cuda")
    fresh, counted = AdamW([p], capturable=True), AdamW([p])
    counted.step()
    torch.cuda.synchronize()
    graph, x = torch.cuda.CUDAGraph(), torch.zeros(4, device="cuda")
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="run a step before"):
            fresh.step()
        with pytest.raises(RuntimeError, match="frozen"):
            counted.step()
        with pytest.raises(RuntimeError, match="frozen"):
            adamw_step([x], [x.clone()], [x.clone()], [x.clone()], lr=1e-3, step=1)
    assert counted.state[p]["step"] == 1


def test_other_streams():
    """Work on a side stream, ordered by events, gives the bits of the current stream."""
    lists = _inputs([100_000])
    other = _clone(lists)
    adamw_step(*lists, **HYPER, step=4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        norm = utils.global_grad_norm(other[1])
        adamw_step(*other, **HYPER, step=4)
    torch.cuda.current_stream().wait_stream(side)
    assert all(_same(a[0], b[0]) for a, b in zip(lists, other))
    assert _same(norm, utils.global_grad_norm(lists[1]))


def test_two_captured_graphs_replayed_at_once():
    """Two graphs of different parameters share no workspace: replayed on two streams they give what they give alone."""
    def build():
        lists = _inputs([300_000, 77])
        grads = lists[1]
        step = torch.ones((), dtype=torch.int64, device="cuda")
        def body():
            norm, coef = utils.clip_coefficient(grads, 1e-2)
            adamw_step(*lists, **HYPER, step=step, grad_scale=coef)
            return norm
        return lists, body

    want, body = build()
    norm = body()
    torch.cuda.synchronize()
    sides = []
    for _ in range(2):
        lists, body = build()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = body()
        sides.append((lists, graph, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _, graph, _, stream in sides:
        with torch.cuda.stream(stream):
            graph.replay()
    torch.cuda.synchronize()
    for lists, _, out, _ in sides:
        assert _same(out, norm)
        assert all(_same(x, y) for k in (0, 2, 3) for x, y in zip(lists[k], want[k]))


def test_many_calls_queued_without_waiting():
    """Workspaces of one call are handed to the next by the allocator while the first still runs."""
    gs = [[_randn(1 << 20, i, 0.1 * (i + 1))] for i in range(8)]
    want = [_norm64(g) for g in gs]
    norms = [utils.global_grad_norm(gs[i % 8]) for i in range(200)]
    for i, n in enumerate(norms):
        assert abs(float(n) - want[i % 8]) <= 2 * ULP * want[i % 8]


def test_zero_dimensional_and_empty_parameters():
    values = (torch.tensor(2.0, device="cuda"), torch.empty(0, 3, device="cuda"), torch.ones(1, 1, device="cuda"))
    params = [torch.nn.Parameter(t) for t in values]
    for bits in (32, 8):
        opt = AdamW(params, lr=0.1, weight_decay=0.0, state_bits=bits)
        for p in params:
            p.grad = torch.ones_like(p)
        before = [p.detach().clone() for p in params]
        opt.step()
        for p, b in zip(params, before):  # the first step moves by lr, whatever the gradient's size
            assert torch.allclose(p.detach(), b - 0.1, rtol=0, atol=1e-6)
        opt.load_state_dict(opt.state_dict())
        assert utils.clip_grad_norm_(params, 1e-3) is not None


def test_unknown_states_are_refused():
    p = torch.nn.Parameter(torch.ones(4, device="cuda"))
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    with pytest.raises(ValueError, match="no state"):
        opt.moments(p)
    assert p not in opt.state
    for key in ("amsgrad", "maximize"):
        other = torch.optim.AdamW([p], **{key: True})
        other.step()
        with pytest.raises(ValueError, match=key):
            opt.load_state_dict(other.state_dict())
    wrong = torch.nn.Parameter(torch.ones(5, device="cuda"))
    wrong.grad = torch.ones_like(wrong)
    third = AdamW([wrong])
    third.step()
    with pytest.raises(ValueError, match="does not fit"):
        opt.load_state_dict(third.state_dict())


def test_autograd_sees_the_step():
    p = torch.nn.Parameter(_randn(10, 1))
    loss = (p * p).sum()  # saves p
    p.grad = torch.ones_like(p)
    AdamW([p]).step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_refusals_on_the_gpu():
    x = torch.zeros(8, device="cuda")
    y = [torch.zeros(8, device="cuda") for _ in range(3)]
    u8 = [torch.zeros(8, dtype=torch.uint8, device="cuda") for _ in range(2)]
    e8 = [torch.zeros(1, dtype=torch.uint8, device="cuda") for _ in range(2)]
    kw = dict(lr=1e-3, step=1)
    with pytest.raises(ValueError, match="elements"):
        adamw_step([x], [x[:4].clone()], [y[0]], [y[1]], **kw)
    with pytest.raises(ValueError, match="tensors where"):
        adamw_step([x], [y[2]], [], [y[1]], **kw)
    with pytest.raises(TypeError, match="exp_avgs"):
        adamw_step([x], [y[2]], [y[0].half()], [y[1]], **kw)
    with pytest.raises(TypeError, match="params"):
        adamw_step([x.double()], [y[2]], [y[0]], [y[1]], **kw)
    with pytest.raises(ValueError, match="contiguous"):
        adamw_step([torch.zeros(8, 2, device="cuda")[:, 0]], [y[2]], [y[0]], [y[1]], **kw)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([x, x], [y[2], y[2]], [y[0], y[1]], [y[0].clone(), y[1].clone()], **kw)
    with pytest.raises(ValueError, match="twice"):
        adamw_step([x], [y[2]], [y[0]], [y[0]], **kw)
    with pytest.raises(ValueError, match="twice"):
        utils.clip_grads_([x, x], 1.0)
    with pytest.raises(ValueError, match="step"):
        adamw_step([x], [y[2]], [y[0]], [y[1]], lr=1e-3, step=0)
    with pytest.raises(TypeError, match="step"):
        adamw_step([x], [y[2]], [y[0]], [y[1]], lr=1e-3, step=torch.ones((), device="cuda"))
    with pytest.raises(TypeError, match="grad_scale"):
        adamw_step([x], [y[2]], [y[0]], [y[1]], **kw, grad_scale=torch.ones(()))
    with pytest.raises(TypeError, match="grad_scale"):
        adamw_step([x], [y[2]], [y[0]], [y[1]], **kw, grad_scale=0.5)
    with pytest.raises(TypeError, match="bf16"):
        adamw_step([x], [y[2]], [y[0]], [y[1]], **kw, remainders=[torch.zeros(8, dtype=torch.int16, device="cuda")])
    with pytest.raises(ValueError, match="exponents"):
        adamw_step_8bit([x], [y[2]], [u8[0]], [e8[0][:0]], [u8[1]], [e8[1]], **kw, seed=0)
    with pytest.raises(ValueError, match="seed"):
        adamw_step_8bit([x], [y[2]], [u8[0]], [e8[0]], [u8[1]], [e8[1]], **kw, seed=-1)
    with pytest.raises(ValueError, match="seed"):
        quantize_blockwise(x, signed=True, seed=1 << 32)
    with pytest.raises(TypeError):
        quantize_blockwise(x.half(), signed=True)
    with pytest.raises(TypeError):
        dequantize_blockwise(u8[0], e8[0], signed=True, dtype=torch.float16)
    with pytest.raises(ValueError, match="exponents"):
        dequantize_blockwise(u8[0], u8[1], signed=True)
    z = torch.zeros(4, 8, device="cuda")
    with pytest.raises(TypeError, match="list of tensors"):
        adamw_step(z, z.clone(), z.clone(), z.clone(), **kw)
    with pytest.raises(TypeError, match="list of tensors"):
        adamw_step([z], z.clone(), [z.clone()], [z.clone()], **kw)
    with pytest.raises(TypeError, match="list of tensors"):
        utils.clip_grads_(z, 1.0)
    with pytest.raises(TypeError, match="not a tensor"):
        adamw_step([x], [None], [y[0]], [y[1]], **kw)
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.zeros(8, device="cuda")
    opt = AdamW([p], capturable=True)
    opt.step()
    with pytest.raises(TypeError, match="grad_scale"):
        opt.step(grad_scale=2.0)
    assert int(opt.state[p]["step"]) == 1  # a step that was refused does not count
    for t in [x, *y, z]:
        assert not bool(t.any())  # no call wrote anything


def test_muon_and_adamw_train_one_model_together():
    """Matrices by Muon, the rest by AdamW with 8-bit moments, one global norm over both: the calls a training loop makes."""
    torch.manual_seed(0)
    layers = torch.nn.Embedding(100, 64), torch.nn.Linear(64, 128), torch.nn.LayerNorm(128), torch.nn.Linear(128, 100)
    model = torch.nn.Sequential(*layers).cuda()
    hidden = [model[1].weight]
    rest = [p for p in model.parameters() if p is not hidden[0]]
    muon = Muon(hidden, lr=0.01)
    adamw = AdamW(rest, lr=1e-2, state_bits=8)
    tokens = torch.randint(0, 100, (32,), device="cuda")
    for step in range(3):
        muon.zero_grad()
        adamw.zero_grad()
        torch.nn.functional.cross_entropy(model(tokens), tokens).backward()
        grads = [p.grad.clone() for p in model.parameters()]
        want = _norm64(grads)
        norm, coef = utils.clip_coefficient([p.grad for p in model.parameters()], 0.1)
        assert abs(float(norm) - want) <= 2 * ULP * want
        utils.clip_grads_([p.grad for p in hidden], float("inf"))  # nothing to clip: left as it is
        before = [p.detach().clone() for p in rest]
        moments = [adamw.moments(p) if adamw.state[p] else (torch.zeros_like(p), torch.zeros_like(p)) for p in rest]
        muon.step()
        adamw.step(grad_scale=coef)
        for p, p0, (m0, v0) in zip(rest, before, moments):
            (p64, _, _), (mag, _, _) = ref.adamw(
                _np64(p0), _np64(p.grad), _np64(m0), _np64(v0), lr=1e-2, betas=(0.9, 0.95), eps=1e-8, wd=0.01, step=step + 1,
                scale=float(coef),
            )  # fmt: skip
            assert np.all(np.abs(_np64(p) - p64) <= 16 * ULP * mag)
    assert all(bool(torch.isfinite(p).all()) for p in model.parameters())

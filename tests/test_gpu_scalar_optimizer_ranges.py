"""AdamW, clipping and the block quantiser on the GPU at the ends of their ranges: second moments that overflow, lists made on
the way, long chunks, unusual layouts and checkpoints that hooks look at."""

import copy
import os
import struct

import numpy as np
import pytest
import torch

from emerging_optimizers_b200 import _native
from emerging_optimizers_b200 import build as eo_build
from emerging_optimizers_b200 import utils
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
HYPER = dict(lr=3e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)


@pytest.fixture(scope="module", autouse=True)
def host_module():
    if not os.path.exists(eo_build.HOST_OUT):
        eo_build.build_host()


def _randn(n, seed, scale=1.0):
    return torch.from_numpy((np.random.default_rng(seed).standard_normal(n) * scale).astype(np.float32)).cuda()


def _np64(t):
    return t.detach().cpu().to(torch.float64).numpy()


def _same(a, b):
    """The same bits, NaN included."""
    width = {1: torch.uint8, 2: torch.int16, 4: torch.int32, 8: torch.int64}[a.element_size()]
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(a.view(width), b.view(width))


# ---- second moments that overflow ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("eps", [1e-8, 1e-10, 1e-15, 1e-30, 0.0])
@pytest.mark.parametrize("method", ["decoupled", "l2"])
def test_second_moments_up_to_infinity(eps, method):
    """Gradients from 1e-14 to 3e38, in any mix within a lane: over several steps the bits of torch's elementary fp32 operations,
    for which the quotient by an infinite root is zero.  (0.05 g^2 of the smallest is 2^-98: a root that is rounded to nearest.)"""
    n = 100_003
    rng = np.random.default_rng(1)
    lr, (b1, b2), wd = HYPER["lr"], HYPER["betas"], HYPER["weight_decay"]
    p, m, v = _randn(n, 2, 0.02), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    p0, m0, v0 = p.clone(), m.clone(), v.clone()
    exponent = rng.uniform(-14, 38.4, n)
    exponent[: n // 2] = rng.uniform(-8, 8, n // 2)  # whole runs without an overflow beside those that have some
    for step in (1, 2, 1000):
        g = rng.choice([-1.0, 1.0], n) * 10.0 ** np.clip(exponent + rng.uniform(-1, 1, n), -14, 38.5)
        g = torch.from_numpy(g.astype(np.float32)).cuda()
        adamw_step([p], [g], [m], [v], **{**HYPER, "eps": eps}, step=step, weight_decay_method=method)
        x = g + p0 * wd if method == "l2" else g
        p0 = p0 * ref.decay_factor(method, lr, wd)
        m0 = m0 * b1 + x * (1 - b1)
        v0 = v0 * b2 + (x * x) * (1 - b2)
        p0 = p0 - (m0 / (v0.sqrt() * (1 / (1 - b2**step) ** 0.5) + eps)) * (lr / (1 - b1**step))
        assert _same(m, m0) and _same(v, v0) and _same(p, p0)
    assert bool(torch.isinf(v).any()) and bool((v > 2.0**92).logical_and(torch.isfinite(v)).any())


@pytest.mark.parametrize("kind", ["8-bit", "remainders", "8-bit remainders", "bf16"])
@pytest.mark.parametrize("eps", [1e-8, 1e-15])
def test_every_form_takes_an_overflowing_second_moment_alike(kind, eps):
    """First steps of the other forms: the bits of the fp32 step above (bf16 weights: rounded), and the codes of its moments.
    Blocks that hold a large first or second moment, or one that is not finite, lie beside blocks that do not."""
    n = 5001
    exponent = np.random.default_rng(4).uniform(-14, 37, n)
    exponent[: n // 2] = np.minimum(exponent[: n // 2], np.repeat([3, 4, 5, 6, 7], 500))  # squares around 2^30
    g = _randn(n, 3) * torch.from_numpy(10.0**exponent).float().cuda()
    start = _randn(n, 5, 0.02).bfloat16().float()
    hyper = {**HYPER, "eps": eps}
    want, m, v = start.clone(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    adamw_step([want], [g], [m], [v], **hyper, step=1)
    p = start.clone() if kind == "8-bit" else start.bfloat16()
    r = [torch.zeros(n, dtype=torch.int16, device="cuda")] if "remainders" in kind else None
    if "8-bit" in kind:
        state = [[torch.zeros(k, dtype=torch.uint8, device="cuda")] for k in (n, -(-n // 256), n, -(-n // 256))]
        adamw_step_8bit([p], [g], *state, **hyper, step=1, seed=0, remainders=r)
        for ((codes,), (exponents,)), wide, signed in ((state[:2], m, True), (state[2:], v, False)):
            want_c, want_e = ref.quantize(wide.cpu().numpy(), signed, ref.random_bits(n, 0, 0, 1, signed))
            assert np.array_equal(codes.cpu().numpy(), want_c) and np.array_equal(exponents.cpu().numpy(), want_e)
    else:
        adamw_step([p], [g], *[[torch.zeros(n, device="cuda")] for _ in range(2)], **hyper, step=1, remainders=r)
    if r is not None:
        p = torch.from_numpy(ref.join(p.view(torch.int16).cpu().numpy(), r[0].cpu().numpy())).cuda()
    assert _same(p, want.bfloat16() if kind == "bf16" else want)


@pytest.mark.parametrize("size,eps", [(1e15, 1e-15), (1e17, 1e-15), (1e18, 0.0), (1e18, 1e-8)])
def test_steps_by_large_second_moments_against_float64(size, eps):
    """Second moments beyond 2^92 that fp32 still holds, with any eps: the first step is about lr."""
    n = 2000
    g = _randn(n, 6, size)
    p, m, v = (torch.zeros(n, device="cuda") for _ in range(3))
    adamw_step([p], [g], [m], [v], lr=1e-2, betas=(0.9, 0.95), eps=eps, weight_decay=0.0, step=1)
    m64, v64 = _np64(m), _np64(v)
    assert np.isfinite(v64).all() and v64.max() > 2.0**92
    want = -(1e-2 / (1 - 0.9)) * m64 / (np.sqrt(v64 / (1 - 0.95)) + eps)
    # the root, three products, a sum, the quotient, two factors: at most ten roundings
    assert np.all(np.abs(_np64(p) - want) <= 15 * ULP * np.abs(want))


def test_moments_that_are_not_finite_give_what_their_quotient_is():
    inf, nan = float("inf"), float("nan")
    m = torch.tensor([1.0, -1.0, inf, nan, 1.0, 0.0], device="cuda")
    v = torch.tensor([inf, inf, inf, inf, nan, inf], device="cuda")
    g, p = torch.zeros(6, device="cuda"), torch.tensor([2.0, 0.0, 2.0, 2.0, 2.0, -0.0], device="cuda")
    adamw_step([p], [g], [m], [v], **{**HYPER, "weight_decay": 0.0}, step=9)
    out = p.cpu()
    assert out[0] == 2 and out[1] == 0 and out[5] == 0 and bool(torch.isnan(out[2:5]).all())


# ---- lists made on the way ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
def test_iterators_give_the_bits_of_lists(bits):
    """Gradients, counters and the rest from generators, with device counters: the scratch that these need is allocated while the
    tensors made on the way are in use."""
    sizes = [4, 300, 5000]
    ps = [_randn(n, i) for i, n in enumerate(sizes)]
    gs = [_randn(n, 10 + i, 1e-3).bfloat16() for i, n in enumerate(sizes)]
    outs = []
    for lazy in (False, True):
        p = [t.clone() for t in ps]
        if bits == 32:
            state = [[torch.zeros_like(t) for t in ps] for _ in range(2)]
        else:
            state = [[torch.zeros(k, dtype=torch.uint8, device="cuda") for k in ks] for ks in 2 * (sizes, [-(-n // 256) for n in sizes])]
        lists = [p, (g.float() for g in gs), *state]
        step = (torch.full((), 3, device="cuda") for _ in sizes)
        if lazy:
            lists = [map(lambda t: t, ts) for ts in lists]
        else:
            lists, step = [list(ts) for ts in lists], list(step)
        call, kw = (adamw_step, {}) if bits == 32 else (adamw_step_8bit, {"seed": 1})
        call(*lists, **HYPER, **kw, step=step, grad_scale=torch.tensor(0.5, device="cuda"))
        outs.append([*p, *(t for ts in state for t in ts)])
    assert all(_same(a, b) for a, b in zip(*outs))


# ---- the C interface ----------------------------------------------------------------------------------------------------


def _c_step(counters, *, step, dev_lr=False, eps=1e-8, sizes=(4, 4)):
    """eo_adamw_step on tensors of ones; counters[i]: whether tensor i has a device step counter."""
    n = len(sizes)
    rows = [[torch.ones(k, device="cuda") for k in sizes] for _ in range(4)]
    count, lr = torch.ones((), dtype=torch.int64, device="cuda"), torch.full((), 0.1, device="cuda")
    scratch = torch.zeros(_native.lib().eo_adamw_scratch_bytes(n), dtype=torch.uint8, device="cuda")
    columns = [[t.data_ptr() for t in ts] for ts in rows] + [[0] * n] * 3
    columns += [[count.data_ptr() if c else 0 for c in counters], list(sizes), [0] * n]
    table = struct.pack(f"{10 * n}q", *[x for column in columns for x in column])
    config = _native._CONFIG.pack(
        0.1, 0.9, 0.95, eps, 0.0, step, lr.data_ptr() if dev_lr else 0, 0, scratch.data_ptr(), scratch.numel(), 0, 32, 0, 0
    )
    rc = _native.lib().eo_adamw_step(n, table, config, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return rc, rows[0]


BAD_ARG = 1


@pytest.mark.parametrize("counters,dev_lr,sizes", [
    ((0, 0), True, (4, 4)), ((1, 0), False, (4, 4)), ((0, 1), True, (4, 4)), ((0, 0), False, (4, 4)), ((0, 1), False, (4, 0)),
])  # fmt: skip
def test_step_numbers_below_one_are_refused_where_a_tensor_uses_them(counters, dev_lr, sizes):
    for step in (0, -3):
        rc, params = _c_step(counters, step=step, dev_lr=dev_lr, sizes=sizes)
        assert rc == BAD_ARG and b"counts from 1" in _native.lib().eo_last_error()
        assert all(bool((p == 1).all()) for p in params)
    rc, params = _c_step(counters, step=1, dev_lr=dev_lr, sizes=sizes)
    assert rc == 0 and all(bool(torch.isfinite(p).all()) and not bool((p == 1).any()) for p in params)


def test_epsilons_at_the_ends():
    """A weight that nothing moves stays where it is, down to the smallest eps, and the smallest eps divides; those beyond are refused."""
    for eps in (2.0**-126, 1e-30, 1e-8, 1e30):
        p, z = torch.tensor([1.0, -2.0], device="cuda"), torch.zeros(2, device="cuda")
        m = torch.tensor([0.0, eps], device="cuda")
        adamw_step([p], [z], [m], [z.clone()], lr=0.25, betas=(0.5, 0.5), eps=eps, weight_decay=0.0, step=1)
        assert p.tolist() == [1.0, -2.0 - 0.25]  # lr / (1 - 0.5) times half of eps over eps
    for eps in (1e-40, 2.0**126, float("inf"), float("nan"), -1e-8):
        rc, params = _c_step((0, 0), step=1, eps=eps)
        assert rc == BAD_ARG and all(bool((p == 1).all()) for p in params)


@pytest.mark.parametrize("counters,sizes", [((1, 1), (4, 4)), ((1, 0), (4, 0))])
def test_step_number_is_free_where_every_tensor_has_a_counter(counters, sizes):
    for dev_lr in (False, True):
        rc, params = _c_step(counters, step=0, dev_lr=dev_lr, sizes=sizes)
        assert rc == 0 and all(bool(torch.isfinite(p).all()) for p in params)


# ---- clipping of other memory orders --------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_clipping_of_dense_gradients_in_any_memory_order(dtype):
    """Transposed and channels-last gradients, with dimensions of one element and an odd offset: the float64 norm, and every element
    scaled where it lies."""
    base = _randn(3 + 33 * 70, 1).to(dtype)
    grads = [
        base[3:].view(33, 70).t(),
        _randn(4 * 6 * 5 * 5, 2).to(dtype).reshape(4, 6, 5, 5).to(memory_format=torch.channels_last),
        _randn(60, 3).to(dtype).reshape(5, 1, 12).transpose(0, 2),
        _randn(7, 4).to(dtype),
        torch.empty(3, 0, device="cuda", dtype=dtype).t(),
    ]
    assert not any(g.is_contiguous() for g in grads[:3])
    before = [g.clone() for g in grads]
    norm = float(np.sqrt(sum((_np64(g) ** 2).sum() for g in grads)))
    params = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
    for p, g in zip(params, grads):
        p.grad = g
    assert abs(float(utils.global_grad_norm(grads)) - norm) <= 2 * ULP * norm
    assert abs(float(utils.clip_coefficient(grads, 1.0)[1]) * norm - 1) <= 1e-6 / norm + 8 * ULP
    got = utils.clip_grad_norm_(params, 0.5 * norm)
    assert abs(float(got) - norm) <= 2 * ULP * norm
    want = 0.5 * norm / (norm + 1e-6)
    for p, g, b in zip(params, grads, before):
        assert p.grad.data_ptr() == g.data_ptr()
        # the coefficient is at most 6 roundings off, the product one; bf16 results are rounded by 2^-8 at most
        bound = 8 * ULP + (2.0**-8 * 1.01 if dtype == BF16 else 0)
        assert np.all(np.abs(_np64(g) - _np64(b) * want) <= bound * np.abs(_np64(b) * want))
    assert torch.equal(base[:3], _randn(3 + 33 * 70, 1).to(dtype)[:3])  # nothing beside them was scaled


def test_gradients_with_gaps_are_refused_by_clipping():
    x = torch.ones(6, 8, device="cuda")
    for g in (x[:, ::2], x[:, :4], x[0].expand(5, 8)):
        p = torch.nn.Parameter(torch.zeros(g.shape, device="cuda"))
        p.grad = g
        with pytest.raises(ValueError, match="not dense"):
            utils.clip_grad_norm_([p], 1e-3)
        with pytest.raises(ValueError, match="not dense"):
            utils.clip_coefficient([g], 1e-3)
    assert bool((x == 1).all())


# ---- copies and layouts ---------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_copied_model_and_optimizer_step_alike(bits, dtype):
    params = [torch.nn.Parameter(_randn(n, n, 0.02).to(dtype)) for n in (5, 700)]
    opt = AdamW(params, lr=1e-2, state_bits=bits, master_remainder=True, seed=3, weight_decay_method="independent")

    def step(ps, o, k):
        for p in ps:
            p.grad = _randn(p.numel(), 10 * k + p.numel(), 1e-3).to(dtype)
        o.step()

    step(params, opt, 0)
    others, other = copy.deepcopy((params, opt))
    for k in (1, 2):
        step(params, opt, k)
        step(others, other, k)
    for p, q in zip(params, others):
        assert p is not q and _same(p.detach(), q.detach())
        for name, value in opt.state[p].items():
            assert _same(value, other.state[q][name]) if torch.is_tensor(value) else value == other.state[q][name]


def test_negated_views_are_refused():
    """A lazily negated view (a part of a conjugate) holds its values with the other sign."""
    x, one = _randn(300, 1), torch.ones((), device="cuda")
    with pytest.raises(ValueError, match="negated"):
        quantize_blockwise(torch._neg_view(x), signed=True)
    lists = [[torch.zeros(4, device="cuda")] for _ in range(4)]
    for kw in (dict(lr=torch._neg_view(one)), dict(lr=0.1, grad_scale=torch._neg_view(one))):
        with pytest.raises(ValueError, match="negated"):
            adamw_step(*lists, **kw, step=1)
    with pytest.raises(ValueError, match="negated"):
        adamw_step(*lists, lr=0.1, step=torch._neg_view(torch.ones((), dtype=torch.int64, device="cuda")))
    assert not any(bool(t.any()) for (t,) in lists)


@pytest.mark.parametrize("capturable", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first,then", [("contiguous_format", "channels_last"), ("channels_last", "contiguous_format")])
def test_a_parameter_that_changes_its_memory_order(first, then, bits, capturable):
    """``model.to(memory_format=...)`` between two steps: refused without a trace, and taken once the state is laid out anew."""
    p = torch.nn.Parameter(_randn(4 * 6 * 5 * 5, 1, 0.02).reshape(4, 6, 5, 5).bfloat16().to(memory_format=getattr(torch, first)))
    other = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = AdamW([p, other], lr=1e-2, state_bits=bits, master_remainder=True, capturable=capturable)
    for q in (p, other):
        q.grad = torch.ones_like(q) * 1e-3
    opt.step()
    p.data = p.data.to(memory_format=getattr(torch, then))
    p.grad = torch.ones_like(p) * 1e-3
    other.grad = None
    before = [p.detach().clone(), *(t.clone() for t in opt.state[p].values() if torch.is_tensor(t))]
    with pytest.raises(ValueError, match="lays the state out anew"):
        opt.step()
    after = [p.detach(), *(t for t in opt.state[p].values() if torch.is_tensor(t))]
    assert all(torch.equal(a, b) for a, b in zip(before, after)) and int(opt.state[p]["step"]) == 1
    moments, remainder = opt.moments(p), opt.state[p]["remainder"].clone()
    opt.load_state_dict(opt.state_dict())
    for x, y in zip(moments, opt.moments(p)):
        assert torch.equal(x, y)  # one value throughout, so that blocks of another order round to it too
    assert torch.equal(opt.state[p]["remainder"], remainder)
    opt.step()
    assert int(opt.state[p]["step"]) == 2 and not torch.equal(opt.moments(p)[0], moments[0])


# ---- long chunks ----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("p_dtype,g_dtype", [(BF16, BF16), (F32, BF16)])
def test_chunks_of_more_runs_than_a_warp_holds_exponents_of(p_dtype, g_dtype):
    """A warp reads the exponent bytes of 32 of its runs (2048 elements apart) at a time; a launch over more than 320 M elements gives it
    more.  Random codes and exponents, so that a byte of another run shows: whole chunks against the fp32 step on the decoded
    moments (weights bit for bit) and the statement of the rounding (codes)."""
    n = 360_000_000 + 12_345
    chunk = n // (2048 * 148 * 32) // 4 * 4 * 2048
    assert chunk > 32 * 2048
    gen = torch.Generator(device="cuda").manual_seed(1)
    blocks = -(-n // 256)
    p = torch.empty(n, dtype=p_dtype, device="cuda").normal_(0, 0.02, generator=gen)
    g = torch.empty(n, dtype=g_dtype, device="cuda").normal_(0, 1, generator=gen)
    mc = torch.randint(0, 0x78, (n,), dtype=torch.uint8, device="cuda", generator=gen)  # below the NaN
    mc += torch.randint(0, 2, (n,), dtype=torch.uint8, device="cuda", generator=gen) * 128
    vc = torch.randint(0, 0xF8, (n,), dtype=torch.uint8, device="cuda", generator=gen)
    me, ve = [torch.randint(117, 137, (blocks,), dtype=torch.uint8, device="cuda", generator=gen) for _ in range(2)]
    parts = []
    for first in (0, 17 * chunk, n // chunk * chunk - chunk, n // chunk * chunk):
        here = slice(first, min(first + chunk, n))
        b = slice(first // 256, -(-here.stop // 256))
        m = dequantize_blockwise(mc[here].clone(), me[b].clone(), signed=True)
        v = dequantize_blockwise(vc[here].clone(), ve[b].clone(), signed=False)
        parts.append((here, b, p[here].clone(), g[here].clone(), m, v))
    adamw_step_8bit([p], [g], [mc], [me], [vc], [ve], **HYPER, step=6, seed=8)
    for here, b, p0, g0, m, v in parts:
        adamw_step([p0], [g0], [m], [v], **HYPER, step=6)
        assert _same(p[here], p0)
        for codes, exponents, wide, signed in ((mc, me, m, True), (vc, ve, v, False)):
            bits = ref.random_bits(wide.numel(), 8, 0, 6, signed, first=here.start)
            want, want_e = ref.quantize(wide.cpu().numpy(), signed, bits)
            assert np.array_equal(codes[here].cpu().numpy(), want) and np.array_equal(exponents[b].cpu().numpy(), want_e)

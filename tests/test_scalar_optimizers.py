"""AdamW, gradient clipping and the block quantiser without a GPU: the statements the GPU tests compare with, and what
is refused."""

import numpy as np
import pytest
import torch

from emerging_optimizers_b200 import _native, registry, utils
from emerging_optimizers_b200 import build as eo_build
from emerging_optimizers_b200.scalar_optimizers import (
    AdamW,
    adamw_step,
    adamw_step_8bit,
    dequantize_blockwise,
    quantize_blockwise,
)
from tests import _scalar_ref as ref


@pytest.fixture(scope="module", autouse=True)
def built():
    eo_build.build()


def _p(*shape, dtype=torch.float32):
    return torch.nn.Parameter(torch.ones(*shape, dtype=dtype))


@pytest.mark.parametrize(
    "kw",
    [{"lr": -1.0}, {"lr": float("nan")}, {"betas": (1.0, 0.9)}, {"betas": (0.9, -0.1)}, {"betas": (0.9,)}, {"eps": -1e-8},
     {"weight_decay": -0.1}, {"weight_decay_method": "other"}, {"state_bits": 16}, {"seed": -1}, {"seed": 1 << 32}],
)  # fmt: skip
def test_adamw_refuses_bad_hyperparameters(kw):
    with pytest.raises(ValueError):
        AdamW([_p(3)], **kw)


def test_adamw_is_registered_and_checks_names():
    assert registry.get_optimizer_cls("fused_adamw") is AdamW
    with pytest.raises(TypeError):
        registry.get_configured_optimizer_cls("fused_adamw", momentum=0.9)


def test_cpu_tensors_are_refused():
    p = _p(5)
    p.grad = torch.ones(5)
    opt = AdamW([p])
    with pytest.raises(_native.NativeLibraryError, match="no CPU path"):
        opt.step()
    assert not opt.state[p]
    x = torch.ones(5)
    for call in (
        lambda: adamw_step([x], [x], [x], [x], lr=1e-3, step=1),
        lambda: adamw_step_8bit([x], [x], [x], [x], [x], [x], lr=1e-3, step=1, seed=0),
        lambda: utils.clip_grads_([x], 1.0),
        lambda: utils.global_grad_norm([x]),
        lambda: utils.clip_grad_norm_([p], 1.0),
        lambda: quantize_blockwise(x, signed=True),
        lambda: dequantize_blockwise(x.to(torch.uint8), x.to(torch.uint8), signed=True),
    ):
        with pytest.raises(_native.NativeLibraryError, match="no CPU path"):
            call()
    assert torch.equal(p.detach(), torch.ones(5))


def test_host_module_of_another_torch_is_refused(monkeypatch):
    monkeypatch.setattr(_native, "_host_module", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(_native.NativeLibraryError, match="built for torch"):
        _native.host()


def test_scratch_queries_need_no_gpu():
    lib = _native.lib()
    assert lib.eo_adamw_scratch_bytes(0) == 0 and lib.eo_adamw_scratch_bytes(7) == 7 * 16
    small = lib.eo_grad_norm_scratch_bytes(3, 5000)
    assert small >= 8 * (3 + 2)  # a partial sum for every begun chunk of 2048 elements
    assert lib.eo_grad_norm_scratch_bytes(-1, 5) == 0
    huge = lib.eo_grad_norm_scratch_bytes(1, 1 << 40)
    assert small < huge < 1 << 20  # the number of chunks is bounded


def test_other_refusals_that_need_no_gpu():
    p = _p(5)
    p.grad = torch.ones(5)
    with pytest.raises(ValueError, match="closure"):
        AdamW([p]).step(lambda: 0.0)
    with pytest.raises(ValueError):
        utils.clip_grads_([], 1.0)
    with pytest.raises(ValueError):
        utils.clip_grads_([p.grad], -1.0)
    with pytest.raises(ValueError):
        utils.clip_grads_([p.grad], float("nan"))
    assert float(utils.clip_grad_norm_([_p(3)], 1.0)) == 0.0  # no gradients: nothing to do
    q = _p(5, dtype=torch.float16)
    q.grad = torch.ones(5, dtype=torch.float16)
    with pytest.raises(TypeError):
        AdamW([q]).step()
    q = _p(4)
    q.grad = torch.sparse_coo_tensor([[1]], [1.0], (4,))
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW([q]).step()
    AdamW([_p(3)]).step()  # nothing has a gradient
    adamw_step([], [], [], [], lr=1e-3, step=1)


@pytest.mark.parametrize("signed", [True, False])
def test_block_format_statement(signed):
    """Every code that a finite value can get reads back as itself, and rounding is to a neighbour."""
    top = 0x78 if signed else 0xF8  # the block's power of two rounded up
    codes = np.arange(0, top + 1)
    values = ref.dequantize(codes, np.array([127], np.uint8), signed)
    assert values[top] == 2.0 and values[1] == 2.0 ** (-16 if signed else -32) and np.all(np.diff(values) > 0)
    block = values[:top]  # below the next power of two, so the exponent byte is that of 1.0
    again, e = ref.quantize(block.astype(np.float32), signed)
    assert e[0] == 127 and np.array_equal(again, codes[:top])
    rng = np.random.default_rng(1)
    x = (rng.standard_normal(1000) * np.exp(2 * rng.standard_normal(1000))).astype(np.float32)
    x = x if signed else x * x
    for bits in (None, ref.random_bits(1000, 3, 1, 7, signed)):
        c, e = ref.quantize(x, signed, bits)
        y = ref.dequantize(c, e, signed)
        scale = np.ldexp(1.0, np.repeat(e.astype(int), 256)[:1000] - 127)
        unit = np.maximum(np.ldexp(1.0, np.frexp(np.abs(x))[1] - 4), scale * 2.0 ** (-16 if signed else -32))
        most = np.where((c == 1) & (not signed), 1.0, 0.5) if bits is None else 1.0  # unsigned values are kept above zero
        assert np.all(np.abs(y - x.astype(np.float64)) <= unit * most * (1 + 1e-12))


def test_random_rounding_is_unbiased():
    """65536 roundings of one value: the mean is off by at most six standard deviations of a mean of fair draws."""
    x = np.full(65536, 1.03, dtype=np.float32)
    c, e = ref.quantize(x, True, ref.random_bits(65536, 5, 0, 1, True))
    y = ref.dequantize(c, e, True)
    f = (1.03 - 1.0) * 8
    assert set(np.unique(y)) == {1.0, 1.125}
    assert abs(y.mean() - 1.03) <= 6 * 0.125 * np.sqrt(f * (1 - f) / 65536)

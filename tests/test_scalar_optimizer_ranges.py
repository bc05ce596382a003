"""AdamW, clipping and the block quantiser without a GPU: what a call keeps, and checkpoints and builds that are unusual."""

import copy
import gc
import os
import pickle
import shutil
import weakref

import pytest
import torch

from emerging_optimizers_b200 import _native
from emerging_optimizers_b200 import build as eo_build
from emerging_optimizers_b200.scalar_optimizers import AdamW, adamw_step, adamw_step_8bit


@pytest.fixture(scope="module", autouse=True)
def built():
    eo_build.build()


class _FakeHost:
    """Stands in for the host module: notes which tensors it was given."""

    def __init__(self):
        self.seen = []

    def adamw_table(self, *columns):
        self.seen += [weakref.ref(t) for ts in columns if ts is not None and not torch.is_tensor(ts) for t in ts]
        return 0, b"", 1

    def stream(self, device):
        return 0, True, False


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_made_on_the_way_live_until_the_launch(bits, monkeypatch):
    """Lists may be iterators that make their tensors as they go: the table holds addresses, so the call has to keep them."""
    host = _FakeHost()
    monkeypatch.setattr(_native, "host", lambda: host)
    alive = []

    def launch(device, n, *args, **kw):
        gc.collect()
        assert n == 3
        alive.extend(r() is not None for r in host.seen)

    monkeypatch.setattr(_native, "adamw_step", launch)

    def made(dtype=torch.float32):
        return (torch.zeros(4, dtype=dtype) for _ in range(3))

    kw = dict(lr=1e-3, step=(torch.ones((), dtype=torch.int64) for _ in range(3)), remainders=made(torch.int16))
    if bits == 32:
        adamw_step(made(), made(), made(), map(torch.abs, made()), **kw)
    else:
        adamw_step_8bit(*[made() for _ in range(6)], **kw, seed=0)
    assert len(alive) == 3 * (6 if bits == 32 else 8) and all(alive)


@pytest.mark.parametrize("eps", [1e-40, 2.0**-127, 2.0**126, 1e39, float("inf"), float("nan"), -1.0])
def test_epsilons_without_a_normal_reciprocal_are_refused(eps):
    with pytest.raises(ValueError, match="epsilon"):
        AdamW(_params(), eps=eps)
    x = [torch.zeros(3)]
    with pytest.raises(ValueError, match="epsilon"):
        adamw_step(x, x, x, x, lr=0.1, step=1, eps=eps)
    for fine in (0.0, 2.0**-126, 1e-30, 1.0, 1e30):
        AdamW(_params(), eps=fine)


def test_the_table_takes_lists_and_tuples_only():
    x = torch.zeros(3)
    for bad in (iter([x]), {0: x}, None, x):
        with pytest.raises(TypeError, match="must be a list of tensors"):
            _native.host().grads_table(bad, False)


@pytest.mark.parametrize("version", ["2.11.0a0+git1234567", "2.12.0.dev20260101", "2.11.0a0"])
def test_host_module_of_a_pre_release_of_torch(version, tmp_path, monkeypatch):
    """A module built for a pre-release is loaded there, and neither loaded nor taken for up to date with another torch."""
    real = eo_build.build_host()
    commands = []

    def compiler(cmd, tmp, out):
        commands.append(cmd)
        shutil.copy(real, out)
        return ""

    monkeypatch.setattr(eo_build, "PKG_DIR", str(tmp_path))
    monkeypatch.setattr(eo_build, "_run", compiler)
    monkeypatch.setattr(_native, "_host_module", None)
    monkeypatch.setattr(torch, "__version__", version)
    with pytest.raises(_native.NativeLibraryError, match="build --force"):
        _native.host()
    path = eo_build.build_host()
    assert len(commands) == 1 and os.path.dirname(path) == str(tmp_path)
    assert _native.host().__file__ == path
    eo_build.build_host()
    assert len(commands) == 1  # up to date
    monkeypatch.setattr(_native, "_host_module", None)
    monkeypatch.setattr(torch, "__version__", "2.11.1")
    with pytest.raises(_native.NativeLibraryError, match="built for torch 2.11.1"):
        _native.host()
    eo_build.build_host()
    assert len(commands) == 2


def test_host_module_that_does_not_load_is_named(tmp_path, monkeypatch):
    monkeypatch.setattr(eo_build, "PKG_DIR", str(tmp_path))
    monkeypatch.setattr(_native, "_host_module", None)
    with open(eo_build.host_path(), "w") as f:
        f.write("not a module")
    with pytest.raises(_native.NativeLibraryError, match="build --force"):
        _native.host()


def _saved(n=3):
    """A state of torch's class, as it comes back from a file."""
    state = {i: {"step": torch.tensor(5.0), "exp_avg": torch.full((n,), 0.5), "exp_avg_sq": torch.full((n,), 2.0)} for i in range(2)}
    return {"state": state, "param_groups": [{"lr": 0.1, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.0, "params": [0, 1]}]}


def _params(n=3):
    return [torch.nn.Parameter(torch.ones(n)) for _ in range(2)]


def test_hooks_of_loading_see_and_change_the_state(monkeypatch):
    monkeypatch.setattr(AdamW, "_loaded_state", lambda self, p, saved: dict(saved))  # what makes GPU tensors of it
    params = _params()
    opt = AdamW(params)
    seen = []

    def renamed(_, state_dict):
        seen.append(("pre", sorted(state_dict["state"])))
        return {**state_dict, "state": {0: state_dict["state"][1]}}

    def doubled(_, state_dict):
        seen.append(("second pre", sorted(state_dict["state"])))
        state_dict["state"] = {0: {**state_dict["state"][0], "exp_avg": 2 * state_dict["state"][0]["exp_avg"]}}

    opt.register_load_state_dict_pre_hook(doubled)
    opt.register_load_state_dict_pre_hook(renamed, prepend=True)
    opt.register_load_state_dict_post_hook(lambda o: seen.append(("post", [p in o.state for p in params])))
    opt.register_load_state_dict_post_hook(lambda o: seen.append(("first post", [p in o.state for p in params])), prepend=True)
    saved = _saved()
    opt.load_state_dict(saved)
    want = [("pre", [0, 1]), ("second pre", [0]), ("first post", [True, False]), ("post", [True, False])]
    assert seen == want
    assert bool((opt.state[params[0]]["exp_avg"] == 1.0).all()) and opt.param_groups[0]["lr"] == 0.1
    assert sorted(saved["state"]) == [0, 1]  # the caller's is as it was
    opt.load_state_dict(_saved())  # hooks of one call are gone at the next
    assert seen == 2 * want


def test_a_refused_load_leaves_no_hook_behind(monkeypatch):
    monkeypatch.setattr(AdamW, "_loaded_state", lambda self, p, saved: dict(saved))
    opt = AdamW(_params())
    bad = _saved()
    bad["param_groups"][0]["amsgrad"] = True
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(bad)
    short = _saved()
    short["param_groups"][0]["params"] = [0]
    with pytest.raises(ValueError):
        opt.load_state_dict(short)
    assert not opt.state
    opt.load_state_dict(_saved())
    assert len(opt.state) == 2


@pytest.mark.parametrize("again", [copy.deepcopy, lambda o: pickle.loads(pickle.dumps(o)), copy.copy])
def test_copies_keep_what_says_how_to_read_the_state(again):
    kw = dict(weight_decay_method="palm", state_bits=8, master_remainder=True, capturable=True, seed=5)
    opt = AdamW(_params(), lr=0.25, **kw)
    other = again(opt)
    assert {name: getattr(other, name) for name in kw} == kw and other.param_groups[0]["lr"] == 0.25
    other.step()  # nothing has a gradient
    other.param_groups[0]["params"][0].grad = torch.ones(3)
    with pytest.raises(_native.NativeLibraryError, match="no CPU path"):
        other.step()

"""group_norm and dropout on the CPU: tests of tests/test_gpu_layers.py called with the simulator's build of the kernels in the HIP
library's place (tests/cpu_sim; test_sim_kernels.py says what that shows and what not). Both forms of the norm, all types and
vector widths, the second draw of the generator, refusals; about a minute together. `pytest tests/test_gpu_layers.py -m gpu --sim`
runs all of them."""
import importlib
import inspect
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from inpc_amd import _lib

CASES = [
    ("test_dropout_is_its_definition_bit_for_bit", dict(count=10007, dtype="bf16")),
    ("test_dropout_is_its_definition_bit_for_bit", dict(count=9, dtype="fp32")),
    ("test_dropout_second_draw_decides_ties", {}),
    ("test_dropout_extremes", dict(dtype="fp32")),
    ("test_dropout_layouts", dict(dtype="fp16")),
    ("test_dropout_seed_on_the_device", {}),
    ("test_group_norm", dict(shape=(3, 30, 11, 7, 5), dtype="fp16")),
    ("test_group_norm", dict(shape=(1, 2064, 3, 2, 1), dtype="fp32")),
    ("test_group_norm", dict(shape=(5, 4, 1, 1, 2), dtype="bf16")),
    ("test_group_norm_of_large_groups", dict(shape=(2, 24, 120, 95, 3, "fp16", "gelu", 0.25))),
    ("test_group_norm_of_large_groups", dict(shape=(1, 33, 200, 200, 33, "fp32", "silu", 0.1))),
    ("test_group_norm_of_large_groups", dict(shape=(1, 40, 120, 75, 5, "fp32", "relu", 0.0))),
    *(("test_group_norm_of_wide_groups", dict(shape=shape))
      for shape in ((2, 1030, 40, 11, 2, "bf16", "silu", 0.25), (1, 8008, 12, 9, 8, "fp16", "gelu", 0.0), (3, 4104, 9, 7, 1, "fp16", "relu", 0.1),
                    (1, 6148, 5, 5, 1, "fp32", "none", 0.5))),
    ("test_group_norm_gradients_of_a_wide_group_with_many_pixels", {}),
    ("test_group_norm_activation_and_dropout", dict(act="silu", p=0.35, dtype="bf16")),
    ("test_group_norm_layouts", dict(dtype="bf16")),
    ("test_group_norm_of_values_far_from_zero", {}),
    ("test_group_norm_of_an_outlier_in_front_of_many_values", dict(shape=(1, 2056, 64, 64, 1, "fp32"))),
    ("test_group_norm_of_an_outlier_in_front_of_many_values", dict(shape=(1, 515, 64, 64, 1, "fp16"))),
    ("test_group_norm_of_an_outlier_in_front_of_many_values", dict(shape=(256, 1, 256, 256, 1, "fp16"))),
    ("test_group_norm_gradient_against_differences", {}),
    ("test_group_norm_keeps_what_is_not_finite_inside_its_group", dict(size=(90, 101))),
    ("test_group_norm_of_nothing", {}),
    ("test_gradients_of_nothing_through_the_c_abi", dict(size=dict(n_images=0, n_pixels=9), param="fp32")),
    ("test_gradients_of_nothing_through_the_c_abi", dict(size=dict(n_images=2, n_pixels=0), param="bf16")),
    ("test_norm_then_dropout_is_the_chain_of_both", {}),
    ("test_a_training_step_from_points_to_loss", {}),
    ("test_checkpoint_of_a_call_whose_seed_tensor_is_let_go", dict(op="group_norm")),
    ("test_checkpoint_of_a_call_whose_seed_tensor_is_let_go", dict(op="dropout")),
    ("test_a_saved_copy_of_the_seed_outlives_a_refill", dict(op="group_norm")),
    ("test_a_saved_copy_of_the_seed_outlives_a_refill", dict(op="dropout")),
    ("test_saved_tensors_that_come_back_with_other_strides", {}),
    *(("test_saved_tensors_that_come_back_as_something_else_are_refused", dict(which=which))
      for which in ("input", "weight", "bias", "moments", "seed")),
    ("test_refusals", {}),
    ("test_forward_mode_is_refused", dict(grad_mode=True)),
    ("test_forward_mode_is_refused", dict(grad_mode=False)),
    ("test_recording_is_refused", dict(requires_grad=True)),
    ("test_recording_is_refused", dict(requires_grad=False)),
]


def _case_id(case):
    name, kwargs = case
    return name[5:] + "".join(f"-{v}".replace(" ", "") for v in kwargs.values())


@pytest.mark.parametrize("case", CASES, ids=_case_id)
def test_on_the_simulator(sim, case):
    name, kwargs = case
    function = getattr(importlib.import_module("tests.test_gpu_layers"), name)
    assert set(inspect.signature(function).parameters) == {"gpu", *kwargs}
    assert "real_gpu" not in [m.name for m in getattr(function, "pytestmark", [])]
    function(gpu=sim, **kwargs)


def test_the_seed_of_a_call_without_dropout_is_not_read(sim):
    """Its address may be anything: none of these runs on a device, where reading it would fault."""
    gen = torch.Generator().manual_seed(1)
    nowhere = 8
    for pixels in (16, 9000):   # either form
        x, dy = (torch.randn(pixels, 8, generator=gen) for _ in range(2))
        results = []
        for seed_dev in (None, nowhere):
            cfg = _lib.GroupNormConfig(1, pixels, 8, 2, _lib.DTYPE_F32, _lib.DTYPE_F32, 2, 1e-5, pixels * 8, 8, pixels * 8, 8, 0.0, 5,
                                       seed_dev, 0)
            y, dx, dw, moments = torch.empty_like(x), torch.empty_like(x), torch.empty(8), torch.empty(4)
            lib = _lib.lib()
            workspace = [torch.empty(lib.inpc_group_norm_workspace_bytes(cfg, backward) + 16, dtype=torch.uint8) for backward in (0, 1)]
            _lib.check(lib.inpc_group_norm_forward(cfg, _lib.ptr(x), None, None, _lib.ptr(y), _lib.ptr(moments), _lib.ptr(workspace[0]),
                                                   workspace[0].numel(), None), "inpc_group_norm_forward")
            _lib.check(lib.inpc_group_norm_backward(cfg, _lib.ptr(dy), _lib.ptr(x), None, None, _lib.ptr(moments), _lib.ptr(dx),
                                                    _lib.ptr(dw), None, _lib.ptr(workspace[1]), workspace[1].numel(), None),
                       "inpc_group_norm_backward")
            copied = torch.empty_like(x)
            _lib.check(lib.inpc_dropout(_lib.ptr(x), _lib.ptr(copied), x.numel(), _lib.DTYPE_F32, 0.0, 5, seed_dev, 0, None), "inpc_dropout")
            assert torch.equal(copied, x)
            results.append((y, dx, dw, moments))
        assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("order", ["reverse", "shuffle"])
def test_results_do_not_depend_on_the_order_of_threads_and_blocks(order):
    chosen = [_case_id(c) for c in CASES if "large_groups" in c[0] or "wide_groups" in c[0] or c[0] in ("test_group_norm", "test_dropout_layouts")]
    nodes = [f"{Path(__file__)}::test_on_the_simulator[{case}]" for case in chosen]
    done = subprocess.run([sys.executable, "-m", "pytest", *nodes, "-q", "-x", "-p", "no:cacheprovider"],
                          env=dict(os.environ, INPC_SIM_ORDER=order), capture_output=True, text=True, stdin=subprocess.DEVNULL,
                          timeout=900, cwd=Path(__file__).resolve().parent.parent)
    assert done.returncode == 0, done.stdout[-3000:] + done.stderr[-2000:]
    assert f"{len(chosen)} passed" in done.stdout, done.stdout[-2000:]

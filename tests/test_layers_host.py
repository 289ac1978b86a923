"""What of the layers (inpc_amd/layers.py, include/inpc_hip.h) can be checked without a kernel launch: the C layout of the
configuration, the refusals of the C calls, the reference's generator against published answers."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from inpc_amd import _lib, dropout, group_norm
from tests import layer_reference as R

HEADER = Path(__file__).resolve().parent.parent / "include" / "inpc_hip.h"


def test_generator_gives_the_published_answers():
    # the known answers that come with the generator's publication (Random123, kat_vectors: philox4x32 10)
    assert [int(v) for v in R.philox(np.array([0]), 0, 0, 0)[0]] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = R.philox(np.array([2**63 + 2**32 - 1 + (2**31 - 1 << 32)], dtype=np.uint64) & np.uint64(2**63 - 1), 1, 2**64 - 1, 2**64 - 1)
    assert [int(v) for v in ones[0]] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]


def test_configuration_has_the_c_layout(tmp_path):
    names = [f for f, _ in _lib.GroupNormConfig._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", f'#include "{HEADER}"', "int main(void) {",
             '  printf("size %zu\\n", sizeof(inpc_group_norm_config));']
    lines += [f'  printf("{f} %zu\\n", offsetof(inpc_group_norm_config, {f}));' for f in names]
    lines += ['  printf("constants %d %d %d %d %d %d %d\\n", INPC_DTYPE_F32, INPC_DTYPE_F16, INPC_DTYPE_BF16, '
              "INPC_ACTIVATION_NONE, INPC_ACTIVATION_RELU, INPC_ACTIVATION_SILU, INPC_ACTIVATION_GELU);", "  return 0; }"]
    source, program = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines))
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-pedantic", str(source), "-o", str(program)], check=True)
    out = dict(line.split(" ", 1) for line in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.splitlines())
    assert int(out["size"]) == C.sizeof(_lib.GroupNormConfig)
    for f in names:
        assert int(out[f]) == getattr(_lib.GroupNormConfig, f).offset, f
    assert out["constants"] == f"{_lib.DTYPE_F32} {_lib.DTYPE_F16} {_lib.DTYPE_BF16} {_lib.ACTIVATION_NONE} " \
                               f"{_lib.ACTIVATION_RELU} {_lib.ACTIVATION_SILU} {_lib.ACTIVATION_GELU}"


def config(**changes):
    values = dict(n_images=1, n_pixels=16, channels=8, groups=2, dtype=_lib.DTYPE_F16, param_dtype=_lib.DTYPE_F32, activation=0,
                  eps=1e-5, input_image_stride=128, input_pixel_stride=8, grad_image_stride=128, grad_pixel_stride=8,
                  dropout_p=0.0, seed=0, seed_dev=None, offset=0)
    values.update(changes)
    return _lib.GroupNormConfig(**values)


@pytest.mark.parametrize("changes,code,word", [
    (dict(groups=3), -1, b"groups"),
    (dict(groups=0), -1, b"groups"),
    (dict(channels=0), -1, b"groups"),
    (dict(dtype=3), -3, b"fp32"),
    (dict(param_dtype=_lib.DTYPE_BF16), -3, b"parameters"),
    (dict(activation=4), -3, b"activation"),
    (dict(activation=-1), -3, b"activation"),
    (dict(eps=-1.0), -1, b"eps"),
    (dict(eps=float("nan")), -1, b"eps"),
    (dict(dropout_p=1.5), -1, b"probability"),
    (dict(dropout_p=float("nan")), -1, b"probability"),
    (dict(channels=131072, groups=1), -3, b"65536"),
    (dict(n_pixels=1 << 30), -3, b"2^30"),
    (dict(n_images=1 << 23), -3, b"images"),
    (dict(n_images=0xFFFFFFFF, channels=8, groups=8), -3, b"images"),
    (dict(input_pixel_stride=1 << 19), -3, b"strides"),
    (dict(grad_pixel_stride=1 << 19), -3, b"strides"),
])
def test_refused_configurations(changes, code, word):
    lib = _lib.lib()
    cfg = config(**changes)
    fake = (C.c_char * 256)()   # never dereferenced: the calls return before they launch anything
    p = C.c_void_p((C.addressof(fake) + 15) & ~15)
    assert lib.inpc_group_norm_forward(C.byref(cfg), p, None, None, p, p, p, 1 << 62, None) == code
    assert word in lib.inpc_last_error()
    assert lib.inpc_group_norm_backward(C.byref(cfg), p, p, None, None, p, p, None, None, p, 1 << 62, None) == code
    assert word in lib.inpc_last_error()


def test_refused_pointers_and_workspaces():
    lib = _lib.lib()
    cfg = config()
    size = lib.inpc_group_norm_workspace_bytes(C.byref(cfg), 0)
    fake = (C.c_char * 256)()
    p = C.c_void_p((C.addressof(fake) + 15) & ~15)
    assert lib.inpc_group_norm_workspace_bytes(C.byref(config(groups=3)), 0) == 0
    assert lib.inpc_group_norm_workspace_bytes(None, 1) == 0
    assert lib.inpc_group_norm_forward(None, p, None, None, p, p, p, size, None) == -1
    for args in ((None, None, None, p, p), (p, None, None, None, p), (p, None, None, p, None)):
        assert lib.inpc_group_norm_forward(C.byref(cfg), *args, p, size, None) == -1
    for args in ((None, p, None, None, p, p, p, p), (p, None, None, None, p, p, p, p), (p, p, None, None, None, p, p, p)):
        assert lib.inpc_group_norm_backward(C.byref(cfg), *args, p, size, None) == -1
    # nothing to do: no pointer is looked at
    empty = config(n_images=0)
    assert lib.inpc_group_norm_forward(C.byref(empty), None, None, None, None, None, None, 0, None) == 0
    assert lib.inpc_group_norm_backward(C.byref(cfg), None, None, None, None, None, None, None, None, None, 0, None) == 0
    large = config(n_pixels=1_000_000, input_image_stride=8_000_000, grad_image_stride=8_000_000)
    sizes = [lib.inpc_group_norm_workspace_bytes(C.byref(large), backward) for backward in (0, 1)]
    assert 0 < sizes[0] < sizes[1]
    for backward, size in enumerate(sizes):
        for workspace, held in ((p, size - 1), (None, size), (C.c_void_p(p.value + 4), size)):
            if backward:
                rc = lib.inpc_group_norm_backward(C.byref(large), p, p, None, None, p, p, None, None, workspace, held, None)
            else:
                rc = lib.inpc_group_norm_forward(C.byref(large), p, None, None, p, p, workspace, held, None)
            assert rc == -2 and b"workspace" in lib.inpc_last_error()
    # small maps need none, except to add up the parameters' gradients of several images
    assert lib.inpc_group_norm_workspace_bytes(C.byref(cfg), 0) == lib.inpc_group_norm_workspace_bytes(C.byref(cfg), 1) == 0
    assert lib.inpc_group_norm_workspace_bytes(C.byref(config(n_images=3)), 1) == 3 * 8 * 8
    assert lib.inpc_dropout(None, p, 4, 0, 0.5, 1, None, 0, None) == -1
    assert lib.inpc_dropout(p, None, 4, 0, 0.5, 1, None, 0, None) == -1
    assert lib.inpc_dropout(p, p, 4, 3, 0.5, 1, None, 0, None) == -3
    assert lib.inpc_dropout(p, p, 4, 0, 1.5, 1, None, 0, None) == -1
    assert lib.inpc_dropout(p, p, 4, 0, float("nan"), 1, None, 0, None) == -1
    assert lib.inpc_dropout(p, p, 1 << 40, 0, 0.5, 1, None, 0, None) == -3
    assert lib.inpc_dropout(None, None, 0, 0, 0.5, 1, None, 0, None) == 0


def test_wide_groups_take_a_workspace_where_they_are_cut_into_parts():
    lib = _lib.lib()

    def sizes(**changes):
        cfg = config(**changes)
        return [lib.inpc_group_norm_workspace_bytes(C.byref(cfg), backward) for backward in (0, 1)]

    wide = dict(channels=65535, groups=1, n_pixels=1, input_pixel_stride=65535, input_image_stride=65535, grad_pixel_stride=65535,
                grad_image_stride=65535)
    # 128 parts of 512 single elements at most, one slab: a pair of sums for each, of each channel, and of each image
    assert sizes(**wide, n_images=1000) == [1000 * 128 * 8, 1000 * 128 * 8 + (1000 * 65535 * 8 + 255) // 256 * 256 + 1000 * 8]
    # more blocks than a launch has: a block for each image
    assert sizes(**wide, n_images=65600) == [0, 65600 * 65535 * 8]
    # 64 KB: one block
    assert sizes(**dict(wide, channels=32768), n_images=2) == [0, 2 * 32768 * 8]


def test_operators_refuse_host_tensors():
    x = torch.randn(1, 4, 2, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        group_norm(x, 2)
    with pytest.raises(RuntimeError, match="GPU"):
        dropout(x, 0.5, 1)
    with pytest.raises(RuntimeError, match="GPU"):
        dropout(None, 0.5, 1)

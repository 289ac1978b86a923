"""group_norm and dropout (inpc_amd/layers.py) against plain 64-bit implementations (tests/layer_reference.py, which
derives the tolerances)."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.utils.checkpoint import checkpoint

from inpc_amd import _lib, dropout, fused_cauchy_loss, group_norm, rasterize_points, synthetic
from tests import helpers as H
from tests import layer_reference as R

pytestmark = pytest.mark.gpu

DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def to_device(t):
    """A CPU tensor on the device, with its strides."""
    return t.to(H.DEVICE, copy=True) if t is not None else None


def bits(t):
    t = t.detach().cpu().contiguous()
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


# ---- dropout -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("count", [0, 1, 7, 8, 9, 2047, 2049, 10007])
def test_dropout_is_its_definition_bit_for_bit(gpu, dtype, count):
    gen = torch.Generator().manual_seed(count)
    x = torch.randn(count, generator=gen).to(DTYPES[dtype])
    dy = torch.randn(count, generator=gen).to(DTYPES[dtype])
    for p, seed, offset in ((0.1, 5, 0), (0.5, 2**64 - 1, 2**64 - 1), (2**-9 + 2**-30, 1234567891011, 2**32)):
        xd = to_device(x).requires_grad_(True)
        y = dropout(xd, p, seed, offset)
        y.backward(to_device(dy))
        assert torch.equal(bits(y), bits(R.dropout(x, p, seed, offset)))
        assert torch.equal(bits(xd.grad), bits(R.dropout(dy, p, seed, offset)))
        assert y.dtype == x.dtype and y.shape == x.shape


def test_dropout_second_draw_decides_ties(gpu):
    # T = 77 * 2^16 + 2^15: elements whose first half is 77 (one in 65536) are decided by the second draw, both ways
    p, seed, count = (77 + 0.5) / 65536, 3, 400_003
    first = R.halves(0, count, 0, 0, seed)
    second = R.halves(0, count, 1, 0, seed)
    tied = first == 77
    assert (tied & (second < 32768)).any() and (tied & (second >= 32768)).any()
    x = torch.ones(count)
    got = dropout(to_device(x), p, seed)
    assert torch.equal(bits(got), bits(R.dropout(x, p, seed)))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_dropout_extremes(gpu, dtype):
    x = torch.randn(1003, generator=torch.Generator().manual_seed(1)).to(DTYPES[dtype])
    x[::3] = float("nan")
    x[1::3] = float("inf")
    xd = to_device(x).requires_grad_(True)
    assert dropout(xd, 0.0, None) is xd and dropout(xd, 0.7, None, training=False) is xd
    y = dropout(xd, 1.0, 9)
    y.backward(torch.full_like(y, float("nan")))
    assert torch.equal(y.detach().cpu(), torch.zeros_like(x)) and torch.equal(xd.grad.cpu(), torch.zeros_like(x))
    # a dropped NaN or infinity is 0, a kept one stays
    keep = torch.from_numpy(R.kept(0, 1003, 0.5, 9, 0))
    y = dropout(to_device(x), 0.5, 9).cpu()
    assert (y[~keep] == 0).all()
    assert torch.equal(torch.isnan(y), keep & torch.isnan(x)) and torch.equal(torch.isinf(y), keep & torch.isinf(x))


def test_dropout_masks_are_uniform_and_independent(gpu):
    count, p = 200_000, 0.3
    x = torch.ones(count, device=H.DEVICE)
    masks = [dropout(x, p, seed, offset).cpu() > 0 for seed, offset in ((1, 0), (1, 1), (2, 0), (1 + 2**32, 0), (1, 2**32))]
    sigma = (p * (1 - p) / count) ** 0.5
    for i, m in enumerate(masks):
        assert abs(m.double().mean() - (1 - p)) < 6 * sigma
        assert abs((m[1:] & m[:-1]).double().mean() - (1 - p) ** 2) < 6 * count**-0.5   # neighbours
        for other in masks[:i]:
            assert abs((m & other).double().mean() - (1 - p) ** 2) < 6 * count**-0.5


@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_dropout_layouts(gpu, dtype):
    gen = torch.Generator().manual_seed(4)
    wide = torch.randn(2, 5, 7, 6, generator=gen).to(DTYPES[dtype])
    p, seed, offset = 0.4, 77, 5
    # channels last: numbered (N, H, W, C), the result lies the same way; also with a gradient that lies otherwise
    x = to_device(wide).to(memory_format=torch.channels_last).requires_grad_(True)
    y = dropout(x, p, seed, offset)
    assert y.stride() == x.stride()
    want = R.dropout(wide.permute(0, 2, 3, 1).contiguous(), p, seed, offset).permute(0, 3, 1, 2)
    assert torch.equal(y.detach().cpu(), want)
    dy = torch.randn(2, 5, 7, 6, generator=gen).to(DTYPES[dtype])
    (grad,) = torch.autograd.grad(y, x, to_device(dy))
    assert torch.equal(grad.cpu(), R.dropout(dy.permute(0, 2, 3, 1).contiguous(), p, seed, offset).permute(0, 3, 1, 2))
    # a transposed matrix is made contiguous first
    m = to_device(wide).view(10, 42).t()
    assert torch.equal(dropout(m, p, seed, offset).cpu(), R.dropout(wide.view(10, 42).t().contiguous(), p, seed, offset))
    # a vector that starts one element behind an aligned address
    v = to_device(wide).view(-1)[1:]
    assert torch.equal(dropout(v, p, seed, offset).cpu(), R.dropout(wide.view(-1)[1:], p, seed, offset))
    # a gradient that is one value expanded
    v = v.detach().requires_grad_(True)
    dropout(v, p, seed, offset).sum().backward()
    assert torch.equal(v.grad.cpu(), R.dropout(torch.ones(v.numel(), dtype=DTYPES[dtype]), p, seed, offset))


def test_dropout_seed_on_the_device(gpu):
    x = torch.randn(5000, device=H.DEVICE).requires_grad_(True)
    for seed in (11, 2**63 + 5):
        held = torch.tensor([seed - 2**64 if seed >= 2**63 else seed], dtype=torch.int64, device=H.DEVICE)
        y = dropout(x, 0.2, held, offset=3)
        assert torch.equal(y, dropout(x, 0.2, seed, offset=3))
        (grad,) = torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
        assert torch.equal(grad != 0, y != 0)
        held += 1   # the mask of a backward pass could no longer be computed again
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, x, torch.ones_like(y))


@pytest.mark.parametrize("offset", [0, 1])
def test_dropout_in_place_through_the_c_abi(gpu, offset):
    x = torch.randn(6001, generator=torch.Generator().manual_seed(2)).half()
    held = to_device(x)[offset:]
    _lib.check(_lib.lib().inpc_dropout(_lib.ptr(held), _lib.ptr(held), held.numel(), _lib.DTYPE_F16, 0.3, 8, None, 0, H.stream()),
               "inpc_dropout")
    assert torch.equal(held.cpu(), R.dropout(x[offset:], 0.3, 8))


# ---- group norm ----------------------------------------------------------------------------------------------------

def make_case(n, c, h, w, dtype, seed, mean=1.0, weighted=True, param_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, h, w, c, generator=gen) * torch.exp(0.5 * torch.randn(c, generator=gen)) + mean * torch.randn(c, generator=gen)
    x = x.to(DTYPES[dtype]).permute(0, 3, 1, 2)
    weight = (1 + 0.3 * torch.randn(c, generator=gen)).to(param_dtype) if weighted else None
    bias = (0.3 * torch.randn(c, generator=gen)).to(param_dtype) if weighted else None
    dy = torch.randn(n, h, w, c, generator=gen).to(DTYPES[dtype]).permute(0, 3, 1, 2)
    return x, weight, bias, dy


def mask_of(shape, p, seed, offset=0):
    n, c, h, w = shape
    if not p:
        return None
    keep = torch.from_numpy(R.kept(0, n * c * h * w, p, seed, offset)).view(n, h, w, c).permute(0, 3, 1, 2)
    return keep.double() * (1.0 / (1.0 - p) if p < 1 else 0.0)


def check(x, weight, bias, dy, groups, act="none", eps=1e-5, p=0.0, seed=1, offset=0, on_device=to_device):
    """Forward and backward pass of the operator against the reference; returns the outputs."""
    keep = mask_of(x.shape, p, seed, offset)
    if act == "relu":   # a value on the border has no gradient to compare: leave those out
        z = R.GroupNorm(x, groups, weight, bias, eps, act)
        dy = torch.where(z.z.abs() <= z.z_bound, torch.zeros((), dtype=dy.dtype), dy)
    ref = R.GroupNorm(x, groups, weight, bias, eps, act, keep, dy)
    xd = on_device(x).requires_grad_(True)
    leaves = [t.requires_grad_(True) if t is not None else None for t in (to_device(weight), to_device(bias))]
    y = group_norm(xd, groups, *leaves, eps=eps, activation=act, dropout_p=p, seed=seed, offset=offset)
    assert y.dtype == x.dtype and y.shape == x.shape
    y.backward(on_device(dy))
    R.assert_within(y, ref.y, ref.y_bound, "y")
    R.assert_within(xd.grad, ref.dx, ref.dx_bound, "dx")
    if weight is not None:
        R.assert_within(leaves[0].grad, ref.dweight, ref.dweight_bound, "dweight")
    if bias is not None:
        R.assert_within(leaves[1].grad, ref.dbias, ref.dbias_bound, "dbias")
    with torch.no_grad():
        again = group_norm(on_device(x), groups, to_device(weight), to_device(bias), eps=eps, activation=act, dropout_p=p,
                           seed=seed, offset=offset)
    assert torch.equal(again, y.detach())
    return y.detach(), xd.grad


SHAPES = [
    # n, c, h, w, groups
    (1, 1, 1, 1, 1),       # one value: variance 0
    (1, 8, 1, 1, 2),       # one pixel
    (2, 3, 5, 7, 3),       # a group per channel, single elements
    (1, 6, 9, 4, 1),       # one group of all channels
    (3, 30, 11, 7, 5),     # six channels per group, vectors of two
    (2, 24, 13, 9, 3),
    (1, 64, 16, 16, 8),
    (1, 16, 40, 33, 4),    # many rows per block
    (2, 20, 17, 3, 20),
    (1, 260, 6, 5, 13),    # columns that do not divide a block
    (1, 2064, 3, 2, 1),    # more columns than a block has threads (of 8 values: 258), one group over all tiles
    (5, 4, 1, 1, 2),
    (1, 512, 5, 4, 1),     # a group wider than a block has threads
]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_group_norm(gpu, shape, dtype):
    *size, groups = shape
    check(*make_case(*size, dtype, sum(shape)), groups)


# maps whose groups are too large for one block each: slabs of pixels in one launch, the result in a second
SPLIT_SHAPES = [
    (1, 8, 150, 161, 1, "fp32", "none", 0.0),
    (1, 8, 150, 161, 1, "bf16", "silu", 0.0),
    (2, 24, 120, 95, 3, "fp16", "gelu", 0.25),      # columns that are no power of two
    (2, 24, 120, 95, 3, "fp32", "silu", 0.25),
    (3, 6, 210, 113, 2, "bf16", "silu", 0.5),       # vectors of two, 170 rows to a block
    (1, 40, 120, 75, 5, "fp32", "relu", 0.0),
    (1, 33, 200, 200, 33, "fp32", "silu", 0.1),     # single elements, two tiles of channels, the second of one group
    (1, 640, 41, 13, 2, "fp16", "none", 0.0),       # 80 columns, 320 channels to a group
]


@pytest.mark.parametrize("shape", SPLIT_SHAPES, ids=str)
def test_group_norm_of_large_groups(gpu, shape):
    *size, groups, dtype, act, p = shape
    check(*make_case(*size, dtype, sum(size)), groups, act, p=p, seed=19)


# groups too wide for a block: each is cut into parts
WIDE_SHAPES = [
    (2, 1030, 40, 11, 2, "bf16", "silu", 0.25),     # vectors of two would end inside a part: single elements, parts of 258 and 257
    (1, 8008, 12, 9, 8, "fp16", "gelu", 0.0),       # 1001 channels to a group, two parts each
    (3, 4104, 9, 7, 1, "fp16", "relu", 0.1),        # 513 vectors of eight
    (1, 6148, 5, 5, 1, "fp32", "none", 0.5),        # four parts, the last one narrower
    (2, 2052, 31, 20, 1, "fp32", "silu", 0.0),
]


@pytest.mark.parametrize("shape", WIDE_SHAPES, ids=str)
def test_group_norm_of_wide_groups(gpu, shape):
    *size, groups, dtype, act, p = shape
    x, weight, bias, dy = make_case(*size, dtype, sum(size))
    check(x, weight, bias, dy, groups, act, p=p, seed=19)
    # from an odd channel of a wider map: single elements
    check(x, weight, bias, dy, groups, act, p=p, seed=19, on_device=lambda t: to_device(torch.cat((t[:, :3], t, t[:, :2]), 1))[:, 3:-2])


def test_group_norm_gradients_of_a_wide_group_with_many_pixels(gpu):
    """Equal values, so that every addition of a long chain would round the same way."""
    x, weight, bias, dy = make_case(1, 515, 200, 200, "fp16", 29)
    check(x, weight, bias, torch.full_like(dy, 0.1), 1)


def test_group_norm_some_gradients_of_large_groups(gpu):
    x, weight, bias, dy = make_case(2, 8, 100, 90, "fp32", 77)
    ref = R.GroupNorm(x, 2, weight, bias, 1e-5, "silu", None, dy)
    for wanted in ("x", "weight", "bias", "x bias"):
        leaves = {name: to_device(t).requires_grad_(name in wanted.split())
                  for name, t in (("x", x), ("weight", weight), ("bias", bias))}
        group_norm(leaves["x"], 2, leaves["weight"], leaves["bias"], activation="silu").backward(to_device(dy))
        for name, t in leaves.items():
            if name in wanted.split():
                R.assert_within(t.grad, getattr(ref, "d" + name), getattr(ref, f"d{name}_bound"), f"d{name} of {wanted}")
            else:
                assert t.grad is None


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("act", ["relu", "silu", "gelu"])
@pytest.mark.parametrize("p", [0.0, 0.35])
def test_group_norm_activation_and_dropout(gpu, act, p, dtype):
    check(*make_case(2, 32, 9, 11, dtype, 5), 4, act, p=p, seed=2**40 + 3, offset=6)
    check(*make_case(1, 5, 7, 3, dtype, 6), 5, act, p=p, seed=8)     # single elements
    check(*make_case(1, 12, 6, 5, dtype, 7), 2, act, p=p, seed=8)    # vectors of four


@pytest.mark.parametrize("dtype,param", [("fp16", torch.float16), ("bf16", torch.bfloat16), ("fp32", torch.float32)])
def test_group_norm_parameters(gpu, dtype, param):
    x, weight, bias, dy = make_case(2, 16, 6, 7, dtype, 9, param_dtype=param)
    check(x, weight, bias, dy, 4, "silu")
    check(x, weight, None, dy, 4, "silu")
    check(x, None, bias, dy, 4, "silu")
    check(x, None, None, dy, 4, "silu")
    # only some gradients are asked for
    xd, wd, bd = to_device(x), to_device(weight).requires_grad_(True), to_device(bias)
    group_norm(xd, 4, wd, bd).backward(to_device(dy))
    ref = R.GroupNorm(x, 4, weight, bias, 1e-5, "none", None, dy)
    R.assert_within(wd.grad, ref.dweight, ref.dweight_bound, "dweight")
    assert xd.grad is None and bd.grad is None


def test_group_norm_of_values_far_from_zero(gpu):
    # a mean of about 1000 standard deviations: nothing may cancel (a sum of squares in fp32 would lose the variance)
    gen = torch.Generator().manual_seed(2)
    x = (torch.randn(2, 8, 33, 21, generator=gen) + 1000.0).to(memory_format=torch.channels_last)
    dy = torch.randn(2, 8, 33, 21, generator=gen).to(memory_format=torch.channels_last)
    y, _ = check(x, None, None, dy, 2)
    assert abs(float(y.std()) - 1.0) < 1e-3
    # an outlier in front of everything else
    x = torch.randn(1, 4, 16, 16, generator=gen).to(memory_format=torch.channels_last)
    x[0, 0, 0, 0] = 1e5
    check(x, None, None, dy[:1, :4, :16, :16].contiguous(memory_format=torch.channels_last), 2)
    # no variance at all
    check(torch.full((1, 4, 5, 5), 3.0).to(memory_format=torch.channels_last), None, None,
          torch.randn(1, 4, 5, 5, generator=gen), 2)


def outlier_in_front(n, c, h, w, dtype, seed):
    """Every image's first value makes up most of its variance: the worst pivot there is."""
    x, _, _, dy = make_case(n, c, h, w, dtype, seed, mean=0.0, weighted=False)
    x[:, 0, 0, 0] = 3e4
    return x, dy


@pytest.mark.parametrize("shape", [(1, 2056, 64, 64, 1, "fp32"), (1, 515, 64, 64, 1, "fp16"), (256, 1, 256, 256, 1, "fp16")], ids=str)
def test_group_norm_of_an_outlier_in_front_of_many_values(gpu, shape):
    *size, groups, dtype = shape
    x, dy = outlier_in_front(*size, dtype, 23)
    check(x, None, None, dy, groups)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_group_norm_layouts(gpu, dtype):
    gen = torch.Generator().manual_seed(12)
    x, weight, bias, dy = make_case(2, 16, 9, 10, dtype, 3)
    want = [t.cpu() for t in check(x, weight, bias, dy, 4, "silu", p=0.2)]

    def same(on_device):
        got = [t.cpu() for t in check(x, weight, bias, dy, 4, "silu", p=0.2, on_device=on_device)]
        assert all(torch.equal(a, b) for a, b in zip(got, want))

    same(lambda t: to_device(t).contiguous())     # (N, C, H, W) in memory
    check(x, weight, bias, dy, 4, "silu", p=0.2, on_device=lambda t: to_device(torch.cat((t, t), 1))[:, 16:])   # half of a wider map

    def slice_at_odd_channel(t):
        wide = torch.randn(2, 9, 10, 21, generator=gen).to(t.dtype).permute(0, 3, 1, 2)
        wide[:, 3:19] = t
        return to_device(wide)[:, 3:19]

    check(x, weight, bias, dy, 4, "silu", p=0.2, on_device=slice_at_odd_channel)

    def crop(t):   # pixels that are not evenly spaced
        wide = torch.zeros(2, 12, 14, 16, dtype=t.dtype).permute(0, 3, 1, 2)
        wide[:, :, 2:11, 3:13] = t
        return to_device(wide)[:, :, 2:11, 3:13]

    same(crop)
    # every second image, every second pixel of a row
    check(x, weight, bias, dy, 4, on_device=lambda t: to_device(t.repeat_interleave(2, 0))[::2])
    check(x, weight, bias, dy, 4, on_device=lambda t: to_device(t.repeat_interleave(2, 3))[:, :, :, ::2])
    # one value expanded as the gradient
    xd = to_device(x).requires_grad_(True)
    group_norm(xd, 4, to_device(weight), to_device(bias), activation="silu").sum().backward()
    ref = R.GroupNorm(x, 4, weight, bias, 1e-5, "silu", None, torch.ones_like(dy))
    R.assert_within(xd.grad, ref.dx, ref.dx_bound, "dx")
    # strided parameters
    both = to_device(torch.stack((weight, bias), 1))
    got = group_norm(to_device(x), 4, both[:, 0], both[:, 1], activation="silu")
    assert torch.equal(got, group_norm(to_device(x), 4, to_device(weight), to_device(bias), activation="silu"))


def test_group_norm_gradient_against_differences(gpu):
    """The operator's own directional derivatives by central differences: they differ from the gradient by what the
    differences cut off (known from the same differences in 64 bits) and by the rounding of y, divided by the step."""
    x, weight, bias, dy = make_case(2, 6, 4, 5, "fp32", 21)
    gen = torch.Generator().manual_seed(5)
    for act in ("none", "silu", "gelu"):
        ref = R.GroupNorm(x, 2, weight, bias, 1e-5, act, None, dy)
        grads = {"x": ref.dx, "weight": ref.dweight, "bias": ref.dbias}
        args = {"x": x, "weight": weight, "bias": bias}
        dev = {k: to_device(v).requires_grad_(True) for k, v in args.items()}
        y = group_norm(dev["x"], 2, dev["weight"], dev["bias"], activation=act)
        got = dict(zip(args, torch.autograd.grad(y, tuple(dev.values()), to_device(dy))))
        for name in args:
            direction = torch.randn(args[name].shape, generator=gen).to(args[name])
            h = 2.0**-7
            ends = []
            for sign in (1, -1):
                moved = dict(args, **{name: args[name] + sign * h * direction})
                here = group_norm(*(to_device(moved[k]) if k == "x" else None for k in ("x",)), 2, to_device(moved["weight"]),
                                  to_device(moved["bias"]), activation=act).cpu().double()
                exact = R.GroupNorm(moved["x"], 2, moved["weight"], moved["bias"], 1e-5, act)
                ends.append(((here * dy.double()).sum(), (exact.y * dy.double()).sum(), (exact.y_bound * dy.double().abs()).sum()))
            difference, exact_difference = ((ends[0][k] - ends[1][k]) / (2 * h) for k in (0, 1))
            slope = (grads[name] * direction.double()).sum()
            tolerance = (exact_difference - slope).abs() + (ends[0][2] + ends[1][2]) / (2 * h)
            assert (difference - (got[name].cpu().double() * direction.double()).sum()).abs() <= 1.01 * tolerance + 1e-4, (act, name)


@pytest.mark.parametrize("size", [(6, 5), (90, 101)], ids=["single", "split"])
def test_group_norm_keeps_what_is_not_finite_inside_its_group(gpu, size):
    x, weight, bias, dy = make_case(2, 8, *size, "fp32", 31)
    bad = x.clone()
    bad[0, 1, 2, 3] = float("nan")     # group 0 of image 0
    bad[1, 6, -1, -1] = float("inf")   # group 3 of image 1
    want = group_norm(to_device(x), 4, to_device(weight), to_device(bias)).cpu()
    got = group_norm(to_device(bad), 4, to_device(weight), to_device(bias)).cpu()
    hit = torch.zeros(2, 8, 1, 1, dtype=torch.bool)
    hit[0, 0:2] = hit[1, 6:8] = True
    assert torch.isnan(got[hit.expand_as(got)]).all()
    assert torch.equal(got[~hit.expand_as(got)], want[~hit.expand_as(got)])


def test_group_norm_of_nothing(gpu):
    for size in ((0, 4, 3, 3), (2, 4, 0, 3)):
        x = torch.empty(size, device=H.DEVICE).requires_grad_(True)
        w = torch.ones(4, device=H.DEVICE).requires_grad_(True)
        y = group_norm(x, 2, w, None, activation="silu")
        assert y.shape == size
        y.sum().backward()
        assert x.grad.shape == size and torch.equal(w.grad.cpu(), torch.zeros(4))


@pytest.mark.parametrize("param", ["fp32", "bf16"])
@pytest.mark.parametrize("size", [dict(n_images=0, n_pixels=9), dict(n_images=2, n_pixels=0)], ids=["no image", "no pixel"])
def test_gradients_of_nothing_through_the_c_abi(gpu, size, param):
    """The parameters' gradients are sums over nothing: zeros, in buffers that held something else."""
    channels = 70
    cfg = _lib.GroupNormConfig(**size, channels=channels, groups=7, dtype=_lib.DTYPE_BF16,
                               param_dtype=_lib.DTYPE_F32 if param == "fp32" else _lib.DTYPE_BF16, activation=0, eps=1e-5,
                               input_image_stride=0, input_pixel_stride=channels, grad_image_stride=0, grad_pixel_stride=channels)
    for wanted in ((True, True), (True, False), (False, True)):
        grads = [torch.full((channels + 1,), 7.0, dtype=DTYPES[param], device=H.DEVICE) for _ in range(2)]
        args = [_lib.ptr(g) if want else None for g, want in zip(grads, wanted)]
        _lib.check(_lib.lib().inpc_group_norm_backward(cfg, None, None, None, None, None, None, *args, None, 0, H.stream()),
                   "inpc_group_norm_backward")
        for g, want in zip(grads, wanted):
            expected = torch.full((channels + 1,), 7.0, dtype=DTYPES[param])
            if want:
                expected[:channels] = 0
            assert torch.equal(g.cpu(), expected)


# ---- together ------------------------------------------------------------------------------------------------------

def test_norm_then_dropout_is_the_chain_of_both(gpu):
    x, weight, bias, _ = make_case(2, 24, 7, 9, "fp32", 41)
    xd, wd, bd = (to_device(t) for t in (x, weight, bias))
    one = group_norm(xd, 3, wd, bd, activation="gelu", dropout_p=0.3, seed=6, offset=2)
    two = dropout(group_norm(xd, 3, wd, bd, activation="gelu"), 0.3, 6, offset=2)
    assert torch.equal(one, two)   # fp32: the chain rounds to fp32 in between anyway
    plain = group_norm(xd, 3, wd, bd, activation="gelu", dropout_p=0.3, training=False)
    assert torch.equal(plain, group_norm(xd, 3, wd, bd, activation="gelu"))


def test_a_training_step_from_points_to_loss(gpu):
    """Rasterizer -> norm, activation, dropout -> 1x1 mixing of channels -> dropout -> loss, and back to the points'
    features, against the same chain in 64 bits behind the same image."""
    hv = synthetic.camera_on_z(40, 28, 30.0, 3.0)
    n, channels = 3000, 8
    pos = synthetic.cube_points(n, 1.8, 3)
    feats, opac = synthetic.point_attributes(n, channels, "normal", 4)
    view = hv.to_view(torch.device(H.DEVICE))
    gen = torch.Generator().manual_seed(8)
    weight, bias = 1 + 0.2 * torch.randn(channels, generator=gen), 0.2 * torch.randn(channels, generator=gen)
    mix, target = torch.randn(3, channels, generator=gen) / 3, torch.rand(1, 3, hv.camera.height, hv.camera.width, generator=gen)

    f = H.dev(feats).requires_grad_(True)
    image, _, _ = rasterize_points(view, H.dev(pos), f, H.dev(opac), tile=16)
    wd, bd, md = (to_device(t).requires_grad_(True) for t in (weight, bias, mix))
    hidden = group_norm(image[None], 2, wd, bd, activation="silu", dropout_p=0.25, seed=5)
    picture = dropout((hidden.permute(0, 2, 3, 1) @ md.t()).permute(0, 3, 1, 2), 0.1, 5, offset=1)
    loss = fused_cauchy_loss(picture.contiguous(), to_device(target))
    grads = torch.autograd.grad(loss, (image, f, wd, bd, md))

    image64 = image.detach().cpu().double()[None].requires_grad_(True)
    leaves = [t.double().requires_grad_(True) for t in (weight, bias, mix)]
    grouped = image64.view(1, 2, -1)
    var, mean = torch.var_mean(grouped, dim=2, correction=0, keepdim=True)
    z = ((grouped - mean) / torch.sqrt(var + 1e-5)).view_as(image64) * leaves[0].view(1, -1, 1, 1) + leaves[1].view(1, -1, 1, 1)
    y = R.activation(z, "silu") * mask_of(image64.shape, 0.25, 5)
    out = torch.einsum("oc,nchw->nohw", leaves[2], y)
    out = out * mask_of(out.shape, 0.1, 5, 1)
    loss64 = torch.log1p(12.5 * (out - target.double()) ** 2).mean()
    want = torch.autograd.grad(loss64, (image64, *leaves))
    # every step is fp32: 2000 roundings of u on the way bound what adds up, relative to the largest value
    loss, loss64 = loss.detach(), loss64.detach()
    assert abs(float(loss) - float(loss64)) < 2000 * R.U * float(loss64)
    for got, ref in zip((grads[0][None], *grads[2:]), want):
        assert float((got.cpu().double() - ref).abs().max()) < 2000 * R.U * float(ref.abs().max())
    assert grads[1].shape == f.shape and bool(torch.isfinite(grads[1]).all()) and float(grads[1].abs().max()) > 0


# ---- saved tensors that come back as others -------------------------------------------------------------------------

SEEDED = {"group_norm": lambda t, seed: group_norm(t, 2, activation="silu", dropout_p=0.5, seed=seed, offset=3),
          "dropout": lambda t, seed: dropout(t, 0.5, seed, offset=3)}


def seeded_gradient(op, x, dy, seed, around=lambda f, t: f(t), before_backward=lambda: None):
    """d(op(x) dy) / dx, where `around` calls the operator and `before_backward` comes between the two passes"""
    xd = to_device(x).requires_grad_(True)
    y = around(lambda t: SEEDED[op](t, seed()), xd)
    before_backward()
    y.backward(to_device(dy))
    return xd.grad.cpu()


@pytest.mark.parametrize("op", list(SEEDED))
def test_checkpoint_of_a_call_whose_seed_tensor_is_let_go(gpu, op):
    gen = torch.Generator().manual_seed(6)
    x, dy = (torch.randn(2, 8, 5, 6, generator=gen) for _ in range(2))
    kept = []

    def refill():   # what the allocator hands out next lies where the seed was
        kept.extend(torch.full((1,), k, dtype=torch.int64, device=H.DEVICE) for k in range(500))

    want = seeded_gradient(op, x, dy, lambda: 1234567)
    got = seeded_gradient(op, x, dy, lambda: torch.tensor([1234567], device=H.DEVICE),
                          lambda f, t: checkpoint(f, t, use_reentrant=False), refill)
    assert torch.equal(got, want)


@pytest.mark.parametrize("op", list(SEEDED))
def test_a_saved_copy_of_the_seed_outlives_a_refill(gpu, op):
    gen = torch.Generator().manual_seed(7)
    x, dy = (torch.randn(2, 8, 5, 6, generator=gen) for _ in range(2))
    held = torch.tensor([77], device=H.DEVICE)

    def copied(f, t):
        with torch.autograd.graph.saved_tensors_hooks(lambda saved: saved.clone(), lambda saved: saved):
            return f(t)

    want = seeded_gradient(op, x, dy, lambda: 77)
    assert torch.equal(seeded_gradient(op, x, dy, lambda: held, copied, lambda: held.fill_(99)), want)


def test_saved_tensors_that_come_back_with_other_strides(gpu):
    """Hooks that keep values alone (as copies into pinned memory do): the input comes back row-major, and a slice of a wider map
    as a map of its own; parameters come back strided."""
    x, weight, bias, dy = make_case(2, 16, 9, 10, "fp32", 3)
    held = torch.tensor([4], device=H.DEVICE)

    def gradients(map_on_device, hooked):
        leaves = [t.requires_grad_(True) for t in (map_on_device(x), to_device(weight), to_device(bias))]
        pack = lambda t: t.clone(memory_format=torch.contiguous_format)  # noqa: E731
        unpack = lambda t: torch.stack((t, t), 1)[:, 0] if t.dim() == 1 else t  # noqa: E731
        with torch.autograd.graph.saved_tensors_hooks(*((pack, unpack) if hooked else (lambda t: t, lambda t: t))):
            y = group_norm(leaves[0], 4, *leaves[1:], activation="silu", dropout_p=0.2, seed=held)
        return torch.autograd.grad(y, leaves, to_device(dy))

    for map_on_device in (to_device, lambda t: to_device(torch.cat((t, t, t), 1))[:, 16:32], lambda t: to_device(t).contiguous()):
        want = gradients(map_on_device, False)
        for got, ref in zip(gradients(map_on_device, True), want):
            assert torch.equal(got, ref)


@pytest.mark.parametrize("which", ["input", "weight", "bias", "moments", "seed"])
def test_saved_tensors_that_come_back_as_something_else_are_refused(gpu, which):
    # in the order in which the operator saves them; sizes, types and places that the kernels would read past
    position = ["input", "weight", "bias", "moments", "seed"].index(which)
    x, weight, bias, dy = make_case(2, 8, 5, 6, "fp32", 3)
    held = torch.tensor([4], device=H.DEVICE)
    for changed in (lambda t: t[:0], lambda t: t.to(torch.bfloat16 if t.is_floating_point() else torch.int32), lambda t: t.to("meta")):
        packed = []

        def pack(t):
            packed.append(t)
            return len(packed) - 1

        leaves = [to_device(t).requires_grad_(True) for t in (x, weight, bias)]
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda i: changed(packed[i]) if i == position else packed[i]):
            y = group_norm(leaves[0], 2, *leaves[1:], dropout_p=0.5, seed=held)
        assert len(packed) == 5
        with pytest.raises(RuntimeError, match="unpacked"):
            torch.autograd.grad(y, leaves, to_device(dy))
        if which == "seed":
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, changed):
                y = dropout(leaves[0], 0.5, held)
            with pytest.raises(RuntimeError, match="unpacked"):
                torch.autograd.grad(y, leaves[0], to_device(dy))


# ---- refusals ------------------------------------------------------------------------------------------------------

def test_refusals(gpu):
    x = torch.randn(1, 6, 4, 4, device=H.DEVICE)
    w = torch.ones(6, device=H.DEVICE)
    for bad in (0, 4, -1, 2.0, True):
        with pytest.raises(ValueError, match="groups"):
            group_norm(x, bad)
    with pytest.raises(ValueError, match="dimensions"):
        group_norm(x[0], 2)
    with pytest.raises(ValueError, match="activation"):
        group_norm(x, 2, activation="tanh")
    with pytest.raises(ValueError, match="eps"):
        group_norm(x, 2, eps=float("nan"))
    with pytest.raises(ValueError, match="shape"):
        group_norm(x, 2, w[:5])
    with pytest.raises(ValueError, match="shape"):
        group_norm(x, 2, w, w[None])
    with pytest.raises(RuntimeError, match="scalar type"):
        group_norm(x, 2, w.double())
    with pytest.raises(RuntimeError, match="scalar type"):
        group_norm(x.half(), 2, w, w.half())
    with pytest.raises(RuntimeError, match="scalar type"):
        group_norm(x.half(), 2, w.bfloat16())
    with pytest.raises(RuntimeError, match="Float"):
        group_norm(x.double(), 2)
    with pytest.raises(ValueError, match="seed"):
        group_norm(x, 2, dropout_p=0.5)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError, match="0, 1"):
            dropout(x, p, 1)
        with pytest.raises(ValueError, match="0, 1"):
            group_norm(x, 2, dropout_p=p, seed=1)
    for seed in (None, -1, 2**64, 1.0, True):
        with pytest.raises(ValueError, match="seed"):
            dropout(x, 0.5, seed)
    for seed in (torch.ones(2, dtype=torch.int64, device=H.DEVICE), torch.ones(1, device=H.DEVICE)):
        with pytest.raises(RuntimeError, match="Long"):
            dropout(x, 0.5, seed)
    for offset in (-1, 2**64, 0.5):
        with pytest.raises(ValueError, match="offset"):
            dropout(x, 0.5, 1, offset)
    with pytest.raises(RuntimeError, match="Float"):
        dropout(torch.ones(4, dtype=torch.int32, device=H.DEVICE), 0.5, 1)
    # nothing differentiates these twice
    xg = x.clone().requires_grad_(True)
    for y in (group_norm(xg, 2, activation="silu"), dropout(xg, 0.5, 1)):
        (g,) = torch.autograd.grad(y.square().sum(), xg, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(g.sum(), xg)


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_is_refused(gpu, grad_mode):
    x, weight, bias, dy = (to_device(t) for t in make_case(1, 8, 4, 5, "fp32", 13))
    xg = x.clone().requires_grad_(grad_mode)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad_mode):
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for call in (lambda: dropout(dual(x), 0.5, 1), lambda: group_norm(dual(x), 2), lambda: dropout(dual(xg), 0.5, 1),
                     lambda: group_norm(x, 2, dual(weight), bias), lambda: group_norm(x, 2, weight, dual(bias)),
                     lambda: group_norm(xg, 2, dual(weight), bias)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        assert forward_ad.unpack_dual(dropout(dual(x), 0.0, None)).tangent is not None   # the input itself
        # no tangent, nothing to lose
        group_norm(x, 2, weight, bias), dropout(x, 0.5, 1)
        if grad_mode:   # forward over reverse
            for y in (group_norm(xg, 2, weight, bias), dropout(xg, 0.5, 1)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    torch.autograd.grad(y, xg, dual(dy))


@pytest.mark.parametrize("requires_grad", [True, False])
def test_recording_is_refused(gpu, requires_grad):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(1, 4, 3, 5, device=H.DEVICE, requires_grad=requires_grad)
    for call in (lambda t: dropout(t, 0.5, 1), lambda t: group_norm(t, 2)):
        with pytest.raises(RuntimeError, match="recorded"):
            make_fx(call)(x)
        with pytest.raises(RuntimeError, match="recorded"):
            torch.jit.trace(call, x, check_trace=False)
        y = call(x)
        if requires_grad:   # the backward pass alone
            with pytest.raises(RuntimeError, match="recorded"):
                make_fx(lambda dy: torch.autograd.grad(y, x, dy))(torch.ones_like(y))
    assert torch.equal(torch.jit.trace(lambda t: 2 * dropout(t, 0.5, None, training=False), x)(x), 2 * x)


# ---- on the device alone: graphs, streams, sizes -------------------------------------------------------------------

@pytest.mark.real_gpu
@pytest.mark.parametrize("dtype", ["fp32", "fp16"])
def test_captured_step_draws_a_new_mask_on_every_replay(gpu, dtype):
    x, weight, bias, dy = (to_device(t) for t in make_case(2, 32, 33, 29, dtype, 51))
    for t in (x, weight, bias):
        t.requires_grad_(True)
    held = torch.tensor([100], dtype=torch.int64, device=gpu)

    def step(seed):
        y = group_norm(x, 4, weight, bias, activation="silu", dropout_p=0.2, seed=seed, offset=7)
        out = dropout(y, 0.1, seed, offset=8)
        return (out, *torch.autograd.grad(out, (x, weight, bias), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [t.detach() for t in step(held)]
    for replay in range(4):
        held.fill_(1000 + replay)
        with torch.no_grad():
            x.copy_(torch.randn_like(x))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        eager = step(1000 + replay)
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b), replay


@pytest.mark.real_gpu
def test_two_captured_graphs_do_not_share_a_workspace(gpu):
    cases = [[to_device(t) for t in make_case(1, 16, 64 + 9 * k, 50, "fp16", 60 + k)] for k in range(2)]
    graphs, outputs = [], []
    for x, weight, bias, _ in cases:
        with torch.no_grad():
            group_norm(x, 4, weight, bias, activation="gelu")
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outputs.append(group_norm(x, 4, weight, bias, activation="gelu"))
            graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for (x, weight, bias, _), out in zip(cases, outputs):
            with torch.no_grad():
                assert torch.equal(out, group_norm(x, 4, weight, bias, activation="gelu"))


@pytest.mark.real_gpu
def test_calls_on_two_streams_at_once(gpu):
    cases = [[to_device(t) for t in make_case(1, 32, 300 + 50 * k, 400, "bf16", 70 + k)] for k in range(2)]
    want = []
    for x, weight, bias, dy in cases:
        x.requires_grad_(True)
        y = group_norm(x, 8, weight, bias, activation="silu", dropout_p=0.1, seed=3)
        want.append((y.detach(), *torch.autograd.grad(y, x, dy)))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in cases], [[], []]
    for _ in range(5):
        for k, (x, weight, bias, dy) in enumerate(cases):
            with torch.cuda.stream(streams[k]):
                y = group_norm(x, 8, weight, bias, activation="silu", dropout_p=0.1, seed=3)
                got[k].append((y.detach(), *torch.autograd.grad(y, x, dy)))
    torch.cuda.synchronize()
    for results, (y, dx) in zip(got, want):
        for a, b in results:
            assert torch.equal(a, y) and torch.equal(b, dx)


def large_step(n, c, h, w, groups, dtype, seed):
    """A training step of a map whose groups are too large for a block each: its slab sums lie in a workspace in both directions.
    Returns the input and step(seed of the mask), which gives the output and all gradients."""
    x, weight, bias, dy = (to_device(t) for t in make_case(n, c, h, w, dtype, seed))
    for t in (x, weight, bias):
        t.requires_grad_(True)

    def step(mask_seed):
        y = group_norm(x, groups, weight, bias, activation="silu", dropout_p=0.2, seed=mask_seed, offset=7)
        return (y, *torch.autograd.grad(y, (x, weight, bias), dy))

    with _lib.KernelTimer() as timer:
        group_norm(x.detach(), groups, weight, bias)
    assert "group_norm_moments" in [name for name, _ in timer.records]
    return x, step


LARGE_STEPS = [(1, 16, 200, 150, 4, "fp16"), (2, 24, 120, 95, 3, "fp32"), (2, 1030, 40, 11, 2, "bf16")]   # the last in parts


@pytest.mark.real_gpu
@pytest.mark.parametrize("shape", LARGE_STEPS, ids=str)
def test_captured_steps_of_large_groups(gpu, shape):
    """Two graphs, replayed on two streams at once, with eager steps and new inputs between the replays."""
    held = torch.tensor([100], dtype=torch.int64, device=gpu)
    graphs, kept = [], []
    for k in range(2):
        x, step = large_step(*shape, 80 + k)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(held)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = [t.detach() for t in step(held)]
        graphs.append(graph)
        kept.append((x, step, captured))
    streams = [torch.cuda.Stream() for _ in graphs]
    for replay in range(4):
        held.fill_(1000 + replay)
        with torch.no_grad():
            for x, _, _ in kept:
                x.copy_(torch.randn_like(x))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, step, captured in kept:
            got = [t.clone() for t in captured]
            eager = step(1000 + replay)
            torch.cuda.synchronize()
            for a, b in zip(got, eager):
                assert torch.equal(a, b), replay


@pytest.mark.real_gpu
@pytest.mark.parametrize("shape", LARGE_STEPS, ids=str)
def test_all_gradients_on_two_streams_at_once(gpu, shape):
    steps = [large_step(*shape, 90 + k)[1] for k in range(2)]
    want = [[t.detach().clone() for t in step(5)] for step in steps]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in steps], [[], []]
    for _ in range(5):
        for k, step in enumerate(steps):
            with torch.cuda.stream(streams[k]):
                got[k].append(step(5))
    torch.cuda.synchronize()
    for results, expected in zip(got, want):
        for result in results:
            for a, b in zip(result, expected):
                assert torch.equal(a, b)


@pytest.mark.real_gpu
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_a_16_bit_map_beyond_the_caches(gpu, dtype):
    """106 MB: results of both directions are stored past the caches."""
    gen = torch.Generator(device=gpu).manual_seed(6)
    x, dy = (torch.randn(1, 1300, 640, 64, generator=gen, device=gpu).to(DTYPES[dtype]).permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = (torch.randn(64, generator=gen, device=gpu) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (x, weight, bias)]
    y = group_norm(x, 8, weight, bias, activation="gelu")
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        ref = R.GroupNorm(x, 8, weight, bias, 1e-5, "gelu", None, dy)
        R.assert_within(y, ref.y, ref.y_bound, "y")
        for got, name in zip(grads, ("dx", "dweight", "dbias")):
            R.assert_within(got, getattr(ref, name), getattr(ref, name + "_bound"), name)


@pytest.mark.real_gpu
@pytest.mark.parametrize("pin_memory", [False, True])
def test_saved_tensors_on_the_host(gpu, pin_memory):
    x, weight, bias, dy = make_case(2, 16, 90, 101, "fp16", 33)
    held = torch.tensor([12], device=gpu)
    for map_on_device in (to_device, lambda t: to_device(torch.cat((t, t, t), 1))[:, 16:32]):
        results = []
        for on_host in (False, True):
            leaves = [t.requires_grad_(True) for t in (map_on_device(x), to_device(weight), to_device(bias))]
            with torch.autograd.graph.save_on_cpu(pin_memory) if on_host else torch.enable_grad():
                y = dropout(group_norm(leaves[0], 4, *leaves[1:], activation="silu", dropout_p=0.2, seed=held), 0.1, held, offset=1)
            results.append((y, *torch.autograd.grad(y, leaves, to_device(dy))))
        for a, b in zip(*results):
            assert torch.equal(a, b)


@pytest.mark.real_gpu
def test_more_than_two_to_the_32_values(gpu):
    # dropout: the block number passes 2^29, element numbers and byte offsets pass 2^32
    count, tail = 2**32 + 2**20 + 5, 5000
    x = torch.ones(count, dtype=torch.float16, device=gpu)
    y = dropout(x, 0.5, 12, offset=4)
    want = R.dropout(torch.ones(tail, dtype=torch.float16), 0.5, 12, 4, first=count - tail)
    assert torch.equal(y[count - tail:].cpu(), want)
    del x, y
    # group norm: the last image starts behind 2^32 values
    n, c, h, w = 5, 64, 4100, 4100
    x = torch.zeros((n, h, w, c), dtype=torch.bfloat16, device=gpu).permute(0, 3, 1, 2)
    x[-1].normal_(generator=torch.Generator(device=gpu).manual_seed(1))
    assert (n - 1) * c * h * w > 2**32
    y = group_norm(x, 4, activation="silu", dropout_p=0.5, seed=12, offset=4)
    assert not y[:-1].any()
    rows = 3   # the last rows of the last image, from the moments torch computes in 64 bits a channel at a time
    for group in (0, 3):
        v = x[-1, 16 * group:16 * group + 16]
        mean = float(torch.stack([t.double().mean() for t in v]).mean())
        var = float(torch.stack([((t.double() - mean) ** 2).mean() for t in v]).mean())
        z = (v[:, -rows:].double().cpu() - mean) / (var + 1e-5) ** 0.5
        first = ((n - 1) * h + h - rows) * w * c
        keep = torch.from_numpy(R.kept(first, rows * w * c, 0.5, 12, 4)).view(rows, w, c)[:, :, 16 * group:16 * group + 16]
        ref = R.activation(z, "silu") * keep.permute(2, 0, 1) * 2.0
        # moments of 16.8 million pixels: a chain of up to 2^12 roundings, and half a step of bf16
        R.assert_within(y[-1, 16 * group:16 * group + 16, -rows:], ref, 4096 * R.U * (z.abs() + 1) + 2.0**-8 * ref.abs(), "y")


@pytest.mark.real_gpu
def test_an_outlier_in_front_of_long_runs(gpu):
    """512 images, so that a block has a whole one and a thread 512 vectors (2.1 GB): two of them against the reference."""
    x = torch.randn(512, 64, 128, 128, generator=torch.Generator(device=gpu).manual_seed(2), device=gpu).permute(0, 3, 1, 2)
    x[:, ::4, 0, 0] = 3e4
    y = group_norm(x, 32)
    for image in (0, 511):
        ref = R.GroupNorm(x[image:image + 1].cpu(), 32, None, None, 1e-5, "none")
        R.assert_within(y[image:image + 1], ref.y, ref.y_bound, "y")


@pytest.mark.real_gpu
def test_wide_groups_of_more_images_than_parts_have_blocks(gpu):
    """65600 images of one pixel, 65535 channels each, in one group: a block for each, and more than 2^32 values in both directions."""
    n, c = 65600, 65535
    assert n * c > 2**32
    gen = torch.Generator(device=gpu).manual_seed(4)
    x, dy = (torch.empty(n, c, dtype=torch.float16, device=gpu).normal_(generator=gen).view(n, c, 1, 1) for _ in range(2))
    x.requires_grad_(True)
    y = group_norm(x, 1, activation="silu", dropout_p=0.25, seed=7)
    (dx,) = torch.autograd.grad(y, x, dy)
    for image in (0, 40000, n - 1):
        keep = torch.from_numpy(R.kept(image * c, c, 0.25, 7, 0)).view(1, c, 1, 1).double() / 0.75
        part = slice(image, image + 1)
        ref = R.GroupNorm(x[part].detach().cpu(), 1, None, None, 1e-5, "silu", keep, dy[part].cpu())
        R.assert_within(y[part], ref.y, ref.y_bound, "y")
        R.assert_within(dx[part], ref.dx, ref.dx_bound, "dx")


@pytest.mark.real_gpu
def test_gradients_of_more_than_two_to_the_32_values(gpu):
    """Five images of 4100x4100x64 bf16. A channel's gradients are sums over 84 million pixels: a thread's own run (512 at most), the
    block's 64 rows, 2600 slabs by 16 threads and those: not 1000 roundings one after the other."""
    roundings = 1000
    n, c, h, w = 5, 64, 4100, 4100
    x, dy = (torch.zeros((n, h, w, c), dtype=torch.bfloat16, device=gpu).permute(0, 3, 1, 2) for _ in range(2))
    weight = torch.ones(c, device=gpu).requires_grad_(True)
    bias = torch.zeros(c, device=gpu).requires_grad_(True)
    # Equal values, 0.1 times the slope at 0.3, which fills the mantissa. Within a binade of its sum every addition of a chain of L is off
    # by the same amount, half a step at most: 2/3 L u 2^k where the sum ends at 2^k + 2^k, so L u / 3, and 0.37 L u where it ends half-way
    # to there. With runs of 512 and 163 slabs to a thread, and 16 u for the slope, the joins and the store: 266 u.
    dy.fill_(0.1)
    at = torch.full((c,), 0.3, device=gpu).requires_grad_(True)
    (dbias,) = torch.autograd.grad(group_norm(x, 4, weight, at, activation="silu"), at, dy)
    each = float(dy[0, 0, 0, 0]) * R.slope(at.detach().cpu().double(), "silu")
    R.assert_within(dbias, n * h * w * each, 266 * R.U * n * h * w * each, "dbias of equal values")
    # the last image alone: its values start behind 2^32
    gen = torch.Generator(device=gpu).manual_seed(1)
    dy.zero_()
    x[-1].normal_(generator=gen)
    dy[-1].normal_(generator=gen)
    x.requires_grad_(True)
    dx, dweight, dbias = torch.autograd.grad(group_norm(x, 4, weight, bias, activation="silu"), (x, weight, bias), dy)
    assert not dx[:-1].any()
    for group in (0, 3):
        part = slice(16 * group, 16 * group + 16)
        with torch.no_grad():
            ref = R.GroupNorm(x[-1:, part], 1, None, None, 1e-5, "silu", None, dy[-1:, part])
        more = roundings / (32 + 8 * 16 + 256 / 16)   # than the reference allows for
        R.assert_within(dx[-1:, part], ref.dx, more * ref.dx_bound, "dx")
        R.assert_within(dweight[part], ref.dweight, more * ref.dweight_bound, "dweight")
        R.assert_within(dbias[part], ref.dbias, more * ref.dbias_bound, "dbias")
        del ref


@pytest.mark.real_gpu
def test_slab_sums_of_two_images_and_tiles_in_a_launch_of_their_own(gpu):
    """Two images of 4200x4200x64 fp16 in 64 groups, two tiles of 32 with 384 slabs each: more sums than every block adds up itself. Longest way
    of a value: a run of 512, a block's 128 rows, 384 slabs by 64 lanes: not 1000 roundings."""
    roundings, n, c, h, w = 1000, 2, 64, 4200, 4200
    gen = torch.Generator(device=gpu).manual_seed(5)
    x, dy = (torch.empty(n, h, w, c, dtype=torch.float16, device=gpu).normal_(generator=gen).permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = (torch.randn(c, generator=gen, device=gpu).requires_grad_(True) for _ in range(2))
    x.requires_grad_(True)
    with _lib.KernelTimer() as timer:
        y = group_norm(x, 64, weight, bias, activation="silu")
    assert [name for name, _ in timer.records] == ["group_norm_moments", "group_norm_combine_moments", "group_norm_apply"]
    dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), dy)
    for channel in (0, 31, 32, 63):
        part = slice(channel, channel + 1)
        with torch.no_grad():
            ref = R.GroupNorm(x[:, part], 1, weight[part], bias[part], 1e-5, "silu", None, dy[:, part])
        more = roundings / (32 + 8 + 256)   # than the reference allows for
        R.assert_within(y[:, part], ref.y, more * ref.y_bound, "y")
        R.assert_within(dx[:, part], ref.dx, more * ref.dx_bound, "dx")
        R.assert_within(dweight[part], ref.dweight, more * ref.dweight_bound, "dweight")
        R.assert_within(dbias[part], ref.dbias, more * ref.dbias_bound, "dbias")


@pytest.mark.real_gpu
def test_a_map_beyond_the_caches(gpu):
    """A map of 102 MB in 20 groups: more slab sums than every block adds up itself, and results that are stored past the caches."""
    gen = torch.Generator(device=gpu).manual_seed(3)
    x, dy = (torch.randn(1, 800, 800, 40, generator=gen, device=gpu).permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = (torch.randn(40, generator=gen, device=gpu) for _ in range(2))
    leaves = [t.requires_grad_(True) for t in (x, weight, bias)]
    y = group_norm(x, 20, weight, bias, activation="silu")
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        ref = R.GroupNorm(x, 20, weight, bias, 1e-5, "silu", None, dy)
        R.assert_within(y, ref.y, ref.y_bound, "y")
        for got, name in zip(grads, ("dx", "dweight", "dbias")):
            R.assert_within(got, getattr(ref, name), getattr(ref, name + "_bound"), name)

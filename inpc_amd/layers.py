"""Layers for networks on either side of the rasterizer: group norm with an activation over channels-last feature
maps (with dropout behind it if asked for), and dropout from a counter-based generator. Neither is among the reference's
operators; they are for networks that a user trains in the places of Modules/UNet.py:1-200 and Modules/AppearanceField.py:1-88.
Both compute in fp32, run as hand-written kernels in both directions and keep neither normalised values nor masks for the
backward pass.
"""
from __future__ import annotations

import ctypes as C
from typing import Any

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16, torch.bfloat16: _lib.DTYPE_BF16}
_ACTIVATIONS = {"none": _lib.ACTIVATION_NONE, "relu": _lib.ACTIVATION_RELU, "silu": _lib.ACTIVATION_SILU,
                "gelu": _lib.ACTIVATION_GELU}


_current_device, _stream_of = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _run(name: str, t: torch.Tensor, *args) -> None:
    """Calls the library with `args` and the current stream of the device that `t` lies on. The library launches on the
    current device, so that is made the tensor's. Where it is already, device and stream are asked for without the layers that
    torch.cuda puts around them (1 us of a small call's 10)."""
    function, index = getattr(_lib.lib(), name), t.get_device()
    if index < 0:
        _lib.check(function(*args, _lib.current_stream()), name)
    elif index == _current_device():
        _lib.check(function(*args, _stream_of(index)), name)
    else:
        with torch.cuda.device(index):
            _lib.check(function(*args, _stream_of(index)), name)


def _address(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


_tracing_state, _dispatch_mode, _PROXY = torch._C._get_tracing_state, torch._C._get_dispatch_mode, torch._C._TorchDispatchModeKey.PROXY


def _require_plain_call(a: torch.Tensor, b: torch.Tensor | None = None, c: torch.Tensor | None = None, d: torch.Tensor | None = None) -> None:
    """Refuses what torch does around its own operators and would leave a kernel out of. The kernels compute no forward-mode
    derivatives, and what they write carries none; a recorded call would replay the allocation of the result alone."""
    if forward_ad._current_level >= 0:   # no dual tensors outside of a level: that alone is asked in most calls (0.07 us)
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in (a, b, c, d)):
            raise RuntimeError("group_norm and dropout have no forward-mode derivative")
    if _tracing_state() is not None or _dispatch_mode(_PROXY) is not None:
        raise RuntimeError("group_norm and dropout cannot be recorded by torch.jit.trace or make_fx; capture a CUDA graph instead")


def _require_values(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"expected {name} to be a tensor on the GPU")
    if t.dtype not in _DTYPES:
        raise RuntimeError(f"expected {name} of scalar type Float, Half or BFloat16, got {t.dtype}")


def _require_probability(p: float, name: str) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"{name} must lie in [0, 1], got {p}")
    return p


def _require_seed(seed: int | torch.Tensor | None, offset: int, device: torch.device) -> tuple[int, torch.Tensor | None, int]:
    """(seed, its place on the GPU or None, offset)"""
    if isinstance(offset, bool) or not isinstance(offset, int) or not 0 <= offset < 2**64:
        raise ValueError("offset must be a whole number in [0, 2^64)")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1 or seed.device != device:
            raise RuntimeError("a seed tensor holds one Long on the device of the input")
        return 0, seed.view(1), offset
    if seed is None or isinstance(seed, bool) or not isinstance(seed, int) or not 0 <= seed < 2**64:
        raise ValueError("dropout needs a seed: a whole number in [0, 2^64) or a tensor that holds one")
    return seed, None, offset


def _unpacked(t: torch.Tensor | None, count: int, dtype: torch.dtype, device: torch.device) -> torch.Tensor | None:
    """A saved vector as the kernels read it. A hook on saved tensors gives back what it likes, and the kernels go by the forward
    pass's sizes and types."""
    if t is None:
        return None
    if t.numel() != count or t.dtype != dtype or t.device != device:
        raise RuntimeError(f"a saved vector, {count} of {dtype} on {device}, was unpacked as {t.numel()} of {t.dtype} on {t.device}")
    return t if t.is_contiguous() else t.contiguous()


# ---- dropout -------------------------------------------------------------------------------------------------------

def _memory_format(t: torch.Tensor) -> torch.memory_format:
    """The order in which a tensor's elements are numbered: channels last where that is how it lies in memory."""
    if t.dim() == 4 and not t.is_contiguous() and t.is_contiguous(memory_format=torch.channels_last):
        return torch.channels_last
    return torch.contiguous_format


def _dropout_call(x: torch.Tensor, p: float, seed: int, seed_tensor: torch.Tensor | None, offset: int) -> torch.Tensor:
    out = torch.empty_like(x)
    _run("inpc_dropout", x, x.data_ptr(), out.data_ptr(), x.numel(), _DTYPES[x.dtype], p, seed, _address(seed_tensor), offset)
    return out


def _dropout_backward(ctx: Any, grad: torch.Tensor):
    _require_plain_call(grad)
    p, seed, seed_tensor, offset = ctx.random
    if seed is None:
        (seed_tensor,) = ctx.saved_tensors   # torch refuses one that has changed; a hook's copy keeps its value
        seed, seed_tensor = 0, _unpacked(seed_tensor, 1, torch.int64, grad.device)
    return _dropout_call(grad.contiguous(memory_format=ctx.order), p, seed, seed_tensor, offset), None, None


# Under create_graph the result must refuse to be differentiated again; otherwise that wrapper's few microseconds are saved.
_dropout_backward_once = once_differentiable(_dropout_backward)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, order: torch.memory_format, random: tuple) -> torch.Tensor:
        ctx.order, ctx.random = order, random
        if random[2] is not None:
            ctx.save_for_backward(random[2])   # torch watches over it
            ctx.random = random[0], None, None, random[3]
        return _dropout_call(x, *random)

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor):
        return (_dropout_backward_once if torch.is_grad_enabled() else _dropout_backward)(ctx, grad)


def dropout(input: torch.Tensor, p: float, seed: int | torch.Tensor | None, offset: int = 0, training: bool = True) -> torch.Tensor:
    """Zeroes each element of `input` with probability `p` and divides the others by 1 - p; differentiable.

    The mask is a function of `seed`, `offset` and an element's number in memory order alone (channels-last tensors
    are numbered that way, all others row-major; tensors that are neither are made contiguous first) and is stored nowhere: the
    backward pass computes it again. Calls with different `seed` or `offset` draw independent masks, so use one seed for
    a training run and step the offset from layer to layer, and another seed for each iteration. `seed` is a whole
    number or a GPU tensor of one int64, which is read when the kernel runs (in a captured graph: on every
    replay); torch refuses a backward pass if that tensor has been changed in between, and under hooks on saved tensors
    (torch.utils.checkpoint, save_on_cpu) the saved value counts. The generator is Philox4x32-10; include/inpc_hip.h
    (inpc_dropout) gives the numbering of its bits. With training=False or p = 0, `input` itself is returned. Second and
    forward-mode derivatives are refused, and so is recording by torch.jit.trace or make_fx.
    """
    _require_values(input, "input")
    p = _require_probability(p, "p")
    if not training or p == 0.0:
        return input
    _require_plain_call(input)
    random = (p, *_require_seed(seed, offset, input.device))
    order = _memory_format(input)
    input = input.contiguous(memory_format=order)
    if torch.is_grad_enabled() and input.requires_grad:
        return _Dropout.apply(input, order, random)
    return _dropout_call(input, *random)


# ---- group norm ----------------------------------------------------------------------------------------------------

def _pixel_strides(t: torch.Tensor) -> tuple[int, int] | None:
    """(from image to image, from pixel to pixel) of a (N, C, H, W) tensor whose channels are adjacent and whose pixels lie
    evenly spaced; None where it lies otherwise. Strides of dimensions of size one mean nothing."""
    n, c, h, w = t.shape
    s_n, s_c, s_h, s_w = t.stride()
    if s_c == 1 and s_w == c and s_h == w * c and s_n == h * w * c:   # dense
        return s_n, c
    if c != 1 and s_c != 1:
        return None
    if w != 1:
        pixel = s_w
        if h != 1 and s_h != w * s_w:
            return None
    else:
        pixel = s_h if h != 1 else c
    image = s_n if n != 1 else h * w * pixel
    if pixel < c or image < h * w * pixel or pixel >= 2**19:   # overlapping, expanded, or beyond the kernels' offsets
        return None
    return image, pixel


def _dense(like: torch.Tensor) -> torch.Tensor:
    """An uninitialised (N, C, H, W) tensor that lies as (N, H, W, C)."""
    n, c, h, w = like.shape
    return torch.empty_strided((n, c, h, w), (h * w * c, 1, w * c, c), dtype=like.dtype, device=like.device)


def _channels_last(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """The tensor, copied to a dense channels-last one where the kernels cannot read it as it lies, and its strides."""
    strides = _pixel_strides(t)
    if strides is None:
        t = _dense(t).copy_(t)
        strides = _pixel_strides(t)
    return t, *strides


def _workspace(cfg: _lib.GroupNormConfig, backward: int, device: torch.device) -> tuple[torch.Tensor | None, int]:
    size = _lib.lib().inpc_group_norm_workspace_bytes(C.byref(cfg), backward)
    return (torch.empty(size, dtype=torch.uint8, device=device) if size else None), size


def _group_norm_call(x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, groups: int, eps: float,
                     activation: int, p: float, seed: int, seed_tensor: torch.Tensor | None, offset: int):
    """(output, the input as the kernels have read it, moments, configuration)"""
    x, image_stride, pixel_stride = _channels_last(x)
    n, c, h, w = x.shape
    param = weight if weight is not None else bias
    cfg = _lib.GroupNormConfig(n, h * w, c, groups, _DTYPES[x.dtype], _lib.DTYPE_F32 if param is None else _DTYPES[param.dtype],
                               activation, eps, image_stride, pixel_stride, 0, 0, p, seed, _address(seed_tensor), offset)
    y = _dense(x)
    moments = torch.empty(2 * n * groups, dtype=torch.float32, device=x.device)
    workspace, size = _workspace(cfg, 0, x.device)
    _run("inpc_group_norm_forward", x, C.byref(cfg), x.data_ptr(), _address(weight), _address(bias), y.data_ptr(),
         moments.data_ptr(), _address(workspace), size)
    return y, x, moments, cfg


def _require_parameter(t: torch.Tensor, name: str, channels: int, input: torch.Tensor) -> torch.Tensor:
    if t.dim() != 1 or t.shape[0] != channels:
        raise ValueError(f"expected {name} of shape ({channels},), got {tuple(t.shape)}")
    if t.dtype != torch.float32 and t.dtype != input.dtype:
        raise RuntimeError("weight and bias have one scalar type, Float or that of the input")
    if t.device != input.device:
        raise RuntimeError("expected all tensors on the same device")
    return t.contiguous()


def _group_norm_backward(ctx: Any, grad: torch.Tensor):
    x, weight, bias, moments, seed_tensor = ctx.saved_tensors
    _require_plain_call(grad, x, weight, bias)
    cfg = _lib.GroupNormConfig.from_buffer_copy(ctx.cfg)   # two backward passes of one forward pass may run at once
    # Hooks on saved tensors may give back others than the forward pass's, which lie elsewhere and with other strides.
    device, (param_dtype, strides) = grad.device, ctx.saved_as
    if x.shape != grad.shape or x.dtype != grad.dtype or x.device != device:
        raise RuntimeError(f"the saved input, {tuple(grad.shape)} of {grad.dtype} on {device}, was unpacked as {tuple(x.shape)} of {x.dtype} "
                           f"on {x.device}")
    if x.stride() != strides:
        x, cfg.input_image_stride, cfg.input_pixel_stride = _channels_last(x)
    weight = _unpacked(weight, cfg.channels, param_dtype, device)
    bias = _unpacked(bias, cfg.channels, param_dtype, device)
    moments = _unpacked(moments, 2 * cfg.n_images * cfg.groups, torch.float32, device)
    seed_tensor = _unpacked(seed_tensor, 1, torch.int64, device)
    cfg.seed_dev = _address(seed_tensor)
    grad, cfg.grad_image_stride, cfg.grad_pixel_stride = _channels_last(grad)
    need_x, need_weight, need_bias, _ = ctx.needs_input_grad
    dx = _dense(x) if need_x else None
    dweight = torch.empty_like(weight) if need_weight else None
    dbias = torch.empty_like(bias) if need_bias else None
    workspace, size = _workspace(cfg, 1, x.device)
    _run("inpc_group_norm_backward", x, C.byref(cfg), grad.data_ptr(), x.data_ptr(), _address(weight), _address(bias),
         moments.data_ptr(), _address(dx), _address(dweight), _address(dbias), _address(workspace), size)
    return dx, dweight, dbias, None


_group_norm_backward_once = once_differentiable(_group_norm_backward)


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, options: tuple) -> torch.Tensor:
        y, x, moments, ctx.cfg = _group_norm_call(x, weight, bias, *options)
        ctx.save_for_backward(x, weight, bias, moments, options[5])   # the last: a seed on the GPU, which torch watches over
        ctx.saved_as = (weight.dtype if weight is not None else bias.dtype if bias is not None else None), x.stride()
        return y

    @staticmethod
    def backward(ctx: Any, grad: torch.Tensor):
        return (_group_norm_backward_once if torch.is_grad_enabled() else _group_norm_backward)(ctx, grad)


def group_norm(input: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, activation: str = "none", dropout_p: float = 0.0, seed: int | torch.Tensor | None = None,
               offset: int = 0, training: bool = True) -> torch.Tensor:
    """Group norm of a (N, C, H, W) feature map, then an activation ("none", "relu", "silu" or "gelu", the exact one), then
    dropout where dropout_p > 0; differentiable in `input`, `weight` and `bias`.

    The kernels work on channels-last maps (torch.channels_last, also a slice of the channels of a wider one); other
    layouts are copied into that first. The result is a dense channels-last tensor of the input's type. `weight` and
    `bias` are (C,) tensors of one type, fp32 or the input's, so fp32 parameters serve 16-bit maps. Everything is
    computed in fp32 and rounded once, at the end of the whole chain. `dropout_p`, `seed`, `offset` and `training` are
    those of `dropout`, which gives the same mask for the same map. For the backward pass only the input and two
    numbers per image and group are kept. What `dropout` refuses is refused here too.
    """
    _require_values(input, "input")
    if input.dim() != 4:
        raise ValueError(f"expected a (N, C, H, W) tensor, got {input.dim()} dimensions")
    channels = input.shape[1]
    if input.shape[2] * input.shape[3] >= 2**30 or input.shape[0] >= 2**31:
        raise ValueError("expected fewer than 2^30 pixels per image and fewer than 2^31 images")
    if isinstance(num_groups, bool) or not isinstance(num_groups, int) or num_groups < 1 or channels < 1 or channels % num_groups != 0:
        raise ValueError(f"{channels} channels cannot be split into {num_groups} groups")
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; choose from {', '.join(_ACTIVATIONS)}")
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    if weight is not None:
        weight = _require_parameter(weight, "weight", channels, input)
    if bias is not None:
        bias = _require_parameter(bias, "bias", channels, input)
        if weight is not None and weight.dtype != bias.dtype:
            raise RuntimeError("weight and bias have one scalar type, Float or that of the input")
    _require_plain_call(input, weight, bias)
    p = _require_probability(dropout_p, "dropout_p") if training else 0.0
    seed, seed_tensor, offset = _require_seed(seed, offset, input.device) if p > 0.0 else (0, None, 0)
    options = num_groups, float(eps), _ACTIVATIONS[activation], p, seed, seed_tensor, offset
    if torch.is_grad_enabled() and (input.requires_grad or (weight is not None and weight.requires_grad)
                                    or (bias is not None and bias.requires_grad)):
        return _GroupNorm.apply(input, weight, bias, options)
    return _group_norm_call(input, weight, bias, *options)[0]

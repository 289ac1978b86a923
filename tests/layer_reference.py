"""Group norm with an activation and counter-based dropout in 64 bits, plainly, with the error bounds that the tests of
inpc_amd/layers.py hold the kernels to."""
from __future__ import annotations

import math

import numpy as np
import torch

U = 2.0**-24   # half a step of fp32


# ---- the generator -------------------------------------------------------------------------------------------------

def philox(blocks: np.ndarray, draw: int, offset: int, seed: int) -> np.ndarray:
    """(len(blocks), 4) uint64 in [0, 2^32): Philox4x32-10 of each block's counter."""
    m = np.uint64(0xFFFFFFFF)
    shift = np.uint64(32)
    blocks = blocks.astype(np.uint64)
    c = [blocks & m, (blocks >> shift) + np.uint64(draw << 31), np.full_like(blocks, offset & 0xFFFFFFFF),
         np.full_like(blocks, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k0), b & m, (a >> shift) ^ c[3] ^ np.uint64(k1), a & m]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def halves(first: int, count: int, draw: int, offset: int, seed: int) -> np.ndarray:
    """The 16-bit halves of elements first .. first + count - 1."""
    number = np.arange(first, first + count, dtype=np.uint64)
    base = first // 8
    words = philox(np.arange(base, (first + count + 7) // 8, dtype=np.uint64), draw, offset, seed)
    lane = (number % np.uint64(8)).astype(np.int64)
    word = words[(number // np.uint64(8)).astype(np.int64) - base, lane // 2]
    return ((word >> (16 * (lane % 2)).astype(np.uint64)) & np.uint64(0xFFFF)).astype(np.int64)


def kept(first: int, count: int, p: float, seed: int, offset: int) -> np.ndarray:
    """True where the element stays."""
    u = halves(first, count, 0, offset, seed) * 65536 + halves(first, count, 1, offset, seed)
    return u >= round(p * 2**32)


def dropout(x: torch.Tensor, p: float, seed: int, offset: int = 0, first: int = 0) -> torch.Tensor:
    """What the operator gives for the elements of x in memory order, bit for bit: an fp32 product rounded once."""
    mask = torch.from_numpy(kept(first, x.numel(), p, seed, offset)).view(x.shape)
    scale = torch.tensor(1.0 / (1.0 - p) if p < 1.0 else 0.0, dtype=torch.float32)
    return torch.where(mask, x.float() * scale, torch.zeros((), dtype=torch.float32)).to(x.dtype)


# ---- group norm ----------------------------------------------------------------------------------------------------

def activation(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros((), dtype=z.dtype))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2.0))
    return z


def slope(z: torch.Tensor, name: str) -> torch.Tensor:
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2.0)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


class GroupNorm:
    """Forward and, given dy, backward pass in 64 bits from the formulas, and bounds on what fp32 arithmetic may add.

    Bounds, with u = 2^-24 and D roundings on the longest way of a value through a sum (a thread's own pixels, the block's
    halving, a group's partial sums: the kernels' sums are at most 32 + 8 * per_group + 256 / per_group deep for the
    sizes here: up to 2048 slabs): a mean is off by D u max|x|, a standard deviation by the relative D u, so
      xhat by E_x = D u (rstd max|x| + |xhat| + 1), z by E_z = |w| E_x + 2 u (|z| + |w xhat|), and y by 1.13 E_z (no slope
      exceeds 1.13) plus the activation's own 8 u (|z| + 1): a few roundings of exp, 1 / (1 + e) and erf. dz takes over z's error
      by the activation's second derivative (below 1 everywhere) and the same 8 u. The sums' errors are
      D u times the sum of magnitudes plus the errors of their terms.
    Rounding the result adds half a step of its type and, for fp16, half of its smallest value 2^-24."""

    def __init__(self, x, groups, weight, bias, eps, act, keep=None, dy=None):
        n, c, h, w = x.shape
        self.shape, self.dtype = x.shape, x.dtype
        per_group = c // groups
        D = 32 + 8 * per_group + 256 / per_group
        split = lambda t: t.double().permute(0, 2, 3, 1).reshape(n, h * w, groups, per_group)  # noqa: E731
        whole = lambda t: t.reshape(n, h, w, c).permute(0, 3, 1, 2)  # noqa: E731
        wt = (x.new_ones(c) if weight is None else weight).double().view(groups, per_group)
        bs = (x.new_zeros(c) if bias is None else bias).double().view(groups, per_group)
        param = next((t.dtype for t in (weight, bias) if t is not None), torch.float32)
        v = split(x)
        mean = v.mean(dim=(1, 3), keepdim=True)
        rstd = 1 / torch.sqrt(((v - mean) ** 2).mean(dim=(1, 3), keepdim=True) + eps)
        xhat = (v - mean) * rstd
        z = xhat * wt + bs
        scale = torch.ones_like(z) if keep is None else split(keep.double())
        e_x = D * U * (rstd * v.abs().amax(dim=(1, 3), keepdim=True) + xhat.abs() + 1)
        e_z = wt.abs() * e_x + 2 * U * (z.abs() + (wt * xhat).abs())
        y = activation(z, act) * scale
        self.y = whole(y)
        self.y_bound = whole((1.13 * e_z + 8 * U * (z.abs() + 1)) * scale + 2 * U * y.abs()) + self._rounding(self.y, x.dtype)
        self.z, self.z_bound = whole(z), whole(e_z)
        if dy is None:
            return
        g = split(dy) * scale
        dz = g * slope(z, act)
        e_dz = g.abs() * (e_z + 8 * U * (z.abs() + 1)) + 4 * U * dz.abs()
        dn, e_dn = wt * dz, wt.abs() * e_dz + U * (wt * dz).abs()
        mean_of = lambda t: t.mean(dim=(1, 3), keepdim=True)  # noqa: E731
        a, b = mean_of(dn), mean_of(dn * xhat)
        e_a = D * U * mean_of(dn.abs()) + mean_of(e_dn)
        e_b = D * U * mean_of((dn * xhat).abs()) + mean_of(e_dn * xhat.abs() + dn.abs() * e_x)
        self.dx = whole(rstd * (dn - a - xhat * b))
        e_dx = rstd * (e_dn + e_a + xhat.abs() * e_b + e_x * b.abs() + (D + 4) * U * (dn.abs() + a.abs() + (xhat * b).abs()))
        self.dx_bound = whole(e_dx) + self._rounding(self.dx, x.dtype)
        total = lambda t: t.sum(dim=(0, 1)).reshape(c)  # noqa: E731
        self.dbias, self.dweight = total(dz), total(dz * xhat)
        self.dbias_bound = total(e_dz + D * U * dz.abs()) + self._rounding(self.dbias, param)
        self.dweight_bound = (total(e_dz * xhat.abs() + dz.abs() * e_x + D * U * (dz * xhat).abs())
                              + self._rounding(self.dweight, param))

    @staticmethod
    def _rounding(values, dtype):
        return torch.finfo(dtype).eps / 2 * values.abs() + (2.0**-25 if dtype == torch.float16 else 0.0)


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    off = (got.detach().to(want.device).double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} values outside their bound; worst {float((off / bound).max()):.3g} "
                           f"times it")

"""The image-space and point-feature operators as a program calls them, and their plain forms.

Two operators: `group_norm` (group norm with an activation over channels-last feature maps, the layers of the network
that takes the rasterizer's images, optionally with dropout behind the activation) and `dropout` (from a counter-based
generator; the mask is a function of seed, offset and element number and is stored nowhere). A case is one call:
forward alone ("infer"), or forward and backward with all gradients ("train").

    z = (x - mean) / sqrt(var + eps) * weight + bias     mean, var over the pixels and the channels of a group
    y = activation(z)
    dropped(i) = u(i) < round(p * 2^32)                  i: number of the element in memory order (N, H, W, C)
    out = 0 where dropped, else y / (1 - p)

    u(i) = h(0, i) * 2^16 + h(1, i); h(d, i) is the 16-bit half i % 8 (low half first) of the four 32-bit words of
    Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011) with the key `seed` and the
    counter (b mod 2^32, b div 2^32 + 2^31 d, offset mod 2^32, offset div 2^32), b = i div 8.
"""
import math

import torch

own = False

EPS = 1e-5
DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
M32 = 0xFFFFFFFF


# The cases use smooth activations: which side of a ReLU's border a value next to it falls on is a matter of the last bit of
# z, and decides its whole gradient.

def listed():
    norm = dict(op="norm", p=0.0, slice_of=0, device_seed=False)
    drop = dict(op="dropout", device_seed=False)
    return [
        # the deepest feature map of a 256x256 view: the call's own latency counts
        dict(norm, name="norm_infer_16x16x64_fp16", mode="infer", n=1, c=64, h=16, w=16, groups=8, act="silu", dtype="fp16"),
        # a rendered frame of 2473x1643 padded to multiples of four, first layer, no gradients
        dict(norm, name="norm_infer_2476x1644x16_fp16", mode="infer", n=1, c=16, h=1644, w=2476, groups=4, act="silu",
             dtype="fp16"),
        # a training view of 1237x822 padded to multiples of four, first layer
        dict(norm, name="norm_train_1240x824x32_fp16", mode="train", n=1, c=32, h=824, w=1240, groups=8, act="silu",
             dtype="fp16"),
        # the same view one level down; the input is the skip half of a concatenated map of twice the channels
        dict(norm, name="norm_train_620x412x64_bf16_slice", mode="train", n=1, c=64, h=412, w=620, groups=32, act="silu",
             dtype="bf16", slice_of=128),
        # a batch of deep maps: little per image, many channels
        dict(norm, name="norm_train_39x26x256_bf16_b8", mode="train", n=8, c=256, h=26, w=39, groups=32, act="gelu",
             dtype="bf16"),
        # full precision, odd image sizes, a group of eight channels that is no power of two of the row
        dict(norm, name="norm_train_317x203x24_fp32", mode="train", n=2, c=24, h=203, w=317, groups=3, act="silu", dtype="fp32"),
        # channels that do not fill vectors: six to a group, rows of sixty bytes
        dict(norm, name="norm_train_77x101x30_bf16_b3", mode="train", n=3, c=30, h=101, w=77, groups=5, act="none", dtype="bf16"),
        # a residual block in training: norm, activation and dropout in one call; the seed lives on the GPU
        dict(norm, name="norm_dropout_train_310x206x128_fp16", mode="train", n=1, c=128, h=206, w=310, groups=16, act="silu",
             dtype="fp16", p=0.1, device_seed=True),
        # the same on a small crop
        dict(norm, name="norm_dropout_train_64x64x32_fp32", mode="train", n=1, c=32, h=64, w=64, groups=8, act="silu",
             dtype="fp32", p=0.25),
        # a ragged handful of values
        dict(drop, name="dropout_train_10007_fp32", mode="train", count=10007, dtype="fp32", p=0.1),
        # the feature map of a training view
        dict(drop, name="dropout_train_1240x824x32_fp16", mode="train", count=1240 * 824 * 32, dtype="fp16", p=0.3,
             device_seed=True),
        # the hidden features of a training draw of 8,388,352 points, 64 each
        dict(drop, name="dropout_train_8388352x64_bf16", mode="train", count=8388352 * 64, dtype="bf16", p=0.5),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    dtype = rng.choice(("fp32", "fp16", "bf16"))
    if rng.random() < 0.35:
        return dict(op="dropout", mode=rng.choice(("train", "train", "infer")), count=_log_int(rng, 1000, 200_000_000), dtype=dtype,
                    p=round(rng.uniform(0.01, 0.9), 3), device_seed=rng.random() < 0.5)
    per_group, groups = rng.choice((1, 2, 3, 4, 6, 8, 16)), rng.choice((1, 2, 3, 4, 5, 8, 16, 32))
    c = per_group * groups
    n = rng.choice((1, 1, 1, 2, 3, 8))
    most = max(64, 30_000_000 // (n * c))
    pixels = _log_int(rng, 64, min(most, 2_000_000))
    h = max(1, int(math.sqrt(pixels) * rng.uniform(0.5, 1.0)))
    p = rng.choice((0.0, 0.0, 0.1, 0.35))
    return dict(op="norm", mode=rng.choice(("train", "train", "infer")), n=n, c=c, h=h, w=max(1, pixels // h), groups=groups,
                act=rng.choice(("none", "silu", "gelu")), dtype=dtype, p=p,
                slice_of=rng.choice((0, 0, 0, 2 * c)), device_seed=p > 0 and rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, train = DTYPES[case["dtype"]], case["mode"] == "train"
    normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    state = {"case": case, "seed": seed * 1_000_003 + 17, "offset": seed % 1000}
    if case["device_seed"]:
        state["seed_tensor"] = torch.tensor([state["seed"]], dtype=torch.int64, device="cuda")
    if case["op"] == "dropout":
        state["x"] = torch.empty(case["count"], dtype=dtype, device="cuda").normal_(generator=g).requires_grad_(train)
        if train:
            state["dy"] = torch.empty(case["count"], dtype=dtype, device="cuda").normal_(generator=g)
        return state
    n, c, h, w = (case[k] for k in "nchw")
    # feature maps as a convolution leaves them: a channel has a mean and a scale of its own, pixels vary around it
    wide = normal(n, h, w, case["slice_of"] or c) * torch.exp(0.5 * normal(case["slice_of"] or c)) + normal(case["slice_of"] or c)
    state["x"] = wide.to(dtype).permute(0, 3, 1, 2)[:, :c].requires_grad_(train)
    state["weight"] = (1.0 + 0.2 * normal(c)).requires_grad_(train)
    state["bias"] = (0.2 * normal(c)).requires_grad_(train)
    if train:
        state["dy"] = normal(n, h, w, c).to(dtype).permute(0, 3, 1, 2)
    return state


# ---- the plain forms ---------------------------------------------------------------------------------------------------

def _philox(c0, c1, offset, seed):
    """The four words of Philox4x32-10, each as int64 in [0, 2^32). A product of two 32-bit values wraps in int64 without
    loss: its bits are those of the unsigned product."""
    c = [c0, c1, torch.full_like(c0, offset & M32), torch.full_like(c0, offset >> 32)]
    k0, k1 = seed & M32, (seed >> 32) & M32
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [((b >> 32) & M32) ^ c[1] ^ k0, b & M32, ((a >> 32) & M32) ^ c[3] ^ k1, a & M32]
        k0, k1 = (k0 + 0x9E3779B9) & M32, (k1 + 0xBB67AE85) & M32
    return c


def _halves(blocks, d, offset, seed, count):
    words = torch.stack(_philox(blocks & M32, (blocks >> 32) + (d << 31), offset, seed), -1)
    return torch.stack((words & 0xFFFF, words >> 16), -1).view(-1)[:count]


def _kept(count, p, seed, offset):
    """True where the element stays, in memory order."""
    blocks = torch.arange((count + 7) // 8, device="cuda")
    u = (_halves(blocks, 0, offset, seed, count) << 16) + _halves(blocks, 1, offset, seed, count)
    return u >= min(M32, round(p * 2**32))


def _dropped_out(v, kept, p):
    """v: float32 in memory order (any shape)."""
    return torch.where(kept.view(v.shape), v * torch.tensor(1.0 / (1.0 - p), dtype=torch.float32), 0.0)


def _activation(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5**0.5))
    return z


def _activation_slope(z, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * 0.5**0.5)) + z * torch.exp(-0.5 * z * z) * (0.5 / math.pi) ** 0.5
    return torch.ones_like(z)


def _plain_norm(s, case):
    n, c, h, w, groups = (case[k] for k in ("n", "c", "h", "w", "groups"))
    x = s["x"].permute(0, 2, 3, 1).float().reshape(n, h * w, groups, c // groups)
    weight, bias = (s[k].float().view(groups, c // groups) for k in ("weight", "bias"))
    mean = x.mean(dim=(1, 3), keepdim=True)
    centred = x - mean
    rstd = 1 / torch.sqrt((centred * centred).mean(dim=(1, 3), keepdim=True) + EPS)
    normed = centred * rstd
    z = normed * weight + bias
    y = _activation(z, case["act"])
    if case["p"]:
        kept = _kept(x.numel(), case["p"], s["seed"], s["offset"])
        y = _dropped_out(y, kept, case["p"])
    picture = lambda v: v.reshape(n, h, w, c).to(s["x"].dtype).permute(0, 3, 1, 2)  # noqa: E731
    if case["mode"] == "infer":
        return picture(y)
    dy = s["dy"].permute(0, 2, 3, 1).float().reshape(n, h * w, groups, c // groups)
    if case["p"]:
        dy = _dropped_out(dy, kept, case["p"])
    dz = dy * _activation_slope(z, case["act"])
    d_normed = dz * weight
    dx = rstd * (d_normed - d_normed.mean(dim=(1, 3), keepdim=True) - normed * (d_normed * normed).mean(dim=(1, 3), keepdim=True))
    return picture(y), picture(dx), (dz * normed).sum(dim=(0, 1)).view(c), dz.sum(dim=(0, 1)).view(c)


def _plain_dropout(s, case):
    dtype = s["x"].dtype
    kept = _kept(s["x"].numel(), case["p"], s["seed"], s["offset"])
    y = _dropped_out(s["x"].float(), kept, case["p"]).to(dtype)
    return y if case["mode"] == "infer" else (y, _dropped_out(s["dy"].float(), kept, case["p"]).to(dtype))


# ---- one pass ----------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return _plain_dropout(state, case) if case["op"] == "dropout" else _plain_norm(state, case)
    import inpc_amd

    x, seed = state["x"], state.get("seed_tensor", state["seed"])
    if case["op"] == "dropout":
        y = inpc_amd.dropout(x, case["p"], seed, offset=state["offset"])
        leaves = (x,)
    else:
        random = dict(dropout_p=case["p"], seed=seed, offset=state["offset"]) if case["p"] else {}
        y = inpc_amd.group_norm(x, case["groups"], state["weight"], state["bias"], eps=EPS, activation=case["act"], **random)
        leaves = (x, state["weight"], state["bias"])
    if case["mode"] == "infer":
        return y
    return (y.detach(), *torch.autograd.grad(y, leaves, state["dy"]))


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    passes = 4 if case["mode"] == "train" else 2     # x in, out; with a backward pass also dy in, dx out
    if case["op"] == "dropout":
        return {"bytes": passes * size * case["count"], "flops": passes / 2 * case["count"]}
    count = case["n"] * case["c"] * case["h"] * case["w"]
    # statistics three, normalisation four, activation about four; the backward pass about twice that
    return {"bytes": passes * size * count + passes * 4 * case["c"], "flops": (11 if passes == 2 else 33) * count}


# ---- the definition in 64 bits -----------------------------------------------------------------------------------------

def _mul_hi_lo(a, m):
    """High and low 32 bits of a * m from 16-bit limbs (nothing wraps)."""
    a1, a0, m1, m0 = a >> 16, a & 0xFFFF, m >> 16, m & 0xFFFF
    low, mid1, mid2 = a0 * m0, a1 * m0, a0 * m1
    mid = (low >> 16) + (mid1 & 0xFFFF) + (mid2 & 0xFFFF)
    return a1 * m1 + (mid1 >> 16) + (mid2 >> 16) + (mid >> 16), ((mid & 0xFFFF) << 16) | (low & 0xFFFF)


def _exact_scale(count, p, seed, offset):
    """What each element is multiplied by: 0 or 1 / (1 - p)."""
    number = torch.arange(count, device="cuda")
    block, lane = torch.arange((count + 7) // 8, device="cuda"), number % 8
    threshold, u = min(M32, round(p * 2**32)), None
    for d in (0, 1):
        w0, w1 = block % 2**32, block // 2**32 + d * 2**31
        w2, w3 = torch.full_like(block, offset % 2**32), torch.full_like(block, offset // 2**32)
        for r in range(10):
            key0, key1 = (seed % 2**32 + r * 0x9E3779B9) % 2**32, (seed // 2**32 + r * 0xBB67AE85) % 2**32
            (hi0, lo0), (hi1, lo1) = _mul_hi_lo(w0, 0xD2511F53), _mul_hi_lo(w2, 0xCD9E8D57)
            w0, w1, w2, w3 = hi1 ^ w1 ^ key0, lo1, hi0 ^ w3 ^ key1, lo0
        table = torch.stack((w0, w1, w2, w3), 1)
        half = (table[number // 8, lane // 2] >> (16 * (lane % 2))) & 0xFFFF
        u = half if u is None else u * 2**16 + half
    return torch.where(u < threshold, 0.0, 1.0 / (1.0 - p)).double()


def exact(case, seed):
    if case["op"] == "dropout" and case["count"] > 300_000_000:
        return None     # tens of gigabytes of 64-bit temporaries
    s = prepare(case, seed)
    x = s["x"].detach().double()
    if case["op"] == "dropout":
        scale = _exact_scale(case["count"], case["p"], s["seed"], s["offset"])
        return x * scale if case["mode"] == "infer" else (x * scale, s["dy"].double() * scale)
    n, c, h, w, groups = (case[k] for k in ("n", "c", "h", "w", "groups"))
    train = case["mode"] == "train"
    weight, bias = (s[k].detach().double().requires_grad_(train) for k in ("weight", "bias"))
    x.requires_grad_(train)
    grouped = x.reshape(n, groups, -1)
    var, mean = torch.var_mean(grouped, dim=2, correction=0, keepdim=True)
    z = ((grouped - mean) / (var + EPS).sqrt()).view(n, c, h, w) * weight.view(1, c, 1, 1) + bias.view(1, c, 1, 1)
    y = {"none": lambda v: v, "silu": lambda v: v * torch.sigmoid(v),
         "gelu": lambda v: v * torch.special.ndtr(v)}[case["act"]](z)
    if case["p"]:
        scale = _exact_scale(x.numel(), case["p"], s["seed"], s["offset"])
        y = y * scale.view(n, h, w, c).permute(0, 3, 1, 2)
    if not train:
        return y
    return (y.detach(), *torch.autograd.grad(y, (x, weight, bias), s["dy"].double()))

"""The 8-bit KV cache and attention over it in 64 bits, token by token, on the CPU: what the kernels are tested against."""
import math

import torch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def least_scale(amax: float, code) -> float:
    e = -100
    while amax * 2.0 ** -e > MOST[code]:
        e += 1
    return 2.0 ** e


def to_codes(x: torch.Tensor, code) -> torch.Tensor:
    return torch.round(x).to(torch.int8) if code == torch.int8 else x.float().to(code)


class Cache:
    """Values [blocks, heads, 16, d] and scales of one tensor (keys or values) in 64 bits."""

    def __init__(self, codes: torch.Tensor, scale: torch.Tensor):
        self.code = codes.dtype
        self.codes = codes.cpu().view(torch.uint8).clone().view(codes.dtype)
        self.scale = scale.cpu().double()

    def append(self, x: torch.Tensor, slots) -> None:
        """x: [tokens, heads, d]; all tokens of a block in one go."""
        blocks = {}
        for t, s in enumerate(slots):
            if s >= 0:
                blocks.setdefault(s // 16, []).append((s % 16, t))
        for b, members in blocks.items():
            lo = min(o for o, _ in members)
            for h in range(x.shape[1]):
                new = torch.stack([x[t, h] for _, t in members]).double()
                old = 0.0 if lo == 0 else float(self.scale[b, h])
                s = least_scale(float(new.abs().max()), self.code) if bool(torch.isfinite(new).all()) else math.nan
                s = math.nan if math.isnan(s) or math.isnan(old) else max(s, old)
                self.scale[b, h] = s
                raw = self.codes.view(torch.uint8)
                if lo and s != old:
                    kept = self.codes[b, h, :lo].double() * old / s if not math.isnan(s) else torch.zeros(lo, x.shape[2])
                    raw[b, h, :lo] = to_codes(kept, self.code).view(torch.uint8)
                for (o, _), v in zip(members, new):
                    raw[b, h, o] = to_codes(v / s if not math.isnan(s) else torch.zeros_like(v), self.code).view(torch.uint8)

    def values(self) -> torch.Tensor:
        return self.codes.double() * self.scale[:, :, None, None]


def rotate(x: torch.Tensor, positions, base: float) -> torch.Tensor:
    """[tokens, heads, d] in its own type, channel pairs (j, j + d / 2)."""
    half = x.shape[-1] // 2
    theta = base ** (-torch.arange(half, dtype=torch.float64) / half)
    ang = torch.as_tensor(positions, dtype=torch.float64)[:, None, None] * theta
    a, b = x[..., :half].double(), x[..., half:].double()
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).to(x.dtype)


def attend(q, kvals, vvals, pages, limit, scale):
    """q [heads, d] over the first ``limit`` keys of ``pages``: out and sum p |v| [heads, d]; for each head the largest
    scale * sum |q k| and the number of keys times the largest |v|."""
    heads, d = q.shape
    kvh = kvals.shape[1]
    if limit <= 0:
        z = torch.zeros(heads, d, dtype=torch.float64)
        return z, z, torch.zeros(heads, dtype=torch.float64), torch.zeros(heads, dtype=torch.float64)
    idx = torch.as_tensor(pages[: -(-limit // 16)], dtype=torch.long)
    k = kvals[idx].transpose(0, 1).reshape(kvh, -1, d)[:, :limit].repeat_interleave(heads // kvh, 0)
    v = vvals[idx].transpose(0, 1).reshape(kvh, -1, d)[:, :limit].repeat_interleave(heads // kvh, 0)
    # a poisoned value block is seen by whoever sees its keys
    qd = q.double()
    s = torch.einsum("hd,hkd->hk", qd, k) * scale
    s = torch.where(torch.isnan(v).any(-1), torch.full_like(s, math.nan), s)
    p = torch.softmax(s, -1)
    size = (torch.einsum("hd,hkd->hk", qd.abs(), k.abs()) * abs(scale)).amax(-1)
    return torch.einsum("hk,hkd->hd", p, v), torch.einsum("hk,hkd->hd", p, v.abs()), size, limit * torch.nan_to_num(v).abs().amax((1, 2))


def bound(ref, weight, size, most, dtype, d, p_round=2.0 ** -11, p_floor=2.0 ** -40, kv_round=0.0):
    """How far a kernel's output may be from ``attend``'s.  Rounding of the result: eps / 2 of its type.  Rounding of the
    probabilities to 16 bits (``p_round``; the sum of them is kept in 32): that fraction of sum p |v|.  The scores are sums
    of d products in 32 bits, with the factors of the scale and of log2 e: (d + 8) * 2^-23 of sum |q k| at most (accumulation
    that truncates costs a whole step), which moves p, and their sum, by that much each; exponentials and the running
    rescaling: 2^-20 of p.  A probability kept as 2^15 p in fp16 has steps of 2^-24 at its smallest, so half of that over 2^15,
    2^-40, of each |v| can be lost (``p_floor``; kept as p itself: half a step, 2^-25).  32-bit arithmetic that takes subnormals for zero loses up to 2^-126 (for |v| up to 1; in proportion above) of each
    product, and of the result.  Keys and values that are rounded on the way (``kv_round`` of each) move a score by that fraction
    of sum |q k|, p and the sum of p by as much each, and v by its own."""
    u = torch.finfo(dtype).eps / 2
    rel = p_round + 2 * ((d + 8) * 2.0 ** -23 + kv_round) * size[..., None] + kv_round + 2.0 ** -20
    return (u * ref.abs() + (1 + u) * rel * weight + most[..., None] * p_floor + (most[..., None] + 2) * 2.0 ** -126
            + torch.finfo(dtype).smallest_normal * u * 2)

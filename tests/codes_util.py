"""Plain restatement in 64 bits of a paged cache of 8-bit codes."""
import math

import torch

from paged_util import HALF_STEP, Batch

MOST = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
CODES = tuple(MOST)


def quantize64(y, kind):
    """(codes, scale) of rows y [..., head_dim], CPU: the scale rounded to 32 bits, then code = y / scale rounded once, to nearest, ties to
    even, from the quotient in 64 bits."""
    y = y.double()
    top = y.abs().amax(-1)
    scale = torch.where(top > 0, (top / MOST[kind]).float().clamp(min=2.0 ** -126), torch.ones_like(top).float())
    z = (y / scale.double()[..., None]).clamp(-MOST[kind], MOST[kind])
    step = torch.ones_like(z) if kind == torch.int8 else torch.ldexp(torch.ones_like(z), (torch.frexp(z).exponent - 4).clamp(min=-9))
    return (torch.round(z / step) * step).float().to(kind), scale


def half_step(y, scale, kind):
    """The most that a value y is off when its row is kept under this scale."""
    if kind == torch.int8:
        return (0.5 * scale.double())[..., None].expand(y.shape)
    return torch.maximum(y.double().abs() * 2.0 ** -4, (scale.double() * 2.0 ** -10)[..., None])


class CodesBatch(Batch):
    """A Batch whose cache holds codes; the rows' magnitudes differ by `spread` powers of two either way."""

    def __init__(self, new, lens, heads, kv_heads, head_dim=128, page=16, dtype=torch.float16, kind=torch.int8, spread=1.0, **more):
        super().__init__(new, lens, heads, kv_heads, head_dim, page, dtype, **more)
        self.kind = kind
        gen = torch.Generator().manual_seed(1 + more.get("seed", 0))
        for w in "kv":
            cache = getattr(self, w + "_cache").float()
            cache *= torch.exp2(spread * (2 * torch.rand(cache.shape[:3], generator=gen) - 1))[..., None]
            codes, scale = quantize64(cache, kind)
            setattr(self, w + "_cache", codes)
            setattr(self, w + "_scale", scale)

    def gpu(self):
        return [t.cuda() for t in (self.k_cache, self.v_cache, self.pages, self.starts, self.lens)]

    def scales(self):
        return dict(k_scale=self.k_scale.cuda(), v_scale=self.v_scale.cuda())

    def values(self, w, b):
        """[positions, kv_heads, head_dim] of sequence b in 64 bits."""
        codes = self.history(getattr(self, w + "_cache").float(), b).double()
        return codes * self.history(getattr(self, w + "_scale"), b).double()[..., None]

    def poison(self):
        """Every slot that no sequence holds gets codes of all ones and scales of NaN."""
        held = torch.zeros(self.k_cache.shape[0], self.page, dtype=torch.bool)
        for b, n in enumerate(self.lens_list):
            p = torch.arange(n)
            held[self.pages[b].long()[p // self.page], p % self.page] = True
        for cache, scale in ((self.k_cache, self.k_scale), (self.v_cache, self.v_scale)):
            cache.view(torch.uint8).transpose(1, 2)[~held] = 255
            scale.transpose(1, 2)[~held] = math.nan


def attend_codes64(batch, scale=None, window=0, first_key=None, alibi_slopes=None, tiles=False):
    """(out, tolerance) [tokens of the sequences, heads, head_dim] in float64.

    The tolerance, first order.  A weight p_j s_j (s_j the scale of the value) is rounded to fp16, by u = 2^-11 of itself; the sum that
    divides is of the rounded weights over s_j, so it is off by u, too.  Below fp16's smallest normal value a weight is off by 2^-25, where the
    largest one is 2^7 or more: 2^-32 of that, times the codes.  A score is a sum of head_dim products in fp32, whose additions may
    be cut off instead of rounded, scaled twice: (2 head_dim + 8) 2^-24 of its sum of magnitudes, which is the relative error of its
    exponential beside that of ex2 and of the running rescaling (2^-19 in all); the same goes for the sum.  q of bf16 enters as fp16 under a
    power of two with the largest value at 2^14 or more, off by 2^-25 at most: 2^-39 of the largest.  The result is rounded by half a
    step.

    tiles: for calls that take tiles of 128 rows, where the weight times the scale is rounded to q's type, and the sum that divides is of weights that
    are not rounded; and for the sequences of few tokens among them as above.  In fp16 a weight is held under a power of two that is at most twice the largest scale among the values that the tile reads, so what
    falls below the smallest normal value is off by 2^-25 of that power where the largest weight is 2^7 or more: 2^-31 of that scale, times the codes."""
    H, D = batch.q.shape[1:]
    K = batch.k_cache.shape[1]
    u = HALF_STEP[batch.dtype] if tiles else 2.0 ** -11
    scale = 1 / math.sqrt(D) if scale is None else scale
    n = sum(batch.new)
    out, tol = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    at = 0
    for b, (t, length) in enumerate(zip(batch.new, batch.lens_list)):
        if t == 0 or length == 0:
            at += t
            continue
        k, v = (batch.values(w, b).repeat_interleave(H // K, 1).transpose(0, 1) for w in "kv")      # [heads][positions][D]
        vs = batch.history(batch.v_scale, b).double().repeat_interleave(H // K, 1).transpose(0, 1)[:, None, :]
        q = batch.q[at:at + t].double().transpose(0, 1)
        p, j = torch.arange(length - t, length)[:, None], torch.arange(length)[None, :]
        seen = j <= p
        if window:
            seen &= j > p - window
        if first_key is not None:
            seen &= j >= first_key[b]
        s = scale * q @ k.transpose(1, 2)
        size = abs(scale) * (q.abs() @ k.abs().transpose(1, 2) +
                             2.0 ** -15 / D * q.abs().amax(-1, keepdim=True) * k.abs().sum(-1)[:, None, :])
        if alibi_slopes is not None:
            bias = alibi_slopes.double()[:, None, None] * (j - p)
            s, size = s + bias, size + bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
        l = e.sum(-1, keepdim=True)
        w = torch.where(l > 0, e / l, 0.0)
        off = (2 * D + 8) * 2.0 ** -24 * size
        off = off.masked_fill(~seen, 0).amax(-1, keepdim=True)
        o, mag = w @ v, w @ v.abs()
        t_o = (2 * u + 2 * off + 2.0 ** -19) * mag + HALF_STEP[batch.dtype] * o.abs() + 2.0 ** -25
        codes = seen.double() @ (v.abs() / vs.transpose(1, 2))
        t_o += (2.0 ** -31 * vs.amax() if tiles else 2.0 ** -32 * (w * vs).amax(-1, keepdim=True)) * codes
        out[at:at + t], tol[at:at + t] = o.transpose(0, 1), t_o.transpose(0, 1)
        at += t
    return out, tol

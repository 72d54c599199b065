"""Plain restatement in 64 bits of the calls on a paged cache, and batches to try them on."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rotate64(x, positions, freqs, interleaved, magnitude=1.0):
    """x [tokens, heads, head_dim], CPU; returns float64."""
    y = x.double().clone()
    angle = positions.double()[:, None, None] * freqs.double()
    c, s = torch.cos(angle) * magnitude, torch.sin(angle) * magnitude
    r = 2 * freqs.numel()
    one = slice(0, r, 2) if interleaved else slice(0, r // 2)
    two = slice(1, r, 2) if interleaved else slice(r // 2, r)
    a, b = x[..., one].double(), x[..., two].double()
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    return y


def rotate_tolerance(x, freqs, interleaved, dtype, magnitude=1.0):
    """Half a step of the result, and fp32 work of a few operations on a pair: the bound of |a| + |b| times 2^-21."""
    y = x.double().abs()
    r = 2 * freqs.numel()
    one = slice(0, r, 2) if interleaved else slice(0, r // 2)
    two = slice(1, r, 2) if interleaved else slice(r // 2, r)
    both = (y[..., one] + y[..., two]) * magnitude
    y[..., one], y[..., two] = both, both
    return y * 2.0 ** -21


class Batch:
    """A paged cache with some sequences in it: `new[b]` tokens of sequence b are to be served, `lens[b]` positions exist."""

    def __init__(self, new, lens, heads, kv_heads, head_dim=128, page=16, dtype=torch.float16, seed=0, spare=3, q_scale=2.0, behind=0):
        gen = torch.Generator().manual_seed(seed)
        self.new, self.lens_list, self.page, self.dtype = list(new), list(lens), page, dtype
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        self.k_cache = torch.randn(total, kv_heads, page, head_dim, generator=gen).to(dtype)
        self.v_cache = torch.randn(total, kv_heads, page, head_dim, generator=gen).to(dtype)
        order = torch.randperm(total, generator=gen).tolist()
        self.pages = torch.full((len(new), max(need + [1])), -1, dtype=torch.int32)   # what is not needed is no page
        for b, n in enumerate(need):
            self.pages[b, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
        self.unused = order
        self.starts = torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32)
        self.lens = torch.tensor(lens, dtype=torch.int32)
        n = sum(new) + behind
        self.q = (q_scale * torch.randn(n, heads, head_dim, generator=gen)).to(dtype)
        self.k = torch.randn(n, kv_heads, head_dim, generator=gen).to(dtype)
        self.v = torch.randn(n, kv_heads, head_dim, generator=gen).to(dtype)

    def history(self, cache, b, length=None):
        """[positions, kv_heads, head_dim] of sequence b."""
        p = torch.arange(self.lens_list[b] if length is None else length)
        return cache[self.pages[b].long()[p // self.page], :, p % self.page]

    def poison(self, value=math.nan):
        """Every slot that no sequence holds gets `value`."""
        held = torch.zeros(self.k_cache.shape[0], self.page, dtype=torch.bool)
        for b, n in enumerate(self.lens_list):
            p = torch.arange(n)
            held[self.pages[b].long()[p // self.page], p % self.page] = True
        for cache in (self.k_cache, self.v_cache):
            cache.transpose(1, 2)[~held] = value

    def positions(self):
        return torch.cat([torch.arange(n - t, n) for t, n in zip(self.new, self.lens_list)])


def attend64(batch, scale=None, window=0, first_key=None, alibi_slopes=None):
    """(out, tolerance) [tokens of the sequences, heads, head_dim] in float64.

    The tolerance, first order: each probability enters the product rounded by at most half a step u of the cache's type, or in
    fp16 by 2^-25 below its smallest normal value (the largest probability is 1 or more, so the sum l is too), the result is
    rounded by u; a score is a sum of head_dim products in fp32, scaled, off by (head_dim + 8) 2^-24 of its sum of magnitudes,
    which is the relative error of its exponential beside that of ex2 and of the running rescaling (2^-20 in all); the same
    goes for the sum that divides."""
    H, D = batch.q.shape[1:]
    K = batch.k_cache.shape[1]
    u = HALF_STEP[batch.dtype]
    scale = 1 / math.sqrt(D) if scale is None else scale
    n = sum(batch.new)
    out, tol = torch.zeros(n, H, D, dtype=torch.float64), torch.zeros(n, H, D, dtype=torch.float64)
    at = 0
    for b, (t, length) in enumerate(zip(batch.new, batch.lens_list)):
        if t == 0:
            continue
        k = batch.history(batch.k_cache, b).double().repeat_interleave(H // K, 1).transpose(0, 1)      # [heads][positions][D]
        v = batch.history(batch.v_cache, b).double().repeat_interleave(H // K, 1).transpose(0, 1)
        q = batch.q[at:at + t].double().transpose(0, 1)
        p, j = torch.arange(length - t, length)[:, None], torch.arange(length)[None, :]
        seen = j <= p
        if window:
            seen &= j > p - window
        if first_key is not None:
            seen &= j >= first_key[b]
        s = scale * q @ k.transpose(1, 2)
        size = abs(scale) * q.abs() @ k.abs().transpose(1, 2) if length else s
        if alibi_slopes is not None:
            bias = alibi_slopes.double()[:, None, None] * (j - p)
            s, size = s + bias, size + bias.abs()
        s = s.masked_fill(~seen, -math.inf)
        e = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if length else s
        l = e.sum(-1, keepdim=True)
        w = torch.where(l > 0, e / l, 0.0)
        off = (size.masked_fill(~seen, 0).amax(-1, keepdim=True) if length else torch.zeros_like(l)) * (D + 8) * 2.0 ** -24
        o, mag = w @ v, w @ v.abs()
        t_o = (u + 2 * off + 2.0 ** -19) * mag + u * o.abs() + 1e-7
        if batch.dtype == torch.float16:
            t_o += 2.0 ** -25 * torch.where(l > 0, (seen.double() @ v.abs()) / l, 0.0)
        out[at:at + t], tol[at:at + t] = o.transpose(0, 1), t_o.transpose(0, 1)
        at += t
    return out, tol

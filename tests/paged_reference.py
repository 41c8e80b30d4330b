"""Plain 64-bit forms of the paged cache's operators, and random cases for
their tests."""
import math

import numpy as np
import torch

U = 2.0 ** -24  # half a step of float32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rotate(x, positions, count, theta_scale):
    """x [tokens, heads, dim] (float64): pairs (i, i + count / 2) turned by
    position * theta_scale^i."""
    h = count // 2
    angle = positions.double()[:, None, None] * float(theta_scale) ** torch.arange(h, dtype=torch.float64)
    c, s = angle.cos(), angle.sin()
    a, b = x[..., :h], x[..., h:count]
    return torch.cat([a * c - b * s, a * s + b * c, x[..., count:]], -1)


def norm(x, gamma, eps):
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * gamma.double()


def softmax_rows(q, keys, values, scale):
    """One row: q [heads, dim], keys and values [tokens, kv_heads, dim], all
    float64.  The output, the sum of weight * |v| per element, and the largest
    scale * sum |q||k| (for error bounds)."""
    heads, kv = q.shape[0], keys.shape[1]
    out, mass, dots = torch.zeros_like(q), torch.zeros_like(q), 0.0
    if keys.shape[0] == 0:
        return out, mass, dots
    for h in range(heads):
        k, v = keys[:, h // (heads // kv)], values[:, h // (heads // kv)]
        p = torch.softmax(k @ q[h] * scale, 0)
        out[h], mass[h] = p @ v, p @ v.abs()
        dots = max(dots, float((k.abs() @ q[h].abs()).max()) * abs(scale))
    return out, mass, dots


def attend_bound(out, mass, dots, tokens, dim, dtype, cache):
    """How far a row's output may be from the 64-bit one.  A score is a dot
    product of `dim` terms summed in 32 bits: off by (dim + 8) U sum |q||k|
    at most, so each weight by twice that, relative (it and the maximum);
    the exponential's argument and value are rounded (4 U and |s| U, covered
    by another dots * U); sums over the tokens are off by tokens * U.  With
    16-bit outputs over a 16-bit cache a weight enters the value product as two
    bfloat16 parts, 2^-16 relative.  The output is rounded once."""
    weights = 2 * (dim + 9) * U * dots + (tokens + 32) * U
    if dtype == torch.bfloat16 and cache == torch.bfloat16:
        weights += 2.0 ** -16
    return weights * mass + half_step(dtype) * out.abs() + 1e-30


class Batch:
    """A random batch over a paged pool: pages dealt at random, slots past
    each row's length and pages of nobody filled with `junk`."""

    def __init__(self, seed, rows, kv_heads, group, dim, page, prefix, lengths, dtype, cache, junk=float("nan"),
                 spare=2, wide=None):
        g = torch.Generator().manual_seed(seed)
        self.page, self.prefix_tokens, self.lengths = page, prefix, lengths
        needed = [-(-max(n, 0) // page) for n in lengths]
        shared = -(-prefix // page)
        total = shared + sum(needed) + spare
        order = torch.randperm(total, generator=g).int()
        self.keys = torch.full((total, page, kv_heads, dim), junk).to(cache)
        self.values = self.keys.clone()
        self.prefix = order[:shared].clone()
        self.table = torch.full((rows, max(1, max(needed)) if wide is None else wide), -1, dtype=torch.int32)
        at = shared

        def fill(pages, n):
            k = torch.randn(n, kv_heads, dim, generator=g).to(cache)
            v = torch.randn(n, kv_heads, dim, generator=g).to(cache)
            i = torch.arange(n)
            self.keys[pages.long()[i // page], i % page] = k
            self.values[pages.long()[i // page], i % page] = v
            return k.double(), v.double()

        self.shared = fill(self.prefix, prefix)
        self.own = []
        for r, n in enumerate(needed):
            self.table[r, :n] = order[at:at + n]
            at += n
            self.own.append(fill(self.table[r, :n], max(lengths[r], 0)))
        self.q = (1.5 * torch.randn(rows, group * kv_heads, dim, generator=g)).to(dtype)
        self.scale = 1.0 / math.sqrt(dim)

    def reference(self, r, skip=()):
        """Row r's output, mass and dots; `skip`: own tokens that a bad page hides."""
        keep = [i for i in range(self.own[r][0].shape[0]) if i not in skip]
        keys, values = (torch.cat([s, o[keep]]) for s, o in zip(self.shared, self.own[r]))
        return softmax_rows(self.q[r].double(), keys, values, self.scale) + (keys.shape[0],)


def np_adjust(logits, u, vocab):
    """The rules on float32 or bfloat16 logits [rows, vocab] (numpy float32):
    64-bit, rounded once to float32, then to the type by the caller."""
    x = logits.astype(np.float64)
    for r in range(x.shape[0]):
        if u.get("history") is not None:
            n = min(int(u["history_lengths"][r]), u["history"].shape[1])
            if n < 0:
                continue
            tokens = u["history"][r, :n].astype(np.int64)
            start = 0 if u.get("prompt_lengths") is None else max(0, int(u["prompt_lengths"][r]))
            valid = (tokens >= 0) & (tokens < vocab)
            seen = np.unique(tokens[valid])
            if u.get("repetition") is not None:
                rep = np.float64(u["repetition"][r])
                x[r, seen] = np.where(x[r, seen] > 0, x[r, seen] / rep, x[r, seen] * rep)
            made, count = np.unique(tokens[start:][valid[start:]], return_counts=True)
            freq = 0.0 if u.get("frequency") is None else np.float64(u["frequency"][r])
            pres = 0.0 if u.get("presence") is None else np.float64(u["presence"][r])
            x[r, made] = x[r, made] - freq * count - pres
        if u.get("bias_ids") is not None:
            n = int(u["bias_lengths"][r])
            sums = {}
            for i, v in zip(u["bias_ids"][r, :n], u["bias_values"][r, :n]):
                if 0 <= i < vocab:
                    sums[int(i)] = sums[int(i)] + np.float64(v) if int(i) in sums else np.float64(v)
            for i, v in sums.items():
                x[r, i] += v
        if u.get("masks") is not None:
            m = r if u.get("mask_of") is None else int(u["mask_of"][r])
            if m >= u["masks"].shape[0]:
                x[r] = -np.inf
            elif m >= 0:
                bits = np.unpackbits(np.ascontiguousarray(u["masks"][m]).view(np.uint8), bitorder="little")[:vocab]
                x[r, bits == 0] = -np.inf
    return x.astype(np.float32)


def np_greedy(values):
    """The lowest index of the highest value of each row; 0xffffffff where only
    NaN and -inf are left."""
    out = []
    for row in values:
        row = np.where(np.isnan(row), -np.inf, row)
        out.append(int(row.argmax()) if row.max() > -np.inf else 0xffffffff)
    return np.array(out, np.uint32)

"""The 8-bit cache in plain numpy and 64 bits: what its levels stand for, one-token attention over it, the choice of the blocks
that eviction keeps, and the rules on logits."""
import math

import numpy as np
import torch

BLOCK = 16


def levels_of(x, fmt):
    """x fp32 [16, D]: (levels as numbers, scale), every operation rounded to fp32 as the definition says."""
    x = x.float().cpu()
    top = torch.tensor(127.0 if fmt == torch.int8 else 448.0)
    scale = torch.clamp(x.abs().max() / top, min=torch.tensor(2.0 ** -126))
    q = torch.clamp(x / scale, -top, top)
    q = torch.round(q) if fmt == torch.int8 else q.to(torch.float8_e4m3fn).float()
    return q, scale


class PlainCache:
    """What each sequence holds, by position: lists of fp32 rows per kv head, finished blocks replaced by what their levels stand for."""

    def __init__(self, kv_heads, dim, fmt):
        self.G, self.D, self.fmt = kv_heads, dim, fmt
        self.rows, self.levels, self.scales = [], [], []      # rows[p] [2, G, D] as they came; levels[b], scales[b] of finished blocks

    def append(self, k, v):
        self.rows.append(torch.stack([k, v]).double().cpu())
        if len(self.rows) % BLOCK == 0:
            x = torch.stack(self.rows[-BLOCK:]).permute(1, 2, 0, 3)              # [2, G, 16, D]
            got = [[levels_of(x[i, g], self.fmt) for g in range(self.G)] for i in range(2)]
            self.levels.append(torch.stack([torch.stack([g[0] for g in h]) for h in got]))
            self.scales.append(torch.stack([torch.stack([g[1] for g in h]) for h in got]))

    def values(self, upto=None):
        """[2, G, positions, D] in 64 bits; the block of position `upto` (the last one) as it came, even if it is finished."""
        n = len(self.rows)
        blk = (n - 1) // BLOCK
        old = [self.levels[b].double() * self.scales[b].double()[..., None, None] for b in range(blk)]
        new = torch.stack(self.rows[blk * BLOCK:]).permute(1, 2, 0, 3)
        return torch.cat(old + [new], 2)


def attend(q, kv, scale, window=0):
    """q [H, D], kv [2, G, n, D] in 64 bits, the newest position last: (outputs [H, D], weights of positions [G, n],
    largest sum of |q_d k_d| * scale over the visible positions)."""
    H, (_, G, n, D) = q.shape[0], kv.shape
    lo = max(0, n - window) if window else 0
    qg = q.double().view(G, H // G, D)
    s = torch.einsum("ghd,gjd->ghj", qg, kv[0][:, lo:]) * scale
    a = torch.softmax(s, -1)
    out = torch.einsum("ghj,gjd->ghd", a, kv[1][:, lo:]).reshape(H, D)
    w = torch.zeros(G, n, dtype=torch.float64)
    w[:, lo:] = a.sum(1)
    spread = torch.einsum("ghd,gjd->ghj", qg.abs(), kv[0][:, lo:].abs()).max().item() * scale
    return out, w, spread


def attend_bounds(D, n, spread, top, out_dtype):
    """How far fp32 arithmetic may be off (outputs, and block weights relative to the group's heads).  A score is a sum of D
    products, each with a relative error below 2^-22 (operands in two 11-bit parts) and D additions of 2^-24: in all below
    (D / 4 + 4) 2^-22 of the sum of magnitudes `spread`, and a factor 2 for what an exponential makes of it and for the normaliser.  Sums
    over n positions in fp32 add n 2^-24, exponentials and divisions 2^-20."""
    rel = 2 * (D / 4 + 4) * 2.0 ** -22 * spread + n * 2.0 ** -24 + 2.0 ** -20
    return rel * top + (top * torch.finfo(out_dtype).eps / 2), rel


def kept_blocks(weight, keep, recent):
    """Numbers of the blocks that stay, of one sequence and head."""
    n = len(weight)
    if n <= keep:
        return list(range(n))
    order = sorted(range(n - recent), key=lambda b: (-(math.inf if math.isnan(weight[b]) else weight[b]), not math.isnan(weight[b]), b))
    return sorted(order[:keep - recent]) + list(range(n - recent, n))


def rules(x, history, prompt_len, penalties, bias, allowed):
    """One row in 64 bits: (results, bound on the fp32 error)."""
    x = np.asarray(x, dtype=np.float64).copy()
    mag = np.abs(x)
    if penalties is not None:
        rep, pres, freq = [float(v) for v in penalties]
        seen = np.zeros(len(x), dtype=np.int64)
        said = np.zeros(len(x), dtype=np.int64)
        for j, t in enumerate(history):
            if 0 <= t < len(x):
                seen[t] += 1
                said[t] += j >= prompt_len
        hit = seen > 0
        x[hit] = np.where(x[hit] > 0, x[hit] / rep, x[hit] * rep)
        x -= np.where(said > 0, freq * said + pres, 0.0)
        mag = np.maximum(mag, np.maximum(mag * rep, mag / rep)) * hit + mag * ~hit + np.where(said > 0, abs(freq) * said + abs(pres), 0.0)
    if bias is not None:
        b = np.asarray(bias, dtype=np.float64)
        x, mag = x + b, mag + np.where(np.isfinite(b), np.abs(b), 0.0)
    if allowed is not None:
        x[~allowed] = -np.inf
    # at most five roundings (quotient, product, two differences, sum), each at most 2^-24 of a number that is no larger than the
    # sum of the magnitudes of all terms
    return x, 5 * 2.0 ** -24 * mag

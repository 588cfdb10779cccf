"""One-token attention over the 8-bit cache where blocks differ in what they contribute: values of very different sizes, a key far above
all others, blocks outside the window, against 64 bits.

The bound on an output is made of sums over the positions, so that large values that have next to no weight do not widen it.  A score is
a sum of D products, each off by 2^-22 of its size (operands in parts of 11 bits), and D additions of 2^-24, in all (D / 4 + 4) 2^-22 of the
sum of magnitudes; queries written in digits are off by 2^-20 (bfloat16 runs) or 2^-27 (float32 runs) of the row's largest; the score
itself and its distance to the reference are rounded, 2^-22 of the two largest scores together.  An exponential turns the sum of these into a relative error of
a weight; sums over n positions add n 2^-24, exponentials and divisions 2^-20.  The normaliser has the weights' mean error.  A weight that
multiplies values is held in fewer bits than fp32 only relative to the heaviest product of weight and value scale near it: off by 2^-22 of
itself or by 2^-21 (bfloat16 runs; float32 runs 2^-25) of the heaviest within seven blocks, whichever is more."""
import pytest
import torch

from block_reference import BLOCK
from test_gpu_block_cache import KERNELS, B, Rig, how

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def bound_of(q, kv, scales, scale, window, dtype):
    """q [H, D], kv [2, G, n, D], scales [G, n] (of the values; 0 where a position is not held in levels), all in 64 bits: (outputs, bound) [H, D]."""
    H, (_, G, n, D) = q.shape[0], kv.shape
    q = q.double().view(G, H // G, D)
    s = torch.einsum("ghd,gjd->ghj", q, kv[0]) * scale
    mag = torch.einsum("ghd,gjd->ghj", q.abs(), kv[0].abs()) * scale
    digits = 2.0 ** -20 if dtype == torch.bfloat16 else 2.0 ** -27
    off = q.abs().amax(-1, keepdim=True) * digits * kv[0].abs().sum(-1)[:, None] * scale
    if window:
        s[..., :max(0, n - window)] = float("-inf")
    a = torch.softmax(s, -1)
    seen = torch.where(a > 0, s, torch.zeros_like(s))
    rel = (D / 4 + 4) * 2.0 ** -22 * mag + off + 2.0 ** -22 * (seen.abs() + seen.abs().amax(-1, keepdim=True)) + n * 2.0 ** -24 + 2.0 ** -20
    rel = rel + (a * rel).sum(-1, keepdim=True)
    v = kv[1].abs()
    bound = torch.einsum("ghj,gjd->ghd", a * (rel + 2.0 ** -22), v)
    # the heaviest product within seven blocks, position by position
    product = torch.nn.functional.pad(a * scales[:, None], (0, -n % BLOCK)).view(G, H // G, -1, BLOCK).amax(-1)
    near = torch.nn.functional.max_pool1d(product, 15, stride=1, padding=7).repeat_interleave(BLOCK, -1)[..., :n]
    floor = 2.0 ** -21 if dtype == torch.bfloat16 else 2.0 ** -25
    levels = torch.where(scales > 0, 1 / scales.clamp(min=1e-300), torch.zeros_like(scales))[..., None] * v
    bound = bound + floor * torch.einsum("ghj,gjd->ghd", near, levels)
    out = torch.einsum("ghj,gjd->ghd", a, kv[1])
    bound = bound + out.abs() * torch.finfo(dtype).eps / 2 + 1e-37
    return out.reshape(H, D), bound.reshape(H, D)


class Apart(Rig):
    """A rig whose rows are given, and whose outputs are held against the bound above."""

    def fill(self, slot, k, v):
        """k, v [n, G, D]: the prompt of a slot."""
        n = k.shape[0]
        x = torch.cat([torch.zeros(n, self.H, self.D), k, v], 1).to(self.dtype)
        view, keep = self.batch([slot], [n], [0])
        B().block_store(x.reshape(n, -1).to(DEV), view, self.view, self.H, self.err, B().stream_ptr())
        for r in x:
            self.cache_of(slot).append(r[self.H:self.H + self.G].float(), r[self.H + self.G:].float())
        torch.cuda.synchronize()

    def ask(self, slots, q, k, v, scale, kernel, splits=0, check=None):
        """q [n, H, D], k, v [n, G, D]: a step; the outputs of `check` (default: all) are compared."""
        b = B()
        x = torch.cat([q, k, v], 1).to(self.dtype)
        view, keep = self.batch(slots, [1] * len(slots), [len(self.cache_of(s).rows) for s in slots])
        out = torch.empty(len(slots), self.H * self.D, dtype=self.dtype, device=DEV)
        scratch = torch.zeros(b.block_attention_scratch_floats(len(slots), self.H, self.view), device=DEV)
        b.block_attention(x.reshape(len(slots), -1).to(DEV), out, view, self.view, self.H, scale, scratch, self.err, b.stream_ptr(),
                          splits=splits, **how(kernel))
        torch.cuda.synchronize()
        assert self.err.item() == 0
        for i, s in enumerate(slots):
            c = self.cache_of(s)
            c.append(x[i, self.H:self.H + self.G].float(), x[i, self.H + self.G:].float())
            if check is not None and s not in check:
                continue
            kv = c.values()
            n = kv.shape[2]
            scales = torch.zeros(self.G, n, dtype=torch.float64)
            for blk in range((n - 1) // BLOCK):
                scales[:, blk * BLOCK:(blk + 1) * BLOCK] = c.scales[blk][1].double()[:, None]
            want, bound = bound_of(x[i, :self.H], kv, scales, scale, self.window, self.dtype)
            got = out[i].view(self.H, self.D).double().cpu()
            assert torch.isfinite(got).all(), (i, s)
            worst = ((got - want).abs() / bound).max().item()
            assert worst <= 1, f"slot {s}: an error of {worst:.3g} bounds"
        return out.view(len(slots), self.H, self.D)


def noise(g, *shape):
    return torch.randn(*shape, generator=g)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("fmt, D, H", [(torch.int8, 128, 8), (torch.int8, 64, 5), (torch.int8, 128, 12), (torch.float8_e4m3fn, 128, 4), (torch.float8_e4m3fn, 64, 8)])
def test_bfloat16_outputs_are_rounded_once(kernel, fmt, D, H):
    """Weights that differ little over few positions, so that all that may be seen beside the output's own rounding is a few 2^-20: a
    weight rounded to 11 bits where it multiplies values moves one output in fifty past a border."""
    r = Apart(2, 2 * H, D, fmt, torch.bfloat16, n_slots=4, width=2, seed=H)
    for slot, n in enumerate((16, 35, 64, 100)):
        r.fill(slot, noise(r.g, n, 2, D), noise(r.g, n, 2, D))
    for _ in range(4):
        r.ask([0, 1, 2, 3], noise(r.g, 4, 2 * H, D) * 0.05, noise(r.g, 4, 2, D), noise(r.g, 4, 2, D), D ** -0.5, kernel)

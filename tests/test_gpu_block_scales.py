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
    weight rounded to 11 bits where it multiplies values moves outputs past a border."""
    r = Apart(2, 2 * H, D, fmt, torch.bfloat16, n_slots=4, width=2, seed=H)
    for slot, n in enumerate((16, 35, 64, 100)):
        r.fill(slot, noise(r.g, n, 2, D), noise(r.g, n, 2, D))
    for _ in range(4):
        r.ask([0, 1, 2, 3], noise(r.g, 4, 2 * H, D) * 0.05, noise(r.g, 4, 2, D), noise(r.g, 4, 2, D), D ** -0.5, kernel)


SHAPES = [(torch.int8, 128, 8), (torch.int8, 64, 5), (torch.float8_e4m3fn, 128, 4)]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt, D, H", SHAPES)
@pytest.mark.parametrize("power", [10, 20, 30, 60])
def test_large_values_that_have_next_to_no_weight(kernel, dtype, fmt, D, H, power):
    """A block whose values are 2^power times the others': its keys lie so far below that it contributes a millionth of the output.  In front, in the middle,
    last, and both the first and the last of a sequence."""
    n, scale = 700, D ** -0.5
    r = Apart(1, H, D, fmt, dtype, n_slots=4, width=11, seed=power)
    below = (power + 20) * 0.6931472
    for slot, where in enumerate([(0,), (21,), (42,), (0, 42)]):
        k, v = noise(r.g, n, 1, D) * 0.5, noise(r.g, n, 1, D)
        k[..., 0] = 0
        for blk in where:
            rows = slice(blk * BLOCK, (blk + 1) * BLOCK)
            k[rows] *= 0.01
            k[rows, :, 0] = -below / (4 * scale)
            v[rows] *= 2.0 ** power
        r.fill(slot, k, v)
    for splits in (0, 1) if kernel is not True else (0,):
        q = noise(r.g, 4, H, D) * 0.3
        q[..., 0] = 4
        k, v = noise(r.g, 4, 1, D) * 0.5, noise(r.g, 4, 1, D)
        k[..., 0] = 0
        r.ask([0, 1, 2, 3], q, k, v, scale, kernel, splits=splits)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt, D, H", SHAPES)
@pytest.mark.parametrize("nats", [12, 18, 24])
def test_a_key_far_above_the_others_with_a_value_near_zero(kernel, dtype, fmt, D, H, nats):
    """What a first token often is: all the weight, and nothing to say.  Its block's values are zeros, or those of its neighbours ordinary."""
    n, scale = 4096 + 5, D ** -0.5
    r = Apart(1, H, D, fmt, dtype, n_slots=3, width=65, seed=nats)
    for slot, (at, alone) in enumerate([(0, True), (0, False), (2000, False)]):
        k, v = noise(r.g, n, 1, D) * 0.5, noise(r.g, n, 1, D)
        k[..., 0] = 0
        v += 0.5                                    # (values that add up)
        blk = slice(at // BLOCK * BLOCK, at // BLOCK * BLOCK + BLOCK)
        if alone:
            v[blk] = 0
        k[blk] *= 0.01
        k[at, :, 0] = nats / (4 * scale)
        v[at] = 0
        r.fill(slot, k, v)
    for splits in (0, 1) if kernel is not True else (0,):
        q = noise(r.g, 3, H, D) * 0.1
        q[..., 0] = 4
        k, v = noise(r.g, 3, 1, D) * 0.5, noise(r.g, 3, 1, D)
        k[..., 0] = 0
        r.ask([0, 1, 2], q, k, v, scale, kernel, splits=splits)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt, D, H", SHAPES)
def test_values_that_grow_and_shrink_from_block_to_block(kernel, dtype, fmt, D, H):
    """Value sizes from 2^-40 to 2^40 in no order, keys alike: the largest block is what counts, wherever it stands.  And all values tiny, or large."""
    n, scale = 1000, D ** -0.5
    r = Apart(1, H, D, fmt, dtype, n_slots=4, width=17, seed=5)
    for slot in range(4):
        k, v = noise(r.g, n, 1, D) * 0.5, noise(r.g, n, 1, D)
        if slot < 2:
            powers = torch.randint(-40, 41, (-(-n // BLOCK),), generator=r.g).repeat_interleave(BLOCK)[:n].view(-1, 1, 1)
            v = v * torch.exp2(powers.float())
        else:
            v = v * (2.0 ** -90 if slot == 2 else 2.0 ** 90)
        r.fill(slot, k, v)
    q, k, v = noise(r.g, 4, H, D) * 0.5, noise(r.g, 4, 1, D) * 0.5, noise(r.g, 4, 1, D)
    v[2:] = 0
    for splits in (0, 1) if kernel is not True else (0,):
        r.ask([0, 1, 2, 3], q, k, v, scale, kernel, splits=splits)


@pytest.mark.parametrize("kernel, splits", [(True, 0), (False, 0), ("digits", 0), ("digits", 1), ("digits", 8), ("digits", 9)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("odd", [float("inf"), float("nan"), 3e38, 2.0 ** 40])
@pytest.mark.parametrize("ring", [None, 5])
def test_blocks_in_front_of_a_window(kernel, splits, dtype, odd, ring):
    """Scales of blocks that the window has left, in the page of its first one, change nothing, not a bit."""
    window, n, D = 260, 700 + 16 * 3, 128
    outs = []
    for poison in (False, True):
        r = Apart(1, 4, D, torch.int8, dtype, n_slots=3, width=17, window=window, ring=ring, seed=3)
        for slot, m in enumerate((n, n - 16, n - 32)):            # the window's first block stands third, second and first in its page
            r.fill(slot, noise(r.g, m, 1, D), noise(r.g, m, 1, D))
            first = (m + 1 - window) // BLOCK
            if poison:
                for blk in range(first // 4 * 4, first):
                    page = int(r.table_host[slot, blk // 4 % r.ring])
                    r.v_scale[page, :, blk % 4] = odd
                    r.k_scale[page, :, blk % 4] = odd
        q, k, v = noise(r.g, 3, 4, D), noise(r.g, 3, 1, D), noise(r.g, 3, 1, D)
        outs.append(r.ask([0, 1, 2], q, k, v, D ** -0.5, kernel, splits=splits))
    assert torch.equal(*outs)

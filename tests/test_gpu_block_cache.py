"""The 8-bit cache: storing prompts and one-token attention against a plain statement in 64 bits (tests/block_reference.py), at the
lengths, types, head layouts, windows and page tables where they can go wrong."""
import numpy as np
import pytest
import torch

from block_reference import BLOCK, PlainCache, attend, attend_bounds, levels_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
FORMATS = [torch.int8, torch.float8_e4m3fn]
KERNELS = [True, False, "digits"]            # plain; by the kernels' rules; on tcgen05 wherever it can be (int8 levels, heads of 128, up to eight to a key head)


def how(plain):
    return {"plain": plain is True, "groups": 1 if plain == "digits" else 0}


def B():
    from inference_engine_rust_b200.csrc import bindings
    return bindings


def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device=DEV)


class Rig:
    """A cache of one layer over pages in no order, everything that nobody wrote poisoned, and the same in plain form."""

    def __init__(self, kv_heads, heads, dim, fmt, dtype, n_slots=3, width=4, window=0, ring=None, weights=False, page_tokens=64, seed=0, shift=None):
        self.g = torch.Generator().manual_seed(seed)
        self.G, self.H, self.D, self.fmt, self.dtype, self.window, self.PT = kv_heads, heads, dim, fmt, dtype, window, page_tokens
        self.per = page_tokens // BLOCK
        n_pages = n_slots * width + 2
        self.n_pages, self.n_slots = n_pages, n_slots
        nan = float("nan")
        poison = torch.full((n_pages, kv_heads, page_tokens, dim), 99.0 if fmt == torch.int8 else nan, device=DEV)
        self.k, self.v = poison.to(fmt), poison.to(fmt)
        self.k_scale, self.v_scale = (torch.full((n_pages, kv_heads, self.per), nan, device=DEV) for _ in range(2))
        self.weight = torch.full((n_pages, kv_heads, self.per), nan, device=DEV) if weights else None
        self.tail_k, self.tail_v = (torch.full((n_slots, kv_heads, BLOCK, dim), nan, device=DEV).to(dtype) for _ in range(2))
        table = np.random.default_rng(seed).permutation(n_pages)[:n_slots * width].reshape(n_slots, width)
        if ring is not None:
            table[:, ring:] = -1
        self.table_host, self.table = table, dev(table)
        self.shift = None if shift is None else dev(shift)
        self.err = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.view = B().block_view(self.k, self.v, self.k_scale, self.v_scale, self.tail_k, self.tail_v, self.table, window=window, ring_pages=ring,
                                   weight=self.weight, shift=self.shift)
        self.ring = ring or width
        self.plain = {}
        self.blocks_weight = {}                 # slot -> list per block of [G] weights

    def rows(self, n, spread=1.0):
        x = torch.randn(n, (self.H + 2 * self.G), self.D, generator=self.g)
        x[:, :, ::5] *= 3                       # a few large channels
        return (x * spread).to(self.dtype)

    def batch(self, slots, q_lens, pos0, pad_seqs=0, pad_tokens=0):
        n, T = len(slots) + pad_seqs, sum(q_lens) + pad_tokens
        cu = np.concatenate([[0], np.cumsum(q_lens), np.full(pad_seqs, sum(q_lens))])
        if pad_seqs and pad_tokens == pad_seqs:               # a padded one-token step: every padding sequence has a token
            cu = np.arange(n + 1)
        arrs = [dev(cu), dev(list(slots) + [-1] * pad_seqs), dev(np.concatenate([np.repeat(np.arange(len(slots)), q_lens), np.full(pad_tokens, -1)])),
                dev(list(pos0) + [0] * pad_seqs)]
        view = B().BatchView(cu_q=arrs[0].data_ptr(), slot_ids=arrs[1].data_ptr(), tok_seq=arrs[2].data_ptr(), pos0=arrs[3].data_ptr(), n_seqs=n, n_tokens=T)
        return view, arrs

    def cache_of(self, slot):
        return self.plain.setdefault(slot, PlainCache(self.G, self.D, self.fmt))

    def store(self, slots, q_lens, **pad):
        pos0 = [len(self.cache_of(s).rows) for s in slots]
        x = self.rows(sum(q_lens))
        view, keep = self.batch(slots, q_lens, pos0, **pad)
        full = torch.cat([x, torch.full((pad.get("pad_tokens", 0),) + x.shape[1:], float("nan"), dtype=x.dtype)])
        B().block_store(full.reshape(len(full), -1).to(DEV), view, self.view, self.H, self.err, B().stream_ptr())
        at = 0
        for s, n in zip(slots, q_lens):
            for r in x[at:at + n]:
                self.cache_of(s).append(r[self.H:self.H + self.G].float(), r[self.H + self.G:].float())
            at += n
        torch.cuda.synchronize()

    def check_content(self, slots):
        """Everything that is visible stands in the cache, to the bit."""
        for s in slots:
            c = self.cache_of(s)
            n = len(c.rows)
            done = n // BLOCK
            for b in range(max(0, done - self.ring * self.per), done):
                page, part = self.table_host[s, (b // self.per) % self.ring], b % self.per
                for i, (q, sc) in enumerate(((self.k, self.k_scale), (self.v, self.v_scale))):
                    got = q[page, :, part * BLOCK:(part + 1) * BLOCK].float().cpu()
                    assert torch.equal(got, c.levels[b][i]), (s, b, i)
                    assert torch.equal(sc[page, :, part].cpu(), c.scales[b][i].float()), (s, b, i)
            for i, t in enumerate((self.tail_k, self.tail_v)):
                want = torch.stack([r[i] for r in c.rows[done * BLOCK:]], 1) if n > done * BLOCK else torch.zeros(self.G, 0, self.D)
                assert torch.equal(t[s, :, :n - done * BLOCK].double().cpu(), want.double()), (s, i)
        assert self.err.item() == 0

    def step(self, slots, pad=0, weight_out=None, plain=True, splits=0, groups=0, scale=None, spread=1.0, check=True, scratch=None):
        """One token for each of `slots`; compares with 64 bits and returns the outputs."""
        b = B()
        if plain == "digits":
            plain, groups = False, 1
        scale = self.D ** -0.5 if scale is None else scale
        x = self.rows(len(slots), spread)
        pos0 = [len(self.cache_of(s).rows) for s in slots]
        for s, r in zip(slots, x):
            self.cache_of(s).append(r[self.H:self.H + self.G].float(), r[self.H + self.G:].float())
        full = torch.cat([x, torch.full((pad,) + x.shape[1:], float("nan"), dtype=x.dtype)]).reshape(len(slots) + pad, -1).to(DEV)
        view, keep = self.batch(slots, [1] * len(slots), pos0, pad_seqs=pad, pad_tokens=pad)
        out = torch.full((len(slots) + pad + 1, self.H * self.D), 7.0, dtype=self.dtype, device=DEV)
        if scratch is None:
            scratch = torch.full((b.block_attention_scratch_floats(len(slots) + pad, self.H, self.view),), float("nan"), device=DEV)
        b.block_attention(full, out, view, self.view, self.H, scale, scratch, self.err, b.stream_ptr(), weight_out=weight_out, plain=plain,
                          splits=splits, groups=groups)
        torch.cuda.synchronize()
        assert (out[-1] == 7).all(), "a row behind the last sequence was written"
        assert (out[len(slots):-1] == 0).all(), "padding sequences"
        for i, s in enumerate(slots if check else []):
            kv = self.cache_of(s).values()
            want, w, mag = attend(x[i, :self.H], kv, scale, self.window)
            bound, rel = attend_bounds(self.D, kv.shape[2], mag, kv[1].abs().max().item(), self.dtype)
            err = (out[i].view(self.H, self.D).double().cpu() - want).abs().max().item()
            assert err <= bound, f"slot {s}: error {err:.3g}, bound {bound:.3g}"
            if self.weight is not None:
                n = kv.shape[2]
                old = self.blocks_weight.setdefault(s, [])
                if pos0[i] % BLOCK == 0:
                    old.append(torch.zeros(self.G, dtype=torch.float64))
                per_block = torch.nn.functional.pad(w, (0, -n % BLOCK)).view(self.G, -1, BLOCK).sum(-1)
                target = weight_out if weight_out is not None else self.weight
                for blk in range(per_block.shape[1]):
                    old[blk] = old[blk] + per_block[:, blk]
                    got = target[self.table_host[s, blk // self.per], :, blk % self.per].double().cpu()
                    off = (got - old[blk]).abs().max().item()
                    # every step adds weights with a relative error `rel` and a rounding of the sum
                    assert off <= (rel + 2.0 ** -22) * (old[blk].max().item() + 1e-30) + 1e-30, (s, blk, off)
        assert self.err.item() == 0
        return out[:len(slots)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G, H, D", [(1, 1, 16), (2, 6, 64), (8, 32, 128), (3, 3, 48), (1, 5, 24), (2, 2, 33)])
def test_prompts(fmt, dtype, G, H, D):
    r = Rig(G, H, D, fmt, dtype, n_slots=5, width=5, weights=True, seed=D)
    r.store([3, 0, 4, 1], [1, 64, 37, 16 * 17 + 15])
    r.check_content([3, 0, 4, 1])
    r.store([2, 3], [15, 1])                    # a prompt of fewer than 16; one more for a sequence that has one
    r.check_content([2, 3, 0])


@pytest.mark.parametrize("q", [1, 14, 15, 16, 17, 31, 33, 100])
@pytest.mark.parametrize("start", [0, 1, 15, 16, 47])
def test_rows_for_a_running_sequence(start, q):
    r = Rig(2, 4, 64, torch.int8, torch.bfloat16, n_slots=2, width=4, seed=start * 131 + q)
    if start:
        r.store([1], [start])
    r.store([1, 0], [q, 5])
    r.check_content([0, 1])


def test_prompts_padded_for_a_graph():
    r = Rig(2, 4, 64, torch.float8_e4m3fn, torch.bfloat16, n_slots=6, width=3, seed=1)
    r.store([5, 0, 2], [20, 1, 90], pad_seqs=5, pad_tokens=17)
    r.check_content([5, 0, 2])
    assert torch.isnan(r.tail_k[[1, 3, 4]].float()).all() and torch.isnan(r.k_scale[r.table.long()[[1, 3, 4]]]).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_of_zeros_and_of_extremes(fmt):
    """All zeros, numbers around fp32's smallest, its largest, one infinite, one NaN: levels and scales to the bit (what is not
    a number reaches the scale, so that whoever reads the block sees it)."""
    r = Rig(1, 1, 32, fmt, torch.float32, n_slots=8, width=1)
    x = torch.randn(8, BLOCK, 32, generator=r.g)
    x[0] = 0
    x[1] *= 1e-42
    x[2] *= 1e-38
    x[3] *= 1e38
    x[4, 3, 4] = float("inf")
    x[5, 2, 2] = float("nan")
    x[6] = -x[6].abs()
    x[7, 0, 0] = 1e6
    qkv = torch.cat([torch.zeros(8 * BLOCK, 32), x.view(-1, 32), x.view(-1, 32) * 0.5], 1).to(DEV)
    view, keep = r.batch(range(8), [BLOCK] * 8, [0] * 8)
    B().block_store(qkv, view, r.view, 1, r.err, B().stream_ptr())
    for s in range(8):
        got, sc = r.k[r.table_host[s, 0], 0, :BLOCK].float().cpu(), r.k_scale[r.table_host[s, 0], 0, 0].cpu()
        if s == 4:
            assert torch.isinf(sc)
        elif s == 5:
            assert torch.isnan(sc)
        else:
            q, scale = levels_of(x[s], fmt)
            assert torch.equal(got, q) and torch.equal(sc, scale.float()), s
            # half a step of what the block's largest number allows (subnormal scales aside)
            step = scale * 0.5 if fmt == torch.int8 else torch.maximum(x[s].abs() * 2.0 ** -4, scale * 2.0 ** -10)
            assert ((q * scale - x[s]).abs() <= step * (1 + 2.0 ** -20) + 2.0 ** -149).all(), s


LENS = [0, 1, 14, 15, 16, 17, 63, 64, 65, 127, 128, 200, 255]


@pytest.mark.parametrize("plain", KERNELS)
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G, H, D", [(1, 1, 64), (2, 8, 128), (8, 32, 128), (2, 24, 64), (1, 20, 128), (1, 5, 24), (3, 6, 48), (1, 2, 256)])
def test_one_token_steps(plain, fmt, dtype, G, H, D):
    """All lengths at once, six tokens in a row: blocks begin and finish on the way."""
    n = len(LENS)
    r = Rig(G, H, D, fmt, dtype, n_slots=n + 1, width=5, weights=True, seed=H)
    slots = list(np.random.default_rng(1).permutation(n + 1)[:n])
    live = [(s, x) for s, x in zip(slots, LENS) if x]
    r.store([s for s, _ in live], [x for _, x in live])
    for s, x in live:
        r.blocks_weight[s] = [torch.zeros(G, dtype=torch.float64) for _ in range(-(-x // BLOCK))]
    for i in range(6):
        r.step(slots, plain=plain, pad=3 if i == 2 else 0)
    r.check_content(slots)
    other = [s for s in range(n + 1) if s not in slots]
    assert torch.isnan(r.tail_k[other].float()).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("groups, splits", [(1, 1), (1, 4), (1, 8), (2, 1), (2, 2), (2, 8), (2, 9), (2, 16)])
@pytest.mark.parametrize("D, H", [(64, 5), (128, 5), (128, 12)])
def test_a_key_head_shared_by_ctas(fmt, groups, splits, D, H):
    """Long and short sequences, more CTAs than blocks among them, more than 64 blocks for a warp."""
    lens = [0, 5, 16, 40, 100, 1023, 2500, 16 * 32 * 4 * 2 + 17]
    r = Rig(1, H, D, fmt, torch.bfloat16, n_slots=8, width=66, weights=True, seed=splits)
    slots = [3, 1, 0, 7, 2, 5, 6, 4]
    live = [(s, x) for s, x in zip(slots, lens) if x]
    r.store([s for s, _ in live], [x for _, x in live])
    for s, x in live:
        r.blocks_weight[s] = [torch.zeros(1, dtype=torch.float64) for _ in range(-(-x // BLOCK))]
    umma = D == 128 and H <= 8 and fmt == torch.int8
    for pad in (0, 8):
        r.step(slots, plain=False, splits=splits if umma or splits != 9 else 8, groups=groups, pad=pad)
    r.check_content(slots)


@pytest.mark.parametrize("plain", KERNELS)
@pytest.mark.parametrize("window, ring", [(1, 1), (16, 1), (17, 1), (64, 1), (65, 2), (100, 2), (128, 2), (1000, None)])
@pytest.mark.parametrize("D", [64, 128, 40])
def test_windows_and_rings(plain, window, ring, D):
    """Windows that end inside a block and rings that have gone round: the prompt brings only what the ring holds, steps go on from there."""
    r = Rig(2, 6, D, torch.int8, torch.bfloat16, n_slots=4, width=8, window=window, ring=ring, seed=window)
    r.store([0, 1, 2, 3], [300, 129, 5, 63])
    r.check_content([0, 1, 2, 3])
    for _ in range(40):
        r.step([3, 0, 2, 1], plain=plain)
    r.check_content([0, 1, 2, 3])


@pytest.mark.parametrize("plain", KERNELS)
def test_pages_of_other_sizes(plain):
    for pt in (16, 48, 128):
        r = Rig(2, 4, 64, torch.int8, torch.bfloat16, n_slots=2, width=9, weights=True, page_tokens=pt, seed=pt)
        r.store([1], [100])
        r.blocks_weight[1] = [torch.zeros(2, dtype=torch.float64) for _ in range(7)]
        for _ in range(20):
            r.step([1, 0], plain=plain)
        r.check_content([0, 1])


@pytest.mark.parametrize("plain", KERNELS)
def test_weights_elsewhere(plain):
    """Weights into another array: the view's own stay, and of the other only the sequences' blocks are written."""
    r = Rig(2, 4, 128, torch.int8, torch.bfloat16, n_slots=2, width=3, weights=True, seed=5)
    r.store([0, 1], [70, 31])
    r.blocks_weight = {0: [torch.zeros(2, dtype=torch.float64) for _ in range(5)], 1: [torch.zeros(2, dtype=torch.float64) for _ in range(2)]}
    r.step([0, 1], plain=plain)                      # in place
    before = r.weight.clone()
    out = torch.full_like(r.weight, 5.0)
    r.step([0, 1], plain=plain, weight_out=out)
    assert torch.equal(torch.nan_to_num(r.weight), torch.nan_to_num(before))
    used = {(int(r.table_host[s, b // 4]), b % 4) for s, n in ((0, 72), (1, 33)) for b in range(-(-n // 16))}
    for page in range(r.n_pages):
        for part in range(4):
            if (page, part) not in used:
                assert (out[page, :, part] == 5).all()


@pytest.mark.parametrize("plain", KERNELS)
@pytest.mark.parametrize("D", [128, 24])
@pytest.mark.parametrize("pairing", [0, 1])
def test_rotation_inside_the_kernel(plain, D, pairing):
    """Rotated in front (the framework's own kernel) and stored, or rotated inside: the same keys, outputs as near as queries in
    fp32 and in bfloat16 are.  Positions lie `shift` above the rows."""
    b = B()
    shift = [0, 37, 5]
    rs = [Rig(2, 4, D, torch.int8, torch.float32, n_slots=3, width=3, seed=9, shift=shift) for _ in range(2)]
    rot = D // 4 * 2
    inv = (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) * 2 / rot)).float().to(DEV)
    for r in rs:
        r.store([0, 1], [50, 15])
    for i in range(3):
        outs = []
        for fused, r in zip((True, False), rs):
            slots, pos0 = [0, 1, 2], [50 + i, 15 + i, i]
            x = torch.randn(3, 8 * D, generator=torch.Generator().manual_seed(i)).to(DEV)
            view, keep = r.batch(slots, [1] * 3, pos0)
            where, keep2 = r.batch(slots, [1] * 3, [p + shift[s] for p, s in zip(pos0, slots)])
            out = torch.empty(3, 4 * D, device=DEV)
            if not fused:
                b.rotate_qk(x, where, inv, 4, 2, D, rot, pairing, r.err, b.stream_ptr(), rot_mul=1.25)
            scratch = torch.empty(b.block_attention_scratch_floats(3, 4, r.view), device=DEV)
            b.block_attention(x, out, view, r.view, 4, D ** -0.5, scratch, r.err, b.stream_ptr(), rope=(inv, rot, pairing, 1.25) if fused else None, **how(plain))
            outs.append(out)
        # the same rotation in fp32 (contracted or not: two roundings of a sum of two products) before the same sums
        assert (outs[0] - outs[1]).abs().max().item() <= 1e-4
    for x, y in ((rs[0].tail_k, rs[1].tail_k), (rs[0].tail_v, rs[1].tail_v)):
        assert (torch.nan_to_num(x) - torch.nan_to_num(y)).abs().max().item() <= 8 * 2.0 ** -22
    assert rs[0].err.item() == 0 and rs[1].err.item() == 0


@pytest.mark.parametrize("plain", KERNELS)
def test_bad_pages_and_slots_set_the_error_word(plain):
    b = B()
    r = Rig(2, 4, 64, torch.int8, torch.bfloat16, n_slots=3, width=2, weights=True, seed=11)
    r.store([0, 1, 2], [40, 40, 40])
    good = r.table.clone()
    for bad in (-1, r.n_pages, 1 << 30):
        r.table[1, 0] = bad
        view, keep = r.batch([0, 1, 2], [1] * 3, [40] * 3)
        x, out = r.rows(3).reshape(3, -1).to(DEV), torch.empty(3, 4 * 64, dtype=torch.bfloat16, device=DEV)
        scratch = torch.zeros(b.block_attention_scratch_floats(3, 4, r.view), device=DEV)
        b.block_attention(x, out, view, r.view, 4, 0.125, scratch, r.err, b.stream_ptr(), **how(plain))
        assert r.err.item() == b.ERR_PAGE_RANGE
        r.err.zero_()
        r.table.copy_(good)
    for slot in (3, 1000):                                      # a slot that the cache does not have: as padding
        view, keep = r.batch([0, slot, 2], [1] * 3, [40] * 3)
        b.block_attention(x, out, view, r.view, 4, 0.125, scratch, r.err, b.stream_ptr(), **how(plain))
        assert r.err.item() == b.ERR_PAGE_RANGE and (out[1] == 0).all() and torch.isfinite(out.float()).all()
        r.err.zero_()
    # a sequence longer than its row of the table
    view, keep = r.batch([0], [1], [128])
    b.block_attention(x[:1], out[:1], view, r.view, 4, 0.125, scratch, r.err, b.stream_ptr(), **how(plain))
    assert r.err.item() == b.ERR_PAGE_RANGE and (out[0] == 0).all()
    r.err.zero_()
    r.table[1, 0] = -1
    view, keep = r.batch([1], [16], [0])
    b.block_store(r.rows(16).reshape(16, -1).to(DEV), view, r.view, 4, r.err, b.stream_ptr())
    assert r.err.item() == b.ERR_PAGE_RANGE


@pytest.mark.parametrize("plain", KERNELS)
def test_what_is_not_a_number_stays_where_it_is_seen(plain):
    """A NaN among one sequence's values reaches that sequence's heads alone; positions outside a window reach nobody."""
    r = Rig(2, 4, 64, torch.int8, torch.bfloat16, n_slots=3, width=3, window=30, seed=13)
    r.store([0, 1, 2], [100, 100, 100])
    clean = r.view
    page = r.table_host[1, 5 // 4]
    r.v_scale[page, 0, 1] = float("nan")                        # block 5 of slot 1 (positions 80 to 95), kv head 0: inside the window
    page = r.table_host[2, 0]
    r.v_scale[page, :, :3] = float("nan")                       # far outside the window of slot 2
    r.k_scale[page, :, :3] = float("inf")
    out = r.step([0, 1, 2], plain=plain, check=False).view(3, 4, 64)
    assert torch.isfinite(out[0].float()).all() and torch.isfinite(out[2].float()).all()
    assert torch.isnan(out[1, :2].float()).all() and torch.isfinite(out[1, 2:].float()).all()
    assert clean is r.view


@pytest.mark.parametrize("plain", KERNELS)
def test_large_scores(plain):
    """Scores of several hundred: one position takes nearly all the weight; nothing overflows."""
    r = Rig(2, 8, 128, torch.int8, torch.float32, n_slots=2, width=4, weights=True, seed=14)
    r.store([0, 1], [150, 33])
    r.blocks_weight = {0: [torch.zeros(2, dtype=torch.float64) for _ in range(10)], 1: [torch.zeros(2, dtype=torch.float64) for _ in range(3)]}
    for spread in (1e-3, 1.0, 8.0):
        r.step([0, 1], plain=plain, spread=spread)


@pytest.mark.parametrize("plain", KERNELS)
def test_on_another_stream_and_captured(plain):
    b = B()
    outs = []
    for mode in ("eager", "stream", "graph"):
        r = Rig(2, 8, 128, torch.int8, torch.bfloat16, n_slots=2, width=4, weights=True, seed=15)
        r.store([0, 1], [150, 31])
        x = r.rows(2).reshape(2, -1).to(DEV)
        view, keep = r.batch([0, 1], [1, 1], [150, 31])
        out, scratch = torch.empty(2, 8 * 128, dtype=torch.bfloat16, device=DEV), torch.zeros(b.block_attention_scratch_floats(2, 8, r.view), device=DEV)

        def go():
            b.block_attention(x, out, view, r.view, 8, 0.1, scratch, r.err, b.stream_ptr(), **how(plain))
        torch.cuda.synchronize()
        if mode == "eager":
            go()
        elif mode == "stream":
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                go()
            side.synchronize()
        else:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                go()
            graph.replay()
        torch.cuda.synchronize()
        outs.append((out, r.weight[r.table.long()], r.tail_k, r.k_scale[r.table.long()]))
    for got in outs[1:]:
        for a, c in zip(outs[0], got):
            assert torch.equal(torch.nan_to_num(a.float()), torch.nan_to_num(c.float()))


@pytest.mark.parametrize("plain", KERNELS)
def test_equal_calls_give_equal_bits(plain):
    """No sum depends on what runs when."""
    got = []
    for _ in range(3):
        r = Rig(4, 16, 128, torch.int8, torch.bfloat16, n_slots=6, width=20, weights=True, seed=16)
        slots = list(range(6))
        r.store(slots, [1200, 3, 700, 64, 1023, 500])
        for s, n in zip(slots, [1200, 3, 700, 64, 1023, 500]):
            r.blocks_weight[s] = [torch.zeros(4, dtype=torch.float64) for _ in range(-(-n // BLOCK))]
        got.append((r.step(slots, plain=plain), torch.nan_to_num(r.weight)))
    for o, w in got[1:]:
        assert torch.equal(o, got[0][0]) and torch.equal(w, got[0][1])


def test_more_tiles_than_a_sum_of_integers_may_take():
    """40,000 positions done by one CTA: the 32-bit sums of products of levels and digits are emptied on the way."""
    r = Rig(1, 3, 128, torch.int8, torch.bfloat16, n_slots=1, width=626, weights=True, seed=17)
    r.store([0], [40_000])
    r.blocks_weight[0] = [torch.zeros(1, dtype=torch.float64) for _ in range(2500)]
    r.step([0], plain=False, splits=1, groups=1)


def test_values_and_probabilities_at_their_largest():
    """Every probability alike and every value's level 127 (or -127): the largest sums there are.  The answer is the value itself: levels
    and scale give it back with the rounding of the scale and of one product."""
    b = B()
    r = Rig(1, 8, 128, torch.int8, torch.float32, n_slots=1, width=626, seed=18)
    x = torch.zeros(40_001, 10, 128)
    x[:, 9, ::2], x[:, 9, 1::2] = 3.7, -3.7
    x = x.reshape(40_001, -1).to(DEV)
    view, keep = r.batch([0], [40_000], [0])
    b.block_store(x[:40_000], view, r.view, 8, r.err, b.stream_ptr())
    view, keep = r.batch([0], [1], [40_000])
    out, scratch = torch.empty(1, 1024, device=DEV), torch.empty(b.block_attention_scratch_floats(1, 8, r.view), device=DEV)
    b.block_attention(x[40_000:], out, view, r.view, 8, 1.0, scratch, r.err, b.stream_ptr(), splits=1, groups=1)
    want = x[40_000:, -128:].repeat(1, 8)
    # scale, product and quotient; the sum of 40,000 weights in one CTA: below 320 additions a thread, then 7 of partial sums, and as many of the outputs
    assert (out - want).abs().max().item() <= 3.7 * (2 * 330 + 6) * 2.0 ** -24
    assert r.err.item() == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("G, n", [(2, 160), (1, 300)])
def test_more_sequences_than_run_at_once(fmt, G, n):
    """The longest first where they can be put in order (up to 256), as they stand where not."""
    r = Rig(G, 4, 128, fmt, torch.bfloat16, n_slots=n, width=4, weights=True, seed=n)
    g = np.random.default_rng(n)
    slots, lens = list(g.permutation(n)), g.integers(1, 250, n)
    lens[:5] = 200                                    # equal ones
    r.store(slots, list(lens))
    for s, x in zip(slots, lens):
        r.blocks_weight[s] = [torch.zeros(G, dtype=torch.float64) for _ in range(-(-int(x) // BLOCK))]
    r.step(slots, plain=False, pad=5)
    r.check_content(slots)


def test_a_table_that_reaches_far():
    """Few sequences that may become long: CTAs that are no cluster, and a second kernel, by the kernel's own rule."""
    r = Rig(1, 5, 128, torch.int8, torch.bfloat16, n_slots=3, width=260, weights=True, seed=19)
    r.store([2, 0], [3000, 15])
    r.blocks_weight = {s: [torch.zeros(1, dtype=torch.float64) for _ in range(-(-n // BLOCK))] for s, n in ((2, 3000), (0, 15))}
    for pad in (0, 1):
        r.step([2, 0, 1], plain=False, pad=pad)
    r.check_content([0, 1, 2])


@pytest.mark.parametrize("groups, splits", [(1, 2), (2, 1), (2, 9)])
def test_bad_pages_and_numbers_where_integers_are_multiplied(groups, splits):
    """Heads of 128 over int8 levels: a page that is not there counts for nothing and sets the error word, a scale that is no number
    reaches the heads of its key head alone."""
    b = B()
    r = Rig(2, 8, 128, torch.int8, torch.bfloat16, n_slots=3, width=5, weights=True, seed=20)
    r.store([0, 1, 2], [300, 300, 300])
    r.weight.zero_()
    good, x = r.table.clone(), r.rows(3).reshape(3, -1).to(DEV)
    scratch = torch.zeros(b.block_attention_scratch_floats(3, 8, r.view), device=DEV)

    def go(slots, pos):
        view, keep = r.batch(slots, [1] * len(slots), pos)
        out = torch.full((len(slots), 8 * 128), 7.0, dtype=torch.bfloat16, device=DEV)
        b.block_attention(x[:len(slots)], out, view, r.view, 8, 0.1, scratch, r.err, b.stream_ptr(), splits=splits, groups=groups)
        torch.cuda.synchronize()
        err = r.err.item()
        r.err.zero_()
        return out.float(), err
    for bad in (-1, r.n_pages, 1 << 30):
        r.table[1, 1] = bad
        out, err = go([0, 1, 2], [300] * 3)
        assert err == b.ERR_PAGE_RANGE and torch.isfinite(out).all()
        r.table.copy_(good)
    out, err = go([0, 3, 2], [300] * 3)                       # a slot that the cache does not have
    assert err == b.ERR_PAGE_RANGE and (out[1] == 0).all() and torch.isfinite(out).all()
    out, err = go([0], [320])                                 # longer than its row of the table
    assert err == b.ERR_PAGE_RANGE and (out == 0).all()
    for scale in (r.k_scale, r.v_scale):
        at = (int(good[1, 2]), 0, 1)
        was = scale[at].item()
        scale[at] = float("nan")
        out, err = go([0, 1, 2], [300] * 3)
        out = out.view(3, 8, 128)
        assert err == 0 and torch.isfinite(out[0]).all() and torch.isfinite(out[2]).all()
        assert torch.isnan(out[1, :4]).all() and torch.isfinite(out[1, 4:]).all()
        scale[at] = was
    out, err = go([0, 1, 2], [300] * 3)
    assert err == 0 and torch.isfinite(out).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_two_steps_at_once(fmt):
    """Two steps of different sequences on two streams, each with scratch of its own."""
    b = B()
    outs = []
    for apart in (False, True):
        rigs = [Rig(2, 8, 128, fmt, torch.bfloat16, n_slots=4, width=20, weights=True, seed=21 + i) for i in range(2)]
        for r in rigs:
            r.store([0, 1, 2, 3], [1000, 31, 700, 16])
            r.weight.zero_()
        torch.cuda.synchronize()
        got, keep = [], []
        for r, stream in zip(rigs, [torch.cuda.Stream() for _ in rigs] if apart else [torch.cuda.current_stream()] * 2):
            with torch.cuda.stream(stream):
                x = r.rows(4).reshape(4, -1).to(DEV)
                view, arrs = r.batch([0, 1, 2, 3], [1] * 4, [1000, 31, 700, 16])
                out, scratch = torch.empty(4, 8 * 128, dtype=torch.bfloat16, device=DEV), torch.empty(b.block_attention_scratch_floats(4, 8, r.view), device=DEV)
                for _ in range(5):
                    b.block_attention(x, out, view, r.view, 8, 0.1, scratch, r.err, b.stream_ptr())
                got.append((out, r.weight))
                keep.append((x, view, arrs, scratch))
        torch.cuda.synchronize()
        outs.append(got)
    for one, two in zip(*outs):
        for a, c in zip(one, two):
            assert torch.equal(a, c)


def test_numbers_of_ctas_that_no_kernel_takes():
    from inference_engine_rust_b200.csrc.bindings import KernelError
    for D, splits in ((128, 3), (128, 200), (64, 9), (64, 32), (24, 2)):
        r = Rig(1, 5, D, torch.int8, torch.bfloat16, n_slots=1, width=2, seed=22)
        with pytest.raises(KernelError):
            r.step([0], plain=False, splits=splits)

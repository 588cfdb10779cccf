"""Penalties, biases and masks on logits against the formulas in 64 bits, at the sizes and rows where they can go wrong."""
import numpy as np
import pytest
import torch

from block_reference import rules as plain_rules

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def B():
    from inference_engine_rust_b200.csrc import bindings
    return bindings


def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device=DEV)


def bits_of(allowed):
    """bool [R, V] -> int32 [R, ceil(V / 32)]."""
    R, V = allowed.shape
    full = np.zeros((R, -(-V // 32) * 32), dtype=np.uint64)
    full[:, :V] = allowed
    words = (full.reshape(R, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)
    return torch.from_numpy(words.view(np.int32)).to(DEV)


class Case:
    def __init__(self, R, V, H=None, width=40, seed=0, pad=0, penalties=True, bias="row", mask=True, rounded=False):
        g = np.random.default_rng(seed)
        H = R + 2 if H is None else H
        store = torch.from_numpy(g.normal(size=(R, V + pad)).astype(np.float32) * 4).to(DEV)
        if rounded:
            store = store.round()                              # many equal logits: ties
        self.store, self.logits = store, store[:, :V]
        self.rows = g.permutation(H)[:R]
        self.lens = g.integers(0, width + 1, size=H)
        self.lens[self.rows] = np.minimum(self.lens[self.rows], width - 1)
        self.prompt = (self.lens * g.uniform(0, 1, H)).astype(int)
        self.history = (g.uniform(0, 1, (H, width)) ** 3 * V * 1.02).astype(np.int64)     # a few ids lie outside the vocabulary
        self.history[:, ::7] = -1
        self.penalties = np.stack([g.uniform(0.7, 1.6, H), g.uniform(-0.5, 1, H), g.uniform(-0.2, 0.6, H)], 1).astype(np.float32) if penalties else None
        self.bias = None if bias is None else (g.normal(size=(R, V) if bias == "rows" else (V,)) * (g.uniform(0, 1, V) < 0.2)).astype(np.float32)
        self.allowed = g.uniform(0, 1, (R, V)) < 0.6 if mask else None
        if mask:
            self.allowed[:, g.integers(0, V)] = True

    def run(self, out=None, append=True, choose=True):
        d = {"history": dev(self.history), "lens": dev(self.lens), "prompt": dev(self.prompt), "rows": dev(self.rows),
             "err": torch.zeros(1, dtype=torch.int32, device=DEV), "chosen": torch.full((len(self.rows),), -5, dtype=torch.int32, device=DEV)}
        d["out"] = torch.empty_like(self.logits) if out is None else out
        B().logit_rules(self.logits, d["out"], d["history"], d["lens"], d["prompt"], d["rows"], d["err"], B().stream_ptr(),
                        penalties=None if self.penalties is None else dev(self.penalties, torch.float32),
                        bias=None if self.bias is None else dev(self.bias, torch.float32),
                        mask=None if self.allowed is None else bits_of(self.allowed), chosen=d["chosen"] if choose else None,
                        lens_out=d["lens"] if append else None)
        torch.cuda.synchronize()
        return d

    def check(self, d, before):
        got = d["out"].cpu().numpy()
        for r, h in enumerate(self.rows):
            want, bound = plain_rules(before[r], self.history[h, :self.lens[h]], self.prompt[h], None if self.penalties is None else self.penalties[h],
                                      None if self.bias is None else self.bias[r] if self.bias.ndim == 2 else self.bias,
                                      None if self.allowed is None else self.allowed[r])
            assert np.array_equal(np.isneginf(got[r]), np.isneginf(want)), r
            ok = np.isfinite(want)
            assert (np.abs(got[r][ok] - want[ok]) <= bound[ok]).all(), r
            chosen = int(d["chosen"][r])
            assert chosen == int(np.argmax(got[r])), r          # the first of the largest
            assert want[chosen] >= want.max() - 2 * bound[ok].max(), r
            n = self.lens[h]
            assert int(d["history"][h, n]) == chosen and int(d["lens"][h]) == n + 1, r
        others = [h for h in range(len(self.lens)) if h not in set(self.rows.tolist())]
        assert torch.equal(d["history"][others].cpu(), torch.from_numpy(self.history[others]).int())
        assert torch.equal(d["lens"][others].cpu(), torch.from_numpy(self.lens[others]).int())
        assert d["err"].item() == 0


@pytest.mark.parametrize("V", [1, 2, 31, 33, 100, 128, 331, 1024, 1027, 4096, 40007, 131072, 200003])
@pytest.mark.parametrize("R", [1, 5])
def test_against_the_formulas(R, V):
    c = Case(R, V, seed=V + R)
    c.check(c.run(), c.logits.cpu().numpy())


@pytest.mark.parametrize("penalties", [False, True])
@pytest.mark.parametrize("bias", [None, "row", "rows"])
@pytest.mark.parametrize("mask", [False, True])
def test_every_set_of_rules(penalties, bias, mask):
    c = Case(3, 1000, seed=3, penalties=penalties, bias=bias, mask=mask)
    c.check(c.run(), c.logits.cpu().numpy())


@pytest.mark.parametrize("pad", [1, 3, 4, 64])
def test_rows_with_a_stride_and_in_place(pad):
    c = Case(4, 512, seed=pad, pad=pad)
    before, tail = c.logits.cpu().numpy().copy(), c.store[:, 512:].clone()
    c.check(c.run(out=c.logits), before)
    assert torch.equal(c.store[:, 512:], tail)                  # what lies between the rows stays


def test_ties_go_to_the_lowest_id():
    c = Case(9, 20000, seed=1, penalties=False, bias=None, mask=False, rounded=True)
    c.check(c.run(), c.logits.cpu().numpy())


def test_a_long_history_and_many_rows():
    c = Case(33, 5000, width=9001, seed=4)
    c.check(c.run(), c.logits.cpu().numpy())


def test_no_choice_and_no_append_leave_the_history():
    c = Case(3, 300, seed=5)
    d = c.run(append=False, choose=False)
    assert torch.equal(d["history"].cpu(), torch.from_numpy(c.history).int()) and torch.equal(d["lens"].cpu(), torch.from_numpy(c.lens).int())
    assert (d["chosen"] == -5).all()
    d2 = c.run(append=False)
    assert torch.equal(d["out"], d2["out"])


def test_without_results():
    c = Case(3, 300, seed=6)
    d = {"chosen": torch.zeros(3, dtype=torch.int32, device=DEV), "err": torch.zeros(1, dtype=torch.int32, device=DEV)}
    B().logit_rules(c.logits, None, None, None, None, None, d["err"], B().stream_ptr(), bias=dev(c.bias, torch.float32), chosen=d["chosen"])
    want = (c.logits.cpu() + torch.from_numpy(c.bias)).argmax(1)
    assert torch.equal(d["chosen"].cpu().long(), want) and d["err"].item() == 0


def test_one_mask_and_one_bias_row_for_all():
    c = Case(4, 700, seed=7, penalties=False, bias="row", mask=True)
    c.allowed[:] = c.allowed[:1]
    full = c.run()
    err, chosen, out = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), torch.empty_like(c.logits)
    B().logit_rules(c.logits, out, None, None, None, None, err, B().stream_ptr(), bias=dev(c.bias, torch.float32), mask=bits_of(c.allowed[:1]),
                    chosen=chosen)
    assert torch.equal(out, full["out"]) and torch.equal(chosen, full["chosen"]) and err.item() == 0


def test_what_sets_the_error_word():
    b = B()
    base = torch.randn(2, 640, device=DEV)

    def go(logits, **kw):
        err, chosen = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((2,), 7, dtype=torch.int32, device=DEV)
        out = torch.empty_like(logits)
        b.logit_rules(logits, out, kw.pop("history", None), kw.pop("lens", None), kw.pop("prompt", None), kw.pop("rows", None), err, b.stream_ptr(),
                      chosen=chosen, **kw)
        return err.item(), chosen.tolist(), out
    nothing = torch.zeros(2, 20, dtype=torch.int32, device=DEV)
    nothing[0, 3] = 1 << 4
    err, chosen, out = go(base, mask=nothing)
    assert err == b.ERR_NOTHING_ALLOWED and chosen == [100, 0]
    assert torch.isneginf(out[1]).all() and torch.isfinite(out[0]).sum() == 1
    for bad in (float("nan"), float("inf"), float("-inf")):
        x = base.clone()
        x[1, 77] = bad
        assert go(x)[0] == b.ERR_NONFINITE_LOGIT
        mask = torch.full((2, 20), -1, dtype=torch.int32, device=DEV)
        mask[1, 2] = ~(1 << 13)                                 # a logit that the mask rules out may be anything
        err, chosen, out = go(x, mask=mask)
        assert err == 0 and torch.isneginf(out[1, 77])
        assert chosen == [int(base[0].argmax()), int(base[1].index_fill(0, torch.tensor([77], device=DEV), float("-inf")).argmax())]
    bias = torch.zeros(640, device=DEV)
    bias[5] = float("-inf")
    err, _, out = go(base, bias=bias)
    assert err == 0 and torch.isneginf(out[:, 5]).all()         # a bias that rules out
    for bad in (float("nan"), float("inf")):
        bias[5] = bad
        assert go(base, bias=bias)[0] == b.ERR_NONFINITE_LOGIT
    # a history that is full, and one that does not exist: the logits come out as far as they can, nothing is written out of place
    hist, lens, prompt = torch.zeros(2, 4, dtype=torch.int32, device=DEV), dev([4, 1]), dev([0, 0])
    kw = dict(history=hist, prompt=prompt)
    lens_out = torch.zeros(2, dtype=torch.int32, device=DEV)
    err, chosen, _ = go(base, lens=lens, lens_out=lens_out, **kw)
    assert err == b.ERR_HISTORY and hist[0].tolist() == [0, 0, 0, 0] and hist[1].tolist() == [0, chosen[1], 0, 0] and lens_out.tolist() == [4, 2]
    assert go(base, lens=dev([1, 1]), rows=dev([0, 2]), **kw)[0] == b.ERR_HISTORY


def test_counts_in_more_than_one_window():
    """A vocabulary whose eighth is larger than the counts that stand in shared memory at a time."""
    for pad in (0, 1):
        c = Case(1, 8 * 24576 + 1000, width=3000, seed=9, pad=pad)
        c.check(c.run(), c.logits.cpu().numpy())


@pytest.mark.parametrize("width", [32767, 32768, 40000])
@pytest.mark.parametrize("V", [1000, 1001])
def test_histories_whose_counts_need_more_than_fifteen_bits(width, V):
    """One id stands in nearly all places of the longest histories: its count is right on both sides of the border between word sizes."""
    c = Case(2, V, width=width, seed=11)
    c.lens[c.rows] = width - 1
    c.prompt[c.rows] = [0, 5]
    c.history[:, 3:] = 77
    c.check(c.run(), c.logits.cpu().numpy())


def test_masked_temperature_never_chooses_what_is_ruled_out():
    """Rows with few allowed ids, at many draws: each is allowed, and frequencies follow the softmax of what is left."""
    b = B()
    g = np.random.default_rng(0)
    V, n = 3001, 4000
    allowed = np.sort(g.permutation(V)[:5])
    x = torch.full((V,), float("-inf"))
    x[allowed] = torch.tensor([0.0, 1.0, -1.0, 0.5, 2.0])
    logits = x.to(DEV).expand(n, V)
    out, err = torch.empty(n, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ids, steps = torch.arange(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
    b.sample_temperature_masked(logits, 0.8, 11, ids, steps, out, err, b.stream_ptr())
    assert err.item() == 0
    got = out.cpu().numpy()
    assert set(got.tolist()) <= set(allowed.tolist())
    p = torch.softmax(x[allowed].double() / 0.8, 0).numpy()
    for i, a in enumerate(allowed):
        # a count of n draws: six standard deviations
        assert abs((got == a).sum() - n * p[i]) <= 6 * np.sqrt(n * p[i] * (1 - p[i])), a
    # the same draws choose the same ids where nothing is ruled out, by the ordinary sampler too
    full = torch.randn(64, V, device=DEV)
    o1, o2 = torch.empty(64, dtype=torch.int32, device=DEV), torch.empty(64, dtype=torch.int32, device=DEV)
    b.sample_temperature(full, 0.8, 5, ids[:64], steps[:64], o1, err, b.stream_ptr())
    b.sample_temperature_masked(full, 0.8, 5, ids[:64], steps[:64], o2, err, b.stream_ptr())
    assert torch.equal(o1, o2) and err.item() == 0
    b.sample_temperature_masked(torch.full((1, V), float("-inf"), device=DEV), 1.0, 5, ids[:1], steps[:1], o1[:1], err, b.stream_ptr())
    assert err.item() == b.ERR_NOTHING_ALLOWED and o1[0].item() == 0


def test_on_another_stream_and_captured():
    c = Case(4, 2000, seed=12)
    want = c.run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = c.run()
    for k in ("out", "chosen", "history", "lens"):
        assert torch.equal(want[k], got[k])
    b = B()
    hist, lens, prompt, rows = dev(c.history), dev(c.lens), dev(c.prompt), dev(c.rows)
    pen, bias, mask = dev(c.penalties, torch.float32), dev(c.bias, torch.float32), bits_of(c.allowed)
    err, chosen, out = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), torch.empty_like(c.logits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.logit_rules(c.logits, out, hist, lens, prompt, rows, err, b.stream_ptr(), penalties=pen, bias=bias, mask=mask, chosen=chosen, lens_out=lens)
    graph.replay()
    assert torch.equal(out, want["out"]) and torch.equal(chosen, want["chosen"]) and torch.equal(lens, want["lens"])
    graph.replay()                                              # the second token: its history has one more
    assert torch.equal(lens, torch.where(torch.isin(torch.arange(len(c.lens), device=DEV), rows), want["lens"] + 1, want["lens"]))


@pytest.mark.parametrize("R, V", [(40, 140_000), (40, 70_001), (100, 70_001), (100, 70_016), (300, 70_016), (300, 4099)])
def test_rows_that_fewer_ctas_share(R, V):
    """Clusters of four, two and one: a CTA's ids then are more than it counts at a time."""
    c = Case(R, V, seed=R + V)
    c.check(c.run(), c.logits.cpu().numpy())

"""Eviction by accumulated weight: which blocks stay, and that what stays is what was there."""
import numpy as np
import pytest
import torch

from block_reference import BLOCK, kept_blocks

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def B():
    from inference_engine_rust_b200.csrc import bindings
    return bindings


def dev(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device=DEV)


def run(lens, keep, recent, layers=2, G=2, D=64, fmt=torch.int8, page_tokens=64, seed=0, weights="spread", slots=False, width=None):
    g = np.random.default_rng(seed)
    per, n = page_tokens // BLOCK, len(lens)
    need = [-(-x // page_tokens) for x in lens]
    width = width or max(1, max(need))
    rows = n + 3 if slots else n
    row_of = g.permutation(rows)[:n] if slots else np.arange(n)
    new_w = -(-(keep * BLOCK + BLOCK) // page_tokens)
    n_pages = sum(need) + n * new_w + 3
    order = g.permutation(n_pages)
    table, at = np.full((rows, width), -1, dtype=np.int32), 0
    for i, m in enumerate(need):
        table[row_of[i], :m] = order[at:at + m]
        at += m
    new = order[at:at + n * new_w].reshape(n, new_w)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    shape = (layers, n_pages, G, page_tokens, D)
    k, v = ((torch.randn(shape, generator=gen, device=DEV) * 60).clamp(-127, 127).to(fmt) for _ in range(2))
    ks, vs, w = (torch.rand((layers, n_pages, G, per), generator=gen, device=DEV) for _ in range(3))
    if weights == "ties":
        w = (w * 3).round()
    elif weights == "equal":
        w = torch.full_like(w, 0.25)
    elif weights == "odd":                       # zeros of both signs, negative numbers, infinities, NaN
        pick = torch.tensor([0.0, -0.0, -1.0, float("inf"), float("nan"), 1e-42, 2.0, 2.0], device=DEV)
        w = pick[torch.randint(0, 8, w.shape, generator=gen, device=DEV)]
    before = [t.clone() for t in (k, v, ks, vs, w)]
    kept = torch.full((layers, n, G, keep), -7, dtype=torch.int32, device=DEV)
    err, shift = torch.zeros(1, dtype=torch.int32, device=DEV), torch.full((rows,), 100, dtype=torch.int32, device=DEV)
    B().block_evict(k, v, ks, vs, w, dev(table), dev(lens), dev(new), keep, recent, kept, err, B().stream_ptr(), slots=dev(row_of) if slots else None,
                    shift=shift)
    torch.cuda.synchronize()
    assert err.item() == 0
    want_shift = np.full(rows, 100)
    new_set, seen = set(new.flatten().tolist()), torch.zeros(n_pages, per, dtype=torch.bool)
    wb = before[4].cpu().double().numpy()
    for i, x in enumerate(lens):
        nb = x // BLOCK
        want_shift[row_of[i]] += max(0, nb - keep) * BLOCK
        for layer in range(layers):
            for h in range(G):
                weight = [wb[layer, table[row_of[i], b // per], h, b % per] for b in range(nb)]
                want = kept_blocks(weight, keep, recent)
                got = kept[layer, i, h].tolist()
                assert got == want + [-1] * (keep - len(want)), (i, layer, h)
                src = [(table[row_of[i], b // per], b % per) for b in want]
                dst = [(new[i, t // per], t % per) for t in range(len(want))]
                sp, se = (torch.tensor(a, dtype=torch.long, device=DEV) for a in ([p for p, _ in src], [e for _, e in src]))
                dp, de = (torch.tensor(a, dtype=torch.long, device=DEV) for a in ([p for p, _ in dst], [e for _, e in dst]))
                for now, was in ((ks, before[2]), (vs, before[3]), (w, before[4])):
                    assert torch.equal(now[layer, dp, h, de].view(torch.int32), was[layer, sp, h, se].view(torch.int32))
                for now, was in ((k, before[0]), (v, before[1])):
                    a, c = now.view(torch.uint8)[layer, :, h].view(n_pages, per, -1), was.view(torch.uint8)[layer, :, h].view(n_pages, per, -1)
                    assert torch.equal(a[dp, de], c[sp, se])
                for p, e in dst:
                    seen[p, e] = True
        if x % BLOCK:                            # the weight of the unfinished block goes along
            t = min(nb, keep)
            a, c = w[:, new[i, t // per], :, t % per], before[4][:, table[row_of[i], nb // per], :, nb % per]
            assert torch.equal(a.view(torch.int32), c.view(torch.int32))
            seen[new[i, t // per], t % per] = True
    # nothing else changed: not the old pages, not the places behind a sequence's last block
    rest = ~seen.to(DEV)
    for now, was in zip((ks, vs, w), before[2:]):
        assert torch.equal(now.view(torch.int32).transpose(2, 3)[:, rest], was.view(torch.int32).transpose(2, 3)[:, rest])
    for now, was in ((k, before[0]), (v, before[1])):
        a, c = (t.view(torch.uint8).view(layers, n_pages, G, per, -1).transpose(2, 3)[:, rest] for t in (now, was))
        assert torch.equal(a, c)
    assert shift.tolist() == want_shift.tolist()
    assert not new_set & {int(p) for p in table.flatten() if p >= 0}


@pytest.mark.parametrize("weights", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("keep, recent", [(1, 0), (1, 1), (4, 0), (5, 2), (7, 7), (16, 3)])
def test_choice_and_copies(weights, keep, recent):
    run([16, 17 * 16 + 5, 0, 15, 300, 16 * 16, 64 * 16 + 15], keep, recent, weights=weights, seed=keep * 10 + recent, slots=True)


@pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("D, page_tokens, G", [(128, 64, 8), (1, 16, 1), (33, 48, 3), (256, 128, 1)])
def test_types_and_sizes(fmt, D, page_tokens, G):
    run([500, 1000, 77], 6, 2, layers=3, G=G, D=D, fmt=fmt, page_tokens=page_tokens, seed=D)


def test_long_sequences():
    run([16 * 3000 + 3, 16 * 257], 1000, 100, layers=1, G=1, D=16, weights="ties", seed=1)
    run([16 * 9000], 4096, 0, layers=1, G=2, D=16, seed=2)


def test_a_wide_table_and_many_layers():
    run([100, 160], 3, 1, layers=40, G=1, D=16, seed=3, width=200)


def test_more_blocks_than_shared_memory_holds():
    run([52_003 * BLOCK + 7, 100 * BLOCK], keep=300, recent=20, layers=1, G=1, D=1, page_tokens=16, weights="ties")


def test_no_room_for_an_unfinished_block_sets_the_error_word():
    k, v = (torch.zeros((1, 6, 1, 16, 16), dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs, w = (torch.ones((1, 6, 1, 1), device=DEV) for _ in range(3))
    for length, want in ((48, 0), (49, 4)):
        err, kept = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros((1, 1, 1, 2), dtype=torch.int32, device=DEV)
        B().block_evict(k, v, ks, vs, w, dev([[0, 1, 2, 3]]), dev([length]), dev([[4, 5]]), 2, 1, kept, err, B().stream_ptr())
        assert err.item() == want


def test_bad_pages_and_rows_set_the_error_word():
    b = B()
    k = torch.zeros(1, 8, 1, 64, 16, dtype=torch.int8, device=DEV)
    s = torch.ones(1, 8, 1, 4, device=DEV)
    for table, new, slots in (([[0, -1]], [[2]], None), ([[0, 8]], [[2]], None), ([[0, 1]], [[8]], None), ([[0, 1]], [[-1]], None), ([[0, 1]], [[2]], [1]),
                              ([[0, 1]], [[2]], [-1])):
        k2, s2, s3, s4 = k.clone() + 1, s.clone(), s.clone(), s.clone()
        err, kept = torch.zeros(1, dtype=torch.int32, device=DEV), torch.zeros(1, 1, 1, 3, dtype=torch.int32, device=DEV)
        b.block_evict(k2, k2.clone(), s2, s3, s4, dev(table), dev([100]), dev(new), 3, 1, kept, err, b.stream_ptr(), slots=None if slots is None else dev(slots))
        assert err.item() == b.ERR_PAGE_RANGE
        assert (k2 == 1).all() and (s4 == 1).all()


def test_captured():
    """A captured eviction, replayed over weights that have changed meanwhile."""
    b = B()
    table, new, lens = dev([[0, 1, 2]]), dev([[3]]), dev([160])
    k = torch.arange(5, device=DEV).to(torch.int8).view(1, 5, 1, 1, 1).expand(1, 5, 1, 64, 16).contiguous()
    s, w = torch.ones(1, 5, 1, 4, device=DEV), torch.zeros(1, 5, 1, 4, device=DEV)
    kept, err = torch.zeros(1, 1, 1, 4, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    v, s2 = k.clone(), s.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.block_evict(k, v, s, s2, w, table, lens, new, 4, 1, kept, err, b.stream_ptr())
    for best in ([0, 5, 8], [2, 3, 7]):
        w.zero_()
        for x in best:
            w[0, x // 4, 0, x % 4] = 1.0
        graph.replay()
        torch.cuda.synchronize()
        assert kept.flatten().tolist() == best + [9] and err.item() == 0
        assert k[0, 3, 0, ::16, 0].tolist() == [x // 4 for x in best + [9]]

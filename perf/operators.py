"""Three operators of a long conversation in little memory, and what each must compute.

attend   one-token attention over a paged cache held in 8 bits.  A block is 16 consecutive positions of one key/value head; its
         16 x D keys share one fp32 scale, its values another, a number stands for level * scale (levels int8 or e4m3).  The
         newest, unfinished block of a sequence is held as it came (bfloat16 or float32) and becomes 8 bits when its sixteenth
         position arrives.  For sequence s at position p, query head h of group G(h), over the visible positions j <= p (under a
         window also j > p - W):  a_hj = softmax_j(scale q_h . k_j),  o_h = sum_j a_hj v_j,  and, where the cache keeps them, the
         accumulated weights of its blocks  w_gb += sum over h of group g and j of block b of a_hj  (a block that starts at p starts at 0).
         The step's own key and value are stored in the same pass.
store    the keys and values of a step's prompts into such a cache: scale = max|x| / 127 (e4m3: 448), at least 2^-126, level =
         round(x / scale); the rest of a prompt, fewer than 16 positions, as it came.
evict    from each sequence's n finished blocks each layer and head keeps `keep`: the last `recent` and, among the others, those with
         the largest accumulated weight (ties: the lower index), in their order, copied to pages of their own.
rules    penalties for repeated tokens, biases and a mask of allowed tokens on a step's logits, and the best token that is left:
         an id seen in prompt or answer: x / r if x > 0 else x * r;  an id with c > 0 occurrences in the answer: x - f c - a;  then
         + bias;  -infinity where the mask has no bit.  The chosen id (ties: the lowest) joins the row's history.

Sizes are those of the repository's presets (32 query heads over 8 of 128; vocabularies of 32,000, 32,768 and 131,072) and odd ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
BLOCK, PAGE = 16, 64
BPP = PAGE // BLOCK


def listed():
    return [
        # one conversation, a short way in: launches and latency are all there is
        {"name": "attend_b1_short", "kind": "attend", "batch": 1, "context": 700, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "format": "int8", "dtype": "bfloat16", "weights": True},
        # the benchmark's batch and context
        {"name": "attend_b8", "kind": "attend", "batch": 8, "context": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "format": "int8", "dtype": "bfloat16", "weights": True},
        # a full server: conversations of very unequal lengths, e4m3 levels, no eviction wanted
        {"name": "attend_b64_e4m3", "kind": "attend", "batch": 64, "context": 4096, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "format": "float8_e4m3", "dtype": "bfloat16", "weights": False},
        # one conversation at the longest position of the 12B preset
        {"name": "attend_long", "kind": "attend", "batch": 1, "context": 131071, "heads": 32, "kv_heads": 8, "dim": 128, "window": 0,
         "format": "int8", "dtype": "bfloat16", "weights": True},
        # a true 32-bit run with heads of 64, six query heads to a key head, and a window that ends inside a block
        {"name": "attend_f32_window", "kind": "attend", "batch": 5, "context": 2500, "heads": 24, "kv_heads": 4, "dim": 64, "window": 1000,
         "format": "int8", "dtype": "float32", "weights": False},
        # the benchmark's prompt into the cache
        {"name": "store_prompt", "kind": "store", "batch": 1, "tokens": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "format": "int8",
         "dtype": "bfloat16"},
        # many prompts of unequal, odd lengths in one step
        {"name": "store_many_e4m3", "kind": "store", "batch": 19, "tokens": 16001, "heads": 24, "kv_heads": 4, "dim": 64,
         "format": "float8_e4m3", "dtype": "bfloat16"},
        # one conversation goes back to 1,024 positions, all layers of the 7B presets at once
        {"name": "evict_one", "kind": "evict", "batch": 1, "layers": 32, "context": 1088, "keep": 64, "recent": 16, "kv_heads": 8, "dim": 128,
         "format": "int8"},
        # eight conversations lose half of what they hold
        {"name": "evict_half", "kind": "evict", "batch": 8, "layers": 8, "context": 4096, "keep": 128, "recent": 32, "kv_heads": 8,
         "dim": 128, "format": "int8"},
        # the next token of one conversation: penalties and biases
        {"name": "rules_b1", "kind": "rules", "rows": 1, "vocab": 32000, "history": 700, "penalties": True, "bias": True, "mask": False},
        # a few rows of an odd vocabulary under a grammar's mask
        {"name": "rules_odd", "kind": "rules", "rows": 7, "vocab": 40007, "history": 2000, "penalties": True, "bias": False, "mask": True},
        # a full server at the 12B preset's vocabulary
        {"name": "rules_b64", "kind": "rules", "rows": 64, "vocab": 131072, "history": 4096, "penalties": True, "bias": True, "mask": True},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "store", "evict", "rules", "rules"])
    kv_heads, group, dim = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 6, 8, 12]), rng.choice([64, 128])
    fmt = rng.choice(["int8", "float8_e4m3"])
    if kind == "attend":
        batch = _log(rng, 1, 64)
        window = rng.choice([0, 0, 0, _log(rng, 17, 5000)])
        return {"kind": kind, "batch": batch, "context": _log(rng, 1, min(131071, 262144 // batch)), "heads": kv_heads * group,
                "kv_heads": kv_heads, "dim": dim, "window": window, "format": fmt, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]),
                "weights": window == 0 and rng.random() < 0.6}
    if kind == "store":
        batch = _log(rng, 1, 32)
        return {"kind": kind, "batch": batch, "tokens": max(batch, _log(rng, 1, 16001)), "heads": kv_heads * group, "kv_heads": kv_heads,
                "dim": dim, "format": fmt, "dtype": rng.choice(["bfloat16", "float32"])}
    if kind == "evict":
        keep = _log(rng, 2, 200)
        return {"kind": kind, "batch": _log(rng, 1, 8), "layers": rng.choice([1, 3, 8]), "context": (keep + _log(rng, 1, 100)) * BLOCK + rng.randrange(16),
                "keep": keep, "recent": rng.randint(0, keep), "kv_heads": kv_heads, "dim": dim, "format": fmt}
    vocab = _log(rng, 100, 131072)
    return {"kind": kind, "rows": _log(rng, 1, 64), "vocab": vocab, "history": _log(rng, 1, 8192), "penalties": rng.random() < 0.8,
            "bias": rng.random() < 0.5, "mask": rng.random() < 0.5}


# ---------------------------------------------------------------------------------------
# inputs, from a seed alone


class _Draws:
    """Tensors in the order they are asked for; the same order gives the same tensors again."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed))

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=self.g, device=DEV) * std).to(dtype)

    def uniform(self, lo, hi, *shape):
        return torch.rand(shape, generator=self.g, device=DEV) * (hi - lo) + lo

    def whole(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device=DEV, dtype=torch.int32)


def _level_type(case):
    return torch.int8 if case["format"] == "int8" else torch.float8_e4m3fn


def _lens(case, seed):
    """Positions that each sequence holds before the step (store: that its prompt brings)."""
    rs = np.random.RandomState(seed % (1 << 31))
    b = case["batch"]
    if case["kind"] == "store":
        w = rs.uniform(0.2, 1.8, b)
        lens = 1 + (w / w.sum() * (case["tokens"] - b)).astype(int)
        lens[int(np.argmax(lens))] += case["tokens"] - int(lens.sum())
        return [int(x) for x in lens]
    if b == 1:
        return [case["context"]]
    low = case["keep"] * BLOCK if case["kind"] == "evict" else case["context"] // 16
    lens = rs.randint(min(low, case["context"]), case["context"] + 1, b)
    lens[0] = case["context"]
    if case["kind"] == "attend" and case["context"] >= BLOCK:
        lens[b // 2] = max(BLOCK - 1, int(lens[b // 2]) // BLOCK * BLOCK - 1)     # one sequence finishes a block in this step
    return [int(x) for x in lens]


def _tables(lens, seed, n_pages):
    """Page tables [sequences, width] (-1: no page) over a pool's pages in no order, and the pages that are left."""
    need = [-(-n // PAGE) for n in lens]
    order = np.random.RandomState((seed + 1) % (1 << 31)).permutation(n_pages)
    table, at = np.full((len(lens), max(need)), -1, dtype=np.int32), 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, [int(x) for x in order[at:]]


def _levels(case, d, *shape):
    if case["format"] == "int8":
        return torch.randn(shape, generator=d.g, device=DEV, dtype=torch.bfloat16).mul_(42).round_().clamp_(-127, 127).to(torch.int8)
    return torch.randn(shape, generator=d.g, device=DEV, dtype=torch.bfloat16).mul_(130).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(case, d, *shape):
    top = 127.0 if case["format"] == "int8" else 448.0
    return d.uniform(2.5, 4.5, *shape) / top


def _dev(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device=DEV)


def prepare(case, seed):
    d = _Draws(seed)
    return {"attend": _prepare_cache, "store": _prepare_cache, "evict": _prepare_evict, "rules": _prepare_rules}[case["kind"]](case, seed, d)


def _prepare_cache(case, seed, d):
    lens, n, G, D = _lens(case, seed), case["batch"], case["kv_heads"], case["dim"]
    attend = case["kind"] == "attend"
    dt = torch.float32 if case["dtype"] == "float32" else torch.bfloat16
    n_pages = n * (case["context"] // PAGE + 1) if attend else case["tokens"] // PAGE + 2 * n
    table, _ = _tables([x + 1 for x in lens] if attend else lens, seed, n_pages)
    T = n if attend else sum(lens)
    s = {"case": case, "lens": lens}
    s["qkv"] = d.normal(T, (case["heads"] + 2 * G) * D, dtype=dt)
    shape = (n_pages, G, PAGE, D)
    if attend:
        s["k"], s["v"] = _levels(case, d, *shape), _levels(case, d, *shape)
        s["k_scale"], s["v_scale"] = _scales(case, d, n_pages, G, BPP), _scales(case, d, n_pages, G, BPP)
        s["tail_k"], s["tail_v"] = d.normal(n, G, BLOCK, D, dtype=dt), d.normal(n, G, BLOCK, D, dtype=dt)
    else:
        s["k"], s["v"] = (torch.zeros(shape, device=DEV).to(_level_type(case)) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros((n_pages, G, BPP), device=DEV) for _ in range(2))
        s["tail_k"], s["tail_v"] = (torch.zeros((n, G, BLOCK, D), dtype=dt, device=DEV) for _ in range(2))
    s["table"] = _dev(table)
    pos0 = lens if attend else [0] * n
    q_lens = [1] * n if attend else lens
    cu = np.concatenate([[0], np.cumsum(q_lens)])
    s["cu"], s["slots"], s["seq"], s["pos0"] = _dev(cu), _dev(range(n)), _dev(np.repeat(np.arange(n), q_lens)), _dev(pos0)
    s["weight"], s["weight_out"] = None, None
    if attend:
        s["out"] = torch.empty((T, case["heads"] * D), dtype=dt, device=DEV)
        if case["weights"]:
            s["weight"], s["weight_out"] = d.uniform(0.0, 2.0, n_pages, G, BPP), torch.zeros((n_pages, G, BPP), device=DEV)
    # host facts that the plain form needs: which page and block a position is in
    s["pages"] = torch.tensor(table, dtype=torch.int64, device=DEV).clamp_(min=0)
    s["n"] = torch.tensor(lens, dtype=torch.int64, device=DEV)
    s["longest"] = max(lens)
    if own:
        from inference_engine_rust_b200.csrc import bindings as B
        s["err"] = torch.zeros(1, dtype=torch.int32, device=DEV)
        s["batch"] = B.BatchView(cu_q=s["cu"].data_ptr(), slot_ids=s["slots"].data_ptr(), tok_seq=s["seq"].data_ptr(),
                                 pos0=s["pos0"].data_ptr(), n_seqs=n, n_tokens=T)
        s["view"] = B.block_view(s["k"], s["v"], s["k_scale"], s["v_scale"], s["tail_k"], s["tail_v"], s["table"],
                                 window=case.get("window", 0), weight=s["weight"])
        if attend:
            s["scratch"] = torch.empty(B.block_attention_scratch_floats(n, case["heads"], s["view"]), device=DEV)
    return s


def _prepare_evict(case, seed, d):
    lens, n, G, D, L = _lens(case, seed), case["batch"], case["kv_heads"], case["dim"], case["layers"]
    per = -(-(case["keep"] * BLOCK + BLOCK - 1) // PAGE)
    n_pages = n * (-(-case["context"] // PAGE) + per)
    table, free = _tables(lens, seed, n_pages)
    s = {"case": case, "lens": lens}
    s["k"], s["v"] = _levels(case, d, L, n_pages, G, PAGE, D), _levels(case, d, L, n_pages, G, PAGE, D)
    s["k_scale"], s["v_scale"] = _scales(case, d, L, n_pages, G, BPP), _scales(case, d, L, n_pages, G, BPP)
    # a few blocks carry most of the weight, many carry almost none, some the very same
    s["weight"] = torch.exp2(torch.round(d.normal(L, n_pages, G, BPP, std=3.0) * 64) / 64)
    s["table"], s["new"] = _dev(table), _dev(np.reshape(free[:n * per], (n, per)))
    s["lengths"] = _dev(lens)
    s["kept"] = torch.zeros((L, n, G, case["keep"]), dtype=torch.int32, device=DEV)
    if own:
        s["err"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    return s


def _prepare_rules(case, seed, d):
    R, V, H = case["rows"], case["vocab"], case["history"]
    s = {"case": case, "logits": d.normal(R, V, std=4.0)}
    rs = np.random.RandomState(seed % (1 << 31))
    lens = rs.randint(max(1, H // 4), H + 1, R)
    prompts = (lens * rs.uniform(0.1, 0.9, R)).astype(int)
    # tokens of a text: few ids make up most of it
    s["history"] = (torch.rand((R, H + 1), generator=d.g, device=DEV) ** 4 * V).to(torch.int32).clamp_(max=V - 1)
    s["lens"], s["prompt_lens"], s["rows"] = _dev(lens), _dev(prompts), _dev(rs.permutation(R))
    s["penalties"] = torch.stack([d.uniform(1.0, 1.4, R), d.uniform(0.0, 0.8, R), d.uniform(0.0, 0.5, R)], 1).contiguous() if case["penalties"] else None
    s["bias"] = d.normal(V, std=1.0) * (d.uniform(0.0, 1.0, V) < 0.02) if case["bias"] else None
    s["mask"] = d.whole(-(1 << 31), (1 << 31) - 1, R, -(-V // 32)) if case["mask"] else None
    s["out"], s["chosen"], s["lens_out"] = torch.empty_like(s["logits"]), torch.zeros(R, dtype=torch.int32, device=DEV), torch.zeros_like(s["lens"])
    if own:
        s["err"] = torch.zeros(1, dtype=torch.int32, device=DEV)
    return s


# ---------------------------------------------------------------------------------------
# one pass


def run(s):
    return {"attend": _attend, "store": _store, "evict": _evict, "rules": _rules}[s["case"]["kind"]](s)


def _values(levels, scale):
    """What 8-bit levels [..., PAGE, D] with scales [..., BPP] stand for, in 32 bits."""
    return levels.float() * scale.repeat_interleave(BLOCK, -1).unsqueeze(-1)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


def _quantize(x, kind):
    """x [..., 16, D] in 32 bits: levels and scales [...]."""
    top = torch.full((), 127.0 if kind == torch.int8 else 448.0, device=x.device)
    scale = (x.abs().amax((-1, -2)) / top).clamp(min=2.0 ** -126)
    level = (x / scale[..., None, None]).clamp(-top, top)
    return (level.round() if kind == torch.int8 else level).to(kind), scale


def _state(s):
    out = {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"], "tail_k": s["tail_k"], "tail_v": s["tail_v"]}
    if s["weight_out"] is not None:
        out["weight"] = s["weight_out"]
    return out


def _attend(s):
    case = s["case"]
    n, H, G, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if own:
        from inference_engine_rust_b200.csrc import bindings as B
        B.block_attention(s["qkv"], s["out"], s["batch"], s["view"], H, D ** -0.5, s["scratch"], s["err"], B.stream_ptr(),
                          weight_out=s["weight_out"])
        return {"out": s["out"], **_state(s)}
    rows = s["qkv"].view(n, H + 2 * G, D)
    seq, pos = torch.arange(n, device=DEV), s["n"]
    at = pos % BLOCK
    s["tail_k"][seq, :, at], s["tail_v"][seq, :, at] = rows[:, H:H + G], rows[:, H + G:]
    blk = pos // BLOCK
    first = blk.view(n, 1) * BLOCK + torch.arange(BLOCK, device=DEV)                     # positions of the unfinished block
    pages = s["pages"][:, :s["longest"] // PAGE + 1]
    W = pages.shape[1] * PAGE

    def whole(name):
        x = _values(_bytes(s[name])[pages].view(s[name].dtype), s[name + "_scale"][pages])  # [n, pages, G, PAGE, D]
        x = x.transpose(1, 2).reshape(n, G, W, D)
        return x.index_put_((seq.view(n, 1, 1), torch.arange(G, device=DEV).view(1, G, 1), first.view(n, 1, BLOCK)), s["tail_" + name].float())
    j = torch.arange(W, device=DEV).view(1, W)
    hidden = j > pos.view(n, 1)
    if case["window"]:
        hidden = hidden | (j <= pos.view(n, 1) - case["window"])
    score = rows[:, :H].float().reshape(n, G, H // G, D) @ whole("k").transpose(2, 3) * D ** -0.5
    score.masked_fill_(hidden.view(n, 1, 1, W), -math.inf)
    a = torch.softmax(score, -1)
    out = (a @ whole("v").masked_fill_(hidden.view(n, 1, W, 1), 0.0)).reshape(n, H * D).to(s["out"].dtype)
    if s["weight_out"] is not None:
        w = a.sum(2).view(n, G, W // PAGE, BPP, BLOCK).sum(-1).transpose(1, 2)           # [n, pages, G, BPP]
        b = torch.arange(W // BLOCK, device=DEV).view(1, W // PAGE, 1, BPP)
        new = (b == blk.view(n, 1, 1, 1)) & (at == 0).view(n, 1, 1, 1)
        w = w + s["weight"][pages].masked_fill(new, 0.0)
        seen = (b <= blk.view(n, 1, 1, 1)).expand_as(w)
        e = torch.arange(BPP, device=DEV).view(1, 1, 1, BPP).expand_as(w)
        g = torch.arange(G, device=DEV).view(1, 1, G, 1).expand_as(w)
        s["weight_out"][pages[:, :, None, None].expand_as(w)[seen], g[seen], e[seen]] = w[seen]
    done = torch.nonzero(at == BLOCK - 1).flatten()                                       # blocks that the step finished
    page, part = s["pages"][done, pos[done] // PAGE], blk[done] % BPP
    cols = part.view(-1, 1) * BLOCK + torch.arange(BLOCK, device=DEV)
    for name in ("k", "v"):
        level, scale = _quantize(s["tail_" + name][done].float(), s[name].dtype)
        _bytes(s[name])[page[:, None, None], torch.arange(G, device=DEV)[None, :, None], cols[:, None, :]] = _bytes(level)
        s[name + "_scale"][page, :, part] = scale
    return {"out": out, **_state(s)}


def _store(s):
    case = s["case"]
    n, H, G, D = case["batch"], case["heads"], case["kv_heads"], case["dim"]
    if own:
        from inference_engine_rust_b200.csrc import bindings as B
        B.block_store(s["qkv"], s["batch"], s["view"], H, s["err"], B.stream_ptr())
        return _state(s)
    rows = s["qkv"].view(-1, H + 2 * G, D)
    seq = s["seq"].long()
    pos = torch.arange(rows.shape[0], device=DEV) - s["cu"][seq]
    ends = s["n"][seq] // BLOCK * BLOCK
    rest = pos >= ends                                                                     # rows of unfinished blocks
    done = torch.nonzero(~rest).flatten().view(-1, BLOCK)                                 # rows of finished blocks
    block, page = pos[done[:, 0]] // BLOCK, s["pages"][seq[done[:, 0]], pos[done[:, 0]] // PAGE]
    cols = (block % BPP).view(-1, 1) * BLOCK + torch.arange(BLOCK, device=DEV)
    for name, lo in (("k", H), ("v", H + G)):
        s["tail_" + name][seq[rest], :, pos[rest] % BLOCK] = rows[rest, lo:lo + G]
        level, scale = _quantize(rows[:, lo:lo + G][done].float().transpose(1, 2), s[name].dtype)   # [blocks, G, 16, D]
        _bytes(s[name])[page[:, None, None], torch.arange(G, device=DEV)[None, :, None], cols[:, None, :]] = _bytes(level)
        s[name + "_scale"][page, :, block % BPP] = scale
    return _state(s)


def _evict(s):
    case = s["case"]
    n, G, L, keep, recent = case["batch"], case["kv_heads"], case["layers"], case["keep"], case["recent"]
    got = {x: s[x] for x in ("k", "v", "k_scale", "v_scale", "weight", "kept")}
    if own:
        from inference_engine_rust_b200.csrc import bindings as B
        B.block_evict(s["k"], s["v"], s["k_scale"], s["v_scale"], s["weight"], s["table"], s["lengths"], s["new"], keep, recent, s["kept"],
                      s["err"], B.stream_ptr())
        return got
    pages, new, blocks = s["table"].long().clamp(min=0), s["new"].long(), s["lengths"].long() // BLOCK
    B_, l = pages.shape[1] * BPP, torch.arange(L, device=DEV).view(L, 1, 1, 1)
    g = torch.arange(G, device=DEV).view(1, 1, G, 1)
    w = s["weight"][:, pages].transpose(2, 3).reshape(L, n, G, B_)                        # [L, n, pages, G, BPP]
    b = torch.arange(B_, device=DEV)
    nb = blocks.view(1, n, 1, 1)
    rank = w.masked_fill(b >= nb - recent, math.inf).masked_fill(b >= nb, -1.0)
    best = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.sort(best, dim=-1).values                                                # [L, n, G, keep]
    s["kept"].copy_(kept)
    i = torch.arange(n, device=DEV).view(1, n, 1, 1)
    to = torch.arange(keep, device=DEV).view(1, 1, 1, keep)
    src_page, dst_page = pages[i, kept // BPP], new[i, to // BPP].expand_as(kept)
    for name in ("k_scale", "v_scale", "weight"):
        s[name][l, dst_page, g, (to % BPP).expand_as(kept)] = s[name][l, src_page, g, kept % BPP]
    for name in ("k", "v"):
        t = _bytes(s[name]).view(L, -1, G, BPP, BLOCK * case["dim"])
        t[l, dst_page, g, (to % BPP).expand_as(kept)] = t[l, src_page, g, kept % BPP]
    open_ = torch.nonzero(s["lengths"] % BLOCK).flatten()                                 # unfinished blocks take their weight along
    s["weight"][:, new[open_, keep // BPP], :, torch.full_like(open_, keep % BPP)] = \
        s["weight"][:, pages[open_, blocks[open_] // BPP], :, blocks[open_] % BPP]
    return got


def _rules(s):
    case = s["case"]
    R, V = case["rows"], case["vocab"]
    if own:
        from inference_engine_rust_b200.csrc import bindings as B
        B.logit_rules(s["logits"], s["out"], s["history"], s["lens"], s["prompt_lens"], s["rows"], s["err"], B.stream_ptr(),
                      penalties=s["penalties"], bias=s["bias"], mask=s["mask"], chosen=s["chosen"], lens_out=s["lens_out"])
        return {"logits": s["out"], "chosen": s["chosen"], "lens": s["lens_out"], "history": s["history"]}
    at, x = s["rows"].long(), s["logits"]
    if s["penalties"] is not None:
        h, lens, prompt = s["history"][at].long(), s["lens"][at].view(R, 1), s["prompt_lens"][at].view(R, 1)
        place = torch.arange(h.shape[1], device=DEV).view(1, -1)
        seen = torch.zeros((R, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, (place < lens).int())
        said = torch.zeros((R, V), dtype=torch.int32, device=DEV).scatter_add_(1, h, ((place >= prompt) & (place < lens)).int())
        rep, pres, freq = (s["penalties"][at][:, i:i + 1] for i in range(3))
        x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = torch.where(said > 0, x - freq * said - pres, x)
    if s["bias"] is not None:
        x = x + s["bias"]
    if s["mask"] is not None:
        ids = torch.arange(V, device=DEV)
        x = x.masked_fill((s["mask"][:, ids // 32] >> (ids % 32)) & 1 == 0, -math.inf)
    best = x.amax(1, keepdim=True)
    chosen = torch.where(x == best, torch.arange(V, device=DEV), V).amin(1).to(torch.int32)
    s["history"][at, s["lens"][at].long()] = chosen
    lens = s["lens"].clone()
    lens[at] += 1
    return {"logits": x, "chosen": chosen, "lens": lens, "history": s["history"]}


# ---------------------------------------------------------------------------------------
# what a pass cannot do without


def work(case):
    if case["kind"] == "rules":
        R, V = case["rows"], case["vocab"]
        b = 8.0 * R * V + (4.0 * V if case["bias"] else 0) + (R * V / 8 if case["mask"] else 0)
        b += R * (0.625 * 4 * case["history"] if case["penalties"] else 0) + 32 * R
        return {"bytes": b, "flops": 4.0 * R * V}
    G, D = case["kv_heads"], case["dim"]
    if case["kind"] == "evict":
        L, n = case["layers"], case["batch"]
        blocks = L * n * G * case["keep"]
        return {"bytes": blocks * (2.0 * 2 * (BLOCK * D + 6) + 4) + 4.0 * L * G * sum(_lens(case, 0)) / BLOCK, "flops": 0.0}
    size = 4 if case["dtype"] == "float32" else 2
    H = case["heads"]
    if case["kind"] == "store":
        return {"bytes": case["tokens"] * G * 2.0 * (D * size + D + 4 / BLOCK), "flops": 4.0 * case["tokens"] * G * D}
    reach = lambda x: min(x + 1, case["window"]) if case["window"] else x + 1   # noqa: E731
    seen = sum(reach(x) for x in _lens(case, 0))
    b = seen * G * (2.0 * D + 8 / BLOCK + (8 / BLOCK if case["weights"] else 0))
    b += case["batch"] * ((2 * H + 2 * G) * D * size + 2 * G * D * size * 8.5)            # queries, outputs, the unfinished block
    return {"bytes": b, "flops": 4.0 * seen * H * D}


# ---------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits, a sequence (or row) at a time


def exact(case, seed):
    d = _Draws(seed)
    if case["kind"] == "rules":
        return _exact_rules(_prepare_rules(case, seed, d))
    if case["kind"] == "evict":
        return None                       # it moves what is there: nothing is computed but whole numbers
    if case["kind"] == "store":
        return _exact_store(_prepare_cache(case, seed, d))
    return _exact_attend(_prepare_cache(case, seed, d))


def _exact_row(s, name, i, j):
    """Rows `j` (a range of finished positions) of sequence i, [kv heads, rows, dim], in 64 bits."""
    table = s["table"][i].tolist()
    out = []
    for p in range(j.start // PAGE, (j.stop + PAGE - 1) // PAGE):
        x = s[name][table[p]].double()
        out.append((x.view(x.shape[0], BPP, BLOCK, -1) * s[name + "_scale"][table[p]].double()[:, :, None, None]).flatten(1, 2))
    lo = j.start // PAGE * PAGE
    return torch.cat(out, 1)[:, j.start - lo:j.stop - lo] if out else torch.zeros((s["tail_k"].shape[1], 0, s["tail_k"].shape[3]), device=DEV, dtype=torch.float64)


def _exact_attend(s):
    case = s["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    outs, weight = [], s["weight_out"].double() if s["weight_out"] is not None else None
    tails = {"k": s["tail_k"].double(), "v": s["tail_v"].double()}
    scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()}
    for i, p in enumerate(s["lens"]):
        row = s["qkv"][i].double().view(H + 2 * G, D)
        base = p - p % BLOCK
        lo = max(0, p + 1 - case["window"]) if case["window"] else 0
        kv = {}
        for name, own_rows in (("k", row[H:H + G]), ("v", row[H + G:])):
            tails[name][i, :, p - base] = own_rows
            kv[name] = torch.cat([_exact_row(s, name, i, range(min(lo, base), base)), tails[name][i, :, max(0, lo - base):p - base + 1]], 1)
            if p - base == BLOCK - 1:
                top = 127.0 if s[name].dtype == torch.int8 else 448.0
                scales[name][int(s["table"][i, p // PAGE]), :, base // BLOCK % BPP] = tails[name][i].abs().amax((1, 2)) / top
        e = torch.einsum("ghd,gjd->ghj", row[:H].view(G, H // G, D), kv["k"]) / math.sqrt(D)
        e = torch.exp(e - e.amax(-1, keepdim=True))
        a = e / e.sum(-1, keepdim=True)
        outs.append(torch.einsum("ghj,gjd->ghd", a, kv["v"]).reshape(-1))
        if weight is not None:
            per = torch.zeros((G, (p // BLOCK + 1) * BLOCK), dtype=torch.float64, device=DEV)
            per[:, :p + 1] = a.sum(1)
            per = per.view(G, -1, BLOCK).sum(-1)
            for b0 in range(0, per.shape[1], BPP):
                m, page = min(BPP, per.shape[1] - b0), int(s["table"][i, b0 // BPP])
                old = s["weight"][page, :, :m].double()
                if p % BLOCK == 0 and b0 + m == per.shape[1]:
                    old = torch.cat([old[:, :m - 1], torch.zeros_like(old[:, :1])], 1)
                weight[page, :, :m] = old + per[:, b0:b0 + m]
    got = {"out": torch.stack(outs), "k": None, "v": None, "k_scale": scales["k"], "v_scale": scales["v"], "tail_k": tails["k"], "tail_v": tails["v"]}
    if weight is not None:
        got["weight"] = weight
    return got


def _exact_store(s):
    case = s["case"]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    got = {x: s[x].double() for x in ("k_scale", "v_scale", "tail_k", "tail_v")}
    at = 0
    for i, n in enumerate(s["lens"]):
        rows = s["qkv"][at:at + n].double().view(n, H + 2 * G, D)
        at += n
        full = n // BLOCK
        for name, lo in (("k", H), ("v", H + G)):
            x = rows[:, lo:lo + G].transpose(0, 1)
            got["tail_" + name][i, :, :n - full * BLOCK] = x[:, full * BLOCK:]
            top = x[:, :full * BLOCK].reshape(G, full, BLOCK * D).abs().amax(-1) / (127.0 if s["k"].dtype == torch.int8 else 448.0) if full else None
            for b in range(full):
                got[name + "_scale"][int(s["table"][i, b // BPP]), :, b % BPP] = top[:, b]
    return {"k": None, "v": None, **got}


def _exact_rules(s):
    case, xs = s["case"], []
    V = case["vocab"]
    for r, h in enumerate(s["rows"].tolist()):
        x = s["logits"][r].double()
        if s["penalties"] is not None:
            n, p = int(s["lens"][h]), int(s["prompt_lens"][h])
            rep, pres, freq = s["penalties"][h].double()
            seen = torch.bincount(s["history"][h, :n].long(), minlength=V)
            said = torch.bincount(s["history"][h, p:n].long(), minlength=V)
            x = torch.where((seen > 0) & (x > 0), x / rep, torch.where(seen > 0, x * rep, x))
            x = x - freq * said - pres * (said > 0)
        if s["bias"] is not None:
            x = x + s["bias"].double()
        if s["mask"] is not None:
            bits = (s["mask"][r][:, None] >> torch.arange(32, device=DEV)) & 1
            x[bits.reshape(-1)[:V] == 0] = -math.inf
        xs.append(x)
    return {"logits": torch.stack(xs), "chosen": None, "lens": None, "history": None}

"""What the 8-bit cache's and the logit rules' entry points refuse, before anything is launched (no GPU needed)."""
import pytest
import torch

from inference_engine_rust_b200.csrc import bindings as B


def rules(**kw):
    a = dict(logits=torch.zeros(2, 40), out=torch.zeros(2, 40), history=torch.zeros(3, 8, dtype=torch.int32), lens=torch.zeros(3, dtype=torch.int32),
             prompt_lens=torch.zeros(3, dtype=torch.int32), rows=torch.zeros(2, dtype=torch.int32))
    opt = dict(penalties=torch.ones(3, 3), bias=torch.zeros(40), mask=torch.zeros(2, 2, dtype=torch.int32), chosen=torch.zeros(2, dtype=torch.int32))
    for k, v in kw.items():
        (a if k in a else opt)[k] = v
    B.logit_rules(a["logits"], a["out"], a["history"], a["lens"], a["prompt_lens"], a["rows"], torch.zeros(1, dtype=torch.int32), 0, **opt)


@pytest.mark.parametrize("kw, says", [
    (dict(logits=torch.zeros(2, 40, dtype=torch.bfloat16)), "logits must be float32"),
    (dict(logits=torch.zeros(40)), "logits must be float32"),
    (dict(logits=torch.zeros(40, 2).t()), "contiguous rows"),
    (dict(out=torch.zeros(2, 41)), "out must be"),
    (dict(history=torch.zeros(3, 8)), "history must be"),
    (dict(history=torch.zeros(8, 3, dtype=torch.int32).t()), "history must be"),
    (dict(lens=torch.zeros(2, dtype=torch.int32)), "lens must be"),
    (dict(prompt_lens=None), "prompt_lens must be"),
    (dict(rows=torch.zeros(3, dtype=torch.int32)), "rows must be"),
    (dict(penalties=torch.ones(2, 3)), "penalties must be"),
    (dict(bias=torch.zeros(39)), "bias must be"),
    (dict(bias=torch.zeros(3, 40)), "bias must be"),
    (dict(mask=torch.zeros(2, 1, dtype=torch.int32)), "mask must be"),
    (dict(mask=torch.zeros(3, 2, dtype=torch.int32)), "mask must be"),
    (dict(chosen=torch.zeros(2)), "chosen must be"),
    (dict(lens_out=torch.zeros(2, dtype=torch.int32)), "lens_out must be"),
    (dict(lens_out=torch.zeros(3, dtype=torch.int32), chosen=None), "lens_out needs chosen"),
    (dict(history=None), "need a history"),
    (dict(), "on one CUDA device"),
])
def test_rules_refuse(kw, says):
    with pytest.raises(B.KernelError, match=says):
        rules(**kw)


def test_history_append_refuses():
    h, n = torch.zeros(3, 8, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    err = torch.zeros(1, dtype=torch.int32)
    for args, says in [((h.float(), n, None, n), "history must be"), ((h, n[:2], None, n), "lens must be"), ((h, n, None, n.float()), "tokens must be"),
                       ((h, n, n[:2], n), "rows must be"), ((h, n, n, n), "on one CUDA device")]:
        with pytest.raises(B.KernelError, match=says):
            B.history_append(*args, err, 0)


def pools(G=2, D=16, pt=64, pages=3, slots=2, width=2, fmt=torch.int8, tail=torch.bfloat16, lead=()):
    k = torch.zeros(*lead, pages, G, pt, D).to(fmt)
    s = torch.zeros(*lead, pages, G, pt // 16)
    return dict(k=k, v=k.clone(), k_scale=s, v_scale=s.clone(), tail_k=torch.zeros(slots, G, 16, D, dtype=tail),
                tail_v=torch.zeros(slots, G, 16, D, dtype=tail), page_table=torch.zeros(slots, width, dtype=torch.int32))


@pytest.mark.parametrize("kw, says", [
    (dict(k=torch.zeros(3, 2, 64, 16)), "must be int8 or float8"),
    (dict(v=torch.zeros(3, 2, 64, 16).to(torch.float8_e4m3fn)), "must be int8 or float8"),
    (dict(k_scale=torch.zeros(3, 2, 3)), "k_scale must be"),
    (dict(v_scale=torch.zeros(3, 2, 4, dtype=torch.float64)), "v_scale must be"),
    (dict(tail_k=torch.zeros(2, 2, 16, 16)), "of one type"),
    (dict(tail_v=torch.zeros(1, 2, 16, 16, dtype=torch.bfloat16)), "tail_k and tail_v must be"),
    (dict(page_table=torch.zeros(2, 2)), "page table must be"),
    (dict(weight=torch.zeros(3, 2, 5)), "weight must be"),
    (dict(weight=torch.zeros(3, 2, 4), window=32), "without a window"),
    (dict(shift=torch.zeros(1, dtype=torch.int32)), "shift must be"),
    (dict(ring_pages=1), "needs a window"),
    (dict(ring_pages=3, window=64), "part of a table row"),
    (dict(ring_pages=1, window=65), "must hold the window"),
])
def test_block_view_refuses(kw, says):
    p = pools()
    p.update(kw)
    with pytest.raises(B.KernelError, match=says):
        B.block_view(**p)


def test_block_view_refuses_pages_that_cut_a_block_and_strides():
    with pytest.raises(B.KernelError, match="multiple of 16"):
        B.block_view(**pools(pt=24))
    p = pools()
    p["k"] = p["k"].transpose(2, 3).contiguous().transpose(2, 3)
    with pytest.raises(B.KernelError, match="k must be contiguous"):
        B.block_view(**p)


def batch(n_seqs, n_tokens):
    return B.BatchView(cu_q=None, slot_ids=None, tok_seq=None, pos0=None, n_seqs=n_seqs, n_tokens=n_tokens)


def test_steps_refuse():
    p = pools()
    weight = torch.zeros(3, 2, 4)
    view = B.block_view(**p, weight=weight)
    err = torch.zeros(1, dtype=torch.int32)
    good = torch.zeros(2, (4 + 4) * 16, dtype=torch.bfloat16)
    out, scratch = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(B.block_attention_scratch_floats(2, 4, view))

    def step(**kw):
        a = dict(qkv=good, out=out, batch=batch(2, 2), heads=4, scratch=scratch)
        a.update(kw)
        B.block_attention(a["qkv"], a["out"], a["batch"], view, a["heads"], 1.0, a["scratch"], err, 0, weight_out=a.get("weight_out"))
    for kw, says in [(dict(qkv=good.float()), "of the tails' type"), (dict(qkv=good[:, :-1]), "projection must be"), (dict(batch=batch(2, 3)), "one row per"),
                     (dict(batch=batch(3, 3)), "one row per"), (dict(heads=3, qkv=torch.zeros(2, 7 * 16, dtype=torch.bfloat16)), "multiple of kv_heads"),
                     (dict(out=out[:1]), "out must be"), (dict(out=out.float()), "out must be"), (dict(scratch=scratch[1:]), "scratch is too small"), ({}, "on one CUDA device")]:
        with pytest.raises(B.KernelError, match=says):
            step(**kw)
    with pytest.raises(B.KernelError, match="fewer rows"):
        B.block_store(good, batch(1, 3), view, 4, err, 0)
    with pytest.raises(B.KernelError, match="on one CUDA device"):
        B.block_store(good, batch(1, 2), view, 4, err, 0)


@pytest.mark.parametrize("kw, says", [
    (dict(keep=0), "must be positive"), (dict(recent=5), "between 0 and keep"), (dict(recent=-1), "between 0 and keep"),
    (dict(new_pages=torch.zeros(2, 0, dtype=torch.int32)), "room for the kept"), (dict(new_pages=torch.zeros(1, 1, dtype=torch.int32)), "new_pages must be"),
    (dict(kept=torch.zeros(1, 2, 2, 3, dtype=torch.int32)), "kept must be"), (dict(weight=None), "weight must be"),
    (dict(lengths=torch.zeros(3, dtype=torch.int32)), "lengths must be"), (dict(slots=torch.zeros(3, dtype=torch.int32)), "slots must be"),
    (dict(shift=torch.zeros(3, dtype=torch.int32)), "shift must be"), ({}, "on one CUDA device")])
def test_evict_refuses(kw, says):
    p = pools(lead=(1,))
    a = dict(k=p["k"], v=p["v"], k_scale=p["k_scale"], v_scale=p["v_scale"], weight=p["k_scale"].clone(), page_table=p["page_table"],
             lengths=torch.zeros(2, dtype=torch.int32), new_pages=torch.zeros(2, 1, dtype=torch.int32), keep=4, recent=2,
             kept=torch.zeros(1, 2, 2, 4, dtype=torch.int32), slots=None, shift=None)
    a.update(kw)
    slots, shift = a.pop("slots"), a.pop("shift")
    with pytest.raises(B.KernelError, match=says):
        B.block_evict(*a.values(), torch.zeros(1, dtype=torch.int32), 0, slots=slots, shift=shift)

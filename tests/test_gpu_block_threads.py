"""Calls of one operator at different sizes from two threads, each on a stream of its own: none makes another's launch fail."""
import sys
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def B():
    from inference_engine_rust_b200.csrc import bindings
    return bindings


class Recorder:
    """The library, whose next call is made and remembered."""

    def __init__(self, lib):
        self.lib, self.call = lib, None

    def __getattr__(self, name):
        entry = getattr(self.lib, name)

        def call(*args):
            self.call = (entry, args)
            return entry(*args)
        return call


def both(monkeypatch, make, sizes, calls=60_000):
    """`make(size)` gives a function that makes one call on a given stream, one that forgets its result and one that looks at it.  The calls that reach the
    library are repeated by two threads at once, with nothing in between but the loop (a launch that fails says so by its status)."""
    wrong, streams, work = [], [torch.cuda.Stream() for _ in sizes], []
    for size, stream in zip(sizes, streams):
        go, forget, check = make(size)
        lib = Recorder(B().core())
        with monkeypatch.context() as m:
            m.setattr(B(), "core", lambda: lib)
            go(stream.cuda_stream)
        torch.cuda.synchronize()
        check()
        forget()
        work.append((lib.call, check, go))            # (what the call points to lives in `go`)
    torch.cuda.synchronize()

    def loop(entry, args):
        try:
            for _ in range(calls):
                if entry(*args) != 0:
                    wrong.append(entry.__name__)
        except Exception as e:
            wrong.append(e)
    threads = [threading.Thread(target=loop, args=call) for call, _, _ in work]
    often = sys.getswitchinterval()
    sys.setswitchinterval(1e-6)                       # the threads take turns as often as they can
    try:
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(often)
    torch.cuda.synchronize()
    assert not wrong, (len(wrong), wrong[:3])
    for _, check, _ in work:
        check()


def test_rules(monkeypatch):
    """Rows enough for a CTA each, which then counts in 41 and 64 KB of shared memory."""
    def make(vocab):
        R = 140
        g = torch.Generator(device=DEV).manual_seed(vocab)
        logits = torch.randn((R, vocab), generator=g, device=DEV)
        history = torch.randint(0, vocab, (R, 64), generator=g, device=DEV, dtype=torch.int32)
        lens, prompt = torch.full((R,), 64, dtype=torch.int32, device=DEV), torch.full((R,), 10, dtype=torch.int32, device=DEV)
        pen, err = torch.tensor([[1.2, 0.1, 0.2]] * R, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
        chosen, want = (torch.zeros(R, dtype=torch.int32, device=DEV) for _ in range(2))

        def go(stream, to=chosen):
            B().logit_rules(logits, None, history, lens, prompt, None, err, stream, penalties=pen, chosen=to)
        go(B().stream_ptr(), want)

        def check():
            assert torch.equal(chosen, want) and err.item() == 0
        return go, chosen.zero_, check
    both(monkeypatch, make, (20_600, 32_768))


def test_eviction(monkeypatch):
    """Tables of 10,400 and 32,000 blocks, whose keys the choice keeps in shared memory."""
    def make(width):
        k, v = (torch.zeros((1, 9, 1, 64, 16), dtype=torch.int8, device=DEV) for _ in range(2))
        ks, vs, w = (torch.ones((1, 9, 1, 4), device=DEV) for _ in range(3))
        w[0, :, 0, :] = torch.arange(36, device=DEV).view(9, 4)
        table = torch.full((1, width), -1, dtype=torch.int32, device=DEV)
        table[0, :5] = torch.arange(5)
        lens, new = torch.tensor([300], dtype=torch.int32, device=DEV), torch.tensor([[7, 8]], dtype=torch.int32, device=DEV)
        kept, err = torch.zeros((1, 1, 1, 4), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)

        def go(stream):
            B().block_evict(k, v, ks, vs, w, table, lens, new, 4, 1, kept, err, stream)

        def check():
            assert kept.flatten().tolist() == [14, 15, 16, 17] and err.item() == 0
        return go, kept.zero_, check
    both(monkeypatch, make, (2_600, 8_000))


def test_attention_as_the_equations_say(monkeypatch):
    """Heads of 176 and of 256, which take 52 and 75 KB."""
    from test_gpu_block_cache import Rig

    def make(D):
        r = Rig(1, 2, D, torch.int8, torch.float32, n_slots=1, width=2, seed=D)
        r.store([0], [50])
        x = r.rows(1).reshape(1, -1).to(DEV)
        view, keep = r.batch([0], [1], [50])
        out, want = (torch.zeros(1, 2 * D, device=DEV) for _ in range(2))
        scratch = torch.zeros(B().block_attention_scratch_floats(1, 2, r.view), device=DEV)

        def go(stream, to=out, keep=keep):
            B().block_attention(x, to, view, r.view, 2, D ** -0.5, scratch, r.err, stream)
        go(B().stream_ptr(), want)

        def check():
            assert torch.equal(out, want) and r.err.item() == 0
        return go, out.zero_, check
    both(monkeypatch, make, (176, 256))

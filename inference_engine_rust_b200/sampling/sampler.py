"""Choice of the next token from logits, on the device.

Reference: `sample_greedy` (first largest logit; empty or non-finite logits are an error,
src/engine/sampling.rs:25-49) and `sample_temperature` (softmax(logits / T), a uniform r
in [0, 1), the first id whose running sum exceeds r, else the last id; T must be positive
and finite, :54-79).  The reference takes the caller's generator; here r is one
Philox4x32-10 draw keyed by the seed with counter (request id, step), so a request draws
the same numbers alone and in any batch.
"""
from __future__ import annotations

import math
import operator
from dataclasses import dataclass
from typing import Dict, List, Mapping, Optional, Sequence, Tuple

import numpy as np
import torch

from ..csrc import bindings as B


class SamplingError(ValueError):
    pass


_F32_MOST, _F32_LEAST = float(np.finfo(np.float32).max), 2.0 ** -149       # the largest and the smallest positive number of 32 bits


@dataclass(frozen=True)
class SamplingParams:
    """temperature 0 = greedy; > 0 = temperature sampling with `seed`.  The penalties and biases are the rules above; `logit_bias` maps
    ids to what is added to their logits (finite, or -infinity)."""
    temperature: float = 0.0
    seed: int = 0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Tuple[Tuple[int, float], ...] = ()

    def __post_init__(self):
        t = self.temperature
        if isinstance(t, bool) or not isinstance(t, (int, float)) or not math.isfinite(t) or t < 0:
            raise SamplingError(f"temperature must be finite and >= 0 (0 = greedy), got {t!r}")
        if isinstance(self.seed, bool) or not isinstance(self.seed, int) or not 0 <= self.seed < 2 ** 64:
            raise SamplingError(f"seed must be an integer in [0, 2^64), got {self.seed!r}")
        for name in ("repetition_penalty", "presence_penalty", "frequency_penalty"):
            v = getattr(self, name)
            if (isinstance(v, bool) or not isinstance(v, (int, float)) or not -_F32_MOST <= v <= _F32_MOST
                    or (name == "repetition_penalty" and v < _F32_LEAST)):
                raise SamplingError(f"{name} must be finite{' and positive' if name == 'repetition_penalty' else ''} in 32 bits, got {v!r}")
        bias = self.logit_bias
        if bias is None:
            bias = ()
        pairs = []
        for pair in bias.items() if isinstance(bias, Mapping) else bias:
            try:
                i, b = pair
                i, b = operator.index(i), float(b)
            except (TypeError, ValueError, OverflowError):
                raise SamplingError(f"logit_bias maps token ids to numbers, got {pair!r}") from None
            if i < 0 or not b <= _F32_MOST:
                raise SamplingError(f"logit_bias: id {i} must be >= 0 and its bias finite or -infinity in 32 bits, got {b!r}")
            pairs.append((i, b))
        if len({i for i, _ in pairs}) != len(pairs):
            raise SamplingError("logit_bias: an id appears twice")
        object.__setattr__(self, "logit_bias", tuple(pairs))

    @property
    def greedy(self) -> bool:
        return self.temperature == 0

    @property
    def penalized(self) -> bool:
        return self.repetition_penalty != 1 or self.presence_penalty != 0 or self.frequency_penalty != 0


def pack_allowed(allowed: Sequence, vocab: int) -> np.ndarray:
    """One row of bits per entry (int32 [rows, ceil(vocab / 32)], bit i % 32 of word i // 32): None = every id, a sequence of ids, or a
    boolean array of the vocabulary's length."""
    words = -(-vocab // 32)
    out = np.empty((len(allowed), words), dtype=np.uint32)
    for r, a in enumerate(allowed):
        if a is None:
            out[r] = 0xFFFFFFFF
            continue
        a = a.cpu().numpy() if isinstance(a, torch.Tensor) else np.asarray(list(a) if not isinstance(a, np.ndarray) else a)
        full = np.zeros(words * 32, dtype=bool)
        if a.dtype == bool:
            if a.shape != (vocab,):
                raise SamplingError(f"a mask of allowed tokens must have the vocabulary's length ({vocab}), got {a.shape}")
            full[:vocab] = a
        else:
            if a.size and (a.ndim != 1 or a.dtype.kind not in "iu" or a.min() < 0 or a.max() >= vocab):
                raise SamplingError(f"allowed tokens must be ids in [0, {vocab})")
            if a.size:
                full[a] = True
        if not full.any():
            raise SamplingError("no token is allowed")
        out[r] = np.packbits(full.reshape(words, 32), axis=1, bitorder="little").view(np.uint32).reshape(words)
    return out.view(np.int32)


class Sampler:
    """Samples one token per row of a float32 [rows, vocab] logits tensor on the device."""

    def __init__(self, params: SamplingParams, err: torch.Tensor):
        self.params = params
        self.err = err
        # page-locked host buffers for the ids on their way back, used in rotation (the generation
        # loop has at most two reads in flight)
        self._host: List[Optional[torch.Tensor]] = [None] * 4
        self._events: list = [None] * 4
        self._turn = 0
        self._ctr_host: List[Optional[torch.Tensor]] = [None] * 4
        self._ctr_events: list = [None] * 4
        self._ctr_turn = 0
        self._bias: Optional[torch.Tensor] = None
        # the running batch's histories, one row per request: ids, lengths, prompt lengths and penalties on the device
        self._row_of: Dict[int, int] = {}
        self._history = self._lens = self._prompt_lens = self._penalties = None

    def begin(self, request_ids: Sequence[int], prompts: Sequence[Sequence[int]], max_new_tokens: int) -> None:
        """Start the histories of a batch (penalties look at the prompt too); those of the batch before are dropped."""
        if not self.params.penalized:
            return
        if len(set(request_ids)) != len(request_ids):
            raise SamplingError("penalties need a different id for every request of a batch")
        self._row_of = {r: i for i, r in enumerate(request_ids)}
        n, width = len(prompts), max((len(p) for p in prompts), default=0) + max(max_new_tokens, 0) + 1
        p, device = self.params, self.err.device
        host = np.full((n, width), -1, dtype=np.int32)
        for i, ids in enumerate(prompts):
            host[i, :len(ids)] = ids
        self._history = torch.from_numpy(host).to(device)
        self._lens = torch.tensor([len(x) for x in prompts], dtype=torch.int32, device=device)
        self._prompt_lens = self._lens.clone()
        self._penalties = torch.tensor([[p.repetition_penalty, p.presence_penalty, p.frequency_penalty]] * n, dtype=torch.float32, device=device)

    def _rules(self, logits: torch.Tensor, request_ids: Sequence[int], allowed) -> Optional[dict]:
        """What `logit_rules` takes for these rows; None where the params ask for nothing."""
        p, vocab = self.params, logits.shape[1]
        if not p.penalized and not p.logit_bias and allowed is None:
            return None
        kw = {"history": None, "lens": None, "prompt_lens": None, "rows": None}
        if p.logit_bias:
            if self._bias is None or self._bias.shape[0] != vocab or self._bias.device != logits.device:
                if max(i for i, _ in p.logit_bias) >= vocab:
                    raise SamplingError(f"logit_bias: id {max(i for i, _ in p.logit_bias)} is outside the vocabulary [0, {vocab})")
                bias = np.zeros(vocab, dtype=np.float32)
                for i, b in p.logit_bias:
                    bias[i] = b
                self._bias = torch.from_numpy(bias).to(logits.device)
            kw["bias"] = self._bias
        if allowed is not None:
            if len(allowed) != logits.shape[0]:
                raise SamplingError("one entry of allowed tokens per row is needed")
            kw["mask"] = torch.from_numpy(pack_allowed(allowed, vocab)).to(logits.device)
        if p.penalized:
            missing = [r for r in request_ids if r not in self._row_of]
            if len(request_ids) != logits.shape[0] or missing or len(set(request_ids)) != len(request_ids):
                raise SamplingError("penalties need the batch's prompts (begin()) and one different request per row"
                                    + (f"; unknown: {missing}" if missing else ""))
            rows = self._counters_to_device([self._row_of[r] for r in request_ids], request_ids, logits.device)[0]
            kw.update(history=self._history, lens=self._lens, prompt_lens=self._prompt_lens, rows=rows, penalties=self._penalties)
        return kw

    def sample_device(self, logits: torch.Tensor, request_ids: Sequence[int],
                      steps: Sequence[int], allowed: Optional[Sequence] = None) -> torch.Tensor:
        """int32 [rows] on the device.  `request_ids[i]`, `steps[i]`: the Philox counter of row i.  With penalties the rows are those
        of requests that `begin` has been told of, and each choice joins its request's history.  `allowed`: for each row the ids
        that may be chosen (a sequence of ids, a boolean array of the vocabulary, or None: all)."""
        rows = logits.shape[0]
        if logits.dim() != 2 or rows == 0 or logits.shape[1] == 0:
            raise SamplingError("logits are empty")          # src/engine/sampling.rs:58-60
        if logits.dtype != torch.float32:
            raise SamplingError(f"logits must be float32, got {logits.dtype}")
        out = torch.empty(rows, dtype=torch.int32, device=logits.device)
        stream = B.stream_ptr()
        rules = self._rules(logits, request_ids, allowed)
        if rules is not None and self.params.greedy:
            B.logit_rules(logits, None, err=self.err, stream=stream, chosen=out, lens_out=rules["lens"], **rules)
        elif rules is not None:
            if len(request_ids) != rows or len(steps) != rows:
                raise SamplingError("one request id and one step per row are needed")
            ruled = torch.empty((rows, logits.shape[1]), dtype=torch.float32, device=logits.device)
            B.logit_rules(logits, ruled, err=self.err, stream=stream, **rules)
            ctr = self._counters_to_device(request_ids, steps, logits.device)
            B.sample_temperature_masked(ruled, float(self.params.temperature), self.params.seed, ctr[0], ctr[1], out, self.err, stream)
            if rules["history"] is not None:
                B.history_append(rules["history"], rules["lens"], rules["rows"], out, self.err, stream)
        elif self.params.greedy:
            B.sample_greedy(logits, out, self.err, stream)
        else:
            if len(request_ids) != rows or len(steps) != rows:
                raise SamplingError("one request id and one step per row are needed")
            ctr = self._counters_to_device(request_ids, steps, logits.device)
            B.sample_temperature(logits, float(self.params.temperature), self.params.seed,
                                 ctr[0], ctr[1], out, self.err, stream)
        return out

    def _counters_to_device(self, request_ids: Sequence[int], steps: Sequence[int], device) -> torch.Tensor:
        """int32 [2, rows] on the device, sent from a page-locked buffer without waiting for the
        device (a copy out of ordinary memory would hold the host until the stream has drained)."""
        rows = len(request_ids)
        i = self._ctr_turn
        self._ctr_turn = (i + 1) % len(self._ctr_host)
        if self._ctr_events[i] is not None:
            self._ctr_events[i].synchronize()          # the copy that last used this buffer is over
        buf = self._ctr_host[i]
        if buf is None or buf.shape[1] < rows:
            buf = self._ctr_host[i] = torch.empty((2, max(rows, 64)), dtype=torch.int32, pin_memory=True)
        view = buf[:, :rows]
        view[0] = torch.tensor(list(request_ids), dtype=torch.int32)
        view[1] = torch.tensor(list(steps), dtype=torch.int32)
        dev = torch.empty((2, rows), dtype=torch.int32, device=device)
        dev.copy_(view, non_blocking=True)
        ev = self._ctr_events[i]
        if ev is None:
            ev = self._ctr_events[i] = torch.cuda.Event()
        ev.record()
        return dev

    def read_async(self, tokens: torch.Tensor) -> "PendingTokens":
        """Start the copy of device token ids (int32 [rows], as `sample_device` returns them) and
        of the device error word to the host, and return at once; `wait()` on the result gives
        the ids.  The caller may launch more work in between: the generation loop starts the
        next step from the ids on the device and reads them on the host one step behind."""
        rows = tokens.shape[0]
        i = self._turn
        self._turn = (i + 1) % len(self._host)
        buf = self._host[i]
        if buf is None or buf.numel() < rows + 1:
            buf = self._host[i] = torch.empty(max(rows + 1, 65), dtype=torch.int32, pin_memory=True)
        buf[:rows].copy_(tokens, non_blocking=True)
        buf[rows:rows + 1].copy_(self.err, non_blocking=True)
        ev = self._events[i]
        if ev is None:
            ev = self._events[i] = torch.cuda.Event()
        ev.record()
        return PendingTokens(self, buf, rows, ev)

    def __call__(self, logits: torch.Tensor, request_ids: Sequence[int], steps: Sequence[int],
                 allowed: Optional[Sequence] = None) -> List[int]:
        """Host token ids (synchronises), after checking the device error word."""
        return self.read_async(self.sample_device(logits, request_ids, steps, allowed)).wait()


class PendingTokens:
    """Token ids on their way to the host (one copy for the ids and the error word, one wait)."""

    def __init__(self, sampler: Sampler, buf: torch.Tensor, rows: int, event):
        self._sampler, self._buf, self._rows, self._event = sampler, buf, rows, event

    def wait(self) -> List[int]:
        """The ids, after checking the device error word as it stood when they were chosen."""
        self._event.synchronize()
        values = self._buf[:self._rows + 1].tolist()
        bits = values.pop()
        if bits:
            self._sampler.err.zero_()
            raise SamplingError(B.describe_error_bits(bits))
        return values

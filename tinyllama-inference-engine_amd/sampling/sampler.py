"""Sampling from the step's logits.

reference: greedy is the first index of the maximum and refuses NaN or Inf
(src/operators.cpp:166-175); with temperature > 0 the server draws from the top-p part of
softmax(logits / T) (app/server.cpp:237-277) with a generator seeded per request (:198).  Here the
draw is made on the device by one kernel for all rows, and the uniform number for a row is a
hash of (the request's seed, the index of the token being generated): it is the same whatever
else is in the batch and however the prompt was cut, also after a preemption.  Rows that ask for top_k or min_p are drawn by
`ops.sample_filtered` with the same number (its order is that of the logits, not of the vocabulary); the others as ever.
"""
from __future__ import annotations

from operator import attrgetter

import numpy as np
import torch

from .. import ops
from ..errors import EngineError, ErrorCode

MASK64 = (1 << 64) - 1


def splitmix64(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & MASK64
    x = ((x ^ (x >> 30)) * 0xBF58476D1CE4E5B9) & MASK64
    x = ((x ^ (x >> 27)) * 0x94D049BB133111EB) & MASK64
    return x ^ (x >> 31)


def uniform01(seed: int, counter: int) -> float:
    """The uniform number in [0, 1) that the kernel uses for (seed, counter): 24 bits."""
    h = splitmix64(splitmix64(seed & MASK64) ^ ((counter * 0xD1342543DE82EF95 + 1) & MASK64))
    return (h >> 40) / 16777216.0


def uniforms01(seeds, counters) -> np.ndarray:
    """`uniform01` of many rows, float32."""
    def mix(x):
        x = x + np.uint64(0x9E3779B97F4A7C15)
        x = (x ^ (x >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        x = (x ^ (x >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
        return x ^ (x >> np.uint64(31))
    seeds = np.array([int(seed) & MASK64 for seed in seeds], dtype=np.uint64)
    counters = np.array([(int(counter) * 0xD1342543DE82EF95 + 1) & MASK64 for counter in counters], dtype=np.uint64)
    return ((mix(mix(seeds) ^ counters) >> np.uint64(40)).astype(np.float64) / 16777216.0).astype(np.float32)


def _signed(value: int) -> int:
    value &= MASK64
    return value - (1 << 64) if value >= (1 << 63) else value


_LOGPROBS, _TOP_K, _MIN_P = attrgetter("logprobs"), attrgetter("top_k"), attrgetter("min_p")


def what_rows_ask(params: list) -> tuple[bool, list[bool] | None]:
    """(whether a row asks for log-probabilities, which rows are drawn with top_k or min_p; None: none).  (Most steps have neither, and
    are asked three questions without any Python a row: of 256 rows 23 us in place of 59.)"""
    try:
        wants_logprobs = any(map(_LOGPROBS, params))
        if not any(map(_TOP_K, params)) and not any(map(_MIN_P, params)):
            return wants_logprobs, None
    except AttributeError:                                # (params need not have these)
        wants_logprobs = any(getattr(p, "logprobs", False) for p in params)
    filtered = [p.temperature > 0.0 and getattr(p, "filtered", False) for p in params]
    return wants_logprobs, filtered if any(filtered) else None


class PendingTokens:
    """A step's sampled tokens on their way to the host.  `read()` waits for them."""

    def __init__(self, host: torch.Tensor, event, rows: int, logprobs: torch.Tensor | None = None):
        self._host, self._event, self.rows, self._logprobs = host, event, rows, logprobs

    def read(self) -> list[int]:
        if self._event is not None:
            self._event.synchronize()
        out = self._host[:self.rows].tolist()
        if any(token < 0 for token in out):
            raise EngineError(ErrorCode.NUMERICAL, "logits contain NaN or Inf")
        return out

    def read_logprobs(self) -> list[float] | None:
        """The tokens' log-probabilities, when a row asked for them (else None).  Waits like `read`."""
        if self._event is not None:
            self._event.synchronize()
        return self._logprobs[:self.rows].tolist() if self._logprobs is not None else None


class Sampler:
    """Samples on the device into a buffer that stays where it is (`device_tokens`: a decode step
    can take its tokens from there before the host has seen them) and copies the tokens to pinned
    host memory without waiting.  Two sets of host buffers are used in turn: a caller may have at
    most one `PendingTokens` unread when it samples again."""

    def __init__(self, device, capacity: int = 64):
        self.device = torch.device(device)
        self.capacity = capacity
        self.device_tokens = torch.zeros(capacity, dtype=torch.int32, device=self.device)
        self._floats = torch.zeros((4, capacity), dtype=torch.float32, device=self.device)      # temperature, top_p, min_p, the random number
        self._top_k = torch.zeros(capacity, dtype=torch.int32, device=self.device)
        self._marks = torch.zeros(capacity, dtype=torch.bool, device=self.device)               # rows that `ops.sample_filtered` draws
        self._logprobs = torch.zeros(capacity, dtype=torch.float32, device=self.device)
        self._host_logprobs = [torch.zeros(capacity, dtype=torch.float32, pin_memory=True) for _ in range(2)]
        self._host_top_k = [torch.zeros(capacity, dtype=torch.int32, pin_memory=True) for _ in range(2)]
        self._host_marks = [torch.zeros(capacity, dtype=torch.bool, pin_memory=True) for _ in range(2)]
        self._longs = torch.zeros((2, capacity), dtype=torch.int64, device=self.device)         # seed, counter
        self._host_tokens = [torch.zeros(capacity, dtype=torch.int32, pin_memory=True) for _ in range(2)]
        self._host_floats = [torch.zeros((4, capacity), dtype=torch.float32, pin_memory=True) for _ in range(2)]
        self._host_longs = [torch.zeros((2, capacity), dtype=torch.int64, pin_memory=True) for _ in range(2)]
        self._events = [torch.cuda.Event(), torch.cuda.Event()]
        self._turn = 0

    def sample_async(self, logits: torch.Tensor, params: list, counters: list[int]) -> PendingTokens:
        """One token per row, left in `device_tokens[:rows]` and on its way to the host.
        params[i] has temperature, top_p and seed, and may have top_k, min_p and logprobs; counters[i] is the index of the
        token row i generates."""
        rows = logits.shape[0]
        if rows == 0:
            return PendingTokens(self._host_tokens[0], None, 0)
        if rows > self.capacity:
            raise EngineError(ErrorCode.INVALID_ARGUMENT, f"the sampler was made for {self.capacity} rows, not {rows}")
        turn = self._turn
        self._turn ^= 1
        out = self.device_tokens[:rows]
        wants_logprobs, filtered = what_rows_ask(params)
        if wants_logprobs or filtered is not None:
            self._sample_filtered(logits, params, counters, filtered or [False] * rows, wants_logprobs, out, turn)
        elif all(not p.temperature > 0.0 for p in params):
            ops.sample(logits, out=out)
        else:
            floats, longs = self._host_floats[turn], self._host_longs[turn]
            floats[0, :rows] = torch.tensor([float(p.temperature) for p in params], dtype=torch.float32)
            floats[1, :rows] = torch.tensor([float(p.top_p) for p in params], dtype=torch.float32)
            longs[0, :rows] = torch.tensor([_signed(int(p.seed)) for p in params], dtype=torch.int64)
            longs[1, :rows] = torch.tensor([int(c) for c in counters], dtype=torch.int64)
            self._floats.copy_(floats, non_blocking=True)
            self._longs.copy_(longs, non_blocking=True)
            ops.sample(logits, self._floats[0, :rows], self._floats[1, :rows], self._longs[0, :rows], self._longs[1, :rows],
                       out=out)
        host = self._host_tokens[turn]
        host[:rows].copy_(out, non_blocking=True)
        if wants_logprobs:
            self._host_logprobs[turn][:rows].copy_(self._logprobs[:rows], non_blocking=True)
        self._events[turn].record()
        return PendingTokens(host, self._events[turn], rows, self._host_logprobs[turn] if wants_logprobs else None)

    def _sample_filtered(self, logits, params, counters, filtered, wants_logprobs, out, turn) -> None:
        """A step with rows that ask for top_k or min_p, or for log-probabilities: `ops.sample_filtered` over all rows, and for the rows that
        ask for neither filter the tokens that `ops.sample` draws (a row's token does not depend on what else is in the step)."""
        rows = logits.shape[0]
        floats, longs, top_k, marks = self._host_floats[turn], self._host_longs[turn], self._host_top_k[turn], self._host_marks[turn]
        floats[0, :rows] = torch.tensor([float(p.temperature) for p in params], dtype=torch.float32)
        floats[1, :rows] = torch.tensor([float(p.top_p) for p in params], dtype=torch.float32)
        floats[2, :rows] = torch.tensor([float(getattr(p, "min_p", 0.0)) for p in params], dtype=torch.float32)
        floats[3, :rows] = torch.from_numpy(uniforms01([p.seed for p in params], counters))
        top_k[:rows] = torch.tensor([int(getattr(p, "top_k", 0)) for p in params], dtype=torch.int32)
        self._floats.copy_(floats, non_blocking=True)
        self._top_k.copy_(top_k, non_blocking=True)
        device = self._floats[:, :rows]
        logprobs = self._logprobs[:rows] if wants_logprobs else None
        ops.sample_filtered(logits, device[3], device[0], top_k=self._top_k[:rows], top_p=device[1], min_p=device[2], logprobs=wants_logprobs, out=out,
                            out_logprobs=logprobs, finite=True)
        if all(filtered):
            return
        longs[0, :rows] = torch.tensor([_signed(int(p.seed)) for p in params], dtype=torch.int64)
        longs[1, :rows] = torch.tensor([int(c) for c in counters], dtype=torch.int64)
        marks[:rows] = torch.tensor(filtered)
        self._longs.copy_(longs, non_blocking=True)
        self._marks.copy_(marks, non_blocking=True)
        plain = ops.sample(logits, device[0], device[1], self._longs[0, :rows], self._longs[1, :rows])
        if wants_logprobs:
            # another token of the same row: its log-probability differs by the difference of the logits
            both = logits.gather(1, torch.stack([plain, out], dim=1).clamp(min=0).long())
            logprobs.add_(torch.where(self._marks[:rows], torch.zeros_like(logprobs), both[:, 0] - both[:, 1]))
        out.copy_(torch.where(self._marks[:rows], out, plain))

    def sample(self, logits: torch.Tensor, params: list, counters: list[int]) -> list[int]:
        """One token per row, on the host.  Raises `numerical_error` on NaN or Inf logits."""
        return self.sample_async(logits, params, counters).read()

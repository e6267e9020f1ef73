"""Sampling: greedy and temperature.

The reference samples greedily only: `logits[:, -1].argmax(-1)` on the host side of
the step (model/inference_paged.py:166,193), ties to the lowest index; temperature is
described as softmax(logits / T) (docs/day_1_docs.md:45-52) and forced to 0 in its
benchmark.  Here both run in one kernel on float32 logits (socrates_b200/csrc/sampling.cu):

* temperature 0: argmax, ties to the lowest index;
* temperature T > 0: a draw from softmax(logits / T) by the Gumbel-max rule,
  token = argmax_i (logit_i / T - log(-log u_i)).

u_i is a counter-based uniform, a pure function of (seed, counter, i): with mix32 the
three-round xorshift-multiply finalizer (constants 0x7FEB352D, 0x846CA68B, shifts
16/15/16) on unsigned 32-bit integers,

    key = mix32(mix32(seed ^ 0x9E3779B9) ^ mix32(counter + 0x85EBCA6B))
    u_i = ((mix32((i + 0x165667B1) ^ key) >> 9) + 0.5) / 2^23

`counter` is the number of tokens the request has produced so far, so a request's
tokens depend on its seed alone: not on the batch it ran in, not on how its prompt was
cut, not on whether it was preempted and recomputed.

Before either rule a request may have its logits adjusted (in the same kernel's pass; see kernels/ops.py
sample_adjusted for the formulas): penalties for tokens that its prompt and output hold already, biases on single
tokens, and a set of allowed tokens, fixed or (a grammar) a function of the output so far.
"""

from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Iterable, Mapping, Optional, Union

import numpy as np

MAX_BIASES = 512                 # of one request
MOST_ADJUSTED = 262144           # tokens of a vocabulary whose logits can be adjusted (see ops.sample_adjusted)
LARGEST = 1e30                   # penalty or bias: with any logit, and counted 10^7 times, it is finite in float32


@dataclass(frozen=True)
class SamplingParams:
    temperature: float = 0.0     # 0 = greedy
    seed: int = 0
    repetition_penalty: float = 1.0      # logits of tokens in the prompt or output: l / r if l > 0 else l * r
    presence_penalty: float = 0.0        # taken off logits of tokens in the output
    frequency_penalty: float = 0.0       # taken off once for every time a token stands in the output
    logit_bias: Optional[Mapping[int, float]] = None        # token -> what is added to its logit
    # The tokens that may come next: ids or a packed mask (`pack_allowed`), or a function from the output so far (a list of
    # ids) to one of these or to None for all.  A function that allows nothing ends the request.
    allowed: Optional[Union[Iterable[int], Callable]] = None

    def __post_init__(self):
        # what walks and changes is kept as it is now: iterators are walked more than once, masks are the caller's arrays
        if isinstance(self.allowed, AllowedMask):
            object.__setattr__(self, "allowed", self.allowed.copy())
        elif self.allowed is not None and not callable(self.allowed):
            object.__setattr__(self, "allowed", list(self.allowed))
        if self.logit_bias is not None:
            object.__setattr__(self, "logit_bias", dict(self.logit_bias))

    def validate(self, vocab: Optional[int] = None, packed: bool = False) -> None:
        """`vocab`: check token ids, too (`packed`: those of a fixed set were, when it was packed)."""
        if not self.temperature >= 0.0:
            raise ValueError(f"temperature must be >= 0, got {self.temperature}")
        if not 1 / LARGEST <= self.repetition_penalty <= LARGEST:
            raise ValueError(f"repetition_penalty must be positive, got {self.repetition_penalty}")
        for name in ("presence_penalty", "frequency_penalty"):
            if not abs(getattr(self, name)) <= LARGEST:
                raise ValueError(f"{name} must be finite, got {getattr(self, name)}")
        if self.logit_bias is not None:
            if len(self.logit_bias) > MAX_BIASES:
                raise ValueError(f"{len(self.logit_bias)} biases; a request has at most {MAX_BIASES}")
            for t, b in self.logit_bias.items():
                if vocab is not None and not 0 <= int(t) < vocab:
                    raise ValueError(f"a bias on token {t}, outside the vocabulary of {vocab}")
                if not (abs(b) <= LARGEST or b == -math.inf):
                    raise ValueError(f"a bias of {b} on token {t}")
        if self.allowed is not None and not callable(self.allowed) and vocab is not None and not packed:
            if pack_allowed(self.allowed, vocab) is None:
                raise ValueError("no token is allowed")

    @property
    def penalizes(self) -> bool:
        return self.repetition_penalty != 1.0 or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0

    @property
    def adjusts(self) -> bool:
        """Whether logits are adjusted at all."""
        return self.penalizes or bool(self.logit_bias) or self.allowed is not None


class AllowedMask(np.ndarray):
    """A packed mask, int32 [ceil(vocab / 32)]: bit t % 32 of word t // 32 allows token t.  `pack_allowed` makes them, `&` and
    `|` of two are masks again, and `words.view(AllowedMask)` says that an array is one: nothing else about an array does,
    as ids may be so many and of that type."""


def pack_allowed(allowed, vocab: int) -> Optional[AllowedMask]:
    """A set of token ids (of any iterable, arrays among them) as the mask that the kernel takes.  An AllowedMask is one already.
    None if nothing is allowed."""
    words = -(-vocab // 32)
    if isinstance(allowed, AllowedMask):
        if allowed.dtype != np.int32 or allowed.shape != (words,):
            raise ValueError(f"a mask of {allowed.dtype} {allowed.shape} with a vocabulary of {vocab}")
        tail = vocab % 32
        last = int(allowed[-1]) & ((1 << tail) - 1 if tail else -1)
        return allowed if last or allowed[:-1].any() else None
    ids = np.fromiter((int(t) for t in allowed), dtype=np.int64)
    if ids.size == 0:
        return None
    if ids.min() < 0 or ids.max() >= vocab:
        raise ValueError(f"allowed tokens from {ids.min()} to {ids.max()} with a vocabulary of {vocab}")
    bits = np.zeros(words * 32, dtype=np.uint8)
    bits[ids] = 1
    return np.packbits(bits, bitorder="little").view("<i4").view(AllowedMask)


__all__ = ["AllowedMask", "MAX_BIASES", "MOST_ADJUSTED", "SamplingParams", "pack_allowed"]

"""Picking tokens from logits.

Greedy: the smallest index attaining the maximum, NaN never wins -- the rule
the reference's host and device argmax share
(/root/reference/crates/imparo-cpu/src/ops.rs:628-640). The reference's
`sample` ignores the temperature it parses
(/root/reference/crates/imparo-server/src/main.rs:3382-3390); here a positive
temperature draws from softmax(logits / T) by inverse CDF with a uniform
number that depends only on (seed, index of the generated token), so a
request's draws do not depend on what it was batched with. top-k, top-p and
min-p leave tokens out before the draw, each by the request's own value.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence, Tuple


_MASK = (1 << 64) - 1


def _splitmix64(x: int) -> int:
    x = (x + 0x9E3779B97F4A7C15) & _MASK
    z = x
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _MASK
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _MASK
    return z ^ (z >> 31)


def uniform_for(seed: int, index: int) -> float:
    """A number in [0, 1) with 24 random bits, a pure function of (seed, index)."""
    h = _splitmix64(_splitmix64(seed & _MASK) ^ ((index * 0xD1342543DE82EF95) & _MASK))
    return (h >> 40) / float(1 << 24)


@dataclass
class SamplingParams:
    """`max_tokens` and `temperature` carry the reference's request fields of
    those names (/root/reference/crates/imparo-server/src/main.rs:1849-1872);
    temperature 0 is greedy. `top_k` keeps the so many likeliest tokens (0:
    all), `top_p` of those the fewest likeliest that hold top_p of their
    probability (1: all), `min_p` of those the ones at least min_p times as
    likely as the likeliest (0: all); equal logits count in the order of
    their ids."""
    temperature: float = 0.0
    max_tokens: int = 16
    seed: int = 0
    stop_token_ids: Tuple[int, ...] = ()
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        if isinstance(self.top_k, bool) or not hasattr(self.top_k, "__index__") or not 0 <= self.top_k < 1 << 31:
            raise ValueError(f"top_k is a whole number of tokens, or 0 for all of them; got {self.top_k!r}")
        if not 0.0 < self.top_p <= 1.0:
            raise ValueError(f"top_p lies above 0 and up to 1 (all tokens); got {self.top_p!r}")
        if not 0.0 <= self.min_p <= 1.0:
            raise ValueError(f"min_p lies between 0 (all tokens) and 1; got {self.min_p!r}")

    @property
    def filters(self) -> Tuple[int, float, float]:
        """(top_k, top_p, min_p)."""
        return self.top_k, self.top_p, self.min_p


NO_FILTERS = (0, 1.0, 0.0)


class PendingPick:
    """Token ids that the sampling kernel has been asked for. `on_device` is
    the int32 vector they land in (to feed the next step from, without
    waiting); `tokens()` waits for the copy to the host and returns them.
    The vectors are the sampler's own and are used again after `Sampler.RING`
    further picks: feed `on_device` to the next step or two, not later (the
    ids themselves are read out in time by the sampler if the caller has not)."""

    def __init__(self, on_device, host, event):
        self.on_device = on_device
        self._host = host
        self._event = event
        self._tokens: Optional[List[int]] = None

    def tokens(self) -> List[int]:
        if self._tokens is None:
            self._event.synchronize()
            self._tokens = self._host.tolist()
        return self._tokens


class _PickBuffers:
    """What one pick needs, allocated once: the ids on the device and in pinned host memory,
    temperatures, uniform numbers and filters (top-k as the bits of an int32) in pinned host memory and on the device."""

    def __init__(self, torch, device, capacity: int):
        self.capacity = capacity
        self.ids = torch.empty(capacity, dtype=torch.int32, device=device)
        self.ids_host = torch.empty(capacity, dtype=torch.int32, pin_memory=True)
        self.params_host = torch.empty(5, capacity, dtype=torch.float32, pin_memory=True)
        self.params = torch.empty(5, capacity, dtype=torch.float32, device=device)
        self.last: Optional[PendingPick] = None


class Sampler:
    """Runs the sampling kernels over the logits rows a step returned. Its
    buffers go round in a ring, so a pick allocates nothing once the ring has
    seen the batch size."""
    RING = 8

    def __init__(self, device):
        import torch
        self.device = device
        self._torch = torch
        self._ring: List[Optional[_PickBuffers]] = [None] * self.RING
        self._turn = 0

    def _buffers(self, n: int) -> _PickBuffers:
        i = self._turn
        self._turn = (i + 1) % self.RING
        b = self._ring[i]
        if b is not None and b.last is not None:
            b.last.tokens()          # whoever still holds that pick finds its ids read out; the buffers are free
            b.last = None
        if b is None or b.capacity < n:
            b = self._ring[i] = _PickBuffers(self._torch, self.device, max(64, 1 << (n - 1).bit_length()))
        return b

    def pick_async(self, logits, temperatures: Sequence[float], uniforms: Sequence[float],
                   filters: Optional[Sequence[Tuple[int, float, float]]] = None) -> PendingPick:
        """Queues the kernel and the copy of its result to the host; returns at once. `filters`: (top_k, top_p, min_p)
        for every row (NO_FILTERS for a row without any)."""
        torch = self._torch
        from ..kernels import ops
        n = logits.shape[0]
        if filters is not None and len(filters) != n:
            raise ValueError(f"filters of {len(filters)} rows were given for {n} rows of logits")
        b = self._buffers(n)
        out = b.ids[:n]
        if all(t <= 0 for t in temperatures):
            ops.argmax_rows(logits, out)
        else:
            # (a greedy row's filters are of no bearing on its pick)
            filtered = filters is not None and any(t > 0 and tuple(f) != NO_FILTERS for t, f in zip(temperatures, filters))
            b.params_host[0, :n] = torch.tensor(list(temperatures), dtype=torch.float32)
            b.params_host[1, :n] = torch.tensor(list(uniforms), dtype=torch.float32)
            if filtered:
                b.params_host[2].view(torch.int32)[:n] = torch.tensor([f[0] for f in filters], dtype=torch.int32)
                b.params_host[3:5, :n] = torch.tensor([[f[1] for f in filters], [f[2] for f in filters]], dtype=torch.float32)
                b.params.copy_(b.params_host, non_blocking=True)
                ops.sample_rows(logits, b.params[0, :n], b.params[1, :n], out, top_k=b.params[2].view(torch.int32)[:n],
                                top_p=b.params[3, :n], min_p=b.params[4, :n])
            else:
                b.params[:2].copy_(b.params_host[:2], non_blocking=True)
                ops.sample_rows(logits, b.params[0, :n], b.params[1, :n], out)
        back = b.ids_host[:n]
        back.copy_(out, non_blocking=True)
        event = torch.cuda.Event()
        event.record()
        b.last = PendingPick(out, back, event)
        return b.last

    def pick(self, logits, temperatures: Sequence[float], uniforms: Sequence[float],
             filters: Optional[Sequence[Tuple[int, float, float]]] = None) -> List[int]:
        return self.pick_async(logits, temperatures, uniforms, filters).tokens()

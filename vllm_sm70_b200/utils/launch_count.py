"""Counts launches of this library's own kernels (not torch's) so a benchmark
can report how many native kernels ran in its timed region. Eager launches
are counted by the op wrappers; CUDA-graph replays add the per-graph count
recorded at capture time."""
from __future__ import annotations

import threading

_lock = threading.Lock()
_total = 0
_others = []  # counters kept elsewhere
_before = 0   # what they held when they did not count yet


def add(n: int = 1) -> None:
    global _total
    with _lock:
        _total += n


def also(counter) -> None:
    """Counts what ``counter()`` grows by from now on, too (launches that
    native code makes on its own, such as a backward pass's)."""
    global _before
    if counter in _others:
        return
    with _lock:
        if counter not in _others:
            _before += counter()
            _others.append(counter)


def total() -> int:
    return _total + sum(c() for c in _others) - _before


def reset() -> None:
    global _total, _before
    with _lock:
        _total = 0
        _before = sum(c() for c in _others)

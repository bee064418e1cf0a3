"""CPU oracle for the rules on logits (numpy, fp32 step by step).

TEST INFRASTRUCTURE ONLY, like the rest of this package.
"""
from __future__ import annotations

import numpy as np

F = np.float32


def adjust(x, ids=None, prompt=0, repetition=1.0, frequency=0.0, presence=0.0, biases=(), allowed=None, offset=0):
    """One row x [N] fp32 -> the row under the rules, and the token (-1: none).

    ids: the row's tokens; biases: (id, value) pairs in order; allowed: truth
    values of the whole vocabulary; offset: token of column 0."""
    x = np.array(x, F)
    N = len(x)
    with np.errstate(all="ignore"):
        if ids is not None:
            seen, times = np.zeros(N, bool), np.zeros(N, np.int64)
            for i, v in enumerate(ids):
                if 0 <= v - offset < N:
                    seen[v - offset] = True
                    times[v - offset] += i >= prompt
            x = np.where(seen, np.where(x > 0, x / F(repetition), x * F(repetition)), x)
            x = np.where(times > 0, (x - F(frequency) * times.astype(F)) - F(presence), x)
        last = {}
        for v, b in biases:
            if 0 <= v - offset < N and v >= 0:
                last[v - offset] = F(b)
        for v, b in last.items():
            x[v] = x[v] + b
    ok = np.ones(N, bool) if allowed is None else np.asarray(allowed[offset:offset + N], bool)
    x = np.where(ok, x, F(-np.inf)).astype(F)
    at = np.flatnonzero(ok)
    if not len(at):
        return x, -1
    nan = np.flatnonzero(np.isnan(x[at]))
    return x, int(at[nan[0]] if len(nan) else at[np.argmax(x[at])]) + offset

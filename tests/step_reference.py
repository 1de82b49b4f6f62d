"""Plain restatements, in 64 bits, of the step operators: metadata from request lengths, the
multi-axis rotation and linear attention with a decay per head; and error bounds of the last two."""
from __future__ import annotations

import numpy as np

# Largest relative error of one rounding to the type.
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def step_metadata(context_lens, query_lens, table, free, num_tokens, block_size, offsets=None):
    """Request by request, token by token: (cu_q, cu_k, slots, positions, cu_new, table)."""
    table = np.array(table, dtype=np.int64)
    width = table.shape[1]
    slots = np.full(num_tokens, -1, np.int64)
    positions = np.zeros(num_tokens, np.int64)
    cu_q, cu_k, cu_new = [0], [0], [0]
    for b, (c, q) in enumerate(zip(map(int, context_lens), map(int, query_lens))):
        held = min(width, -(-c // block_size))
        need = min(width, -(-(c + q) // block_size))
        cu_new.append(cu_new[-1] + need - held)
        if cu_new[-1] <= len(free):
            table[b, held:need] = free[cu_new[-2]:cu_new[-1]]
            reach = need
        else:
            reach = held
        for i in range(q):
            row, p = cu_q[-1] + i, c + i
            if row >= num_tokens:
                break
            positions[row] = p + (0 if offsets is None else int(offsets[b]))
            if p // block_size < reach:
                slots[row] = table[b, p // block_size] * block_size + p % block_size
        cu_q.append(cu_q[-1] + q)
        cu_k.append(cu_k[-1] + c + q)
    return np.array(cu_q), np.array(cu_k), slots, positions, np.array(cu_new), table


def axis_of(sections, interleaved):
    """The axis of each frequency."""
    if not interleaved:
        return np.repeat(np.arange(len(sections)), sections)
    owner = np.zeros(sum(sections), np.int64)
    for a in range(1, len(sections)):
        owner[a:len(sections) * sections[a]:len(sections)] = a
    return owner


def norm_rotate(x, weight, eps, table, positions, sections, interleaved):
    """x [T, H, D] float64 -> normed (weight None: not) and rotated; positions [A, T]."""
    x = np.asarray(x, np.float64)
    half = x.shape[-1] // 2
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    row = np.clip(positions, 0, table.shape[0] - 1)[axis_of(sections, interleaved)].T  # [T, half]
    j = np.arange(half)
    cos, sin = (table.astype(np.float64)[row, j + o][:, None] for o in (0, half))
    a, b = x[..., :half], x[..., half:]
    return np.concatenate([a * cos - b * sin, b * cos + a * sin], -1)


def rotate_bound(x, weight, eps, table, positions, sections, interleaved, dtype, want):
    """Elementwise bound of |got - want| for fp32 arithmetic rounded once: half a step of the
    result, plus 2^-24 of the two products' sizes for each operation before it: at most D + 4 in
    the mean of squares and the reciprocal of its root, 2 for the weight, 2 for the rotation."""
    half = x.shape[-1] // 2
    size = np.abs(x)
    if weight is not None:
        size = size / np.sqrt((size * size).mean(-1, keepdims=True) + eps) * np.abs(weight)
    row = np.clip(positions, 0, table.shape[0] - 1)[axis_of(sections, interleaved)].T
    j = np.arange(half)
    cos, sin = (np.abs(table.astype(np.float64))[row, j + o][:, None] for o in (0, half))
    a, b = size[..., :half], size[..., half:]
    size = np.concatenate([a * cos + b * sin, b * cos + a * sin], -1)
    return HALF_STEP[dtype] * np.abs(want) + (x.shape[-1] + 8) * HALF_STEP["f32"] * size + _TINY[dtype]


# Half the spacing of the type's subnormal numbers.
_TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def linear_attention(q, k, v, log_decay, state, slots, lens, scale, fresh=None, out=None):
    """The recurrence over each sequence's tokens, float64.  Returns out, state and, with the
    same shapes, the sums of absolute values that bound their errors.  Sequences with a slot
    outside the state are skipped, those without tokens leave their slot alone."""
    q, k, v, state = (np.asarray(x, np.float64) for x in (q, k, v, state))
    state = state.copy()
    size = np.abs(state)
    out = np.zeros_like(q) if out is None else np.array(out, np.float64)
    out_size = np.zeros_like(q)
    group = q.shape[1] // k.shape[1]
    with np.errstate(over="ignore"):
        decay = np.exp(np.asarray(log_decay, np.float64))[:, None, None]
    at = 0
    for b, n in enumerate(map(int, lens)):
        s = int(slots[b])
        if n == 0 or not 0 <= s < state.shape[0]:
            at += n
            continue
        now, mag = state[s], size[s]
        if fresh is not None and fresh[b]:
            now, mag = np.zeros_like(now), np.zeros_like(mag)
        for t in range(at, at + n):
            now = now * decay + k[t][:, :, None] * v[t][:, None, :]
            mag = mag * decay + np.abs(k[t][:, :, None] * v[t][:, None, :])
            qt = q[t].reshape(-1, group, q.shape[2])
            out[t] = scale * (qt @ now).reshape(q.shape[1:])
            out_size[t] = abs(scale) * (np.abs(qt) @ mag).reshape(q.shape[1:])
        state[s], size[s] = now, mag
        at += n
    return out, state, out_size, size


def assert_linear_close(got, want, size, dtype, longest, what):
    """Outputs and states of linear attention against the 64-bit recurrence.

    Elementwise: an output is rounded once (half a step of itself); before that the scores and
    the state are each rounded once to the type on their way into the matrix products (half a
    step of the sum of absolute values that they are part of); fp32 sums over at most D + longest
    terms add 2^-24 of that sum each.  A state is held in fp32; the values that are added to it
    go through the matrix products as 16-bit parts, together off by at most 2^-16.
    In the 2-norm, for inputs of independent signs, where errors add as the terms do: the three
    roundings together stay under twice a half step, the state's under 2^-19."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape
    assert np.array_equal(np.isfinite(got), np.isfinite(want)), f"{what}: finite values differ"
    fine = np.isfinite(want)
    got, want, size = got[fine], want[fine], size[fine]
    if not got.size:
        return
    sums = (128 + longest) * HALF_STEP["f32"]
    if dtype == "f32":
        bound = (2.0 ** -16 + sums) * size
        norm = 2.0 ** -19
    else:
        u = HALF_STEP[dtype]
        bound = u * np.abs(want) + (u + sums) * size + _TINY[dtype]
        norm = 2 * u
    err = np.abs(got - want)
    rel = float(np.linalg.norm(err) / max(np.linalg.norm(want), 1e-300))
    print(f"{what}: relative error {rel:.2e}, largest error / bound {float((err / np.maximum(bound, 1e-300)).max()):.2f}",
          flush=True)
    assert np.all(err <= bound), f"{what}: error {err.max():.3e}, over its bound by {float((err / bound).max()):.2f}"
    assert rel <= norm, f"{what}: relative error {rel:.2e} > {norm:.2e}"

"""The multi-axis prologue on the GPU against norm and rotation in 64 bits; v rows and rows that
are not written, bit for bit."""
import numpy as np
import pytest

import oracle
import step_reference as ref
from helpers import normal_bits, to_bits, to_torch

pytestmark = pytest.mark.gpu

EPS, MAX_POS = 1e-6, 700


def _inputs(seed, T, Hq, Hkv, D, dtype, axes, pad=0, weights=True):
    rng = np.random.default_rng(seed)
    row = (Hq + 2 * Hkv) * D
    table = rng.standard_normal((MAX_POS, D)).astype(np.float32)
    angle = rng.uniform(0, 2 * np.pi, (MAX_POS, D // 2))
    table[:, :D // 2], table[:, D // 2:] = np.cos(angle), np.sin(angle)
    pos = rng.integers(-3, MAX_POS + 3, (axes, T)).astype(np.int32)  # clamped at both ends
    w = [oracle.float_to_half((1 + 0.2 * rng.standard_normal(D)).astype(np.float32), dtype) if weights else None
         for _ in range(2)]
    NB, BS = -(-T // 16) + 2, 16
    slots = rng.permutation(NB * BS)[:T].astype(np.int64)
    caches = [normal_bits(rng, (NB, BS, Hkv, D), dtype) for _ in range(2)]
    return normal_bits(rng, (T, row + pad), dtype, 2.0), w, table, pos, slots, caches


def _value(bits, dtype):
    return oracle.bits_to_f32(bits.reshape(-1, bits.shape[-1]), dtype).astype(np.float64).reshape(bits.shape)


def _call(device, dtype, D, Hq, Hkv, x, w, table, pos, sections, caches, slots, **kw):
    import torch
    import oxide_paged_kv as ox

    row = (Hq + 2 * Hkv) * D
    qkv = to_torch(x, dtype, device)[:, :row]
    wq, wk = (None if v is None else to_torch(v, dtype, device) for v in w)
    kc, vc = (None, None) if caches is None else (to_torch(c, dtype, device) for c in caches)
    r = ox.qk_norm_mrope_and_cache(qkv, Hq, Hkv, wq, wk, EPS, torch.from_numpy(table).to(device),
                                   torch.from_numpy(pos).to(device), sections, kc, vc,
                                   None if slots is None else torch.from_numpy(slots).to(device), **kw)
    return r, kc, vc


def _check(device, seed, T, Hq, Hkv, D, dtype, sections, interleaved=False, pad=0, weights=True):
    x, w, table, pos, slots, caches = _inputs(seed, T, Hq, Hkv, D, dtype, len(sections), pad, weights)
    if T > 3:
        slots[1], slots[2], slots[3] = -1, -7, caches[0].shape[0] * 16  # no slot, no slot, past the cache
    (q, k), kc, vc = _call(device, dtype, D, Hq, Hkv, x, w, table, pos, sections, caches, slots,
                           interleaved=interleaved, return_k=True)
    val = _value(x[:, :(Hq + 2 * Hkv) * D].reshape(T, -1, D), dtype)
    wv = [None if v is None else _value(v[None], dtype)[0] for v in w]
    for got, part, wt in ((q, val[:, :Hq], wv[0]), (k, val[:, Hq:Hq + Hkv], wv[1])):
        want = ref.norm_rotate(part, wt, EPS, table, pos, sections, interleaved)
        err = np.abs(_value(to_bits(got), dtype) - want)
        bound = ref.rotate_bound(part, wt, EPS, table, pos, sections, interleaved, dtype, want)
        assert np.all(err <= bound), f"error over its bound by {float((err / bound).max()):.3f}"
    keep = (slots >= 0) & (slots < caches[0].shape[0] * 16)
    kw, vw = (c.reshape(-1, Hkv, D).copy() for c in caches)
    kw[slots[keep]] = to_bits(k)[keep]
    vw[slots[keep]] = x[:, (Hq + Hkv) * D:(Hq + 2 * Hkv) * D].reshape(T, Hkv, D)[keep]
    assert np.array_equal(to_bits(kc).reshape(kw.shape), kw) and np.array_equal(to_bits(vc).reshape(vw.shape), vw)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("T,Hq,Hkv,D,sections,interleaved", [
    (1, 32, 8, 128, (16, 24, 24), False), (5, 16, 8, 128, (24, 20, 20), True), (64, 28, 4, 64, (12, 10, 10), True),
    (333, 5, 5, 64, (11, 10, 11), False), (17, 1, 1, 128, (1, 62, 1), False), (200, 40, 8, 128, (64,), False),
    (9, 7, 1, 64, (0, 32), False), (31, 2, 2, 128, (20, 16, 14, 14), True), (12, 3, 1, 64, (8, 8, 8, 8), False),
    (700, 64, 8, 128, (22, 21, 21), True), (3, 130, 3, 64, (32, 0, 0), True)])
def test_rotation_by_axes(device, T, Hq, Hkv, D, sections, interleaved, dtype):
    _check(device, T + D, T, Hq, Hkv, D, dtype, sections, interleaved)


@pytest.mark.parametrize("pad", [8, 5])
@pytest.mark.parametrize("weights", [True, False])
def test_row_strides_and_no_norm(device, pad, weights):
    """A row stride of whole 16 bytes and one that leaves the rows unaligned."""
    _check(device, pad, 50, 6, 2, 64, "f16", (12, 10, 10), True, pad, weights)
    _check(device, pad, 50, 6, 2, 128, "bf16", (16, 24, 24), False, pad, weights)


def test_extreme_rows(device):
    """Zeros, one huge element, tiny rows: the mean of squares neither overflows nor vanishes for bf16 rows
    up to 2^60; NaN and infinity stay in their own heads."""
    T, Hq, Hkv, D = 6, 3, 1, 64
    x, w, table, pos, slots, caches = _inputs(0, T, Hq, Hkv, D, "bf16", 2)
    x[0] = 0
    x[1, 5] = oracle.float_to_half(np.array([2.0 ** 60], np.float32), "bf16")[0]
    x[2] = oracle.float_to_half(np.full(x.shape[1], 2.0 ** -40, np.float32), "bf16")
    x[3, 2] = 0x7FC0  # NaN in head 0
    x[4, D + 1] = 0x7F80  # infinity in head 1
    (q, k), kc, vc = _call(device, "bf16", D, Hq, Hkv, x, w, table, pos, (16, 16), caches, slots, return_k=True)
    got = _value(to_bits(q), "bf16")
    val, wq = _value(x.reshape(T, -1, D), "bf16")[:, :Hq], _value(w[0][None], "bf16")[0]
    clean = np.ones((T, Hq), bool)
    clean[3, 0] = clean[4, 1] = False
    with np.errstate(invalid="ignore"):
        want = ref.norm_rotate(val, wq, EPS, table, pos, (16, 16), False)
        bound = ref.rotate_bound(val, wq, EPS, table, pos, (16, 16), False, "bf16", want)
    assert np.all(np.abs(got - want)[clean] <= bound[clean])
    assert np.isnan(got[3, 0]).all() and np.isnan(got[4, 1]).any()


def test_equal_axes_agree_with_the_single_axis_prologue(device):
    """The single-axis entry rounds after norm, weight and rotation: within four half steps of the pair."""
    import torch
    import oxide_paged_kv as ox

    T, Hq, Hkv, D = 77, 8, 2, 128
    x, w, table, pos, slots, caches = _inputs(3, T, Hq, Hkv, D, "bf16", 1)
    (q3, k3), kc, vc = _call(device, "bf16", D, Hq, Hkv, x, w, table, np.repeat(pos, 3, 0), (16, 24, 24), caches, slots,
                             return_k=True)
    t = lambda b: to_torch(b, "bf16", device)  # noqa: E731
    k1c, v1c = t(caches[0]), t(caches[1])
    q1, k1 = ox.qk_norm_rope_and_cache(t(x), Hq, Hkv, t(w[0]), t(w[1]), EPS, torch.from_numpy(table).to(device),
                                       torch.from_numpy(pos[0]).to(device), k1c, v1c, torch.from_numpy(slots).to(device),
                                       return_k=True)
    assert torch.equal(vc, v1c)
    for a, b in ((q3, q1), (k3, k1)):
        a, b = a.double().cpu().numpy(), b.double().cpu().numpy()
        pair = np.hypot(a, np.roll(a, D // 2, -1))
        assert np.all(np.abs(a - b) <= 4 * 2.0 ** -8 * pair + 1e-30)


def test_without_caches_and_into_given_outputs(device):
    import torch

    T, Hq, Hkv, D = 20, 4, 2, 64
    x, w, table, pos, slots, caches = _inputs(5, T, Hq, Hkv, D, "f16", 3)
    args = (device, "f16", D, Hq, Hkv, x, w, table, pos, (12, 10, 10))
    (q, k), kc, _ = _call(*args, caches, slots, return_k=True)
    only_q, none, _ = _call(*args, None, None)
    assert none is None and torch.equal(only_q, q)
    q_out, k_out = torch.zeros_like(q), torch.zeros_like(k)
    (a, b), _, _ = _call(*args, caches, slots, q_out=q_out, k_out=k_out)
    assert a is q_out and b is k_out and torch.equal(a, q) and torch.equal(b, k)


def test_captured_and_on_another_stream(device):
    import torch
    import oxide_paged_kv as ox

    T, Hq, Hkv, D = 40, 8, 4, 128
    x, w, table, pos, slots, caches = _inputs(8, T, Hq, Hkv, D, "bf16", 3)
    t = lambda b: to_torch(b, "bf16", device)  # noqa: E731
    qkv, wq, wk, kc, vc = t(x), t(w[0]), t(w[1]), t(caches[0]), t(caches[1])
    rope, p, s = (torch.from_numpy(a).to(device) for a in (table, pos, slots))
    call = lambda: ox.qk_norm_mrope_and_cache(qkv, Hq, Hkv, wq, wk, EPS, rope, p, (24, 20, 20), kc, vc, s,  # noqa: E731
                                              interleaved=True)
    want = call().clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(3):
        qkv.copy_(t(x).roll(1, 0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())
        qkv.copy_(t(x))
        graph.replay()
        assert torch.equal(out, want)

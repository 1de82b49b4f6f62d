"""Linear attention with a decay per head on the GPU against the recurrence in 64 bits."""
import math

import numpy as np
import pytest

import oracle
import step_reference as ref
from helpers import normal_bits, to_bits, to_torch

pytestmark = pytest.mark.gpu

DTYPES = ["bf16", "f16"]


def _value(bits, dtype):
    return oracle.bits_to_f32(bits.reshape(-1, bits.shape[-1]), dtype).astype(np.float64).reshape(bits.shape)


def _decays(Hkv):
    """No decay, ever faster ones, no memory at all."""
    ld = -np.exp2(-np.linspace(9, 0.5, Hkv)).astype(np.float32)
    if Hkv > 2:
        ld[0], ld[-1] = 0.0, -np.inf
    return ld


class Case:
    """Rows of a merged projection, a pool of states and the calls on them."""

    def __init__(self, device, seed, dtype, D, Hq, Hkv, lens, behind=3, scale=1.0, pool=None, decays=None):
        import torch

        rng = np.random.default_rng(seed)
        self.device, self.dtype, self.D, self.lens = device, dtype, D, np.asarray(lens)
        T = int(self.lens.sum()) + behind
        self.parts = [normal_bits(rng, (T, h, D), dtype, scale) for h in (Hq, Hkv, Hkv)]
        merged = to_torch(np.concatenate(self.parts, 1), dtype, device)
        self.q, self.k, self.v = merged.split([Hq, Hkv, Hkv], 1)
        B = len(self.lens)
        n = pool or B + 2
        self.slots = rng.permutation(n)[:B].astype(np.int32)
        self.ld = _decays(Hkv) if decays is None else np.asarray(decays, np.float32)
        self.start = (4 * rng.standard_normal((n, Hkv, D, D))).astype(np.float32)
        self.ctx = np.where(rng.random(B) < 0.4, 0, 100).astype(np.int32)
        self.scale = 1 / math.sqrt(D)
        self.i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
        self.state = torch.from_numpy(self.start).to(device)
        self.out = torch.full((T, Hq, D), 7.0, dtype=self.q.dtype, device=device)
        self.ld_t = torch.from_numpy(self.ld).to(device)
        self.cu = self.i32(np.concatenate([[0], np.cumsum(self.lens)]))
        self.slots_t, self.ctx_t = self.i32(self.slots), self.i32(self.ctx)

    def prefill(self, with_ctx=True, **kw):
        import oxide_paged_kv as ox

        return ox.linear_attn_prefill(self.q, self.k, self.v, self.ld_t, self.state, self.slots_t, self.cu,
                                      int(self.lens.max(initial=0)), self.scale,
                                      context_lens=self.ctx_t if with_ctx else None, out=self.out, **kw)

    def decode(self):
        import oxide_paged_kv as ox

        return ox.linear_attn_decode(self.q, self.k, self.v, self.ld_t, self.state, self.slots_t, self.scale,
                                     out=self.out)

    def check(self, with_ctx=True, what=""):
        got, state = _value(to_bits(self.out), self.dtype), self.state.double().cpu().numpy()
        q, k, v = (_value(p, self.dtype) for p in self.parts)
        want, s_want, size, s_size = ref.linear_attention(
            q, k, v, self.ld, self.start, self.slots, self.lens, self.scale, self.ctx == 0 if with_ctx else None,
            np.full_like(q, 7.0))
        n = int(self.lens.max(initial=0))
        ref.assert_linear_close(got, want, size, self.dtype, n, f"{what} out")
        ref.assert_linear_close(state, s_want, s_size, "f32", n, f"{what} state")
        # What nothing belongs to is as it was.
        live = np.zeros(self.start.shape[0], bool)
        for s, length in zip(self.slots, self.lens):
            if length and 0 <= s < len(live):
                live[s] = True
        assert np.array_equal(state[~live], self.start[~live].astype(np.float64))
        assert np.all(got[int(self.lens.sum()):] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hq,Hkv,D", [(1, 1, 1, 64), (1, 16, 16, 128), (4, 32, 8, 128), (23, 28, 4, 64), (3, 5, 5, 128),
                                        (2, 34, 2, 64), (70, 8, 8, 64), (40, 32, 8, 128), (64, 32, 32, 128),
                                        (64, 64, 32, 128)])
def test_decode(device, B, Hq, Hkv, D, dtype):
    c = Case(device, B + Hq, dtype, D, Hq, Hkv, [1] * B, behind=0)
    if B > 2:
        c.slots[1], c.slots[2] = -1, c.start.shape[0]  # skipped
        c.slots_t = c.i32(c.slots)
    c.decode()
    c.check(with_ctx=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(3, 3, 128), (8, 4, 64), (7, 1, 128)])
@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [128], [0, 5], [130, 0, 1, 64, 17, 200], [1000]],
                         ids=lambda x: "-".join(map(str, x)))
def test_prefill(device, lens, Hq, Hkv, D, dtype):
    for with_ctx in (True, False):
        c = Case(device, sum(lens) + D + Hq, dtype, D, Hq, Hkv, lens)
        c.prefill(with_ctx)
        c.check(with_ctx, f"{lens}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[4000], [2500, 1, 700, 0, 3000], [3] * 150 + [3000] + [0, 0, 65] * 20 + [1200]],
                         ids=["one", "ragged", "among many"])
def test_prefill_of_long_sequences(device, lens, dtype):
    """Long enough that pieces are worked on side by side, with the workspace and without one."""
    import torch

    for given in (None, torch.empty(1, dtype=torch.uint8, device=device)):
        c = Case(device, len(lens), dtype, 128, 4, 2, lens, decays=[0.0, -0.002])
        c.prefill(workspace=given)
        c.check(what="no workspace" if given is not None else "workspace")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq,Hkv,D", [(20, 4, 128), (7, 1, 64), (33, 3, 64)])
def test_heads_of_a_group_on_several_workgroups(device, Hq, Hkv, D, dtype):
    """Few pieces: a group's query heads are dealt out, not always evenly; short sequences are not cut."""
    c = Case(device, 43, dtype, D, Hq, Hkv, [2000, 70, 500], decays=np.linspace(-0.01, 0, Hkv))
    c.prefill()
    c.check()


@pytest.mark.parametrize("longest", [700, 6000])
def test_a_longest_length_that_is_only_a_bound(device, longest):
    """A captured step's maximum is its rows, whatever the lengths; the rows may begin behind others."""
    import oxide_paged_kv as ox

    c = Case(device, 21, "bf16", 128, 2, 2, [600, 10, 90], behind=6000)
    skip = 77  # rows of nobody
    cu = c.i32(np.concatenate([[0], np.cumsum(c.lens)]) + skip)
    ox.linear_attn_prefill(c.q, c.k, c.v, c.ld_t, c.state, c.slots_t, cu, longest, c.scale, context_lens=c.ctx_t,
                           out=c.out)
    got = _value(to_bits(c.out), "bf16")
    q, k, v = (_value(p, "bf16")[skip:skip + 700] for p in c.parts)
    want, s_want, size, s_size = ref.linear_attention(q, k, v, c.ld, c.start, c.slots, c.lens, c.scale, c.ctx == 0)
    ref.assert_linear_close(got[skip:skip + 700], want, size, "bf16", 600, "out")
    ref.assert_linear_close(c.state.cpu().numpy(), s_want, s_size, "f32", 600, "state")
    assert np.all(got[:skip] == 7.0) and np.all(got[skip + 700:] == 7.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [2.0 ** -10, 2.0 ** 6])
def test_prefill_of_small_and_large_values(device, scale, dtype):
    """Scores and states far from 1: f16 products of three values of 2^6 pass its largest number, those of
    2^-10 lie under its smallest."""
    c = Case(device, 11, dtype, 64, 4, 2, [150, 70], scale=scale, decays=[0.0, -0.05])
    c.start *= np.float32(scale * scale)
    c.state.copy_(__import__("torch").from_numpy(c.start))
    c.scale = 1 / scale / scale
    c.prefill()
    c.check()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_then_tokens_equal_one_prompt(device, dtype):
    """Chunks and single tokens leave the state that one call leaves."""
    import torch
    import oxide_paged_kv as ox

    D, H = 128, 4
    c = Case(device, 2, dtype, D, H, H, [150], behind=0)
    zeros = torch.zeros_like(c.state)
    whole = zeros.clone()
    one = c.i32([1])
    ox.linear_attn_prefill(c.q, c.k, c.v, c.ld_t, whole, one, c.cu, 150, c.scale)
    parts = zeros.clone()
    at = 0
    for n in (70, 1, 64, 13):
        ox.linear_attn_prefill(c.q[at:at + n], c.k[at:at + n], c.v[at:at + n], c.ld_t, parts, one, c.i32([0, n]), n,
                               c.scale)
        at += n
    for t in range(at, 150):
        ox.linear_attn_decode(c.q[t:t + 1], c.k[t:t + 1], c.v[t:t + 1], c.ld_t, parts, one, c.scale)
    q, k, v = (_value(p, dtype) for p in c.parts)
    _, want, _, size = ref.linear_attention(q, k, v, c.ld, zeros.cpu().numpy(), [1], [150], c.scale)
    for got in (whole, parts):
        ref.assert_linear_close(got.cpu().numpy(), want, size, "f32", 150, "state")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("part", [1, 2], ids=["k", "v"])
def test_nothing_reaches_earlier_tokens(device, part, bad, dtype):
    """A NaN or infinity in a token's k or v leaves the tokens before it, other heads and other sequences as they
    are, and reaches the state that it is added to."""
    lens, at = [40, 100, 30], 40 + 37  # token 37 of the second sequence
    bits = {"bf16": {"nan": 0x7FC0, "inf": 0x7F80}, "f16": {"nan": 0x7E00, "inf": 0x7C00}}[dtype][bad]
    c = Case(device, 5, dtype, 64, 4, 2, lens)
    clean = Case(device, 5, dtype, 64, 4, 2, lens)
    c.parts[part][at, 1, 3] = bits
    c.q, c.k, c.v = to_torch(np.concatenate(c.parts, 1), dtype, device).split([4, 2, 2], 1)
    c.prefill()
    clean.prefill()
    got, want = _value(to_bits(c.out), dtype), _value(to_bits(clean.out), dtype)
    assert np.all(np.isfinite(want))
    other = np.ones(got.shape[:2], bool)
    other[at:140, 2:] = False  # kv head 1's query heads, from that token on
    u = ref.HALF_STEP[dtype]
    q, k, v = (_value(p, dtype) for p in clean.parts)
    _, _, size, _ = ref.linear_attention(q, k, v, c.ld, c.start, c.slots, lens, c.scale, c.ctx == 0)
    assert np.all(np.isfinite(got[other]))
    assert np.all(np.abs(got - want)[other] <= (2 * u * np.abs(want) + 3 * u * size)[other])
    cols = slice(None) if part == 1 else 3
    assert not np.isfinite(got[at, 2:, cols]).any()
    state = c.state.cpu().numpy()
    s = c.slots[1]
    assert not np.isfinite(state[s, 1, 3] if part == 1 else state[s, 1, :, 3]).any()
    others = np.arange(len(state)) != s
    assert np.all(np.isfinite(state[others])) and np.all(np.isfinite(state[s, 0]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("bad", [np.inf, np.nan])
def test_other_columns_keep_their_values(device, bad, D, dtype):
    """An infinity or NaN in one value column, of a token's v or of the state before: the others as without it."""
    import torch

    bits = {"bf16": {"inf": 0x7F80, "nan": 0x7FC0}, "f16": {"inf": 0x7C00, "nan": 0x7E00}}[dtype][str(bad)]
    c = Case(device, 41, dtype, D, 2, 1, [150, 90], decays=[-0.01])
    c.ctx[:] = 100
    c.ctx_t = c.i32(c.ctx)
    c.parts[2][70, 0, 5] = bits
    c.start[c.slots[1], 0, :, 9] = bad
    c.q, c.k, c.v = to_torch(np.concatenate(c.parts, 1), dtype, device).split([2, 1, 1], 1)
    c.state.copy_(torch.from_numpy(c.start))
    c.prefill()
    got, state = _value(to_bits(c.out), dtype), c.state.double().cpu().numpy()
    q, k, v = (_value(p, dtype) for p in c.parts)
    with np.errstate(invalid="ignore"):
        want, s_want, size, s_size = ref.linear_attention(q, k, v, c.ld, c.start, c.slots, c.lens, c.scale)
    for rows, column in ((slice(0, 150), 5), (slice(150, 240), 9)):
        rest = np.arange(D) != column
        ref.assert_linear_close(got[rows][..., rest], want[rows][..., rest], size[rows][..., rest], dtype, 150, "out")
    for b, column in enumerate((5, 9)):
        rest, s = np.arange(D) != column, c.slots[b]
        ref.assert_linear_close(state[s][..., rest], s_want[s][..., rest], s_size[s][..., rest], "f32", 150, "state")
    assert not np.isfinite(got[70:150, :, 5]).any() and not np.isfinite(got[150:240, :, 9]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,growth", [([20, 64], 0.4), ([100, 3], 0.1), ([64, 150], 0.05), ([3000], 0.004)], ids=str)
def test_states_that_grow(device, lens, growth, dtype):
    """A decay over 1: weights of up to e^25 in a chunk, of e^12 over pieces; rows padded in front have none."""
    import torch

    c = Case(device, 42, dtype, 128, 2, 2, lens, decays=[growth, 0.0])
    c.start *= np.float32(2.0 ** -6)
    c.state.copy_(torch.from_numpy(c.start))
    c.scale = math.exp(-growth * max(lens)) / 8  # the largest outputs are a few hundred
    c.prefill()
    c.check()


def test_fresh_sequences_do_not_read_their_slots(device):
    c = Case(device, 9, "bf16", 64, 2, 2, [70, 5])
    c.ctx[:] = 0
    c.ctx_t = c.i32(c.ctx)
    c.state[c.slots_t.long()] = float("nan")
    c.prefill()
    c.start[c.slots] = 0
    c.check()


def test_skipped_sequences(device):
    """Slots outside the state: rows and states left as they are."""
    c = Case(device, 4, "bf16", 64, 2, 2, [70, 65, 3, 200])
    c.slots[1], c.slots[3] = -1, c.start.shape[0]
    c.slots_t = c.i32(c.slots)
    c.prefill()
    c.check()


def test_lengths_over_the_maximum_and_the_rows(device):
    """Sequences are cut at max_seqlen_q and at the rows that there are."""
    import oxide_paged_kv as ox

    c = Case(device, 6, "f16", 64, 2, 2, [100, 90], behind=0)
    ox.linear_attn_prefill(c.q, c.k, c.v, c.ld_t, c.state, c.slots_t, c.i32([0, 100, 500]), 95, c.scale,
                           context_lens=c.ctx_t, out=c.out)
    got = _value(to_bits(c.out), "f16")
    q, k, v = (_value(p, "f16") for p in c.parts)
    rows = np.r_[0:95, 100:190]
    want, s_want, size, s_size = ref.linear_attention(q[rows], k[rows], v[rows], c.ld, c.start, c.slots, [95, 90],
                                                      c.scale, c.ctx == 0)
    ref.assert_linear_close(got[rows], want, size, "f16", 95, "out")
    ref.assert_linear_close(c.state.cpu().numpy(), s_want, s_size, "f32", 95, "state")
    assert np.all(got[95:100] == 7.0)


def test_offsets_past_32_bits(device):
    """Rows and state slots whose offsets pass 2^31 elements."""
    import torch
    import oxide_paged_kv as ox

    D, H, T = 64, 4, 2_900_000
    merged = torch.empty(T, 3 * H, D, dtype=torch.bfloat16, device=device)  # 2.2e9 elements
    state = torch.empty(135_000, H, D, D, device=device)  # 2.2e9 elements
    c = Case(device, 8, "bf16", D, H, H, [70], behind=0)
    merged[T - 70:] = torch.cat([c.q, c.k, c.v], 1)
    slot = 134_999
    state[slot] = c.state[c.slots[0]]
    q, k, v = merged.split([H, H, H], 1)
    out = torch.empty(T, H, D, dtype=torch.bfloat16, device=device)
    ox.linear_attn_prefill(q, k, v, c.ld_t, state, c.i32([slot]), c.i32([T - 70, T]), 70, c.scale, out=out)
    c.prefill(with_ctx=False)
    assert torch.equal(out[T - 70:], c.out) and torch.equal(state[slot], c.state[c.slots[0]])
    ox.linear_attn_decode(q[T - 1:], k[T - 1:], v[T - 1:], c.ld_t, state, c.i32([slot]), c.scale)
    ox.linear_attn_decode(c.q[69:], c.k[69:], c.v[69:], c.ld_t, c.state, c.slots_t, c.scale)
    assert torch.equal(state[slot], c.state[c.slots[0]])


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_as_far_apart_as_they_may_be(device, dtype):
    """The last chunk's rows are 2^26 bytes apart: offsets of almost 2^32."""
    import torch
    import oxide_paged_kv as ox

    c = Case(device, 40, dtype, 128, 2, 2, [64 + 61], behind=0)
    far = torch.empty(125, 1 << 25, dtype=c.q.dtype, device=device)
    far[:, :6 * 128] = torch.cat([c.q, c.k, c.v], 1).view(125, -1)
    q, k, v = far[:, :6 * 128].view(125, 6, 128).split([2, 2, 2], 1)
    ox.linear_attn_prefill(q, k, v, c.ld_t, c.state, c.slots_t, c.cu, 125, c.scale, context_lens=c.ctx_t, out=c.out)
    c.check()


def test_captured_calls_replay(device):
    """A captured prompt and a captured token, replayed between eager work: as eager calls from the same state."""
    import torch

    p = Case(device, 12, "bf16", 128, 2, 2, [3000, 40])
    d = Case(device, 13, "bf16", 128, 4, 2, [1] * 5, behind=0)
    for c, call in ((p, p.prefill), (d, d.decode)):
        start = c.state.clone()
        call()
        torch.cuda.synchronize()
        c.state.copy_(start)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        for _ in range(3):
            c.state.copy_(start)
            graph.replay()
            torch.cuda.synchronize()
            out, state = c.out.clone(), c.state.clone()
            c.state.copy_(start)
            call()
            torch.cuda.synchronize()
            assert torch.equal(out[:int(c.lens.sum())], c.out[:int(c.lens.sum())]) and torch.equal(state, c.state)


def test_calls_on_two_streams(device):
    """Calls on two streams at once, each with a workspace of its own, as one after the other."""
    import torch

    cases = [Case(device, 20 + i, "bf16", 128, 2, 2, [2800, 100]) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in cases]
    for c, s in zip(cases, streams):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            c.prefill()
    torch.cuda.synchronize()
    for i, c in enumerate(cases):
        again = Case(device, 20 + i, "bf16", 128, 2, 2, [2800, 100])
        again.prefill()
        assert torch.equal(c.out, again.out) and torch.equal(c.state, again.state)


def test_same_bits_every_time(device):
    import torch

    got = []
    for _ in range(3):
        c = Case(device, 30, "f16", 128, 4, 2, [2500, 77])
        c.prefill()
        got.append((c.out.clone(), c.state.clone()))
    for out, state in got[1:]:
        assert torch.equal(out, got[0][0]) and torch.equal(state, got[0][1])

"""Serving steps as an engine makes them: metadata from request lengths, the multi-axis prologue into the
paged cache, paged attention, and a linear attention layer beside it -- prompts, a mixed step, captured
single-token steps.  Each stage is checked on what the stage before it gave."""
import math

import numpy as np
import pytest

import step_reference as ref
from helpers import assert_attn_close

pytestmark = pytest.mark.gpu

HQ, HKV, LIN, D, BS, MAX_POS, EPS = 8, 2, 4, 128, 16, 2048, 1e-6
SECTIONS = (16, 24, 24)


class Engine:
    """State of a small hybrid model: a paged layer and a linear one, tables and lengths on the device."""

    def __init__(self, device, requests, dtype):
        import torch

        self.device, self.dtype = device, dtype
        g = torch.Generator(device=device).manual_seed(1)
        self.rnd = lambda *s: torch.randn(s, generator=g, device=device).to(dtype)  # noqa: E731
        self.i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
        angle = np.random.default_rng(2).uniform(0, 2 * np.pi, (MAX_POS, D // 2))
        self.rope = torch.from_numpy(np.concatenate([np.cos(angle), np.sin(angle)], 1).astype(np.float32)).to(device)
        self.wq, self.wk = 1 + 0.1 * self.rnd(D), 1 + 0.1 * self.rnd(D)
        blocks = 400
        self.k_cache, self.v_cache = self.rnd(blocks, BS, HKV, D), self.rnd(blocks, BS, HKV, D)
        self.free = np.random.default_rng(3).permutation(blocks).astype(np.int32)
        self.table = self.i32(np.zeros((requests, 40)))
        self.state = torch.full((requests + 2, LIN, D, D), float("nan"), device=device)  # of no request yet
        self.slots = self.i32(np.random.default_rng(4).permutation(requests + 2)[:requests])
        self.log_decay = -torch.tensor([0.0, 0.003, 0.05, 1.0], device=device)
        self.context = np.zeros(requests, np.int64)
        self.offsets = -np.arange(requests) * 3 % 7  # images behind a prompt's token count

    def inputs(self, tokens):
        return self.rnd(tokens, (HQ + 2 * HKV) * D), self.rnd(tokens, 3 * LIN, D)

    def step(self, context, query, free, tokens, longest, qkv, lin, decode):
        """The calls of one step, on device tensors only."""
        import oxide_paged_kv as ox

        scale = 1 / math.sqrt(D)
        cu_q, cu_k, slots, pos, cu_new = ox.build_step_metadata(
            context, query, self.table, free, tokens, BS, position_offsets=self.i32_offsets, num_axes=3)
        q = ox.qk_norm_mrope_and_cache(qkv, HQ, HKV, self.wq, self.wk, EPS, self.rope, pos, SECTIONS, self.k_cache,
                                       self.v_cache, slots)
        lq, lk, lv = lin.split(LIN, 1)
        if decode:
            attn = ox.decode_attn(q, self.k_cache, self.v_cache, cu_k, self.table, longest[1], scale, page_block_size=BS)
            out = ox.linear_attn_decode(lq, lk, lv, self.log_decay, self.state, self.slots, scale)
        else:
            attn = ox.prefill_attn(q, self.k_cache, self.v_cache, cu_q, cu_k, longest[0], longest[1], scale, self.table)
            out = ox.linear_attn_prefill(lq, lk, lv, self.log_decay, self.state, self.slots, cu_q, longest[0], scale,
                                         context_lens=context)
        return cu_q, cu_k, slots, pos, cu_new, q, attn, out


def _f64(t):
    return t.double().cpu().numpy()


def _check_step(e, name, before, query, free, qkv, lin, got):
    """One step's results, stage by stage; `before`: table and states as they were."""
    table, state = before
    cu_q, cu_k, slots, pos, cu_new, q, attn, out = got
    T = qkv.shape[0]
    w_q, w_k, w_slots, w_pos, w_new, w_table = ref.step_metadata(e.context, query, table, free, T, BS, e.offsets)
    for a, b in ((cu_q, w_q), (cu_k, w_k), (slots, w_slots), (cu_new, w_new), (e.table, w_table)):
        assert np.array_equal(a.cpu().numpy(), b)
    assert np.array_equal(pos.cpu().numpy(), np.broadcast_to(w_pos, (3, T)))
    x = _f64(qkv).reshape(T, -1, D)
    rope, positions = e.rope.cpu().numpy(), np.broadcast_to(w_pos, (3, T))
    args = (EPS, rope, positions, SECTIONS, False)
    want = ref.norm_rotate(x[:, :HQ], _f64(e.wq), *args)
    err = np.abs(_f64(q) - want)
    assert np.all(err <= ref.rotate_bound(x[:, :HQ], _f64(e.wq), *args, e.name, want))
    k_rows, v_rows = (_f64(c).reshape(-1, HKV, D) for c in (e.k_cache, e.v_cache))
    want = ref.norm_rotate(x[:, HQ:HQ + HKV], _f64(e.wk), *args)
    err = np.abs(k_rows[w_slots] - want)
    assert np.all(err <= ref.rotate_bound(x[:, HQ:HQ + HKV], _f64(e.wk), *args, e.name, want))
    assert np.array_equal(v_rows[w_slots], x[:, HQ + HKV:])
    # Softmax attention over the pages.
    qd, want = _f64(q), np.zeros((T, HQ, D))
    for b, n in enumerate(query):
        total = int(e.context[b] + n)
        p = np.arange(total)
        rows = w_table[b, p // BS] * BS + p % BS
        for i in range(n):
            t, seen = w_q[b] + i, rows[:e.context[b] + i + 1]
            for h in range(HQ):
                s = k_rows[seen, h // (HQ // HKV)] @ qd[t, h] / math.sqrt(D)
                s = np.exp(s - s.max())
                want[t, h] = s @ v_rows[seen, h // (HQ // HKV)] / s.sum()
    assert_attn_close(attn.float().cpu().numpy(), want)
    # Linear attention.
    lq, lk, lv = (_f64(t) for t in lin.split(LIN, 1))
    start = np.where(np.isnan(state), 0.0, state)
    w_out, w_state, size, s_size = ref.linear_attention(lq, lk, lv, e.log_decay.cpu().numpy(), start, e.slots.cpu().numpy(),
                                                        query, 1 / math.sqrt(D), e.context == 0)
    longest = int(max(query)) + 64
    ref.assert_linear_close(_f64(out), w_out, size, e.name, longest, f"{name} out")
    used = e.slots.cpu().numpy()[(e.context + query) > 0]
    ref.assert_linear_close(_f64(e.state)[used], w_state[used], s_size[used], "f32", longest, f"{name} state")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_serving_steps(device, dtype):
    import torch

    e = Engine(device, 4, torch.bfloat16 if dtype == "bf16" else torch.float16)
    e.name, e.i32_offsets = dtype, e.i32(e.offsets)
    taken = 0
    # Prompts of three requests; then two single tokens, a chunk and a new prompt; then idle ones beside a token.
    for name, query in (("prompts", [70, 1, 33, 0]), ("mixed", [1, 1, 40, 90]), ("mostly idle", [0, 1, 0, 0])):
        query = np.array(query)
        qkv, lin = e.inputs(int(query.sum()))
        free = e.free[taken:]
        before = e.table.cpu().numpy(), _f64(e.state)
        longest = int(query.max()), int((e.context + query).max())
        got = e.step(e.i32(e.context), e.i32(query), e.i32(free), int(query.sum()), longest, qkv, lin, False)
        _check_step(e, name, before, query, free, qkv, lin, got)
        taken += int(got[4][-1])
        e.context += query
    # Single tokens: one captured step, replayed, with eager work in between.
    ones = np.ones(4, np.int64)
    context_t, query_t = e.i32(e.context), e.i32(ones)
    # A captured step takes its blocks from one list: those that it has taken are moved to its end.
    free_t = e.i32(np.resize(e.free[taken:], 300))
    qkv, lin = e.inputs(4)
    longest = (1, int(e.context.max()) + 40)
    saved = [t.clone() for t in (e.table, e.state, e.k_cache, e.v_cache)]
    e.step(context_t, query_t, free_t, 4, longest, qkv, lin, True)
    torch.cuda.synchronize()
    for t, s in zip((e.table, e.state, e.k_cache, e.v_cache), saved):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = e.step(context_t, query_t, free_t, 4, longest, qkv, lin, True)
    for i in range(20):
        new_qkv, new_lin = e.inputs(4)
        qkv.copy_(new_qkv)
        lin.copy_(new_lin)
        before = e.table.cpu().numpy(), _f64(e.state)
        free = free_t.cpu().numpy()
        graph.replay()
        torch.cuda.synchronize()
        _check_step(e, f"token {i}", before, ones, free, qkv, lin, got)
        used = int(got[4][-1])
        free_t.copy_(free_t.roll(-used))
        e.context += ones
        context_t.copy_(e.i32(e.context))


@pytest.mark.parametrize("general", [False, True], ids=["native", "general"])
def test_front_ends_agree(device, general, monkeypatch):
    """The native front end takes the calls of a step; the general code gives the same bits."""
    import torch
    import oxide_paged_kv as ox
    from oxide_paged_kv import ops

    results = []
    taken = []
    native = ops._native

    class Front:
        def __init__(self, decline):
            self.decline = decline

        def __getattr__(self, name):
            def call(*args):
                r = None if self.decline else getattr(native, name)(*args)
                taken.append((name, r is not None))
                return r
            return call

    for decline in (general, True):
        monkeypatch.setattr(ops, "_native", Front(decline))
        e = Engine(device, 3, torch.bfloat16)
        e.i32_offsets = e.i32(e.offsets)
        query = np.array([20, 5, 300])
        qkv, lin = e.inputs(325)
        a = e.step(e.i32(e.context), e.i32(query).view(torch.uint32), e.i32(e.free), 325, (300, 300), qkv, lin, False)
        qkv, lin = e.inputs(3)
        b = e.step(e.i32(query), e.i32([1, 1, 1]), e.i32(e.free[100:]), 3, (1, 301), qkv, lin, True)
        results.append([*a, *b, e.table, e.state, e.k_cache, e.v_cache])
    mine = ("step_metadata", "mrope", "linear_prefill", "linear_decode")
    first = [x for x in taken[:len(taken) // 2] if x[0] in mine]
    assert len(first) == 6 and all(took is not general for _, took in first)
    for x, y in zip(*results):
        assert x.dtype == y.dtype and x.shape == y.shape
        assert torch.equal(torch.nan_to_num(x.float(), 7.5), torch.nan_to_num(y.float(), 7.5))
    del ox

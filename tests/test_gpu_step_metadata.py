"""build_step_metadata on the GPU against the request-by-request restatement: whole numbers, equal."""
import numpy as np
import pytest

import step_reference as ref

pytestmark = pytest.mark.gpu


def _case(seed, B, bs, max_ctx, max_new, spare=5, width_extra=1, idle=0.2):
    rng = np.random.default_rng(seed)
    ctx = rng.integers(0, max_ctx + 1, B)
    new = np.where(rng.random(B) < idle, 0, rng.integers(0, max_new + 1, B))
    ctx[rng.random(B) < 0.2] = 0
    need = -(-(ctx + new) // bs)
    width = max(1, int(need.max()) + width_extra)
    table = rng.integers(0, 10 ** 6, (B, width)).astype(np.int32)  # stale entries behind those held
    free = rng.permutation(10 ** 6)[:int((need - -(-ctx // bs)).sum()) + spare].astype(np.int32)
    offsets = rng.integers(-2000, 2000, B).astype(np.int32)
    return ctx, new, table, free, offsets


def _run(device, ctx, new, table, free, tokens, bs, offsets=None, axes=None, u32=False):
    import torch
    import oxide_paged_kv as ox

    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
    lens = lambda a: t(a).view(torch.uint32) if u32 else t(a)  # noqa: E731
    tab = t(table)
    r = ox.build_step_metadata(lens(ctx), lens(new), tab, None if free is None else t(free), tokens, bs,
                               position_offsets=None if offsets is None else t(offsets), num_axes=axes)
    return [x.cpu().numpy() for x in r] + [tab.cpu().numpy()]


def _check(got, ctx, new, table, free, tokens, bs, offsets=None, axes=None):
    want = ref.step_metadata(ctx, new, table, [] if free is None else free, tokens, bs, offsets)
    cu_q, cu_k, slots, positions, cu_new, tab = got
    assert np.array_equal(cu_q.view(np.uint32), want[0]) and np.array_equal(cu_k.view(np.uint32), want[1])
    assert slots.dtype == np.int64 and np.array_equal(slots, want[2])
    assert positions.shape == ((tokens,) if axes is None else (axes, tokens))
    assert np.array_equal(positions.reshape(axes or 1, tokens), np.broadcast_to(want[3], (axes or 1, tokens)))
    assert np.array_equal(cu_new.view(np.uint32), want[4])
    assert np.array_equal(tab, want[5])


@pytest.mark.parametrize("B,bs,max_ctx,max_new,axes", [
    (1, 256, 5000, 1, None), (1, 16, 0, 700, 3), (64, 256, 8192, 1, 1), (63, 16, 300, 40, None), (257, 64, 1000, 70, 3),
    (1024, 16, 500, 30, 2), (1025, 16, 500, 30, None), (3000, 24, 400, 9, 4), (5, 1, 30, 9, None)])
@pytest.mark.parametrize("fit", ["exact", "spare rows", "short"])
def test_step_metadata(device, B, bs, max_ctx, max_new, axes, fit):
    ctx, new, table, free, offsets = _case(B + bs, B, bs, max_ctx, max_new)
    tokens = int(new.sum())
    tokens = tokens + 37 if fit == "spare rows" else tokens - tokens // 3 if fit == "short" else tokens
    off = offsets if axes else None
    _check(_run(device, ctx, new, table, free, tokens, bs, off, axes, u32=B % 2 == 0), ctx, new, table, free, tokens,
           bs, off, axes)


@pytest.mark.parametrize("B", [7, 1500])
@pytest.mark.parametrize("left", [0, 1, 9, 40])
def test_free_list_that_ends_inside_the_step(device, B, left):
    """Requests behind the list's end take nothing: no slot in a block they do not have, entries left alone."""
    ctx, new, table, free, _ = _case(B + left, B, 16, 100, 60)
    free = free[:left] if left else None
    tokens = int(new.sum())
    _check(_run(device, ctx, new, table, free, tokens, 16), ctx, new, table, free, tokens, 16)


def test_tokens_past_the_table(device):
    """A request longer than its row: the tokens past it have no slot, its blocks end with the row."""
    ctx, new = np.array([30, 0, 64]), np.array([40, 100, 8])
    table = np.arange(12, dtype=np.int32).reshape(3, 4) + 50
    free = np.arange(20, dtype=np.int32)
    _check(_run(device, ctx, new, table, free, 148, 16), ctx, new, table, free, 148, 16)


def test_nothing_to_do(device):
    for ctx, new, tokens in (([], [], 0), ([], [], 5), ([7, 0], [0, 0], 3)):
        ctx, new = np.array(ctx, np.int64), np.array(new, np.int64)
        table, free = np.full((len(ctx), 2), 9, np.int32), np.arange(3, dtype=np.int32)
        _check(_run(device, ctx, new, table, free, tokens, 16), ctx, new, table, free, tokens, 16)


def test_lengths_near_32_bits(device):
    """Positions past 2^31 and sums past 2^32: slots in 64 bits, prefix sums modulo 2^32."""
    ctx, new = np.array([2 ** 32 - 5, 2 ** 31, 3], np.uint32), np.array([3, 2, 4], np.uint32)
    bs = 1 << 22
    table = np.arange(3 * 1025, dtype=np.int32).reshape(3, 1025)
    free = np.arange(5000, 5004, dtype=np.int32)
    cu_q, cu_k, slots, positions, cu_new, tab = _run(device, ctx.view(np.int32), new.view(np.int32), table, free, 9, bs)
    want = ref.step_metadata(ctx, new, table, free, 9, bs)
    assert np.array_equal(cu_q, want[0]) and np.array_equal(cu_k.view(np.uint32), want[1].astype(np.uint32))
    assert np.array_equal(slots, want[2]) and np.array_equal(positions, want[3].astype(np.uint32).view(np.int32))
    assert np.array_equal(cu_new, want[4]) and np.array_equal(tab, want[5])


def test_captured_step_replays(device):
    """A captured call follows its inputs' values; eager work runs between the replays."""
    import torch
    import oxide_paged_kv as ox

    B, bs, tokens = 40, 16, 500
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(device)  # noqa: E731
    ctx_t, new_t, table_t, free_t = t(np.zeros(B)), t(np.zeros(B)), t(np.zeros((B, 20))), t(np.zeros(200))
    call = lambda: ox.build_step_metadata(ctx_t, new_t, table_t, free_t, tokens, bs)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for seed in range(4):
        ctx, new, table, free, _ = _case(seed, B, bs, 200, 20)
        table, free = np.resize(table, (B, 20)).astype(np.int32), np.resize(free, 200).astype(np.int32)
        for dst, src in ((ctx_t, ctx), (new_t, new), (table_t, table), (free_t, free)):
            dst.copy_(t(src))
        graph.replay()
        torch.cuda.synchronize()
        _check([x.cpu().numpy() for x in out] + [table_t.cpu().numpy()], ctx, new, table, free, tokens, bs)
        call()  # the same table again: nothing changes
        torch.cuda.synchronize()
        assert np.array_equal(table_t.cpu().numpy(), ref.step_metadata(ctx, new, table, free, tokens, bs)[5])


def test_decode_step_agrees_with_decode_metadata(device):
    """One new token each, tables complete: the slots of build_decode_metadata."""
    import torch
    import oxide_paged_kv as ox

    rng = np.random.default_rng(0)
    ctx = rng.integers(1, 999, 33)
    table = rng.integers(0, 4000, (33, 64)).astype(np.int32)
    ctx = np.where(ctx % 16 == 0, ctx + 1, ctx)  # the new token's block is held
    cu_q, cu_k, slots, positions, cu_new, tab = _run(device, ctx, np.ones(33), table, None, 33, 16)
    t = torch.from_numpy(table).to(device)
    cu, want = ox.build_decode_metadata(torch.from_numpy((ctx + 1).astype(np.int32)).to(device), t, 16)
    assert np.array_equal(cu_k, cu.cpu().numpy()) and np.array_equal(slots, want.cpu().numpy())
    assert np.array_equal(positions, ctx) and not cu_new.any() and np.array_equal(tab, table)

"""Refusals of step metadata, the multi-axis prologue and linear attention: C error codes without a
launch, and the Python checks (which come before the device check, so host tensors show them)."""
import ctypes

import pytest
import torch

import oxide_paged_kv as ox
from oxide_paged_kv import _lib

INVALID, DTYPE, SHAPE = 1, 2, 3
P = [ctypes.c_void_p(1 << 20 | i << 32) for i in range(1, 12)]  # aligned addresses, 4 GB apart; never read


def _code(name, *args):
    L = _lib.load()
    L.oxide_clear_error()
    getattr(L, name)(*args)
    code = L.oxide_last_error()
    L.oxide_clear_error()
    return code


def _metadata(batch=2, width=4, free=3, block=16, tokens=8, axes=1, context=P[0], cu=P[6], table=P[3], positions=P[10],
              free_list=P[4], slots=P[9]):
    return _code("build_step_metadata_device", context, P[1], None, table, width, free_list, free, batch, block, tokens,
                 axes, cu, P[7], P[8], slots, positions, None)


@pytest.mark.parametrize("change", [
    {"batch": -1}, {"batch": 65536}, {"width": -1}, {"batch": 60000, "width": 40000}, {"width": 1 << 31}, {"free": -1},
    {"block": 0}, {"block": 1 << 31}, {"tokens": -1}, {"tokens": 1 << 31}, {"axes": 0}, {"axes": 5}, {"context": None},
    {"cu": None}, {"table": None}, {"free_list": None}, {"slots": None}], ids=str)
def test_step_metadata_refuses(change):
    assert _metadata(**change) == INVALID


def _mrope(q_out=P[0], k_out=None, qkv=P[2], stride=6 * 128, rope=P[3], max_pos=10, pos=P[4], sections=(16, 24, 24),
           axes=None, dealt=0, kc=P[5], vc=P[6], slots=32, sm=P[7], T=3, Hq=4, Hkv=1, D=128, dtype=1):
    s = None if sections is None else (ctypes.c_int32 * len(sections))(*sections)
    return _code("qk_norm_mrope_and_cache", q_out, k_out, qkv, stride, None, None, 1e-6, rope, max_pos, pos,
                 len(sections or ()) if axes is None else axes, None if s is None else ctypes.addressof(s), dealt, kc, vc,
                 slots, sm, T, Hq, Hkv, D, dtype, None)


@pytest.mark.parametrize("change,code", [
    ({"dtype": 2}, DTYPE), ({"dtype": 9}, DTYPE), ({"D": 96}, SHAPE), ({"D": 256}, SHAPE), ({"T": -1}, INVALID),
    ({"T": 1 << 26}, INVALID), ({"Hq": 0}, INVALID), ({"Hkv": 0}, INVALID), ({"stride": 6 * 128 - 1}, INVALID),
    ({"max_pos": 0}, INVALID), ({"sections": None, "axes": 3}, INVALID), ({"axes": 0}, INVALID),
    ({"sections": (16, 16, 16, 8, 8)}, INVALID), ({"sections": (16, 24, 23)}, INVALID),
    ({"sections": (65, -1, 0)}, INVALID), ({"sections": (1 << 30, 1 << 30, 64)}, INVALID),
    ({"sections": (10, 32, 22), "dealt": 1}, INVALID), ({"slots": -1}, INVALID), ({"q_out": None}, INVALID),
    ({"qkv": None}, INVALID), ({"rope": None}, INVALID), ({"pos": None}, INVALID), ({"kc": None}, INVALID),
    ({"vc": None}, INVALID), ({"q_out": P[2]}, INVALID), ({"k_out": P[2]}, INVALID)], ids=str)
def test_prologue_refuses(change, code):
    assert _mrope(**change) == code


def test_prologue_of_nothing():
    assert _mrope(T=0) == 0


def _decode(out=P[0], q=P[1], k=P[2], v=P[3], sq=256, sk=128, sv=128, ld=P[4], state=P[5], slots=P[6], n=4, B=2, Hq=2,
            Hkv=1, D=128, dtype=1):
    return _code("linear_attention_decode", out, q, k, v, sq, sk, sv, ld, state, slots, n, B, Hq, Hkv, D, 0.1, dtype, None)


def _prefill(out=P[0], q=P[1], k=P[2], v=P[3], sq=256, sk=128, sv=128, ld=P[4], state=P[5], slots=P[6], n=4, B=2, Hq=2,
             Hkv=1, D=128, dtype=1, cu=P[7], T=9, longest=5):
    return _code("linear_attention_prefill", out, q, k, v, sq, sk, sv, ld, state, slots, None, cu, n, T, B, Hq, Hkv, D,
                 longest, 0.1, None, 0, dtype, None)


@pytest.mark.parametrize("call", [_decode, _prefill])
@pytest.mark.parametrize("change,code", [
    ({"dtype": 2}, DTYPE), ({"dtype": -1}, DTYPE), ({"D": 32}, SHAPE), ({"D": 256}, SHAPE), ({"B": -1}, INVALID),
    ({"B": 65536}, INVALID), ({"Hq": 0}, INVALID), ({"Hkv": 0}, INVALID), ({"Hq": 3, "Hkv": 2}, INVALID),
    ({"Hq": 4097}, INVALID), ({"n": -1}, INVALID), ({"sq": 255}, INVALID), ({"sq": 260}, INVALID),
    ({"sk": 120}, INVALID), ({"sv": 132}, INVALID), ({"q": None}, INVALID), ({"k": None}, INVALID),
    ({"v": None}, INVALID), ({"out": None}, INVALID), ({"state": None}, INVALID), ({"ld": None}, INVALID),
    ({"slots": None}, INVALID), ({"q": ctypes.c_void_p(P[1].value + 8)}, INVALID),
    ({"state": ctypes.c_void_p(P[5].value + 4)}, INVALID), ({"out": P[1]}, INVALID), ({"out": P[2]}, INVALID),
    ({"out": P[3]}, INVALID)], ids=str)
def test_linear_attention_refuses(call, change, code):
    assert call(**change) == code


@pytest.mark.parametrize("call", [_decode, _prefill])
@pytest.mark.parametrize("stride", ["sq", "sk", "sv"])
def test_linear_attention_refuses_rows_too_far_apart(call, stride):
    """64 rows' offsets in bytes have to fit 32 bits."""
    far = ctypes.c_void_p(1 << 46)  # not between the rows
    assert call(out=far, **{stride: (1 << 25) + 8}) == INVALID


def test_prefill_refuses():
    assert _prefill(cu=None) == INVALID and _prefill(T=-1) == INVALID and _prefill(longest=-1) == INVALID


def test_linear_attention_of_nothing():
    assert _decode(B=0) == 0 and _prefill(B=0) == 0 and _prefill(T=0) == 0 and _prefill(longest=0) == 0


def test_workspace_size_of_refused_arguments_is_zero():
    for args in ((-1, 1, 1, 1, 128, 9), (9, -1, 1, 1, 128, 9), (9, 1, 3, 2, 128, 9), (9, 1, 1, 0, 128, 9),
                 (9, 1, 1, 1, 100, 9), (9, 1, 1, 1, 128, -9), (0, 1, 1, 1, 128, 0)):
        assert ox.linear_workspace_size(*args) == 0


def _raises(call, text):
    with pytest.raises(ox.OxideError, match=text):
        call()


def test_python_step_metadata_refuses():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    call = lambda ctx=i(2), new=i(2), table=i(2, 3), free=i(4), n=5, **kw: ox.build_step_metadata(  # noqa: E731
        ctx, new, table, free, n, 16, **kw)
    _raises(lambda: call(ctx=i(2).long()), "32-bit")
    _raises(lambda: call(new=i(3)), "32-bit")
    _raises(lambda: call(table=i(3, 3)), "block_table")
    _raises(lambda: call(table=i(2, 3).long()), "block_table")
    _raises(lambda: call(free=i(4).long()), "free_blocks")
    _raises(lambda: call(position_offsets=i(3)), "position_offsets")
    _raises(lambda: call(n=-1), "num_tokens")
    _raises(lambda: call(num_axes=0), "num_axes")
    _raises(lambda: call(num_axes=5), "num_axes")
    _raises(call, "device tensor")


def test_python_prologue_refuses():
    h = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    base = {"qkv": h(5, 6 * 64), "num_heads": 4, "num_kv_heads": 1, "q_norm_weight": h(64), "k_norm_weight": h(64),
            "eps": 1e-6, "cos_sin_cache": torch.zeros(9, 64), "positions": torch.zeros(3, 5, dtype=torch.int32),
            "sections": (12, 10, 10), "key_cache": h(2, 16, 1, 64), "value_cache": h(2, 16, 1, 64),
            "slot_mapping": torch.zeros(5, dtype=torch.int64)}
    call = lambda **kw: ox.qk_norm_mrope_and_cache(**{**base, **kw})  # noqa: E731
    _raises(lambda: call(qkv=h(5, 5 * 64)), "shorter")
    _raises(lambda: call(qkv=h(6 * 64, 5).t()), "unit element stride")
    _raises(lambda: call(positions=torch.zeros(2, 5, dtype=torch.int32)), "positions")
    _raises(lambda: call(positions=torch.zeros(3, 4, dtype=torch.int32)), "positions")
    _raises(lambda: call(positions=torch.zeros(3, 5)), "positions")
    _raises(lambda: call(q_norm_weight=h(32)), "q_norm_weight")
    _raises(lambda: call(k_norm_weight=torch.zeros(64)), "k_norm_weight")
    _raises(lambda: call(slot_mapping=torch.zeros(5, dtype=torch.int32)), "slot_mapping")
    _raises(lambda: call(slot_mapping=torch.zeros(4, dtype=torch.int64)), "slot_mapping")
    _raises(lambda: call(slot_mapping=None), "together")
    _raises(lambda: call(key_cache=None), "together")
    _raises(lambda: call(value_cache=h(2, 16, 2, 64)), "value_cache")
    _raises(lambda: call(key_cache=torch.zeros(2, 16, 1, 64)), "key_cache")
    _raises(lambda: call(q_out=h(5, 3, 64)), "q_out")
    _raises(call, "device tensor")


def test_python_linear_attention_refuses():
    h = lambda *s: torch.zeros(s, dtype=torch.float16)  # noqa: E731
    i = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    base = {"q": h(5, 4, 64), "k": h(5, 2, 64), "v": h(5, 2, 64), "log_decay": torch.zeros(2),
            "state": torch.zeros(6, 2, 64, 64), "state_slots": i(5), "scale": 0.1}
    decode = lambda **kw: ox.linear_attn_decode(**{**base, **kw})  # noqa: E731
    prefill = lambda **kw: ox.linear_attn_prefill(**{**base, "state_slots": i(2), "cu_seqlens_q": i(3),  # noqa: E731
                                                     "max_seqlen_q": 5, **kw})
    for call in (decode, prefill):
        _raises(lambda: call(k=h(4, 2, 64)), "expected")
        _raises(lambda: call(v=h(5, 4, 64)), "expected")
        _raises(lambda: call(q=h(5, 3, 64)), "multiple")
        _raises(lambda: call(k=h(5, 2, 64).bfloat16()), "dtype")
        _raises(lambda: call(log_decay=torch.zeros(3)), "log_decay")
        _raises(lambda: call(log_decay=torch.zeros(2).double()), "log_decay")
        _raises(lambda: call(state=torch.zeros(6, 2, 64, 32)), "state")
        _raises(lambda: call(state=h(6, 2, 64, 64)), "state")
        _raises(lambda: call(state_slots=i(4)), "state_slots")
        _raises(lambda: call(out=h(5, 4, 32)), "out")
        _raises(call, "device tensor")
    _raises(lambda: prefill(cu_seqlens_q=i(3).long()), "cu_seqlens_q")
    _raises(lambda: prefill(context_lens=i(3)), "context_lens")

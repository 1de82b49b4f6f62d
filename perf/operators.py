"""Timed cases of a serving step's further operators: metadata from request lengths, the prologue with positions on
several axes, and linear attention with a decay for each head (prompts and single tokens).

A case is a dict of plain values.  Lengths and head layouts belong to the case, so that its work is known without a
seed; values, page orders, image sizes and state slots come from the seed.  `own` false: the operators in elementary
torch operations, in 32 bits; true: the calls a user makes of `oxide_paged_kv`.
"""
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16}
_EPS = 1e-6
_MAX_POSITION = 40960
_DEVICE = "cuda:0"

# Query heads, kv heads of the attention layers that the repository's benchmark configurations and header name.
_HEADS = ((16, 8), (32, 8), (40, 8), (64, 8), (28, 4))
# Heads of linear attention layers: a state for each head, or one that a group of query heads shares.
_LINEAR_HEADS = ((16, 16), (32, 32), (8, 8), (32, 8), (28, 4), (40, 8), (5, 5))


_imported = None


def _package():
    """The framework's package, imported at the first call: its parent folder is not a package itself."""
    global _imported
    if _imported is None:
        parent = str(Path.cwd() / "vllm-oxide_amd")
        if parent not in sys.path:
            sys.path.insert(0, parent)
        import oxide_paged_kv
        _imported = oxide_paged_kv
    return _imported


def _metadata(name, batch, new_lo, new_hi, ctx_lo, ctx_hi, page, axes=1):
    return {"name": name, "kind": "metadata", "batch": batch, "new_lo": new_lo, "new_hi": new_hi, "ctx_lo": ctx_lo,
            "ctx_hi": ctx_hi, "page": page, "axes": axes}


def _prologue(name, tokens, heads, kv_heads, dim, dtype, sections, interleaved, page):
    return {"name": name, "kind": "prologue", "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "time": sections[0], "height": sections[1], "width": sections[2],
            "interleaved": interleaved, "page": page}


def _decode(name, batch, heads, kv_heads, dim, dtype):
    return {"name": name, "kind": "linear_decode", "batch": batch, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype}


def _prefill(name, batch, lo, hi, heads, kv_heads, dim, dtype, fresh):
    return {"name": name, "kind": "linear_prefill", "batch": batch, "lo": lo, "hi": hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "fresh": fresh}


def listed():
    return [
        # The metadata of a decode step: one new token for each of 64 requests.
        _metadata("metadata_decode_b64", 64, 1, 1, 2048, 8192, 256),
        # A large mixed step over small pages: whole prompts, chunks and single tokens, positions on three axes.
        _metadata("metadata_mixed_b700", 700, 1, 180, 0, 4000, 16, axes=3),
        # The prologue of a decode step of an image-and-text model, 64 requests.
        _prologue("prologue_decode_b64", 64, 32, 8, 128, "bf16", (16, 24, 24), False, 256),
        # Prompts with images: the prologue's largest pass.
        _prologue("prologue_images_16k", 16384, 32, 8, 128, "bf16", (16, 24, 24), False, 256),
        # Small heads in f16, frequencies dealt to the axes in turn, an odd number of tokens, small pages.
        _prologue("prologue_f16_interleaved", 1777, 28, 4, 64, "f16", (12, 10, 10), True, 16),
        # One token each for four users, a state for each head: the smallest decode call of a linear layer.
        _decode("linear_decode_b4", 4, 16, 16, 128, "bf16"),
        # The serving batch: 256 MB of state read and written.
        _decode("linear_decode_b64", 64, 32, 32, 128, "bf16"),
        # An odd batch in f16, seven query heads on a state, small heads.
        _decode("linear_decode_f16_grouped", 23, 28, 4, 64, "f16"),
        # A short prompt of one user: latency.
        _prefill("linear_prefill_1x100", 1, 100, 100, 16, 16, 128, "bf16", True),
        # One long prompt: few rows, so the work is split over its length.
        _prefill("linear_prefill_1x8192", 1, 8192, 8192, 32, 32, 128, "bf16", True),
        # Chunks of many prompts behind earlier ones, ragged, grouped heads.
        _prefill("linear_prefill_ragged", 16, 1, 1500, 32, 8, 128, "bf16", False),
        # The largest: prompts in full, f16.
        _prefill("linear_prefill_4x4096_f16", 4, 4096, 4096, 32, 32, 128, "f16", True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("metadata", "prologue", "linear_decode", "linear_prefill", "linear_prefill"))
    dim = rng.choice((128, 128, 64))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    case = {"kind": kind}
    if kind == "metadata":
        batch = _log_int(rng, 1, 700)
        new_hi = min(_log_int(rng, 1, 8192), 63000 // batch)
        case.update(batch=batch, new_lo=rng.choice((1, max(1, new_hi // 2))), new_hi=new_hi, ctx_lo=0,
                    ctx_hi=_log_int(rng, 1, 8192), page=rng.choice((256, 64, 16)), axes=rng.choice((1, 3)))
    elif kind == "prologue":
        heads, kv_heads = rng.choice(_HEADS)
        interleaved = rng.random() < 0.5
        # Dealt in turn, height and width hold at most a third of the frequencies; in runs, any share.
        most = dim // 6 if interleaved else dim // 2 - 2
        height = rng.randint(1, most)
        width = rng.randint(1, min(most, dim // 2 - height - 1))
        # At most the listed 16k prompt's rows.
        tokens = _log_int(rng, 1, min(16384, 16384 * 48 * 128 // ((heads + 2 * kv_heads) * dim)))
        case.update(tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                    time=dim // 2 - height - width, height=height, width=width, interleaved=interleaved,
                    page=rng.choice((256, 64, 16)))
    else:
        heads, kv_heads = rng.choice(_LINEAR_HEADS)
        case.update(heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype)
        if kind == "linear_decode":
            # At most the listed serving batch's state.
            case.update(batch=_log_int(rng, 1, min(200, 64 * 32 * 128 * 128 // (kv_heads * dim * dim))))
        else:
            batch = _log_int(rng, 1, 24)
            # At most the listed largest prompts' rows in total.
            hi = _log_int(rng, 1, min(16384, 16384 * 64 // (batch * (heads + kv_heads))))
            case.update(batch=batch, lo=max(1, int(hi * rng.choice((0.05, 0.5, 1.0)))), hi=hi,
                        fresh=rng.random() < 0.5)
    return case


def _lengths(lo, hi, n, salt):
    """n lengths in [lo, hi] with both ends among them, the same for every seed."""
    r = np.random.default_rng([salt, lo, hi, n])
    out = r.integers(lo, hi, size=n, endpoint=True)
    out[0] = hi
    if n > 1:
        out[n // 2] = lo
    return out


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=_DEVICE) * scale).to(dtype)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(_DEVICE)


def _cu(lens):
    return _i32(np.concatenate([[0], np.cumsum(lens)]))


# ------------------------------------------------------------------------------------------------ metadata


def _metadata_lens(case):
    return (_lengths(case["ctx_lo"], case["ctx_hi"], case["batch"], 1),
            _lengths(case["new_lo"], case["new_hi"], case["batch"], 2))


def _prepare_metadata(case, seed):
    r = np.random.default_rng([seed, 3])
    ctx, new = _metadata_lens(case)
    page = case["page"]
    held, need = -(-ctx // page), -(-(ctx + new) // page)
    taken = int(need.sum() - held.sum())
    ids = r.permutation(int(need.sum()) + 64).astype(np.int32)  # a pool with 64 blocks to spare
    table = np.zeros((case["batch"], int(need.max()) + 1), np.int32)
    at = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[at:at + n]
        at += n
    # Images make a request's positions run behind its token count.
    offsets = -r.integers(0, ctx + 1).astype(np.int32) if case["axes"] > 1 else None
    # A captured step has room for a fixed number of tokens: the last rows belong to no request.
    return {"context_lens": _i32(ctx), "query_lens": _i32(new), "table": _i32(table),
            "free": _i32(ids[at:at + taken + 64]), "tokens": (int(new.sum()) + 63) // 64 * 64, "page": page,
            "axes": case["axes"] if case["axes"] > 1 else None,
            "offsets": None if offsets is None else _i32(offsets)}


def _plain_metadata(s):
    ctx, new, page = s["context_lens"].long(), s["query_lens"].long(), s["page"]
    table, free, tokens = s["table"], s["free"], s["tokens"]
    zero = ctx.new_zeros(1)
    prefix = lambda x: torch.cat([zero, x.cumsum(0)])  # noqa: E731
    cu_q, cu_k = prefix(new), prefix(ctx + new)
    width = table.shape[1]
    held = ((ctx + page - 1) // page).clamp(max=width)
    need = ((ctx + new + page - 1) // page).clamp(max=width)
    cu_new = prefix(need - held)
    served = (need == held) | (cu_new[1:] <= free.shape[0])
    j = torch.arange(width, device=ctx.device)[None]
    takes = (j >= held[:, None]) & (j < need[:, None]) & served[:, None]
    at = (cu_new[:-1, None] + j - held[:, None]).clamp(0, free.shape[0] - 1)
    table.copy_(torch.where(takes, free[at], table))
    t = torch.arange(tokens, device=ctx.device)
    b = torch.searchsorted(cu_q[1:], t, right=True).clamp(max=ctx.shape[0] - 1)
    real = t < cu_q[-1]
    pos = ctx[b] + t - cu_q[b]
    block = pos // page
    ok = real & (block < width) & ((block < held[b]) | served[b])
    slot = torch.where(ok, table[b, block.clamp(max=width - 1)].long() * page + pos % page, -1)
    if s["offsets"] is not None:
        pos = pos + s["offsets"][b]
    pos = torch.where(real, pos, 0).int()
    if s["axes"] is not None:
        pos = pos[None].expand(s["axes"], tokens).contiguous()
    return {"cu_seqlens_q": cu_q.int(), "cu_seqlens_k": cu_k.int(), "slot_mapping": slot, "positions": pos,
            "cu_new_blocks": cu_new.int(), "block_table": table}


def _own_metadata(s):
    cu_q, cu_k, slots, positions, cu_new = _package().build_step_metadata(
        s["context_lens"], s["query_lens"], s["table"], s["free"], s["tokens"], s["page"],
        position_offsets=s["offsets"], num_axes=s["axes"])
    return {"cu_seqlens_q": cu_q, "cu_seqlens_k": cu_k, "slot_mapping": slots, "positions": positions,
            "cu_new_blocks": cu_new, "block_table": s["table"]}


# ------------------------------------------------------------------------------------------------ prologue


def _rope_table(dim):
    """cos | sin of position * 10^6^(-2 j / dim), rounded from 64 bits."""
    f = 1e6 ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device=_DEVICE) / dim)
    a = torch.arange(_MAX_POSITION, dtype=torch.float64, device=_DEVICE)[:, None] * f
    return torch.cat([a.cos(), a.sin()], 1).float()


def _image_positions(r, tokens):
    """Positions on three axes of text with images in between: text counts up on all three; an image's patches share
    a time and have their row and column; the text behind it goes on after its larger side."""
    out = np.zeros((3, tokens), np.int32)
    at, p = 0, int(r.integers(0, 2000))
    while at < tokens:
        n = min(tokens - at, int(r.integers(1, 300)))
        out[:, at:at + n] = p + np.arange(n)
        at, p = at + n, p + n
        h, w = (int(x) for x in r.integers(4, 40, size=2))
        n = min(tokens - at, h * w)
        i = np.arange(n)
        out[:, at:at + n] = p + np.stack([np.zeros(n, np.int64), i // w, i % w])
        at, p = at + n, p + max(h, w)
    return out


def _prepare_prologue(case, seed):
    r = np.random.default_rng([seed, 4])
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    t, heads, kv_heads, dim, page = (case[k] for k in ("tokens", "heads", "kv_heads", "dim", "page"))
    dtype = _DTYPE[case["dtype"]]
    blocks = -(-t // page)
    pages = r.permutation(blocks + 2)[:blocks]
    i = np.arange(t)
    slots = pages[i // page].astype(np.int64) * page + i % page
    cache = lambda: _randn(g, (blocks + 2, page, kv_heads, dim), dtype)  # noqa: E731
    return {"qkv": _randn(g, (t, (heads + 2 * kv_heads) * dim), dtype, 2.0), "heads": heads, "kv_heads": kv_heads,
            "q_weight": (1 + _randn(g, (dim,), torch.float32, 0.1)).to(dtype),
            "k_weight": (1 + _randn(g, (dim,), torch.float32, 0.1)).to(dtype), "rope": _rope_table(dim),
            "positions": _i32(_image_positions(r, t)), "sections": (case["time"], case["height"], case["width"]),
            "interleaved": case["interleaved"], "k_cache": cache(), "v_cache": cache(),
            "slots": torch.from_numpy(slots).to(_DEVICE)}


def _axis_of(sections, interleaved, device):
    """The axis whose position turns each of the frequencies."""
    j = torch.arange(sum(sections), device=device)
    if not interleaved:
        return (j >= sections[0]).long() + (j >= sections[0] + sections[1]).long()
    return torch.where((j % 3 == 1) & (j < 3 * sections[1]), 1,
                       torch.where((j % 3 == 2) & (j < 3 * sections[2]), 2, 0))


def _plain_prologue(s):
    t, dim, heads, kv_heads = s["qkv"].shape[0], s["rope"].shape[1], s["heads"], s["kv_heads"]
    q, k, v = s["qkv"].view(t, -1, dim).split([heads, kv_heads, kv_heads], 1)
    axis = _axis_of(s["sections"], s["interleaved"], q.device)
    row = s["positions"].long().clamp(0, s["rope"].shape[0] - 1)[axis].T  # [T, dim / 2]
    j = torch.arange(dim // 2, device=q.device)
    cos, sin = s["rope"][row, j][:, None], s["rope"][row, j + dim // 2][:, None]

    def turned(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS) * w.float()
        a, b = x[..., :dim // 2], x[..., dim // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(q.dtype)

    s["k_cache"].view(-1, kv_heads, dim)[s["slots"]] = turned(k, s["k_weight"])
    s["v_cache"].view(-1, kv_heads, dim)[s["slots"]] = v
    return {"q": turned(q, s["q_weight"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_prologue(s):
    q = _package().qk_norm_mrope_and_cache(
        s["qkv"], s["heads"], s["kv_heads"], s["q_weight"], s["k_weight"], _EPS, s["rope"], s["positions"],
        s["sections"], s["k_cache"], s["v_cache"], s["slots"], interleaved=s["interleaved"])
    return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _exact_prologue(case, seed):
    s = _prepare_prologue(case, seed)
    dim, kv_heads = case["dim"], case["kv_heads"]
    x = s["qkv"].double().view(case["tokens"], -1, dim)
    pos = s["positions"].cpu().numpy()
    rope = s["rope"].double()
    # The turn of each pair as a complex number, frequency by frequency.
    owner = np.zeros(dim // 2, np.int64)
    if case["interleaved"]:
        for a, n in ((1, case["height"]), (2, case["width"])):
            owner[a:3 * n:3] = a
    else:
        owner[case["time"]:] = 1
        owner[case["time"] + case["height"]:] = 2
    turn = torch.stack([torch.complex(rope[p, j], rope[p, j + dim // 2]) for j, p in
                        ((j, torch.from_numpy(pos[owner[j]]).to(_DEVICE).long()) for j in range(dim // 2))], 1)

    def rotated(x, w):
        y = x / torch.sqrt(x.square().mean(-1, keepdim=True) + _EPS) * w.double()
        z = torch.complex(y[..., :dim // 2], y[..., dim // 2:]) * turn[:, None]
        return torch.cat([z.real, z.imag], -1)

    h = case["heads"]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    kc.view(-1, kv_heads, dim)[s["slots"]] = rotated(x[:, h:h + kv_heads], s["k_weight"])
    vc.view(-1, kv_heads, dim)[s["slots"]] = x[:, h + kv_heads:]
    return {"q": rotated(x[:, :h], s["q_weight"]), "k_cache": kc, "v_cache": vc}


# ------------------------------------------------------------------------------------------------ linear attention


def _log_decay(kv_heads):
    """Rates spread evenly over their logarithm: the fastest head forgets within two tokens, the slowest in 256."""
    return -torch.exp2(-8.0 * torch.arange(1, kv_heads + 1, device=_DEVICE) / kv_heads).float()


def _prepare_linear(case, seed, tokens):
    g = torch.Generator(device=_DEVICE).manual_seed(seed)
    heads, kv_heads, dim, dtype = case["heads"], case["kv_heads"], case["dim"], _DTYPE[case["dtype"]]
    # q, k and v are the parts of a merged projection's rows.
    qkv = _randn(g, (tokens, heads + 2 * kv_heads, dim), dtype)
    q, k, v = qkv.split([heads, kv_heads, kv_heads], 1)
    r = np.random.default_rng([seed, 5])
    batch = case["batch"]
    return {"q": q, "k": k, "v": v, "log_decay": _log_decay(kv_heads),
            "state": _randn(g, (batch + 3, kv_heads, dim, dim), torch.float32, 4.0),
            "slots": _i32(r.permutation(batch + 3)[:batch]), "scale": dim ** -0.5}


def _plain_decode(s):
    kv_heads, group = s["k"].shape[1], s["q"].shape[1] // s["k"].shape[1]
    k, v, slots = s["k"].float(), s["v"].float(), s["slots"].long()
    decay = s["log_decay"].exp()[:, None, None]
    new = s["state"][slots] * decay + k[..., :, None] * v[..., None, :]
    s["state"][slots] = new
    q = s["q"].float().view(-1, kv_heads, group, k.shape[2])
    return {"out": (torch.matmul(q, new) * s["scale"]).to(s["q"].dtype).view(s["q"].shape), "state": s["state"]}


def _own_decode(s):
    out = _package().linear_attn_decode(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["slots"], s["scale"])
    return {"out": out, "state": s["state"]}


def _prefill_lens(case):
    return _lengths(case["lo"], case["hi"], case["batch"], 6)


def _prepare_prefill(case, seed):
    lens = _prefill_lens(case)
    s = _prepare_linear(case, seed, int(lens.sum()))
    # Without `fresh`, two requests in three go on behind an earlier chunk.
    ctx = np.where(np.arange(case["batch"]) % 3 == 1, 0, 512) * (not case["fresh"])
    return dict(s, cu=_cu(lens), max_len=int(lens.max()), context_lens=_i32(ctx))


def _plain_prefill(s):
    """Pieces of 64 tokens: the products inside a piece, and every piece's state from the sums of those before it."""
    size = 64
    cu, ld, scale = s["cu"].long(), s["log_decay"], s["scale"]
    t, heads, dim = s["q"].shape
    kv_heads, batch = s["k"].shape[1], cu.shape[0] - 1
    dev = cu.device
    lens = cu[1:] - cu[:-1]
    first = torch.cat([cu.new_zeros(1), ((lens + size - 1) // size).cumsum(0)])  # each request's first piece
    n = torch.arange(t // size + batch, device=dev)  # at least as many pieces as there are
    seq = torch.searchsorted(first[1:], n, right=True).clamp(max=batch - 1)
    begin = (n - first[seq]) * size
    filled = (lens[seq] - begin).clamp(0, size)
    i = torch.arange(size, device=dev)
    held = i < filled[:, None]
    row = torch.where(held, cu[seq][:, None] + begin[:, None] + i, 0)
    piece = lambda x: (x[row].float() * held[:, :, None, None]).transpose(1, 2)  # noqa: E731  [N, H, 64, D]
    q, k, v = piece(s["q"]).reshape(n.shape[0], kv_heads, -1, dim), piece(s["k"]), piece(s["v"])
    group = heads // kv_heads
    power = lambda x: torch.exp(ld.view(-1, *[1] * x.dim()) * x.float())  # noqa: E731  [Hkv, ...]
    past = i[:, None] - i
    inside = torch.where(past >= 0, power(past.clamp(min=0)), 0.0).repeat(1, group, 1)
    out = torch.matmul(torch.matmul(q, k.transpose(2, 3)) * inside, v)
    weight = power((filled[:, None] - 1 - i).clamp(min=0)).transpose(0, 1)[..., None]
    added = torch.matmul((k * weight).transpose(2, 3), v)  # [N, Hkv, D, D]
    start = torch.where(s["context_lens"][:, None, None, None] == 0, 0.0, s["state"][s["slots"].long()])
    # States at each piece's begin, then at each request's end: sums over the pieces before, decayed by the way to go.
    to_seq = torch.cat([seq, torch.arange(batch, device=dev)])
    to = torch.cat([begin, lens])
    way = to[:, None] - (begin + filled)
    before = (to_seq[:, None] == seq) & (way >= 0) & (filled > 0)
    mix = torch.where(before, power(way.clamp(min=0)), 0.0)  # [Hkv, N + B, N]
    states = torch.matmul(mix, added.transpose(0, 1).reshape(kv_heads, n.shape[0], -1))
    states = states.view(kv_heads, -1, dim, dim) + power(to)[..., None, None] * start[to_seq].transpose(0, 1)
    at_begin, at_end = states.split([n.shape[0], batch], 1)
    out = out + torch.matmul(q, at_begin.transpose(0, 1)) * power(i + 1).repeat(1, group)[None, :, :, None]
    s["state"][s["slots"].long()] = at_end.transpose(0, 1)
    # Back to rows.
    token = torch.arange(t, device=dev)
    b = torch.searchsorted(cu[1:], token, right=True)
    rel = token - cu[b]
    out = out.view(n.shape[0], kv_heads, group, size, dim)[first[b] + rel // size, :, :, rel % size]
    return {"out": (out.reshape(t, heads, dim) * scale).to(s["q"].dtype), "state": s["state"]}


def _own_prefill(s):
    out = _package().linear_attn_prefill(s["q"], s["k"], s["v"], s["log_decay"], s["state"], s["slots"], s["cu"],
                                         s["max_len"], s["scale"], context_lens=s["context_lens"])
    return {"out": out, "state": s["state"]}


def _exact_linear(s, lens, context_lens):
    """The recurrence itself, token by token, in 64 bits."""
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    kv_heads, dim = k.shape[1:]
    group = q.shape[1] // kv_heads
    decay = torch.exp(s["log_decay"].double())[:, None, None]
    slots = s["slots"].long()
    state, out = s["state"].double(), torch.zeros_like(q)
    now = state[slots] * torch.from_numpy((context_lens != 0).astype(np.float64)).to(_DEVICE)[:, None, None, None]
    order = np.argsort(-lens, kind="stable")  # the longest first: those still running are the first ones
    now = now[torch.from_numpy(order).to(_DEVICE)]
    begins = torch.from_numpy((np.cumsum(lens) - lens)[order]).to(_DEVICE)
    for i in range(int(lens.max())):
        m = int((lens > i).sum())
        at = begins[:m] + i
        now[:m] = now[:m] * decay + k[at][..., :, None] * v[at][..., None, :]
        out[at] = (q[at].view(m, kv_heads, group, 1, dim) @ now[:m, :, None]).reshape(m, -1, dim) * s["scale"]
    state[slots[torch.from_numpy(order).to(_DEVICE)]] = now
    return {"out": out, "state": state}


# ------------------------------------------------------------------------------------------------ what is called


def prepare(case, seed):
    kind = case["kind"]
    if kind == "metadata":
        s = _prepare_metadata(case, seed)
    elif kind == "prologue":
        s = _prepare_prologue(case, seed)
    elif kind == "linear_decode":
        s = _prepare_linear(case, seed, case["batch"])
    else:
        s = _prepare_prefill(case, seed)
    return dict(s, kind=kind)


_PLAIN = {"metadata": _plain_metadata, "prologue": _plain_prologue, "linear_decode": _plain_decode,
          "linear_prefill": _plain_prefill}
_OWN = {"metadata": _own_metadata, "prologue": _own_prologue, "linear_decode": _own_decode,
        "linear_prefill": _own_prefill}


def run(state):
    return (_OWN if own else _PLAIN)[state["kind"]](state)


def exact(case, seed):
    if case["kind"] == "prologue":
        return _exact_prologue(case, seed)
    if case["kind"] == "linear_decode":
        ones = np.ones(case["batch"], np.int64)
        return _exact_linear(_prepare_linear(case, seed, case["batch"]), ones, ones)
    if case["kind"] == "linear_prefill":
        s = _prepare_prefill(case, seed)
        return _exact_linear(s, _prefill_lens(case), s["context_lens"].cpu().numpy())
    return None  # whole numbers


def work(case):
    kind = case["kind"]
    if kind == "metadata":
        ctx, new = _metadata_lens(case)
        page, tokens = case["page"], (int(new.sum()) + 63) // 64 * 64
        last = int((ctx % page != 0).sum())  # table entries that a step's first tokens go on in
        taken = int((-(-(ctx + new) // page) + ctx // -page).sum())
        # Lengths and offsets, prefix sums, blocks handed out (read, written), a slot and the positions of each row.
        return {"bytes": case["batch"] * (12 if case["axes"] > 1 else 8) + 3 * 4 * (case["batch"] + 1) + 4 * last
                + 8 * taken + tokens * (8 + 4 * case["axes"]), "flops": 0}
    dim = case["dim"]
    if kind == "prologue":
        values = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * dim
        turned = case["tokens"] * (case["heads"] + case["kv_heads"]) * dim
        # Rows in and out, positions and slots; the rotation table's rows are few and shared.
        return {"bytes": 4 * values + case["tokens"] * (3 * 4 + 8), "flops": 7 * turned}
    kv_state = case["batch"] * case["kv_heads"] * dim * dim
    tokens = case["batch"] if kind == "linear_decode" else int(_prefill_lens(case).sum())
    rows = tokens * (2 * case["heads"] + 2 * case["kv_heads"]) * dim * 2
    reads = 1
    if kind == "linear_prefill":
        reads = 0 if case["fresh"] else float(np.mean(np.arange(case["batch"]) % 3 != 1))
    return {"bytes": rows + (1 + reads) * kv_state * 4,
            "flops": tokens * dim * dim * (2 * case["heads"] + 3 * case["kv_heads"])}

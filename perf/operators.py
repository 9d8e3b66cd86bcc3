"""The operators of batched serving on an 8-bit KV cache, as they are timed:
the batch map (block tables and slots from request lengths), the cache write,
decode attention and ragged prefill attention over the cache.

A cache block holds block_tokens tokens; for each (block, kv head) K and V have
one f32 scale each, a power of two when the write chose it.  Values are e4m3 or
int8 codes times that scale.  A case is a dict of plain values; "op" names the
operator and the rest its sizes and options.  Inputs are drawn on the GPU from
the seed alone.  `own` selects the library's kernels; without it the operators
are computed by elementary torch operations.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

# (heads, kv heads, head size): a 1.1B-shaped and an 8B-shaped attention, and
# the small grouped and the ungrouped head counts of the tests
GEOMETRIES = ((32, 4, 64), (32, 8, 128), (8, 2, 128), (12, 12, 64))
TOP = {"e4m3": 448.0, "int8": 127.0}
# 448 = 0.875 * 2^9, 127 = 0.9921875 * 2^7
TOP_MANTISSA = {"e4m3": 0.875, "int8": 0.9921875}
TOP_EXPONENT = {"e4m3": 9, "int8": 7}

DECODE_BYTES_MAX = 560_000_000
PREFILL_CELLS_MAX = 8192 * 8192 * 32
PREFILL_FLOPS_MAX = 550_000_000_000
WRITE_VALUES_MAX = 8192 * 8 * 128
MAP_ROWS_MAX = 65536


def _library():
    path = os.path.join(ROOT, "nyion.rs_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import nyion_hip

    return nyion_hip


def listed():
    return [
        # one decode step's slots and new pages of a full continuous batch
        dict(name="map_decode_batch64", op="map", batch=64, cached_lo=512, cached_hi=32767,
             new_lo=1, new_hi=1, block_tokens=16),
        # many prompts admitted at once, some onto a cached prefix
        dict(name="map_prompts_batch250", op="map", batch=250, cached_lo=0, cached_hi=1000,
             new_lo=1, new_hi=500, block_tokens=16),
        # the token that each sequence of a full batch appends in one layer
        dict(name="write_append_batch64", op="write", code="e4m3", io="f32", heads=32, kv_heads=4,
             head_dim=64, batch=64, cached_lo=512, cached_hi=4096, new_lo=1, new_hi=1,
             block_tokens=16),
        # a long prompt's K/V of one layer, 8B-shaped
        dict(name="write_prompt_8192", op="write", code="e4m3", io="bf16", heads=32, kv_heads=8,
             head_dim=128, batch=1, cached_lo=0, cached_hi=0, new_lo=8192, new_hi=8192,
             block_tokens=16),
        # chunks of several prompts that continue blocks half full, 8-bit integers
        dict(name="write_chunks_int8", op="write", code="int8", io="bf16", heads=32, kv_heads=8,
             head_dim=128, batch=7, cached_lo=100, cached_hi=3000, new_lo=100, new_hi=700,
             block_tokens=64),
        # the first tokens of a short chat: one call, almost no work
        dict(name="decode_ctx128", op="decode", code="e4m3", io="f32", heads=32, kv_heads=4,
             head_dim=64, batch=1, ctx_lo=128, ctx_hi=128, block_tokens=16, softcap=0.0, window=0,
             bias=False),
        # continuous batching at its fullest
        dict(name="decode_batch64", op="decode", code="e4m3", io="f32", heads=32, kv_heads=4,
             head_dim=64, batch=64, ctx_lo=512, ctx_hi=32768, block_tokens=16, softcap=0.0,
             window=0, bias=False),
        # an 8B-shaped batch with capped scores on 8-bit integers, ragged lengths
        dict(name="decode_capped_int8_batch24", op="decode", code="int8", io="bf16", heads=32,
             kv_heads=8, head_dim=128, batch=24, ctx_lo=200, ctx_hi=16000, block_tokens=32,
             softcap=50.0, window=0, bias=False),
        # a few long contexts, scores biased by distance
        dict(name="decode_biased_batch3", op="decode", code="e4m3", io="bf16", heads=32,
             kv_heads=8, head_dim=128, batch=3, ctx_lo=3000, ctx_hi=9001, block_tokens=16,
             softcap=0.0, window=0, bias=True),
        # a long prompt in one call
        dict(name="prefill_8192", op="prefill", code="e4m3", heads=32, kv_heads=8, head_dim=128,
             batch=1, history_lo=0, history_hi=0, rows_lo=8192, rows_hi=8192, block_tokens=16,
             softcap=0.0, window=0, bias=False, prefix=False),
        # a later chunk of a chat's prompt, capped scores, 8-bit integers
        dict(name="prefill_chunk_capped", op="prefill", code="int8", heads=32, kv_heads=4,
             head_dim=64, batch=1, history_lo=3001, history_hi=3001, rows_lo=500, rows_hi=500,
             block_tokens=16, softcap=30.0, window=0, bias=False, prefix=False),
        # a mixed batch: prompts, chunks and short turns, each behind a prefix
        # that all its rows see, scores biased by distance
        dict(name="prefill_ragged_prefix", op="prefill", code="e4m3", heads=32, kv_heads=8,
             head_dim=128, batch=9, history_lo=0, history_hi=2000, rows_lo=1, rows_hi=900,
             block_tokens=32, softcap=0.0, window=0, bias=True, prefix=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("map", "write", "write", "decode", "decode", "decode", "prefill", "prefill"))
    heads, kv_heads, head_dim = rng.choice(GEOMETRIES)
    block_tokens = rng.choice((16, 16, 32, 64, 128))
    geo = dict(heads=heads, kv_heads=kv_heads, head_dim=head_dim, block_tokens=block_tokens)
    if op == "map":
        batch = _log_int(rng, 1, 1000)
        new_hi = _log_int(rng, 1, max(1, MAP_ROWS_MAX // batch))
        cached_hi = _log_int(rng, 16, 16384)
        return dict(op="map", batch=batch, cached_lo=rng.choice((0, cached_hi // 2)),
                    cached_hi=cached_hi, new_lo=1, new_hi=new_hi, block_tokens=block_tokens)
    if op == "write":
        batch = _log_int(rng, 1, 64)
        most = max(1, WRITE_VALUES_MAX // (kv_heads * head_dim * batch))
        new_hi = rng.choice((1, _log_int(rng, 1, most)))
        return dict(op="write", code=rng.choice(("e4m3", "e4m3", "int8")),
                    io=rng.choice(("f32", "bf16")), batch=batch, cached_lo=0,
                    cached_hi=_log_int(rng, 16, 4096), new_lo=max(1, new_hi // 3), new_hi=new_hi,
                    **geo)
    softcap = rng.choice((0.0, 0.0, 30.0, 50.0))
    bias = rng.random() < 0.3
    code = rng.choice(("e4m3", "e4m3", "int8"))
    if op == "decode":
        window = rng.choice((0, 0, 0, 500, 4096))
        hi = _log_int(rng, 2 * window if window else 64, 32768)
        lo = max(1, int(hi * rng.choice((1.0, 0.5, 0.02))))
        batch = max(1, min(_log_int(rng, 1, 64), DECODE_BYTES_MAX // (2 * kv_heads * hi * head_dim)))
        return dict(op="decode", code=code, io=rng.choice(("f32", "f32", "bf16")), batch=batch,
                    ctx_lo=lo, ctx_hi=hi, softcap=softcap, window=window, bias=bias, **geo)
    rows = _log_int(rng, 2, 8192)
    history = rng.choice((0, _log_int(rng, 16, 16384)))
    while (heads * rows * (history + rows) > PREFILL_CELLS_MAX
           or 4 * heads * head_dim * rows * (history + (rows + 1) / 2) > PREFILL_FLOPS_MAX):
        history //= 2
    cost = heads * rows * (history + rows)
    batch = max(1, min(_log_int(rng, 1, 16), PREFILL_CELLS_MAX // 4 // cost))
    return dict(op="prefill", code=code, batch=batch, history_lo=history // 3, history_hi=history,
                rows_lo=max(1, rows // 4) if batch > 1 else rows, rows_hi=rows, softcap=softcap,
                window=rng.choice((0, 0, 1000)), bias=bias, prefix=rng.random() < 0.25, **geo)


# ------------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, device="cuda", generator=g)


def _between(g, lo, hi, n):
    return torch.randint(lo, hi + 1, (n,), generator=g, device="cuda").to(torch.int32)


def _sharing(g, lo, hi, n):
    """n numbers of lo..hi whose sum is n times their mean, whatever the seed."""
    x = torch.randint(lo, hi + 1, (n,), generator=g, device="cuda")
    for side in (hi, lo):  # what is missing, or too much, goes to the first that have room
        room, want = (x - side).abs(), n * (lo + hi) // 2 - x.sum()
        if (want > 0) == (side == hi):
            part = torch.minimum((want.abs() - (room.cumsum(0) - room)).clamp(min=0), room)
            x = x + part * want.sign()
    return x.to(torch.int32)


def _scale(amax, code):
    """The smallest power of two (2^-126 at least) by which amax fits the codes."""
    mantissa, exponent = torch.frexp(amax)
    exponent = exponent - TOP_EXPONENT[code] + (mantissa > TOP_MANTISSA[code]).to(exponent.dtype)
    return torch.ldexp(torch.ones_like(amax), exponent.clamp(min=-126))


def _encode(x, code):
    """Codes of values that are within the codes' range already."""
    if code == "e4m3":
        return x.to(torch.float8_e4m3fn).view(torch.uint8)
    return x.round().to(torch.int8).view(torch.uint8)


def _values(codes, code):
    """The codes' values in f32, without the scale."""
    return codes.view(torch.float8_e4m3fn if code == "e4m3" else torch.int8).float()


def _pool(g, c, blocks):
    """A pool of N(0, 1) rows, each (block, head) at a level of its own, in slices."""
    h, bt, d = c["kv_heads"], c["block_tokens"], c["head_dim"]
    codes = torch.empty((blocks, h, bt, d), dtype=torch.uint8, device="cuda")
    scales = torch.empty((blocks, h), device="cuda")
    per = max(1, (64 << 20) // (h * bt * d))
    for b in range(0, blocks, per):
        n = min(per, blocks - b)
        x = _normal(g, n, h, bt, d) * torch.exp(0.3 * _normal(g, n, h, 1, 1))
        s = _scale(x.abs().amax((2, 3)), c["code"])
        codes[b:b + n] = _encode(x / s[:, :, None, None], c["code"])
        scales[b:b + n] = s
    return codes, scales


def _tables(g, lens, block_tokens, max_blocks, empty=0):
    """Block tables of sequences that share one shuffled pool, and how many blocks they hold."""
    need = (lens.long() + block_tokens - 1) // block_tokens
    total = int(need.sum())
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    tables = torch.full((len(lens), max_blocks), empty, dtype=torch.int32, device="cuda")
    mask = torch.arange(max_blocks, device="cuda")[None, :] < need[:, None]
    tables[mask] = order
    return tables, total


def _slots(tables, cached, new, block_tokens):
    """Row starts and the flat slot of each new row (block * block_tokens + place in it)."""
    starts = torch.zeros(len(new) + 1, dtype=torch.int32, device="cuda")
    starts[1:] = new.cumsum(0)
    rows = torch.arange(int(starts[-1]), device="cuda")
    seq = torch.searchsorted(starts[1:].contiguous(), rows.to(torch.int32), right=True)
    pos = cached.long()[seq] + rows - starts.long()[seq]
    block = tables[seq, pos // block_tokens].long()
    return starts, block * block_tokens + pos % block_tokens


def _slopes(c):
    if not c["bias"]:
        return None
    at = torch.arange(1, c["heads"] + 1, device="cuda", dtype=torch.float32)
    return torch.exp2(-8.0 * at / c["heads"])


def prepare(case, seed):
    g, c = _generator(seed), case
    bt = c["block_tokens"]
    if c["op"] == "map":
        cached = _between(g, c["cached_lo"], c["cached_hi"], c["batch"])
        new = _sharing(g, c["new_lo"], c["new_hi"], c["batch"])
        max_blocks = -(-(c["cached_hi"] + c["new_hi"]) // bt)
        tables, held = _tables(g, cached, bt, max_blocks, empty=-1)
        n_rows = int(new.sum())
        wanted = n_rows // bt + c["batch"]
        free = held + torch.randperm(wanted, generator=g, device="cuda").to(torch.int32)
        out = dict(tables=tables, ctx_lens=torch.empty_like(cached),
                   row_starts=torch.empty(c["batch"] + 1, dtype=torch.int32, device="cuda"),
                   slots=torch.empty(n_rows, dtype=torch.int64, device="cuda"),
                   positions=torch.empty(n_rows, dtype=torch.int32, device="cuda"),
                   counts=torch.empty(2, dtype=torch.int32, device="cuda"))
        return dict(case=c, cached=cached, new=new, free=free, num_blocks=held + wanted, out=out)
    if c["op"] == "write":
        cached = _between(g, c["cached_lo"], c["cached_hi"], c["batch"])
        new = _sharing(g, c["new_lo"], c["new_hi"], c["batch"])
        max_blocks = -(-(c["cached_hi"] + c["new_hi"]) // bt)
        tables, _ = _tables(g, cached + new, bt, max_blocks)
        _, slots = _slots(tables, cached, new, bt)
        blocks = c["batch"] * max_blocks
        k_pool, k_scales = _pool(g, c, blocks)
        v_pool, v_scales = _pool(g, c, blocks)
        dtype = torch.float32 if c["io"] == "f32" else torch.bfloat16
        shape = (len(slots), c["kv_heads"], c["head_dim"])
        return dict(case=c, k_pool=k_pool, v_pool=v_pool, k_scales=k_scales, v_scales=v_scales,
                    tables=tables, cached=cached, slots=slots, k=_normal(g, *shape).to(dtype),
                    v=_normal(g, *shape).to(dtype))
    slopes = _slopes(c)
    if c["op"] == "decode":
        lens = _between(g, c["ctx_lo"], c["ctx_hi"], c["batch"])
        rows, starts, max_rows, prefix = c["batch"], None, 1, None
        dtype = torch.float32 if c["io"] == "f32" else torch.bfloat16
    else:
        new = _sharing(g, c["rows_lo"], c["rows_hi"], c["batch"])
        history = _between(g, c["history_lo"], c["history_hi"], c["batch"])
        lens = history + new
        starts = torch.zeros(c["batch"] + 1, dtype=torch.int32, device="cuda")
        starts[1:] = new.cumsum(0)
        rows, max_rows, dtype = int(starts[-1]), int(new.max()), torch.bfloat16
        share = torch.rand(c["batch"], generator=g, device="cuda")
        prefix = (share * lens).to(torch.int32) if c["prefix"] else None
    max_ctx = int(lens.max())
    tables, blocks = _tables(g, lens, bt, -(-max_ctx // bt))
    k_pool, k_scales = _pool(g, c, blocks)
    v_pool, v_scales = _pool(g, c, blocks)
    q = _normal(g, rows, c["heads"], c["head_dim"]).to(dtype)
    return dict(case=c, k_pool=k_pool, v_pool=v_pool, k_scales=k_scales, v_scales=v_scales,
                tables=tables, lens=lens, max_ctx=max_ctx, starts=starts, max_rows=max_rows,
                prefix=prefix, slopes=slopes, q=q, out=torch.empty_like(q))


# ------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if op == "map":
        return _map_own(state) if own else _map_plain(state)
    if op == "write":
        if own:
            _write_own(state)
        else:
            _write_plain(state)
        held = torch.float8_e4m3fn if state["case"]["code"] == "e4m3" else torch.int8
        return dict(k=state["k_pool"].view(held), v=state["v_pool"].view(held),
                    k_scales=state["k_scales"], v_scales=state["v_scales"])
    if own:
        return _decode_own(state) if op == "decode" else _prefill_own(state)
    return _attention_plain(state)


def _cache(state):
    """The cache handle that a program keeps, made at its first use."""
    if "cache" not in state:
        nh = _library()
        nh.init(0)
        code = {"e4m3": nh.KV8_E4M3, "int8": nh.KV8_INT8}[state["case"]["code"]]
        state["cache"] = nh.Kv8Cache(state["k_pool"], state["v_pool"], state["k_scales"],
                                     state["v_scales"], code)
    return state["cache"]


def _options(state):
    if "options" not in state:
        c = state["case"]
        state["options"] = _library().ScoreOptions(softcap=c["softcap"], window=c["window"],
                                                   slopes=state["slopes"],
                                                   prefix_lens=state["prefix"])
    return state["options"]


def _map_own(state):
    nh, o = _library(), state["out"]
    nh.batch_map(state["cached"], state["new"], state["free"], o["tables"],
                 state["case"]["block_tokens"], state["num_blocks"], o["ctx_lens"],
                 o["row_starts"], o["slots"], o["positions"], o["counts"])
    return o


def _write_own(state):
    _library().kv8_write(_cache(state), state["slots"], state["k"], state["v"])


def _decode_own(state):
    nh, cache = _library(), _cache(state)
    if "workspace" not in state:
        need = nh.kv8_decode_workspace_size(cache, len(state["lens"]), state["case"]["heads"],
                                            state["max_ctx"], state["case"]["window"])
        state["workspace"] = nh.alloc_workspace(need)
    nh.kv8_decode(cache, state["q"], state["tables"], state["lens"], state["out"],
                  max_ctx=state["max_ctx"], options=_options(state),
                  workspace=state["workspace"])
    return state["out"]


def _prefill_own(state):
    nh, cache = _library(), _cache(state)
    if "workspace" not in state:
        need = nh.kv8_prefill_workspace_size(cache, len(state["lens"]), state["case"]["heads"],
                                             len(state["q"]), state["max_rows"],
                                             state["max_ctx"], state["case"]["window"])
        state["workspace"] = nh.alloc_workspace(need)
    nh.kv8_prefill_bf16(cache, state["q"], state["tables"], state["lens"], state["starts"],
                        state["out"], max_rows=state["max_rows"], max_ctx=state["max_ctx"],
                        options=_options(state), workspace=state["workspace"])
    return state["out"]


def _map_plain(state):
    bt, o = state["case"]["block_tokens"], state["out"]
    cached, new, free, tables = (state["cached"].long(), state["new"].long(), state["free"],
                                 o["tables"])
    ctx = cached + new
    held, last = (cached + bt - 1) // bt, (ctx + bt - 1) // bt
    ends, taken = new.cumsum(0), (last - held).cumsum(0)
    page = torch.arange(tables.shape[1], device=tables.device)[None, :]
    fresh = (page >= held[:, None]) & (page < last[:, None])
    at = (taken - (last - held))[:, None] + page - held[:, None]
    given = torch.where(at < len(free), free[at.clamp(0, len(free) - 1)], -1)
    tables.copy_(torch.where(fresh, given, tables))
    rows = torch.arange(len(o["slots"]), device=tables.device)
    seq = torch.searchsorted(ends, rows, right=True)
    pos = cached[seq] + rows - (ends - new)[seq]
    block = tables[seq, pos // bt].long()
    starts = torch.cat((torch.zeros_like(ends[:1]), ends))
    o.update(ctx_lens=ctx.to(torch.int32), row_starts=starts.to(torch.int32),
             slots=torch.where(block >= 0, block * bt + pos % bt, -1),
             positions=pos.to(torch.int32),
             counts=torch.stack((taken[-1], ends[-1])).to(torch.int32))
    return o


def _write_plain(state):
    _write_plain_half(state, state["k_pool"], state["k_scales"], state["k"])
    _write_plain_half(state, state["v_pool"], state["v_scales"], state["v"])


def _write_plain_half(state, pool, scales, x):
    code, bt = state["case"]["code"], state["case"]["block_tokens"]
    slots, cached, tables = state["slots"], state["cached"].long(), state["tables"]
    x = x.float()
    block = slots // bt
    # the largest value that each (block, head) takes in; blocks without one keep 0
    top = torch.zeros_like(scales).index_reduce_(0, block, x.abs().amax(2), "amax")
    fresh = torch.where(top > 0, _scale(top, code), 0)
    # the block that each sequence continues holds `live` tokens in front of the new ones
    live = cached % bt
    ahead = tables.gather(1, (cached // bt)[:, None])[:, 0].long()
    before = torch.where(live[:, None] > 0, scales[ahead], 0)
    after = torch.maximum(before, fresh[ahead])
    place = torch.arange(bt, device=pool.device)[None, None, :, None] < live[:, None, None, None]
    old = pool[ahead]
    again = _encode(_values(old, code) * (before / after)[:, :, None, None], code)
    pool[ahead] = torch.where(place, again, old)
    fresh[ahead] = after
    scales.copy_(torch.where(top > 0, fresh, scales))
    pool[block, :, slots % bt] = _encode(x / scales[block][:, :, None], code)


def _attention_plain(state):
    c = state["case"]
    b, hk, d, bt = c["batch"], c["kv_heads"], c["head_dim"], c["block_tokens"]
    group = c["heads"] // hk
    q, tables, lens, r = state["q"].float(), state["tables"].long(), state["lens"], state["max_rows"]

    def rows_of(pool, scales):
        x = _values(pool[tables], c["code"]) * scales[tables][:, :, :, None, None]
        return x.permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)

    device = q.device
    if state["starts"] is None:
        at = torch.arange(b, device=device)[:, None]
        pos = lens.long()[:, None] - 1
    else:
        starts = state["starts"].long()
        i = torch.arange(r, device=device)[None, :]
        at = (starts[:-1, None] + i).clamp(max=len(q) - 1)
        pos = lens.long()[:, None] - (starts[1:] - starts[:-1])[:, None] + i
    # [b][kv head][row, head of the group][d]
    rows = q[at].view(b, r, hk, group, d).permute(0, 2, 1, 3, 4).reshape(b, hk, r * group, d)
    s = rows @ rows_of(state["k_pool"], state["k_scales"]).transpose(2, 3)
    s = s.view(b, hk, r, group, -1) / math.sqrt(d)
    if c["softcap"] > 0:
        s = c["softcap"] * torch.tanh(s / c["softcap"])
    key = torch.arange(s.shape[-1], device=device)
    back = pos[:, :, None] - key[None, None, :]
    if state["slopes"] is not None:
        s = s - (state["slopes"].view(1, hk, 1, group, 1) * back.abs().float()[:, None, :, None, :])
    seen = back >= 0
    if state["prefix"] is not None:
        seen = seen | (key[None, None, :] < state["prefix"].long()[:, None, None])
    if c["window"] > 0:
        seen = seen & (back < c["window"])
    seen = (seen & (key[None, None, :] < lens.long()[:, None, None]))[:, None, :, None, :]
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    o = (p.view(b, hk, r * group, -1) @ rows_of(state["v_pool"], state["v_scales"]))
    o = o.view(b, hk, r, group, d) / total
    o = o.permute(0, 2, 1, 3, 4).reshape(b * r, c["heads"], d)
    if state["starts"] is not None:
        row = torch.arange(len(q), device=device)
        seq = torch.searchsorted(starts[1:].contiguous(), row, right=True)
        o = o[seq * r + row - starts[seq]]
    return o.to(state["q"].dtype)


# ------------------------------------------------------------- 64 bits

def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "map":
        return None
    if case["op"] == "write":
        k, k_scales = _write_exact(state, state["k_pool"], state["k_scales"], state["k"])
        v, v_scales = _write_exact(state, state["v_pool"], state["v_scales"], state["v"])
        return dict(k=k, v=v, k_scales=k_scales, v_scales=v_scales)
    c, q = case, state["q"].double()
    out, bt, group = torch.zeros_like(q), c["block_tokens"], c["heads"] // c["kv_heads"]
    lens = state["lens"].tolist()
    starts = list(range(c["batch"] + 1)) if state["starts"] is None else state["starts"].tolist()
    for b, n in enumerate(lens):
        blocks = state["tables"][b, :-(-n // bt)].long()
        position = torch.arange(n - (starts[b + 1] - starts[b]), n, device="cuda")
        key = torch.arange(n, device="cuda")
        distance = position[:, None] - key[None, :]
        hidden = distance < 0
        if state["prefix"] is not None:
            hidden &= key[None, :] >= int(state["prefix"][b])
        if c["window"] > 0:
            hidden |= distance >= c["window"]
        for h in range(c["heads"]):
            k, v = (_decoded(p[blocks, h // group], c["code"]).mul_(
                s[blocks, h // group].double()[:, None, None]).view(-1, c["head_dim"])[:n]
                for p, s in ((state["k_pool"], state["k_scales"]),
                             (state["v_pool"], state["v_scales"])))
            s = q[starts[b]:starts[b + 1], h] @ k.T
            s *= c["head_dim"] ** -0.5
            if c["softcap"] > 0:
                s = torch.tanh(s / c["softcap"]) * c["softcap"]
            if c["bias"]:
                s -= float(state["slopes"][h]) * distance.abs()
            s.masked_fill_(hidden, -math.inf)
            out[starts[b]:starts[b + 1], h] = torch.softmax(s, 1) @ v
    return out


def _decoded(codes, code):
    """The codes' values in 64 bits, from their bits."""
    x = codes.to(torch.int64)
    if code == "int8":
        return torch.where(x > 127, x - 256, x).double()
    e, m = (x >> 3) & 15, x & 7
    size = torch.where(e > 0, (8 + m).double() * torch.exp2((e - 10).double()),
                       m.double() * 2.0 ** -9)
    return torch.where(x > 127, -size, size)


def _rounded(x, code):
    """The nearest value that a code has, ties to even, of |x| within their range."""
    if code == "int8":
        return torch.round(x)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _write_exact(state, pool, scales, x):
    c = state["case"]
    code, bt = c["code"], c["block_tokens"]
    values, held = _decoded(pool, code), scales.double()
    x, slots = x.double(), state["slots"]
    block, place = slots // bt, slots % bt
    for b in block.unique().tolist():
        at = (block == b).nonzero()[:, 0]
        first = int(place[at].min())
        for h in range(c["kv_heads"]):
            top = float(x[at, h].abs().max())
            scale = 2.0 ** max(-126, math.ceil(math.log2(top / TOP[code]))) if top > 0 else 2.0 ** -126
            if first > 0:
                was = float(held[b, h])
                scale = max(scale, was)
                values[b, h, :first] = _rounded(values[b, h, :first] * (was / scale), code)
            held[b, h] = scale
            values[b, h, place[at]] = _rounded(x[at, h] / scale, code)
    return values, held


# ------------------------------------------------------------- work

def work(case):
    c, bt = case, case["block_tokens"]
    if c["op"] == "map":
        # the mean of the drawn lengths; each row's slot and position, each new page's table entry
        rows = c["batch"] * (c["new_lo"] + c["new_hi"]) // 2
        return {"bytes": 12 * rows + 8 * (rows // bt + c["batch"]) + 16 * c["batch"], "flops": 0}
    hk, d = c["kv_heads"], c["head_dim"]
    if c["op"] == "write":
        rows = c["batch"] * (c["new_lo"] + c["new_hi"]) // 2
        size = 4 if c["io"] == "f32" else 2
        return {"bytes": 2 * rows * hk * d * (size + 1) + 8 * rows + 16 * hk * (rows // bt + c["batch"]),
                "flops": 2 * rows * hk * d * 3}
    if c["op"] == "decode":
        rows, size = 1, 4 if c["io"] == "f32" else 2
        keys = (c["ctx_lo"] + c["ctx_hi"]) // 2
        pairs = held = min(keys, c["window"]) if c["window"] > 0 else keys
    else:
        rows, size = (c["rows_lo"] + c["rows_hi"]) // 2, 2
        history = (c["history_lo"] + c["history_hi"]) // 2
        keys = history + rows
        held = min(keys, rows + c["window"]) if c["window"] > 0 else keys
        pairs = rows * (history + (rows + 1) / 2)
        if c["window"] > 0:
            pairs = min(pairs, rows * c["window"])
        if c["prefix"] and c["window"] <= 0:  # half of the keys, seen by the rows in front of them too
            pairs += max(0, keys / 2 - history) ** 2 / 2
    blocks = -(-held // bt)
    return {"bytes": c["batch"] * (2 * held * hk * d + 8 * blocks * hk + 4 * blocks
                                   + 2 * rows * c["heads"] * d * size),
            "flops": 4 * c["batch"] * c["heads"] * d * pairs}

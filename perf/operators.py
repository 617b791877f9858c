"""The operators of a cache held in 4 bits, timed in plain torch and on the framework's kernels: rows packed into pages and read back,
attention over such pages, and a step's index arrays made on the GPU from its requests' lengths.

The page.  Neighbouring elements of one head of one token, 32 at a time, share a power of two 2^(b - 127), b in 2 .. 252 one byte (255: none of
them is a number), and an element is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 in 4 bits, the lower half of a byte first.  With `a` the
largest magnitude of a block, b + 2 is the biased exponent of a, one more where a's significand is 1.75 or larger; elements are
divided by the block's power, rounded to the nearest of the eight (ties to the even code) and no larger than 6.  What a page holds of one
kv head lies in one run of bytes, for `ps` keys of `D` elements: key codes [ps][D / 2], value codes [ps / 8][D / 8][8 keys][4 bytes], key
powers [ps][D / 32], value powers [ps / 8][D / 32][8 keys].
"""

from __future__ import annotations

import math

import torch

own = False

DEVICE = "cuda:0"
# heads, kv heads and head size of the layer sizes under configs/, and two that no file there has
LAYERS = ((12, 2, 128), (28, 4, 128), (40, 8, 128), (16, 4, 64), (9, 3, 96))
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one user in the middle of an answer: a layer's attention of one token, where launches count
        {"name": "attend 1", "op": "attend", "heads": 12, "kv_heads": 2, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 1, "context": 640, "portion": 0, "behind": 0, "window": 0},
        # a full batch of a busy server over ragged contexts of some thousand tokens
        {"name": "attend 64", "op": "attend", "heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 64, "context": 4096, "portion": 0, "behind": 0, "window": 0},
        # eight long documents: the cache is what the step reads
        {"name": "attend 8 long", "op": "attend", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 8, "context": 30000, "portion": 0, "behind": 0, "window": 0},
        # the true 32-bit mode, narrow heads, large pages, a sliding window
        {"name": "attend float32 window", "op": "attend", "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "float32", "page": 64, "decodes": 17, "context": 2011, "portion": 0, "behind": 0, "window": 1024},
        # a new prompt of an odd length
        {"name": "attend prompt 2047", "op": "attend", "heads": 12, "kv_heads": 2, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 0, "context": 0, "portion": 2047, "behind": 0, "window": 0},
        # the last portion of a long document's prompt
        {"name": "attend 2048 behind 30000", "op": "attend", "heads": 12, "kv_heads": 2, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 0, "context": 0, "portion": 2048, "behind": 30000, "window": 0},
        # continuous batching: a portion of a prompt beside 31 requests that decode
        {"name": "attend 31+256", "op": "attend", "heads": 28, "kv_heads": 4, "dim": 128, "dtype": "bfloat16", "page": 16, "decodes": 31, "context": 640, "portion": 256, "behind": 300, "window": 0},
        # the keys and values of a decode step's tokens, and a look at what was kept of them
        {"name": "store 8", "op": "store", "heads": 12, "kv_heads": 2, "dim": 128, "dtype": "bfloat16", "page": 16, "tokens": 8, "singles": True},
        # those of a portion of the largest layer sizes
        {"name": "store 8192", "op": "store", "heads": 40, "kv_heads": 8, "dim": 128, "dtype": "bfloat16", "page": 16, "tokens": 8192, "singles": False},
        # 32-bit rows, an odd number of them, pages of 8
        {"name": "store float32 1021", "op": "store", "heads": 16, "kv_heads": 4, "dim": 64, "dtype": "float32", "page": 8, "tokens": 1021, "singles": False},
        # the index arrays of a step of one token
        {"name": "place 1", "op": "place", "decodes": 1, "context": 640, "portion": 0, "behind": 0, "groups": 1, "page": 16, "blocks": 2048},
        # ... of 63 decoded tokens beside a portion, for a model with two kinds of layers
        {"name": "place 63+2048", "op": "place", "decodes": 63, "context": 8192, "portion": 2048, "behind": 5000, "groups": 2, "page": 16, "blocks": 2048},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choices(("attend", "store", "place"), weights=(6, 2, 2))[0]
    page = rng.choice((8, 16, 16, 24, 64))
    if op == "place":
        decodes, portion = _spread(rng, 1, 128), rng.choice((0, _spread(rng, 2, 4096)))
        return {"op": op, "decodes": decodes, "context": _spread(rng, 2, 10000), "portion": portion, "behind": rng.choice((0, _spread(rng, 1, 8000))),
                "groups": rng.choice((1, 1, 2, 3)), "page": page, "blocks": -(-16384 // page)}
    heads, kv_heads, dim = rng.choice(LAYERS)
    dtype = rng.choice(("bfloat16", "bfloat16", "float32"))
    if op == "store":
        singles = rng.random() < 0.4
        return {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page,
                "tokens": _spread(rng, 1, 128) if singles else _spread(rng, 2, 6000), "singles": singles}
    case = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "page": page, "decodes": 0, "context": 0, "portion": 0, "behind": 0,
            "window": rng.choice((0, 0, 0, _spread(rng, 1, 2000)))}
    kind = rng.choices(("decode", "prompt", "mixed"), weights=(4, 2, 2))[0]
    if kind != "prompt":
        case["decodes"] = _spread(rng, 1, 64 if kind == "decode" else 32)
        case["context"] = _spread(rng, 1, min(30000, 200000 // case["decodes"]) if kind == "decode" else 4000)
    if kind != "decode":
        case["portion"] = _spread(rng, 2, 2048 if kind == "prompt" else 512)
        case["behind"] = rng.choice((0, _spread(rng, 1, 12000 if kind == "prompt" else 4000)))
    return case


def _requests(case):
    """(cached tokens before the step, tokens in it) of every request: contexts ragged from half to one and a half times their mean, the portion last."""
    count, mean = case["decodes"], case["context"]
    found = [(max(0, round(mean * (0.5 + i / (count - 1)) if count > 1 else mean) - 1), 1) for i in range(count)]
    return found + ([(case["behind"], case["portion"])] if case["portion"] else [])


def _visible(before, tokens, window):
    """Keys seen by the queries at before .. before + tokens - 1, added up."""
    if not window:
        return tokens * before + tokens * (tokens + 1) // 2
    short = max(0, min(tokens, window - before))  # queries that see fewer keys than the window holds
    return short * before + short * (short + 1) // 2 + (tokens - short) * window


def work(case):
    if case["op"] == "place":
        requests = _requests(case)
        tokens, groups = sum(n for _, n in requests), case["groups"]
        width = max(-(-(before + n) // case["page"]) for before, n in requests)
        held = sum(-(-(before + n) // case["page"]) for before, n in requests)
        return {"bytes": 4 * (3 * len(requests) + groups * held + 2 * tokens + 2 * len(requests) + 1 + groups * (tokens + len(requests) * width)), "flops": 0}
    size = 2 if case["dtype"] == "bfloat16" else 4
    row = case["kv_heads"] * case["dim"]
    if case["op"] == "store":  # rows read, packed, read as packed, written
        return {"bytes": case["tokens"] * 2 * row * (2 * size + 2 * 17 / 32), "flops": 0}
    keys = queries = pairs = 0
    for before, tokens in _requests(case):
        first = max(0, before + 1 - case["window"]) if case["window"] else 0
        keys += before + tokens - first
        queries += tokens
        pairs += _visible(before, tokens, case["window"])
    width = case["heads"] * case["dim"]
    return {"bytes": keys * 2 * row * 17 / 32 + queries * 2 * width * size, "flops": 4 * width * pairs}


# ---------------------------------------------------------------------------- pages in plain torch


def _packed(x):
    """float32 [..., D] -> (codes uint8 [..., D], powers uint8 [..., D / 32])."""
    blocks = x.unflatten(-1, (-1, 32))
    largest = blocks.abs().amax(-1)
    power = ((largest.view(torch.int32) + 0x200000) >> 23).sub(2).clamp(2, 252)
    scaled = blocks * torch.exp2(127.0 - power.float()).unsqueeze(-1)
    size = scaled.abs()
    code = ((size > 0.25).int() + (size >= 0.75).int() + (size > 1.25).int() + (size >= 1.75).int() + (size > 2.5).int() + (size >= 3.5).int() + (size > 5.0).int())
    code = torch.where(torch.isfinite(largest).unsqueeze(-1), code + 8 * torch.signbit(scaled).int(), 0)
    power = torch.where(torch.isfinite(largest), power, 255)
    return code.to(torch.uint8).flatten(-2), power.to(torch.uint8)


def _pairs(codes):
    """Two codes to a byte, the first in the lower half."""
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _fields(pages, ps, dim):
    """Views of the four runs of pages [..., bytes]."""
    a, b = ps * dim // 2, ps * dim // 32
    lead = pages.shape[:-1]
    return (pages[..., :a].view(*lead, ps, dim // 2), pages[..., a:2 * a].view(*lead, ps // 8, dim // 8, 8, 4),
            pages[..., 2 * a:2 * a + b].view(*lead, ps, dim // 32), pages[..., 2 * a + b:].view(*lead, ps // 8, dim // 32, 8))


def _values(codes, powers):
    """Bytes of two codes [..., D / 2] and powers [..., D / 32] -> float32 [..., D]."""
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    both = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    power = torch.where(powers == 255, torch.nan, torch.exp2(powers.float() - 127.0))
    return (table[both.int()].unflatten(-1, (-1, 32)) * power.unsqueeze(-1)).flatten(-2)


def _rows(pages, ps, dim):
    """Pages [..., bytes] -> keys and values float32 [..., ps, D]."""
    kc, vc, kp, vp = _fields(pages, ps, dim)
    # (pieces of eight keys, granules of eight elements, keys, bytes) -> keys, bytes of a row
    return _values(kc, kp), _values(vc.transpose(-3, -2).flatten(-2).flatten(-3, -2), vp.transpose(-2, -1).flatten(-3, -2))


def _write(pages, slots, keys, values, ps):
    """Packs keys and values float32 [T, kv, D] into the pages [pages, kv, bytes] at slots [T]; a negative slot's rows go nowhere."""
    dim = keys.shape[-1]
    kept = slots >= 0
    page, offset = (slots.long() // ps)[kept], (slots.long() % ps)[kept]
    kc, vc, kp, vp = _fields(pages, ps, dim)
    codes, powers = _packed(keys[kept])
    kc[page, :, offset], kp[page, :, offset] = _pairs(codes), powers
    codes, powers = _packed(values[kept])
    vc[page, :, offset // 8, :, offset % 8] = _pairs(codes).unflatten(-1, (-1, 4))
    vp[page, :, offset // 8, :, offset % 8] = powers


# ---------------------------------------------------------------------------- states


def prepare(case, seed):
    generator = torch.Generator(device=DEVICE).manual_seed(seed)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=DEVICE)
    if case["op"] == "place":
        requests, ps, blocks = _requests(case), case["page"], case["blocks"]
        slots = torch.randperm(256, generator=generator, device=DEVICE)[:len(requests)].int()
        held = ints([-(-(before + n) // ps) for before, n in requests])
        # a cache's tables: a row a request slot, pages in any order, -1 behind the last one
        tables = torch.randint(0, 1 << 20, (case["groups"], 256, blocks), generator=generator, device=DEVICE, dtype=torch.int32)
        tables[:, slots.long()] = torch.where(torch.arange(blocks, device=DEVICE) < held[:, None], tables[:, slots.long()], -1)
        return {"op": "place", "tables": tables, "slots": slots, "starts": ints([before for before, _ in requests]), "counts": ints([n for _, n in requests]),
                "page": ps, "tokens": sum(n for _, n in requests), "width": int(held.max())}
    dtype, dim, kv, ps = getattr(torch, case["dtype"]), case["dim"], case["kv_heads"], case["page"]
    heads = case["heads"]
    state = {"op": case["op"], "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "page": ps}
    normal = lambda *shape: torch.randn(shape, generator=generator, device=DEVICE)
    # keys and values as projections leave them: channels of different sizes, some an order larger than others
    spread = torch.exp(0.7 * normal(2, kv, 1, dim))
    if case["op"] == "store":
        tokens = case["tokens"]
        pages = -(-tokens // ps) + 3 if not case["singles"] else tokens + 3
        order = torch.randperm(pages, generator=generator, device=DEVICE)
        at = torch.arange(tokens, device=DEVICE)
        if case["singles"]:  # a token of each of so many requests
            slots = order[at] * ps + torch.randint(0, ps, (tokens,), generator=generator, device=DEVICE)
        else:  # a run of tokens of one request, from somewhere inside a page
            at = at + 3
            slots = order[at // ps] * ps + at % ps
        rows = torch.cat([normal(tokens, heads * dim), (normal(kv, tokens, dim) * spread[0]).transpose(0, 1).flatten(1),
                          (normal(kv, tokens, dim) * spread[1]).transpose(0, 1).flatten(1)], dim=1)
        return state | {"qkv": rows.to(dtype), "slots": slots.int(), "pages": torch.zeros((pages, kv, ps * (dim + dim // 16)), dtype=torch.uint8, device=DEVICE)}
    requests = _requests(case)
    held = [-(-(before + n) // ps) for before, n in requests]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=generator, device=DEVICE).int()
    tables = torch.full((len(requests), max(held)), -1, dtype=torch.int32, device=DEVICE)
    places = torch.arange(max(held), device=DEVICE) < ints(held)[:, None]
    tables[places] = order[:sum(held)]
    storage = torch.empty((pages, kv, ps * (dim + dim // 16)), dtype=torch.uint8, device=DEVICE)
    kc, vc, kp, vp = _fields(storage, ps, dim)
    for first in range(0, pages, 4096):  # (in pieces: float32 rows of a whole cache are many times its size)
        some = slice(first, min(pages, first + 4096))
        number = some.stop - first
        codes, powers = _packed(normal(number, kv, ps, dim) * spread[0])
        kc[some], kp[some] = _pairs(codes), powers
        codes, powers = _packed(normal(number, kv, ps, dim) * spread[1])
        vc[some] = _pairs(codes).unflatten(-2, (-1, 8)).unflatten(-1, (-1, 4)).transpose(-3, -2)
        vp[some] = powers.unflatten(-2, (-1, 8)).transpose(-2, -1)
    tokens = sum(n for _, n in requests)
    # queries that prefer some keys: scores of a spread of about two
    qkv = torch.cat([normal(tokens, heads * dim), torch.zeros((tokens, 2 * kv * dim), device=DEVICE)], dim=1)
    return state | {
        "qkv": qkv.to(dtype), "pages": storage, "tables": tables, "scale": dim ** -0.5, "window": case["window"], "requests": requests, "decodes": case["decodes"],
        "contexts": ints([before + n for before, n in requests]), "starts": ints([0] + [sum(n for _, n in requests[:i + 1]) for i in range(len(requests))]),
        "positions": torch.cat([torch.arange(before, before + n, device=DEVICE) for before, n in requests]).int(),
        "sequence": torch.cat([torch.full((n,), i, device=DEVICE) for i, (_, n) in enumerate(requests)]).int(),
    }


# ---------------------------------------------------------------------------- plain forms


def _attend(q, pages, tables, contexts, state):
    """q float32 [R, n, heads, D], the last n tokens of R requests -> [R, n, heads * D]."""
    ps, dim, kv = state["page"], state["dim"], state["kv_heads"]
    count, n = q.shape[:2]
    keys, values = (x.transpose(1, 2).flatten(2, 3) for x in _rows(pages[tables.clamp(min=0).long()], ps, dim))  # [R, kv, keys, D]
    position = contexts[:, None] - n + torch.arange(n, device=q.device)
    key = torch.arange(keys.shape[2], device=q.device)
    seen = key <= position[..., None]
    if state["window"]:
        seen &= key > position[..., None] - state["window"]
    group = q.shape[2] // kv
    rows = q.view(count, n, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(count, kv, group * n, dim)
    scores = (rows @ keys.transpose(-2, -1).contiguous()).view(count, kv, group, n, -1) * state["scale"]
    scores = scores.masked_fill(~seen[:, None, None], -torch.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = (weights / weights.sum(-1, keepdim=True)).view(count, kv, group * n, -1)
    mixed = weights @ values.masked_fill(key[:, None] >= contexts[:, None, None, None], 0.0)
    return mixed.view(count, kv, group, n, dim).permute(0, 3, 1, 2, 4).reshape(count, n, -1)


def _plain_place(state):
    tables, slots, counts, starts, ps = state["tables"], state["slots"], state["counts"], state["starts"], state["page"]
    ends = counts.cumsum(0, dtype=torch.int32)
    query_start = torch.cat([ends.new_zeros(1), ends])
    token = torch.arange(state["tokens"], device=ends.device, dtype=torch.int32)
    sequence = torch.searchsorted(ends, token, right=True, out_int32=True)
    positions = starts[sequence] + token - query_start[sequence]
    page = tables[:, slots[sequence].long(), (positions // ps).long()]
    contexts = starts + counts
    mine = torch.arange(state["width"], device=ends.device) < ((contexts + ps - 1) // ps)[:, None]
    return [positions, sequence, query_start, contexts, torch.where(page < 0, -1, page * ps + positions % ps),
            torch.where(mine, tables[:, slots.long(), :state["width"]], -1)]


def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "place":
        return _plain_place(state)
    heads, kv, dim, dtype = state["heads"], state["kv_heads"], state["dim"], state["dtype"]
    if state["op"] == "store":
        keys, values = state["qkv"][:, heads * dim:].float().view(-1, 2, kv, dim).unbind(1)
        _write(state["pages"], state["slots"], keys, values, state["page"])
        page, offset = state["slots"].long() // state["page"], state["slots"].long() % state["page"]
        kc, vc, kp, vp = _fields(state["pages"], state["page"], dim)
        kept = (_values(kc[page, :, offset], kp[page, :, offset]),
                _values(vc[page, :, offset // 8, :, offset % 8].flatten(-2), vp[page, :, offset // 8, :, offset % 8]))
        return [torch.where((state["slots"] < 0)[:, None, None], 0.0, x).to(dtype) for x in kept]
    q = state["qkv"][:, :heads * dim].float().view(-1, heads, dim)
    singles, out = state["decodes"], []
    if singles:
        out.append(_attend(q[:singles].unsqueeze(1), state["pages"], state["tables"][:singles], state["contexts"][:singles], state).flatten(0, 1))
    if q.shape[0] > singles:
        out.append(_attend(q[singles:].unsqueeze(0), state["pages"], state["tables"][singles:], state["contexts"][singles:], state).flatten(0, 1))
    return torch.cat(out).to(dtype)


# ---------------------------------------------------------------------------- the framework's operators

_LIBRARIES = {}  # a program keeps one kernel library a run dtype


def _library(dtype):
    if dtype not in _LIBRARIES:
        from llmserve_amd.kernels import HipKernels

        _LIBRARIES[dtype] = HipKernels(dtype, DEVICE)
    return _LIBRARIES[dtype]


def _step(state):
    """The step's batch, the layer's cell and the rows' layout, which an engine makes once a step and not once a layer."""
    if "step" not in state:
        from llmserve_amd.cache import CacheCell
        from llmserve_amd.engine.batch import GroupBatch, SequenceChunk, StepBatch
        from llmserve_amd.parts import HeadLayout, PackedKeyValue

        none = torch.zeros(0, dtype=torch.int32, device=DEVICE)
        tokens = state["qkv"].shape[0]
        requests = state.get("requests", [(0, tokens)])
        group = GroupBatch(state["page"], state.get("tables", none), state.get("slots", none), state["tables"].shape[1] if "tables" in state else 0)
        batch = StepBatch(
            num_tokens=tokens, chunks=[SequenceChunk(str(i), i, before, n) for i, (before, n) in enumerate(requests)], token_ids=none,
            positions=state.get("positions", none), token_sequence=state.get("sequence", none), query_start=state.get("starts", none),
            context_lengths=state.get("contexts", none), state_slots=none, groups=[group], logit_rows=none, num_logit_rows=0,
            max_query_length=max(n for _, n in requests), max_context_length=max(before + n for before, n in requests),
        )
        need = PackedKeyValue(state["kv_heads"], state["dim"], state.get("window") or None)
        state["step"] = batch, CacheCell(need, fields={"packed": state["pages"]}, group=0), HeadLayout(state["heads"], state["kv_heads"], state["dim"])
    return state["step"]


def _run_own(state):
    if state["op"] == "place":
        kernels = _library(torch.bfloat16)
        return list(kernels.place_tokens(state["tables"], state["slots"], state["starts"], state["counts"], state["page"], state["tokens"], state["width"]))
    kernels = _library(state["dtype"])
    batch, cell, layout = _step(state)
    if state["op"] == "store":
        kernels.store_packed(state["qkv"], layout, batch, cell)
        return list(kernels.packed_rows(cell, state["slots"], state["page"]))
    return kernels.paged_attention(state["qkv"], layout, batch, cell, state["scale"], state["window"] or None)


# ---------------------------------------------------------------------------- 64 bits


def _exact_block(x):
    """What is kept of float64 [..., 32], from the definition: the nearest of the sixteen numbers times the block's power."""
    largest = x.abs().amax(-1, keepdim=True)
    significand, exponent = torch.frexp(largest)  # largest = significand * 2^exponent, 0.5 <= significand < 1
    exponent = exponent + (significand >= 0.875) - 1 - 2
    unit = torch.ldexp(torch.ones_like(largest), exponent.clamp(-125, 125))
    size = (x / unit).abs().clamp(max=6.0)
    step = torch.where(size < 2.0, 0.5, torch.where(size < 4.0, 1.0, 2.0)).to(x.dtype)
    return torch.copysign(torch.round(size / step) * step, x) * unit  # (a tie goes to the even multiple of the step, which is the even code)


def _exact_rows(pages, page, ps, dim):
    """Pages `page` [n] as keys and values float64 [kv, n * ps, D], taken apart byte by byte."""
    data = pages[page.long()].transpose(0, 1)  # [kv, n, bytes]
    n, a, b = page.shape[0], ps * dim // 2, ps * dim // 32
    number = lambda c: (1 - 2 * (c >> 3).double()) * torch.where((c & 6) == 0, (c & 1).double() / 2, (1 + (c & 1).double() / 2) * torch.exp2(((c >> 1) & 3).double() - 1))
    keys = data[..., :a].reshape(-1, n * ps, dim // 2, 1)
    keys = number(torch.cat([keys & 15, keys >> 4], -1)).view(-1, n * ps, dim // 32, 32)
    keys = keys * torch.exp2(data[..., 2 * a:2 * a + b].reshape(-1, n * ps, dim // 32, 1).double() - 127)
    values = data[..., a:2 * a].reshape(-1, n, ps // 8, dim // 8, 8, 4, 1)
    values = number(torch.cat([values & 15, values >> 4], -1)).permute(0, 1, 2, 4, 3, 5, 6).reshape(-1, n * ps, dim // 32, 32)
    power = data[..., 2 * a + b:].reshape(-1, n, ps // 8, dim // 32, 8).transpose(-2, -1).reshape(-1, n * ps, dim // 32, 1)
    return keys.flatten(-2), (values * torch.exp2(power.double() - 127)).flatten(-2)


def _exact_place(case, state):
    """The arrays as a host program writes them down, request by request."""
    requests, ps, tables, slots = _requests(case), case["page"], state["tables"].tolist(), state["slots"].tolist()
    token, ends, compact = [], [0], [[] for _ in tables]
    for b, (before, n) in enumerate(requests):
        token += [(before + i, b, [rows[slots[b]][(before + i) // ps] * ps + (before + i) % ps for rows in tables]) for i in range(n)]
        ends.append(len(token))
        held = -(-(before + n) // ps)
        for mine, rows in zip(compact, tables):
            mine.append(rows[slots[b]][:held] + [-1] * (state["width"] - held))
    found = [[p for p, _, _ in token], [b for _, b, _ in token], ends, [before + n for before, n in requests], [[s[g] for _, _, s in token] for g in range(len(tables))], compact]
    return [torch.tensor(x, dtype=torch.int32, device=DEVICE) for x in found]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "place":
        return _exact_place(case, state)
    heads, kv, dim, ps = case["heads"], case["kv_heads"], case["dim"], case["page"]
    rows = state["qkv"].double()
    if case["op"] == "store":
        found = [_exact_block(x.reshape(-1, kv, dim // 32, 32)).flatten(-2) for x in (rows[:, heads * dim:(heads + kv) * dim], rows[:, (heads + kv) * dim:])]
        return [torch.where((state["slots"] >= 0)[:, None, None], x, 0.0) for x in found]
    out, first = [], 0
    for i, (before, n) in enumerate(_requests(case)):
        length = before + n
        keys, values = (x[:, :length] for x in _exact_rows(state["pages"], state["tables"][i, :-(-length // ps)], ps, dim))
        mine = rows[first:first + n, :heads * dim].view(n, heads, dim)
        first += n
        mixed = torch.empty((n, heads, dim), dtype=torch.float64, device=rows.device)
        distance = torch.arange(before, length, device=rows.device)[:, None] - torch.arange(length, device=rows.device)
        hidden = (distance < 0) | (distance >= (case["window"] or length))
        for h in range(heads):
            scores = (mine[:, h].contiguous() @ keys[h // (heads // kv)].t().contiguous()) * state["scale"]
            mixed[:, h] = torch.softmax(scores.masked_fill_(hidden, -torch.inf), -1) @ values[h // (heads // kv)].contiguous()
        out.append(mixed.flatten(1))
    return torch.cat(out)

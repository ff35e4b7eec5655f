"""Cases and plain forms of the operators around K/V rows held in 8 bits, for measuring them.

Four operators (Backend methods of straydog_b200.backend):

  kv8_write         new keys and values of a batch of sequences into states of 8-bit rows that share one scale a block of 32 positions and head
  kv8_attention     queries over such states, one row a sequence (decode), a few (verification) or a prompt chunk; scores capped by a tanh,
                    biased by distance, limited to a window, opened over a prefix; optionally the keys' attention weights added up
  masked_attention  the same attention over 16-bit keys and values of packed documents
  kv8_evict         the rows that hold the least accumulated attention weight left out, the others moved together into a new state

The definition they share. Row i of a sequence of `length` keys and `rows` queries sits at position p = length - rows + i (below 0: before the
first key). It sees key j < length when j <= p and (no window, or j > p - window), or when j < prefix. Score: s = scale * q . k, then
s = cap * tanh(s / cap) when cap > 0, then s -= slope[head] * |p - j| when there are slopes. Out = softmax(s) . v over the seen keys, zeros
where none is seen. A code c of a block with scale s stands for c * s; the scale is the largest magnitude / 127 (int8) or / 448 (e4m3). Rows
appended to a begun block keep its scale unless they need a larger one; then the block's older codes are rounded again in the new scale.
"""
import functools
import math

import numpy as np
import torch

own = False

BLOCK = 32
TOP = {"int8": 127.0, "e4m3": 448.0}
TYPE = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---- the cases ----

def _case(op, **given):
    base = {
        "write": dict(sequences=1, context=1024, rows=1, kv_heads=2, dim=256, code="int8", dtype="f16"),
        "cached": dict(sequences=1, context=1024, rows=1, heads=16, kv_heads=2, dim=256, code="int8", dtype="f16", cap=0.0, bias=False,
                       window=0, prefix=0, weights=False),
        "masked": dict(documents=1, rows=64, past=0, heads=16, kv_heads=2, dim=256, dtype="bf16", cap=0.0, bias=False, window=0, prefix=0),
        "evict": dict(sequences=1, context=2048, keep=1024, sinks=4, recent=128, kv_heads=2, dim=256, code="int8"),
    }[op]
    return {"op": op, **base, **given}


def listed():
    return [
        # a decode step's append of a running batch: one row a sequence, into blocks that are partly filled
        _case("write", name="append 32 x 1", sequences=32, context=4096, rows=1, kv_heads=8, dim=128, dtype="bf16"),
        # a long prompt chunk of a model with two wide K/V heads, from a position inside a block
        _case("write", name="write 8191 rows", context=32768, rows=8191, kv_heads=2, dim=256, code="e4m3", dtype="f16"),
        # one user's token early in a conversation: latency
        _case("cached", name="decode 1 x 1000", context=1000),
        # the framework's headline batch: 64 ragged sequences of up to 32768 positions, one token each
        _case("cached", name="decode 64 x 32768", sequences=64, context=32768),
        # a layer with capped scores and a sliding window, a small batch
        _case("cached", name="decode 8 capped window", sequences=8, context=16384, heads=32, kv_heads=8, dim=128, code="e4m3", dtype="bf16",
              cap=50.0, window=4095),
        # verification rows of 16 sequences, scores biased by distance, weights added up for a later eviction
        _case("cached", name="verify 16 x 4 weights", sequences=16, context=8192, rows=4, heads=32, kv_heads=8, dim=128, dtype="bf16", bias=True,
              weights=True),
        # a prompt chunk behind cached positions, with a prefix (an instruction, an image) that every row sees
        _case("cached", name="chunk 2048 of 8192", context=8192, rows=2048, heads=32, kv_heads=8, dim=128, dtype="bf16", prefix=700),
        # many short documents packed in one call (a re-ranker's batch), distance bias
        _case("masked", name="documents 24 short", documents=24, rows=64, heads=8, kv_heads=8, dim=64, dtype="f16", bias=True),
        # ordinary prompts of several users packed in one call: about 8 thousand tokens
        _case("masked", name="documents 7 of 2100", documents=7, rows=2100, heads=32, kv_heads=8, dim=128),
        # a chunk of a long document behind 16-bit keys and values, capped scores, wide heads
        _case("masked", name="chunk 4096 after 12288", rows=4096, past=12288, cap=30.0),
        # one conversation brought back to its budget
        _case("evict", name="evict 1 x 2047", context=2047, keep=1024),
        # a batch of long sequences halved
        _case("evict", name="evict 16 x 16384", sequences=16, context=16384, keep=8191, recent=1024, kv_heads=8, dim=128, code="e4m3"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(16, 2, 256), (24, 2, 256), (32, 8, 128), (16, 16, 64), (8, 1, 128), (12, 4, 64), (4, 4, 256)])
    code, dtype = rng.choice(["int8", "e4m3"]), rng.choice(["f16", "bf16"])
    rule = dict(cap=rng.choice([0.0, 0.0, 20.0, 50.0]), bias=rng.random() < 0.3)
    op = rng.choice(["write", "cached", "cached", "prompt", "masked", "masked", "evict"])
    if op == "write":
        rows = rng.choice([1, _log(rng, 1, 16), _log(rng, 16, 8192)])
        context = max(rows + 40, _log(rng, 64, 16384))
        many = max(1, min(64, (1 << 24) // (context * kv_heads * dim // 16)))
        return _case("write", sequences=_log(rng, 1, many), context=context, rows=rows, kv_heads=kv_heads, dim=dim, code=code,
                     dtype=rng.choice(["f32", "f16", "bf16"]))
    if op == "cached":
        context = _log(rng, 2, 32768)
        many = max(1, min(64, (1 << 29) // (context * kv_heads * dim)))
        rows = rng.choice([1, 1, 1, rng.randint(2, 8)])
        return _case("cached", sequences=_log(rng, 1, many), context=context, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, code=code,
                     dtype=dtype, window=rng.choice([0, 0, _log(rng, 1, context)]), prefix=rng.choice([0, 0, rng.randint(0, context)]),
                     weights=rng.random() < 0.3 and rows * (heads // kv_heads) <= 16, **rule)
    if op == "prompt":
        rows = _log(rng, 9, 2048)
        context = _log(rng, max(rows // 2, 2), 8192)
        return _case("cached", sequences=rng.choice([1, 2, 3]), context=context, rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, code=code,
                     dtype=dtype, window=rng.choice([0, 0, _log(rng, 1, context)]), prefix=rng.choice([0, 0, rng.randint(0, context)]), **rule)
    if op == "masked":
        rows = _log(rng, 1, 4096)
        documents = _log(rng, 1, max(1, min(64, 6000 // rows)))
        past = rng.choice([0, 0, _log(rng, 1, max(2, 8192 // documents))])
        return _case("masked", documents=documents, rows=rows, past=past, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                     window=rng.choice([0, 0, _log(rng, 1, rows + past)]), prefix=rng.choice([0, 0, rng.randint(0, rows + past)]), **rule)
    context = _log(rng, 64, 32768)
    keep = _log(rng, 2, context - 1)
    many = max(1, min(32, (1 << 28) // (context * kv_heads * dim)))
    return _case("evict", sequences=_log(rng, 1, many), context=context, keep=keep, sinks=rng.randint(0, min(8, keep // 2)),
                 recent=rng.randint(0, keep // 2), kv_heads=kv_heads, dim=dim, code=code)


def _part(i, salt):
    """A fixed fraction in [0, 1) for sequence i: the ragged sizes of a case, the same for every seed."""
    return ((i + 1) * 0.6180339887498949 + salt * 0.3490731) % 1.0


def _sizes(case):
    """Sequences' (rows, lengths, prefixes); the first sequence has the largest sizes."""
    if case["op"] == "masked":
        n = case["documents"]
        rows = [case["rows"] if i == 0 else 1 + int((case["rows"] - 1) * _part(i, 1)) for i in range(n)]
        past = [case["past"] if i == 0 else int(case["past"] * _part(i, 2)) for i in range(n)]
        lengths = [r + p for r, p in zip(rows, past)]
    else:
        n = case["sequences"]
        rows = [case["rows"] if i == 0 or case["op"] != "cached" else 1 + int((case["rows"] - 1) * _part(i, 1)) for i in range(n)]
        lengths = [case["context"] if i == 0 else max(1, int(case["context"] * (0.1 + 0.9 * _part(i, 2)))) for i in range(n)]
    prefixes = [min(case["prefix"] if i == 0 else int(case["prefix"] * _part(i, 3)), lengths[i]) for i in range(n)] if "prefix" in case else None
    return rows, lengths, prefixes


def _bases(case):
    """Where a write's rows begin: anywhere they fit."""
    room = case["context"] - case["rows"]
    return [int(room * (0.25 + 0.7 * _part(i, 4))) for i in range(case["sequences"])]


def _kept_sizes(case):
    """An eviction's lengths: every sequence holds more than is kept."""
    keep, room = case["keep"], case["context"] - case["keep"]
    return [case["context"] if i == 0 else keep + 1 + int((room - 1) * _part(i, 2)) for i in range(case["sequences"])]


def _rounded(context):
    return -(-context // BLOCK) * BLOCK


# ---- a state: 2 * kv_heads planes (keys, then values) of `context` rows of `dim` codes, then the planes' block scales (F32) ----

def _state_bytes(context, kv_heads, dim):
    return -(-2 * kv_heads * (context * dim + context // BLOCK * 4) // 16) * 16


def _codes(states, case):
    """The codes of a batch's states as [sequences, planes, context, dim], in the type they are held in."""
    planes, context, dim = 2 * case["kv_heads"], _rounded(case["context"]), case["dim"]
    held = torch.int8 if case["code"] == "int8" else torch.float8_e4m3fn
    return states[:, : planes * context * dim].view(held).view(-1, planes, context, dim)


def _scales(states, case):
    planes, context, dim = 2 * case["kv_heads"], _rounded(case["context"]), case["dim"]
    return states[:, planes * context * dim: planes * (context * dim + context // BLOCK * 4)].view(torch.float32).view(-1, planes, context // BLOCK)


def _encode(x, code):
    return torch.round(x).clamp(-127, 127).to(torch.int8) if code == "int8" else x.clamp(-448, 448).to(torch.float8_e4m3fn)


def _over(x, scale):
    """x / scale, 0 under a zero scale."""
    return torch.where(scale > 0, x / torch.where(scale > 0, scale, torch.ones_like(scale)), torch.zeros_like(x))


def _made_states(case, g, lengths):
    """States filled as a run of the model fills them: normal values, some channels of the keys much larger than the rest."""
    planes, context, dim, code = 2 * case["kv_heads"], _rounded(case["context"]), case["dim"], case["code"]
    states = torch.zeros(len(lengths), _state_bytes(context, case["kv_heads"], dim), dtype=torch.uint8, device="cuda")
    codes, scales = _codes(states, case), _scales(states, case)
    channel = torch.exp(0.6 * torch.randn(planes, 1, dim, generator=g, device="cuda"))
    top = torch.tensor(TOP[code], device="cuda")
    for s, length in enumerate(lengths):
        filled = _rounded(length)
        x = torch.randn(planes, filled, dim, generator=g, device="cuda") * channel
        x[:, length:] = 0
        blocks = x.view(planes, filled // BLOCK, BLOCK, dim)
        scale = blocks.abs().amax((2, 3)) / top
        codes[s, :, :filled] = _encode(_over(blocks, scale[:, :, None, None]), code).view(planes, filled, dim)
        scales[s, :, : filled // BLOCK] = scale
    return states


def _pointers(t):
    """The addresses of t's parts along its first axis, as the calls take them."""
    return np.asarray([t.data_ptr() + i * t.stride(0) * t.element_size() for i in range(t.shape[0])], np.uint64)


def _counts(values):
    return np.asarray(values, np.uint64)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dim, kv_heads = case["op"], case["dim"], case["kv_heads"]
    normal = lambda *shape, dtype: torch.randn(*shape, generator=g, device="cuda").to(TYPE[dtype])  # noqa: E731
    st = {"case": case}
    if op == "write":
        n, rows, bases = case["sequences"], case["rows"], _bases(case)
        st["states"] = _made_states(case, g, bases)
        st["keys"], st["values"] = (1.3 * normal(n * rows, kv_heads, dim, dtype=case["dtype"]) for _ in range(2))
        st["bases"], st["base_at"] = _counts(bases), torch.tensor(bases, device="cuda")
        st["steps"] = _counts([rows] * n)
    elif op == "cached":
        rows, lengths, prefixes = _sizes(case)
        n, heads = case["sequences"], case["heads"]
        st["states"] = _made_states(case, g, lengths)
        st["q"] = normal(sum(rows), heads, dim, dtype=case["dtype"])
        st["out"] = torch.empty_like(st["q"])
        # weights come with the history of the steps before
        st["weights"] = 4 * torch.rand(n, kv_heads, _rounded(case["context"]), generator=g, device="cuda") if case["weights"] else None
        st["weights_at"] = _pointers(st["weights"]) if case["weights"] else None
        st["rows"], st["lengths"] = _counts(rows), _counts(lengths)
    elif op == "masked":
        rows, lengths, prefixes = _sizes(case)
        heads, total, keys = case["heads"], sum(rows), sum(lengths)
        if case["past"] == 0:   # queries, keys and values are parts of one projection's rows
            fused = normal(total, (heads + 2 * kv_heads) * dim, dtype=case["dtype"])
            q, k, v = fused.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
            st["q"], st["k"], st["v"] = q.unflatten(1, (heads, dim)), k.unflatten(1, (kv_heads, dim)), v.unflatten(1, (kv_heads, dim))
        else:
            st["q"] = normal(total, heads, dim, dtype=case["dtype"])
            st["k"], st["v"] = (normal(keys, kv_heads, dim, dtype=case["dtype"]) for _ in range(2))
        st["out"] = torch.empty(total, heads, dim, dtype=TYPE[case["dtype"]], device="cuda")
        st["rows"], st["lengths"] = _counts(rows), _counts(lengths)
    else:
        lengths, n, kept = _kept_sizes(case), case["sequences"], _rounded(case["keep"])
        st["states"] = _made_states(case, g, lengths)
        st["lengths"] = _counts(lengths)
        # what attention leaves: a few keys with most of the weight, ties among the rest (weights that were never more than rounding)
        w = torch.rand(n, kv_heads, _rounded(case["context"]), generator=g, device="cuda")
        st["weights"] = torch.where(w < 0.2, torch.zeros_like(w), torch.exp(6 * w) / 64)
        st["targets"] = torch.zeros(n, _state_bytes(kept, kv_heads, dim), dtype=torch.uint8, device="cuda")
        st["target_weights"] = torch.zeros(n, kv_heads, kept, device="cuda")
        st["kept"] = torch.zeros(n, kv_heads, case["keep"], dtype=torch.int32, device="cuda")
        st["weights_at"], st["targets_at"], st["target_weights_at"] = (_pointers(st[k]) for k in ("weights", "targets", "target_weights"))
        st["target_contexts"] = _counts([kept] * n)
    if op in ("cached", "masked"):
        st["prefixes"] = _counts(prefixes) if case["prefix"] else None
        st["slopes"] = torch.exp2(-8 * (1 + torch.arange(case["heads"], device="cuda")) / case["heads"]).float() if case["bias"] else None
        # the rows' and keys' places, for the plain form
        device = dict(device="cuda")
        r, ln = torch.tensor(rows, **device), torch.tensor(lengths, **device)
        st["row_of"] = torch.repeat_interleave(torch.arange(len(rows), **device), r)
        st["row_at"] = torch.arange(sum(rows), **device) - (r.cumsum(0) - r)[st["row_of"]]
        st["row_position"] = st["row_at"] + (ln - r)[st["row_of"]]
        st["prefix_of"], st["length_of"] = torch.tensor(prefixes, **device), ln
    if "states" in st:
        st["states_at"] = _pointers(st["states"])
        st["contexts"] = _counts([_rounded(case["context"])] * case["sequences"])
    return st


# ---- the framework's calls ----

@functools.lru_cache(maxsize=None)
def _backend(device, stream):   # (the default stream is 0 on every device)
    from straydog_b200.backend import Backend
    return Backend.adopt(device, stream)


def _own(st):
    from straydog_b200 import backend as b
    case = st["case"]
    gpu = _backend(torch.cuda.current_device(), torch.cuda.current_stream().cuda_stream)
    kind = {"f32": b.F32, "f16": b.F16, "bf16": b.BF16}.get(case.get("dtype"))
    code = {"int8": b.INT8, "e4m3": b.E4M3}.get(case.get("code"))
    op, kv_heads, dim = case["op"], case["kv_heads"], case["dim"]
    if op == "write":
        gpu.kv8_write(st["states_at"], st["contexts"], st["bases"], st["steps"], kv_heads, dim, code, st["keys"].data_ptr(),
                      st["values"].data_ptr(), kind)
        return {"codes": _codes(st["states"], case), "scales": _scales(st["states"], case)}
    slopes = st["slopes"].data_ptr() if st.get("slopes") is not None else None
    if op == "cached":
        gpu.kv8_attention(st["states_at"], st["contexts"], st["lengths"], st["rows"], case["heads"], kv_heads, dim, code, 1 / math.sqrt(dim),
                          st["q"].data_ptr(), st["out"].data_ptr(), kind, cap=case["cap"], slopes=slopes, window=case["window"],
                          prefixes=st["prefixes"], weights=st["weights_at"])
        return {"out": st["out"], "weights": st["weights"]}
    if op == "masked":
        gpu.masked_attention(st["q"].data_ptr(), st["k"].data_ptr(), st["v"].data_ptr(), st["out"].data_ptr(), st["rows"], st["lengths"],
                             case["heads"], kv_heads, dim, kind, 1 / math.sqrt(dim), cap=case["cap"], slopes=slopes, window=case["window"],
                             prefixes=st["prefixes"], q_stride=st["q"].stride(0), k_stride=st["k"].stride(0), v_stride=st["v"].stride(0))
        return {"out": st["out"]}
    gpu.kv8_evict(st["states_at"], st["contexts"], st["lengths"], st["weights_at"], case["keep"], case["sinks"], case["recent"], kv_heads, dim,
                  code, st["targets_at"], st["target_contexts"], st["target_weights_at"], st["kept"].data_ptr())
    return _evicted(st)


def _evicted(st):
    case, keep = st["case"], st["case"]["keep"]
    target = {**case, "context": keep}
    return {"codes": _codes(st["targets"], target)[:, :, :keep], "scales": _scales(st["targets"], target),
            "weights": st["target_weights"][:, :, :keep], "kept": st["kept"]}


# ---- the plain forms ----

def _plain_write(st):
    case = st["case"]
    n, rows, planes, dim, code = case["sequences"], case["rows"], 2 * case["kv_heads"], case["dim"], case["code"]
    codes, scales = _codes(st["states"], case), _scales(st["states"], case)
    base = st["base_at"]
    first = base // BLOCK
    blocks = (BLOCK - 1 + rows + BLOCK - 1) // BLOCK
    at_block = (first[:, None] + torch.arange(blocks, device="cuda")).clamp(max=scales.shape[2] - 1)       # [n, blocks]
    local = torch.arange(blocks * BLOCK, device="cuda") - (base - first * BLOCK)[:, None]                   # row of the call, or outside it
    new = ((local >= 0) & (local < rows)).view(n, 1, blocks, BLOCK, 1)
    given = torch.cat([st["keys"], st["values"]], 1).float().view(n, rows, planes, dim)
    x = given.gather(1, local.clamp(0, rows - 1)[:, :, None, None].expand(-1, -1, planes, dim)).permute(0, 2, 1, 3)
    x = x.reshape(n, planes, blocks, BLOCK, dim)
    need = torch.where(new, x.abs(), torch.zeros_like(x)).amax((3, 4)) / torch.tensor(TOP[code], device="cuda")
    seq, plane = torch.arange(n, device="cuda")[:, None, None], torch.arange(planes, device="cuda")[None, :, None]
    old = scales[seq, plane, at_block[:, None, :]]
    begun = ((at_block * BLOCK < base[:, None]) & (torch.arange(blocks, device="cuda") == 0))[:, None, :]   # a block with older rows
    touched = new.any(3).view(n, 1, blocks)
    scale = torch.where(begun, torch.maximum(old, need), need)
    row = (at_block[:, :, None] * BLOCK + torch.arange(BLOCK, device="cuda")).view(n, 1, -1)
    held = codes.view(torch.uint8)[seq, plane, row].view(codes.dtype)
    again = held.float().view(x.shape) * _over(old, scale)[..., None, None]
    older = begun[..., None, None] & (local < 0).view(n, 1, blocks, BLOCK, 1)
    fresh = torch.where(new, _encode(_over(x, scale[..., None, None]), code).float(), held.float().view(x.shape))
    fresh = torch.where(older, _encode(again, code).float(), fresh).to(codes.dtype).view(n, planes, blocks * BLOCK, dim)
    keep = touched.expand(n, planes, blocks)
    where = keep.nonzero(as_tuple=True)
    scales[where[0], where[1], at_block[where[0], where[2]]] = scale[where]
    by_block = codes.view(torch.uint8).view(n, planes, -1, BLOCK, dim)
    by_block[where[0], where[1], at_block[where[0], where[2]]] = fresh.view(torch.uint8).view(n, planes, blocks, BLOCK, dim)[where]
    return {"codes": codes, "scales": scales}


def _plain_softmax(s, seen, v_of):
    """softmax over the seen keys (last axis of s), zeros where none is; v_of(p): the products with the values. (out, p)"""
    s = s.masked_fill_(~seen, -math.inf)
    m = s.amax(-1, keepdim=True).clamp(min=-3e38)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    return v_of(p), p


def _plain_rule(s, case, slopes, distance):
    if case["cap"]:
        s = s.div_(case["cap"]).tanh_().mul_(case["cap"])
    if slopes is not None:
        s = s.sub_(slopes * distance)
    return s


def _plain_seen(position, key, length, prefix, window):
    seen = key <= position
    if window:
        seen = seen & (key > position - window)
    return (seen | (key < prefix)) & (key < length)


def _plain_cached(st):
    case = st["case"]
    n, heads, kv_heads, dim, most = case["sequences"], case["heads"], case["kv_heads"], case["dim"], case["rows"]
    group, context = heads // kv_heads, _rounded(case["context"])
    blocks = _codes(st["states"], case).float().view(n, 2 * kv_heads, -1, BLOCK, dim)
    kv = blocks.mul_(_scales(st["states"], case)[..., None, None]).view(n, 2, kv_heads, context, dim)
    q = torch.zeros(n, most, heads, dim, device="cuda")
    q[st["row_of"], st["row_at"]] = st["q"].float()
    position = torch.full((n, most), -1, device="cuda")
    position[st["row_of"], st["row_at"]] = st["row_position"]
    q = q.view(n, most, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv_heads, group * most, dim)
    s = (q @ kv[:, 0].transpose(2, 3)).mul_(1 / math.sqrt(dim)).view(n, kv_heads, group, most, context)
    key = torch.arange(context, device="cuda")
    at = position[:, None, None, :, None]
    slopes = st["slopes"].view(1, kv_heads, group, 1, 1) if st["slopes"] is not None else None
    s = _plain_rule(s, case, slopes, (at - key).abs())
    real = torch.zeros(n, most, dtype=torch.bool, device="cuda")
    real[st["row_of"], st["row_at"]] = True
    seen = _plain_seen(at, key, st["length_of"].view(n, 1, 1, 1, 1), st["prefix_of"].view(n, 1, 1, 1, 1), case["window"])
    out, p = _plain_softmax(s, seen & real[:, None, None, :, None], lambda p: p.view(n, kv_heads, group * most, context) @ kv[:, 1])
    if st["weights"] is not None:
        st["weights"] += p.sum((2, 3))
    out = out.view(n, kv_heads, group, most, dim).permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)
    st["out"].copy_(out[st["row_of"], st["row_at"]])
    return {"out": st["out"], "weights": st["weights"]}


def _plain_masked(st):
    case = st["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    group, total = heads // kv_heads, st["q"].shape[0]
    lengths = st["length_of"]
    key_of = torch.repeat_interleave(torch.arange(len(lengths), device="cuda"), lengths)
    key_at = torch.arange(key_of.numel(), device="cuda") - (lengths.cumsum(0) - lengths)[key_of]
    q = st["q"].float().view(total, kv_heads, group, dim).permute(1, 2, 0, 3).reshape(kv_heads, group * total, dim)
    k, v = st["k"].float().transpose(0, 1), st["v"].float().transpose(0, 1)
    s = (q @ k.transpose(1, 2)).mul_(1 / math.sqrt(dim)).view(kv_heads, group, total, -1)
    at = st["row_position"][:, None]
    slopes = st["slopes"].view(kv_heads, group, 1, 1) if st["slopes"] is not None else None
    s = _plain_rule(s, case, slopes, (at - key_at).abs() if slopes is not None else None)
    seen = _plain_seen(at, key_at, lengths[key_of], st["prefix_of"][key_of], case["window"]) & (st["row_of"][:, None] == key_of)
    out, _ = _plain_softmax(s, seen, lambda p: p.view(kv_heads, group * total, -1) @ v)
    st["out"].copy_(out.view(kv_heads, group, total, dim).permute(2, 0, 1, 3).reshape(total, heads, dim))
    return {"out": st["out"]}


def _plain_evict(st):
    case, keep, code = st["case"], st["case"]["keep"], st["case"]["code"]
    n, kv_heads, dim, kept = case["sequences"], case["kv_heads"], case["dim"], _rounded(case["keep"])
    lengths = torch.tensor(st["lengths"].astype(np.int64), device="cuda")[:, None, None]
    key = torch.arange(st["weights"].shape[2], device="cuda")
    always = (key < case["sinks"]) | ((key >= lengths - case["recent"]) & (key < lengths))
    order = torch.where(always, math.inf, st["weights"].masked_fill(key >= lengths, -math.inf))
    at = torch.sort(order, dim=2, descending=True, stable=True).indices[:, :, :keep].sort(dim=2).values           # [n, kv_heads, keep]
    st["kept"].copy_(at)
    st["target_weights"][:, :, :keep] = st["weights"].gather(2, at)
    at = at.repeat(1, 2, 1)                                                                                       # keys, then values
    held = _codes(st["states"], case).view(torch.uint8)
    moved = held.gather(2, at[..., None].expand(-1, -1, -1, dim)).view(_codes(st["states"], case).dtype).float()
    from_scale = _scales(st["states"], case).gather(2, at // BLOCK)
    padded = torch.nn.functional.pad(from_scale, (0, kept - keep)).view(n, 2 * kv_heads, kept // BLOCK, BLOCK)
    scale = padded.amax(3)
    again = moved * _over(from_scale, scale.repeat_interleave(BLOCK, 2)[:, :, :keep])[..., None]
    target = {**case, "context": keep}
    _codes(st["targets"], target).view(torch.uint8)[:, :, :keep] = _encode(again, code).view(torch.uint8)
    _scales(st["targets"], target).copy_(scale)
    return _evicted(st)


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "cached": _plain_cached, "masked": _plain_masked, "evict": _plain_evict}[state["case"]["op"]](state)


# ---- what a pass has to read, write and compute ----

def _seen_count(rows, length, window, prefix):
    """Seen (row, key) pairs of one sequence and head, and the keys that any row sees."""
    p = np.arange(length - rows, length, dtype=np.int64)
    low = np.maximum(p - window + 1, 0) if window else np.zeros_like(p)
    causal = np.where(p >= 0, p + 1 - np.minimum(low, p + 1), 0)
    both = np.clip(np.minimum(prefix, p + 1) - low, 0, None) * (p >= 0)
    first = int(low[p >= 0][0]) if (p >= 0).any() else length
    return int((causal + prefix - both).sum()), (length - first) + min(prefix, first)


def work(case):
    op, kv_heads, dim = case["op"], case["kv_heads"], case["dim"]
    if op == "write":
        rows = case["sequences"] * case["rows"] * 2 * kv_heads * dim
        # (the new rows read and written; the begun blocks' older rows only change when their scale grows: not counted)
        return {"bytes": rows * ({"f32": 4}.get(case["dtype"], 2) + 1) + rows // dim * 4 // BLOCK, "flops": 2 * rows}
    if op == "evict":
        lengths, n, keep = _kept_sizes(case), case["sequences"], case["keep"]
        moved = n * 2 * kv_heads * keep * dim
        return {"bytes": 2 * moved + sum(lengths) * kv_heads * 4 + n * kv_heads * keep * 8 + 2 * moved // dim // BLOCK * 4, "flops": moved}
    rows, lengths, prefixes = _sizes(case)
    counts = [_seen_count(r, n, case["window"], p) for r, n, p in zip(rows, lengths, prefixes)]
    pairs, keys = sum(c[0] for c in counts), sum(c[1] for c in counts)
    q = 2 * 2 * sum(rows) * case["heads"] * dim
    if op == "cached":
        weights = 8 * keys * kv_heads if case["weights"] else 0
        return {"bytes": q + keys * 2 * kv_heads * (dim + 4 / BLOCK) + weights, "flops": 4 * pairs * case["heads"] * dim}
    return {"bytes": q + keys * 2 * kv_heads * dim * 2, "flops": 4 * pairs * case["heads"] * dim}


# ---- the definition in 64 bits, sequence by sequence ----

def _exact_attention(q, k, v, case, slopes, prefix):
    """q [rows, heads, dim], k and v [length, kv_heads, dim], all in 64 bits: (out, the weights' sums over rows and a K/V head's queries)."""
    rows, heads, dim = q.shape
    length, kv_heads = k.shape[0], k.shape[1]
    out, sums = torch.zeros_like(q), torch.zeros(kv_heads, length, dtype=torch.float64, device="cuda")
    i, j = torch.arange(rows, device="cuda")[:, None] + (length - rows), torch.arange(length, device="cuda")[None, :]
    open_ = (j <= i) & ((i - j < case["window"]) if case["window"] else True) | (j < prefix)
    for h in range(heads):
        kv = h * kv_heads // heads
        z = q[:, h] @ k[:, kv].T / math.sqrt(dim)
        if case["cap"]:
            z = torch.tanh(z / case["cap"]) * case["cap"]
        if slopes is not None:
            z = z - slopes[h].double() * (i - j).abs()
        e = torch.where(open_, z - torch.where(open_, z, -math.inf).max(1, keepdim=True).values.nan_to_num(neginf=0.0), -math.inf).exp()
        d = e.sum(1, keepdim=True)
        e = torch.where(d > 0, e / d, 0.0)
        out[:, h] = e @ v[:, kv]
        sums[kv] += e.sum(0)
    return out, sums


def exact(case, seed):
    st = prepare(case, seed)
    op, kv_heads, dim = case["op"], case["kv_heads"], case["dim"]
    if op in ("cached", "masked"):
        rows, lengths, prefixes = _sizes(case)
        row, key, outs = 0, 0, []
        weights = st["weights"].double() if st.get("weights") is not None else None
        for s, (r, n) in enumerate(zip(rows, lengths)):
            if op == "cached":
                c = _codes(st["states"], case)[s, :, :n].to(torch.float32).double()
                kv = c * _scales(st["states"], case)[s].double().repeat_interleave(BLOCK, 1)[:, :n, None]
                k, v = kv[:kv_heads].transpose(0, 1), kv[kv_heads:].transpose(0, 1)
            else:
                k, v = st["k"][key: key + n].double(), st["v"][key: key + n].double()
            o, sums = _exact_attention(st["q"][row: row + r].double(), k, v, case, st["slopes"], prefixes[s])
            outs.append(o)
            if weights is not None:
                weights[s, :, :n] += sums
            row, key = row + r, key + n
        return {"out": torch.cat(outs), "weights": weights} if op == "cached" else {"out": torch.cat(outs)}
    if op == "evict":
        # the moved weights are copies; the scales the largest of the kept rows' blocks, row by row
        keep, lengths = case["keep"], _kept_sizes(case)
        scales, weights = [], []
        for s, n in enumerate(lengths):
            w = st["weights"][s, :, :n].double().cpu().numpy()
            held = _scales(st["states"], case)[s].double().cpu().numpy()
            middle = np.arange(case["sinks"], n - case["recent"])
            ends = np.concatenate([np.arange(case["sinks"]), np.arange(n - case["recent"], n)])
            at = [np.sort(np.concatenate([ends, middle[np.lexsort((middle, -w[h, middle]))][: keep - len(ends)]])) for h in range(kv_heads)]
            weights.append(np.stack([w[h, at[h]] for h in range(kv_heads)]))
            scales.append(np.stack([np.maximum.reduceat(held[p, at[p % kv_heads] // BLOCK], np.arange(0, keep, BLOCK)) for p in range(2 * kv_heads)]))
        return {"codes": None, "scales": torch.tensor(np.stack(scales)), "weights": torch.tensor(np.stack(weights)), "kept": None}
    scales = _scales(st["states"], case).double()
    planes = 2 * kv_heads
    given = torch.cat([st["keys"], st["values"]], 1).double().abs().amax(2).view(case["sequences"], case["rows"], planes)
    for s, base in enumerate(_bases(case)):
        for block in range(base // BLOCK, (base + case["rows"] - 1) // BLOCK + 1):
            low, high = max(block * BLOCK, base) - base, min((block + 1) * BLOCK, base + case["rows"]) - base
            need = given[s, low:high].amax(0) / TOP[case["code"]]
            scales[s, :, block] = torch.maximum(scales[s, :, block], need) if block * BLOCK < base else need
    return {"codes": None, "scales": scales}

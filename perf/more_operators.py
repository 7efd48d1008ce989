"""Rotary positions, the paged cache with the attention over it, and beam search: the cases they are measured on, and
their plain forms.

Kinds of a case ("kind"):
  rotary   rotary positions of x [S][L][H][D]; with "train" the gradient's way back too: y, and dx
  append   keys and values of new tokens into a paged cache, rotated on the way, and the blocks that they went to, read
           back as the values that the cache now holds
  attend   attention of new tokens' queries, rotated on the way, over such a cache
  beams    one step of beam search: the best continuations of each sequence's beams over the vocabulary
  reorder  the beams' page tables in the order of their parents, with the last pages copied and read back

Caches hold bf16, or 8 bits with a scale for every 16 tokens and head.  dim 64 heads, 8 of them, and 801 frames of an
8 s window are the benchmark configuration's; the rest are generic.  Activations are N(0, 1), keys with a gain of their
own for each head and dim (logarithms N(0, 0.3)), logits N(0, 3).  "ragged": lengths fall evenly from the whole to about
a third of it, and from 8 sequences on the last one is an empty slot.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

DEV = "cuda:0"
BLOCK = 16  # tokens that share a scale
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # one token's queries far into a long context whose angles are scaled, half of the head turning: a call's latency
        {"name": "rotary_step_bf16", "kind": "rotary", "type": "bf16", "sequences": 1, "length": 1, "heads": 32,
         "head_dim": 128, "dim": 64, "interleaved": False, "start": 100_003, "factor": 8.0, "train": False},
        # a training step's queries of the windows of a device pass
        {"name": "rotary_train_fp32", "kind": "rotary", "type": "fp32", "sequences": 8, "length": 801, "heads": 8,
         "head_dim": 64, "dim": 64, "interleaved": True, "start": 0, "factor": 1.0, "train": True},
        # a step of decoding: a token of each request at the end of what it has
        {"name": "append_step_int8", "kind": "append", "type": "bf16", "cache": "int8", "sequences": 32, "length": 1,
         "start": 700, "kv_heads": 8, "head_dim": 64, "page": 64, "dim": 64, "interleaved": True, "ragged": True},
        # the prompts of a batch of requests, padded to the longest
        {"name": "append_prompt_int8", "kind": "append", "type": "bf16", "cache": "int8", "sequences": 8,
         "length": 4001, "start": 0, "kv_heads": 8, "head_dim": 128, "page": 64, "dim": 128, "interleaved": False,
         "ragged": True},
        # one request's token over a short past, everything but the cache in full precision: the smallest call
        {"name": "attend_first_fp32", "kind": "attend", "type": "fp32", "cache": "bf16", "sequences": 1, "heads": 8,
         "kv_heads": 8, "head_dim": 64, "q": 1, "k": 77, "page": 16, "dim": 64, "interleaved": True, "ragged": False,
         "causal": False},
        # single tokens of a batch of requests over long pasts of uneven lengths, shared heads, one slot idle
        {"name": "attend_step_int8", "kind": "attend", "type": "bf16", "cache": "int8", "sequences": 16, "heads": 32,
         "kv_heads": 8, "head_dim": 64, "q": 1, "k": 8192, "page": 64, "dim": 64, "interleaved": True, "ragged": True,
         "causal": False},
        # single tokens of a large batch of long contexts: the largest
        {"name": "attend_step_large_int8", "kind": "attend", "type": "bf16", "cache": "int8", "sequences": 32,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "q": 1, "k": 16384, "page": 128, "dim": 128,
         "interleaved": False, "ragged": False, "causal": False},
        # a piece of long prompts, each token over the ones before it
        {"name": "attend_chunk_int8", "kind": "attend", "type": "bf16", "cache": "int8", "sequences": 4, "heads": 16,
         "kv_heads": 4, "head_dim": 64, "q": 517, "k": 4613, "page": 64, "dim": 64, "interleaved": True,
         "ragged": True, "causal": True},
        # one request's beams over a small vocabulary: a call's latency
        {"name": "beams_one_fp32", "kind": "beams", "type": "fp32", "sequences": 1, "beams": 4, "vocab": 5003,
         "picks": 4},
        # a batch of requests over a large vocabulary, twice the beams kept for those that end
        {"name": "beams_batch_bf16", "kind": "beams", "type": "bf16", "sequences": 32, "beams": 8, "vocab": 120_001,
         "picks": 16},
        # one request's beams
        {"name": "reorder_one_bf16", "kind": "reorder", "type": "bf16", "cache": "bf16", "groups": 1, "beams": 4,
         "kv_heads": 8, "head_dim": 64, "page": 16, "length": 203},
        # a batch of requests' beams with large pages
        {"name": "reorder_batch_int8", "kind": "reorder", "type": "bf16", "cache": "int8", "groups": 32, "beams": 8,
         "kv_heads": 8, "head_dim": 128, "page": 128, "length": 2037},
    ]


def draw(rng):
    def between(lo, hi):  # log-uniform whole number
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["rotary", "append", "attend", "attend", "attend", "beams", "reorder"])
    c = {"kind": kind, "type": rng.choice(["fp32", "bf16"])}
    if kind == "beams":
        c.update(sequences=between(1, 64), beams=rng.choice([1, 2, 3, 4, 5, 8, 12, 16]), vocab=between(100, 130_000))
        c["picks"] = min(c["vocab"], c["beams"] * rng.choice([1, 1, 2]))
        while c["sequences"] * c["beams"] * c["vocab"] > 31_000_000:
            c["sequences"] = (c["sequences"] + 1) // 2 if c["sequences"] > 1 else 1
            c["vocab"] = c["vocab"] if c["sequences"] > 1 else c["vocab"] // 2
        return c
    if kind == "rotary":
        D = rng.choice([64, 64, 128, 96, 80])
        c.update(sequences=between(1, 16), length=between(1, 8192), heads=rng.choice([1, 2, 7, 8, 16, 32]), head_dim=D,
                 dim=rng.choice([D, D, D // 2, D // 4]), interleaved=rng.random() < 0.5, train=rng.random() < 0.5)
        c.update(start=rng.choice([0, between(1, 100_000)]), factor=rng.choice([1.0, 4.0, 8.0]))
        while c["sequences"] * c["length"] * c["heads"] * D > 16_000_000:
            c["length"] = (c["length"] + 1) // 2
        return c
    D = rng.choice([64, 128])
    c.update(cache=rng.choice(["int8", "int8", "bf16"]), kv_heads=rng.choice([1, 2, 4, 8, 8, 12]), head_dim=D,
             page=rng.choice([16, 64, 64, 128, 256]))
    if kind == "reorder":
        c.update(groups=between(1, 48), beams=rng.choice([2, 3, 4, 5, 8, 16]), length=between(1, 4096))
        while c["groups"] * c["beams"] * (c["length"] + c["page"]) * c["kv_heads"] * D > 700_000_000:
            c["groups"] = (c["groups"] + 1) // 2 if c["groups"] > 1 else 1
            c["length"] = c["length"] if c["groups"] > 1 else c["length"] // 2
        return c
    c.update(dim=rng.choice([D, D, D // 2]), interleaved=rng.random() < 0.5, ragged=rng.random() < 0.6,
             sequences=between(1, 32))
    if kind == "append":
        c.update(length=rng.choice([1, rng.randint(2, 9), between(10, 4096)]), start=rng.choice([0, between(1, 5000)]))
        while c["sequences"] * c["length"] * c["kv_heads"] * D > 34_000_000:
            c["sequences"] = (c["sequences"] + 1) // 2
        while c["sequences"] * c["start"] * c["kv_heads"] * D > 200_000_000:
            c["start"] //= 2
        return c
    step = rng.random() < 0.6
    c.update(heads=c["kv_heads"] * rng.choice([1, 2, 4, 4, 8]), q=rng.choice([1, 1, 1, 2, 5]) if step else between(8, 2048))
    c.update(k=c["q"] + between(8, 16384 if step else 4096), causal=c["q"] > 1 and rng.random() < 0.8)
    # at most the listed ones' cache and scores
    while c["sequences"] * c["k"] * c["kv_heads"] * D > 500_000_000 or \
            c["sequences"] * c["heads"] * c["q"] * c["k"] * D > 9.0e9 * (1.0 if c["type"] == "bf16" else 0.5):
        if c["sequences"] > 1:
            c["sequences"] = (c["sequences"] + 1) // 2
        elif c["q"] > 64:
            c["k"], c["q"] = c["k"] - c["q"] + c["q"] * 2 // 3, c["q"] * 2 // 3
        else:
            c["k"] = c["q"] + (c["k"] - c["q"]) * 2 // 3
    return c


# ---------------------------------------------------------------- sizes that follow from a case

def _fall(whole, S, ragged):
    if not ragged:
        return [whole] * S
    n = [max(1, whole - (2 * whole * s) // (3 * S)) for s in range(S)]
    if S >= 8:
        n[-1] = 0
    return n


def _lengths(case):
    """New tokens of each sequence: a step's one token each but for the empty slot."""
    if case["kind"] == "append":
        n = _fall(case["length"], case["sequences"], case["ragged"])
        return n if case["length"] > 1 else [min(1, x) for x in n]
    return [min(case["q"], n) for n in _fall(case["k"], case["sequences"], case["ragged"])]


def _starts(case):
    """Tokens that each sequence held before."""
    if case["kind"] == "append":
        return [case["start"] - (case["start"] * s) // (2 * case["sequences"]) if case["ragged"] else case["start"]
                for s in range(case["sequences"])]
    return [n - m for n, m in zip(_fall(case["k"], case["sequences"], case["ragged"]), _lengths(case))]


def _capacity(case):
    """Tokens that a sequence's row of the page table has room for."""
    if case["kind"] == "append":
        return case["start"] + case["length"]
    return case["k"] if case["kind"] == "attend" else case["length"] + 1


def _rows(case):
    return case["groups"] * case["beams"] if case["kind"] == "reorder" else case["sequences"]


# ---------------------------------------------------------------- inputs

def _generator(seed, stream):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 16 + stream) & 0x7FFFFFFFFFFF)
    return g


def _randn(seed, stream, *shape):
    return torch.randn(*shape, device=DEV, generator=_generator(seed, stream))


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _native():
    path = os.path.join(os.getcwd(), "karaoke-platform-sidecar-native_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from vocalarc_hip import native
    return native


def _buffer(nbytes):
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=DEV)


def prepare(case, seed):
    kind = case["kind"]
    s = {"case": case}
    if own:
        s["ctx"] = _native().Context()
    if kind == "rotary":
        return _prepare_rotary(s, case, seed)
    if kind == "beams":
        return _prepare_beams(s, case, seed)
    return _prepare_cache(s, case, seed)


SCALING = {"original": 8192, "low": 1.0, "high": 32.0}  # with a factor: turns in the first context that keep their angle
BASE = 10000.0


def _angles(positions, dim, factor):
    """The angles of positions in 64 bits [n][dim / 2], and what the rotation is multiplied by."""
    theta = BASE ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=DEV) / dim)
    if factor == 1.0:
        return positions.double()[:, None] * theta, 1.0
    turns = SCALING["original"] * theta / (2 * math.pi)
    keep = ((turns - SCALING["low"]) / (SCALING["high"] - SCALING["low"])).clamp(0, 1)
    return positions.double()[:, None] * (theta * (keep + (1 - keep) / factor)), 1 + 0.1 * math.log(factor)


def _rotation(s, positions, dim, interleaved, factor=1.0):
    """What a program keeps of the rotation: the table of every position."""
    if own:
        more = dict(SCALING, factor=factor, magnitude=1 + 0.1 * math.log(factor)) if factor != 1.0 else {}
        s["rotary"] = _native().Rotary(s["ctx"], positions, dim, interleaved=interleaved, base=BASE, **more)
    else:
        a, m = _angles(torch.arange(positions, device=DEV), dim, factor)
        s["cos"], s["sin"] = (a.cos() * m).float(), (a.sin() * m).float()


def _prepare_rotary(s, case, seed):
    S, L, H, D = case["sequences"], case["length"], case["heads"], case["head_dim"]
    s["x"] = _randn(seed, 0, S, L, H, D).to(TYPES[case["type"]])
    if case["train"]:
        s["dy"] = _randn(seed, 1, S, L, H, D).to(TYPES[case["type"]])
    s["start"] = _ints([case["start"] // (i + 1) for i in range(S)])
    _rotation(s, case["start"] + L, case["dim"], case["interleaved"], case["factor"])
    if own:
        s["y"] = torch.empty_like(s["x"])
        if case["train"]:
            s["dx"] = torch.empty_like(s["x"])
    return s


def _prepare_beams(s, case, seed):
    S, B, V = case["sequences"], case["beams"], case["vocab"]
    s["logits"] = (3 * _randn(seed, 0, S, B, V)).to(TYPES[case["type"]])
    s["scores"] = -4 - _randn(seed, 1, S, B).abs()
    s["ended"] = (torch.rand(S, B, device=DEV, generator=_generator(seed, 2)) < 0.1).int()
    s["end_token"] = 2
    if own:
        native = _native()
        s["search"] = native.BeamSearch(s["ctx"], s["logits"], picks=case["picks"], end_token=2)
        s["workspace"] = _buffer(s["search"].workspace_bytes())
        s["out"] = [torch.empty(S, case["picks"], dtype=t, device=DEV)
                    for t in (torch.int32, torch.int32, torch.float32, torch.int32)]
    return s


def _prepare_cache(s, case, seed):
    kind, S, KV, D, page = case["kind"], _rows(case), case["kv_heads"], case["head_dim"], case["page"]
    t = TYPES[case["type"]]
    each = -(-_capacity(case) // page)
    pages = S * each + (S if kind == "reorder" else 0)
    ids = torch.randperm(pages, device=DEV, generator=_generator(seed, 9)).int()
    s["table"] = ids[:S * each].view(S, each).contiguous()
    if own:
        native = _native()
        s["cache"] = native.PagedCache(s["ctx"], case["cache"], kv_heads=KV, head_dim=D, page_tokens=page, pages=pages)
    else:  # one page more, for what is masked
        q = torch.int8 if case["cache"] == "int8" else torch.bfloat16
        s["pages"] = pages
        s["pool"] = [torch.zeros(pages + 1, KV, page, D, dtype=q, device=DEV) for _ in "kv"]
        s["pool_scale"] = [torch.zeros(pages + 1, KV, page // BLOCK, device=DEV) for _ in "kv"]
    rotary = kind != "reorder"
    if rotary:
        _rotation(s, _capacity(case), case["dim"], case["interleaved"])
    if kind == "append":
        held, starts, new = case["start"], _starts(case), case["length"]
    else:
        held = case["k"] if kind == "attend" else case["length"]
        starts = _fall(held, S, case["ragged"]) if kind == "attend" else [held] * S
        new = case.get("q", 0)
    gain = torch.exp(0.3 * _randn(seed, 2, KV, D))
    if held:  # what the sequences hold already
        k, v = (_randn(seed, 3, S, held, KV, D) * gain).to(t), _randn(seed, 4, S, held, KV, D).to(t)
        if own:
            s["cache"].tokens(s["table"], k, v, lengths=_ints(starts), rotary=s.get("rotary")).append(k, v)
        else:
            _append(s, case, k, v, [0] * S, starts, rotary)
        del k, v
    if kind == "append":
        n = _lengths(case)
        s["start"], s["lengths"] = _ints(starts), _ints(n)
        s["k"], s["v"] = (_randn(seed, 0, S, new, KV, D) * gain).to(t), _randn(seed, 1, S, new, KV, D).to(t)
        # the blocks that the new tokens go to
        first = [x // BLOCK * BLOCK for x in starts]
        rows = _touched(case)
        s["first"], s["upto"] = _ints(first), _ints([a + b - f if b else 0 for a, b, f in zip(starts, n, first)])
        if own:
            s["k_out"], s["v_out"] = torch.empty(S, rows, KV, D, dtype=t, device=DEV), \
                torch.empty(S, rows, KV, D, dtype=t, device=DEV)
            s["append"] = s["cache"].tokens(s["table"], s["k"], s["v"], start=s["start"], lengths=s["lengths"],
                                            rotary=s["rotary"])
            s["read"] = s["cache"].tokens(s["table"], s["k_out"], s["v_out"], start=s["first"], lengths=s["upto"])
    elif kind == "attend":
        H = case["heads"]
        s["q"] = _randn(seed, 0, S, new, H, D).to(t)
        s["scale"] = D ** -0.5
        s["key_lengths"], s["query_lengths"] = _ints(starts), _ints(_lengths(case))
        s["start"] = _ints(_starts(case))
        if own:
            s["out"] = torch.empty_like(s["q"])
            s["attend"] = s["cache"].queries(s["table"], s["q"], s["out"], most_keys=case["k"], causal=case["causal"],
                                             scale=s["scale"], query_lengths=s["query_lengths"],
                                             key_lengths=s["key_lengths"], query_start=s["start"], rotary=s["rotary"])
            s["workspace"] = _buffer(s["attend"].workspace_bytes())
    else:
        G, B = case["groups"], case["beams"]
        # a beam goes on in its place or in another's
        r = torch.rand(G, B, device=DEV, generator=_generator(seed, 5))
        s["parents"] = torch.where(r < 0.4, torch.arange(B, device=DEV), (r * 7919).long() % B).int().flatten()
        s["group_lengths"] = _ints([case["length"]] * G)
        s["spare"] = ids[S * each:].contiguous()
        last = case["length"] // page * page
        if own:
            s["table_out"], s["spare_out"] = torch.empty_like(s["table"]), torch.empty_like(s["spare"])
            s["k_out"], s["v_out"] = torch.empty(S, page, KV, D, dtype=t, device=DEV), \
                torch.empty(S, page, KV, D, dtype=t, device=DEV)
            s["read"] = s["cache"].tokens(s["table_out"], s["k_out"], s["v_out"], start=_ints([last] * S),
                                          lengths=_ints([case["length"] - last] * S))
    return s


def _touched(case):
    """Rows of the blocks that a call's new tokens may lie in."""
    off = max(x % BLOCK for x in _starts(case))
    return -(-(off + case["length"]) // BLOCK) * BLOCK


# ---------------------------------------------------------------- one pass

def run(s):
    return (_own if own else _plain)[s["case"]["kind"]](s)


def _rotary_own(s):
    s["rotary"].apply(s["x"], s["y"], start=s["start"])
    if not s["case"]["train"]:
        return {"y": s["y"]}
    s["rotary"].apply(s["dy"], s["dx"], start=s["start"], backward=True)
    return {"y": s["y"], "dx": s["dx"]}


def _append_own(s):
    s["append"].append(s["k"], s["v"])
    s["read"].read(s["k_out"], s["v_out"])
    return {"k": s["k_out"], "v": s["v_out"]}


def _attend_own(s):
    s["attend"].forward(s["q"], s["out"], workspace=s["workspace"])
    return {"out": s["out"]}


def _beams_own(s):
    tokens, parents, scores, ended = s["out"]
    s["search"].select(s["logits"], s["scores"], tokens, parents, scores, ended=s["ended"], new_ended=ended,
                       workspace=s["workspace"])
    return {"tokens": tokens, "parents": parents, "scores": scores, "ended": ended}


def _reorder_own(s):
    s["cache"].reorder(s["table"], s["parents"], s["group_lengths"], s["spare"], s["table_out"], s["spare_out"],
                       beams=s["case"]["beams"])
    s["read"].read(s["k_out"], s["v_out"])
    return {"table": s["table_out"], "spare": s["spare_out"], "k": s["k_out"], "v": s["v_out"]}


_own = {"rotary": _rotary_own, "append": _append_own, "attend": _attend_own, "beams": _beams_own,
        "reorder": _reorder_own}


def _turn(x, c, sn, dim, interleaved):
    """x [..., D] of 32 bits by the angles whose cosines and sines are c and sn [..., dim / 2]."""
    r, rest = x[..., :dim], x[..., dim:]
    a, b = (r[..., 0::2], r[..., 1::2]) if interleaved else (r[..., :dim // 2], r[..., dim // 2:])
    u, w = a * c - b * sn, a * sn + b * c
    r = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((r, rest), -1)


def _turn_rows(s, x, start, sign=1):
    """x [S][L][H][D] by the positions from start [S] on (-1: back again)."""
    at = (start.long()[:, None] + torch.arange(x.shape[1], device=DEV)).clamp(max=s["cos"].shape[0] - 1)
    return _turn(x.float(), s["cos"][at][:, :, None], sign * s["sin"][at][:, :, None], s["case"]["dim"],
                 s["case"]["interleaved"])


def _rotary_plain(s):
    t = s["x"].dtype
    y = _turn_rows(s, s["x"], s["start"]).to(t)
    if not s["case"]["train"]:
        return {"y": y}
    return {"y": y, "dx": _turn_rows(s, s["dy"], s["start"], -1).to(t)}


def _append(s, case, k, v, starts, lengths, rotary):
    """Tokens into the pages, with the starts and lengths on the device or in lists; the touched blocks' values."""
    page, KV, D, S = case["page"], case["kv_heads"], case["head_dim"], k.shape[0]
    start = starts if torch.is_tensor(starts) else _ints(starts)
    count = lengths if torch.is_tensor(lengths) else _ints(lengths)
    nb = (_touched(case) if torch.is_tensor(starts) else -(-k.shape[1] // BLOCK) * BLOCK) // BLOCK
    first = start.long() // BLOCK
    at = (first[:, None] * BLOCK + torch.arange(nb * BLOCK, device=DEV))
    old, new = at < start[:, None], (at >= start[:, None]) & (at < (start + count)[:, None])
    block = first[:, None] + torch.arange(nb, device=DEV)  # [S][nb]
    ids = s["table"].long().gather(1, (block * BLOCK // page).clamp(max=s["table"].shape[1] - 1))
    ids = torch.where(new.view(S, nb, BLOCK).any(-1), ids, s["pages"])
    slot = block % (page // BLOCK)
    old, new = old.view(S, nb, 1, BLOCK, 1), new.view(S, nb, 1, BLOCK, 1)
    from_row = (at - start[:, None]).clamp(0, k.shape[1] - 1)[:, :, None, None].expand(-1, -1, KV, D)
    values = []
    for i, x in enumerate((k, v)):
        x = _turn_rows(s, x, start) if i == 0 and rotary else x.float()
        x = x.gather(1, from_row).view(S, nb, BLOCK, KV, D).transpose(2, 3)  # [S][nb][KV][16][D]
        pool = s["pool"][i].view(-1, KV, page // BLOCK, BLOCK, D)
        was = pool[ids, :, slot]
        if case["cache"] == "int8":
            scale = (torch.where(new, x.abs(), 0).amax((3, 4)) * (1 / 127)).clamp(min=2.0 ** -100)
            before = s["pool_scale"][i][ids, :, slot]
            scale = torch.where(old.any(3)[..., 0], torch.maximum(scale, before), scale)
            inv = scale.reciprocal()
            q = torch.round(x * inv[..., None, None]).clamp(-127, 127)
            q = torch.where(new, q, torch.where(old, torch.round(was.float() * (before * inv)[..., None, None]), 0))
            s["pool_scale"][i][ids, :, slot] = scale
            pool[ids, :, slot] = q.to(torch.int8)
            got = q * scale[..., None, None]
        else:
            got = torch.where(new, x.bfloat16(), torch.where(old, was, 0))
            pool[ids, :, slot] = got
        got = torch.where(new.any(3, keepdim=True), got.float(), 0)
        values.append(got.transpose(2, 3).reshape(S, nb * BLOCK, KV, D).to(k.dtype))
    return values


def _append_plain(s):
    k, v = _append(s, s["case"], s["k"], s["v"], s["start"], s["lengths"], True)
    return {"k": k, "v": v}


def _gathered(s, i, table):
    """Values of the pages that a table [S][n] names: [S][KV][n * page][D], in 32 bits."""
    x = s["pool"][i][table.long()].float()  # [S][n][KV][page][D]
    if s["case"]["cache"] == "int8":
        x = x * s["pool_scale"][i][table.long()].repeat_interleave(BLOCK, -1)[..., None]
    return x.transpose(1, 2).flatten(2, 3)


def _attend_plain(s):
    case, t = s["case"], s["q"].dtype
    S, H, KV, Lq, D = (case[n] for n in ("sequences", "heads", "kv_heads", "q", "head_dim"))
    q = _turn_rows(s, s["q"], s["start"]).view(S, Lq, KV, H // KV, D).permute(0, 2, 3, 1, 4).flatten(2, 3)
    k, v = _gathered(s, 0, s["table"]), _gathered(s, 1, s["table"])
    x = torch.matmul(q, k.transpose(2, 3)) * s["scale"]  # [S][KV][G Lq][Lk]
    at = torch.arange(k.shape[2], device=DEV)
    row = torch.arange(Lq, device=DEV)
    sees = (at < s["key_lengths"][:, None])[:, None, :] & (row < s["query_lengths"][:, None])[:, :, None]
    if case["causal"]:
        sees = sees & (at <= (s["start"][:, None] + row)[:, :, None])
    sees = sees[:, None].expand(-1, H // KV, -1, -1).flatten(1, 2)[:, None]
    x = torch.where(sees, x, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)  # finite where a row has no key
    p = torch.exp(x - m)
    p = p / p.sum(-1, keepdim=True).clamp(min=1.0)  # the largest adds 1: less only without a key
    out = torch.matmul(p, v).unflatten(2, (H // KV, Lq))
    return {"out": out.permute(0, 3, 1, 2, 4).reshape(S, Lq, H, D).to(t)}


def _beams_plain(s):
    case = s["case"]
    B, V, n = case["beams"], case["vocab"], case["picks"]
    x = s["logits"].double()  # candidates next to each other differ by less than 32 bits hold of their scores
    m = x.amax(-1, keepdim=True)
    x = x - (m + (x - m).exp().sum(-1, keepdim=True).log())
    ends = torch.arange(V, device=DEV) == s["end_token"]
    x = torch.where(s["ended"][..., None] != 0, torch.where(ends, 0.0, -math.inf), x) + s["scores"].double()[..., None]
    best, at = x.flatten(1).sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    tokens, parents = at % V, at // V
    ended = (s["ended"].gather(1, parents) != 0) | (tokens == s["end_token"])
    return {"tokens": tokens.int(), "parents": parents.int(), "scores": best.float(), "ended": ended.int()}


def _reorder_plain(s):
    case = s["case"]
    B, page, S, n = case["beams"], case["page"], _rows(case), case["length"]
    row = torch.arange(S, device=DEV)
    parent = row // B * B + s["parents"].long()
    last, used = n // page, n % page
    column = torch.arange(s["table"].shape[1], device=DEV)
    table = torch.where(column < last, s["table"][parent], s["table"])
    spare = s["spare"].clone()
    if used:
        moved = parent != row
        table[:, last] = torch.where(moved, s["spare"], s["table"][:, last])
        spare = torch.where(moved, s["table"][:, last], s["spare"])
        source, target = s["table"][parent, last].long(), torch.where(moved, s["spare"], s["pages"]).long()
        for pool in s["pool"] + s["pool_scale"]:
            pool[target] = pool[source]
    got = {"table": table, "spare": spare}
    held = torch.arange(page, device=DEV)[:, None, None] < used
    for i, name in enumerate("kv"):
        x = _gathered(s, i, table[:, min(last, table.shape[1] - 1)][:, None]).transpose(1, 2)
        got[name] = torch.where(held, x, 0).to(TYPES[case["type"]])
    return got


_plain = {"rotary": _rotary_plain, "append": _append_plain, "attend": _attend_plain, "beams": _beams_plain,
          "reorder": _reorder_plain}


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    size, kind = 2 if case["type"] == "bf16" else 4, case["kind"]
    if kind == "rotary":
        n = case["sequences"] * case["length"] * case["heads"] * case["head_dim"] * (2 if case["train"] else 1)
        table = case["sequences"] * case["length"] * case["dim"] * 4
        return {"bytes": 2 * n * size + table, "flops": 3 * n * case["dim"] // case["head_dim"]}
    if kind == "beams":
        n = case["sequences"] * case["beams"] * case["vocab"]
        return {"bytes": n * size + 16 * case["sequences"] * case["picks"], "flops": 4 * n}
    KV, D = case["kv_heads"], case["head_dim"]
    # of a token's key or value in the cache
    held = KV * (D + 4 / BLOCK if case["cache"] == "int8" else 2 * D)
    if kind == "append":
        n, starts = _lengths(case), _starts(case)
        old = sum(x % BLOCK for x, m in zip(starts, n) if m)  # tokens of the first blocks, whose scale may change
        new, rows = sum(n), case["sequences"] * _touched(case)
        again = 2 * old * held if case["cache"] == "int8" else 0  # read and written once more
        # k and v in, into the cache, and the touched blocks' values out
        return {"bytes": 2 * (new * KV * D * size + new * held + again + rows * KV * D * size) + new * case["dim"] * 4,
                "flops": 10 * new * KV * D}
    if kind == "reorder":
        S, used = _rows(case), case["length"] % case["page"]
        moved = S * 0.6 * (1 - 1 / case["beams"])  # beams in another's place
        # the last pages in, those that move out again, and their values
        return {"bytes": 2 * used * held * (S + moved) + 2 * S * case["page"] * KV * D * size +
                8 * S * (case["length"] // case["page"] + 1), "flops": 2 * S * used * KV * D}
    S, H, Lq = case["sequences"], case["heads"], case["q"]
    pairs, keys = 0, 0
    for n, m, a in zip(_fall(case["k"], S, case["ragged"]), _lengths(case), _starts(case)):
        keys += n
        pairs += m * a + m * (m + 1) // 2 if case["causal"] else m * n
    return {"bytes": 2 * keys * held + 2 * S * Lq * H * D * size, "flops": 4 * D * pairs * H}


# ---------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    global own
    before, own = own, False  # the inputs, and for attention the cache's values, as the plain form has them
    try:
        s = prepare(case, seed)
    finally:
        own = before
    return _exact[case["kind"]](s)


def _spin(x, positions, case, sign=1):
    """x [L][H][D] in 64 bits as complex numbers times exp(i angle), position by position."""
    dim = case["dim"]
    a, m = _angles(positions, dim, case.get("factor", 1.0))
    turn = torch.polar(torch.full_like(a, m), sign * a)[:, None]
    pair = x[..., :dim].unflatten(-1, (dim // 2, 2)) if case["interleaved"] else \
        x[..., :dim].unflatten(-1, (2, dim // 2)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    z = z if case["interleaved"] else z.transpose(-1, -2)
    return torch.cat((z.flatten(-2), x[..., dim:]), -1)


def _each(s, x, case, sign=1):
    L = x.shape[1]
    return torch.stack([_spin(x[i].double(), torch.arange(a, a + L, device=DEV), case, sign)
                        for i, a in enumerate(s["start"].tolist())])


def _rotary_exact(s):
    case = s["case"]
    y = _each(s, s["x"], case)
    # the rotation's transpose: the other way round, with the same magnitude
    return {"y": y, "dx": _each(s, s["dy"], case, -1)} if case["train"] else {"y": y}


def _append_exact(s):
    """Block by block of the sequences' own order, from the values in the cache before the call."""
    case = s["case"]
    S, KV, D, page = case["sequences"], case["kv_heads"], case["head_dim"], case["page"]
    rows = _touched(case)
    got = {n: torch.zeros(S, rows, KV, D, dtype=torch.float64, device=DEV) for n in "kv"}
    turned = _each(s, s["k"], case)
    for b, (a, n) in enumerate(zip(_starts(case), _lengths(case))):
        if not n:
            continue
        first, off = a // BLOCK, a % BLOCK
        blocks = -(-(off + n) // BLOCK)
        for i, (name, x) in enumerate((("k", turned[b]), ("v", s["v"][b].double()))):
            z = torch.zeros(blocks * BLOCK, KV, D, dtype=torch.float64, device=DEV)
            z[off:off + n] = x[:n]
            if case["cache"] == "bf16":
                if off:
                    id, slot = int(s["table"][b, a // page]), first % (page // BLOCK) * BLOCK
                    z[:off] = s["pool"][i][id, :, slot:slot + off].double().transpose(0, 1)
                got[name][b, :len(z)] = z.bfloat16().double()
                continue
            top = z.abs().view(blocks, BLOCK, KV, D).amax((1, 3)) / 127
            if off:
                id, slot = int(s["table"][b, a // page]), first % (page // BLOCK)
                before = s["pool_scale"][i][id, :, slot].double()
                top[0] = torch.maximum(top[0], before)
                z[:off] = (s["pool"][i][id, :, slot * BLOCK:slot * BLOCK + off].double() * before[:, None, None]).transpose(0, 1)
            unit = top.repeat_interleave(BLOCK, 0)[..., None].clamp(min=2.0 ** -100)
            got[name][b, :len(z)] = torch.round(z / unit).clamp(-127, 127) * unit
    return got


def _attend_exact(s):
    case = s["case"]
    H, KV, page = case["heads"], case["kv_heads"], case["page"]
    if case["sequences"] * KV > 600:
        return None
    q = _each(s, s["q"], case)
    out = torch.zeros_like(q)
    for b, n in enumerate(_fall(case["k"], case["sequences"], case["ragged"])):
        m, a = _lengths(case)[b], _starts(case)[b]
        if not n:
            continue
        ids = s["table"][b].long()
        for g in range(KV):
            held = []
            for i in (0, 1):
                x = s["pool"][i][ids, g].double()
                if case["cache"] == "int8":
                    x = (x.unflatten(1, (-1, BLOCK)) * s["pool_scale"][i][ids, g].double()[:, :, None, None]).flatten(1, 2)
                held.append(x.flatten(0, 1)[:n])
            heads = slice(g * (H // KV), (g + 1) * (H // KV))
            x = torch.einsum("lhd,kd->hlk", q[b, :m, heads], held[0]) * s["scale"]
            if case["causal"]:
                late = torch.arange(n, device=DEV) > torch.arange(a, a + m, device=DEV)[:, None]
                x = x.masked_fill(late, -math.inf)
            out[b, :m, heads] = torch.einsum("hlk,kd->lhd", torch.softmax(x, -1), held[1])
    return {"out": out}


def _beams_exact(s):
    """The scores alone: their order has no rounding to be off by."""
    n, best = s["case"]["picks"], []
    for b in range(s["case"]["sequences"]):
        x = torch.log_softmax(s["logits"][b].double(), -1)
        done = s["ended"][b] != 0
        x[done] = -math.inf
        x[done, s["end_token"]] = 0
        best.append((x + s["scores"][b].double()[:, None]).flatten().topk(n).values)
    return {"tokens": None, "parents": None, "scores": torch.stack(best), "ended": None}


def _reorder_exact(s):
    """What the parents' last pages hold."""
    case = s["case"]
    B, page, n = case["beams"], case["page"], case["length"]
    last, used = n // page, n % page
    got = {"table": None, "spare": None}
    for i, name in enumerate("kv"):
        got[name] = z = torch.zeros(_rows(case), page, case["kv_heads"], case["head_dim"], dtype=torch.float64, device=DEV)
        if not used:
            continue
        for r, p in enumerate(s["parents"].tolist()):
            id = int(s["table"][r // B * B + p, last])
            x = s["pool"][i][id, :, :used].double()
            if case["cache"] == "int8":
                x = x * s["pool_scale"][i][id].double().repeat_interleave(BLOCK, -1)[:, :used, None]
            z[r, :used] = x.transpose(0, 1)
    return got


_exact = {"rotary": _rotary_exact, "append": _append_exact, "attend": _attend_exact, "beams": _beams_exact,
          "reorder": _reorder_exact}

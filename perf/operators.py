"""Operators on the 8-bit context cache: what a user has them do, over the sizes they are used at.

The cache keeps the context keys and values of ``heads`` heads in blocks of 64 rows.  Of every (group, head, block)

  codes    uint8 [G,H,blocks,2,64*Dh]   keys row by row, then values transposed, [Dh][64], the rows of a block in
                                        ROW_ORDER; the value of a code is (code - 128) * scale
  scales   fp32  [G,H,blocks,2]         largest magnitude / 127, of the keys and of the values
  bounds   fp16  [G,H,blocks,2,Dh]      smallest and largest key code of a channel over the block's rows (less 128)
  lens     int32 [G]                    rows in use

A group is one context: shared by the whole batch, or one per batch element (``shared`` False).  A case is one of

  quantize   write the rows of whole contexts into a new cache, and read them back
  append     put ``new`` rows behind those of every group, and read the blocks back that hold them
  attend     softmax attention of the queries over the whole cache: output and log-sum-exp
  select     the ``pick`` blocks with the largest upper bound of a score, for every query
  blocks     attention over a list of blocks for every query

``type`` is that of queries, keys and values.  ``ragged``: the groups hold different numbers of rows, the last one
of eight or more none at all.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

BLOCK = 64
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
# row of a block at each place of a value row: place 16 t + 4 s + 2 h + e holds row 16 s + 8 h + 2 t + e
ROW_ORDER = [16 * s + 8 * h + 2 * t + e for t in range(4) for s in range(4) for h in range(2) for e in range(2)]


def _case(name, op, type, shared, batch, heads, head_dim, ctx, queries=1, ragged=False, new=0, pick=0):
    return dict(name=name, op=op, type=type, shared=shared, batch=batch, heads=heads, head_dim=head_dim, ctx=ctx,
                queries=queries, ragged=ragged, new=new, pick=pick)


def listed():
    return [
        # smallest: one small table is cached, fp32, narrow heads
        _case("quantize_small_fp32", "quantize", "fp32", True, 1, 4, 16, 128),
        # the contexts of a batch of datasets of different lengths
        _case("quantize_datasets_bf16", "quantize", "bf16", False, 64, 6, 32, 2048, ragged=True),
        # a decode step keeps one new row of every stream
        _case("append_row_bf16", "append", "bf16", False, 512, 6, 32, 256, ragged=True, new=1),
        # more labelled rows arrive for every dataset, a different number each
        _case("append_rows_fp32", "append", "fp32", False, 64, 8, 64, 2048, ragged=True, new=100),
        # smallest attention: a few streams on one small table with an odd number of rows
        _case("attend_small_fp32", "attend", "fp32", True, 8, 4, 16, 125),
        # one decode step (buffer and target query) of datasets with a context each
        _case("attend_datasets_bf16", "attend", "bf16", False, 64, 6, 32, 2048, queries=2, ragged=True),
        # single queries over a few very long contexts
        _case("attend_long_bf16", "attend", "bf16", False, 8, 8, 64, 65536),
        # thousands of streams on one context: a decode step of the largest sampling jobs
        _case("attend_4096_bf16", "attend", "bf16", True, 4096, 6, 32, 8192, queries=2),
        # blocks for every query of a decode step of 512 streams on a long context
        _case("select_512_bf16", "select", "bf16", True, 512, 6, 32, 16384, queries=2, pick=16),
        # single queries of datasets with a context each
        _case("select_datasets_fp32", "select", "fp32", False, 64, 8, 64, 2048, ragged=True, pick=8),
        # the attention behind either selection
        _case("blocks_512_bf16", "blocks", "bf16", True, 512, 6, 32, 16384, queries=2, pick=16),
        _case("blocks_datasets_fp32", "blocks", "fp32", False, 64, 8, 64, 2048, ragged=True, pick=8),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["quantize", "append", "attend", "attend", "select", "blocks"])
        shared = op not in ("quantize", "append") and rng.random() < 0.5
        batch = _log(rng, 1, 2048 if shared else 128)
        ctx = _log(rng, 40, 16384)
        new = min(_log(rng, 1, 300), ctx) if op == "append" else 0
        c = _case(None, op, rng.choice(["fp32", "bf16"]), shared, batch, rng.choice([1, 2, 3, 4, 6, 8]),
                  rng.choice([16, 32, 64]), ctx, 1 if op in ("quantize", "append") else rng.choice([1, 1, 2, 3, 5]),
                  not shared and rng.random() < 0.6, new, _log(rng, 1, 24) if op in ("select", "blocks") else 0)
        del c["name"]
        if _cost(c) <= top:
            return c


def _cost(c):
    w = work(c)
    rows = c["batch"] * c["queries"] * c["heads"]
    # the plain form of "blocks" copies the rows of every list, that of "select" a product per (query, block, channel)
    copies = {"blocks": rows * c["pick"] * BLOCK * c["head_dim"] * 8, "select": rows * c["ctx"] / BLOCK * c["head_dim"] * 4}
    return max(w["bytes"], w["flops"] / 50, copies.get(c["op"], 0) / 4)


def _held(c):
    """Rows in use, summed over the groups (mean of what prepare draws)."""
    groups = 1 if c["shared"] else c["batch"]
    return groups * c["ctx"] * (0.625 if c["ragged"] else 1.0)


def work(case):
    c = case
    e = 4 if c["type"] == "fp32" else 2
    H, D = c["heads"], c["head_dim"]
    held = _held(c) * H
    rows = c["batch"] * c["queries"] * H
    record = 128 * D + 8 + 4 * D          # codes, scales and bounds of a block
    if c["op"] == "quantize":             # rows in, records out and in again, fp32 rows out
        return {"bytes": held * 2 * D * (e + 4) + held / BLOCK * 2 * record, "flops": held * 2 * D * 4}
    if c["op"] == "append":               # new rows in, the blocks that they touch in and out, and read back as fp32
        n, blocks = c["new"] * (0.75 if c["ragged"] else 1.0), (c["new"] + 126) // BLOCK + 1
        n, blocks = n * c["batch"] * H, (n + 63) / BLOCK * c["batch"] * H
        return {"bytes": n * 2 * D * e + blocks * (3 * record + 2 * BLOCK * D * 4), "flops": blocks * 2 * BLOCK * D * 4}
    queries = rows * (D * e + 4)
    if c["op"] == "attend":
        pairs = rows * _held(c) / (1 if c["shared"] else c["batch"])
        return {"bytes": held / BLOCK * (128 * D + 8) + queries + rows * D * e, "flops": pairs * 4 * D}
    if c["op"] == "select":
        pairs = rows * _held(c) / (1 if c["shared"] else c["batch"]) / BLOCK
        return {"bytes": held / BLOCK * (4 * D + 4) + rows * D * e + rows * c["pick"] * 4, "flops": pairs * 4 * D}
    pick = min(c["pick"], _held(c) / (1 if c["shared"] else c["batch"]) / BLOCK)
    read = min(held / BLOCK, rows * pick) * (128 * D + 8)
    return {"bytes": read + queries + rows * (D * e + c["pick"] * 4), "flops": rows * pick * BLOCK * 4 * D}


# ------------------------------------------------------------------ the plain form

def _order(device):
    return torch.tensor(ROW_ORDER, device=device)


def _nearest(x, scale):
    """The whole number nearest to x / scale (64 bits: quotients next to a half), zero where the scale is."""
    y = torch.where(scale > 0, x.double() / scale.double(), 0.0)
    return torch.round(y).clamp(-127, 127).float()


def _scale(top):
    return (top.double() / torch.full((), 127.0, dtype=torch.float64, device=top.device)).float()


def _blocked(x, blocks):
    """[G,H,N,D] -> [G,H,blocks,64,D], zeros behind the last row."""
    G, H, N, D = x.shape
    y = x.new_zeros(G, H, blocks * BLOCK, D)
    y[:, :, :N] = x
    return y.view(G, H, blocks, BLOCK, D)


def _fields(k, v, ks, vs, live):
    """Codes, scales and bounds of blocks of rows [..., 64, D] with given scales; live [..., 64]."""
    ck = _nearest(k, ks[..., None, None]) * live[..., None]
    cv = _nearest(v, vs[..., None, None]) * live[..., None]
    lead, D = ck.shape[:-2], ck.shape[-1]
    codes = torch.stack([ck.reshape(*lead, BLOCK * D),
                         cv.transpose(-1, -2)[..., _order(k.device)].reshape(*lead, BLOCK * D)], dim=-2)
    lo = torch.where(live[..., None], ck, 127.0).amin(-2)
    hi = torch.where(live[..., None], ck, -127.0).amax(-2)
    return ((codes + 128).to(torch.uint8), torch.stack([ks, vs], dim=-1), torch.stack([lo, hi], dim=-2).half())


def _quantized(k, v, lens):
    """Cache tensors of rows [G,H,N,D]; rows behind lens[g] are not in use."""
    G, H, N, D = k.shape
    blocks = (N + BLOCK - 1) // BLOCK
    live = (torch.arange(blocks * BLOCK, device=k.device) < lens[:, None]).view(G, 1, blocks, BLOCK).expand(G, H, -1, -1)
    kb, vb = (torch.where(live[..., None], _blocked(x.float(), blocks), 0.0) for x in (k, v))
    ks, vs = (_scale(x.abs().amax((-1, -2))) for x in (kb, vb))
    return _fields(kb, vb, ks, vs, live)


def _values(codes, scales):
    """codes [..., 2, 64 D] -> k, v [..., 64, D] fp32."""
    lead, D = codes.shape[:-2], codes.shape[-1] // BLOCK
    y = codes.float() - 128.0
    k = y[..., 0, :].reshape(*lead, BLOCK, D)
    place = torch.argsort(_order(codes.device))
    v = y[..., 1, :].reshape(*lead, D, BLOCK)[..., place].transpose(-1, -2)
    return k * scales[..., 0, None, None], v * scales[..., 1, None, None]


def _grouped(q, G):
    """[B,H,Lq,D] -> [G,H,rows of a group,D]"""
    B, H, L, D = q.shape
    return q if G == B else q.permute(1, 0, 2, 3).reshape(1, H, B * L, D)


def _ungrouped(x, B, L):
    G, H = x.shape[:2]
    return x if G == B else x.reshape(H, B, L, *x.shape[3:]).transpose(0, 1)


def _softmax(s, v, zero):
    """Weights from scores [..., keys] with -inf where nothing is seen, values [..., keys, D]: output and log-sum-exp."""
    m = s.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), zero, m)
    e = torch.exp(s - m)
    total = e.sum(-1, keepdim=True)
    out = (e @ v) / torch.where(total > 0, total, 1.0)
    return out, (m + torch.log(total))[..., 0]


def _plain(state):
    c, op = state["case"], state["case"]["op"]
    if op == "quantize":
        k, v, lens = state["k"], state["v"], state["lens"]
        codes, scales, bounds = _quantized(k, v, lens)
        N = k.shape[2]
        kk, vv = (x.flatten(2, 3)[:, :, :N] for x in _values(codes, scales))
        used = (torch.arange(scales.shape[2], device=k.device) * BLOCK < lens[:, None])[:, None, :, None]
        return {"k": kk, "v": vv, "scales": torch.where(used, scales, 0.0),
                "bounds": torch.where(used[..., None], bounds, 0.0), "lens": lens}
    codes, scales, bounds = state["codes"], state["scales"], state["bounds"]
    G, H, blocks = scales.shape[:3]
    if op == "append":
        start, counts, first, J = state["start"], state["counts"], state["first"], state["span"] // BLOCK
        n = state["k_new"].shape[2]
        b = (first[:, None].long() // BLOCK + torch.arange(J, device=first.device))          # [G,J]
        at = (torch.arange(G, device=b.device)[:, None, None], torch.arange(H, device=b.device)[None, :, None], b[:, None])
        row = (b[:, :, None] * BLOCK + torch.arange(BLOCK, device=b.device))                    # [G,J,64]
        old = row < start[:, None, None]
        which = row - start[:, None, None]
        fresh = ~old & (which < counts[:, None, None])
        was_c, was_s, was_b = codes[at], scales[at], bounds[at]
        src = which.clamp(0, n - 1)
        g = torch.arange(G, device=b.device)[:, None, None, None]
        h = torch.arange(H, device=b.device)[None, :, None, None]
        rows, tops = [], []
        has_old = old.any(-1)[:, None]
        for i, (x, was) in enumerate(zip((state["k_new"], state["v_new"]), _values64(was_c, was_s))):
            new = torch.where(fresh[:, None, ..., None], x.float()[g, h, src[:, None]], 0.0)
            top = _scale(new.abs().amax((-1, -2)))
            tops.append(torch.maximum(top, torch.where(has_old, was_s[..., i], 0.0)))
            rows.append(torch.where(old[:, None, ..., None], was, new.double()))
        live = (old | fresh)[:, None].expand(G, H, J, BLOCK)
        new_c, new_s, new_b = _fields(*rows, *tops, live)
        touched = fresh.any(-1)[:, None].expand(G, H, J)
        codes[at] = torch.where(touched[..., None, None], new_c, was_c)
        scales[at] = torch.where(touched[..., None], new_s, was_s)
        bounds[at] = torch.where(touched[..., None, None], new_b, was_b)
        end = start + counts
        state["lens"].copy_(end)
        seen = (row < end[:, None, None])[:, None, ..., None]
        k, v = (torch.where(seen, x, 0.0).reshape(G, H, J * BLOCK, -1) for x in _values(codes[at], scales[at]))
        return {"k": k, "v": v, "lens": state["lens"]}
    q, lens = state["q"].float(), state["lens"]
    B, _, L, D = q.shape
    if op == "attend":
        k, v = (x.flatten(2, 3) for x in _values(codes, scales))
        s = _grouped(q, G) @ k.transpose(-1, -2) * D ** -0.5
        seen = torch.arange(blocks * BLOCK, device=q.device) < lens[:, None, None, None]
        out, lse = _softmax(s.masked_fill(~seen, -math.inf), v, s.new_zeros(()))
        return _ungrouped(out, B, L).to(state["q"].dtype), _ungrouped(lse, B, L)
    if op == "select":
        r = _scale(q.abs().amax(-1, keepdim=True))
        qi = _grouped(_nearest(q, r), G)                               # whole numbers: the sums are exact
        lo, hi = bounds[..., 0, :].float(), bounds[..., 1, :].float()
        top = qi.clamp(min=0) @ hi.transpose(-1, -2) + qi.clamp(max=0) @ lo.transpose(-1, -2)
        score = top * scales[..., None, :, 0]
        there = torch.arange(blocks, device=q.device) * BLOCK < lens[:, None, None, None]
        score = score.masked_fill(~there, -math.inf)
        n = min(state["pick"], blocks)
        best, index = torch.sort(score, dim=-1, descending=True, stable=True)
        index = torch.where(torch.isinf(best[..., :n]), blocks, index[..., :n]).sort(dim=-1).values
        index = torch.where(index == blocks, -1, index).int()
        full = index.new_full((*index.shape[:-1], state["pick"]), -1)
        full[..., :n] = index
        return _ungrouped(full, B, L)
    index = state["index"].long()                                      # [B,H,L,S]
    b = torch.arange(B, device=q.device).clamp(max=G - 1).view(B, 1, 1, 1)
    h = torch.arange(H, device=q.device).view(1, H, 1, 1)
    i = index.clamp(min=0)
    k, v = (x.flatten(3, 4) for x in _values(codes[b, h, i], scales[b, h, i]))
    s = (k @ q[..., None])[..., 0] * D ** -0.5
    row = (i[..., None] * BLOCK + torch.arange(BLOCK, device=q.device))
    seen = (index >= 0)[..., None] & (row < lens[b][..., None])
    out, lse = _softmax(s.masked_fill(~seen.flatten(3), -math.inf)[..., None, :], v, s.new_zeros(()))
    return out[..., 0, :].to(state["q"].dtype), lse[..., 0]


def _values64(codes, scales):
    return _values(codes, scales.double())


# ------------------------------------------------------------------ the framework's operators

def _package():
    root = os.path.join(os.getcwd(), "ar-nanotabpfn_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from ar_tabpfn.model import context_cache
    return context_cache


def _own(state):
    cc, op = _package(), state["case"]["op"]
    if op == "quantize":
        cache = cc.quantize_context(state["k"], state["v"], lens=state["lens"] if state["case"]["ragged"] else None)
        k, v = cc.read_context(cache)
        return {"k": k, "v": v, "scales": cache.scales, "bounds": cache.bounds, "lens": cache.lens}
    cache = cc.ContextCache(state["codes"], state["scales"], state["bounds"], state["lens"])
    if op == "append":
        cc.append_context(cache, state["k_new"], state["v_new"], counts=state["counts"], start=state["start"])
        k, v = cc.read_context(cache, start=state["first"], n=state["span"])
        return {"k": k, "v": v, "lens": cache.lens}
    if op == "attend":
        return cc.context_cache_attention(state["q"], cache)
    if op == "select":
        return cc.select_context_blocks(state["q"], cache, state["pick"])
    return cc.block_context_attention(state["q"], cache, state["index"])


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ inputs

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)
    randn = lambda *s: torch.randn(*s, device="cuda", generator=g)
    dtype = TYPES[c["type"]]
    B, H, D, N, L = c["batch"], c["heads"], c["head_dim"], c["ctx"], c["queries"]
    G = 1 if c["shared"] else B
    lens = torch.full((G,), N, dtype=torch.int32, device="cuda")
    if c["ragged"]:
        lens = (N // 4 + rand(G) * (N - N // 4 + 1)).int().clamp(max=N)
        if G >= 8:
            lens[-1] = 0
    # keys and values as a layer projects them: channels of different spread and offset, rows that drift
    spread, offset = 0.3 + 1.2 * rand(2, 1, H, 1, D), randn(2, 1, H, 1, D)
    drift = 1.0 + 0.5 * torch.sin(torch.arange(N, device="cuda") / 97.0)[:, None]
    k, v = (randn(G, H, N, D).mul_(drift).mul_(spread[i]).add_(offset[i]).to(dtype) for i in range(2))
    state = {"case": c, "lens": lens}
    if c["op"] == "quantize":
        return state | {"k": k, "v": v}
    if c["op"] == "append":
        n = c["new"]
        span = ((n + 63 + 63) // BLOCK) * BLOCK
        blocks = (N + span + BLOCK - 1) // BLOCK
        wide = lambda x: torch.cat([x, x.new_zeros(G, H, blocks * BLOCK - N, D)], dim=2)
        counts = torch.full_like(lens, n)
        if c["ragged"]:
            counts = (n // 2 + rand(G) * (n - n // 2 + 1)).int().clamp(max=n)
        codes, scales, bounds = _quantized(wide(k), wide(v), lens)
        k_new, v_new = (randn(G, H, n, D).mul_(1.3).mul_(spread[i]).add_(offset[i]).to(dtype) for i in range(2))
        return state | {"codes": codes, "scales": scales, "bounds": bounds, "k_new": k_new, "v_new": v_new,
                        "start": lens.clone(), "counts": counts, "first": lens // BLOCK * BLOCK, "span": span}
    codes, scales, bounds = _quantized(k, v, lens)
    del k, v
    q = (randn(B, H, L, D) + 0.3 * offset[0]).to(dtype)
    state |= {"codes": codes, "scales": scales, "bounds": bounds, "q": q}
    if c["op"] == "select":
        state["pick"] = c["pick"]
    if c["op"] == "blocks":
        held = ((lens + BLOCK - 1) // BLOCK).view(G, 1, 1, 1)
        blocks, S = scales.shape[2], c["pick"]
        key = torch.where(torch.arange(blocks, device="cuda") < held, rand(B, H, L, blocks), 2.0)
        n = min(S, blocks)
        low, index = torch.topk(key, n, dim=-1, largest=False)
        index = torch.where(low < 2.0, index, blocks).sort(dim=-1).values
        full = torch.full((B, H, L, S), -1, dtype=torch.int32, device="cuda")
        full[..., :n] = torch.where(index < blocks, index, -1).int()
        state["index"] = full
    return state


# ------------------------------------------------------------------ in 64 bits, from the definitions

def _row_place():
    place = [0] * BLOCK
    for p, r in enumerate(ROW_ORDER):
        place[r] = p
    return place


def _decoded(codes, scales):
    """Real keys and values [G,H,rows,D] that the fields stand for."""
    G, H, nb, _, size = codes.shape
    D = size // BLOCK
    whole = codes.to(torch.float64).sub_(128)
    k = whole[:, :, :, 0].reshape(G, H, nb * BLOCK, D)
    v = whole[:, :, :, 1].reshape(G, H, nb, D, BLOCK)[..., _row_place()].permute(0, 1, 2, 4, 3).reshape(G, H, nb * BLOCK, D)
    per_row = scales.double().repeat_interleave(BLOCK, dim=2)
    return k * per_row[..., :1], v * per_row[..., 1:]


def _rounded_rows(x, lens):
    """What 8 bits keep of rows [G,H,N,D]; with the scale of every block."""
    G, H, N, D = x.shape
    nb = -(-N // BLOCK)
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, nb * BLOCK - N))
    row = torch.arange(nb * BLOCK, device=x.device)
    x = x * (row[None, :] < lens[:, None])[:, None, :, None]
    x = x.reshape(G, H, nb, BLOCK * D)
    step = (x.abs().max(-1).values / 127.0).float().double()
    whole = torch.nan_to_num(x / step[..., None]).round()
    return whole.reshape(G, H, nb, BLOCK, D), step


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "select":
        return None
    if op == "quantize":
        lens, N = s["lens"], s["k"].shape[2]
        out, steps = {}, []
        for name in ("k", "v"):
            whole, step = _rounded_rows(s[name], lens)
            out[name] = (whole * step[..., None, None]).flatten(2, 3)[:, :, :N]
            steps.append(step)
            if name == "k":
                row = torch.arange(whole.shape[2] * BLOCK, device=whole.device).view(1, 1, -1, BLOCK, 1)
                gone = row >= lens.view(-1, 1, 1, 1, 1)
                lo = whole.masked_fill(gone, math.inf).min(3).values
                hi = whole.masked_fill(gone, -math.inf).max(3).values
                edges = torch.stack([lo, hi], dim=3)
                edges[torch.isinf(edges)] = 0.0
        return {**out, "scales": torch.stack(steps, dim=-1), "bounds": edges, "lens": None}
    if op == "append":
        k, v = _decoded(s["codes"], s["scales"])
        G, H, rows, D = k.shape
        out = {"lens": None}
        row = torch.arange(rows, device=k.device)
        start, end = s["start"].long(), (s["start"] + s["counts"]).long()
        nb = rows // BLOCK
        for i, (name, x) in enumerate((("k", k), ("v", v))):
            fresh = (row >= start[:, None]) & (row < end[:, None])
            src = (row - start[:, None]).clamp(0, s[name + "_new"].shape[2] - 1)
            new = s[name + "_new"].double().gather(2, src[:, None, :, None].expand(G, H, rows, D))
            f, o = fresh[:, None, :, None], (row < start[:, None])[:, None, :, None]
            x = torch.where(f, new, torch.where(o, x, 0.0)).reshape(G, H, nb, BLOCK, D)
            f, o = f.reshape(G, 1, nb, BLOCK, 1), o.reshape(G, 1, nb, BLOCK, 1)
            top = ((x * f).abs().flatten(3).max(-1).values / 127.0).float().double()
            was = s["scales"][..., i].double()
            step = torch.maximum(top, torch.where(o.any(3)[..., 0], was, 0.0))
            step = torch.where(f.any(3)[..., 0], step, was)[..., None, None]
            x = (torch.nan_to_num(x / step).round().clamp(-127, 127) * step).reshape(G, H, rows, D)
            at = (s["first"].long()[:, None] + torch.arange(s["span"], device=k.device))
            got = x.gather(2, at[:, None, :, None].expand(G, H, -1, D))
            out[name] = got * (at < end[:, None])[:, None, :, None]
        return out
    q = s["q"].double()
    B, H, L, D = q.shape
    if B * H * L * case["ctx"] > 5e8:
        return None
    k, v = _decoded(s["codes"], s["scales"])
    G, rows = k.shape[0], k.shape[2]
    row = torch.arange(rows, device=k.device)
    if op == "attend":
        weight = torch.einsum("bhld,bhnd->bhln", q, k.expand(B, -1, -1, -1)) / math.sqrt(D)
        weight = weight.masked_fill((row >= s["lens"][:, None]).view(G, 1, 1, rows), -math.inf)
        lse = torch.logsumexp(weight, dim=-1)
        part = torch.nan_to_num(torch.exp(weight - lse[..., None]))
        return torch.einsum("bhln,bhnd->bhld", part, v.expand(B, -1, -1, -1)), lse
    times = torch.zeros(B, H, L, rows // BLOCK + 1, dtype=torch.float64, device=k.device)
    index = s["index"].long()
    times.scatter_add_(3, torch.where(index < 0, rows // BLOCK, index), torch.ones_like(index, dtype=torch.float64))
    often = times[..., :-1].repeat_interleave(BLOCK, dim=3) * (row < s["lens"].view(-1, 1, 1, 1))
    weight = torch.einsum("bhld,bhnd->bhln", q, k.expand(B, -1, -1, -1)) / math.sqrt(D) + torch.log(often)
    lse = torch.logsumexp(weight, dim=-1)
    part = torch.nan_to_num(torch.exp(weight - lse[..., None]))
    return torch.einsum("bhln,bhnd->bhld", part, v.expand(B, -1, -1, -1)), lse

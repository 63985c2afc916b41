"""Operators over a paged K/V cache held in 8 bits (e4m3) with a scale for each block of tokens and head, as timed cases.

  write   ``ops.reshape_and_cache_flash(..., "fp8", k_scale, v_scale)``: rows of prompts or single new tokens into the blocks
  decode  ``attention.paged_decode_attention(..., k_scale=, v_scale=)``: one query row per request over its blocks
  prefix  ``attention.paged_prefix_attention``: several new tokens per request over the request's whole context, causal
  step    ``FlashAttentionImpl.forward`` with ``kv_cache_dtype="fp8"`` on decode tokens: write and attention in one call

Element x of a row of block b and head h is held as the e4m3 number nearest to x / s[b, h]; s is the smallest power of two (not
below 2^-118) with |x| <= 448 s for every finite element of the rows that the block was given.  A write that reaches a block's first
slot starts the block anew; one that starts later keeps the larger of the two scales and rounds the block's other rows to it.

``own`` is False: ``run`` computes the plain forms in fp32.  True: it calls the package.
Lengths belong to the case (drawn from its ``mix`` number), values to the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn
# heads, head size: 125m, 1.3b, 13b and one rank of eight of 66b
HEADS = [(12, 64), (32, 64), (40, 128), (9, 128)]


def _case(op, heads, head_size, dtype, batch, context, new, mix, longest=2048, block=16):
    return {"op": op, "heads": heads, "head_size": head_size, "dtype": dtype, "batch": batch, "context": context, "new": new,
            "mix": mix, "longest": longest, "block": block}


def listed():
    def named(name, *a, **kw):
        return dict(_case(*a, **kw), name=name)
    return [
        # prompts of a prefill batch: rows of whole blocks, the last of each prompt partly filled
        named("write prompts 13b", "write", 40, 128, "fp16", 24, 700, 700, 61),
        # a short prompt of a small model: launch latency
        named("write prompt 125m", "write", 12, 64, "fp32", 1, 37, 37, 62),
        # the new tokens of a full decode batch: blocks that are partly filled, some of them just begun
        named("write tokens 13b", "write", 40, 128, "bf16", 256, 700, 1, 63),
        # a full decode batch of a large model: the largest amount of cache
        named("decode 13b b256", "decode", 40, 128, "fp16", 256, 900, 1, 64),
        # one user with a very long context: one request's blocks for the whole GPU
        named("decode 1.3b long", "decode", 32, 64, "bf16", 1, 30011, 1, 65, longest=32768, block=32),
        # a handful of short chats on the smallest model in fp32: latency
        named("decode 125m fp32", "decode", 12, 64, "fp32", 8, 230, 1, 66),
        # plain serving, one rank of eight: few heads, ragged lengths
        named("step 66b tp8 b128", "step", 9, 128, "bf16", 128, 900, 1, 67),
        # a few short chats: launches and host work of one layer
        named("step 1.3b b5", "step", 32, 64, "fp16", 5, 90, 1, 68),
        # chunks of prompts behind what is cached already
        named("prefix 13b chunks", "prefix", 40, 128, "fp16", 6, 1500, 500, 69),
        # drafted tokens of many requests to be verified: a few query rows over long contexts
        named("prefix 13b drafts", "prefix", 40, 128, "bf16", 64, 700, 5, 70),
        # the last chunk of one long document
        named("prefix 1.3b document", "prefix", 32, 64, "fp16", 1, 16001, 2048, 71, longest=32768),
        # one short turn behind a cached system prompt on the smallest model: latency
        named("prefix 125m turn", "prefix", 12, 64, "bf16", 2, 300, 23, 72, block=32),
    ]


def draw(rng):
    def log_int(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["write", "decode", "decode", "step", "step", "prefix", "prefix"])
    heads, head_size = rng.choice(HEADS)
    dtype = rng.choice(["fp16", "fp16", "bf16", "bf16", "fp32"])
    if dtype == "fp32" and (op == "prefix" or (heads, head_size) != (12, 64)):
        dtype = "bf16"
    long = rng.random() < 0.2
    longest = 32768 if long else 2048
    batch = log_int(1, 4 if long else 256)
    context = log_int(2048, 30000) if long else log_int(20, 1500)
    new = 1
    if op == "write":
        new = rng.choice([1, context])
    elif op == "prefix":
        new = log_int(1, min(2048, context))
    c = _case(op, heads, head_size, dtype, batch, context, new, rng.randrange(10 ** 6), longest, rng.choice([16, 16, 32]))
    most_bytes = max(work(x)["bytes"] for x in listed() if x["op"] == ("decode" if op == "step" else op))
    most_flops = max(work(x)["flops"] for x in listed())
    while c["batch"] > 1 and (work(c)["bytes"] > most_bytes or work(c)["flops"] > most_flops):
        c["batch"] = max(1, c["batch"] * 3 // 4)
    while work(c)["bytes"] > most_bytes or work(c)["flops"] > most_flops:
        c["context"] = c["context"] * 3 // 4
        c["new"] = c["context"] if op == "write" and c["new"] > 1 else min(c["new"], c["context"])
    return c


# ---- sizes ------------------------------------------------------------------------------
def _lengths(case):
    """Tokens of each request after the call, and how many of them are new."""
    rng = np.random.default_rng(case["mix"])
    n = case["batch"]
    lens = np.clip(np.rint(rng.lognormal(math.log(case["context"]), 0.5, size=n)), 1, case["longest"]).astype(int)
    if n == 1:
        lens[0] = case["context"]
    if case["new"] == 1:
        new = np.ones(n, dtype=int)
    elif case["op"] == "write":
        new = lens.copy()
    else:
        new = np.clip(np.rint(rng.lognormal(math.log(case["new"]), 0.3, size=n)), 1, 2048).astype(int)
        if n == 1:
            new[0] = case["new"]
        new = np.minimum(new, lens)
    return lens, new


def work(case):
    """Bytes and operations of one pass, each input read and each output written once."""
    lens, new = _lengths(case)
    h, d, bs = case["heads"], case["head_size"], case["block"]
    es = 4 if case["dtype"] == "fp32" else 2
    t, row = int(new.sum()), case["heads"] * case["head_size"]
    blocks = int(sum(-(-n // bs) for n in lens))
    touched = int(sum((n - 1) // bs - (n - k) // bs + 1 for n, k in zip(lens, new)))
    write = t * row * 2 * (es + 1) + t * 8 + touched * h * 8 * 2
    attend = int(lens.sum()) * row * 2 + blocks * (h * 8 + 4) + t * row * 2 * es
    pairs = float(sum(k * (n - k) + k * (k + 1) / 2 for n, k in zip(lens, new)))
    flops = 4.0 * pairs * row
    if case["op"] == "write":
        return {"bytes": float(write), "flops": 4.0 * t * row}
    if case["op"] == "step":
        return {"bytes": float(attend + write), "flops": flops}
    return {"bytes": float(attend), "flops": flops}


# ---- inputs -----------------------------------------------------------------------------
def _power_of_two(top):
    """The smallest power of two s >= 2^-118 with top <= 448 s."""
    mantissa, exponent = torch.frexp(top.clamp_min(2.0 ** -120))
    return torch.ldexp(torch.ones_like(top), (exponent - 9 + (mantissa > 0.875)).clamp(-118, 120))


def prepare(case, seed):
    lens, new = _lengths(case)
    h, d, bs, n = case["heads"], case["head_size"], case["block"], case["batch"]
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    dev, dtype = "cuda", DTYPES[case["dtype"]]
    per = [-(-int(x) // bs) for x in lens]
    nb = sum(per) + 8
    ids = torch.randperm(nb, generator=g, device=dev, dtype=torch.int32)   # blocks are handed out in any order
    tables = torch.zeros(n, max(per), dtype=torch.int32, device=dev)
    at = torch.tensor([r * max(per) + j for r in range(n) for j in range(per[r])], device=dev)
    tables.view(-1)[at] = ids[:sum(per)]
    # heads differ in size; a head's cached values are normal
    spread = torch.exp(0.5 * torch.randn(2, h, generator=g, device=dev))
    cache = torch.empty(2, nb, bs, h, d, dtype=E4M3, device=dev)
    scales = torch.empty(2, nb, h, device=dev)
    for plane in (0, 1):
        x = torch.randn(nb, bs, h, d, generator=g, device=dev).mul_(spread[plane].view(h, 1))
        scales[plane] = _power_of_two(x.abs().amax(dim=(1, 3)))
        cache[plane] = x.div_(scales[plane].view(nb, 1, h, 1)).to(E4M3)
        del x
    t = int(new.sum())
    qkv = torch.randn(t, 3, h, d, generator=g, device=dev)   # the step's projection, query, key and value its thirds
    qkv[:, 1:] *= spread.view(2, h, 1)
    qkv = qkv.to(dtype).view(t, 3 * h * d)
    q, k, v = qkv.split(h * d, dim=1)
    req = np.repeat(np.arange(n), new)
    pos = np.concatenate([np.arange(a - b, a) for a, b in zip(lens, new)])
    req_d, pos_d = torch.from_numpy(req).to(dev), torch.from_numpy(pos).to(dev)
    slots = tables[req_d, pos_d // bs].long() * bs + pos_d % bs
    blocks, groups = np.unique(req * (case["longest"] // bs + 1) + pos // bs, return_inverse=True)
    first = torch.from_numpy(blocks).to(dev)
    width = case["longest"] // bs + 1
    state = {"case": dict(case), "cache": cache, "scales": scales, "q": q, "k": k.view(t, h, d), "v": v.view(t, h, d), "tables": tables,
             "lens": torch.tensor(lens, dtype=torch.int32, device=dev), "slots": slots, "scale": d ** -0.5,
             "starts": torch.tensor(np.concatenate([[0], np.cumsum(new)]), dtype=torch.int32, device=dev), "most_new": int(new.max()),
             # of the plain form: the blocks that the rows go to, each row's place among them, and the padded query
             "blocks": tables[first // width, first % width].long(), "groups": torch.from_numpy(groups.reshape(-1)).to(dev),
             "rows": req_d, "row_in": torch.from_numpy(np.concatenate([np.arange(b) for b in new])).to(dev)}
    return state


# ---- plain forms ------------------------------------------------------------------------
def _plain_write(cache, scales, x, s):
    """One plane: cache [NB, BS, H, D], scales [NB, H], x [T, H, D]."""
    bs = cache.shape[1]
    x = x.float()
    top = torch.where(torch.isfinite(x), x.abs(), torch.zeros_like(x)).amax(dim=2)
    g, h = s["blocks"].numel(), x.shape[1]
    need = torch.zeros(g, h, device=x.device).scatter_reduce_(0, s["groups"][:, None].expand(-1, h), top, "amax")
    anew = torch.zeros(g, device=x.device).scatter_reduce_(0, s["groups"], (s["slots"] % bs == 0).float(), "amax")[:, None] > 0
    old = scales[s["blocks"]]
    new = torch.where(anew, _power_of_two(need), torch.maximum(old, _power_of_two(need)))
    ratio = torch.where(anew, torch.ones_like(new), old / new)
    held = cache.view(torch.uint8)
    kept = held[s["blocks"]].view(E4M3).float() * ratio[:, None, :, None]
    held[s["blocks"]] = kept.to(E4M3).view(torch.uint8)
    held.view(-1, *x.shape[1:])[s["slots"]] = (x / new[s["groups"]][:, :, None]).to(E4M3).view(torch.uint8)
    scales[s["blocks"]] = new


def _plain_rows(cache, scales, s):
    """One plane's rows by request, [B, L, H, D] in fp32, zeros behind a request's last token."""
    ids = s["tables"].long()
    b, w = ids.shape
    _, bs, h, d = cache.shape
    x = cache.view(torch.uint8)[ids].view(E4M3).float() * scales[ids][:, :, None, :, None]
    x = x.view(b, w * bs, h, d)
    behind = torch.arange(w * bs, device=x.device)[None, :] >= s["lens"][:, None]
    return x.masked_fill_(behind[:, :, None, None], 0.0)


def _plain_attention(s):
    """Every request's new tokens, the last of its context, over the tokens up to each."""
    kc, vc = s["cache"]
    _, _, h, d = kc.shape
    b, m = s["tables"].shape[0], s["most_new"]
    q = torch.zeros(b, m, h, d, device=kc.device)
    q[s["rows"], s["row_in"]] = s["q"].float().view(-1, h, d)
    scores = torch.matmul(q.transpose(1, 2), _plain_rows(kc, s["scales"][0], s).permute(0, 2, 3, 1)) * s["scale"]   # [B, H, M, L]
    new = s["starts"][1:] - s["starts"][:-1]
    last = (s["lens"] - new)[:, None] + torch.arange(m, device=kc.device)   # a query row's own position
    ahead = torch.arange(scores.shape[3], device=kc.device)[None, None, :] > last[:, :, None]
    scores.masked_fill_(ahead[:, None], float("-inf"))
    scores -= scores.amax(dim=3, keepdim=True)
    scores.exp_()
    total = scores.sum(dim=3, keepdim=True)
    out = torch.matmul(scores, _plain_rows(vc, s["scales"][1], s).transpose(1, 2)) / total
    out = out.transpose(1, 2)[s["rows"], s["row_in"]]
    return out.reshape(-1, h * d).to(s["q"].dtype)


def _metadata(s):
    """What the engine's model runner hands to every layer of a decode step."""
    from apt_serve_b200 import attention as A
    n = s["tables"].shape[0]
    none = s["slots"][:0]
    return A.FlashAttentionMetadata(
        num_prefills=0, num_prefill_tokens=0, num_decode_tokens=n, num_hidden_cache_tokens=0, num_tot_tokens=n,
        slot_mapping=s["slots"], slot_mapping_shared=none, hidden_cache_use_tot=none, kv_cache_use_tot=none,
        hidden_cache_use_input=none, hidden_cache_store_tot=none, hidden_holder_upd=none, hidden_holder_pull=none, seq_lens=None,
        seq_lens_tensor=s["lens"], max_query_len=1, max_prefill_seq_len=0, max_decode_seq_len=s["case"]["longest"],
        query_start_loc=None, seq_start_loc=None, context_lens_tensor=None, block_tables=s["tables"], use_cuda_graph=False)


def run(state):
    s, op = state, state["case"]["op"]
    if own:
        from apt_serve_b200 import attention as A
        from apt_serve_b200 import ops
        if op == "write":
            ops.reshape_and_cache_flash(s["k"], s["v"], s["cache"][0], s["cache"][1], s["slots"], "fp8", s["scales"][0], s["scales"][1])
            return {"cache": s["cache"], "scales": s["scales"]}
        if op == "decode":
            return A.paged_decode_attention(s["q"], s["cache"][0], s["cache"][1], s["tables"], s["lens"], s["scale"],
                                            k_scale=s["scales"][0], v_scale=s["scales"][1])
        if op == "prefix":
            return A.paged_prefix_attention(s["q"], s["cache"][0], s["cache"][1], s["tables"], s["starts"], s["lens"], s["most_new"],
                                            s["scale"], s["scales"][0], s["scales"][1])
        if "layer" not in s:   # what an engine keeps: the layer's attention and the step's metadata
            h, d = s["case"]["heads"], s["case"]["head_size"]
            s["layer"] = A.FlashAttentionImpl(h, d, s["scale"], h, None, None, "fp8"), _metadata(s)
        impl, meta = s["layer"]
        t, h, d = s["k"].shape
        out = impl.forward(s["q"], s["k"].view(t, h * d), s["v"].view(t, h * d), s["cache"], None, meta, s["scales"])
        return {"out": out, "cache": s["cache"], "scales": s["scales"]}
    if op in ("write", "step"):
        _plain_write(s["cache"][0], s["scales"][0], s["k"], s)
        _plain_write(s["cache"][1], s["scales"][1], s["v"], s)
        if op == "write":
            return {"cache": s["cache"], "scales": s["scales"]}
        return {"out": _plain_attention(s), "cache": s["cache"], "scales": s["scales"]}
    return _plain_attention(s)


# ---- the definition in 64 bits ------------------------------------------------------------
def _exact_write(s, plane, x, values):
    """The blocks' values over their scales (not rounded) into ``values``; returns the scales."""
    codes, scales = s["cache"][plane], s["scales"][plane].double()
    bs = codes.shape[1]
    values.copy_(codes)
    slots = s["slots"].tolist()
    of_block = {}
    for t, slot in enumerate(slots):
        of_block.setdefault(slot // bs, []).append((t, slot % bs))
    # blocks that take the same number of rows, from the same slot on, are handled together
    alike = {}
    for b, rows in of_block.items():
        alike.setdefault((len(rows), rows[0][1]), []).append((b, rows[0][0]))
    for (count, offset), some in alike.items():
        ids = torch.tensor([b for b, _ in some], device=codes.device)
        t = torch.tensor([a for _, a in some], device=codes.device)[:, None] + torch.arange(count, device=codes.device)
        new = x[t].double()                                              # [blocks, count, H, D]
        part, power = torch.frexp(new.abs().amax(dim=(1, 3)).clamp_min(1e-60) / 448)   # a half exactly: the ratio is a power of two
        need = torch.ldexp(torch.ones_like(part), (power - (part == 0.5).int()).clamp_min(-118))
        if offset > 0:
            s_new = torch.maximum(need, scales[ids])
            block = values[ids] * (scales[ids] / s_new)[:, None, :, None]
        else:
            s_new, block = need, values[ids]
        block[:, offset:offset + count] = new / s_new[:, None, :, None]
        values[ids] = block
        scales[ids] = s_new
    return scales


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    answer = {}
    if op in ("write", "step"):
        values = torch.empty(s["cache"].shape, dtype=torch.float64, device="cuda")
        answer = {"cache": values, "scales": torch.stack([_exact_write(s, p, s[n], values[p]) for p, n in ((0, "k"), (1, "v"))])}
        if op == "write":
            return answer
        # what is attended is what the 8 bits hold, which the rounding decides: to the nearest, as the definition says
        s["cache"].copy_(values.to(E4M3))
        s["scales"].copy_(answer["scales"])
    _, _, bs, h, d = s["cache"].shape
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for r, n in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        ids = s["tables"][r, :-(-n // bs)].long()
        q = s["q"][a:b].double().view(b - a, h, d).transpose(0, 1)
        k, v = ((s["cache"][p].view(torch.uint8)[ids].view(E4M3).double() * s["scales"][p][ids].double()[:, None, :, None])
                .flatten(0, 1)[:n].transpose(0, 1) for p in (0, 1))
        row, col = torch.arange(n - (b - a), n, device="cuda")[:, None], torch.arange(n, device="cuda")[None, :]
        for lo in range(0, h, 8):   # some heads at a time: a document's scores take gigabytes
            p = torch.softmax((q[lo:lo + 8] @ k[lo:lo + 8].transpose(1, 2) * s["scale"]).masked_fill(col > row, -math.inf), dim=2)
            out[a:b, lo * d:(lo + 8) * d] = (p @ v[lo:lo + 8]).transpose(0, 1).reshape(b - a, -1)
            del p
    return {**answer, "out": out} if answer else out

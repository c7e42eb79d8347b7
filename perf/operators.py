"""Measured cases of the KV-cache operators: writing new tokens into a cache (append_kv, 8 bits or
as they are), reading a cache back (gather_kv), attention of a chunk of new tokens over a cache
(extend) and the single-token decode over an 8-bit cache (decode with scales).

A case is a batch of sequences: sequence b has a context of lens[b] keys, of which the last new[b]
are the tokens of this call. Caches are contiguous [B, S_max, H_kv, D] or paged
[num_blocks, page, H_kv, D] with shuffled pages; an 8-bit cache has one fp32 scale per token and
KV head. The plain form works on padded sequences in fp32 and rounds once at the end.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16}
_TINY = 2.0 ** -100   # smallest scale of an 8-bit row


# --------------------------------------------------------------------------------------------
# Cases
# --------------------------------------------------------------------------------------------

def _case(op, batch, new, ctx, heads, heads_kv, dim, dtype, int8, page, causal=True, spread=0,
          **more):
    """new / ctx: (lowest, highest) new tokens and earlier keys per sequence."""
    return dict(op=op, batch=batch, new_lo=new[0], new_hi=new[1], ctx_lo=ctx[0], ctx_hi=ctx[1],
                heads=heads, heads_kv=heads_kv, dim=dim, dtype=dtype, int8=int8, page=page,
                causal=causal, spread=spread, **more)


def listed():
    def named(name, *args, **kw):
        return dict(_case(*args, **kw), name=name)

    return [
        # One decode step's K/V of 8 short sequences written to an 8-bit paged cache and read back:
        # a call whose launch latency is all that counts.
        named("append_i8_step", "append", 8, (1, 1), (5, 40), 32, 8, 128, "bf16", True, 16),
        # Eight ragged prompts, about 16K tokens, quantised as they are written and read back (a
        # prefix handed to another worker).
        named("append_i8_prompts", "append", 8, (900, 3300), (0, 0), 32, 8, 128, "bf16", True, 16),
        # The same path without quantisation: ragged multi-head chunks into a contiguous cache.
        named("append_f16_chunks", "append", 6, (301, 1500), (0, 700), 32, 32, 64, "fp16", False, 0),
        # Reading back a short shared prefix of an 8-bit cache.
        named("gather_i8_prefix", "gather", 3, (0, 0), (33, 200), 32, 8, 128, "fp16", True, 32),
        # Whole long contexts read back from 8 bits, contiguous cache.
        named("gather_i8_long", "gather", 8, (0, 0), (5000, 16384), 32, 8, 128, "bf16", True, 0),
        # Speculative decoding: five proposed tokens per sequence checked against 1K-2K keys.
        named("extend_verify", "extend", 4, (5, 5), (1000, 2040), 32, 8, 128, "bf16", False, 16),
        # Chunked prefill: a chunk of 2048 prompt tokens after 16K keys already in 64-row pages.
        named("extend_chunk", "extend", 1, (2048, 2048), (16384, 16384), 32, 8, 128, "bf16", False, 64),
        # A serving step that mixes decoding sequences with prompt chunks, 8-bit paged cache.
        named("extend_i8_mixed", "extend", 10, (1, 600), (300, 6000), 32, 8, 128, "bf16", True, 16,
              ones=8),
        # Ragged prompts from scratch, multi-head, head_dim 64, contiguous cache (odd lengths).
        named("extend_f16_prompts", "extend", 4, (2500, 4095), (0, 0), 16, 16, 64, "fp16", False, 0),
        # One sequence, one token, a short multi-head cache in 8 bits: latency.
        named("decode_i8_short", "decode", 1, (1, 1), (2047, 2047), 32, 32, 128, "bf16", True, 0),
        # The benchmark's grouped-query decode (8 sequences of 16K to 32K keys), 8-bit 16-row pages.
        named("decode_i8_long", "decode", 8, (1, 1), (16383, 32767), 32, 8, 128, "bf16", True, 16),
        # A larger batch of medium contexts, head_dim 64, contiguous 8-bit cache.
        named("decode_i8_d64", "decode", 24, (1, 1), (200, 8000), 32, 4, 64, "fp16", True, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "gather", "extend", "extend", "decode"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["bf16", "fp16"])
    heads_kv = rng.choice([1, 2, 4, 5, 8, 16, 32])
    group = rng.choice([g for g in (1, 2, 3, 4, 6, 7, 8, 16) if g * heads_kv <= 40])
    page = rng.choice([0, 8, 16, 32, 64, 128, 192])
    spread = rng.randrange(1 << 20)
    while True:
        batch = _log_int(rng, 1, 64)
        if op == "append":
            new, ctx = _log_int(rng, 1, 4096), _log_int(rng, 1, 512)
            case = _case(op, batch, (max(1, new // 3), new), (0, ctx), heads_kv * group, heads_kv,
                         dim, dtype, rng.random() < 0.7, page, spread=spread)
        elif op == "gather":
            ctx = _log_int(rng, 20, 16384)
            case = _case(op, batch, (0, 0), (ctx // 4, ctx), heads_kv * group, heads_kv, dim, dtype,
                         True, page, spread=spread)
        elif op == "extend":
            new, ctx = _log_int(rng, 2, 4096), _log_int(rng, 2, 20000)
            case = _case(op, batch, (max(1, new // 2), new), (rng.choice([0, ctx // 2]), ctx),
                         heads_kv * group, heads_kv, dim, dtype, rng.random() < 0.5, page,
                         causal=rng.random() < 0.8, spread=spread,
                         ones=rng.choice([0, 0, batch // 2]))
        else:
            ctx = _log_int(rng, 1, 32767)
            case = _case(op, batch, (1, 1), (ctx // 3, ctx), heads_kv * group, heads_kv, dim, dtype,
                         True, page, spread=spread)
        w = work(case)
        new_, lens_ = _lengths(case)
        scores = batch * max(new_) * max(lens_) * heads_kv * group
        if w["bytes"] <= 6e8 and w["flops"] <= 5e11 and (op in ("append", "gather") or scores <= 1.2e9) \
                and batch * max(lens_) * heads_kv * dim <= 3e8:
            return case


def _lengths(case):
    """(new tokens, keys with them) of each sequence: a fixed spread over the case's ranges."""
    rng = random.Random(case["spread"])
    new, lens = [], []
    for b in range(case["batch"]):
        n = rng.randint(case["new_lo"], case["new_hi"])
        if b < case.get("ones", 0):
            n = 1
        new.append(n)
        lens.append(max(1, rng.randint(case["ctx_lo"], case["ctx_hi"]) + n))
    return new, lens


def work(case):
    new, lens = _lengths(case)
    tokens, keys = sum(new), sum(lens)
    hkv, d = case["heads_kv"], case["dim"]
    row = d + 4 if case["int8"] else 2 * d          # bytes of one cached row of one head
    if case["op"] == "append":
        moved = 2 * tokens * hkv * (2 * d + row)
        if case["int8"]:
            moved += 2 * keys * hkv * (row + 2 * d)   # the pass reads the sequences back
        return {"bytes": moved, "flops": 2 * tokens * hkv * d * 2}
    if case["op"] == "gather":
        return {"bytes": 2 * keys * hkv * (row + 2 * d), "flops": 2 * keys * hkv * d}
    pairs = 0
    for n, length in zip(new, lens):
        pairs += n * length - (n * (n - 1) // 2 if case["causal"] else 0)
    return {"bytes": 2 * keys * hkv * row + 2 * tokens * case["heads"] * d * 2,
            "flops": 4 * case["heads"] * d * pairs}


# --------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------

def _rows(gen, rows, hkv, d, dev):
    """K-like and V-like rows: a few strong K channels, V of a different size per head."""
    k = torch.randn(rows, hkv, d, device=dev, generator=gen)
    k *= torch.exp2(2.0 * torch.rand(d, device=dev, generator=gen) - 1.0)
    v = torch.randn(rows, hkv, d, device=dev, generator=gen)
    v *= torch.exp2(2.0 * torch.rand(hkv, 1, device=dev, generator=gen) - 1.0)
    return k, v


def _quantise(x):
    """[..., D] fp32 -> (int8 codes, fp32 scales [...])."""
    amax = x.abs().amax(dim=-1)
    codes = torch.round(x * (127.0 / amax).clamp_max(1.0 / _TINY)[..., None]).clamp(-127, 127)
    return codes.to(torch.int8), (amax / 127.0).clamp_min(_TINY)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    new, lens = _lengths(case)
    dtype, hkv, d, page = _DTYPE[case["dtype"]], case["heads_kv"], case["dim"], case["page"]
    batch, longest = case["batch"], max(lens)
    s = dict(op=case["op"], dtype=dtype, causal=case["causal"], int8=case["int8"],
             longest=longest, most_new=max(new), keys=sum(lens), tokens=sum(new),
             scale=1.0 / math.sqrt(d))

    # The cache: pages in shuffled order with a few unused ones, or rows up to a capacity that is
    # no multiple of anything.
    if page:
        need = [-(-n // page) for n in lens]
        blocks = sum(need) + 3
        ids = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).tolist()
        width = max(need)
        table, at = [], 0
        for n in need:
            table.append(ids[at:at + n] + [0] * (width - n))
            at += n
        s["block_tables"] = torch.tensor(table, dtype=torch.int32, device=dev)
        outer, rows = blocks, page
    else:
        s["block_tables"] = None
        outer, rows = batch, longest + 5
    k, v = _rows(gen, outer * rows, hkv, d, dev)
    for name, x in (("k", k), ("v", v)):
        if case["int8"]:
            codes, scale = _quantise(x)
            # Scales are kept head by head, a row's scales side by side along the keys.
            s[name + "_scale"] = scale.view(outer, rows, hkv).transpose(1, 2).contiguous().transpose(1, 2)
            s[name + "_cache"] = codes.view(outer, rows, hkv, d)
        else:
            s[name + "_scale"] = None
            s[name + "_cache"] = x.to(dtype).view(outer, rows, hkv, d)
    del k, v

    def offsets(n):
        return torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], dtype=torch.int32, device=dev)

    s["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    s["cu_new"], s["cu_keys"] = offsets(new), offsets(lens)
    heads = case["heads"]
    if case["op"] == "append":
        # k and v are slices of a packed q, k, v projection.
        k, v = _rows(gen, s["tokens"], hkv, d, dev)
        packed = torch.randn(s["tokens"], heads + 2 * hkv, d, device=dev, generator=gen)
        packed[:, heads:heads + hkv], packed[:, heads + hkv:] = k, v
        packed = packed.to(dtype)
        s["k"], s["v"] = packed[:, heads:heads + hkv], packed[:, heads + hkv:]
    elif case["op"] != "gather":
        s["q"] = torch.randn(s["tokens"], heads, d, device=dev, generator=gen).to(dtype)
    return s


# --------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------

def run(state):
    return _own(state) if own else _plain(state)


def _flash_lab():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "flash-attention-lab_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import flash_lab
    return flash_lab


def _own(s):
    fl = _flash_lab()
    cache = dict(block_tables=s["block_tables"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if s["op"] == "append":
        fl.append_kv(s["k"], s["v"], s["k_cache"], s["v_cache"], s["seq_lens"], s["cu_new"], **cache)
        if not s["int8"]:
            return s["k_cache"], s["v_cache"]
    if s["op"] in ("append", "gather"):
        return fl.gather_kv(s["k_cache"], s["v_cache"], s["seq_lens"], s["cu_keys"], s["keys"],
                            dtype=s["dtype"], **cache)
    if s["op"] == "extend":
        return fl.extend(s["q"], s["k_cache"], s["v_cache"], s["seq_lens"], s["cu_new"],
                         causal=s["causal"], return_lse=True, **cache)
    return fl.decode(s["q"], s["k_cache"], s["v_cache"], s["seq_lens"], return_lse=True, **cache)


def _token_places(cu, tokens):
    """For each of the ragged tokens: its sequence and its place in it."""
    at = torch.arange(tokens, device=cu.device)
    b = torch.searchsorted(cu[1:].long().contiguous(), at, right=True)
    return b, at - cu[b]


def _slots(s, b, pos):
    """(outer, row) of key pos of sequence b in the cache."""
    if s["block_tables"] is None:
        return b, pos
    page = s["k_cache"].shape[1]
    return s["block_tables"][b, pos // page].long(), pos % page


def _values(s, name, outer, row, dtype):
    """Cached rows as the values they stand for."""
    x = s[name + "_cache"][outer, row].to(dtype)
    return x * s[name + "_scale"][outer, row][..., None].to(dtype) if s["int8"] else x


def _plain(s):
    if s["op"] == "append":
        b, i = _token_places(s["cu_new"], s["tokens"])
        n = s["cu_new"][1:] - s["cu_new"][:-1]
        at = _slots(s, b, s["seq_lens"][b] - n[b] + i)
        if not s["int8"]:
            s["k_cache"][at], s["v_cache"][at] = s["k"], s["v"]
            return s["k_cache"], s["v_cache"]
        s["k_cache"][at], s["k_scale"][at] = _quantise(s["k"].float())
        s["v_cache"][at], s["v_scale"][at] = _quantise(s["v"].float())
    if s["op"] in ("append", "gather"):
        at = _slots(s, *_token_places(s["cu_keys"], s["keys"]))
        return (_values(s, "k", *at, torch.float32).to(s["dtype"]),
                _values(s, "v", *at, torch.float32).to(s["dtype"]))

    q = s["q"].float()
    tokens, heads, d = q.shape
    batch, device = s["seq_lens"].shape[0], q.device
    hkv = s["k_cache"].shape[2]
    group, cu = heads // hkv, s["cu_new"].long()
    n = cu[1:] - cu[:-1]
    # Padded queries [B, H_kv, most_new * group, D] and keys [B, H_kv, longest, D].
    i = torch.arange(s["most_new"], device=device)
    q = q[(cu[:-1, None] + i).clamp(max=tokens - 1)].view(batch, -1, hkv, group, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(batch, hkv, -1, d)
    j = torch.arange(s["longest"], device=device)
    at = _slots(s, torch.arange(batch, device=device)[:, None], j[None, :])
    k = _values(s, "k", *at, torch.float32).transpose(1, 2)
    v = _values(s, "v", *at, torch.float32).transpose(1, 2)
    length = s["seq_lens"].long()[:, None, None]
    last = length - n[:, None, None] + i[None, :, None] if s["causal"] else length - 1
    seen = (j <= last) & (j < length)
    scores = torch.matmul(q, k.transpose(2, 3)) * s["scale"]
    scores.masked_fill_(~seen.repeat_interleave(group if s["causal"] else 1, dim=1)[:, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores.sub_(top))
    total = p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p, v) / total
    lse = top + torch.log(total)
    # Back to ragged rows.
    b, i = _token_places(s["cu_new"], tokens)
    out = out.view(batch, hkv, -1, group, d)[b, :, i].reshape(tokens, heads, d)
    lse = lse.view(batch, hkv, -1, group)[b, :, i].reshape(tokens, heads)
    return out.to(s["dtype"]), lse


# --------------------------------------------------------------------------------------------
# The definition in 64 bits, sequence by sequence
# --------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    new, lens = _lengths(case)
    hkv, d, page = case["heads_kv"], case["dim"], case["page"]

    def stored(name, b, first, count):
        """Keys first..first + count - 1 of sequence b: flat indices into the cache's rows."""
        pos = torch.arange(first, first + count, device="cuda")
        if page:
            return s["block_tables"][b].long()[pos // page] * page + pos % page
        return pos + b * s[name + "_cache"].shape[1]

    flat = {}
    for name in ("k", "v"):
        flat[name] = s[name + "_cache"].reshape(-1, hkv, d)
        if case["int8"]:
            flat[name + "_scale"] = s[name + "_scale"].reshape(-1, hkv)

    def values(name, where):
        x = flat[name][where].double()
        return x * flat[name + "_scale"][where].double().unsqueeze(2) if case["int8"] else x

    if case["op"] == "append" and not case["int8"]:
        done = {}
        for name in ("k", "v"):
            full, t = flat[name].double(), 0
            for b, (n, length) in enumerate(zip(new, lens)):
                full[stored(name, b, length - n, n)] = s[name][t:t + n].double()
                t += n
            done[name] = full.view(s[name + "_cache"].shape)
        return done["k"], done["v"]
    if case["op"] in ("append", "gather"):
        done = {}
        for name in ("k", "v"):
            parts, t = [], 0
            for b, (n, length) in enumerate(zip(new, lens)):
                parts.append(values(name, stored(name, b, 0, length - n)))
                if n:
                    x = s[name][t:t + n].double()
                    step = (x.abs().max(dim=2, keepdim=True).values / 127).clamp_min(_TINY)
                    parts.append(torch.round(x / step) * step)
                t += n
            done[name] = torch.cat(parts)
        return done["k"], done["v"]

    group = case["heads"] // hkv
    out = torch.empty(s["tokens"], case["heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.empty(s["tokens"], case["heads"], dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, length) in enumerate(zip(new, lens)):
        k, v = (values(name, stored(name, b, 0, length)) for name in ("k", "v"))
        row = torch.arange(n, device="cuda").unsqueeze(1)
        hidden = torch.arange(length, device="cuda").unsqueeze(0) > row + (length - n)
        for h in range(case["heads"]):
            z = s["q"][t:t + n, h].double() @ k[:, h // group].T / math.sqrt(d)
            if case["causal"]:
                z[hidden] = -math.inf
            lse[t:t + n, h] = torch.logsumexp(z, dim=1)
            out[t:t + n, h] = torch.exp(z - lse[t:t + n, h].unsqueeze(1)) @ v[:, h // group]
        t += n
    return out, lse

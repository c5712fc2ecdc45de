"""A key and value cache held in 4 bits: appending to it, reading it back, attending over it.

A head's numbers lie in groups of sixteen.  A number is a code of 4 bits times its group's scale of 8 bits: code n (0 to
15) in nibble order stands for n - 8, scale byte b for the half-precision number with the bits b << 7, over 64.  Codes are
``[blocks, kv_heads, block_size, dim / 2]`` bytes, scales ``[blocks, kv_heads, block_size, dim / 16]``, for keys and for values.

  append     the queries and keys of float32 q|k|v rows are rotated, keys and values quantised into the cache, and the
             blocks that were written to are read back as the bfloat16 numbers they stand for
  attend     causal grouped-query attention of 1 or more new tokens a sequence over what is cached, window or not

The ranges (``draw``): 1 to 32 query heads on 1 to 32 key heads of 16 to 128 numbers, blocks of 16 to 64 positions, batches
of 1 to 64 equal or ragged sequences, contexts of 1 to 131,072 positions, 1 to 2,048 new tokens, windows or none.
"""
import math
import random

import torch

own = False

GROUP = 16
SCALE_STEPS = 64
LARGEST = 246                                  # the largest scale byte that is written
NOT_FINITE = 255                               # the scale byte of a group that held an infinity or a NaN
THETA = 500000.0


def attend(name, heads, kv, dim, batch, before, new, block=64, window=0, ragged=False):
    return dict({"name": name} if name else {}, op="attend", heads=heads, kv=kv, dim=dim, batch=batch, before=before, new=new,
                block=block, window=window, ragged=ragged)


def append(name, heads, kv, dim, batch, before, new, block=64, ragged=False):
    return dict({"name": name} if name else {}, op="append", heads=heads, kv=kv, dim=dim, batch=batch, before=before, new=new,
                block=block, window=0, ragged=ragged)


def listed():
    return [
        # a decode step's new token of eight sequences, at the headline benchmark's heads
        append("append-step-8", 32, 4, 64, 8, 2000, 1),
        # a long prompt of the wider model in one step
        append("append-prompt-2048", 32, 8, 128, 1, 0, 2048),
        # a batch of short prompts of unequal length, small blocks
        append("append-ragged-8", 32, 32, 128, 8, 0, 333, block=16, ragged=True),
        # one short chat: latency
        attend("step-1x300", 32, 4, 64, 1, 299, 1),
        # the headline benchmark's decode step
        attend("step-8x2048", 32, 4, 64, 8, 2047, 1),
        # a full batch at a middle context
        attend("step-64x4096", 32, 8, 128, 64, 4095, 1),
        # one very long document
        attend("step-1x131072", 32, 8, 128, 1, 131071, 1),
        # sequences of unequal length, a key head per query head, small blocks
        attend("step-ragged-12-mha", 32, 32, 128, 12, 5000, 1, block=16, ragged=True),
        # a sliding window over long contexts
        attend("step-window-32", 32, 8, 128, 32, 9000, 1, window=1024, ragged=True),
        # a few tokens a sequence: drafted ones that are checked at once
        attend("few-4x5", 32, 8, 128, 4, 4000, 5, ragged=True),
        # a whole prompt
        attend("prompt-2048", 32, 4, 64, 1, 0, 2048),
        # a further piece of a long prompt
        attend("prompt-512-behind-8192", 32, 8, 128, 1, 8192, 512),
    ]


MOST_KEYS = 64 * 4096 * 8 * 128                # what the largest listed step keeps: positions x key heads x head size
MOST_PAIRS = 512 * 8704 * 32 * 128             # and the largest prompt multiplies: pairs x heads x head size


def draw(rng):
    heads, kv, dim = rng.choice(((32, 4, 64), (32, 8, 128), (32, 32, 128), (32, 8, 128), (32, 4, 64), (8, 1, 128), (7, 1, 16),
                                 (3, 3, 80), (24, 8, 64), (6, 2, 96)))
    block = rng.choice((16, 32, 64, 64))
    batch = round(2 ** rng.uniform(0, 6))
    kind = rng.random()
    if kind < 0.25:
        case = append("", heads, kv, dim, batch, rng.choice((0, round(2 ** rng.uniform(0, 12)))),
                      1 if rng.random() < 0.4 else round(2 ** rng.uniform(1, 11)), block, rng.random() < 0.6)
    elif kind < 0.7:
        case = attend("", heads, kv, dim, batch, round(2 ** rng.uniform(0, 17)) - 1, 1, block,
                      rng.choice((0, 0, 0, round(2 ** rng.uniform(5, 12)))), rng.random() < 0.6)
    else:
        case = attend("", heads, kv, dim, batch, rng.choice((0, round(2 ** rng.uniform(0, 13)))), round(2 ** rng.uniform(1, 11)), block,
                      rng.choice((0, 0, 0, round(2 ** rng.uniform(5, 12)))), rng.random() < 0.6)
    while True:
        longest = case["before"] + case["new"]
        if (case["batch"] * longest * kv * dim <= MOST_KEYS and case["batch"] * case["new"] * longest * heads * dim <= MOST_PAIRS
                and case["batch"] * case["new"] <= 8192):
            return case
        key = "batch" if case["batch"] > 1 and rng.random() < 0.5 else "before" if case["before"] > case["new"] else "new"
        case[key] = max(1, case[key] // 2)


def lengths(case):
    """(positions cached before the call, new tokens) of each sequence."""
    rng = random.Random(repr([case[k] for k in ("heads", "kv", "dim", "batch", "before", "new", "block", "window")]))
    pick = lambda most, least: rng.randint(min(most, max(least, most // 8)), most) if case["ragged"] else most  # noqa: E731
    before = [pick(case["before"], 0) for _ in range(case["batch"])]
    return before, [pick(case["new"], 1) for _ in range(case["batch"])]


# ---- inputs ----------------------------------------------------------------------------------------------------------

def half_of_byte(device):
    """The half-precision number of each scale byte, as float32."""
    return (torch.arange(256, device=device, dtype=torch.int16) << 7).view(torch.float16).float()


def quantize(x):
    """Codes (packed, two a byte) and scale bytes of float32 numbers ``[..., dim]``."""
    table = half_of_byte(x.device)[:LARGEST + 1] / SCALE_STEPS
    groups = x.unflatten(-1, (-1, GROUP))
    most = groups.abs().amax(-1)
    finite = torch.isfinite(most)
    # the smallest scale of which seven steps reach the largest number (seven times a scale is exact)
    scale = torch.searchsorted(7.0 * table, torch.where(finite, most, torch.zeros_like(most))).clamp(max=LARGEST)
    inverse = torch.where(scale > 0, 1.0 / table[scale], torch.zeros_like(most))
    codes = (groups * inverse[..., None]).round().clamp(-7.0, 7.0)
    codes = torch.where(finite[..., None], codes, torch.zeros_like(codes)).to(torch.int16).flatten(-2) + 8
    packed = (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)
    return packed, torch.where(finite, scale, torch.full_like(scale, NOT_FINITE)).to(torch.uint8)


def dequantize(packed, scale):
    """The float32 numbers that codes and scale bytes stand for."""
    n = torch.stack([packed & 15, packed >> 4], dim=-1).flatten(-2).float() - 8.0
    steps = half_of_byte(packed.device)[scale.long()] / SCALE_STEPS
    return (n.unflatten(-1, (-1, GROUP)) * steps[..., None]).flatten(-2)


def prepare(case, seed):
    device = "cuda"
    gen = torch.Generator(device=device).manual_seed(seed)
    randn = lambda *shape: torch.randn(shape, generator=gen, device=device)  # noqa: E731
    heads, kv, dim, block, batch = (case[k] for k in ("heads", "kv", "dim", "block", "batch"))
    before, new = lengths(case)
    after = [b + n for b, n in zip(before, new)]
    width = -(-max(after) // block)
    total = batch * width
    tokens = sum(new)
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device=device)  # noqa: E731
    state = {"case": case, "max_q_len": max(new), "block_table": torch.randperm(total, generator=gen, device=device).int().view(batch, width).contiguous(),
             "ctx_after": ints(after), "cu_q": ints([0] + list(torch.tensor(new).cumsum(0).tolist())),
             "positions": torch.cat([torch.arange(b, a, dtype=torch.int32) for b, a in zip(before, after)]).to(device),
             "token_seq": torch.repeat_interleave(torch.arange(batch), torch.tensor(new)).int().to(device)}
    # keys have a few loud channels, as rotated keys do; a block holds keys, then values
    loud = 1.0 + 3.0 * (torch.rand(kv, 1, dim, generator=gen, device=device) < 0.05)
    for name, by in (("k", loud), ("v", torch.ones_like(loud))):
        state[name] = torch.empty(total + 1, kv, block, dim // 2, dtype=torch.uint8, device=device)
        state[name + "_scale"] = torch.empty(total + 1, kv, block, dim // GROUP, dtype=torch.uint8, device=device)
        piece = max(1, (1 << 27) // (kv * block * dim))
        for at in range(0, total + 1, piece):
            count = min(piece, total + 1 - at)
            state[name][at:at + count], state[name + "_scale"][at:at + count] = quantize(randn(count, kv, block, dim) * by)
    if case["op"] == "append":
        inverse = THETA ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64) / dim)
        angle = torch.arange(max(after), dtype=torch.float64)[:, None] * inverse.float().double()[None, :]
        state["cos_sin"] = torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous().to(device)
        state["qkv"] = randn(tokens, (heads + 2 * kv) * dim)
        # the blocks that hold the newest position (a step) or every position (a prompt) are read back
        state["keep"] = 1 if max(new) == 1 else 0
        state["out_width"] = 1 if state["keep"] else width
        state["q_out"] = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=device)
        for name in ("k_out", "v_out"):
            state[name] = torch.empty(batch * state["out_width"], kv, block, dim, dtype=torch.bfloat16, device=device)
        state["out_table"] = torch.empty(batch, width, dtype=torch.int32, device=device)
    else:
        state["q"] = randn(tokens, heads * dim).bfloat16()
        state["out"] = torch.empty(tokens, heads * dim, dtype=torch.bfloat16, device=device)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return (run_append if case["op"] == "append" else run_attend)(state)
    return (plain_append if case["op"] == "append" else plain_attend)(state)


def run_append(s):
    from stratakv_b200 import ops
    c = s["case"]
    k = ops.kernels_for(torch.bfloat16, c["dim"], verbose=False)
    k.append_kv4(s["qkv"], s["cos_sin"], s["positions"], s["token_seq"], s["block_table"], s["q_out"], s["k"], s["v"], s["k_scale"],
                 s["v_scale"], c["heads"], c["kv"], c["dim"], c["block"])
    k.unpack_kv4(s["k"], s["v"], s["k_scale"], s["v_scale"], s["block_table"], s["ctx_after"], s["k_out"], s["v_out"], s["out_table"],
                 c["kv"], c["dim"], c["block"], s["keep"])
    return s["q_out"], s["k_out"], s["v_out"]


def run_attend(s):
    from stratakv_b200 import ops
    c = s["case"]
    k = ops.kernels_for(torch.bfloat16, c["dim"], verbose=False)
    if "scratch" not in s:
        wanted = k.attention_kv4_scratch(c["batch"], s["q"].shape[0], s["max_q_len"], s["block_table"].shape[1], c["heads"], c["kv"],
                                         c["dim"], c["block"], c["window"])
        s["scratch"] = torch.empty(wanted, dtype=torch.uint8, device="cuda")
    k.attention_kv4(s["q"], s["k"], s["v"], s["k_scale"], s["v_scale"], s["block_table"], s["cu_q"], s["ctx_after"], s["out"],
                    s["max_q_len"], c["heads"], c["kv"], c["dim"], c["block"], 1.0 / math.sqrt(c["dim"]), c["window"], s["scratch"])
    return s["out"]


def plain_append(s):
    c = s["case"]
    heads, kv, dim, block = c["heads"], c["kv"], c["dim"], c["block"]
    rows = s["qkv"].unflatten(-1, (-1, dim))
    cos, sin = s["cos_sin"][s["positions"].long()][:, None].unbind(-1)
    low, high = rows[:, :heads + kv].chunk(2, dim=-1)
    rotated = torch.cat([low * cos - high * sin, low * sin + high * cos], dim=-1)
    at = s["positions"].long()
    blocks, offsets = s["block_table"][s["token_seq"].long(), at // block].long(), at % block
    s["k"][blocks, :, offsets], s["k_scale"][blocks, :, offsets] = quantize(rotated[:, heads:])
    s["v"][blocks, :, offsets], s["v_scale"][blocks, :, offsets] = quantize(rows[:, heads + kv:])
    # what the blocks that are read back stand for; rows behind a sequence's end are zero
    after = s["ctx_after"].long()[:, None]
    logical = ((after - 1) // block if s["keep"] else torch.zeros_like(after)) + torch.arange(s["out_width"], device=after.device)
    read = s["block_table"].gather(1, logical.clamp(max=s["block_table"].shape[1] - 1)).long()
    live = (logical[..., None] * block + torch.arange(block, device=after.device) < after[..., None])[:, :, None, :, None]
    k = torch.where(live, dequantize(s["k"][read], s["k_scale"][read]), 0.0).bfloat16().flatten(0, 1)
    v = torch.where(live, dequantize(s["v"][read], s["v_scale"][read]), 0.0).bfloat16().flatten(0, 1)
    return rotated[:, :heads].flatten(1).bfloat16(), k, v


def plain_attend(s):
    c = s["case"]
    heads, kv, dim = c["heads"], c["kv"], c["dim"]
    read = s["block_table"].long()
    # [sequences, key heads, positions, head size]
    keys = dequantize(s["k"][read], s["k_scale"][read]).transpose(1, 2).flatten(2, 3)
    values = dequantize(s["v"][read], s["v_scale"][read]).transpose(1, 2).flatten(2, 3)
    # queries padded to the longest sequence: [sequences, key heads, heads of one x queries, head size]
    cu, after = s["cu_q"].long(), s["ctx_after"].long()
    count = (cu[1:] - cu[:-1])[:, None]
    local = torch.arange(s["max_q_len"], device=cu.device)[None, :]
    rows = (cu[:-1, None] + local).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[rows].unflatten(-1, (kv, heads // kv, dim)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    scores = torch.matmul(q, keys.transpose(-1, -2)) * (1.0 / math.sqrt(dim))
    scores = scores.unflatten(2, (heads // kv, s["max_q_len"]))
    at = (after[:, None] - count + local)[:, :, None]
    key_at = torch.arange(keys.shape[2], device=cu.device)[None, None, :]
    hidden = (key_at > at) | (key_at >= after[:, None, None])
    if c["window"]:
        hidden = hidden | (key_at <= at - c["window"])
    scores.masked_fill_(hidden[:, None, None], -math.inf)
    # (rows that pad a sequence see every key of it; they are left out at the end)
    weights = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    weights = weights.div_(weights.sum(-1, keepdim=True))
    out = torch.matmul(weights.flatten(2, 3), values).unflatten(2, (heads // kv, s["max_q_len"]))
    out = out.permute(0, 3, 1, 2, 4).flatten(2)
    return out[local.expand(count.shape[0], -1) < count].bfloat16()


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------

def exact_scales(device):
    """Scale of each byte that is written (the one for what is not finite stands for NaN)."""
    finite = [((8 + (b & 7)) * 2.0 ** ((b >> 3) - 18) if b >= 8 else b * 2.0 ** -17) / 64.0 for b in range(LARGEST + 1)]
    return torch.tensor(finite + [math.nan] * (255 - LARGEST), dtype=torch.float64, device=device)


def exact_values(codes, scale, dim):
    """``[..., dim]`` float64 numbers that codes ``[..., dim / 2]`` and scales ``[..., dim / 16]`` stand for."""
    out = torch.empty(codes.shape[:-1] + (dim,), dtype=torch.float64, device=codes.device)
    out[..., 0::2] = codes.remainder(16).double() - 8
    out[..., 1::2] = codes.div(16, rounding_mode="floor").double() - 8
    return out * exact_scales(codes.device)[scale.long()].repeat_interleave(16, dim=-1)


def exact_rounded(x):
    """Float64 numbers ``[..., dim]`` brought to the nearest number that the cache holds."""
    scales = exact_scales(x.device)[:LARGEST + 1].contiguous()
    groups = x.reshape(x.shape[:-1] + (-1, 16))
    step = scales[torch.searchsorted(7.0 * scales, groups.abs().amax(-1)).clamp(max=LARGEST)][..., None]
    return (torch.clamp(torch.round(groups / step.clamp(min=1e-30)), -7, 7) * step).reshape(x.shape)


def exact(case, seed):
    s = prepare(case, seed)
    heads, kv, dim, block, batch = (case[k] for k in ("heads", "kv", "dim", "block", "batch"))
    before, new = lengths(case)
    firsts = s["cu_q"].tolist()
    if case["op"] == "append":
        x = s["qkv"].double().reshape(-1, heads + 2 * kv, dim)
        turn = torch.view_as_complex(s["cos_sin"].double())[s["positions"].long()][:, None, :]
        pairs = torch.complex(x[:, :heads + kv, :dim // 2], x[:, :heads + kv, dim // 2:]) * turn
        turned = torch.cat([pairs.real, pairs.imag], dim=-1)
        fresh = {"k": exact_rounded(turned[:, heads:]), "v": exact_rounded(x[:, heads + kv:])}
        found = {}
        for name in ("k", "v"):
            out = torch.zeros(batch, s["out_width"], kv, block, dim, dtype=torch.float64, device="cuda")
            for i in range(batch):
                after = before[i] + new[i]
                first = (after - 1) // block if s["keep"] else 0
                for b in range(first, -(-after // block)):
                    at = int(s["block_table"][i, b])
                    out[i, b - first] = exact_values(s[name][at], s[name + "_scale"][at], dim)
                    out[i, b - first, :, max(0, after - b * block):] = 0.0
                    lo, hi = max(b * block, before[i]), min((b + 1) * block, after)
                    if lo < hi:
                        own_rows = fresh[name][firsts[i] + lo - before[i]:firsts[i] + hi - before[i]]
                        out[i, b - first, :, lo - b * block:hi - b * block] = own_rows.transpose(0, 1)
            found[name] = out.reshape(-1, kv, block, dim)
        return turned[:, :heads].reshape(-1, heads * dim), found["k"], found["v"]
    out = torch.empty(s["q"].shape[0], heads, dim, dtype=torch.float64, device="cuda")
    for i in range(batch):
        after = before[i] + new[i]
        blocks = s["block_table"][i, :-(-after // block)].long()
        k, v = (exact_values(s[name][blocks], s[name + "_scale"][blocks], dim).permute(1, 0, 2, 3).reshape(kv, -1, dim)[:, :after]
                for name in ("k", "v"))
        q = s["q"][firsts[i]:firsts[i + 1]].double().reshape(new[i], kv, heads // kv, dim)
        behind = torch.arange(before[i], after, device="cuda")[:, None] - torch.arange(after, device="cuda")[None, :]
        seen = (behind >= 0) & (behind < (case["window"] or after + 1))
        for h in range(kv):
            score = torch.einsum("qgd,kd->gqk", q[:, h], k[h]) / math.sqrt(dim)
            weight = torch.softmax(score.masked_fill(~seen, -math.inf), dim=-1)
            out[firsts[i]:firsts[i + 1], h * (heads // kv):(h + 1) * (heads // kv)] = torch.einsum("gqk,kd->qgd", weight, v[h])
    return out.reshape(-1, heads * dim)


def work(case):
    heads, kv, dim, block = case["heads"], case["kv"], case["dim"], case["block"]
    before, new = lengths(case)
    tokens, row = sum(new), kv * (dim + dim // 8)                 # bytes of a position: codes and scales, keys and values
    if case["op"] == "append":
        # read: the rows and the angles; written: queries and codes; then what is read back
        keep = max(new) == 1
        back = sum(((a - 1) % block + 1) if keep else a for a in (b + n for b, n in zip(before, new)))
        zeros = len(new) * (block if keep else -(-max(b + n for b, n in zip(before, new)) // block) * block)
        return {"bytes": tokens * ((heads + 2 * kv) * dim * 4 + dim * 4 + heads * dim * 2 + row) + back * row + zeros * kv * dim * 4,
                "flops": tokens * (heads + kv) * dim * 3}
    keys = pairs = 0
    for b, n in zip(before, new):
        reach = case["window"] or b + n
        keys += min(b + n, reach + n - 1)
        if b + 1 >= reach:
            pairs += n * reach
        else:
            short = min(n, reach - b)                              # queries that see every position before them
            pairs += short * b + short * (short + 1) // 2 + (n - short) * reach
    return {"bytes": keys * row + 2 * tokens * heads * dim * 2, "flops": 4 * pairs * heads * dim}

"""The operators of serving with drafted tokens over a paged cache of 4-bit numbers (xalm_b200/paged.py), as a serving loop calls them, from the smallest call to the largest.

  append4     keys and values of a ragged batch of new tokens, keys turned by their positions, into pages of 4-bit blocks, queries turned beside them; and the stored rows
              read back as the numbers they stand for.
  attend4     causal attention of the new tokens over their sequences' 4-bit pages; groups of sequences share their first pages.
  verify      drafted tokens against the target's probabilities, from given random numbers: how many are taken, and the token drawn behind them.

`own` is false: plain torch operations.  `exact` restates the operators in float64.

A block is 32 neighbouring entries of a head (behind the last entry, zeros).  With M its entry of the largest magnitude, the positive one of two: scale = fp16(-M / 8), code =
clamp(rint(x / scale) + 8, 0, 15), and the block stands for scale (code - 8).  A page has a run of bytes for each kv head: the slots' key codes, their scales, value codes, scales.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1000000.0


# ---- the cases ---------------------------------------------------------------------------------------------------------------------------
def cached(name, op, type, heads, kv_heads, dim, seqs, new, past, page=64, vdim=None, groups=0, shared=(0, 0), rot=None, neighbours=False):
    """`new`, `past`: (least, most) tokens per sequence of this call and before it, shared ones not counted; `shared`: tokens each group has in common."""
    c = {"op": op, "type": type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim or dim, "page": page, "seqs": seqs, "new_lo": new[0], "new_hi": new[1],
         "past_lo": past[0], "past_hi": past[1], "groups": groups, "shared_lo": shared[0], "shared_hi": shared[1], "rot": dim // 2 if rot is None else rot, "neighbours": neighbours}
    return c if name is None else dict(c, name=name)


def drafted(name, type, seqs, drafts, vocab, known=True):
    """`drafts`: (least, most) drafted tokens per sequence; `known`: the drafts' probabilities are given, else each draft is certain."""
    c = {"op": "verify", "type": type, "seqs": seqs, "drafts_lo": drafts[0], "drafts_hi": drafts[1], "vocab": vocab, "known": known}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        cached("append4_16", "append4", "bf16", 32, 8, 128, 16, (1, 1), (200, 3000)),                                # a step of sixteen chats: latency
        cached("append4_prompts", "append4", "f16", 32, 8, 128, 9, (300, 1500), (0, 700)),                           # prompts of several users in one pass
        cached("attend4_4", "attend4", "f16", 8, 2, 128, 4, (1, 1), (100, 400), page=16),                            # four short chats: latency
        cached("attend4_64", "attend4", "bf16", 32, 8, 128, 64, (1, 1), (1000, 8000)),                               # an ordinary batch of long chats
        cached("attend4_128", "attend4", "bf16", 32, 8, 128, 128, (1, 1), (8000, 32000)),                            # the largest: long documents, a question each
        cached("attend4_drafts", "attend4", "f16", 32, 8, 128, 32, (3, 6), (1000, 6000)),                            # a step that verifies drafts
        cached("attend4_shared", "attend4", "bf16", 32, 8, 128, 64, (1, 1), (1, 1500), groups=1, shared=(8192, 8192)),  # chats under one long system prompt
        cached("attend4_prompts", "attend4", "bf16", 32, 8, 128, 5, (150, 700), (1000, 3000)),                       # prompts that continue long texts
        cached("attend4_8_f32", "attend4", "f32", 8, 2, 64, 8, (1, 1), (100, 2500), page=16),                        # fp32 queries, small heads and pages
        drafted("verify_8", "f32", 8, (1, 4), 32000),                                                               # eight chats: latency
        drafted("verify_64", "f32", 64, (0, 8), 131072),                                                            # a full batch over a large vocabulary
        drafted("verify_33_sure", "f32", 33, (2, 5), 50021, known=False),                                           # drafts looked up in the text itself, odd vocabulary
    ]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append4", "attend4", "attend4", "attend4", "verify"])
    if op == "verify":
        most = rng.choice([1, 4, 8])
        return drafted(None, rng.choice(["f32", "f32", "f16", "bf16"]), log_uniform(rng, 1, 64), (rng.randint(0, most), most), log_uniform(rng, 1000, 131072), known=rng.random() < 0.75)
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 4, 4, 5, 8])
    dim = rng.choice([64, 96, 128, 128, 256])
    kw = dict(page=rng.choice([16, 32, 64, 64, 128]), vdim=rng.choice([dim, dim, 64]))
    type = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    if op == "append4":
        kw.update(neighbours=rng.random() < 0.5, rot=rng.choice([dim // 2, dim // 4]))
        if rng.random() < 0.5:
            return cached(None, op, type, heads, kv_heads, dim, log_uniform(rng, 1, 256), (1, 1), (0, log_uniform(rng, 16, 8000)), **kw)
        return cached(None, op, type, heads, kv_heads, dim, rng.randint(1, 6), (1, log_uniform(rng, 16, 1500)), (0, log_uniform(rng, 1, 2000)), **kw)
    if rng.random() < 0.7:
        most = rng.choice([1, 1, 5])
        if rng.random() < 0.4:
            shared = log_uniform(rng, 100, 16000)
            kw.update(groups=rng.randint(1, 3), shared=(shared // 2, shared))
        return cached(None, op, type, heads, kv_heads, dim, log_uniform(rng, 4, 128), (1, most), (0, log_uniform(rng, 16, 12000)), **kw)
    kw.update(groups=rng.randint(0, 1), shared=(500, 1000))
    return cached(None, op, type, heads, kv_heads, dim, rng.randint(2, 6), (1, log_uniform(rng, 2, 600)), (0, log_uniform(rng, 16, 3000)), **kw)


# ---- sizes of a case, by its values alone ---------------------------------------------------------------------------------------------------
def spread(i, lo, hi):
    return lo + int((hi - lo + 1) * (((i + 1) * 0.6180339887498949) % 1.0))


def sizes(c):
    """(new tokens, tokens before them and outside the shared part, tokens shared) per sequence, and the groups' bounds."""
    B, n = c["seqs"], c["groups"]
    new = [spread(i, c["new_lo"], c["new_hi"]) for i in range(B)]
    past = [spread(3 * i + 1, c["past_lo"], c["past_hi"]) for i in range(B)]
    bounds = [i * B // n for i in range(n + 1)] if n else [0]
    common = [spread(2 * i, c["shared_lo"], c["shared_hi"]) // c["page"] * c["page"] for i in range(n)]
    shared = [0] * B
    for i in range(n):
        for s in range(bounds[i], bounds[i + 1]):
            shared[s] = common[i]
    return new, past, shared, bounds, common


def work(c):
    if c["op"] == "verify":
        return {"bytes": c["seqs"] * c["vocab"] * BYTES[c["type"]] * (2 if c["known"] else 1), "flops": c["seqs"] * c["vocab"] * 3}
    new, past, shared, bounds, common = sizes(c)
    H, G, d, dv = c["heads"], c["kv_heads"], c["dim"], c["vdim"]
    e, N = BYTES[c["type"]], sum(new)
    blocks = lambda n: (d + dv) * n * G * 9 // 16  # 4 bits an entry, 16 a block
    if c["op"] == "append4":
        return {"bytes": N * (2 * H * d + G * (d + dv)) * e + 2 * blocks(N) + N * G * (d + dv) * 4, "flops": N * ((H + G) * c["rot"] * 6 + G * (d + dv) * 4)}
    last = [a + b + s for a, b, s in zip(new, past, shared)]
    keys = sum(common) + sum(t - s for t, s in zip(last, shared))
    seen = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, last))
    return {"bytes": N * H * (d + dv) * e + blocks(keys), "flops": 2 * seen * H * (d + dv)}


# ---- the 4-bit format ----------------------------------------------------------------------------------------------------------------------
def width(n):
    """Codes to a slot and head: heads of other sizes lie in rows of 64, 128 or 256."""
    return 64 if n <= 64 else 128 if n <= 128 else 256


def scales_of(blocks):
    """fp16 scales of (.., 32) blocks of fp32 numbers."""
    hi, lo = blocks.amax(dim=-1), blocks.amin(dim=-1)
    return (torch.where(hi >= -lo, hi, lo) * -0.125).clamp(-65504.0, 65504.0).half()


def codes_of(blocks, scales):
    d = scales.double()[..., None]
    return torch.where(d == 0, 8.0, (blocks.double() / d).round() + 8).clamp(0, 15)


def rounded(x):
    """The fp32 numbers (.., n) that x's 4-bit blocks stand for."""
    n = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, -n % 32)).unflatten(-1, (-1, 32))
    scales = scales_of(blocks)
    return ((codes_of(blocks, scales) - 8).float() * scales.float()[..., None]).flatten(-2)[..., :n]


def packed(x, lanes):
    """(.., n) numbers as bytes: codes (.., width / 2) and scales (.., width / 16).  A block's bytes go to `lanes` lanes in turn, and each lane's bytes of all blocks lie together."""
    n = x.shape[-1]
    blocks = torch.nn.functional.pad(x.float(), (0, width(n) - n)).unflatten(-1, (-1, 32))
    scales = scales_of(blocks)
    code = codes_of(blocks, scales).to(torch.uint8)
    both = code[..., 0::2] | code[..., 1::2] << 4
    return both.unflatten(-1, (lanes, -1)).transpose(-3, -2).flatten(-3), scales.contiguous().view(torch.uint8)


def unpacked(codes, scales, lanes, n):
    """The numbers (.., n) in fp32."""
    both = codes.unflatten(-1, (lanes, scales.shape[-1] // 2, -1)).transpose(-3, -2).flatten(-2)
    code = torch.stack((both & 15, both >> 4), dim=-1).flatten(-2)
    return ((code.float() - 8) * scales.contiguous().view(torch.float16).float()[..., None]).flatten(-2)[..., :n]


KEY_LANES, VALUE_LANES = 4, 8


def sections(c):
    P, k, v = c["page"], width(c["dim"]), width(c["vdim"])
    return [P * k // 2, P * k // 16, P * v // 2, P * v // 16]


def page_bytes(c, k, v):
    """Keys and values (n, heads, slots, entries) as pages' bytes (n, heads, bytes)."""
    kc, ks = packed(k, KEY_LANES)
    vc, vs = packed(v, VALUE_LANES)
    return torch.cat([t.flatten(2) for t in (kc, ks, vc, vs)], dim=2)


def page_numbers(c, block):
    """The reverse: (n, heads, slots, entries) in fp32."""
    kc, ks, vc, vs = (t.unflatten(2, (c["page"], -1)) for t in block.split(sections(c), dim=2))
    return unpacked(kc, ks, KEY_LANES, c["dim"]), unpacked(vc, vs, VALUE_LANES, c["vdim"])


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------
def inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return verify_inputs(c, g) if c["op"] == "verify" else cache_inputs(c, g)


def verify_inputs(c, g):
    """The target's and the drafts' distributions, peaked and alike; drafts drawn from theirs, or the likeliest tokens where drafts are certain."""
    B, V = c["seqs"], c["vocab"]
    starts = [0]
    for i in range(B):
        starts.append(starts[-1] + 1 + spread(i, c["drafts_lo"], c["drafts_hi"]))
    N = starts[-1]
    logits = torch.randn(N, V, generator=g, device="cuda").mul_(3.0)
    target = logits.softmax(dim=1)
    draft = logits.add_(torch.randn(N, V, generator=g, device="cuda")).softmax(dim=1)
    del logits
    drawn = torch.multinomial(draft, 1, generator=g).squeeze(1) if c["known"] else draft.argmax(dim=1)
    t = TYPES[c["type"]]
    return {"case": c, "starts": torch.tensor(starts, device="cuda", dtype=torch.int32), "host_starts": starts, "target": target.to(t), "draft": draft.to(t) if c["known"] else None,
            "tokens": torch.cat((drawn[:1], drawn[:-1])).to(torch.int32), "accept": torch.rand(N, generator=g, device="cuda"), "pick": torch.rand(B, generator=g, device="cuda")}


def cache_inputs(c, g):
    """A pool of pages that hold keys and values in every slot, as sequences before these left it."""
    new, past, shared, bounds, common = sizes(c)
    B, H, G, d, dv, P = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    t = TYPES[c["type"]]
    lens = [a + b + s for a, b, s in zip(new, past, shared)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    N = starts[-1]

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    need = sum(x // P for x in common) + sum((x - s + P - 1) // P for x, s in zip(lens, shared))
    pages = need + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, max((x + P - 1) // P for x in lens)), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i in range(len(common)):
        k = common[i] // P
        table[bounds[i]:bounds[i + 1], :k] = order[at:at + k]
        at += k
    for s in range(B):
        a, b = shared[s] // P, (lens[s] + P - 1) // P
        table[s, a:b] = order[at:at + b - a]
        at += b - a
    # different pages up to 16384 slots, which large pools repeat in any order
    kinds = min(pages, max(1, 16384 // P))
    bank = page_bytes(c, normal(kinds, G, P, d), normal(kinds, G, P, dv))
    pool = bank if kinds == pages else bank[torch.randint(kinds, (pages,), generator=g, device="cuda")]
    st = {"case": c, "starts": torch.tensor(starts, device="cuda", dtype=torch.int32), "lens": torch.tensor(lens, device="cuda", dtype=torch.int32), "table": table,
          "host_starts": starts, "host_lens": lens, "pool": pool, "scale": d ** -0.5, "groups": None, "shared": None}
    if c["groups"]:
        st["groups"] = torch.tensor(bounds, device="cuda", dtype=torch.int32)
        st["shared"] = torch.tensor(common, device="cuda", dtype=torch.int32)
    if c["op"] == "append4":
        st["new_q"], st["new_k"], st["new_v"] = normal(N, H, d, dtype=t), normal(N, G, d, dtype=t), normal(N, G, dv, dtype=t)
        st["freq"] = (THETA ** (-torch.arange(c["rot"], device="cuda", dtype=torch.float64) / c["rot"])).float()
    else:
        st["q"] = normal(N, H, d, dtype=t).mul_(1.5)  # some keys stand out
    return st


def where(st):
    """Sequence and position of every row."""
    starts, lens = st["starts"].long(), st["lens"].long()
    row = torch.arange(st["host_starts"][-1], device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    return seq, lens[seq] - starts[seq + 1] + row


def prepare(c, seed):
    st = inputs(c, seed)
    if own:
        from xalm_b200 import paged
        if c["op"] != "verify":
            st["cache"] = paged.PagedCache4(st["pool"], c["page"], c["dim"], c["vdim"])
            st["batch"] = paged.Batch(st["starts"], st["lens"], st["table"], groups=st["groups"], shared=st["shared"])
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        return {"append4": plain_append, "attend4": plain_attend, "verify": plain_verify}[c["op"]](st)
    from xalm_b200 import paged
    if c["op"] == "verify":
        out, taken = paged.verify(st["starts"], st["tokens"], st["target"], st["accept"], st["pick"], draft=st["draft"])
        return {"out": out, "taken": taken}
    cache, batch = st["cache"], st["batch"]
    if c["op"] == "append4":
        q = paged.append4(cache, batch, st["new_k"], st["new_v"], q=st["new_q"], freq=st["freq"], neighbours=c["neighbours"])
        k, v = paged.read4(cache, batch, st["host_starts"][-1])
        return {"q": q, "k": k, "v": v}
    out, lse = paged.attend4(cache, batch, st["q"], st["scale"], want_lse=True)
    return {"out": out, "lse": lse}


def turned(x, pos, freq, neighbours):
    """The first 2 len(freq) entries of every head of x (N, heads, d) in 64 bits, turned by pos * freq."""
    angle = pos.double()[:, None] * freq.double()
    cs, sn = angle.cos()[:, None], angle.sin()[:, None]
    n = freq.numel()
    x = x.double()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if neighbours else (x[..., :n], x[..., n:2 * n])
    u, w = a * cs - b * sn, b * cs + a * sn
    head = torch.stack((u, w), dim=-1).flatten(-2) if neighbours else torch.cat((u, w), dim=-1)
    return torch.cat((head, x[..., 2 * n:]), dim=-1).float()


def plain_append(st):
    """Keys and values as their blocks stand for them."""
    c, pos = st["case"], where(st)[1]
    q = turned(st["new_q"], pos, st["freq"], c["neighbours"]).to(st["new_q"].dtype)
    return {"q": q, "k": rounded(turned(st["new_k"], pos, st["freq"], c["neighbours"])), "v": rounded(st["new_v"])}


def plain_attend(st):
    c, P, G = st["case"], st["case"]["page"], st["case"]["kv_heads"]
    outs, lses = [], []
    for s, t in enumerate(st["host_lens"]):
        a, b = st["host_starts"][s], st["host_starts"][s + 1]
        keys, values = (x.transpose(1, 2).flatten(0, 1)[:t] for x in page_numbers(c, st["pool"][st["table"][s, :(t + P - 1) // P].long()]))
        q = st["q"][a:b].float().unflatten(1, (G, -1))
        score = torch.einsum("ngrd,jgd->ngrj", q, keys) * st["scale"]
        if b - a > 1:
            later = torch.arange(t, device="cuda") > torch.arange(t - (b - a), t, device="cuda")[:, None]
            score.masked_fill_(later[:, None, None], -math.inf)
        top = score.amax(dim=-1, keepdim=True)
        p = (score - top).exp()
        total = p.sum(dim=-1, keepdim=True)
        outs.append((torch.einsum("ngrj,jgd->ngrd", p, values) / total).flatten(1, 2))
        lses.append((top + total.log()).squeeze(-1).flatten(1))
    return {"out": torch.cat(outs).to(st["q"].dtype), "lse": torch.cat(lses)}


def plain_verify(st):
    starts, target, draft, tokens = st["starts"].long(), st["target"], st["draft"], st["tokens"].long()
    first, n = starts[:-1], starts[1:] - starts[:-1]
    N, V = target.shape
    row = torch.arange(N, device="cuda")
    seq = torch.searchsorted(starts[1:], row, right=True)
    following = tokens[(row + 1).clamp_max(N - 1)]
    p = target[row, following].double()
    q = torch.ones_like(p) if draft is None else draft[row, following].double()
    refused = (st["accept"].double() * q >= p) | (row + 1 == starts[seq + 1])  # the last row has no draft behind it
    taken = torch.where(refused, row - first[seq], N).new_full((len(n),), N).scatter_reduce(0, seq, torch.where(refused, row - first[seq], N), "amin")
    at = first + taken
    left = target[at].double()
    some = taken < n - 1  # a draft was refused: what the draft's distribution has too much of is left out
    if draft is None:
        left[some, following[at][some]] = 0
    else:
        left = torch.where(some[:, None], (left - draft[at].double()).clamp_min(0), left)
    total = left.cumsum(dim=1)
    drawn = torch.searchsorted(total, st["pick"].double()[:, None] * total[:, -1:], right=True).squeeze(1).clamp_max(V - 1)
    i = row - first[seq]
    out = torch.where(i < taken[seq], following, torch.where(i == taken[seq], drawn[seq], -1))
    return {"out": out.to(torch.int32), "taken": taken.to(torch.int32)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------
def exact_pages(c, block):
    """Keys and values (n, heads, slots, entries) in 64 bits, entry by entry from where it lies."""
    P, at, out = c["page"], 0, []
    for dim, lanes in ((c["dim"], 4), (c["vdim"], 8)):
        W = 64 if dim <= 64 else 128 if dim <= 128 else 256
        e = torch.arange(dim, device="cuda")
        per, part = 32 // lanes, W // 2 // lanes  # a lane's entries of a block, its bytes
        byte = e % 32 // per * part + e // 32 * (per // 2) + e % per // 2
        code = block[:, :, at:at + P * W // 2].reshape(*block.shape[:2], P, W // 2)[..., byte].to(torch.int32)
        code = torch.where(e % 2 == 1, torch.div(code, 16, rounding_mode="floor"), code % 16)
        at += P * W // 2
        scale = block[:, :, at:at + P * W // 16].contiguous().view(torch.float16).reshape(*block.shape[:2], P, W // 32)[..., e // 32]
        at += P * W // 16
        out.append((code - 8).double() * scale.double())
    return out


def exact_rows(x):
    """Rows (N, heads, n) of fp32 numbers as their blocks stand for them, by the distance to the codes."""
    out = torch.zeros_like(x, dtype=torch.float64)
    codes = torch.arange(-8, 8, device="cuda", dtype=torch.float64)
    for a in range(0, x.shape[-1], 32):
        part = x[..., a:a + 32].double()
        top, at = part.abs().max(dim=-1, keepdim=True)
        largest = torch.where((part == top).any(dim=-1, keepdim=True), top, -top)
        scale = (largest / -8).clamp(-65504, 65504).float().half().double()
        ratio = part / torch.where(scale == 0, 1.0, scale)
        near = (ratio[..., None] - codes).abs()
        pick = near.argmin(dim=-1)
        even = (near == near.amin(dim=-1, keepdim=True)) & (codes % 2 == 0)  # half way between two, the even one
        pick = torch.where((near == near.amin(dim=-1, keepdim=True)).sum(dim=-1) > 1, even.to(torch.int32).argmax(dim=-1), pick)
        out[..., a:a + 32] = codes[pick] * scale
    return out


def exact(c, seed):
    st = inputs(c, seed)
    starts = st["host_starts"]
    if c["op"] == "verify":
        out, taken = torch.full((starts[-1],), -1, dtype=torch.int32), []
        tokens, u = st["tokens"].tolist(), st["accept"].double().tolist()
        for s in range(c["seqs"]):
            i = starts[s]
            while i + 1 < starts[s + 1]:
                x = tokens[i + 1]
                if not u[i] * (1.0 if st["draft"] is None else float(st["draft"][i, x])) < float(st["target"][i, x]):
                    break
                out[i] = x
                i += 1
            taken.append(i - starts[s])
            rest = st["target"][i].double()
            if i + 1 < starts[s + 1]:
                if st["draft"] is None:
                    rest[tokens[i + 1]] = 0
                else:
                    rest = torch.relu(rest - st["draft"][i].double())
            upto = rest.cpu().cumsum(0)
            out[i] = int((upto <= float(st["pick"][s].double()) * float(upto[-1])).sum())
        return {"out": out.cuda(), "taken": torch.tensor(taken, dtype=torch.int32, device="cuda")}
    H, G, P, lens = c["heads"], c["kv_heads"], c["page"], st["host_lens"]
    if c["op"] == "append4":
        pos = torch.cat([torch.arange(t - b + a, t, device="cuda") for a, b, t in zip(starts, starts[1:], lens)])
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * st["freq"].double())[:, None]
        n = c["rot"]

        def rotate(x):
            x = x.double().clone()
            a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["neighbours"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
            x[..., a], x[..., b] = z.real, z.imag
            return x

        return {"q": rotate(st["new_q"]), "k": exact_rows(rotate(st["new_k"]).float()), "v": exact_rows(st["new_v"].float())}
    rep = H // G
    out = torch.zeros(starts[-1], H, c["vdim"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(starts[-1], H, dtype=torch.float64, device="cuda")
    for s, t in enumerate(lens):
        at = torch.arange(t, device="cuda")
        k, v = exact_pages(c, st["pool"][st["table"][s, :(t + P - 1) // P].long()])
        for a in range(starts[s], starts[s + 1], 256):
            b = min(a + 256, starts[s + 1])
            seen = at <= t - starts[s + 1] + torch.arange(a, b, device="cuda")[:, None]
            for g in range(G):
                s64 = st["q"][a:b, g * rep:(g + 1) * rep].double() @ k[:, g].flatten(0, 1)[:t].T * st["scale"]
                s64 = s64.masked_fill(~seen[:, None], -math.inf)
                lse[a:b, g * rep:(g + 1) * rep] = s64.logsumexp(dim=-1)
                out[a:b, g * rep:(g + 1) * rep] = s64.softmax(dim=-1) @ v[:, g].flatten(0, 1)[:t]
    return {"out": out, "lse": lse}

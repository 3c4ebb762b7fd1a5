"""The operators of batched serving over a paged cache (xalm_b200/paged.py), as a serving loop calls them, from the smallest call to the largest.

  append      keys and values of a ragged batch of new tokens into the pages of their sequences, the position rotation applied on the way, queries turned
              beside them, and the mean key of every page that fills up.
  attend      causal attention of the new tokens over their sequences' pages; groups of sequences share their first pages, which are read once for all.
  select      the pages each new token reads, by the product of its queries with the pages' mean keys.
  selected    attention of each new token over the pages of its own list.

`own` is false: plain torch operations.  `exact` restates the operators in float64.
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}
THETA = 1000000.0


# ---- the cases ---------------------------------------------------------------------------------------------------------------------------
def case(name, op, type, heads, kv_heads, dim, seqs, new, past, page=64, vdim=None, layout="position", groups=0, shared=(0, 0), in_type=None, rot=None,
         neighbours=False, means=False, top=0, first=1, recent=1):
    """`new`, `past`: (least, most) tokens per sequence of this call and before it, shared ones not counted; `shared`: tokens each group has in common."""
    c = {"op": op, "type": type, "in_type": in_type or type, "heads": heads, "kv_heads": kv_heads, "dim": dim, "vdim": vdim or dim, "page": page, "layout": layout,
         "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "past_lo": past[0], "past_hi": past[1], "groups": groups, "shared_lo": shared[0], "shared_hi": shared[1],
         "rot": dim // 2 if rot is None else rot, "neighbours": neighbours, "means": means, "top": top, "first": first, "recent": recent}
    return c if name is None else dict(c, name=name)


def listed():
    return [
        case("append_16", "append", "bf16", 32, 8, 128, 16, (1, 1), (200, 3000)),                           # a step of sixteen chats: latency
        case("append_250_f16", "append", "f16", 16, 4, 64, 250, (1, 1), (1, 9000), page=32, in_type="f32", neighbours=True, means=True, layout="head"),  # a full batch of a small model, fp32 projections
        case("append_prompts", "append", "bf16", 32, 8, 128, 9, (300, 1500), (0, 700), means=True),         # prompts of several users in one pass
        case("attend_4", "attend", "f16", 8, 2, 128, 4, (1, 1), (10, 100), groups=1, shared=(256, 256)),    # four short chats under one system prompt: latency
        case("attend_64", "attend", "bf16", 32, 8, 128, 64, (1, 1), (1, 1500), groups=1, shared=(8192, 8192)),  # an ordinary batch of one application
        case("attend_128", "attend", "bf16", 32, 8, 128, 128, (1, 1), (50, 2500), groups=2, shared=(16384, 32768)),  # the largest: two long documents, many questions each
        case("attend_chunks", "attend", "bf16", 32, 8, 128, 5, (150, 700), (0, 900), groups=1, shared=(2048, 2048), layout="head"),  # prompts that continue a shared text
        case("attend_8_f32", "attend", "f32", 8, 2, 64, 8, (1, 1), (100, 2500), page=16),                   # fp32 cache, nothing shared, small pages
        case("select_8", "select", "bf16", 32, 8, 128, 8, (1, 1), (8000, 32000), top=32),                   # long chats, one token each
        case("select_prompt", "select", "f16", 32, 8, 128, 2, (500, 900), (7000, 15000), top=16),           # prompts behind long texts
        case("selected_16", "selected", "bf16", 32, 8, 128, 16, (1, 1), (4000, 32000), top=32),             # a step of long chats
        case("selected_prompt", "selected", "f16", 32, 8, 128, 2, (500, 900), (3000, 8000), top=16),        # prompts behind long texts
    ]


def log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "select", "selected"])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 4, 4, 5, 8])
    dim = rng.choice([64, 80, 128, 128])
    kw = dict(page=rng.choice([16, 32, 64, 64, 128]), layout=rng.choice(["position", "position", "head"]))
    type = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    if op == "append":
        kw.update(in_type=rng.choice([type, "f32"]), neighbours=rng.random() < 0.5, means=rng.random() < 0.5, rot=rng.choice([dim // 2, dim // 4]))
        if rng.random() < 0.5:
            return case(None, op, type, heads, kv_heads, dim, log_uniform(rng, 1, 256), (1, 1), (0, log_uniform(rng, 16, 8000)), **kw)
        return case(None, op, type, heads, kv_heads, dim, rng.randint(1, 6), (1, log_uniform(rng, 16, 1500)), (0, log_uniform(rng, 1, 2000)), **kw)
    if op == "attend":
        kw.update(vdim=rng.choice([dim, dim, 64]))
        if rng.random() < 0.6:
            seqs, past = log_uniform(rng, 1, 128 if type != "f32" else 32), log_uniform(rng, 16, 4000)
            if rng.random() < 0.6:
                shared = log_uniform(rng, 100, 16000 if type != "f32" else 2000)
                kw.update(groups=rng.randint(1, min(seqs, 3)), shared=(shared // 2, shared))
            return case(None, op, type, heads, kv_heads, dim, seqs, (1, 1), (0, past), **kw)
        new = log_uniform(rng, 2, 800 if type != "f32" else 200)
        kw.update(groups=rng.randint(0, 1), shared=(500, 1000))
        return case(None, op, type, heads, kv_heads, dim, rng.randint(2, 6), (1, new), (0, log_uniform(rng, 16, 2000)), **kw)
    top = rng.choice([8, 16, 32])
    kw.update(top=top, first=rng.randint(0, 2), recent=rng.randint(0, 3))
    if rng.random() < 0.6:
        return case(None, op, type, heads, kv_heads, dim, log_uniform(rng, 1, 32), (1, 1), (100, log_uniform(rng, 500, 24000)), **kw)
    return case(None, op, type, heads, kv_heads, dim, rng.randint(1, 3), (1, log_uniform(rng, 16, 600 if type != "f32" else 100)), (0, log_uniform(rng, 500, 8000)), **kw)


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
    new, past, shared, bounds, common = sizes(c)
    H, G, d, dv, P = c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    e, ei, N = BYTES[c["type"]], BYTES[c["in_type"]], sum(new)
    last = [a + b + s for a, b, s in zip(new, past, shared)]
    if c["op"] == "append":
        filled = sum(t // P - (t - n) // P for t, n in zip(last, new)) if c["means"] else 0
        return {"bytes": N * (H * d + G * (d + dv)) * (ei + e) + filled * G * d * e, "flops": N * (H + G) * c["rot"] * 6}
    if c["op"] == "select":
        pages = [t // P for t in last]
        return {"bytes": sum(pages) * G * d * e + N * H * d * e + N * G * c["top"] * 4, "flops": 2 * sum(n * p for n, p in zip(new, pages)) * G * d}
    if c["op"] == "attend":
        keys = sum(common) + sum(t - s for t, s in zip(last, shared))
        seen = sum(n * (t - n) + n * (n + 1) // 2 for n, t in zip(new, last))
    else:
        keys = sum(min(t, n * c["top"] * P) for n, t in zip(new, last))
        seen = sum(min(t - n + i + 1, c["top"] * P) for n, t in zip(new, last) for i in range(n))
    return {"bytes": (N * H + keys * G) * (d + dv) * e, "flops": 2 * seen * H * (d + dv)}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------------
def inputs(c, seed):
    """Tensors of a case: a pool of pages that hold random keys and values in every slot, as sequences before these left it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, past, shared, bounds, common = sizes(c)
    B, H, G, d, dv, P = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["vdim"], c["page"]
    t, ti = TYPES[c["type"]], TYPES[c["in_type"]]
    lens = [a + b + s for a, b, s in zip(new, past, shared)]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    N = starts[-1]

    def normal(*shape, dtype=t, scale=1.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=dtype)
        return x if scale == 1.0 else x.mul_(scale)

    width = max((x + P - 1) // P for x in lens)
    need = sum(x // P for x in common) + sum((x - s + P - 1) // P for x, s in zip(lens, shared))
    pages = need + 5
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((B, width), -1, device="cuda", dtype=torch.int32)
    at = 0
    for i in range(len(common)):
        k = common[i] // P
        table[bounds[i]:bounds[i + 1], :k] = order[at:at + k]
        at += k
    for s in range(B):
        a, b = shared[s] // P, (lens[s] + P - 1) // P
        table[s, a:b] = order[at:at + b - a]
        at += b - a

    def pool(n):
        return normal(pages, G, P, n).transpose(1, 2) if c["layout"] == "head" else normal(pages, P, G, n)

    st = {"case": c, "starts": torch.tensor(starts, device="cuda", dtype=torch.int32), "lens": torch.tensor(lens, device="cuda", dtype=torch.int32), "table": table,
          "host_starts": starts, "host_lens": lens, "k": pool(d), "v": pool(dv), "scale": d ** -0.5, "means": None, "groups": None, "shared": None}
    if c["groups"]:
        st["groups"] = torch.tensor(bounds, device="cuda", dtype=torch.int32)
        st["shared"] = torch.tensor(common, device="cuda", dtype=torch.int32)
    if c["op"] == "append":
        st["new_q"], st["new_k"], st["new_v"] = normal(N, H, d, dtype=ti), normal(N, G, d, dtype=ti), normal(N, G, dv, dtype=ti)
        st["freq"] = (THETA ** (-torch.arange(c["rot"], device="cuda", dtype=torch.float64) / c["rot"])).float()
    else:
        st["q"] = normal(N, H, d, scale=1.5)  # some pages and keys stand out
    if c["means"] or c["op"] == "select":
        st["means"] = normal(pages, G, d, scale=P ** -0.5)
    if c["op"] == "selected":
        last = where(st)[1] // P  # the page of the token itself, and others at random
        j = torch.arange(width, device="cuda")
        rank = torch.rand(N, G, width, generator=g, device="cuda")
        rank = torch.where(j == last[:, None, None], 2.0, torch.where(j > last[:, None, None], -1.0, rank))
        best, at = rank.topk(min(c["top"], width), dim=2)
        lists = torch.where(best >= 0, at, width).sort(dim=2).values
        lists = torch.where(lists < width, lists, -1)
        st["lists"] = torch.nn.functional.pad(lists, (0, c["top"] - lists.shape[2]), value=-1).to(torch.int32).contiguous()
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
        st["cache"] = paged.PagedCache(st["k"], st["v"], st["means"])
        st["batch"] = paged.Batch(st["starts"], st["lens"], st["table"], groups=st["groups"], shared=st["shared"])
    return st


# ---- one pass ----------------------------------------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        return {"append": plain_append, "attend": plain_attend, "select": plain_select, "selected": plain_selected}[c["op"]](st)
    from xalm_b200 import paged
    cache, batch = st["cache"], st["batch"]
    if c["op"] == "append":
        q = paged.append(cache, batch, st["new_k"], st["new_v"], q=st["new_q"], freq=st["freq"], neighbours=c["neighbours"])
        return {"q": q, "k": st["k"], "v": st["v"], **({"means": st["means"]} if c["means"] else {})}
    if c["op"] == "select":
        return paged.select(cache, batch, st["q"], c["top"], first=c["first"], recent=c["recent"])
    if c["op"] == "attend":
        out, lse = paged.attend(cache, batch, st["q"], st["scale"], want_lse=True)
    else:
        out, lse = paged.attend_selected(cache, batch, st["q"], st["lists"], st["scale"], want_lse=True)
    return {"out": out, "lse": lse}


def turned(x, pos, freq, neighbours):
    """The first 2 len(freq) entries of every head of x (N, heads, d), turned by pos * freq."""
    angle = pos.double()[:, None] * freq.double()
    cs, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    n = freq.numel()
    x = x.float()
    a, b = (x[..., 0:2 * n:2], x[..., 1:2 * n:2]) if neighbours else (x[..., :n], x[..., n:2 * n])
    u, w = a * cs - b * sn, b * cs + a * sn
    head = torch.stack((u, w), dim=-1).flatten(-2) if neighbours else torch.cat((u, w), dim=-1)
    return torch.cat((head, x[..., 2 * n:]), dim=-1)


def plain_append(st):
    c, k, v, P = st["case"], st["k"], st["v"], st["case"]["page"]
    seq, pos = where(st)
    page, slot = st["table"][seq, pos // P].long(), pos % P
    k[page, slot] = turned(st["new_k"], pos, st["freq"], c["neighbours"]).to(k.dtype)
    v[page, slot] = st["new_v"].to(v.dtype)
    out = {"q": turned(st["new_q"], pos, st["freq"], c["neighbours"]).to(k.dtype), "k": k, "v": v}
    if c["means"]:
        full = page[slot == P - 1]
        st["means"][full] = k[full].float().mean(dim=1).to(k.dtype)
        out["means"] = st["means"]
    return out


def plain_attend(st):
    c, P, G = st["case"], st["case"]["page"], st["case"]["kv_heads"]
    outs, lses = [], []
    for s, t in enumerate(st["host_lens"]):
        a, b = st["host_starts"][s], st["host_starts"][s + 1]
        pages = st["table"][s, :(t + P - 1) // P].long()
        keys, values = st["k"][pages].flatten(0, 1)[:t].float(), st["v"][pages].flatten(0, 1)[:t].float()
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


def plain_select(st):
    c, P, G, top = st["case"], st["case"]["page"], st["case"]["kv_heads"], st["case"]["top"]
    big = torch.finfo(torch.float64).max
    out = []
    for s, t in enumerate(st["host_lens"]):
        a, b = st["host_starts"][s], st["host_starts"][s + 1]
        n = (t + P - 1) // P
        means = st["means"][st["table"][s, :n].long()].double()
        q = st["q"][a:b].double().unflatten(1, (G, -1)).sum(dim=2)
        score = torch.einsum("ngd,jgd->ngj", q, means).nan_to_num(nan=-big, posinf=big, neginf=-big)
        last = (torch.arange(t - (b - a), t, device="cuda") // P)[:, None, None]
        j = torch.arange(n, device="cuda")
        score = torch.where((j < c["first"]) | (j >= last - c["recent"]), math.inf, score)
        score = torch.where(j > last, -math.inf, score)
        best, at = score.sort(dim=-1, descending=True, stable=True)
        best, at = best[..., :top], at[..., :top]
        at = torch.where(best > -math.inf, at, n).sort(dim=-1).values
        at = torch.where(at < n, at, -1)
        out.append(torch.nn.functional.pad(at, (0, top - at.shape[-1]), value=-1))
    return torch.cat(out).to(torch.int32)


def plain_selected(st):
    c, P, G = st["case"], st["case"]["page"], st["case"]["kv_heads"]
    seq, pos = where(st)
    lists = st["lists"].long()
    kh, vh, head = st["k"].transpose(1, 2), st["v"].transpose(1, 2), torch.arange(G, device="cuda")[None, :, None]
    step = max(1, (1 << 28) // (G * lists.shape[2] * P * max(c["dim"], c["vdim"])))
    outs, lses = [], []
    for a in range(0, len(pos), step):
        rows = slice(a, a + step)
        j = lists[rows]
        page = torch.gather(st["table"][seq[rows]].long()[:, None].expand(-1, G, -1), 2, j.clamp_min(0))
        keys, values = kh[page, head].flatten(2, 3).float(), vh[page, head].flatten(2, 3).float()
        q = st["q"][rows].float().unflatten(1, (G, -1))
        at = (j[..., None] * P + torch.arange(P, device="cuda")).flatten(2)
        seen = (at >= 0) & (at <= pos[rows, None, None]) & (j >= 0)[..., None].expand(*j.shape, P).flatten(2)
        score = torch.matmul(q, keys.transpose(2, 3)) * st["scale"]
        score.masked_fill_(~seen[:, :, None], -math.inf)
        top = score.amax(dim=-1, keepdim=True)
        p = (score - top).exp()
        total = p.sum(dim=-1, keepdim=True)
        outs.append((torch.matmul(p, values) / total).flatten(1, 2))
        lses.append((top + total.log()).squeeze(-1).flatten(1))
    return {"out": torch.cat(outs).to(st["q"].dtype), "lse": torch.cat(lses)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------
def exact(c, seed):
    st = inputs(c, seed)
    H, G, P = c["heads"], c["kv_heads"], c["page"]
    rep, starts, lens, table = H // G, st["host_starts"], st["host_lens"], st["table"].tolist()
    if c["op"] == "append":
        k, v, means = st["k"].double(), st["v"].double(), None if st["means"] is None else st["means"].double()
        q = st["new_q"].double()
        place = [(table[s][p // P], p % P, p) for s in range(len(lens)) for p in range(lens[s] - starts[s + 1] + starts[s], lens[s])]
        pg, sl, pos = (torch.tensor(x, device="cuda") for x in zip(*place))
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), pos.double()[:, None] * st["freq"].double())[:, None]
        n = c["rot"]

        def rotate(x):
            x = x.double().clone()
            a, b = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["neighbours"] else (slice(0, n), slice(n, 2 * n))
            z = torch.complex(x[..., a].contiguous(), x[..., b].contiguous()) * turn
            x[..., a], x[..., b] = z.real, z.imag
            return x

        k[pg, sl], v[pg, sl] = rotate(st["new_k"]), st["new_v"].double()
        out = {"q": rotate(q), "k": k, "v": v}
        if c["means"]:
            for page, slot, _ in place:
                if slot == P - 1:
                    means[page] = k[page].sum(dim=0) / P  # of keys before they are rounded
            out["means"] = means
        return out
    if c["op"] == "select":
        lists = []
        q, means = st["q"].double().cpu(), st["means"].double().cpu()
        for s, t in enumerate(lens):
            score = torch.stack([means[table[s][:t // P + 1], g] @ q[starts[s]:starts[s + 1], g * rep:(g + 1) * rep].sum(dim=1).T for g in range(G)]).tolist()
            for i in range(starts[s + 1] - starts[s]):
                last = (t - starts[s + 1] + starts[s] + i) // P
                for g in range(G):
                    always = {j for j in range(last + 1) if j < c["first"] or j >= last - c["recent"]}
                    rest = sorted((-score[g][j][i], j) for j in range(last + 1) if j not in always)
                    pick = sorted(always | {j for _, j in rest[:c["top"] - len(always)]})
                    lists.append(pick + [-1] * (c["top"] - len(pick)))
        return torch.tensor(lists, dtype=torch.int32, device="cuda").view(-1, G, c["top"])
    out = torch.zeros(starts[-1], H, c["vdim"], dtype=torch.float64, device="cuda")
    lse = torch.zeros(starts[-1], H, dtype=torch.float64, device="cuda")
    for s, t in enumerate(lens):
        at = torch.arange(t, device="cuda")
        pg, sl = torch.tensor(table[s], device="cuda")[at // P], at % P
        for a in range(starts[s], starts[s + 1], 256):
            b = min(a + 256, starts[s + 1])
            pos = t - starts[s + 1] + torch.arange(a, b, device="cuda")
            for g in range(G):
                seen = at <= pos[:, None]
                if c["op"] == "selected":
                    listed = torch.zeros(b - a, t // P + 2, dtype=torch.bool, device="cuda")
                    j = st["lists"][a:b, g].long()
                    listed.scatter_(1, torch.where(j < 0, t // P + 1, j), True)
                    seen = seen & listed[:, at // P]
                s64 = st["q"][a:b, g * rep:(g + 1) * rep].double() @ st["k"][pg, sl, g].double().T * st["scale"]
                s64 = s64.masked_fill(~seen[:, None], -math.inf)
                lse[a:b, g * rep:(g + 1) * rep] = s64.logsumexp(dim=-1)
                out[a:b, g * rep:(g + 1) * rep] = s64.softmax(dim=-1) @ st["v"][pg, sl, g].double()
    return {"out": out, "lse": lse}

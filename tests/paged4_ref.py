"""Plain 64-bit restatement of the 4-bit paged cache's operators and of the verification of drafts on the CPU, and problems for them."""
import math

import torch

from paged_ref import F32, HALF, TYPES

BLOCKS = lambda n: 2 if n <= 64 else 4 if n <= 128 else 8
MANY = 64  # (token, head) rows


def quantise(x):
    """Scales (.., blocks) in fp16 and codes (.., blocks, 32) of fp32 rows x (.., n), block by block from the definition."""
    n = x.shape[-1]
    b = torch.zeros(*x.shape[:-1], BLOCKS(n) * 32)
    b[..., :n] = x
    b = b.unflatten(-1, (-1, 32)).double()
    hi, lo = b.max(dim=-1).values, b.min(dim=-1).values
    top = torch.where(hi >= -lo, hi, lo)
    d = (top / -8).clamp(-65504, 65504).float().half()
    d64 = d.double()[..., None]
    c = torch.where(d64 == 0, torch.full_like(b, 8.0), torch.clamp(torch.round(b / torch.where(d64 == 0, 1.0, d64)) + 8, 0, 15))
    odd = ~torch.isfinite(b).all(dim=-1)
    c[odd] = 8
    d[odd] = math.nan
    return d, c.nan_to_num(8).to(torch.int64)


def values(d, c, n):
    return ((c - 8).double() * d.double()[..., None]).flatten(-2)[..., :n]


def place(entry, lanes, blocks):
    """Byte and half of an entry's code in its slot's row."""
    per = 32 // lanes
    g, e = divmod(entry, 32)
    t, i = divmod(e, per)
    return t * (per // 2) * blocks + g * (per // 2) + i // 2, i % 2


def pack(k, v):
    """Pages' bytes (pages, G, bytes) of keys and values (pages, G, P, n), entry by entry."""
    out = []
    for x, lanes in ((k, 4), (v, 8)):
        d, c = quantise(x)
        n = BLOCKS(x.shape[-1])
        rows = torch.zeros(*x.shape[:-1], n * 16, dtype=torch.uint8)
        for e in range(n * 32):
            at, half = place(e, lanes, n)
            rows[..., at] |= (c[..., e // 32, e % 32] << (4 * half)).to(torch.uint8)
        out += [rows.flatten(2), d.contiguous().view(torch.uint8).flatten(2)]
    return torch.cat(out, dim=2)


def unpack(pool, P, d, dv):
    """The numbers of all slots: (pages, G, P, d) and (pages, G, P, dv) in 64 bits."""
    at, out = 0, []
    for n, lanes in ((d, 4), (dv, 8)):
        b = BLOCKS(n)
        rows = pool[:, :, at:at + P * b * 16].unflatten(2, (P, -1)).to(torch.int64)
        at += P * b * 16
        scales = pool[:, :, at:at + P * b * 2].contiguous().view(torch.float16).unflatten(2, (P, -1)).double()
        at += P * b * 2
        x = torch.zeros(*rows.shape[:3], n, dtype=torch.float64)
        for e in range(n):
            byte, half = place(e, lanes, b)
            x[..., e] = ((rows[..., byte] >> (4 * half) & 15) - 8) * scales[..., e // 32]
        out.append(x)
    return out


class Problem4:
    """A batch over a pool of random 4-bit pages.  What no position of a sequence lies in is all ones: scales that are no numbers."""

    def __init__(self, type, new, lens, G=2, rep=4, d=64, dv=None, page=16, order="head", groups=None, spare=3, seed=0, pad_rows=0, offset=0, k=None, v=None):
        self.type, self.t, self.new, self.lens, self.G, self.rep, self.H = type, TYPES[type], list(new), list(lens), G, rep, G * rep
        self.d, self.dv, self.page, self.groups, self.offset, self.order = d, dv or d, page, groups, offset, order
        g = self.gen = torch.Generator().manual_seed(seed)
        self.starts = [offset]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + pad_rows
        B = len(new)
        self.pages = sum(-(-x // page) for x in lens) + spare
        left = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((B, max([1] + [-(-x // page) for x in lens])), -1, dtype=torch.int32)
        for s in range(B):
            for j in range(-(-lens[s] // page)):
                self.table[s, j] = left.pop()
        if groups:
            for i, m in enumerate(groups[1]):
                for s in range(groups[0][i], groups[0][i + 1]):
                    self.table[s, :m // page] = self.table[groups[0][i], :m // page]
        self.scale = self.d ** -0.5
        self.q = torch.randn(self.rows, self.H, self.d, generator=g).to(self.t)
        self.fill(torch.randn(self.pages, G, page, self.d, generator=g) if k is None else k, torch.randn(self.pages, G, page, self.dv, generator=g) if v is None else v)

    def fill(self, k, v):
        """Keys and values (pages, G, page, n) into the slots that some position lies in."""
        self.pool = pack(k, v)
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for s, n in enumerate(self.lens):
            if n:
                at = torch.arange(n)
                used[self.table[s].long()[at // self.page], at % self.page] = True
        at = 0
        for n in (BLOCKS(self.d), BLOCKS(self.dv)):
            for size in (16 * n, 2 * n):
                self.pool[:, :, at:at + self.page * size].unflatten(2, (self.page, size)).masked_fill_(~used[:, None, :, None], 255)
                at += self.page * size
        self.k, self.v = unpack(self.pool, self.page, self.d, self.dv)

    def row(self, n):
        for s in range(len(self.new)):
            if self.starts[s] <= n < self.starts[s + 1]:
                return s, self.lens[s] - self.new[s] + n - self.starts[s]
        return None

    def attend(self, only=None):
        """(out, lse, tolerance of out, tolerance of lse) in 64 bits; rows outside every sequence, and those not in `only`, are NaN in `out`.

        Tolerances.  A product of 16 terms and what was there lines 17 numbers up by the largest exponent and keeps 23 bits behind it: it is off by at most 17 2^-23 of the largest number in it.
        With codes c - 8 of up to 2^3, two products to a block of 32 and queries that fp16 holds, a score is off by ds <= scale max|q| sum_blocks |d| 2 17 2^-20, and by (dim + 16) 2^-24 scale sum
        |q| |d| 16 for the fp32 additions; fp32 queries have two parts, which twice as many products and 2^-22 of each entry add to.  A probability is off by the factor 1 + 2 ds (its own score's and the
        denominator's); the sums over n keys add n 2^-24, exp2 and its argument (1 + |s| log2 e) 2^-22, all relative to sum p |v|.  The second product, in the same way: 2 17 2^-20 sum p |d|, n / 16
        17 2^-23 sum p |v| for what was there, and 2^-21 15 sum p |d| for p d in two parts.  bf16 queries have p d in one part: 2^-11 sum p |v|.  Where more than MANY rows of a kv head (of 16-bit
        queries, heads of up to 128 entries) read the same keys, p and p d are rounded to fp16, each 2^-11 sum p |v|.  The result is rounded once to its type."""
        out = torch.full((self.rows, self.H, self.dv), math.nan, dtype=torch.float64)
        lse, tol_o, tol_l = out[..., 0].clone(), torch.zeros_like(out), torch.zeros(self.rows, self.H, dtype=torch.float64)
        half, wide = HALF[self.type], self.type == "f32"
        dk = self.pool_scales(0)
        dvs = self.pool_scales(1)
        for n in range(self.rows) if only is None else only:
            w = self.row(n)
            if w is None:
                continue
            s, p = w
            at = torch.arange(max(p + 1, 0))
            pg, sl = self.table[s].long()[at // self.page], at % self.page
            for g in range(self.G):
                hs = slice(g * self.rep, (g + 1) * self.rep)
                if len(at) == 0:
                    out[n, hs], lse[n, hs] = 0.0, -math.inf
                    continue
                k, v, q = self.k[pg, g, sl], self.v[pg, g, sl], self.q[n, hs].double()
                sc = q @ k.T * self.scale
                pr = sc.softmax(dim=1)
                out[n, hs], lse[n, hs] = pr @ v, sc.logsumexp(dim=1)
                a, b = dk[pg, g, sl].double().abs(), dvs[pg, g, sl].double().abs()
                top, size = q.abs().max(dim=1).values * abs(self.scale), a.sum(dim=1).max()
                ds = top * size * (4 * 17 * 2.0 ** -20 + 2.0 ** -15 if wide else 2 * 17 * 2.0 ** -20)
                ds = ds + (self.d + 16) * F32 * (q.abs().sum(dim=1) * abs(self.scale)) * a.max() * 16
                rough = 0.0
                if not wide:
                    rough = 2.0 ** -11 if self.type == "bf16" else 0.0
                    if self.many(s):
                        rough = 2 * 2.0 ** -11
                rel = 2 * ds + rough + 2 * len(at) * F32 + 8 * (1 + sc.abs().max(dim=1).values * 1.4427) * F32
                spread, step = pr @ v.abs(), (pr @ b).repeat_interleave(32, dim=1)[:, :self.dv]
                tol_o[n, hs] = spread * (rel[:, None] + len(at) * 17 * 2.0 ** -27) + step * 2 * 17 * 2.0 ** -20 + step * 15 * 2.0 ** -21 + out[n, hs].abs() * half
                tol_l[n, hs] = rel + 2 * F32 * lse[n, hs].abs()
        if self.type == "f16":
            tol_o += 2.0 ** -25
        return out, lse, tol_o, tol_l

    def many(self, s):
        """Whether some of a sequence's keys may be read by many rows."""
        rows = self.new[s]
        if self.groups:
            for i in range(len(self.groups[1])):
                a, b = self.groups[0][i], self.groups[0][i + 1]
                if a <= s < b:
                    rows = max(rows, sum(self.new[a:b]))
        return rows * self.rep > MANY and max(self.d, self.dv) <= 128

    def pool_scales(self, which):
        a, b, P = BLOCKS(self.d), BLOCKS(self.dv), self.page
        at, n = (P * a * 16, a) if which == 0 else (P * (a * 18 + b * 16), b)
        return self.pool[:, :, at:at + P * n * 2].contiguous().view(torch.float16).unflatten(2, (P, -1))

    def on_gpu(self):
        """A cache and a batch of copies on the GPU; pages in another order of dimensions, and apart, on request."""
        from xalm_b200 import paged
        dev = torch.device("cuda", 0)
        n, G, b = self.pool.shape
        if self.order == "head":
            self.gpool = self.pool.to(dev)
        elif self.order == "page":  # all pages of a head together
            self.gpool = torch.empty(G, n, b, dtype=torch.uint8, device=dev).transpose(0, 1)
        else:  # one layer of several
            self.gpool = torch.full((n, 3, G, b + 48), 255, dtype=torch.uint8, device=dev)[:, 1, :, :b]
        self.gpool.copy_(self.pool)
        self.gq = self.q.to(dev)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        bounds = dict(groups=i32(self.groups[0]), shared=i32(self.groups[1])) if self.groups else {}
        return paged.PagedCache4(self.gpool, self.page, self.d, self.dv), paged.Batch(i32(self.starts), i32(self.lens), self.table.to(dev), **bounds)


def turned(x, pos, freq, mag, neighbours):
    """A row (heads, n) at a position, turned in 64 bits."""
    x = x.double().clone()
    n = 0 if freq is None else freq.numel()
    if n:
        angle = pos * freq.double()
        cs, sn, i = angle.cos(), angle.sin(), torch.arange(n)
        a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + n)
        u, w = x[:, a].clone(), x[:, b].clone()
        x[:, a], x[:, b] = (u * cs - w * sn) * mag, (w * cs + u * sn) * mag
    return x


def verify(starts, tokens, target, accept, pick, draft=None):
    """Tokens and how many drafts are taken, from the definition."""
    rows, V = target.shape
    out, taken = [None] * rows, []
    for s in range(len(starts) - 1):
        a, b = starts[s], starts[s + 1]
        i = a
        while i + 1 < b:
            x = int(tokens[i + 1])
            if not (0 <= x < V and float(accept[i]) * (1.0 if draft is None else float(draft[i, x])) < float(target[i, x])):
                break
            out[i] = x
            i += 1
        taken.append(max(i - a, 0))
        if a == b:
            continue
        refused = i + 1 < b
        weights = []
        for use_draft in ([True, False] if refused else [False]):
            p = target[i].double()
            p = torch.where(p > 0, p, 0.0)
            if use_draft:
                if draft is None:
                    x = int(tokens[i + 1])
                    if 0 <= x < V:
                        p[x] = 0.0
                else:
                    q = draft[i].double()
                    p = (p - torch.where(q > 0, q, 0.0)).clamp_min(0.0)
            weights = p
            if float(p.sum()) > 0:
                break
        total, goal, last = 0.0, float(pick[s]) * math.fsum(weights.tolist()), -1
        out[i] = -1
        for v in torch.nonzero(weights).flatten().tolist():
            total += float(weights[v])
            last = v
            if total > goal:
                break
        out[i] = last
        for j in range(i + 1, b):
            out[j] = -1
    return out, taken

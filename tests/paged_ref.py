"""Plain 64-bit restatement of the paged cache's operators on the CPU, and problems for them."""
import math

import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # the most a rounding is off, relative to the value
F32 = 2.0 ** -24


class Problem:
    """A batch over a pool with random pages.  new, lens: tokens of this call and all tokens, per sequence; shared: (groups' bounds, shared tokens)."""

    def __init__(self, type, new, lens, G=2, rep=4, d=64, dv=None, page=16, layout="position", groups=None, spare=3, seed=0, pad_rows=0, offset=0, max_pages=None, key_scale=1.0):
        self.type, self.t, self.new, self.lens, self.G, self.rep, self.H = type, TYPES[type], list(new), list(lens), G, rep, G * rep
        self.d, self.dv, self.page, self.groups = d, dv or d, page, groups
        g = torch.Generator().manual_seed(seed)
        self.gen = g
        self.offset = offset
        self.starts = [offset]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.rows = self.starts[-1] + pad_rows
        B = len(new)
        self.max_pages = max_pages or max([1] + [-(-x // page) for x in lens])
        need = sum(-(-x // page) for x in lens)
        self.pages = need + spare
        order = torch.randperm(self.pages, generator=g).tolist()
        self.table = torch.full((B, self.max_pages), -1, dtype=torch.int32)
        for s in range(B):
            for j in range(-(-lens[s] // page)):
                self.table[s, j] = order.pop()
        if groups:
            bounds, shared = groups
            for i, m in enumerate(shared):
                for s in range(bounds[i], bounds[i + 1]):
                    self.table[s, :m // page] = self.table[bounds[i], :m // page]
        self.k, self.v = self.pool(self.d, key_scale), self.pool(self.dv)
        if layout == "head":
            self.k, self.v = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (self.k, self.v))
        self.q = self.normal(self.rows, self.H, self.d)
        self.scale = self.d ** -0.5

    def normal(self, *shape, scale=1.0, dtype=None):
        return (torch.randn(*shape, generator=self.gen) * scale).to(dtype or self.t)

    def pool(self, n, scale=1.0):
        return self.normal(self.pages, self.page, self.G, n, scale=scale)

    def row(self, n):
        """(sequence, position) of a row; None outside every sequence."""
        for s in range(len(self.new)):
            if self.starts[s] <= n < self.starts[s + 1]:
                return s, self.lens[s] - self.new[s] + n - self.starts[s]
        return None

    def slots(self, s, at):
        at = torch.as_tensor(at)
        return self.table[s].long()[at // self.page], at % self.page

    def written_only(self, fill=math.nan):
        """Fills what no position of any sequence lies in."""
        used = torch.zeros(self.pages, self.page, dtype=torch.bool)
        for s, n in enumerate(self.lens):
            if n:
                used[self.slots(s, torch.arange(n))] = True
        self.k[~used], self.v[~used] = fill, fill

    def attend(self, lists=None, round_p=True, only=None):
        """(out, lse, tolerance of out, tolerance of lse) in 64 bits; rows outside every sequence, and those not in `only`, are NaN in `out`.

        Tolerances: scores are sums of d products in fp32, each off by at most 2^-24 of the sum of absolute products per addition, so a score is off by
        ds <= (d + 2) 2^-24 scale sum |q k|, and a probability by the factor 1 + 2 ds (its own score's and the denominator's).  The sums over n keys in fp32 add n 2^-24, exp2 and the scaling of its
        argument (1 + |s| log2 e) 2^-22, the joins of partial results as much again; the probabilities' rounding to the matrix operand's type adds half a step of it.  All are
        relative to sum p |v|.  The result is rounded once to its type."""
        out = torch.full((self.rows, self.H, self.dv), math.nan, dtype=torch.float64)
        lse, tol_o, tol_l = out[..., 0].clone(), torch.zeros_like(out), torch.zeros(self.rows, self.H, dtype=torch.float64)
        half = HALF[self.type]
        for n in range(self.rows) if only is None else only:
            w = self.row(n)
            if w is None:
                continue
            s, p = w
            for g in range(self.G):
                at = torch.arange(max(p + 1, 0))
                if lists is not None:
                    named = set(int(x) for x in lists[n, g])
                    at = torch.tensor([j for j in at.tolist() if j // self.page in named], dtype=torch.long)
                hs = slice(g * self.rep, (g + 1) * self.rep)
                if len(at) == 0:
                    out[n, hs], lse[n, hs] = 0.0, -math.inf
                    continue
                pg, sl = self.slots(s, at)
                k, v, q = self.k[pg, sl, g].double(), self.v[pg, sl, g].double(), self.q[n, hs].double()
                sc = q @ k.T * self.scale
                pr = sc.softmax(dim=1)
                out[n, hs], lse[n, hs] = pr @ v, sc.logsumexp(dim=1)
                ds = (self.d + 2) * F32 * (q.abs() @ k.abs().T * abs(self.scale)).max(dim=1).values
                rel = 2 * ds + 2 * len(at) * F32 + 8 * (1 + sc.abs().max(dim=1).values * 1.4427) * F32
                spread = pr @ v.abs()
                tol_o[n, hs] = spread * (rel + (half if round_p and self.type != "f32" else 0))[:, None] + out[n, hs].abs() * half
                tol_l[n, hs] = rel + 2 * F32 * lse[n, hs].abs()
        if self.type == "f16":
            tol_o += 2.0 ** -25  # half a step of the smallest numbers
        return out, lse, tol_o, tol_l

    def turned(self, x, n_rot, freq, mag, neighbours):
        """Rows x (rows, heads, d) turned by their positions, in 64 bits."""
        x = x.double().clone()
        for n in range(self.rows):
            w = self.row(n)
            if w is None or n_rot == 0:
                continue
            angle = w[1] * freq.double()
            cs, sn = angle.cos() * mag, angle.sin() * mag
            i = torch.arange(n_rot)
            a, b = (2 * i, 2 * i + 1) if neighbours else (i, i + n_rot)
            u, z = x[n][:, a].clone(), x[n][:, b].clone()
            x[n][:, a], x[n][:, b] = u * cs - z * sn, z * cs + u * sn
        return x

    def select(self, means, top, first, recent):
        big = torch.finfo(torch.float64).max
        out = torch.full((self.rows, self.G, top), -1, dtype=torch.int32)
        for n in range(self.rows):
            w = self.row(n)
            if w is None or w[1] < 0:
                continue
            s, last = w[0], w[1] // self.page
            for g in range(self.G):
                always = [j for j in range(last + 1) if j < first or j >= last - recent]
                rest = [j for j in range(last + 1) if j not in always]
                q = self.q[n, g * self.rep:(g + 1) * self.rep].double().sum(dim=0)
                score = {j: float(torch.nan_to_num(means[int(self.table[s, j]), g].double() @ q, nan=-big, posinf=big, neginf=-big)) for j in rest}
                pick = sorted(always + sorted(rest, key=lambda j: (-score[j], j))[:top - len(always)])
                out[n, g, :len(pick)] = torch.tensor(pick, dtype=torch.int32)
        return out

    def on_gpu(self):
        """The operators' arguments: a cache and a batch of copies on the GPU."""
        from xalm_b200 import paged
        dev = torch.device("cuda", 0)

        def copy(x):
            y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev)
            return y.copy_(x)

        self.gk, self.gv, self.gq = copy(self.k), copy(self.v), self.q.to(dev)
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
        bounds = dict(groups=i32(self.groups[0]), shared=i32(self.groups[1])) if self.groups else {}
        return paged.PagedCache(self.gk, self.gv, getattr(self, "means", None) if getattr(self, "means", None) is None else self.means.to(dev)), \
            paged.Batch(i32(self.starts), i32(self.lens), self.table.to(dev), **bounds)

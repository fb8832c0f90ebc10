"""Plain 64-bit forms of the rotation and paged-cache operators, and how far
their results may be off, for the GPU tests."""

import math

import torch

from moba.kernels.paged import PagedKV

U24 = 2.0 ** -24  # half a step of float32 at 1


def half_step(dtype) -> float:
    """Most a rounding to `dtype` moves a value, relative to it."""
    return torch.finfo(dtype).eps / 2


def tables(positions, rotary, base=10000.0):
    freq = base ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def rotate(x, cos, sin, interleaved):
    """x [..., D] turned by cos, sin [..., rotary / 2]."""
    half = cos.shape[-1]
    y = x.clone()
    a, b = (x[..., 0:2 * half:2], x[..., 1:2 * half:2]) if interleaved else \
        (x[..., :half], x[..., half:2 * half])
    ya, yb = a * cos - b * sin, b * cos + a * sin
    if interleaved:
        y = torch.cat((torch.stack((ya, yb), -1).flatten(-2), x[..., 2 * half:]), -1)
    else:
        y = torch.cat((ya, yb, x[..., 2 * half:]), -1)
    return y


def norm_rotate64(x, w, cos, sin, pos, eps, interleaved):
    """[..., H, D] at positions pos [...], in float64; differentiable."""
    n = x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    if cos is None:
        return n
    return rotate(n, cos.double()[pos][..., None, :], sin.double()[pos][..., None, :], interleaved)


def pair_size(x, w, cos, eps, interleaved):
    """|n_a| + |n_b| of every feature's pair: what bounds a rotation's rounding."""
    n = (x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w).abs()
    if cos is None:
        return n
    half = cos.shape[-1]
    out = n.clone()
    if interleaved:
        s = n[..., 0:2 * half:2] + n[..., 1:2 * half:2]
        out[..., :2 * half] = torch.stack((s, s), -1).flatten(-2)
    else:
        s = n[..., :half] + n[..., half:2 * half]
        out[..., :2 * half] = torch.cat((s, s), -1)
    return out


def forward_bound(ref, size, dtype):
    """A row's sum of squares: 16 terms in a lane, up to 6 sums across lanes,
    so at most 22 roundings, halved by the root; the mean, eps, the root, two
    products, two products and a sum of the rotation: under 32 in all. Then
    the rounding to the type (subnormal float16: 2^-25)."""
    return half_step(dtype) * ref.abs() + 32 * U24 * size + (2.0 ** -25 if dtype == torch.float16 else 0)


class Paged:
    """Sequences on the pages of a cache, on the CPU, everything that no
    sequence's token owns NaN."""

    def __init__(self, lens, h_kv, block, d, dtype, seed, spare=2, width=None, tokens=None):
        g = torch.Generator().manual_seed(seed)
        self.g, self.lens, self.block, self.h_kv, self.d, self.dtype = g, lens, block, h_kv, d, dtype
        counts = [-(-n // block) for n in lens]
        pages = max(1, sum(counts)) + spare
        order = torch.randperm(pages, generator=g).to(torch.int32)
        width = max(1, max(counts)) if width is None else width
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        self.k = torch.full((pages, h_kv, block, d), math.nan, dtype=dtype)
        self.v = self.k.clone()
        self.kbar = torch.full((pages, h_kv, d), math.nan, dtype=dtype)
        at = 0
        for s, n in enumerate(counts):
            self.table[s, :n] = order[at:at + n]
            at += n
            if tokens is None:
                self.put(s, self.randn(lens[s], h_kv, d), self.randn(lens[s], h_kv, d))
        # Unused entries: pages that hold nothing, or no pages at all.
        for s, n in enumerate(counts):
            for j in range(n, width):
                self.table[s, j] = (-1, pages, 2 ** 31 - 1, int(order[-1]) if spare else -7)[(s + j) % 4]

    def randn(self, *shape):
        return torch.randn(shape, generator=self.g).to(self.dtype)

    def put(self, s, k, v, first=0):
        """Tokens [n, H, D] of sequence s from position `first`, and kbar of full blocks."""
        for i in range(k.shape[0]):
            p, r = int(self.table[s, (first + i) // self.block]), (first + i) % self.block
            if not 0 <= p < self.k.shape[0]:
                continue
            self.k[p, :, r], self.v[p, :, r] = k[i], v[i]
            if r == self.block - 1:
                total = self.k[p].double().sum(1).float().to(self.dtype).float()
                self.kbar[p] = (total / self.block).to(self.dtype)

    def gpu(self):
        return (PagedKV(self.k.cuda(), self.v.cuda(), self.kbar.cuda()), self.table.cuda(),
                torch.tensor(self.lens, dtype=torch.int32, device="cuda"))


def cu_of(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return torch.tensor(cu, dtype=torch.int32)


def select64(p, s, q, pos, cfg):
    """Ids of one token's heads: q [H, D]. Lists, ascending."""
    own = pos // p.block
    take = cfg.past_blocks_selected(p.table.shape[1])
    group = q.shape[0] // p.h_kv
    ids = []
    for h in range(q.shape[0]):
        ranked = []
        for j in range(min(own, p.table.shape[1])):
            page = int(p.table[s, j])
            if 0 <= page < p.k.shape[0]:
                x = (q[h].double() @ p.kbar[page, h // group].double()).float().to(p.dtype).item()
                if x > -math.inf:
                    ranked.append((-x, j))
        chosen = sorted(j for _, j in sorted(ranked)[:take])
        if cfg.always_select_current and own < p.table.shape[1] and \
                0 <= int(p.table[s, own]) < p.k.shape[0]:
            chosen.append(own)
        ids.append(chosen)
    return ids


def attend64(p, s, q, pos, ids):
    """(out, lse in log2 units, bound) of one token's heads over blocks `ids`.

    The bound counts: per score at most 16 + 6 + 2 roundings of float32 of the
    sum of |q k| (eight or four terms in a lane, sums across lanes; on matrix
    units at most D / 8 + 8 additions of one chain), twice over (numerator and
    sum); exp2 and the sums over keys, 64 more of the weights. 16-bit inputs
    may round each weight and each block's result once to the type: half a
    step each of the weighted mean of |v|; then the rounding of the output."""
    group = q.shape[0] // p.h_kv
    out, lse, bound = torch.zeros(q.shape, dtype=torch.float64), [], []
    for h in range(q.shape[0]):
        ks, vs = [], []
        for j in ids[h]:
            page = int(p.table[s, j])
            n = min(p.block, pos - j * p.block + 1)
            if n > 0:
                ks.append(p.k[page, h // group, :n].double())
                vs.append(p.v[page, h // group, :n].double())
        if not ks:
            lse.append(-math.inf)
            bound.append(torch.zeros(q.shape[1], dtype=torch.float64))
            continue
        k, v = torch.cat(ks), torch.cat(vs)
        scale = q.shape[1] ** -0.5
        x = k @ q[h].double() * scale
        w = torch.softmax(x, 0)
        out[h] = w @ v
        lse.append((torch.logsumexp(x, 0) / math.log(2)).item())
        terms = (k.abs() @ q[h].double().abs()).max().item() * scale
        spread = v.abs().max().item()
        delta = U24 * ((q.shape[1] / 8 + 24) * terms + 64)
        b = half_step(p.dtype) * out[h].abs() + 2 * delta * spread
        if p.dtype != torch.float32:
            b = b + 2 * half_step(p.dtype) * (w @ v.abs())
        if p.dtype == torch.float16:
            b = b + 2.0 ** -24
        bound.append(b)
    return out, torch.tensor(lse, dtype=torch.float64), torch.stack(bound)

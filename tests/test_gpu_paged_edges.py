"""Calls over a paged cache at the edges of what they take: scores that are not
numbers, lengths and bounds that make no sense."""

import math

import pytest
import torch

from moba.config import MoBAConfig
from moba.kernels.paged import PagedKV, append_tokens, paged_attention, paged_gate_select
from paged_util import Paged, cu_of, half_step, select64

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def one_by_one(p, new, q, cfg):
    """(ids, out, lse) of a chunk's tokens as short calls, which take the kernels
    of single tokens."""
    cache, table, _ = p.gpu()
    ids, out, lse, at = [], [], [], 0
    for s, n in enumerate(new):
        for i in range(0, n, 3):
            m = min(3, n - i)
            lens = torch.tensor([p.lens[s] - n + i + m], dtype=torch.int32, device="cuda")
            part = q[at + i:at + i + m].cuda()
            ids.append(paged_gate_select(part, cache, table[s:s + 1], lens, cfg))
            o, e = paged_attention(part, cache, table[s:s + 1], lens, cfg, return_lse=True)
            out.append(o)
            lse.append(e)
        at += n
    return torch.cat(ids), torch.cat(out), torch.cat(lse, 1)


# -- representatives far below 1 --------------------------------------------------

def check_small_representatives(length, n, h, unit):
    """Representatives whose squares are below float32's smallest number, and
    whose scores are what sums of their products lose: c + a - c, with a 2^-26
    of c and another one for every block."""
    d, block = 64, 16
    p = Paged([length], 1, block, d, BF, 31)
    blocks = torch.arange(length // block)
    kbar = torch.zeros(len(blocks), 1, d)
    kbar[:, 0, 0], kbar[:, 0, 32] = unit, -unit
    kbar[:, 0, 16] = unit * 2.0 ** -26 * (1 + (blocks * 37 % 128) / 128)
    p.kbar[p.table[0, :len(blocks)].long()] = kbar.to(BF)
    q = torch.zeros(n, h, d, dtype=BF)
    q[..., ::16] = 1.0
    q[..., 48] = p.randn(n, h)
    cfg = MoBAConfig(block_size=block, top_k=4)
    cache, table, lens = p.gpu()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg).cpu()
    for i in range(0, n, max(1, n // 10)):
        want = select64(p, 0, q[i], length - n + i, cfg)
        assert [x.tolist() for x in ids[i]] == want, i


@pytest.mark.parametrize("unit", [2.0 ** -60, 2.0 ** -80, 2.0 ** -95])
def test_small_representatives_of_a_chunk(device, unit):
    check_small_representatives(2000, 300, 32, unit)


# -- layouts ----------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("h", [1, 4])
def test_one_token_of_odd_rows(device, dtype, h):
    """A token of a projection whose rows are no multiple of 16 bytes, appended:
    the pages and queries of contiguous tensors."""
    d, block = 64, 16
    p = Paged([block], 1, block, d, dtype, 28)
    x = p.randn(1, (h + 2) * d + 5).cuda()
    q, k, v = x[:, :h * d].unflatten(1, (h, d)), x[:, None, h * d:h * d + d], x[:, None, h * d + d:h * d + 2 * d]
    got = []
    for q, k, v in ((q, k, v), [torch.empty(t.shape, dtype=dtype, device="cuda").copy_(t) for t in (q, k, v)]):
        cache, table, lens = p.gpu()
        got.append([append_tokens(q, k, v, cache, table, lens), cache.k, cache.v, cache.kbar])
    for a, b in zip(*got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


# -- scores that are not numbers --------------------------------------------------

def check_scores_that_are_not_numbers(dtype, d, block, length, n, h, hk=2):
    """Queries with NaN, a key of NaN that is the first of its token's own block,
    a block whose keys are all NaN: whoever sees one has NaN for a result and for
    its lse, and nobody else, as in short calls."""
    cfg = MoBAConfig(block_size=block, top_k=4)
    p = Paged([length], hk, block, d, dtype, 21)
    q = p.randn(n, h, d)
    q[7, -1, 5], q[12], q[n - 1, 0] = math.nan, math.nan, math.nan
    first = -(-(length - n) // block) * block  # a new token whose block begins with it
    p.k[p.table[0, first // block], 0, 0, 9] = math.nan
    p.k[p.table[0, 2], 1] = math.nan  # kbar stays: the block is chosen
    cache, table, lens = p.gpu()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg)
    out, lse = paged_attention(q.cuda(), cache, table, lens, cfg, return_lse=True)
    want_ids, want, want_lse = one_by_one(p, [n], q, cfg)
    assert torch.equal(ids, want_ids)
    # By the definition: any NaN among the query and the keys that it sees.
    pos = torch.arange(length - n, length)[:, None]
    chosen, group = ids.cpu(), h // hk
    bad = q.isnan().any(-1)
    bad[:, :group] |= ((chosen == first // block).any(-1) & (pos >= first))[:, :group]
    bad[:, group:] |= (chosen == 2).any(-1)[:, group:]
    assert bool(bad[first - (length - n), :group].all()) and 0 < int(bad.sum()) < bad.numel()
    for o, e in ((want, want_lse), (out, lse)):
        assert torch.equal(o.cpu().isnan(), bad[..., None].expand(-1, -1, d))
        assert torch.equal(e.cpu().isnan(), bad.t())
        assert bool(o.cpu()[~bad].isfinite().all()) and bool(e.cpu().t()[~bad].isfinite().all())


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("d,block", [(128, 128), (64, 96)])
def test_chunks_with_scores_that_are_not_numbers(device, dtype, d, block):
    check_scores_that_are_not_numbers(dtype, d, block, 1000, 300, 32)


# -- numbers that make no sense ---------------------------------------------------

def check_farthest_length(dtype, d, block, ctx, new, h, hk=2):
    """A sequence of 2^31 - 1 tokens between two ordinary ones: it sees its past
    blocks, and they have every bit that they have beside an ordinary one."""
    cfg = MoBAConfig(block_size=block, top_k=4)
    p = Paged([c + n for c, n in zip(ctx, new)], hk, block, d, dtype, 22,
              width=max(-(-(c + n) // block) for c, n in zip(ctx, new)) + 2)
    q = p.randn(sum(new), h, d)
    cu = cu_of(new).cuda()
    a, b = new[0], new[0] + new[1]
    cache, table, lens = p.gpu()
    want = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    p.lens[1] = 2 ** 31 - 1
    cache, table, lens = p.gpu()
    out = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    assert torch.equal(out[:a], want[:a]) and torch.equal(out[b:], want[b:])
    alone = one_by_one(p, new, q, cfg)[1]
    # Weights and results rounded, half a step of max |v| each on each side.
    far = (out[a:b].double() - alone[a:b].double()).abs().max().item()
    assert far <= 4 * half_step(dtype) * p.v[p.v.isfinite()].abs().max().item()


@pytest.mark.parametrize("dtype,d,block", [(BF, 128, 128), (FH, 64, 64)])
def test_the_farthest_length_in_a_chunk(device, dtype, d, block):
    check_farthest_length(dtype, d, block, [900, 300, 700], [200, 60, 150], 32)


def check_bounds(dtype, d, block, bounds, counted, tokens, ctx, h, hk=2):
    """Bounds that fall, leave the token axis or overlap: sequences that make
    sense by themselves and begin where no earlier such one reaches are served,
    the others have no new tokens, in every call alike."""
    seqs = len(bounds) - 1
    cfg = MoBAConfig(block_size=block, top_k=4)
    new = [max(0, b - a) if b <= tokens else 7 for a, b in zip(bounds, bounds[1:])]
    p = Paged([ctx + n for n in new], hk, block, d, dtype, 23, width=-(-(ctx + max(new)) // block) + 1)
    x = p.randn(tokens, h + 2 * hk, d).cuda()
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    cu = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    cache, table, lens = p.gpu()
    want_cache, _, _ = p.gpu()
    mine = torch.zeros(tokens, dtype=torch.bool)
    for s in counted:
        mine[bounds[s]:bounds[s + 1]] = True
    mine = mine.to(q.device)
    out = torch.full((tokens, h, d), 5.0, dtype=dtype, device="cuda")
    append_tokens(q, k, v, cache, table, lens, cu_seqlens=cu, out=out)
    assert torch.equal(out[mine], q[mine]) and bool((out[~mine] == 5).all())
    ids = paged_gate_select(q, cache, table, lens, cfg, cu_seqlens=cu)
    out.fill_(5.0)
    _, lse = paged_attention(q, cache, table, lens, cfg, cu_seqlens=cu, out=out, return_lse=True)
    assert bool((out[~mine] == 5).all()) and bool((ids[~mine] == -1).all())
    for s in counted:
        at = slice(bounds[s], bounds[s + 1])
        one = (table[s:s + 1].contiguous(), lens[s:s + 1])
        append_tokens(q[at], k[at], v[at], want_cache, *one)
        assert torch.equal(ids[at], paged_gate_select(q[at], want_cache, *one, cfg))
        want, want_lse = paged_attention(q[at], want_cache, *one, cfg, return_lse=True)
        # Weights and results rounded, half a step of max |v| each on each
        # side; float32: sums of up to 4 blocks in any order.
        most = p.v[p.v.isfinite()].abs().max().item()
        bar = 4 * half_step(dtype) * most if dtype != F32 else 2.0 ** -24 * 8 * block * most
        assert (out[at].double() - want.double()).abs().max().item() <= bar
        assert (lse[:, at] - want_lse).abs().max().item() <= 1e-4 + 2.0 ** -7 * (dtype != F32)
    for name in ("k", "v", "kbar"):
        a, b = (getattr(c, name).view(torch.uint8) for c in (cache, want_cache))
        assert torch.equal(a, b), name


# bounds, sequences that count
BOUNDS = [
    ([0, 999, 20, 60, 60], [2]),                       # the first leaves the axis
    ([0, 50, 30, 70, 100], [0, 3]),                    # the third begins inside the first
    ([-3, 10, 90, 5, 100], [1]),                       # the last begins before the second ends
    ([0, 40, 10, 100, 70, 90], [0]),                   # and so do all behind the first
    ([0] * 66 + [30, 20, 60, 100], [65, 68]),          # across 64 sequences
]


@pytest.mark.parametrize("bounds,counted", BOUNDS, ids=str)
@pytest.mark.parametrize("dtype,d,block", [(BF, 128, 128), (FH, 64, 64), (F32, 64, 32)])
@pytest.mark.parametrize("scale,h", [(1, 4), (3, 32)])
def test_bounds_that_make_no_sense(device, dtype, d, block, bounds, counted, scale, h):
    check_bounds(dtype, d, block, [scale * b for b in bounds], counted, 100 * scale, 700, h)


# -- values of very different sizes -----------------------------------------------

def attend_exactly(p, q, ids, pos):
    """One query's head of a kv head 0 .. by 64 bits: (out, weighted mean of |v|,
    largest |v| of each feature, bound on a weight's relative error by float32).

    Scores: at most D / 8 + 8 additions of one chain and two products, of sums
    of |q k| scaled; twice, in the row and in its sum; exp2 and the sums over
    keys and blocks, 64 roundings more."""
    ks, vs = [], []
    for j in ids:
        page, seen = int(p.table[0, j]), min(p.block, pos - j * p.block + 1)
        ks.append(p.k[page, :, :seen].double())
        vs.append(p.v[page, :, :seen].double())
    k, v = torch.cat(ks, 1), torch.cat(vs, 1)
    scale = q.shape[-1] ** -0.5
    w = torch.softmax((k[0] @ q.double()) * scale, 0)
    terms = (k[0].abs() @ q.double().abs()).max().item() * scale
    delta = 2 * 2.0 ** -24 * ((q.shape[-1] / 8 + 24) * terms + 64)
    return w @ v[0], w @ v[0].abs(), v[0].abs().amax(0), delta


def check_values(p, q, cfg, weights, tokens):
    """Every feature of a chunk's result (one kv head) within its own bound: half
    a step of the result, `weights` of the weighted mean of |v|, float32 sums."""
    n, h, d = q.shape
    cache, table, lens = p.gpu()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg).cpu()
    out = paged_attention(q.cuda(), cache, table, lens, cfg).cpu().double()
    for i in tokens:
        for hd in range(h):
            pos = p.lens[0] - n + i
            ref, mean, most, delta = attend_exactly(p, q[i, hd], [j for j in ids[i, hd].tolist() if j >= 0], pos)
            bound = half_step(p.dtype) * ref.abs() + weights * mean + delta * most
            if p.dtype == FH:
                bound = bound + 2.0 ** -25
            far = (out[i, hd] - ref).abs()
            assert bool((far <= bound).all()), (i, hd, (far / bound).max().item())


def check_large_channels(dtype, d, block, length, n, h, ratio):
    """A feature of every 64 that is `ratio` times the others leaves them as
    exact as they are without it."""
    p = Paged([length], 1, block, d, dtype, 24)
    p.v[..., 5] *= ratio
    p.v[..., d - 9] *= ratio
    cfg = MoBAConfig(block_size=block, top_k=4)
    check_values(p, p.randn(n, h, d), cfg, half_step(dtype), range(0, n, max(1, n // 12)))


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("d,block", [(128, 128), (64, 96)])
@pytest.mark.parametrize("ratio", [100, 4000])
def test_large_channels_leave_the_others_exact(device, dtype, d, block, ratio):
    check_large_channels(dtype, d, block, 1000, 300, 16, ratio)


def check_largest_values(block, length, n, h):
    """bf16 values behind 2^126, whose reciprocals are subnormal: one key of
    every block, at most three blocks to a query, so no sum passes float32."""
    p = Paged([length], 1, block, 64, BF, 25)
    p.v[p.v.isfinite()] = 0.0
    for j in range(length // block):
        p.v[p.table[0, j], 0, j % 3, 3] = 1e38
        p.v[p.table[0, j], 0, j % 5, 40] = -9e37
    cfg = MoBAConfig(block_size=block, top_k=3)
    check_values(p, p.randn(n, h, 64), cfg, half_step(BF), range(0, n, max(1, n // 12)))


def test_the_largest_values_in_a_chunk(device):
    check_largest_values(64, 1500, 600, 32)


def check_weights(dtype, block, length, n, h):
    """Weights are no rounder than float32 sums show: scores without rounding
    (one feature of a query counts), three keys of a block that matter, at s = 0
    and close below, and others whose weights are exactly 0.

    Roundings of float32, relative to the weighted mean of |v|: the scale and
    the two numbers that the exponent is formed of, at most 17 in size, 35 times
    ln 2; exp2 2; at most 12 weights summed, and as two numbers each in the
    product, 36; four blocks merged, 8: under 80, in the row and in its sum. A
    weight in two numbers of the type is off by half a step squared."""
    d = 64
    p = Paged([length], 1, block, d, dtype, 26)
    real = p.k.isfinite()
    p.k[real] = -24.0
    for j, page in enumerate(p.table[0].tolist()):
        for i, row in enumerate((1, block // 2, block - 2)):
            p.k[page, 0, row] = torch.where(p.k[page, 0, row].isfinite(),
                                            -torch.arange(d).add(j * 5 + i * 7).remainder(13) / 64, math.nan).to(dtype)
    q = torch.zeros(n, h, d, dtype=dtype)
    for i in range(n):
        for hd in range(h):
            q[i, hd, (i * 3 + hd * 11) % d] = 96.0
    cfg = MoBAConfig(block_size=block, top_k=4)
    cache, table, lens = p.gpu()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg).cpu()
    out = paged_attention(q.cuda(), cache, table, lens, cfg).cpu().double()
    for i in range(0, n, max(1, n // 25)):
        for hd in range(h):
            ref, mean, _, _ = attend_exactly(p, q[i, hd], [j for j in ids[i, hd].tolist() if j >= 0], length - n + i)
            bound = half_step(dtype) * ref.abs() + (half_step(dtype) ** 2 + 160 * 2.0 ** -24) * mean
            if dtype == FH:
                bound = bound + 2.0 ** -25
            far = (out[i, hd] - ref).abs()
            assert bool((far <= bound).all()), (i, hd, (far / bound).max().item())


@pytest.mark.parametrize("dtype", [BF, FH])
def test_weights_of_a_chunk_keep_their_bits(device, dtype):
    check_weights(dtype, 64, 1500, 600, 32)


def check_far_scores(dtype, block, length, n, h, size):
    """Scores so large that neighbours are far apart in float32: nothing but the
    best key of every query counts, and no weight leaves the type's range."""
    d = 64
    p = Paged([length], 1, block, d, dtype, 27)
    real = p.k.isfinite()
    p.k[real] = (p.k[real].float() * size).to(dtype)
    q = (p.randn(n, h, d).float() * size).to(dtype)
    cfg = MoBAConfig(block_size=block, top_k=4)
    cache, table, lens = p.gpu()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg).cpu()
    out, lse = paged_attention(q.cuda(), cache, table, lens, cfg, return_lse=True)
    assert bool(out.isfinite().all()) and bool(lse.isfinite().all())
    out = out.cpu().double()
    sure = 0
    for i in range(0, n, max(1, n // 25)):
        for hd in range(h):
            ks, vs = [], []
            for j in (j for j in ids[i, hd].tolist() if j >= 0):
                page, seen = int(p.table[0, j]), min(block, length - n + i - j * block + 1)
                ks.append(p.k[page, 0, :seen].double())
                vs.append(p.v[page, 0, :seen].double())
            k, v = torch.cat(ks), torch.cat(vs)
            x = k @ q[i, hd].double() / 8
            best, second = x.topk(2).values.tolist() if len(x) > 1 else (x[0].item(), -math.inf)
            # float32's sums of 64 products: 16 additions of a chain, and two
            # products, of sums of |q k| / 8, on both sides; 40 beyond leaves e^-40.
            terms = (k.abs() @ q[i, hd].double().abs()).max().item() / 8
            if best - second > 2 * 20 * 2.0 ** -24 * terms + 40:
                sure += 1
                far = (out[i, hd] - v[x.argmax()]).abs()
                assert bool((far <= half_step(dtype) * v[x.argmax()].abs() + 2.0 ** -25).all()), (i, hd)
    assert sure > 0


@pytest.mark.parametrize("dtype,size", [(FH, 700), (FH, 6000), (FH, 12000), (BF, 12000), (BF, 1e9)])
def test_chunks_of_far_scores(device, dtype, size):
    check_far_scores(dtype, 64, 1500, 600, 32, size)


# -- sizes ------------------------------------------------------------------------

def test_more_rows_than_a_launch_holds(device):
    """2^24 query rows and more, each with its own block only: the last sequence
    has the result that it has by itself."""
    seqs, n, h, d, block = 8, 65541, 32, 64, 16
    assert seqs * n * h > 1 << 24
    cfg = MoBAConfig(block_size=block, top_k=1, dtype=F32)
    width = -(-n // block)
    g = torch.Generator(device="cuda").manual_seed(29)
    q = torch.randn(seqs * n, h, d, generator=g, device="cuda")
    k, v = (torch.randn(seqs * width, 1, block, d, generator=g, device="cuda") for _ in range(2))
    cache = PagedKV(k, v, torch.zeros(seqs * width, 1, d, device="cuda"))
    table = torch.arange(seqs * width, dtype=torch.int32, device="cuda").view(seqs, width)
    lens = torch.full((seqs,), n, dtype=torch.int32, device="cuda")
    out, lse = paged_attention(q, cache, table, lens, cfg, return_lse=True)
    for s in (0, seqs - 1):
        at = slice(s * n, s * n + n)
        want, want_lse = paged_attention(q[at], cache, table[s:s + 1], lens[:1], cfg, return_lse=True)
        assert torch.equal(out[at], want) and torch.equal(lse[:, at], want_lse)


@pytest.mark.parametrize("dtype,d,block", [(FH, 64, 64), (BF, 128, 128)])
def test_chunks_of_several_slices(device, dtype, d, block):
    """A call whose partial rows take more than one slice of scratch, prompts from
    an empty cache and a chunk behind one, slices ending inside sequences: every
    sequence has the bits that it has by itself."""
    h, hk, ctx, new = 32, 2, [0, 100, 0], [9000, 700, 11000]
    cfg = MoBAConfig(block_size=block, top_k=4, dtype=dtype)
    assert sum(new) * h * 4 * d * 4 > 2 ** 29
    g = torch.Generator(device="cuda").manual_seed(32)
    lens = [c + n for c, n in zip(ctx, new)]
    counts = [-(-n // block) for n in lens]
    pages, width = sum(counts) + 1, max(counts)
    k, v = (torch.randn(pages, hk, block, d, generator=g, device="cuda").to(dtype) for _ in range(2))
    cache = PagedKV(k, v, k.float().mean(2).to(dtype))
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((3, width), -1, dtype=torch.int32, device="cuda")
    for s, n in enumerate(counts):
        table[s, :n] = order[sum(counts[:s]):sum(counts[:s]) + n]
    q = torch.randn(sum(new) + 5, h, d, generator=g, device="cuda").to(dtype)
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 5.0)
    _, lse = paged_attention(q, cache, table, seq_lens, cfg, cu_seqlens=cu_of(new).cuda(), out=out, return_lse=True)
    assert bool((out[sum(new):] == 5).all())
    at = 0
    for s, n in enumerate(new):
        part = slice(at, at + n)
        want, want_lse = paged_attention(q[part], cache, table[s:s + 1], seq_lens[s:s + 1], cfg, return_lse=True)
        assert torch.equal(out[part], want) and torch.equal(lse[:, part], want_lse), s
        # The last tokens again, in a call that has others in its slice.
        tail, tail_lse = paged_attention(q[at + n - 400:at + n], cache, table[s:s + 1], seq_lens[s:s + 1], cfg,
                                         return_lse=True)
        assert torch.equal(out[at + n - 400:at + n], tail) and torch.equal(lse[:, at + n - 400:at + n], tail_lse), s
        at += n

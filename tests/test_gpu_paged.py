"""The paged cache's operators against their definitions in 64 bits: appended
pages, routing (exact), attention; then a run of them together."""

import math

import pytest
import torch

from moba import paged as P
from moba.config import MoBAConfig
from moba.kernels.gating import gate_select
from moba.kernels.moba_fwd import moba_forward
from moba.kernels.paged import (PagedKV, append_tokens, copy_pages, paged_attention,
                                paged_gate_select)
from moba.kernels.pooling import pool_blocks
from moba.kernels.rotary import norm_rotate
from paged_util import (Paged, attend64, cu_of, forward_bound, half_step, norm_rotate64, pair_size, select64,
                        tables)

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def same(a, b):
    """Bit for bit, NaN included."""
    return torch.equal(a.cpu().contiguous().view(torch.uint8), b.cpu().contiguous().view(torch.uint8))


# -- append ---------------------------------------------------------------------

# contexts, new tokens, heads, kv heads, head_dim, block, dtype, rotary, neighbours, weights
APPENDS = [
    ([0], [1], 1, 1, 64, 16, BF, 64, False, F32),
    ([0, 15, 16, 17, 100, 5], [1, 1, 1, 1, 1, 0], 4, 2, 64, 16, BF, 64, False, F32),
    ([3, 0, 64, 127], [70, 200, 64, 1], 8, 2, 128, 64, BF, 64, True, BF),
    ([0, 31, 40], [33, 1, 130], 6, 3, 64, 48, FH, 32, False, FH),
    ([10, 130], [300, 129], 5, 1, 256, 128, F32, 256, False, F32),
    ([50] * 70, [1, 3] * 35, 2, 1, 64, 32, BF, 64, False, None),
    ([7, 0], [40, 20], 2, 2, 128, 16, BF, 0, False, F32),
    ([0], [1500], 4, 4, 64, 1024, BF, 64, False, F32),
]


def append_inputs(case, seed=0):
    ctx, new, h, hk, d, block, dt, rot, il, wd = case
    p = Paged([c + n for c, n in zip(ctx, new)], hk, block, d, dt, seed, tokens="none")
    for s, c in enumerate(ctx):
        p.put(s, p.randn(c, hk, d), p.randn(c, hk, d))
    x = p.randn(sum(new) + 2, h + 2 * hk, d)  # two rows of no sequence behind
    wq, wk = (None if wd is None else (1 + 0.2 * torch.randn(d, generator=p.g)).to(wd) for _ in range(2))
    cos, sin = tables(max(p.lens), rot) if rot else (None, None)
    return p, x, wq, wk, cos, sin


@pytest.mark.parametrize("case", APPENDS, ids=str)
def test_append(device, case):
    ctx, new, h, hk, d, block, dt, rot, il, wd = case
    p, x, wq, wk, cos, sin = append_inputs(case)
    cache, table, lens = p.gpu()
    xg = x.cuda()
    xg[-2:] = math.nan
    out = torch.full((x.shape[0], h, d), 7.0, dtype=dt, device="cuda")
    cuda = [None if t is None else t.cuda() for t in (cos, sin, wq, wk)]
    got = append_tokens(xg[:, :h], xg[:, h:h + hk], xg[:, h + hk:], cache, table, lens,
                        cu_seqlens=cu_of(new).cuda(), cos=cuda[0], sin=cuda[1], q_weight=cuda[2],
                        k_weight=cuda[3], interleaved=il, out=out)
    assert got is out and bool((out[-2:] == 7).all())
    at = 0
    for s, (c, n) in enumerate(zip(ctx, new)):
        pos = torch.arange(c, c + n)
        rows = x[at:at + n]
        for part, w, y in ((rows[:, :h], wq, out[at:at + n].cpu()), (rows[:, h:h + hk], wk, None)):
            w = None if w is None else w.double()
            ref = norm_rotate64(part.double(), w, cos, sin, pos, 1e-6, il)
            if y is None:  # keys, from where the table says they are
                page = p.table[s].long()[pos // block]
                y = cache.k.cpu()[page, :, pos % block]
            bound = forward_bound(ref, pair_size(part.double(), w, cos, 1e-6, il), dt)
            assert bool(((y.double() - ref).abs() <= bound).all())
        # What stands in the pages is what the plain form puts there.
        p.put(s, cache.k.cpu()[page, :, pos % block], rows[:, h + hk:], first=c)
        at += n
    for name in ("k", "v", "kbar"):
        assert same(getattr(cache, name), getattr(p, name)), name


def test_append_matches_norm_rotate_and_pool(device):
    """Bit for bit the training path's keys, queries and representatives."""
    g = torch.Generator().manual_seed(1)
    n, h, hk, d, block = 300, 4, 2, 128, 64
    x = torch.randn(n, h + 2 * hk, d, generator=g).to(BF).cuda()
    q, k, v = x[:, :h], x[:, h:h + hk], x[:, h + hk:]
    w = torch.rand(d, generator=g).cuda() + 0.5
    cos, sin = (t.cuda() for t in tables(n, d))
    cache = PagedKV.empty(5, hk, block, d)
    table = torch.tensor([[3, 0, 4, 1, 2]], dtype=torch.int32, device="cuda")
    done = 0
    for m in (1, 62, 2, 64, 100, 71):
        done += m
        lens = torch.tensor([done], dtype=torch.int32, device="cuda")
        part = slice(done - m, done)
        qa = append_tokens(q[part], k[part], v[part], cache, table, lens, cos=cos, sin=sin,
                           q_weight=w, k_weight=w)
        pos = torch.arange(done - m, done, device="cuda")
        assert torch.equal(qa, norm_rotate(q[part][None], k[part][None], cos, sin, positions=pos,
                                           q_weight=w, k_weight=w)[0][0])
    assert done == n
    kn = norm_rotate(q[None], k[None], cos, sin, q_weight=w, k_weight=w)[1]
    order = table[0].long()
    assert torch.equal(cache.k[order].transpose(1, 2).reshape(-1, hk, d)[:n], kn[0])
    assert torch.equal(cache.v[order].transpose(1, 2).reshape(-1, hk, d)[:n], v)
    want = pool_blocks(kn, MoBAConfig(block_size=block, top_k=4))
    assert torch.equal(cache.kbar[order[:4]].transpose(0, 1), want[0, :, :4])


def test_append_drops_what_has_no_place(device):
    """Tokens whose page is no page, and sequences whose numbers make no sense."""
    p = Paged([40, 20, 20, 5], 1, 16, 64, BF, 0, tokens="none")
    p.table[0, 1] = -3
    p.table[1, 0] = p.k.shape[0]
    cache, table, _ = p.gpu()
    before = [t.clone() for t in (cache.k, cache.v, cache.kbar)]
    lens = torch.tensor([40, 20, 3, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    x = p.randn(90, 1, 64).cuda()
    out = torch.full_like(x, 3.0)
    cu = torch.tensor([0, 40, 60, 80, 85], dtype=torch.int32, device="cuda")  # 20 new of 3: nonsense
    append_tokens(x, x, x, cache, table, lens, cu_seqlens=cu, out=out)
    assert torch.equal(out[:60], x[:60]) and bool((out[60:80] == 3).all()) and bool((out[85:] == 3).all())
    for s, c, n, first in ((0, 0, 40, 0), (1, 0, 20, 40)):
        p.put(s, x[first:first + n].cpu(), x[first:first + n].cpu())
    assert same(cache.k, p.k) and same(cache.v, p.v) and same(cache.kbar, p.kbar)
    # Bounds that fall or leave the token axis.
    cache2 = PagedKV(*before)
    for bad in ([0, -5, 60, 80, 85], [0, 40, 30, 95, 96], [5, 4, 3, 2, 1]):
        cu = torch.tensor(bad, dtype=torch.int32, device="cuda")
        append_tokens(x, x, x, cache2, table, torch.full_like(lens, 1000), cu_seqlens=cu)
    torch.cuda.synchronize()


# -- attention --------------------------------------------------------------------

def cfg_of(block, top_k, **more):
    return MoBAConfig(block_size=block, top_k=top_k, **more)


# contexts, new tokens, heads, kv heads, head_dim, dtype, config
ATTENDS = [
    ([0], [1], 1, 1, 64, BF, cfg_of(16, 3)),
    ([0, 15, 16, 17, 700, 5, 400], [1, 1, 1, 1, 1, 0, 1], 4, 2, 64, BF, cfg_of(16, 4)),
    ([300, 0, 63, 64, 1000], [1, 40, 1, 64, 5], 8, 2, 128, BF, cfg_of(64, 4)),
    ([300, 0, 63, 64, 1000], [70, 40, 1, 64, 33], 8, 2, 128, FH, cfg_of(32, 8)),
    ([2000], [100], 4, 4, 64, BF, cfg_of(128, 3)),
    ([0], [300], 4, 1, 64, FH, cfg_of(64, 2)),
    ([129, 500], [64, 1], 6, 3, 64, FH, cfg_of(48, 5)),
    ([900, 3], [20, 9], 4, 2, 256, BF, cfg_of(64, 3)),
    ([900, 3], [20, 9], 4, 2, 64, F32, cfg_of(64, 3)),
    ([600, 1], [3, 9], 8, 1, 128, F32, cfg_of(80, 4)),
    ([500], [17], 3, 1, 256, F32, cfg_of(32, 6)),
    ([1500, 200], [2, 1], 4, 2, 64, BF, cfg_of(16, 33)),
    ([1500, 200], [2, 40], 4, 2, 64, BF, cfg_of(16, 17)),
    ([700, 2], [20, 5], 4, 2, 64, BF, cfg_of(32, 1)),
    ([700, 2], [20, 40], 4, 2, 64, BF, cfg_of(32, 3, always_select_current=False)),
    ([700, 2], [20, 40], 4, 2, 128, BF, cfg_of(32, 3, top_k_includes_current=False)),
    ([100] * 40 + [17], [1] * 40 + [130], 16, 2, 64, BF, cfg_of(32, 4)),
    ([50, 90] * 40, [1, 2] * 40, 2, 1, 64, BF, cfg_of(16, 3)),
    ([3000, 1023], [1, 9], 4, 2, 64, BF, cfg_of(1024, 3)),
    ([2100], [3], 2, 1, 256, F32, cfg_of(1024, 2)),
]


def check_attention(p, new, q, cfg, tail=2, tokens=None):
    """Routing exact, outputs and lse within the bound, rows of no sequence untouched;
    of all new tokens or those of a set."""
    cache, table, lens = p.gpu()
    cu = cu_of(new).cuda()
    qg = torch.cat((q, torch.full((tail, *q.shape[1:]), math.nan, dtype=q.dtype))).cuda()
    ids = paged_gate_select(qg, cache, table, lens, cfg, cu_seqlens=cu).cpu()
    out = torch.full_like(qg, 5.0)
    got, lse = paged_attention(qg, cache, table, lens, cfg, cu_seqlens=cu, out=out, return_lse=True)
    assert got is out and bool((out[len(q):] == 5).all()) and bool((ids[len(q):] == -1).all())
    out, lse = out.cpu().double(), lse.cpu().double()
    at = 0
    for s, n in enumerate(new):
        for i in range(n):
            if tokens is not None and at not in tokens:
                at += 1
                continue
            pos = p.lens[s] - n + i
            want = select64(p, s, q[at], pos, cfg)
            for h, w in enumerate(want):
                assert ids[at, h].tolist() == w + [-1] * (ids.shape[2] - len(w)), (s, i, h)
            ref, ref_lse, bound = attend64(p, s, q[at], pos, want)
            far = (out[at] - ref).abs()
            assert bool((far <= bound).all()), (s, i, (far - bound).max().item())
            # A lse is off by what every score may be, and by its own rounding.
            near = (lse[:, at] - ref_lse).abs() <= 1e-4 + 2.0 ** -7 * (p.dtype != F32)
            assert bool((near | (lse[:, at] == ref_lse)).all())
            at += 1
    return ids


@pytest.mark.parametrize("case", ATTENDS, ids=str)
def test_attention(device, case):
    ctx, new, h, hk, d, dt, cfg = case
    p = Paged([c + n for c, n in zip(ctx, new)], hk, cfg.block_size, d, dt, 3,
              width=max(-(-(c + n) // cfg.block_size) for c, n in zip(ctx, new)) + 2)
    q = p.randn(sum(new), h, d)
    check_attention(p, new, q, cfg)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_wide_table(device, dtype):
    """The widest table: its entries past the sequences' blocks do not count."""
    cfg = cfg_of(16, 3)
    p = Paged([270, 20], 2, 16, 64, dtype, 17, width=1 << 16)
    check_attention(p, [70, 1], p.randn(71, 4, 64), cfg)


# Chunks that go tile by tile and block by block: the same.
CHUNKS = [
    ([1000, 0, 333], [400, 100, 61], 8, 2, 128, BF, cfg_of(128, 4)),
    ([1500], [300], 16, 4, 128, FH, cfg_of(64, 9)),
    ([2000, 64, 7], [200, 64, 130], 16, 2, 64, FH, cfg_of(32, 17)),
    ([300, 2500], [600, 40], 8, 8, 64, BF, cfg_of(96, 6)),
    ([700, 70], [300, 250], 12, 4, 64, BF, cfg_of(128, 3, always_select_current=False)),
    ([400, 200, 9], [500, 0, 77], 10, 2, 128, BF, cfg_of(100, 3, top_k_includes_current=False)),
    ([900, 3], [300, 300], 8, 1, 256, BF, cfg_of(64, 3)),
    ([1500], [400], 16, 4, 64, BF, cfg_of(16, 33)),
    ([1100], [129], 128, 1, 128, FH, cfg_of(128, 2)),
]


def edges(p, new, n=24):
    """First, last and some tokens of every chunk."""
    out, at = set(), 0
    for k in new:
        out |= {at, at + k - 1} | {at + int(i) for i in torch.randint(0, k, (n,), generator=p.g)} if k else set()
        at += k
    return out


def row_by_row(p, new, q, cfg):
    """The chunk's tokens as many short calls, which take the single-token kernels."""
    cache, table, _ = p.gpu()
    ids, out, at = [], [], 0
    for s, n in enumerate(new):
        for i in range(0, n, 3):
            m = min(3, n - i)
            lens = torch.tensor([p.lens[s] - n + i + m], dtype=torch.int32, device="cuda")
            part = q[at + i:at + i + m].cuda()
            ids.append(paged_gate_select(part, cache, table[s:s + 1], lens, cfg))
            out.append(paged_attention(part, cache, table[s:s + 1], lens, cfg))
        at += n
    return torch.cat(ids), torch.cat(out)


def check_chunk(p, new, q, cfg, finite=True):
    """Some tokens against 64 bits (where values are finite), all of them against
    the single-token kernels."""
    if finite:
        check_attention(p, new, q, cfg, tokens=edges(p, new))
    cache, table, lens = p.gpu()
    cu = cu_of(new).cuda()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    out = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    given = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu, block_idx=ids)
    assert bool(((given == out) | (given.isnan() & out.isnan())).all())
    want_ids, want = row_by_row(p, new, q, cfg)
    assert torch.equal(ids, want_ids)
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isposinf(), want.isposinf())
    assert torch.equal(out.isneginf(), want.isneginf())
    # Both round their result, block by block the weights too: half a step of
    # the weighted mean of |v| each; codes and float32 sums are below 2^-14 of it.
    most = p.v[p.v.isfinite()].abs().max().double()
    far = torch.where(out.isfinite(), out.double() - want.double(), 0.0).abs().max()
    assert far <= (3 * half_step(p.dtype) + 2.0 ** -13) * most


@pytest.mark.parametrize("case", CHUNKS, ids=str)
def test_chunks(device, case):
    ctx, new, h, hk, d, dt, cfg = case
    p = Paged([c + n for c, n in zip(ctx, new)], hk, cfg.block_size, d, dt, 13,
              width=max(-(-(c + n) // cfg.block_size) for c, n in zip(ctx, new)) + 2)
    check_chunk(p, new, p.randn(sum(new), h, d), cfg)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("size", [2.0 ** -12, 1.0, 2.0 ** 6])
def test_chunks_of_correlated_keys(device, dtype, size):
    """Representatives that drift from block to block and lie far from zero:
    neighbours score nearly alike, and many scores round to the same value."""
    cfg = cfg_of(16, 12)
    p = Paged([4000], 2, 16, 64, dtype, 14)
    drift = torch.randn(p.kbar.shape[0], 2, 64, generator=p.g).cumsum(0) * 0.05 + 3
    p.kbar[p.table[0, :250].long()] = (drift[:250] * size).to(dtype)
    check_chunk(p, [300], p.randn(300, 16, 64) + 1, cfg)


@pytest.mark.parametrize("dtype", [BF, FH])
def test_chunks_without_pages(device, dtype):
    cfg = cfg_of(128, 3)
    new = [300, 1, 150]
    p = Paged([1200, 1, 500], 2, 128, 128, dtype, 15)
    p.table[0, 2], p.table[0, 5], p.table[0, 8] = -1, p.k.shape[0], 2 ** 31 - 1
    p.table[1, 0] = -2
    p.table[2, :4] = -1
    check_chunk(p, new, p.randn(451, 12, 128), cfg)


@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("d,block", [(128, 128), (64, 96)])
def test_chunks_with_special_values(device, dtype, d, block):
    """Infinities and NaN, in values that all, some and none of the queries
    see; a value of each where every query sees it; large values."""
    cfg = cfg_of(block, 3)
    n = 300
    p = Paged([1000], 2, block, d, dtype, 16)
    q = p.randn(n, 32, d)
    p.v[p.v.isfinite()] *= 100
    for row, feature, value in ((999, 3, math.nan), (998, 5, math.inf), (900, 7, -math.inf), (800, 9, math.nan),
                                (650, d - 1, math.inf), (20, 0, -math.inf), (21, 0, math.inf), (5, 2, math.inf)):
        p.v[p.table[0, row // block], :, row % block, feature] = value
    check_chunk(p, [n], q, cfg, finite=False)


def test_replays_of_a_chunk(device):
    """A captured chunk call replayed on other lengths, pages and queries, eager
    calls and a second captured call between the replays."""
    cfg = cfg_of(128, 4)
    p = Paged([2000, 900], 2, 128, 128, BF, 18)
    cache, table, lens = p.gpu()
    q, cu = p.randn(400, 12, 128).cuda(), cu_of([250, 150]).cuda()
    tables = [table, table.flip(1).contiguous(), table.roll(1, 1).contiguous(), table]
    lengths = [lens, lens - 640, torch.tensor([260, 150], dtype=torch.int32, device="cuda"), lens]
    cache.kbar.nan_to_num_(0.0)
    cache.k.nan_to_num_(0.0)
    cache.v.nan_to_num_(0.0)

    def run(q, table, lens):
        return paged_attention(q, cache, table, lens, cfg, cu_seqlens=cu, return_lse=True)

    static = [t.clone() for t in (q, table, lens)]
    run(*static)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                outs.append(run(*static))
            graphs.append(g)
    torch.cuda.synchronize()
    for i, (t, n) in enumerate(zip(tables, lengths)):
        x = q.roll(i, 0)
        want = run(x, t, n)
        for buf, value in zip(static, (x, t, n)):
            buf.copy_(value)
        for g, (out, lse) in zip(graphs, outs):
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want[0]) and torch.equal(lse, want[1]), i
            assert torch.equal(run(x, t, n)[0], want[0])


def test_two_chunks_at_once(device):
    cfg = cfg_of(128, 4)
    p = Paged([1500], 2, 128, 128, FH, 19)
    cache, table, lens = p.gpu()
    qs = [p.randn(400, 12, 128).cuda() for _ in range(2)]
    want = [paged_attention(q, cache, table, lens, cfg) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(paged_attention(qs[i], cache, table, lens, cfg))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_result_over_the_queries(device):
    """`out` may be `q`: rows, split rows and chunks."""
    for n, cfg in ((1, cfg_of(128, 9)), (400, cfg_of(128, 4))):
        p = Paged([2500], 2, 128, 128, BF, 20)
        cache, table, lens = p.gpu()
        q = p.randn(n, 12, 128).cuda()
        want = paged_attention(q, cache, table, lens, cfg)
        assert torch.equal(paged_attention(q, cache, table, lens, cfg, out=q), want)


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("new", [[1, 1], [40, 33], [300, 290]])
def test_ties_and_special_scores(device, dtype, new):
    """Integer-valued queries and keys (equal scores everywhere), and
    representatives with infinities and NaN."""
    cfg = cfg_of(16, 4)
    p = Paged([300 + new[0], 200 + new[1]], 2, 16, 64, dtype, 5)
    q = torch.randint(-1, 2, (sum(new), 8, 64), generator=p.g).to(dtype)
    tokens = edges(p, new) if sum(new) > 100 else None
    p.kbar[:] = torch.randint(-1, 2, p.kbar.shape, generator=p.g).to(dtype)
    check_attention(p, new, q, cfg, tokens=tokens)
    p.kbar[p.table[0, 3], :, 5], p.kbar[p.table[0, 7], :, 5] = math.inf, -math.inf
    p.kbar[p.table[1, 2], :, 9], p.kbar[p.table[1, 4]] = math.nan, 0.0
    check_attention(p, new, q, cfg, tokens=tokens)
    p.kbar[:] = torch.randn(p.kbar.shape, generator=p.g).to(dtype) * 2.0 ** -100 if dtype != FH else \
        torch.randn(p.kbar.shape, generator=p.g).to(dtype) * 2.0 ** -20
    check_attention(p, new, q, cfg, tokens=tokens)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [40, 1, 70]])
def test_missing_pages(device, dtype, new):
    """Blocks without a page are never chosen; a query whose own block has
    none and that has no other sees nothing."""
    cfg = cfg_of(16, 3)
    p = Paged([200 + new[0], new[1], 60 + new[2]], 2, 16, 64, dtype, 6)
    p.table[0, 2], p.table[0, 5], p.table[0, 12] = -1, p.k.shape[0], 2 ** 31 - 1
    p.table[1, 0] = -2
    p.table[2, :3] = -1
    check_attention(p, new, p.randn(sum(new), 4, 64), cfg)


def test_shared_pages_and_even_chunks(device):
    """Two sequences on the same prefix pages; no cu_seqlens."""
    cfg = cfg_of(32, 3)
    p = Paged([100, 100, 100], 1, 32, 64, BF, 7)
    p.table[1, :3] = p.table[0, :3]
    q = p.randn(9, 2, 64)
    check_attention(p, [3, 3, 3], q, cfg)
    cache, table, lens = p.gpu()
    a = paged_attention(q.cuda(), cache, table, lens, cfg)
    b = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu_of([3, 3, 3]).cuda())
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("n", [1, 64, 200])
def test_hidden_values_do_not_reach_a_query(device, dtype, n):
    """Infinities and NaN in keys and values of later tokens of the same block:
    the outputs of earlier tokens keep every bit."""
    cfg = cfg_of(64, 2)
    p = Paged([500], 2, 64, 64, dtype, 8)
    q = p.randn(n, 4, 64)
    cu = cu_of([n]).cuda()

    def run():
        cache, table, lens = p.gpu()
        return paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)

    want = run()
    last = 499
    for row, value in ((last, math.nan), (last - 1, math.inf), (last - 3, -math.inf)):
        page = p.table[0, row // 64]
        p.v[page, :, row % 64, ::3] = value
        p.k[page, :, row % 64, ::5] = value
    got = run()
    clean = max(0, n - 4)
    assert torch.equal(got[:clean], want[:clean])
    if n > 1:
        assert bool(got[-1].isnan().any())


def test_values_of_padding_are_not_read(device):
    """seq_lens and cu_seqlens that make no sense: no rows are touched."""
    cfg = cfg_of(16, 3)
    p = Paged([40, 40], 1, 16, 64, BF, 9)
    cache, table, _ = p.gpu()
    q = p.randn(20, 2, 64).cuda()
    for lens, cu in (([5, 40], [0, 10, 20]), ([40, 2 ** 31 - 1], [0, 10, 20]), ([40, 40], [0, -3, 25]),
                     ([-4, 40], [0, 10, 5]), ([40, 40], [30, 20, 10])):
        out = torch.full_like(q, 2.0)
        paged_attention(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), cfg,
                        cu_seqlens=torch.tensor(cu, dtype=torch.int32, device="cuda"), out=out)
        torch.cuda.synchronize()
        if lens[0] < 10:
            assert bool((out[:10] == 2).all())
    # A length far behind the table: no page there, nothing but chosen past blocks.
    assert bool(out.isfinite().all())


def test_given_blocks(device):
    """block_idx instead of the gate's choice, out-of-range ids included."""
    cfg = cfg_of(16, 3)
    p = Paged([100, 70], 2, 16, 64, BF, 10)
    new = [20, 1]
    q = p.randn(21, 4, 64)
    cache, table, lens = p.gpu()
    cu = cu_of(new).cuda()
    ids = paged_gate_select(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    want = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu)
    assert torch.equal(paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu, block_idx=ids), want)
    odd = torch.cat((ids, torch.tensor([1000, -9, 2 ** 31 - 1], device="cuda", dtype=torch.int32)
                     .expand(21, 4, 3)), -1)
    got = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu, block_idx=odd)
    assert bool((got.double() - want.double()).abs().max() <= 2 ** -7 * want.double().abs().max())
    none, lse = paged_attention(q.cuda(), cache, table, lens, cfg, cu_seqlens=cu,
                                block_idx=torch.full_like(ids, -1), return_lse=True)
    assert bool((none == 0).all()) and bool((lse == -math.inf).all())


def test_no_tokens(device):
    p = Paged([10], 1, 16, 64, BF, 11)
    cache, table, lens = p.gpu()
    q = torch.zeros(0, 2, 64, dtype=BF, device="cuda")
    cu = cu_of([0]).cuda()
    assert paged_attention(q, cache, table, lens, cfg_of(16, 3), cu_seqlens=cu).shape == q.shape
    assert paged_gate_select(q, cache, table, lens, cfg_of(16, 3), cu_seqlens=cu).shape == (0, 2, 2)
    k = torch.zeros(0, 1, 64, dtype=BF, device="cuda")
    assert append_tokens(q, k, k, cache, table, lens, cu_seqlens=cu).shape == q.shape


@pytest.mark.parametrize("dtype,d,block,top_k", [(BF, 64, 128, 8), (BF, 128, 64, 4), (FH, 64, 32, 12),
                                                 (F32, 64, 64, 4)])
def test_matches_whole_sequences(device, dtype, d, block, top_k):
    """A prompt in chunks and single tokens: the routing of gate_select, and
    moba_forward's results within two roundings each side."""
    n, h, hk = 1500, 4, 2
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn(1, n, m, d, generator=g).to(dtype).cuda() for m in (h, hk, hk))
    k += torch.randn(1, 1, hk, d, generator=g).to(dtype).cuda()
    cfg = MoBAConfig(block_size=block, top_k=top_k, dtype=dtype)
    want = moba_forward(q, k, v, cfg)
    ids = gate_select(q, pool_blocks(k, cfg), cfg)
    cache = PagedKV.empty(-(-n // block) + 1, hk, block, d, dtype)
    table = torch.randperm(-(-n // block) + 1, generator=g).to(torch.int32).cuda()[None].contiguous()
    done = 0
    for m in (1, 700, 1, 1, 300, 64, 400, 33):
        part = slice(done, done + m)
        done += m
        lens = torch.tensor([done], dtype=torch.int32, device="cuda")
        qa = append_tokens(q[0, part], k[0, part], v[0, part], cache, table, lens)
        got_ids = paged_gate_select(qa, cache, table, lens, cfg)
        assert torch.equal(got_ids.transpose(0, 1), ids[0, :, part, :got_ids.shape[2]])
        out = paged_attention(qa, cache, table, lens, cfg)
        # Both sides: weights, block results and outputs rounded, half a step
        # of max |v| each; float32: the bar of the float32 path on each side.
        far = (out.double() - want[0, part].double()).abs().max().item()
        bar = 2e-5 if dtype == F32 else 6 * torch.finfo(dtype).eps / 2 * v.abs().max().item()
        assert far <= bar
    assert done == n


# -- pages ----------------------------------------------------------------------

@pytest.mark.parametrize("layers,pages,h_kv,block,d,dtype,n", [
    (None, 3, 1, 16, 64, BF, 1), (3, 9, 2, 48, 64, FH, 4), (2, 700, 1, 16, 64, F32, 300),
    (5, 40, 8, 128, 128, BF, 20)])
@pytest.mark.parametrize("where", ["list", "host", "device"])
def test_copy_pages(device, layers, pages, h_kv, block, d, dtype, n, where):
    g = torch.Generator().manual_seed(13)
    lead = (pages,) if layers is None else (layers, pages)
    k, v = (torch.randn(*lead, h_kv, block, d, generator=g).to(dtype).cuda() for _ in range(2))
    cache = PagedKV(k, v, torch.randn(*lead, h_kv, d, generator=g).to(dtype).cuda())
    k.view(-1)[::7] = math.nan
    perm = torch.randperm(pages, generator=g).to(torch.int32)
    src, dst = perm[:n].clone(), perm[n:2 * n].clone()
    if n > 1:
        src[1] = src[0]  # one page to two places
    want = [t.clone() for t in (cache.k, cache.v, cache.kbar)]
    for t in want:
        at = t if layers is None else t.transpose(0, 1)
        at[dst.long().cuda()] = at[src.long().cuda()]
    args = (src.tolist(), dst.tolist()) if where == "list" else (src, dst) if where == "host" else \
        (src.cuda(), dst.cuda())
    copy_pages(cache, *args)
    for got, w in zip((cache.k, cache.v, cache.kbar), want):
        assert same(got, w)
    if where == "device":  # pairs outside the cache are skipped
        copy_pages(cache, torch.tensor([0, -1, pages], dtype=torch.int32, device="cuda"),
                   torch.tensor([pages, 1, 1], dtype=torch.int32, device="cuda"))
        assert same(cache.k, want[0])
    copy_pages(cache, [], [])


# -- together -------------------------------------------------------------------

def test_serving_run(device):
    """Prompts, a fork, decoding, an ended sequence, compaction: every token's
    output is that of its whole sequence."""
    cfg = MoBAConfig(block_size=32, top_k=3)
    h, hk, d, layers = 4, 2, 64, 2
    g = torch.Generator().manual_seed(14)
    cache = P.PagedCache(layers, 40, hk, d, cfg)
    for t in (cache.kv.k, cache.kv.v, cache.kv.kbar):
        t.fill_(math.nan)
    w = [1 + 0.1 * torch.randn(d, generator=g).cuda() for _ in range(2)]
    cos, sin = (t.cuda() for t in tables(2000, d))
    history = {}  # sequence: rows of x per layer
    results = {}

    def step(seqs, new):
        x = torch.randn(layers, sum(new), h + 2 * hk, d, generator=g).to(BF).cuda()
        st = cache.grow(seqs, new)
        outs = []
        for i in range(layers):
            kv = cache.kv.layer(i)
            q = append_tokens(x[i, :, :h], x[i, :, h:h + hk], x[i, :, h + hk:], kv, *st.args,
                              cos=cos, sin=sin, q_weight=w[0], k_weight=w[1])
            outs.append(paged_attention(q, kv, st.block_table, st.seq_lens, cfg, st.cu_seqlens))
        at = 0
        for s, n in zip(seqs, new):
            history.setdefault(s, []).append(x[:, at:at + n])
            results.setdefault(s, []).append(torch.stack(outs)[:, at:at + n])
            at += n

    a, b = cache.create(), cache.create()
    step([a, b], [100, 333])
    step([a, b], [1, 1])
    c = cache.fork(b)
    history[c], results[c] = list(history[b]), list(results[b])
    for _ in range(3):
        step([a, b, c], [1, 1, 1])
    cache.free(a)
    assert cache.compact() > 0
    e = cache.create()
    step([b, e, c], [40, 70, 1])
    for _ in range(30):
        step([c, e, b], [1, 1, 1])
    for s in (a, b, c, e):
        x, got = torch.cat(history[s], 1), torch.cat(results[s], 1)
        for i in range(layers):
            q, k = norm_rotate(x[i, None, :, :h], x[i, None, :, h:h + hk], cos, sin, q_weight=w[0],
                               k_weight=w[1])
            v = x[i, None, :, h + hk:]
            want = moba_forward(q, k, v.contiguous(), cfg)[0]
            far = (got[i].double() - want.double()).abs().max().item()
            assert far <= 6 * 2.0 ** -8 * v.abs().max().item(), (s, i, far)


def decode_state(seed=15, n=6):
    cfg = MoBAConfig(block_size=16, top_k=3)
    p = Paged([30 + 17 * i for i in range(n)], 2, 16, 64, BF, seed)
    return cfg, p


def test_replays_of_a_decoding_step(device):
    """append + attention captured once, replayed as the sequences grow across
    block boundaries, a padded sequence among them; eager calls in between.
    A second graph of the same shapes runs beside it."""
    cfg, p = decode_state()
    n = len(p.lens)
    cos, sin = (t.cuda() for t in tables(400, 64))
    w = torch.rand(64, generator=p.g).cuda() + 0.5
    width = 16
    pages = n * width
    table = torch.randperm(pages, generator=p.g).view(n, width).to(torch.int32).cuda()
    table[-1] = -1  # padding of the batch
    caches = [PagedKV.empty(pages, 2, 16, 64) for _ in range(3)]
    for c in caches:
        for t in (c.k, c.v, c.kbar):
            t.zero_()
    lens = torch.tensor(p.lens, dtype=torch.int32, device="cuda")
    x = p.randn(n, 8, 64).cuda()

    def step(cache):
        q = append_tokens(x[:, :4], x[:, 4:6], x[:, 6:], cache, table, lens, cos=cos, sin=sin,
                          q_weight=w, k_weight=w)
        return paged_attention(q, cache, table, lens, cfg)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[2])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for c in caches[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(c))
        graphs.append(graph)
    for c in caches:
        for t in (c.k, c.v, c.kbar):
            t.zero_()
    streams = [torch.cuda.Stream() for _ in graphs]
    for i in range(40):
        x.copy_(p.randn(n, 8, 64))
        lens += 1
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):  # both at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        want = step(caches[2])
        torch.cuda.synchronize()
        for c, out in zip(caches, outs):
            assert same(out, want), i
            assert same(c.k, caches[2].k) and same(c.kbar, caches[2].kbar), i


def test_on_another_stream(device):
    cfg, p = decode_state(16)
    cache, table, lens = p.gpu()
    q = p.randn(len(p.lens), 4, 64).cuda()
    want = paged_attention(q, cache, table, lens, cfg)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = paged_attention(q, cache, table, lens, cfg)
    side.synchronize()
    assert torch.equal(got, want)

"""norm_rotate against its definition in 64 bits: values, gradients, layouts,
captured replays."""

import math

import pytest
import torch

from moba.kernels.rotary import norm_rotate
from paged_util import U24, forward_bound, half_step, norm_rotate64, pair_size, tables

pytestmark = pytest.mark.gpu

BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-6

# batch, seq, heads, kv heads, head_dim, rotary (0: none), neighbours, dtype, weights
CASES = [
    (1, 1, 1, 1, 64, 64, False, BF, F32),
    (2, 37, 4, 2, 64, 64, False, BF, F32),
    (2, 37, 4, 2, 64, 16, True, FH, FH),
    (1, 130, 8, 8, 128, 128, True, BF, BF),
    (3, 5, 16, 2, 128, 32, False, F32, F32),
    (1, 67, 5, 1, 256, 256, False, FH, F32),
    (1, 33, 6, 3, 512, 128, False, BF, F32),
    (1, 9, 2, 1, 1024, 1024, True, BF, F32),
    (2, 19, 3, 1, 32, 32, False, F32, F32),
    (1, 41, 4, 4, 128, 128, False, BF, None),
    (1, 41, 4, 2, 128, 0, False, BF, F32),
    (2, 2500, 7, 3, 64, 64, False, BF, F32),  # more than 2^15 rows: four to a lane group
]


def inputs(case, seed=0):
    b, s, h, hk, d, rot, il, dt, wd = case
    g = torch.Generator().manual_seed(seed)
    q, k = (torch.randn(b, s, n, d, generator=g).to(dt) for n in (h, hk))
    gq, gk = (torch.randn(b, s, n, d, generator=g).to(dt) for n in (h, hk))
    wq, wk = (None if wd is None else (1 + 0.2 * torch.randn(d, generator=g)).to(wd) for _ in range(2))
    cos, sin = tables(s + 50, rot) if rot else (None, None)
    pos = torch.randint(0, s + 50, (b, s), generator=g)
    return q, k, gq, gk, wq, wk, cos, sin, pos


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@pytest.mark.parametrize("case", CASES, ids=str)
def test_values(device, case):
    q, k, _, _, wq, wk, cos, sin, pos = inputs(case)
    il, dt = case[6], case[7]
    got = norm_rotate(*cuda(q, k, cos, sin), positions=pos.cuda(), q_weight=cuda(wq)[0],
                      k_weight=cuda(wk)[0], eps=EPS, interleaved=il)
    for x, w, y in ((q, wq, got[0]), (k, wk, got[1])):
        w = None if w is None else w.double()
        ref = norm_rotate64(x.double(), w, cos, sin, pos, EPS, il)
        size = pair_size(x.double(), w, cos, EPS, il)
        assert y.dtype == dt and y.is_contiguous()
        assert bool(((y.cpu().double() - ref).abs() <= forward_bound(ref, size, dt)).all())


@pytest.mark.parametrize("case", CASES, ids=str)
def test_gradients(device, case):
    q, k, gq, gk, wq, wk, cos, sin, pos = inputs(case, 1)
    il, dt, d = case[6], case[7], case[4]
    leaves = [None if t is None else t.cuda().requires_grad_() for t in (q, k, wq, wk)]
    out = norm_rotate(leaves[0], leaves[1], *cuda(cos, sin), positions=pos.cuda(),
                      q_weight=leaves[2], k_weight=leaves[3], eps=EPS, interleaved=il)
    torch.autograd.backward(out, cuda(gq, gk))
    for x, w, g, lx, lw in ((q, wq, gq, leaves[0], leaves[2]), (k, wk, gk, leaves[1], leaves[3])):
        x64 = x.double().requires_grad_()
        w64 = None if w is None else w.double().requires_grad_()
        norm_rotate64(x64, w64, cos, sin, pos, EPS, il).backward(g.double())
        # The turned gradient's rounding goes by its pair; then the norm's row:
        # h and the mean of |h x r| times x r, each times r. At most 64 roundings.
        with torch.no_grad():
            size = pair_size(g.double(), None, cos, EPS, il)
            if w is None:
                scale = size
            else:
                r = 1 / torch.sqrt((x64 * x64).mean(-1, keepdim=True) + EPS)
                xr = (x64 * r).abs()
                h = size * w.double().abs()
                scale = r * (h + xr * (h * xr).mean(-1, keepdim=True))
            bound = half_step(dt) * x64.grad.abs() + 64 * U24 * scale + \
                (2.0 ** -25 if dt == FH else 0)
            assert bool(((lx.grad.cpu().double() - x64.grad).abs() <= bound).all())
            if w is not None:
                # Up to 2^7 rows in a lane and 16 sums after it.
                total = (size * xr).flatten(0, -2).sum(0)
                bound = half_step(w.dtype) * w64.grad.abs() + (128 + 64) * U24 * total
                assert lw.grad.dtype == w.dtype
                assert bool(((lw.grad.cpu().double() - w64.grad).abs() <= bound).all())


def test_gradients_against_differences(device):
    """Directional derivatives of the 64-bit forward, step 1e-5 (truncation
    below 1e-9 of the third derivative), against the kernel's gradients."""
    case = (1, 6, 3, 2, 64, 32, False, F32, F32)
    q, k, gq, gk, wq, wk, cos, sin, pos = inputs(case, 2)
    leaves = [t.cuda().requires_grad_() for t in (q, k, wq, wk)]
    out = norm_rotate(leaves[0], leaves[1], *cuda(cos, sin), positions=pos.cuda(),
                      q_weight=leaves[2], k_weight=leaves[3], eps=EPS)
    grads = [t.cpu().double() for t in torch.autograd.grad(out, leaves, cuda(gq, gk))]

    def value(ts):
        return sum((norm_rotate64(x, w, cos, sin, pos, EPS, False) * g.double()).sum()
                   for x, w, g in ((ts[0], ts[2], gq), (ts[1], ts[3], gk)))

    base = [t.double() for t in (q, k, wq, wk)]
    gen = torch.Generator().manual_seed(3)
    for i in range(4):
        u = torch.randn(base[i].shape, generator=gen).double()
        plus, minus = list(base), list(base)
        plus[i], minus[i] = base[i] + 1e-5 * u, base[i] - 1e-5 * u
        diff = ((value(plus) - value(minus)) / 2e-5).item()
        # 192 roundings of every gradient element at most; elements are O(10).
        slack = 256 * U24 * (grads[i].abs() * u.abs()).sum().item() + 256 * U24 * 10 * u.abs().sum().item()
        assert abs((grads[i] * u).sum().item() - diff) <= slack + 1e-5


@pytest.mark.parametrize("dtype", [BF, F32])
def test_layouts_agree(device, dtype):
    """Views of a fused projection, transposed and broadcast inputs, odd
    offsets, an expanded gradient: the results of contiguous tensors."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 21, 8, 64, generator=g).to(dtype).cuda()
    cos, sin = cuda(*tables(21, 64))
    w = torch.rand(64, generator=g).cuda() + 0.5

    def run(q, k):
        q, k = q.detach().requires_grad_(), k.detach().requires_grad_()
        out = norm_rotate(q, k, cos, sin, q_weight=w, k_weight=w)
        grads = torch.autograd.grad([o.float().sum() for o in out], (q, k))
        return [*out, *grads]

    def check(q, k):
        want = run(q.contiguous(), k.contiguous())
        for a, b in zip(run(q, k), want):
            assert torch.equal(a, b)

    check(x[:, :, :6], x[:, :, 6:])
    t = x.transpose(1, 2).contiguous().transpose(1, 2)
    check(t[:, :, :6], t[:, :, 6:])
    check(x[:1, :, :6].expand(2, -1, -1, -1), x[:, :1, 6:].expand(-1, 21, -1, -1))
    flat = torch.randn(2 * 21 * 8 * 64 + 1, generator=g).to(dtype).cuda()[1:].view(2, 21, 8, 64)
    check(flat[:, :, :6], flat[:, :, 6:])
    wide = torch.randn(2, 21, 8, 67, generator=g).to(dtype).cuda()[..., 2:66]
    check(wide[:, :, :6], wide[:, :, 6:])


def test_positions(device):
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(2, 9, 2, 64, generator=g).to(BF).cuda(), torch.randn(2, 9, 1, 64, generator=g).to(BF).cuda()
    cos, sin = cuda(*tables(20, 64))
    plain = norm_rotate(q, k, cos, sin)
    for pos in (torch.arange(9), torch.arange(9).expand(2, 9), torch.arange(9, dtype=torch.int32)):
        for a, b in zip(norm_rotate(q, k, cos, sin, positions=pos.cuda()), plain):
            assert torch.equal(a, b)
    # Outside the tables: NaN in the rotated part, the rest as it is.
    half = [t[:, :16].contiguous() for t in (cos, sin)]
    pos = torch.arange(9).expand(2, 9).clone()
    pos[0, 3], pos[1, 0] = 20, -1
    out, ok = norm_rotate(q, k, *half, positions=pos.cuda())[0], norm_rotate(q, k, *half)[0]
    bad = torch.zeros(2, 9, dtype=torch.bool)
    bad[0, 3] = bad[1, 0] = True
    assert bool(out[bad.cuda()][..., :32].isnan().all())
    assert torch.equal(out[bad.cuda()][..., 32:], ok[bad.cuda()][..., 32:])
    assert torch.equal(out[~bad.cuda()], ok[~bad.cuda()])


def test_no_tokens(device):
    w = torch.ones(64, device="cuda", requires_grad=True)
    q = torch.zeros(2, 0, 4, 64, device="cuda", dtype=BF, requires_grad=True)
    k = torch.zeros(2, 0, 2, 64, device="cuda", dtype=BF)
    cos, sin = cuda(*tables(4, 64))
    out = norm_rotate(q, k, cos, sin, q_weight=w)
    assert out[0].shape == q.shape and out[1].shape == k.shape
    out[0].sum().backward()
    assert q.grad.shape == q.shape and bool((w.grad == 0).all())


def test_one_output_used(device):
    g = torch.Generator().manual_seed(6)
    q, k = (torch.randn(1, 7, n, 64, generator=g).cuda().requires_grad_() for n in (2, 1))
    w = torch.ones(64, device="cuda", requires_grad=True)
    norm_rotate(q, k, *cuda(*tables(7, 64)), q_weight=w, k_weight=w)[1].sum().backward()
    assert bool((q.grad == 0).all()) and bool((k.grad != 0).any())


def test_second_derivatives_are_refused(device):
    q = torch.randn(1, 3, 1, 64, device="cuda", requires_grad=True)
    w = torch.ones(64, device="cuda")
    out = norm_rotate(q, q, None, None, q_weight=w, k_weight=w)
    grad, = torch.autograd.grad(out[0].sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_replays_match_eager(device):
    case = (2, 33, 4, 2, 128, 64, False, BF, F32)
    q, k, gq, gk, wq, wk, cos, sin, pos = cuda(*inputs(case, 7))
    static = [t.clone().requires_grad_() for t in (q, k, wq, wk)]
    grads = [gq.clone(), gk.clone()]
    pos = pos.to(torch.int32)

    def step(leaves, g, pos):
        out = norm_rotate(leaves[0], leaves[1], cos, sin, positions=pos, q_weight=leaves[2],
                          k_weight=leaves[3])
        return [*out, *torch.autograd.grad(out, leaves, g)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static, grads, pos)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static, grads, pos)
    for seed in (8, 9, 10):
        new = cuda(*inputs(case, seed))
        with torch.no_grad():
            for s, t in zip(static, (new[0], new[1], new[4], new[5])):
                s.copy_(t)
            for s, t in zip(grads, new[2:4]):
                s.copy_(t)
            pos.copy_(new[8])
        graph.replay()
        torch.cuda.synchronize()
        eager = step([t.clone().requires_grad_() for t in (new[0], new[1], new[4], new[5])],
                     new[2:4], new[8])
        torch.cuda.synchronize()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)


def test_zero_rows_without_eps_are_not_a_number(device):
    """0 / 0, as the formula gives it; a row of zeros with eps stays zero."""
    q = torch.zeros(1, 2, 1, 64, device="cuda", dtype=BF)
    w = torch.ones(64, device="cuda")
    assert bool((norm_rotate(q, q, None, None, q_weight=w)[0] == 0).all())
    assert math.isnan(norm_rotate(q, q, None, None, q_weight=w, eps=0.0)[0].flatten()[0].item())


def test_far_positions_are_outside_the_tables(device):
    """int64 positions past 32 bits do not wrap around into the tables."""
    q, k = torch.ones(1, 4, 1, 64, device="cuda"), torch.ones(1, 4, 1, 64, device="cuda")
    cos, sin = (t.cuda() for t in tables(8, 64))
    pos = torch.tensor([3, 2 ** 32 + 3, -2 ** 32 + 3, 2 ** 31], device="cuda")
    for out in norm_rotate(q, k, cos, sin, positions=pos):
        assert bool(out[0, 0].isfinite().all()) and bool(out[0, 1:].isnan().all())

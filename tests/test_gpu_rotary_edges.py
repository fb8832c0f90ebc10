"""norm_rotate at the edges of what it takes: one token, one head,
forward-mode derivatives."""

import pytest
import torch
from torch.autograd import forward_ad

from moba.kernels.rotary import norm_rotate
from paged_util import tables

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("batch,seq,h,hk", [(1, 1, 4, 2), (1, 1, 1, 1), (3, 1, 4, 1), (1, 5, 1, 1)])
def test_one_token_or_head_of_odd_rows(device, dtype, batch, seq, h, hk):
    """Slices of a projection whose rows are no multiple of 16 bytes: values and
    gradients of the contiguous tensors, bit for bit."""
    d = 64
    g = torch.Generator().manual_seed(30)
    x = torch.randn(batch, seq, (h + hk) * d + 3, generator=g).to(dtype).cuda()
    cos, sin = (t.cuda() for t in tables(seq, d))
    w = torch.rand(d, generator=g).cuda() + 0.5
    grads = [torch.randn(batch, seq, n, d, generator=g).to(dtype).cuda() for n in (h, hk)]

    def run(q, k):
        leaves = [t.detach().requires_grad_() for t in (q, k, w)]
        out = norm_rotate(leaves[0], leaves[1], cos, sin, q_weight=leaves[2], k_weight=w)
        return [*out, *torch.autograd.grad(out, leaves, grads)]

    q, k = x[..., :h * d].unflatten(-1, (h, d)), x[..., h * d:(h + hk) * d].unflatten(-1, (hk, d))
    want = run(torch.empty(q.shape, dtype=dtype, device="cuda").copy_(q),
               torch.empty(k.shape, dtype=dtype, device="cuda").copy_(k))
    for a, b in zip(run(q, k), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["q", "k", "q_weight", "k_weight"])
def test_forward_mode_is_refused(device, which):
    """A tangent is never dropped in silence, with gradients enabled or not."""
    args = {"q": torch.randn(1, 3, 2, 64, device="cuda"), "k": torch.randn(1, 3, 1, 64, device="cuda"),
            "q_weight": torch.rand(64, device="cuda"), "k_weight": torch.rand(64, device="cuda")}
    cos, sin = (t.cuda() for t in tables(3, 64))
    want = norm_rotate(**args, cos=cos, sin=sin)
    with forward_ad.dual_level():
        # Without a dual tensor the call stands.
        for a, b in zip(norm_rotate(**args, cos=cos, sin=sin), want):
            assert torch.equal(a, b)
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        for grad in (True, False):
            with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward"):
                norm_rotate(**args, cos=cos, sin=sin)

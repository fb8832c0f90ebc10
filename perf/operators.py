"""Operators of MoBA serving and of the layer around the attention: what they
compute, and the calls whose times and results are tracked.

* norm_rotate: queries and keys of a layer, each head normalised by its root
  mean square, scaled by a learned weight and rotated by position; for
  training with its backward.
* append_tokens: the same for new tokens of cached sequences, whose keys and
  values go into the pages of a cache, with the representative (mean key) of
  every block that became full.
* paged_attention: MoBA attention of new tokens (a chunk of a prompt, or the
  one token of a decoding step) over such a cache.
* copy_pages: pages copied within a cache, in all layers.

A page holds one MoBA block: K and V [pages, kv heads, block, D], block
representatives [pages, kv heads, D]; a sequence's row of the block table
lists its pages in order.

The ranges (`draw`): one token to 128K; 1 to 64 sequences, contexts up to
128K tokens, lengths mostly no multiple of the block; 1 to 32 query heads over
1 to 8 kv heads; head_dim 64, 128 and 256; block size 16 to 128; top_k 2 to 16;
bfloat16, float16, float32; queries and keys as views of one fused projection
or by themselves; rotation of all features or of a part, of halves or of
neighbours.
"""

import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


def _package():
    # The package folder's name is no module name: its modules are found there.
    pkg = str(Path.cwd() / "moba-triton_amd")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)


# -- cases ------------------------------------------------------------------

def _qk(name, mode, dtype, batch, seq, heads, kv_heads, dim, rotary, interleaved=False,
        fused=True):
    return {"name": name, "op": "norm_rotate", "mode": mode, "dtype": dtype, "batch": batch,
            "seq": seq, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rotary": rotary,
            "interleaved": interleaved, "fused": fused}


def _append(name, dtype, seqs, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim, block):
    """`seqs` sequences of ctx_lo..ctx_hi cached tokens get new_lo..new_hi each."""
    return {"name": name, "op": "append", "dtype": dtype, "seqs": seqs, "new_lo": new_lo,
            "new_hi": new_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi, "heads": heads,
            "kv_heads": kv_heads, "dim": dim, "block": block}


def _attend(name, dtype, seqs, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim, block,
            top_k, keys="iid"):
    """As `_append`; the new tokens are already in the cache, behind ctx."""
    return dict(_append(name, dtype, seqs, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim,
                        block), op="attend", top_k=top_k, keys=keys)


def _copy(name, dtype, layers, pages, copies, kv_heads, dim, block):
    return {"name": name, "op": "copy", "dtype": dtype, "layers": layers, "pages": pages,
            "copies": copies, "kv_heads": kv_heads, "dim": dim, "block": block}


def listed():
    return [
        # A decoding step of a small batch, one layer's queries and keys.
        _qk("qk_decode_8", "infer", "bf16", 8, 1, 16, 4, 128, 128),
        # A training step in half precision at a ragged length, a quarter of
        # the features rotated, neighbours as pairs.
        _qk("qk_train_fp16_ragged", "train", "fp16", 2, 20011, 8, 2, 64, 16, interleaved=True),
        # A training step of a grouped-query layer of a large model.
        _qk("qk_train_gqa_32k", "train", "bf16", 1, 32768, 32, 8, 128, 128),
        # A decoding step of a full batch: one token for each sequence.
        _append("append_decode_64", "bf16", 64, 1, 1, 1, 2000, 32, 8, 128, 128),
        # Prompts of a few sequences behind cached prefixes of any length.
        _append("append_prompts", "bf16", 5, 1000, 4096, 0, 4000, 16, 4, 128, 64),
        # Decoding of one sequence at a long context: latency.
        _attend("decode_1_64k", "bf16", 1, 1, 1, 65536, 65536, 4, 4, 64, 128, 8),
        # Decoding of a batch of grouped-query sequences of all lengths.
        _attend("decode_32", "bf16", 32, 1, 1, 0, 100000, 32, 8, 128, 128, 8),
        # One chunk of a long prompt, most of it already cached.
        _attend("chunk_2k_at_128k", "bf16", 1, 2048, 2048, 129001, 129001, 32, 8, 128, 128, 8),
        # Chunks and single tokens in one call, half precision, small blocks,
        # keys with the per-channel offset that trained keys have.
        _attend("mixed_fp16", "fp16", 12, 1, 700, 0, 30000, 16, 4, 64, 64, 12, keys="offset"),
        # Full precision, as reference runs ask for it.
        _attend("chunk_fp32", "fp32", 1, 500, 500, 8000, 8000, 8, 2, 64, 64, 8),
        # Shared pages made a sequence's own before it writes into them.
        _copy("copy_on_write_8", "bf16", 16, 64, 8, 8, 128, 128),
        # Compaction of a cache after many sequences have ended.
        _copy("compact_180", "bf16", 16, 400, 180, 8, 128, 128),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limits = {}
    for c in listed():
        w = work(c)
        at = limits.setdefault(c["op"], {"bytes": 0, "flops": 0})
        at["bytes"], at["flops"] = max(at["bytes"], w["bytes"]), max(at["flops"], w["flops"])
    while True:
        kv_heads = rng.choice([1, 2, 4, 4, 8])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 8])
        dim = rng.choice([64, 64, 128, 128, 128, 256])
        block = rng.choice([16, 32, 64, 80, 128, 128])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp16", "fp32"])
        op = rng.choice(["norm_rotate", "append", "attend", "attend", "attend", "copy"])
        if heads > 32:
            continue
        if op == "norm_rotate":
            case = _qk("", rng.choice(["train", "infer"]), dtype, rng.choice([1, 1, 2, 3, 8]),
                       _log_int(rng, 1, 131072), heads, kv_heads, dim,
                       rng.choice([dim, dim, dim // 2, dim // 4]), rng.random() < 0.3,
                       rng.random() < 0.6)
        elif op == "copy":
            copies = _log_int(rng, 1, 200)
            case = _copy("", dtype, rng.choice([1, 4, 16, 24]), 2 * copies + rng.randint(0, 50),
                         copies, kv_heads, dim, block)
        else:
            seqs = _log_int(rng, 1, 64)
            new_hi = 1 if rng.random() < 0.4 else _log_int(rng, 2, 4096)
            new_lo = rng.choice([1, new_hi, max(1, new_hi // 8)])
            ctx_hi = _log_int(rng, 16, 131072 if op == "attend" else 8192)
            ctx_lo = rng.choice([0, ctx_hi, ctx_hi // 2])
            args = ("", dtype, seqs, new_lo, new_hi, ctx_lo, ctx_hi, heads, kv_heads, dim, block)
            if op == "append":
                case = _append(*args)
            else:
                case = _attend(*args, rng.choice([2, 3, 4, 8, 8, 12, 16]),
                               rng.choice(["iid", "iid", "offset", "walk"]))
            # Pages held: what the case needs of memory.
            held = _pages(case) * kv_heads * block * dim
            if held > (1 << 30) or sum(_lengths(case)[0]) * heads * dim > 1 << 26:
                continue
        w, top = work(case), limits[op]
        share = 1 / 8 if dtype == "fp32" and op == "attend" else 1
        if w["bytes"] <= top["bytes"] and w["flops"] <= share * top["flops"]:
            del case["name"]
            return case


def _lengths(case):
    """(new tokens, cached tokens before them) of every sequence, from the
    sizes alone."""
    rng = random.Random(case["seqs"] * 1000003 + case["new_hi"] * 1009 + case["ctx_hi"])
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["seqs"])]
    ctx = [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    return new, ctx


def _pages(case):
    new, ctx = _lengths(case)
    return sum(-(-(n + c) // case["block"]) for n, c in zip(new, ctx))


def work(case):
    size = torch.empty((), dtype=DTYPES[case["dtype"]]).element_size()
    dim, kv_heads = case["dim"], case["kv_heads"]
    if case["op"] == "copy":
        page = kv_heads * dim * (2 * case["block"] + 1) * size
        return {"bytes": 2 * case["layers"] * case["copies"] * page, "flops": 0}
    heads = case["heads"]
    if case["op"] == "norm_rotate":
        rows = case["batch"] * case["seq"] * (heads + kv_heads)
        passes, ops = (5, 25) if case["mode"] == "train" else (2, 8)
        return {"bytes": rows * dim * passes * size, "flops": rows * dim * ops}
    new, ctx = _lengths(case)
    if case["op"] == "append":
        # q, k and v read and written; every full block's older keys read.
        rows = sum(new) * (heads + 2 * kv_heads)
        full = sum((n + c) // case["block"] - c // case["block"] for n, c in zip(new, ctx))
        old = sum(c % case["block"] for n, c in zip(new, ctx)
                  if (n + c) // case["block"] > c // case["block"])
        return {"bytes": (2 * rows + (full + old) * kv_heads) * dim * size,
                "flops": sum(new) * (heads + kv_heads) * dim * 8}
    bs, take, group = case["block"], case["top_k"] - 1, heads // kv_heads
    rows = 2 * sum(new) * heads  # q and out
    keys = pairs = past_pairs = 0
    for n, c in zip(new, ctx):
        for first in range(c - c % bs, c + n, bs):  # the queries of one own block
            a, b = max(first, c), min(first + bs, c + n)
            own_block = first // bs
            pairs += (b - a) * min(take, own_block) * bs + (b - a) * (a + b + 1 - 2 * first) // 2
            past_pairs += (b - a) * own_block
        # Distinct blocks that independent choices touch, the new tokens' own
        # blocks among them.
        full = c // bs
        chosen = full if full <= take else full * (1 - (1 - take / full) ** (group * n))
        keys += kv_heads * (min(chosen * bs, c) + n + c % bs)
        rows += kv_heads * ((c + n - 1) // bs)  # representatives
    return {"bytes": int((rows + 2 * keys) * dim * size),
            "flops": heads * dim * (4 * pairs + 2 * past_pairs)}


# -- inputs -----------------------------------------------------------------

def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _tables(positions, rotary):
    """cos, sin [positions, rotary / 2] float32, from angles in 64 bits."""
    freq = 10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device="cuda") / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device="cuda")[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _projection(gen, case, *lead, fused=True):
    """q, k, v [..., heads, D] of one fused projection, or each by itself."""
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    x = _randn(gen, *lead, h + 2 * hk, d, dtype=DTYPES[case["dtype"]])
    q, k, v = x[..., :h, :], x[..., h:h + hk, :], x[..., h + hk:, :]
    return (q, k, v) if fused else (q.contiguous(), k.contiguous(), v.contiguous())


def _kbar(k):
    """Block representatives of pages [..., block, D]: the exact sum rounded
    to float32 and to the type, the quotient rounded to the type."""
    total = torch.cat([part.double().sum(-2) for part in k.split(1024)])
    return (total.float().to(k.dtype).float() / k.shape[-2]).to(k.dtype)


def _cache(gen, case):
    """A cache's pages and the sequences on them, in random order."""
    new, ctx = _lengths(case)
    bs, hk, d, dtype = case["block"], case["kv_heads"], case["dim"], DTYPES[case["dtype"]]
    lens = [n + c for n, c in zip(new, ctx)]
    counts = [-(-length // bs) for length in lens]
    pages = sum(counts) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lens), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = order[at:at + n]
        at += n
    k = _randn(gen, pages, hk, bs, d, dtype=dtype)
    v = _randn(gen, pages, hk, bs, d, dtype=dtype)
    if case.get("keys") == "offset":
        k += _randn(gen, 1, hk, 1, d, dtype=dtype)
    elif case.get("keys") == "walk":
        for s, n in enumerate(counts):  # a drift along each sequence
            k[table[s, :n].long()] += (_randn(gen, n, hk, 1, d).cumsum(0) * 0.1).to(dtype)
    cu = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    return {"k": k, "v": v, "table": table, "cu": cu, "new": new, "ctx": ctx,
            "lens": torch.tensor(lens, dtype=torch.int32, device="cuda")}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    state = {"case": case}
    if case["op"] == "copy":
        shape = (case["layers"], case["pages"], case["kv_heads"], case["block"], case["dim"])
        k, v = torch.empty(shape, dtype=dtype, device="cuda"), torch.empty(shape, dtype=dtype, device="cuda")
        for layer in range(case["layers"]):
            k[layer], v[layer] = _randn(gen, *shape[1:]), _randn(gen, *shape[1:])
        perm = torch.randperm(case["pages"], generator=torch.Generator().manual_seed(seed))
        n = case["copies"]
        state.update(k=k, v=v, kbar=_randn(gen, *shape[:3], case["dim"], dtype=dtype),
                     src=perm[:n].to(torch.int32), dst=perm[n:2 * n].to(torch.int32))
        return state
    if case["op"] == "norm_rotate":
        b, s = case["batch"], case["seq"]
        q, k, _ = _projection(gen, case, b, s, fused=case["fused"])
        state.update(q=q, k=k)
        if case["mode"] == "train":
            state.update(gq=_randn(gen, *q.shape, dtype=dtype), gk=_randn(gen, *k.shape, dtype=dtype))
        # Decoding steps stand at any position, training rows start at 0.
        first = 1000 if s == 1 else 0
        pos = torch.arange(first, first + s, dtype=torch.int32, device="cuda")
        state["positions"] = pos.expand(b, s).contiguous()
        state["cos"], state["sin"] = _tables(first + s, case["rotary"])
    else:
        state.update(_cache(gen, case))
        if case["op"] == "attend":
            state["q"] = _randn(gen, sum(state["new"]), case["heads"], case["dim"], dtype=dtype)
            state["kbar"] = _kbar(state["k"])
            return state
        state["kbar"] = torch.zeros_like(state["k"][:, :, 0])
        state["q"], state["k_new"], state["v_new"] = _projection(gen, case, sum(state["new"]))
        state["cos"], state["sin"] = _tables(int(state["lens"].max()), case["dim"])
    state["wq"] = 1 + 0.1 * _randn(gen, case["dim"])
    state["wk"] = 1 + 0.1 * _randn(gen, case["dim"])
    return state


# -- one pass ---------------------------------------------------------------

def run(state):
    op = state["case"]["op"]
    if own:
        _package()
    return {"norm_rotate": _run_norm_rotate, "append": _run_append, "attend": _run_attend,
            "copy": _run_copy}[op](state)


def _run_norm_rotate(s):
    case = s["case"]
    train = case["mode"] == "train"
    if own:
        from moba.kernels.rotary import norm_rotate
        leaves = [s[n].detach().requires_grad_(train) for n in ("q", "k", "wq", "wk")]
        q, k, wq, wk = leaves
        out = norm_rotate(q, k, s["cos"], s["sin"], positions=s["positions"], q_weight=wq,
                          k_weight=wk, eps=EPS, interleaved=case["interleaved"])
        if not train:
            return tuple(out)
        return tuple(out) + torch.autograd.grad(out, leaves, (s["gq"], s["gk"]))
    pos = s["positions"].long()
    cos, sin = s["cos"][pos][:, :, None], s["sin"][pos][:, :, None]
    outs, grads = [], []
    for x, w, g in ((s["q"], s["wq"], s.get("gq")), (s["k"], s["wk"], s.get("gk"))):
        x = x.float()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        xr = x * r
        outs.append(_rotate(xr * w, cos, sin, case["interleaved"]).to(DTYPES[case["dtype"]]))
        if train:
            g = _rotate(g.float(), cos, -sin, case["interleaved"])
            dw = (g * xr).flatten(0, -2).sum(0, dtype=torch.float64).float()
            h = g * w
            dx = r * (h - xr * (h * xr).mean(-1, keepdim=True))
            grads.append((dx.to(DTYPES[case["dtype"]]), dw))
    if not train:
        return tuple(outs)
    return tuple(outs) + (grads[0][0], grads[1][0], grads[0][1], grads[1][1])


def _rotate(x, cos, sin, interleaved):
    """The first 2 * cos.shape[-1] features of x rotated: halves or neighbours."""
    half = cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * half:]), -1)


def _positions(s):
    """Sequence and position of every new token."""
    dev = s["q"].device
    new, ctx = torch.tensor(s["new"], device=dev), torch.tensor(s["ctx"], device=dev)
    seq = torch.repeat_interleave(torch.arange(len(s["new"]), device=dev), new,
                                  output_size=sum(s["new"]))
    pos = torch.arange(sum(s["new"]), device=dev) - s["cu"].long()[seq] + ctx[seq]
    return seq, pos


def _run_append(s):
    bs = s["case"]["block"]
    if own:
        from moba.kernels.paged import PagedKV, append_tokens
        q = append_tokens(s["q"], s["k_new"], s["v_new"], PagedKV(s["k"], s["v"], s["kbar"]),
                          s["table"], s["lens"], cu_seqlens=s["cu"], cos=s["cos"], sin=s["sin"],
                          q_weight=s["wq"], k_weight=s["wk"], eps=EPS)
        return q, s["k"], s["v"], s["kbar"]
    seq, pos = _positions(s)
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    rows = []
    for x, w in ((s["q"], s["wq"]), (s["k_new"], s["wk"])):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        rows.append(_rotate(x, cos, sin, False).to(s["k"].dtype))
    page = s["table"].long()[seq, pos // bs]
    s["k"][page, :, pos % bs] = rows[1]
    s["v"][page, :, pos % bs] = s["v_new"]
    full = page[pos % bs == bs - 1]
    if full.numel():
        s["kbar"][full] = _kbar(s["k"][full])
    return rows[0], s["k"], s["v"], s["kbar"]


def _select(s, q, pos, pages):
    """Block ids [tokens, heads, slots] of queries at `pos` whose sequences'
    pages are `pages` [tokens, blocks]; -1 for none."""
    bs, take, hk = s["case"]["block"], s["case"]["top_k"] - 1, s["case"]["kv_heads"]
    kbar = s["kbar"][pages].double().transpose(1, 2).contiguous()  # [tokens, kv heads, blocks, D]
    heads = q.double().unflatten(1, (hk, -1)).mT.contiguous()      # [tokens, kv heads, D, group]
    score = torch.matmul(kbar, heads).mT.flatten(1, 2)             # exact: [tokens, heads, blocks]
    score = score.float().to(q.dtype).float()
    own_block = (pos // bs)[:, None, None]
    past = torch.arange(pages.shape[1], device=q.device) < own_block
    score = torch.where(past, score, -math.inf)
    best, ids = torch.sort(score, dim=-1, descending=True, stable=True)
    ids = torch.where(best[..., :take] > -math.inf, ids[..., :take], -1)
    return torch.cat((ids, own_block.expand(-1, ids.shape[1], 1)), -1)


def _run_attend(s):
    case = s["case"]
    if own:
        from moba.config import MoBAConfig
        from moba.kernels.paged import PagedKV, paged_attention
        cfg = MoBAConfig(block_size=case["block"], top_k=case["top_k"], dtype=s["q"].dtype)
        return paged_attention(s["q"], PagedKV(s["k"], s["v"], s["kbar"]), s["table"], s["lens"],
                               cfg, cu_seqlens=s["cu"])
    out = torch.empty_like(s["q"])
    bs, dim, heads, hk = case["block"], case["dim"], case["heads"], case["kv_heads"]
    head = torch.arange(heads, device=out.device)[:, None] // (heads // hk)
    seq, position = _positions(s)
    # Tokens at a time: gathered keys and representatives of at most 2^28 elements.
    step = max(1, (1 << 28) // (dim * max(heads * case["top_k"] * bs, hk * s["table"].shape[1])))
    for t in range(0, out.shape[0], step):
        q, pos = s["q"][t:t + step], position[t:t + step]
        pages = s["table"][seq[t:t + step]].long().clamp(min=0)
        ids = _select(s, q, pos, pages)
        at = torch.gather(pages[:, None].expand(-1, heads, -1), 2, ids.clamp(min=0))
        k = s["k"][at, head].float().flatten(2, 3)  # [tokens, heads, slots * block, D]
        key = ids[..., None] * bs + torch.arange(bs, device=q.device)
        seen = ((ids[..., None] >= 0) & (key <= pos[:, None, None, None])).flatten(2)
        x = torch.matmul(k, q.float()[..., None])[..., 0] * dim ** -0.5
        x = torch.where(seen, x, -math.inf)
        p = torch.exp(x - x.amax(-1, keepdim=True))
        del k
        v = s["v"][at, head].float().flatten(2, 3)
        o = torch.matmul(p[:, :, None], v)[:, :, 0] / p.sum(-1, keepdim=True)
        out[t:t + step] = o.to(q.dtype)
    return out


def _run_copy(s):
    if own:
        from moba.kernels.paged import PagedKV, copy_pages
        copy_pages(PagedKV(s["k"], s["v"], s["kbar"]), s["src"], s["dst"])
    else:
        src, dst = s["src"].to("cuda").long(), s["dst"].to("cuda").long()
        for t in (s["k"], s["v"], s["kbar"]):
            t[:, dst] = t[:, src]
    return s["k"], s["v"], s["kbar"]


# -- 64-bit results ---------------------------------------------------------

def exact(case, seed):
    """What `run` returns, from the definitions in 64 bits."""
    if case["op"] == "copy":
        return None  # copies: nothing is computed
    s = prepare(case, seed)
    if case["op"] == "norm_rotate":
        train = case["mode"] == "train"
        leaves = [s[n].detach().double().requires_grad_(train) for n in ("q", "k", "wq", "wk")]
        turn = _turns(s["positions"].long(), case["rotary"])
        out = tuple(_turned(leaves[i], leaves[2 + i], turn, case["interleaved"]) for i in (0, 1))
        if not train:
            return out
        return tuple(o.detach() for o in out) + torch.autograd.grad(
            out, leaves, (s["gq"].double(), s["gk"].double()))
    if case["op"] == "append":
        return _exact_append(s)
    return _exact_attend(s)


def _turns(pos, rotary):
    """The rotations of `pos` as complex numbers [..., 1, rotary / 2]. Their
    parts are rounded to float32: the tables are inputs."""
    freq = torch.exp(torch.arange(0, rotary, 2, dtype=torch.float64, device=pos.device)
                     * (-math.log(10000.0) / rotary))
    angle = pos.double()[..., None, None] * freq
    return torch.complex(angle.cos().float().double(), angle.sin().float().double())


def _turned(x, w, turn, interleaved):
    y = w * x / torch.sqrt(x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS)
    half = turn.shape[-1]
    head, tail = y[..., :2 * half], y[..., 2 * half:]
    pair = head.unflatten(-1, (half, 2)) if interleaved else head.unflatten(-1, (2, half)).mT
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    return torch.cat(((z if interleaved else z.mT).flatten(-2), tail), -1)


def _exact_append(s):
    case, bs = s["case"], s["case"]["block"]
    k, v, kbar = s["k"].double(), s["v"].double(), s["kbar"].double()
    out = []
    at = 0
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        pos = torch.arange(c, c + n, device=k.device)
        turn = _turns(pos, case["dim"])
        out.append(_turned(s["q"][at:at + n].double(), s["wq"].double(), turn, False))
        kn = _turned(s["k_new"][at:at + n].double(), s["wk"].double(), turn, False)
        for block in range(c // bs, (c + n - 1) // bs + 1):
            a, b = max(block * bs, c), min(block * bs + bs, c + n)
            page = int(s["table"][i, block])
            k[page, :, a - block * bs:b - block * bs] = kn[a - c:b - c].transpose(0, 1)
            v[page, :, a - block * bs:b - block * bs] = \
                s["v_new"][at + a - c:at + b - c].double().transpose(0, 1)
            if b == block * bs + bs:
                kbar[page] = k[page].mean(1)
        at += n
    return torch.cat(out), k, v, kbar


def _exact_attend(s):
    """Kv head by kv head and slot by slot with a running maximum; the routing
    is that of the inputs' type, by an order over (score, id)."""
    case, bs, hk = s["case"], s["case"]["block"], s["case"]["kv_heads"]
    group, take, scale = case["heads"] // hk, case["top_k"] - 1, case["dim"] ** -0.5
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, c) in enumerate(zip(s["new"], s["ctx"])):
        pages = s["table"][i, :(c + n - 1) // bs + 1].long()
        step = max(1, (1 << 26) // (group * bs * case["dim"]))
        for h in range(hk):
            kb = s["kbar"][pages, h].double()
            for t in range(0, n, step):
                q = s["q"][at + t:at + min(t + step, n), h * group:(h + 1) * group].double()
                pos = torch.arange(c + t, c + t + q.shape[0], device="cuda")[:, None].expand(-1, group)
                score = torch.einsum("tgd,nd->tgn", q, kb).float().to(s["q"].dtype).double()
                index = torch.arange(kb.shape[0], device="cuda")
                score = score.masked_fill(index >= (pos // bs)[..., None], -math.inf)
                top = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
                total, acc = torch.zeros_like(top), torch.zeros_like(q)
                for slot in range(take + 1):
                    if slot == 0:
                        pick, live = pos // bs, torch.ones_like(top, dtype=torch.bool)
                    else:
                        best = score.amax(-1, keepdim=True)
                        pick = torch.where(score == best, index, kb.shape[0]).amin(-1)
                        live = best[..., 0] > -math.inf
                        pick = torch.where(live, pick, 0)
                        score = score.scatter(-1, pick[..., None], -math.inf)
                    keys, values = s["k"][pages[pick], h].double(), s["v"][pages[pick], h].double()
                    x = (keys * q[:, :, None]).sum(-1) * scale
                    seen = (pick[..., None] * bs + torch.arange(bs, device="cuda")) <= pos[..., None]
                    x = x.masked_fill(~(seen & live[..., None]), -math.inf)
                    m = torch.maximum(top, x.amax(-1))
                    p, old = torch.exp(x - m[..., None]), torch.exp(top - m)
                    total = total * old + p.sum(-1)
                    acc = acc * old[..., None] + (p[..., None] * values).sum(2)
                    top = m
                out[at + t:at + t + q.shape[0], h * group:(h + 1) * group] = acc / total[..., None]
        at += n
    return out

"""The 4-bit cache's format and its attention in 64 bits, element by element from the definition."""

import math

import torch


def decoded(pool):
    """Keys and values [blocks, tokens of a page, kv heads, hd] fp64 that the bytes of ``pool`` stand for."""
    blocks, hkv, tiles, width = pool.shape
    hd = width // 18
    ng = hd // 32
    raw = pool.cpu()
    scales = raw[..., 16 * hd:].contiguous().view(torch.float16).double()      # [..., 16 tokens * 2 * ng]
    out = torch.zeros((2, blocks, hkv, tiles, 16, hd), dtype=torch.float64)
    for t in range(16):
        for d in range(hd):
            word = (t // 8) * ng + d // 32
            start = word // 4 * 512 + word % 4 * 4
            key = raw[..., start + (t % 8 * 4 + d % 32 // 8) * 16 + d % 8 // 2]
            value = raw[..., 8 * hd + start + (d % 32 // 4 * 4 + t % 8 // 2) * 16 + t % 2 * 2 + d % 4 // 2]
            for i, byte in enumerate((key, value)):
                n = (byte >> 4 if d % 2 else byte & 15).double() - 8
                out[i, ..., t, d] = n * scales[..., t * 2 * ng + i * ng + d // 32]
    return tuple(x.permute(0, 2, 3, 1, 4).reshape(blocks, tiles * 16, hkv, hd) for x in out)


def quantised(x):
    """fp64 values that rows x [..., hd] have in the cache."""
    g = x.double().unflatten(-1, (-1, 32))
    most, least = g.amax(-1, keepdim=True), g.amin(-1, keepdim=True)
    step = (torch.where(most >= -least, most, least) / -8).clamp(-65504, 65504).half().double()
    n = torch.where(step == 0, torch.zeros_like(g), g / torch.where(step == 0, torch.ones_like(step), step))
    return (n.round().clamp(-8, 7) * step).flatten(-2)


def attention(q, k, v, table, lens, hq, scale, seqs=None):
    """(out, tolerance) fp64 [T, hq, hd]. k, v as :func:`decoded` gives them. The tolerance is what the kernel's roundings
    can add up to, times 1.1 for products of them:

    * probability times value scale is rounded to fp16, half a step of at most 2^-11 relative (the value's code counts from
      0 there, at most 15 scales; with |v| >= 0 it is at most 15 |scale|, bounded here by 15 / 7 of the group's largest
      or, all elements being codes of one scale, by 15 scales): 2^-11 * sum p 15 |scale| / sum p;
    * a score: fp32 sums of hd products of at most 15 |q| |scale| each and of the constant 8 sum |q| |scale|, every
      addition relative 2^-22 of the sum of magnitudes (matrix instructions cut instead of rounding), hd / 16 + 8 of them in
      a row; exp2 and the subtraction of the maximum 2^-21 of max(1, |score| range): an error e of the natural score moves
      out by at most 2 e sum p |v| / sum p;
    * the output's own rounding: eps / 2 of its type."""
    t, hd = q.shape[0], q.shape[1] // hq
    blocks, bs, hkv, _ = k.shape
    out = torch.zeros((t, hq, hd), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for i in range(t):
        row = i if seqs is None else int(seqs[i])
        n = min(int(lens[i]), table.shape[1] * bs) if 0 <= row < table.shape[0] else 0
        rows = [(int(table[row, p // bs]), p % bs) for p in range(max(n, 0))]
        rows = [(b, o) for b, o in rows if 0 <= b < blocks]
        if not rows:
            continue
        b, o = torch.tensor(rows).T
        for h in range(hq):
            kk, vv = k[b, o, h * hkv // hq], v[b, o, h * hkv // hq]
            x = q[i].view(hq, hd)[h].double().cpu()
            s = (kk @ x) * scale
            p = torch.softmax(s, 0)
            out[i, h] = p @ vv
            # |scale| of a group is at least a 1/8 of its largest element: codes reach -8 .. 7
            step_k = kk.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2) / 7
            step_v = vv.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2) / 7
            magnitude = (23 * step_k * x.abs()).sum(-1).max() * abs(scale)
            err = (hd / 16 + 8) * 2.0 ** -22 * magnitude + 2.0 ** -21 * max(1.0, float(s.max() - s.min()))
            tol[i, h] = 1.1 * (2.0 ** -11 * 15 * (p @ step_v) + 2 * err * (p @ vv.abs())
                               + torch.finfo(q.dtype).eps / 2 * out[i, h].abs()) + torch.finfo(q.dtype).tiny
    return out.view(t, -1), tol.view(t, -1)


def cache(lens, hkv, hd, bs, dtype, seed=0, spare=3, spread=False, device="cpu"):
    """(pool with Gaussian rows everywhere, its table, rows) for sequences of the given lengths, pages in random order.
    ``spread``: magnitudes of the values' tokens over 2^-12 .. 2^8, of the keys' channels over 1 .. 8."""
    from ironcore_b200.ops import paged

    g = torch.Generator().manual_seed(seed)
    need = [-(-n // bs) for n in lens]
    blocks = sum(need) + spare
    k, v = (torch.randn((blocks * bs, hkv * hd), generator=g) for _ in range(2))
    if spread:
        k *= 8.0 ** torch.rand(hkv * hd, generator=g)
        v *= 2.0 ** (20 * torch.rand((blocks * bs, 1), generator=g) - 12)
    pool = torch.zeros(paged.q4_pool_shape(blocks, hkv, bs, hd), dtype=torch.uint8)
    paged.kv_append_q4_reference(k.to(dtype), v.to(dtype), pool, torch.arange(blocks * bs))
    order = torch.randperm(blocks, generator=g)
    table = torch.zeros((len(lens), max(max(need), 1)), dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n].int()
        at += n
    return pool.to(device), table.to(device), torch.tensor(lens, dtype=torch.int32, device=device)


def scale_of(hd):
    return 1 / math.sqrt(hd)

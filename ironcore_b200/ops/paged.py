"""Attention over paged K / V caches in 16 or 4 bits, rows into and out of them, copies of their pages: native kernels on
CUDA, PyTorch restatements elsewhere (oracle / CPU path).

The 4-bit cache (``csrc/q4.cuh`` has the byte order): a pool ``[num_blocks, kv_heads, block_size / 16, 18 * head_dim]`` uint8
holds keys and values; every 32 neighbouring elements of a token's head share an fp16 scale, a code n in 0..15 stands for
``scale * (n - 8)``. 4.5 bits an element, so a token costs 9/32 of its 16-bit rows."""

from __future__ import annotations

import ctypes
import functools
import struct
from typing import Optional, Sequence, Tuple, Union

import torch

from . import native
from .native import call, dtype_code, ptr, stream_ptr

P, I, L, F = native.P, native.I, native.L, native.F
native.register("icb_kv_append", [P, P, P, P, P, I, I, L, L, P])
native.register("icb_paged_decode", [P, L, P, P, P, P, P, P, I, I, I, I, I, I, F, I, P, P, I, P, I, I, I, P, L])
# these take their arguments as one packed record: see csrc/paged_q4.cu and csrc/paged_q4_decode.cu
native.register("icb_kv_append_q4", [ctypes.c_char_p, P])
native.register("icb_kv_read_q4", [ctypes.c_char_p, P])
native.register("icb_paged_decode_q4", [ctypes.c_char_p, P])
_ROWS_CALL = struct.Struct("12q").pack
_DECODE_CALL = struct.Struct("18qdq").pack
native.register("icb_paged_decode_q4_plan", [I, I, I, L, L])
native.register("icb_copy_pages", [P, I, P, P, I, P])
_SMS = None
_HALF = {dt: dtype_code(dt) for dt in (torch.bfloat16, torch.float16)}
Q4_GROUP = 32                                       # elements that share a scale
Q4_HEAD_DIMS = (64, 128, 192, 256)


def _decode_splits(rows: int, groups: int, max_tokens: int) -> int:
    """Context ranges per (row, kv head) for the tensor-core decode kernel: enough CTAs for two per SM, at least four
    16-token steps per range."""
    global _SMS
    if _SMS is None:
        _SMS = torch.cuda.get_device_properties(torch.cuda.current_device()).multi_processor_count
    want = -(-2 * _SMS // max(1, rows * groups))
    return max(1, min(want, 8, max(1, max_tokens // 64)))


def kv_append(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor):
    """k, v: [T, hkv*hd] (row views with arbitrary pitch); caches [blocks, bs, hkv, hd]; slots int64 [T]."""
    t, row = k.shape
    if k.is_cuda and k.dtype in (torch.bfloat16, torch.float16):
        call("icb_kv_append", ptr(k), ptr(v), ptr(k_cache), ptr(v_cache), ptr(slots), t, row, k.stride(0), v.stride(0),
             stream_ptr())
        return
    kc = k_cache.view(-1, row)
    vc = v_cache.view(-1, row)
    ok = slots >= 0
    kc[slots[ok]] = k[ok]
    vc[slots[ok]] = v[ok]


def paged_decode_reference(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, hd, scale):
    s = q.shape[0]
    bs = k_cache.shape[1]
    out = torch.zeros((s, hq * hd), dtype=q.dtype, device=q.device)
    g = hq // hkv
    for i in range(s):
        n = int(seq_lens[i])
        if n == 0:
            continue
        pages = (n + bs - 1) // bs
        blocks = block_table[i, :pages].long()
        k = k_cache[blocks].reshape(-1, hkv, hd)[:n].float()
        v = v_cache[blocks].reshape(-1, hkv, hd)[:n].float()
        qi = q[i].view(hq, hd).float()
        k = k.repeat_interleave(g, dim=1)
        v = v.repeat_interleave(g, dim=1)
        sc = torch.einsum("hd,nhd->hn", qi, k) * scale
        p = torch.softmax(sc, dim=-1)
        out[i] = torch.einsum("hn,nhd->hd", p, v).reshape(-1).to(q.dtype)
    return out


def mma_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor,
               hq: int, hkv: int, hd: int, *, block_size: int, max_keys: int, scale: float, out: torch.Tensor,
               seqs: Optional[torch.Tensor] = None, len_bias: int = 0, window: int = 0, chunk: int = 0,
               gate: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The tensor-core kernel (16-bit, head size 64 or 128): query row i (q [T, hq*hd], any 16-byte pitch) against the
    pages of sequence ``seqs[i]`` (None: i) up to position ``lens[i] + len_bias - 1``. ``out``: [T, hq*hd], any pitch.
    ``max_keys`` bounds how many keys a row sees."""
    t = q.shape[0]
    nsplit = _decode_splits(t, hkv * ((hq // hkv + 7) // 8), max_keys)
    scratch = torch.empty(max(1, t * hq * nsplit * (hd + 2) if nsplit > 1 else 1), dtype=torch.float32, device=q.device)
    call("icb_paged_decode", ptr(q), q.stride(0), ptr(k_cache), ptr(v_cache), ptr(block_table), ptr(lens), ptr(out), None,
         t, hq, hkv, hd, int(block_size), block_table.shape[1], float(scale), dtype_code(q.dtype), stream_ptr(),
         ptr(scratch), int(nsplit), ptr(seqs), int(len_bias), int(window), int(chunk), ptr(gate), out.stride(0))
    return out


def paged_decode(q: torch.Tensor, k_cache, v_cache, block_table, seq_lens, hq: int, hkv: int, hd: int,
                 scale: Optional[float] = None) -> torch.Tensor:
    """q: [S, hq*hd] (row view, any pitch) -> [S, hq*hd]: attention of one token per sequence over its pages."""
    scale = scale if scale is not None else hd ** -0.5
    s = q.shape[0]
    if q.is_cuda and q.dtype in (torch.bfloat16, torch.float16) and hd in (64, 128):
        out = torch.empty((s, hq * hd), dtype=q.dtype, device=q.device)
        if q.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0:
            # tensor-core kernel (mma.sync over the GQA group), the context split over several CTAs
            return mma_decode(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, hd, block_size=k_cache.shape[1],
                              max_keys=block_table.shape[1] * k_cache.shape[1], scale=scale, out=out)
        if hq // hkv <= 8:
            call("icb_paged_decode", ptr(q), q.stride(0), ptr(k_cache), ptr(v_cache), ptr(block_table), ptr(seq_lens),
                 ptr(out), None, s, hq, hkv, hd, k_cache.shape[1], block_table.shape[1], float(scale),
                 dtype_code(q.dtype), stream_ptr(), None, 0, None, 0, 0, 0, None, 0)
            return out
    return paged_decode_reference(q, k_cache, v_cache, block_table, seq_lens, hq, hkv, hd, scale)


# --------------------------------------------------------------------------- pages
def _elsewhere(dev: int) -> bool:
    """Whether launches for tensors on CUDA device ``dev`` need another current device."""
    return dev != native.current_device()


def _page_numbers(x, name: str) -> torch.Tensor:
    if not isinstance(x, torch.Tensor):
        if not all(isinstance(n, int) for n in x):
            raise ValueError(f"{name} must be a list of page numbers")
        x = torch.tensor(list(x), dtype=torch.int64)
    if x.dim() != 1 or x.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be a list of page numbers")
    return x


def copy_pages(pools: Union[torch.Tensor, Sequence[torch.Tensor]], src, dst) -> None:
    """Page ``dst[i]`` becomes page ``src[i]`` in every pool, all pools in one launch. ``pools``: one stacked tensor
    [layers, pages, ...], or a sequence of tensors [pages, ...] (any shapes and types, contiguous). No page may be written
    twice or be both written and read. ``src``, ``dst`` on the host (lists, CPU tensors) are checked for that and for their
    range; int32 tensors on the device are taken as they are, pairs with a page outside a pool being left out."""
    stacked = isinstance(pools, torch.Tensor)
    tensors: Sequence[torch.Tensor] = (pools,) if stacked else pools
    src, dst = _page_numbers(src, "src"), _page_numbers(dst, "dst")
    n = src.shape[0]
    if n != dst.shape[0]:
        raise ValueError(f"{n} source pages for {dst.shape[0]} destinations")
    if not tensors:
        return
    lead = 1 if stacked else 0
    dev = tensors[0].get_device()
    records = []
    for t in tensors:
        if t.dim() <= lead or not t.is_contiguous():
            raise ValueError("a pool must be contiguous, pages first" + (" after the layers" if stacked else ""))
        if t.get_device() != dev:
            raise ValueError("the pools must be on one device")
        if t.numel():
            layers, pages = (t.shape[0] if stacked else 1), t.shape[lead]
            page = t.numel() // (layers * pages) * t.element_size()      # strides of single layers and pages say nothing
            records += (t.data_ptr(), layers, pages * page, pages, page)
    if src.get_device() >= 0 or dst.get_device() >= 0:
        if not src.get_device() == dst.get_device() == dev or not src.dtype == dst.dtype == torch.int32:
            raise ValueError("page numbers on the device must be int32, both on the pools' device")
    else:
        pages = min(t.shape[lead] for t in tensors)
        a, b = src.tolist(), dst.tolist()
        if any(not 0 <= x < pages for x in a + b):
            raise ValueError(f"page numbers must be in [0, {pages})")
        if len(set(b)) != len(b) or not set(a).isdisjoint(b):
            raise ValueError("a page may be written once, and not be read by another pair")
    if n == 0 or not records:
        return
    if dev < 0:
        a, b = src.long(), dst.long()
        for t in tensors:
            if stacked:
                t[:, b] = t[:, a]
            else:
                t[b] = t[a]
        return
    if src.get_device() < 0:
        both = torch.stack((src, dst)).to(tensors[0].device, torch.int32)
        src, dst = both[0], both[1]
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            copy_pages(pools, src, dst)
        return
    src, dst = src.contiguous(), dst.contiguous()
    call("icb_copy_pages", _records(len(records))(*records), len(records) // 5, src.data_ptr(), dst.data_ptr(), n, stream_ptr())


@functools.lru_cache(maxsize=64)
def _records(n: int):
    return ctypes.c_longlong * n


# --------------------------------------------------------------------------- the 4-bit cache
def q4_pool_shape(num_blocks: int, kv_heads: int, block_size: int, head_dim: int) -> Tuple[int, int, int, int]:
    if block_size < 16 or block_size % 16:
        raise ValueError("block_size must be a multiple of 16")
    if head_dim not in Q4_HEAD_DIMS:
        raise ValueError(f"a 4-bit cache holds heads of {', '.join(map(str, Q4_HEAD_DIMS))}, not {head_dim}")
    return num_blocks, kv_heads, block_size // 16, 18 * head_dim


@functools.lru_cache(maxsize=64)
def _q4_shape(shape: torch.Size) -> Optional[Tuple[int, int, int, int]]:
    if len(shape) != 4 or shape[3] % 18 or shape[3] // 18 not in Q4_HEAD_DIMS or shape[1] < 1 or shape[2] < 1:
        return None
    return shape[0], shape[1], shape[2], shape[3] // 18


def _q4_sizes(pool: torch.Tensor) -> Tuple[int, int, int, int]:
    """(blocks, kv heads, tiles of a page, head size) of a pool."""
    sizes = _q4_shape(pool.shape)
    if sizes is None or pool.dtype != torch.uint8:
        raise ValueError(f"not a 4-bit pool: {pool.dtype} {tuple(pool.shape)}")
    if not pool.is_contiguous() or pool.data_ptr() % 16:
        raise ValueError("a 4-bit pool must be contiguous and start on a 16-byte boundary")
    return sizes


def _not_together(pool: torch.Tensor, **others) -> None:
    for name, t in others.items():
        if t is not None and t.device != pool.device:
            raise ValueError(f"{name} is on {t.device}, the pool on {pool.device}")


def _rows16(x: torch.Tensor) -> torch.Tensor:
    """Rows that 16-byte loads can read: neighbouring elements, aligned starts."""
    row, col = x.stride()
    return x if col == 1 and row % 8 == 0 and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


@functools.lru_cache(maxsize=512)
def _q4_plan(hd: int, per: int, dtype: torch.dtype, units: int, tiles: int) -> Tuple[int, int]:
    """(how the attention kernel runs a call, floats of scratch memory that it needs)."""
    plan = native.query("icb_paged_decode_q4_plan", hd, per, dtype_code(dtype), units, tiles)
    if plan == 0:
        raise RuntimeError(f"icb_paged_decode_q4 has no kernel for heads of {hd} in {dtype}")
    return plan, -plan * (16 + 8 * min(8, per) * (hd + 4)) if plan < 0 else 0


@functools.lru_cache(maxsize=16)
def _q4_places(hd: int, device: torch.device) -> torch.Tensor:
    """Byte of a tile for [token 0..15, byte]: hd / 2 bytes of key codes (elements 2 i, 2 i + 1), hd / 2 of value codes, the
    scales."""
    ng = hd // 32
    t = torch.arange(16, device=device)[:, None]
    d = torch.arange(0, hd, 2, device=device)[None, :]
    word = (t // 8) * ng + d // 32
    at = word // 4 * 512 + word % 4 * 4
    keys = at + (4 * (t % 8) + d % 32 // 8) * 16 + d % 8 // 2
    values = 8 * hd + at + (4 * (d % 32 // 4) + t % 8 // 2) * 16 + t % 2 * 2 + d % 4 // 2
    return torch.cat((keys, values, 16 * hd + t * 4 * ng + torch.arange(4 * ng, device=device)), 1)


def q4_quantize_reference(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """x [..., hd] -> codes uint8 [..., hd], scales fp16 [..., hd / 32]."""
    g = x.float().unflatten(-1, (-1, Q4_GROUP))
    most, least = g.amax(-1), g.amin(-1)
    scale = (torch.where(most >= -least, most, least) / -8.0).clamp(-65504.0, 65504.0).half()
    scale = torch.where(scale == 0, torch.zeros_like(scale), scale)
    n = torch.round(g / scale.float().unsqueeze(-1)).clamp(-8.0, 7.0)
    n = torch.where((scale == 0).unsqueeze(-1), torch.zeros_like(n), torch.nan_to_num(n, nan=0.0))
    return (n + 8.0).to(torch.uint8).flatten(-2), scale


def _q4_bytes_at(pool: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Index of every byte of the rows ``slots`` (valid ones) in the flat pool: [T, kv heads, 9 hd / 8]."""
    _, hkv, tiles, width = pool.shape
    block, inside = slots // (16 * tiles), slots % (16 * tiles)
    tile = (block[:, None] * hkv + torch.arange(hkv, device=pool.device)) * tiles + inside[:, None] // 16
    return tile[..., None] * width + _q4_places(width // 18, pool.device)[inside % 16][:, None, :]


def kv_append_q4_reference(k, v, pool, slots):
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    ok = (slots >= 0) & (slots < blocks * tiles * 16)
    (kc, ks), (vc, vs) = (q4_quantize_reference(x[ok].unflatten(1, (hkv, hd))) for x in (k, v))
    scales = torch.stack((ks, vs), 2).flatten(2).contiguous().view(torch.uint8)
    pool.view(-1)[_q4_bytes_at(pool, slots[ok])] = torch.cat((kc[..., 0::2] | kc[..., 1::2] << 4,
                                                              vc[..., 0::2] | vc[..., 1::2] << 4, scales), -1)


def kv_read_q4_reference(pool, slots, dtype=torch.float32):
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    ok = (slots >= 0) & (slots < blocks * tiles * 16)
    data = pool.view(-1)[_q4_bytes_at(pool, torch.where(ok, slots, torch.zeros_like(slots)))] if blocks else \
        torch.zeros((slots.numel(), hkv, 9 * hd // 8), dtype=torch.uint8, device=pool.device)
    n = torch.stack((data[..., :hd] & 15, data[..., :hd] >> 4), -1).flatten(-2).float() - 8.0
    both = n * data[..., hd:].contiguous().view(torch.float16).float().repeat_interleave(Q4_GROUP, -1)
    both = torch.where(ok[:, None, None], both, torch.zeros_like(both)).to(dtype)
    return both[..., :hd].flatten(1), both[..., hd:].flatten(1)


def paged_decode_q4_reference(q, pool, block_table, seq_lens, hq, scale, seqs=None):
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    bs, out = 16 * tiles, torch.zeros((q.shape[0], hq * hd), dtype=q.dtype, device=q.device)
    for i in range(q.shape[0]):
        row = i if seqs is None else int(seqs[i])
        n = min(int(seq_lens[i]), block_table.shape[1] * bs) if 0 <= row < block_table.shape[0] else 0
        if n <= 0:
            continue
        tok = torch.arange(n, device=q.device)
        page = block_table[row, tok // bs].long()
        tok, page = tok[(page >= 0) & (page < blocks)], page[(page >= 0) & (page < blocks)]
        if tok.numel() == 0:
            continue
        k, v = (x.view(-1, hkv, hd).repeat_interleave(hq // hkv, 1)
                for x in kv_read_q4_reference(pool, page * bs + tok % bs))
        # 64 bits: products of a query, a key and the scale pass the range of 32
        p = torch.softmax(torch.einsum("hd,nhd->hn", q[i].view(hq, hd).double(), k.double()) * scale, dim=-1).float()
        out[i] = torch.einsum("hn,nhd->hd", p, v).reshape(-1).to(q.dtype)
    return out


def kv_append_q4(k: torch.Tensor, v: torch.Tensor, pool: torch.Tensor, slots: torch.Tensor) -> None:
    """Quantise k, v [T, hkv * hd] (row views with arbitrary pitch) and write them to the cache rows ``slots`` (int64 [T],
    block * block_size + offset; rows with a slot outside the pool are left out). No two rows may have one slot: what it holds
    then is a mixture of both, codes and scales. Other slots are as they should be."""
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    shape, dtype = k.shape, k.dtype
    if len(shape) != 2 or shape != v.shape or shape[1] != hkv * hd or dtype != v.dtype:
        raise ValueError(f"rows of {hkv} heads of {hd} expected, got {tuple(shape)} {dtype} and {tuple(v.shape)} {v.dtype}")
    if slots.dtype != torch.int64 or slots.shape != shape[:1]:
        raise ValueError(f"slots must be int64 [{shape[0]}], got {slots.dtype} {tuple(slots.shape)}")
    dev = pool.get_device()
    if not k.get_device() == v.get_device() == slots.get_device() == dev:
        _not_together(pool, k=k, v=v, slots=slots)
    if dev < 0 or dtype not in _HALF:
        kv_append_q4_reference(k, v, pool, slots)
        return
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            kv_append_q4(k, v, pool, slots)
        return
    k, v, slots = _rows16(k), _rows16(v), slots.contiguous()
    call("icb_kv_append_q4", _ROWS_CALL(k.data_ptr(), v.data_ptr(), pool.data_ptr(), slots.data_ptr(), shape[0], hkv, hd, tiles,
                                        blocks * tiles * 16, k.stride(0), v.stride(0), _HALF[dtype]), stream_ptr())


def kv_read_q4(pool: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16
               ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [T, hkv * hd] of the cache rows ``slots`` (int64 [T]); zeros for a slot outside the pool."""
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise ValueError(f"slots must be int64 [T], got {slots.dtype} {tuple(slots.shape)}")
    dev = pool.get_device()
    if slots.get_device() != dev:
        _not_together(pool, slots=slots)
    if dev < 0 or dtype not in _HALF:
        if not dtype.is_floating_point:
            raise ValueError(f"cannot read a cache as {dtype}")
        return kv_read_q4_reference(pool, slots, dtype)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return kv_read_q4(pool, slots, dtype)
    t = slots.shape[0]
    k = pool.new_empty((t, hkv * hd), dtype=dtype)
    v = torch.empty_like(k)
    slots = slots.contiguous()
    call("icb_kv_read_q4", _ROWS_CALL(k.data_ptr(), v.data_ptr(), pool.data_ptr(), slots.data_ptr(), t, hkv, hd, tiles,
                                      blocks * tiles * 16, 0, 0, _HALF[dtype]), stream_ptr())
    return k, v


def paged_decode_q4(q: torch.Tensor, pool: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, hq: int,
                    scale: Optional[float] = None, *, seqs: Optional[torch.Tensor] = None,
                    out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, hq * hd] (row view, any pitch): row i against the first ``seq_lens[i]`` tokens of the sequence whose pages are
    row ``seqs[i]`` of ``block_table`` (int32; None: row i) -> [T, hq * hd], into ``out`` (rows of any pitch, apart) if given.
    A row without tokens gives zeros. Page numbers outside the pool and table rows outside the table hold no tokens. A NaN
    among the keys or values of a sequence makes the heads that read it NaN. ``scale``: up to 1e38 of either sign."""
    blocks, hkv, tiles, hd = _q4_sizes(pool)
    shape, dtype, i32 = q.shape, q.dtype, torch.int32
    if hq < 1 or hq % hkv:
        raise ValueError(f"{hq} query heads do not share {hkv} key / value heads evenly")
    if len(shape) != 2 or shape[1] != hq * hd:
        raise ValueError(f"query rows of {hq} heads of {hd} expected, got {tuple(shape)}")
    t, rows, per = shape[0], shape[:1], hq // hkv
    scale = hd ** -0.5 if scale is None else float(scale)
    if not abs(scale) <= 1e38:
        raise ValueError(f"a scale of {scale}")
    if block_table.dim() != 2 or block_table.dtype != i32 or seq_lens.dtype != i32 or seq_lens.shape != rows \
            or (seqs is not None and (seqs.dtype != i32 or seqs.shape != rows)):
        raise ValueError("block_table [S, pages], seq_lens [T] and seqs [T] must be int32")
    table_rows, pages = block_table.shape
    if seqs is None and table_rows < t:
        raise ValueError(f"{t} rows for {table_rows} rows of pages")
    if out is not None and (out.shape != shape or out.dtype != dtype or out.stride(1) != 1
                            or (t > 1 and out.stride(0) < shape[1])):
        raise ValueError("out must have q's shape and type, neighbouring elements and rows that do not overlap")
    dev = pool.get_device()
    if not q.get_device() == block_table.get_device() == seq_lens.get_device() == dev \
            or (seqs is not None and seqs.get_device() != dev) or (out is not None and out.get_device() != dev):
        _not_together(pool, q=q, block_table=block_table, seq_lens=seq_lens, seqs=seqs, out=out)
    if dev < 0 or dtype not in _HALF:
        res = paged_decode_q4_reference(q, pool, block_table, seq_lens, hq, scale, seqs)
        return res if out is None else out.copy_(res)
    if _elsewhere(dev):
        with torch.cuda.device(dev):
            return paged_decode_q4(q, pool, block_table, seq_lens, hq, scale, seqs=seqs, out=out)
    q, block_table, seq_lens = _rows16(q), block_table.contiguous(), seq_lens.contiguous()
    if out is None:     # the quicker of the two where rows do not overlap: contiguous rows then too
        out = torch.empty_like(q) if q.stride(0) >= shape[1] else q.new_empty(shape)
    if seqs is not None:
        seqs = seqs.contiguous()
    plan, floats = _q4_plan(hd, per, dtype, t * hkv * ((per + 7) // 8), pages * tiles)
    scratch = q.new_empty(floats, dtype=torch.float32) if floats else None
    call("icb_paged_decode_q4",
         _DECODE_CALL(q.data_ptr(), q.stride(0), pool.data_ptr(), block_table.data_ptr(),
                      seqs.data_ptr() if seqs is not None else 0, seq_lens.data_ptr(), out.data_ptr(), out.stride(0),
                      scratch.data_ptr() if scratch is not None else 0, t, hq, hkv, hd, tiles, pages, table_rows, blocks, plan,
                      scale, _HALF[dtype]), stream_ptr())
    return out

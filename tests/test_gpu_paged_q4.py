"""Kernels of the 4-bit paged cache and of page copies against the definition in 64 bits."""

import pytest
import torch

import q4_oracle as O
from helpers import tiny_config

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _rows(t, hkv, hd, dtype, seed=0, device="cuda"):
    """k, v as views of a packed projection, with groups of every kind among them."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((t, 3 * hkv * hd), generator=g) * 2.0 ** (16 * torch.rand((t, 3 * hkv * hd // 32), generator=g) - 8
                                                            ).repeat_interleave(32, 1)
    x = x.to(dtype)
    k, v = x[:, hkv * hd:2 * hkv * hd], x[:, 2 * hkv * hd:]
    k[0, :32] = 0
    v[t // 2] = torch.tensor([1.0, -1.0]).to(dtype).repeat(hkv * hd // 2)
    k[t - 1, :64] = torch.arange(-32, 32).to(dtype) / 4                      # quotients that are ties
    x = x.to(device)
    return x[:, hkv * hd:2 * hkv * hd], x[:, 2 * hkv * hd:]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hkv,hd,bs,t", [(2, 128, 16, 1), (12, 64, 32, 77), (1, 256, 16, 300), (3, 192, 48, 130), (8, 128, 64, 1000),
                                         (8, 128, 64, 2100), (2, 256, 16, 4200), (12, 64, 32, 2800), (5, 192, 48, 2200)])
def test_append_and_read(hkv, hd, bs, t, dtype):
    from ironcore_b200.ops import paged

    k, v = _rows(t, hkv, hd, dtype)
    blocks = -(-t // bs) + 3
    g = torch.Generator().manual_seed(1)
    start = torch.randint(0, 255, paged.q4_pool_shape(blocks, hkv, bs, hd), dtype=torch.uint8, generator=g)
    order = torch.randperm(blocks, generator=g)
    first = 5 % bs if t < blocks * bs - 5 else 0
    for name, slots in (("scattered", torch.randperm(blocks * bs, generator=g)[:t]),
                        ("in order", order[(torch.arange(t) + first) // bs] * bs + (torch.arange(t) + first) % bs),
                        ("some left out", torch.where(torch.rand(t, generator=g) < 0.3, -torch.ones(t, dtype=torch.int64),
                                                      order[torch.arange(t) // bs] * bs + torch.arange(t) % bs))):
        if t > 3 and name == "some left out":
            slots[1], slots[2] = blocks * bs, 2 ** 40
        want, got = start.clone(), start.clone().cuda()
        paged.kv_append_q4_reference(k.cpu(), v.cpu(), want, slots)
        paged.kv_append_q4(k, v, got, slots.cuda())
        assert torch.equal(got.cpu(), want), name
        for x, y in zip(paged.kv_read_q4(got, slots.cuda(), dtype), paged.kv_read_q4_reference(want, slots, dtype)):
            assert torch.equal(x.cpu().nan_to_num(), y.nan_to_num()), name
    # every row of the pool, stale ones included, in order and with both ends beyond it
    every = torch.arange(-3, blocks * bs + 5)
    for x, y in zip(paged.kv_read_q4(got, every.cuda(), dtype), paged.kv_read_q4_reference(want, every, dtype)):
        assert torch.equal(x.cpu().nan_to_num(), y.nan_to_num()) and torch.equal(x.cpu().isnan(), y.isnan())


def test_append_extreme_groups():
    from ironcore_b200.ops import paged

    for dtype, big in ((BF, 3e38), (HF, 65504.0)):
        k = torch.ones((7, 64), dtype=dtype)
        k[0, :32] = 0
        k[1, :32] = torch.tensor([1e-38, -1e-39] * 16).to(dtype)
        k[2, 3] = big
        k[3, 5] = float("-inf")
        k[4, 7] = float("nan")
        k[5, :32] = torch.tensor([2.0, -2.0] * 16)
        k[6, 0] = -1.0
        want = torch.zeros(paged.q4_pool_shape(1, 1, 16, 64), dtype=torch.uint8)
        got = want.cuda()
        paged.kv_append_q4_reference(k, k, want, torch.arange(7))
        paged.kv_append_q4(k.cuda(), k.cuda(), got, torch.arange(7).cuda())
        for x, y in zip(paged.kv_read_q4(got, torch.arange(7).cuda(), BF), paged.kv_read_q4_reference(want, torch.arange(7), BF)):
            assert torch.equal(x.cpu().nan_to_num(7.0), y.nan_to_num(7.0))
        codes = 16 * 64                                     # NaN scales may differ in their bits, codes may not
        assert torch.equal(got.cpu()[..., :codes], want[..., :codes])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_append_extreme_groups_among_many_rows(dtype):
    """Whole tiles with a group that fp16 scales do not hold exactly, that has none, or that is not finite."""
    from ironcore_b200.ops import paged

    hkv, hd, t = 8, 128, 2304
    k, v = (x.clone() for x in _rows(t, hkv, hd, dtype, seed=9, device="cpu"))
    for i, (x, value) in enumerate([(k, float("nan")), (v, float("-inf")), (v, float("nan")), (k, 3e38), (v, float("inf")), (k, 0.0)]):
        x[100 + 37 * i, 64 + i] = value
    for i, x in enumerate((k, v, k, v)):
        x[900 + 50 * i, 128:160] = torch.linspace(-3, 2.9, 32).to(dtype) * 2.0 ** -(23 + i)
        x[1500 + 50 * i, 32 * i:32 * i + 64] = 0
    blocks = t // 16 + 2
    slots = torch.randperm(blocks, generator=torch.Generator().manual_seed(0))[torch.arange(t) // 16] * 16 + torch.arange(t) % 16
    want = torch.zeros(paged.q4_pool_shape(blocks, hkv, 16, hd), dtype=torch.uint8)
    got = want.cuda()
    paged.kv_append_q4_reference(k, v, want, slots)
    paged.kv_append_q4(k.cuda(), v.cuda(), got, slots.cuda())
    codes = 16 * hd
    assert torch.equal(got.cpu()[..., :codes], want[..., :codes])
    scales = [x.cpu()[..., codes:].contiguous().view(HF) for x in (got, want)]
    assert torch.equal(scales[0].isnan(), scales[1].isnan()) and torch.equal(scales[0].nan_to_num(), scales[1].nan_to_num())
    for x, y in zip(paged.kv_read_q4(got, slots.cuda(), dtype), paged.kv_read_q4_reference(want, slots, dtype)):
        assert torch.equal(x.cpu().nan_to_num(), y.nan_to_num()) and torch.equal(x.cpu().isnan(), y.isnan())


def _widened(table, bs):
    """The table with room for 20000 tokens, which sends a call to the kernel that cuts all tiles into ranges."""
    return torch.cat((table, torch.full((table.shape[0], 20000 // bs), -1, dtype=torch.int32, device=table.device)), 1)


def _check(q, pool, table, lens, hq, scale=None, **kw):
    """Both kernels, by the width of the table; the result of the first."""
    from ironcore_b200.ops import paged

    hd, bs = pool.shape[3] // 18, 16 * pool.shape[2]
    want, tol = O.attention(q.cpu(), *O.decoded(pool), table.cpu(), lens.cpu(), hq, O.scale_of(hd) if scale is None else scale,
                            kw["seqs"].cpu() if "seqs" in kw else None)
    outs = []
    for t in (table, _widened(table, bs)):
        out = paged.paged_decode_q4(q, pool, t, lens, hq, scale, **kw)
        off = (out.cpu().double() - want).abs()
        assert bool(torch.isfinite(out).all())
        assert bool((off <= tol).all()), f"{float((off / tol).max()):.2f} of the tolerance"
        outs.append(out)
    return outs[0]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hq,hkv,hd,bs", [(2, 1, 64, 16), (12, 2, 128, 16), (12, 12, 64, 64), (8, 1, 256, 32), (16, 1, 128, 16),
                                          (11, 1, 192, 48), (10, 2, 64, 16), (32, 8, 128, 64)])
def test_attention(hq, hkv, hd, bs, dtype):
    lens = [1, 0, 15, 16, 17, 33, 2 * bs, 2 * bs + 1, 200, 129]
    pool, table, lens = O.cache(lens, hkv, hd, bs, dtype, seed=hq, device="cuda")
    q = (2 * torch.randn((10, (hq + 2 * hkv) * hd), generator=torch.Generator().manual_seed(1))).to(dtype).cuda()[:, :hq * hd]
    out = _check(q, pool, table, lens, hq)
    assert not out[1].any()


def test_attention_over_many_rows():
    """More (row, head) pairs than warps on the GPU, some rows empty."""
    g = torch.Generator().manual_seed(0)
    lens = [0 if x < 20 else x - 19 for x in torch.randint(0, 220, (304,), generator=g).tolist()]
    pool, table, lens = O.cache(lens, 8, 128, 16, BF, seed=11, device="cuda")
    q = torch.randn((304, 8 * 128), generator=g).to(BF).cuda()
    _check(q, pool, table, lens, 8)


@pytest.mark.parametrize("spread", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_over_long_contexts(hd, spread):
    pool, table, lens = O.cache([9000, 3, 0, 2777, 5000], 2, hd, 16, BF, seed=5, spread=spread, device="cuda")
    q = torch.randn((5, 6 * hd), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    _check(q, pool, table, lens, 6)


@pytest.mark.parametrize("hd,group", [(128, 6), (128, 2), (64, 3), (256, 1)])
def test_attention_of_blocks_over_long_rows(hd, group):
    """A block's warps at their longest: 16 (8 for larger heads) with 32 tiles each, beside rows of all lengths."""
    from ironcore_b200.ops import paged

    longest = 8192 if hd <= 128 else 4096
    lens = [longest, 1, 0, longest - 1, 17, 511, 513, longest // 2 + 5] + [16 * i + i % 3 for i in range(24)]
    pool, table, lens = O.cache(lens, 4, hd, 16, BF, seed=4, device="cuda")
    plan, _ = paged._q4_plan(hd, group, BF, 32 * 4, table.shape[1])
    assert plan == (16 if hd <= 128 else 8)
    _check(torch.randn((32, 4 * group * hd), generator=torch.Generator().manual_seed(1)).to(BF).cuda(), pool, table, lens,
           4 * group)


def test_attention_with_one_dominant_token():
    """A first token that takes nearly all probability and has tiny values, among values of ordinary size."""
    from ironcore_b200.ops import paged

    hd, n = 128, 2500
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn((n + 12, hd), generator=g) for _ in range(2))
    q = torch.randn((1, hd), generator=g)
    k[0] = q[0]
    v[0] *= 2.0 ** -13
    pool = torch.zeros(paged.q4_pool_shape(157, 1, 16, hd), dtype=torch.uint8)
    paged.kv_append_q4_reference(k.to(BF), v.to(BF), pool, torch.arange(n + 12))
    table, lens = torch.arange(157, dtype=torch.int32)[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda()
    for factor in (0.05, 0.15, 1.0):
        _check(q.to(BF).cuda(), pool.cuda(), table, lens, 1, factor)


@pytest.mark.parametrize("size", [2.0 ** -60, 1.0, 2.0 ** 60])
def test_attention_with_queries_of_any_size(size):
    pool, table, lens = O.cache([77, 300], 1, 128, 16, BF, seed=2, device="cuda")
    q = torch.randn((2, 4 * 128), generator=torch.Generator().manual_seed(1))
    q[0, 3:60] *= 2.0 ** -20                                # small elements beside large ones
    _check((q * size).to(BF).cuda(), pool, table, lens, 4, 0.09 / size)


@pytest.mark.parametrize("scale", [-0.1, 0.0, 1e-38])
@pytest.mark.parametrize("hq", [2, 8])
def test_attention_with_scales_of_any_sign(hq, scale):
    """Tokens outside the sequence stay outside whatever the scores are multiplied with."""
    pool, table, lens = O.cache([77, 300, 0, 1], 1, 128, 16, BF, seed=2, device="cuda")
    _check(torch.randn((4, hq * 128), generator=torch.Generator().manual_seed(1)).to(BF).cuda(), pool, table, lens, hq, scale)


def test_attention_in_place_and_over_nothing():
    """The output over the query rows; no rows, tables without pages or rows, pools without pages."""
    from ironcore_b200.ops import paged

    pool, table, lens = O.cache([77, 3000, 0, 16], 2, 64, 16, BF, seed=2, device="cuda")
    q = torch.randn((4, 6 * 64), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    for wide in (table, _widened(table, 16)):
        want, over = paged.paged_decode_q4(q, pool, wide, lens, 6), q.clone()
        assert paged.paged_decode_q4(over, pool, wide, lens, 6, out=over) is over and torch.equal(over, want)
    assert paged.paged_decode_q4(q[:0], pool, table, lens[:0], 6).shape == (0, 6 * 64)
    assert not paged.paged_decode_q4(q, pool, table[:, :0], lens, 6).any()
    assert not paged.paged_decode_q4(q, pool[:0], table, lens, 6).any()
    assert not paged.paged_decode_q4(q, pool, table[:0], lens, 6, seqs=torch.zeros(4, dtype=torch.int32, device="cuda")).any()
    none = torch.zeros(0, dtype=torch.int64, device="cuda")
    before = pool.clone()
    paged.kv_append_q4(q[:0, :128], q[:0, 128:256], pool, none)
    paged.kv_append_q4(q[:, :128], q[:, 128:256], pool[:0], torch.arange(4, device="cuda"))
    assert torch.equal(pool, before)
    assert paged.kv_read_q4(pool, none)[0].shape == (0, 128)
    assert not paged.kv_read_q4(pool[:0], torch.arange(4, device="cuda"))[1].any()


def test_attention_over_stale_pages():
    """NaN scales and any codes behind the last token, in unused pages and in pages of other sequences."""
    hkv, hd, bs = 2, 128, 32
    lens = [1, 17, 40, 0, 64]
    pool, table, dev_lens = O.cache(lens, hkv, hd, bs, BF, seed=3)
    stale = torch.ones((pool.shape[0], bs), dtype=torch.bool)
    for i, n in enumerate(lens):
        for p in range(n):
            stale[table[i, p // bs], p % bs] = False
    half = pool[..., 16 * hd:].contiguous().view(torch.float16).view(-1, hkv, bs // 16, 16, 8)
    mask = stale.view(-1, 1, bs // 16, 16, 1).expand_as(half)
    half = torch.where(mask, torch.tensor(float("nan"), dtype=HF), half)
    pool[..., 16 * hd:] = half.view(pool.shape[0], hkv, bs // 16, 128).contiguous().view(torch.uint8)
    q = torch.randn((5, 4 * hd), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    from ironcore_b200.ops import paged

    k, v = O.decoded(pool)
    want, tol = O.attention(q.cpu(), k.nan_to_num(), v.nan_to_num(), table, dev_lens, 4, O.scale_of(hd))
    for t in (_widened(table, bs), table):
        out = paged.paged_decode_q4(q, pool.cuda(), t.cuda(), dev_lens.cuda(), 4)
        assert bool(((out.cpu().double() - want).abs() <= tol).all())
    # a NaN among the tokens does reach its sequence, and no other
    row = pool[table[1, 0], 0, 0, 16 * hd:].view(torch.float16)
    row[0] = float("nan")
    again = paged.paged_decode_q4(q, pool.cuda(), table.cuda(), dev_lens.cuda(), 4)
    assert again[1, :2 * hd].isnan().all() and torch.equal(again[[0, 2, 3, 4]], out[[0, 2, 3, 4]])
    assert torch.equal(again[1, 2 * hd:], out[1, 2 * hd:])
    pool[table[0, 0], 1, 0, 16 * hd:16 * hd + 2] = torch.tensor([float("nan")], dtype=HF).view(torch.uint8)
    for t in (_widened(table, bs), table):
        again = paged.paged_decode_q4(q, pool.cuda(), t.cuda(), dev_lens.cuda(), 4)          # the only token of a sequence
        assert again[0, 2 * hd:].isnan().all() and bool(again[0, :2 * hd].isfinite().all())
    assert torch.equal(again[0, :2 * hd], out[0, :2 * hd])


def test_attention_calls_of_every_form():
    """Rows that name their sequence, one sequence several times, outputs and queries of odd pitch and alignment, page
    numbers and rows outside, lengths beyond the table."""
    from ironcore_b200.ops import paged

    hkv, hd, bs, hq = 2, 64, 16, 6
    pool, table, _ = O.cache([100, 60, 90], hkv, hd, bs, HF, seed=4)
    table[1, 1], table[2, 0] = -1, pool.shape[0]
    seqs = torch.tensor([2, 0, 0, 0, 1, 3, -1, 0], dtype=torch.int32).cuda()
    lens = torch.tensor([90, 100, 1, 50, 60, 9, 9, 112], dtype=torch.int32).cuda()
    assert table.shape[1] * bs == 112
    table[0, 6] = table[0, 5]                               # the whole row of the table holds pages
    wide = torch.randn((8, hq * hd + 24), generator=torch.Generator().manual_seed(1)).to(HF).cuda()
    pool, table = pool.cuda(), table.cuda()
    first = _check(wide[:, :hq * hd], pool, table, lens, hq, seqs=seqs)
    beyond = lens.clone()
    beyond[7] = 10 ** 9                                     # as many as the table has
    assert torch.equal(paged.paged_decode_q4(wide[:, :hq * hd], pool, table, beyond, hq, seqs=seqs), first)
    assert not first[5].any() and not first[6].any()
    for lo in (1, 8, 3):
        _check(wide[:, lo:lo + hq * hd], pool, table, lens, hq, seqs=seqs)
    # one query for all rows, columns before rows, a single row: as their contiguous copies
    for x in (wide[:1, :hq * hd].expand(8, -1), wide[:, :hq * hd].t().contiguous().t(), wide[2:3, 8:8 + hq * hd]):
        n = x.shape[0]
        got = paged.paged_decode_q4(x, pool, table, lens[:n], hq, seqs=seqs[:n])
        assert torch.equal(got, paged.paged_decode_q4(x.contiguous(), pool, table, lens[:n], hq, seqs=seqs[:n]))
        assert got.is_contiguous()
    into = torch.full((8, hq * hd + 3), 9.0, dtype=HF, device="cuda")
    paged.paged_decode_q4(wide[:, :hq * hd], pool, table, lens, hq, seqs=seqs, out=into[:, 1:1 + hq * hd])
    assert torch.equal(into[:, 1:1 + hq * hd], first) and bool((into[:, 0] == 9).all()) and bool((into[:, -2:] == 9).all())
    assert paged.paged_decode_q4(wide[:0, :hq * hd], pool, table, lens[:0], hq).shape == (0, hq * hd)
    nothing = paged.paged_decode_q4(wide[:, :hq * hd], pool, table[:, :0], lens, hq, seqs=seqs)
    assert not nothing.any()


def test_attention_is_reproducible_and_runs_on_other_streams():
    from ironcore_b200.ops import paged

    pool, table, lens = O.cache([1500, 700, 3, 0, 999], 4, 128, 16, BF, seed=6, device="cuda")
    q = torch.randn((5, 16 * 128), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    for table in (table, _widened(table, 16)):
        first = paged.paged_decode_q4(q, pool, table, lens, 16)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = []
        for i in range(6):
            with torch.cuda.stream(streams[i % 2]):
                outs.append(paged.paged_decode_q4(q, pool, table, lens, 16))
        torch.cuda.synchronize()
        assert all(torch.equal(o, first) for o in outs)


def test_attention_in_graphs():
    """Captured calls that share nothing, replayed in turn with lengths that change between replays."""
    from ironcore_b200.ops import paged

    sets = []
    for seed, hd, wide in ((7, 128, False), (8, 64, False), (9, 128, True), (10, 64, True)):
        pool, table, lens = O.cache([800, 50, 300], 2, hd, 16, BF, seed=seed, device="cuda")
        table = _widened(table, 16) if wide else table
        q = torch.randn((3, 8 * hd), generator=torch.Generator().manual_seed(seed)).to(BF).cuda()
        paged.paged_decode_q4(q, pool, table, lens, 8)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = paged.paged_decode_q4(q, pool, table, lens, 8)
        sets.append((q, pool, table, lens, graph, out))
    for now in ([800, 50, 300], [1, 0, 299], [17, 49, 0], [799, 16, 1]):
        for q, pool, table, lens, graph, out in sets:
            lens.copy_(torch.tensor(now, dtype=torch.int32))
            out.fill_(float("nan"))
        for _ in range(2):
            for s in sets:
                s[4].replay()
        for q, pool, table, lens, graph, out in sets:
            assert torch.equal(out, paged.paged_decode_q4(q, pool, table, lens, 8))
    q, pool, table, lens, graph, out = sets[0]
    want, tol = O.attention(q.cpu(), *O.decoded(pool), table.cpu(), lens.cpu(), 8, O.scale_of(128))
    assert bool(((out.cpu().double() - want).abs() <= tol).all())


@pytest.mark.parametrize("wide", [False, True])
def test_calls_follow_one_another(wide):
    """Every call reads what the one before wrote, with nothing in between: as with a synchronisation after each. Also from a
    graph that forks to another stream and joins."""
    from ironcore_b200.ops import paged

    hkv, hd, hq, bs = 2, 128, 8, 16
    first, table, lens = O.cache([40, 300, 5], hkv, hd, bs, BF, seed=3, device="cuda")
    lens = lens - 1
    table = _widened(table, bs) if wide else table
    blocks = first.shape[0]
    src, dst = (torch.tensor([b], dtype=torch.int32, device="cuda") for b in (int(table[1, 0]), blocks - 1))
    index = torch.arange(3, device="cuda")
    start = torch.randn((3, hq * hd), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    side = torch.cuda.Stream()

    def steps(pool, q, after, fork=False):
        outs = []
        for i in range(20):
            slots = table[index, (lens // bs).long()].long() * bs + lens.long() % bs
            paged.kv_append_q4(q[:, :hkv * hd], q[:, hkv * hd:2 * hkv * hd], pool, slots)
            after()
            out = paged.paged_decode_q4(q, pool, table, lens + 1, hq)
            after()
            if fork and i % 5 == 0:
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    extra = out.float().sum()
            paged.copy_pages(pool[None], src, dst)
            after()
            k, v = paged.kv_read_q4(pool, torch.arange(bs, device="cuda") + (blocks - 1) * bs)
            after()
            if fork and i % 5 == 0:
                torch.cuda.current_stream().wait_stream(side)
            q = paged.paged_decode_q4(out, pool, table, lens + 1, hq, out=out)
            after()
            paged.kv_append_q4(k[:1], v[:1], pool, slots[:1])
            after()
            outs += [q, k, v]
        return outs

    pool = first.clone()
    want = steps(pool, start, torch.cuda.synchronize)
    again = first.clone()
    for a, b in zip(steps(again, start, lambda: None), want):
        assert torch.equal(a, b)
    assert torch.equal(again, pool)
    pool.copy_(first)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = steps(again, start, lambda: None, fork=True)
    for _ in range(3):
        again.copy_(first)
        graph.replay()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_pools_larger_than_32_bit_offsets():
    """Pages on both sides of 2^31 and 2^32 bytes."""
    from ironcore_b200.ops import paged

    hkv, hd, bs = 8, 128, 64
    size = hkv * hd * 18 // 16 * bs
    blocks = 2 ** 32 // size + 3
    pool = torch.empty(paged.q4_pool_shape(blocks, hkv, bs, hd), dtype=torch.uint8, device="cuda")
    pages = torch.tensor([blocks - 1, 0, 2 ** 31 // size, blocks - 2, 2 ** 32 // size])
    k, v = _rows(5 * bs, hkv, hd, BF, seed=2)
    slots = (pages[:, None] * bs + torch.arange(bs)).flatten().cuda()
    small = torch.zeros(paged.q4_pool_shape(5, hkv, bs, hd), dtype=torch.uint8, device="cuda")
    paged.kv_append_q4(k, v, pool, slots)
    paged.kv_append_q4(k, v, small, torch.arange(5 * bs).cuda())
    assert torch.equal(pool[pages.cuda()], small)
    for x, y in zip(paged.kv_read_q4(pool, slots), paged.kv_read_q4(small, torch.arange(5 * bs).cuda())):
        assert torch.equal(x, y)
    q = torch.randn((1, 16 * hd), generator=torch.Generator().manual_seed(1)).to(BF).cuda()
    lens = torch.tensor([5 * bs - 7], dtype=torch.int32).cuda()
    assert torch.equal(paged.paged_decode_q4(q, pool, pages[None].int().cuda(), lens, 16),
                       paged.paged_decode_q4(q, small, torch.arange(5, dtype=torch.int32)[None].cuda(), lens, 16))
    paged.copy_pages([pool], [blocks - 1], [1])
    assert torch.equal(pool[1], small[0])


def test_copy_pages_kernel():
    from ironcore_b200.ops import paged

    g = torch.Generator().manual_seed(0)
    shapes = [((40, 16, 2, 64), BF), ((40, 5), torch.float32), ((41, 3), torch.uint8), ((40, 1, 7), HF), ((40, 33000), torch.uint8),
              ((40, 0), BF), ((50, 4096), torch.float32)]
    pools = [(100 * torch.randn(s, generator=g)).to(t) for s, t in shapes] * 15          # more than one launch
    dev = [p.cuda() for p in pools]
    src, dst = [3, 3, 0, 39], [1, 38, 2, 10]
    paged.copy_pages(dev, src, dst)
    for p, d in zip(pools, dev):
        p = p.clone()
        p[dst] = p[src]
        assert torch.equal(p, d.cpu())
    stack = torch.randint(0, 255, (3, 20, 2, 1, 18 * 64), dtype=torch.uint8, generator=g)
    got = stack.cuda()
    # device lists: pairs outside the pool are left out
    paged.copy_pages(got, torch.tensor([4, -1, 5, 20, 6], dtype=torch.int32).cuda(),
                     torch.tensor([0, 1, 20, 2, 19], dtype=torch.int32).cuda())
    stack[:, [0, 19]] = stack[:, [4, 6]]
    assert torch.equal(stack, got.cpu())
    one = torch.zeros(4000, dtype=torch.uint8, device="cuda").as_strided((1, 5), (3995, 1))     # a page by itself, an odd stride
    assert one.is_contiguous()
    paged.copy_pages([one], torch.zeros(1, dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32).cuda())
    views = torch.zeros((9, 5), dtype=torch.uint8, device="cuda").view(-1)[1:41].view(8, 5)      # odd addresses
    views[2] = torch.arange(5)
    paged.copy_pages([views], [2], [7])
    assert views[7].tolist() == [0, 1, 2, 3, 4] and int(views.sum()) == 20
    with pytest.raises(ValueError):
        paged.copy_pages(got, torch.tensor([4]).cuda(), torch.tensor([0]).cuda())
    with pytest.raises(ValueError):
        paged.copy_pages(got, torch.tensor([4], dtype=torch.int32).cuda(), [0])


def test_layer_caches_fork_rows_and_states():
    from ironcore_b200.layers.mixer import CacheSpec
    from ironcore_b200.rl import BlockKVCache, LayerCache

    spec = CacheSpec(rows={"k": 24, "v": 8}, states={"s": ((3, 5), torch.float32), "t": ((7,), None), "u": ((1,), None)})
    c = LayerCache([spec, spec], max_seqs=5, max_seq_len=64, device="cuda")
    b = BlockKVCache(3, 2, 64, 20, 16, 5, 64)
    pos = torch.arange(19, device="cuda")
    for cache in (c, b):
        a = cache.acquire()
        cache.reserve(a, 19)
        cache.advance(a, 19)
    for t in (*c.rows[0].values(), *c.rows[1].values(), *c.states[0].values(), *c.states[1].values(), *b.k, *b.v):
        t.normal_()
    before = [t.clone() for run in c.states for t in run.values()]
    forks, others = c.fork(a, 2), b.fork(a, 2)
    for i in forks:
        for run in c.rows:
            for t in run.values():
                assert torch.equal(t[c.slots_for(torch.full_like(pos, i), pos)], t[c.slots_for(torch.full_like(pos, a), pos)])
    for t, old in zip((t for run in c.states for t in run.values()), before):
        want = old.clone()
        want[forks] = old[a]
        assert torch.equal(t, want)
    for i in others:
        for t in b.k + b.v:
            t = t.view(-1, 128)
            assert torch.equal(t[b.slots_for(torch.full_like(pos, i), pos)], t[b.slots_for(torch.full_like(pos, a), pos)])


def test_refusals_on_the_gpu():
    from ironcore_b200.ops import paged

    pool = torch.zeros(paged.q4_pool_shape(2, 2, 16, 64), dtype=torch.uint8, device="cuda")
    rows, slots = torch.zeros((3, 128), dtype=BF, device="cuda"), torch.arange(3, device="cuda")
    for bad in ((rows.cpu(), rows.cpu(), slots), (rows, rows, slots.cpu())):
        with pytest.raises(ValueError):
            paged.kv_append_q4(bad[0], bad[1], pool, bad[2])
    q = torch.zeros((3, 256), dtype=BF, device="cuda")
    table, lens = torch.zeros((3, 1), dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
    for kw in (dict(q=q.cpu()), dict(block_table=table.cpu()), dict(seq_lens=lens.cpu()), dict(seqs=lens.cpu())):
        with pytest.raises(ValueError):
            paged.paged_decode_q4(**{**dict(q=q, pool=pool, block_table=table, seq_lens=lens, hq=4), **kw})
    with pytest.raises(ValueError):
        paged.kv_read_q4(pool, slots.cpu())
    # fp32 rows run on PyTorch operators
    k = torch.randn((3, 128), generator=torch.Generator().manual_seed(0))
    paged.kv_append_q4(k.cuda(), k.cuda(), pool, slots)
    assert torch.equal(paged.kv_read_q4(pool, slots, torch.float32)[0].cpu().double(), O.quantised(k.view(3, 2, 64)).flatten(1))


def _engine(bits, **kw):
    from ironcore_b200.config import validate_config
    from ironcore_b200.models import LanguageModel
    from ironcore_b200.parallel import mesh
    from ironcore_b200.rl import RolloutEngine

    mesh.destroy_model_parallel()
    cfg = tiny_config("qwen", d_model=256, d_ffn=512, num_layers=2, num_attention_heads=4, num_attention_groups=2, head_dim=128,
                      max_seq_len=128, max_position_embeddings=128, precision="bf16", vocab_size=1024, qkv_bias=True)
    cfg.data.vocab_size = 1024
    cfg.rl.kv_cache_bits = bits
    validate_config(cfg)
    torch.manual_seed(3)
    model = LanguageModel(cfg, device=torch.device("cuda")).cuda().eval()
    return model, RolloutEngine(model, cfg, max_seqs=6, max_seq_len=128, **kw)


@pytest.mark.parametrize("bits", [4, 16])
def test_rollouts(bits):
    """The whole path: prompt, quantised rows, captured decode steps, forks."""
    prompts = torch.randint(0, 1024, (2, 37), generator=torch.Generator().manual_seed(1))
    model, eager = _engine(bits, use_cuda_graph=False)
    t1, lp1 = eager.generate(prompts.repeat_interleave(3, dim=0), 24, temperature=0.0)
    _, graph = _engine(bits, use_cuda_graph=True)
    t2, lp2 = graph.generate(prompts, 24, temperature=0.0, samples=3)
    assert graph.cache.free_blocks == graph.cache.num_blocks
    full = model.token_logprobs(t1[:, :-1], t1[:, 1:])[:, 36:]
    assert bool(torch.isfinite(lp1).all()) and (full - lp1).abs().max().item() < (0.5 if bits == 4 else 0.15)
    assert t2.shape == t1.shape and torch.equal(t2[0], t2[1]) and torch.equal(t2[0], t2[2])
    again, lp3 = graph.generate(prompts, 24, temperature=0.0, samples=3)
    assert torch.equal(t2, again) and torch.equal(lp2, lp3)


@pytest.mark.parametrize("rows,heads", [(5, 2), (500, 8)])
def test_lengths_that_change_under_a_call(rows, heads):
    """Another stream overwrites the lengths while calls over ranges of tiles run: what such calls give is worthless, but nothing
    outside of their output is touched, and later calls are right. An entry for each unit, and one for each warp."""
    from ironcore_b200.ops import paged

    hd, bs = 64, 16
    g = torch.Generator().manual_seed(rows)
    most = 2000 if rows < 10 else 200
    pool, table, lens = O.cache([most] * rows, heads, hd, bs, BF, seed=1, device="cuda")
    table = _widened(table, bs)
    q = torch.randn((rows, heads * 2 * hd), generator=g).to(BF).cuda()
    plan, _ = paged._q4_plan(hd, 2, BF, rows * heads, table.shape[1])
    assert plan < 0 and (rows * heads <= -4 * plan) == (rows < 10)
    want = paged.paged_decode_q4(q, pool, table, lens, 2 * heads)
    now = lens.clone()
    others = [(torch.rand(rows, generator=g) ** 3 * (torch.rand(rows, generator=g) > 0.3) * most).int().cuda() for _ in range(20)]
    guarded = torch.full((rows + 4, heads * 2 * hd), 7.0, dtype=BF, device="cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for i in range(200):
        with torch.cuda.stream(side):
            for j in range(4):
                now.copy_(others[(i + j) % 20] if j % 2 else lens)
        paged.paged_decode_q4(q, pool, table, now, 2 * heads, out=guarded[2:-2])
    torch.cuda.synchronize()
    assert bool((guarded[:2] == 7).all()) and bool((guarded[-2:] == 7).all())
    assert torch.equal(paged.paged_decode_q4(q, pool, table, lens, 2 * heads), want)


@pytest.mark.parametrize("hq", [2, 8])
@pytest.mark.parametrize("scale", [1.0, 16.0, -64.0, 2.0 ** 12, 2.0 ** 30, -2.0 ** 30, 1e31, -1e31, 1e36, 1e38, -1e38])
@pytest.mark.parametrize("base", [-(2.0 ** 20), 2.0 ** 20, -3.0])
def test_attention_with_scores_of_any_size(hq, scale, base):
    """Scores ``scale`` * (``base`` + k / 8), k in -8 .. 7, whose dot products fp32 holds exactly: the softmax is that of the
    differences, equal ones share, and scores that are all very negative are no empty row. Tolerance: a weight is off by 2^-21 of
    1 + its distance in base 2 from the largest (the factor, its product with the difference and exp2, 2^-23 each); the product
    with the value's scale by 2^-11, times codes of up to 15; the output by half a step of bf16."""
    from ironcore_b200.ops import paged

    hd, n = 128, 700
    g = torch.Generator().manual_seed(5)
    k, v = torch.zeros((n + 4, hd)), torch.randn((n + 4, hd), generator=g)
    k[:, 0] = -4.0 if base > -4 and base < 0 else 4.0
    k[:, 32] = -1.0                                         # the scale of the second group, whatever the element that counts
    k[:, 40] = torch.randint(-8, 8, (n + 4,), generator=g) / 8.0
    q = torch.zeros((2, hq, hd))
    q[..., 0] = base / float(k[0, 0])
    q[..., 40] = 1.0
    q = q.view(2, hq * hd).to(BF)
    pool = torch.zeros(paged.q4_pool_shape(44, 1, 16, hd), dtype=torch.uint8)
    paged.kv_append_q4_reference(k.to(BF), v.to(BF), pool, torch.arange(n + 4))
    kk, vv = (x.flatten(0, 1)[:, 0] for x in O.decoded(pool))
    assert torch.equal(kk[:n + 4], k.double())
    table = torch.arange(44, dtype=torch.int32)[None].repeat(2, 1).cuda()
    lens = torch.tensor([n, 5], dtype=torch.int32).cuda()
    for t in (table, _widened(table, 16)):
        out = paged.paged_decode_q4(q.cuda(), pool.cuda(), t, lens, hq, scale).cpu().double().view(2, hq, hd)
        for row, m in enumerate((n, 5)):
            s = (kk[:m] @ q[row, :hd].double()) * scale
            p = torch.softmax(s, 0)
            off = 2.0 ** -21 * (1 + (s.max() - s).clamp(max=1e6) / 0.693)
            step = vv[:m].abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2) / 7
            want = p @ vv[:m]
            tol = 1.1 * (2.0 ** -11 * 15 * (p @ step) + 2 * ((p * off) @ vv[:m].abs()) + 2.0 ** -8 * want.abs()) + 1e-30
            assert bool(((out[row] - want).abs() <= tol).all())


@pytest.mark.parametrize("hq", [2, 8])
@pytest.mark.parametrize("big", [2.0 ** 18, -(2.0 ** 18)])
def test_attention_with_scores_of_all_sizes(hq, big):
    """Scores around ``big`` * {-4, 0, 3} * 64 in one row, the largest first, last or in between: between them only the largest
    count, in either kernel's order and where parts of a row are joined. Tolerance as above."""
    from ironcore_b200.ops import paged

    hd, n, scale = 128, 1500, 64.0
    g = torch.Generator().manual_seed(6)
    pools, rows = [], []
    for part in ((0, 400), (700, 720), (1100, n), (0, n), (n, n)):
        k, v = torch.zeros((n + 4, hd)), torch.randn((n + 4, hd), generator=g)
        low = torch.arange(n + 4) % 3 == 0                  # some very small ones everywhere
        k[:, 0] = torch.where(low, 3.0 if big < 0 else -4.0, 0.0)
        k[part[0]:part[1], 0] = torch.where(torch.rand(part[1] - part[0], generator=g) < 0.5, -4.0 if big < 0 else 3.0, 0.0)
        k[:, 1] = torch.where(torch.arange(n + 4) % 2 == 0, -4.0, 3.5)      # the scale of the first group, whatever counts
        k[:, 32] = -1.0
        k[:, 40] = torch.randint(-8, 8, (n + 4,), generator=g) / 8.0
        pools.append((k, v))
    pool = torch.zeros(paged.q4_pool_shape(94 * 5, 1, 16, hd), dtype=torch.uint8)
    for i, (k, v) in enumerate(pools):
        paged.kv_append_q4_reference(k.to(BF), v.to(BF), pool, torch.arange(n + 4) + 94 * 16 * i)
    q = torch.zeros((5, hq, hd))
    q[..., 0], q[..., 40] = big, 1.0
    q = q.view(5, hq * hd).to(BF)
    keys, values = (x.flatten(0, 1)[:, 0] for x in O.decoded(pool))
    table = torch.arange(94 * 5, dtype=torch.int32).view(5, 94).cuda()
    lens = torch.full((5,), n, dtype=torch.int32, device="cuda")
    for t in (table, _widened(table, 16)):
        out = paged.paged_decode_q4(q.cuda(), pool.cuda(), t, lens, hq, scale).cpu().double().view(5, hq, hd)
        for row in range(5):
            kk, vv = keys[94 * 16 * row:][:n], values[94 * 16 * row:][:n]
            s = (kk @ q[row, :hd].double()) * scale
            p = torch.softmax(s, 0)
            off = 2.0 ** -21 * (1 + (s.max() - s).clamp(max=1e6) / 0.693)
            step = vv.abs().unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(-1, -1, 32).flatten(-2) / 7
            want = p @ vv
            tol = 1.1 * (2.0 ** -11 * 15 * (p @ step) + 2 * ((p * off) @ vv.abs()) + 2.0 ** -8 * want.abs()) + 1e-30
            assert bool(((out[row] - want).abs() <= tol).all())


@pytest.mark.parametrize("size", [2.0 ** -126, 2.0 ** -110, 2.0 ** 116, 2.0 ** 120, 2.0 ** 125])
@pytest.mark.parametrize("hq", [2, 8])
def test_attention_with_queries_at_the_ends_of_their_type(hq, size):
    pool, table, lens = O.cache([77, 300], 1, 128, 16, BF, seed=2, device="cuda")
    q = torch.randn((2, hq * 128), generator=torch.Generator().manual_seed(1)).clamp(-3.5, 3.5)
    q = (q.double() * size).to(BF)
    assert bool(torch.isfinite(q).all())
    _check(q.cuda(), pool, table, lens, hq, 0.09 / size if size > 1 else 1e37)


@pytest.mark.parametrize("graph", [None, True])
@pytest.mark.parametrize("bits,precision,head_dim", [(4, "fp32", 64), (16, "fp32", 64), (4, "bf16", 256), (16, "bf16", 256)])
def test_rollouts_without_kernels_for_the_cache(bits, precision, head_dim, graph):
    """Types and head sizes for which the cache's operators are PyTorch's run eagerly, whatever is asked for; the others captured."""
    from ironcore_b200.config import validate_config
    from ironcore_b200.models import LanguageModel
    from ironcore_b200.parallel import mesh
    from ironcore_b200.rl import RolloutEngine

    mesh.destroy_model_parallel()
    cfg = tiny_config("qwen", d_model=256, d_ffn=512, num_layers=2, num_attention_heads=4, num_attention_groups=2, head_dim=head_dim,
                      max_seq_len=64, max_position_embeddings=64, precision=precision, vocab_size=512, qkv_bias=True)
    cfg.trainer.use_flash_attn = False
    cfg.rl.kv_cache_bits = bits
    validate_config(cfg)
    torch.manual_seed(3)
    model = LanguageModel(cfg, device=torch.device("cuda")).cuda().eval()
    eng = RolloutEngine(model, cfg, max_seqs=4, max_seq_len=64, use_cuda_graph=graph)
    prompts = torch.randint(0, 512, (2, 19), generator=torch.Generator().manual_seed(1))
    tokens, logps = eng.generate(prompts, 8, temperature=0.0, samples=2)
    assert eng.use_graph == (bits == 4 and precision == "bf16")
    assert any(g.graph is not None for g in eng._graphs.values()) == eng.use_graph
    full = model.token_logprobs(tokens[:, :-1], tokens[:, 1:])[:, 18:]
    assert bool(torch.isfinite(logps).all()) and (full - logps).abs().max().item() < (0.5 if bits == 4 else 0.15)


@pytest.mark.parametrize("bits", [4, 16])
def test_forked_captured_rollouts_follow_the_model(bits):
    """Log-probs of samples that share their prompt's pages and run in captured steps, against the model without a cache. Sampled,
    so that the forks differ; long enough for pages of their own."""
    _, graph = _engine(bits, use_cuda_graph=True)
    model = graph.model
    prompts = torch.randint(0, 1024, (2, 37), generator=torch.Generator().manual_seed(1))
    g = torch.Generator(device="cuda").manual_seed(2)
    for _ in range(2):                                      # the second time on graphs from the first step on
        tokens, logps = graph.generate(prompts, 40, temperature=1.0, samples=3, generator=g)
        assert any(x.graph is not None for x in graph._graphs.values())
        full = model.token_logprobs(tokens[:, :-1], tokens[:, 1:])[:, 36:]
        assert bool(torch.isfinite(logps).all()) and (full - logps).abs().max().item() < (0.5 if bits == 4 else 0.15)
        assert len({tuple(t) for t in tokens[:, 37:].tolist()}) == 6
    assert graph.cache.free_blocks == graph.cache.num_blocks


@pytest.mark.parametrize("t,hkv,hd", [(64, 2, 128), (4096, 8, 128)])
def test_append_to_a_row_twice(t, hkv, hd):
    """Rows of a call that share a slot leave something finite there and every other row of the pool as it should be."""
    from ironcore_b200.ops import paged

    k, v = _rows(t, hkv, hd, BF, seed=4)
    slots = torch.arange(t)
    for a in range(0, t, 50):
        slots[a + 7] = a + 3                                # breaks up tiles, and shares a slot of one
    shared = torch.zeros(t, dtype=torch.bool)
    shared[torch.arange(0, t, 50) + 3] = True
    want = torch.zeros(paged.q4_pool_shape(t // 16, hkv, 16, hd), dtype=torch.uint8)
    got = want.cuda()
    paged.kv_append_q4_reference(k.cpu(), v.cpu(), want, slots)
    paged.kv_append_q4(k, v, got, slots.cuda())
    for x, y in zip(paged.kv_read_q4(got, torch.arange(t).cuda(), BF), paged.kv_read_q4_reference(want, torch.arange(t), BF)):
        assert torch.equal(x.cpu()[~shared], y[~shared]) and bool(torch.isfinite(x).all())

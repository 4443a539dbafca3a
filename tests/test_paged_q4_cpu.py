"""The 4-bit paged cache on CPU: its format against the definition, its refusals, page copies, forks of sequences, rollouts
on it."""

import pytest
import torch

import q4_oracle as O
from helpers import tiny_config
from ironcore_b200.ops import paged


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("hd,hkv,bs", [(64, 3, 16), (128, 2, 32), (192, 1, 16), (256, 1, 48)])
def test_rows_go_in_and_come_out(hd, hkv, bs, dtype):
    g = torch.Generator().manual_seed(1)
    blocks, t = 3, 29
    k, v = (3 * torch.randn((t, hkv * hd), generator=g).to(dtype) for _ in range(2))
    pool = torch.randint(0, 255, paged.q4_pool_shape(blocks, hkv, bs, hd), dtype=torch.uint8, generator=g)
    before = pool.clone()
    slots = torch.randperm(blocks * bs, generator=g)[:t]
    slots[4], slots[5] = -1, blocks * bs                     # left out
    paged.kv_append_q4(k, v, pool, slots)
    ok = (slots >= 0) & (slots < blocks * bs)
    want = [O.quantised(x.unflatten(1, (hkv, hd))) for x in (k, v)]
    got = O.decoded(pool)
    for x, y in zip(got, want):
        assert torch.equal(x.flatten(0, 1)[slots[ok]], y[ok])
    untouched = torch.ones(blocks * bs, dtype=torch.bool)
    untouched[slots[ok]] = False
    for x, y in zip(got, O.decoded(before)):
        assert torch.equal(x.flatten(0, 1)[untouched].nan_to_num(), y.flatten(0, 1)[untouched].nan_to_num())
    out = paged.kv_read_q4(pool, slots, dtype)
    for x, y in zip(out, want):
        y = torch.where(ok[:, None, None], y, torch.zeros_like(y)).flatten(1)
        assert x.dtype == dtype and torch.equal(x, y.to(dtype))
    # a group of 32 is off by at most half a scale, the end opposite to its largest element by at most one
    far = k.double().unflatten(-1, (-1, 32)).abs().amax(-1, keepdim=True)
    off = (want[0].flatten(1) - k.double()).unflatten(-1, (-1, 32)).abs()
    assert bool((off <= far / 8 * (1 + 2 ** -10)).all())


def test_extreme_groups():
    """Zero groups, the smallest and the largest numbers, infinities, NaN: only the group that has them is touched."""
    hd = 64
    k = torch.ones((7, hd), dtype=torch.bfloat16)
    k[0, :32] = 0
    k[1, :32] = torch.tensor([1e-38, -1e-39] * 16)
    k[2, 3] = 3e38
    k[3, 5] = float("-inf")
    k[4, 7] = float("nan")
    k[5, :32] = torch.tensor([2.0, -2.0] * 16)               # equally far: the positive one is exact
    k[6, 0] = -1.0
    pool = torch.zeros(paged.q4_pool_shape(1, 1, 16, hd), dtype=torch.uint8)
    paged.kv_append_q4(k, k, pool, torch.arange(7))
    for x in paged.kv_read_q4(pool, torch.arange(7), torch.float32):
        assert torch.equal(x[:, 32:], torch.ones(7, 32))
        assert not x[0].any(dim=-1) or not x[0, :32].any()
        assert not x[1, :32].any()
        assert x[2, 3] == 8 * 65504 and x[3, 5] == -8 * 65504
        assert x[4, :32].isnan().all()
        assert torch.equal(x[5, :32], torch.tensor([2.0, -1.75] * 16))
        assert x[6, 0] == -0.875 and x[6, 1] == 1.0


@pytest.mark.parametrize("hq,hkv,hd,bs", [(4, 2, 64, 16), (6, 1, 128, 32), (2, 2, 192, 16), (10, 1, 256, 16)])
def test_attention_restatement(hq, hkv, hd, bs):
    lens = [1, 0, 17, 40, 2 * bs]
    pool, table, lens = O.cache(lens, hkv, hd, bs, torch.float32)
    q = torch.randn((5, hq * hd), generator=torch.Generator().manual_seed(2))
    out = paged.paged_decode_q4(q, pool, table, lens, hq)
    want, _ = O.attention(q, *O.decoded(pool), table, lens, hq, O.scale_of(hd))
    assert torch.allclose(out.double(), want, atol=1e-5)
    assert not out[1].any()
    seqs = torch.tensor([3, 3, 0], dtype=torch.int32)
    some = torch.tensor([40, 7, 1], dtype=torch.int32)
    into = torch.full((3, hq * hd + 8), 5.0)
    paged.paged_decode_q4(q[:3], pool, table, some, hq, 0.1, seqs=seqs, out=into[:, :hq * hd])
    want, _ = O.attention(q[:3], *O.decoded(pool), table, some, hq, 0.1, seqs)
    assert torch.allclose(into[:, :hq * hd].double(), want, atol=1e-5) and bool((into[:, hq * hd:] == 5).all())


def test_pages_and_rows_outside_hold_nothing():
    pool, table, _ = O.cache([40, 40], 2, 64, 16, torch.float32)
    q = torch.randn((4, 4 * 64), generator=torch.Generator().manual_seed(3))
    table[0, 1], table[1, 0] = -1, pool.shape[0]
    lens = torch.tensor([40, 40, 999, -3], dtype=torch.int32)
    seqs = torch.tensor([0, 1, 2, 1], dtype=torch.int32)
    out = paged.paged_decode_q4(q, pool, table, lens, 4, seqs=seqs)
    want, _ = O.attention(q, *O.decoded(pool), table, lens, 4, O.scale_of(64), seqs)
    assert torch.allclose(out.double(), want, atol=1e-5)
    assert not out[2].any() and not out[3].any()


def test_refusals():
    pool = torch.zeros(paged.q4_pool_shape(2, 2, 16, 64), dtype=torch.uint8)
    rows, slots = torch.zeros((3, 128)), torch.arange(3)
    for bad in ((2, 2, 8, 64), (2, 2, 24, 64), (2, 2, 16, 80), (2, 2, 16, 96), (2, 2, 16, 320)):
        with pytest.raises(ValueError):
            paged.q4_pool_shape(*bad)
    for p in (pool.int(), pool[0], pool[..., :600], pool[:, :1], torch.zeros((2, 2, 1, 18 * 80), dtype=torch.uint8)):
        with pytest.raises(ValueError):
            paged.kv_append_q4(rows, rows, p, slots)
        with pytest.raises(ValueError):
            paged.kv_read_q4(p, slots)
    for k, v, s in ((rows[:, :64], rows[:, :64], slots), (rows, rows[:2], slots), (rows, rows.half(), slots),
                    (rows, rows, slots.int()), (rows, rows, slots[:2]), (rows[0], rows[0], slots)):
        with pytest.raises(ValueError):
            paged.kv_append_q4(k, v, pool, s)
    with pytest.raises(ValueError):
        paged.kv_read_q4(pool, slots.int())
    with pytest.raises(ValueError):
        paged.kv_read_q4(pool, slots, torch.int8)
    q, table, lens = torch.zeros((3, 256)), torch.zeros((3, 1), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    paged.paged_decode_q4(q, pool, table, lens, 4)
    for a, kw in (((q, pool, table, lens, 3), {}), ((q, pool, table, lens, 2), {}), ((q, pool, table.long(), lens, 4), {}),
                  ((q, pool, table, lens.long(), 4), {}), ((q, pool, table, lens[:2], 4), {}), ((q, pool, table[:2], lens, 4), {}),
                  ((q, pool, table, lens, 4), {"seqs": lens.long()}), ((q, pool, table, lens, 4), {"out": torch.zeros((3, 128))}),
                  ((q, pool, table, lens, 4), {"out": torch.zeros((3, 256)).half()}), ((q, pool, table, lens, 0), {}),
                  ((q, pool, table, lens, 4, float("nan")), {}), ((q, pool, table, lens, 4, float("-inf")), {})):
        with pytest.raises(ValueError):
            paged.paged_decode_q4(*a, **kw)


def test_copy_pages():
    g = torch.Generator().manual_seed(0)
    pools = [torch.randn(6, 3, generator=g), torch.randint(0, 9, (7, 2, 5), generator=g)]
    before = [p.clone() for p in pools]
    paged.copy_pages(pools, [0, 0, 4], [1, 3, 5])
    for p, b in zip(pools, before):
        want = b.clone()
        want[[1, 3, 5]] = b[[0, 0, 4]]
        assert torch.equal(p, want)
    stack = torch.arange(24).view(2, 6, 2)
    want = stack.clone()
    want[:, 2] = want[:, 5]
    paged.copy_pages(stack, torch.tensor([5]), torch.tensor([2]))
    assert torch.equal(stack, want)
    paged.copy_pages(stack, [], [])
    paged.copy_pages([], [0], [1])
    for src, dst in (([0], [1, 2]), ([0], [6]), ([-1], [1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([0], [0]), ([0.5], [1])):
        with pytest.raises(ValueError):
            paged.copy_pages(pools, src, dst)
    with pytest.raises(ValueError):
        paged.copy_pages([pools[0].t()], [0], [1])


def test_forks_share_full_pages():
    from ironcore_b200.rl import QuantizedKVCache

    c = QuantizedKVCache(2, 1, 64, num_blocks=12, block_size=16, max_seqs=6, max_seq_len=96, device="cpu")
    a = c.acquire()
    c.reserve(a, 37)
    k = torch.randn((37, 64), generator=torch.Generator().manual_seed(0))
    slots = c.slots_for(torch.full((37,), a), torch.arange(37))
    for layer in range(2):
        c.append(layer, k + layer, -k, slots)
    c.advance(a, 37)
    c.seq_lens[a] = 37
    (b, d), = c.fork_many([a], 2)
    assert c.free_blocks == 12 - 3 - 2
    assert c.block_table[a, :2].tolist() == c.block_table[b, :2].tolist() == c.block_table[d, :2].tolist()
    assert len({int(c.block_table[s, 2]) for s in (a, b, d)}) == 3
    assert c.seq_lens[[a, b, d]].tolist() == [37] * 3 and c.length(d) == 37
    for layer in range(2):
        for x, y, z in zip(*(c.read(layer, s, torch.float32) for s in (a, b, d))):
            assert torch.equal(x, y) and torch.equal(x, z)
    # each goes on alone
    for s, val in ((a, 1.0), (b, 2.0), (d, 3.0)):
        c.reserve(s, 38)
        row = torch.full((1, 64), val)
        c.append(0, row, row, c.slots_for(torch.tensor([s]), torch.tensor([37])))
        c.advance(s, 38)
    for s, val in ((a, 1.0), (b, 2.0), (d, 3.0)):
        assert torch.equal(c.read(0, s, torch.float32)[0][37], torch.full((64,), val))
    c.release(a)
    assert c.free_blocks == 12 - 4                          # two shared pages are still held, two last pages
    c.drop_before(b, 32)
    assert c.free_blocks == 12 - 4
    assert not c.read(0, b, torch.float32)[0][:32].any() and c.read(0, d, torch.float32)[0][:32].any()
    c.release(d)
    assert c.free_blocks == 12 - 1
    c.release(b)
    assert c.free_blocks == 12
    assert sorted(c._free) == list(range(12)) and not any(c._holders)


def test_fork_is_all_or_nothing():
    from ironcore_b200.rl import BlockKVCache

    c = BlockKVCache(1, 1, 8, num_blocks=3, block_size=16, max_seqs=3, max_seq_len=64, dtype=torch.float32, device="cpu")
    a = c.acquire()
    c.reserve(a, 20)
    c.advance(a, 20)
    with pytest.raises(RuntimeError):
        c.fork(a, 3)                                        # sequences
    with pytest.raises(RuntimeError):
        c.fork(a, 2)                                        # pages
    with pytest.raises(ValueError):
        c.fork(a, -1)
    with pytest.raises(ValueError):
        c.fork(c._idle[0])                                  # nobody's sequence
    assert c.free_blocks == 1 and len(c._idle) == 2 and c.fork(a, 0) == []
    b, = c.fork(a)
    assert c.free_blocks == 0 and c.length(b) == 20


def _model(**kw):
    from ironcore_b200.config import validate_config
    from ironcore_b200.models import LanguageModel
    from ironcore_b200.parallel import mesh

    mesh.destroy_model_parallel()
    cfg = tiny_config("llama", max_seq_len=64, max_position_embeddings=64, **kw)
    cfg.trainer.use_flash_attn = False
    validate_config(cfg)
    torch.manual_seed(0)
    return cfg, LanguageModel(cfg).eval()


@pytest.mark.parametrize("bits", [16, 4])
def test_rollouts_with_forked_prompts(bits):
    """Greedy samples of a forked prompt are those of the prompt run by itself; sampled ones differ among each other."""
    from ironcore_b200.rl import RolloutEngine

    cfg, model = _model(head_dim=64, num_attention_heads=4)
    cfg.rl.kv_cache_bits = bits
    eng = RolloutEngine(model, cfg, max_seqs=6, max_seq_len=64, block_size=16)
    free = eng.cache.free_blocks
    prompts = torch.randint(0, 512, (2, 21), generator=torch.Generator().manual_seed(4))
    one, lp1 = eng.generate(prompts, 9, temperature=0.0)
    many, lp3 = eng.generate(prompts, 9, temperature=0.0, samples=3)
    assert torch.equal(many, one.repeat_interleave(3, dim=0))
    assert torch.allclose(lp3, lp1.repeat_interleave(3, dim=0), atol=1e-5)
    drawn, _ = eng.generate(prompts, 9, temperature=1.0, samples=3, generator=torch.Generator().manual_seed(0))
    assert torch.equal(drawn[:, :21], prompts.repeat_interleave(3, dim=0)) and not torch.equal(drawn[0], drawn[1])
    lists = [prompts[0].tolist(), prompts[1, :5].tolist(), prompts[1, :16].tolist()]
    alone, _ = eng.generate(lists, [4, 0, 6], temperature=0.0)
    got, _ = eng.generate(lists, [4, 0, 6], temperature=0.0, samples=2)
    assert got == [t for t in alone for _ in range(2)]
    assert eng.cache.free_blocks == free
    with pytest.raises(ValueError):
        eng.generate(prompts, 2, samples=7)
    eng.step([("a", lists[0], None)])
    eng.fork("a", ["b", "c"])
    logits = eng.step([("a", [7], None), ("b", [7], None), ("c", [9], None)])
    assert torch.allclose(logits[0], logits[1], atol=1e-5) and not torch.allclose(logits[0], logits[2], atol=1e-3)
    for bad in (("z", ["d"]), ("a", ["b"]), ("a", ["d", "d"])):
        with pytest.raises(ValueError):
            eng.fork(*bad)
    eng.end(["a", "b", "c"])
    assert eng.cache.free_blocks == free


def test_rollouts_on_four_bits():
    """The decode path equals the model run on the quantised keys and values: its own cache read back, in 64 bits."""
    from ironcore_b200.rl import RolloutEngine

    cfg, model = _model(head_dim=64, num_attention_heads=4, num_layers=1)
    cfg.rl.kv_cache_bits = 4
    eng = RolloutEngine(model, cfg, max_seqs=2, max_seq_len=64, block_size=16)
    toks = torch.randint(0, 512, (30,), generator=torch.Generator().manual_seed(5)).tolist()
    full = RolloutEngine(model, _model(head_dim=64, num_attention_heads=4, num_layers=1)[0], max_seqs=2, max_seq_len=64)
    a = eng.step([("r", toks, None)])
    b = full.step([("r", toks, None)])
    assert torch.allclose(a, b, atol=1e-5)                  # prompts attend in full precision
    got, near = eng.step([("r", [3], None)]), full.step([("r", [3], None)])
    assert not torch.equal(got, near)
    seq, other = eng._requests["r"], full._requests["r"]
    k, v = eng.cache.read(0, seq, torch.float32)
    pages = full.cache.block_table[other, :2].long()
    full.cache.k[0][pages] = torch.cat((k, torch.zeros(1, k.shape[1]))).view(2, 16, 2, 64)
    full.cache.v[0][pages] = torch.cat((v, torch.zeros(1, v.shape[1]))).view(2, 16, 2, 64)
    full.cache.advance(other, 30)
    full.cache.seq_lens[other] = 30
    # the same step again over the read-back rows; its own row is written in full precision, so set it afterwards
    real = full.cache.append
    full.cache.append = lambda li, kk, vv, s: (real(li, kk, vv, s), full.cache.k[0].view(-1, 128).__setitem__(s, k[30:31]),
                                               full.cache.v[0].view(-1, 128).__setitem__(s, v[30:31]))
    again = full.step([("r", [3], None)])
    assert torch.allclose(got, again, atol=1e-5)


def test_configuration_of_the_cache():
    from ironcore_b200.rl import QuantizedKVCache, RolloutEngine

    cfg, model = _model(head_dim=64, num_attention_heads=4)
    cfg.rl.kv_cache_bits = 4
    eng = RolloutEngine(model, cfg, max_seqs=2, max_seq_len=64)
    assert isinstance(eng.cache, QuantizedKVCache) and eng.cache.bytes_per_token() == 2 * 2 * 64 * 2 * 9 // 16
    cfg.rl.kv_cache_bits = 8
    with pytest.raises(ValueError):
        RolloutEngine(model, cfg, max_seqs=2, max_seq_len=64)
    cfg, model = _model()                                   # heads of 16
    cfg.rl.kv_cache_bits = 4
    with pytest.raises(ValueError):
        RolloutEngine(model, cfg, max_seqs=2, max_seq_len=64)


def test_layer_caches_fork_rows_and_states():
    from ironcore_b200.layers.mixer import CacheSpec
    from ironcore_b200.rl import LayerCache

    spec = CacheSpec(rows={"k": 8, "v": 4}, states={"s": ((3, 5), torch.float32), "t": ((7,), None)})
    c = LayerCache([spec], max_seqs=4, max_seq_len=64, dtype=torch.float32, device="cpu")
    a = c.acquire()
    c.reserve(a, 19)
    c.advance(a, 19)
    for t in (*c.rows[0].values(), *c.states[0].values()):
        t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(1)))
    b, d = c.fork(a, 2)
    pos = torch.arange(19)
    for name in ("k", "v"):
        rows = [c.rows[0][name][c.slots_for(torch.full((19,), s), pos)] for s in (a, b, d)]
        assert torch.equal(rows[0], rows[1]) and torch.equal(rows[0], rows[2])
    for name in ("s", "t"):
        assert torch.equal(c.states[0][name][a], c.states[0][name][b]) and torch.equal(c.states[0][name][a], c.states[0][name][d])


@pytest.mark.parametrize("family", ["tetepel", "kedavik"])
def test_residual_stream_models_fork_prompts(family):
    """Caches of rows and fixed-size states: forked prompts go on as the prompt run by itself, windows included."""
    import kedavik_cases as K
    import tetepel_cases as T

    if family == "tetepel":
        C, cfg = T, T.config([T.layer(window=5), T.layer(heads=2, window=11, ff=None)], streams=3, width=24)
        w = T.weights(cfg)
    else:
        C, cfg = K, K.config([K.mamba(), K.pair(chunk=9)])
        w = K.weights(cfg)
    model, c = C.build(cfg, w)
    eng = T.engine(model, c, max_seqs=6)
    prompts = [T.tokens(cfg, n, n) for n in (7, 16, 19)]
    alone, _ = eng.generate(prompts, 20, temperature=0.0)
    got, _ = eng.generate(prompts, 20, temperature=0.0, samples=3)
    assert got == [t for t in alone for _ in range(3)]
    assert eng.cache.free_blocks == eng.cache.num_blocks
    c.rl.kv_cache_bits = 4
    with pytest.raises(ValueError):
        T.engine(model, c)


@pytest.mark.parametrize("bits,share", [(16, True), (4, False), (4, True)])
def test_grpo_on_shared_prompts_and_four_bits(bits, share):
    from ironcore_b200.config import validate_config
    from ironcore_b200.parallel import mesh
    from ironcore_b200.rl.trainer import GRPOTrainer

    mesh.destroy_model_parallel()
    cfg = tiny_config("llama", max_seq_len=48, max_position_embeddings=48, head_dim=64)
    cfg.trainer.use_flash_attn = False
    cfg.rl(num_prompts=2, prompt_len=19, group_size=4, max_new_tokens=8, reward_vocab_subset=64, kv_cache_bits=bits,
           share_prompts=share)
    cfg.trainer(micro_batch_size=4, train_batch_size=4, gradient_accumulation_steps=None)
    cfg.operation.train_steps = 1
    validate_config(cfg)
    tr = GRPOTrainer(cfg)
    batch = tr.rollout()
    assert batch["tokens"].shape == (8, 27) and batch["logp_old"].shape == (8, 8)
    for i in range(0, 8, 4):
        assert bool((batch["tokens"][i:i + 4, :19] == batch["tokens"][i, :19]).all())
    st = tr.policy_update(batch)
    # the cache's rounding reaches the sampled tokens' log-probs, no more
    assert abs(st["ratio_mean"] - 1.0) < (1e-3 if bits == 16 else 0.2)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int16, torch.uint8, torch.float32])
@pytest.mark.parametrize("family", ["llama", "tetepel"])
def test_prompts_of_any_type(family, dtype):
    """Token ids reach the model in 64 bits, which its kernels read, whatever the prompts' type."""
    import tetepel_cases as T
    from ironcore_b200.rl import RolloutEngine

    if family == "llama":
        c, model = _model()
        eng, vocab = RolloutEngine(model, c, max_seqs=4, max_seq_len=64, block_size=16), 200
    else:
        cfg = T.config([T.layer(window=5)], streams=3, width=24)
        model, c = T.build(cfg, T.weights(cfg))
        eng, vocab = T.engine(model, c), min(200, cfg["vocab"])
    prompts = torch.randint(0, vocab, (2, 9), generator=torch.Generator().manual_seed(4))
    want, lp = eng.generate(prompts, 5, temperature=0.0)
    seen, real = [], eng.program.logits
    eng.program.logits = lambda batch: (seen.append(batch.tokens.dtype), real(batch))[1]
    got, lp2 = eng.generate(prompts.to(dtype), 5, temperature=0.0)
    assert set(seen) == {torch.int64}
    assert torch.equal(got, want) and torch.equal(lp, lp2)


@pytest.mark.parametrize("scale,size", [(1e31, 1.0), (-1e31, 1.0), (1e38, 1.0), (-1e38, 1.0), (1e38, 2.0 ** 120), (1e-42, 2.0 ** 125)])
def test_attention_restatement_at_the_ends(scale, size):
    """Scores beyond what fp32 holds: the largest takes all, equal ones share."""
    pool, table, lens = O.cache([30, 1, 17], 1, 64, 16, torch.float32)
    q = torch.randn((3, 2 * 64), generator=torch.Generator().manual_seed(2)) * size
    out = paged.paged_decode_q4(q, pool, table, lens, 2, scale)
    want, _ = O.attention(q, *O.decoded(pool), table, lens, 2, scale)
    assert torch.allclose(out.double(), want, atol=1e-5)


def test_which_decode_steps_a_graph_can_hold():
    """The restatements of the cache's operators read lengths on the host."""
    from ironcore_b200.rl import BlockKVCache, QuantizedKVCache, RolloutEngine

    sizes = dict(num_blocks=2, block_size=16, max_seqs=1, max_seq_len=32, device="cpu")
    for hd, dtype, plain, four in ((64, torch.bfloat16, True, True), (128, torch.float16, True, True), (256, torch.bfloat16, False, True),
                                   (64, torch.float32, False, False), (192, torch.float16, False, True)):
        assert BlockKVCache(1, 1, hd, dtype=dtype, **sizes).on_kernels(dtype) == plain
        assert QuantizedKVCache(1, 1, hd, **sizes).on_kernels(dtype) == four
    for bits in (16, 4):
        for kw in ({}, {"precision": "bf16"}):
            cfg, model = _model(head_dim=64, num_attention_heads=4, **kw)
            cfg.rl.kv_cache_bits = bits
            assert RolloutEngine(model, cfg, max_seqs=2, max_seq_len=64).program.capturable == bool(kw)


def test_outputs_that_overlap_are_refused():
    pool, table, lens = O.cache([7, 20], 1, 64, 16, torch.float32)
    q = torch.randn((2, 128), generator=torch.Generator().manual_seed(1))
    room = torch.zeros(400)
    for stride in (0, 1, 127):
        with pytest.raises(ValueError):
            paged.paged_decode_q4(q, pool, table, lens, 2, out=room.as_strided((2, 128), (stride, 1)))
    for n, stride in ((2, 128), (2, 131), (1, 0)):          # a single row has nothing to overlap
        got = paged.paged_decode_q4(q[:n], pool, table[:n], lens[:n], 2, out=room.as_strided((n, 128), (stride, 1)))
        assert torch.equal(got, paged.paged_decode_q4(q[:n], pool, table[:n], lens[:n], 2))


def _tp_rollout_worker(rank, world, out_path):
    from ironcore_b200.config import validate_config
    from ironcore_b200.models import LanguageModel
    from ironcore_b200.parallel import mesh
    from ironcore_b200.rl import RolloutEngine

    cfg = tiny_config("llama", max_seq_len=64, max_position_embeddings=64, head_dim=64, num_attention_heads=4)
    cfg.trainer.use_flash_attn = False
    cfg.trainer(tensor_model_parallel_size=world)
    cfg.parallel(world_size=world, rank=rank)
    cfg.rl.kv_cache_bits = 4
    validate_config(cfg)
    mesh.initialize_model_parallel(world)
    model = LanguageModel(cfg).eval()
    eng = RolloutEngine(model, cfg, max_seqs=6, max_seq_len=64, block_size=16)
    assert eng.cache.kv_heads == 2 // world
    prompts = torch.randint(0, 512, (2, 21), generator=torch.Generator().manual_seed(4))
    got = eng.generate(prompts, 12, temperature=0.0, samples=3)
    assert eng.cache.free_blocks == eng.cache.num_blocks
    if rank == 0:
        torch.save(got, out_path)


def test_rollouts_on_two_tensor_parallel_ranks_match_one(tmp_path):
    """Each rank holds its kv heads in 4 bits, groups being within heads: the same codes, forks and tokens as on one rank."""
    from helpers import run_distributed
    from ironcore_b200.parallel import mesh

    mesh.destroy_model_parallel()
    a, b = str(tmp_path / "one.pt"), str(tmp_path / "two.pt")
    run_distributed(_tp_rollout_worker, 1, a)
    run_distributed(_tp_rollout_worker, 2, b)
    (t1, lp1), (t2, lp2) = torch.load(a), torch.load(b)
    assert torch.equal(t1, t2) and torch.allclose(lp1, lp2, atol=1e-4)

"""The quantised decoder-layer operators on the GPU against 64-bit plain implementations (quant_oracle.py, which also
derives the tolerances): norm with 8-bit output, 8-bit product, 4-bit cache write, load and attention, and all of them in a
row."""
import math

import pytest
import torch

import quant_oracle as qo

pytestmark = pytest.mark.gpu
DTYPES = [torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def _randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen) * scale).to(dtype)


# ---- norm

NORM_SIZES = [(1, 1), (1, 7), (3, 64), (5, 100), (2, 4096), (64, 4096), (7, 4104), (3, 8192), (2, 16384), (2, 16392), (2, 20000),
              (300, 256), (129, 2048), (1, 65536)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,dim", NORM_SIZES)
def test_norm_quant_sizes(ops, dev, rows, dim, dtype):
    gen = _gen(rows * 100003 + dim)
    x, r = _randn(gen, (rows, dim), dtype), _randn(gen, (rows, dim), dtype, 5.0)
    gamma = _randn(gen, (dim,), dtype)
    for residual in (None, r):
        codes, scale, out = ops.rms_norm_quant(x.to(dev), gamma.to(dev), residual=None if residual is None else residual.to(dev))
        assert qo.norm_quant_ok(x, residual, gamma, 1e-5, codes.cpu(), scale.cpu(), out.cpu())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim,x_gap,r_gap", [(4096, 512, 8), (4096, 3, 1), (100, 28, 5)])
def test_norm_quant_strided_rows(ops, dev, dim, x_gap, r_gap, dtype):
    gen = _gen(dim + x_gap)
    x, r, gamma = _randn(gen, (9, dim + x_gap), dtype), _randn(gen, (9, dim + r_gap), dtype), _randn(gen, (dim,), dtype)
    dx, dr = x.to(dev), r.to(dev)
    codes, scale, out = ops.rms_norm_quant(dx[:, x_gap:], gamma.to(dev), residual=dr[:, :dim], epsilon=1e-6)
    assert qo.norm_quant_ok(x[:, x_gap:], r[:, :dim], gamma, 1e-6, codes.cpu(), scale.cpu(), out.cpu())
    assert torch.equal(dx.cpu(), x) and torch.equal(dr.cpu(), r)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [4096, 4099])
@pytest.mark.parametrize("into", ["x", "residual"])
def test_norm_quant_adds_in_place(ops, dev, into, dim, dtype):
    gen = _gen(dim)
    x, r, gamma = _randn(gen, (33, dim), dtype), _randn(gen, (33, dim), dtype), _randn(gen, (dim,), dtype)
    dx, dr = x.to(dev), r.to(dev)
    target = dx if into == "x" else dr
    codes, scale, out = ops.rms_norm_quant(dx, gamma.to(dev), residual=dr, residual_out=target)
    assert out is target
    assert qo.norm_quant_ok(x, r, gamma, 1e-5, codes.cpu(), scale.cpu(), out.cpu())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("dim", [256, 4096, 4099])
def test_norm_quant_special_rows(ops, dev, dim, dtype):
    """Zeros, subnormal and largest values; rows with an infinity or a NaN stand for NaN and do not touch the others."""
    gen = _gen(7)
    x = _randn(gen, (8, dim), dtype)
    big = torch.finfo(dtype).max
    x[0] = 0
    x[1] = x[1].sign() * big
    x[2] = x[2].sign() * (2.0 ** -24 if dtype == torch.float16 else 2.0 ** -130)
    x[3, dim // 2] = big
    x[4, dim - 1] = math.inf
    x[5, 0] = math.nan
    x[6] = 0
    x[6, 1] = -big
    gamma = _randn(gen, (dim,), dtype)
    codes, scale, _ = ops.rms_norm_quant(x.to(dev), gamma.to(dev))
    codes, scale = codes.cpu(), scale.cpu()
    for row in (4, 5):
        assert scale[row].isnan() and (codes[row] == 0).all()
    keep = [0, 1, 2, 3, 6, 7]
    assert qo.norm_quant_ok(x[keep], None, gamma, 1e-5, codes[keep], scale[keep], None)
    gamma[dim // 3] = math.nan
    codes, scale, _ = ops.rms_norm_quant(x.to(dev), gamma.to(dev))
    assert scale.cpu().isnan().all() and (codes.cpu() == 0).all()


# ---- linear

LINEAR_SIZES = [(1, 1, 1), (1, 16, 64), (3, 5, 17), (7, 48, 130), (16, 64, 256), (17, 4096, 512), (33, 1000, 1936), (64, 6144, 256),
                (64, 512, 4096), (65, 130, 96), (100, 257, 1023), (128, 256, 128), (129, 384, 640), (255, 512, 384), (256, 256, 4096),
                (300, 777, 555), (513, 640, 320), (1024, 1024, 256), (1, 10240, 8192), (5, 48, 16384), (2, 32, 65536)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("m,n,k", LINEAR_SIZES)
def test_linear_sizes(ops, dev, m, n, k, dtype):
    gen = _gen(m * 7919 + n * 31 + k)
    x = torch.randint(-128, 128, (m, k), generator=gen, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=gen, dtype=torch.int8)
    xs, ws = torch.rand((m,), generator=gen) + 0.01, (torch.rand((n,), generator=gen) + 0.01) * (0.01 / math.sqrt(k))
    for bias in (None, torch.randn((n,), generator=gen)):
        got = ops.linear_int8(x.to(dev), w.to(dev), xs.to(dev), ws.to(dev), bias=None if bias is None else bias.to(dev),
                              out_dtype=dtype).cpu().double()
        want, bound = qo.linear(x, w, xs, ws, bias, dtype)
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())


@pytest.mark.parametrize("m,n,k,off,x_gap,w_gap,o_gap", [(40, 96, 256, 0, 16, 32, 8), (40, 96, 256, 1, 3, 5, 1), (300, 520, 384, 16, 16, 16, 24),
                                                         (300, 520, 384, 0, 8, 0, 2), (3, 200, 1000, 0, 24, 8, 0),
                                                         (270, 300, 256, 4, 4, 4, 4)])
def test_linear_strided_matrices(ops, dev, m, n, k, off, x_gap, w_gap, o_gap):
    gen = _gen(m + n + k)
    x = torch.randint(-128, 128, (m, k + x_gap + off), generator=gen, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k + w_gap + off), generator=gen, dtype=torch.int8)
    xs, ws = torch.rand((m,), generator=gen), torch.rand((n,), generator=gen) * 1e-3
    out = torch.full((m, n + o_gap), 7.0, dtype=torch.float16, device=dev)
    ops.linear_int8(x.to(dev)[:, off:off + k], w.to(dev)[:, off:off + k], xs.to(dev), ws.to(dev), out=out[:, :n])
    want, bound = qo.linear(x[:, off:off + k], w[:, off:off + k], xs, ws, None, torch.float16)
    assert bool(((out[:, :n].cpu().double() - want).abs() <= bound).all())
    assert bool((out[:, n:] == 7.0).all())


@pytest.mark.parametrize("m,n", [(64, 96), (257, 300)])
@pytest.mark.parametrize("k", [131071, 131056])
def test_linear_longest_sums_stay_exact(ops, dev, m, n, k):
    """All factors at their extremes: the largest sums that 32 bits hold, of both signs."""
    x = torch.full((m, k), -128, dtype=torch.int8, device=dev)
    w = torch.full((n, k), -128, dtype=torch.int8, device=dev)
    w[1::2] = 127
    one = torch.ones((max(m, n),), device=dev)
    got = ops.linear_int8(x, w, one[:m], one[:n] * 2.0 ** -20, out_dtype=torch.bfloat16).cpu().double()
    want = torch.tensor([128.0 * 128 * k, -128.0 * 127 * k], dtype=torch.float64).repeat(n // 2) * 2.0 ** -20
    assert bool(((got - want).abs() <= (qo.U[torch.bfloat16] + 4 * qo.F32) * want.abs()).all())


# ---- 4-bit cache write and load


def _fresh(ops, blocks, heads, block, d, dtype, dev):
    """A cache whose every byte is known, so that what a call leaves alone can be seen."""
    cache = ops.new_int4_cache(blocks, heads, block, d, dtype, dev)
    cache[0].fill_(0x5A)
    cache[1].fill_(0xA5)
    cache[2].fill_(3.0)
    cache[3].fill_(-3.0)
    return cache


WRITE_SHAPES = [(1, 1, 64, 16), (5, 3, 64, 48), (33, 8, 128, 16), (200, 2, 128, 128), (77, 1, 256, 32), (130, 5, 256, 1024), (64, 8, 128, 128)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("order", ["runs", "shuffled"])
@pytest.mark.parametrize("tokens,heads,d,block", WRITE_SHAPES)
def test_write_then_rows(ops, dev, tokens, heads, d, block, order, dtype):
    """Written rows are what the definition makes of them; all other slots keep every byte. Slots in runs that begin
    anywhere and cross blocks (a prompt), or shuffled; skipped tokens among them."""
    gen = _gen(tokens * 31 + d)
    blocks = (tokens + 37) // block + 2
    slots = torch.randperm(blocks * block, generator=gen)[:tokens] if order == "shuffled" else torch.arange(tokens) + 13
    slots = slots.to(torch.int32)
    skipped = torch.zeros(tokens, dtype=torch.bool)
    if tokens > 4:
        skipped[torch.tensor([1, 3, tokens - 2])] = True
        slots[1], slots[3], slots[tokens - 2] = -1, blocks * block, -(2 ** 31)
    key, value = _randn(gen, (tokens, heads, d), dtype, 2.0), _randn(gen, (tokens, heads, d), dtype) + 1
    cache = _fresh(ops, blocks, heads, block, d, dtype, dev)
    before = [t.clone().cpu() for t in cache]
    ops.reshape_and_cache_int4(key.to(dev), value.to(dev), *cache, slots.to(dev))
    s = slots[~skipped].long()
    kc, vc, kp, vp = qo.token_rows(cache, s // block, s % block)
    assert qo.quantised_row_ok(key[~skipped], kc, kp)
    assert qo.quantised_row_ok(value[~skipped], vc, vp)
    after = [t.cpu() for t in cache]
    for old, new in ((before[0], after[0]), (before[2], after[2]), (before[3], after[3])):
        old[s // block, :, s % block] = new[s // block, :, s % block]
        assert torch.equal(old, new)
    before[1][s // block, :, :, s % block] = after[1][s // block, :, :, s % block]
    assert torch.equal(before[1], after[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gap", [64, 8, 1])
def test_write_from_a_fused_projection(ops, dev, gap, dtype):
    gen = _gen(gap)
    tokens, heads, d, block = 45, 4, 128, 32
    rows = _randn(gen, (tokens, 2 * heads * d + gap), dtype)
    key = rows[:, gap: gap + heads * d].unflatten(1, (heads, d))
    value = rows[:, gap + heads * d:].unflatten(1, (heads, d))
    dr = rows.to(dev)
    dk, dv = dr[:, gap: gap + heads * d].unflatten(1, (heads, d)), dr[:, gap + heads * d:].unflatten(1, (heads, d))
    cache = _fresh(ops, 3, heads, block, d, dtype, dev)
    slots = torch.arange(tokens, dtype=torch.int32) + 5
    ops.reshape_and_cache_int4(dk, dv, *cache, slots.to(dev))
    s = slots.long()
    kc, vc, kp, vp = qo.token_rows(cache, s // block, s % block)
    assert qo.quantised_row_ok(key, kc, kp) and qo.quantised_row_ok(value, vc, vp)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_write_special_rows(ops, dev, dtype):
    """Constant rows, zeros, the type's largest and smallest values, infinities and NaN."""
    gen = _gen(3)
    d, block = 128, 16
    big, small = torch.finfo(dtype).max, torch.finfo(dtype).smallest_normal
    x = _randn(gen, (10, 1, d), dtype)
    x[0] = 0
    x[1] = 1.5
    x[2] = x[2].sign() * big
    x[3] = x[3].sign() * small
    x[4] = small / 2
    x[4, 0, 5] = 0
    x[5, 0, 100] = math.inf
    x[6, 0, 3] = -math.inf
    x[7, 0, 0] = math.nan
    x[8] = -big
    x[8, 0, 77] = big
    cache = _fresh(ops, 1, 1, block, d, dtype, dev)
    slots = torch.arange(10, dtype=torch.int32)
    ops.reshape_and_cache_int4(x.to(dev), x.flip(0).contiguous().to(dev), *cache, slots.to(dev))
    kc, vc, kp, vp = qo.token_rows(cache, slots.long() // block, slots.long() % block)
    assert qo.quantised_row_ok(x, kc, kp)
    assert qo.quantised_row_ok(x.flip(0), vc, vp)
    assert kp[5:8].isnan().all()


def _random_cache(ops, gen, blocks, heads, block, d, dtype, dev):
    cache = ops.new_int4_cache(blocks, heads, block, d, dtype, dev)
    cache[0].copy_(torch.randint(0, 256, cache[0].shape, generator=gen, dtype=torch.uint8))
    cache[1].copy_(torch.randint(0, 256, cache[1].shape, generator=gen, dtype=torch.uint8))
    for p in cache[2:]:
        p[..., 0] = (torch.rand(p.shape[:-1], generator=gen) * 0.4 + 0.1).to(dtype).to(dev)
        p[..., 1] = torch.randn(p.shape[:-1], generator=gen).to(dtype).to(dev)
    return cache


def _tables(gen, lens, block, extra=0):
    """Shuffled pages with one owner each; entries behind a sequence's pages are no ids."""
    need = [max(0, -(-int(n) // block)) for n in lens]
    pool = sum(need) + 3
    perm = torch.randperm(pool, generator=gen).to(torch.int32)
    table = torch.full((len(need), max(need + [1]) + extra), -7, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at: at + n]
        at += n
    return table, pool


LOADS = [([1], None, 16, 2, 64), ([5, 0, 33, 16], None, 16, 3, 128), ([300, 17, 1, 128], [0, 5, 127, 40], 128, 2, 128),
         ([64, 64], [16, 15], 32, 1, 256), ([700, 3], [1, 0], 48, 8, 64), ([0, 0], None, 16, 1, 64)]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lens,starts,block,heads,d", LOADS)
def test_load_rows(ops, dev, lens, starts, block, heads, d, dtype):
    gen = _gen(sum(lens) + d)
    first = starts or [0] * len(lens)
    tables, pool = _tables(gen, [a + n for a, n in zip(first, lens)], block)
    cache = _random_cache(ops, gen, pool, heads, block, d, dtype, dev)
    total = sum(lens) + 2  # two rows behind the last sequence stay as they are
    key = torch.full((total, heads, d), 9.0, dtype=dtype, device=dev)
    value = torch.full((total, heads, d), -9.0, dtype=dtype, device=dev)
    ops.paged_cache_load_int4(*cache, tables.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev), total,
                              seq_starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=dev),
                              key=key, value=value)
    at = 0
    for b, n in enumerate(lens):
        kc, vc, kp, vp = (t[first[b]:] for t in qo.sequence_rows(cache, tables[b], first[b] + n, block))
        for got, codes, params in ((key, kc, kp), (value, vc, vp)):
            want = qo.decode(codes, params)
            size = params[..., 1:].double().abs() + 7.5 * params[..., :1].double()
            assert bool(((got[at: at + n].cpu().double() - want).abs() <= qo.U[dtype] * want.abs() + 4 * qo.F32 * size + qo.TINY[dtype]).all())
        at += n
    assert bool((key[at:] == 9.0).all()) and bool((value[at:] == -9.0).all())


def test_load_leaves_what_has_no_row(ops, dev):
    """Pages outside the pool, positions past the table, lengths below zero and past max_seq_len, rows past the output."""
    gen = _gen(11)
    cache = _random_cache(ops, gen, 6, 2, 16, 64, torch.float16, dev)
    tables = torch.tensor([[0, -1, 2], [5, 6, 1], [3, 4, 2 ** 31 - 1], [1, 1, 1]], dtype=torch.int32, device=dev)
    lens = torch.tensor([48, 40, -5, 60], dtype=torch.int32, device=dev)
    starts = torch.tensor([0, 0, 0, 20], dtype=torch.int32, device=dev)
    key = torch.full((140, 2, 64), 9.0, dtype=torch.float16, device=dev)
    value = key.clone()
    ops.paged_cache_load_int4(*cache, tables, lens, 140, seq_starts=starts, max_seq_len=45, key=key, value=value)
    touched = (key.cpu() != 9.0).any(-1).any(-1)
    want = torch.zeros(140, dtype=torch.bool)
    want[0:16] = want[32:45] = True            # sequence 0: its page -1 and its tokens past 45 stay
    want[48:64] = want[80:88] = True           # sequence 1: page 6 is outside the pool
    want[88:116] = True                        # sequence 3: positions 20 .. 47 of 48 that the table reaches
    assert torch.equal(touched, want)
    short = torch.full((50, 2, 64), 9.0, dtype=torch.float16, device=dev)
    ops.paged_cache_load_int4(*cache, tables, lens, 50, seq_starts=starts, key=short, value=short.clone())
    assert torch.equal(short[:16], key[:16]) and torch.equal(short[48:50], key[48:50])


# ---- attention


def _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens, mask=None):
    tables, pool = _tables(gen, lens, block)
    cache = _random_cache(ops, gen, pool, kv_heads, block, d, dtype, dev)
    query = _randn(gen, (len(lens) * tokens, heads, d), dtype)
    return query, cache, tables, torch.tensor(lens, dtype=torch.int32), 1.0 / math.sqrt(d)


def _check_attention(ops, dev, query, cache, tables, lens, scale, tokens, block, mask=None):
    got = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), lens.to(dev), scale, query_tokens=tokens,
                                   mask=None if mask is None else mask.to(dev)).cpu().double()
    want, bound = qo.attention(query, cache, tables, lens, scale, tokens, block, mask=mask)
    worst = ((got - want).abs() / bound.clamp_min(1e-30)).max()
    assert bool(((got - want).abs() <= bound).all()), float(worst)
    return got


ATTENTION = [
    # lens, heads, kv_heads, d, block, tokens
    ([1], 1, 1, 64, 16, 1),
    ([1, 2, 63, 64, 65], 4, 2, 64, 16, 1),
    ([500], 8, 2, 128, 128, 1),
    ([300, 0, 17, 1, 129], 8, 1, 128, 32, 1),
    ([257, 255], 20, 1, 128, 64, 1),       # more query heads a KV head than one tile of columns
    ([130, 70, 4], 8, 2, 128, 48, 4),      # several query tokens
    ([3, 2, 1, 200], 4, 4, 64, 16, 3),     # contexts no longer than the query tokens
    ([90, 190], 10, 2, 64, 16, 8),         # 40 columns a KV head
    ([140, 33], 4, 2, 256, 16, 1),
    ([600], 8, 2, 256, 128, 2),
    ([2500, 40], 4, 1, 128, 128, 1),       # cut over many workgroups
    ([37] * 70, 2, 1, 64, 16, 1),          # more sequences than a wave has lanes
    ([0, 0, 0], 2, 1, 64, 16, 2),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lens,heads,kv_heads,d,block,tokens", ATTENTION)
def test_attention_shapes(ops, dev, lens, heads, kv_heads, d, block, tokens, dtype):
    gen = _gen(sum(lens) + heads + d)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    _check_attention(ops, dev, query, cache, tables, n, scale, tokens, block)


def _mask(gen, kind, batch, heads, tokens, positions, dtype):
    if kind == "alibi":
        slope = torch.exp2(-torch.arange(1, heads + 1) * 8.0 / heads)
        return (-slope[:, None] * torch.arange(positions - 1, -1, -1)).to(dtype).reshape(1, heads, 1, positions)
    if kind == "rows":  # a mask row for each query token, with strides of its own
        m = torch.randn((batch, 1, tokens, positions), generator=gen).to(dtype)
        m[torch.rand(m.shape, generator=gen) < 0.4] = -math.inf
        return m
    low = -math.inf if kind == "-inf" else torch.finfo(dtype).min
    m = torch.zeros((batch, 1, 1, positions), dtype=dtype)
    for b in range(batch):
        m[b, :, :, : 5 * b] = low
    m[-1] = low  # a sequence that the mask empties
    return m


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["alibi", "rows", "-inf", "lowest"])
@pytest.mark.parametrize("d,tokens,extra", [(128, 1, 0), (64, 3, 5), (256, 2, -20)])
def test_attention_masks(ops, dev, d, tokens, extra, kind, dtype):
    """Additive masks of every broadcast form; -inf hides, the type's lowest value weighs a row of nothing else evenly;
    positions past the mask's length are hidden."""
    gen = _gen(d + tokens)
    lens, heads, kv_heads, block = [150, 64, 7, 201], 4, 2, 16
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    mask = _mask(gen, kind, len(lens), heads, tokens, max(lens) + extra, dtype)
    got = _check_attention(ops, dev, query, cache, tables, n, scale, tokens, block, mask)
    if kind == "-inf":
        assert bool((got[-tokens:] == 0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_never_sees_hidden_rows(ops, dev, dtype):
    """Codes and params of positions that no query sees may hold anything, NaN and infinities as well: past the length, in
    the future of a query token, behind a mask of -inf, in pages outside the pool."""
    gen = _gen(5)
    lens, heads, kv_heads, d, block, tokens = [100, 77, 40], 4, 2, 128, 16, 2
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    mask = torch.zeros((3, 1, 1, 100), dtype=dtype)
    mask[:, :, :, 10:30] = -math.inf
    tables[1, 2] = 10 ** 6
    tables[2, 1] = -1
    want = _check_attention(ops, dev, query, cache, tables, n, scale, tokens, block, mask)
    for b, length in enumerate(lens):
        places = list(range(10, 30)) + list(range(length, tables.shape[1] * block))
        for i, p in enumerate(places):
            page = int(tables[b, p // block])
            if 0 <= page < cache[0].shape[0]:
                for params in cache[2:]:
                    params[page, :, p % block] = math.nan if i % 2 else math.inf
    got = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), n.to(dev), scale, query_tokens=tokens,
                                   mask=mask.to(dev)).cpu().double()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_attention_nan_stays_in_its_row(ops, dev, dtype):
    """A NaN that is seen reaches the heads and sequences that see it, and no other."""
    gen = _gen(6)
    lens, heads, kv_heads, d, block = [70, 90], 4, 2, 64, 16
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, 1)
    want = _check_attention(ops, dev, query, cache, tables, n, scale, 1, block)
    cache[2][int(tables[0, 2]), 1, 3] = math.nan
    got = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), n.to(dev), scale).cpu().double()
    assert got[0, 2:].isnan().all()
    assert torch.equal(got[0, :2], want[0, :2]) and torch.equal(got[1], want[1])
    cache[2][int(tables[0, 2]), 1, 3] = 1.0
    cache[3][int(tables[1, 0]), 0, 7] = math.nan
    got = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), n.to(dev), scale).cpu().double()
    assert got[1, :2].isnan().all() and not got[1, 2:].isnan().any() and not got[0].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("values", [1e-3, 1.0, 300.0])
def test_attention_ranges_of_values(ops, dev, values, dtype):
    """Value scales far from one and scores that spread the weights over many powers of two."""
    gen = _gen(8)
    lens, heads, kv_heads, d, block = [400, 130], 8, 2, 128, 32
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, 1)
    cache[3].mul_(values)
    _check_attention(ops, dev, query * 4, cache, tables, n, scale, 1, block)


def test_attention_lengths_out_of_range(ops, dev):
    """Lengths below zero count as zero, those past the table as its reach; rows of empty sequences are zeros."""
    gen = _gen(9)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, [48, 48, 48], 4, 2, 64, 16, torch.float16, 1)
    n = torch.tensor([-3, 2 ** 31 - 1, 49], dtype=torch.int32)
    got = _check_attention(ops, dev, query, cache, tables, n, scale, 1, 16)
    assert bool((got[0] == 0).all())


# ---- together


def test_layer_half_in_a_row_and_captured(ops, dev):
    """Norm, projection, cache write, attention, projection for two decode steps, against the same steps from the 64-bit
    definitions; then captured into a graph and replayed, with eager work in between, bit for bit."""
    gen = _gen(21)
    dtype, batch, heads, kv_heads, d, block = torch.bfloat16, 3, 8, 2, 64, 16
    hidden = heads * d
    lens = [40, 17, 64]
    x = _randn(gen, (batch, hidden), dtype)
    residual = _randn(gen, (batch, hidden), dtype)
    gamma = _randn(gen, (hidden,), dtype, 0.1) + 1
    n_qkv = (heads + 2 * kv_heads) * d
    w1 = torch.randint(-127, 128, (n_qkv, hidden), generator=gen, dtype=torch.int8)
    w2 = torch.randint(-127, 128, (hidden, heads * d), generator=gen, dtype=torch.int8)
    s1 = torch.rand((n_qkv,), generator=gen) * 2e-3
    s2 = torch.rand((hidden,), generator=gen) * 2e-3
    tables, pool = _tables(gen, [n + 2 for n in lens], block)
    cache = _random_cache(ops, gen, pool, kv_heads, block, d, dtype, dev)
    on = lambda t: t.to(dev)  # noqa: E731
    dx, dres, dgamma, dw1, dw2, ds1, ds2, dtab = map(on, (x, residual, gamma, w1, w2, s1, s2, tables))
    dlens = torch.tensor([n + 1 for n in lens], dtype=torch.int32, device=dev)
    seq = torch.arange(batch)
    pos = torch.tensor(lens)
    slots = on((tables[seq, pos // block] * block + pos % block).to(torch.int32))
    scale = 1.0 / math.sqrt(d)

    def step():
        q8, qs, res = ops.rms_norm_quant(dx, dgamma, residual=dres)
        qkv = ops.linear_int8(q8, dw1, qs, ds1, out_dtype=dtype).unflatten(1, (-1, d))
        query = qkv[:, :heads].contiguous()
        ops.reshape_and_cache_int4(qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:], *cache, slots)
        att = ops.paged_attention_int4(query, *cache, dtab, dlens, scale)
        a8, as_, _ = ops.rms_norm_quant(att.flatten(1), torch.ones_like(dgamma))
        return q8, qs, res, qkv, att, a8, as_, ops.linear_int8(a8, dw2, as_, ds2, out_dtype=dtype)

    q8, qs, res, qkv, att, a8, as_, y = step()
    assert qo.norm_quant_ok(x, residual, gamma, 1e-5, q8.cpu(), qs.cpu(), res.cpu())
    want, bound = qo.linear(q8.cpu(), w1, qs.cpu(), s1, None, dtype)
    assert bool(((qkv.flatten(1).cpu().double() - want).abs() <= bound).all())
    kc, vc, kp, vp = qo.token_rows(cache, slots.cpu().long() // block, slots.cpu().long() % block)
    assert qo.quantised_row_ok(qkv[:, heads:heads + kv_heads].cpu(), kc, kp)
    assert qo.quantised_row_ok(qkv[:, heads + kv_heads:].cpu(), vc, vp)
    want, bound = qo.attention(qkv[:, :heads].cpu(), cache, tables, dlens, scale, 1, block)
    assert bool(((att.cpu().double() - want).abs() <= bound).all())
    assert qo.norm_quant_ok(att.flatten(1).cpu(), None, torch.ones_like(gamma), 1e-5, a8.cpu(), as_.cpu(), None)
    want, bound = qo.linear(a8.cpu(), w2, as_.cpu(), s2, None, dtype)
    assert bool(((y.cpu().double() - want).abs() <= bound).all())

    side = torch.cuda.Stream(device=dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(dev).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(4):
        dx.copy_(_randn(gen, (batch, hidden), dtype).to(dev))
        dlens.fill_(0).add_(torch.tensor([n + 1 for n in lens], dtype=torch.int32, device=dev) - i)
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in captured]
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(replayed, eager):
            assert torch.equal(a, b)


def test_calls_on_two_streams_and_repeated(ops, dev):
    """Two calls at once on streams of their own, and the same call again, give the same bits."""
    gen = _gen(22)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, [3000, 1200], 8, 2, 128, 128, torch.bfloat16, 1)
    args = (query.to(dev), *cache, tables.to(dev), n.to(dev), scale)
    want = ops.paged_attention_int4(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device=dev) for _ in range(2)]
    for _ in range(5):
        outs = []
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(ops.paged_attention_int4(*args))
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)


def test_a_moved_page_reads_the_same(ops, binding, dev):
    """atbmi_block_copy moves blocks of the 4-bit cache: codes in one call, params in another."""
    gen = _gen(23)
    heads, d, block = 2, 128, 16
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, [45], 4, heads, d, block, torch.float16, 1)
    want = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), n.to(dev), scale)
    free = [p for p in range(cache[0].shape[0]) if p not in tables.tolist()[0]][0]
    src = torch.tensor([int(tables[0, 1])], dtype=torch.int32, device=dev)
    dst = torch.tensor([free], dtype=torch.int32, device=dev)
    one = torch.tensor([1], dtype=torch.int32, device=dev)
    stream = torch.cuda.current_stream(dev).cuda_stream
    for a, b in ((cache[0], cache[1]), (cache[2], cache[3])):
        size = a[0].numel() * a.element_size()
        assert binding.kernels().atbmi_block_copy(a.data_ptr(), b.data_ptr(), src.data_ptr(), dst.data_ptr(), one.data_ptr(), 1, 1,
                                                  a.shape[0], size, size, stream) == 0
    cache[2][int(tables[0, 1])] = math.nan
    tables[0, 1] = free
    assert torch.equal(ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), n.to(dev), scale), want)

"""The quantised decoder-layer operators where offsets pass 32 bits: blocks at the end of a cache of more than 4 GB, matrices of more
than 2^32 values."""
import pytest
import torch

import quant_oracle as qo
from test_gpu_quantized import _gen, _randn

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    yield torch.device("cuda:0")
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d,block,tokens", [(128, 128, 700), (256, 48, 1100)])
def test_blocks_past_four_gigabytes(ops, dev, d, block, tokens):
    """Rows written into blocks at both ends of a large cache, read by the load and by attention: the bits of a small cache."""
    gen = _gen(d)
    heads, kv_heads, dtype = 8, 4, torch.bfloat16
    blocks = 2 ** 32 // (kv_heads * block * d // 2) + 40
    far = [torch.empty(shape, dtype=of, device=dev) for shape, of in (
        ((blocks, kv_heads, block, d // 2), torch.uint8), ((blocks, kv_heads, d // 2, block), torch.uint8),
        ((blocks, kv_heads, block, 2), dtype), ((blocks, kv_heads, block, 2), dtype))]
    assert far[0].numel() > 2 ** 32
    pages = -(-tokens // block)
    small = ops.new_int4_cache(pages, kv_heads, block, d, dtype, dev)
    near = torch.randperm(pages, generator=gen).to(torch.int32)
    ids = torch.where(near % 2 == 0, near, blocks - 1 - near).to(torch.int32)  # every other page at the far end
    key, value = _randn(gen, (tokens, kv_heads, d), dtype).to(dev), _randn(gen, (tokens, kv_heads, d), dtype).to(dev)
    query = _randn(gen, (1, heads, d), dtype).to(dev)
    lens = torch.tensor([tokens], dtype=torch.int32, device=dev)
    pos = torch.arange(tokens)
    got = []
    for cache, table in ((small, near), (far, ids)):
        slots = (table[pos // block].long() * block + pos % block).to(torch.int32).to(dev)
        ops.reshape_and_cache_int4(key, value, *cache, slots)
        tables = table.view(1, -1).contiguous().to(dev)
        got.append([*ops.paged_cache_load_int4(*cache, tables, lens, tokens),
                    ops.paged_attention_int4(query, *cache, tables, lens, 0.1)])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    kc, vc, kp, vp = qo.token_rows(small, near[pos // block].long(), pos % block)
    assert qo.quantised_row_ok(key.cpu(), kc, kp) and qo.quantised_row_ok(value.cpu(), vc, vp)


def test_linear_of_more_than_two_to_the_32_outputs(ops, dev):
    m, n, k = 2 ** 17 + 3, 2 ** 15 + 5, 64
    gen = torch.Generator(device=dev)
    gen.manual_seed(1)
    x = torch.randint(-128, 128, (m, k), generator=gen, device=dev, dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=gen, device=dev, dtype=torch.int8)
    xs, ws = torch.rand((m,), generator=gen, device=dev) + 0.01, torch.rand((n,), generator=gen, device=dev) * 1e-3
    out = ops.linear_int8(x, w, xs, ws, out_dtype=torch.bfloat16)
    assert out.numel() > 2 ** 32
    for rows in (slice(0, 300), slice(2 ** 16 - 100, 2 ** 16 + 100), slice(m - 300, m)):
        want, bound = qo.linear(x[rows], w, xs[rows], ws, None, torch.bfloat16)
        assert bool(((out[rows].double() - want).abs() <= bound).all())


def test_norm_of_more_than_two_to_the_32_values(ops, dev):
    rows, dim = 2 ** 19 + 9, 8192
    gen = torch.Generator(device=dev)
    gen.manual_seed(2)
    x = torch.randn((rows, dim), generator=gen, device=dev, dtype=torch.bfloat16)
    gamma = torch.randn((dim,), generator=gen, device=dev, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 32
    codes, scale, total = ops.rms_norm_quant(x, gamma, residual=x)
    for part in (slice(0, 20), slice(2 ** 18 - 10, 2 ** 18 + 10), slice(rows - 20, rows)):
        assert qo.norm_quant_ok(x[part].cpu(), x[part].cpu(), gamma.cpu(), 1e-5, codes[part].cpu(), scale[part].cpu(),
                                total[part].cpu())

"""Masked attention over the 4-bit cache with mask rows on 16-byte boundaries, which come through LDS a tile ahead, for every number
of columns that has a kernel of its own; and whole against cut sequences."""
import pytest
import torch

import quant_oracle as qo
from test_gpu_quantized import DTYPES, _attention_case, _gen, _mask
from test_gpu_quantized_cut import _wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _run(ops, dev, query, cache, tables, lens, scale, tokens, mask):
    got = ops.paged_attention_int4(query.to(dev), *cache, tables.to(dev), lens.to(dev), scale, query_tokens=tokens, mask=mask)
    return got.cpu().double()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["alibi", "rows", "-inf", "lowest"])
@pytest.mark.parametrize("d,heads,block,tokens,positions", [
    (64, 4, 64, 1, 704), (64, 8, 64, 1, 640), (64, 8, 16, 2, 704), (128, 8, 16, 1, 704), (128, 6, 128, 1, 712), (128, 2, 48, 4, 720),
    (128, 8, 128, 3, 704), (256, 4, 128, 1, 704), (256, 8, 32, 1, 648), (256, 5, 128, 3, 704)])
def test_masks_through_lds(ops, dev, d, heads, block, tokens, positions, kind, dtype):
    """Both with tables that let a workgroup take whole sequences and with wide ones, and the two against each other."""
    gen = _gen(d + heads + tokens + positions)
    lens = [650, 64, 7, 701, 129]
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, 1, d, block, dtype, tokens)
    mask = _mask(gen, kind, len(lens), heads, tokens, positions, dtype).to(dev)
    assert mask.data_ptr() % 16 == 0 and positions % 8 == 0
    want, bound = qo.attention(query, cache, tables, n, scale, tokens, block, mask=mask)
    whole = _run(ops, dev, query, cache, tables, n, scale, tokens, mask)
    cut = _run(ops, dev, query, cache, _wide(tables, block), n, scale, tokens, mask)
    for got in (whole, cut):
        assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound.clamp_min(1e-30)).max())
    assert bool(((whole - cut).abs() <= 2 * bound).all())
    # the same mask from an address that keeps it from LDS: the same bits
    room = torch.empty((mask.numel() + 1,), dtype=dtype, device=dev)
    odd = room[1:].view(mask.shape)
    odd.copy_(mask)
    assert torch.equal(_run(ops, dev, query, cache, tables, n, scale, tokens, odd), whole)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("heads,kv_heads,d,block,tokens", [(8, 2, 128, 128, 1), (8, 1, 64, 64, 1), (4, 1, 256, 16, 4)])
def test_whole_and_cut_lie_within_their_bounds_of_each_other(ops, dev, heads, kv_heads, d, block, tokens, dtype):
    gen = _gen(d)
    lens = [1000, 64, 1, 0, 513]
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    assert tables.shape[1] * block <= 1024
    whole = _run(ops, dev, query, cache, tables, n, scale, tokens, None)
    cut = _run(ops, dev, query, cache, _wide(tables, block, 4096), n, scale, tokens, None)
    want, bound = qo.attention(query, cache, tables, n, scale, tokens, block)
    assert bool(((whole - want).abs() <= bound).all()) and bool(((cut - want).abs() <= bound).all())
    assert bool(((whole - cut).abs() <= 2 * bound).all())

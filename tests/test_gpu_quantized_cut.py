"""Attention over the 4-bit cache where sequences are cut over workgroups: tables that reach far (whatever the lengths are),
every number of columns that has a kernel of its own, masks, empty and short sequences beside long ones; and its workspace."""
import ctypes
import math

import pytest
import torch

import quant_oracle as qo
from test_gpu_quantized import DTYPES, _attention_case, _check_attention, _gen, _mask

pytestmark = pytest.mark.gpu
REACH = 2200  # positions: more than any number of whole sequences is worked on for


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _wide(tables, block, reach=REACH):
    """The same tables with entries that are no ids behind them."""
    more = max(0, -(-reach // block) - tables.shape[1])
    return torch.cat([tables, torch.full((tables.shape[0], more), -1, dtype=torch.int32)], 1).contiguous()


SHAPES = [
    # lens, heads, kv_heads, d, block, tokens
    ([1], 4, 1, 64, 16, 1),
    ([65, 0, 64, 1, 700, 127], 8, 2, 128, 128, 1),
    ([1100, 3, 0, 0, 320], 2, 2, 128, 16, 1),
    ([640, 500], 8, 1, 128, 64, 1),             # 8 columns
    ([513, 20, 900], 16, 2, 64, 128, 1),
    ([410, 130], 8, 2, 256, 128, 2),
    ([150, 1000], 4, 1, 256, 48, 4),            # 16 columns
    ([333, 256, 2], 10, 2, 128, 128, 8),        # 40 columns
    ([2200, 17], 2, 1, 128, 128, 3),
    ([40] * 67 + [1000], 4, 2, 64, 16, 1),
]


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("lens,heads,kv_heads,d,block,tokens", SHAPES)
def test_cut_sequences(ops, dev, lens, heads, kv_heads, d, block, tokens, dtype):
    gen = _gen(sum(lens) + heads * 3 + d)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    _check_attention(ops, dev, query, cache, _wide(tables, block), n, scale, tokens, block)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("kind", ["alibi", "rows", "-inf", "lowest"])
@pytest.mark.parametrize("d,heads,block,tokens,positions", [(128, 4, 128, 1, 704), (128, 8, 16, 1, 705), (64, 4, 64, 3, 640),
                                                            (256, 2, 32, 2, 600), (128, 8, 128, 4, 701)])
def test_cut_sequences_with_masks(ops, dev, d, heads, block, tokens, positions, kind, dtype):
    gen = _gen(d + tokens + positions)
    lens, kv_heads = [650, 64, 7, 701], 1
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, dtype, tokens)
    mask = _mask(gen, kind, len(lens), heads, tokens, positions, dtype)
    got = _check_attention(ops, dev, query, cache, _wide(tables, block), n, scale, tokens, block, mask)
    if kind == "-inf":
        assert bool((got[-tokens:] == 0).all())


@pytest.mark.parametrize("d,tokens", [(64, 1), (128, 2), (256, 1)])
def test_workspace_is_enough_and_needs_no_content(ops, binding, dev, d, tokens):
    gen = _gen(d)
    lens, heads, kv_heads, block = [1500, 900, 30], 4, 2, 32
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, torch.float16, tokens)
    tables = _wide(tables, block)
    call = binding.AtbmiPaInt4Call(dtype=binding.ATBMI_F16, numHeads=heads, numKvHeads=kv_heads, headDim=d, blockSize=block,
                                   numBlocks=cache[0].shape[0], maxBlocksPerSeq=tables.shape[1], batch=len(lens),
                                   queryTokens=tokens, qkScale=scale)
    need = ctypes.c_uint64()
    assert binding.kernels().atbmi_pa_int4_workspace_size(ctypes.byref(call), ctypes.byref(need)) == 0 and need.value > 0
    room = torch.full((need.value + 4096,), 0xFF, dtype=torch.uint8, device=dev)  # (NaN where it is read as numbers)
    args = (query.to(dev), *cache, tables.to(dev), n.to(dev), scale)
    want = ops.paged_attention_int4(*args, query_tokens=tokens)
    for _ in range(2):
        got = ops.paged_attention_int4(*args, query_tokens=tokens, workspace=room[:need.value])
        assert torch.equal(got, want)
    assert bool((room[need.value:] == 0xFF).all())
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_attention_int4(*args, query_tokens=tokens, workspace=room[:need.value - 16])
    bad, bound = qo.attention(query, cache, tables, n, scale, tokens, block)
    assert bool(((want.cpu().double() - bad).abs() <= bound).all())


def test_two_captured_graphs_in_turn(ops, dev):
    """Two graphs whose calls took their workspaces while being captured, replayed in turn with eager calls in between."""
    gen = _gen(5)
    cases = []
    for lens, block in (([1800, 40], 128), ([700, 1300, 5], 16)):
        query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, 8, 2, 128, block, torch.bfloat16, 1)
        args = (query.to(dev), *cache, _wide(tables, block).to(dev), n.to(dev), scale)
        want = ops.paged_attention_int4(*args)
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = ops.paged_attention_int4(*args)
        cases.append((args, want, graph, out))
    for i in range(4):
        for args, want, graph, out in cases if i % 2 else reversed(cases):
            graph.replay()
            assert torch.equal(ops.paged_attention_int4(*args), want)
            torch.cuda.synchronize()
            assert torch.equal(out, want)
            out.zero_()


def test_whole_and_cut_agree(ops, dev):
    """The same call with tables that reach 1024 positions and 4096: one workgroup a sequence, and cut."""
    gen = _gen(8)
    lens = [1000, 64, 1, 0, 513]
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, 8, 2, 128, 128, torch.float16, 1)
    assert tables.shape[1] * 128 <= 1024
    a = _check_attention(ops, dev, query, cache, tables, n, scale, 1, 128)
    b = _check_attention(ops, dev, query, cache, _wide(tables, 128, 4096), n, scale, 1, 128)
    assert bool((a[3] == 0).all()) and bool((b[3] == 0).all()) and not math.isnan(float((a - b).abs().max()))

"""The quantised decoder-layer operators as atb::Operations on the GPU (the same bits as the torch functions, whose results
test_gpu_quantized.py holds against 64 bits), and the write of many tokens at once."""
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


def _same(a, b):
    return a.dtype == b.dtype and a.shape == b.shape and torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


def _layer(gen, dtype, d, block, dev):
    """Tensors of a decode step of three sequences: 8 query heads over 2 KV heads."""
    batch, heads, kv_heads, hidden = 3, 8, 2, 512
    n = (heads + 2 * kv_heads) * d
    t = dict(x=torch.randn(batch, hidden, generator=gen).to(dtype), residual=torch.randn(batch, hidden, generator=gen).to(dtype),
             gamma=(1 + 0.1 * torch.randn(hidden, generator=gen)).to(dtype),
             w=torch.randint(-127, 128, (n, hidden), generator=gen, dtype=torch.int8), ws=torch.rand(n, generator=gen) * 2e-3,
             bias=torch.randn(n, generator=gen))
    lens = [70, 1, 33]
    reach = 5 * 16 // block + 1
    t["tables"] = torch.randperm(batch * reach, generator=gen).view(batch, reach).to(torch.int32)
    seq, pos = torch.arange(batch), torch.tensor(lens) - 1
    t["slots"] = (t["tables"][seq, pos // block] * block + pos % block).to(torch.int32)
    t["lens"] = torch.tensor(lens, dtype=torch.int32)
    old = torch.randn(2, batch * reach * block, kv_heads, d, generator=gen).to(dtype)
    t["old_key"], t["old_value"] = old[0].contiguous(), old[1].contiguous()
    t["all_slots"] = torch.arange(batch * reach * block, dtype=torch.int32)
    return {k: v.to(dev) for k, v in t.items()}, heads, kv_heads, batch * reach


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d,block", [(64, 16), (128, 48), (256, 32)])
def test_operations_in_a_row(ops, binding, dev, d, block, dtype):
    """A decode step through atb::Operations on a stream of its own, against the functions."""
    t, heads, kv_heads, blocks = _layer(_gen(d), dtype, d, block, dev)
    split = (heads * d, kv_heads * d, kv_heads * d)
    scale = 1.0 / math.sqrt(d)
    mask = (torch.randn(1, heads, 1, 90, generator=_gen(1)) * 2).to(dtype).to(dev)
    starts, lens = torch.tensor([5, 0, 20], dtype=torch.int32, device=dev), torch.tensor([60, 1, 13], dtype=torch.int32, device=dev)

    want_cache = ops.new_int4_cache(blocks, kv_heads, block, d, dtype, dev)
    ops.reshape_and_cache_int4(t["old_key"], t["old_value"], *want_cache, t["all_slots"])
    want = list(ops.rms_norm_quant(t["x"], t["gamma"], residual=t["residual"], epsilon=1e-6))
    want.append(ops.linear_int8(want[0], t["w"], want[1], t["ws"], bias=t["bias"], out_dtype=dtype))
    q, k, v = (p.unflatten(1, (-1, d)).contiguous() for p in want[3].split(split, 1))
    ops.reshape_and_cache_int4(k, v, *want_cache, t["slots"])
    want.append(ops.paged_attention_int4(q, *want_cache, t["tables"], t["lens"], scale, mask=mask))
    want.append(ops.paged_attention_int4(q, *want_cache, t["tables"], t["lens"], scale))
    rows = torch.full((80, kv_heads, d), 7.0, dtype=dtype, device=dev), torch.full((80, kv_heads, d), 7.0, dtype=dtype, device=dev)
    want += ops.paged_cache_load_int4(*want_cache, t["tables"], lens, 80, seq_starts=starts, key=rows[0], value=rows[1])

    torch.cuda.synchronize()
    stream = torch.cuda.Stream(device=dev)
    context = binding.Context(stream)
    cache = ops.new_int4_cache(blocks, kv_heads, block, d, dtype, dev)
    torch.cuda.synchronize()

    def run(name, inputs, outputs=None, **param):
        runner = binding.OperationRunner(name + "Operation", getattr(binding, name + "Param")(**param), context)
        out = runner.run(inputs, outputs)
        stream.synchronize()
        return out

    with torch.cuda.stream(stream):
        run("ReshapeAndCacheInt4", [t["old_key"], t["old_value"], *cache, t["all_slots"]], list(cache))
        got = run("RmsNormQuant", [t["x"], t["gamma"], t["residual"]], hasResidual=True, epsilon=1e-6)
        got += run("LinearInt8", [got[0], t["w"], got[1], t["ws"], t["bias"]], hasBias=True, outDataType=binding._torch_acl_dtype(t["x"]))
        run("ReshapeAndCacheInt4", [k, v, *cache, t["slots"]], list(cache))
        heads_param = dict(headNum=heads, kvHeadNum=kv_heads, qkScale=scale)
        got += run("PagedAttentionInt4", [q, *cache, t["tables"], t["lens"], mask], hasMask=True, **heads_param)
        got += run("PagedAttentionInt4", [q, *cache, t["tables"], t["lens"]], **heads_param)
        rows = [torch.full((80, kv_heads, d), 7.0, dtype=dtype, device=dev) for _ in range(2)]
        got += run("PagedCacheLoadInt4", [*cache, t["tables"], lens, *rows, starts], rows, hasSeqStarts=True)
    assert len(got) == len(want) == 8
    for i, (a, b) in enumerate(zip(got, want)):
        assert _same(a, b), i
    assert all(_same(a, b) for a, b in zip(cache, want_cache))
    assert bool((got[6][74:] == 7.0).all()) and bool((got[7][74:] == 7.0).all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_torch_atb_forward(pkg, ops, dev, dtype):
    """The same operations through torch_atb.Operation(param).forward."""
    ta = pkg.torch_atb
    d, block = 128, 16
    t, heads, kv_heads, blocks = _layer(_gen(4), dtype, d, block, dev)
    cache = ops.new_int4_cache(blocks, kv_heads, block, d, dtype, dev)
    want_cache = [c.clone() for c in cache]
    out_type = 27 if dtype == torch.bfloat16 else 1

    codes, scale = ta.Operation(ta.RmsNormQuantParam()).forward([t["x"], t["gamma"]])
    want = ops.rms_norm_quant(t["x"], t["gamma"])
    assert _same(codes, want[0]) and _same(scale, want[1])
    y, = ta.Operation(ta.LinearInt8Param(out_data_type=out_type)).forward([codes, t["w"], scale, t["ws"]])
    assert _same(y, ops.linear_int8(codes, t["w"], scale, t["ws"], out_dtype=dtype))
    written = ta.Operation(ta.ReshapeAndCacheInt4Param()).forward([t["old_key"], t["old_value"], *cache, t["all_slots"]])
    ops.reshape_and_cache_int4(t["old_key"], t["old_value"], *want_cache, t["all_slots"])
    assert all(a is b for a, b in zip(written, cache)) and all(_same(a, b) for a, b in zip(cache, want_cache))
    q = y[:, :heads * d].unflatten(1, (heads, d)).contiguous()
    op = ta.Operation(ta.PagedAttentionInt4Param(head_num=heads, kv_head_num=kv_heads, qk_scale=0.1))
    for _ in range(2):
        out, = op.forward([q, *cache, t["tables"], t["lens"]])
        assert _same(out, ops.paged_attention_int4(q, *cache, t["tables"], t["lens"], 0.1))
    key, value = (torch.zeros(104, kv_heads, d, dtype=dtype, device=dev) for _ in range(2))
    loaded = ta.Operation(ta.PagedCacheLoadInt4Param()).forward([*cache, t["tables"], t["lens"], key, value])
    assert loaded[0] is key and loaded[1] is value
    want = ops.paged_cache_load_int4(*cache, t["tables"], t["lens"], 104)
    assert _same(key, want[0]) and _same(value, want[1])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("order", ["runs", "shuffled"])
@pytest.mark.parametrize("tokens,heads,d,block,gap", [(1024, 1, 64, 16, 0), (1100, 3, 128, 48, 8), (1087, 2, 256, 128, 0),
                                                      (2113, 1, 128, 1024, 3), (1025, 2, 64, 32, 1)])
def test_write_of_many_tokens(ops, dev, tokens, heads, d, block, gap, order, dtype):
    """Prompts: slots in runs that begin anywhere and cross blocks, or shuffled; skipped tokens; token strides with and
    without whole 16-byte pieces. Written rows are what the definition makes of them, all other slots keep every byte, and
    the rows are bit for bit those of calls with few tokens."""
    gen = _gen(tokens + d)
    blocks = (tokens + 37) // block + 2
    slots = torch.randperm(blocks * block, generator=gen)[:tokens] if order == "shuffled" else torch.arange(tokens) + 13
    slots = slots.to(torch.int32)
    skipped = torch.zeros(tokens, dtype=torch.bool)
    skipped[torch.tensor([0, 63, 64, 700, tokens - 1])] = True
    slots[0], slots[63], slots[64], slots[700], slots[tokens - 1] = -1, blocks * block, 2 ** 31 - 1, -(2 ** 31), -5
    rows = (torch.randn(2, tokens, heads * d + gap, generator=gen) * 2).to(dtype)
    rows[0, 5, gap + 3], rows[1, 77, gap + 1] = math.inf, math.nan
    rows[:, 9] = 0.25
    key, value = (r[:, gap:].unflatten(1, (heads, d)) for r in rows)
    dr = rows.to(dev)
    dk, dv = (r[:, gap:].unflatten(1, (heads, d)) for r in dr)
    cache = ops.new_int4_cache(blocks, heads, block, d, dtype, dev)
    for c, fill in zip(cache, (0x5A, 0xA5, 3.0, -3.0)):
        c.fill_(fill)
    parts = [c.clone() for c in cache]
    before = [c.clone().cpu() for c in cache]
    ds = slots.to(dev)
    ops.reshape_and_cache_int4(dk, dv, *cache, ds)
    for at in range(0, tokens, 300):
        ops.reshape_and_cache_int4(dk[at:at + 300], dv[at:at + 300], *parts, ds[at:at + 300])
    assert all(_same(a, b) for a, b in zip(cache, parts))
    s = slots[~skipped].long()
    kc, vc, kp, vp = qo.token_rows(cache, s // block, s % block)
    assert qo.quantised_row_ok(key[~skipped], kc, kp) and qo.quantised_row_ok(value[~skipped], vc, vp)
    after = [c.cpu() for c in cache]
    for i in (0, 2, 3):
        before[i][s // block, :, s % block] = after[i][s // block, :, s % block]
    before[1][s // block, :, :, s % block] = after[1][s // block, :, :, s % block]
    assert all(_same(a, b) for a, b in zip(before, after))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,dim", [(515, 4096), (513, 8192), (512, 8200), (600, 1032), (530, 16384), (512, 40000), (700, 777)])
def test_norm_of_many_rows(ops, dev, rows, dim, dtype):
    """Rows enough to fill the chip, where a row gets fewer threads; with special rows among them."""
    gen = _gen(rows + dim)
    x = torch.randn(rows, dim, generator=gen).to(dtype)
    r = torch.randn(rows, dim, generator=gen).to(dtype)
    x[3], r[3] = 0, 0
    x[5] = (x[5].float() * 1e-3).to(dtype)
    gamma = torch.randn(dim, generator=gen).to(dtype)
    for residual in (None, r):
        codes, scale, out = ops.rms_norm_quant(x.to(dev), gamma.to(dev), residual=None if residual is None else residual.to(dev))
        assert qo.norm_quant_ok(x, residual, gamma, 1e-5, codes.cpu(), scale.cpu(), out.cpu())
        assert float(scale[3]) == 0 and bool((codes[3] == 0).all())

"""The quantised decoder-layer operators at the edges of what their definition allows, against 64-bit plain implementations:
outputs that only the C ABI offers, values at the ends of the types' ranges, launches of many rows."""
import math

import pytest
import torch

import quant_oracle as qo
from test_gpu_quantized import DTYPES, _attention_case, _check_attention, _gen, _mask, _random_cache, _randn
from test_gpu_quantized_cut import _wide

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.quantized


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    return torch.device("cuda:0")


def _norm_c(binding, dev, x, gamma, eps, residual_out, out, scale):
    """atbmi_rms_norm_quant without a residual."""
    code = binding.ATBMI_F16 if x.dtype == torch.float16 else binding.ATBMI_BF16
    rc = binding.kernels().atbmi_rms_norm_quant(x.data_ptr(), None, gamma.data_ptr(), out.data_ptr(), scale.data_ptr(),
                                                residual_out.data_ptr(), x.shape[0], x.shape[1], x.stride(0), 0, code, eps,
                                                torch.cuda.current_stream(dev).cuda_stream)
    assert rc == 0, binding.kernels().atbmi_last_error()
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("gap", [0, 8])
@pytest.mark.parametrize("rows,dim", [(3, 64), (600, 2048), (7, 4096), (7, 4099), (600, 8192), (2, 65536)])
def test_norm_quant_gives_its_rows_without_a_residual(binding, dev, rows, dim, gap, dtype):
    """residualOut holds x where there is no residual, whatever the rows' length and stride; so it does where it is x."""
    gen = _gen(rows + dim)
    x, gamma = _randn(gen, (rows, dim + gap), dtype), _randn(gen, (dim,), dtype)
    dx, dgamma = x.to(dev), gamma.to(dev)
    out = torch.full((rows, dim), 99, dtype=torch.int8, device=dev)
    scale = torch.full((rows,), -1.0, device=dev)
    kept = torch.full((rows + 1, dim), -7.0, dtype=dtype, device=dev)
    _norm_c(binding, dev, dx[:, :dim], dgamma, 1e-5, kept, out, scale)
    assert torch.equal(kept[:rows].cpu(), x[:, :dim]) and bool((kept[rows] == -7.0).all())
    assert torch.equal(dx.cpu(), x)
    assert qo.norm_quant_ok(x[:, :dim], None, gamma, 1e-5, out.cpu(), scale.cpu(), None)
    if gap == 0:
        again, again_scale = torch.empty_like(out), torch.empty_like(scale)
        _norm_c(binding, dev, dx, dgamma, 1e-5, dx, again, again_scale)
        assert torch.equal(dx.cpu(), x) and torch.equal(again, out) and torch.equal(again_scale, scale)


def test_functions_under_vmap_raise(ops, dev):
    """torch.vmap's tensors have no memory of their own: the call raises, and the next one runs as ever."""
    x, gamma = torch.ones(3, 5, 96, dtype=torch.bfloat16, device=dev), torch.ones(96, dtype=torch.bfloat16, device=dev)
    with pytest.raises(RuntimeError, match="data pointer"):
        torch.vmap(lambda t: ops.rms_norm_quant(t, gamma)[1])(x)
    x8, w = torch.ones(3, 5, 96, dtype=torch.int8, device=dev), torch.ones(8, 96, dtype=torch.int8, device=dev)
    one = torch.ones(8, device=dev)
    with pytest.raises(RuntimeError, match="data pointer"):
        torch.vmap(lambda t: ops.linear_int8(t, w, one[:5], one, out_dtype=torch.bfloat16))(x8)
    assert bool((ops.linear_int8(x8[0], w, one[:5], one, out_dtype=torch.bfloat16) == 96.0).all())


@pytest.mark.parametrize("dim", [256, 259])
@pytest.mark.parametrize("epsilon", [0.0, 1e-30, 1e-5, 4.0, 1e30, 3.4e38])
@pytest.mark.parametrize("gamma_power", [0, -110, 100, 127])
def test_norm_quant_rows_anywhere_in_the_range(ops, dev, gamma_power, epsilon, dim):
    """A row for every power of two of the bf16 range, and epsilons whose sum with the squares leaves fp32's unless both are
    brought down: codes and scales as for any other row, wherever the scale is an fp32 number."""
    gen = _gen(dim + gamma_power)
    powers = torch.arange(-133, 128, dtype=torch.float64)
    rows = (torch.rand((len(powers), dim), generator=gen, dtype=torch.float64) * 2 - 1)
    rows[:, 0] = 1.0
    x = (rows * torch.exp2(powers)[:, None]).to(torch.bfloat16)
    gamma = ((torch.rand((dim,), generator=gen, dtype=torch.float64) + 0.9) * 2.0 ** gamma_power / 2).to(torch.bfloat16)
    assert bool(x.isfinite().all()) and bool(gamma.isfinite().all())
    codes, scale, _ = ops.rms_norm_quant(x.to(dev), gamma.to(dev), epsilon=epsilon)
    codes, scale = codes.cpu(), scale.cpu()
    epsilon = float(torch.tensor(epsilon))  # as the call takes it
    s = x.double()
    y = (s * gamma.double()).abs().amax(-1) / torch.sqrt((s * s).mean(-1) + epsilon)  # (held in fp32)
    none = (scale == 0) & (y / 127.0 < 2.0 ** -149)  # a scale of 0: the codes do not matter
    keep = ~none & (y < 3.4e38)
    assert int(keep.sum()) >= 100 or epsilon >= 1e30
    assert not bool(scale[keep].isnan().any())
    assert qo.norm_quant_ok(x[keep], None, gamma, epsilon, codes[keep], scale[keep], None)


@pytest.mark.parametrize("rows,dim", [(2 ** 24 + 5, 7), (2 ** 26 + 3, 8)])
def test_norm_quant_more_rows_than_a_launch_holds(ops, dev, rows, dim):
    """Rows past 2^32 threads of one launch: every row is written, those around the seams are what they should be."""
    gen = torch.Generator(device=dev)
    gen.manual_seed(rows)
    x = torch.randn((rows, dim), generator=gen, device=dev, dtype=torch.bfloat16)
    gamma = torch.randn((dim,), generator=gen, device=dev, dtype=torch.bfloat16)
    scale = torch.full((rows,), -1.0, device=dev)
    out = torch.full((rows, dim), -128, device=dev, dtype=torch.int8)
    residual_out = torch.full((rows, dim), -9.0, device=dev, dtype=torch.bfloat16)
    ops.rms_norm_quant(x, gamma, residual=x, out=out, scale=scale, residual_out=residual_out)
    assert bool((scale >= 0).all()) and bool((out > -128).all()) and torch.equal(residual_out, x + x)
    seams = torch.arange(0, rows, 2 ** 21)
    for first in [0, rows - 64] + (seams[1:] - 32).tolist():
        part = slice(first, min(first + 64, rows))
        assert qo.norm_quant_ok(x[part].cpu(), x[part].cpu(), gamma.cpu(), 1e-5, out[part].cpu(), scale[part].cpu(),
                                residual_out[part].cpu())


def test_load_with_the_widest_table(ops, dev):
    """A table that reaches almost 2^30 positions and no bound on the lengths: the launch follows the rows there are."""
    gen = _gen(31)
    cache = _random_cache(ops, gen, 4, 1, 16, 256, torch.bfloat16, dev)
    tables = torch.full((1, 2 ** 26 - 1), -1, dtype=torch.int32, device=dev)
    tables[0, :4] = torch.tensor([2, 0, 3, 1], dtype=torch.int32, device=dev)
    lens = torch.tensor([61], dtype=torch.int32, device=dev)
    got = ops.paged_cache_load_int4(*cache, tables, lens, 50)
    want = ops.paged_cache_load_int4(*cache, tables[:, :4].contiguous(), lens, 61)
    for a, b in zip(got, want):
        assert a.shape == (50, 1, 256) and torch.equal(a, b[:50])


LARGE = [
    # lens, heads, kv_heads, d, block, tokens, cut
    ([1, 300, 40], 4, 1, 128, 16, 1, False),
    ([700, 65], 8, 1, 64, 64, 1, False),
    ([129, 400], 4, 1, 256, 32, 4, False),
    ([2100, 30, 0, 900], 8, 2, 128, 128, 1, True),
    ([640, 1700], 8, 1, 128, 64, 1, True),
    ([1500, 200], 4, 1, 256, 16, 5, True),
    ([900, 1100, 3], 4, 2, 64, 128, 2, True),
]


@pytest.mark.parametrize("mask", [None, "-inf"])
@pytest.mark.parametrize("power", [88, 96, 112, 124])
@pytest.mark.parametrize("lens,heads,kv_heads,d,block,tokens,cut", LARGE)
def test_attention_over_the_largest_bf16_values(ops, dev, lens, heads, kv_heads, d, block, tokens, cut, power, mask):
    """Value rows up to the type's largest numbers, whose weighted sums leave fp32: the means are finite and as near as
    elsewhere, in one sequence of the batch; the others keep every bit."""
    gen = _gen(sum(lens) + d)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, torch.bfloat16, tokens)
    if cut:
        tables = _wide(tables, block)
    m = None if mask is None else _mask(gen, mask, len(lens), heads, tokens, max(lens), torch.bfloat16)
    before = _check_attention(ops, dev, query, cache, tables, n, scale, tokens, block, m)
    own = tables[1][: -(-lens[1] // block)].long().to(dev)
    cache[3][own] *= 2.0 ** power
    got = _check_attention(ops, dev, query, cache, tables, n, scale, tokens, block, m)
    assert bool(got.isfinite().all())
    rows = torch.arange(len(lens)).repeat_interleave(tokens)
    assert torch.equal(got[rows != 1], before[rows != 1])


@pytest.mark.parametrize("length", [5, 1024, 3000])
def test_attention_over_rows_of_the_largest_number(ops, dev, length):
    """Every value is the largest bf16 number: so is the mean."""
    gen = _gen(length)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, [length], 4, 1, 128, 128, torch.bfloat16, 1)
    cache[3][..., 0], cache[3][..., 1] = 0.0, torch.finfo(torch.bfloat16).max
    got = _check_attention(ops, dev, query, cache, tables, n, scale, 1, 128)
    assert bool((got == torch.finfo(torch.bfloat16).max).all())


@pytest.mark.parametrize("heads,d,block,tokens,cut", [(4, 128, 128, 1, False), (8, 64, 16, 1, False), (8, 256, 32, 2, True), (4, 128, 64, 1, True)])
def test_attention_masks_of_the_largest_numbers(ops, dev, heads, d, block, tokens, cut):
    """Different masks of the bf16 type's largest numbers, of either sign: positions under the highest of a row share it, the
    others have no part in it."""
    gen = _gen(heads + d)
    big = torch.finfo(torch.bfloat16).max
    lens = [150, 64, 7, 201, 333, 90]
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, 1, d, block, torch.bfloat16, tokens)
    low = torch.tensor([-big, -0.97 * big, -0.9 * big, -0.5 * big, -0.3 * big, -math.inf])
    mask = torch.empty((len(lens), 1, 1, max(lens)))
    for b, chosen in enumerate(([0, 1], [0, 1, 2, 5], [2, 3], [0, 4, 5], [0, 5])):
        mask[b, 0, 0] = low[chosen][torch.randint(0, len(chosen), (max(lens),), generator=gen)]
    mask[5, 0, 0] = (torch.rand((max(lens),), generator=gen) < 0.3).float() * big - big * (torch.arange(max(lens)) % 2)
    mask = mask.to(torch.bfloat16)
    got = _check_attention(ops, dev, query, cache, _wide(tables, block) if cut else tables, n, scale, tokens, block, mask)
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("d", [64, 256])
def test_load_from_positions_in_front_of_the_first(ops, dev, d, dtype):
    """A start below zero: the positions in front of the sequence have no row, their places stay as they are, and the others lie
    where they would."""
    gen = _gen(d)
    cache = _random_cache(ops, gen, 6, 2, 16, d, dtype, dev)
    tables = torch.tensor([[3, 1, 4], [0, 5, 2], [1, 2, 3], [4, 0, 5]], dtype=torch.int32, device=dev)
    starts, lens = [-5, -16, -2 ** 31, 2], [30, 20, 25, 7]
    rows = sum(lens)
    key = torch.full((rows, 2, d), 9.0, dtype=dtype, device=dev)
    value = torch.full((rows, 2, d), -9.0, dtype=dtype, device=dev)
    put = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)  # noqa: E731
    ops.paged_cache_load_int4(*cache, tables, put(lens), rows, seq_starts=put(starts), key=key, value=value)
    all_rows = ops.paged_cache_load_int4(*cache, tables, put([48] * 4), 4 * 48)
    for got, full, empty in ((key, all_rows[0], 9.0), (value, all_rows[1], -9.0)):
        want = torch.full_like(got, empty)
        at = 0
        for b in range(4):
            for t in range(lens[b]):
                if starts[b] + t >= 0:
                    want[at + t] = full[48 * b + starts[b] + t]
            at += lens[b]
        assert torch.equal(got, want)


@pytest.mark.parametrize("values", ["ordinary", "largest", "NaN"])
@pytest.mark.parametrize("lens,heads,kv_heads,d,block,tokens,cut", LARGE + [([300, 40], 20, 1, 128, 16, 2, False)])
def test_attention_in_the_place_of_its_query(ops, dev, lens, heads, kv_heads, d, block, tokens, cut, values):
    """`out` may be the query: the same bits as into another tensor, where sums leave fp32 or a column is NaN as well."""
    gen = _gen(sum(lens) + d)
    query, cache, tables, n, scale = _attention_case(ops, dev, gen, lens, heads, kv_heads, d, block, torch.bfloat16, tokens)
    if cut:
        tables = _wide(tables, block)
    own = tables[1][: -(-lens[1] // block)].long().to(dev)
    if values == "largest":
        cache[3][own] *= 2.0 ** 124
    elif values == "NaN":
        query[tokens, 0, 3] = math.nan
        cache[3][own[:1], 0, :1] = math.nan
    query, tables, n = query.to(dev), tables.to(dev), n.to(dev)
    want = ops.paged_attention_int4(query, *cache, tables, n, scale, query_tokens=tokens)
    got = ops.paged_attention_int4(query, *cache, tables, n, scale, query_tokens=tokens, out=query)
    assert got is query and torch.equal(got.view(torch.int16), want.view(torch.int16))

"""The quantised decoder-layer operators on torch tensors: 8-bit activations and weights, a paged cache in 4 bits.

    import importlib
    ops = importlib.import_module("ascend-transformer-boost_amd").quantized
    q, scale, residual = ops.rms_norm_quant(x, gamma, residual=residual)
    qkv = ops.linear_int8(q, w_qkv, scale, w_qkv_scale, out_dtype=x.dtype)
    ops.reshape_and_cache_int4(key, value, *cache, slot_mapping)       # cache = ops.new_int4_cache(...)
    out = ops.paged_attention_int4(query, *cache, block_tables, context_lens, qk_scale)

Each function checks its arguments (ValueError), launches the HIP kernel through the C ABI (include/atbmi_kernels.h, which
defines the operators) on torch's current stream of the tensors' device, and returns without waiting; a failure of the
launch raises RuntimeError, as do tensors without memory of their own (those of torch.vmap). The functions have no gradients.
Nothing is read back from the device, so all of them can be captured into a HIP graph; results
and workspaces come from torch's allocator unless they are handed in (`out=` and its like).

The calls themselves are made by an extension module (torch_ext/quantized_ext.cpp). It does nothing and returns None when an
argument is not what it should be; the functions named _refuse_* here then say what is wrong.
"""
import importlib.util
import os

from . import binding as _b

torch = None  # imported by the first call: the package is usable without it
_module = None


def _ext():
    """The extension module, loaded by the first call."""
    global torch, _module
    import torch as imported
    torch = imported
    path = os.path.join(_b._LIB, "quantized_ext.so")
    if not os.path.exists(path):
        raise RuntimeError("%s is not built; run `python3 %s`" % (path, os.path.join(_b._PKG, "build.py")))
    _b.kernels()  # the extension depends on it
    spec = importlib.util.spec_from_file_location("quantized_ext", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    _module = module
    return module


def rms_norm_quant(x, gamma, residual=None, epsilon=1e-5, out=None, scale=None, residual_out=None):
    """(codes int8 [rows, dim], scale float32 [rows], x + residual in x's type; x itself without a residual) of x [rows, dim].

    x and residual may be row-strided views. residual_out may be x or residual (contiguous ones) to add in place."""
    got = (_module or _ext()).rms_norm_quant(x, gamma, residual, epsilon, out, scale, residual_out)
    return got if got is not None else _refuse_norm(x, gamma, residual, out, scale, residual_out)


def linear_int8(x, weight, x_scale, weight_scale, bias=None, out_dtype=None, out=None):
    """x_scale[i] * weight_scale[j] * (x @ weight.T)[i, j] + bias[j] for int8 x [m, k] and weight [n, k]; the scales and
    the bias are float32. The result has out_dtype (float16 or bfloat16), or goes to `out`; x, weight and out may be
    row-strided views."""
    got = (_module or _ext()).linear_int8(x, weight, x_scale, weight_scale, bias, out_dtype, out)
    return got if got is not None else _refuse_linear(x, weight, x_scale, weight_scale, bias, out_dtype, out)


def new_int4_cache(num_blocks, kv_heads, block_size, head_dim, dtype, device):
    """(key_cache, value_cache, key_params, value_params) of an empty 4-bit cache (every row stands for zeros)."""
    if torch is None:
        _ext()
    _model_type(dtype)

    def zeros(*shape, of):
        return torch.zeros(shape, dtype=of, device=device)

    return (zeros(num_blocks, kv_heads, block_size, head_dim // 2, of=torch.uint8),
            zeros(num_blocks, kv_heads, head_dim // 2, block_size, of=torch.uint8),
            zeros(num_blocks, kv_heads, block_size, 2, of=dtype), zeros(num_blocks, kv_heads, block_size, 2, of=dtype))


def reshape_and_cache_int4(key, value, key_cache, value_cache, key_params, value_params, slot_mapping):
    """Quantises key and value [tokens, kv_heads, head_dim] (token-strided views allowed) into the slots of a 4-bit cache;
    slots (int32) outside the pool skip their token, and those of one call must differ."""
    if (_module or _ext()).reshape_and_cache_int4(key, value, key_cache, value_cache, key_params, value_params,
                                                  slot_mapping) is None:
        _refuse_write(key, value, (key_cache, value_cache, key_params, value_params), slot_mapping)


def paged_cache_load_int4(key_cache, value_cache, key_params, value_params, block_tables, seq_lens, total_rows,
                          seq_starts=None, max_seq_len=None, key=None, value=None):
    """(key, value) [total_rows, kv_heads, head_dim]: the cached rows of positions seq_starts[b] .. + seq_lens[b] of every
    sequence, one sequence after the other. Rows that no cached row lands in are left as they are (new tensors: unset).
    max_seq_len bounds the lengths (default: what a row of block_tables reaches)."""
    got = (_module or _ext()).paged_cache_load_int4(key_cache, value_cache, key_params, value_params, block_tables, seq_lens,
                                                    total_rows, seq_starts, max_seq_len, key, value)
    return got if got is not None else _refuse_load((key_cache, value_cache, key_params, value_params), block_tables,
                                                    seq_lens, total_rows, seq_starts, max_seq_len, key, value)


def paged_attention_int4(query, key_cache, value_cache, key_params, value_params, block_tables, context_lens, qk_scale,
                         query_tokens=1, mask=None, out=None, workspace=None):
    """Attention of query [batch * query_tokens, heads, head_dim] over a 4-bit cache; query token j of a sequence sees its
    first context_lens[b] - query_tokens + 1 + j positions. mask, in the query's type and [batch | 1, heads | 1,
    query_tokens | 1, positions] with positions next to each other, is added to the scaled scores; positions past its
    length are hidden. `out` may be the query. `workspace`: a uint8 tensor to use instead of a new one. Tables that reach much further than the
    contexts cost short ones a few microseconds (see AtbmiPaInt4Call)."""
    got = (_module or _ext()).paged_attention_int4(query, key_cache, value_cache, key_params, value_params, block_tables,
                                                   context_lens, qk_scale, query_tokens, mask, out, workspace)
    return got if got is not None else _refuse_attention(query, (key_cache, value_cache, key_params, value_params),
                                                         block_tables, context_lens, query_tokens, mask, out, workspace)


# ---- what is wrong with a call that the extension did not take

def _fail(text, *args):
    raise ValueError(text % args)


def _model_type(dtype):
    if dtype not in (torch.float16, torch.bfloat16):
        _fail("the model's type is float16 or bfloat16, got %s", dtype)


def _check(name, t, dtype, shape, device, contiguous=True):
    """A tensor argument: type, shape, device, and no gaps unless strides are allowed."""
    if not isinstance(t, torch.Tensor):
        _fail("%s should be a tensor, got %s", name, type(t).__name__)
    if t.dtype is not dtype:
        _fail("%s should be %s, got %s", name, dtype, t.dtype)
    if t.shape != shape:
        _fail("%s should have the shape %s, got %s", name, list(shape), list(t.shape))
    if t.device != device:
        _fail("%s is on %s, other tensors on %s", name, t.device, device)
    if contiguous and not t.is_contiguous():
        _fail("%s should be contiguous", name)


def _dims(name, t, count):
    """The shape of a tensor of `count` dimensions."""
    if not isinstance(t, torch.Tensor):
        _fail("%s should be a tensor, got %s", name, type(t).__name__)
    if t.dim() != count:
        _fail("%s should have %d dimensions, got the shape %s", name, count, list(t.shape))
    return t.shape


def _rows(name, t):
    """A matrix whose rows have no gaps."""
    if t.shape[1] > 1 and t.stride(1) != 1:
        _fail("the rows of %s should have no gaps", name)


def _tokens(name, t):
    """[tokens, heads, channels] whose tokens have no gaps."""
    if (t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        _fail("the tokens of %s should have no gaps", name)


def _int(name, value, least):
    if not isinstance(value, int) or value < least:
        _fail("%s should be a whole number of at least %d, got %r", name, least, value)


def _refused(device):
    if device.type != "cuda":
        _fail("the tensors should be on a GPU, got %s", device)
    _fail("the arguments are not what the operator takes")


def _refuse_norm(x, gamma, residual, out, scale, residual_out):
    shape = _dims("x", x, 2)
    dtype, device = x.dtype, x.device
    _model_type(dtype)
    if shape[1] == 0:
        _fail("x has no columns")
    _check("gamma", gamma, dtype, shape[1:], device)
    _rows("x", x)
    if residual is not None:
        _check("residual", residual, dtype, shape, device, False)
        _rows("residual", residual)
        if residual_out is not None:
            _check("residual_out", residual_out, dtype, shape, device)
    elif residual_out is not None:
        _fail("residual_out without a residual")
    if out is not None:
        _check("out", out, torch.int8, shape, device)
    if scale is not None:
        _check("scale", scale, torch.float32, shape[:1], device)
    _refused(device)


def _refuse_linear(x, weight, x_scale, weight_scale, bias, out_dtype, out):
    m, k = _dims("x", x, 2)
    n = _dims("weight", weight, 2)[0]
    device = x.device
    _check("x", x, torch.int8, (m, k), device, False)
    _check("weight", weight, torch.int8, (n, k), device, False)
    _check("x_scale", x_scale, torch.float32, (m,), device)
    _check("weight_scale", weight_scale, torch.float32, (n,), device)
    if bias is not None:
        _check("bias", bias, torch.float32, (n,), device)
    _rows("x", x)
    _rows("weight", weight)
    if out is not None:
        if out_dtype is not None and out_dtype is not out.dtype:
            _fail("out is %s, out_dtype %s", out.dtype, out_dtype)
        _model_type(out.dtype)
        _check("out", out, out.dtype, (m, n), device, False)
        _rows("out", out)
    else:
        _model_type(out_dtype)
    _refused(device)


def _check_cache(key_cache, value_cache, key_params, value_params):
    """(device, dtype, heads, head size) of a 4-bit cache."""
    shape = _dims("key_cache", key_cache, 4)
    blocks, heads, block, half = shape
    device = key_cache.device
    dtype = _dims("key_params", key_params, 4) and key_params.dtype
    _model_type(dtype)
    _check("key_cache", key_cache, torch.uint8, shape, device)
    _check("value_cache", value_cache, torch.uint8, (blocks, heads, half, block), device)
    _check("key_params", key_params, dtype, (blocks, heads, block, 2), device)
    _check("value_params", value_params, dtype, (blocks, heads, block, 2), device)
    return device, dtype, heads, 2 * half


def _refuse_write(key, value, cache, slot_mapping):
    device, dtype, heads, d = _check_cache(*cache)
    tokens = _dims("key", key, 3)[0]
    _check("key", key, dtype, (tokens, heads, d), device, False)
    _check("value", value, dtype, (tokens, heads, d), device, False)
    _check("slot_mapping", slot_mapping, torch.int32, (tokens,), device)
    _tokens("key", key)
    _tokens("value", value)
    _refused(device)


def _refuse_load(cache, block_tables, seq_lens, total_rows, seq_starts, max_seq_len, key, value):
    device, dtype, heads, d = _check_cache(*cache)
    shape = _dims("block_tables", block_tables, 2)
    _check("block_tables", block_tables, torch.int32, shape, device)
    _check("seq_lens", seq_lens, torch.int32, shape[:1], device)
    if seq_starts is not None:
        _check("seq_starts", seq_starts, torch.int32, shape[:1], device)
    _int("total_rows", total_rows, 0)
    if max_seq_len is not None:
        _int("max_seq_len", max_seq_len, 0)
    for name, t in (("key", key), ("value", value)):
        if t is not None:
            _check(name, t, dtype, (total_rows, heads, d), device)
    _refused(device)


def _refuse_attention(query, cache, block_tables, context_lens, query_tokens, mask, out, workspace):
    device, dtype, kv_heads, d = _check_cache(*cache)
    shape = _dims("block_tables", block_tables, 2)
    _check("block_tables", block_tables, torch.int32, shape, device)
    batch = shape[0]
    _int("query_tokens", query_tokens, 1)
    heads = _dims("query", query, 3)[1]
    _check("query", query, dtype, (batch * query_tokens, heads, d), device)
    _check("context_lens", context_lens, torch.int32, (batch,), device)
    if mask is not None:
        got = _dims("mask", mask, 4)
        _check("mask", mask, dtype, got, device, False)
        if any(have not in (1, want) for have, want in zip(got, (batch, heads, query_tokens))):
            _fail("mask should have the shape [%d | 1, %d | 1, %d | 1, positions], got %s", batch, heads, query_tokens,
                  list(got))
        if got[3] == 0 or (got[3] > 1 and mask.stride(3) != 1):
            _fail("the positions of mask should lie next to each other")
    if out is not None:
        _check("out", out, dtype, query.shape, device)
    if workspace is not None:
        _check("workspace", workspace, torch.uint8, (workspace.numel(),), device)
    _refused(device)

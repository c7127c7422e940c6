"""The quantised decoder-layer operators on torch tensors: 8-bit activations and weights, a paged cache in 4 bits.

    import importlib
    ops = importlib.import_module("ascend-transformer-boost_amd").quantized
    q, scale, residual = ops.rms_norm_quant(x, gamma, residual=residual)
    qkv = ops.linear_int8(q, w_qkv, scale, w_qkv_scale, out_dtype=x.dtype)
    ops.reshape_and_cache_int4(key, value, *cache, slot_mapping)       # cache = ops.new_int4_cache(...)
    out = ops.paged_attention_int4(query, *cache, block_tables, context_lens, qk_scale)

Each function checks its arguments (ValueError), launches the HIP kernel through the C ABI (include/atbmi_kernels.h, which
defines the operators) on torch's current stream of the first tensor's device, and returns without waiting; a failure of
the launch raises RuntimeError. Nothing is read back from the device, so all of them can be captured into a HIP graph; results and
workspaces come from torch's allocator unless they are handed in (`out=` and its like).
"""
import ctypes
import functools
import struct

from . import binding as _b

# AtbmiPaInt4Call, filled at once
_CALL = struct.Struct("@10ifi3q9P")
assert _CALL.size == ctypes.sizeof(_b.AtbmiPaInt4Call)

torch = None  # imported by the first call: the package is usable without it
_raw_stream = None


def _need_torch():
    global torch, _raw_stream
    import torch as module
    # (a stream's handle without an object around it, where this torch has it)
    _raw_stream = getattr(module._C, "_cuda_getCurrentRawStream", None) or (
        lambda index: module.cuda.current_stream(index).cuda_stream)
    torch = module


def _operator(function):
    """Runs an operator with the device of its first tensor as the current one."""
    name = function.__code__.co_varnames[0]

    @functools.wraps(function)
    def call(*args, **kwargs):
        if torch is None:
            _need_torch()
        index = (args[0] if args else kwargs[name]).get_device()
        if index < 0 or index == torch.cuda.current_device():
            return function(*args, **kwargs)
        with torch.cuda.device(index):
            return function(*args, **kwargs)
    return call


def _fail(text, *args):
    raise ValueError(text % args)


def _code(dtype):
    if dtype is torch.float16:
        return _b.ATBMI_F16
    if dtype is torch.bfloat16:
        return _b.ATBMI_BF16
    _fail("the model's type is float16 or bfloat16, got %s", dtype)


def _check(name, t, dtype, shape, index, contiguous=True):
    """A tensor argument: type, shape, device (-1: the CPU), and no gaps unless strides are allowed."""
    if t.dtype is not dtype:
        _fail("%s should be %s, got %s", name, dtype, t.dtype)
    if t.shape != shape:
        _fail("%s should have the shape %s, got %s", name, list(shape), list(t.shape))
    if t.get_device() != index:
        _fail("%s is on %s, not on the device of the first input", name, t.device)
    if contiguous and not t.is_contiguous():
        _fail("%s should be contiguous", name)


def _dims(name, t, count):
    """The shape of a tensor of `count` dimensions."""
    shape = t.shape
    if len(shape) != count:
        _fail("%s should have %d dimensions, got the shape %s", name, count, list(shape))
    return shape


def _rows(name, t):
    """Row stride of a matrix whose rows have no gaps."""
    rows, columns = t.shape
    if columns > 1 and t.stride(1) != 1:
        _fail("the rows of %s should have no gaps", name)
    return t.stride(0) if rows > 1 else columns


def _tokens(name, t):
    """Token stride of [tokens, heads, channels] whose tokens have no gaps."""
    tokens, heads, channels = t.shape
    if (channels > 1 and t.stride(2) != 1) or (heads > 1 and t.stride(1) != channels):
        _fail("the tokens of %s should have no gaps", name)
    return t.stride(0) if tokens > 1 else heads * channels


def _stream(index):
    """The current stream of the device that the tensors are on."""
    if index < 0:
        _fail("the tensors should be on a GPU")
    return _raw_stream(index)


def _done(rc):
    """Raises what the library reports."""
    if rc != 0:
        raise (ValueError if _b.ERROR_NAMES[rc] == "ERROR_INVALID_PARAM" else RuntimeError)("%s (%s)" % (_b.last_kernel_error(), _b.ERROR_NAMES[rc]))


@_operator
def rms_norm_quant(x, gamma, residual=None, epsilon=1e-5, out=None, scale=None, residual_out=None):
    """(codes int8 [rows, dim], scale float32 [rows], x + residual in x's type; x itself without a residual) of x [rows, dim].

    x and residual may be row-strided views. residual_out may be x or residual (contiguous ones) to add in place."""
    index = x.get_device()
    dtype = x.dtype
    code = _code(dtype)
    shape = _dims("x", x, 2)
    rows, dim = shape
    if dim == 0:
        _fail("x has no columns")
    _check("gamma", gamma, dtype, (dim,), index)
    x_stride = _rows("x", x)
    r_stride = r_ptr = ro_ptr = 0
    if residual is not None:
        _check("residual", residual, dtype, shape, index, False)
        r_stride, r_ptr = _rows("residual", residual), residual.data_ptr()
        if residual_out is None:
            residual_out = torch.empty(shape, dtype=dtype, device=x.device)
        else:
            _check("residual_out", residual_out, dtype, shape, index)
        ro_ptr = residual_out.data_ptr()
    elif residual_out is not None:
        _fail("residual_out without a residual")
    else:
        residual_out = x
    if out is None:
        out = torch.empty(shape, dtype=torch.int8, device=x.device)
    else:
        _check("out", out, torch.int8, shape, index)
    if scale is None:
        scale = torch.empty((rows,), dtype=torch.float32, device=x.device)
    else:
        _check("scale", scale, torch.float32, (rows,), index)
    stream = _stream(index)
    if rows:
        _done(_b.kernels().atbmi_rms_norm_quant(x.data_ptr(), r_ptr, gamma.data_ptr(), out.data_ptr(), scale.data_ptr(),
                                                ro_ptr, rows, dim, x_stride, r_stride, code, epsilon, stream))
    return out, scale, residual_out


@_operator
def linear_int8(x, weight, x_scale, weight_scale, bias=None, out_dtype=None, out=None):
    """x_scale[i] * weight_scale[j] * (x @ weight.T)[i, j] + bias[j] for int8 x [m, k] and weight [n, k]; the scales and
    the bias are float32. The result has out_dtype (float16 or bfloat16), or goes to `out`; x, weight and out may be
    row-strided views."""
    index = x.get_device()
    m, k = _dims("x", x, 2)
    n = _dims("weight", weight, 2)[0]
    _check("x", x, torch.int8, (m, k), index, False)
    _check("weight", weight, torch.int8, (n, k), index, False)
    _check("x_scale", x_scale, torch.float32, (m,), index)
    _check("weight_scale", weight_scale, torch.float32, (n,), index)
    if bias is not None:
        _check("bias", bias, torch.float32, (n,), index)
    if out is None:
        code = _code(out_dtype)
        out = torch.empty((m, n), dtype=out_dtype, device=x.device)
    else:
        if out_dtype is not None and out_dtype is not out.dtype:
            _fail("out is %s, out_dtype %s", out.dtype, out_dtype)
        code = _code(out.dtype)
        _check("out", out, out.dtype, (m, n), index, False)
    x_stride, w_stride, out_stride = _rows("x", x), _rows("weight", weight), _rows("out", out)
    stream = _stream(index)
    if m == 0 or n == 0:
        return out
    lib = _b.kernels()
    need = ctypes.c_uint64()
    _done(lib.atbmi_linear_int8_workspace_size(m, n, k, need))
    need = need.value
    workspace = torch.empty((need,), dtype=torch.uint8, device=x.device) if need else None
    _done(lib.atbmi_linear_int8(x.data_ptr(), weight.data_ptr(), x_scale.data_ptr(), weight_scale.data_ptr(),
                                0 if bias is None else bias.data_ptr(), out.data_ptr(), m, n, k, x_stride, w_stride,
                                out_stride, code, workspace.data_ptr() if need else 0, need, stream))
    return out


def new_int4_cache(num_blocks, kv_heads, block_size, head_dim, dtype, device):
    """(key_cache, value_cache, key_params, value_params) of an empty 4-bit cache (every row stands for zeros)."""
    if torch is None:
        _need_torch()
    _code(dtype)

    def zeros(*shape, of):
        return torch.zeros(shape, dtype=of, device=device)

    return (zeros(num_blocks, kv_heads, block_size, head_dim // 2, of=torch.uint8),
            zeros(num_blocks, kv_heads, head_dim // 2, block_size, of=torch.uint8),
            zeros(num_blocks, kv_heads, block_size, 2, of=dtype), zeros(num_blocks, kv_heads, block_size, 2, of=dtype))


def _cache(key_cache, value_cache, key_params, value_params):
    """(device index, dtype, blocks, heads, block size, head size) of a 4-bit cache."""
    index = key_cache.get_device()
    shape = _dims("key_cache", key_cache, 4)
    blocks, heads, block, half = shape
    dtype = key_params.dtype
    params = (blocks, heads, block, 2)
    _check("key_cache", key_cache, torch.uint8, shape, index)
    _check("value_cache", value_cache, torch.uint8, (blocks, heads, half, block), index)
    _check("key_params", key_params, dtype, params, index)
    _check("value_params", value_params, dtype, params, index)
    return index, dtype, blocks, heads, block, 2 * half


@_operator
def reshape_and_cache_int4(key, value, key_cache, value_cache, key_params, value_params, slot_mapping):
    """Quantises key and value [tokens, kv_heads, head_dim] (token-strided views allowed) into the slots of a 4-bit cache;
    slots (int32) outside the pool skip their token, and those of one call must differ."""
    index, dtype, blocks, heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    code = _code(dtype)
    tokens = _dims("key", key, 3)[0]
    _check("key", key, dtype, (tokens, heads, d), index, False)
    _check("value", value, dtype, (tokens, heads, d), index, False)
    _check("slot_mapping", slot_mapping, torch.int32, (tokens,), index)
    k_stride, v_stride = _tokens("key", key), _tokens("value", value)
    stream = _stream(index)
    if tokens:
        _done(_b.kernels().atbmi_reshape_and_cache_int4(
            key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_params.data_ptr(),
            value_params.data_ptr(), slot_mapping.data_ptr(), tokens, heads, d, block, blocks, k_stride, v_stride, code,
            stream))


@_operator
def paged_cache_load_int4(key_cache, value_cache, key_params, value_params, block_tables, seq_lens, total_rows,
                          seq_starts=None, max_seq_len=None, key=None, value=None):
    """(key, value) [total_rows, kv_heads, head_dim]: the cached rows of positions seq_starts[b] .. + seq_lens[b] of every
    sequence, one sequence after the other. Rows that no cached row lands in are left as they are (new tensors: unset).
    max_seq_len bounds the lengths (default: what a row of block_tables reaches)."""
    index, dtype, blocks, heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    code = _code(dtype)
    batch, reach = _dims("block_tables", block_tables, 2)
    _check("block_tables", block_tables, torch.int32, (batch, reach), index)
    _check("seq_lens", seq_lens, torch.int32, (batch,), index)
    if seq_starts is not None:
        _check("seq_starts", seq_starts, torch.int32, (batch,), index)
    shape = (total_rows, heads, d)
    if key is None:
        key = torch.empty(shape, dtype=dtype, device=key_cache.device)
    else:
        _check("key", key, dtype, shape, index)
    if value is None:
        value = torch.empty(shape, dtype=dtype, device=key_cache.device)
    else:
        _check("value", value, dtype, shape, index)
    stream = _stream(index)
    if batch and reach and total_rows:
        _done(_b.kernels().atbmi_paged_cache_load_int4(
            key_cache.data_ptr(), value_cache.data_ptr(), key_params.data_ptr(), value_params.data_ptr(),
            block_tables.data_ptr(), seq_lens.data_ptr(), 0 if seq_starts is None else seq_starts.data_ptr(),
            key.data_ptr(), value.data_ptr(), batch, reach, heads, d, block, blocks, total_rows,
            reach * block if max_seq_len is None else max_seq_len, code, stream))
    return key, value


def _mask(mask, dtype, index, batch, heads, query_tokens):
    """(sequence, head and row stride, positions, address) of a mask."""
    shape = _dims("mask", mask, 4)
    _check("mask", mask, dtype, shape, index, False)
    for have, want in zip(shape, (batch, heads, query_tokens)):
        if have != 1 and have != want:
            _fail("mask should have the shape [%d | 1, %d | 1, %d | 1, positions], got %s", batch, heads, query_tokens,
                  list(shape))
    if shape[3] == 0 or (shape[3] > 1 and mask.stride(3) != 1):
        _fail("the positions of mask should lie next to each other")
    return [mask.stride(i) if shape[i] > 1 else 0 for i in range(3)], shape[3], mask.data_ptr()


@_operator
def paged_attention_int4(query, key_cache, value_cache, key_params, value_params, block_tables, context_lens, qk_scale,
                         query_tokens=1, mask=None, out=None, workspace=None):
    """Attention of query [batch * query_tokens, heads, head_dim] over a 4-bit cache; query token j of a sequence sees its
    first context_lens[b] - query_tokens + 1 + j positions. mask, in the query's type and [batch | 1, heads | 1,
    query_tokens | 1, positions] with positions next to each other, is added to the scaled scores; positions past its
    length are hidden. `workspace`: a uint8 tensor to use instead of a new one."""
    index, dtype, blocks, kv_heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    code = _code(dtype)
    batch, reach = _dims("block_tables", block_tables, 2)
    _check("block_tables", block_tables, torch.int32, (batch, reach), index)
    heads = _dims("query", query, 3)[1]
    shape = (batch * query_tokens, heads, d)
    _check("query", query, dtype, shape, index)
    _check("context_lens", context_lens, torch.int32, (batch,), index)
    strides, mask_len, mask_ptr = (0, 0, 0), 0, 0
    if mask is not None:
        strides, mask_len, mask_ptr = _mask(mask, dtype, index, batch, heads, query_tokens)
    if out is None:
        out = torch.empty(shape, dtype=dtype, device=query.device)
    else:
        _check("out", out, dtype, shape, index)
    if workspace is not None:
        _check("workspace", workspace, torch.uint8, (workspace.numel(),), index)
    stream = _stream(index)
    if batch == 0:
        return out
    call = _b.AtbmiPaInt4Call.from_buffer_copy(_CALL.pack(
        code, heads, kv_heads, d, block, blocks, reach, batch, query_tokens, mask_len, qk_scale, 0, *strides,
        query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_params.data_ptr(), value_params.data_ptr(),
        block_tables.data_ptr(), context_lens.data_ptr(), mask_ptr, out.data_ptr()))
    lib = _b.kernels()
    if workspace is None:
        need = ctypes.c_uint64()
        _done(lib.atbmi_pa_int4_workspace_size(call, need))
        need = need.value
        workspace = torch.empty((need,), dtype=torch.uint8, device=query.device) if need else None
    else:
        need = workspace.numel()
    _done(lib.atbmi_pa_int4_decode(call, workspace.data_ptr() if need else 0, need, stream))
    return out

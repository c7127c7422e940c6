"""The quantised decoder-layer operators on torch tensors: 8-bit activations and weights, a paged cache in 4 bits.

    import importlib
    ops = importlib.import_module("ascend-transformer-boost_amd").quantized
    q, scale, residual = ops.rms_norm_quant(x, gamma, residual=residual)
    qkv = ops.linear_int8(q, w_qkv, scale, w_qkv_scale, out_dtype=x.dtype)
    ops.reshape_and_cache_int4(key, value, *cache, slot_mapping)       # cache = ops.new_int4_cache(...)
    out = ops.paged_attention_int4(query, *cache, block_tables, context_lens, qk_scale)

Each function checks its arguments (ValueError), launches the HIP kernel through the C ABI (include/atbmi_kernels.h, which
defines the operators) on torch's current stream of the tensors' device, and returns without waiting; a failure of the
launch raises RuntimeError. Nothing is read back from the device, so all of them can be captured into a HIP graph; results and
workspaces come from torch's allocator unless they are handed in (`out=` and its like).
"""
import ctypes

from . import binding as _b


def _torch():
    import torch
    return torch


def _fail(text, *args):
    raise ValueError(text % args)


def _code(dtype):
    torch = _torch()
    if dtype == torch.float16:
        return _b.ATBMI_F16
    if dtype == torch.bfloat16:
        return _b.ATBMI_BF16
    _fail("the model's type is float16 or bfloat16, got %s", dtype)


def _check(name, t, dtype, shape, device, contiguous=True):
    """A tensor argument: type, shape (None: any length there), device, and no gaps unless strides are allowed."""
    if t.dtype != dtype:
        _fail("%s should be %s, got %s", name, dtype, t.dtype)
    if t.dim() != len(shape) or any(want is not None and want != have for want, have in zip(shape, t.shape)):
        _fail("%s should have the shape %s, got %s", name, list(shape), list(t.shape))
    if t.device != device:
        _fail("%s is on %s, the first input is on %s", name, t.device, device)
    if contiguous and not t.is_contiguous():
        _fail("%s should be contiguous", name)


def _device_of(t, name):
    if not t.is_cuda:
        _fail("%s should be on a GPU", name)
    return t.device


def _rows(name, t):
    """Row stride of a matrix whose rows have no gaps."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        _fail("the rows of %s should have no gaps", name)
    return t.stride(0) if t.shape[0] > 1 else t.shape[-1]


def _tokens(name, t):
    """Token stride of [tokens, heads, channels] whose tokens have no gaps."""
    if (t.shape[2] > 1 and t.stride(2) != 1) or (t.shape[1] > 1 and t.stride(1) != t.shape[2]):
        _fail("the tokens of %s should have no gaps", name)
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2]


def _launch(device, call):
    """Runs call(stream) with `device` current; raises what the library reports."""
    torch = _torch()
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            rc = call(torch.cuda.current_stream(device).cuda_stream)
    else:
        rc = call(torch.cuda.current_stream(device).cuda_stream)
    if rc != 0:
        raise RuntimeError("%s (%s)" % (_b.last_kernel_error(), _b.ERROR_NAMES[rc]))


def rms_norm_quant(x, gamma, residual=None, epsilon=1e-5, out=None, scale=None, residual_out=None):
    """(codes int8 [rows, dim], scale float32 [rows], x + residual in x's type; x itself without a residual) of x [rows, dim].

    x and residual may be row-strided views. residual_out may be x or residual (contiguous ones) to add in place."""
    torch = _torch()
    device = _device_of(x, "x")
    code = _code(x.dtype)
    if x.dim() != 2:
        _fail("x should be a matrix, got %s", list(x.shape))
    rows, dim = x.shape
    _check("gamma", gamma, x.dtype, (dim,), device)
    x_stride = _rows("x", x)
    r_stride = 0
    if residual is not None:
        _check("residual", residual, x.dtype, (rows, dim), device, contiguous=False)
        r_stride = _rows("residual", residual)
    elif residual_out is not None:
        _fail("residual_out without a residual")
    out = torch.empty((rows, dim), dtype=torch.int8, device=device) if out is None else out
    scale = torch.empty((rows,), dtype=torch.float32, device=device) if scale is None else scale
    _check("out", out, torch.int8, (rows, dim), device)
    _check("scale", scale, torch.float32, (rows,), device)
    if residual is not None:
        residual_out = torch.empty((rows, dim), dtype=x.dtype, device=device) if residual_out is None else residual_out
        _check("residual_out", residual_out, x.dtype, (rows, dim), device)
    if rows and dim == 0:
        _fail("x has no columns")
    if rows:
        _launch(device, lambda stream: _b.kernels().atbmi_rms_norm_quant(
            x.data_ptr(), residual.data_ptr() if residual is not None else None, gamma.data_ptr(), out.data_ptr(),
            scale.data_ptr(), residual_out.data_ptr() if residual is not None else None, rows, dim, x_stride, r_stride, code,
            epsilon, stream))
    return out, scale, (x if residual is None else residual_out)


def linear_int8(x, weight, x_scale, weight_scale, bias=None, out_dtype=None, out=None):
    """x_scale[i] * weight_scale[j] * (x @ weight.T)[i, j] + bias[j] for int8 x [m, k] and weight [n, k]; the scales and
    the bias are float32. The result has out_dtype (float16 or bfloat16), or goes to `out`; x, weight and out may be
    row-strided views."""
    torch = _torch()
    device = _device_of(x, "x")
    _check("x", x, torch.int8, (None, None), device, contiguous=False)
    m, k = x.shape
    _check("weight", weight, torch.int8, (None, k), device, contiguous=False)
    n = weight.shape[0]
    _check("x_scale", x_scale, torch.float32, (m,), device)
    _check("weight_scale", weight_scale, torch.float32, (n,), device)
    if bias is not None:
        _check("bias", bias, torch.float32, (n,), device)
    if out is None:
        _code(out_dtype)
        out = torch.empty((m, n), dtype=out_dtype, device=device)
    elif out_dtype is not None and out_dtype != out.dtype:
        _fail("out is %s, out_dtype %s", out.dtype, out_dtype)
    _check("out", out, out.dtype, (m, n), device, contiguous=False)
    code = _code(out.dtype)
    if m == 0 or n == 0:
        return out
    x_stride, w_stride, out_stride = _rows("x", x), _rows("weight", weight), _rows("out", out)
    lib = _b.kernels()

    def call(stream):
        need = ctypes.c_uint64(0)
        rc = lib.atbmi_linear_int8_workspace_size(m, n, k, ctypes.byref(need))
        if rc != 0:
            return rc
        workspace = torch.empty((need.value,), dtype=torch.uint8, device=device) if need.value else None
        return lib.atbmi_linear_int8(x.data_ptr(), weight.data_ptr(), x_scale.data_ptr(), weight_scale.data_ptr(),
                                     bias.data_ptr() if bias is not None else None, out.data_ptr(), m, n, k, x_stride,
                                     w_stride, out_stride, code, workspace.data_ptr() if need.value else None, need.value,
                                     stream)

    _launch(device, call)
    return out


def new_int4_cache(num_blocks, kv_heads, block_size, head_dim, dtype, device):
    """(key_cache, value_cache, key_params, value_params) of an empty 4-bit cache (every row stands for zeros)."""
    torch = _torch()
    _code(dtype)

    def zeros(*shape, of):
        return torch.zeros(shape, dtype=of, device=device)

    return (zeros(num_blocks, kv_heads, block_size, head_dim // 2, of=torch.uint8),
            zeros(num_blocks, kv_heads, head_dim // 2, block_size, of=torch.uint8),
            zeros(num_blocks, kv_heads, block_size, 2, of=dtype), zeros(num_blocks, kv_heads, block_size, 2, of=dtype))


def _cache(key_cache, value_cache, key_params, value_params):
    """(device, dtype, blocks, heads, block size, head size) of a 4-bit cache."""
    torch = _torch()
    device = _device_of(key_cache, "key_cache")
    _check("key_cache", key_cache, torch.uint8, (None, None, None, None), device)
    blocks, heads, block, half = key_cache.shape
    _check("value_cache", value_cache, torch.uint8, (blocks, heads, half, block), device)
    _check("key_params", key_params, key_params.dtype, (blocks, heads, block, 2), device)
    _code(key_params.dtype)
    _check("value_params", value_params, key_params.dtype, (blocks, heads, block, 2), device)
    return device, key_params.dtype, blocks, heads, block, 2 * half


def reshape_and_cache_int4(key, value, key_cache, value_cache, key_params, value_params, slot_mapping):
    """Quantises key and value [tokens, kv_heads, head_dim] (token-strided views allowed) into the slots of a 4-bit cache;
    slots (int32) outside the pool skip their token, and those of one call must differ."""
    torch = _torch()
    device, dtype, blocks, heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    _check("key", key, dtype, (None, heads, d), device, contiguous=False)
    tokens = key.shape[0]
    _check("value", value, dtype, (tokens, heads, d), device, contiguous=False)
    _check("slot_mapping", slot_mapping, torch.int32, (tokens,), device)
    if tokens == 0:
        return
    k_stride, v_stride = _tokens("key", key), _tokens("value", value)
    _launch(device, lambda stream: _b.kernels().atbmi_reshape_and_cache_int4(
        key.data_ptr(), value.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr(), key_params.data_ptr(),
        value_params.data_ptr(), slot_mapping.data_ptr(), tokens, heads, d, block, blocks, k_stride, v_stride, _code(dtype),
        stream))


def paged_cache_load_int4(key_cache, value_cache, key_params, value_params, block_tables, seq_lens, total_rows,
                          seq_starts=None, max_seq_len=None, key=None, value=None):
    """(key, value) [total_rows, kv_heads, head_dim]: the cached rows of positions seq_starts[b] .. + seq_lens[b] of every
    sequence, one sequence after the other. Rows that no cached row lands in are left as they are (new tensors: unset).
    max_seq_len bounds the lengths (default: what a row of block_tables reaches)."""
    torch = _torch()
    device, dtype, blocks, heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    _check("block_tables", block_tables, torch.int32, (None, None), device)
    batch, reach = block_tables.shape
    _check("seq_lens", seq_lens, torch.int32, (batch,), device)
    if seq_starts is not None:
        _check("seq_starts", seq_starts, torch.int32, (batch,), device)
    key = torch.empty((total_rows, heads, d), dtype=dtype, device=device) if key is None else key
    value = torch.empty((total_rows, heads, d), dtype=dtype, device=device) if value is None else value
    _check("key", key, dtype, (total_rows, heads, d), device)
    _check("value", value, dtype, (total_rows, heads, d), device)
    if batch and reach and total_rows:
        longest = reach * block if max_seq_len is None else int(max_seq_len)
        _launch(device, lambda stream: _b.kernels().atbmi_paged_cache_load_int4(
            key_cache.data_ptr(), value_cache.data_ptr(), key_params.data_ptr(), value_params.data_ptr(),
            block_tables.data_ptr(), seq_lens.data_ptr(), seq_starts.data_ptr() if seq_starts is not None else None,
            key.data_ptr(), value.data_ptr(), batch, reach, heads, d, block, blocks, total_rows, longest, _code(dtype),
            stream))
    return key, value


def paged_attention_int4(query, key_cache, value_cache, key_params, value_params, block_tables, context_lens, qk_scale,
                         query_tokens=1, mask=None, out=None, workspace=None):
    """Attention of query [batch * query_tokens, heads, head_dim] over a 4-bit cache; query token j of a sequence sees its
    first context_lens[b] - query_tokens + 1 + j positions. mask, in the query's type and [batch | 1, heads | 1,
    query_tokens | 1, positions] with positions next to each other, is added to the scaled scores; positions past its
    length are hidden. `workspace`: a uint8 tensor to use instead of a new one (paged_attention_int4_workspace)."""
    torch = _torch()
    device, dtype, blocks, kv_heads, block, d = _cache(key_cache, value_cache, key_params, value_params)
    _check("block_tables", block_tables, torch.int32, (None, None), device)
    batch, reach = block_tables.shape
    _check("query", query, dtype, (batch * query_tokens, None, d), device)
    heads = query.shape[1]
    _check("context_lens", context_lens, torch.int32, (batch,), device)
    call = _b.AtbmiPaInt4Call()
    call.dtype, call.numHeads, call.numKvHeads, call.headDim = _code(dtype), heads, kv_heads, d
    call.blockSize, call.numBlocks, call.maxBlocksPerSeq, call.batch = block, blocks, reach, batch
    call.queryTokens, call.qkScale = query_tokens, qk_scale
    if mask is not None:
        _check("mask", mask, dtype, (None, None, None, None), device, contiguous=False)
        for have, want in zip(mask.shape, (batch, heads, query_tokens)):
            if have not in (1, want):
                _fail("mask should have the shape [%d | 1, %d | 1, %d | 1, positions], got %s", batch, heads, query_tokens,
                      list(mask.shape))
        if mask.shape[3] == 0 or (mask.shape[3] > 1 and mask.stride(3) != 1):
            _fail("the positions of mask should lie next to each other")
        strides = [mask.stride(i) if mask.shape[i] > 1 else 0 for i in range(3)]
        call.maskSeqStride, call.maskHeadStride, call.maskRowStride = strides
        call.maskLen, call.mask = mask.shape[3], mask.data_ptr()
    out = torch.empty_like(query) if out is None else out
    _check("out", out, dtype, query.shape, device)
    if batch == 0:
        return out
    call.query, call.keyCache, call.valueCache = query.data_ptr(), key_cache.data_ptr(), value_cache.data_ptr()
    call.keyParams, call.valueParams = key_params.data_ptr(), value_params.data_ptr()
    call.blockTables, call.contextLens, call.out = block_tables.data_ptr(), context_lens.data_ptr(), out.data_ptr()
    lib = _b.kernels()

    def launch(stream):
        need = ctypes.c_uint64(0)
        rc = lib.atbmi_pa_int4_workspace_size(ctypes.byref(call), ctypes.byref(need))
        if rc != 0:
            return rc
        ws = workspace
        if ws is None and need.value:
            ws = torch.empty((need.value,), dtype=torch.uint8, device=device)
        elif ws is not None:
            _check("workspace", ws, torch.uint8, (None,), device)
        return lib.atbmi_pa_int4_decode(ctypes.byref(call), ws.data_ptr() if ws is not None else None,
                                        ws.numel() if ws is not None else 0, stream)

    _launch(device, launch)
    return out

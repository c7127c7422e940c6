"""The quantised decoder-layer operators without a GPU: what the atb::Operations, the C ABI and the torch functions refuse,
and the shapes that the operations infer. Nothing here launches a kernel: every refused call returns before it touches the
device, so addresses may be made up."""
import ctypes

import pytest
import torch

FAKE = 0x100000
NONE, PARAM, NUM, INI, DIM, RANK = ("NO_ERROR", "ERROR_INVALID_PARAM", "ERROR_INVALID_IN_TENSOR_NUM",
                                    "ERROR_INVALID_TENSOR_INI_MATCH", "ERROR_INVALID_TENSOR_DIM",
                                    "ERROR_INVALID_TENSOR_DIM_NUM")


def _tensors(binding, descs):
    return [binding.make_tensor(t, shape, device_ptr=FAKE + 0x10000 * i) for i, (t, shape) in enumerate(descs)]


def _cache(t="float16", blocks=4, heads=2, block=32, d=128):
    return [("uint8", [blocks, heads, block, d // 2]), ("uint8", [blocks, heads, d // 2, block]), (t, [blocks, heads, block, 2]),
            (t, [blocks, heads, block, 2])]


def _norm(binding, t="bf16", residual=True, **kw):
    ins = [(t, [5, 96]), (t, [96])] + ([(t, [5, 96])] if residual else [])
    outs = [("int8", [5, 96]), ("float", [5])] + ([(t, [5, 96])] if residual else [])
    return "RmsNormQuantOperation", binding.RmsNormQuantParam(hasResidual=residual, **kw), ins, outs, {}


def _linear(binding, t="bf16", bias=True):
    ins = [("int8", [5, 96]), ("int8", [40, 96]), ("float", [5]), ("float", [40])] + ([("float", [40])] if bias else [])
    param = binding.LinearInt8Param(hasBias=bias, outDataType=binding.ACL_DTYPE_BY_NAME[t])
    return "LinearInt8Operation", param, ins, [(t, [5, 40])], {}


def _write(binding, t="bf16", d=128):
    ins = [(t, [7, 2, d])] * 2 + _cache(t, d=d) + [("int32", [7])]
    return "ReshapeAndCacheInt4Operation", binding.ReshapeAndCacheInt4Param(), ins, ins[2:6], {0: 2, 1: 3, 2: 4, 3: 5}


def _load(binding, t="bf16", starts=True, d=128):
    ins = _cache(t, d=d) + [("int32", [3, 4]), ("int32", [3])] + [(t, [50, 2, d])] * 2 + ([("int32", [3])] if starts else [])
    return "PagedCacheLoadInt4Operation", binding.PagedCacheLoadInt4Param(hasSeqStarts=starts), ins, ins[6:8], {0: 6, 1: 7}


def _attend(binding, t="bf16", tokens=2, mask=(3, 1, 2, 100), d=128, **kw):
    ins = [(t, [3 * tokens, 8, d])] + _cache(t, d=d) + [("int32", [3, 4]), ("int32", [3])] + ([(t, list(mask))] if mask else [])
    param = binding.PagedAttentionInt4Param(**{**dict(headNum=8, kvHeadNum=2, qkScale=0.1, queryTokens=tokens, hasMask=bool(mask)), **kw})
    return "PagedAttentionInt4Operation", param, ins, [(t, [3 * tokens, 8, d])], {}


def _run(binding, case, change=None):
    """Status of CreateOperation, InferShape and Setup in turn, with one input changed."""
    name, param, ins, outs, alias = case
    op = binding.Operation(name, param)
    if not op.ok:
        return "C", binding.ERROR_NAMES[op.status]
    ins = [list(i) for i in ins]
    if change is not None:
        ins[change[0]] = list(change[1])
    tensors = _tensors(binding, ins)
    st, descs = op.infer_shape(tensors)
    if st != 0:
        return "I", binding.ERROR_NAMES[st]
    assert [(binding.ACL_DTYPE_BY_NAME[t], s) for t, s in outs] == [(d.dtype, list(d.dims[:d.dimNum])) for d in descs]
    outputs = _tensors(binding, outs)
    for i, source in alias.items():
        outputs[i].deviceData = tensors[source].deviceData
    st, workspace = op.setup(tensors, outputs, binding.Context(0x77))
    return "S", binding.ERROR_NAMES[st]


ALL = [_norm, _linear, _write, _load, _attend]


@pytest.mark.parametrize("t", ["float16", "bf16"])
@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_operations_are_set_up(binding, make, t):
    assert _run(binding, make(binding, t)) == ("S", NONE)


@pytest.mark.parametrize("make,without", [(_norm, dict(residual=False)), (_linear, dict(bias=False)), (_load, dict(starts=False)),
                                          (_attend, dict(mask=None)), (_attend, dict(mask=(1, 8, 1, 1)))])
def test_optional_inputs(binding, make, without):
    assert _run(binding, make(binding, **without)) == ("S", NONE)


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("make", [_write, _load, _attend], ids=lambda f: f.__name__)
def test_head_sizes(binding, make, d):
    assert _run(binding, make(binding, d=d)) == ("S", NONE)


@pytest.mark.parametrize("make,at,desc,status", [
    (_norm, 0, ("int8", [5, 96]), INI), (_norm, 0, ("bf16", [5, 96, 1]), RANK), (_norm, 1, ("bf16", [95]), DIM),
    (_norm, 2, ("bf16", [4, 96]), DIM), (_norm, 0, ("bf16", [1, 65537]), DIM), (_norm, 1, ("float16", [96]), INI),
    (_linear, 0, ("int8", [5, 95]), DIM), (_linear, 1, ("int8", [40]), RANK), (_linear, 2, ("float", [6]), DIM),
    (_linear, 3, ("float", [5]), DIM), (_linear, 4, ("float", [39]), DIM), (_linear, 1, ("uint8", [40, 96]), INI),
    (_linear, 4, ("bf16", [40]), INI),
    (_write, 0, ("bf16", [7, 256]), RANK), (_write, 0, ("bf16", [7, 3, 128]), DIM), (_write, 1, ("bf16", [6, 2, 128]), DIM),
    (_write, 2, ("uint8", [4, 2, 64]), RANK), (_write, 3, ("uint8", [4, 2, 32, 64]), DIM),
    (_write, 4, ("bf16", [4, 2, 32, 1]), DIM), (_write, 5, ("float16", [4, 2, 32, 2]), INI), (_write, 6, ("int32", [8]), DIM),
    (_write, 2, ("int8", [4, 2, 32, 64]), INI), (_write, 6, ("int64", [7]), INI),
    (_load, 4, ("int32", [12]), RANK), (_load, 5, ("int32", [4]), DIM), (_load, 6, ("bf16", [50, 2, 64]), DIM),
    (_load, 7, ("bf16", [51, 2, 128]), DIM), (_load, 8, ("int32", [2]), DIM),
    (_attend, 0, ("bf16", [5, 8, 128]), DIM), (_attend, 0, ("bf16", [6, 4, 128]), DIM), (_attend, 5, ("int32", [12]), RANK),
    (_attend, 6, ("int32", [2]), DIM), (_attend, 7, ("bf16", [3, 100]), RANK), (_attend, 7, ("bf16", [2, 1, 2, 100]), DIM),
    (_attend, 7, ("bf16", [3, 8, 3, 100]), DIM), (_attend, 7, ("float16", [3, 1, 2, 100]), INI),
    (_attend, 5, ("int32", [3, 1 << 25]), DIM)])
def test_operations_refuse_inputs(binding, make, at, desc, status):
    assert _run(binding, make(binding), (at, desc)) == ("I", status)


@pytest.mark.parametrize("shape", [dict(block=24), dict(block=1040), dict(d=96), dict(d=32), dict(heads=3)])
def test_cache_shapes_that_are_not_built(binding, shape):
    name, param, ins, outs, alias = _attend(binding)
    cache = _cache("bf16", **shape)
    d = shape.get("d", 128)
    ins = [("bf16", [6, 8, d])] + cache + ins[5:]
    assert _run(binding, (name, param, ins, [("bf16", [6, 8, d])], alias)) == ("I", DIM)


@pytest.mark.parametrize("bad", [dict(headNum=0), dict(headNum=9), dict(kvHeadNum=0), dict(kvHeadNum=-2), dict(queryTokens=0),
                                 dict(queryTokens=65), dict(qkScale=0.0), dict(qkScale=float("nan")), dict(qkScale=float("inf"))])
def test_attention_params_refused(binding, bad):
    param = binding.PagedAttentionInt4Param(**{**dict(headNum=8, kvHeadNum=2, qkScale=0.1), **bad})
    assert binding.ERROR_NAMES[binding.Operation("PagedAttentionInt4Operation", param).status] == PARAM


@pytest.mark.parametrize("make", ALL, ids=lambda f: f.__name__)
def test_reserved_bytes_and_counts(binding, make):
    name, param, ins, outs, alias = make(binding)
    op = binding.Operation(name, param)
    assert op.ok and op.get_name() == name and op.input_num() == len(ins) and op.output_num() == len(outs)
    assert binding.ERROR_NAMES[op.infer_shape(_tensors(binding, ins[:-1]))[0]] == NUM
    param.rsv[len(param.rsv) - 1] = 1
    assert binding.ERROR_NAMES[binding.Operation(name, param).status] == PARAM


@pytest.mark.parametrize("name,param", [("RmsNormQuantOperation", dict(epsilon=-1e-5)),
                                        ("RmsNormQuantOperation", dict(epsilon=float("nan"))),
                                        ("LinearInt8Operation", dict(outDataType=0)), ("LinearInt8Operation", dict(outDataType=2))])
def test_params_refused(binding, name, param):
    made = getattr(binding, name.replace("Operation", "Param"))(**param)
    assert binding.ERROR_NAMES[binding.Operation(name, made).status] == PARAM


def test_outputs_of_another_shape_or_place(binding):
    for make in (_norm, _linear, _attend):
        name, param, ins, outs, alias = make(binding)
        op = binding.Operation(name, param)
        wrong = [(outs[0][0], [outs[0][1][0] + 1] + outs[0][1][1:])] + outs[1:]
        assert binding.ERROR_NAMES[op.setup(_tensors(binding, ins), _tensors(binding, wrong), binding.Context(0x77))[0]] == DIM
    for make in (_write, _load):
        name, param, ins, outs, alias = make(binding)
        op = binding.Operation(name, param)
        assert binding.ERROR_NAMES[op.setup(_tensors(binding, ins), _tensors(binding, outs), binding.Context(0x77))[0]] == PARAM
    name, param, ins, outs, alias = _attend(binding)
    tensors = _tensors(binding, ins)
    tensors[6].hostData, tensors[6].deviceData = tensors[6].deviceData, None
    op = binding.Operation(name, param)
    assert binding.ERROR_NAMES[op.setup(tensors, _tensors(binding, outs), binding.Context(0x77))[0]] == PARAM


def test_execute_wants_the_workspace(binding):
    """A long context is worked on by several workgroups, whose parts need room."""
    name, param, ins, outs, alias = _attend(binding)
    ins[5] = ("int32", [3, 400])
    op = binding.Operation(name, param)
    context = binding.Context(0x77)
    tensors, outputs = _tensors(binding, ins), _tensors(binding, outs)
    st, need = op.setup(tensors, outputs, context)
    assert st == 0 and need > 0
    assert binding.ERROR_NAMES[op.execute(tensors, outputs, None, 0, context)] == PARAM
    assert binding.ERROR_NAMES[op.execute(tensors, outputs, FAKE, need - 1, context)] == PARAM


# ---- the C ABI

NORM = dict(x=FAKE, residual=FAKE, gamma=FAKE, out=FAKE, scale=FAKE, residual_out=FAKE + 64, rows=4, dim=96, xs=96, rs=96, dtype=1,
            eps=1e-5, stream=None)
LINEAR = dict(x=FAKE, w=FAKE, xs=FAKE, ws=FAKE, bias=None, out=FAKE, m=5, n=40, k=96, x_stride=96, w_stride=96, out_stride=40, dtype=1,
              workspace=None, bytes=0, stream=None)
WRITE = dict(key=FAKE, value=FAKE, kc=FAKE, vc=FAKE, kp=FAKE, vp=FAKE, slots=FAKE, tokens=3, heads=2, d=128, block=16, blocks=4,
             ks=256, vs=256, dtype=0, stream=None)
LOAD = dict(kc=FAKE, vc=FAKE, kp=FAKE, vp=FAKE, tables=FAKE, lens=FAKE, starts=None, key=FAKE, value=FAKE, batch=2, reach=3, heads=2,
            d=128, block=16, blocks=4, rows=10, longest=10, dtype=0, stream=None)


@pytest.mark.parametrize("call,good,bad", [
    ("atbmi_rms_norm_quant", NORM, b) for b in (dict(dtype=2), dict(rows=-1), dict(dim=0), dict(dim=65537), dict(xs=95), dict(rs=95),
                                                dict(eps=-1.0), dict(eps=float("inf")), dict(x=None), dict(gamma=None), dict(out=None),
                                                dict(scale=None), dict(residual_out=FAKE, xs=97), dict(rows=1 << 31))
] + [
    ("atbmi_linear_int8", LINEAR, b) for b in (dict(dtype=2), dict(m=-1), dict(k=0), dict(k=131072), dict(x_stride=95),
                                               dict(w_stride=95), dict(out_stride=39), dict(x=None), dict(ws=None), dict(out=None),
                                               dict(x_stride=(1 << 23) + 1), dict(w_stride=(1 << 23) + 1))
] + [
    ("atbmi_reshape_and_cache_int4", WRITE, b) for b in (dict(dtype=2), dict(tokens=-1), dict(heads=0), dict(d=96), dict(block=8),
                                                         dict(block=2048), dict(blocks=0), dict(blocks=1 << 30), dict(ks=255),
                                                         dict(vs=255), dict(key=None), dict(slots=None), dict(vc=FAKE + 8),
                                                         dict(kp=FAKE + 4))
] + [
    ("atbmi_paged_cache_load_int4", LOAD, b) for b in (dict(dtype=3), dict(batch=-1), dict(batch=70000), dict(heads=70000),
                                                       dict(reach=0), dict(reach=1 << 28), dict(rows=-1), dict(longest=-1),
                                                       dict(lens=None), dict(key=FAKE + 2), dict(kc=FAKE + 8), dict(d=80))
])
def test_c_calls_refused(binding, call, good, bad):
    lib = binding.kernels()
    assert getattr(lib, call)(*{**good, **bad}.values()) == 1
    assert call[6:].encode() in lib.atbmi_last_error()


PA = dict(dtype=1, numHeads=8, numKvHeads=2, headDim=128, blockSize=16, numBlocks=4, maxBlocksPerSeq=3, batch=2, queryTokens=1, maskLen=0,
          qkScale=0.1, reserved=0, maskSeqStride=0, maskHeadStride=0, maskRowStride=0, query=FAKE, keyCache=FAKE, valueCache=FAKE,
          keyParams=FAKE, valueParams=FAKE, blockTables=FAKE, contextLens=FAKE, mask=None, out=FAKE)


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(numHeads=0), dict(numHeads=7), dict(numKvHeads=0), dict(headDim=192), dict(blockSize=40),
                                 dict(numBlocks=0), dict(maxBlocksPerSeq=0), dict(maxBlocksPerSeq=1 << 26), dict(batch=-1),
                                 dict(queryTokens=0), dict(queryTokens=65), dict(qkScale=0.0), dict(qkScale=float("nan")),
                                 dict(reserved=1), dict(mask=FAKE), dict(mask=FAKE, maskLen=4, maskRowStride=-4),
                                 dict(batch=1 << 30), dict(query=None), dict(out=None), dict(contextLens=None),
                                 dict(query=FAKE + 8), dict(valueCache=FAKE + 8), dict(out=FAKE + 2)])
def test_c_attention_refused(binding, bad):
    lib = binding.kernels()
    call = binding.AtbmiPaInt4Call(**{**PA, **bad})
    assert lib.atbmi_pa_int4_decode(ctypes.byref(call), FAKE, 1 << 40, None) == 1
    assert b"pa_int4" in lib.atbmi_last_error()


def test_c_workspace(binding):
    lib = binding.kernels()
    call = binding.AtbmiPaInt4Call(**{**PA, "maxBlocksPerSeq": 100})
    need = ctypes.c_uint64()
    assert lib.atbmi_pa_int4_workspace_size(ctypes.byref(call), ctypes.byref(need)) == 0 and need.value > 0
    assert lib.atbmi_pa_int4_workspace_size(ctypes.byref(call), None) == 1
    assert lib.atbmi_pa_int4_workspace_size(None, ctypes.byref(need)) == 1
    for workspace, size in ((None, need.value), (FAKE, need.value - 1), (FAKE + 8, need.value)):
        assert lib.atbmi_pa_int4_decode(ctypes.byref(call), workspace, size, None) == 1
    assert lib.atbmi_linear_int8_workspace_size(64, 64, 64, None) == 1
    # nothing to do: no launch, whatever the pointers are
    assert lib.atbmi_pa_int4_decode(ctypes.byref(binding.AtbmiPaInt4Call(**{**PA, "batch": 0})), None, 0, None) == 0
    assert lib.atbmi_rms_norm_quant(*{**NORM, "rows": 0}.values()) == 0
    assert lib.atbmi_linear_int8(*{**LINEAR, "m": 0}.values()) == 0
    assert lib.atbmi_reshape_and_cache_int4(*{**WRITE, "tokens": 0}.values()) == 0
    for nothing in ("batch", "rows", "longest"):
        assert lib.atbmi_paged_cache_load_int4(*{**LOAD, nothing: 0}.values()) == 0


# ---- the torch functions

def _cpu_cache(d=128, heads=2, block=32, dtype=torch.bfloat16):
    return (torch.zeros(4, heads, block, d // 2, dtype=torch.uint8), torch.zeros(4, heads, d // 2, block, dtype=torch.uint8),
            torch.zeros(4, heads, block, 2, dtype=dtype), torch.zeros(4, heads, block, 2, dtype=dtype))


def test_functions_refuse(pkg):
    ops = pkg.quantized
    bf, i8, i32, f32 = torch.bfloat16, torch.int8, torch.int32, torch.float32
    x, gamma = torch.zeros(4, 96, dtype=bf), torch.zeros(96, dtype=bf)

    def refused(text, function, *args, **kw):
        with pytest.raises(ValueError, match=text):
            function(*args, **kw)

    refused("on a GPU", ops.rms_norm_quant, x, gamma)
    refused("float16 or bfloat16", ops.rms_norm_quant, x.float(), gamma)
    refused("2 dimensions", ops.rms_norm_quant, x[0], gamma)
    refused("no columns", ops.rms_norm_quant, x[:, :0], gamma[:0])
    refused("gamma", ops.rms_norm_quant, x, gamma[1:])
    refused("residual", ops.rms_norm_quant, x, gamma, residual=x[1:])
    refused("without a residual", ops.rms_norm_quant, x, gamma, residual_out=x)
    refused("no gaps", ops.rms_norm_quant, torch.zeros(96, 4, dtype=bf).t(), gamma)
    refused("out", ops.rms_norm_quant, x, gamma, out=torch.zeros(4, 96, dtype=torch.uint8))
    refused("contiguous", ops.rms_norm_quant, x, gamma, out=torch.zeros(4, 97, dtype=i8)[:, 1:])
    refused("scale", ops.rms_norm_quant, x, gamma, scale=torch.zeros(5))
    refused("residual_out", ops.rms_norm_quant, x, gamma, residual=x, residual_out=gamma)

    a, w, xs, ws = torch.zeros(4, 96, dtype=i8), torch.zeros(8, 96, dtype=i8), torch.zeros(4), torch.zeros(8)
    refused("on a GPU", ops.linear_int8, a, w, xs, ws, out_dtype=bf)
    refused("float16 or bfloat16", ops.linear_int8, a, w, xs, ws)
    refused("float16 or bfloat16", ops.linear_int8, a, w, xs, ws, out_dtype=f32)
    refused("x should be", ops.linear_int8, a.float(), w, xs, ws, out_dtype=bf)
    refused("weight", ops.linear_int8, a, w[:, 1:], xs, ws, out_dtype=bf)
    refused("x_scale", ops.linear_int8, a, w, xs[1:], ws, out_dtype=bf)
    refused("weight_scale", ops.linear_int8, a, w, xs, ws.half(), out_dtype=bf)
    refused("bias", ops.linear_int8, a, w, xs, ws, bias=xs, out_dtype=bf)
    refused("out_dtype", ops.linear_int8, a, w, xs, ws, out_dtype=bf, out=torch.zeros(4, 8).half())
    refused("out should", ops.linear_int8, a, w, xs, ws, out=torch.zeros(4, 9).half())

    cache = _cpu_cache()
    k, slots = torch.zeros(3, 2, 128, dtype=bf), torch.zeros(3, dtype=i32)
    refused("on a GPU", ops.reshape_and_cache_int4, k, k, *cache, slots)
    refused("key", ops.reshape_and_cache_int4, k[:, :1], k, *cache, slots)
    refused("value should be", ops.reshape_and_cache_int4, k, k.half(), *cache, slots)
    refused("slot_mapping", ops.reshape_and_cache_int4, k, k, *cache, slots.long())
    refused("tokens of key", ops.reshape_and_cache_int4, torch.zeros(3, 128, 2, dtype=bf).transpose(1, 2), k, *cache, slots)
    refused("value_cache", ops.reshape_and_cache_int4, k, k, cache[0], cache[0], *cache[2:], slots)
    refused("key_params", ops.reshape_and_cache_int4, k, k, *cache[:2], cache[2][:, :1], cache[3], slots)
    refused("float16 or bfloat16", ops.reshape_and_cache_int4, k, k, *cache[:2], cache[2].float(), cache[3].float(), slots)
    refused("4 dimensions", ops.reshape_and_cache_int4, k, k, cache[0][0], *cache[1:], slots)

    tables, lens = torch.zeros(2, 3, dtype=i32), torch.zeros(2, dtype=i32)
    refused("on a GPU", ops.paged_cache_load_int4, *cache, tables, lens, 10)
    refused("block_tables", ops.paged_cache_load_int4, *cache, tables[0], lens, 10)
    refused("seq_lens", ops.paged_cache_load_int4, *cache, tables, lens[1:], 10)
    refused("seq_starts", ops.paged_cache_load_int4, *cache, tables, lens, 10, seq_starts=lens.long())
    refused("key should", ops.paged_cache_load_int4, *cache, tables, lens, 10, key=torch.zeros(9, 2, 128, dtype=bf))

    q = torch.zeros(2, 8, 128, dtype=bf)
    refused("on a GPU", ops.paged_attention_int4, q, *cache, tables, lens, 0.1)
    refused("query should", ops.paged_attention_int4, q.half(), *cache, tables, lens, 0.1)
    refused("query should", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, query_tokens=2)
    refused("context_lens", ops.paged_attention_int4, q, *cache, tables, lens[:1], 0.1)
    refused("contiguous", ops.paged_attention_int4, torch.zeros(2, 9, 128, dtype=bf)[:, 1:], *cache, tables, lens, 0.1)
    mask = torch.zeros(2, 8, 1, 50, dtype=bf)
    refused("mask should have", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, mask=mask[:, :3])
    refused("mask should be", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, mask=mask.float())
    refused("next to each other", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, mask=mask[:, :, :, ::2])
    refused("next to each other", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, mask=mask[:, :, :, :0])
    refused("out should", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, out=mask)
    refused("workspace", ops.paged_attention_int4, q, *cache, tables, lens, 0.1, workspace=xs)

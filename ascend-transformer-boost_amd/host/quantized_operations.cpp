// The operators of a decoder layer's attention half with 8-bit activations and weights and a 4-bit KV cache, as
// atb::Operations: RmsNormQuant, LinearInt8, ReshapeAndCacheInt4, PagedCacheLoadInt4, PagedAttentionInt4. This library's
// own additions to the operators of the reference; tensors and params are described in atb/infer_op_params.h, the
// arithmetic in atbmi_kernels.h.
#include <algorithm>
#include <cmath>
#include <new>
#include "atb/infer_op_params.h"
#include "atb/utils.h"
#include "atbmi_kernels.h"
#include "log.h"
#include "operation_base.h"

namespace atb {
namespace {
using Types = std::vector<aclDataType>;

IrCombo Row(const Types &in, const Types &out)
{
    IrCombo c;
    c.inDtypes = in;
    c.inFormats.assign(in.size(), ACL_FORMAT_ND);
    c.outDtypes = out;
    c.outFormats.assign(out.size(), ACL_FORMAT_ND);
    return c;
}

// A row of the dtype table for each of the model's types.
template <typename F> OpIr BothTypes(F row)
{
    return {row(ACL_FLOAT16), row(ACL_BF16)};
}

int32_t ModelType(const TensorDesc &desc)
{
    return desc.dtype == ACL_BF16 ? ATBMI_BF16 : ATBMI_F16;
}

bool Is(const TensorDesc &desc, std::initializer_list<int64_t> dims)
{
    return desc.shape.dimNum == dims.size() && std::equal(dims.begin(), dims.end(), desc.shape.dims);
}

Status WrongShape(const std::string &op, const char *what)
{
    ATB_LOG(ERROR) << op << ": " << what;
    return ERROR_INVALID_TENSOR_DIM;
}

Status WrongRank(const std::string &op, const char *what)
{
    ATB_LOG(ERROR) << op << ": " << what;
    return ERROR_INVALID_TENSOR_DIM_NUM;
}

const void *At(const SVector<Tensor> &tensors, size_t i)
{
    return tensors.at(i).deviceData;
}

int64_t Dim(const SVector<Tensor> &tensors, size_t i, size_t d)
{
    return tensors.at(i).desc.shape.dims[d];
}

// What the five share: one check of the input descriptions for InferShape and Setup, outputs that have the shapes InferShape
// gives them, operands on the device, and the kernel library's code on a failed launch.
class QuantizedOperation : public OperationBase {
public:
    QuantizedOperation(const char *name, const OpIr &ir, uint32_t inputs, uint32_t outputs)
        : OperationBase(name), op_(name), inputs_(inputs), outputs_(outputs)
    {
        ir_ = &ir;
    }
    uint32_t GetInputNum() const override { return inputs_; }
    uint32_t GetOutputNum() const override { return outputs_; }

protected:
    virtual Status DimCheck(const SVector<TensorDesc> &in) const = 0;
    // Input that output i is, updated in place; -1: none.
    virtual int InPlace(size_t i) const
    {
        (void)i;
        return -1;
    }
    virtual uint64_t Workspace(const VariantPack &pack, int &rc) const
    {
        (void)pack;
        rc = 0;
        return 0;
    }
    virtual int Launch(const VariantPack &pack, uint8_t *workspace, uint64_t workspaceSize, aclrtStream stream) const = 0;

    Status InferShapeCheckImpl(const SVector<TensorDesc> &in) const override { return DimCheck(in); }

    Status SetupCheckImpl(const SVector<Tensor> &inTensors, const SVector<Tensor> &outTensors) const override
    {
        SVector<TensorDesc> in, want;
        for (size_t i = 0; i < inTensors.size(); ++i) {
            in.push_back(inTensors.at(i).desc);
        }
        Status st = DimCheck(in);
        if (st != NO_ERROR) {
            return st;
        }
        want.resize(outputs_);
        st = InferShapeImpl(in, want);
        if (st != NO_ERROR) {
            return st;
        }
        for (size_t i = 0; i < outputs_; ++i) {
            const TensorDesc &have = outTensors.at(i).desc;
            if (have.shape.dimNum != want.at(i).shape.dimNum ||
                !std::equal(have.shape.dims, have.shape.dims + have.shape.dimNum, want.at(i).shape.dims)) {
                return WrongShape(op_, "the outputs should have the shapes that InferShape gives");
            }
        }
        return NO_ERROR;
    }

    Status PlanImpl(const VariantPack &pack, uint64_t &workspaceSize) override
    {
        for (size_t i = 0; i < inputs_; ++i) {
            if (!pack.inTensors.at(i).deviceData) {
                ATB_LOG(ERROR) << op_ << ": input " << i << " should be on the device";
                return ERROR_INVALID_PARAM;
            }
        }
        for (size_t i = 0; i < outputs_; ++i) {
            const int from = InPlace(i);
            if (!pack.outTensors.at(i).deviceData ||
                (from >= 0 && pack.outTensors.at(i).deviceData != pack.inTensors.at(from).deviceData)) {
                ATB_LOG(ERROR) << op_ << ": output " << i << " should be on the device"
                               << (from >= 0 ? ", the same tensor as the input that is updated in place" : "");
                return ERROR_INVALID_PARAM;
            }
        }
        int rc = 0;
        workspaceSize = Workspace(pack, rc);
        if (rc != 0) {
            ATB_LOG(ERROR) << op_ << ": " << atbmi_last_error();
        }
        return rc;
    }

    Status LaunchImpl(const VariantPack &pack, uint8_t *workspace, uint64_t workspaceSize, aclrtStream stream) override
    {
        const int rc = Launch(pack, workspace, workspaceSize, stream);
        if (rc != 0) {
            ATB_LOG(ERROR) << op_ << " launch failed: " << atbmi_last_error();
        }
        return rc;
    }

    const std::string op_;

private:
    uint32_t inputs_;
    uint32_t outputs_;
};

class RmsNormQuantOperation : public QuantizedOperation {
public:
    explicit RmsNormQuantOperation(const infer::RmsNormQuantParam &param)
        : QuantizedOperation("RmsNormQuantOperation", Table(param.hasResidual), param.hasResidual ? 3 : 2,
                             param.hasResidual ? 3 : 2),
          param_(param)
    {
    }

protected:
    Status DimCheck(const SVector<TensorDesc> &in) const override
    {
        const Dims &x = in.at(0).shape;
        if (x.dimNum != 2 || in.at(1).shape.dimNum != 1) {
            return WrongRank(op_, "x should have 2 dims, gamma 1");
        }
        if (x.dims[1] > 65536 || x.dims[0] > 0x7fffffffLL) {
            return WrongShape(op_, "rows of up to 65536 values, up to 2^31 - 1 of them");
        }
        if (!Is(in.at(1), {x.dims[1]}) || (param_.hasResidual && !Is(in.at(2), {x.dims[0], x.dims[1]}))) {
            return WrongShape(op_, "gamma should be as long as a row, the residual as large as x");
        }
        return NO_ERROR;
    }

    Status InferShapeImpl(const SVector<TensorDesc> &in, SVector<TensorDesc> &out) const override
    {
        out.at(0) = in.at(0);
        out.at(0).dtype = ACL_INT8;
        out.at(1) = in.at(0);
        out.at(1).dtype = ACL_FLOAT;
        out.at(1).shape.dimNum = 1;
        if (param_.hasResidual) {
            out.at(2) = in.at(0);
        }
        return NO_ERROR;
    }

    int Launch(const VariantPack &pack, uint8_t *, uint64_t, aclrtStream stream) const override
    {
        const int64_t rows = Dim(pack.inTensors, 0, 0), dim = Dim(pack.inTensors, 0, 1);
        const bool residual = param_.hasResidual;
        return atbmi_rms_norm_quant(At(pack.inTensors, 0), residual ? At(pack.inTensors, 2) : nullptr,
                                    At(pack.inTensors, 1), static_cast<int8_t *>(pack.outTensors.at(0).deviceData),
                                    static_cast<float *>(pack.outTensors.at(1).deviceData),
                                    residual ? pack.outTensors.at(2).deviceData : nullptr, rows, dim, dim, dim,
                                    ModelType(pack.inTensors.at(0).desc), param_.epsilon, stream);
    }

private:
    static const OpIr &Table(bool residual)
    {
        static const OpIr plain = BothTypes([](aclDataType t) { return Row({t, t}, {ACL_INT8, ACL_FLOAT}); });
        static const OpIr added = BothTypes([](aclDataType t) { return Row({t, t, t}, {ACL_INT8, ACL_FLOAT, t}); });
        return residual ? added : plain;
    }
    infer::RmsNormQuantParam param_;
};

class LinearInt8Operation : public QuantizedOperation {
public:
    explicit LinearInt8Operation(const infer::LinearInt8Param &param)
        : QuantizedOperation("LinearInt8Operation", Table(param.hasBias, param.outDataType == ACL_BF16),
                             param.hasBias ? 5 : 4, 1),
          param_(param)
    {
    }

protected:
    Status DimCheck(const SVector<TensorDesc> &in) const override
    {
        const Dims &x = in.at(0).shape, &w = in.at(1).shape;
        if (x.dimNum != 2 || w.dimNum != 2) {
            return WrongRank(op_, "x and weight should have 2 dims");
        }
        if (x.dims[1] != w.dims[1] || !Is(in.at(2), {x.dims[0]}) || !Is(in.at(3), {w.dims[0]}) ||
            (param_.hasBias && !Is(in.at(4), {w.dims[0]}))) {
            return WrongShape(op_, "x [m, k], weight [n, k], xScale [m], weightScale and bias [n] are expected");
        }
        return NO_ERROR;
    }

    Status InferShapeImpl(const SVector<TensorDesc> &in, SVector<TensorDesc> &out) const override
    {
        out.at(0) = in.at(0);
        out.at(0).dtype = param_.outDataType;
        out.at(0).shape.dims[1] = in.at(1).shape.dims[0];
        return NO_ERROR;
    }

    uint64_t Workspace(const VariantPack &pack, int &rc) const override
    {
        uint64_t bytes = 0;
        rc = atbmi_linear_int8_workspace_size(Dim(pack.inTensors, 0, 0), Dim(pack.inTensors, 1, 0),
                                              Dim(pack.inTensors, 0, 1), &bytes);
        return bytes;
    }

    int Launch(const VariantPack &pack, uint8_t *workspace, uint64_t workspaceSize, aclrtStream stream) const override
    {
        const int64_t m = Dim(pack.inTensors, 0, 0), n = Dim(pack.inTensors, 1, 0), k = Dim(pack.inTensors, 0, 1);
        return atbmi_linear_int8(
            static_cast<const int8_t *>(At(pack.inTensors, 0)), static_cast<const int8_t *>(At(pack.inTensors, 1)),
            static_cast<const float *>(At(pack.inTensors, 2)), static_cast<const float *>(At(pack.inTensors, 3)),
            param_.hasBias ? static_cast<const float *>(At(pack.inTensors, 4)) : nullptr, pack.outTensors.at(0).deviceData,
            m, n, k, k, k, n, param_.outDataType == ACL_BF16 ? ATBMI_BF16 : ATBMI_F16, workspace, workspaceSize, stream);
    }

private:
    static const OpIr &Table(bool bias, bool bf16)
    {
        auto make = [](bool withBias, aclDataType out) {
            Types in = {ACL_INT8, ACL_INT8, ACL_FLOAT, ACL_FLOAT};
            if (withBias) {
                in.push_back(ACL_FLOAT);
            }
            return OpIr{Row(in, {out})};
        };
        static const OpIr tables[2][2] = {{make(false, ACL_FLOAT16), make(false, ACL_BF16)},
                                          {make(true, ACL_FLOAT16), make(true, ACL_BF16)}};
        return tables[bias][bf16];
    }
    infer::LinearInt8Param param_;
};

// The cache's four tensors, from input `at` on: their dims agree and are what the kernels take.
Status CacheCheck(const std::string &op, const SVector<TensorDesc> &in, size_t at)
{
    const Dims &k = in.at(at).shape;
    if (k.dimNum != 4) {
        return WrongRank(op, "keyCache should have 4 dims");
    }
    const int64_t blocks = k.dims[0], heads = k.dims[1], blockSize = k.dims[2], half = k.dims[3];
    if (!Is(in.at(at + 1), {blocks, heads, half, blockSize}) || !Is(in.at(at + 2), {blocks, heads, blockSize, 2}) ||
        !Is(in.at(at + 3), {blocks, heads, blockSize, 2})) {
        return WrongShape(op, "keyCache [blocks, heads, blockSize, headSize / 2], valueCache [blocks, heads, headSize / 2, "
                              "blockSize] and params [blocks, heads, blockSize, 2] are expected");
    }
    if ((half != 32 && half != 64 && half != 128) || blockSize % 16 != 0 || blockSize > 1024 ||
        blocks > 0x7fffffffLL / blockSize) {
        return WrongShape(op, "head sizes of 64, 128 and 256, blocks of a multiple of 16 up to 1024 tokens, 32-bit slots");
    }
    return NO_ERROR;
}

class ReshapeAndCacheInt4Operation : public QuantizedOperation {
public:
    explicit ReshapeAndCacheInt4Operation(const infer::ReshapeAndCacheInt4Param &)
        : QuantizedOperation("ReshapeAndCacheInt4Operation", Table(), 7, 4)
    {
    }

protected:
    Status DimCheck(const SVector<TensorDesc> &in) const override
    {
        Status st = CacheCheck(op_, in, 2);
        if (st != NO_ERROR) {
            return st;
        }
        const Dims &key = in.at(0).shape, &cache = in.at(2).shape;
        if (key.dimNum != 3) {
            return WrongRank(op_, "key should have 3 dims");
        }
        if (key.dims[1] != cache.dims[1] || key.dims[2] != 2 * cache.dims[3] ||
            !Is(in.at(1), {key.dims[0], key.dims[1], key.dims[2]}) || !Is(in.at(6), {key.dims[0]})) {
            return WrongShape(op_, "key and value [tokens, heads, headSize] as in the cache, slotMapping [tokens] are expected");
        }
        return NO_ERROR;
    }
    Status InferShapeImpl(const SVector<TensorDesc> &in, SVector<TensorDesc> &out) const override
    {
        for (size_t i = 0; i < 4; ++i) {
            out.at(i) = in.at(2 + i);
        }
        return NO_ERROR;
    }
    int InPlace(size_t i) const override { return static_cast<int>(2 + i); }

    int Launch(const VariantPack &pack, uint8_t *, uint64_t, aclrtStream stream) const override
    {
        const SVector<Tensor> &in = pack.inTensors;
        const int64_t heads = Dim(in, 0, 1), d = Dim(in, 0, 2);
        return atbmi_reshape_and_cache_int4(
            At(in, 0), At(in, 1), static_cast<uint8_t *>(in.at(2).deviceData), static_cast<uint8_t *>(in.at(3).deviceData),
            in.at(4).deviceData, in.at(5).deviceData, static_cast<const int32_t *>(At(in, 6)), Dim(in, 0, 0), heads, d,
            Dim(in, 2, 2), Dim(in, 2, 0), heads * d, heads * d, ModelType(in.at(0).desc), stream);
    }

private:
    static const OpIr &Table()
    {
        static const OpIr table = BothTypes([](aclDataType t) {
            return Row({t, t, ACL_UINT8, ACL_UINT8, t, t, ACL_INT32}, {ACL_UINT8, ACL_UINT8, t, t});
        });
        return table;
    }
};

class PagedCacheLoadInt4Operation : public QuantizedOperation {
public:
    explicit PagedCacheLoadInt4Operation(const infer::PagedCacheLoadInt4Param &param)
        : QuantizedOperation("PagedCacheLoadInt4Operation", Table(param.hasSeqStarts), param.hasSeqStarts ? 9 : 8, 2),
          param_(param)
    {
    }

protected:
    Status DimCheck(const SVector<TensorDesc> &in) const override
    {
        Status st = CacheCheck(op_, in, 0);
        if (st != NO_ERROR) {
            return st;
        }
        const Dims &cache = in.at(0).shape, &tables = in.at(4).shape, &key = in.at(6).shape;
        if (tables.dimNum != 2 || key.dimNum != 3) {
            return WrongRank(op_, "blockTables should have 2 dims, key and value 3");
        }
        if (!Is(in.at(5), {tables.dims[0]}) || key.dims[1] != cache.dims[1] || key.dims[2] != 2 * cache.dims[3] ||
            !Is(in.at(7), {key.dims[0], key.dims[1], key.dims[2]}) ||
            (param_.hasSeqStarts && !Is(in.at(8), {tables.dims[0]}))) {
            return WrongShape(op_, "seqLens and seqStarts [batch], key and value [tokens, heads, headSize] are expected");
        }
        if (tables.dims[0] > 65535 || cache.dims[1] > 65535 || tables.dims[1] > ((1LL << 30) - 1) / cache.dims[2]) {
            return WrongShape(op_, "up to 65535 sequences and heads, tables that reach less than 2^30 positions");
        }
        return NO_ERROR;
    }
    Status InferShapeImpl(const SVector<TensorDesc> &in, SVector<TensorDesc> &out) const override
    {
        out.at(0) = in.at(6);
        out.at(1) = in.at(7);
        return NO_ERROR;
    }
    int InPlace(size_t i) const override { return static_cast<int>(6 + i); }

    int Launch(const VariantPack &pack, uint8_t *, uint64_t, aclrtStream stream) const override
    {
        const SVector<Tensor> &in = pack.inTensors;
        const int64_t blockSize = Dim(in, 0, 2), reach = Dim(in, 4, 1), rows = Dim(in, 6, 0);
        // (a sequence is no longer than the output holds)
        return atbmi_paged_cache_load_int4(
            static_cast<const uint8_t *>(At(in, 0)), static_cast<const uint8_t *>(At(in, 1)), At(in, 2), At(in, 3),
            static_cast<const int32_t *>(At(in, 4)), static_cast<const int32_t *>(At(in, 5)),
            param_.hasSeqStarts ? static_cast<const int32_t *>(At(in, 8)) : nullptr, in.at(6).deviceData,
            in.at(7).deviceData, Dim(in, 4, 0), reach, Dim(in, 0, 1), Dim(in, 6, 2), blockSize, Dim(in, 0, 0), rows,
            std::min(rows, reach * blockSize), ModelType(in.at(2).desc), stream);
    }

private:
    static const OpIr &Table(bool starts)
    {
        auto make = [](bool withStarts) {
            return BothTypes([withStarts](aclDataType t) {
                Types in = {ACL_UINT8, ACL_UINT8, t, t, ACL_INT32, ACL_INT32, t, t};
                if (withStarts) {
                    in.push_back(ACL_INT32);
                }
                return Row(in, {t, t});
            });
        };
        static const OpIr tables[2] = {make(false), make(true)};
        return tables[starts];
    }
    infer::PagedCacheLoadInt4Param param_;
};

class PagedAttentionInt4Operation : public QuantizedOperation {
public:
    explicit PagedAttentionInt4Operation(const infer::PagedAttentionInt4Param &param)
        : QuantizedOperation("PagedAttentionInt4Operation", Table(param.hasMask), param.hasMask ? 8 : 7, 1), param_(param)
    {
    }

protected:
    Status DimCheck(const SVector<TensorDesc> &in) const override
    {
        Status st = CacheCheck(op_, in, 1);
        if (st != NO_ERROR) {
            return st;
        }
        const Dims &cache = in.at(1).shape, &tables = in.at(5).shape;
        if (tables.dimNum != 2 || (param_.hasMask && in.at(7).shape.dimNum != 4)) {
            return WrongRank(op_, "blockTables should have 2 dims, a mask 4");
        }
        if (cache.dims[1] != param_.kvHeadNum) {
            return WrongShape(op_, "the cache should have kvHeadNum heads");
        }
        const int64_t batch = tables.dims[0];
        if (batch > 0x7fffffffLL / param_.queryTokens || tables.dims[1] * cache.dims[2] >= (1LL << 30) ||
            !Is(in.at(0), {batch * param_.queryTokens, param_.headNum, 2 * cache.dims[3]}) || !Is(in.at(6), {batch})) {
            return WrongShape(op_, "query [batch * queryTokens, headNum, headSize], contextLens [batch], tables that reach "
                                   "less than 2^30 positions are expected");
        }
        if (param_.hasMask) {
            const int64_t want[3] = {batch, param_.headNum, param_.queryTokens};
            const Dims &mask = in.at(7).shape;
            for (int i = 0; i < 3; ++i) {
                if (mask.dims[i] != 1 && mask.dims[i] != want[i]) {
                    return WrongShape(op_, "mask [batch | 1, headNum | 1, queryTokens | 1, positions] is expected");
                }
            }
            if (mask.dims[3] > 0x7fffffffLL) {
                return WrongShape(op_, "a mask of less than 2^31 positions is expected");
            }
        }
        return NO_ERROR;
    }
    Status InferShapeImpl(const SVector<TensorDesc> &in, SVector<TensorDesc> &out) const override
    {
        out.at(0) = in.at(0);
        return NO_ERROR;
    }

    uint64_t Workspace(const VariantPack &pack, int &rc) const override
    {
        uint64_t bytes = 0;
        const AtbmiPaInt4Call call = Call(pack);
        rc = atbmi_pa_int4_workspace_size(&call, &bytes);
        return bytes;
    }

    int Launch(const VariantPack &pack, uint8_t *workspace, uint64_t workspaceSize, aclrtStream stream) const override
    {
        const AtbmiPaInt4Call call = Call(pack);
        return atbmi_pa_int4_decode(&call, workspace, workspaceSize, stream);
    }

private:
    AtbmiPaInt4Call Call(const VariantPack &pack) const
    {
        const SVector<Tensor> &in = pack.inTensors;
        AtbmiPaInt4Call c{};
        c.dtype = ModelType(in.at(0).desc);
        c.numHeads = param_.headNum;
        c.numKvHeads = param_.kvHeadNum;
        c.headDim = static_cast<int32_t>(Dim(in, 0, 2));
        c.blockSize = static_cast<int32_t>(Dim(in, 1, 2));
        c.numBlocks = static_cast<int32_t>(Dim(in, 1, 0));
        c.maxBlocksPerSeq = static_cast<int32_t>(Dim(in, 5, 1));
        c.batch = static_cast<int32_t>(Dim(in, 5, 0));
        c.queryTokens = param_.queryTokens;
        c.qkScale = param_.qkScale;
        c.query = At(in, 0);
        c.keyCache = static_cast<const uint8_t *>(At(in, 1));
        c.valueCache = static_cast<const uint8_t *>(At(in, 2));
        c.keyParams = At(in, 3);
        c.valueParams = At(in, 4);
        c.blockTables = static_cast<const int32_t *>(At(in, 5));
        c.contextLens = static_cast<const int32_t *>(At(in, 6));
        c.out = pack.outTensors.at(0).deviceData;
        if (param_.hasMask) {
            const int64_t *d = in.at(7).desc.shape.dims;
            c.mask = At(in, 7);
            c.maskLen = static_cast<int32_t>(d[3]);
            c.maskSeqStride = d[0] > 1 ? d[1] * d[2] * d[3] : 0;
            c.maskHeadStride = d[1] > 1 ? d[2] * d[3] : 0;
            c.maskRowStride = d[2] > 1 ? d[3] : 0;
        }
        return c;
    }
    static const OpIr &Table(bool mask)
    {
        auto make = [](bool withMask) {
            return BothTypes([withMask](aclDataType t) {
                Types in = {t, ACL_UINT8, ACL_UINT8, t, t, ACL_INT32, ACL_INT32};
                if (withMask) {
                    in.push_back(t);
                }
                return Row(in, {t});
            });
        };
        static const OpIr tables[2] = {make(false), make(true)};
        return tables[mask];
    }
    infer::PagedAttentionInt4Param param_;
};

template <typename Op, typename Param> Status Create(const Param &param, bool valid, const char *why, Operation **operation)
{
    if (operation == nullptr) {
        return ERROR_INVALID_PARAM;
    }
    if (!ReservedIsZero(param)) {
        ATB_LOG(ERROR) << "a reserved byte of the param is not zero";
        return ERROR_INVALID_PARAM;
    }
    if (!valid) {
        ATB_LOG(ERROR) << why;
        return ERROR_INVALID_PARAM;
    }
    *operation = new (std::nothrow) Op(param);
    return *operation == nullptr ? ERROR_OUT_OF_HOST_MEMORY : NO_ERROR;
}
} // namespace

template <> Status CreateOperation(const infer::RmsNormQuantParam &opParam, Operation **operation)
{
    return Create<RmsNormQuantOperation>(opParam, std::isfinite(opParam.epsilon) && opParam.epsilon >= 0.0f,
                                         "RmsNormQuantParam epsilon should be finite and not below 0", operation);
}

template <> Status CreateOperation(const infer::LinearInt8Param &opParam, Operation **operation)
{
    return Create<LinearInt8Operation>(opParam, opParam.outDataType == ACL_FLOAT16 || opParam.outDataType == ACL_BF16,
                                       "LinearInt8Param outDataType should be ACL_FLOAT16 or ACL_BF16", operation);
}

template <> Status CreateOperation(const infer::ReshapeAndCacheInt4Param &opParam, Operation **operation)
{
    return Create<ReshapeAndCacheInt4Operation>(opParam, true, "", operation);
}

template <> Status CreateOperation(const infer::PagedCacheLoadInt4Param &opParam, Operation **operation)
{
    return Create<PagedCacheLoadInt4Operation>(opParam, true, "", operation);
}

template <> Status CreateOperation(const infer::PagedAttentionInt4Param &opParam, Operation **operation)
{
    const bool heads = opParam.kvHeadNum > 0 && opParam.headNum > 0 && opParam.headNum <= (1 << 20) &&
                       opParam.headNum % opParam.kvHeadNum == 0;
    return Create<PagedAttentionInt4Operation>(
        opParam, heads && opParam.queryTokens >= 1 && opParam.queryTokens <= 64 && std::isfinite(opParam.qkScale) && opParam.qkScale > 0.0f,
        "PagedAttentionInt4Param: headNum should be a multiple of kvHeadNum, queryTokens 1 .. 64, qkScale finite and above 0",
        operation);
}
} // namespace atb

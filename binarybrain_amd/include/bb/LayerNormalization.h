// Layer normalisation: every frame is normalised over all nodes of the layer, then each node is mapped by a gamma and beta of its own, which are trained.  Unlike
// StochasticBatchNormalization it keeps no running statistics, and training and inference compute the same.  (The reference has no such layer.)
// BinType Bit: packed bits in, read as 0 and 1; the output and both gradients are fp32.
// Serialized as  version 1 | Model part | shape | eps | gamma | beta (both as typed tensor objects).
#pragma once

#include "bb/Model.h"
#include "bb/Workspace.h"

namespace bb {

template <typename BinType = float, typename RealType = float>
class LayerNormalization : public Model {
    static_assert(std::is_same<RealType, float>::value, "outputs and gradients are fp32");
    static_assert(std::is_same<BinType, float>::value || std::is_same<BinType, Bit>::value, "inputs are fp32 or packed bits");
    static constexpr bool kBit = std::is_same<BinType, Bit>::value;

    indices_t m_shape;
    float     m_eps = 1.0e-5f;
    std::shared_ptr<Tensor_<float>> m_gamma  = std::make_shared<Tensor_<float>>(), m_beta  = std::make_shared<Tensor_<float>>();
    std::shared_ptr<Tensor_<float>> m_dgamma = std::make_shared<Tensor_<float>>(), m_dbeta = std::make_shared<Tensor_<float>>();
    Workspace m_work;

public:
    struct create_t {
        float eps = 1.0e-5f;
    };

protected:
    explicit LayerNormalization(create_t const &create) : m_eps(create.eps)
    {
        m_gamma->Resize(0); m_beta->Resize(0); m_dgamma->Resize(0); m_dbeta->Resize(0);        // (no nodes before SetInputShape)
    }

    void DumpObjectData(std::ostream &os) const override
    {
        SaveValue(os, (std::int64_t)1);
        Model::DumpObjectData(os);
        SaveIndices(os, m_shape);
        SaveValue(os, m_eps);
        m_gamma->DumpObject(os);
        m_beta->DumpObject(os);
    }

    void LoadObjectData(std::istream &is) override
    {
        std::int64_t ver = -1;
        LoadValue(is, ver);
        BB_ASSERT(ver == 1);
        Model::LoadObjectData(is);
        m_shape = LoadIndices(is);
        LoadValue(is, m_eps);
        m_gamma->LoadObject(is);
        m_beta->LoadObject(is);
        index_t const nodes = m_shape.empty() ? 0 : CalcShapeSize(m_shape);
        BB_ASSERT(is.good() && m_gamma->GetSize() == nodes && m_beta->GetSize() == nodes);
        m_dgamma->Resize(m_gamma->GetShape()); m_dgamma->FillZero();
        m_dbeta->Resize(m_beta->GetShape());   m_dbeta->FillZero();
    }

    void RequireDevice(FrameBuffer const &buf) const
    {
        if (!buf.IsDeviceAvailable()) { throw Exception("LayerNormalization: host-only execution is not provided by this library (device path only)"); }
    }

public:
    static std::string ModelName(void)  { return "LayerNormalization"; }
    static std::string ObjectName(void) { return ModelName() + "_" + DataType<BinType>::Name() + "_" + DataType<RealType>::Name(); }
    std::string GetModelName(void) const override  { return ModelName(); }
    std::string GetObjectName(void) const override { return ObjectName(); }

    static std::shared_ptr<LayerNormalization> Create(create_t const &create) { return std::shared_ptr<LayerNormalization>(new LayerNormalization(create)); }
    static std::shared_ptr<LayerNormalization> Create(float eps = 1.0e-5f)
    {
        create_t c;
        c.eps = eps;
        return Create(c);
    }

    float   GetEps(void) const { return m_eps; }
    Tensor &gamma(void)  { return *m_gamma; }
    Tensor &beta(void)   { return *m_beta; }
    Tensor &dgamma(void) { return *m_dgamma; }
    Tensor &dbeta(void)  { return *m_dbeta; }
    auto lock_gamma(void)        { return m_gamma->Lock(); }
    auto lock_gamma_const(void) const { return m_gamma->LockConst(); }
    auto lock_beta(void)         { return m_beta->Lock(); }
    auto lock_beta_const(void) const  { return m_beta->LockConst(); }
    auto lock_dgamma_const(void) const { return m_dgamma->LockConst(); }
    auto lock_dbeta_const(void) const  { return m_dbeta->LockConst(); }

    Variables GetParameters(void) override
    {
        Variables v;
        if (!m_parameter_lock) { v.PushBack(m_gamma); v.PushBack(m_beta); }
        return v;
    }
    Variables GetGradients(void) override
    {
        Variables v;
        if (!m_parameter_lock) { v.PushBack(m_dgamma); v.PushBack(m_dbeta); }
        return v;
    }

    // a repeated shape changes nothing; a new one starts at gamma 1, beta 0
    indices_t SetInputShape(indices_t shape) override
    {
        if (shape == m_shape) { return m_shape; }
        m_shape = shape;
        index_t const nodes = CalcShapeSize(shape);
        m_gamma->Resize(nodes);  *m_gamma = 1.0f;
        m_beta->Resize(nodes);   *m_beta  = 0.0f;
        m_dgamma->Resize(nodes); m_dgamma->FillZero();
        m_dbeta->Resize(nodes);  m_dbeta->FillZero();
        return m_shape;
    }
    indices_t GetInputShape(void) const override  { return m_shape; }
    indices_t GetOutputShape(void) const override { return m_shape; }

    std::vector<double> ForwardNode(index_t, std::vector<double>) const override
    {
        throw Exception("LayerNormalization: a node's value depends on all nodes of its frame");
    }

    FrameBuffer Forward(FrameBuffer x_buf, bool train = true) override
    {
        RequireDevice(x_buf);
        BB_ASSERT(x_buf.GetType() == DataType<BinType>::type);
        if (x_buf.GetShape() != m_shape) { SetInputShape(x_buf.GetShape()); }
        FrameBuffer y_buf(x_buf.GetFrameSize(), x_buf.GetShape(), BB_TYPE_FP32);
        FrameBuffer stat_buf;
        if (train) { stat_buf = FrameBuffer(x_buf.GetFrameSize(), indices_t({2}), BB_TYPE_FP32); }         // mean and rstd of every frame
        int const nodes = (int)x_buf.GetNodeSize(), frames = (int)x_buf.GetFrameSize();
        std::size_t const size = bbhip_LayerNormalization_WorkspaceBytes(nodes, frames);
        {
            auto px = x_buf.LockDeviceMemoryConst();
            auto py = y_buf.LockDeviceMemory(true);
            auto pg = m_gamma->LockDeviceMemoryConst();
            auto pb = m_beta->LockDeviceMemoryConst();
            float *mean = train ? (float *)stat_buf.LockDeviceMemory(true).GetAddr() : nullptr;
            float *rstd = train ? mean + stat_buf.GetFrameStride() / 4 : nullptr;
            int const x_stride = (int)(x_buf.GetFrameStride() / 4), y_stride = (int)(y_buf.GetFrameStride() / 4);
            if (kBit) {
                CheckDevice(bbhip_bit_fp32_LayerNormalization_Forward((int const *)px.GetAddr(), (float *)py.GetAddr(), (float const *)pg.GetAddr(), (float const *)pb.GetAddr(),
                                mean, rstd, m_eps, nodes, frames, x_stride, y_stride, m_work.Get(size), size, nullptr), "bbhip_bit_fp32_LayerNormalization_Forward");
            }
            else {
                CheckDevice(bbhip_fp32_LayerNormalization_Forward((float const *)px.GetAddr(), (float *)py.GetAddr(), (float const *)pg.GetAddr(), (float const *)pb.GetAddr(),
                                mean, rstd, m_eps, nodes, frames, x_stride, y_stride, m_work.Get(size), size, nullptr), "bbhip_fp32_LayerNormalization_Forward");
            }
        }
        if (train) { PushFrameBuffer(x_buf); PushFrameBuffer(stat_buf); }
        return y_buf;
    }

    // the gradients of gamma and beta accumulate until the optimizer or FillZero clears them, as those of the other layers
    FrameBuffer Backward(FrameBuffer dy_buf) override
    {
        if (dy_buf.Empty()) { return FrameBuffer(); }
        RequireDevice(dy_buf);
        BB_ASSERT(dy_buf.GetType() == BB_TYPE_FP32);
        FrameBuffer stat_buf = PopFrameBuffer();
        FrameBuffer x_buf = PopFrameBuffer();
        BB_ASSERT(x_buf.GetFrameSize() == dy_buf.GetFrameSize() && x_buf.GetNodeSize() == dy_buf.GetNodeSize());
        FrameBuffer dx_buf(dy_buf.GetFrameSize(), dy_buf.GetShape(), BB_TYPE_FP32);
        int const nodes = (int)dy_buf.GetNodeSize(), frames = (int)dy_buf.GetFrameSize();
        std::size_t const size = bbhip_LayerNormalization_WorkspaceBytes(nodes, frames);
        auto px  = x_buf.LockDeviceMemoryConst();
        auto pdy = dy_buf.LockDeviceMemoryConst();
        auto pdx = dx_buf.LockDeviceMemory(true);
        auto ps  = stat_buf.LockDeviceMemoryConst();
        auto pg  = m_gamma->LockDeviceMemoryConst();
        auto pdg = m_dgamma->LockDeviceMemory();
        auto pdb = m_dbeta->LockDeviceMemory();
        float const *mean = (float const *)ps.GetAddr(), *rstd = mean + stat_buf.GetFrameStride() / 4;
        int const x_stride = (int)(x_buf.GetFrameStride() / 4), stride = (int)(dy_buf.GetFrameStride() / 4);
        if (kBit) {
            CheckDevice(bbhip_bit_fp32_LayerNormalization_Backward((int const *)px.GetAddr(), (float const *)pdy.GetAddr(), (float *)pdx.GetAddr(), (float const *)pg.GetAddr(),
                            mean, rstd, (float *)pdg.GetAddr(), (float *)pdb.GetAddr(), 1, nodes, frames, x_stride, stride, m_work.Get(size), size, nullptr),
                        "bbhip_bit_fp32_LayerNormalization_Backward");
        }
        else {
            CheckDevice(bbhip_fp32_LayerNormalization_Backward((float const *)px.GetAddr(), (float const *)pdy.GetAddr(), (float *)pdx.GetAddr(), (float const *)pg.GetAddr(),
                            mean, rstd, (float *)pdg.GetAddr(), (float *)pdb.GetAddr(), 1, nodes, frames, x_stride, stride, m_work.Get(size), size, nullptr),
                        "bbhip_fp32_LayerNormalization_Backward");
        }
        return dx_buf;
    }
};

}  // namespace bb

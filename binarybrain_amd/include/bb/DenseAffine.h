// A dense layer: every output node sees every input node, y = activation(W x + b), W and b are trained.  BinType Bit: packed bits in, read as 0 and 1; output and gradients are fp32.
// A residual of the output's shape may be added ahead of the activation.  (The reference's layer of this name is a host loop or a BLAS product without the epilogue; its objects are others.)
// Serialized as  version 1 | Model part | input shape | output shape | activation | W | b (both as typed tensor objects).
#pragma once

#include "bb/Model.h"
#include "bb/Workspace.h"

namespace bb {

template <typename BinType = float, typename RealType = float>
class DenseAffine : public Model {
    static_assert(std::is_same<RealType, float>::value, "outputs and gradients are fp32");
    static_assert(std::is_same<BinType, float>::value || std::is_same<BinType, Bit>::value, "inputs are fp32 or packed bits");
    static constexpr bool kBit = std::is_same<BinType, Bit>::value;

public:
    struct create_t {
        indices_t   output_shape;
        std::string activation = "none";            // none, relu, sigmoid, hard_tanh (limits -1 and 1)
        double      initialize_std = 0;             // of W; 0: 1 / sqrt(input nodes)
        std::uint64_t seed = 1;
    };

protected:
    create_t  m_create;
    int       m_activation = 0;
    indices_t m_input_shape;
    std::shared_ptr<Tensor_<float>> m_W  = std::make_shared<Tensor_<float>>(), m_b  = std::make_shared<Tensor_<float>>();
    std::shared_ptr<Tensor_<float>> m_dW = std::make_shared<Tensor_<float>>(), m_db = std::make_shared<Tensor_<float>>();
    Workspace m_work;

    static int ActivationByName(std::string const &name)
    {
        char const *const names[] = {"none", "relu", "sigmoid", "hard_tanh"};
        for (int i = 0; i < 4; ++i) { if (name == names[i]) { return i; } }
        throw Exception("DenseAffine: activation " + name + " is none of none, relu, sigmoid, hard_tanh");
    }

    explicit DenseAffine(create_t const &create) : m_create(create), m_activation(ActivationByName(create.activation))
    {
        m_W->Resize(0); m_b->Resize(0); m_dW->Resize(0); m_db->Resize(0);          // (no weights before SetInputShape)
    }

    void DumpObjectData(std::ostream &os) const override
    {
        SaveValue(os, (std::int64_t)1);
        Model::DumpObjectData(os);
        SaveIndices(os, m_input_shape);
        SaveIndices(os, m_create.output_shape);
        SaveValue(os, (std::int64_t)m_activation);
        m_W->DumpObject(os);
        m_b->DumpObject(os);
    }

    void LoadObjectData(std::istream &is) override
    {
        std::int64_t ver = -1, activation = -1;
        LoadValue(is, ver);
        BB_ASSERT(ver == 1);
        Model::LoadObjectData(is);
        m_input_shape = LoadIndices(is);
        m_create.output_shape = LoadIndices(is);
        LoadValue(is, activation);
        BB_ASSERT(is.good() && activation >= 0 && activation < 4);
        m_activation = (int)activation;
        m_W->LoadObject(is);
        m_b->LoadObject(is);
        index_t const in = m_input_shape.empty() ? 0 : CalcShapeSize(m_input_shape), out = CalcShapeSize(m_create.output_shape);
        BB_ASSERT(is.good() && m_W->GetSize() == in * out && m_b->GetSize() == (in ? out : 0));
        m_dW->Resize(m_W->GetShape()); m_dW->FillZero();
        m_db->Resize(m_b->GetShape()); m_db->FillZero();
    }

    void RequireDevice(FrameBuffer const &buf) const
    {
        if (!buf.IsDeviceAvailable()) { throw Exception("DenseAffine: host-only execution is not provided by this library (device path only)"); }
    }
    static int Stride(FrameBuffer const &buf) { return (int)(buf.GetFrameStride() / 4); }
    std::size_t ForwardWorkspaceSize(index_t frames) const { return bbhip_DenseAffine_Forward_WorkspaceBytes((int)GetInputNodeSize(), (int)GetOutputNodeSize(), (int)frames, kBit); }
    std::size_t WorkspaceSize(index_t frames) const { return bbhip_DenseAffine_WorkspaceBytes((int)GetInputNodeSize(), (int)GetOutputNodeSize(), (int)frames); }

public:
    static std::string ModelName(void)  { return "DenseAffine"; }
    static std::string ObjectName(void) { return ModelName() + "_" + DataType<BinType>::Name() + "_" + DataType<RealType>::Name(); }
    std::string GetModelName(void) const override  { return ModelName(); }
    std::string GetObjectName(void) const override { return ObjectName(); }

    static std::shared_ptr<DenseAffine> Create(create_t const &create)
    {
        BB_ASSERT(!create.output_shape.empty());
        return std::shared_ptr<DenseAffine>(new DenseAffine(create));
    }
    static std::shared_ptr<DenseAffine> Create(indices_t const &output_shape, std::string activation = "none", std::uint64_t seed = 1)
    {
        create_t c;
        c.output_shape = output_shape; c.activation = activation; c.seed = seed;
        return Create(c);
    }
    static std::shared_ptr<DenseAffine> Create(index_t output_node_size, std::string activation = "none", std::uint64_t seed = 1)
    {
        return Create(indices_t({output_node_size}), activation, seed);
    }

    int GetActivation(void) const { return m_activation; }
    std::shared_ptr<Tensor_<float>> W(void)  { return m_W; }
    std::shared_ptr<Tensor_<float>> b(void)  { return m_b; }
    std::shared_ptr<Tensor_<float>> dW(void) { return m_dW; }
    std::shared_ptr<Tensor_<float>> db(void) { return m_db; }
    auto lock_W(void)              { return m_W->Lock(); }
    auto lock_W_const(void) const  { return m_W->LockConst(); }
    auto lock_b(void)              { return m_b->Lock(); }
    auto lock_b_const(void) const  { return m_b->LockConst(); }
    auto lock_dW_const(void) const { return m_dW->LockConst(); }
    auto lock_db_const(void) const { return m_db->LockConst(); }

    Variables GetParameters(void) override
    {
        Variables v;
        if (!m_parameter_lock) { v.PushBack(m_W); v.PushBack(m_b); }
        return v;
    }
    Variables GetGradients(void) override
    {
        Variables v;
        if (!m_parameter_lock) { v.PushBack(m_dW); v.PushBack(m_db); }
        return v;
    }

    // a repeated shape changes nothing; a new one starts with weights of its own
    indices_t SetInputShape(indices_t shape) override
    {
        if (shape == m_input_shape) { return m_create.output_shape; }
        m_input_shape = shape;
        index_t const in = CalcShapeSize(shape), out = CalcShapeSize(m_create.output_shape);
        m_W->Resize(indices_t({out, in}));
        m_W->InitNormalDistribution(0.0, m_create.initialize_std > 0 ? m_create.initialize_std : 1.0 / std::sqrt((double)in), m_create.seed);
        m_b->Resize(out);  *m_b = 0.0f;
        m_dW->Resize(indices_t({out, in})); m_dW->FillZero();
        m_db->Resize(out); m_db->FillZero();
        return m_create.output_shape;
    }
    indices_t GetInputShape(void) const override  { return m_input_shape; }
    indices_t GetOutputShape(void) const override { return m_create.output_shape; }

    FrameBuffer Forward(FrameBuffer x_buf, bool train = true) override { return Forward(x_buf, FrameBuffer(), train); }

    // residual_buf (empty: none) has the output's nodes
    FrameBuffer Forward(FrameBuffer x_buf, FrameBuffer residual_buf, bool train)
    {
        RequireDevice(x_buf);
        BB_ASSERT(x_buf.GetType() == DataType<BinType>::type);
        if (x_buf.GetShape() != m_input_shape) { SetInputShape(x_buf.GetShape()); }
        FrameBuffer y_buf(x_buf.GetFrameSize(), m_create.output_shape, BB_TYPE_FP32);
        bool const more = !residual_buf.Empty();
        BB_ASSERT(!more || (residual_buf.GetType() == BB_TYPE_FP32 && residual_buf.GetNodeSize() == y_buf.GetNodeSize() && residual_buf.GetFrameSize() == x_buf.GetFrameSize()));
        int const in = (int)x_buf.GetNodeSize(), out = (int)y_buf.GetNodeSize(), frames = (int)x_buf.GetFrameSize();
        std::size_t const size = ForwardWorkspaceSize(frames);
        {
            auto px = x_buf.LockDeviceMemoryConst();
            auto py = y_buf.LockDeviceMemory(true);
            auto pW = m_W->LockDeviceMemoryConst();
            auto pb = m_b->LockDeviceMemoryConst();
            float const *r = more ? (float const *)residual_buf.LockDeviceMemoryConst().GetAddr() : nullptr;
            int const r_stride = more ? Stride(residual_buf) : 0;
            if (kBit) {
                CheckDevice(bbhip_bit_fp32_DenseAffine_Forward((int const *)px.GetAddr(), (float *)py.GetAddr(), (float const *)pW.GetAddr(), (float const *)pb.GetAddr(), r,
                                m_activation, in, out, frames, Stride(x_buf), Stride(y_buf), r_stride, m_work.Get(size), size, nullptr), "bbhip_bit_fp32_DenseAffine_Forward");
            }
            else {
                CheckDevice(bbhip_fp32_DenseAffine_Forward((float const *)px.GetAddr(), (float *)py.GetAddr(), (float const *)pW.GetAddr(), (float const *)pb.GetAddr(), r,
                                m_activation, in, out, frames, Stride(x_buf), Stride(y_buf), r_stride, m_work.Get(size), size, nullptr), "bbhip_fp32_DenseAffine_Forward");
            }
        }
        if (train) { PushFrameBuffer(x_buf); PushFrameBuffer(m_activation ? y_buf : FrameBuffer()); }
        return y_buf;
    }

    // the gradients of W and b accumulate until the optimizer or FillZero clears them, as those of the other layers
    FrameBuffer Backward(FrameBuffer dy_buf) override { return Backward(dy_buf, nullptr); }

    // residual_gradient: receives the gradient of the residual
    FrameBuffer Backward(FrameBuffer dy_buf, FrameBuffer *residual_gradient)
    {
        if (dy_buf.Empty()) { return FrameBuffer(); }
        RequireDevice(dy_buf);
        BB_ASSERT(dy_buf.GetType() == BB_TYPE_FP32);
        FrameBuffer y_buf = PopFrameBuffer();
        FrameBuffer x_buf = PopFrameBuffer();
        BB_ASSERT(x_buf.GetFrameSize() == dy_buf.GetFrameSize() && dy_buf.GetNodeSize() == GetOutputNodeSize());
        FrameBuffer dx_buf(dy_buf.GetFrameSize(), m_input_shape, BB_TYPE_FP32);
        if (residual_gradient) { *residual_gradient = FrameBuffer(dy_buf.GetFrameSize(), m_create.output_shape, BB_TYPE_FP32); }
        int const in = (int)x_buf.GetNodeSize(), out = (int)dy_buf.GetNodeSize(), frames = (int)dy_buf.GetFrameSize();
        std::size_t const size = WorkspaceSize(frames);
        auto px  = x_buf.LockDeviceMemoryConst();
        auto pdy = dy_buf.LockDeviceMemoryConst();
        auto pdx = dx_buf.LockDeviceMemory(true);
        auto pW  = m_W->LockDeviceMemoryConst();
        auto pdW = m_dW->LockDeviceMemory();
        auto pdb = m_db->LockDeviceMemory();
        float const *y = m_activation ? (float const *)y_buf.LockDeviceMemoryConst().GetAddr() : nullptr;
        float *dr = residual_gradient ? (float *)residual_gradient->LockDeviceMemory(true).GetAddr() : nullptr;
        if (kBit) {
            CheckDevice(bbhip_bit_fp32_DenseAffine_Backward((int const *)px.GetAddr(), (float const *)pdy.GetAddr(), y, (float const *)pW.GetAddr(), (float *)pdx.GetAddr(),
                            (float *)pdW.GetAddr(), (float *)pdb.GetAddr(), dr, m_activation, 1, in, out, frames, Stride(x_buf), Stride(dx_buf), Stride(dy_buf), m_work.Get(size),
                            size, nullptr), "bbhip_bit_fp32_DenseAffine_Backward");
        }
        else {
            CheckDevice(bbhip_fp32_DenseAffine_Backward((float const *)px.GetAddr(), (float const *)pdy.GetAddr(), y, (float const *)pW.GetAddr(), (float *)pdx.GetAddr(),
                            (float *)pdW.GetAddr(), (float *)pdb.GetAddr(), dr, m_activation, 1, in, out, frames, Stride(x_buf), Stride(dx_buf), Stride(dy_buf), m_work.Get(size),
                            size, nullptr), "bbhip_fp32_DenseAffine_Backward");
        }
        return dx_buf;
    }

    std::vector<double> ForwardNode(index_t node, std::vector<double> x) const override
    {
        index_t const in = GetInputNodeSize();
        BB_ASSERT((index_t)x.size() == in && node >= 0 && node < GetOutputNodeSize());
        auto W = m_W->LockConst();
        auto b = m_b->LockConst();
        double z = b[node];
        for (index_t i = 0; i < in; ++i) { z += (double)W[node * in + i] * x[(std::size_t)i]; }
        if (m_activation == 1) { z = z <= 0 ? 0 : z; }
        if (m_activation == 2) { z = 1.0 / (1.0 + std::exp(-z)); }
        if (m_activation == 3) { z = z <= -1 ? -1 : z >= 1 ? 1 : z; }
        return {z};
    }
};

}  // namespace bb

// The softmax cross entropy on top of a dense layer, in pieces of its channels: at most 64 Mi logits (or those of 256 channels) are held at a time.  CalculateLoss takes the layer's INPUT and the
// labels, adds to the layer's gradients and returns the input's; accumulated over batches like the other losses.  (The reference has no such loss: there the layer's
// output goes through LossSoftmaxCrossEntropy.)
#pragma once

#include "bb/DenseAffine.h"
#include "bb/LossSoftmaxCrossEntropy.h"

namespace bb {

template <typename BinType = float>
class LossDenseSoftmaxCrossEntropy : public LossFunction {
    static constexpr bool kBit = std::is_same<BinType, Bit>::value;

    std::shared_ptr<DenseAffine<BinType, float>> m_layer;
    Workspace m_work;
    double    m_loss = 0, m_weight = 0;

    explicit LossDenseSoftmaxCrossEntropy(std::shared_ptr<DenseAffine<BinType, float>> layer) : m_layer(layer)
    {
        if (!layer || layer->GetActivation() != 0) { throw Exception("LossDenseSoftmaxCrossEntropy: a dense layer without an activation is needed"); }
    }

public:
    static std::string LossFunctionName(void) { return "LossDenseSoftmaxCrossEntropy"; }
    std::string GetLossFunctionName(void) const override { return LossFunctionName(); }

    static std::shared_ptr<LossDenseSoftmaxCrossEntropy> Create(std::shared_ptr<DenseAffine<BinType, float>> layer)
    {
        return std::shared_ptr<LossDenseSoftmaxCrossEntropy>(new LossDenseSoftmaxCrossEntropy(layer));
    }

    void   Clear(void) override { m_loss = 0; m_weight = 0; }
    double GetLoss(void) const override { return m_weight == 0 ? 0 : m_loss / m_weight; }

    // label_buf: one int32 node; a negative label, or no channel of the layer: the frame does not count
    FrameBuffer CalculateLoss(FrameBuffer x_buf, FrameBuffer label_buf, index_t) override { return CalculateLoss(x_buf, label_buf, FrameBuffer(), true); }

    // weight_buf: of every frame (empty: 1); without gradients an empty buffer is returned
    FrameBuffer CalculateLoss(FrameBuffer x_buf, FrameBuffer label_buf, FrameBuffer weight_buf, bool gradients)
    {
        BB_ASSERT(x_buf.GetType() == DataType<BinType>::type && label_buf.GetType() == BB_TYPE_INT32);
        if (!Manager::IsDeviceAvailable()) { throw Exception("LossDenseSoftmaxCrossEntropy: host-only execution is not provided by this library (device path only)"); }
        if (x_buf.GetShape() != m_layer->GetInputShape()) { m_layer->SetInputShape(x_buf.GetShape()); }
        index_t const frame_size = x_buf.GetFrameSize(), ch_size = m_layer->GetOutputNodeSize();
        bool const weighted = !weight_buf.Empty();
        BB_ASSERT(label_buf.GetNodeSize() == 1 && label_buf.GetFrameSize() == frame_size);
        BB_ASSERT(!weighted || (weight_buf.GetType() == BB_TYPE_FP32 && weight_buf.GetNodeSize() == 1 && weight_buf.GetFrameSize() == frame_size));
        double weight_sum = 0;
        {
            auto label = label_buf.LockConst<std::int32_t>();
            for (index_t f = 0; f < frame_size; ++f) {
                std::int32_t const t = label.Get(f, 0);
                if (t >= 0 && t < ch_size) { weight_sum += weighted ? (double)weight_buf.LockConst<float>().Get(f, 0) : 1.0; }
            }
        }
        FrameBuffer loss_buf(frame_size, indices_t({1}), BB_TYPE_FP32), dx_buf;
        if (gradients) { dx_buf = FrameBuffer(frame_size, x_buf.GetShape(), BB_TYPE_FP32); }
        int const in = (int)x_buf.GetNodeSize();
        std::size_t const size = bbhip_LossDenseSoftmaxCrossEntropy_WorkspaceBytes(in, (int)ch_size, (int)frame_size, gradients);
        {
            auto px    = x_buf.LockDeviceMemoryConst();
            auto pW    = m_layer->W()->LockDeviceMemoryConst();
            auto pb    = m_layer->b()->LockDeviceMemoryConst();
            auto label = label_buf.LockDeviceMemoryConst();
            auto loss  = loss_buf.LockDeviceMemory(true);
            float const *weight = weighted ? (float const *)weight_buf.LockDeviceMemoryConst().GetAddr() : nullptr;
            float *dx = gradients ? (float *)dx_buf.LockDeviceMemory(true).GetAddr() : nullptr;
            float *dW = gradients ? (float *)m_layer->dW()->LockDeviceMemory().GetAddr() : nullptr;
            float *db = gradients ? (float *)m_layer->db()->LockDeviceMemory().GetAddr() : nullptr;
            int const x_stride = (int)(x_buf.GetFrameStride() / 4), dx_stride = gradients ? (int)(dx_buf.GetFrameStride() / 4) : 0;
            if (kBit) {
                CheckDevice(bbhip_bit_fp32_LossDenseSoftmaxCrossEntropy((int const *)px.GetAddr(), (float const *)pW.GetAddr(), (float const *)pb.GetAddr(),
                                (int const *)label.GetAddr(), weight, dx, dW, db, (float *)loss.GetAddr(), (float)weight_sum, 1, in, (int)ch_size, (int)frame_size, x_stride,
                                dx_stride, m_work.Get(size), size, nullptr), "bbhip_bit_fp32_LossDenseSoftmaxCrossEntropy");
            }
            else {
                CheckDevice(bbhip_fp32_LossDenseSoftmaxCrossEntropy((float const *)px.GetAddr(), (float const *)pW.GetAddr(), (float const *)pb.GetAddr(),
                                (int const *)label.GetAddr(), weight, dx, dW, db, (float *)loss.GetAddr(), (float)weight_sum, 1, in, (int)ch_size, (int)frame_size, x_stride,
                                dx_stride, m_work.Get(size), size, nullptr), "bbhip_fp32_LossDenseSoftmaxCrossEntropy");
            }
        }
        m_loss += loss_buf.Sum();
        m_weight += weight_sum;
        return dx_buf;
    }
};

}  // namespace bb

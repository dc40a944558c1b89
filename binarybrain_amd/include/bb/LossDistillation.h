// Distillation from a teacher's largest logits, accumulated over batches like the other losses: dy of CalculateLoss is the gradient of
//   sum over places of w T^2 KL(softmax(teacher / T) over its kept logits || softmax(y / T)) / sum of w,
// GetLoss the same quotient over all batches since Clear.  Nodes are [ch][pix].  (The reference has no such loss.)
#pragma once

#include "bb/LossSoftmaxCrossEntropy.h"
#include "bb/TopLogits.h"

namespace bb {

template <typename T = float>
class LossDistillation : public LossFunction {
    static_assert(std::is_same<T, float>::value, "the device path is fp32");

public:
    struct create_t {
        float   temperature = 1.0f;
        index_t top_size    = 64;           // of a teacher's logits that are given whole: kept are so many (all of fewer channels)
    };

protected:
    create_t  m_create;
    TopLogits m_top;
    Workspace m_work;
    double    m_loss = 0, m_weight = 0;

    explicit LossDistillation(create_t const &create) : m_create(create) {}

public:
    static std::string LossFunctionName(void) { return "LossDistillation"; }
    std::string GetLossFunctionName(void) const override { return LossFunctionName(); }

    static std::shared_ptr<LossDistillation> Create(create_t const &create) { return std::shared_ptr<LossDistillation>(new LossDistillation(create)); }
    static std::shared_ptr<LossDistillation> Create(float temperature = 1.0f, index_t top_size = 64)
    {
        create_t c;
        c.temperature = temperature; c.top_size = top_size;
        return Create(c);
    }

    void   Clear(void) override { m_loss = 0; m_weight = 0; }
    double GetLoss(void) const override { return m_weight == 0 ? 0 : m_loss / m_weight; }

    // t_buf: the teacher's logits, of the shape of y_buf
    FrameBuffer CalculateLoss(FrameBuffer y_buf, FrameBuffer t_buf, index_t) override
    {
        BB_ASSERT(y_buf.GetNodeSize() == t_buf.GetNodeSize() && y_buf.GetFrameSize() == t_buf.GetFrameSize() && y_buf.GetShape()[0] == t_buf.GetShape()[0]);
        index_t const ch_size = y_buf.GetShape()[0];
        TopLogits::list_t const list = m_top.Calculate(t_buf, m_create.top_size < ch_size ? m_create.top_size : ch_size);
        return CalculateLoss(y_buf, list, FrameBuffer());
    }

    // a teacher's kept logits, and the weight of every pixel and frame (an empty buffer: 1)
    FrameBuffer CalculateLoss(FrameBuffer y_buf, TopLogits::list_t const &list, FrameBuffer weight_buf)
    {
        BB_ASSERT(y_buf.GetType() == BB_TYPE_FP32 && list.index.GetType() == BB_TYPE_INT32 && list.logit.GetType() == BB_TYPE_FP32);
        if (!Manager::IsDeviceAvailable()) { throw Exception("LossDistillation: host-only execution is not provided by this library (device path only)"); }
        index_t const ch_size = y_buf.GetShape()[0], pix_size = y_buf.GetNodeSize() / ch_size, frame_size = y_buf.GetFrameSize(), top_size = list.index.GetNodeSize() / pix_size;
        BB_ASSERT(top_size * pix_size == list.index.GetNodeSize() && list.logit.GetNodeSize() == list.index.GetNodeSize());
        BB_ASSERT(list.index.GetFrameSize() == frame_size && list.logit.GetFrameSize() == frame_size);
        bool const weighted = !weight_buf.Empty();
        BB_ASSERT(!weighted || (weight_buf.GetType() == BB_TYPE_FP32 && weight_buf.GetNodeSize() == pix_size && weight_buf.GetFrameSize() == frame_size));
        double const weight_sum = weighted ? weight_buf.Sum() : (double)(pix_size * frame_size);
        FrameBuffer dy_buf(frame_size, y_buf.GetShape(), BB_TYPE_FP32), loss_buf(frame_size, PixelShape(y_buf.GetShape(), 0), BB_TYPE_FP32);
        std::size_t const size = bbhip_LossDistillation_WorkspaceBytes((int)pix_size, (int)ch_size, (int)frame_size);
        {
            auto y_ptr     = y_buf.LockDeviceMemoryConst();
            auto index_ptr = list.index.LockDeviceMemoryConst();
            auto logit_ptr = list.logit.LockDeviceMemoryConst();
            auto dy_ptr    = dy_buf.LockDeviceMemory(true);
            auto loss_ptr  = loss_buf.LockDeviceMemory(true);
            float const *weight = weighted ? (float const *)weight_buf.LockDeviceMemoryConst().GetAddr() : nullptr;
            CheckDevice(bbhip_fp32_LossDistillation((float const *)y_ptr.GetAddr(), (int const *)index_ptr.GetAddr(), (float const *)logit_ptr.GetAddr(), weight,
                            (float *)dy_ptr.GetAddr(), (float *)loss_ptr.GetAddr(), m_create.temperature, (float)weight_sum, (int)top_size, (int)pix_size, (int)ch_size,
                            (int)frame_size, (int)(y_buf.GetFrameStride() / 4), (int)(list.index.GetFrameStride() / 4), m_work.Get(size), size, nullptr),
                        "bbhip_fp32_LossDistillation");
        }
        m_loss += loss_buf.Sum();
        m_weight += weight_sum;
        return dy_buf;
    }
};

}  // namespace bb

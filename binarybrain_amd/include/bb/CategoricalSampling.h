// A category of every pixel and frame drawn from a network's logits by given random numbers: temperature, the largest logits (top_size), the shortest prefix of
// them that holds top_p of their probability, of it those of at least min_p times the largest.  Nodes are [ch][pix].  (The reference has no such operation.)
#pragma once

#include "bb/TopLogits.h"

namespace bb {

class CategoricalSampling {
public:
    struct create_t {
        float   temperature = 1.0f;
        index_t top_size    = 50;           // 1: the largest logit; of fewer channels all
        float   top_p       = 1.0f;
        float   min_p       = 0.0f;
    };

protected:
    create_t  m_create;
    Workspace m_work;
    explicit CategoricalSampling(create_t const &create) : m_create(create) {}

public:
    static std::shared_ptr<CategoricalSampling> Create(create_t const &create) { return std::shared_ptr<CategoricalSampling>(new CategoricalSampling(create)); }
    static std::shared_ptr<CategoricalSampling> Create(void) { return Create(create_t()); }

    // u_buf: numbers in [0, 1), one for every pixel and frame.  int32 channels (-1 where nothing can be drawn); share: their probability among the kept
    FrameBuffer Sample(FrameBuffer y_buf, FrameBuffer u_buf, FrameBuffer *share = nullptr)
    {
        BB_ASSERT(y_buf.GetType() == BB_TYPE_FP32 && u_buf.GetType() == BB_TYPE_FP32);
        if (!y_buf.IsDeviceAvailable()) { throw Exception("CategoricalSampling: host-only execution is not provided by this library (device path only)"); }
        index_t const ch_size = y_buf.GetShape()[0], pix_size = y_buf.GetNodeSize() / ch_size, frame_size = y_buf.GetFrameSize();
        BB_ASSERT(u_buf.GetNodeSize() == pix_size && u_buf.GetFrameSize() == frame_size);
        int const top_size = (int)(m_create.top_size < ch_size ? m_create.top_size : ch_size);
        FrameBuffer category_buf(frame_size, PixelShape(y_buf.GetShape(), 0), BB_TYPE_INT32);
        if (share) { *share = FrameBuffer(frame_size, PixelShape(y_buf.GetShape(), 0), BB_TYPE_FP32); }
        std::size_t const size = bbhip_TopLogits_WorkspaceBytes(top_size, (int)pix_size, (int)ch_size, (int)frame_size);
        auto y_ptr = y_buf.LockDeviceMemoryConst();
        auto u_ptr = u_buf.LockDeviceMemoryConst();
        auto c_ptr = category_buf.LockDeviceMemory(true);
        float *s = share ? (float *)share->LockDeviceMemory(true).GetAddr() : nullptr;
        CheckDevice(bbhip_fp32_CategoricalSampling((float const *)y_ptr.GetAddr(), (float const *)u_ptr.GetAddr(), (int *)c_ptr.GetAddr(), s, m_create.temperature, top_size,
                        m_create.top_p, m_create.min_p, (int)pix_size, (int)ch_size, (int)frame_size, (int)(y_buf.GetFrameStride() / 4), m_work.Get(size), size, nullptr),
                    "bbhip_fp32_CategoricalSampling");
        return category_buf;
    }
};

}  // namespace bb

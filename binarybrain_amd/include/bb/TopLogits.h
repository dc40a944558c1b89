// The largest logits of every pixel and frame: what a teacher keeps of its output for LossDistillation.  Nodes are [ch][pix], the channel index first in the shape.
// (The reference has no such operation.)
#pragma once

#include "bb/FrameBuffer.h"
#include "bb/Workspace.h"

namespace bb {

// the shape of what has `channels` entries for every pixel of `shape` (0: one value, the channel index falls away)
inline indices_t PixelShape(indices_t shape, index_t channels)
{
    BB_ASSERT(!shape.empty());
    if (channels > 0) { shape[0] = channels; return shape; }
    shape.erase(shape.begin());
    return shape.empty() ? indices_t({1}) : shape;
}

class TopLogits {
    Workspace m_work;

public:
    struct list_t {
        FrameBuffer index;          // int32 channels, [top][pix] nodes
        FrameBuffer logit;          // their logits, descending
    };

    list_t Calculate(FrameBuffer y_buf, index_t top_size)
    {
        BB_ASSERT(y_buf.GetType() == BB_TYPE_FP32);
        if (!y_buf.IsDeviceAvailable()) { throw Exception("TopLogits: host-only execution is not provided by this library (device path only)"); }
        index_t const ch_size = y_buf.GetShape()[0], pix_size = y_buf.GetNodeSize() / ch_size, frame_size = y_buf.GetFrameSize();
        list_t list{FrameBuffer(frame_size, PixelShape(y_buf.GetShape(), top_size), BB_TYPE_INT32), FrameBuffer(frame_size, PixelShape(y_buf.GetShape(), top_size), BB_TYPE_FP32)};
        BB_ASSERT(list.index.GetFrameStride() == list.logit.GetFrameStride());
        std::size_t const size = bbhip_TopLogits_WorkspaceBytes((int)top_size, (int)pix_size, (int)ch_size, (int)frame_size);
        auto y_ptr     = y_buf.LockDeviceMemoryConst();
        auto index_ptr = list.index.LockDeviceMemory(true);
        auto logit_ptr = list.logit.LockDeviceMemory(true);
        CheckDevice(bbhip_fp32_TopLogits((float const *)y_ptr.GetAddr(), (int *)index_ptr.GetAddr(), (float *)logit_ptr.GetAddr(), (int)top_size, (int)pix_size, (int)ch_size,
                        (int)frame_size, (int)(y_buf.GetFrameStride() / 4), (int)(list.index.GetFrameStride() / 4), m_work.Get(size), size, nullptr), "bbhip_fp32_TopLogits");
        return list;
    }
};

}  // namespace bb

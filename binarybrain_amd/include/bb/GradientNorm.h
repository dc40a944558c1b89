// The norm of a list of gradients as if they were one vector, and the list scaled to a norm.  (The reference has neither.)
#pragma once

#include "bb/Core.h"
#include "bb/Tensor.h"
#include "bb/Workspace.h"

namespace bb {

class GradientNorm {
    Variables m_grads;
    std::shared_ptr<Memory> m_size_table, m_grad_table, m_norm;
    Workspace m_work;

    void Apply(bool clip, float max_norm)
    {
        if (!Manager::IsDeviceAvailable()) { throw Exception("GradientNorm: no device available (there is no host path)"); }
        index_t const n = m_grads.GetSize();
        for (index_t i = 0; i < n; ++i) { if (clip) { m_grads[i].LockDeviceMemory(); } else { m_grads[i].LockDeviceMemoryConst(); } }
        auto const entry = clip ? bbhip_fp32_GradientClip : bbhip_fp32_GradientNorm;
        std::size_t const size = bbhip_GradientNorm_WorkspaceBytes();
        CheckDevice(entry((int)n, n ? (int const *)m_size_table->LockDeviceConst() : nullptr, n ? (float *const *)m_grad_table->LockDeviceConst() : nullptr, max_norm,
                          (float *)m_norm->LockDevice(true), m_work.Get(size), size, nullptr), clip ? "bbhip_fp32_GradientClip" : "bbhip_fp32_GradientNorm");
    }

public:
    // The tensors must keep their storage (no Resize) while they are bound.  One that is in the list twice is refused: it would be counted and scaled twice, by two workgroups at once.
    explicit GradientNorm(Variables grads) : m_grads(grads), m_norm(Memory::Create(2 * sizeof(float)))
    {
        if (grads.HasOneTwice()) { throw Exception("GradientNorm: a tensor is in the list twice"); }
        index_t const n = grads.GetSize();
        std::vector<std::int32_t> sizes;
        std::vector<void *> addresses;
        for (index_t i = 0; i < n; ++i) {
            BB_ASSERT(grads[i].GetType() == BB_TYPE_FP32 && grads[i].GetSize() <= 0x7fffffff);
            if (!grads[i].IsDeviceAvailable()) { throw Exception("GradientNorm: no device path for host-only tensors"); }
            sizes.push_back((std::int32_t)grads[i].GetSize());
            addresses.push_back(grads[i].LockDeviceMemory().GetAddr());
        }
        if (n == 0) { return; }
        m_size_table = Memory::Create(sizes.size() * sizeof(std::int32_t));
        std::memcpy(m_size_table->Lock(true), sizes.data(), sizes.size() * sizeof(std::int32_t));
        m_grad_table = Memory::Create(addresses.size() * sizeof(void *));
        std::memcpy(m_grad_table->Lock(true), addresses.data(), addresses.size() * sizeof(void *));
    }

    // the norm of the gradients as they are
    double Calculate(void) { Apply(false, INFINITY); return ((float const *)m_norm->LockConst())[0]; }
    // scales them to max_norm where theirs is larger; returns what it was
    double Clip(double max_norm) { Apply(true, (float)max_norm); return ((float const *)m_norm->LockConst())[0]; }
};

}  // namespace bb

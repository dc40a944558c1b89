// Device scratch that an operator's object keeps for its calls: grown when a call needs more, never cleared, never read between calls.
#pragma once

#include "bb/Core.h"

namespace bb {

class Workspace {
    std::shared_ptr<Memory> m_mem;
public:
    // `size` bytes on the device (nullptr for 0), the same place as long as it suffices
    void *Get(std::size_t size)
    {
        if (size == 0) { return nullptr; }
        if (!m_mem || m_mem->GetSize() < size) { m_mem = Memory::Create(size); }
        return m_mem->LockDevice(true);
    }
};

}  // namespace bb

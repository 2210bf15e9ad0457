// Host side of the attention kernels' launches.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>

namespace w34 {

// One attribute call per kernel instantiation and device.  The record is process-wide and
// lock-free: slot i belongs to the first kernel that claims it, bit d of its mask says that
// device d is configured.  Kernels that address their dequantisation table absolutely
// (lds_base_zero) also have their static LDS size checked here: it must be zero, so that the
// dynamic block starts at LDS address 0.
constexpr int kLdsRecordSlots = 128;
static std::atomic<const void*> g_lds_fn[kLdsRecordSlots];
static std::atomic<unsigned long long> g_lds_devs[kLdsRecordSlots];

template <typename KernelT>
static int ensure_dynamic_lds(KernelT kernel, int bytes, bool lds_base_zero = false) {
    int dev = 0;
    hipError_t rc = hipGetDevice(&dev);
    if (rc != hipSuccess) return (int)rc;
    const void* fn = (const void*)kernel;
    int slot = -1;
    for (int i = 0; i < kLdsRecordSlots; ++i) {
        const void* cur = g_lds_fn[i].load(std::memory_order_acquire);
        if (cur == nullptr) {
            const void* expect = nullptr;
            if (g_lds_fn[i].compare_exchange_strong(expect, fn, std::memory_order_acq_rel)) cur = fn;
            else cur = expect;
        }
        if (cur == fn) {
            slot = i;
            break;
        }
    }
    const bool tracked = slot >= 0 && dev >= 0 && dev < 64;
    if (tracked && ((g_lds_devs[slot].load(std::memory_order_acquire) >> dev) & 1ull)) return 0;
    if (lds_base_zero) {
        hipFuncAttributes attr;
        rc = hipFuncGetAttributes(&attr, fn);
        if (rc != hipSuccess) return (int)rc;
        if (attr.sharedSizeBytes != 0) return (int)hipErrorInvalidConfiguration;
    }
    rc = hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (rc != hipSuccess) return (int)rc;
    if (tracked) g_lds_devs[slot].fetch_or(1ull << dev, std::memory_order_release);
    return 0;
}

// Whether a launch of so many workgroups side by side is one: a grid has less than 2^32 threads along each axis.
inline bool grid_fits(long long workgroups, int threads) { return workgroups < (1ll << 32) / threads; }

// ceil(2^16 / q_group), for the division of a workgroup's column by the q heads of its tile
inline uint32_t q_group_magic_for(int q_group) { return (65536u + (uint32_t)q_group - 1u) / (uint32_t)q_group; }

}  // namespace w34

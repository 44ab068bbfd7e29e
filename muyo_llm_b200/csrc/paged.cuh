// Shared by the paged-cache entry points: the checked device view of MuyoPagedCache.
#pragma once

#include <atomic>
#include <climits>
#include <cmath>

#include <cuda_fp8.h>

#include "common.cuh"

namespace muyo {

struct PagedDev {
    int heads, kv_heads, group, head_dim, page_size, num_pages;
    float k_scale, v_scale;
    long long page_stride, head_stride, slot_stride;  // elements
};

inline int kv_bytes(uint32_t kv_dtype) { return kv_dtype == MUYO_KV_F32 ? 4 : kv_dtype == MUYO_KV_F16 ? 2 : 1; }

// Validates a cache description (no CUDA call) and resolves its defaults.
inline int paged_prepare(const MuyoPagedCache& c, const char* what, PagedDev& d)
{
    MUYO_REQUIRE(c.heads > 0 && c.kv_heads > 0 && c.heads % c.kv_heads == 0,
                 "%s: heads %u must be a positive multiple of kv_heads %u", what, c.heads, c.kv_heads);
    MUYO_REQUIRE(c.heads / c.kv_heads <= 16, "%s: more than 16 query heads per KV head", what);
    MUYO_REQUIRE(c.heads <= 65535, "%s: %u heads exceed 65535", what, c.heads);
    if (!(c.head_dim == 16 || c.head_dim == 32 || c.head_dim == 64 || c.head_dim == 128)) {
        set_error("%s: head_dim %u not supported (16, 32, 64, 128)", what, c.head_dim);
        return MUYO_EUNSUPPORTED;
    }
    MUYO_REQUIRE(c.kv_dtype == MUYO_KV_F32 || c.kv_dtype == MUYO_KV_F16 || c.kv_dtype == MUYO_KV_F8, "%s: kv_dtype %u", what,
                 c.kv_dtype);
    MUYO_REQUIRE(c.page_size > 0 && c.num_pages > 0, "%s: page_size and num_pages must be positive", what);
    MUYO_REQUIRE((uint64_t)c.page_size * c.num_pages <= (uint64_t)INT_MAX, "%s: %u pages of %u slots exceed INT32_MAX slots",
                 what, c.num_pages, c.page_size);
    const auto fits = [](float s) { return s == 0.0f || (s >= 0x1p-100f && s <= 0x1p100f); };
    MUYO_REQUIRE(fits(c.k_scale) && fits(c.v_scale), "%s: k_scale and v_scale must be 0 or in [2^-100, 2^100]", what);
    d.heads = (int)c.heads, d.kv_heads = (int)c.kv_heads, d.group = (int)(c.heads / c.kv_heads);
    d.head_dim = (int)c.head_dim, d.page_size = (int)c.page_size, d.num_pages = (int)c.num_pages;
    d.k_scale = c.k_scale == 0.0f ? 1.0f : c.k_scale;
    d.v_scale = c.v_scale == 0.0f ? 1.0f : c.v_scale;
    const bool packed = c.page_stride == 0 && c.head_stride == 0 && c.slot_stride == 0;
    const uint64_t hd = c.head_dim;
    const uint64_t ps = packed ? hd * c.page_size * c.kv_heads : c.page_stride;
    const uint64_t hs = packed ? hd * c.page_size : c.head_stride;
    const uint64_t ss = packed ? hd : c.slot_stride;
    MUYO_REQUIRE(ps >= hd && hs >= hd && ss >= hd, "%s: strides %llu, %llu, %llu (page, head, slot) are below head_dim", what,
                 (unsigned long long)ps, (unsigned long long)hs, (unsigned long long)ss);
    const uint64_t unit = 16 / kv_bytes(c.kv_dtype);
    MUYO_REQUIRE(ps % unit == 0 && hs % unit == 0 && ss % unit == 0, "%s: strides must be multiples of 16 bytes", what);
    const uint64_t most = (uint64_t)1 << 46;  // far beyond device memory; keeps every offset in 63 bits
    MUYO_REQUIRE(ps <= most / c.num_pages && hs <= most / c.kv_heads && ss <= most / c.page_size, "%s: strides too large",
                 what);
    d.page_stride = (long long)ps, d.head_stride = (long long)hs, d.slot_stride = (long long)ss;
    return MUYO_OK;
}

// Lets `kernel` use `bytes` of dynamic shared memory on the current device. The setting stays with the function, so it
// is made once per device (`done`: a bit each); the call costs the host as much as a fifth of a launch.
template <typename Kernel>
inline cudaError_t allow_smem(Kernel kernel, size_t bytes, std::atomic<unsigned long long>& done)
{
    int device = 0;
    const cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess)
        return e;
    const unsigned long long bit = device < 64 ? 1ull << device : 0ull;
    if (done.load(std::memory_order_acquire) & bit)
        return cudaSuccess;
    const cudaError_t r = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (r == cudaSuccess)
        done.fetch_or(bit, std::memory_order_release);
    return r;
}

// log2 of a power of two, or -1.
inline int page_shift_of(int page_size)
{
    for (int s = 0; s < 31; ++s)
        if (page_size == 1 << s)
            return s;
    return -1;
}

inline bool aligned_to(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

}  // namespace muyo

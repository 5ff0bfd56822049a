// Host side of the delta rule's launches: the build of a kernel for a window's sizes.
#pragma once
#include <hip/hip_runtime.h>

#include <type_traits>

#include "../../../include/inet_policy.h"

namespace pol {

constexpr size_t LDS_MAX = 160 * 1024;

// a workgroup above 64 KiB of LDS has to be allowed it, once a kernel and device
inline bool allow_lds(const void* kernel, size_t bytes) {
    return bytes > 64 * 1024 &&
           hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess;
}

template <typename V> struct Type { typedef V type; };
template <int V> using Int = std::integral_constant<int, V>;

// (more planes fill the LDS with fewer steps: 32-bit values and large float16 heads go by chunks of 32 alone)
template <typename F, typename T> int delta_dispatch_t(const InetDelta& d, T t, F&& f) {
    constexpr bool F32 = std::is_same<typename T::type, float>::value;
    constexpr bool B16 = std::is_same<typename T::type, __bf16>::value;
    if (d.chunk == 32)
        return d.K <= 32 ? f(t, Int<32>{}, Int<32>{}) : d.K <= 64 ? f(t, Int<32>{}, Int<64>{})
                                                                  : f(t, Int<32>{}, Int<128>{});
    if constexpr (!F32) {
        if (d.K <= 32) return f(t, Int<64>{}, Int<32>{});
        if (d.K <= 64) return f(t, Int<64>{}, Int<64>{});
    }
    if constexpr (B16) return f(t, Int<64>{}, Int<128>{});
    return INET_POLICY_EINVAL;
}

// f(type, chunk, padded key size) for a window's sizes
template <typename F> int delta_dispatch(const InetDelta& d, F&& f) {
    if (d.dtype == INET_POLICY_F32) return delta_dispatch_t(d, Type<float>{}, f);
    if (d.dtype == INET_POLICY_BF16) return delta_dispatch_t(d, Type<__bf16>{}, f);
    return delta_dispatch_t(d, Type<_Float16>{}, f);
}

// vec: all rows start on 16 bytes and hold whole groups of eight
int delta_forward(const InetDelta& d, bool vec, hipStream_t st);
int delta_backward(const InetDelta& d, const InetDeltaGrad& g, bool vec, hipStream_t st);
int delta_step(const InetDelta& d, hipStream_t st);
// the long-window forms (delta_split.hip), taken where d.work is given
int delta_split(const InetDelta& d, const InetDeltaGrad* g, bool vec, hipStream_t st);
size_t delta_split_bytes(const InetDelta& d, bool back);

}  // namespace pol

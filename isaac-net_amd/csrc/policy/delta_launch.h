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

template <typename T, typename F> int delta_dispatch_keys(const InetDelta& d, F&& f) {
    constexpr Type<T> t{};
    if constexpr (std::is_same<T, __bf16>::value)
        if (d.chunk == 64)
            return d.K <= 32 ? f(t, Int<64>{}, Int<32>{}) : d.K <= 64 ? f(t, Int<64>{}, Int<64>{})
                                                                      : f(t, Int<64>{}, Int<128>{});
    if (d.chunk != 32) return INET_POLICY_EINVAL;
    return d.K <= 32 ? f(t, Int<32>{}, Int<32>{}) : d.K <= 64 ? f(t, Int<32>{}, Int<64>{})
                                                              : f(t, Int<32>{}, Int<128>{});
}

// f(type, chunk, padded key size) for a window's sizes
template <typename F> int delta_dispatch(const InetDelta& d, F&& f) {
    if (d.dtype == INET_POLICY_F32) return delta_dispatch_keys<float>(d, f);
    if (d.dtype == INET_POLICY_BF16) return delta_dispatch_keys<__bf16>(d, f);
    return delta_dispatch_keys<_Float16>(d, f);
}

// vec: all rows start on 16 bytes and hold whole groups of eight
int delta_forward(const InetDelta& d, bool vec, hipStream_t st);
int delta_backward(const InetDelta& d, const InetDeltaGrad& g, bool vec, hipStream_t st);
int delta_step(const InetDelta& d, hipStream_t st);
// the long-window forms (delta_split.hip), taken where d.work is given
int delta_split(const InetDelta& d, const InetDeltaGrad* g, bool vec, hipStream_t st);
size_t delta_split_bytes(const InetDelta& d, bool back);

}  // namespace pol

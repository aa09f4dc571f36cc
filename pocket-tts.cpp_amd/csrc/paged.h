// Launch interface of the paged-cache kernels (paged_plan.hip, paged_rotary.hip, paged_attention.hip).  The argument structures
// are the public ones of pocket_tts_amd.h.  The check_ functions read the structure alone, need no GPU and throw
// std::runtime_error; the launches take what has passed them, with the device current.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "pocket_tts/pocket_tts_amd.h"

namespace ptts {

void check_paged_plan(const PttsPagedPlan& p);
void check_rotary_append(const PttsRotaryAppend& p);
void check_paged_attention(const PttsPagedAttention& p);
void launch_paged_plan(const PttsPagedPlan& p, hipStream_t s);
void launch_rotary_append(const PttsRotaryAppend& a, hipStream_t s);
long long paged_attention_workspace(const PttsPagedAttention& a, int cus);
void launch_paged_attention(const PttsPagedAttention& a, int cus, hipStream_t s);

// One launch, its own error thrown.  The thread's last error is not asked: it may come from any earlier call of the program (a poll of a
// stream that is not ready sets it), and is left as it was.
template <typename A> void launch_paged(void (*kernel)(A), dim3 grid, hipStream_t s, A a) {
    void* args[] = {&a};
    const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(256), args, 0, s);
    if (e != hipSuccess) {
        (void)hipGetLastError();          // this one has been reported
        throw std::runtime_error(std::string("kernel launch failed: ") + hipGetErrorString(e));
    }
}

// The part of the checks that two of them share.
void check_pages(const PttsPages& p, const char* who);

constexpr int kStatusPage = 1, kStatusRows = 2, kStatusLength = 4;

// Whether all of these addresses (null ones too) are multiples of n.
inline bool aligned(std::initializer_list<const void*> ptrs, unsigned n) {
    uintptr_t low = 0;
    for (const void* p : ptrs) low |= reinterpret_cast<uintptr_t>(p);
    return low % n == 0;
}

inline int type_size(int t) { return t == PTTS_TYPE_F32 ? 4 : 2; }

// Quotients of non-negative 31-bit numbers by a number fixed at launch: q = n * m >> s with s = 31 + ceil(log2 d) and
// m = floor(2^s / d) + 1 < 2^32 (n * (m - 2^s / d) / 2^s < 2^31 / 2^s <= 1 / d, so the quotient is exact).
struct FastDiv {
    unsigned m, s, d;
    static FastDiv of(unsigned d) {
        unsigned l = 0;
        while ((1ull << l) < d) ++l;
        return FastDiv{static_cast<unsigned>((1ull << (31 + l)) / d + 1), 31 + l, d};
    }
    __device__ __forceinline__ unsigned div(unsigned n) const { return static_cast<unsigned>((static_cast<unsigned long long>(n) * m) >> s); }
};

}  // namespace ptts

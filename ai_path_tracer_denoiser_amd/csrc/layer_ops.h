// layer_ops.h -- what the layer operators (linear.hip, block_norm.hip, adamw.hip) share: element types, argument checks, launches.
#pragma once
#include "internal.h"

#include <algorithm>
#include <initializer_list>
#include <type_traits>

namespace aipt {

using bf16 = __bf16;
using f16 = _Float16;

inline int type_bytes(int type) { return type == AIPT_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == AIPT_TYPE_F32 || type == AIPT_TYPE_BF16 || type == AIPT_TYPE_F16; }

// behind an entry's checks of its arguments, which need no GPU and so come first: what they refuse a host without one is told too
// (aipt_last_error(NULL))
#define AIPT_NEED_CTX(ctx) \
    do { if (!(ctx)) return aipt::fail(nullptr, AIPT_E_INVALID, "%s: ctx is NULL", __func__); } while (0)

// 16 bytes of elements: the unit every aligned load and store moves
template <typename T> struct alignas(16) Chunk { T v[16 / sizeof(T)]; };

// The caller's current device is put back: these entries sit between a host program's own GPU calls.
struct DeviceScope {
    int prev = -1, want;
    hipError_t err;
    explicit DeviceScope(int device) : want(device) {
        err = hipGetDevice(&prev);
        if (err == hipSuccess && prev != want) err = hipSetDevice(want);
    }
    ~DeviceScope() {
        if (prev >= 0 && prev != want) (void)hipSetDevice(prev);
    }
};

// hipLaunchKernel answers for this launch alone (hipGetLastError would also hand over an error somebody else left behind)
template <typename... Args, typename... Given>
inline hipError_t launch(void (*kernel)(Args...), size_t blocks, unsigned threads, unsigned lds, hipStream_t st, const Given&... args) {
    static_assert((std::is_same_v<std::remove_const_t<Args>, Given> && ...), "the kernel's arguments");
    void* p[] = {(void*)&args...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)blocks), dim3(threads), p, lds, st);
}

// zeros to `bytes` bytes (a multiple of 2): a kernel, since a fill that a captured graph replays must not be a memset node
hipError_t zero_fill(hipStream_t st, const void* data, size_t bytes);

// most workgroups of a launch: the runtime counts a grid's threads in 32 bits
inline bool grid_fits(size_t blocks, unsigned threads) { return blocks <= 0xffffffffull / threads; }

// One matrix operand's memory, for the checks of overlap: `lines` lines of `len` contiguous elements, `stride` apart.
struct Extent {
    const char* data = nullptr;
    long long lines = 0, len = 0, stride = 0;   // in bytes but for `lines`
    long long span() const { return lines > 0 && len > 0 ? (lines - 1) * stride + len : 0; }
};
inline bool overlap(const Extent& a, const Extent& b) {
    if (!a.data || !b.data || !a.span() || !b.span()) return false;
    if (a.data + a.span() <= b.data || b.data + b.span() <= a.data) return false;
    if (a.stride == b.stride && a.stride > 0 && a.lines > 1 && b.lines > 1) {   // windows side by side in lines of one buffer
        long long d = (b.data - a.data) % a.stride;
        if (d < 0) d += a.stride;
        if (d >= a.len && d + b.len <= a.stride) return false;
    }
    return true;
}

// Sums over 16 neighbouring lanes (rotations within a row of 16, which the vector unit does itself) and over the 64 of a wave: the same value in
// each lane, always added in the same order.
template <int N> __device__ inline float rotate16(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + N, 0xf, 0xf, true));
}
__device__ inline float sum4(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xb1, 0xf, 0xf, true));   // the other of a pair
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4e, 0xf, 0xf, true));   // the other pair
}
__device__ inline float sum16(float v) {
    v += rotate16<8>(v);
    v += rotate16<4>(v);
    v += rotate16<2>(v);
    v += rotate16<1>(v);
    return v;
}
__device__ inline float wave_sum(float v) {
    v = sum16(v);
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    return v;
}
// The largest of 64 magnitudes, each at least +0: as whole numbers they are in the same order, and a NaN is above infinity (the chip's maximum of
// floats would pass over it).
__device__ inline float wave_max_magnitude(float v) {
    unsigned m = __float_as_uint(v);
    auto rotate = [&](auto n) { m = max(m, (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x120 + decltype(n)::value, 0xf, 0xf, true)); };
    rotate(std::integral_constant<int, 8>{});
    rotate(std::integral_constant<int, 4>{});
    rotate(std::integral_constant<int, 2>{});
    rotate(std::integral_constant<int, 1>{});
    m = max(m, (unsigned)__shfl_xor((int)m, 16));
    return __uint_as_float(max(m, (unsigned)__shfl_xor((int)m, 32)));
}
__device__ inline float max_magnitude(float a, float b) { return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b))); }

}  // namespace aipt

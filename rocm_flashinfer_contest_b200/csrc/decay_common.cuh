// Shared pieces of the kernels for linear attention with a decay per head.
#pragma once

#include "../../include/gdn_decay_b200.h"
#include "gdn_common.cuh"

namespace gdn {
namespace decay {

// exp() of anything below this rounds to zero in fp32, so log decays are
// clamped here: -inf then stays out of the sums and differences of log decays
// (-inf - -inf is NaN).  NaN is kept.
constexpr float kMinLogDecay = -104.0f;

__device__ __forceinline__ float clamp_log_decay(float g) { return g < kMinLogDecay ? kMinLogDecay : g; }

// A clamped log decay as a multiple of 2^-10 and the rest, at most 2^-11.  Up to 64
// of them are summed part by part: the first sum is exact (at most 64 * 151 in
// magnitude, so 24 bits hold it), the second is off by 2^-28 at most, and so
// differences of two sums are as exact as the decays between them.  In one float
// each, behind gates that forget (-104), a sum is in the thousands and a difference
// of a tenth was off by 5e-4.
constexpr float kPartUnit = 12288.0f;  // 1.5 * 2^13: its last bit is 2^-10
__device__ __forceinline__ float2 split_log_decay(float g) {
    const float x = (g + kPartUnit) - kPartUnit;
    return make_float2(x, g - x);
}
// The same of g / ln 2, 1 / ln 2 itself in two floats.
__device__ __forceinline__ float2 split_log2_decay(float g) {
    constexpr double kLog2e = 1.4426950408889634;
    constexpr float kNear = (float)kLog2e, kRest = (float)(kLog2e - (double)kNear);
    const float x = fmaf(g, kNear, kPartUnit) - kPartUnit;
    return make_float2(x, fmaf(g, kRest, fmaf(g, kNear, -x)));
}

__device__ __forceinline__ long long slot_at(const void* idx, int is64, int i) {
    if (idx == nullptr) return i;
    return is64 ? static_cast<const long long*>(idx)[i] : (long long)static_cast<const int*>(idx)[i];
}

// The 16 state columns a lane of a row's 8 holds, as four float4: a row is
// read 128 bytes at a time by 8 neighbouring lanes in either type, so fp32
// lanes hold columns 4 sub + 32 j + {0..3} and bf16 lanes 8 sub + 64 (j / 2) +
// 4 (j % 2) + {0..3}.
template <bool kBf16>
__device__ __forceinline__ int col_of(int sub, int j) {
    return kBf16 ? 8 * sub + 64 * (j >> 1) + 4 * (j & 1) : 4 * sub + 32 * j;
}

template <bool kBf16>
struct StateRow;

template <>
struct StateRow<false> {
    using Raw = float4;
    static constexpr int kRaw = 4;
    static __device__ __forceinline__ void load(const void* base, size_t row, int sub, Raw (&r)[4]) {
        const float* p = static_cast<const float*>(base) + row * kDim + 4 * sub;
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = __ldcs(reinterpret_cast<const float4*>(p + 32 * j));
    }
    static __device__ __forceinline__ void widen(const Raw (&r)[4], float4 (&s)[4]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = r[j];
    }
    static __device__ __forceinline__ void store(void* base, size_t row, int sub, const float4 (&s)[4]) {
        float* p = static_cast<float*>(base) + row * kDim + 4 * sub;
#pragma unroll
        for (int j = 0; j < 4; ++j) __stcs(reinterpret_cast<float4*>(p + 32 * j), s[j]);
    }
};

__device__ __forceinline__ float2 widen2(uint32_t x) {
    return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}
// {lo, hi} rounded to nearest-even and packed
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
}

// True in one lane of a converged warp, always the same.
__device__ __forceinline__ bool elect_one() {
    uint32_t x;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(x));
    return x != 0;
}

// The upper halves of two floats, packed: their first 8 significant bits.
__device__ __forceinline__ uint32_t upper2(float2 x) {
    return __byte_perm(__float_as_uint(x.x), __float_as_uint(x.y), 0x7632);
}
// y minus the lower / upper bf16 of t, exactly rounded once (exact where t holds y's
// leading bits): one mixed-precision fma on the FMA pipe, where masking t out
// and subtracting it would be an integer operation on the busier ALU pipe.
__device__ __forceinline__ float2 minus_bf16(float2 y, uint32_t t) {
    float2 d;
    asm("{\n\t.reg .b16 l, h, m;\n\tmov.b32 {l, h}, %2;\n\tmov.b16 m, 0xbf80;\n\t"
        "fma.rn.f32.bf16 %0, l, m, %3;\n\tfma.rn.f32.bf16 %1, h, m, %4;\n\t}"
        : "=f"(d.x), "=f"(d.y)
        : "r"(t), "f"(y.x), "f"(y.y));
    return d;
}

template <>
struct StateRow<true> {
    using Raw = uint4;
    static constexpr int kRaw = 2;
    static __device__ __forceinline__ void load(const void* base, size_t row, int sub, Raw (&r)[2]) {
        const __nv_bfloat16* p = static_cast<const __nv_bfloat16*>(base) + row * kDim + 8 * sub;
#pragma unroll
        for (int j = 0; j < 2; ++j) r[j] = __ldcs(reinterpret_cast<const uint4*>(p + 64 * j));
    }
    static __device__ __forceinline__ void widen(const Raw (&r)[2], float4 (&s)[4]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 a = widen2(r[j].x), b = widen2(r[j].y), c = widen2(r[j].z), d = widen2(r[j].w);
            s[2 * j] = make_float4(a.x, a.y, b.x, b.y);
            s[2 * j + 1] = make_float4(c.x, c.y, d.x, d.y);
        }
    }
    static __device__ __forceinline__ void store(void* base, size_t row, int sub, const float4 (&s)[4]) {
        __nv_bfloat16* p = static_cast<__nv_bfloat16*>(base) + row * kDim + 8 * sub;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float4 a = s[2 * j], b = s[2 * j + 1];
            __stcs(reinterpret_cast<uint4*>(p + 64 * j),
                   make_uint4(pack_bf16(a.x, a.y), pack_bf16(a.z, a.w), pack_bf16(b.x, b.y), pack_bf16(b.z, b.w)));
        }
    }
};

}  // namespace decay
}  // namespace gdn

// Argument checks common to the entry points over a pool.
static inline int gdn_decay_check_pool(int state_bf16, int indices_int64, int per_token, int B, int T, int H, int HV,
                                       int K, int V, int pool_size) {
    if (B < 0 || T < 0 || H <= 0 || HV <= 0 || pool_size < 0 || (state_bf16 != 0 && state_bf16 != 1) ||
        (indices_int64 != 0 && indices_int64 != 1) || (per_token != 0 && per_token != 1))
        return GDN_ERR_INVALID;
    if (K != gdn::kDim || V != gdn::kDim || HV % H != 0) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

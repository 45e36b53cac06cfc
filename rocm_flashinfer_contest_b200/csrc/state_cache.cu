// state_cache.cu — pool slots written to an 8-bit cache and read back.
//
// Per group of 32 values: e = the smallest integer >= -127 with
// max|x| <= top 2^e (top = 127 for int8, 448 for e4m3), code = x 2^-e rounded
// to nearest-even, read back as code 2^e.  The scale is a power of two, so
// scaling is exact and the only rounding is the code's own; an int8 code is
// off by at most 2^(e-1), an e4m3 code by 2^-4 of its value (2^(e-10) below
// 2^(e-6)).
//
// Both directions stream: 4 + 33/32 bytes (fp32) or 2 + 33/32 (bf16) a value,
// nothing re-read; bound by HBM bandwidth.  A warp takes 512 consecutive values as
// 4 steps of 128: a lane reads 16 (8) bytes and writes 4 code bytes a step, so 8
// lanes share a group, its maximum takes three shuffles, and the warp's 16 exponent
// bytes leave as one store.  All 4 steps' loads are on their way before the first is
// needed.  48 slots of 32 heads, fp32 to int8 and back (248 MB): 45.8 us both, 5.4
// TB/s, with two launches' starts and ends in it (back alone 24.9); 8 steps a warp
// 47.4, 2 steps 49.4; CTAs of 1, 2 and 8 warps instead of 4 (8 steps): 47.1, 47.5 and
// 47.9.  bf16 to int8 and back (150 MB) 38.4, back alone 18.2, with half the bytes
// of a state on their way in a lane; e4m3 takes the same in both.
#include <cuda_fp8.h>

#include "decay_common.cuh"

namespace gdn {
namespace cache {

constexpr int kGroup = GDN_STATE_CACHE_GROUP;
constexpr int kSteps = 4, kWarpElems = kSteps * 128, kWarps = 4;

struct Params {
    void* pool;
    uint8_t* codes;
    uint8_t* exps;
    const void* slots;
    const void* cache_slots;
    int idx64, pool_size, cache_size;
    long long elems;
    unsigned tiles;  // CTAs for one slot
};

// Which slot pair and which values a warp has; false: padding or past the end.
__device__ __forceinline__ bool locate(const Params& p, long long& slot, long long& cslot, long long& at) {
    const int i = blockIdx.x / p.tiles;
    slot = decay::slot_at(p.slots, p.idx64, i);
    cslot = decay::slot_at(p.cache_slots, p.idx64, i);
    at = ((long long)(blockIdx.x % p.tiles) * kWarps + (threadIdx.x >> 5)) * kWarpElems;
    return slot >= 0 && slot < p.pool_size && cslot >= 0 && cslot < p.cache_size && at < p.elems;
}

template <bool kBf16>
__device__ __forceinline__ float4 load4(const void* pool, long long at) {
    if (kBf16) {
        const uint2 r = __ldcs(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(pool) + at));
        const float2 a = decay::widen2(r.x), b = decay::widen2(r.y);
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(pool) + at));
}

// 2^e for -149 <= e <= 127, exact (subnormal below -126).
__device__ __forceinline__ float pow2(int e) {
    return __int_as_float(e >= -126 ? (e + 127) << 23 : e >= -149 ? 1 << (e + 149) : 0);
}

// The larger one; NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// The exponent byte of a group with largest magnitude `top` (as the bits of a
// non-negative float).  top = f 2^x with 1 <= f < 2 (normal): the smallest e with
// f 2^x <= 127 2^e is x - 6 while f <= 127/64, else x - 5; for 448 = 1.75 2^8 it
// is x - 8 while f <= 1.75, else x - 7.  Subnormals (x < -126) clamp to -127.
template <bool kE4m3>
__device__ __forceinline__ int exponent_byte(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    const int x = (int)(top >> 23);  // biased; 0 for zero and subnormals
    const uint32_t frac = top & 0x7fffffu;
    const int byte = kE4m3 ? x - 8 + (frac > 0x600000u) : x - 6 + (frac > 0x7e0000u);
    return byte < 0 ? 0 : byte;
}

template <bool kE4m3>
__device__ __forceinline__ uint32_t encode4(float4 x, int byte) {
    if (byte == 255) return 0;
    const float inv = pow2(127 - byte);  // 2^-e, -127 <= -e <= 127: normal, or 2^-127
    x.x *= inv, x.y *= inv, x.z *= inv, x.w *= inv;
    if (kE4m3) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(x.x, x.y), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(x.z, x.w), __NV_SATFINITE, __NV_E4M3);
        return lo | hi << 16;
    }
    // |x| <= 127: adding 1.5 * 2^23 rounds to an integer, nearest-even, whose low byte is the code (the
    // conversion instruction has a quarter of the rate)
    constexpr float kMagic = 12582912.0f;
    const uint32_t a = __float_as_uint(x.x + kMagic), b = __float_as_uint(x.y + kMagic);
    const uint32_t c = __float_as_uint(x.z + kMagic), d = __float_as_uint(x.w + kMagic);
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <bool kE4m3>
__device__ __forceinline__ float4 decode4(uint32_t c, int byte) {
    const float s = byte == 255 ? __int_as_float(0x7fffffff) : pow2(byte - 127);
    float4 x;
    if (kE4m3) {
        const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c & 0xffffu), __NV_E4M3);
        const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(c >> 16), __NV_E4M3);
        const float2 a = __half22float2(__half2(lo)), b = __half22float2(__half2(hi));
        x = make_float4(a.x, a.y, b.x, b.y);
    } else {
        // 2^23 + (code + 128), exactly, in the low byte of that float
        const uint32_t u = c ^ 0x80808080u;
        constexpr float kOff = 8388608.0f + 128.0f;
        x = make_float4(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - kOff, __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - kOff,
                        __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - kOff, __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - kOff);
    }
    return make_float4(x.x * s, x.y * s, x.z * s, x.w * s);
}

template <bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(32 * kWarps) store_kernel(const Params p) {
    long long slot, cslot, at;
    if (!locate(p, slot, cslot, at)) return;
    const int lane = threadIdx.x & 31;
    const long long left = p.elems - at;  // a multiple of 32: groups are whole
    const long long src = slot * p.elems + at + 4 * lane, dst = cslot * p.elems + at + 4 * lane;
    float4 x[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u)
        x[u] = 128 * u + 4 * lane < left ? load4<kBf16>(p.pool, src + 128 * u) : make_float4(0.f, 0.f, 0.f, 0.f);
    int mine = 0;  // exponent byte of the warp's group number `lane`
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        float t = max_nan(max_nan(fabsf(x[u].x), fabsf(x[u].y)), max_nan(fabsf(x[u].z), fabsf(x[u].w)));
        t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, 1));
        t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, 2));
        t = max_nan(t, __shfl_xor_sync(0xffffffffu, t, 4));
        const uint32_t m = __float_as_uint(t) & 0x7fffffffu;
        const int byte = exponent_byte<kE4m3>(m);
        if (128 * u + 4 * lane < left)
            __stcs(reinterpret_cast<uint32_t*>(p.codes + dst + 128 * u), encode4<kE4m3>(x[u], byte));
        const int got = __shfl_sync(0xffffffffu, byte, 8 * (lane & 3));
        if (lane >> 2 == u) mine = got;
    }
    if (lane < 4 * kSteps && kGroup * lane < left) p.exps[(cslot * p.elems + at) / kGroup + lane] = (uint8_t)mine;
}

template <bool kBf16, bool kE4m3>
__global__ void __launch_bounds__(32 * kWarps) load_kernel(const Params p) {
    long long slot, cslot, at;
    if (!locate(p, slot, cslot, at)) return;
    const int lane = threadIdx.x & 31;
    const long long left = p.elems - at;
    const long long dst = slot * p.elems + at + 4 * lane, src = cslot * p.elems + at + 4 * lane;
    const uint8_t* ex = p.exps + (cslot * p.elems + at) / kGroup + (lane >> 3);
    uint32_t c[kSteps];
    int byte[kSteps];
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        const bool in = 128 * u + 4 * lane < left;
        c[u] = in ? __ldcs(reinterpret_cast<const uint32_t*>(p.codes + src + 128 * u)) : 0u;
        byte[u] = in ? ex[4 * u] : 0;
    }
#pragma unroll
    for (int u = 0; u < kSteps; ++u) {
        if (128 * u + 4 * lane >= left) break;
        const float4 x = decode4<kE4m3>(c[u], byte[u]);
        if (kBf16)
            __stcs(reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.pool) + dst + 128 * u),
                   make_uint2(decay::pack_bf16(x.x, x.y), decay::pack_bf16(x.z, x.w)));
        else
            __stcs(reinterpret_cast<float4*>(static_cast<float*>(p.pool) + dst + 128 * u), x);
    }
}

template <bool kStore>
static int run(const Params& p, int B, int bf16, int e4m3, void* stream) {
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)B * p.tiles, thr = 32 * kWarps;
    if (kStore) {
        if (bf16 && e4m3) store_kernel<true, true><<<grid, thr, 0, st>>>(p);
        else if (bf16) store_kernel<true, false><<<grid, thr, 0, st>>>(p);
        else if (e4m3) store_kernel<false, true><<<grid, thr, 0, st>>>(p);
        else store_kernel<false, false><<<grid, thr, 0, st>>>(p);
    } else {
        if (bf16 && e4m3) load_kernel<true, true><<<grid, thr, 0, st>>>(p);
        else if (bf16) load_kernel<true, false><<<grid, thr, 0, st>>>(p);
        else if (e4m3) load_kernel<false, true><<<grid, thr, 0, st>>>(p);
        else load_kernel<false, false><<<grid, thr, 0, st>>>(p);
    }
    return gdn_launch_status();
}

template <bool kStore>
static int entry(const void* pool, int bf16, const void* slots, const void* cache_slots, int idx64, const void* codes,
                 int e4m3, const void* exps, int B, long long elems, int pool_size, int cache_size, void* stream) {
    if (B < 0 || elems <= 0 || pool_size < 0 || cache_size < 0 || (bf16 != 0 && bf16 != 1) ||
        (e4m3 != 0 && e4m3 != 1) || (idx64 != 0 && idx64 != 1))
        return GDN_ERR_INVALID;
    if (elems % kGroup != 0) return GDN_ERR_UNSUPPORTED;
    const long long per = (long long)kWarps * kWarpElems, tiles = (elems + per - 1) / per;
    if (tiles > (1ll << 30) || tiles * B > (1ll << 30)) return GDN_ERR_UNSUPPORTED;  // grid index
    if (B == 0) return GDN_OK;
    // (without slots on a side there may be no address)
    if (!slots || !cache_slots || (pool_size > 0 && !pool) || (cache_size > 0 && (!codes || !exps))) return GDN_ERR_INVALID;
    if (!gdn_aligned(pool, 16) || !gdn_aligned(codes, 16) || !gdn_aligned(slots, idx64 ? 8 : 4) ||
        !gdn_aligned(cache_slots, idx64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    if (pool_size == 0 || cache_size == 0) return GDN_OK;  // every pair is padding
    Params p;
    p.pool = const_cast<void*>(pool);
    p.codes = static_cast<uint8_t*>(const_cast<void*>(codes));
    p.exps = static_cast<uint8_t*>(const_cast<void*>(exps));
    p.slots = slots;
    p.cache_slots = cache_slots;
    p.idx64 = idx64;
    p.pool_size = pool_size;
    p.cache_size = cache_size;
    p.elems = elems;
    p.tiles = (unsigned)tiles;
    return run<kStore>(p, B, bf16, e4m3, stream);
}

}  // namespace cache
}  // namespace gdn

extern "C" int gdn_state_cache_store(const void* pool, int state_bf16, const void* slots, const void* cache_slots,
                                     int slots_int64, void* codes, int e4m3, unsigned char* exps, int B,
                                     long long slot_elems, int pool_size, int cache_size, void* stream) {
    return gdn::cache::entry<true>(pool, state_bf16, slots, cache_slots, slots_int64, codes, e4m3, exps, B, slot_elems,
                                   pool_size, cache_size, stream);
}

extern "C" int gdn_state_cache_load(const void* codes, int e4m3, const unsigned char* exps, const void* cache_slots,
                                    const void* slots, int slots_int64, void* pool, int state_bf16, int B,
                                    long long slot_elems, int pool_size, int cache_size, void* stream) {
    return gdn::cache::entry<false>(pool, state_bf16, slots, cache_slots, slots_int64, codes, e4m3, exps, B, slot_elems,
                                    pool_size, cache_size, stream);
}

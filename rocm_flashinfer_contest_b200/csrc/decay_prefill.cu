// decay_prefill.cu — prefill of packed prompts for linear attention with a
// decay per head (sm_100a).
#include "decay_common.cuh"

namespace gdn {
namespace decay {

struct PrefillParams {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const float* state;  // nullable: zero
    const float* log_decay;
    const void* cu;
    __nv_bfloat16* out;
    float* new_state;
    float scale;
    int cu64, per_token, N, T, H, HV, rep;
};

__device__ __forceinline__ int cu_at(const void* cu, int is64, int i, int T) {
    const long long x = is64 ? static_cast<const long long*>(cu)[i] : (long long)static_cast<const int*>(cu)[i];
    return (int)(x < 0 ? 0 : x > T ? T : x);
}

// Token-serial form: 32 rows of one sequence's v-head per CTA, 8 lanes to a
// row, the state in registers over all tokens.
__global__ void __launch_bounds__(128) decay_prefill_serial_kernel(const PrefillParams p) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
    const int rb = blockIdx.x % 4, nh = blockIdx.x / 4, n = nh / p.HV, h = nh % p.HV, hq = h / p.rep;
    const int row = rb * 32 + warp * 8 + (lane >> 3);
    if (n == p.N) {  // tokens of no sequence: zero outputs
        const int c0 = cu_at(p.cu, p.cu64, 0, p.T), c1 = cu_at(p.cu, p.cu64, p.N, p.T);
        for (int t = warp; t < p.T; t += 4)
            if (t < c0 || t >= c1) p.out[((size_t)t * p.HV + h) * kDim + rb * 32 + lane] = __float2bfloat16_rn(0.f);
        return;
    }
    const int t0 = cu_at(p.cu, p.cu64, n, p.T), t1 = cu_at(p.cu, p.cu64, n + 1, p.T);
    float4 s[2][4];
#pragma unroll
    for (int ps = 0; ps < 2; ++ps) {
        if (p.state != nullptr)
            StateRow<false>::load(p.state, (size_t)nh * kDim + row + 4 * ps, sub, s[ps]);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) s[ps][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int t = t0; t < t1; ++t) {
        const size_t qk = ((size_t)t * p.H + hq) * kDim, vo = ((size_t)t * p.HV + h) * kDim + row;
        const float a = expf(clamp_log_decay(p.log_decay[p.per_token ? (size_t)t * p.HV + h : h]));
        float4 q[4], k[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            q[j] = load_bf16x4(p.q + qk + 4 * sub + 32 * j);
            k[j] = load_bf16x4(p.k + qk + 4 * sub + 32 * j);
        }
#pragma unroll
        for (int ps = 0; ps < 2; ++ps) {
            const float vv = bf16_to_f32(p.v[vo + 4 * ps]);
            float2 acc = make_float2(0.f, 0.f);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                s[ps][j] = gs_plus_dk(a, s[ps][j], vv, k[j]);
                acc = dot4_acc2(s[ps][j], q[j], acc);
            }
            float o = acc.x + acc.y;
            o += __shfl_xor_sync(0xffffffffu, o, 1);
            o += __shfl_xor_sync(0xffffffffu, o, 2);
            o += __shfl_xor_sync(0xffffffffu, o, 4);
            if (sub == 0) p.out[vo + 4 * ps] = __float2bfloat16_rn(p.scale * o);
        }
    }
#pragma unroll
    for (int ps = 0; ps < 2; ++ps) StateRow<false>::store(p.new_state, (size_t)nh * kDim + row + 4 * ps, sub, s[ps]);
}

}  // namespace decay
}  // namespace gdn

extern "C" size_t gdn_decay_prefill_workspace_bytes(int N, int T, int HV) {
    (void)N, (void)T, (void)HV;
    return 0;
}

extern "C" int gdn_decay_prefill_fwd(const void* q, const void* k, const void* v, const float* state,
                                     const float* log_decay, int decay_per_token, const void* cu_seqlens,
                                     int cu_seqlens_is_int64, int N, int T, float scale, int H, int HV, int K, int V,
                                     void* out, float* new_state, void* workspace, size_t workspace_bytes,
                                     void* stream) {
    using namespace gdn::decay;
    if (N < 0 || T < 0 || H <= 0 || HV <= 0 || (cu_seqlens_is_int64 != 0 && cu_seqlens_is_int64 != 1) ||
        (decay_per_token != 0 && decay_per_token != 1))
        return GDN_ERR_INVALID;
    if (K != gdn::kDim || V != gdn::kDim || HV % H != 0) return GDN_ERR_UNSUPPORTED;
    if (((long long)N + 1) * HV > (1ll << 27)) return GDN_ERR_UNSUPPORTED;  // grid index
    if (N == 0 && T == 0) return GDN_OK;
    if (!cu_seqlens || (T > 0 && (!q || !k || !v || !out)) || !log_decay || (N > 0 && !new_state))
        return GDN_ERR_INVALID;
    if (!gdn_aligned(q, 16) || !gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(out, 16) ||
        !gdn_aligned(state, 16) || !gdn_aligned(new_state, 16) || !gdn_aligned(log_decay, 4) ||
        !gdn_aligned(cu_seqlens, cu_seqlens_is_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    const size_t need = gdn_decay_prefill_workspace_bytes(N, T, HV);
    if (need && (!workspace || workspace_bytes < need)) return GDN_ERR_INVALID;
    if (!gdn_aligned(workspace, 16)) return GDN_ERR_ALIGN;
    PrefillParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.v = static_cast<const __nv_bfloat16*>(v);
    p.state = state;
    p.log_decay = log_decay;
    p.cu = cu_seqlens;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.new_state = new_state;
    p.scale = scale == 0.0f ? 1.0f / sqrtf((float)K) : scale;
    p.cu64 = cu_seqlens_is_int64;
    p.per_token = decay_per_token;
    p.N = N;
    p.T = T;
    p.H = H;
    p.HV = HV;
    p.rep = HV / H;
    decay_prefill_serial_kernel<<<(unsigned)((N + 1) * HV * 4), 128, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return gdn_launch_status();
}

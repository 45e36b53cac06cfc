// decay_decode.cu — single-token step of linear attention with a decay per
// head over pooled states (sm_100a).
//
// Per v-head, with the k-last state row S[v, :]:
//   S'[v,:] = e^g S[v,:] + v[v] k        o[v] = scale * (S'[v,:] . q)
//
// Rows are independent, so the kernel is one streaming pass: every state row
// is read once and written once, 8 bytes (fp32) or 4 bytes (bf16) of HBM
// traffic per state element, and nothing else of size moves.  It is bound by
// HBM bandwidth from about 16 entries of 32 heads on, by the latency of one
// load-compute-store chain below that.
//
// 8 lanes share a row, so a warp-wide 16-byte load covers four whole 128-byte
// lines, and a row's dot product takes three shuffles.  Each lane starts all
// the loads of its rows before it needs any: 128 bytes a lane, 16 KiB a CTA, so
// 32 rows of fp32 or 64 of bf16.  Measured, by rows per CTA: 64 entries of 32
// heads in fp32 (268 MB) 43.4 us with 16, 43.3 with 32 (6.2 TB/s), 43.5 with 64
// and 44.4 with 128; 221 entries of 32 heads in bf16 (463 MB) 87.2, 77.4, 74.0
// (6.3 TB/s) and 74.4.
#include "decay_common.cuh"

namespace gdn {
namespace decay {

struct DecodeParams {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const void* pool_in;  // nullable: zero states
    void* pool_out;
    const void* indices;
    const void* out_indices;
    const float* log_decay;
    __nv_bfloat16* out;
    float scale;
    int idx64, per_token, H, HV, rep, pool_size;
};

template <bool kBf16>
constexpr int kDecodeRows = kBf16 ? 64 : 32;

// 4 warps, kRows rows of one v-head per CTA; a warp pass covers 4 rows.
template <bool kBf16>
__global__ void __launch_bounds__(128) decay_decode_kernel(const DecodeParams p) {
    using Row = StateRow<kBf16>;
    constexpr int kRows = kDecodeRows<kBf16>, kPasses = kRows / 16, kBlocks = kDim / kRows;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane & 7;
    const int head = blockIdx.x / kBlocks;  // entry * HV + h
    const int row0 = (blockIdx.x % kBlocks) * kRows + warp * (kRows / 4) + (lane >> 3);
    const int b = head / p.HV, h = head % p.HV, hq = h / p.rep;

    const long long slot = slot_at(p.indices, p.idx64, b);
    if (slot < 0 || slot >= p.pool_size) {  // padding: zero output, no state touched
        if (sub == 0)
#pragma unroll
            for (int ps = 0; ps < kPasses; ++ps) p.out[(size_t)head * kDim + row0 + 4 * ps] = __float2bfloat16_rn(0.f);
        return;
    }
    const size_t srow = ((size_t)slot * p.HV + h) * kDim + row0;
    typename Row::Raw raw[kPasses][Row::kRaw];
    if (p.pool_in != nullptr) {
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) Row::load(p.pool_in, srow + 4 * ps, sub, raw[ps]);
    } else {
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps)
#pragma unroll
            for (int j = 0; j < Row::kRaw; ++j) raw[ps][j] = typename Row::Raw{};
    }
    const size_t qk = ((size_t)b * p.H + hq) * kDim;
    float4 q[4], k[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j] = load_bf16x4(p.q + qk + col_of<kBf16>(sub, j));
        k[j] = load_bf16x4(p.k + qk + col_of<kBf16>(sub, j));
    }
    float vv[kPasses];
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) vv[ps] = bf16_to_f32(p.v[(size_t)head * kDim + row0 + 4 * ps]);
    const float a = expf(clamp_log_decay(p.log_decay[p.per_token ? head : h]));
    const long long oslot = p.out_indices ? slot_at(p.out_indices, p.idx64, b) : slot;
    const bool put = oslot >= 0 && oslot < p.pool_size;
    const size_t drow = ((size_t)(put ? oslot : 0) * p.HV + h) * kDim + row0;

#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) {
        float4 s[4];
        Row::widen(raw[ps], s);
        float2 acc = make_float2(0.f, 0.f);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            s[j] = gs_plus_dk(a, s[j], vv[ps], k[j]);
            acc = dot4_acc2(s[j], q[j], acc);
        }
        if (put) Row::store(p.pool_out, drow + 4 * ps, sub, s);
        float o = acc.x + acc.y;
        o += __shfl_xor_sync(0xffffffffu, o, 1);
        o += __shfl_xor_sync(0xffffffffu, o, 2);
        o += __shfl_xor_sync(0xffffffffu, o, 4);
        if (sub == 0) p.out[(size_t)head * kDim + row0 + 4 * ps] = __float2bfloat16_rn(p.scale * o);
    }
}

template <bool kBf16>
static void launch_decode(const DecodeParams& p, long long heads, cudaStream_t st) {
    decay_decode_kernel<kBf16><<<(unsigned)(heads * (kDim / kDecodeRows<kBf16>)), 128, 0, st>>>(p);
}

}  // namespace decay
}  // namespace gdn

extern "C" int gdn_decay_decode_fwd(const void* q, const void* k, const void* v, const void* pool_in, void* pool_out,
                                    int state_bf16, const void* indices, const void* out_indices, int indices_int64,
                                    const float* log_decay, int decay_per_token, float scale, int B, int H, int HV,
                                    int K, int V, int pool_size, void* out, void* stream) {
    const int bad = gdn_decay_check_pool(state_bf16, indices_int64, decay_per_token, B, 1, H, HV, K, V, pool_size);
    if (bad) return bad;
    if ((long long)B * HV > (1ll << 27)) return GDN_ERR_UNSUPPORTED;  // grid index
    if (B == 0) return GDN_OK;
    // (a pool without slots may have no address: every entry is padding then)
    if (!q || !k || !v || !log_decay || !out || (!pool_out && pool_size > 0)) return GDN_ERR_INVALID;
    if (!gdn_aligned(q, 16) || !gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(out, 16) ||
        !gdn_aligned(pool_in, 16) || !gdn_aligned(pool_out, 16) || !gdn_aligned(log_decay, 4) ||
        !gdn_aligned(indices, indices_int64 ? 8 : 4) || !gdn_aligned(out_indices, indices_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    // the pools are one buffer or two that do not overlap
    const size_t bytes = (size_t)pool_size * HV * gdn::kDim * gdn::kDim * (state_bf16 ? 2 : 4);
    const uintptr_t pi = (uintptr_t)pool_in, po = (uintptr_t)pool_out;
    if (pool_in && pi != po && pi < po + bytes && po < pi + bytes) return GDN_ERR_INVALID;

    gdn::decay::DecodeParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.v = static_cast<const __nv_bfloat16*>(v);
    p.pool_in = pool_in;
    p.pool_out = pool_out;
    p.indices = indices;
    p.out_indices = out_indices;
    p.log_decay = log_decay;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.scale = scale == 0.0f ? 1.0f / sqrtf((float)K) : scale;
    p.idx64 = indices_int64;
    p.per_token = decay_per_token;
    p.H = H;
    p.HV = HV;
    p.rep = HV / H;
    p.pool_size = pool_size;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const long long heads = (long long)B * HV;
    if (state_bf16)
        gdn::decay::launch_decode<true>(p, heads, st);
    else
        gdn::decay::launch_decode<false>(p, heads, st);
    return gdn_launch_status();
}

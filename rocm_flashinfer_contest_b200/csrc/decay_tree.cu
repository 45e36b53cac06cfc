// decay_tree.cu — linear attention with a decay per head for trees of drafted
// tokens over pooled states, and the update by the accepted path (sm_100a).
//
// With c_t the sum of the log decays on node t's path from the cached state S
// (node t included) and j <= t meaning "j is on node t's path":
//   o_t = scale * ( e^{c_t} S q_t + sum_{j <= t} e^{c_t - c_j} (q_t . k_j) v_j )
//   S'  = e^{c_a} S + sum_{j <= a} e^{c_a - c_j} v_j k_j^T      (a: accepted)
#include <cuda.h>

#include <atomic>
#include <mutex>

#include "decay_common.cuh"
#include "umma.cuh"

namespace gdn {
namespace decay {

constexpr int kTreeMax = GDN_DECAY_TREE_MAX;

// ---------------------------------------------------------------------------
// Verification: persistent CTAs of 8 warps, one entry's v-head after the other,
// two CTAs per SM up to 32 nodes.
//
// The state (64 KiB in fp32) is the traffic.  It is read once, by TMA into shared
// memory while the CTA works on the item before it; a thread then turns half a
// row into bf16 terms in tensor memory, where they are the A operand of
// o^T[v, t] = S[v, :] . q_t on tcgen05, and the next state may come.  q, k and v of
// the tree come by TMA too, each asked for as soon as the last item is done with
// its place.  The scores and their product with v are small (T x T x 128) and cut
// by the paths: warp-level products on operands from ldmatrix, which run beside the
// tcgen05 ones.  One warp finds the next item's paths meanwhile.
//
// 64 entries, 32 v-heads, 32 nodes (182 MB): 37.6 us, 4.8 TB/s.  Two CTAs take turns
// at load, conversion, products and outputs, 7,300 cycles an item each, and shared
// memory holds no third.  With S q on warp-level products too, 54 us: two terms of a
// state times 32 tokens kept that path, an eighth of tcgen05's rate, busy for 3,700
// cycles a state, as long as its bytes take.  With q, k and v by 16-byte copies of all
// threads 43, by a copy a row 54; operands of the small products by plain loads +2;
// padding's v zeroed in shared memory, and every thread asking for the next slot,
// +2; the next slot and output place found by every thread +1; the paths found by
// one warp before the item +0.5.  64 such entries without a pause between calls, fp32
// / bf16 states: 8 nodes 32.0 / 25.3 us, 16 33.7 / 27.0, 32 38.3 / 31.4, 64 (one CTA
// an SM) 74 / 68.
// bf16 and 16 nodes would leave shared memory for four CTAs; their 256 columns of
// tensor memory each let two run.
//
// Precision: q, k, v are bf16 as given.  An fp32 state is split into two bf16
// terms (hi, its first 8 bits, and lo, what is left, below 2^-7 of its power of two,
// rounded to 8 bits: off by at most 2^-16 of it) and the decayed scores P likewise,
// so the products lose nothing next to the output's own rounding to bf16 (2^-8);
// one bf16 term each would about double the output's error.  Sums of log decays
// are exact to 2^-28 (split_log_decay).
// ---------------------------------------------------------------------------

struct VerifyParams {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const void* indices;
    const int* parents;
    const float* log_decay;
    __nv_bfloat16* out;
    float scale;
    int idx64, per_token, T, Tp, H, HV, rep, pool_size, items;  // Tp: T rounded up to 16; items: entries * HV
};

constexpr int kVS = 136, kPS = 72;  // row strides in bf16 elements of the outputs, of P

// tensor-memory columns: S's two terms, o^T
constexpr uint32_t kTmHi = 0, kTmLo = 64, kTmO = 128;

// Shared memory: the next state in boxes of 128 rows x 128 bytes (128-byte swizzle),
// then q, k and v in boxes of Tp rows x 128 bytes (same swizzle: q is a K-major
// operand as it lies), outputs and the two terms of P.
constexpr uint32_t kStateBox = 128 * 128;
__host__ __device__ constexpr uint32_t state_bytes(bool bf16) { return bf16 ? 2 * kStateBox : 4 * kStateBox; }
__host__ __device__ constexpr size_t verify_smem(int Tp, bool bf16) {
    return state_bytes(bf16) + (size_t)Tp * 2 * (3 * kDim + kVS + 2 * kPS);
}

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// Four 8 x 8 matrices, rows from the addresses of lanes 8 i .. 8 i + 7; turned or not.
__device__ __forceinline__ void ldmatrix4(const void* p, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(const void* p, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(smem_addr(p))
                 : "memory");
}

// hi + lo split of a pair: hi = the first 8 bits, lo = the rest rounded to bf16.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = upper2(make_float2(x, y));
    const float2 r = minus_bf16(make_float2(x, y), hi);
    lo = pack_bf16(r.x, r.y);
}

// 16 lanes x 16 columns in the fragment layout of a 16 x 8 product's result, two of
// them: a lane's rows lane / 4 and 8 on, columns 2 (lane % 4) + {0, 1} and 8 on.
__device__ __forceinline__ void tmem_ld_frag(uint32_t ta, float (&a)[4], float (&b)[4]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
        : "=f"(a[0]), "=f"(a[1]), "=f"(a[2]), "=f"(a[3]), "=f"(b[0]), "=f"(b[1]), "=f"(b[2]), "=f"(b[3])
        : "r"(ta)
        : "memory");
}

template <bool kBf16>
__global__ void __launch_bounds__(256, 2)
    decay_verify_kernel(const VerifyParams p, const __grid_constant__ CUtensorMap m_pool, const __grid_constant__ CUtensorMap m_q,
                        const __grid_constant__ CUtensorMap m_k, const __grid_constant__ CUtensorMap m_v) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    // of an item and the next one
    __shared__ unsigned long long paths[2][kTreeMax];        // bit j: j is on the node's path; 0: padding
    __shared__ float2 sums[2][kTreeMax];                      // c_t in two parts (split_log_decay)
    __shared__ float decays[2][kTreeMax];                     // e^{c_t}
    __shared__ unsigned long long used_nodes[2];              // bit t: node t is not padding
    __shared__ size_t s_out;               // the next item's first output
    __shared__ int s_padding;              // the next item has no state
    __shared__ uint64_t s_full, s_done, s_qk, s_v;
    __shared__ uint32_t s_tmem;

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int T = p.T, Tp = p.Tp, mt = Tp / 16;
    const int quarter = warp & 3, half = warp >> 2;  // tensor-memory lanes; columns of S, and rows of o^T
    const int rows = 32 * quarter + 16 * half;       // this warp's rows of o^T
    uint8_t* qs = smem_raw + state_bytes(kBf16);
    uint8_t* ks_ = qs + Tp * 256;
    uint8_t* vs = ks_ + Tp * 256;
    __nv_bfloat16* os = reinterpret_cast<__nv_bfloat16*>(vs + Tp * 256);
    __nv_bfloat16* ph = os + Tp * kVS;
    __nv_bfloat16* pl = ph + Tp * kPS;

    auto slot_of = [&](int item) -> long long {  // -1: padding
        const long long slot = slot_at(p.indices, p.idx64, item / p.HV);
        return slot < 0 || slot >= p.pool_size ? -1 : slot;
    };
    // one thread asks for the state of an item; padding has none
    auto ask_state = [&](int item) {
        if (item >= p.items) return;
        const long long slot = slot_of(item);
        if (slot < 0) return;
        const int number = (int)slot * p.HV + item % p.HV;
        umma::mbar_arrive_expect_tx(&s_full, state_bytes(kBf16));
#pragma unroll
        for (int x = 0; x < (kBf16 ? 2 : 4); ++x)
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                    smem_addr(smem_raw) + x * kStateBox),
                "l"(reinterpret_cast<uint64_t>(&m_pool)), "r"(x * (kBf16 ? 64 : 32)), "r"(0), "r"(number), "r"(smem_addr(&s_full))
                : "memory");
    };
    auto look_at = [&](int item) {
        if (item >= p.items) return;
        s_out = ((size_t)(item / p.HV) * T * p.HV + item % p.HV) * kDim;
        s_padding = slot_of(item) < 0;
    };
    // one thread asks for the tree's q and k, and then for its v
    auto ask_box = [&](uint8_t* dst, const CUtensorMap& map, int head, int b, uint64_t* bar) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
            asm volatile(
                "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                    smem_addr(dst) + x * Tp * 128),
                "l"(reinterpret_cast<uint64_t>(&map)), "r"(64 * x), "r"(head), "r"(b * T), "r"(smem_addr(bar))
                : "memory");
    };
    auto ask_qk = [&](int item) {
        if (item >= p.items) return;
        const int b = item / p.HV, hq = item % p.HV / p.rep;
        umma::mbar_arrive_expect_tx(&s_qk, T * 512);
        ask_box(qs, m_q, hq, b, &s_qk);
        ask_box(ks_, m_k, hq, b, &s_qk);
    };
    auto ask_v = [&](int item) {
        if (item >= p.items) return;
        umma::mbar_arrive_expect_tx(&s_v, T * 256);
        ask_box(vs, m_v, item % p.HV, item / p.HV, &s_v);
    };
    // warp 7 asks for its parents and log decays (nodes lane, lane + 32)
    int par[2];
    float gg[2];
    auto ask_path = [&](int item) {
        if (item >= p.items) return;
        const int b = item / p.HV, h = item % p.HV;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = lane + 32 * i;
            par[i] = -2, gg[i] = 0.f;
            if (t < T) {
                par[i] = p.parents[(size_t)b * T + t];
                gg[i] = p.log_decay[p.per_token ? ((size_t)b * T + t) * p.HV + h : h];
            }
        }
    };

    // Paths and their decays by pointer doubling, a lane's two nodes in registers:
    // after r rounds a node knows the last 2^r nodes of its path; -1 ends a path, -2
    // marks padding.
    auto find_paths = [&](int buf) {
        unsigned long long m[2];
        float2 cc[2];
        int up[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = lane + 32 * i;
            up[i] = par[i] < -1 || par[i] >= t ? -2 : par[i];
            cc[i] = split_log_decay(clamp_log_decay(gg[i]));
            m[i] = t < T ? 1ull << t : 0ull;
        }
#pragma unroll 1
        for (int hop = 1; hop < T; hop *= 2) {
            unsigned long long mm[2];
            float2 dc[2];
            int uu[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {  // what node up[i] knows
                const int u = up[i] & 31;
                mm[i] = __shfl_sync(0xffffffffu, m[0], u);
                dc[i].x = __shfl_sync(0xffffffffu, cc[0].x, u), dc[i].y = __shfl_sync(0xffffffffu, cc[0].y, u);
                uu[i] = __shfl_sync(0xffffffffu, up[0], u);
                if (T > 32) {
                    const unsigned long long m1 = __shfl_sync(0xffffffffu, m[1], u);
                    const float2 d1 = make_float2(__shfl_sync(0xffffffffu, cc[1].x, u), __shfl_sync(0xffffffffu, cc[1].y, u));
                    const int u1 = __shfl_sync(0xffffffffu, up[1], u);
                    if (up[i] >= 32) mm[i] = m1, dc[i] = d1, uu[i] = u1;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (up[i] >= 0) cc[i].x += dc[i].x, cc[i].y += dc[i].y, m[i] |= mm[i], up[i] = uu[i];
        }
        unsigned used[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = lane + 32 * i;
            paths[buf][t] = up[i] == -1 ? m[i] : 0ull;
            sums[buf][t] = cc[i];
            decays[buf][t] = expf(cc[i].x + cc[i].y);
            used[i] = __ballot_sync(0xffffffffu, up[i] == -1);
        }
        if (lane == 0) used_nodes[buf] = (unsigned long long)used[1] << 32 | used[0];
    };

    if (tid == 0) {
        umma::mbar_init(&s_full, 1);
        umma::mbar_init(&s_done, 1);
        umma::mbar_init(&s_qk, 1);
        umma::mbar_init(&s_v, 1);
        umma::fence_mbar_init();
        ask_state(blockIdx.x);
    }
    if (warp == 1) {
        umma::tmem_alloc(&s_tmem, 256);
        umma::tmem_relinquish();
    }
    // rows T .. Tp - 1 of q, k and v stay zero
    for (int i = tid; i < (Tp - T) * 16; i += 256) {
        const int t = T + (i >> 4), x = 8 * (i & 15);
        *reinterpret_cast<uint4*>(qs + umma::kmaj_off(t, x, Tp)) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(ks_ + umma::kmaj_off(t, x, Tp)) = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(vs + umma::kmaj_off(t, x, Tp)) = make_uint4(0, 0, 0, 0);
    }
    if (warp == 7) ask_path(blockIdx.x), find_paths(0), ask_path(blockIdx.x + gridDim.x);
    if (tid == 192) look_at(blockIdx.x);
    umma::fence_before_sync();
    __syncthreads();
    umma::fence_after_sync();
    if (tid == 192) ask_qk(blockIdx.x), ask_v(blockIdx.x);
    const uint32_t tm = s_tmem;
    uint32_t phase = 0, turn = 0;  // states and items so far
    bool lost = false;  // a wait has run out

#pragma unroll 1
    for (int item = blockIdx.x; item < p.items; item += gridDim.x, ++turn) {
        const int next = item + gridDim.x;
        __nv_bfloat16* out = p.out + s_out;  // + t * HV * 128
        const bool padding = s_padding;
        const unsigned long long* s_path = paths[turn & 1];
        const float2* s_c = sums[turn & 1];
        const float* s_e = decays[turn & 1];

        float acc[8][4];  // o^T rows `rows` + {g, g + 8}, tokens 8 n + 2 c + {0, 1}
        if (!padding) {
            // half of state row 32 quarter + lane, in bf16 terms, into tensor memory
            lost = !umma::mbar_wait(&s_full, phase & 1u);
            __syncwarp();
            const uint32_t tl = tm + ((uint32_t)(32 * quarter) << 16);
            const uint8_t* row = smem_raw + (32 * quarter + lane) * 128;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                uint32_t hi[16], lo[16];
                if (kBf16) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint4 y = *reinterpret_cast<const uint4*>(row + half * kStateBox + (((4 * x + j) ^ (lane & 7)) << 4));
                        hi[4 * j] = y.x, hi[4 * j + 1] = y.y, hi[4 * j + 2] = y.z, hi[4 * j + 3] = y.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float4 y = *reinterpret_cast<const float4*>(row + (2 * half + x) * kStateBox + ((j ^ (lane & 7)) << 4));
                        split2(y.x, y.y, hi[2 * j], lo[2 * j]);
                        split2(y.z, y.w, hi[2 * j + 1], lo[2 * j + 1]);
                    }
                    umma::tmem_st16_u32_nowait(tl + kTmLo + 32 * half + 16 * x, lo);
                }
                umma::tmem_st16_u32_nowait(tl + kTmHi + 32 * half + 16 * x, hi);
            }
            umma::tmem_wait_st();
            umma::fence_before_sync();
        }
        if (!umma::mbar_wait(&s_qk, turn & 1u)) lost = true;
        umma::fence_proxy_async_smem();  // q is read, and the state's place written, by the async proxy
        if (__syncthreads_or(lost)) break;
        if (tid == 0) ask_state(next);
        if (tid == 192) look_at(next);

        if (!padding) {
            if (warp == 7) {  // the last to have a tile of scores
                umma::fence_after_sync();
                const uint32_t tu = __shfl_sync(0xffffffffu, tm, 0), id = umma::idesc_f16(128, Tp, 1, 1, 0, 0);
                const uint64_t dq = umma::desc_kmaj(__shfl_sync(0xffffffffu, smem_addr(qs), 0), Tp, 0);
                if (elect_one()) {
#pragma unroll
                    for (int term = kBf16 ? 0 : 1; term >= 0; --term)  // the small one first
#pragma unroll
                        for (int ks = 0; ks < 8; ++ks)
                            umma::mma_f16_ts(tu + kTmO, tu + (term ? kTmLo : kTmHi) + 8 * ks,
                                             umma::desc_add(dq, (ks >> 2) * Tp * 128 + (ks & 3) * 32), id, ks > 0 || (!kBf16 && term == 0));
                    umma::mma_commit(&s_done);
                }
                __syncwarp();
            }
        }
        if (warp == 7 && next < p.items) find_paths((turn + 1) & 1);
        if (!padding) {

            // P[t, j] = e^{c_t - c_j} (q_t . k_j) on the paths, 0 elsewhere; nodes come after their parents, so
            // 16 x 8 tiles with every j > t stay out (they are not read either)
#pragma unroll 1
            for (int tile = warp; tile < mt * (mt + 1); tile += 8) {
                int m = 0, n = tile;  // row block m has 2 (m + 1) column tiles
                while (n >= 2 * (m + 1)) n -= 2 * (m + 1), ++m;
                float x[4] = {0.f, 0.f, 0.f, 0.f}, x2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < 8; ks += 2) {
                    uint32_t a[4], a2[4], bb[4];
                    const int arow = 16 * m + (lane & 15), acol = 16 * ks + 8 * (lane >> 4);
                    ldmatrix4(qs + umma::kmaj_off(arow, acol, Tp), a);
                    ldmatrix4(qs + umma::kmaj_off(arow, acol + 16, Tp), a2);
                    ldmatrix4(ks_ + umma::kmaj_off(8 * n + (lane & 7), 16 * ks + 8 * (lane >> 3), Tp), bb);
                    mma16816(x, a, bb[0], bb[1]);
                    mma16816(x2, a2, bb[2], bb[3]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] += x2[e];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const int t = 16 * m + g + 8 * r, j = 8 * n + 2 * c;
                    const unsigned long long path = s_path[t];
                    const float2 ct = s_c[t], cj = s_c[j], cj1 = s_c[j + 1];
                    const float y = path >> j & 1 ? x[2 * r] * expf((ct.x - cj.x) + (ct.y - cj.y)) : 0.f;
                    const float z = path >> (j + 1) & 1 ? x[2 * r + 1] * expf((ct.x - cj1.x) + (ct.y - cj1.y)) : 0.f;
                    uint32_t hi, low;
                    split2(y, z, hi, low);
                    *reinterpret_cast<uint32_t*>(ph + t * kPS + j) = hi;
                    *reinterpret_cast<uint32_t*>(pl + t * kPS + j) = low;
                }
            }
            if (!umma::mbar_wait(&s_done, phase & 1u)) lost = true;
            __syncwarp();
            ++phase;
            umma::fence_after_sync();
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < mt) {
                    tmem_ld_frag(tm + ((uint32_t)rows << 16) + kTmO + 16 * i, acc[2 * i], acc[2 * i + 1]);
#pragma unroll
                    for (int n = 2 * i; n < 2 * i + 2; ++n) {
                        const float2 e = *reinterpret_cast<const float2*>(&s_e[8 * n + 2 * c]);
                        acc[n][0] *= e.x, acc[n][1] *= e.y, acc[n][2] *= e.x, acc[n][3] *= e.y;
                    }
                }
            umma::fence_before_sync();
        }
        if (!umma::mbar_wait(&s_v, turn & 1u)) lost = true;
        if (__syncthreads_or(lost)) break;
        if (tid == 192) ask_qk(next);  // their place is free
        if (warp == 7) ask_path(next + gridDim.x);
        if (!padding) {
#pragma unroll 1
            for (int js = 0; js < mt; ++js) {
                uint32_t a[4];
                ldmatrix4_trans(vs + umma::kmaj_off(16 * js + (lane >> 4) * 8 + (lane & 7), rows + (lane >> 3 & 1) * 8, Tp), a);
                // what padding nodes hold must not meet a zero weight as 0 * NaN
                const unsigned use = (unsigned)(used_nodes[turn & 1] >> (16 * js + 2 * c));
                const uint32_t keep = (use & 1 ? 0xffffu : 0u) | (use & 2 ? 0xffff0000u : 0u);
                const uint32_t keep8 = (use & 0x100 ? 0xffffu : 0u) | (use & 0x200 ? 0xffff0000u : 0u);
                a[0] &= keep, a[1] &= keep, a[2] &= keep8, a[3] &= keep8;
                // 16 tokens at a time: their two terms of P as two column blocks of 8 tokens each
                const int at = ((lane >> 4) * 8 + (lane & 7)) * kPS + 16 * js + (lane >> 3 & 1) * 8;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i < mt && i >= js) {
                        uint32_t low[4], high[4];
                        ldmatrix4(pl + 16 * i * kPS + at, low);
                        ldmatrix4(ph + 16 * i * kPS + at, high);
                        mma16816(acc[2 * i], a, low[0], low[1]);
                        mma16816(acc[2 * i + 1], a, low[2], low[3]);
                        mma16816(acc[2 * i], a, high[0], high[1]);
                        mma16816(acc[2 * i + 1], a, high[2], high[3]);
                    }
            }
#pragma unroll
            for (int n = 0; n < 8; ++n)
                if (n < 2 * mt) {
                    // turned by stmatrix: 8 tokens x 8 v, 16 bytes of a token's row each
                    const uint32_t y0 = pack_bf16(p.scale * acc[n][0], p.scale * acc[n][1]);
                    const uint32_t y1 = pack_bf16(p.scale * acc[n][2], p.scale * acc[n][3]);
                    asm volatile("stmatrix.sync.aligned.m8n8.x2.trans.shared.b16 [%0], {%1, %2};" ::"r"(
                                     smem_addr(os + (8 * n + (lane & 7)) * kVS + rows + 8 * (lane >> 3 & 1))),
                                 "r"(y0), "r"(y1)
                                 : "memory");
                }
        }
        __syncthreads();
        if (tid == 192) ask_v(next);
        for (int i = tid; i < T * 16; i += 256) {
            const int t = i >> 4, x = 8 * (i & 15);
            uint4 val = *reinterpret_cast<const uint4*>(os + t * kVS + x);
            if (padding || s_path[t] == 0ull) val = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(out + (size_t)t * p.HV * kDim + x) = val;
        }
        __syncthreads();
    }
    if (__syncthreads_or(lost) && tid == 0) {  // given up: what is in flight gets as long again to end before the CTA does
        umma::mbar_wait(&s_full, phase & 1u);
        umma::mbar_wait(&s_done, phase & 1u);
        umma::mbar_wait(&s_qk, turn & 1u), umma::mbar_wait(&s_qk, ~turn & 1u);
        umma::mbar_wait(&s_v, turn & 1u), umma::mbar_wait(&s_v, ~turn & 1u);
    }
    __syncthreads();
    if (warp == 1) umma::tmem_dealloc(tm, 256);
}

// ---------------------------------------------------------------------------
// Commit: the decode kernel's streaming pass (64 rows of one v-head per CTA, 8
// lanes to a row), with one update for each node of the accepted path.  The
// state's read and write are the traffic (8 or 4 bytes an element); the path
// costs 2 operations an element and node.  Every warp walks the path by itself:
// lanes hold the parents and log decays of two nodes each, and a step is a
// shuffle, so no warp waits for another.  The first walk, while the state is on
// its way, finds the path's decay (and whether it reaches the cached state); the
// second adds the nodes, newest first, with the next two nodes' k and v on their
// way.
//
// 64 entries of 32 heads, fp32 (270 MB): 45 us with one node accepted, 48 with
// four (5.7 TB/s), 57 with nine, 149 with 32, where the steps of a path, one after
// the other, are what it takes; bf16 27, 34, 48 and 129.  With 32 rows a CTA, 45,
// 48, 60 and 175; bf16 27, 35, 56 and 160 (a step's loads and shuffles serve half
// the rows); with 128 rows 46, 52, 64 and 165.  With one node ahead only, 45, 48, 58
// and 163.  With the path's k and v asked into L1 at the first walk, 45, 49, 72 and
// 213 (of 32 rows).  With one thread walking for the CTA and k and v staged in shared
// memory, the two barriers and the longer chain of waits made four nodes 57.
// ---------------------------------------------------------------------------

struct CommitParams {
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    void* pool;
    const void* indices;
    const void* out_indices;
    const int* parents;
    const int* accepted;
    const float* log_decay;
    int idx64, per_token, T, H, HV, rep, pool_size;
};

constexpr int kCommitRows = 64;

template <bool kBf16>
__global__ void __launch_bounds__(128, 4) decay_commit_kernel(const CommitParams p) {
    using Row = StateRow<kBf16>;
    constexpr int kRows = kCommitRows, kPasses = kRows / 16, kBlocks = kDim / kRows;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, sub = lane & 7;
    const int head = blockIdx.x / kBlocks, row = (blockIdx.x % kBlocks) * kRows + warp * (kRows / 4) + (lane >> 3);
    const int b = head / p.HV, h = head % p.HV, hq = h / p.rep, T = p.T;

    const long long slot = slot_at(p.indices, p.idx64, b);
    if (slot < 0 || slot >= p.pool_size) return;
    const long long oslot = p.out_indices ? slot_at(p.out_indices, p.idx64, b) : slot;
    if (oslot < 0 || oslot >= p.pool_size) return;
    const int last = p.accepted[b];
    const bool some = last >= 0 && last < T;
    if (!some && oslot == slot) return;  // nothing accepted, in place

    const size_t srow = ((size_t)slot * p.HV + h) * kDim + row;
    typename Row::Raw raw[kPasses][Row::kRaw];
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) Row::load(p.pool, srow + 4 * ps, sub, raw[ps]);

    // nodes lane and lane + 32; a parent that is not before its node counts as padding
    int par[2] = {-2, -2};
    float g[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = lane + 32 * i;
        if (t < T && (i == 0 || last >= 32)) {
            par[i] = p.parents[(size_t)b * T + t];
            if (par[i] >= t) par[i] = -2;
            g[i] = clamp_log_decay(p.log_decay[p.per_token ? ((size_t)b * T + t) * p.HV + h : h]);
        }
    }
    auto parent_of = [&](int t) {
        const int x = __shfl_sync(0xffffffffu, par[0], t & 31), y = __shfl_sync(0xffffffffu, par[1], t & 31);
        return t < 32 ? x : y;
    };
    auto decay_of = [&](int t) {
        const float x = __shfl_sync(0xffffffffu, g[0], t & 31), y = __shfl_sync(0xffffffffu, g[1], t & 31);
        return t < 32 ? x : y;
    };
    // k and v of the newest two nodes come with the state, those of the others two steps ahead
    uint2 kn[2][4];
    __nv_bfloat16 vn[2][kPasses];
    auto fetch = [&](int t, uint2 (&kk)[4], __nv_bfloat16 (&vv)[kPasses]) {
        if (t < 0) return;
        const __nv_bfloat16* kp = p.k + (((size_t)b * T + t) * p.H + hq) * kDim;
#pragma unroll
        for (int j = 0; j < 4; ++j) kk[j] = *reinterpret_cast<const uint2*>(kp + col_of<kBf16>(sub, j));
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) vv[ps] = p.v[(((size_t)b * T + t) * p.HV + h) * kDim + row + 4 * ps];
    };
    int t = some ? last : -1, ahead = -1;  // the node that is next, and the one after it
    if (some) {
        ahead = parent_of(t);
        fetch(t, kn[0], vn[0]), fetch(ahead, kn[1], vn[1]);
    }
    float all = 0.f;
    int end = some ? last : -2;
    while (end >= 0) {
        all += decay_of(end);
        end = parent_of(end);
    }
    const bool path = some && end == -1;  // else padding lies on the path: nothing is accepted
    if (!path && oslot == slot) return;

    const float a = path ? expf(all) : 1.f;
    float4 s[kPasses][4];
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) {
        Row::widen(raw[ps], s[ps]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[ps][j].x *= a, s[ps][j].y *= a, s[ps][j].z *= a, s[ps][j].w *= a;
    }
    float behind = 0.f;  // log decays of the nodes behind this one
    if (!path) t = -1;
    while (t >= 0) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            if (t < 0) break;
            float2 k[8];
            float2 f[kPasses];
            const float w = expf(behind);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[2 * j] = widen2(kn[u][j].x), k[2 * j + 1] = widen2(kn[u][j].y);
#pragma unroll
            for (int ps = 0; ps < kPasses; ++ps) f[ps].x = f[ps].y = w * bf16_to_f32(vn[u][ps]);
            behind += decay_of(t);
            t = ahead;
            ahead = ahead >= 0 ? parent_of(ahead) : -1;
            fetch(ahead, kn[u], vn[u]);
#pragma unroll
            for (int ps = 0; ps < kPasses; ++ps)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 x = __ffma2_rn(f[ps], k[2 * j], lo2(s[ps][j])), y = __ffma2_rn(f[ps], k[2 * j + 1], hi2(s[ps][j]));
                    s[ps][j] = make_float4(x.x, x.y, y.x, y.y);
                }
        }
    }
    const size_t drow = ((size_t)oslot * p.HV + h) * kDim + row;
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) Row::store(p.pool, drow + 4 * ps, sub, s[ps]);
}

static int check_tree(int state_bf16, int idx64, int per_token, int B, int T, int H, int HV, int K, int V,
                      int pool_size) {
    const int bad = gdn_decay_check_pool(state_bf16, idx64, per_token, B, T, H, HV, K, V, pool_size);
    if (bad) return bad;
    if (T > kTreeMax || (long long)B * HV > (1ll << 27)) return GDN_ERR_UNSUPPORTED;
    return GDN_OK;
}

// The driver's tensor-map encoder, looked up through the runtime once (no
// link-time dependency on the driver library).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn tree_encode_fn() {
    static std::once_flag once;
    static EncodeFn fn = nullptr;
    std::call_once(once, []() {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeFn>(ptr);
    });
    return fn;
}

template <bool kBf16>
static int launch_verify(const VerifyParams& p, const void* pool, cudaStream_t st) {
    // the pool, [states, 128, 128], in boxes of 128 rows x 128 bytes
    const EncodeFn encode = tree_encode_fn();
    if (encode == nullptr) return GDN_ERR_CUDA;
    CUtensorMap map{};
    const cuuint64_t el = kBf16 ? 2 : 4, n = (cuuint64_t)p.pool_size * p.HV;
    const cuuint64_t dims[3] = {(cuuint64_t)kDim, (cuuint64_t)kDim, n}, strides[2] = {kDim * el, kDim * kDim * el};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / el), (cuuint32_t)kDim, 1u}, estr[3] = {1u, 1u, 1u};
    if (encode(&map, kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(pool),
               dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return GDN_ERR_CUDA;
    // q, k and v, [entries * T, heads, 128], in boxes of T nodes x 64
    CUtensorMap m_qkv[3] = {};
    const __nv_bfloat16* from[3] = {p.q, p.k, p.v};
    for (int i = 0; i < 3; ++i) {
        const cuuint64_t heads = i < 2 ? p.H : p.HV;
        const cuuint64_t tdims[3] = {(cuuint64_t)kDim, heads, (cuuint64_t)(p.items / p.HV) * p.T}, tstrides[2] = {kDim * 2, heads * kDim * 2};
        const cuuint32_t tbox[3] = {64u, 1u, (cuuint32_t)p.T};
        if (encode(&m_qkv[i], CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<__nv_bfloat16*>(from[i]), tdims, tstrides, tbox, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return GDN_ERR_CUDA;
    }
    const size_t smem = verify_smem(p.Tp, kBf16);
    static std::atomic<unsigned long long> done{0};  // the kernel's attribute, once per device (again after a failure)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return GDN_ERR_CUDA;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev >= 64 || !(done.load() & bit)) {
        if (cudaFuncSetAttribute(decay_verify_kernel<kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)verify_smem(kTreeMax, kBf16)) != cudaSuccess) {
            cudaGetLastError();
            return GDN_ERR_CUDA;
        }
        if (dev < 64) done.fetch_or(bit);
    }
    const int per_sm = 2 * (smem + 4096) <= 227 * 1024 ? 2 : 1, most = per_sm * 148;
    decay_verify_kernel<kBf16><<<p.items < most ? p.items : most, 256, smem, st>>>(p, map, m_qkv[0], m_qkv[1], m_qkv[2]);
    return gdn_launch_status();
}

static int tree_status_bits(bool clear) {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_status, sizeof(v)) != cudaSuccess) return -1;
    if (clear && v) {
        const unsigned int z = 0;
        if (cudaMemcpyToSymbol(g_device_status, &z, sizeof(z)) != cudaSuccess) return -1;
    }
    return (int)v;
}

}  // namespace decay

int decay_tree_status(bool clear) { return decay::tree_status_bits(clear); }

}  // namespace gdn

extern "C" int gdn_decay_verify_fwd(const void* q, const void* k, const void* v, const void* pool, int state_bf16,
                                    const void* indices, int indices_int64, const int* parents, const float* log_decay,
                                    int decay_per_token, float scale, int B, int T, int H, int HV, int K, int V,
                                    int pool_size, void* out, void* stream) {
    using namespace gdn::decay;
    const int bad = check_tree(state_bf16, indices_int64, decay_per_token, B, T, H, HV, K, V, pool_size);
    if (bad) return bad;
    if ((long long)pool_size * HV > 0x7fffffffll) return GDN_ERR_UNSUPPORTED;  // state number
    if (B == 0 || T == 0) return GDN_OK;
    if (!q || !k || !v || (!pool && pool_size > 0) || !indices || !parents || !log_decay || !out) return GDN_ERR_INVALID;
    if (!gdn_aligned(q, 16) || !gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(out, 16) ||
        !gdn_aligned(pool, 16) || !gdn_aligned(log_decay, 4) || !gdn_aligned(parents, 4) ||
        !gdn_aligned(indices, indices_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    if (pool_size == 0)  // every entry is padding, and there is no state to make a tensor map of
        return cudaMemsetAsync(out, 0, (size_t)B * T * HV * gdn::kDim * 2, static_cast<cudaStream_t>(stream)) == cudaSuccess
                   ? GDN_OK
                   : GDN_ERR_CUDA;
    VerifyParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.v = static_cast<const __nv_bfloat16*>(v);
    p.indices = indices;
    p.parents = parents;
    p.log_decay = log_decay;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.scale = scale == 0.0f ? 1.0f / sqrtf((float)K) : scale;
    p.idx64 = indices_int64;
    p.per_token = decay_per_token;
    p.T = T;
    p.Tp = (T + 15) / 16 * 16;
    p.H = H;
    p.HV = HV;
    p.rep = HV / H;
    p.pool_size = pool_size;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    p.items = B * HV;
    return state_bf16 ? launch_verify<true>(p, pool, st) : launch_verify<false>(p, pool, st);
}

extern "C" int gdn_decay_commit(const void* k, const void* v, void* pool, int state_bf16, const void* indices,
                                const void* out_indices, int indices_int64, const int* parents, const int* accepted,
                                const float* log_decay, int decay_per_token, int B, int T, int H, int HV, int K, int V,
                                int pool_size, void* stream) {
    using namespace gdn::decay;
    const int bad = check_tree(state_bf16, indices_int64, decay_per_token, B, T, H, HV, K, V, pool_size);
    if (bad) return bad;
    if (B == 0) return GDN_OK;
    if ((!pool && pool_size > 0) || !indices || !accepted || (T > 0 && (!k || !v || !parents || !log_decay))) return GDN_ERR_INVALID;
    if (!gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(pool, 16) || !gdn_aligned(log_decay, 4) ||
        !gdn_aligned(parents, 4) || !gdn_aligned(accepted, 4) || !gdn_aligned(indices, indices_int64 ? 8 : 4) ||
        !gdn_aligned(out_indices, indices_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    if (pool_size == 0) return GDN_OK;  // every entry is padding
    CommitParams p;
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.v = static_cast<const __nv_bfloat16*>(v);
    p.pool = pool;
    p.indices = indices;
    p.out_indices = out_indices;
    p.parents = parents;
    p.accepted = accepted;
    p.log_decay = log_decay;
    p.idx64 = indices_int64;
    p.per_token = decay_per_token;
    p.T = T;
    p.H = H;
    p.HV = HV;
    p.rep = HV / H;
    p.pool_size = pool_size;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const unsigned grid = (unsigned)((long long)B * HV * (gdn::kDim / kCommitRows));
    if (state_bf16)
        decay_commit_kernel<true><<<grid, 128, 0, st>>>(p);
    else
        decay_commit_kernel<false><<<grid, 128, 0, st>>>(p);
    return gdn_launch_status();
}

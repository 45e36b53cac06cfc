// decay_tree.cu — linear attention with a decay per head for trees of drafted
// tokens over pooled states, and the update by the accepted path (sm_100a).
//
// With c_t the sum of the log decays on node t's path from the cached state S
// (node t included) and j <= t meaning "j is on node t's path":
//   o_t = scale * ( e^{c_t} S q_t + sum_{j <= t} e^{c_t - c_j} (q_t . k_j) v_j )
//   S'  = e^{c_a} S + sum_{j <= a} e^{c_a - c_j} v_j k_j^T      (a: accepted)
#include "decay_common.cuh"

namespace gdn {
namespace decay {

constexpr int kTreeMax = GDN_DECAY_TREE_MAX;

// ---------------------------------------------------------------------------
// Verification: one CTA per entry and v-head, 8 warps of 16 state rows each.
//
// The state (64 KiB in fp32) is the traffic: it is read once, straight into
// the A fragments of warp-level matrix products, o^T[v, t] = S[v, :] . q_t,
// and q, k, v of the tree (3 T KiB / 4) come through shared memory.  At T = 64 the
// products are 4.7 M multiply-adds a state (two for each of S q's, S being
// split as below), about as long on the warp-level tensor path as the state's
// 64 KiB take from HBM; below that HBM bounds the kernel.  tcgen05 would need
// the state staged in shared or tensor memory first and a 512-column CTA per
// SM, for products of at most 64 columns.
//
// Precision: q, k, v are bf16 as given.  An fp32 state is split into two bf16
// terms (hi + lo, off by at most 2^-17 of it) and the decayed scores P likewise,
// so the products lose nothing next to the output's own rounding to bf16 (2^-8);
// one bf16 term each would about double the output's error.
//
// Fragment layout: the contraction index may be permuted in both operands
// alike, so that a lane's four k-slots {2c, 2c+1, 2c+8, 2c+9} of a 16-step hold
// columns 4c..4c+3: the state comes by 16-byte (fp32) loads and q and k by 8-byte
// loads from rows 288 bytes apart (no bank conflict).
// ---------------------------------------------------------------------------

struct VerifyParams {
    const __nv_bfloat16* q;
    const __nv_bfloat16* k;
    const __nv_bfloat16* v;
    const void* pool;
    const void* indices;
    const int* parents;
    const float* log_decay;
    __nv_bfloat16* out;
    float scale;
    int idx64, per_token, T, Tp, H, HV, rep, pool_size;  // Tp: T rounded up to 16
};

constexpr int kQS = 144, kVS = 136, kPS = 72;  // row strides in bf16 elements

__host__ __device__ constexpr size_t verify_smem(int Tp) {
    return (size_t)Tp * 2 * (2 * kQS + kVS + 2 * kPS);
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
__device__ __forceinline__ void cp_async16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(dst)), "l"(src) : "memory");
}

// hi + lo split of a pair: hi = bf16(x), lo = bf16(x - hi).  A value that bf16
// rounds to infinity, or that is not finite, keeps lo = 0 (inf - inf is NaN).
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16(x, y);
    const float2 h = widen2(hi);
    const float rx = isinf(h.x) ? 0.f : x - h.x, ry = isinf(h.y) ? 0.f : y - h.y;
    lo = pack_bf16(rx, ry);
}

template <bool kBf16>
__global__ void __launch_bounds__(256, 2) decay_verify_kernel(const VerifyParams p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    __shared__ unsigned long long s_path[kTreeMax];  // bit j: j is on the node's path; 0: padding
    __shared__ float s_c[kTreeMax], s_e[kTreeMax];   // c_t and e^{c_t}
    __shared__ int s_up[kTreeMax];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int b = blockIdx.x / p.HV, h = blockIdx.x % p.HV, hq = h / p.rep, T = p.T, Tp = p.Tp;
    const size_t row_out = ((size_t)b * T * p.HV + h) * kDim;  // + t * HV * 128

    const long long slot = slot_at(p.indices, p.idx64, b);
    if (slot < 0 || slot >= p.pool_size) {
        for (int i = tid; i < T * 16; i += 256)
            *reinterpret_cast<uint4*>(p.out + row_out + (size_t)(i >> 4) * p.HV * kDim + 8 * (i & 15)) =
                make_uint4(0, 0, 0, 0);
        return;
    }

    // the state, first: rows g and g + 8 of this warp's 16, columns 16 ks + 4 c + {0..3}
    const size_t srow = ((size_t)slot * p.HV + h) * kDim + 16 * warp + g;
    float4 sf[kBf16 ? 1 : 8][2];
    uint2 sb[kBf16 ? 8 : 1][2];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const size_t at = (srow + 8 * r) * kDim + 16 * ks + 4 * c;
            if (kBf16)
                sb[ks][r] = __ldcs(reinterpret_cast<const uint2*>(static_cast<const __nv_bfloat16*>(p.pool) + at));
            else
                sf[ks][r] = __ldcs(reinterpret_cast<const float4*>(static_cast<const float*>(p.pool) + at));
        }

    __nv_bfloat16* qs = reinterpret_cast<__nv_bfloat16*>(smem_raw);
    __nv_bfloat16* ks_ = qs + Tp * kQS;
    __nv_bfloat16* vs = ks_ + Tp * kQS;
    __nv_bfloat16* ph = vs + Tp * kVS;
    __nv_bfloat16* pl = ph + Tp * kPS;
    for (int i = tid; i < Tp * 16; i += 256) {
        const int t = i >> 4, x = 8 * (i & 15);
        if (t < T) {
            const size_t qk = (((size_t)b * T + t) * p.H + hq) * kDim + x;
            cp_async16(qs + t * kQS + x, p.q + qk);
            cp_async16(ks_ + t * kQS + x, p.k + qk);
            cp_async16(vs + t * kVS + x, p.v + row_out + (size_t)t * p.HV * kDim + x);
        } else {
            *reinterpret_cast<uint4*>(qs + t * kQS + x) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(ks_ + t * kQS + x) = make_uint4(0, 0, 0, 0);
        }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");

    // Paths and their decays by pointer doubling: after r rounds a node knows the
    // last 2^r nodes of its path; -1 ends a path, -2 marks padding.
    if (warp == 0) {
        unsigned long long m[2];
        float cc[2];
        int up[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = lane + 32 * i;
            up[i] = -2, cc[i] = 0.f, m[i] = 0ull;
            if (t < T) {
                const int par = p.parents[(size_t)b * T + t];
                up[i] = par < -1 || par >= t ? -2 : par;
                cc[i] = clamp_log_decay(p.log_decay[p.per_token ? ((size_t)b * T + t) * p.HV + h : h]);
                m[i] = 1ull << t;
            }
            s_up[t] = up[i], s_c[t] = cc[i], s_path[t] = m[i];
        }
        __syncwarp();
        for (int hop = 1; hop < T; hop *= 2) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
                if (up[i] >= 0) {
                    const int u = up[i];
                    cc[i] += s_c[u], m[i] |= s_path[u], up[i] = s_up[u];
                }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 2; ++i) s_up[lane + 32 * i] = up[i], s_c[lane + 32 * i] = cc[i], s_path[lane + 32 * i] = m[i];
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (up[i] != -1) s_path[lane + 32 * i] = 0ull;
            s_e[lane + 32 * i] = expf(cc[i]);
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();

    // what padding nodes hold must not meet a zero weight as 0 * NaN
    for (int i = tid; i < Tp * 16; i += 256)
        if (s_path[i >> 4] == 0ull) *reinterpret_cast<uint4*>(vs + (i >> 4) * kVS + 8 * (i & 15)) = make_uint4(0, 0, 0, 0);

    // P[t, j] = e^{c_t - c_j} (q_t . k_j) on the paths, 0 elsewhere; nodes come after
    // their parents, so 16 x 8 tiles with every j > t stay out (they are not read either)
    const int mt = Tp / 16;
    for (int tile = warp; tile < mt * (mt + 1); tile += 8) {
        int m = 0, n = tile;  // row block m has 2 (m + 1) column tiles
        while (n >= 2 * (m + 1)) n -= 2 * (m + 1), ++m;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
            const uint2 a0 = *reinterpret_cast<const uint2*>(qs + (16 * m + g) * kQS + 16 * ks + 4 * c);
            const uint2 a1 = *reinterpret_cast<const uint2*>(qs + (16 * m + g + 8) * kQS + 16 * ks + 4 * c);
            const uint2 bb = *reinterpret_cast<const uint2*>(ks_ + (8 * n + g) * kQS + 16 * ks + 4 * c);
            const uint32_t a[4] = {a0.x, a1.x, a0.y, a1.y};
            mma16816(acc, a, bb.x, bb.y);
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int t = 16 * m + g + 8 * r, j = 8 * n + 2 * c;
            const unsigned long long path = s_path[t];
            const float x = path >> j & 1 ? acc[2 * r] * expf(s_c[t] - s_c[j]) : 0.f;
            const float y = path >> (j + 1) & 1 ? acc[2 * r + 1] * expf(s_c[t] - s_c[j + 1]) : 0.f;
            uint32_t hi, lo;
            split2(x, y, hi, lo);
            *reinterpret_cast<uint32_t*>(ph + t * kPS + j) = hi;
            *reinterpret_cast<uint32_t*>(pl + t * kPS + j) = lo;
        }
    }
    __syncthreads();

    uint32_t shi[8][4], slo[kBf16 ? 1 : 8][4];
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
        if (kBf16) {
            shi[ks][0] = sb[ks][0].x, shi[ks][1] = sb[ks][1].x, shi[ks][2] = sb[ks][0].y, shi[ks][3] = sb[ks][1].y;
        } else {
            split2(sf[ks][0].x, sf[ks][0].y, shi[ks][0], slo[ks][0]);
            split2(sf[ks][1].x, sf[ks][1].y, shi[ks][1], slo[ks][1]);
            split2(sf[ks][0].z, sf[ks][0].w, shi[ks][2], slo[ks][2]);
            split2(sf[ks][1].z, sf[ks][1].w, shi[ks][3], slo[ks][3]);
        }
    }
    // o^T rows 16 warp + {g, g + 8}, columns 8 n + 2 c + {0, 1}, two column tiles at a time
    float o[4][2][4];  // [pair of tiles][tile][fragment]
    for (int np = 0; np < mt; ++np) {
        float hi[2][4], lo[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) hi[i][e] = lo[i][e] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint2 bb = *reinterpret_cast<const uint2*>(qs + (16 * np + 8 * i + g) * kQS + 16 * ks + 4 * c);
                mma16816(hi[i], shi[ks], bb.x, bb.y);
                if (!kBf16) mma16816(lo[i], slo[ks], bb.x, bb.y);
            }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float e0 = s_e[16 * np + 8 * i + 2 * c], e1 = s_e[16 * np + 8 * i + 2 * c + 1];
            hi[i][0] = (hi[i][0] + lo[i][0]) * e0, hi[i][1] = (hi[i][1] + lo[i][1]) * e1;
            hi[i][2] = (hi[i][2] + lo[i][2]) * e0, hi[i][3] = (hi[i][3] + lo[i][3]) * e1;
        }
        for (int js = 0; js <= np; ++js) {
            uint32_t a[4];
            const __nv_bfloat16* src =
                vs + (16 * js + (lane >> 4) * 8 + (lane & 7)) * kVS + 16 * warp + (lane >> 3 & 1) * 8;
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                         : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
                         : "r"(smem_addr(src)));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int at = (16 * np + 8 * i + g) * kPS + 16 * js + 2 * c;
                const uint32_t* h0 = reinterpret_cast<const uint32_t*>(ph + at);
                const uint32_t* l0 = reinterpret_cast<const uint32_t*>(pl + at);
                mma16816(hi[i], a, h0[0], h0[4]);
                mma16816(hi[i], a, l0[0], l0[4]);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (k == np)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[k][i][e] = hi[i][e] * p.scale;
    }
    // turned through shared memory (q's place) so that a token's row leaves in 16-byte stores
    __syncthreads();
#pragma unroll
    for (int np = 0; np < 4; ++np)
        if (np < mt)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    qs[(16 * np + 8 * i + 2 * c + (e & 1)) * kVS + 16 * warp + g + 8 * (e >> 1)] =
                        __float2bfloat16_rn(o[np][i][e]);
    __syncthreads();
    for (int i = tid; i < T * 16; i += 256) {
        const int t = i >> 4, x = 8 * (i & 15);
        uint4 val = *reinterpret_cast<const uint4*>(qs + t * kVS + x);
        if (s_path[t] == 0ull) val = make_uint4(0, 0, 0, 0);
        *reinterpret_cast<uint4*>(p.out + row_out + (size_t)t * p.HV * kDim + x) = val;
    }
}

// ---------------------------------------------------------------------------
// Commit: the decode kernel's streaming pass (32 rows of one v-head per CTA, 8
// lanes to a row), with one update for each node of the accepted path.  The
// state's read and write are the traffic (8 or 4 bytes an element); the path
// costs 2 operations an element and node.  Every warp walks the path by itself:
// lanes hold the parents and log decays of two nodes each, and a step is a
// shuffle, so no warp waits for another.  The first walk, while the state is on
// its way, finds the path's decay (and whether it reaches the cached state); the
// second adds the nodes, newest first, with the next node's k and v on their way.
// (With one thread walking for the CTA and k and v staged in shared memory, two
// barriers and the longer chain of waits made the 64-entry commit 57 us, not 45.)
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

template <bool kBf16>
__global__ void __launch_bounds__(128) decay_commit_kernel(const CommitParams p) {
    using Row = StateRow<kBf16>;
    constexpr int kRows = 32, kPasses = kRows / 16, kBlocks = kDim / kRows;
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
    float all = 0.f;
    int end = some ? last : -2;
    while (end >= 0) {
        all += decay_of(end);
        end = parent_of(end);
    }
    const bool path = some && end == -1;  // else padding lies on the path: nothing is accepted
    if (!path && oslot == slot) return;

    uint2 kn[4];
    float vn[kPasses];
    auto fetch = [&](int t) {
        const __nv_bfloat16* kk = p.k + (((size_t)b * T + t) * p.H + hq) * kDim;
#pragma unroll
        for (int j = 0; j < 4; ++j) kn[j] = *reinterpret_cast<const uint2*>(kk + col_of<kBf16>(sub, j));
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) vn[ps] = bf16_to_f32(p.v[(((size_t)b * T + t) * p.HV + h) * kDim + row + 4 * ps]);
    };
    if (path) fetch(last);
    const float a = path ? expf(all) : 1.f;
    float4 s[kPasses][4];
#pragma unroll
    for (int ps = 0; ps < kPasses; ++ps) {
        Row::widen(raw[ps], s[ps]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[ps][j].x *= a, s[ps][j].y *= a, s[ps][j].z *= a, s[ps][j].w *= a;
    }
    float behind = 0.f;  // log decays of the nodes behind this one
    for (int t = path ? last : -1; t >= 0;) {
        float2 k[8];
        float2 f[kPasses];
        const float w = expf(behind);
#pragma unroll
        for (int j = 0; j < 4; ++j) k[2 * j] = widen2(kn[j].x), k[2 * j + 1] = widen2(kn[j].y);
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps) f[ps] = make_float2(w * vn[ps], w * vn[ps]);
        behind += decay_of(t);
        t = parent_of(t);
        if (t >= 0) fetch(t);
#pragma unroll
        for (int ps = 0; ps < kPasses; ++ps)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 x = __ffma2_rn(f[ps], k[2 * j], lo2(s[ps][j])), y = __ffma2_rn(f[ps], k[2 * j + 1], hi2(s[ps][j]));
                s[ps][j] = make_float4(x.x, x.y, y.x, y.y);
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

template <bool kBf16>
static int launch_verify(const VerifyParams& p, int B, cudaStream_t st) {
    const size_t smem = verify_smem(p.Tp);
    // above 48 KiB with the kernel's static arrays: set on each such call, for the current device
    if (smem > 40 * 1024 &&
        cudaFuncSetAttribute(decay_verify_kernel<kBf16>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             (int)verify_smem(kTreeMax)) != cudaSuccess) {
        cudaGetLastError();
        return GDN_ERR_CUDA;
    }
    decay_verify_kernel<kBf16><<<(unsigned)(B * p.HV), 256, smem, st>>>(p);
    return gdn_launch_status();
}

}  // namespace decay
}  // namespace gdn

extern "C" int gdn_decay_verify_fwd(const void* q, const void* k, const void* v, const void* pool, int state_bf16,
                                    const void* indices, int indices_int64, const int* parents, const float* log_decay,
                                    int decay_per_token, float scale, int B, int T, int H, int HV, int K, int V,
                                    int pool_size, void* out, void* stream) {
    using namespace gdn::decay;
    const int bad = check_tree(state_bf16, indices_int64, decay_per_token, B, T, H, HV, K, V, pool_size);
    if (bad) return bad;
    if (B == 0 || T == 0) return GDN_OK;
    if (!q || !k || !v || !pool || !indices || !parents || !log_decay || !out) return GDN_ERR_INVALID;
    if (!gdn_aligned(q, 16) || !gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(out, 16) ||
        !gdn_aligned(pool, 16) || !gdn_aligned(log_decay, 4) || !gdn_aligned(parents, 4) ||
        !gdn_aligned(indices, indices_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    VerifyParams p;
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.k = static_cast<const __nv_bfloat16*>(k);
    p.v = static_cast<const __nv_bfloat16*>(v);
    p.pool = pool;
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
    return state_bf16 ? launch_verify<true>(p, B, st) : launch_verify<false>(p, B, st);
}

extern "C" int gdn_decay_commit(const void* k, const void* v, void* pool, int state_bf16, const void* indices,
                                const void* out_indices, int indices_int64, const int* parents, const int* accepted,
                                const float* log_decay, int decay_per_token, int B, int T, int H, int HV, int K, int V,
                                int pool_size, void* stream) {
    using namespace gdn::decay;
    const int bad = check_tree(state_bf16, indices_int64, decay_per_token, B, T, H, HV, K, V, pool_size);
    if (bad) return bad;
    if (B == 0) return GDN_OK;
    if (!pool || !indices || !accepted || !log_decay || (T > 0 && (!k || !v || !parents))) return GDN_ERR_INVALID;
    if (!gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(pool, 16) || !gdn_aligned(log_decay, 4) ||
        !gdn_aligned(parents, 4) || !gdn_aligned(accepted, 4) || !gdn_aligned(indices, indices_int64 ? 8 : 4) ||
        !gdn_aligned(out_indices, indices_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
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
    const unsigned grid = (unsigned)((long long)B * HV * 4);
    if (state_bf16)
        decay_commit_kernel<true><<<grid, 128, 0, st>>>(p);
    else
        decay_commit_kernel<false><<<grid, 128, 0, st>>>(p);
    return gdn_launch_status();
}

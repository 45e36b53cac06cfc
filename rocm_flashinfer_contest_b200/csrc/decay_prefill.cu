// decay_prefill.cu — prefill of packed prompts for linear attention with a
// decay per head (sm_100a).
//
// Over a chunk of 64 tokens with log decays g, c_i = g_0 + .. + g_i, and the
// state S [V, K] before it:
//   o_i = scale * ( e^{c_i} S q_i  +  sum_{j <= i} e^{c_i - c_j} (q_i . k_j) v_j )
//   S'  = e^{c_63} S + sum_j v_j (w_j k_j)^T,     w_j = e^{c_63 - c_j}
//
// A CTA walks the chunks of segments: up to seg_len tokens of one sequence, for
// one v-head.  Long sequences are cut into segments so that 148 CTAs have work,
// and these run in two launches of the same kernel: the first takes every
// segment that another one follows, a sequence's first segment from its state
// (and is done with it), the others from a zero state, for what they add to the
// state (their outputs are dropped); a small kernel turns that into the state
// before each segment; the second launch takes the segments that are not a
// sequence's first.  With n segments the work is 2 (n - 1) / n of one pass, on
// n - 1 times as many CTAs.  Sequences of one segment run in the second launch,
// which is the only one of a call whose T fits a segment.
//
// Products, all on tcgen05 with fp32 accumulators in tensor memory:
//   U   [v, k] = (V w)^T K      A: in tensor memory, B: K tile (MN-major)
//   P   [i, j] = Q K^T          rows 64..127 of the M = 128 tile are not used
//   O2^T[v, i] = S Q^T          A: S (bf16) in tensor memory, B: Q tile
//   O1^T[v, i] = V^T P^T        A: V^T in tensor memory, B: decayed P (bf16)
// Tiles arrive token-major by TMA.  V is turned once, by 8 x 8 matrices in
// registers, and the weights w are put on it there: as an operand in tensor memory
// it costs shared memory no bandwidth, and K's tile stays as it came.
//
// Precision: inputs are bf16.  V w is split into three bf16 terms of 8 bits each
// (exact), so the fp32 state loses nothing beside its accumulation: 8e-8 of it
// measured, where two terms would give 3e-6.  S and P only meet the output, which
// is rounded to bf16 itself; they are rounded to bf16 once each, one for each of
// the output's two parts, so the output's error is sqrt(2) times that of the last
// rounding alone (measured 0.0023 against 0.0017 of the output; second terms
// bring it to 0.0017 and cost 12 more products and 1,000 more instructions a
// chunk).  It is bounded by 2^-8 of scale (|S| |q| + |P| |v|), so an output that
// cancels loses more of itself.  Sums of log decays are exact to 2^-28
// (split_log2_decay).
//
// Measured: 8,192 tokens of 32 v-heads and 16 q/k heads 92 us (its 205 MB alone
// take 31; called without a pause the GPU reaches its 1,000 W and lowers its clock
// from 1.97 to 1.6 GHz: 104 to 107), a chunk every 2,400 cycles in each CTA.  The chunk's
// 32 products alone take 1,540, issued without a pause and in turn (at the pipe's
// full rate 1,408); those that add to one accumulator with N = 64 follow each other
// at 80 cycles, so 12 for an output are 700 from the first to the end.  The rest are
// three loops of nearly the same length, which share issue slots, shared memory and
// the pipe: U's sums into S, S to bf16, S q, the next S; U, V's terms into the place
// that it leaves, the next U; outputs out of the accumulators, the next output's
// products.
// 61 prompts of 1 to 640 tokens (82 on average), 32 v-heads: 108 us, for two
// reasons.  States (64 KiB in and 64 KiB out a prompt and head) are read and written
// one after the other: in a segment of one chunk 4,700 of 8,500 cycles are the wait
// for its start state, 7 us in all for its rows lying 512 bytes apart in a warp's
// loads.  And a CTA has every 148th segment, whatever their lengths: the busiest has
// 36 chunks, the mean is 24.6.
// 13 prompts of 7 to 3,353 tokens, 8 v-heads: 62 us.  Two launches of 96 and 152
// segments on 148 SMs: 1.3 passes over the chunks, but the busiest CTAs have 14 and
// 14 chunks, 34 us, where the means are 9.1 and 9.6; the rest are the two launches'
// starts and ends and the kernel between them.
//
// Tried and not kept, at the first two (91 and 106.5 us then): K scaled instead of
// V, in shared memory (97 and 117 us); that with its lower terms double-buffered (104); V turned by the state
// warps (100 and 117) or by the output warps (111 and 117); scaling unrolled (96 and
// 113); eight output warps (91 and 109); all of V's terms made before the place is
// free (92 and 108); an output's two chains of products issued in turn (92 and 108);
// the next state by TMA into the place that the last one leaves (95 and 120, from 96
// and 118 then); leaving out what only the dropped outputs need, in the first launch
// (101 without a pause, but 112, and ragged prompts 61.5 from 60, as every chunk then
// asks); that as a kernel of its own, with all outputs in the second launch (109, 115
// and 77).
#include <cuda.h>

#include <atomic>
#include <mutex>

#include "decay_common.cuh"
#include "umma.cuh"

namespace gdn {
namespace decay {

using namespace umma;

constexpr int C = 64;                // tokens per chunk
constexpr uint32_t kTile = C * 256;  // bytes of a [64][128] bf16 tile
constexpr int kSms = 148;

struct PrefillParams {
    const float* state;  // nullable: zero
    const float* log_decay;
    const void* cu;
    __nv_bfloat16* out;
    float* new_state;
    float* ws_state;  // [ws slots][HV][V][K]: the state before a segment (after the first launch: what its
                      // predecessor adds to it)
    float* ws_decay;  // [ws slots][HV]: e^(sum of the predecessor's log decays)
    float scale;
    int cu64, per_token, N, T, HV, rep, seg_len, ws_slots;
    int first;  // the first of the two launches
};

__device__ __forceinline__ int cu_at(const void* cu, int is64, int i, int T) {
    const long long x = is64 ? static_cast<const long long*>(cu)[i] : (long long)static_cast<const int*>(cu)[i];
    return (int)(x < 0 ? 0 : x > T ? T : x);
}

// Segments of a launch in order of their sequences, found by one warp that asks
// for ascending numbers: it keeps the block of 32 sequences where it last
// looked and what came before it.
struct Finder {
    int base = 0, before = 0, ws = 0;
};

// A segment: tokens [t0, t1) of sequence n, number s of nseg, and the workspace
// slot of the sequence's first segment (sequences of one segment have none).
struct Item {
    int n, s, nseg, t0, t1, ws;
};

__device__ __forceinline__ int n_segments(const PrefillParams& p, int n, int& t0, int& len) {
    t0 = cu_at(p.cu, p.cu64, n, p.T);
    const int t1 = cu_at(p.cu, p.cu64, n + 1, p.T);
    len = t1 > t0 ? t1 - t0 : 0;
    return len > p.seg_len ? (len + p.seg_len - 1) / p.seg_len : 1;
}

// The launch's segment number `slot`; n = N: there is none.  Malformed
// cu_seqlens can make sequences overlap; segments whose workspace slots would
// lie past the end are then left out.
__device__ __forceinline__ Item find_item(const PrefillParams& p, Finder& f, int slot) {
    const int lane = threadIdx.x & 31;
    Item it{p.N, 0, 0, 0, 0, 0};
#pragma unroll 1
    for (; f.base < p.N; f.base += 32) {
        int t0 = 0, len = 0, nseg = 0;
        if (f.base + lane < p.N) nseg = n_segments(p, f.base + lane, t0, len);
        const int wcnt = nseg > 1 ? nseg : 0, cnt = nseg > 1 ? nseg - 1 : p.first ? 0 : nseg;
        int cs = cnt, wsum = wcnt;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, cs, d), y = __shfl_up_sync(0xffffffffu, wsum, d);
            if (lane >= d) cs += x, wsum += y;
        }
        const unsigned who = __ballot_sync(0xffffffffu, slot >= f.before + cs - cnt && slot < f.before + cs);
        if (who) {
            const int src = __ffs(who) - 1;
            it.n = f.base + src;
            it.nseg = __shfl_sync(0xffffffffu, nseg, src);
            it.s = slot - (f.before + __shfl_sync(0xffffffffu, cs - cnt, src)) + (!p.first && it.nseg > 1);
            it.ws = f.ws + __shfl_sync(0xffffffffu, wsum - wcnt, src);
            t0 = __shfl_sync(0xffffffffu, t0, src), len = __shfl_sync(0xffffffffu, len, src);
            it.t0 = t0 + it.s * p.seg_len;
            it.t1 = min(t0 + len, it.t0 + p.seg_len);
            if (it.nseg > 1 && it.ws + it.nseg > p.ws_slots) it.n = p.N;
            return it;
        }
        f.before += __shfl_sync(0xffffffffu, cs, 31);
        f.ws += __shfl_sync(0xffffffffu, wsum, 31);
    }
    return it;
}

// ---------------------------------------------------------------------------
// The kernel: one CTA per SM, walking the chunks of segment after segment
// without a break (a segment without tokens is one chunk without tokens).  Each
// chunk goes through all of its warps:
//   warps  0..7       state: half a row of S each thread, fp32, in registers
//   warps  8..15      V^T, and V^T w in three bf16 terms: 32 v and 32 tokens each warp
//   warps 16..19      outputs: 32 v each warp, turned on the way to shared memory, rows sent by TMA
//   warps 20, 21, 25  decayed scores: one row i each thread, 32 columns j
//   warp  22          TMA loads
//   warps 23, 27      one thread each that issues the products
//   warp  24          gates, and what the chunk belongs to
//   warp  26          finished states on their way out
// (a warp reads the 32 tensor-memory lanes of its number modulo 4, hence 25).
// ---------------------------------------------------------------------------

constexpr int kThreads = 28 * 32;
// Registers per thread by warpgroup; 256 * (104 + 64) + 128 * (72 + 48 + 48) is
// the 896 * 72 the CTA is launched with.
constexpr int kRegsState = 104, kRegsScale = 64, kRegsOut = 72, kRegsRest = 48;
static_assert(256 * (kRegsState + kRegsScale) + 128 * (kRegsOut + 2 * kRegsRest) <= kThreads * 72, "register split");

// Shared memory, in bytes from its start.
struct L {
    static constexpr int kStages = 3;
    static constexpr int kGates = kStages + 2;  // gates outlive their tiles (read by the state and output warps)
    static constexpr uint32_t kStage = 3 * kTile, oK = kTile, oV = 2 * kTile;  // a stage: q, k, v
    static constexpr uint32_t ps = kStages * kStage;  // two buffers of P
    static constexpr uint32_t kP = C * C * 2;
    static constexpr uint32_t os = ps + 2 * kP;       // two buffers of a chunk's outputs, [token][v]
    static constexpr uint32_t tail = os + 2 * kTile;  // 24 KiB of a state on its way out
    static constexpr uint32_t gates = tail + 24 * 1024;
    static constexpr uint32_t kGate = 1088;
    static constexpr uint32_t bars = gates + kGates * kGate;
    static constexpr uint32_t total = bars + 320;
};
static_assert(L::total <= 227 * 1024, "shared memory");

enum : int { kLast = 1, kFinal = 2 };

// What a chunk's warps need to know of it.
struct Gate {
    float minus[C];  // the first part of c_i / ln 2 (split_log2_decay), negated
    float near[C];   // 2^-(the second part)
    float e[C];   // scale * e^{c_i}
    float w[C];   // e^{c_63 - c_i}
    float a;      // e^{c_63}
    int flags;    // last chunk of its segment, last chunk of this CTA
    int t, live;  // first token; tokens of the segment from there on, at most 64
    int rows;     // rows of output to write: live, or none
    int h;
    const float* src;  // first chunk: the state before it (null: zero)
    int out;           // last chunk: where the state after it goes: a number in the workspace (first launch) or in
                       // new_state, or nowhere (-1)
    int decay;         // last chunk: the number in the workspace where the segment's decay goes, or -1
};
static_assert(sizeof(Gate) <= L::kGate, "gate slot");

struct Bars {
    uint64_t full[3], empty[3], pv_done[2], qk_full[2], u_full[2], u_free, p_read, p_ready[2], p_free[2], v_ready[2], s_ready, s_free,
        o_full, o_free, st_full, st_free, drain[2];
    uint32_t tmem;
    volatile int abort;
    int none;
    int st_out, st_m, st_final;  // for the store warp: the state's number, its last chunk, no more to come
};
static_assert(sizeof(Bars) <= 320, "barrier block");

// Bounded wait: false once it has run out (2^30 cycles, about half a second; the
// CTA is then given up).  Kept short: the warps run some 25 waits, and
// instructions that do not fit the instruction cache cost more than anything else
// here (64 KiB of them: 2.7 warps a scheduler waited for instructions at any time,
// 104 us at 8,192 tokens; 56 KiB, mostly by shorter waits: 0.5 warps, 98 us).
__device__ __forceinline__ bool wait_one(Bars& B, uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 t0, t;\n\t"
        "mov.u32 t0, %%clock;\n"
        "AGAIN:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "@p bra DONE;\n\t"
        "mov.u32 t, %%clock;\n\t"
        "sub.u32 t, t, t0;\n\t"
        "setp.lt.u32 q, t, 0x40000000;\n\t"
        "@q bra AGAIN;\n"
        "DONE:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity & 1u)
        : "memory");
    if (!ok) B.abort = 1;
    return ok != 0;
}
// The same for a whole warp, which goes on together.
__device__ __forceinline__ bool wait_bar(Bars& B, uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, wait_one(B, bar, parity));
}
// Waits for one, and says in `too` whether another one's phase is over as well.
__device__ __forceinline__ bool wait_and_test(Bars& B, uint64_t* bar, uint32_t parity, uint64_t* bar2, uint32_t parity2, bool& too) {
    const bool ok = wait_one(B, bar, parity);
    uint32_t over;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(over)
                 : "r"(smem_u32(bar2)), "r"(parity2 & 1u)
                 : "memory");
    too = __all_sync(0xffffffffu, over != 0);
    return __all_sync(0xffffffffu, ok);
}
// Both of two: a wait takes some 100 cycles where there is nothing to wait for, two at once hardly more.
__device__ __forceinline__ bool wait_two(Bars& B, uint64_t* bar, uint32_t parity, uint64_t* bar2, uint32_t parity2) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .u32 t0, t;\n\t"
        "mov.u32 t0, %%clock;\n"
        "AGAIN:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 q, [%3], %4;\n\t"
        "and.pred p, p, q;\n\t"
        "@p bra DONE;\n\t"
        "mov.u32 t, %%clock;\n\t"
        "sub.u32 t, t, t0;\n\t"
        "setp.lt.u32 q, t, 0x40000000;\n\t"
        "@q bra AGAIN;\n"
        "DONE:\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity & 1u), "r"(smem_u32(bar2)), "r"(parity2 & 1u)
        : "memory");
    if (!ok) B.abort = 1;
    return __all_sync(0xffffffffu, ok != 0);
}
__device__ __forceinline__ void arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// The same for a whole warp's work, as one arrival: those of 32 lanes take their
// turns in shared memory (8,192 tokens: 98 -> 94 us).
__device__ __forceinline__ void arrive_warp(uint64_t* bar, int lane) {
    __syncwarp();
    if (lane == 0) arrive(bar);
}

// One [64 tokens][64] box of a [T, heads, 128] bf16 tensor, 128-byte swizzle.
__device__ __forceinline__ void tma_box(uint32_t dst, const CUtensorMap* map, int x, int head, int t, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(t), "r"(smem_u32(bar))
        : "memory");
}

// 32 columns of a state, 128-byte swizzle, sent in two boxes of 64 rows.
constexpr uint32_t kBox = 128 * 32 * 4;
__device__ __forceinline__ void tma_store(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(map), "r"(x), "r"(y),
                 "r"(z), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// 16 lanes x 16 columns from the registers of 16 x 8 products' A operands: y[2 n + r] is
// lane lane / 4 + 8 r, column 4 n + lane % 4.
__device__ __forceinline__ void tmem_st_frag(uint32_t ta, const uint32_t (&y)[8]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(ta), "r"(y[0]),
                 "r"(y[1]), "r"(y[2]), "r"(y[3]), "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
                 : "memory");
}

// 16 lanes x 16 columns of two accumulators in the fragment layout, there after the wait: x[8 k + 4 n + 2 r + i]
// is accumulator k, lane lane / 4 + 8 r, column 8 n + 2 (lane % 4) + i.
__device__ __forceinline__ void tmem_ld_frag2(uint32_t ta, uint32_t tb, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n\t"
        "tcgen05.ld.sync.aligned.16x256b.x2.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(ta), "r"(tb)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Products issued by the lane of a converged warp that has a non-zero `me`.  The
// low words of descriptors move by bytes >> 4, the high ones do not change.
__device__ __forceinline__ void mma_ss(uint32_t me, uint32_t d, uint32_t a, uint32_t a_high, uint32_t b, uint32_t b_high, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %7, 0;\n\t"
        "mov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], x, y, %6, p;\n\t}" ::"r"(me),
        "r"(d), "r"(a), "r"(a_high), "r"(b), "r"(b_high), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t me, uint32_t d, uint32_t a, uint32_t b, uint32_t b_high, uint32_t idesc, bool add) {
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t.reg .b64 y;\n\tsetp.ne.b32 q, %0, 0;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "mov.b64 y, {%3, %4};\n\t"
        "@q tcgen05.mma.cta_group::1.kind::f16 [%1], [%2], y, %5, p;\n\t}" ::"r"(me),
        "r"(d), "r"(a), "r"(b), "r"(b_high), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void commit_to(uint32_t me, uint64_t* bar) {
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %0, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}" ::"r"(me),
                 "r"(smem_u32(bar))
                 : "memory");
}

// A barrier of n threads, and whether x holds for all of them.
__device__ __forceinline__ bool bar_all(int id, int n, bool x) {
    uint32_t y;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 q, %3, 0;\n\tbar.red.and.pred p, %1, %2, q;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(y)
                 : "r"(id), "r"(n), "r"((uint32_t)x)
                 : "memory");
    return y != 0;
}

// The launches of a call overlap: one may start its CTAs once every CTA of the one
// before it has started, and waits for that one's end and its writes where it
// needs them.
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_last_launch() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <int kN>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kN));
}
template <int kN>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kN));
}

// Tensor-memory columns
constexpr uint32_t kColU = 0, kColS = 128, kColP = 192, kColO1 = 256, kColO2 = 320;
constexpr uint32_t kColV = 384;  // V^T, and the three terms of V^T w: 32 each

__global__ void __launch_bounds__(kThreads, 1)
    decay_prefill_kernel(const PrefillParams p, const __grid_constant__ CUtensorMap mq,
                         const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                         const __grid_constant__ CUtensorMap m_state, const __grid_constant__ CUtensorMap m_out) {
    extern __shared__ __align__(1024) uint8_t sm[];
    Bars& B = *reinterpret_cast<Bars*>(sm + L::bars);
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t sb = smem_u32(sm);
    auto gate = [&](int m) { return reinterpret_cast<Gate*>(sm + L::gates + (m % L::kGates) * L::kGate); };

    Finder finder;
    Item it{p.N, 0, 0, 0, 0, 0};
    if (warp == 22 || warp == 24) it = find_item(p, finder, blockIdx.x / p.HV);
    if (tid == 22 * 32) {
        B.abort = 0;
        B.none = it.n >= p.N;
#pragma unroll
        for (int i = 0; i < 3; ++i) mbar_init(&B.full[i], 2), mbar_init(&B.empty[i], 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            mbar_init(&B.qk_full[i], 1), mbar_init(&B.pv_done[i], 1), mbar_init(&B.u_full[i], 1);
            mbar_init(&B.p_ready[i], 3), mbar_init(&B.p_free[i], 1), mbar_init(&B.drain[i], 1), mbar_init(&B.v_ready[i], 8);
        }
        mbar_init(&B.u_free, 8), mbar_init(&B.o_full, 1), mbar_init(&B.o_free, 4);
        mbar_init(&B.p_read, 3), mbar_init(&B.s_ready, 8), mbar_init(&B.s_free, 1);
        mbar_init(&B.st_full, 8), mbar_init(&B.st_free, 1);
        fence_mbar_init();
    }
    if (warp == 23) {
        tmem_alloc(&B.tmem, 512);
        tmem_relinquish();
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    constexpr uint32_t tm = 0;  // all 512 columns, so they start at the first
    const bool work = B.none == 0 && B.tmem == tm;
    let_next_launch_start();

    if (warp < 8) {
        // ---- state: row v of 128, half the columns, in registers ----
        more_registers<kRegsState>();
        wait_for_last_launch();  // states
        const int half = warp >> 2, v0 = 32 * (warp & 3), v = v0 + lane;
        const uint32_t tl = tm + ((uint32_t)v0 << 16);
        float s[64];
        float prod = 1.f;
        bool first = true;
        int stored = 0;
#pragma unroll 1
        for (int m = 0; work; ++m) {
            const Gate* gt = gate(m);
            if (first) {
                if (!wait_bar(B, &B.full[m % L::kStages], m / L::kStages)) break;
                prod = 1.f;
                const float* src = gt->src;
                if (src != nullptr) {
                    src += v * kDim + 64 * half;
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        asm volatile("ld.global.L1::no_allocate.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                     : "=f"(s[8 * i]), "=f"(s[8 * i + 1]), "=f"(s[8 * i + 2]), "=f"(s[8 * i + 3]),
                                       "=f"(s[8 * i + 4]), "=f"(s[8 * i + 5]), "=f"(s[8 * i + 6]), "=f"(s[8 * i + 7])
                                     : "l"(src + 8 * i)
                                     : "memory");
                } else {
#pragma unroll
                    for (int i = 0; i < 64; ++i) s[i] = 0.f;
                }
            }
            // S's operand is free once the products with it are done
            if (m > 0 && !wait_bar(B, &B.s_free, m - 1)) break;
            fence_after_sync();
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t x[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) x[j] = pack_bf16(s[32 * i + 2 * j], s[32 * i + 2 * j + 1]);
                tmem_st16_u32_nowait(tl + kColS + 32 * half + 16 * i, x);
            }
            tmem_wait_st();
            fence_before_sync();
            arrive_warp(&B.s_ready, lane);
            if (!wait_bar(B, &B.u_full[m & 1], m >> 1)) break;
            fence_after_sync();
            const float a = gt->a;
            const int flags = gt->flags, out = gt->out, decay = gt->decay;
            prod *= a;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float x[16];
                tmem_ld16(tl + kColU + 64 * half + 16 * i, x);
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float2 y = __ffma2_rn(make_float2(a, a), make_float2(s[16 * i + j], s[16 * i + j + 1]), make_float2(x[j], x[j + 1]));
                    s[16 * i + j] = y.x, s[16 * i + j + 1] = y.y;
                }
            }
            fence_before_sync();
            arrive_warp(&B.u_free, lane);
            first = flags & kLast;
            if (first) {
                // the state leaves by way of its last chunk's k and v (32 KiB) and buffer of P (8 KiB), free after
                // that chunk's U and P V, and 24 KiB beside them; the store warp sends it on and gives them back
                if (!wait_bar(B, &B.pv_done[m & 1], m >> 1)) break;
                if (stored > 0 && !wait_bar(B, &B.st_free, stored - 1)) break;
                ++stored;
                if (out >= 0) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t box = !half            ? (m % L::kStages) * L::kStage + L::oK + x * kBox
                                             : !x || v < 64 ? L::tail + x * kBox
                                                            : L::ps + (m & 1) * L::kP - 64 * 128;
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            *reinterpret_cast<float4*>(sm + box + v * 128 + ((i ^ (v & 7)) << 4)) =
                                make_float4(s[32 * x + 4 * i], s[32 * x + 4 * i + 1], s[32 * x + 4 * i + 2], s[32 * x + 4 * i + 3]);
                    }
                    fence_proxy_async_smem();
                }
                if (tid == 0) {
                    B.st_out = out, B.st_m = m, B.st_final = flags & kFinal;
                    if (decay >= 0) p.ws_decay[decay] = prod;
                }
                arrive_warp(&B.st_full, lane);
            }
            if (flags & kFinal) break;
        }
    } else if (warp < 16) {
        // ---- V^T, and V^T w in three terms of 8 bits each (exact), to tensor memory ----
        fewer_registers<kRegsScale>();
        const int th = (warp - 8) >> 2, v0 = 32 * (warp & 3);  // 32 tokens, 32 v
        const uint32_t to = tm + ((uint32_t)v0 << 16) + kColV + 16 * th;
        const int row = 32 * th + 8 * (lane >> 4) + (lane & 7), piece = v0 / 8 + (lane >> 3 & 1);
        const uint32_t from = sb + L::oV + (piece >> 3) * (kTile / 2) + row * 128;
#pragma unroll 1
        for (int m = 0; work; ++m) {
            const int st = m % L::kStages;
            if (!wait_bar(B, &B.full[st], m / L::kStages)) break;
            const Gate* gt = gate(m);
            const int live = gt->live, flags = gt->flags;
            // transposed 8 x 8 matrices come in the layout in which 16 lanes x 4 columns are stored: y[i][2 n + r] is
            // v 16 i + lane / 4 + 8 r, tokens 8 n + 2 (lane % 4) + {0, 1}
            uint32_t y[2][8];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int n = 0; n < 4; n += 2)
                    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(y[i][2 * n]), "=r"(y[i][2 * n + 1]), "=r"(y[i][2 * n + 2]), "=r"(y[i][2 * n + 3])
                                 : "r"(from + st * L::kStage + 8 * n * 128 + ((((piece + 2 * i) ^ row) & 7) << 4))
                                 : "memory");
            float2 w[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) w[n] = *reinterpret_cast<const float2*>(&gt->w[32 * th + 8 * n + 2 * (lane & 3)]);
            if (live < C) {  // what follows the segment must not meet a zero weight as 0 * NaN, in neither operand
#pragma unroll
                for (int n = 0; n < 4; ++n) {
                    const int left = live - (32 * th + 8 * n + 2 * (lane & 3));
                    const uint32_t keep = left >= 2 ? 0xffffffffu : left == 1 ? 0xffffu : 0u;
#pragma unroll
                    for (int i = 0; i < 2; ++i) y[i][2 * n] &= keep, y[i][2 * n + 1] &= keep;
                }
#pragma unroll 1
                for (int i = tid - 256; i < (C - live) * 16; i += 256)
                    *reinterpret_cast<uint4*>(sm + st * L::kStage + L::oK + (i >> 3 & 1) * (kTile / 2) + (live + (i >> 4)) * 128 + 16 * (i & 7)) =
                        make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                uint32_t t0[8], t1[8], t2[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float2 x = __fmul2_rn(w[e >> 1], widen2(y[i][e]));
                    t0[e] = upper2(x);
                    x = minus_bf16(x, t0[e]);
                    t1[e] = upper2(x);
                    t2[e] = upper2(minus_bf16(x, t1[e]));
                }
                if (i == 0) {  // the products with the chunk before are done
                    if (m > 0 && !wait_two(B, &B.pv_done[(m - 1) & 1], (m - 1) >> 1, &B.u_full[(m - 1) & 1], (m - 1) >> 1)) goto out;
                    fence_after_sync();
                }
                const uint32_t at = to + ((uint32_t)(16 * i) << 16);
                tmem_st_frag(at, y[i]);
                tmem_st_frag(at + 32, t0);
                tmem_st_frag(at + 64, t1);
                tmem_st_frag(at + 96, t2);
            }
            tmem_wait_st();
            fence_before_sync();
            arrive_warp(&B.v_ready[m & 1], lane);
            if (flags & kFinal) break;
        }
    out:;
    } else if (warp < 20) {
        fewer_registers<kRegsOut>();
        {
            // ---- outputs ----
            wait_for_last_launch();
            const int wq = warp - 16;
            const uint32_t tl = tm + ((uint32_t)(32 * wq) << 16);
            const size_t step = (size_t)p.HV * kDim;
            if (!p.first) {  // tokens of no sequence: zeros
                const int c0 = cu_at(p.cu, p.cu64, 0, p.T), c1 = max(c0, cu_at(p.cu, p.cu64, p.N, p.T));
                const int rows = c0 + p.T - c1;  // a row is HV * 16 pieces of 16 bytes
#pragma unroll 1
                for (int r = blockIdx.x; r < rows; r += gridDim.x)
#pragma unroll 1
                    for (int i = tid - 512; i < p.HV * 16; i += 128)
                        *reinterpret_cast<uint4*>(p.out + (size_t)(r < c0 ? r : r - c0 + c1) * step + 8 * i) = make_uint4(0, 0, 0, 0);
            }
#pragma unroll 1
            for (int m = 0; work; ++m) {
                const bool ok = wait_bar(B, &B.o_full, m);
                fence_after_sync();
                const uint32_t os = L::os + (m & 1) * kTile;
                const Gate* gt = gate(m);
                const int rows = gt->rows, flags = gt->flags, t = gt->t, h = gt->h;
                // 16 v x 16 tokens at a time, the next ones on their way, in the fragment layout of 8 x 8 matrices, which
                // stmatrix turns into 8 tokens x 8 v: 16 bytes of a token's row, at their place under the 128-byte
                // swizzle.  Matrices of a store: tokens 0, v 0 and 8; tokens 8, v 0 and 8; this lane's address: token
                // lane % 8 of matrix lane / 8
                uint32_t x[2][16];
                auto load = [&](int b, uint32_t (&r)[16]) {  // v 16 (b & 1), tokens 16 (b >> 1)
                    const uint32_t at = tl + ((uint32_t)(16 * (b & 1)) << 16) + 16 * (b >> 1);
                    tmem_ld_frag2(at + kColO1, at + kColO2, r);
                };
                load(0, x[0]);
#pragma unroll 1
                for (int c = 0; c < 4; ++c) {
                    const float2 e[2] = {*reinterpret_cast<const float2*>(&gt->e[16 * c + 2 * (lane & 3)]),
                                         *reinterpret_cast<const float2*>(&gt->e[16 * c + 8 + 2 * (lane & 3)])};
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        tmem_ld_wait(x[b]);
                        if (b == 0)
                            load(2 * c + 1, x[1]);
                        else if (c < 3)
                            load(2 * c + 2, x[0]);
                        else {
                            fence_before_sync();
                            arrive_warp(&B.o_free, lane);
                        }
                        uint32_t y[4];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {  // tokens 8 (n / 2), v 8 (n % 2)
                            const float2 z = __ffma2_rn(e[n >> 1], make_float2(__uint_as_float(x[b][8 + 2 * n]), __uint_as_float(x[b][9 + 2 * n])),
                                                        make_float2(__uint_as_float(x[b][2 * n]), __uint_as_float(x[b][2 * n + 1])));
                            y[n] = pack_bf16(z.x, z.y);
                        }
                        const int chunk = (4 * wq + 2 * b + (lane >> 3 & 1)) & 7, t8 = 16 * c + 8 * (lane >> 4) + (lane & 7);
                        const uint32_t to = sb + os + (wq >> 1) * (kTile / 2) + t8 * 128 + ((chunk ^ (lane & 7)) << 4);
                        asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(to), "r"(y[0]),
                                     "r"(y[1]), "r"(y[2]), "r"(y[3])
                                     : "memory");
                    }
                }
                fence_proxy_async_smem();
                if (tid == 512) bulk_wait_read0();  // the rows of the chunk before have left: the other buffer is free
                if (!bar_all(1, 128, ok)) break;    // (together: none is left at a barrier)
                if (rows == C) {
                    if (tid == 512) {
                        tma_store(&m_out, sb + os, 0, h, t);
                        tma_store(&m_out, sb + os + kTile / 2, 64, h, t);
                    }
                } else {  // the segment ends in this chunk: its rows only
#pragma unroll 1
                    for (int i = tid - 512; i < rows * 16; i += 128) {
                        const int r = i >> 4, x = i & 15;
                        *reinterpret_cast<uint4*>(p.out + ((size_t)(t + r) * p.HV + h) * kDim + 8 * x) =
                            *reinterpret_cast<const uint4*>(sm + os + (x >> 3) * (kTile / 2) + r * 128 + (((x & 7) ^ (r & 7)) << 4));
                    }
                }
                if (flags & kFinal) break;
            }
            if (tid == 512) bulk_wait_read0();  // shared memory is read until then
        }
    } else {
        fewer_registers<kRegsRest>();
        if (warp < 22 || warp == 25) {
            {
                // ---- decayed scores ----
                const int wq = warp & 1, i = 32 * wq + lane, jb = warp == 25 ? 1 : 0;
                const uint32_t tl = tm + ((uint32_t)(32 * wq) << 16);
#pragma unroll 1
                for (int m = 0; work; ++m) {
                    if (!wait_bar(B, &B.qk_full[m & 1], m >> 1)) break;
                    fence_after_sync();
                    const Gate* gt = gate(m);
                    const int flags = gt->flags;
                    const float ci = -gt->minus[i], f = __fdividef(p.scale, gt->near[i]);
                    uint8_t* row = sm + L::ps + (m & 1) * L::kP + i * 128;
                    // this buffer's last products are those of chunk m - 2
                    if (m > 1 && !wait_bar(B, &B.p_free[m & 1], (m >> 1) - 1)) break;
                    if (warp == 20)  // rows 0 .. 31: nothing in columns 32 .. 63
#pragma unroll
                        for (int q = 4; q < 8; ++q) *reinterpret_cast<uint4*>(row + ((q ^ (i & 7)) << 4)) = make_uint4(0, 0, 0, 0);
#pragma unroll 1
                    for (int c = 0; c < 2; ++c) {
                        float x[16];
                        tmem_ld16(tl + kColP + 32 * jb + 16 * c, x);
                        if (c) {
                            fence_before_sync();
                            arrive_warp(&B.p_read, lane);  // the next chunk's scores may follow
                        }
                        const int low = warp == 21 ? 32 : lane - 16 * c;  // the blocks on the diagonal end there
#pragma unroll
                        for (int j = 0; j < 16; j += 4) {
                            // e^{c_i - c_j}: the first parts' difference is exact, the second parts are factors near 1
                            const float4 cj = *reinterpret_cast<const float4*>(&gt->minus[32 * jb + 16 * c + j]);
                            const float4 nj = *reinterpret_cast<const float4*>(&gt->near[32 * jb + 16 * c + j]);
                            const float2 y = __fadd2_rn(make_float2(ci, ci), make_float2(cj.x, cj.y)), z = __fadd2_rn(make_float2(ci, ci), make_float2(cj.z, cj.w));
                            const float2 a = __fmul2_rn(make_float2(ex2(y.x), ex2(y.y)), __fmul2_rn(make_float2(nj.x, nj.y), make_float2(x[j], x[j + 1])));
                            const float2 d = __fmul2_rn(make_float2(ex2(z.x), ex2(z.y)), __fmul2_rn(make_float2(nj.z, nj.w), make_float2(x[j + 2], x[j + 3])));
                            x[j] = j <= low ? a.x : 0.f, x[j + 1] = j + 1 <= low ? a.y : 0.f, x[j + 2] = j + 2 <= low ? d.x : 0.f, x[j + 3] = j + 3 <= low ? d.y : 0.f;
                        }
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            uint32_t t[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float2 z = __fmul2_rn(make_float2(f, f), make_float2(x[8 * q + 2 * e], x[8 * q + 2 * e + 1]));
                                t[e] = pack_bf16(z.x, z.y);
                            }
                            *reinterpret_cast<uint4*>(row + (((4 * jb + 2 * c + q) ^ (i & 7)) << 4)) = make_uint4(t[0], t[1], t[2], t[3]);
                        }
                    }
                    fence_before_sync();
                    fence_proxy_async_smem();
                    arrive_warp(&B.p_ready[m & 1], lane);
                    if (flags & kFinal) break;
                }
            }
        } else if (warp == 22 || warp == 24) {
            // ---- one warp starts the loads, another writes the gates and what the chunk belongs to ----
            const bool loads = warp == 22;
            int m = 0, idx = blockIdx.x;
            bool ok = work;
            auto source = [&](const Item& it, int h) -> const float* {  // the state a segment starts from
                const size_t mat = (size_t)kDim * kDim;
                if (it.s > 0) return p.first ? nullptr : p.ws_state + ((size_t)(it.ws + it.s) * p.HV + h) * mat;
                return p.state ? p.state + ((size_t)it.n * p.HV + h) * mat : nullptr;
            };
            while (ok && it.n < p.N) {
                const int h = idx % p.HV, hq = h / p.rep, len = it.t1 - it.t0, nch = len > C ? (len + C - 1) / C : 1;
                idx += gridDim.x;
                if (loads) {
                    Item next;
#pragma unroll 1
                    for (int c = 0; c < nch; ++c, ++m) {
                        const int st = m % L::kStages;
                        if (m >= L::kStages && !wait_bar(B, &B.empty[st], m / L::kStages - 1)) {
                            ok = false;
                            break;
                        }
                        if (lane == 0) {
                            const uint32_t d = sb + st * L::kStage;
                            const int t = it.t0 + c * C;
                            mbar_arrive_expect_tx(&B.full[st], L::kStage);
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                tma_box(d + x * (kTile / 2), &mq, 64 * x, hq, t, &B.full[st]);
                                tma_box(d + L::oK + x * (kTile / 2), &mk, 64 * x, hq, t, &B.full[st]);
                                tma_box(d + L::oV + x * (kTile / 2), &mv, 64 * x, h, t, &B.full[st]);
                            }
                        }
                        __syncwarp();
                        if (c == 0) {
                            next = find_item(p, finder, idx / p.HV);
                            if (lane == 0 && next.n < p.N) {  // the next segment's state: into L2
                                const float* src = source(next, idx % p.HV);
                                if (src != nullptr)
                                    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(65536) : "memory");
                            }
                        }
                    }
                    it = next;
                    continue;
                }
                const bool last = it.s == it.nseg - 1;
                const int after = (it.ws + it.s + 1) * p.HV + h;  // the next segment's number in the workspace
                const float* src = source(it, h);
                const int out = p.first ? after : last ? it.n * p.HV + h : -1, decay = p.first && it.s > 0 ? after : -1;
                // lane l has tokens 2 l and 2 l + 1 of a chunk; a chunk's log decays are asked for one chunk ahead
                const float* gl = p.log_decay + (p.per_token ? (size_t)(it.t0 + 2 * lane) * p.HV + h : h);
                const size_t one = p.per_token ? p.HV : 0;
                auto ask = [&](int c, float& g0, float& g1) {
                    const int a = c * C + 2 * lane;
                    g0 = g1 = 0.f;
                    if (a < len) g0 = gl[c * C * one];
                    if (a + 1 < len) g1 = gl[c * C * one + one];
                };
                float n0, n1;
                ask(0, n0, n1);
                const Item next = find_item(p, finder, idx / p.HV);
#pragma unroll 1
                for (int c = 0; c < nch; ++c, ++m) {
                    const float g0 = clamp_log_decay(n0), g1 = clamp_log_decay(n1);
                    if (c + 1 < nch) ask(c + 1, n0, n1);
                    // sums to base 2 up to and including token 2 l + 1, in two parts (split_log2_decay)
                    const float2 x0 = split_log2_decay(g0), x1 = split_log2_decay(g1);
                    float2 c1 = make_float2(x0.x + x1.x, x0.y + x1.y);
#pragma unroll
                    for (int d = 1; d < 32; d *= 2) {
                        const float a = __shfl_up_sync(0xffffffffu, c1.x, d), r = __shfl_up_sync(0xffffffffu, c1.y, d);
                        if (lane >= d) c1.x += a, c1.y += r;
                    }
                    // (not c1 - x1: a gate that is NaN stays out of the token before it)
                    float2 c0 = make_float2(__shfl_up_sync(0xffffffffu, c1.x, 1), __shfl_up_sync(0xffffffffu, c1.y, 1));
                    c0 = lane == 0 ? x0 : make_float2(c0.x + x0.x, c0.y + x0.y);
                    const float2 end = make_float2(__shfl_sync(0xffffffffu, c1.x, 31), __shfl_sync(0xffffffffu, c1.y, 31));
                    const float2 e = make_float2(p.scale * exp2f(c0.x + c0.y), p.scale * exp2f(c1.x + c1.y));
                    // (these weigh the fp32 state: expf is a few times as accurate as exp2f)
                    constexpr float kLn2 = 0.6931471805599453f;
                    const float2 w = make_float2(expf(kLn2 * ((end.x - c0.x) + (end.y - c0.y))), expf(kLn2 * ((end.x - c1.x) + (end.y - c1.y))));
                    const float all = expf(kLn2 * (end.x + end.y));
                    // the stage is free, so the products of chunk m - 3 are done, and before them the last reader of
                    // gate slot m - 5 was
                    if (m >= L::kStages && !wait_bar(B, &B.empty[m % L::kStages], m / L::kStages - 1)) {
                        ok = false;
                        break;
                    }
                    Gate* gt = gate(m);
                    *reinterpret_cast<float2*>(&gt->minus[2 * lane]) = make_float2(-c0.x, -c1.x);
                    *reinterpret_cast<float2*>(&gt->near[2 * lane]) = make_float2(ex2(-c0.y), ex2(-c1.y));
                    *reinterpret_cast<float2*>(&gt->e[2 * lane]) = e;
                    *reinterpret_cast<float2*>(&gt->w[2 * lane]) = w;
                    if (lane == 0) {
                        gt->a = all;
                        gt->flags = c < nch - 1 ? 0 : next.n >= p.N ? kLast | kFinal : kLast;
                        gt->t = it.t0 + c * C, gt->live = min(C, len - c * C);
                        gt->rows = p.first && it.s > 0 ? 0 : gt->live;
                        gt->h = h, gt->src = src, gt->out = out, gt->decay = decay;
                    }
                    __syncwarp();
                    if (lane == 0) arrive(&B.full[m % L::kStages]);
                }
                it = next;
            }
            if (loads && !ok && lane == 0)  // given up: copies in flight land before the CTA ends
                // (their gates may be missing: only the bytes are waited for, as long as they can take)
#pragma unroll 1
                for (int k = m > L::kStages ? m - L::kStages : 0; k < m; ++k)
                    for (const int t0 = (int)clock(); !mbar_try_wait(&B.full[k % L::kStages], (k / L::kStages) & 1) && (int)clock() - t0 < 1 << 24;) {}
        } else if (warp == 23 || warp == 27) {
            // ---- products, each warp's issued by one elected thread: warp 23 the scores and U, warp 27 the outputs ----
            constexpr uint32_t id_u = idesc_f16(128, 128, 1, 1, 0, 1), id_qk = idesc_f16(128, 64, 1, 1, 0, 0);
            const uint32_t me = elect_one();
            const uint32_t q0 = (uint32_t)desc_kmaj(sb, C, 0), high = (uint32_t)(desc_kmaj(0, C, 0) >> 32);
            if (warp == 23) {
                const uint64_t dk = desc_mnmaj(sb + L::oK, C, 0);
                const uint32_t k0 = (uint32_t)desc_kmaj(sb + L::oK, C, 0), kt0 = (uint32_t)dk, mn_high = (uint32_t)(dk >> 32);
                auto scores = [&](int st) {
                    const uint32_t at = st * (L::kStage >> 4);
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks) {
                            const uint32_t off = at + ((x * (kTile / 2) + 32 * ks) >> 4);
                            mma_ss(me, tm + kColP, q0 + off, high, k0 + off, high, id_qk, (x | ks) > 0);
                        }
                };
                bool ok = work;
                if (ok) {
                    ok = wait_bar(B, &B.full[0], 0);
                    fence_after_sync();
                    if (ok) {
                        scores(0);
                        commit_to(me, &B.qk_full[0]);
                    }
                }
                int st = 0;
#pragma unroll 1
                for (int m = 0; ok; ++m) {
                    const int st1 = st == L::kStages - 1 ? 0 : st + 1;
                    const int flags = gate(m)->flags;
                    const bool final = flags & kFinal;
                    if (!final) {
                        if (!wait_two(B, &B.full[st1], (m + 1) / L::kStages, &B.p_read, m)) break;  // P's columns are free
                        fence_after_sync();
                        scores(st1);
                        commit_to(me, &B.qk_full[(m + 1) & 1]);
                    }
                    // (u_free: of the chunk before, or a phase that counts as over)
                    if (!wait_two(B, &B.v_ready[m & 1], m >> 1, &B.u_free, m - 1)) break;
                    fence_after_sync();
                    const uint32_t kt = kt0 + st * (L::kStage >> 4);
#pragma unroll
                    for (int term = 3; term > 0; --term)  // small terms first
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_ts(me, tm + kColU, tm + kColV + 32 * term + 8 * ks, kt + (koff_mnmaj(16 * ks) >> 4), mn_high, id_u,
                                   term < 3 || ks > 0);
                    commit_to(me, &B.u_full[m & 1]);
                    if (!(flags & kLast)) commit_to(me, &B.empty[st]);  // a last chunk's k and v take the state out first
                    if (final) break;
                    st = st1;
                }
            } else {
                const uint32_t p0 = (uint32_t)desc_kmaj(sb + L::ps, C, 0);
                int st = 0;
#pragma unroll 1
                for (int m = 0; work; ++m, st = st == L::kStages - 1 ? 0 : st + 1) {
                    if (!wait_two(B, &B.v_ready[m & 1], m >> 1, &B.p_ready[m & 1], m >> 1)) break;
                    bool s_too;  // (o_free: of the chunk before, or a phase that counts as over)
                    if (!wait_and_test(B, &B.o_free, m - 1, &B.s_ready, m, s_too)) break;
                    fence_after_sync();
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        mma_ts(me, tm + kColO1, tm + kColV + 8 * ks, p0 + (m & 1) * (L::kP >> 4) + (koff_kmaj(C, 16 * ks) >> 4), high, id_qk, ks > 0);
                    commit_to(me, &B.pv_done[m & 1]);
                    const int flags = gate(m)->flags;
                    if (!s_too && !wait_bar(B, &B.s_ready, m)) break;
                    fence_after_sync();
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int ks = 0; ks < 4; ++ks)
                            mma_ts(me, tm + kColO2, tm + kColS + 32 * x + 8 * ks,
                                   q0 + st * (L::kStage >> 4) + ((x * (kTile / 2) + 32 * ks) >> 4), high, id_qk, (x | ks) > 0);
                    commit_to(me, &B.s_free);
                    commit_to(me, &B.o_full);
                    commit_to(me, &B.empty[st]);
                    if (!(flags & kLast)) commit_to(me, &B.p_free[m & 1]);  // (nor is this free)
                    if (flags & kFinal) break;
                }
            }
        }
    }
    if (warp == 26 && lane == 0)
        // ---- finished states on their way out (of the state warps, which have waited for the last launch) ----
        for (int i = 0; work; ++i) {
            if (!wait_one(B, &B.st_full, i)) break;
            const int out = B.st_out, m = B.st_m, final = B.st_final, st = m % L::kStages;
            if (out >= 0) {
#pragma unroll
                for (int x = 0; x < 8; ++x)
                    tma_store(&m_state,
                              sb + (x < 4   ? st * L::kStage + L::oK + x * (kBox / 2)
                                    : x < 7 ? L::tail + (x - 4) * (kBox / 2)
                                            : L::ps + (m & 1) * L::kP),
                              32 * (x >> 1), 64 * (x & 1), out);
                bulk_wait_read0();
            }
            arrive(&B.empty[st]);
            arrive(&B.p_free[m & 1]);
            arrive(&B.st_free);
            if (final) break;
        }
    __syncwarp();
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    if (B.abort) {  // given up: products in flight end before the tensor memory is given back
        if ((warp == 23 || warp == 27) && elect_one()) {
            uint64_t* drain = &B.drain[warp == 27];
            mma_commit(drain);
            for (const int t0 = (int)clock(); !mbar_try_wait(drain, 0) && (int)clock() - t0 < 1 << 30;) {}
        }
        __syncthreads();
    }
    if (tid == 0 && (B.abort || B.tmem != tm)) atomicOr(&g_device_status, kDevStatTimeout);
    if (warp == 23) tmem_dealloc(B.tmem, 512);
}

// The state before every segment of the sequences that have several: slot 1 holds
// the state after the first segment already, ws[i] = decay[i] ws[i - 1] + ws[i]
// from slot 2 on.  1,024 elements of one v-head of one such sequence per CTA; the
// j-th of them is found by going through the lengths.
__global__ void __launch_bounds__(256) decay_prefill_carry_kernel(const PrefillParams p) {
    const int part = blockIdx.x & 15, j = (blockIdx.x >> 4) / p.HV, h = (blockIdx.x >> 4) % p.HV, lane = threadIdx.x & 31;
    int nseg = 0, ws = 0, before = 0;
    bool found = false;
    let_next_launch_start();
#pragma unroll 1
    for (int base = 0; base < p.N && !found; base += 32) {
        int t0, len, k = 0;
        if (base + lane < p.N) k = n_segments(p, base + lane, t0, len);
        const int mine = k > 1 ? k : 0;
        int wsum = mine;
#pragma unroll
        for (int d = 1; d < 32; d *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, wsum, d);
            if (lane >= d) wsum += x;
        }
        const unsigned long3 = __ballot_sync(0xffffffffu, k > 2);
        const unsigned who = __ballot_sync(0xffffffffu, k > 2 && before + __popc(long3 & ((1u << lane) - 1)) == j);
        if (who) {
            const int src = __ffs(who) - 1;
            nseg = __shfl_sync(0xffffffffu, k, src);
            ws += __shfl_sync(0xffffffffu, wsum - mine, src);
            found = true;
        } else {
            ws += __shfl_sync(0xffffffffu, wsum, 31);
            before += __popc(long3);
        }
    }
    wait_for_last_launch();  // also where there is nothing to do: the next launch takes this one's end for both
    if (!found || ws + nseg > p.ws_slots) return;
    const size_t at = (size_t)part * 1024 + 4 * threadIdx.x, step = (size_t)p.HV * kDim * kDim;
    float* w = p.ws_state + ((size_t)(ws + 1) * p.HV + h) * kDim * kDim + at;
    const float* d = p.ws_decay + (size_t)(ws + 1) * p.HV + h;
    float4 s = *reinterpret_cast<const float4*>(w), u = *reinterpret_cast<const float4*>(w + step);
#pragma unroll 2
    for (int i = 1; i < nseg - 1; ++i) {
        float4 next = u;
        if (i + 1 < nseg - 1) next = *reinterpret_cast<const float4*>(w + (i + 1) * step);
        const float a = d[i * p.HV];
        s = make_float4(fmaf(a, s.x, u.x), fmaf(a, s.y, u.y), fmaf(a, s.z, u.z), fmaf(a, s.w, u.w));
        *reinterpret_cast<float4*>(w + i * step) = s;
        u = next;
    }
}

// ---------------------------------------------------------------------------

// The driver's tensor-map encoder, looked up through the runtime once (no
// link-time dependency on the driver library).
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn encode_fn() {
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

// [T, heads, 128] bf16 in boxes of 64 tokens x 64 elements, 128-byte swizzle.
static bool encode(CUtensorMap* map, const void* x, int heads, int T) {
    const EncodeFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)kDim, (cuuint64_t)heads, (cuuint64_t)T};
    const cuuint64_t strides[2] = {(cuuint64_t)kDim * 2, (cuuint64_t)heads * kDim * 2};
    const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)C}, estr[3] = {1u, 1u, 1u};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(x), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// [states, 128, 128] fp32 in boxes of 32 columns x 64 rows, 128-byte swizzle.
static bool encode_states(CUtensorMap* map, const void* x, long long states) {
    const EncodeFn fn = encode_fn();
    if (fn == nullptr) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)kDim, (cuuint64_t)kDim, (cuuint64_t)states};
    const cuuint64_t strides[2] = {(cuuint64_t)kDim * 4, (cuuint64_t)kDim * kDim * 4};
    const cuuint32_t box[3] = {32u, 64u, 1u}, estr[3] = {1u, 1u, 1u};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, const_cast<void*>(x), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The kernel's attribute, once per device (again after a failure).
static bool set_attribute() {
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return false;
    const unsigned long long bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load() & bit)) return true;
    if (cudaFuncSetAttribute(decay_prefill_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::total) !=
        cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (dev < 64) done.fetch_or(bit);
    return true;
}

// Tokens of a segment, at least 256: with P = 148 / HV CTAs for each v-head, T
// over P + 1 segments gives both launches P of them.  (HV > 74: whole sequences,
// as two launches of one CTA a head would gain nothing.)
static int segment_tokens(int T, int HV) {
    const int parts = HV <= kSms / 2 ? kSms / HV + 1 : 1;
    const int x = T / parts + (T % parts != 0), r = x > 1 << 30 ? 1 << 30 : (x + C - 1) / C * C;
    return r < 256 ? 256 : r;
}
// Workspace slots: a sequence of n > 1 segments has n of them, at most 2 len / segment.
static int workspace_slots(int T, int HV) {
    const int seg = segment_tokens(T, HV);
    return T > seg ? (int)(2ll * T / seg) : 0;
}

static int status_bits(bool clear) {
    unsigned int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_device_status, sizeof(v)) != cudaSuccess) return -1;
    if (clear && v) {
        const unsigned int z = 0;
        if (cudaMemcpyToSymbol(g_device_status, &z, sizeof(z)) != cudaSuccess) return -1;
    }
    return (int)v;
}

}  // namespace decay

int decay_prefill_status(bool clear) { return decay::status_bits(clear); }

}  // namespace gdn

extern "C" size_t gdn_decay_prefill_workspace_bytes(int N, int T, int HV) {
    if (N <= 0 || T <= 0 || HV <= 0) return 0;
    const size_t slots = gdn::decay::workspace_slots(T, HV);
    return slots * HV * (gdn::kDim * gdn::kDim + 1) * sizeof(float);
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
    const int seg = segment_tokens(T, HV), ws_slots = N > 0 ? workspace_slots(T, HV) : 0;
    const long long slots = (long long)(T / seg) + N;                // (an int could overflow)
    if (slots + 1 > (1ll << 26) / HV) return GDN_ERR_UNSUPPORTED;  // grid index
    if (N == 0 && T == 0) return GDN_OK;
    if (!cu_seqlens || (T > 0 && (!q || !k || !v || !out || !log_decay)) || (N > 0 && !new_state)) return GDN_ERR_INVALID;
    if (!gdn_aligned(q, 16) || !gdn_aligned(k, 16) || !gdn_aligned(v, 16) || !gdn_aligned(out, 16) ||
        !gdn_aligned(state, 32) || !gdn_aligned(new_state, 32) || !gdn_aligned(log_decay, 4) ||
        !gdn_aligned(cu_seqlens, cu_seqlens_is_int64 ? 8 : 4))
        return GDN_ERR_ALIGN;
    // the states are one buffer or two that do not overlap
    const size_t bytes = (size_t)N * HV * gdn::kDim * gdn::kDim * sizeof(float);
    const uintptr_t si = (uintptr_t)state, so = (uintptr_t)new_state;
    if (state && si != so && si < so + bytes && so < si + bytes) return GDN_ERR_INVALID;
    const size_t need = gdn_decay_prefill_workspace_bytes(N, T, HV);
    if (need && (!workspace || workspace_bytes < need)) return GDN_ERR_INVALID;
    if (need && !gdn_aligned(workspace, 32)) return GDN_ERR_ALIGN;
    PrefillParams p;
    p.state = state;
    p.log_decay = log_decay;
    p.cu = cu_seqlens;
    p.out = static_cast<__nv_bfloat16*>(out);
    p.new_state = new_state;
    p.ws_state = static_cast<float*>(workspace);
    p.ws_decay = p.ws_state + (size_t)ws_slots * HV * gdn::kDim * gdn::kDim;
    p.scale = scale == 0.0f ? 1.0f / sqrtf((float)K) : scale;
    p.cu64 = cu_seqlens_is_int64;
    p.per_token = decay_per_token;
    p.N = N;
    p.T = T;
    p.HV = HV;
    p.rep = HV / H;
    p.seg_len = seg;
    p.ws_slots = ws_slots;
    p.first = 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (T == 0) {  // every sequence keeps its state
        cudaError_t e = cudaSuccess;
        if (state == nullptr)
            e = cudaMemsetAsync(new_state, 0, bytes, st);
        else if (state != new_state)
            e = cudaMemcpyAsync(new_state, state, bytes, cudaMemcpyDeviceToDevice, st);
        return e == cudaSuccess ? GDN_OK : GDN_ERR_CUDA;
    }
    CUtensorMap mq{}, mk{}, mv{}, mn{}, mo{}, mw{};
    if (!encode(&mq, q, H, T) || !encode(&mk, k, H, T) || !encode(&mv, v, HV, T) || !encode(&mo, out, HV, T) ||
        (N > 0 && !encode_states(&mn, new_state, (long long)N * HV)) ||
        (ws_slots > 0 && !encode_states(&mw, workspace, (long long)ws_slots * HV)))
        return GDN_ERR_CUDA;
    if (!set_attribute()) return GDN_ERR_CUDA;
    // kernel after kernel, each but the first allowed to start before the one before it ends
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = st;
    cfg.attrs = attr;
    cudaError_t e = cudaSuccess;
    if (ws_slots > 0) {
        const int inner = T / seg * HV;  // at most: segments that another one follows
        p.first = 1;
        cfg.gridDim = dim3(inner < kSms ? inner : kSms), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = L::total;
        e = cudaLaunchKernelEx(&cfg, decay_prefill_kernel, p, mq, mk, mv, mw, mo);
        cfg.numAttrs = 1;
        // at most T / (2 seg) sequences have more than two segments (any number, if they overlap: the first are taken)
        const int longs = T / 2 / seg;
        if (e == cudaSuccess && longs > 0) {
            cfg.gridDim = dim3(longs * HV * 16), cfg.blockDim = dim3(256), cfg.dynamicSmemBytes = 0;
            e = cudaLaunchKernelEx(&cfg, decay_prefill_carry_kernel, p);
        }
        p.first = 0;
    }
    const int items = (int)(slots * HV);
    cfg.gridDim = dim3(items < kSms ? (items > 0 ? items : 1) : kSms), cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = L::total;
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, decay_prefill_kernel, p, mq, mk, mv, mn, mo);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return GDN_ERR_CUDA;
    }
    return gdn_launch_status();
}

// fsb_head_many.cu - the LM head (fsb_head.cu) for more hidden states than a warp's own tensor instructions are good for: tcgen05.mma with
// the weights as operand A in tensor memory, unpacked there by the warps that later take the sums out again.
//
// A CTA takes 256 vocabulary rows at a time and all hidden states of the pass (up to 144).  Two groups of four warps have 128 rows each, a
// thread for every row.  Per block of 64 weights a warp unpacks its 32 rows to q - 8 in bf16 / fp16 (exact), stores them to tensor
// memory as 32 columns of pairs, and one thread issues the products for the group's 128 rows; sums of one group of weights come back as
// one fp32 column per hidden state, are multiplied by the row's scale and added up in registers, two to an instruction.  Taking sums out
// (groups of 32: 2 N columns a block) and unpacking (64 logic instructions a warp and block) bound it up to N = 64, with the weights' bytes
// close behind.  Weights, scales and hidden states come through one ring of stages of two blocks, by bulk and tensor copies of one warp.
#include <cuda.h>

#include <algorithm>

#include "../../include/ferro_sampler_b200.h"
#include "fsb_head.cuh"

namespace fsb {
namespace {

constexpr int kManyThreads = 384;        // two groups of four warps; issuers (8, 9), copies (10), one idle warp that completes the third group
constexpr int kRows = 256;               // vocabulary rows of a unit
constexpr int kPairs = kRows / 32;
constexpr int kTokensMax = 144;
constexpr int kSharedMax = 227 * 1024;
constexpr int kStagesMax = 8;

struct ManyPlan {
    HeadArgs a;
    int tokens;      // hidden states a pass
    int columns;     // ... rounded up to 16
    int slots;       // tensor memory columns sets for sums
    int stages;
    int stage_bytes;
};

struct Barriers {
    u64 full[kStagesMax], empty[kStagesMax];
    u64 a_full[2][2], a_empty[2][2];
    u64 d_full[2][4], d_empty[2][4];
    u64 done[2];
    unsigned tmem;
    volatile int dead;
};

__device__ __forceinline__ void barrier_init(u64* bar, unsigned count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count) : "memory"); }
__device__ __forceinline__ void barrier_arrive(u64* bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory"); }
// Waits for the phase of this parity to end.  Gives up after a million looks (a second or so), or when somebody else of the CTA has.
__device__ __forceinline__ bool barrier_wait(u64* bar, unsigned parity, volatile int* dead) {
    for (int i = 0, looks = FSB_INBOX_LOOKS; i < looks; ++i) {
        unsigned done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(smem_u32(bar)), "r"(parity) : "memory");
        if (done) return true;
        if ((i & 15) == 15 && *dead) return false;
    }
    *dead = 1;
    return false;
}
__device__ __forceinline__ bool warp_wait(u64* bar, unsigned parity, volatile int* dead) { return __all_sync(0xffffffffu, barrier_wait(bar, parity, dead)); }

__device__ __forceinline__ void tc_before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(u64* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_mma(unsigned d, unsigned a, u64 b, unsigned what, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(what),
                 "r"((unsigned)add)
                 : "memory");
}
// 16 lanes x 32 columns: register 2 j and 2 j + 1 are column 4 j + lane % 4 of lanes lane / 4 and lane / 4 + 8.
__device__ __forceinline__ void tc_store(unsigned addr, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
                 "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tc_load16(unsigned addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr)
                 : "memory");
}
// The loads before it have arrived: their registers are handed through so that nobody reads them earlier.
__device__ __forceinline__ void tc_loaded(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tc_use(uint32_t* r) {   // (behind a wait that was given other registers)
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                      "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
// acc[2 i .. 2 i + 1] += s * (d0, d1)
__device__ __forceinline__ void add_scaled(u64& acc, u64 s, uint32_t d0, uint32_t d1) {
    asm("{\n\t.reg .b64 d;\n\tmov.b64 d, {%2, %3};\n\tfma.rn.f32x2 %0, d, %1, %0;\n\t}" : "+l"(acc) : "l"(s), "r"(d0), "r"(d1));
}

// NMAX: columns that a thread has registers for.
template <class X, int GS, int NMAX>
__global__ void __launch_bounds__(kManyThreads, 1) head_many_kernel(const __grid_constant__ ManyPlan P, const __grid_constant__ CUtensorMap hidden_map) {
    extern __shared__ __align__(1024) unsigned char smem_any[];
    __shared__ Barriers B;
    unsigned char* smem = smem_any + (-smem_u32(smem_any) & 1023u);   // (swizzled rows want 1024-byte boundaries)
    const HeadArgs& a = P.a;
    const int tid = (int)threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int blocks = row_blocks(a.n_hidden), chunks = (blocks + 1) / 2;
    const int m0 = (int)blockIdx.y * P.tokens, mt = min(P.tokens, a.n_rows - m0);
    const int units = (a.n_vocab + kRows - 1) / kRows;
    const int mine = (units - (int)blockIdx.x + (int)gridDim.x - 1) / (int)gridDim.x;   // units of this CTA
    const int N = P.columns, slots = P.slots, stages = P.stages;
    // a stage: hidden states [2 blocks][N][128 bytes], weights [8 pairs][2 blocks][1024], scales [8 pairs][...]
    constexpr int kScales = GS == 1 ? 256 : GS == 2 ? 128 : 64;   // of a pair for two blocks
    const int x_bytes = 2 * N * 128;
    volatile int* dead = &B.dead;

    if (tid == 0) {
        for (int i = 0; i < stages; ++i) {
            barrier_init(&B.full[i], 1);
            barrier_init(&B.empty[i], 10);     // eight warps have their weights, two issuers their products
        }
        for (int g = 0; g < 2; ++g) {
            for (int i = 0; i < 2; ++i) barrier_init(&B.a_full[g][i], 4), barrier_init(&B.a_empty[g][i], 1);
            for (int i = 0; i < 4; ++i) barrier_init(&B.d_full[g][i], 1), barrier_init(&B.d_empty[g][i], 4);
            barrier_init(&B.done[g], 1);
        }
        B.dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&B.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_before_sync();
    }
    __syncthreads();
    tc_after_sync();
    const unsigned tmem = B.tmem;

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp == 10) {
            // ------------------------------------------------------------------------------------ copies
            const int64_t pair_w = pair_weights(a.n_hidden), pairs_all = padded_pairs(a.n_vocab);
            const int64_t pair_s = pair_scales(a.n_hidden, 32 * GS);
            int s = 0;
            unsigned phase = 1;    // (a fresh barrier's phase before the first has ended)
            bool ok = true;
            int64_t issued = 0;
            for (int u = 0; u < mine && ok; ++u) {
                const int64_t unit = (int64_t)blockIdx.x + (int64_t)u * gridDim.x;
                const int64_t pair = min(unit * kPairs + (lane & 7), pairs_all - 1);   // behind the vocabulary: any row will do
                for (int c = 0; c < chunks; ++c) {
                    ok = warp_wait(&B.empty[s], phase, dead);
                    if (!ok) break;
                    const int nb = min(2, blocks - 2 * c);
                    const unsigned w_bytes = nb * 1024, s_bytes = GS == 4 ? 64 : nb * (GS == 1 ? 128 : 64);
                    unsigned char* st = smem + s * P.stage_bytes;
                    if (lane == 0) inbox_expect(&B.full[s], nb * N * 128 + kPairs * (w_bytes + s_bytes));
                    __syncwarp();
                    if (lane < 8) bulk_copy(st + x_bytes + lane * 2048, a.weights + pair * pair_w + (int64_t)c * 2048, w_bytes, &B.full[s]);
                    else if (lane < 16)
                        bulk_copy(st + x_bytes + kPairs * 2048 + (lane - 8) * kScales, a.scales + pair * pair_s + (int64_t)c * kScales, s_bytes, &B.full[s]);
                    else if (lane < 16 + nb)
                        asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
                                         smem_u32(st + (lane - 16) * N * 128)),
                                     "l"(&hidden_map), "r"((2 * c + lane - 16) * 64), "r"(m0), "r"(smem_u32(&B.full[s]))
                                     : "memory");
                    ++issued;
                    if (++s == stages) s = 0, phase ^= 1;
                }
            }
            // Nobody leaves while copies are on their way (they are all waited for unless somebody gave up).
            if (*dead) {
                for (int i = 0; i < stages; ++i)
                    if (issued > i) {
                        const int64_t n = (issued - 1 - i) / stages;   // last use of stage i
                        int never = 0;
                        barrier_wait(&B.full[i], (unsigned)(n & 1), &never);
                    }
            }
        } else if (warp < 10) {
            // ------------------------------------------------------------------------------------ products of group `wg`
            const int wg = warp - 8;
            if (lane == 0) {
                constexpr bool bf16 = std::is_same<X, __nv_bfloat16>::value;
                const unsigned what = 1u << 4 | (bf16 ? 1u : 0u) << 7 | (bf16 ? 1u : 0u) << 10 | (unsigned)(N >> 3) << 17 | (128u >> 4) << 24;
                const unsigned a0 = tmem + wg * 256, d0 = a0 + 64;
                // K-major rows of 128 bytes, swizzled, eight rows every 1024 bytes
                const u64 desc0 = 1ull << 16 | (u64)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
                int s = 0, slot = 0;
                unsigned phase = 0, ab = 0, a_phase = 0, d_phase = 1;
                bool ok = true;
                for (int u = 0; u < mine && ok; ++u)
                    for (int c = 0; c < chunks && ok; ++c) {
                        ok = barrier_wait(&B.full[s], phase, dead);
                        const int nb = min(2, blocks - 2 * c);
                        for (int k = 0; k < nb && ok; ++k) {
                            ok = barrier_wait(&B.a_full[wg][ab], a_phase, dead);
                            if (!ok) break;
                            tc_after_sync();
                            const u64 desc = desc0 | (u64)((smem_u32(smem + s * P.stage_bytes + k * N * 128) & 0x3FFFF) >> 4);
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const bool begins = GS == 1 || (half == 0 && (GS == 2 || k == 0)), ends = GS == 1 || (half == 1 && (GS == 2 || k == 1));
                                if (begins) {
                                    ok = ok && barrier_wait(&B.d_empty[wg][slot], d_phase, dead);
                                    tc_after_sync();
                                }
                                if (ok) {
#pragma unroll
                                    for (int q = 0; q < 2; ++q)
                                        tc_mma(d0 + slot * N, a0 + ab * 32 + half * 16 + q * 8, desc + (half * 4 + q * 2), what, !(begins && q == 0));
                                    if (ends) {
                                        tc_commit(&B.d_full[wg][slot]);
                                        if (++slot == slots) slot = 0, d_phase ^= 1;
                                    }
                                }
                            }
                            if (ok) tc_commit(&B.a_empty[wg][ab]);
                            ab ^= 1;
                            if (ab == 0) a_phase ^= 1;
                        }
                        if (ok) tc_commit(&B.empty[s]);
                        if (++s == stages) s = 0, phase ^= 1;
                    }
                // what has been issued is complete before anybody frees its memory
                tc_commit(&B.done[wg]);
                int never = 0;
                barrier_wait(&B.done[wg], 0, &never);
            }
            __syncwarp();
        }
    } else {
        // ---------------------------------------------------------------------------------------- a thread for every row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        const int wg = warp >> 2, wr = warp & 3, r16 = lane >> 4, in16 = lane & 15;
        const unsigned a0 = tmem + ((unsigned)(wr * 32) << 16) + wg * 256, d0 = a0 + 64;
        const Unpack<X> unpack;
        const bool bf16_scales = a.scale_type == FSB_BF16;
        u64 acc[NMAX / 2];
#pragma unroll
        for (int i = 0; i < NMAX / 2; ++i) acc[i] = 0ull;
        int s = 0, slot = 0;
        unsigned phase = 0, ab = 0, a_phase = 1, d_phase = 0;
        bool ok = true;
        constexpr int kEnds = GS == 1 ? 2 : 1;      // groups that end in a block (GS == 4: in every second)
        float scale[kEnds];                         // of the groups that are being added up
        int waiting = 0, last_unit = -1;            // groups whose sums have not been taken out yet; a unit whose last ones they are

        auto take = [&]() {
#pragma unroll
            for (int e = 0; e < kEnds; ++e) {
                if (e >= waiting || !ok) break;
                ok = warp_wait(&B.d_full[wg][slot], d_phase, dead);
                if (!ok) break;
                tc_after_sync();
                const unsigned from = d0 + slot * N;
                u64 s2;
                asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(scale[e]));
#pragma unroll
                for (int c = 0; c < NMAX; c += 32) {
                    if (c >= N) break;
                    uint32_t v[32];
                    const bool two = c + 16 < NMAX && c + 16 < N;
                    tc_load16(from + c, v);
                    if (two) tc_load16(from + c + 16, v + 16);
                    tc_loaded(v);
                    if (two) tc_use(v + 16);
                    if (c + 32 >= N) {   // the last ones: the columns may be written again
                        tc_before_sync();
                        __syncwarp();
                        if (lane == 0) barrier_arrive(&B.d_empty[wg][slot]);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) add_scaled(acc[c / 2 + i], s2, v[2 * i], v[2 * i + 1]);
                    if (two) {
#pragma unroll
                        for (int i = 8; i < 16; ++i)
                            if (c / 2 + i < NMAX / 2) add_scaled(acc[c / 2 + i < NMAX / 2 ? c / 2 + i : 0], s2, v[2 * i], v[2 * i + 1]);
                    }
                }
                if (++slot == slots) slot = 0, d_phase ^= 1;
            }
            waiting = 0;
            if (last_unit >= 0 && ok) {
                const int row = last_unit * kRows + wg * 128 + wr * 32 + lane;
                float* to = a.logits + (int64_t)m0 * a.ld + row;
#pragma unroll
                for (int i = 0; i < NMAX / 2; ++i) {
                    float lo, hi;
                    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(acc[i]));
                    if (row < a.n_vocab) {
                        if (2 * i < mt) to[(int64_t)(2 * i) * a.ld] = lo;
                        if (2 * i + 1 < mt) to[(int64_t)(2 * i + 1) * a.ld] = hi;
                    }
                    acc[i] = 0ull;
                }
                last_unit = -1;
            }
        };

        for (int u = 0; u < mine && ok; ++u)
            for (int c = 0; c < chunks && ok; ++c) {
                ok = warp_wait(&B.full[s], phase, dead);
                if (!ok) break;
                const unsigned char* st = smem + s * P.stage_bytes + x_bytes;
                const unsigned char* sp = st + kPairs * 2048 + (wg * 4 + wr) * kScales;
                const int nb = min(2, blocks - 2 * c);
                for (int k = 0; k < nb && ok; ++k) {
                    uint4 w[2];
#pragma unroll
                    for (int r = 0; r < 2; ++r) w[r] = *reinterpret_cast<const uint4*>(st + (wg * 4 + wr) * 2048 + k * 1024 + r * 512 + lane * 16);
                    // this row's scales
                    float now[kEnds];
#pragma unroll
                    for (int e = 0; e < kEnds; ++e) {
                        const int at = GS == 1 ? k * 128 + r16 * 64 + (in16 & 7) * 8 + e * 4 + (in16 >> 3) * 2
                                               : (GS == 2 ? k * 64 : 0) + r16 * 32 + (in16 & 7) * 4 + (in16 >> 3) * 2;
                        const unsigned short raw = *reinterpret_cast<const unsigned short*>(sp + at);
                        now[e] = bf16_scales ? __uint_as_float((uint32_t)raw << 16) : __half2float(__ushort_as_half(raw));
                    }
                    if (k == nb - 1) {   // the stage's weights and scales have been read
                        __syncwarp();
                        if (lane == 0) barrier_arrive(&B.empty[s]);
                    }
                    uint32_t p[2][16];
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int half = 0; half < 2; ++half)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                p[r][(half * 4 + i) * 2] = unpack.value(half ? w[r].z : w[r].x, i);
                                p[r][(half * 4 + i) * 2 + 1] = unpack.value(half ? w[r].w : w[r].y, i);
                            }
                    ok = warp_wait(&B.a_empty[wg][ab], a_phase, dead);
                    if (!ok) break;
                    tc_after_sync();
                    tc_store(a0 + ab * 32, p[0]);
                    tc_store(a0 + (16u << 16) + ab * 32, p[1]);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    tc_before_sync();
                    __syncwarp();
                    if (lane == 0) barrier_arrive(&B.a_full[wg][ab]);
                    ab ^= 1;
                    if (ab == 0) a_phase ^= 1;
                    // the block before this one (groups of 128: the two before)
                    if (GS != 4 || k == 0) take();
                    if (GS != 4 || k == 1) {
                        waiting = kEnds;
#pragma unroll
                        for (int e = 0; e < kEnds; ++e) scale[e] = now[e];
                        if (2 * c + k == blocks - 1) last_unit = (int)blockIdx.x + u * (int)gridDim.x;
                    }
                }
                if (++s == stages) s = 0, phase ^= 1;
            }
        take();
        tc_before_sync();
    }
    __syncthreads();
    if (warp == 8) {
        tc_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
    if (tid == 0 && B.dead) {
        *static_cast<volatile uint32_t*>(a.late) = 1u;
        __threadfence_system();
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult r;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &r) != cudaSuccess || r != cudaDriverEntryPointSuccess) {
            cudaGetLastError();
            return (EncodeTiled) nullptr;
        }
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return f;
}

template <class X, int GS, int NMAX>
int run(const ManyPlan& p, const CUtensorMap& map, cudaStream_t stream) {
    const int units = (p.a.n_vocab + kRows - 1) / kRows;
    const dim3 grid((unsigned)std::min(units, p.a.sms), (unsigned)((p.a.n_rows + p.tokens - 1) / p.tokens));
    head_many_kernel<X, GS, NMAX><<<grid, kManyThreads, (size_t)(p.stages * p.stage_bytes + 1024), stream>>>(p, map);
    return (int)cudaGetLastError();
}
template <class X, int GS>
int run_columns(const ManyPlan& p, const CUtensorMap& map, cudaStream_t stream) {
    return p.columns <= 32 ? run<X, GS, 32>(p, map, stream) : p.columns <= 64 ? run<X, GS, 64>(p, map, stream)
           : p.columns <= 96 ? run<X, GS, 96>(p, map, stream) : run<X, GS, 144>(p, map, stream);
}
template <class X>
int run_group(const ManyPlan& p, const CUtensorMap& map, cudaStream_t stream) {
    return p.a.group == 32 ? run_columns<X, 1>(p, map, stream) : p.a.group == 64 ? run_columns<X, 2>(p, map, stream) : run_columns<X, 4>(p, map, stream);
}

template <class X, int GS>
int prepare_columns() {
    cudaError_t e = cudaFuncSetAttribute(head_many_kernel<X, GS, 32>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(head_many_kernel<X, GS, 64>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(head_many_kernel<X, GS, 96>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(head_many_kernel<X, GS, 144>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax - 1024);
    return (int)e;
}
template <class X>
int prepare_type() {
    int e = prepare_columns<X, 1>();
    if (e == 0) e = prepare_columns<X, 2>();
    return e ? e : prepare_columns<X, 4>();
}

}  // namespace

int prepare_head_many() {
    const int e = prepare_type<__nv_bfloat16>();
    return e ? e : prepare_type<__half>();
}

bool launch_head_many(const HeadArgs& a, void* stream, int* error) {
    // tensor copies want rows on 16-byte boundaries
    if (reinterpret_cast<uintptr_t>(a.hidden) % 16 != 0 || a.ld_hidden % 8 != 0) return false;
    const EncodeTiled encode = encode_tiled();
    if (!encode) return false;
    ManyPlan p{};
    p.a = a;
    const int passes = (a.n_rows + kTokensMax - 1) / kTokensMax;
    p.tokens = (a.n_rows + passes - 1) / passes;
    p.columns = (p.tokens + 15) / 16 * 16;
    p.slots = std::min(4, (256 - 64) / p.columns);
    p.stage_bytes = 2 * p.columns * 128 + kPairs * (2048 + (a.group == 32 ? 256 : a.group == 64 ? 128 : 64));
    p.stage_bytes = (p.stage_bytes + 1023) / 1024 * 1024;
    p.stages = std::min(kStagesMax, (kSharedMax - 3072) / p.stage_bytes);
    CUtensorMap map;
    const cuuint64_t dims[2] = {(cuuint64_t)a.n_hidden, (cuuint64_t)a.n_rows}, strides[1] = {(cuuint64_t)a.ld_hidden * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)p.columns}, step[2] = {1, 1};
    if (encode(&map, a.hidden_type == FSB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(a.hidden), dims, strides, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
        return false;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    *error = a.hidden_type == FSB_BF16 ? run_group<__nv_bfloat16>(p, map, s) : run_group<__half>(p, map, s);
    return true;
}

}  // namespace fsb

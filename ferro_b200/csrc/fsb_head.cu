// fsb_head.cu - the LM head with 4-bit weights and a scale per group: logits[m][v] = sum_g s[v][g] sum_{k in g} (q[v][k] - 8) x[m][k].
//
// Weights are never rounded: a 4-bit weight becomes the 16-bit float 16 + q by one logic operation (its bits are the upper
// mantissa bits of a number between 16 and 32), tensor cores add up (16 + q) x in fp32 for one group on top of -24 times the
// group's sum of x, and the scale is multiplied in fp32.  For up to 16 hidden states a pass the weights' bytes bound it.
//
// Layout (laid out once): tiles of 16 vocabulary rows, within a tile blocks of 64 weights a row, within a block 16 bytes per lane
// of the warp that multiplies it.  Lane 4 g + t holds, of rows g and g + 8, the weights 8 t .. 8 t + 7 of the block's two halves
// of 32: words (g, half 0), (g + 8, half 0), (g, half 1), (g + 8, half 1), each rotated left by three bits so that its first pair
// of weights already lies where bf16 wants it.  A lane's word is one lane's part of an operand fragment, with the k of a half
// taken in the order that makes it so; hidden states are put in the same order.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/ferro_sampler_b200.h"
#include "fsb_device.cuh"

namespace fsb {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kAhead = 4;                    // blocks of 64 weights that a warp has on their way
constexpr int kSharedMax = 227 * 1024;

// Blocks of 64 weights a row is padded to, and 16-bit scales a lane's row pair needs per block.
__host__ __device__ constexpr int row_blocks(int n_hidden) { return (n_hidden + 63) / 64; }
// Scales lie as [tile][block or pair of blocks][g 0..7][...]: for groups of 32 the lane's (row g, half 0), (g + 8, 0), (g, 1), (g + 8, 1),
// otherwise (g), (g + 8) of the block's (128: of the two blocks') group.
__host__ __device__ constexpr int scale_bytes_per_tile(int n_hidden, int group) {
    return group == 32 ? row_blocks(n_hidden) * 64 : group == 64 ? row_blocks(n_hidden) * 32 : row_blocks(n_hidden) / 2 * 32;
}

// ------------------------------------------------------------------------------------------------ layout
__global__ void layout_weights_kernel(const unsigned char* __restrict__ w, int n_vocab, int n_hidden, uint32_t* __restrict__ out) {
    const int blocks = row_blocks(n_hidden);
    const int64_t words = (int64_t)((n_vocab + 127) / 128) * 8 * blocks * 128;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < words; i += (int64_t)gridDim.x * blockDim.x) {
        const int slot = (int)(i & 3), lane = (int)(i >> 2) & 31;
        const int64_t tb = i >> 7;
        const int block = (int)(tb % blocks);
        const int64_t row = tb / blocks * 16 + (lane >> 2) + (slot & 1) * 8;
        const int k = block * 64 + (slot >> 1) * 32 + (lane & 3) * 8;
        uint32_t v = 0x88888888u;   // weights of value 0
        if (row < n_vocab && k < n_hidden) {
            const unsigned char* p = w + row * (n_hidden / 2) + k / 2;
            v = (uint32_t)p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16 | (uint32_t)p[3] << 24;
        }
        out[i] = __funnelshift_l(v, v, 3);
    }
}
__global__ void layout_scales_kernel(const unsigned short* __restrict__ s, int n_vocab, int n_hidden, int group, unsigned short* __restrict__ out) {
    const int per_tile = scale_bytes_per_tile(n_hidden, group) / 2, groups = n_hidden / group;
    const int64_t n = (int64_t)((n_vocab + 127) / 128) * 8 * per_tile;
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) {
        const int j = (int)(i % per_tile);
        int g, r8, lane_row;
        if (group == 32) {
            g = (j >> 5) * 2 + (j >> 1 & 1);
            lane_row = j >> 2 & 7;
            r8 = j & 1;
        } else {
            g = j >> 4;
            lane_row = j >> 1 & 7;
            r8 = j & 1;
        }
        const int64_t row = i / per_tile * 16 + lane_row + r8 * 8;
        out[i] = row < n_vocab && g < groups ? s[row * groups + g] : (unsigned short)0;
    }
}

// ------------------------------------------------------------------------------------------------ up to 16 rows a pass
struct HeadPlan {
    HeadArgs a;
    int ksplit;        // warps that share a tile pair's k; the CTA's other warps take other tile pairs
    int tokens;        // hidden states a pass
    int vec;           // hidden states may be read 16 bytes at a time
};

// Two of a word's weights as 16-bit floats 16 + q: pair i holds weights i and i + 4 of the word's eight.
template <class X>
__device__ __forceinline__ uint32_t weight_pair(uint32_t w, int i) {
    if constexpr (std::is_same<X, __nv_bfloat16>::value) return (__funnelshift_r(w, w, 4 * i) & 0x00780078u) | 0x41804180u;
    else return (__funnelshift_r(w, w, (4 * i + 29) & 31) & 0x03C003C0u) | 0x4C004C00u;
}

template <class X>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<X, __nv_bfloat16>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint4 load_stream(const unsigned char* p) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ float2 two_scales(uint32_t s, bool bf16) {
    if (bf16) return make_float2(__uint_as_float(s << 16), __uint_as_float(s & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&s));
}

// GS: halves of 32 per group.  NT: eights of hidden states.
template <class X, int GS, int NT>
__global__ void __launch_bounds__(kThreads, 1) head_kernel(const __grid_constant__ HeadPlan P) {
    extern __shared__ __align__(16) unsigned char smem[];
    const HeadArgs& a = P.a;
    constexpr int kBuffers = 2;
    const int tid = (int)threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int blocks = row_blocks(a.n_hidden), ks = P.ksplit, kw = warp % ks, rg = warp / ks, groups_of_warps = kWarps / ks;
    const int m0 = (int)blockIdx.y * P.tokens, mt = min(P.tokens, a.n_rows - m0);
    // a warp's share of k, in pieces that hold whole groups
    constexpr int kPiece = GS == 4 ? 2 : 1;
    const int pieces = blocks / kPiece;
    const int p0 = pieces * kw / ks * kPiece, steps = pieces * (kw + 1) / ks * kPiece - p0;
    const int pairs = (a.n_vocab + 31) / 32;                                  // tile pairs: 32 vocabulary rows
    const int unit_stride = (int)gridDim.x * groups_of_warps;
    const int first = (int)blockIdx.x * groups_of_warps + rg;
    const int units = first < pairs ? (pairs - first + unit_stride - 1) / unit_stride : 0;

    float* part = reinterpret_cast<float*>(smem);                              // [buffer][warp][8 NT][36]
    constexpr int kPart = NT * 8 * 36;
    float* xsum = part + kBuffers * kWarps * kPart;                            // [group][8 NT]: -24 times the group's sum
    const int groups = (2 * blocks + GS - 1) / GS;
    unsigned char* xs = reinterpret_cast<unsigned char*>(xsum + groups * NT * 8);   // [half][hidden state][t] x 16 bytes

    const size_t tile_w = (size_t)blocks * 512, tile_s = (size_t)scale_bytes_per_tile(a.n_hidden, 32 * GS);
    constexpr int kScaleStep = GS == 1 ? 64 : 32;
    // what is fetched next
    int f_unit = 0, f_step = 0;
    const unsigned char* f_w = a.weights + (size_t)first * 2 * tile_w + (size_t)p0 * 512 + lane * 16;
    const unsigned char* f_s = a.scales + (size_t)first * 2 * tile_s + (size_t)(p0 / kPiece) * kScaleStep + g * (GS == 1 ? 8 : 4);
    uint4 w[kAhead][2];
    uint2 sc[kAhead][2];
    auto fetch = [&](int i) {
        if (f_unit >= units) return;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            w[i][r] = load_stream(f_w + r * tile_w);
            if constexpr (GS == 1) sc[i][r] = __ldg(reinterpret_cast<const uint2*>(f_s + r * tile_s));
            else sc[i][r].x = __ldg(reinterpret_cast<const unsigned*>(f_s + r * tile_s));
        }
        ++f_step;
        f_w += 512;
        if (GS != 4 || (f_step & 1) == 0) f_s += kScaleStep;
        if (f_step == steps) {
            f_step = 0;
            ++f_unit;
            f_w += (size_t)unit_stride * 2 * tile_w - (size_t)steps * 512;
            f_s += (size_t)unit_stride * 2 * tile_s - (size_t)(steps / kPiece) * kScaleStep;
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) fetch(i);

    // hidden states into shared memory, eight at a time, in the order of weight_pair
    const X* hidden = static_cast<const X*>(a.hidden);
    for (int i = tid; i < mt * blocks * 8; i += kThreads) {
        const int m = i / (blocks * 8), o = i - m * (blocks * 8);
        const X* p = hidden + (int64_t)(m0 + m) * a.ld_hidden + o * 8;
        alignas(16) unsigned short v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (o * 8 < a.n_hidden) {
            if (P.vec) {
                *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(p));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __ldg(reinterpret_cast<const unsigned short*>(p) + j);
            }
        }
        uint4 u;
        u.x = (uint32_t)v[0] | (uint32_t)v[4] << 16;
        u.y = (uint32_t)v[1] | (uint32_t)v[5] << 16;
        u.z = (uint32_t)v[2] | (uint32_t)v[6] << 16;
        u.w = (uint32_t)v[3] | (uint32_t)v[7] << 16;
        *reinterpret_cast<uint4*>(xs + ((size_t)((o >> 2) * mt + m) * 4 + (o & 3)) * 16) = u;
    }
    __syncthreads();
    for (int i = tid; i < groups * NT * 8; i += kThreads) {
        const int gr = i / (NT * 8), m = i - gr * (NT * 8);
        float sum = 0.0f;
        if (m < mt)
            for (int h = gr * GS; h < min(2 * blocks, gr * GS + GS); ++h) {
                const X* p = reinterpret_cast<const X*>(xs + (size_t)(h * mt + m) * 64);
#pragma unroll 8
                for (int j = 0; j < 32; ++j) sum += (float)p[(j + 8 * (tid & 3)) & 31];
            }
        xsum[i] = -24.0f * sum;
    }
    __syncthreads();

    float acc[2][NT][4];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[r][n][j] = 0.0f;
    float d[2][NT][4];
    const bool bf16_scales = a.scale_type == FSB_BF16;
    int unit = 0, step = 0;
    while (unit < units) {
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (unit >= units) break;
            const int block = p0 + step;
            float2 s[2][GS == 1 ? 2 : 1];
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                s[r][0] = two_scales(sc[i][r].x, bf16_scales);
                if constexpr (GS == 1) s[r][1] = two_scales(sc[i][r].y, bf16_scales);
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bool begins = GS == 1 || (half == 0 && (GS == 2 || (i & 1) == 0));
                const bool ends = GS == 1 || (half == 1 && (GS == 2 || (i & 1) == 1));
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint4 b = make_uint4(0u, 0u, 0u, 0u);
                    if (n * 8 + g < mt) b = *reinterpret_cast<const uint4*>(xs + ((size_t)((block * 2 + half) * mt + n * 8 + g) * 4 + t) * 16);
                    if (begins) {
                        const float2 c = *reinterpret_cast<const float2*>(&xsum[(block * 2 + half) / GS * (NT * 8) + n * 8 + 2 * t]);
#pragma unroll
                        for (int r = 0; r < 2; ++r) d[r][n][0] = d[r][n][2] = c.x, d[r][n][1] = d[r][n][3] = c.y;
                    }
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const uint32_t lo = half ? w[i][r].z : w[i][r].x, hi = half ? w[i][r].w : w[i][r].y;
                        mma<X>(d[r][n], weight_pair<X>(lo, 0), weight_pair<X>(hi, 0), weight_pair<X>(lo, 1), weight_pair<X>(hi, 1), b.x, b.y);
                        mma<X>(d[r][n], weight_pair<X>(lo, 2), weight_pair<X>(hi, 2), weight_pair<X>(lo, 3), weight_pair<X>(hi, 3), b.z, b.w);
                    }
                    if (ends) {
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float2 f = s[r][GS == 1 ? half : 0];
                            acc[r][n][0] = fmaf(f.x, d[r][n][0], acc[r][n][0]);
                            acc[r][n][1] = fmaf(f.x, d[r][n][1], acc[r][n][1]);
                            acc[r][n][2] = fmaf(f.y, d[r][n][2], acc[r][n][2]);
                            acc[r][n][3] = fmaf(f.y, d[r][n][3], acc[r][n][3]);
                        }
                    }
                }
            }
            fetch(i);
            if (++step == steps) {   // the unit's 32 rows: the warps that share them add up their parts
                float* to = part + ((unit & 1) * kWarps + warp) * kPart;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int r = 0; r < 2; ++r)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int col = n * 8 + 2 * t + (j & 1);
                            if (col < mt) to[col * 36 + r * 16 + g + (j >> 1) * 8] = acc[r][n][j];
                            acc[r][n][j] = 0.0f;
                        }
                if (ks == 1) __syncwarp();
                else asm volatile("bar.sync %0, %1;" ::"r"(1 + rg), "r"(32 * ks) : "memory");
                const float* from = part + ((unit & 1) * kWarps + rg * ks) * kPart;
                const int v0 = (first + unit * unit_stride) * 32;
                for (int o = kw * 32 + lane; o < mt * 32; o += ks * 32) {
                    const int col = o >> 5, row = o & 31;
                    float sum = 0.0f;
                    for (int q = 0; q < ks; ++q) sum += from[q * kPart + col * 36 + row];
                    if (v0 + row < a.n_vocab) a.logits[(int64_t)(m0 + col) * a.ld + v0 + row] = sum;
                }
                step = 0;
                ++unit;
            }
        }
    }
}

int shared_bytes(const HeadArgs& a, int nt, int tokens) {
    const int blocks = row_blocks(a.n_hidden), groups = (2 * blocks * 32 + a.group - 1) / a.group;
    return 4 * (2 * kWarps * nt * 8 * 36 + groups * nt * 8) + blocks * 128 * tokens;
}

template <class X, int GS, int NT>
int launch_plan(const HeadPlan& p, int grid_x, cudaStream_t stream) {
    const int bytes = shared_bytes(p.a, NT, p.tokens);
    const dim3 grid((unsigned)grid_x, (unsigned)((p.a.n_rows + p.tokens - 1) / p.tokens));
    head_kernel<X, GS, NT><<<grid, kThreads, (size_t)bytes, stream>>>(p);
    return (int)cudaGetLastError();
}
template <class X, int GS>
int launch_tokens(const HeadPlan& p, int nt, int grid_x, cudaStream_t stream) {
    return nt == 1 ? launch_plan<X, GS, 1>(p, grid_x, stream) : launch_plan<X, GS, 2>(p, grid_x, stream);
}
template <class X>
int launch_group(const HeadPlan& p, int nt, int grid_x, cudaStream_t stream) {
    return p.a.group == 32 ? launch_tokens<X, 1>(p, nt, grid_x, stream)
           : p.a.group == 64 ? launch_tokens<X, 2>(p, nt, grid_x, stream) : launch_tokens<X, 4>(p, nt, grid_x, stream);
}

template <class X, int GS>
int prepare_group() {
    cudaError_t e = cudaFuncSetAttribute(head_kernel<X, GS, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(head_kernel<X, GS, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMax);
    return (int)e;
}
template <class X>
int prepare_type() {
    int e = prepare_group<X, 1>();
    if (e == 0) e = prepare_group<X, 2>();
    return e ? e : prepare_group<X, 4>();
}

}  // namespace

int prepare_head_kernels() {
    const int e = prepare_type<__nv_bfloat16>();
    return e ? e : prepare_type<__half>();
}

int64_t head_weight_bytes(int n_vocab, int n_hidden) { return (int64_t)((n_vocab + 127) / 128) * 8 * row_blocks(n_hidden) * 512; }
int64_t head_scale_bytes(int n_vocab, int n_hidden, int group) { return (int64_t)((n_vocab + 127) / 128) * 8 * scale_bytes_per_tile(n_hidden, group); }

int launch_head_layout(const unsigned char* weights, const void* scales, int n_vocab, int n_hidden, int group, unsigned char* weights_out,
                       unsigned char* scales_out, void* stream) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    layout_weights_kernel<<<148 * 8, 256, 0, s>>>(weights, n_vocab, n_hidden, reinterpret_cast<uint32_t*>(weights_out));
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    layout_scales_kernel<<<148 * 4, 256, 0, s>>>(static_cast<const unsigned short*>(scales), n_vocab, n_hidden, group,
                                                 reinterpret_cast<unsigned short*>(scales_out));
    return (int)cudaGetLastError();
}

int launch_head(const HeadArgs& a, void* stream, int* launches) {
    HeadPlan p{};
    p.a = a;
    p.vec = reinterpret_cast<uintptr_t>(a.hidden) % 16 == 0 && a.ld_hidden % 8 == 0;
    // as many hidden states a pass as shared memory holds beside the partial sums, up to 16
    int nt = a.n_rows > 8 ? 2 : 1;
    p.tokens = std::min(8 * nt, a.n_rows);
    if (shared_bytes(a, nt, p.tokens) > kSharedMax) {
        nt = 1;
        p.tokens = std::min(8, a.n_rows);
        while (shared_bytes(a, 1, p.tokens) > kSharedMax) --p.tokens;
    }
    // How many warps share the k of 32 rows: the fewest steps of the CTA with the most, its waves times the longest share.
    const int pairs = (a.n_vocab + 31) / 32, pieces = row_blocks(a.n_hidden) / (a.group == 128 ? 2 : 1);
    int64_t best = 0;
    int grid_x = 1;
    for (int ks = 1; ks <= kWarps; ks *= 2) {
        if (ks > pieces) break;
        const int per_cta = kWarps / ks, ctas = std::min(a.sms, (pairs + per_cta - 1) / per_cta);
        const int64_t waves = ((int64_t)pairs + (int64_t)ctas * per_cta - 1) / ((int64_t)ctas * per_cta), longest = (pieces + ks - 1) / ks;
        const int64_t cost = waves * (longest * 16 + 8 + ks);   // (a share's end costs about half a step, and more for every part that is added)
        if (best == 0 || cost < best) {
            best = cost;
            p.ksplit = ks;
            grid_x = ctas;
        }
    }
    ++*launches;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a.hidden_type == FSB_BF16 ? launch_group<__nv_bfloat16>(p, nt, grid_x, s) : launch_group<__half>(p, nt, grid_x, s);
}

}  // namespace fsb

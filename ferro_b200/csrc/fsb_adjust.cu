// fsb_adjust.cu - what requests ask of their logits before a token is drawn: softcap, repetition / frequency / presence
// penalty over the penalty window, biases, grammar masks; from fp32, bf16 or fp16 logits to the rows that are sampled.
//
// Per row and column v, c(v) = occurrences of v in the row's window:
//     x = cap * tanhf(x / cap);  c(v) > 0: x = (x > 0 ? x / p : x * p) - (f * c(v) + q);  x += bias(v);  masked: x = -inf
// in fp32, rounded once when it is stored.
//
// One pass over the logits, bound by its bytes.  A CTA takes kTile columns of one row.  Its mask bits come first, and vectors
// of logits that are masked altogether are not read (a grammar leaves a handful of tokens as often as not).  Few columns stand
// in the window or have a bias: they are marked in a bitmap, and only marked columns look at the counts (in shared memory,
// cleared where they are marked and nowhere else) and the bias list.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "../../include/ferro_sampler_b200.h"
#include "fsb_device.cuh"

namespace fsb {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 4096;                     // columns of a CTA
constexpr int kCols = kTile / kThreads;         // ... and of a thread
constexpr int kBlockRows = 512;                 // rows whose descriptors go with one launch

template <int ROWS>
struct Params {
    AdjustArgs a;
    AdjustRow rows[ROWS];
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }

// N elements that are loaded and stored together, 16 bytes at a time.
template <class T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

// The mask bits of the N <= 16 columns whose first token id is `id`.  A word is read where one of the columns [id, id + n) lies in it.
__device__ __forceinline__ unsigned mask_bits(const uint32_t* mask, int id, int n) {
    const int w = id >> 5, shift = id & 31;
    const unsigned lo = __ldg(mask + w);
    const unsigned hi = shift + n > 32 ? __ldg(mask + w + 1) : 0u;
    return __funnelshift_r(lo, hi, shift);
}

template <class TI, class TO, int VEC, int ROWS>
__global__ void __launch_bounds__(kThreads) adjust_kernel(const __grid_constant__ Params<ROWS> P) {
    constexpr int kVecs = kCols / VEC;
    __shared__ unsigned marked[kTile / 32];
    __shared__ int count[kTile];
    const AdjustArgs& a = P.a;
    const int row = (int)blockIdx.y, tid = (int)threadIdx.x;
    const AdjustRow& R = P.rows[row];
    const int c0 = (int)blockIdx.x * kTile, n = min(kTile, a.n_vocab - c0);   // this CTA's columns
    const int id0 = c0 + a.vocab_offset;                                      // token id of its first one
    const TI* in = static_cast<const TI*>(a.in) + (int64_t)row * a.ld + c0;
    TO* out = static_cast<TO*>(a.out) + (int64_t)row * a.out_ld + c0;

    // mask bits, then the logits that they leave
    unsigned keep[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = (i * kThreads + tid) * VEC;
        const int m = min(VEC, n - c);
        keep[i] = m <= 0 ? 0u : (1u << m) - 1u;
        if (R.mask_row >= 0 && m > 0) keep[i] &= mask_bits(a.masks + (int64_t)R.mask_row * a.mask_ld, id0 + c, m);
    }
    Pack<TI, VEC> x[kVecs];
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = (i * kThreads + tid) * VEC;
        if (keep[i] == 0u) continue;
        if (c + VEC <= n) {
            x[i] = *reinterpret_cast<const Pack<TI, VEC>*>(in + c);
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < n) x[i].v[j] = in[c + j];
        }
    }

    const bool special = R.hist_len > 0 || R.n_bias > 0;
    const int32_t* hist = a.pool + R.hist_begin;
    const int32_t* bias_ids = a.pool + R.bias_begin;
    if (special) {
        if (tid < kTile / 32) marked[tid] = 0u;
        __syncthreads();
        for (int i = tid; i < R.hist_len; i += kThreads) {
            const unsigned c = (unsigned)__ldg(hist + i) - (unsigned)id0;
            if (c < (unsigned)n) {
                atomicOr(&marked[c >> 5], 1u << (c & 31));
                count[c] = 0;
            }
        }
        for (int i = tid; i < R.n_bias; i += kThreads) {
            const unsigned c = (unsigned)__ldg(bias_ids + i) - (unsigned)id0;
            if (c < (unsigned)n) {
                atomicOr(&marked[c >> 5], 1u << (c & 31));
                count[c] = 0;
            }
        }
        __syncthreads();
        for (int i = tid; i < R.hist_len; i += kThreads) {
            const unsigned c = (unsigned)__ldg(hist + i) - (unsigned)id0;
            if (c < (unsigned)n) atomicAdd(&count[c], 1);
        }
        __syncthreads();
    }

    const float none = -__int_as_float(0x7f800000);
    bool any = false;
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
        const int c = (i * kThreads + tid) * VEC;
        Pack<TO, VEC> y;
        unsigned mark = 0u;
        if (special && keep[i] != 0u) mark = (marked[c >> 5] >> (c & 31)) & ((1u << VEC) - 1u);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            float v = none;
            if (keep[i] >> j & 1u) {
                v = to_f32(x[i].v[j]);
                if (a.softcap > 0.0f) v = __fmul_rn(a.softcap, tanhf(__fdiv_rn(v, a.softcap)));
                if (mark >> j & 1u) {
                    const int k = count[c + j];
                    if (k > 0) {
                        v = v > 0.0f ? __fdiv_rn(v, R.repetition) : __fmul_rn(v, R.repetition);
                        v -= __fmaf_rn(R.frequency, (float)k, R.presence);
                    }
                    // its place in the bias list, if it has one: ids ascend
                    int lo = 0, hi = R.n_bias;
                    while (lo < hi) {
                        const int mid = (lo + hi) >> 1;
                        if (__ldg(bias_ids + mid) < id0 + c + j) lo = mid + 1;
                        else hi = mid;
                    }
                    if (lo < R.n_bias && __ldg(bias_ids + lo) == id0 + c + j) {
                        const float b = __int_as_float(__ldg(bias_ids + R.n_bias + lo));
                        v = b == none ? none : v + b;
                    }
                }
            }
            any = any || v > none;
            y.v[j] = from_f32<TO>(v);
        }
        if (c + VEC <= n) {
            *reinterpret_cast<Pack<TO, VEC>*>(out + c) = y;
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (c + j < n) out[c + j] = y.v[j];
        }
    }

    if (a.row_state) {   // whoever is the row's last CTA knows whether anything is left
        any = __syncthreads_or(any);
        if (tid == 0) {
            const unsigned tiles = gridDim.x;
            if (any) atomicOr(&a.row_state[row], 0x80000000u);
            __threadfence();
            const unsigned before = atomicAdd(&a.row_state[row], 1u);
            if ((before & 0x7fffffffu) + 1u == tiles) {
                if (!(before & 0x80000000u)) {
                    *static_cast<volatile uint32_t*>(a.empty) = 1u + (unsigned)(a.first_row + row);
                    __threadfence_system();
                }
                a.row_state[row] = 0u;
            }
        }
    }
}

template <class TI, class TO, int VEC, int ROWS>
int launch_rows(const AdjustArgs& a, const AdjustRow* rows, int n_rows, cudaStream_t stream) {
    Params<ROWS> p;
    p.a = a;
    std::copy(rows, rows + n_rows, p.rows);
    const dim3 grid((unsigned)((a.n_vocab + kTile - 1) / kTile), (unsigned)n_rows);
    adjust_kernel<TI, TO, VEC, ROWS><<<grid, kThreads, 0, stream>>>(p);
    return (int)cudaGetLastError();
}

template <class TI, class TO, int VEC>
int launch_vec(const AdjustArgs& a, const AdjustRow* rows, cudaStream_t stream, int* launches) {
    for (int at = 0; at < a.n_rows; at += kBlockRows) {
        const int n = std::min(kBlockRows, a.n_rows - at);
        AdjustArgs b = a;
        b.in = static_cast<const TI*>(a.in) + (int64_t)at * a.ld;
        b.out = static_cast<TO*>(a.out) + (int64_t)at * a.out_ld;
        b.first_row = at;
        b.row_state = a.row_state ? a.row_state + at : nullptr;
        int e;
        if (n <= 16) e = launch_rows<TI, TO, VEC, 16>(b, rows + at, n, stream);
        else if (n <= 96) e = launch_rows<TI, TO, VEC, 96>(b, rows + at, n, stream);
        else e = launch_rows<TI, TO, VEC, kBlockRows>(b, rows + at, n, stream);
        if (e != 0) return e;
        ++*launches;
    }
    return 0;
}

template <class TI, class TO>
int launch_types(const AdjustArgs& a, const AdjustRow* rows, cudaStream_t stream, int* launches) {
    // whole vectors where every row of both matrices starts on a vector's boundary
    constexpr int kVec = 16 / sizeof(TI);
    constexpr size_t out_bytes = std::min<size_t>(16, sizeof(TO) * kVec);
    const bool aligned = reinterpret_cast<uintptr_t>(a.in) % 16 == 0 && a.ld * (int64_t)sizeof(TI) % 16 == 0 &&
                         reinterpret_cast<uintptr_t>(a.out) % out_bytes == 0 && a.out_ld * (int64_t)sizeof(TO) % (int64_t)out_bytes == 0;
    return aligned ? launch_vec<TI, TO, kVec>(a, rows, stream, launches) : launch_vec<TI, TO, 1>(a, rows, stream, launches);
}

}  // namespace

int launch_adjust(const AdjustArgs& a, const AdjustRow* rows, void* stream, int* launches) {
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (a.in_type == FSB_F32) return launch_types<float, float>(a, rows, s, launches);
    if (a.in_type == FSB_BF16)
        return a.out_type == FSB_F32 ? launch_types<__nv_bfloat16, float>(a, rows, s, launches) : launch_types<__nv_bfloat16, __nv_bfloat16>(a, rows, s, launches);
    return a.out_type == FSB_F32 ? launch_types<__half, float>(a, rows, s, launches) : launch_types<__half, __half>(a, rows, s, launches);
}

}  // namespace fsb

// late_head.cuh - compiled into the head's kernels for late_head.cu: now and then a wait gives up at once, in one thread, while what it waits
// for is still on its way.
#pragma once
#ifdef __CUDACC__
static __device__ __forceinline__ int looks_before_giving_up() {
    unsigned long long now;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(now));
    unsigned h = (unsigned)clock64() ^ (threadIdx.x * 2654435761u) ^ (blockIdx.x << 20) ^ (unsigned)(now >> 10);
    h = (h ^ (h >> 16)) * 0x7feb352du;
    h = (h ^ (h >> 15)) * 0x846ca68bu;
    h ^= h >> 16;
    return h % 60000u == 0u ? (int)(h >> 30) : 1 << 20;
}
#define FSB_INBOX_LOOKS looks_before_giving_up()
#endif

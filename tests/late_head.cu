// late_head.cu - launches of the LM head's tensor-memory kernel in which waits now and then give up at once, while what they wait for is still
// on its way.  A launch either tells so, or its logits are right; every launch ends, and the next one is as good as the first.  Prints how
// many told.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <vector>

#include <cuda_runtime.h>

#include "../ferro_b200/csrc/fsb_internal.h"
#include "../include/ferro_sampler_b200.h"

#define CHECK(call)                                                                       \
    do {                                                                                  \
        const cudaError_t e_ = (cudaError_t)(call);                                       \
        if (e_ != cudaSuccess) {                                                          \
            std::printf("%s: %s\n", #call, cudaGetErrorString(e_));                       \
            return 1;                                                                     \
        }                                                                                 \
    } while (0)

template <class T>
T* device(const std::vector<T>& v) {
    T* p = nullptr;
    if (cudaMalloc(reinterpret_cast<void**>(&p), v.size() * sizeof(T)) != cudaSuccess || cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess) {
        std::puts("no memory");
        std::exit(1);
    }
    return p;
}

int main() {
    cudaDeviceProp prop;
    CHECK(cudaGetDeviceProperties(&prop, 0));
    CHECK(fsb::prepare_head_kernels());
    int told[2] = {0, 0}, right[2] = {0, 0};
    for (int c = 0; c < 2; ++c) {
        const int rows = c ? 120 : 40, V = 100000, K = 320, group = c ? 64 : 32;
        std::srand(5 + c);
        std::vector<unsigned char> w((size_t)V * K / 2);
        std::vector<unsigned short> s((size_t)V * K / group, 0x3c00), x((size_t)rows * K);   // scales of 1 (fp16)
        for (auto& b : w) b = (unsigned char)(std::rand() >> 7);
        std::vector<int> xi(x.size());
        for (size_t i = 0; i < x.size(); ++i) {
            xi[i] = (std::rand() >> 7) % 15 - 7;
            const float f = (float)xi[i];
            unsigned u;
            std::memcpy(&u, &f, 4);
            x[i] = (unsigned short)(u >> 16);                                                // bf16, exactly
        }
        unsigned char *ww = nullptr, *ss = nullptr;
        CHECK(cudaMalloc(reinterpret_cast<void**>(&ww), (size_t)fsb::head_weight_bytes(V, K)));
        CHECK(cudaMalloc(reinterpret_cast<void**>(&ss), (size_t)fsb::head_scale_bytes(V, K, group)));
        CHECK(fsb::launch_head_layout(device(w), device(s), V, K, group, ww, ss, nullptr));
        std::vector<float> want((size_t)rows * V), got(want.size());
        for (int v = 0; v < V; v += 7)      // every seventh row of the vocabulary
            for (int m = 0; m < rows; ++m) {
                int sum = 0;
                for (int k = 0; k < K; ++k) sum += ((w[(size_t)v * K / 2 + k / 2] >> (k & 1) * 4 & 15) - 8) * xi[(size_t)m * K + k];
                want[(size_t)m * V + v] = (float)sum;
            }
        uint32_t *late = nullptr, *late_dev = nullptr;
        CHECK(cudaMallocHost(reinterpret_cast<void**>(&late), 4));
        CHECK(cudaHostGetDevicePointer(reinterpret_cast<void**>(&late_dev), late, 0));
        fsb::HeadArgs a{};
        a.weights = ww, a.scales = ss, a.hidden = device(x), a.logits = device(got);
        a.ld_hidden = K, a.ld = V, a.n_rows = rows, a.n_vocab = V, a.n_hidden = K, a.group = group;
        a.scale_type = FSB_F16, a.hidden_type = FSB_BF16, a.sms = prop.multiProcessorCount, a.late = late_dev;
        for (int call = 0; call < 300; ++call) {
            a.chained = call & 1;
            *late = 0u;
            CHECK(cudaMemset(a.logits, 0xff, got.size() * 4));
            int launches = 0;
            CHECK(fsb::launch_head(a, nullptr, &launches));
            CHECK(cudaDeviceSynchronize());
            if (*static_cast<volatile uint32_t*>(late)) {
                ++told[c];
                continue;
            }
            ++right[c];
            if (right[c] % 20 != 1) continue;
            CHECK(cudaMemcpy(got.data(), a.logits, got.size() * 4, cudaMemcpyDeviceToHost));
            for (int v = 0; v < V; v += 7)
                for (int m = 0; m < rows; ++m)
                    if (got[(size_t)m * V + v] != want[(size_t)m * V + v]) {
                        std::printf("call %d, row %d, column %d: %g, not %g\n", call, m, v, got[(size_t)m * V + v], want[(size_t)m * V + v]);
                        return 1;
                    }
        }
    }
    std::printf("%d %d %d %d\n", told[0], right[0], told[1], right[1]);
    return 0;
}

// What the waits of rows128_kernel do when nothing arrives, and how the next call learns of it: one CTA per case, for test_gpu_paged_wait.py.
#include <cstdio>

#include "paged_tensor.cuh"
using namespace lmrs;
using namespace lmrs::paged;

// case 0: nothing arrives | 1: the phase has ended | 2: the end of a part, whose tiles do not go on | 3: they go on for some five seconds, then the part ends
static __global__ void wait_kernel(int which, int* out, unsigned long long* ns, int* err) {
    __shared__ __align__(8) uint64_t bar, flips;
    __shared__ int gave_up;
    if (threadIdx.x == 0) {
        mbar_init(&bar, 1);
        mbar_init(&flips, 1);
        fence_barrier_init();
        gave_up = 0;
    }
    __syncthreads();
    if (threadIdx.x == 32) {
        for (int i = 0; which == 3 && i < 5000; i++) {
            __nanosleep(1000000);
            arrive(&flips);
        }
        if (which == 1 || which == 3) arrive(&bar);
    }
    if (threadIdx.x < 32) {
        unsigned long long a, b;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(a));
        const bool ok = which < 2 ? wait_warp(&bar, 0, &gave_up, dense::TG_SCORES) : wait_part(&bar, 0, &flips, &gave_up);
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(b));
        if (threadIdx.x == 0) { out[0] = ok; *ns = b - a; }
    }
    __syncthreads();
    if (threadIdx.x == 0 && gave_up) *err = gave_up;
}

int main() {
    int *out, res;
    unsigned long long *ns, took;
    GaveUpWord word;
    if (word.take() || !word.get() || word.get() != word.get() || word.take()) return 1;
    if (cudaMalloc(&out, 4) != cudaSuccess || cudaMalloc(&ns, 8) != cudaSuccess) return 1;
    for (int which = 0; which < 4; which++) {
        wait_kernel<<<1, 64>>>(which, out, ns, word.get());
        if (cudaMemcpy(&res, out, 4, cudaMemcpyDeviceToHost) != cudaSuccess || cudaMemcpy(&took, ns, 8, cudaMemcpyDeviceToHost) != cudaSuccess) return 1;
        const int status = word.take();
        printf("%d|%llu|%s|%d\n", res, took / 1000000, status ? dense::tg_gave_up(status).c_str() : "", word.take());
    }
    return 0;
}

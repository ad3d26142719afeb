// What attention over 8-bit pages leaves when one of its waits has run out, and what the next call says: for test_gpu_paged8_wait.py.  The kernels' own copies and products all arrive; so a wait is told
// here that it has waited long enough, one of one warp of one CTA, and what it waited for lands while the kernel clears up.
#include <cstdio>
#include <vector>

#include "dense_gemm.cuh"
namespace lmrs {
namespace dense {
__device__ int loses[4];   // kernel and wait, CTA, warp, how many such waits of it are left
DN_DEVINL bool wait_or_lose_patience(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int what) {
    if (what == loses[0] && (int)blockIdx.x == loses[1] && (int)(threadIdx.x >> 5) == loses[2] && (threadIdx.x & 31) == 0 && loses[3]-- == 0) {
        if (!*abort_flag) *abort_flag = what;
        return false;
    }
    return mbar_wait_bounded(bar, parity, abort_flag, what);
}
}  // namespace dense
}  // namespace lmrs
#define mbar_wait_bounded wait_or_lose_patience
#include "paged8_checks.h"
// (one type and one format are enough here)
template <typename F> static int as_half(F f) { return f(__half()); }
template <typename F> static int as_int8(F f) { return f(std::integral_constant<int, lmrs::paged::FORM_INT8>()); }
#define by_type(dtype, ...) as_half(__VA_ARGS__)
#define by_form(form, ...) as_int8(__VA_ARGS__)
#include "paged8.cu"

static std::string last;
namespace lmrs { int set_error(const std::string& m) { last = m; return 1; } }

static uint32_t seed = 1;
static uint32_t next() { return (seed = seed * 1664525u + 1013904223u) >> 8; }
template <typename T> static T* upload(const std::vector<T>& v) {
    T* p = nullptr;
    if (cudaMalloc(&p, v.size() * sizeof(T) + 16) != cudaSuccess || cudaMemcpy(p, v.data(), v.size() * sizeof(T), cudaMemcpyHostToDevice) != cudaSuccess) exit(1);
    return p;
}

// argv: head size, sequences, rows of each, tokens of the prefix; then kernel and wait, CTA, warp, waits before, as often as wanted
int main(int argc, char** argv) {
    const int D = atoi(argv[1]), seqs = atoi(argv[2]), each = atoi(argv[3]), prefix = atoi(argv[4]);
    const int kv = 8, group = 2, heads = kv * group, page = 16, block = 8, pages = 256, n = seqs * each, table = 26;
    std::vector<int8_t> codes((size_t)pages * page * kv * D);
    std::vector<float> scales((size_t)pages * (page / block) * kv);
    std::vector<__half> q((size_t)n * heads * D);
    std::vector<int> lens(seqs), rows(seqs + 1), tables((size_t)seqs * table), front(prefix / page + 1);
    for (auto& c : codes) c = (int8_t)((int)(next() % 255) - 127);
    for (auto& s : scales) s = (1 + next() % 100) / 6000.0f;
    for (auto& x : q) x = __float2half(((int)(next() % 2001) - 1000) / 500.0f);
    for (auto& t : tables) t = (int)(next() % pages);
    for (auto& t : front) t = (int)(next() % pages);
    for (int b = 0; b < seqs; b++) { lens[b] = 130 + (int)(next() % 270); rows[b] = b * each; }
    rows[seqs] = n;
    int8_t *k = upload(codes), *v = k + 0;
    float* s = upload(scales);
    __half *qd = upload(q), *out = upload(std::vector<__half>((size_t)n * heads * D));
    float* lse = upload(std::vector<float>((size_t)n * heads));
    const int64_t slot = (int64_t)kv * D;
    const lmrs_b200_pages8_t p = {k, v, s, s, page * slot, slot, D, page * slot, slot, D, page / block * kv, kv, 1, page / block * kv, kv, 1, pages, page, kv, D, block, 0};
    const lmrs_b200_batch_t batch = {upload(lens), upload(rows), upload(tables), prefix ? upload(front) : nullptr, table, seqs, table, each, prefix};
    const lmrs_b200_rows_t qr = {qd, (int64_t)heads * D, D}, outr = {out, (int64_t)heads * D, D};
    size_t bytes = 0;
    if (lmrs_b200_paged8_attention_workspace(&p, &batch, 2, n, heads, &bytes)) { puts(last.c_str()); return 1; }
    void* work = nullptr;
    if (cudaMalloc(&work, bytes + 256) != cudaSuccess) return 1;
    std::vector<__half> want(q.size()), got(q.size());
    std::vector<float> want_lse((size_t)n * heads), got_lse(want_lse.size());
    auto call = [&](std::vector<__half>& o, std::vector<float>& l) {   // into a result and a workspace that hold other numbers
        cudaMemset(out, 0x45, o.size() * 2);
        cudaMemset(lse, 0x45, l.size() * 4);
        cudaMemset(work, 0x3f, bytes);
        const int rc = lmrs_b200_paged8_attention(&p, &batch, 2, n, &qr, &outr, heads, 0.125f, 0.0f, lse, work, bytes, nullptr);
        if (cudaMemcpy(o.data(), out, o.size() * 2, cudaMemcpyDeviceToHost) != cudaSuccess || cudaMemcpy(l.data(), lse, l.size() * 4, cudaMemcpyDeviceToHost) != cudaSuccess) exit(1);
        return rc;
    };
    int lose[4] = {0, 0, 0, 0};
    if (cudaMemcpyToSymbol(dense::loses, lose, sizeof lose) != cudaSuccess || call(want, want_lse)) { puts(last.c_str()); return 1; }
    for (int a = 5; a + 3 < argc; a += 4) {
        for (int i = 0; i < 4; i++) lose[i] = atoi(argv[a + i]);
        if (cudaMemcpyToSymbol(dense::loses, lose, sizeof lose) != cudaSuccess || call(got, got_lse)) { puts(last.c_str()); return 1; }
        // a head of a row is right, or all of it is NaN
        size_t nan = 0, wrong = 0;
        for (size_t i = 0; i < got_lse.size(); i++) {
            const bool gone = isnan(got_lse[i]);
            nan += gone;
            bool fine = gone || got_lse[i] == want_lse[i];
            for (int c = 0; c < D; c++) {
                const float x = __half2float(got[i * D + c]);
                fine = fine && (gone ? isnan(x) : x == __half2float(want[i * D + c]));
            }
            wrong += !fine;
        }
        const int said = call(got, got_lse);
        const std::string what = last;
        const int after = call(got, got_lse);
        bool same = true;
        for (size_t i = 0; i < got_lse.size(); i++) same = same && got_lse[i] == want_lse[i];
        printf("%zu|%zu|%zu|%d|%s|%d|%d\n", nan, wrong, got_lse.size(), said, said ? what.c_str() : "", after, (int)same);
    }
    return 0;
}

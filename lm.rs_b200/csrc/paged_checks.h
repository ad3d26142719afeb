// paged_checks.h -- what the entry points over many sequences share on the host (paged.cu, paged8.cu): checks of arguments, how many warps share a row, launches.
#pragma once
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>
#include <string>

#include "paged_attn.cuh"
#include "paged_rows.cuh"

namespace lmrs {
namespace paged {

inline int refuse(const char* where, const std::string& why) { return set_error(std::string("lmrs_b200_") + where + ": " + why); }

inline int launched(const char* where) {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : refuse(where, std::string("launch failed: ") + cudaGetErrorString(e));
}

// the current device: its number of SMs, or 0 with an error set
inline int device_sms(const char* where, int* device) {
    int n = 0, major = 0, sms = 0;
    if (cudaGetDeviceCount(&n) != cudaSuccess || n == 0) {
        cudaGetLastError();
        refuse(where, "no CUDA device available (this library has no CPU fallback)");
        return 0;
    }
    if (cudaGetDevice(device) != cudaSuccess || cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, *device) != cudaSuccess ||
        cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, *device) != cudaSuccess || major != 10) {
        cudaGetLastError();
        refuse(where, "the current device is not sm_100; this library contains sm_100a code only");
        return 0;
    }
    return sms;
}
// a pointer that kernels on the current device may follow
inline bool on_device(const void* p, int device) {
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) { cudaGetLastError(); return false; }
    return (a.type == cudaMemoryTypeDevice && a.device == device) || a.type == cudaMemoryTypeManaged;
}
inline bool aligned(const void* p, size_t n) { return (uintptr_t)p % n == 0; }
inline size_t size_of(int dtype) { return dtype == 1 ? 4 : 2; }
template <typename F> int by_type(int dtype, F f) {
    return dtype == 0 ? f(__nv_bfloat16()) : dtype == 1 ? f(float()) : f(__half());
}
template <typename T> Rows<T> rows_as(const lmrs_b200_rows_t* r) { return Rows<T>{(T*)r->data, r->row, r->head}; }
inline Positions pos_as(const lmrs_b200_positions_t* p) { return p ? Positions{p->data, p->axis, p->row} : Positions{nullptr, 0, 0}; }

inline std::string bad_dtype(int dtype) { return dtype < 0 || dtype > 2 ? "dtype must be 0 (bfloat16), 1 (float32) or 2 (float16)" : ""; }
inline std::string bad_rows(const lmrs_b200_rows_t* r, const char* name, int dtype, int device) {
    if (!r || !r->data) return std::string("null ") + name;
    if (!aligned(r->data, size_of(dtype))) return std::string(name) + " does not lie on a boundary of its elements";
    if (r->row < 0 || r->head < 0) return std::string("negative stride of ") + name;
    if (!on_device(r->data, device)) return std::string(name) + " is not memory of the current device";
    return "";
}
// Do two arrays of a call share bytes?  Exact for equal strides (also where they interleave, as parts of one projection do): the second is the first moved by d, so they meet if
// d + i row + j head comes within a head's size of 0 for distances i, j that rows and heads can have.  With other strides, arrays whose extents meet count as meeting, but for parts of one array's rows.
inline bool meet(const lmrs_b200_rows_t* a, int64_t a_heads, const lmrs_b200_rows_t* b, int64_t b_heads, int64_t n_rows, int64_t head_size, int dtype) {
    if (n_rows < 1 || a_heads < 1 || b_heads < 1) return false;
    const int64_t size = (int64_t)size_of(dtype);
    int64_t a_row = a->row, a_head = a->head, b_row = b->row, b_head = b->head;
    if (n_rows == 1) a_row = b_row = 0;   // (strides that nothing is reached by)
    if (a_heads == 1) a_head = b_heads == 1 ? 0 : b_head;
    if (b_heads == 1) b_head = a_head;
    typedef __int128 wide;   // in bytes: the arrays may lie any number of them apart
    const wide a0 = (wide)(uintptr_t)a->data, b0 = (wide)(uintptr_t)b->data, d = b0 - a0, row = (wide)a_row * size, near = (wide)head_size * size;
    const wide a_span = (wide)(a_heads - 1) * a_head * size + near, b_span = (wide)(b_heads - 1) * b_head * size + near;
    if (a0 + (wide)(n_rows - 1) * a_row * size + a_span <= b0 || b0 + (wide)(n_rows - 1) * b_row * size + b_span <= a0) return false;
    if (a_row == b_row && row > 0) {   // parts of one array's rows, whatever their heads: a's begin at 0 of a row, b's behind them
        const wide at = (d % row + row) % row;
        if (at >= a_span && at + b_span <= row) return false;
    }
    if (a_row != b_row || a_head != b_head || (a_row == 0 && n_rows > 1)) return true;
    for (int64_t j = -(a_heads - 1); j < b_heads; j++) {
        const wide at = d + (wide)j * a_head * size;   // + i row for i in -(n_rows - 1) .. n_rows - 1: the nearest to 0 from either side
        wide i = row ? -at / row : 0;
        for (wide k = i - 1; k <= i + 1; k++) {
            const wide t = at + (k < 1 - (wide)n_rows ? 1 - (wide)n_rows : k > (wide)n_rows - 1 ? (wide)n_rows - 1 : k) * row;
            if (t < near && -t < near) return true;
        }
    }
    return false;
}
inline bool same(const lmrs_b200_rows_t* a, const lmrs_b200_rows_t* b, int64_t n_rows, int64_t heads) {   // the same elements in the same places
    return a->data == b->data && (n_rows < 2 || a->row == b->row) && (heads < 2 || a->head == b->head);
}
inline std::string bad_ints(const int32_t* p, const char* name, int device) {
    if (!aligned(p, 4)) return std::string(name) + " does not lie on a boundary of its elements";
    return on_device(p, device) ? "" : std::string(name) + " is not memory of the current device";
}
inline std::string bad_rope(const lmrs_b200_rope_t* r, int head_size) {
    if (r->pairs < 1 || r->pairs > 128 || r->axes < 1 || (r->layout != 0 && r->layout != 1)) return "rope was not filled by lmrs_b200_rope_init";
    return 2 * r->pairs > head_size ? "rope turns " + std::to_string(2 * r->pairs) + " elements, head_size is " + std::to_string(head_size) : "";
}
inline std::string bad_pages(const lmrs_b200_pages_t* p) {
    if (!p || !p->k || !p->v) return "null pages";
    const std::string why = bad_dtype(p->dtype);
    if (!why.empty()) return why;
    if (p->pages < 1 || p->page_size < 1 || p->kv_heads < 1 || p->kv_heads > MAX_HEADS) return "pages, page_size and kv_heads must be positive, kv_heads at most 65535";
    if (p->head_size < 1 || p->head_size > 256) return "head_size must be 1 .. 256";
    if (p->k_page < 0 || p->k_slot < 0 || p->k_head < 0 || p->v_page < 0 || p->v_slot < 0 || p->v_head < 0) return "negative stride of pages";
    return "";
}
inline std::string bad_batch(const lmrs_b200_batch_t* b, int64_t n_rows, int page_size) {
    if (!b) return "null batch";
    if (b->seqs < 0 || b->seqs > 1 << 30 || n_rows < 0 || n_rows > 0x7fffffff) return "seqs must be 0 .. 2^30, n_rows 0 .. 2^31 - 1";   // (sequences are looked at in strides of up to 384 threads)
    if (b->table_len < 0 || b->table_stride < 0) return "negative table_len or table_stride";
    if (b->prefix_len < 0 || (b->prefix_len > 0 && !b->prefix)) return "prefix_len without prefix";
    if ((int64_t)b->table_len * page_size + b->prefix_len > 0x7fffffff) return "prefix_len + table_len * page_size is beyond 2^31 - 1";
    if (b->seqs > 0 && (!b->lens || (b->table_len > 0 && !b->tables))) return "null lens or tables";
    if (b->max_rows < 1 && n_rows > 0) return "max_rows must be positive";
    if (!b->rows && n_rows != b->seqs) return "without rows, n_rows must be seqs (one row each)";
    return "";
}
inline std::string bad_batch_memory(const lmrs_b200_batch_t* b, int device) {
    std::string why = bad_ints(b->lens, "lens", device);
    if (why.empty() && b->rows) why = bad_ints(b->rows, "rows", device);
    if (why.empty() && b->table_len) why = bad_ints(b->tables, "tables", device);
    if (why.empty() && b->prefix_len) why = bad_ints(b->prefix, "prefix", device);
    return why;
}
inline Batch batch_as(const lmrs_b200_batch_t* b, const lmrs_b200_pages_t* p, int64_t n_rows) {
    return Batch{b->lens, b->rows, b->tables, b->prefix, b->table_stride, b->seqs, b->table_len, b->prefix_len, p->pages, p->page_size, n_rows};
}
template <typename F> int guarded(const char* where, F f) {   // no exception leaves a C entry point
    try {
        return f();
    } catch (...) {
        try { return refuse(where, "out of host memory"); } catch (...) { return 1; }
    }
}
// do an array's heads all begin on 16-byte boundaries?
inline bool vectors(const void* p, int64_t row, int64_t head, int dtype) {
    const int64_t vec = 16 / (int64_t)size_of(dtype);
    return aligned(p, 16) && row % vec == 0 && head % vec == 0;
}
inline bool vectors(const lmrs_b200_rows_t* r, int dtype) { return vectors(r->data, r->row, r->head, dtype); }
// Warps for a row's pieces: one, or more where the rows alone would not give every SM's schedulers a few each; a warp keeps at least one piece a lane.
// One warp a row / this rule, us a call: one row of 40 heads 3.6 / 2.5, keys of one row 6.4 / 4.3, of 64 rows 9.9 / 4.7; from a few thousand rows on it is one in both
inline int parts_of(int64_t n_rows, int64_t pieces, int sms) {
    const int64_t want = ((int64_t)sms * 16 + n_rows - 1) / n_rows, most = (pieces + 31) / 32;
    return (int)std::max<int64_t>(1, std::min(want, most));
}
inline unsigned warps_grid(int64_t warps, int sms) { return (unsigned)std::min<int64_t>((warps + ROW_WARPS - 1) / ROW_WARPS, (int64_t)sms * ROW_CTAS); }

// The number of CTAs that share a call's work counts a B200's SMs: it is part of how a call is cut, and a workspace's size goes by it
constexpr int SMS = 148;
// a line's places in the workspace, counted from `base` (null: only their sizes matter)
inline void place_line(Line& l, int64_t rows, int kv_heads, int head_size, char* base, size_t& bytes) {
    auto take = [&](size_t n) { char* at = base + bytes; bytes += (n + 255) / 256 * 256; return at; };
    l.slots = l.front_units + l.ctas + (l.seqs ? (rows / l.tile_rows + l.seqs) * kv_heads : 0);   // (a sequence's last unit may be a part of one)
    l.plan = (Plan*)take(sizeof(Plan) * ((size_t)l.seqs + 1));
    l.ml = (float2*)take(sizeof(float2) * (size_t)l.slots * l.tile_rows);
    l.o = (float*)take(sizeof(float) * (size_t)l.slots * l.tile_rows * head_size);
}
// lets a kernel use more than 48 KB of shared memory: once a device
template <typename K> cudaError_t allow_smem(K kernel, int device, int bytes, std::atomic<uint64_t>& done) {
    const uint64_t bit = 1ull << (device & 63);
    if (device < 64 && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && device < 64) done.fetch_or(bit, std::memory_order_release);
    return e;
}
// a kernel that may be set up while the one before it still runs, and waits for its results by itself
template <typename K, typename... P> cudaError_t launch_after(K kernel, unsigned grid, unsigned threads, size_t smem, cudaStream_t stream, const P&... p) {
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(grid);
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute a = {};
    a.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a.val.programmaticStreamSerializationAllowed = 1;
    c.attrs = &a;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, p...);
}

}  // namespace paged
}  // namespace lmrs

// C ABI of the gfx950 GEMM library: argument validation, per-stream scratch,
// dispatch to the kernel launchers.  Declarations and the reference interface
// each entry point replaces: include/clove/gemm_c.h.
#include <hip/hip_runtime.h>

#include <map>
#include <mutex>
#include <tuple>
#include <utility>
#include <vector>

#include "clove/gemm_c.h"
#include "common.hpp"
#include "decode.hpp"
#include "dispatch.hpp"
#include "moe.hpp"

namespace clove {
using hw::cdiv64;
namespace {

constexpr int kAbiVersion = 1;

// ---------------------------------------------------------------------------
// device info (cached per device)
// ---------------------------------------------------------------------------
std::mutex g_dev_mu;
std::map<int, int> g_num_cus;

// ---------------------------------------------------------------------------
// scratch per (device, stream)
// ---------------------------------------------------------------------------
struct ScratchEntry {
    void* base = nullptr;
    Scratch view;
};
std::mutex g_scratch_mu;
std::map<std::pair<int, void*>, ScratchEntry> g_scratch;

// other library buffers per (device, stream, slot)
struct BufferEntry {
    void* base = nullptr;
    size_t bytes = 0;
};
std::map<std::tuple<int, void*, int>, BufferEntry> g_buffers;  // guarded by g_scratch_mu

// A call whose launches hand each other data through these buffers (a selection
// and its moves, scores and the weights added up from them, a repacked operand
// and its GEMM) has the stream's to itself from the first acquisition to its end:
// another host thread's launches on the stream would come between its own and
// write what they are still to read.  The locks stay for good.
std::map<std::pair<int, void*>, std::mutex> g_stream_mu;  // the map guarded by g_scratch_mu
thread_local std::unique_lock<std::mutex> t_stream;       // of the current call; let go by CallScope

// (never taken inside g_scratch_mu, which is taken inside it)
void hold_stream(int dev, hipStream_t stream) {
    if (t_stream.owns_lock()) return;
    std::mutex* mu;
    {
        std::lock_guard<std::mutex> lk(g_scratch_mu);
        mu = &g_stream_mu[{dev, reinterpret_cast<void*>(stream)}];
    }
    t_stream = std::unique_lock<std::mutex>(*mu);
}

// Buffers replaced by larger ones, per device, freed by clove_release_scratch
// (after a device synchronize).  A replaced buffer is not freed on the spot: a
// call on another host thread may have taken it and not yet launched the
// kernel that uses it.  Sizes grow by powers of two, so the retired buffers
// of a stream add up to less than its current one.
std::map<int, std::vector<void*>> g_retired;  // guarded by g_scratch_mu

__global__ void zero_u16(uint16_t* p, size_t n) {
    size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0;
}

__global__ void zero_u32(unsigned* p, size_t n) {
    size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x;
    for (; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0u;
}

// Test hook (clove_test_alloc_excess): bytes added to this thread's allocations
thread_local size_t t_alloc_excess = 0;

// hipMalloc whose failure leaves nothing behind: the status is the only report
// of it, and the error HIP keeps for the thread would come back from the next
// check_launch, also from the launch of a call that goes on without scratch.
bool device_malloc(void** p, size_t bytes) {
    if (hipMalloc(p, bytes + t_alloc_excess) == hipSuccess) return true;
    (void)hipGetLastError();
    return false;
}

size_t round_up_pow2(size_t x, size_t floor_bytes) {
    size_t r = floor_bytes;
    while (r < x) r <<= 1;
    return r;
}

bool overlaps(const void* a, size_t abytes, const void* b, size_t bbytes) {
    if (!a || !b || abytes == 0 || bbytes == 0) return false;
    const uintptr_t a0 = reinterpret_cast<uintptr_t>(a), b0 = reinterpret_cast<uintptr_t>(b);
    return a0 < b0 + bbytes && b0 < a0 + abytes;
}

// Rows of one tensor: `rows` of `width` bytes, `stride` bytes apart.
struct Rows {
    const void* p;
    int64_t stride, width, rows;
};

// Whether two such tensors share a byte.  Rows of the same stride may lie
// between each other's (parts of one wider tensor); otherwise their whole
// extents must be apart.
bool overlaps(const Rows& a, const Rows& b) {
    if (!a.p || !b.p || a.rows <= 0 || b.rows <= 0 || a.width <= 0 || b.width <= 0) return false;
    if (!overlaps(a.p, (size_t)((a.rows - 1) * a.stride + a.width), b.p, (size_t)((b.rows - 1) * b.stride + b.width)))
        return false;
    if (a.stride != b.stride || a.width > a.stride || b.width > a.stride) return true;
    const int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
    const int64_t off = ((d % a.stride) + a.stride) % a.stride;  // of b's rows within a's stride
    return off < a.width || a.stride - off < b.width;
}

// Whether an output is its input: the same rows.  (How far apart a single row would
// have its next one does not matter.)
bool same_rows(const Rows& a, const Rows& b) { return a.p == b.p && (a.stride == b.stride || (a.rows <= 1 && b.rows <= 1)); }

bool aligned2(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 1u) == 0; }
bool aligned4(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }

}  // namespace

clove_status_t ensure_lds(const void* kernel, int bytes) {
    if (bytes <= 64 * 1024) return CLOVE_OK;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    static std::mutex mu;
    static std::vector<std::tuple<int, const void*, int>> done;  // (device, kernel, bytes set)
    std::lock_guard<std::mutex> lock(mu);
    for (const auto& e : done)
        if (std::get<0>(e) == dev && std::get<1>(e) == kernel && std::get<2>(e) >= bytes) return CLOVE_OK;
    if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess)
        return CLOVE_ERR_LAUNCH;
    done.emplace_back(dev, kernel, bytes);
    return CLOVE_OK;
}

namespace {

// ---------------------------------------------------------------------------
// caller-owned workspace (clove_workspace_bind / clove_workspace_query_*), per
// host thread.  Layout of a bound workspace: the completion counters at its
// start (a fixed region, so a counter never lands where an earlier call left
// partial sums), then each acquisition of the call at 256-byte offsets.
// ---------------------------------------------------------------------------
enum class WsMode { kLibrary, kBound, kQuery };
struct ThreadWs {
    WsMode mode = WsMode::kLibrary;
    char* ptr = nullptr;
    size_t bytes = 0;
    size_t used = 0;  // carve offset of the current call
    size_t need = 0;  // query: the largest call so far
};
thread_local ThreadWs t_ws;
thread_local ThreadWs t_ws_saved;  // the mode a query interrupted
constexpr size_t kWsCounterBytes = CLOVE_WORKSPACE_MIN_BYTES;
constexpr size_t kWsCounters = kWsCounterBytes / sizeof(unsigned);

size_t round256(size_t x) { return (x + 255) & ~(size_t)255; }

// Carves `bytes` for the current call; nullptr-based in a query (nothing is
// launched, so nothing reads it).
clove_status_t ws_carve(size_t bytes, char** out) {
    const size_t off = t_ws.used, end = off + round256(bytes);
    if (t_ws.mode == WsMode::kBound && end > t_ws.bytes) return CLOVE_ERR_WORKSPACE;
    t_ws.used = end;
    *out = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(t_ws.ptr) + off);
    return CLOVE_OK;
}

// One per C entry point that dispatches: starts the call's carving after the
// counters and, in a query, records what the call took; at its end, when all of
// the call is queued, the stream's library buffers are other threads' again.
struct CallScope {
    CallScope() { t_ws.used = kWsCounterBytes; }
    ~CallScope() {
        if (t_stream.owns_lock()) t_stream.unlock();
        if (t_ws.mode == WsMode::kQuery && t_ws.used > kWsCounterBytes && t_ws.used > t_ws.need)
            t_ws.need = t_ws.used;
    }
};

// ---------------------------------------------------------------------------
// clove_gemm_fp16_noalloc: the fixed device array its calls carve their
// scratch from (counters in its first CLOVE_WORKSPACE_MIN_BYTES, as in a bound
// workspace).  In host code `scratch` is a host-side stand-in for the symbol,
// not a device address: the address each device holds its copy at comes from
// hipGetSymbolAddress, once per device, and only that address is used.
// ---------------------------------------------------------------------------
constexpr size_t kNoAllocBytes = CLOVE_NOALLOC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kNoAllocBytes];
std::mutex g_noalloc_mu;
std::map<int, char*> g_noalloc_ptr;  // device -> address of its `scratch`

clove_status_t noalloc_scratch(hipStream_t stream, char** out) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    std::lock_guard<std::mutex> lk(g_noalloc_mu);
    auto it = g_noalloc_ptr.find(dev);
    if (it == g_noalloc_ptr.end()) {
        void* ptr = nullptr;
        if (hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)) != hipSuccess || ptr == nullptr)
            return CLOVE_ERR_NO_DEVICE;
        // the counters start at zero (every call leaves them zero again)
        hipLaunchKernelGGL(zero_u32, dim3(16), dim3(256), 0, stream, static_cast<unsigned*>(ptr), kWsCounters);
        if (hipGetLastError() != hipSuccess) return CLOVE_ERR_LAUNCH;
        it = g_noalloc_ptr.emplace(dev, static_cast<char*>(ptr)).first;
    }
    *out = it->second;
    return CLOVE_OK;
}

}  // namespace

bool dry_run() { return t_ws.mode == WsMode::kQuery; }

clove_status_t current_device_info(DeviceInfo* out) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    std::lock_guard<std::mutex> lk(g_dev_mu);
    auto it = g_num_cus.find(dev);
    if (it == g_num_cus.end()) {
        int cus = 0;
        if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess ||
            cus <= 0)
            return CLOVE_ERR_NO_DEVICE;
        it = g_num_cus.emplace(dev, cus).first;
    }
    out->device = dev;
    out->num_cus = it->second;
    return CLOVE_OK;
}

clove_status_t acquire_scratch(hipStream_t stream, size_t partial_bytes, size_t num_counters,
                               Scratch* out, bool optional) {
    if (t_ws.mode != WsMode::kLibrary) {
        if (num_counters > kWsCounters) return CLOVE_ERR_WORKSPACE;
        char* part = nullptr;
        const clove_status_t st = ws_carve(partial_bytes, &part);
        if (st != CLOVE_OK) return st;
        out->partials = reinterpret_cast<float*>(part);
        out->partial_bytes = round256(partial_bytes);
        out->counters = reinterpret_cast<unsigned*>(t_ws.ptr);
        out->num_counters = kWsCounters;
        return CLOVE_OK;
    }
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    hold_stream(dev, stream);
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    ScratchEntry& e = g_scratch[{dev, reinterpret_cast<void*>(stream)}];
    if (e.base && e.view.partial_bytes >= partial_bytes && e.view.num_counters >= num_counters) {
        *out = e.view;
        return CLOVE_OK;
    }
    if (optional) {
        hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
        const bool known = hipStreamIsCapturing(stream, &cap) == hipSuccess;
        if (!known) (void)hipGetLastError();
        if (!known || cap != hipStreamCaptureStatusNone) return CLOVE_ERR_OUT_OF_MEMORY;
    }
    const size_t pb = round_up_pow2(partial_bytes, (size_t)4 << 20);
    const size_t nc = round_up_pow2(num_counters, 4096);
    void* base = nullptr;
    if (!device_malloc(&base, pb + nc * sizeof(unsigned))) return CLOVE_ERR_OUT_OF_MEMORY;
    if (e.base) {
        // queued work (and calls of other host threads) may still use the old buffer
        g_retired[dev].push_back(e.base);
        e = ScratchEntry{};
    }
    unsigned* counters = reinterpret_cast<unsigned*>(static_cast<char*>(base) + pb);
    hipLaunchKernelGGL(zero_u32, dim3(64), dim3(256), 0, stream, counters, nc);
    if (hipGetLastError() != hipSuccess) {
        (void)hipFree(base);
        return CLOVE_ERR_LAUNCH;
    }
    e.base = base;
    e.view.partials = static_cast<float*>(base);
    e.view.partial_bytes = pb;
    e.view.counters = counters;
    e.view.num_counters = nc;
    *out = e.view;
    return CLOVE_OK;
}

clove_status_t acquire_buffer(hipStream_t stream, int slot, size_t bytes, void** out) {
    if (t_ws.mode != WsMode::kLibrary) {
        char* p = nullptr;
        const clove_status_t st = ws_carve(bytes, &p);
        *out = p;
        return st;
    }
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    hold_stream(dev, stream);
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    BufferEntry& e = g_buffers[std::make_tuple(dev, reinterpret_cast<void*>(stream), slot)];
    if (e.base && e.bytes >= bytes) {
        *out = e.base;
        return CLOVE_OK;
    }
    const size_t nb = round_up_pow2(bytes, (size_t)1 << 20);
    void* base = nullptr;
    if (!device_malloc(&base, nb)) return CLOVE_ERR_OUT_OF_MEMORY;
    if (e.base) g_retired[dev].push_back(e.base);  // as in acquire_scratch
    e.base = base;
    e.bytes = nb;
    *out = e.base;
    return CLOVE_OK;
}

}  // namespace clove

using namespace clove;

extern "C" {

const char* clove_status_string(clove_status_t status) {
    switch (status) {
        case CLOVE_OK: return "CLOVE_OK";
        case CLOVE_ERR_NULL_POINTER: return "CLOVE_ERR_NULL_POINTER: a required pointer is NULL";
        case CLOVE_ERR_INVALID_DIM: return "CLOVE_ERR_INVALID_DIM: a dimension is negative or too large";
        case CLOVE_ERR_INVALID_ARG: return "CLOVE_ERR_INVALID_ARG: invalid argument (odd K for INT4, mode, alignment)";
        case CLOVE_ERR_ALIASING: return "CLOVE_ERR_ALIASING: output overlaps an input";
        case CLOVE_ERR_OUT_OF_MEMORY: return "CLOVE_ERR_OUT_OF_MEMORY: scratch allocation failed";
        case CLOVE_ERR_LAUNCH: return "CLOVE_ERR_LAUNCH: kernel launch failed";
        case CLOVE_ERR_NO_DEVICE: return "CLOVE_ERR_NO_DEVICE: no usable HIP device";
        case CLOVE_ERR_WORKSPACE: return "CLOVE_ERR_WORKSPACE: the bound workspace is too small for the call";
        case CLOVE_ERR_SCRATCH_LIMIT:
            return "CLOVE_ERR_SCRATCH_LIMIT: the call needs more scratch than the fixed array of "
                   "clove_gemm_fp16_noalloc holds (CLOVE_NOALLOC_SCRATCH_BYTES)";
    }
    return "CLOVE_ERR_UNKNOWN";
}

int clove_abi_version(void) { return kAbiVersion; }

clove_status_t clove_gemm_fp16_batched(const void* A, const void* B, void* C, int batch, int M,
                                       int N, int K, float alpha, float beta, void* stream) {
    CallScope scope;
    if (batch < 0 || M < 0 || N < 0 || K < 0) return CLOVE_ERR_INVALID_DIM;
    if (batch == 0 || M == 0 || N == 0) return CLOVE_OK;
    if (!C || (K > 0 && (!A || !B))) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(A) || !aligned2(B) || !aligned2(C)) return CLOVE_ERR_INVALID_ARG;
    const size_t bc = (size_t)batch * M * N * 2;
    if (overlaps(C, bc, A, (size_t)batch * M * K * 2) || overlaps(C, bc, B, (size_t)batch * K * N * 2))
        return CLOVE_ERR_ALIASING;
    if ((int64_t)batch * (int64_t)cdiv64(M, 32) * (int64_t)cdiv64(N, 128) > 0x3fffffff)
        return CLOVE_ERR_INVALID_DIM;
    return launch_gemm_fp16(static_cast<const uint16_t*>(A), static_cast<const uint16_t*>(B),
                            static_cast<uint16_t*>(C), batch, M, N, K, alpha, beta,
                            static_cast<hipStream_t>(stream));
}

clove_status_t clove_gemm_fp16(const void* A, const void* B, void* C, int M, int N, int K,
                               float alpha, float beta, void* stream) {
    return clove_gemm_fp16_batched(A, B, C, 1, M, N, K, alpha, beta, stream);
}

clove_status_t clove_gemm_fp16_noalloc(const void* A, const void* B, void* C, int M, int N, int K,
                                       float alpha, float beta, void* stream) {
    if (t_ws.mode == WsMode::kQuery) {
        // plan and validate as clove_gemm_fp16, and report a call the fixed
        // array cannot hold as the real call would; the array is not the
        // caller's workspace, so the query's size is left as it was
        const size_t need = t_ws.need;
        t_ws.need = 0;
        clove_status_t st = clove_gemm_fp16(A, B, C, M, N, K, alpha, beta, stream);
        if (st == CLOVE_OK && t_ws.need > kNoAllocBytes) st = CLOVE_ERR_SCRATCH_LIMIT;
        t_ws.need = need;
        return st;
    }
    char* ptr = nullptr;
    clove_status_t st = noalloc_scratch(static_cast<hipStream_t>(stream), &ptr);
    if (st != CLOVE_OK) return st;
    // the call runs with this thread's workspace bound to the array, then the
    // thread's own mode is restored
    const ThreadWs saved = t_ws;
    t_ws = ThreadWs{};
    t_ws.mode = WsMode::kBound;
    t_ws.ptr = ptr;
    t_ws.bytes = kNoAllocBytes;
    st = clove_gemm_fp16(A, B, C, M, N, K, alpha, beta, stream);
    t_ws = saved;
    return st == CLOVE_ERR_WORKSPACE ? CLOVE_ERR_SCRATCH_LIMIT : st;
}

static clove_status_t int8_common(Int8Args& a, void* stream) {
    CallScope scope;
    if (a.M < 0 || a.N < 0 || a.K < 0) return CLOVE_ERR_INVALID_DIM;
    if (a.M == 0 || a.N == 0) return CLOVE_OK;
    if (!a.C || (a.K > 0 && (!a.A || !a.B))) return CLOVE_ERR_NULL_POINTER;
    const size_t out_elt = a.out == Int8Out::kAcc32 ? 4 : 2;
    if (a.out == Int8Out::kAcc32 ? (reinterpret_cast<uintptr_t>(a.C) & 3u) != 0 : !aligned2(a.C))
        return CLOVE_ERR_INVALID_ARG;
    const size_t bc = (size_t)a.M * a.N * out_elt;
    if (overlaps(a.C, bc, a.A, (size_t)a.M * a.K) || overlaps(a.C, bc, a.B, (size_t)a.K * a.N))
        return CLOVE_ERR_ALIASING;
    if (a.out == Int8Out::kHalfRowCol) {
        if (!a.sa || !a.sb) return CLOVE_ERR_NULL_POINTER;
        if (!aligned2(a.sa) || !aligned2(a.sb)) return CLOVE_ERR_INVALID_ARG;
        if (overlaps(a.C, bc, a.sa, (size_t)a.M * 2) || overlaps(a.C, bc, a.sb, (size_t)a.N * 2))
            return CLOVE_ERR_ALIASING;
    }
    return launch_gemm_int8(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_gemm_int8(const int8_t* A_q, const int8_t* B_q, void* C, int M, int N, int K,
                               float A_scale, int8_t A_zero, float B_scale, int8_t B_zero,
                               void* stream) {
    Int8Args a;
    a.A = A_q; a.B = B_q; a.C = C; a.M = M; a.N = N; a.K = K;
    a.scale = A_scale * B_scale;  // combined in fp32 (src/kernels/gemm_int8.cu:40)
    a.za = A_zero; a.zb = B_zero;
    a.out = Int8Out::kHalfPerTensor;
    return int8_common(a, stream);
}

clove_status_t clove_gemm_int8_ex(const int8_t* A_q, const int8_t* B_q, void* C, int M, int N, int K,
                                  float A_scale, int8_t A_zero, float B_scale, int8_t B_zero, int mode,
                                  void* stream) {
    if (mode != CLOVE_INT8_EXACT && mode != CLOVE_INT8_REFERENCE_LITERAL) return CLOVE_ERR_INVALID_ARG;
    Int8Args a;
    a.A = A_q; a.B = B_q; a.C = C; a.M = M; a.N = N; a.K = K;
    a.scale = A_scale * B_scale;  // combined in fp32 (src/kernels/gemm_int8.cu:40)
    a.za = A_zero; a.zb = B_zero;
    if (mode == CLOVE_INT8_REFERENCE_LITERAL && K > 0) {
        // the reference walks K in 32-wide tiles, loads 0 past K and subtracts
        // the zero points from it (src/kernels/gemm_int8.cu:43, 52-54, 63-64,
        // 89-93): each padded k adds za * zb
        const unsigned pad = (unsigned)(32 * ((K + 31) / 32) - K);
        a.acc_add = (int)(pad * (unsigned)(int)A_zero * (unsigned)(int)B_zero);
    }
    a.out = Int8Out::kHalfPerTensor;
    return int8_common(a, stream);
}

clove_status_t clove_gemm_int8_rowcol(const int8_t* A_q, const int8_t* B_q, const void* A_scale,
                                      const void* B_scale, void* C, int M, int N, int K,
                                      int8_t A_zero, int8_t B_zero, void* stream) {
    Int8Args a;
    a.A = A_q; a.B = B_q; a.C = C; a.M = M; a.N = N; a.K = K;
    a.sa = static_cast<const uint16_t*>(A_scale);
    a.sb = static_cast<const uint16_t*>(B_scale);
    a.za = A_zero; a.zb = B_zero;
    a.out = Int8Out::kHalfRowCol;
    return int8_common(a, stream);
}

clove_status_t clove_gemm_int8_acc32(const int8_t* A_q, const int8_t* B_q, int32_t* acc, int M,
                                     int N, int K, int8_t A_zero, int8_t B_zero, void* stream) {
    Int8Args a;
    a.A = A_q; a.B = B_q; a.C = acc; a.M = M; a.N = N; a.K = K;
    a.za = A_zero; a.zb = B_zero;
    a.out = Int8Out::kAcc32;
    return int8_common(a, stream);
}

clove_status_t clove_gemm_int4_ex(const uint8_t* A_q, const void* A_scale, const void* A_zero,
                                  const uint8_t* B_q, const void* B_scale, const void* B_zero,
                                  void* C, int M, int N, int K, clove_int4_mode_t mode,
                                  void* stream) {
    CallScope scope;
    if (mode != CLOVE_INT4_GROUPWISE && mode != CLOVE_INT4_REFERENCE_LITERAL)
        return CLOVE_ERR_INVALID_ARG;
    if (M < 0 || N < 0 || K < 0) return CLOVE_ERR_INVALID_DIM;
    if (K % 2 != 0) return CLOVE_ERR_INVALID_ARG;
    if (M == 0 || N == 0) return CLOVE_OK;
    const bool literal = mode == CLOVE_INT4_REFERENCE_LITERAL;
    if (!C) return CLOVE_ERR_NULL_POINTER;
    if (K > 0) {
        if (!A_q || !A_scale || !B_scale) return CLOVE_ERR_NULL_POINTER;
        if (!literal && (!A_zero || !B_zero || !B_q)) return CLOVE_ERR_NULL_POINTER;
        if (literal && N >= 2 && !B_q) return CLOVE_ERR_NULL_POINTER;
    }
    if (!aligned2(C) || !aligned2(A_scale) || !aligned2(B_scale) || !aligned2(A_zero) ||
        !aligned2(B_zero))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t G = cdiv64(K, 128);
    const size_t bc = (size_t)M * N * 2;
    const size_t bstride = literal ? (size_t)(N / 2) : (size_t)((N + 1) / 2);
    if (overlaps(C, bc, A_q, (size_t)M * (K / 2)) || overlaps(C, bc, B_q, (size_t)K * bstride) ||
        overlaps(C, bc, A_scale, (size_t)M * G * 2) || overlaps(C, bc, B_scale, (size_t)G * N * 2) ||
        (!literal && (overlaps(C, bc, A_zero, (size_t)M * G * 2) ||
                      overlaps(C, bc, B_zero, (size_t)G * N * 2))))
        return CLOVE_ERR_ALIASING;
    Int4Args a;
    a.A = A_q;
    a.A_scale = static_cast<const uint16_t*>(A_scale);
    a.A_zero = static_cast<const uint16_t*>(A_zero);
    a.B = B_q;
    a.B_scale = static_cast<const uint16_t*>(B_scale);
    a.B_zero = static_cast<const uint16_t*>(B_zero);
    a.C = static_cast<uint16_t*>(C);
    a.M = M; a.N = N; a.K = K;
    a.mode = mode;
    return launch_gemm_int4(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_gemm_int4(const uint8_t* A_q, const void* A_scale, const void* A_zero,
                               const uint8_t* B_q, const void* B_scale, const void* B_zero,
                               void* C, int M, int N, int K, void* stream) {
    return clove_gemm_int4_ex(A_q, A_scale, A_zero, B_q, B_scale, B_zero, C, M, N, K,
                              CLOVE_INT4_GROUPWISE, stream);
}

clove_status_t clove_gemm_int4_group_acc32(const uint8_t* A_q, const void* A_zero, const uint8_t* B_q,
                                           const void* B_zero, int32_t* P, int M, int N, int K,
                                           void* stream) {
    CallScope scope;
    if (M < 0 || N < 0 || K < 0) return CLOVE_ERR_INVALID_DIM;
    if (M == 0 || N == 0 || K == 0) return CLOVE_OK;
    if (!A_q || !A_zero || !B_q || !B_zero || !P) return CLOVE_ERR_NULL_POINTER;
    if (K % 256 != 0 || !aligned16(A_q) || !aligned4(P) || !aligned2(A_zero) || !aligned2(B_zero))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t G = K / 128;
    const size_t bp = (size_t)M * N * G * 4;
    if (overlaps(P, bp, A_q, (size_t)M * (K / 2)) || overlaps(P, bp, B_q, (size_t)K * ((N + 1) / 2)) ||
        overlaps(P, bp, A_zero, (size_t)M * G * 2) || overlaps(P, bp, B_zero, (size_t)G * N * 2))
        return CLOVE_ERR_ALIASING;
    DeviceInfo dev;
    clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    Int4Args a;
    a.A = A_q;
    a.A_zero = static_cast<const uint16_t*>(A_zero);
    a.B = B_q;
    a.B_zero = static_cast<const uint16_t*>(B_zero);
    a.M = M; a.N = N; a.K = K;
    return launch_i4i4_partials(a, P, dev.num_cus, static_cast<hipStream_t>(stream));
}

clove_status_t clove_gemm_w4a16(const void* X, const uint8_t* W_q, const void* W_scale,
                                const void* W_zero, void* Y, int T, int O, int K, float alpha,
                                float beta, void* stream) {
    CallScope scope;
    if (T < 0 || O < 0 || K < 0) return CLOVE_ERR_INVALID_DIM;
    if (K % 2 != 0) return CLOVE_ERR_INVALID_ARG;
    if (T == 0 || O == 0) return CLOVE_OK;
    if (!Y || (K > 0 && (!X || !W_q || !W_scale || !W_zero))) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(X) || !aligned2(Y) || !aligned2(W_scale) || !aligned2(W_zero))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t G = cdiv64(K, 128);
    const size_t by = (size_t)T * O * 2;
    if (overlaps(Y, by, X, (size_t)T * K * 2) || overlaps(Y, by, W_q, (size_t)O * (K / 2)) ||
        overlaps(Y, by, W_scale, (size_t)O * G * 2) || overlaps(Y, by, W_zero, (size_t)O * G * 2))
        return CLOVE_ERR_ALIASING;
    W4A16Args a;
    a.X = static_cast<const uint16_t*>(X);
    a.W = W_q;
    a.scale = static_cast<const uint16_t*>(W_scale);
    a.zero = static_cast<const uint16_t*>(W_zero);
    a.Y = static_cast<uint16_t*>(Y);
    a.T = T; a.O = O; a.K = K;
    a.alpha = alpha; a.beta = beta;
    return launch_w4a16(a, static_cast<hipStream_t>(stream));
}

static bool same_or_disjoint(const void* a, const void* b, size_t bytes) {
    return a == b || !overlaps(a, bytes, b, bytes);
}

clove_status_t clove_swiglu(const void* gate, const void* up, void* output, int size, void* stream) {
    CallScope scope;
    if (size < 0) return CLOVE_ERR_INVALID_DIM;
    if (size == 0) return CLOVE_OK;
    if (!gate || !up || !output) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(gate) || !aligned2(up) || !aligned2(output)) return CLOVE_ERR_INVALID_ARG;
    // elementwise: the output may be one of the inputs, but not shifted against it
    const size_t b = (size_t)size * 2;
    if (!same_or_disjoint(output, gate, b) || !same_or_disjoint(output, up, b)) return CLOVE_ERR_ALIASING;
    return launch_swiglu(static_cast<const uint16_t*>(gate), static_cast<const uint16_t*>(up),
                         static_cast<uint16_t*>(output), size, static_cast<hipStream_t>(stream));
}

clove_status_t clove_swiglu_fused(const void* input, const void* W_gate, const void* W_up, void* output,
                                  int batch_seq, int hidden_dim, int intermediate_dim, void* stream) {
    CallScope scope;
    const int T = batch_seq, H = hidden_dim, I = intermediate_dim;
    if (T < 0 || H < 0 || I < 0) return CLOVE_ERR_INVALID_DIM;
    if (T == 0 || I == 0) return CLOVE_OK;
    if (!output || (H > 0 && (!input || !W_gate || !W_up))) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(input) || !aligned2(W_gate) || !aligned2(W_up) || !aligned2(output))
        return CLOVE_ERR_INVALID_ARG;
    const size_t bo = (size_t)T * I * 2;
    if (overlaps(output, bo, input, (size_t)T * H * 2) || overlaps(output, bo, W_gate, (size_t)H * I * 2) ||
        overlaps(output, bo, W_up, (size_t)H * I * 2))
        return CLOVE_ERR_ALIASING;
    if ((int64_t)cdiv64(T, 32) * (int64_t)cdiv64(I, 128) > 0x3fffffff) return CLOVE_ERR_INVALID_DIM;
    return launch_swiglu_fused_fp16(static_cast<const uint16_t*>(input), static_cast<const uint16_t*>(W_gate),
                                    static_cast<const uint16_t*>(W_up), static_cast<uint16_t*>(output), T, H,
                                    I, static_cast<hipStream_t>(stream));
}

clove_status_t clove_w4a16_swiglu(const void* X, const uint8_t* W_q, const void* W_scale,
                                  const void* W_zero, void* H, int T, int I, int K, void* stream) {
    CallScope scope;
    if (T < 0 || I < 0 || K < 0) return CLOVE_ERR_INVALID_DIM;
    if (K % 2 != 0) return CLOVE_ERR_INVALID_ARG;
    if (T == 0 || I == 0) return CLOVE_OK;
    if (!H || (K > 0 && (!X || !W_q || !W_scale || !W_zero))) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(X) || !aligned2(H) || !aligned2(W_scale) || !aligned2(W_zero)) return CLOVE_ERR_INVALID_ARG;
    if ((int64_t)2 * I > 0x7fffffff) return CLOVE_ERR_INVALID_DIM;
    const int64_t G = cdiv64(K, 128);
    const size_t bh = (size_t)T * I * 2;
    if (overlaps(H, bh, X, (size_t)T * K * 2) || overlaps(H, bh, W_q, (size_t)2 * I * (K / 2)) ||
        overlaps(H, bh, W_scale, (size_t)2 * I * G * 2) || overlaps(H, bh, W_zero, (size_t)2 * I * G * 2))
        return CLOVE_ERR_ALIASING;
    hipStream_t s = static_cast<hipStream_t>(stream);
    if (K == 0) {  // gate = up = 0: swiglu(0, 0) = +0
        CLOVE_LAUNCH(zero_u16, dim3(256), dim3(256), 0, s, static_cast<uint16_t*>(H), (size_t)T * I);
        return check_launch();
    }
    W4A16Args a;
    a.X = static_cast<const uint16_t*>(X);
    a.W = W_q;
    a.scale = static_cast<const uint16_t*>(W_scale);
    a.zero = static_cast<const uint16_t*>(W_zero);
    a.Y = static_cast<uint16_t*>(H);
    a.T = T; a.O = I; a.K = K;
    return launch_w4a16_swiglu(a, s);
}

// The descriptor of a cache checked and laid out for kernels.
static clove_status_t read_cache(const clove_kv_cache_t* c, PagedCache* out) {
    if (c->dtype != CLOVE_DTYPE_FP16 && c->dtype != CLOVE_DTYPE_BF16) return CLOVE_ERR_INVALID_ARG;
    if (c->num_pages < 0 || c->page_size <= 0 || c->kv_heads <= 0 || c->kv_heads > 0x10000 ||
        c->head_dim <= 0 || c->head_dim > CLOVE_MAX_HEAD_DIM)
        return CLOVE_ERR_INVALID_DIM;
    const int64_t rows = (int64_t)c->kv_heads * c->page_size;
    if (rows > ((int64_t)1 << 40) / c->head_dim) return CLOVE_ERR_INVALID_DIM;
    const int64_t dense = rows * c->head_dim;
    if (c->page_stride != 0 && c->page_stride < dense) return CLOVE_ERR_INVALID_ARG;
    if (c->num_pages > 0 && (!c->k || !c->v)) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(c->k) || !aligned2(c->v)) return CLOVE_ERR_INVALID_ARG;
    out->k = static_cast<uint16_t*>(c->k);
    out->v = static_cast<uint16_t*>(c->v);
    out->page_stride = c->page_stride ? c->page_stride : dense;
    out->num_pages = c->num_pages;
    out->page_size = c->page_size;
    out->kv_heads = c->kv_heads;
    out->head_dim = c->head_dim;
    out->dtype = c->dtype;
    return CLOVE_OK;
}

static Rows cache_rows(const PagedCache& c, const void* p) {
    return Rows{p, c.page_stride * 2, (int64_t)c.kv_heads * c.page_size * c.head_dim * 2, c.num_pages};
}

// The entries of a table's row, which may be part of a wider one
static int64_t table_bytes(int max_context, const PagedCache& c) { return hw::cdiv64(max_context, c.page_size) * 4; }

clove_status_t clove_qk_norm_rope(const void* qkv, int64_t qkv_stride, const void* q_weight, const void* k_weight,
                                  float eps, const float* rope_cos, const float* rope_sin, int max_position,
                                  const int32_t* positions, void* q_out, int64_t q_out_stride, void* k_out,
                                  int64_t k_out_stride, const clove_kv_cache_t* cache, const int32_t* slots, int T,
                                  int q_heads, int kv_heads, int head_dim, int rot_dim, int interleaved, int dtype,
                                  void* stream) {
    CallScope scope;
    if (dtype != CLOVE_DTYPE_FP16 && dtype != CLOVE_DTYPE_BF16) return CLOVE_ERR_INVALID_ARG;
    if (T < 0 || q_heads < 0 || kv_heads < 0 || head_dim < 1 || head_dim > CLOVE_MAX_HEAD_DIM || rot_dim < 0 ||
        max_position < 0 || q_heads > 0x10000 || kv_heads > 0x10000)
        return CLOVE_ERR_INVALID_DIM;
    if (rot_dim > head_dim || rot_dim % 2 != 0) return CLOVE_ERR_INVALID_ARG;
    const int64_t qw = (int64_t)q_heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    if (T == 0 || q_heads + kv_heads == 0) return CLOVE_OK;
    if (!qkv || (q_heads > 0 && !q_out)) return CLOVE_ERR_NULL_POINTER;
    if (rot_dim > 0 && (!positions || (max_position > 0 && (!rope_cos || !rope_sin)))) return CLOVE_ERR_NULL_POINTER;
    if (qkv_stride < qw + 2 * kw || (q_heads > 0 && q_out_stride < qw) || (k_out && k_out_stride < kw))
        return CLOVE_ERR_INVALID_ARG;
    if (!aligned2(qkv) || !aligned2(q_weight) || !aligned2(k_weight) || !aligned2(q_out) || !aligned2(k_out) ||
        !aligned4(rope_cos) || !aligned4(rope_sin) || !aligned4(positions) || !aligned4(slots))
        return CLOVE_ERR_INVALID_ARG;
    RopeArgs a;
    if (cache) {
        const clove_status_t st = read_cache(cache, &a.cache);
        if (st != CLOVE_OK) return st;
        if (cache->dtype != dtype || cache->kv_heads != kv_heads || cache->head_dim != head_dim) return CLOVE_ERR_INVALID_ARG;
        if (!slots) return CLOVE_ERR_NULL_POINTER;
        if (cache->num_pages == 0) a.cache.k = a.cache.v = nullptr;
    }
    // outputs against inputs: the queries / keys of qkv may be their own output
    const char* x = static_cast<const char*>(qkv);
    const Rows in[] = {{x, qkv_stride * 2, qw * 2, T}, {x + qw * 2, qkv_stride * 2, kw * 2, T},
                       {x + (qw + kw) * 2, qkv_stride * 2, kw * 2, T}};
    const Rows outs[] = {{q_heads > 0 ? q_out : nullptr, q_out_stride * 2, qw * 2, T}, {k_out, k_out_stride * 2, kw * 2, T},
                         cache_rows(a.cache, a.cache.k), cache_rows(a.cache, a.cache.v)};
    const int64_t half = rot_dim / 2;
    const Rows small[] = {{q_weight, 0, head_dim * 2, 1}, {k_weight, 0, head_dim * 2, 1},
                          {rope_cos, 0, max_position * half * 4, 1}, {rope_sin, 0, max_position * half * 4, 1},
                          {positions, 0, (int64_t)T * 4, 1}, {slots, 0, (int64_t)T * 4, 1}};
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 3; ++i) {
            const bool own = o == i && same_rows(outs[o], in[i]);
            if (!own && overlaps(outs[o], in[i])) return CLOVE_ERR_ALIASING;
        }
        for (const Rows& r : small)
            if (overlaps(outs[o], r)) return CLOVE_ERR_ALIASING;
        for (int i = 0; i < o; ++i)
            if (overlaps(outs[o], outs[i])) return CLOVE_ERR_ALIASING;
    }
    a.qkv = static_cast<const uint16_t*>(qkv);
    a.qkv_stride = qkv_stride;
    a.q_weight = static_cast<const uint16_t*>(q_weight);
    a.k_weight = static_cast<const uint16_t*>(k_weight);
    a.eps = eps;
    a.cos = rope_cos;
    a.sin = rope_sin;
    a.max_position = max_position;
    a.positions = positions;
    a.q_out = static_cast<uint16_t*>(q_out);
    a.q_out_stride = q_out_stride;
    a.k_out = static_cast<uint16_t*>(k_out);
    a.k_out_stride = k_out_stride;
    a.slots = slots;
    a.T = T; a.q_heads = q_heads; a.kv_heads = kv_heads; a.head_dim = head_dim; a.rot_dim = rot_dim;
    a.interleaved = interleaved != 0;
    a.dtype = dtype;
    return launch_qk_norm_rope(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_paged_attention(const void* q, int64_t q_stride, const clove_kv_cache_t* cache,
                                     const int32_t* block_table, int64_t table_stride, const int32_t* context_lens,
                                     void* out, int64_t out_stride, float* weights, int64_t weights_stride, int batch,
                                     int q_heads, int max_context, float scale, float softcap, int window,
                                     void* stream) {
    CallScope scope;
    if (!cache) return CLOVE_ERR_NULL_POINTER;
    PagedAttentionArgs a;
    const clove_status_t st = read_cache(cache, &a.cache);
    if (st != CLOVE_OK) return st;
    if (batch < 0 || q_heads < 0 || max_context < 0 || window < 0 || table_stride < 0) return CLOVE_ERR_INVALID_DIM;
    if (q_heads % a.cache.kv_heads != 0 || !(softcap >= 0.0f)) return CLOVE_ERR_INVALID_ARG;
    if (batch == 0 || q_heads == 0) return CLOVE_OK;
    if (!q || !out || !context_lens || (max_context > 0 && !block_table)) return CLOVE_ERR_NULL_POINTER;
    const int64_t width = (int64_t)q_heads * a.cache.head_dim;
    if (q_stride < width || out_stride < width || (weights && weights_stride < max_context) ||
        (int64_t)max_context > table_stride * a.cache.page_size)
        return CLOVE_ERR_INVALID_ARG;
    if (max_context > CLOVE_MAX_CONTEXT || (int64_t)batch * q_heads > 0x1000000 ||
        (weights && batch * hw::cdiv64(max_context, 64) > 0x7fffffff))
        return CLOVE_ERR_INVALID_DIM;
    if (!aligned2(q) || !aligned2(out) || !aligned4(block_table) || !aligned4(context_lens) || !aligned4(weights))
        return CLOVE_ERR_INVALID_ARG;
    const Rows in[] = {{q, q_stride * 2, width * 2, batch}, cache_rows(a.cache, a.cache.k), cache_rows(a.cache, a.cache.v),
                       {block_table, table_stride * 4, table_bytes(max_context, a.cache), batch}, {context_lens, 0, (int64_t)batch * 4, 1}};
    const Rows outs[] = {{out, out_stride * 2, width * 2, batch}, {weights, weights_stride * 4, (int64_t)max_context * 4, batch}};
    for (const Rows& o : outs)
        for (const Rows& i : in)
            if (overlaps(o, i)) return CLOVE_ERR_ALIASING;
    if (overlaps(outs[0], outs[1])) return CLOVE_ERR_ALIASING;
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.block_table = block_table;
    a.table_stride = table_stride;
    a.context_lens = context_lens;
    a.out = static_cast<uint16_t*>(out);
    a.out_stride = out_stride;
    a.weights = weights;
    a.weights_stride = weights_stride;
    a.batch = batch; a.q_heads = q_heads; a.max_context = max_context;
    a.scale = scale;
    a.softcap = softcap;
    a.window = window;
    return launch_paged_attention(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_cache_evict(const clove_kv_cache_t* cache, const int32_t* block_table, int64_t table_stride,
                                 const int32_t* context_lens, const float* weights, int64_t weights_stride,
                                 const int32_t* positions, int64_t positions_stride, float* weights_out,
                                 int64_t weights_out_stride, int32_t* positions_out, int64_t positions_out_stride,
                                 int32_t* lens_out, int batch, int max_context, int budget, int sinks, int recent,
                                 void* stream) {
    CallScope scope;
    if (!cache) return CLOVE_ERR_NULL_POINTER;
    EvictArgs a;
    const clove_status_t st = read_cache(cache, &a.cache);
    if (st != CLOVE_OK) return st;
    if (batch < 0 || batch > 0x10000 || max_context < 0 || max_context > CLOVE_MAX_CONTEXT || budget < 0 || sinks < 0 || recent < 0 || table_stride < 0)
        return CLOVE_ERR_INVALID_DIM;
    if (batch == 0) return CLOVE_OK;
    if (!context_lens || !lens_out) return CLOVE_ERR_NULL_POINTER;
    if (max_context > 0 && (!block_table || !weights || !positions || !weights_out || !positions_out))
        return CLOVE_ERR_NULL_POINTER;
    if ((int64_t)max_context > table_stride * a.cache.page_size || weights_stride < max_context ||
        positions_stride < max_context || weights_out_stride < max_context || positions_out_stride < max_context)
        return CLOVE_ERR_INVALID_ARG;
    if (!aligned4(block_table) || !aligned4(context_lens) || !aligned4(weights) || !aligned4(positions) ||
        !aligned4(weights_out) || !aligned4(positions_out) || !aligned4(lens_out))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t row = (int64_t)max_context * 4, ints = (int64_t)batch * 4;
    const Rows in[] = {{weights, weights_stride * 4, row, batch}, {positions, positions_stride * 4, row, batch},
                       {context_lens, 0, ints, 1}, {block_table, table_stride * 4, table_bytes(max_context, a.cache), batch}};
    const Rows outs[] = {{weights_out, weights_out_stride * 4, row, batch},
                         {positions_out, positions_out_stride * 4, row, batch},
                         {lens_out, 0, ints, 1},
                         cache_rows(a.cache, a.cache.k),
                         cache_rows(a.cache, a.cache.v)};
    for (int o = 0; o < 5; ++o) {
        for (int i = 0; i < 4; ++i) {
            const bool own = o == i && same_rows(outs[o], in[i]);
            if (!own && overlaps(outs[o], in[i])) return CLOVE_ERR_ALIASING;
        }
        for (int i = 0; i < o; ++i)
            if (overlaps(outs[o], outs[i])) return CLOVE_ERR_ALIASING;
    }
    a.block_table = block_table;
    a.table_stride = table_stride;
    a.context_lens = context_lens;
    a.weights = weights;
    a.weights_stride = weights_stride;
    a.positions = positions;
    a.positions_stride = positions_stride;
    a.weights_out = weights_out;
    a.weights_out_stride = weights_out_stride;
    a.positions_out = positions_out;
    a.positions_out_stride = positions_out_stride;
    a.lens_out = lens_out;
    a.batch = batch; a.max_context = max_context; a.budget = budget; a.sinks = sinks; a.recent = recent;
    return launch_cache_evict(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_penalize_logits(const void* logits, int64_t logits_stride, int dtype, void* out,
                                     int64_t out_stride, int out_dtype, int batch, int vocab, const int32_t* history,
                                     int64_t history_stride, const int32_t* history_lens, const int32_t* prompt_lens,
                                     const float* repetition, const float* presence, const float* frequency,
                                     const int32_t* bias_ids, const float* bias_values, int64_t bias_stride,
                                     const int32_t* bias_counts, const uint32_t* allowed, int64_t allowed_stride,
                                     void* stream) {
    CallScope scope;
    if (dtype < CLOVE_DTYPE_FP16 || dtype > CLOVE_DTYPE_FP32 || (out_dtype != dtype && out_dtype != CLOVE_DTYPE_FP32))
        return CLOVE_ERR_INVALID_ARG;
    if (batch < 0 || vocab < 0 || (history && history_stride < 0) || (bias_ids && bias_stride < 0)) return CLOVE_ERR_INVALID_DIM;
    if ((history && history_stride > 0x7fffffff) || (bias_ids && bias_stride > 0x7fffffff)) return CLOVE_ERR_INVALID_DIM;
    if (batch == 0 || vocab == 0) return CLOVE_OK;
    if (!logits || !out || (history && !history_lens) || (bias_ids && !bias_values)) return CLOVE_ERR_NULL_POINTER;
    const int64_t words = hw::cdiv64(vocab, 32);
    if (logits_stride < vocab || out_stride < vocab || (allowed && allowed_stride < words)) return CLOVE_ERR_INVALID_ARG;
    const int64_t is = dtype == CLOVE_DTYPE_FP32 ? 4 : 2, os = out_dtype == CLOVE_DTYPE_FP32 ? 4 : 2;
    if (!(is == 4 ? aligned4(logits) : aligned2(logits)) || !(os == 4 ? aligned4(out) : aligned2(out)) ||
        !aligned4(history) || !aligned4(history_lens) || !aligned4(prompt_lens) || !aligned4(repetition) ||
        !aligned4(presence) || !aligned4(frequency) || !aligned4(bias_ids) || !aligned4(bias_values) ||
        !aligned4(bias_counts) || !aligned4(allowed))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t per = (int64_t)batch * 4;
    const Rows o{out, out_stride * os, (int64_t)vocab * os, batch}, x{logits, logits_stride * is, (int64_t)vocab * is, batch};
    const bool own = os == is && same_rows(o, x);
    if (!own && overlaps(o, x)) return CLOVE_ERR_ALIASING;
    const Rows in[] = {{history, history_stride * 4, history_stride * 4, batch}, {history_lens, 0, per, 1},
                       {prompt_lens, 0, per, 1}, {repetition, 0, per, 1}, {presence, 0, per, 1}, {frequency, 0, per, 1},
                       {bias_ids, bias_stride * 4, bias_stride * 4, batch}, {bias_values, bias_stride * 4, bias_stride * 4, batch},
                       {bias_counts, 0, per, 1}, {allowed, allowed_stride * 4, words * 4, batch}};
    for (const Rows& i : in)
        if (overlaps(o, i)) return CLOVE_ERR_ALIASING;
    LogitsArgs a;
    a.logits = logits;
    a.logits_stride = logits_stride;
    a.dtype = dtype;
    a.out = out;
    a.out_stride = out_stride;
    a.out_dtype = out_dtype;
    a.batch = batch; a.vocab = vocab;
    a.history = history;
    a.history_stride = history_stride;
    a.history_lens = history_lens;
    a.prompt_lens = prompt_lens;
    a.repetition = repetition;
    a.presence = presence;
    a.frequency = frequency;
    a.bias_ids = bias_ids;
    a.bias_values = bias_values;
    a.bias_stride = bias_stride;
    a.bias_counts = bias_counts;
    a.allowed = allowed;
    a.allowed_stride = allowed_stride;
    return launch_penalize_logits(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_block_norm(const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                                const void* post_weight, const void* gate, int64_t gate_stride, float scale,
                                const void* pre_weight, void* y_out, int64_t y_out_stride, void* h_out,
                                int64_t h_out_stride, int T, int D, float eps, int dtype, int residual_dtype,
                                void* stream) {
    CallScope scope;
    if (dtype != CLOVE_DTYPE_FP16 && dtype != CLOVE_DTYPE_BF16) return CLOVE_ERR_INVALID_ARG;
    if (residual_dtype != dtype && residual_dtype != CLOVE_DTYPE_FP32) return CLOVE_ERR_INVALID_ARG;
    if (T < 0 || D < 0 || D > CLOVE_MAX_NORM_DIM) return CLOVE_ERR_INVALID_DIM;
    if (T == 0 || D == 0) return CLOVE_OK;
    if ((!x && !residual) || (!y_out && !h_out)) return CLOVE_ERR_NULL_POINTER;
    if ((x && x_stride < D) || (residual && residual_stride < D) || (gate && gate_stride != 0 && gate_stride < D) ||
        (y_out && y_out_stride < D) || (h_out && h_out_stride < D))
        return CLOVE_ERR_INVALID_ARG;
    const bool wide = residual_dtype == CLOVE_DTYPE_FP32;
    if (!aligned2(x) || !aligned2(gate) || !aligned2(post_weight) || !aligned2(pre_weight) || !aligned2(h_out) ||
        !(wide ? aligned4(residual) && aligned4(y_out) : aligned2(residual) && aligned2(y_out)))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t rs = wide ? 4 : 2;
    // (an output may be the input that each thread has read all of before it writes)
    struct In {
        Rows r;
        bool by_y, by_h;
    };
    const In in[] = {{{x, x_stride * 2, (int64_t)D * 2, T}, !wide, true},
                     {{residual, residual_stride * rs, D * rs, T}, true, !wide},
                     {{gate, gate_stride * 2, (int64_t)D * 2, gate_stride ? T : 1}, !wide && (gate_stride || T == 1),
                      gate_stride || T == 1},
                     {{post_weight, 0, (int64_t)D * 2, 1}, false, false},
                     {{pre_weight, 0, (int64_t)D * 2, 1}, false, false}};
    const Rows oy{y_out, y_out_stride * rs, D * rs, T}, oh{h_out, h_out_stride * 2, (int64_t)D * 2, T};
    for (const In& i : in) {
        if (overlaps(oy, i.r) && !(i.by_y && same_rows(oy, i.r))) return CLOVE_ERR_ALIASING;
        if (overlaps(oh, i.r) && !(i.by_h && same_rows(oh, i.r))) return CLOVE_ERR_ALIASING;
    }
    if (overlaps(oy, oh)) return CLOVE_ERR_ALIASING;
    BlockNormArgs a;
    a.x = x;
    a.x_stride = x_stride;
    a.residual = residual;
    a.residual_stride = residual_stride;
    a.post_weight = x ? post_weight : nullptr;
    a.gate = x ? gate : nullptr;
    a.gate_stride = gate_stride;
    a.scale = scale;
    a.pre_weight = pre_weight;
    a.y_out = y_out;
    a.y_out_stride = y_out_stride;
    a.h_out = h_out;
    a.h_out_stride = h_out_stride;
    a.T = T; a.D = D;
    a.eps = eps;
    a.dtype = dtype;
    a.residual_dtype = residual_dtype;
    return launch_block_norm(a, static_cast<hipStream_t>(stream));
}

clove_status_t clove_moe_route(const void* logits, int64_t logits_stride, int dtype, const float* bias, int score,
                               int groups, int top_groups, int group_top, int top_k, int renormalize, float scale,
                               int32_t* ids, float* weights, int T, int experts, void* stream) {
    CallScope scope;
    if (dtype < CLOVE_DTYPE_FP16 || dtype > CLOVE_DTYPE_FP32 ||
        (score != CLOVE_ROUTE_SOFTMAX && score != CLOVE_ROUTE_SIGMOID) || (group_top != 1 && group_top != 2))
        return CLOVE_ERR_INVALID_ARG;
    if (T < 0 || experts < 1 || experts > CLOVE_MAX_EXPERTS || top_k < 1 || top_k > CLOVE_MAX_TOP_K || groups < 1 ||
        top_groups < 1)
        return CLOVE_ERR_INVALID_DIM;
    if (top_k > experts || experts % groups != 0 || top_groups > groups || groups > 64) return CLOVE_ERR_INVALID_ARG;
    if (T == 0) return CLOVE_OK;
    if (!logits || !ids || !weights) return CLOVE_ERR_NULL_POINTER;
    if (logits_stride < experts) return CLOVE_ERR_INVALID_ARG;
    const int64_t es = dtype == CLOVE_DTYPE_FP32 ? 4 : 2;
    if (!(es == 4 ? aligned4(logits) : aligned2(logits)) || !aligned4(bias) || !aligned4(ids) || !aligned4(weights))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t out = (int64_t)T * top_k * 4;
    const Rows in[] = {{logits, logits_stride * es, experts * es, T}, {bias, 0, (int64_t)experts * 4, 1}};
    const Rows outs[] = {{ids, 0, out, 1}, {weights, 0, out, 1}};
    for (const Rows& o : outs)
        for (const Rows& i : in)
            if (overlaps(o, i)) return CLOVE_ERR_ALIASING;
    if (overlaps(outs[0], outs[1])) return CLOVE_ERR_ALIASING;
    RouteArgs a;
    a.logits = logits;
    a.logits_stride = logits_stride;
    a.dtype = dtype;
    a.bias = bias;
    a.score = score;
    a.groups = groups; a.top_groups = top_groups; a.group_top = group_top; a.top_k = top_k;
    a.renormalize = renormalize != 0;
    a.scale = scale;
    a.ids = ids;
    a.weights = weights;
    a.T = T; a.experts = experts;
    return launch_moe_route(a, static_cast<hipStream_t>(stream));
}

// Both products of a sparse MLP block (MoeArgs): `rows` weight rows an expert
static clove_status_t moe_common(MoeArgs& a, bool swiglu, void* stream) {
    CallScope scope;
    if (a.T < 0 || a.O < 0 || a.K < 0 || a.top_k < 1 || a.top_k > CLOVE_MAX_TOP_K || a.experts < 1 ||
        a.experts > CLOVE_MAX_EXPERTS)
        return CLOVE_ERR_INVALID_DIM;
    if (a.K % 2 != 0) return CLOVE_ERR_INVALID_ARG;
    if (a.T == 0 || a.O == 0) return CLOVE_OK;
    // (pairs, and rows in tiles that may end past the last one, are counted in 31 bits; a row of
    // weights is at most 2^30 bytes)
    const int64_t pairs = (int64_t)a.T * a.top_k, rows = (int64_t)a.O * (swiglu ? 2 : 1), G = cdiv64(a.K, 128);
    if (pairs > 0x3fffffff || rows > 0x7fff0000 || (pairs / 32 + a.experts + 1) * cdiv64(rows, 32) > 0x7fffffff)
        return CLOVE_ERR_INVALID_DIM;
    if (rows * (a.K / 2) > ((int64_t)1 << 50) / a.experts) return CLOVE_ERR_INVALID_DIM;
    if (!a.Y || !a.ids || (a.K > 0 && (!a.X || !a.W || !a.scale || !a.zero))) return CLOVE_ERR_NULL_POINTER;
    if (!aligned2(a.X) || !aligned2(a.Y) || !aligned2(a.scale) || !aligned2(a.zero) || !aligned4(a.ids) ||
        !aligned4(a.weights))
        return CLOVE_ERR_INVALID_ARG;
    const int64_t all = a.experts * rows;
    const Rows y{a.Y, 0, (swiglu ? pairs : a.T) * a.O * 2, 1};
    const Rows in[] = {{a.X, 0, (swiglu ? a.T : pairs) * a.K * 2, 1}, {a.ids, 0, pairs * 4, 1}, {a.weights, 0, pairs * 4, 1},
                       {a.W, 0, all * (a.K / 2), 1}, {a.scale, 0, all * G * 2, 1}, {a.zero, 0, all * G * 2, 1}};
    for (const Rows& i : in)
        if (overlaps(y, i)) return CLOVE_ERR_ALIASING;
    return launch_moe_w4a16(a, swiglu, static_cast<hipStream_t>(stream));
}

clove_status_t clove_moe_w4a16_swiglu(const void* X, const int32_t* expert_ids, const uint8_t* W_q,
                                      const void* W_scale, const void* W_zero, void* H, int T, int top_k, int experts,
                                      int I, int K, void* stream) {
    MoeArgs a;
    a.X = static_cast<const uint16_t*>(X);
    a.ids = expert_ids;
    a.W = W_q;
    a.scale = static_cast<const uint16_t*>(W_scale);
    a.zero = static_cast<const uint16_t*>(W_zero);
    a.Y = static_cast<uint16_t*>(H);
    a.T = T; a.top_k = top_k; a.experts = experts; a.O = I; a.K = K;
    return moe_common(a, true, stream);
}

clove_status_t clove_moe_w4a16(const void* H, const int32_t* expert_ids, const float* weights, const uint8_t* W_q,
                               const void* W_scale, const void* W_zero, void* Y, int T, int top_k, int experts, int O,
                               int K, float alpha, float beta, void* stream) {
    MoeArgs a;
    a.X = static_cast<const uint16_t*>(H);
    a.ids = expert_ids;
    a.weights = weights;
    a.W = W_q;
    a.scale = static_cast<const uint16_t*>(W_scale);
    a.zero = static_cast<const uint16_t*>(W_zero);
    a.Y = static_cast<uint16_t*>(Y);
    a.T = T; a.top_k = top_k; a.experts = experts; a.O = O; a.K = K;
    a.alpha = alpha; a.beta = beta;
    return moe_common(a, false, stream);
}

clove_status_t clove_workspace_bind(void* ptr, size_t bytes) {
    if (t_ws.mode == WsMode::kQuery) return CLOVE_ERR_INVALID_ARG;
    if (!ptr) {
        if (bytes != 0) return CLOVE_ERR_NULL_POINTER;
        t_ws = ThreadWs{};
        return CLOVE_OK;
    }
    if ((reinterpret_cast<uintptr_t>(ptr) & 255u) != 0) return CLOVE_ERR_INVALID_ARG;
    if (bytes < kWsCounterBytes) return CLOVE_ERR_WORKSPACE;
    t_ws = ThreadWs{};
    t_ws.mode = WsMode::kBound;
    t_ws.ptr = static_cast<char*>(ptr);
    t_ws.bytes = bytes;
    return CLOVE_OK;
}

// Test hook, not part of the ABI: the calling thread's scratch allocations ask
// for `bytes` more than they need (an amount no device holds makes them fail).
void clove_test_alloc_excess(size_t bytes) { t_alloc_excess = bytes; }

clove_status_t clove_workspace_query_begin(void) {
    if (t_ws.mode == WsMode::kQuery) return CLOVE_ERR_INVALID_ARG;
    t_ws_saved = t_ws;
    t_ws = ThreadWs{};
    t_ws.mode = WsMode::kQuery;
    return CLOVE_OK;
}

size_t clove_workspace_query_end(void) {
    if (t_ws.mode != WsMode::kQuery) return 0;
    const size_t need = t_ws.need;
    t_ws = t_ws_saved;
    t_ws_saved = ThreadWs{};
    return need;
}

clove_status_t clove_release_scratch(void) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return CLOVE_ERR_NO_DEVICE;
    if (hipDeviceSynchronize() != hipSuccess) return CLOVE_ERR_LAUNCH;
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    for (auto it = g_scratch.begin(); it != g_scratch.end();) {
        if (it->first.first == dev) {
            (void)hipFree(it->second.base);
            it = g_scratch.erase(it);
        } else {
            ++it;
        }
    }
    for (auto it = g_buffers.begin(); it != g_buffers.end();) {
        if (std::get<0>(it->first) == dev) {
            (void)hipFree(it->second.base);
            it = g_buffers.erase(it);
        } else {
            ++it;
        }
    }
    for (void* p : g_retired[dev]) (void)hipFree(p);
    g_retired.erase(dev);
    return CLOVE_OK;
}

}  // extern "C"

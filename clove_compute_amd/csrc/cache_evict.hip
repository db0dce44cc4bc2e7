// Eviction from the paged cache by accumulated attention weight.
//
// Of a sequence's n tokens the `keep` best stay: first those of protected
// positions, then the largest weights, ties to the lowest slot.  Kept tokens
// past slot `keep` move into the holes below it, the j-th into the j-th, so
// nothing is copied that can stay where it is and no row is both read and
// written: the moves are independent of each other.
//
//  * select: one workgroup per sequence.  Each token's rank is one 32-bit key
//    (the ordered bits of its weight; all ones for a token that stays in any
//    case, 0 for one that cannot), in LDS up to 32768 tokens; four 8-bit digits
//    from the top find the keep-th largest key, ties are counted in slot order,
//    and the lists of moving slots and holes come out in order.  It also writes
//    the weights, positions and lengths.  A CU takes 8 bytes a token from memory
//    at about 47 GB/s, and each of its dozen passes waits for the one before, so
//    loads and LDS reads of a pass are issued together (8 of each per thread; one
//    by one, 24576 tokens took 68 us).
//  * move: the rows of K and V, 16 bytes per lane; few rows are moved by select
//    itself, which saves the second launch.
#include <algorithm>
#include <type_traits>

#include "decode.hpp"

namespace clove {
namespace evict {

using namespace hw;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kLdsKeys = 32768;  // 128 KB of the CU's 160
constexpr int kCopies = 16;      // of the digit histogram, by lane: same-address atomics serialise
constexpr unsigned kStays = 0xffffffffu, kGoes = 0u;

// Ordered bits of a weight: a larger weight has the larger key; -0 as 0; NaN
// below -infinity.  Never kStays (a NaN's) or kGoes.
__device__ __forceinline__ unsigned order_key(float w) {
    if (w != w) return 1u;
    const unsigned u = bitcast<unsigned>(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
    for (int m = 32; m; m >>= 1) v = max(v, __shfl_xor(v, m));
    return v;
}

// Element offset of slot `i`'s row of head 0, or -1 where its page is absent.
__device__ __forceinline__ int64_t row_at(const PagedCache& c, const FastDiv& by_page, const int32_t* table, int i) {
    const int page = by_page.div(i), row = i - page * c.page_size;
    const int id = table[page];
    if ((unsigned)id >= (unsigned)c.num_pages) return -1;
    return (int64_t)id * c.page_stride + (int64_t)row * c.head_dim;
}

struct Params {
    EvictArgs a;
    FastDiv page;   // by the page size
    int moves;      // most that one sequence can move
    int* counts;    // [batch]
    int* lists;     // [batch][2][moves]: slots that move, holes
    unsigned* keys; // [batch][key_stride] where they do not fit LDS
    int64_t key_stride;
    FastDiv per;    // by the accesses of a row
    FastDiv heads;  // by the KV heads
    bool vec;       // 8 elements an access, else 1
    bool fused;     // select moves the rows
};

// Accesses first, first + step, .. of a sequence's moves: (move, head, access of the row).
template <int V>
__device__ __forceinline__ void move_rows(const Params& p, const int32_t* table, const int* src, const int* dst, int count, int64_t first,
                                          int64_t step) {
    const PagedCache& c = p.a.cache;
    const int64_t head = (int64_t)c.page_size * c.head_dim, total = (int64_t)count * c.kv_heads * p.per.d;
    for (int64_t i = first; i < total; i += step) {
        int64_t row = total <= INT32_MAX ? p.per.div((int)i) : i / p.per.d;
        const int at = (int)(i - row * p.per.d), j = total <= INT32_MAX ? p.heads.div((int)row) : (int)(row / c.kv_heads);
        const int h = (int)(row - (int64_t)j * c.kv_heads);
        const int64_t from = row_at(c, p.page, table, src[j]), to = row_at(c, p.page, table, dst[j]);
        if (from < 0 || to < 0) continue;
        const int64_t in_row = h * head + (int64_t)at * V;
        if constexpr (V == 8) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(c.k + from + in_row);
            const u32x4 v = *reinterpret_cast<const u32x4*>(c.v + from + in_row);
            *reinterpret_cast<u32x4*>(c.k + to + in_row) = k;
            *reinterpret_cast<u32x4*>(c.v + to + in_row) = v;
        } else {
            c.k[to + in_row] = c.k[from + in_row];
            c.v[to + in_row] = c.v[from + in_row];
        }
    }
}

struct Lds {
    unsigned hist[256 * kCopies];
    unsigned total[256];
    int part[kWaves][3];
    int pick[2];
};

// One value per wave summed or maximised over the workgroup; two barriers.
template <bool MAX>
__device__ __forceinline__ int block_reduce(int v, Lds& s) {
    v = MAX ? wave_max(v) : wave_sum(v);
    if ((threadIdx.x & 63) == 0) s.part[threadIdx.x >> 6][0] = v;
    __syncthreads();
    int r = s.part[0][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) r = MAX ? max(r, s.part[w][0]) : r + s.part[w][0];
    __syncthreads();
    return r;
}

constexpr int kBatch = 8;  // global loads of a thread in flight

template <bool IN_LDS>
__global__ void __launch_bounds__(kThreads) select(const Params p) {
    extern __shared__ __align__(16) unsigned lds_keys[];
    __shared__ Lds s;
    const EvictArgs& a = p.a;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(max(a.context_lens[b], 0), a.max_context);
    const int keep = min(n, a.budget);
    const float* weights = a.weights + b * a.weights_stride;
    const int32_t* positions = a.positions + b * a.positions_stride;
    float* weights_out = a.weights_out + b * a.weights_out_stride;
    int32_t* positions_out = a.positions_out + b * a.positions_out_stride;
    int* const src = p.lists + (int64_t)b * 2 * p.moves;
    int* const dst = src + p.moves;
    int moving = 0;
    if (n > keep && keep > 0) {
        unsigned* const keys = IN_LDS ? lds_keys : p.keys + b * p.key_stride;
        const int padded = cdiv(n, 4) * 4;  // keys are read by fours; past n they are kGoes
        int newest = INT32_MIN;
        for (int i0 = tid; i0 < n; i0 += kBatch * kThreads) {
            int v[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) v[u] = i0 + u * kThreads < n ? positions[i0 + u * kThreads] : INT32_MIN;
#pragma unroll
            for (int u = 0; u < kBatch; ++u) newest = max(newest, v[u]);
        }
        newest = block_reduce<true>(newest, s);
        const int64_t from = (int64_t)newest - a.recent;
        auto safe_at = [&](int pos) { return pos < a.sinks || (int64_t)pos > from; };
        int safes = 0;
        for (int i0 = tid; i0 < padded; i0 += kBatch * kThreads) {
            int v[kBatch];
            float w[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kThreads;
                v[u] = i < n ? positions[i] : INT32_MAX;
                w[u] = i < n ? weights[i] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kBatch; ++u) {
                const int i = i0 + u * kThreads;
                if (i >= padded) continue;
                const bool safe = i < n && safe_at(v[u]);
                safes += safe ? 1 : 0;
                keys[i] = i >= n ? kGoes : safe ? kStays : order_key(w[u]);
            }
        }
        safes = block_reduce<false>(safes, s);
        if (safes >= keep) {  // the protected compete among themselves
            for (int i = tid; i < n; i += kThreads) keys[i] = safe_at(positions[i]) ? order_key(weights[i]) : kGoes;
            __syncthreads();
        }
        // the keep-th largest key, digit by digit: `prefix` its bits so far,
        // `need` how many of the keys with that prefix are kept
        unsigned prefix = 0, mask = 0;
        int need = keep;
        for (int shift = 24; shift >= 0; shift -= 8) {
            *reinterpret_cast<u32x4*>(s.hist + 4 * tid) = u32x4{0u, 0u, 0u, 0u};
            static_assert(4 * kThreads == 256 * kCopies, "one access a thread");
            __syncthreads();
            for (int i = 4 * tid; i < padded; i += 4 * kThreads) {
                const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if ((k[e] & mask) == prefix) atomicAdd(&s.hist[((k[e] >> shift) & 255u) * kCopies + (lane & (kCopies - 1))], 1u);
            }
            __syncthreads();
            {  // the copies of a digit: four lanes of four
                const u32x4 c = *reinterpret_cast<const u32x4*>(s.hist + 4 * tid);
                int v = (int)(c[0] + c[1] + c[2] + c[3]);
                v += __builtin_amdgcn_mov_dpp(v, 0xb1, 0xf, 0xf, false);
                v += __builtin_amdgcn_mov_dpp(v, 0x4e, 0xf, 0xf, false);
                if ((tid & 3) == 0) s.total[255 - tid / 4] = (unsigned)v;  // from the top
            }
            __syncthreads();
            if (wave == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l
                const u32x4 c = *reinterpret_cast<const u32x4*>(s.total + 4 * lane);
                const int sum = (int)(c[0] + c[1] + c[2] + c[3]);
                int above = sum;  // keys of this lane's digits and all higher ones
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const int o = __shfl_up(above, m);
                    if (lane >= m) above += o;
                }
                above -= sum;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above < need && above + (int)c[j] >= need) {
                        s.pick[0] = 255 - 4 * lane - j;
                        s.pick[1] = need - above;
                    }
                    above += (int)c[j];
                }
            }
            __syncthreads();
            prefix |= (unsigned)s.pick[0] << shift;
            mask |= 255u << shift;
            need = s.pick[1];
        }
        // in slot order from here: wave w has slots [w seg, (w + 1) seg), 256 at a
        // time, four adjacent ones a lane
        const int seg = cdiv(cdiv(n, kWaves), 256) * 256;
        const int i0 = min(wave * seg, padded), i1 = min(i0 + seg, padded);
        const unsigned long long below = (1ull << lane) - 1ull;
        int equal = 0;
        for (int i = i0 + 4 * lane; i < i1; i += 256) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) equal += k[e] == prefix ? 1 : 0;
        }
        equal = wave_sum(equal);
        if (lane == 0) s.part[wave][0] = equal;
        __syncthreads();
        int before = 0;  // equal keys of lower slots
        for (int w = 0; w < wave; ++w) before += s.part[w][0];
        // the lists of slots that move and of holes: counted, then written
        int at_src = 0, at_dst = 0;
        for (int pass = 0; pass < 2; ++pass) {
            int ties = before;
            for (int i = i0; i < i1; i += 256) {
                const int at = i + 4 * lane;
                const u32x4 k = at < i1 ? *reinterpret_cast<const u32x4*>(keys + at) : u32x4{kGoes, kGoes, kGoes, kGoes};
                int rank = ties, n_eq = 0;  // of this lane's first slot among the equal keys
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned long long eq = __ballot(k[e] == prefix);
                    rank += __popcll(eq & below);
                    n_eq += __popcll(eq);
                }
                ties += n_eq;
                unsigned out = 0, hole = 0;  // this lane's four
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool kept = k[e] > prefix || (k[e] == prefix && rank < need);
                    rank += k[e] == prefix ? 1 : 0;
                    out |= (kept && at + e >= keep ? 1u : 0u) << e;
                    hole |= (!kept && at + e < keep ? 1u : 0u) << e;
                }
                int my_src = at_src, my_dst = at_dst;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const unsigned long long x = __ballot((out >> e) & 1u), y = __ballot((hole >> e) & 1u);
                    my_src += __popcll(x & below);
                    my_dst += __popcll(y & below);
                    at_src += __popcll(x);
                    at_dst += __popcll(y);
                }
                if (pass) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if ((out >> e) & 1u) src[my_src++] = at + e;
                        if ((hole >> e) & 1u) dst[my_dst++] = at + e;
                    }
                }
            }
            if (!pass) {
                if (lane == 0) {
                    s.part[wave][1] = at_src;
                    s.part[wave][2] = at_dst;
                }
                __syncthreads();
                at_src = at_dst = 0;
                for (int w = 0; w < kWaves; ++w) {
                    if (w < wave) {
                        at_src += s.part[w][1];
                        at_dst += s.part[w][2];
                    }
                    moving += s.part[w][1];
                }
            }
        }
        __syncthreads();
    }
    // the slots as they are now; the moved ones are read past `keep` and
    // written below it, so in-place outputs need only the barrier before the
    // rest of the row is cleared
    auto copy = [&](const auto* from, auto* to) {
        if (to == from) return;
        for (int i0 = tid; i0 < keep; i0 += 4 * kThreads) {
            std::remove_reference_t<decltype(*to)> v[4];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * kThreads < keep) v[u] = from[i0 + u * kThreads];
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * kThreads < keep) to[i0 + u * kThreads] = v[u];
        }
    };
    copy(weights, weights_out);
    copy(positions, positions_out);
    __syncthreads();
    for (int j = tid; j < moving; j += kThreads) {
        const int from = src[j], to = dst[j];
        weights_out[to] = weights[from];
        positions_out[to] = positions[from];
    }
    __syncthreads();
    for (int i = keep + tid; i < a.max_context; i += kThreads) {
        weights_out[i] = 0.0f;
        positions_out[i] = -1;
    }
    if (tid == 0) {
        a.lens_out[b] = keep;
        if (p.moves && !p.fused) p.counts[b] = moving;
    }
    if (p.fused && moving) {
        const int32_t* table = a.block_table + b * a.table_stride;
        p.vec ? move_rows<8>(p, table, src, dst, moving, tid, kThreads) : move_rows<1>(p, table, src, dst, moving, tid, kThreads);
    }
}

template <int V>
__global__ void __launch_bounds__(256) move(const Params p, FastDiv blocks) {
    const int b = blocks.div(blockIdx.x);
    const int* src = p.lists + (int64_t)b * 2 * p.moves;
    move_rows<V>(p, p.a.block_table + b * p.a.table_stride, src, src + p.moves, p.counts[b],
                 (int64_t)(blockIdx.x - b * blocks.d) * 256 + threadIdx.x, (int64_t)blocks.d * 256);
}

}  // namespace evict

clove_status_t launch_cache_evict(const EvictArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    evict::Params p{};
    p.a = a;
    p.page = FastDiv(a.cache.page_size);
    // no sequence can move more slots than lie past the budget, or than it keeps
    p.moves = std::max(0, std::min(a.budget, a.max_context - a.budget));
    p.vec = a.cache.head_dim % 8 == 0 && a.cache.page_stride % 8 == 0 && aligned16(a.cache.k) && aligned16(a.cache.v);
    p.per = FastDiv(p.vec ? a.cache.head_dim / 8 : a.cache.head_dim);
    p.heads = FastDiv(a.cache.kv_heads);
    const int64_t most = (int64_t)p.moves * a.cache.kv_heads * p.per.d;  // accesses of a sequence's moves
    p.fused = most <= 4 * evict::kThreads;
    const bool cuts = a.max_context > a.budget;
    const bool in_lds = !cuts || a.max_context <= evict::kLdsKeys;
    p.key_stride = (int64_t)hw::cdiv(a.max_context, 4) * 4;
    const size_t ints = ((size_t)a.batch * (1 + 2 * (size_t)p.moves) + 3) / 4 * 4, keys = in_lds ? 0 : (size_t)(a.batch * p.key_stride);
    if (p.moves) {
        void* buf = nullptr;
        if ((st = acquire_buffer(stream, kBufDecode, (ints + keys) * 4, &buf)) != CLOVE_OK) return st;
        p.counts = static_cast<int*>(buf);
        p.lists = p.counts + a.batch;
        p.keys = reinterpret_cast<unsigned*>(p.counts + ints);
    }
    const int lds = in_lds && cuts ? (int)p.key_stride * 4 : 0;
    const auto kernel = in_lds ? evict::select<true> : evict::select<false>;
    if ((st = ensure_lds(reinterpret_cast<const void*>(kernel), lds)) != CLOVE_OK) return st;
    CLOVE_LAUNCH(kernel, dim3((unsigned)a.batch), dim3(evict::kThreads), lds, stream, p);
    if ((st = check_launch()) != CLOVE_OK || p.fused) return st;
    const int64_t x = std::min<int64_t>(hw::cdiv64(most, 256), std::max<int64_t>(1, hw::cdiv64(16 * dev.num_cus, a.batch)));
    CLOVE_LAUNCH(p.vec ? evict::move<8> : evict::move<1>, dim3((unsigned)(x * a.batch)), dim3(256), 0, stream, p, FastDiv((int)x));
    return check_launch();
}

}  // namespace clove

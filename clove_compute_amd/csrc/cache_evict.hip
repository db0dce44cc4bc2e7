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
//    case, 0 for one that cannot); four 8-bit digits from the top find the
//    keep-th largest key, ties are counted in slot order, and the lists of
//    moving slots and holes come out in order.  It also writes the weights,
//    positions and lengths.
//  * move: the rows of K and V, 16 bytes per lane.
#include <algorithm>

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

struct Lds {
    unsigned hist[256 * kCopies];
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
    for (int w = 1; w < kWaves; ++w) r = MAX ? max(r, s.part[w][0]) : r + s.part[w][0];
    __syncthreads();
    return r;
}

template <bool IN_LDS>
__global__ void __launch_bounds__(kThreads) select(const EvictArgs a, int moves, int* counts, int* lists,
                                                   unsigned* key_buffer) {
    extern __shared__ unsigned lds_keys[];
    __shared__ Lds s;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = min(max(a.context_lens[b], 0), a.max_context);
    const int keep = min(n, a.budget);
    const float* weights = a.weights + b * a.weights_stride;
    const int32_t* positions = a.positions + b * a.positions_stride;
    float* weights_out = a.weights_out + b * a.weights_out_stride;
    int32_t* positions_out = a.positions_out + b * a.positions_out_stride;
    int* const src = lists + (int64_t)b * 2 * moves;
    int* const dst = src + moves;
    int moving = 0;
    if (n > keep && keep > 0) {
        unsigned* const keys = IN_LDS ? lds_keys : key_buffer + (int64_t)b * a.max_context;
        int newest = INT32_MIN;
        for (int i = tid; i < n; i += kThreads) newest = max(newest, positions[i]);
        newest = block_reduce<true>(newest, s);
        const int64_t from = (int64_t)newest - a.recent;
        auto safe = [&](int i) { return positions[i] < a.sinks || (int64_t)positions[i] > from; };
        int safes = 0;
        for (int i = tid; i < n; i += kThreads) safes += safe(i) ? 1 : 0;
        safes = block_reduce<false>(safes, s);
        const bool only_safe = safes >= keep;  // the protected compete among themselves
        for (int i = tid; i < n; i += kThreads) {
            const unsigned k = order_key(weights[i]);
            keys[i] = only_safe ? (safe(i) ? k : kGoes) : (safe(i) ? kStays : k);
        }
        // the keep-th largest key, digit by digit: `prefix` its bits so far,
        // `need` how many of the keys with that prefix are kept
        unsigned prefix = 0, mask = 0;
        int need = keep;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256 * kCopies; i += kThreads) s.hist[i] = 0u;
            __syncthreads();
            for (int i = tid; i < n; i += kThreads) {
                const unsigned k = keys[i];
                if ((k & mask) == prefix) atomicAdd(&s.hist[((k >> shift) & 255u) * kCopies + (lane & (kCopies - 1))], 1u);
            }
            __syncthreads();
            if (wave == 0) {  // lane l: digits 255 - 4 l .. 252 - 4 l, from the top
                int c[4], sum = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[j] = 0;
                    for (int r = 0; r < kCopies; ++r) c[j] += (int)s.hist[(255 - 4 * lane - j) * kCopies + r];
                    sum += c[j];
                }
                int above = sum;  // keys of this lane's digits and all higher ones
#pragma unroll
                for (int m = 1; m < 64; m <<= 1) {
                    const int o = __shfl_up(above, m);
                    if (lane >= m) above += o;
                }
                above -= sum;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (above < need && above + c[j] >= need) {
                        s.pick[0] = 255 - 4 * lane - j;
                        s.pick[1] = need - above;
                    }
                    above += c[j];
                }
            }
            __syncthreads();
            prefix |= (unsigned)s.pick[0] << shift;
            mask |= 255u << shift;
            need = s.pick[1];
        }
        // in slot order from here: wave w has slots [w seg, (w + 1) seg)
        const int seg = cdiv(cdiv(n, kWaves), 64) * 64;
        const int i0 = min(wave * seg, n), i1 = min(i0 + seg, n);
        int equal = 0;
        for (int i = i0; i < i1; i += 64)
            equal += __popcll(__ballot(i + lane < i1 && keys[min(i + lane, n - 1)] == prefix));
        if (lane == 0) s.part[wave][0] = equal;
        __syncthreads();
        int before = 0;  // equal keys of lower slots
        for (int w = 0; w < wave; ++w) before += s.part[w][0];
        // the lists of slots that move and of holes: counted, then written
        const unsigned long long below = (1ull << lane) - 1ull;
        int at_src = 0, at_dst = 0;
        for (int pass = 0; pass < 2; ++pass) {
            int ties = before;
            for (int i = i0; i < i1; i += 64) {
                const int at = i + lane;
                const unsigned k = at < i1 ? keys[at] : kGoes;
                const unsigned long long eq = __ballot(at < i1 && k == prefix);
                const bool kept = at < i1 && (k > prefix || (k == prefix && ties + __popcll(eq & below) < need));
                ties += __popcll(eq);
                const unsigned long long out = __ballot(kept && at >= keep), hole = __ballot(!kept && at < min(keep, i1));
                if (pass) {
                    if (kept && at >= keep) src[at_src + __popcll(out & below)] = at;
                    if (!kept && at < min(keep, i1)) dst[at_dst + __popcll(hole & below)] = at;
                }
                at_src += __popcll(out);
                at_dst += __popcll(hole);
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
    if (weights_out != weights)
        for (int i = tid; i < keep; i += kThreads) weights_out[i] = weights[i];
    if (positions_out != positions)
        for (int i = tid; i < keep; i += kThreads) positions_out[i] = positions[i];
    __syncthreads();
    for (int j = tid; j < moving; j += kThreads) {
        weights_out[dst[j]] = weights[src[j]];
        positions_out[dst[j]] = positions[src[j]];
    }
    __syncthreads();
    for (int i = keep + tid; i < a.max_context; i += kThreads) {
        weights_out[i] = 0.0f;
        positions_out[i] = -1;
    }
    if (tid == 0) {
        a.lens_out[b] = keep;
        if (moves) counts[b] = moving;
    }
}

// Element offset of slot `i`'s row of head 0, or -1 where its page is absent.
__device__ __forceinline__ int64_t row_at(const EvictArgs& a, const int32_t* table, int i) {
    const int page = i / a.cache.page_size, row = i - page * a.cache.page_size;
    const int id = table[page];
    if ((unsigned)id >= (unsigned)a.cache.num_pages) return -1;
    return (int64_t)id * a.cache.page_stride + (int64_t)row * a.cache.head_dim;
}

// V: elements per access (8, or 1 for any alignment).  A workgroup takes
// (move, head) rows of one sequence in turn.
template <int V>
__global__ void __launch_bounds__(256) move(const EvictArgs a, int moves, int blocks, const int* counts,
                                              const int* lists) {
    const int b = blockIdx.x / blocks, D = a.cache.head_dim, H = a.cache.kv_heads;
    const int* src = lists + (int64_t)b * 2 * moves;
    const int* dst = src + moves;
    const int32_t* table = a.block_table + b * a.table_stride;
    const int per = D / V;  // accesses per row
    const int64_t head = (int64_t)a.cache.page_size * D, total = (int64_t)counts[b] * H * per;
    for (int64_t i = (int64_t)(blockIdx.x - b * blocks) * 256 + threadIdx.x; i < total; i += (int64_t)blocks * 256) {
        const int64_t row = i / per;
        const int c = (int)(i - row * per), j = (int)(row / H), h = (int)(row - (int64_t)j * H);
        const int64_t from = row_at(a, table, src[j]), to = row_at(a, table, dst[j]);
        if (from < 0 || to < 0) continue;
        const int64_t at = h * head + (int64_t)c * V;
        if constexpr (V == 8) {
            const u32x4 k = *reinterpret_cast<const u32x4*>(a.cache.k + from + at);
            const u32x4 v = *reinterpret_cast<const u32x4*>(a.cache.v + from + at);
            *reinterpret_cast<u32x4*>(a.cache.k + to + at) = k;
            *reinterpret_cast<u32x4*>(a.cache.v + to + at) = v;
        } else {
            a.cache.k[to + at] = a.cache.k[from + at];
            a.cache.v[to + at] = a.cache.v[from + at];
        }
    }
}

}  // namespace evict

clove_status_t launch_cache_evict(const EvictArgs& a, hipStream_t stream) {
    DeviceInfo dev;
    clove_status_t st = current_device_info(&dev);
    if (st != CLOVE_OK) return st;
    // no sequence can move more slots than lie past the budget, or than it holds
    const int moves = std::max(0, std::min(a.budget, a.max_context - a.budget));
    const bool cuts = a.max_context > a.budget;
    const bool in_lds = !cuts || a.max_context <= evict::kLdsKeys;
    const size_t ints = (size_t)a.batch * (1 + 2 * (size_t)moves), keys = in_lds ? 0 : (size_t)a.batch * a.max_context;
    int* counts = nullptr;
    if (ints + keys > (size_t)a.batch) {
        void* p = nullptr;
        if ((st = acquire_buffer(stream, kBufDecode, (ints + keys) * 4, &p)) != CLOVE_OK) return st;
        counts = static_cast<int*>(p);
    }
    int* lists = counts ? counts + a.batch : nullptr;
    unsigned* key_buffer = in_lds ? nullptr : reinterpret_cast<unsigned*>(lists + (size_t)a.batch * 2 * moves);
    const int lds = in_lds && cuts ? a.max_context * 4 : 0;
    const auto kernel = in_lds ? evict::select<true> : evict::select<false>;
    if ((st = ensure_lds(reinterpret_cast<const void*>(kernel), lds)) != CLOVE_OK) return st;
    CLOVE_LAUNCH(kernel, dim3((unsigned)a.batch), dim3(evict::kThreads), lds, stream, a, moves, counts, lists,
                 key_buffer);
    if ((st = check_launch()) != CLOVE_OK || moves == 0) return st;
    const bool vec = a.cache.head_dim % 8 == 0 && a.cache.page_stride % 8 == 0 && aligned16(a.cache.k) && aligned16(a.cache.v);
    const int64_t most = (int64_t)moves * a.cache.kv_heads * (vec ? a.cache.head_dim / 8 : a.cache.head_dim);
    const int64_t x = std::min<int64_t>(hw::cdiv64(most, 256), std::max<int64_t>(1, hw::cdiv64(16 * dev.num_cus, a.batch)));
    CLOVE_LAUNCH(vec ? evict::move<8> : evict::move<1>, dim3((unsigned)(x * a.batch)), dim3(256), 0, stream, a, moves,
                 (int)x, counts, lists);
    return check_launch();
}

}  // namespace clove

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
//    case, 0 for one that cannot), in LDS up to 32768 tokens; three digits from
//    the top find the keep-th largest key, ties are counted in slot order,
//    and the lists of moving slots and holes come out in order.  It also writes
//    the weights, positions and lengths.  A CU takes 8 bytes a token from memory
//    at about 47 GB/s, and each of its dozen passes waits for the one before, so
//    loads and LDS reads of a pass are issued together (8 of each per thread):
//    12 sequences of up to 24576 tokens take 24 us (one by one 68), 2049 tokens 8.
//  * move: the rows of K and V, 16 bytes per lane where rows are multiples of
//    that; few rows are moved by select itself, which saves the second launch.
//    HBM-bound: 97 MB read and as much written in 36 us, 5.4 TB/s.  Where rows are whole
//    64-byte parts of lines the stores pass the L2 by, as nothing reads the rows
//    soon: 32 x 8192 tokens to 2048 of 8 heads with 32, 64, 96, 160 elements take
//    44, 56, 94, 136 us so and 55, 62, 104, 150 with ordinary stores, which other
//    rows are better with (72 elements 109 against 120).
#include <algorithm>
#include <type_traits>

#include "decode.hpp"

namespace clove {
namespace evict {

using namespace hw;

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kLdsKeys = 32768;  // 128 KB of the CU's 160
constexpr int kBins = 2048;      // of a digit of 11 bits: the first holds sign, exponent and two bits of a weight
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
    bool whole;     // rows are whole 64-byte parts of lines
    int team;       // lanes of a move: a power of two up to 64
    int vec;        // elements of an access: the most of 8, 4, 2, 1 that rows and addresses are multiples of
    bool fused;     // select moves the rows
};

// Moves first, first + step, .. of a sequence, a team of p.team lanes (`at` of it)
// each: its accesses are those of the row of every head, four of K and V in flight.
template <int V, bool WHOLE = false>
__device__ __forceinline__ void move_rows(const Params& p, const int32_t* table, const int* src, const int* dst, int count, int first,
                                          int step, int at) {
    typedef std::conditional_t<V == 8, u32x4, std::conditional_t<V == 4, u32x2, std::conditional_t<V == 2, unsigned, uint16_t>>> Word;
    const PagedCache& c = p.a.cache;
    const int64_t head = (int64_t)c.page_size * c.head_dim;
    const int items = c.kv_heads * p.per.d;
    for (int64_t j = first; j < count; j += step) {
        const int64_t from = row_at(c, p.page, table, src[j]), to = row_at(c, p.page, table, dst[j]);
        if (from < 0 || to < 0) continue;
        for (int i0 = at; i0 < items; i0 += 4 * p.team) {
            Word k[4], v[4];
            int64_t in_row[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int i = i0 + u * p.team, h = p.per.div(i);
                in_row[u] = h * head + (int64_t)(i - h * p.per.d) * V;
                if (i < items) {
                    k[u] = *reinterpret_cast<const Word*>(c.k + from + in_row[u]);
                    v[u] = *reinterpret_cast<const Word*>(c.v + from + in_row[u]);
                }
            }
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (i0 + u * p.team < items) {
                    if constexpr (WHOLE) {
                        __builtin_nontemporal_store(k[u], reinterpret_cast<Word*>(c.k + to + in_row[u]));
                        __builtin_nontemporal_store(v[u], reinterpret_cast<Word*>(c.v + to + in_row[u]));
                    } else {
                        *reinterpret_cast<Word*>(c.k + to + in_row[u]) = k[u];
                        *reinterpret_cast<Word*>(c.v + to + in_row[u]) = v[u];
                    }
                }
        }
    }
}

// The end of a selection, after a barrier: the lists hold `moving` slots each.
__device__ __forceinline__ void finish(const Params& p, int b, int keep, int moving, const int* src, const int* dst, bool apart) {
    const EvictArgs& a = p.a;
    const int tid = threadIdx.x;
    const float* weights = a.weights + b * a.weights_stride;
    const int32_t* positions = a.positions + b * a.positions_stride;
    float* weights_out = a.weights_out + b * a.weights_out_stride;
    int32_t* positions_out = a.positions_out + b * a.positions_out_stride;
    if (p.fused && moving) {
        const int32_t* table = a.block_table + b * a.table_stride;
        const int first = tid / p.team, step = kThreads / p.team, at = tid & (p.team - 1);
        if (p.whole) move_rows<8, true>(p, table, src, dst, moving, first, step, at);
        else if (p.vec == 8) move_rows<8>(p, table, src, dst, moving, first, step, at);
        else if (p.vec == 4) move_rows<4>(p, table, src, dst, moving, first, step, at);
        else if (p.vec == 2) move_rows<2>(p, table, src, dst, moving, first, step, at);
        else move_rows<1>(p, table, src, dst, moving, first, step, at);
    }
    // Moved slots are read at or past `keep` and written below it.  Where an output
    // is its input, they are moved before the rest of its row is cleared.
    if (!apart && weights_out != weights)
        for (int i = tid; i < keep; i += kThreads) weights_out[i] = weights[i];
    if (!apart && positions_out != positions)
        for (int i = tid; i < keep; i += kThreads) positions_out[i] = positions[i];
    if (!apart) __syncthreads();
    // (the last threads first: the first ones move rows)
    for (int j0 = kThreads - 1 - tid; j0 < moving; j0 += 4 * kThreads) {
        int from[4], to[4];
        float w[4];
        int32_t pos[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = min(j0 + u * kThreads, moving - 1);
            from[u] = src[j];
            to[u] = dst[j];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            w[u] = weights[from[u]];
            pos[u] = positions[from[u]];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (j0 + u * kThreads >= moving) break;
            weights_out[to[u]] = w[u];
            positions_out[to[u]] = pos[u];
        }
    }
    if (p.fused) {  // (else the second kernel clears it)
        if (!apart) __syncthreads();
        for (int i = keep + tid; i < a.max_context; i += kThreads) {
            weights_out[i] = 0.0f;
            positions_out[i] = -1;
        }
    }
    if (tid == 0) {
        a.lens_out[b] = keep;
        if (p.moves && !p.fused) p.counts[b] = moving;
    }
}

// Up to this many tokens past the budget are found one by one, each as the
// smallest (protected, key, slot from the end) above the last: a step of a full
// cache, one token over, takes one reduction where the digits, ties and lists
// take seven barriers (48 x 2049 tokens 12.0 -> 7.4 us).
constexpr int kFew = 4;

struct Lds {
    unsigned hist[3][kBins];
    int part[kWaves][2];
};

// The smallest value of the wave, in every lane: the order of wave_sum.
__device__ __forceinline__ unsigned wave_min(unsigned v) {
    v = min(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x128, 0xf, 0xf, false));  // row_ror:8
    v = min(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x124, 0xf, 0xf, false));  // row_ror:4
    v = min(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x4e, 0xf, 0xf, false));   // quad_perm 2301
    v = min(v, (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0xb1, 0xf, 0xf, false));   // quad_perm 1032
    return min(min((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               min((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}
__device__ __forceinline__ uint64_t wave_min(uint64_t v) {
    const unsigned hi = wave_min((unsigned)(v >> 32));
    return ((uint64_t)hi << 32) | wave_min((unsigned)(v >> 32) == hi ? (unsigned)v : 0xffffffffu);
}

constexpr int kHeld = 16;  // tokens of a thread that stay in registers from the first load on
constexpr int kRest = 8;   // tokens of a thread loaded at once after them

template <bool IN_LDS>
__global__ void __launch_bounds__(kThreads) select(const Params p) {
    extern __shared__ __align__(16) unsigned lds_keys[];
    __shared__ __align__(16) Lds s;
    const EvictArgs& a = p.a;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* weights = a.weights + b * a.weights_stride;
    const int32_t* positions = a.positions + b * a.positions_stride;
    float* weights_out = a.weights_out + b * a.weights_out_stride;
    int32_t* positions_out = a.positions_out + b * a.positions_out_stride;
    const int n = min(max(a.context_lens[b], 0), a.max_context);
    const int keep = min(n, a.budget);
    // rows hold max_context tokens whatever the length is, which is not awaited
    int32_t held_pos[kHeld];
    float held_w[kHeld];
#pragma unroll
    for (int u = 0; u < kHeld; ++u) {
        const int i = tid + u * kThreads;
        held_pos[u] = i < a.max_context ? positions[i] : 0;
        held_w[u] = i < a.max_context ? weights[i] : 0.0f;
    }
    // f(first of the workgroup's slots, slot, position, weight) for each of the
    // first `most` slots that this thread has
    auto each = [&](int most, auto f) {
#pragma unroll
        for (int u = 0; u < kHeld; ++u)
            if (u * kThreads < most && tid + u * kThreads < most) f(u * kThreads, tid + u * kThreads, held_pos[u], held_w[u]);
        for (int base = kHeld * kThreads; base < most; base += kRest * kThreads) {
            int32_t v[kRest];
            float w[kRest];
#pragma unroll
            for (int u = 0; u < kRest; ++u) {
                const int i = base + tid + u * kThreads;
                v[u] = i < most ? positions[i] : 0;
                w[u] = i < most ? weights[i] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < kRest; ++u)
                if (base + u * kThreads < most && base + tid + u * kThreads < most) f(base + u * kThreads, base + tid + u * kThreads, v[u], w[u]);
        }
    };
    const bool apart = weights_out != weights && positions_out != positions;
    // outputs apart from their inputs, before the moved tokens are written over them
    auto pass_on = [&](int base, int i, int32_t pos, float w) {
        if (!apart || base >= keep || i >= keep) return;
        weights_out[i] = w;
        positions_out[i] = pos;
    };
    int* const src = p.lists + (int64_t)b * 2 * p.moves;
    int* const dst = src + p.moves;
    int moving = 0;
    if (n <= keep || keep == 0) {  // nothing to choose
        if (apart) each(keep, pass_on);
    } else {
        unsigned* const keys = IN_LDS ? lds_keys : p.keys + b * p.key_stride;
        const int padded = cdiv(n, 4) * 4;  // keys are read by fours; past n they are kGoes
        int newest = INT32_MIN;
        each(n, [&](int, int, int32_t pos, float) { newest = max(newest, pos); });
        newest = wave_max(newest);
        if (lane == 0) s.part[wave][0] = newest;
        reinterpret_cast<u32x2*>(s.hist[0])[tid] = u32x2{0u, 0u};
        static_assert(kBins == 2 * kThreads, "one access a thread");
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWaves; ++w) newest = max(newest, s.part[w][0]);
        const int64_t from = (int64_t)newest - a.recent;
        auto safe_at = [&](int32_t pos) { return pos < a.sinks || (int64_t)pos > from; };
        int safes = 0;
        each(n, [&](int base, int i, int32_t pos, float w) {
            const bool safe = safe_at(pos);
            const unsigned k = safe ? kStays : order_key(w);
            safes += safe ? 1 : 0;
            keys[i] = k;
            atomicAdd(&s.hist[0][k >> 21], 1u);
            pass_on(base, i, pos, w);
        });
        if (tid < padded - n) keys[n + tid] = kGoes;
        safes = wave_sum(safes);
        if (lane == 0) s.part[wave][1] = safes;
        reinterpret_cast<u32x2*>(s.hist[1])[tid] = u32x2{0u, 0u};
        __syncthreads();
        safes = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) safes += s.part[w][1];
        if (safes >= keep) {  // the protected compete among themselves: keys and first digits anew
            reinterpret_cast<u32x2*>(s.hist[0])[tid] = u32x2{0u, 0u};
            __syncthreads();
            each(n, [&](int, int i, int32_t pos, float w) {
                const unsigned k = safe_at(pos) ? order_key(w) : kGoes;
                keys[i] = k;
                atomicAdd(&s.hist[0][k >> 21], 1u);
            });
            __syncthreads();
        }
        // the keep-th largest key, by digits of 11, 11 and 10 bits: `prefix` its bits so
        // far, `need` how many of the `equal` keys with that prefix are kept.  Every
        // wave reads the counts for itself, so a digit costs one barrier.
        unsigned prefix = 0;
        int need = keep, equal = 0;
#pragma unroll
        for (int digit = 0; digit < 3; ++digit) {
            constexpr int kShift[3] = {21, 10, 0};
            const int shift = kShift[digit];
            unsigned* const hist = s.hist[digit];
            if (digit) {
                const int above_shift = kShift[digit - 1];
                if (digit < 2) reinterpret_cast<u32x2*>(s.hist[digit + 1])[tid] = u32x2{0u, 0u};
                for (int i = 4 * tid; i < padded; i += 4 * kThreads) {
                    const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (k[e] >> above_shift == prefix >> above_shift) atomicAdd(&hist[(k[e] >> shift) & (digit == 2 ? 1023u : 2047u)], 1u);
                }
                __syncthreads();
            }
            // lane l: bins 32 l .. 32 l + 31 summed (read in an order of their own, which
            // keeps the lanes on different banks) and how many keys lie above them
            u32x4 c = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int r = 0; r < 8; ++r) c += *reinterpret_cast<const u32x4*>(hist + 32 * lane + 4 * ((r + lane) & 7));
            const int sum = (int)(c[0] + c[1] + c[2] + c[3]), upto = wave_scan(sum);
            const int above = __builtin_amdgcn_readlane(upto, 63) - upto;
            const int who = __ffsll((long long)__ballot(above < need && above + sum >= need)) - 1;  // one lane has it
            // then its 32 bins, one a lane
            const int bin = lane < 32 ? (int)hist[32 * who + lane] : 0, to_bin = wave_scan(bin);
            const int higher = __builtin_amdgcn_readlane(above, who) + __builtin_amdgcn_readlane(sum, who) - to_bin;
            const int at = __ffsll((long long)__ballot(higher < need && higher + bin >= need)) - 1;
            prefix |= (unsigned)(32 * who + at) << shift;
            need -= __builtin_amdgcn_readlane(higher, at);
            equal = __builtin_amdgcn_readlane(bin, at);
        }
        // in slot order from here: wave w has slots [w seg, (w + 1) seg), 256 at a time
        const int seg = cdiv(cdiv(n, kWaves), 256) * 256;
        const int i0 = min(wave * seg, padded), i1 = min(i0 + seg, padded);
        if (need < equal) {  // of the equal keys the lowest slots stay, the others drop below them
            int count = 0;
            for (int i = i0 + 4 * lane; i < i1; i += 256) {
                const u32x4 k = *reinterpret_cast<const u32x4*>(keys + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) count += k[e] == prefix ? 1 : 0;
            }
            count = wave_sum(count);
            if (lane == 0) s.part[wave][0] = count;
            __syncthreads();
            int ties = 0;
            for (int w = 0; w < wave; ++w) ties += s.part[w][0];
            for (int i = i0; i < i1; i += 256) {
                const int at = i + 4 * lane;
                const u32x4 k = at < i1 ? *reinterpret_cast<const u32x4*>(keys + at) : u32x4{kGoes, kGoes, kGoes, kGoes};
                int own = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) own += k[e] == prefix ? 1 : 0;
                const int upto = wave_scan(own);
                int rank = ties + upto - own;
                ties += __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (k[e] != prefix) continue;
                    if (rank >= need) keys[at + e] = prefix - 1u;
                    ++rank;
                }
            }
            __syncthreads();
        }
        // The lists of slots that move and of holes.  A wave takes its slots 64 at a
        // time; lane c keeps the bits of the c-th 64, so that the second pass over
        // them, with the lists' beginnings known, needs the keys again only where
        // it has more than 64 of them.
        const int groups = cdiv(i1 - i0, 4096);
        uint64_t outs = 0, holes = 0;
        auto bits = [&](int g) {
            const int first = i0 + 4096 * g, chunks = min(64, cdiv(i1 - first, 64));
            uint64_t kept = 0;
            for (int c0 = 0; c0 < chunks; c0 += 4) {
                unsigned k[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) k[u] = keys[min(first + 64 * (c0 + u) + lane, padded - 1)];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const uint64_t m = __ballot(k[u] >= prefix);
                    kept = lane == c0 + u ? m : kept;
                }
            }
            const int base = first + 64 * lane;
            auto up_to = [&](int end) { return end <= base ? 0ull : end >= base + 64 ? ~0ull : (1ull << (end - base)) - 1ull; };
            const uint64_t low = up_to(keep), mine = lane < chunks ? up_to(min(i1, n)) : 0ull;
            outs = kept & mine & ~low;
            holes = ~kept & mine & low;
        };
        int n_src = 0, n_dst = 0;
        for (int g = 0; g < groups; ++g) {
            bits(g);
            n_src += __popcll(outs);
            n_dst += __popcll(holes);
        }
        const int all_src = wave_sum(n_src), all_dst = wave_sum(n_dst);
        __syncthreads();  // (s.part may still be read as the counts of ties)
        if (lane == 0) {
            s.part[wave][0] = all_src;
            s.part[wave][1] = all_dst;
        }
        __syncthreads();
        int at_src = 0, at_dst = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            at_src += w < wave ? s.part[w][0] : 0;
            at_dst += w < wave ? s.part[w][1] : 0;
            moving += s.part[w][0];
        }
        for (int g = 0; g < groups; ++g) {
            if (groups > 1) bits(g);
            const int first = i0 + 4096 * g, chunks = min(64, cdiv(i1 - first, 64));
            const int own = __popcll(outs) | __popcll(holes) << 16, upto = wave_scan(own);  // at most 4096 of each
            if (chunks > 16) {
                // many 64s: each lane its own, bit by bit, as few of them are in a list
                // (24576 tokens to 4096: 4 us, 6 the other way)
                auto write = [&](uint64_t mask, int* list) {
                    for (; mask; mask &= mask - 1ull) *list++ = first + 64 * lane + __ffsll((long long)mask) - 1;
                };
                write(outs, src + at_src + ((upto - own) & 0xffff));
                write(holes, dst + at_dst + ((unsigned)(upto - own) >> 16));
            } else {
                // few: one after the other, a lane a slot (8192 to 4096: 2.8 us, 4.7 the other way)
                for (int c = 0; c < chunks; ++c) {
                    const unsigned before = (unsigned)(__builtin_amdgcn_readlane(upto, c) - __builtin_amdgcn_readlane(own, c));
                    auto write = [&](uint64_t mask, int* list) {
                        const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)mask, c);
                        const unsigned hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(mask >> 32), c);
                        if (!(lo | hi)) return;
                        if (((lane < 32 ? lo : hi) >> (lane & 31)) & 1u)
                            list[__builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0u))] = first + 64 * c + lane;
                    };
                    write(outs, src + at_src + (int)(before & 0xffffu));
                    write(holes, dst + at_dst + (int)(before >> 16));
                }
            }
            const int all = __builtin_amdgcn_readlane(upto, 63);
            at_src += all & 0xffff;
            at_dst += (int)((unsigned)all >> 16);
        }
    }
    __syncthreads();
    finish(p, b, keep, moving, src, dst, apart);
}

// Rows of at most budget + kFew tokens.
__global__ void __launch_bounds__(kThreads) select_few(const Params p) {
    __shared__ uint64_t least_of[2][kWaves];
    __shared__ int newest_of[kWaves], lists[2][kFew];
    const EvictArgs& a = p.a;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* weights = a.weights + b * a.weights_stride;
    const int32_t* positions = a.positions + b * a.positions_stride;
    float* weights_out = a.weights_out + b * a.weights_out_stride;
    int32_t* positions_out = a.positions_out + b * a.positions_out_stride;
    const int n = min(max(a.context_lens[b], 0), a.max_context);
    const int keep = min(n, a.budget);
    const bool apart = weights_out != weights && positions_out != positions;
    // rows hold max_context tokens whatever the length is, which is not awaited
    constexpr int kBatch = 8;
    int32_t pos[kBatch];
    float w[kBatch];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + u * kThreads;
            pos[u] = i < a.max_context ? positions[i] : 0;
            w[u] = i < a.max_context ? weights[i] : 0.0f;
        }
    };
    load(tid);
    int newest = INT32_MIN;
    for (int i0 = tid; i0 < a.max_context; i0 += kBatch * kThreads) {
        if (i0 != tid) load(i0);
#pragma unroll
        for (int u = 0; u < kBatch; ++u) {
            const int i = i0 + u * kThreads;
            if (i < n) newest = max(newest, pos[u]);
            if (apart && i < keep) {
                weights_out[i] = w[u];
                positions_out[i] = pos[u];
            }
        }
    }
    int moving = 0;
    if (n > keep && keep > 0) {
        newest = wave_max(newest);
        if (lane == 0) newest_of[wave] = newest;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kWaves; ++x) newest = max(newest, newest_of[x]);
        const int64_t from = (int64_t)newest - a.recent;
        const bool held = a.max_context <= kBatch * kThreads;  // the registers still have every token
        uint64_t last = 0;
        int gone[kFew];
#pragma unroll
        for (int d = 0; d < kFew; ++d) {
            gone[d] = INT32_MAX;
            if (d >= n - keep) continue;
            uint64_t least = ~(uint64_t)0;
#pragma unroll 1
            for (int i0 = tid; i0 < n; i0 += kBatch * kThreads) {
                if (!held) load(i0);
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    const int i = i0 + u * kThreads;
                    const bool safe = pos[u] < a.sinks || (int64_t)pos[u] > from;
                    const uint64_t c = ((uint64_t)safe << 63) | ((uint64_t)order_key(w[u]) << 31) | (unsigned)(INT32_MAX - i);
                    if (i < n && c > last) least = min(least, c);
                }
            }
            least = wave_min(least);
            if (lane == 0) least_of[d & 1][wave] = least;
            __syncthreads();
#pragma unroll
            for (int x = 0; x < kWaves; ++x) least = min(least, least_of[d & 1][x]);
            last = least;
            gone[d] = INT32_MAX - (int)(least & INT32_MAX);
        }
        // in slot order: those gone below `keep` are holes, those past it that are not gone move
#pragma unroll
        for (int x = 0; x < kFew; ++x)
#pragma unroll
            for (int y = x + 1; y < kFew; ++y) {
                const int lo = min(gone[x], gone[y]), hi = max(gone[x], gone[y]);
                gone[x] = lo;
                gone[y] = hi;
            }
        int holes = 0;
#pragma unroll
        for (int d = 0; d < kFew; ++d) {
            if (gone[d] < keep) {
                if (tid == 0) lists[1][holes] = gone[d];
                ++holes;
            }
            const int i = keep + d;
            bool moves = i < n;
#pragma unroll
            for (int e = 0; e < kFew; ++e) moves = moves && gone[e] != i;
            if (moves) {
                if (tid == 0) lists[0][moving] = i;
                ++moving;
            }
        }
    }
    __syncthreads();
    if (!p.fused && tid < moving) {  // the second kernel's
        int* const src = p.lists + (int64_t)b * 2 * p.moves;
        src[tid] = lists[0][tid];
        src[p.moves + tid] = lists[1][tid];
    }
    finish(p, b, keep, moving, lists[0], lists[1], apart);
}

template <int V, bool WHOLE>
__global__ void __launch_bounds__(256) move(const Params p, FastDiv blocks) {
    const int b = blocks.div(blockIdx.x);
    const int* src = p.lists + (int64_t)b * 2 * p.moves;
    for (int64_t i = p.a.lens_out[b] + (int64_t)(blockIdx.x - b * blocks.d) * 256 + threadIdx.x; i < p.a.max_context; i += (int64_t)blocks.d * 256) {
        p.a.weights_out[b * p.a.weights_out_stride + i] = 0.0f;
        p.a.positions_out[b * p.a.positions_out_stride + i] = -1;
    }
    move_rows<V, WHOLE>(p, p.a.block_table + b * p.a.table_stride, src, src + p.moves, p.counts[b],
                 ((blockIdx.x - b * blocks.d) * 256 + threadIdx.x) / p.team, blocks.d * 256 / p.team, threadIdx.x & (p.team - 1));
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
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.cache.k) | reinterpret_cast<uintptr_t>(a.cache.v);
    for (p.vec = 8; a.cache.head_dim % p.vec || a.cache.page_stride % p.vec || at % (2 * p.vec); p.vec /= 2) {}
    p.whole = a.cache.head_dim % 32 == 0 && a.cache.page_stride % 32 == 0 && at % 64 == 0;
    p.per = FastDiv(a.cache.head_dim / p.vec);
    const int64_t items = (int64_t)a.cache.kv_heads * p.per.d, most = p.moves * items;  // accesses of one move, of a sequence's
    p.team = 1;
    while (p.team < 64 && p.team < items) p.team *= 2;
    p.fused = most <= 4 * evict::kThreads;
    const bool few = a.max_context - a.budget <= evict::kFew;  // (or no row can be cut at all)
    const bool in_lds = few || a.max_context <= evict::kLdsKeys;
    p.key_stride = (int64_t)hw::cdiv(a.max_context, 4) * 4;
    const size_t ints = ((size_t)a.batch * (1 + 2 * (size_t)p.moves) + 3) / 4 * 4, keys = in_lds ? 0 : (size_t)(a.batch * p.key_stride);
    if (p.moves) {
        void* buf = nullptr;
        if ((st = acquire_buffer(stream, kBufDecode, (ints + keys) * 4, &buf)) != CLOVE_OK) return st;
        p.counts = static_cast<int*>(buf);
        p.lists = p.counts + a.batch;
        p.keys = reinterpret_cast<unsigned*>(p.counts + ints);
    }
    const int lds = in_lds && !few ? (int)p.key_stride * 4 : 0;
    const auto kernel = few ? evict::select_few : in_lds ? evict::select<true> : evict::select<false>;
    if ((st = ensure_lds(reinterpret_cast<const void*>(kernel), lds)) != CLOVE_OK) return st;
    CLOVE_LAUNCH(kernel, dim3((unsigned)a.batch), dim3(evict::kThreads), lds, stream, p);
    if ((st = check_launch()) != CLOVE_OK || p.fused) return st;
    // a move a team, at most 32 workgroups per CU
    const int64_t x = std::min<int64_t>(hw::cdiv64((int64_t)p.moves * p.team, 256), std::max<int64_t>(1, hw::cdiv64(32 * dev.num_cus, a.batch)));
    const auto move = p.whole      ? evict::move<8, true>
                      : p.vec == 8 ? evict::move<8, false>
                      : p.vec == 4 ? evict::move<4, false>
                      : p.vec == 2 ? evict::move<2, false>
                                   : evict::move<1, false>;
    CLOVE_LAUNCH(move, dim3((unsigned)(x * a.batch)), dim3(256), 0, stream, p, FastDiv((int)x));
    return check_launch();
}

}  // namespace clove

// Products of (token, place) pairs with the INT4 weights of the experts chosen
// for them:
//
//   SwiGLU:  H[p, i] = fp16(silu(X[t] . W[e, i]) * (X[t] . W[e, I + i]))
//   down:    Y[t, o] = alpha sum_j w[t, j] (H[p] . W[e, o]) + beta Y[t, o]
//   W[e, r, k] = (q - z[e, r, k / 128]) s[e, r, k / 128]
//
// q - z is exact in fp16, so a group's sum on MFMA is an fp32 sum of exact
// products, folded into the fp32 accumulator with its scale; SwiGLU and the
// weighted sum over a token's places are fp32, and a result is rounded once.
//
// The pairs are sorted by expert first (moe_sort), a tile of weight rows then
// meets the pairs of one expert (moe_any), and the places of a token are added
// up from fp32 partial results in place order (moe_combine), so that a call
// gives the same bits every time.
#include "i4w_bits.hpp"
#include "moe.hpp"

namespace clove {
namespace moe {

using namespace hw;

struct Params {
    MoeArgs a;
    int* off;      // [experts + 1]: where an expert's pairs begin in `order`
    int* order;    // [T top_k]: pairs, those of one expert after those of the one before
    float* part;   // down: [T top_k, O] products
    FastDiv k;     // by top_k
    int rows_t;    // tiles of weight rows
    int P, G;
};

// Workgroup e lists the pairs of expert e in order; where they begin is the
// number of pairs of lower experts, which it counts itself: no workgroup waits
// for another.  (128 experts read 65536 ids each from the L2s.)
__global__ void __launch_bounds__(256) moe_sort(const int32_t* ids, int P, int E, int* off, int* order) {
    __shared__ int lds[2][4];
    const int e = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int less = 0, mine = 0;
    for (int p = tid; p < P; p += 256) {
        const int id = ids[p];
        less += id >= 0 && id < e;
        mine += id == e;
    }
    less = wave_sum(less), mine = wave_sum(mine);
    if (lane == 0) lds[0][wave] = less, lds[1][wave] = mine;
    __syncthreads();
    int at = lds[0][0] + lds[0][1] + lds[0][2] + lds[0][3];
    const int count = lds[1][0] + lds[1][1] + lds[1][2] + lds[1][3];
    if (tid == 0) {
        off[e] = at;
        if (e == E - 1) off[E] = at + count;
    }
    if (count == 0) return;
    for (int p0 = 0; p0 < P; p0 += 256) {
        const int p = p0 + tid;
        const bool is = p < P && ids[p] == e;
        const uint64_t m = __ballot(is);
        __syncthreads();
        if (lane == 0) lds[0][wave] = __popcll(m);
        __syncthreads();
        int before = at;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) before += lds[0][w];
            at += lds[0][w];
        }
        if (is) order[before + __popcll(m & (((uint64_t)1 << lane) - 1))] = p;
    }
}

// Tile `tile` of BC pairs.  Expert e's tiles are numbered off[e] / BC + e and on:
// there are at most off[e + 1] / BC + 1 - off[e] / BC of them, so no two experts'
// meet and the last number is below P / BC + experts.  False: a number that no
// tile has.
struct Tile {
    int e, first, count;  // its pairs: order[first ..), at most BC of them
};
__device__ __forceinline__ bool find_tile(const int* off, int E, int tile, int BC, int lane, Tile* t) {
    int n = 0;
    for (int e = lane; e - lane < E; e += 64) n += __popcll(__ballot(e < E && off[min(e, E)] / BC + e <= tile));
    t->e = n - 1;
    const int begin = off[t->e], end = off[t->e + 1];
    t->first = begin + (tile - (begin / BC + t->e)) * BC;
    t->count = min(BC, end - t->first);
    return t->count > 0;
}

// Any K and alignment.  64 weight rows (SwiGLU: 32 gate and the 32 up rows of the
// same outputs) by 32 pairs, four waves of 16 rows; a 128-k group at a time comes
// through registers to LDS, the weights unpacked on the way.
constexpr int AR = 64, AC = 32, ALD = 136;

template <bool SWIGLU>
__global__ void __launch_bounds__(256) moe_any(const Params p) {
    __shared__ __attribute__((aligned(16))) uint16_t ws[AR][ALD];
    __shared__ __attribute__((aligned(16))) uint16_t xs[AC][ALD];
    __shared__ int pair[AC];
    const MoeArgs& a = p.a;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, h = lane >> 4;
    const int tr = blockIdx.x % p.rows_t;
    Tile t;
    if (!find_tile(p.off, a.experts, blockIdx.x / p.rows_t, AC, lane, &t)) return;
    if (tid < AC) pair[tid] = p.order[t.first + min(tid, t.count - 1)];
    __syncthreads();
    constexpr int OR = SWIGLU ? AR / 2 : AR;  // outputs of a tile
    const int r0 = tr * OR, O = a.O, K = a.K, G = p.G;
    const int64_t R = SWIGLU ? 2 * (int64_t)O : O;
    // weight row of tile row i (past the end: the last one, whose results go nowhere)
    auto row = [&](int i) { return (SWIGLU && i >= OR ? (int64_t)O : 0) + min(r0 + i % OR, O - 1) + t.e * R; };
    f32x4 acc[2] = {};
    for (int g = 0; g < G; ++g) {
        {
            // weights: 64 rows x 4 pieces of 16 bytes
            const int i = tid >> 2, c = tid & 3;
            const int64_t r = row(i);
            const uint8_t* src = a.W + r * (K / 2) + 64 * g + 16 * c;
            const int n = K / 2 - (64 * g + 16 * c);
            u32x4 w = {0u, 0u, 0u, 0u};
            if (n >= 16) w = load_any16(src);
            else
                for (int b = 0; b < n; ++b) w[b >> 2] |= (unsigned)src[b] << (8 * (b & 3));
            const float z = rintf(h2f(a.zero[r * G + g]));
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                unsigned o[4];
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    o[b] = pack2h((float)((w[d] >> (8 * b + 4)) & 15u) - z, (float)((w[d] >> (8 * b)) & 15u) - z);
                *reinterpret_cast<u32x4*>(&ws[i][32 * c + 8 * d]) = u32x4{o[0], o[1], o[2], o[3]};
            }
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {  // rows of X: 32 x 16 pieces of 8
            const int i = (tid >> 4) + 16 * j, c = tid & 15;
            const int q = pair[i];
            const uint16_t* src = a.X + (int64_t)(SWIGLU ? p.k.div(q) : q) * K + 128 * g + 8 * c;
            const int n = K - (128 * g + 8 * c);
            u32x4 x = {0u, 0u, 0u, 0u};
            if (n >= 8) x = load_any16(reinterpret_cast<const unsigned char*>(src));
            else
                for (int b = 0; b < n; ++b) x[b >> 1] |= (unsigned)src[b] << (16 * (b & 1));
            *reinterpret_cast<u32x4*>(&xs[i][8 * c]) = x;
        }
        __syncthreads();
        f32x4 P[2] = {};
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f16x8 wf = bitcast<f16x8>(*reinterpret_cast<const u32x4*>(&ws[16 * wave + l16][32 * s + 8 * h]));
#pragma unroll
            for (int j = 0; j < 2; ++j)
                P[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    bitcast<f16x8>(*reinterpret_cast<const u32x4*>(&xs[16 * j + l16][32 * s + 8 * h])), wf, P[j], 0, 0, 0);
        }
        const float sc = h2f(a.scale[row(16 * wave + l16) * G + g]);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) acc[j][v] = fmaf(sc, P[j][v], acc[j][v]);
        __syncthreads();
    }
    // a lane holds weight row l16 of its wave and pairs 4 h .. 4 h + 3 of each 16
    if constexpr (SWIGLU) {
        float* up = reinterpret_cast<float*>(ws);  // [32 outputs][32 pairs], one more apart
        if (wave >= 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int v = 0; v < 4; ++v) up[(16 * (wave - 2) + l16) * 33 + 16 * j + 4 * h + v] = acc[j][v];
        }
        __syncthreads();
        if (wave >= 2) return;
        const int o = r0 + 16 * wave + l16;
        if (o >= O) return;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = 16 * j + 4 * h + v;
                if (c >= t.count) continue;
                const float x = acc[j][v];
                a.Y[(int64_t)pair[c] * O + o] = f2h(x / (1.0f + expf(-x)) * up[(16 * wave + l16) * 33 + c]);
            }
    } else {
        const int o = r0 + 16 * wave + l16;
        if (o >= O) return;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int c = 16 * j + 4 * h + v;
                if (c < t.count) p.part[(int64_t)pair[c] * O + o] = acc[j][v];
            }
    }
}

// Y[t] = alpha sum_j w[t, j] part[t top_k + j] + beta Y[t], places in order; a
// place without an expert is left out.
__global__ void __launch_bounds__(256) moe_combine(const Params p) {
    const MoeArgs& a = p.a;
    const int64_t n = (int64_t)a.T * a.O, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += step) {
        const int t = (int)(i / a.O), o = (int)(i - (int64_t)t * a.O);
        float sum = 0.0f;
        for (int j = 0; j < a.top_k; ++j) {
            const int q = t * a.top_k + j;
            if ((unsigned)a.ids[q] >= (unsigned)a.experts) continue;
            sum = fmaf(a.weights ? a.weights[q] : 1.0f, p.part[(int64_t)q * a.O + o], sum);
        }
        float y = a.alpha * sum;
        if (a.beta != 0.0f) y = fmaf(a.beta, h2f(a.Y[i]), y);
        a.Y[i] = f2h(y);
    }
}

namespace {

size_t round256(size_t b) { return (b + 255) & ~(size_t)255; }

}  // namespace
}  // namespace moe

clove_status_t launch_moe_w4a16(const MoeArgs& a, bool swiglu, hipStream_t stream) {
    using namespace moe;
    DeviceInfo dev;
    if (const clove_status_t st = current_device_info(&dev); st != CLOVE_OK) return st;
    Params p;
    p.a = a;
    p.P = a.T * a.top_k;
    p.G = cdiv(a.K, 128);
    p.k = FastDiv(a.top_k);
    const size_t off = round256((size_t)(a.experts + 1) * 4), order = round256((size_t)p.P * 4);
    const size_t part = swiglu ? 0 : (size_t)p.P * a.O * 4;
    void* buf = nullptr;
    clove_status_t st = acquire_buffer(stream, kBufMoe, off + order + part, &buf);
    if (st != CLOVE_OK) return st;
    char* at = static_cast<char*>(buf);
    p.off = reinterpret_cast<int*>(at);
    p.order = reinterpret_cast<int*>(at + off);
    p.part = reinterpret_cast<float*>(at + off + order);
    CLOVE_LAUNCH(moe_sort, dim3((unsigned)a.experts), dim3(256), 0, stream, a.ids, p.P, a.experts, p.off, p.order);
    p.rows_t = cdiv(a.O, swiglu ? AR / 2 : AR);
    const int64_t tiles = ((int64_t)p.P / AC + a.experts) * p.rows_t;
    if (swiglu) CLOVE_LAUNCH(moe_any<true>, dim3((unsigned)tiles), dim3(256), 0, stream, p);
    else CLOVE_LAUNCH(moe_any<false>, dim3((unsigned)tiles), dim3(256), 0, stream, p);
    if (!swiglu) {
        const int64_t n = cdiv64((int64_t)a.T * a.O, 256);
        CLOVE_LAUNCH(moe_combine, dim3((unsigned)(n < 16384 ? n : 16384)), dim3(256), 0, stream, p);
    }
    return check_launch();
}

}  // namespace clove

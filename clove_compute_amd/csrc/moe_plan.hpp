// Which kernels a call of the experts' products takes, by its sizes and the number of
// CUs alone.  Plain C++ without device code: tests/test_moe_plan.py builds it for the
// host and holds the kernels' tests to the kernels that they name.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>

namespace clove {
namespace moe {

constexpr int NG = 4;      // 128-k groups of a unit (few pairs)
constexpr int SCAN = 16;   // ids a thread holds where the workgroups make their tile's list themselves
constexpr int AR = 64, AC = 32;  // moe_any: weight rows and pairs of a tile

constexpr int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// More threads than a launch counts (2^32 in a dimension)
constexpr bool too_many(int64_t workgroups, int threads) { return workgroups > ((int64_t)0xffffffff) / threads; }

// One part of a call (MoeArgs): `aligned`: K > 0, K % 32 == 0, X and W on 16 bytes
struct Call {
    bool swiglu, aligned;
    int T, top_k, experts, O, K, cus;
    int P() const { return T * top_k; }
    int G() const { return (int)up(K, 128); }
};

// Tokens at a time: X below the 2^31 bytes that a buffer's offsets reach, at most 2^19 pairs, so
// that the lists and launches are small beside the products.  (0: not even one.  In std::min's 64
// bits: HIP's own min on the host is of 32.)
inline int64_t tokens_at_a_time(bool swiglu, int top_k, int K) {
    const int64_t per_token = (int64_t)(swiglu ? 1 : top_k) * K * 2, pairs = (int64_t)1 << 19;
    return std::min(pairs, per_token ? (((int64_t)1 << 31) - 1) / per_token * top_k : pairs) / top_k;
}

enum class Way { kToken, kExpert, kTiles, kAny };  // moe_few_down, moe_few, moe_tile, moe_any
enum class Shape { kMany, kSome, kThin, kSmall };
struct Dims {
    int rows, pairs;  // of a tile
};
constexpr Dims dims(Shape s) {
    return s == Shape::kMany ? Dims{256, 128} : s == Shape::kSome ? Dims{128, 64} : s == Shape::kThin ? Dims{128, 32} : Dims{64, 32};
}

struct Choice {
    Way way = Way::kAny;
    int blocks = 1, waves = 4;     // kToken: 16-row blocks and waves of a workgroup
    int pairs = 8;                 // kExpert: pairs at a time
    Shape shape = Shape::kThin;    // kTiles
    int splits = 1;                // kTiles: parts of K asked for
    int chunk = 0;                 // outputs at a time
};

// Tiles of `on` outputs (about: half of an expert's last tile is empty, and an expert hit has one)
inline int64_t tiles(Shape s, const Call& c, int on) {
    const Dims d = dims(s);
    return up(on, c.swiglu ? d.rows / 2 : d.rows) * std::max(c.P() / d.pairs + (c.experts + 1) / 2, std::min(c.P(), c.experts));
}

// What runs first to its end by an estimate.  Workgroups: whole rounds of as many as the CUs
// hold, and the rest, which takes less time the fewer of them share a CU (`time`: of one beside
// 0, 1, 2 others, 1 for a 128 x 64 tile alone on its CU, which takes 0.8 us for a group and ten
// groups' worth to begin and end).  Where they leave CUs idle K is split: more workgroups, and
// fp32 sums of the parts to write and add up (for SwiGLU by a launch more).  Over 187 drawn
// shapes that go to tiles the choice is 1.4 % off the best of all kernels, shapes and splits on
// average and 1.4 times at worst; of the 108 of few pairs (choose()) 2.9 % and 2.3 times.
// Some (us, weights from HBM):
//                                             256 x 128  128 x 64  128 x 32
//   up 4096 on 8 experts of 22016 rows of 4096     747       898
//   up 20000 on 128 of 768 of 4896                 296       229
//   up 7388 on 16 of 1536 of 8192                  257       288       411
//   up 4736 on 128 of 11008 of 512                 219       171       176
//   up 1090 on 64 of 1024 of 1024, 5 an expert                37        34
//   down 3000 on 64 of 2048 of 1408                           52        57
//   up 600 on 64 of 2816 of 2048                              71        57
//                                              parts of K:  1    2    4    8
//   down 107 on 8 of 256 of 8192, 128 x 32                  42   26   19   16
//   down 42 on 8 of 2048 of 8192                            43   28   28   31
//   down 184 on 8 of 1408 of 14336                          75   44   45   41
//   up 216 on 8 of 1536 of 14336                            73   54   50   49
//   up 857 on 16 of 4096 of 1408                            32   43   57   75
// (128 x 32 with two stages ahead and three workgroups a CU; two with three stages 42.5
// against 38.6 for 15 pairs of 2048 rows of 1408 down.)  And 64 x 32 where 128 x 32 leaves half
// of the CUs idle (4 experts of 2 x 1024 rows of 4096, 25 pairs: 23.6, 24.3).  Half-group stages
// pay where stages of whole groups leave a CU one workgroup (256 x 128); elsewhere their
// 32-byte pieces of weight rows cost more than they bring (256 x 32, 7 pairs: 66 against 57).
template <int SLOTS>
inline float rounds(int64_t items, int cus, const float (&time)[SLOTS]) {
    const int64_t full = items / (SLOTS * cus), rest = items - full * SLOTS * cus;
    return full * time[SLOTS - 1] + (rest ? time[up(rest, cus) - 1] : 0.0f);
}

struct Plan {
    Shape shape = Shape::kThin;
    int splits = 1;
    float us = 0.0f;
};

inline Plan plan(const Call& c, int on) {
    Plan best;
    auto take = [&](Shape shape, int splits, float time) {
        const float sums = splits > 1 ? (float)splits * (0.5f + (float)c.P() * on * (c.swiglu ? 16 : 8) / 4.5e6f) + (c.swiglu ? 4.0f : 0.0f) : 0.0f;
        const float us = 0.8f * time * (up(c.G(), splits) + 10) + sums;
        if (best.us == 0.0f || us < best.us) best = {shape, splits, us};
    };
    take(Shape::kMany, 1, rounds(tiles(Shape::kMany, c, on), c.cus, {2.0f, 3.2f}));
    for (int splits : {1, 2, 3, 4, 6, 8}) {
        if (splits > 1 && ((int64_t)splits * c.P() * on * (c.swiglu ? 8 : 4) > (64 << 20) || c.G() < 4 * splits)) break;
        take(Shape::kSome, splits, rounds(splits * tiles(Shape::kSome, c, on), c.cus, {1.0f, 1.15f, 1.5f}));
        take(Shape::kThin, splits, rounds(splits * tiles(Shape::kThin, c, on), c.cus, {0.8f, 1.05f, 1.3f}));
    }
    if (best.shape == Shape::kThin && best.splits == 1 && 2 * tiles(Shape::kThin, c, on) < c.cus) best.shape = Shape::kSmall;
    return best;
}

// What a call takes, settled by its first part, whose pairs are the most
inline Choice choose(const Call& c) {
    Choice r;
    const int P = c.P(), G = c.G();
    // As many outputs at a time as workgroups of 256 threads for 16 of them and 32 pairs make a
    // launch; for down as their products have room in 512 MB, and as moe_combine's 65535
    // workgroups of 512 outputs cover
    int64_t most = (int64_t)16 * ((1 << 24) - 8) / (P / 32 + c.experts) / 256 * 256;
    if (!c.swiglu)
        most = std::min(std::min(most, (int64_t)512 * 65535), std::max((int64_t)256, ((int64_t)512 << 20) / ((int64_t)P * 4) / 256 * 256));
    r.chunk = most < c.O ? (int)(up(up(c.O, up(c.O, most)), 256) * 256) : c.O;
    // Below three pairs an expert on average: no lists, no tiles (64 experts of 2 x 1408 rows of
    // 2048, 6 a token: 20 tokens 45 us against 47 with tiles, 40 60 and 55, 80 89 and 59); below
    // eight where there are fewer tiles than half of the CUs and K is too short to be split (8
    // experts: 28 pairs down to 768 from 768 7.9 us and 11.0, 50 from 14336 to 1408 59 and 40)
    if (c.aligned && (P < 3 * c.experts || (P < 8 * c.experts && G <= 16 && 2 * tiles(Shape::kThin, c, c.O) < c.cus))) {
        // (2 pairs of an expert at a time while most have one or none, else 8: 1 token on 2 of 8
        // experts of 2 x 14336 rows of 4096 28.3 us against 32.2, 32 on 8 of 128 71 against 47)
        r.way = Way::kExpert;
        r.pairs = 2 * P <= c.experts ? 2 : 8;
        const int64_t grid = (int64_t)c.T * up(c.O, 16);
        if (!c.swiglu && 4 * P <= 3 * c.experts && !too_many(grid, 256)) {
            // Most experts hit have one pair: a workgroup for each token and 16 outputs (32 where that leaves
            // one a CU, or the waves with little: 41 tokens on 1 of 128, 2752 rows of 256 7.3 and 9.4 us)
            // takes one launch and no memory between.  It reads the weights of an expert hit twice twice, and
            // all of a token's places through one CU: by expert where that takes more than the second launch's
            // 4 us, at the 19 GB/s of a CU and 4.2 TB/s of all that both kernels reach (us, by token and by
            // expert: 1 token on 8 of 16 experts, 704 rows of 8192 31.6 and 15.2, 6 of 16, 1472 of 2048 8.6
            // and 10.0; 10 on 6 of 128, 2048 of 8192 128 and 107; 8 on 1 of 128, 1024 of 4096 7.3 and 10.6)
            const float mb = (float)c.O * c.K * 0.53e-6f, places = std::min(c.top_k, c.experts), units = up(G, NG);
            const float hit = c.experts * (1.0f - powf(1.0f - places / c.experts, c.T));
            if (std::max(units * c.top_k * 0.215f, P * mb / 4.2f) <= std::max(units * 0.43f, hit * mb / 4.2f) + 4.0f) {
                r.way = Way::kToken;
                if (grid <= 2 * (int64_t)c.cus) r.blocks = grid <= c.cus ? 1 : 2, r.waves = 16;
                else r.blocks = units * c.top_k <= 2 ? 2 : 1, r.waves = 4;
            }
        }
        return r;
    }
    // (tiles: an expert's weights below the 2^31 bytes that a buffer's offsets reach; launch_moe_w4a16 bounds X)
    if (c.aligned && (int64_t)(c.swiglu ? 2 : 1) * c.O * (c.K / 2) < ((int64_t)1 << 31)) {
        r.way = Way::kTiles;
        const Plan best = plan(c, r.chunk);
        r.shape = best.shape;
        r.splits = best.splits;
    }
    return r;
}

}  // namespace moe
}  // namespace clove

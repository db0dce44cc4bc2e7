// How the attention kernel shares the keys out to its workgroups.  Plain C++
// without device code: tests/test_paged_plan.py builds it for the host.
#pragma once

#include <cstdint>

namespace clove {
namespace paged {

constexpr int kW = 4;         // waves of a workgroup
constexpr int kLongest = 64;  // x 32 keys: longer chunks only where kRounds are not enough
constexpr int kRounds = 6;    // times the CUs' fill: the most chunks, but for remainders
constexpr int kRoom = 16384;  // completion counters: what a bound workspace holds

constexpr int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The host's part, by the bound of the lengths: `span` keys at most in each of
// `batch` sequences, `per` (KV head, tile)s in each of those, `fill` workgroups that
// the CUs hold at once.
struct Plan {
    bool cuts;       // sequences are cut at all
    int64_t rounds;  // most times `fill` workgroups
    int64_t slots;   // most workgroups with keys
};

// Chunks: the CUs' fill a whole number of rounds, and a remainder of each sequence,
// but no more than whole sequences make of the shortest chunks.  Rounds even out what
// one does not fill: 17 x 32 heads of 128 with 8192 keys 456 us in one, 419 in up to
// four, 407 in up to six, 406 in eight; 33 x 8 of 256 567, 431, 416, 416.  But their
// number goes by the bound of the lengths, and workgroups without keys take time: 32
// sequences of 1000 keys, 8 heads of 128, behind a bound of 131072, 29, 30, 34, 35 us,
// and 58 with the 31 that the bound has.  Where counters have no room for six there are
// fewer; where they have none for one, from about 7900 sequences x KV heads x tiles on,
// each of those is one workgroup's.
constexpr Plan plan(int64_t batch, int64_t per, int64_t span, int64_t fill) {
    const int64_t pairs = batch * per, wanted = up(pairs * up(span, 32), fill * kLongest);
    const int64_t fits = ((kRoom - pairs) / per - batch) * per / fill, most = fits < kRounds ? fits : kRounds;
    const int64_t rounds = wanted < 1 || most < 1 ? 1 : wanted < most ? wanted : most;
    const int64_t full = (up(fill * rounds, per) + batch) * per, fewest = pairs * up(span, 32 * kW);
    const int64_t slots = full < fewest ? full : fewest;
    return Plan{span > 32 * kW && pairs + slots <= kRoom, rounds, slots};
}

// The device's part: the chunk, in 32s of keys, for `sum` 32s in all sequences.
constexpr int chunk_of(int64_t sum, int per, int fill, int most_rounds) {
    const int64_t all = sum * per;
    int64_t rounds = most_rounds;
    if (rounds > 1) {  // (a 64-bit division is 0.1 us of a short call)
        const int64_t wanted = up(all, (int64_t)fill * kLongest);
        rounds = wanted < 1 ? 1 : wanted < rounds ? wanted : rounds;
    }
    const int64_t chunk = up(up(all, fill * rounds), kW) * kW;  // a wave takes every fourth of them
    return (int)(chunk < kW ? kW : chunk);
}

// Splits of a sequence of `t` 32s of keys, and the chunk of each
constexpr int splits_of(int t, int chunk) { return t <= chunk ? 1 : (t + chunk - 1) / chunk; }
constexpr int own_chunk(int t, int splits) { return ((t + splits - 1) / splits + kW - 1) / kW * kW; }

}  // namespace paged
}  // namespace clove

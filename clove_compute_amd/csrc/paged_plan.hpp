// How the attention kernel shares the keys out to its workgroups.  Plain C++
// without device code: tests/test_paged_plan.py builds it for the host.
#pragma once

#include <cstdint>

namespace clove {
namespace paged {

constexpr int kW = 4;         // waves of a workgroup
constexpr int kRoom = 16384;  // completion counters: what a bound workspace holds

constexpr int64_t up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The host's part, by the bound of the lengths: `span` keys at most in each of
// `batch` sequences, `per` (KV head, tile)s in each of those, `fill` workgroups that
// the CUs hold at once.
struct Plan {
    bool cuts;      // sequences are cut at all
    int64_t slots;  // most workgroups with keys
};

// As many workgroups as the CUs hold, and a remainder of each sequence, but no more
// than whole sequences make of the shortest chunks.  The bound of the lengths does not
// count beyond that: chunks of at most 2048 keys, and workgroups for as many of those
// as the bound has, were slower (32 sequences of 8 KV heads of 128 behind a bound of
// 131072, 1000 keys each, 57 and 29 us, workgroups without keys taking the difference;
// 16 x 4096 keys of 32 heads 187 and 181; 32 of 131072 keys down to 130 505 and 518)
// and had no room for their counters in bounds that are not rare.  Where this has
// none, from about 7900 sequences x KV heads x tiles on, each of those is one
// workgroup's.
constexpr Plan plan(int64_t batch, int64_t per, int64_t span, int64_t fill) {
    const int64_t full = (up(fill, per) + batch) * per, fewest = batch * per * up(span, 32 * kW);
    const int64_t slots = full < fewest ? full : fewest;
    return Plan{span > 32 * kW && batch * per + slots <= kRoom, slots};
}

// The device's part: the chunk, in 32s of keys, for `sum` 32s in all sequences.
constexpr int chunk_of(int64_t sum, int per, int fill) {
    const int64_t chunk = up(up(sum * per, fill), kW) * kW;  // a wave takes every fourth of them
    return (int)(chunk < kW ? kW : chunk);
}

// Splits of a sequence of `t` 32s of keys, and the chunk of each
constexpr int splits_of(int t, int chunk) { return t <= chunk ? 1 : (t + chunk - 1) / chunk; }
constexpr int own_chunk(int t, int splits) { return ((t + splits - 1) / splits + kW - 1) / kW * kW; }

}  // namespace paged
}  // namespace clove

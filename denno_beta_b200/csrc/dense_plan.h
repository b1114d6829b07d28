// How a dense product is divided among clusters of blocks (dense_tc.cuh, dense_pair.cuh): host code without a CUDA call, so that it is tested without a device.
// at_once[s]: clusters of s (blocks or pairs) that the device holds at once, 0 where it holds none or could not say.  at_once[1] is at least 1.
#pragma once

namespace dnb {

// Into how many parts K is split.  A block costs its chunks of K and, in chunks, what starting and joining it takes (about 100 KB of weights' time);
// a second block on an SM costs 0.85 of another turn, as an SM's share of the memory's rate is nearly that of one block; another wave costs a whole
// turn.  us a call for 1 to 8 parts: 4 tokens, 4096 -> 10240 gated in bf16 (80 tiles) 36, 39, 33, 39, 35, 35, 40, 38; dx of 77 tokens (17 tiles, one
// block an SM) - , -, 32, 28, 25, 24, 36, 34 (beyond 6 parts the clusters take two waves); 4-bit 12288 -> 4096 (32 tiles) -, -, 9.7, 8.5, 8.6, 8.3, 7.8, 7.6.
inline int best_splits(const int (&at_once)[9], int sm_count, int stage_bytes, int tiles, int chunks) {
    const float start = 100.f * 1024.f / stage_bytes;
    int best = 1;
    float least = 0.f;
    for (int s = 1; s <= 8 && s <= chunks; ++s) {
        if (at_once[s] < 1) continue;
        const int waves = (tiles + at_once[s] - 1) / at_once[s], blocks = (tiles < at_once[s] ? tiles : at_once[s]) * s;
        const float turns = 1.f + 0.85f * ((blocks + sm_count - 1) / sm_count - 1);
        const float cost = waves * (start + (chunks + s - 1) / s * turns) + 0.15f * s;
        if (s == 1 || cost < least) best = s, least = cost;
    }
    return best;
}

// Pairs a cluster and how many tiles are not split.  A tile costs its chunks of K and about four more; a split one a part of the chunks and about
// fourteen (shares written, the cluster waited for, sums read).  us a call without / with: dx of 256 tokens, 2048 -> 5632 (8 tiles of 176 chunks) 65 / 31, of
// 1024 tokens 66 / 43; 4-bit 512 tokens, 12288 -> 4096 (32 tiles of 48) 23.8 / 18; gated 512 tokens, 2560 -> 9728 in fp16 (152 tiles of 40) 48.4 / 43;
// 4-bit 256 tokens, 4096 -> 4096 (16 tiles of 16) 10.2 / 10.9, gated 1024 tokens, 1024 -> 2560 (80 tiles of 16) 15.2 / 16.8.
struct PairPlan {
    int parts, whole;       // pairs a cluster; tiles that are not split (the rest: one a cluster)
    int pairs, each, more;  // launched; whole tiles a pair, one more for the first `more` pairs
};
inline PairPlan pair_plan(const int (&at_once)[5], int tiles, int chunks) {
    PairPlan p = {};
    int clusters = 1;
    float least = 0.f;
    for (int s = 1; s <= 4; ++s) {
        const int n = at_once[s];
        if (n < 1) continue;
        const int turns = tiles / (n * s), rest = tiles - turns * n * s;
        const bool split = s > 1 && rest > 0 && rest <= n && chunks >= s;
        const float cost = turns * (chunks + 4.f) + (rest == 0 ? 0.f : split ? (float)((chunks + s - 1) / s) + 14.f : chunks + 4.f);
        if (s == 1 || cost < least) least = cost, p.parts = s, p.whole = split ? turns * n * s : tiles, clusters = n;
    }
    const int used = p.parts > 1 && p.whole > 0 ? clusters : tiles < clusters ? tiles : clusters;
    p.pairs = used * p.parts;
    p.each = p.whole / p.pairs;
    p.more = p.whole % p.pairs;
    return p;
}

}  // namespace dnb

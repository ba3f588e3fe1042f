// Which sequences of a batched step read their common leading pages once (host code without CUDA: tests/test_shared_group_host.py runs it).
#pragma once
#include <stdint.h>

namespace b2 {

constexpr int SHARED_GROUP_MAX = 64;      // sequences: members are bits

// the members, and the tokens of the pages that all their tables begin with. n 0: no group of which reading them once is worth the launches
struct SharedGroup { int n = 0, tokens = 0; uint64_t members = 0; };

// Measured per layer (32 heads over 8 KV heads of 128; saved, us): three launches instead of one cost about 7 us, won back from about 16384 tokens in all:
// 8 sequences behind 512 tokens -1.3, 1024: 1.4, 4096: 19; 16 behind 512 -1.7, 1024: 3.5, 4096: 36; 32 behind 256 -7, 512: -0.9, 1024: 13, 4096: 87; 64 behind
// 128 -7, 256: -0.5, 512: 13, 4096: 183. Where prefix and own tokens are one launch (16 rows a KV head): 4 behind 128 0.9, 4096: 6. The other sequences of the
// step take a launch more: with one of those, 16 behind 1024 -3.4, 4096: 24; 32 behind 512 -13, 1024: 0.6, 4096: 70; 63 behind 512 5, 4096: 170.
inline bool shared_group_pays(int n, int n_all, long tokens, int heads_a_kv) {
    return n < 2 ? false : n == n_all && n * heads_a_kv <= 16 ? tokens >= 128 : tokens * n >= (n == n_all ? 16384 : 32768);
}

// Of all sets of sequences whose tables begin with the same pages, the one with most tokens to read once (members times common tokens) of those that pay.
// Sequence i has n_pages[i] whole pages pages[i][..] behind which it writes. Tables that begin alike are the nodes of a tree: a node is the sequences that share its
// pages, it goes on as long as all of them do and then splits by their next page. Every page is looked at once for each table, as in comparing them with the
// first one's; a node whose sequences could not make a larger set is not looked into.
inline SharedGroup shared_group_of(const int32_t* const* pages, const int* n_pages, int n_all, int block_tokens, int heads_a_kv) {
    SharedGroup best;
    struct Node { uint64_t members; int depth; } open[SHARED_GROUP_MAX];      // (disjoint sets of two or more: half as many at most)
    int n_open = 0;
    open[n_open++] = {n_all < 64 ? (1ull << n_all) - 1 : ~0ull, 0};
    while (n_open) {
        const Node node = open[--n_open];
        uint64_t left = node.members;
        for (int i = 0; i < n_all; i++) {
            if (!(left >> i & 1) || n_pages[i] <= node.depth) continue;
            uint64_t with = 0;
            int n = 0, shortest = n_pages[i], longest = shortest;
            for (int j = i; j < n_all; j++) {
                if (!(left >> j & 1) || n_pages[j] <= node.depth || pages[j][node.depth] != pages[i][node.depth]) continue;
                with |= 1ull << j; n++;
                shortest = shortest < n_pages[j] ? shortest : n_pages[j];
                longest = longest > n_pages[j] ? longest : n_pages[j];
            }
            left &= ~with;
            if (n < 2) continue;
            for (int j = i + 1; j < n_all; j++) {                // the pages that all of them begin with
                if (!(with >> j & 1)) continue;
                int same = node.depth + 1;
                while (same < shortest && pages[j][same] == pages[i][same]) same++;
                shortest = same;
            }
            const long tokens = (long)shortest * block_tokens;
            if (tokens * n > (long)best.n * best.tokens && shared_group_pays(n, n_all, tokens, heads_a_kv)) { best.n = n; best.tokens = (int)tokens; best.members = with; }
            // (a part of them has fewer members and at most the longest one's pages)
            if (n > 2 && (long)(n - 1) * longest * block_tokens > (long)best.n * best.tokens) open[n_open++] = {with, shortest};
        }
    }
    return best;
}

}  // namespace b2

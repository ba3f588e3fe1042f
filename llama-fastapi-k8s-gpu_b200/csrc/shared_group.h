// Which sequences of a batched step read their common leading pages once (host code without CUDA: tests/test_shared_group_host.py runs it).
#pragma once
#include <stdint.h>

namespace b2 {

constexpr int SHARED_GROUP_MAX = 64;      // sequences: members are bits

// the members, and the tokens of the pages that all their tables begin with. n 0: no group of which reading them once is worth the launches
struct SharedGroup { int n = 0, tokens = 0; uint64_t members = 0; };

// The same tables read by every sequence for itself, or the common pages once: us a layer that the second saves (4 layers, 22 of the 4 x 64 shape, Q4_K_M).
//   whole step, 32 heads over 8 KV heads of 128: 8 sequences behind 512 tokens -1.7, 1024: 0.9, 2048: 1.0, 4096: 13; 16 behind 512 -3.1, 1024: 2.5, 4096: 35; 32 behind
//     512 -2.5, 1024: 9, 4096: 79; 64 behind 256 -2.3, 512: 10, 4096: 176. 64 over 8 of 128: 16 behind 512 -2.1, 1024: 3.7; 32 behind 512 -2.7, 1024: 8.7; 64
//     behind 256 -0.4, 512: 9. 32 over 4 of 64: 8 to 64 behind 64 to 2048 11 to 55; 32 over 32 of 128: 8 to 32 behind 64 to 2048 12 to 189 (here the chain of launches
//     behind the other form is slower, whatever the lengths). 16 rows a KV head, one launch for both parts: 4 of 32 over 8 of 128 behind 128 0.5, 2048: -0.3, 4096: 4.
//   beside others, which take a launch more; 32 sequences of 33, 57 of 64 and 26 of 33: 32 over 32 of 128, 1024 tokens: 74, 133, 47; 32 over 8 of 128 (4 heads a KV
//     head), 1024: -2, 19, -6, 2048: 20, 63, 14; 64 over 8 of 128 (8), 1024: -8, 13, -13, 2048: 13, 57, 5; 32 over 4 of 64 (8), 1024: -6, 0, -6, 2048: 3.5, 21, 2.8.
// What is lost goes with the query heads (queries, partial results, joining), what is saved with the KV heads; so the bar goes with the heads a KV head has.
inline bool shared_group_pays(int n, int n_all, long tokens, int heads_a_kv, int kv_width) {
    if (n < 2) return false;
    if (n < n_all) return tokens * n >= (heads_a_kv > 5 ? 6144 * heads_a_kv : 32768);
    if (n * heads_a_kv <= 16) return tokens >= 128;
    return tokens * n >= (n > 16 && heads_a_kv >= 4 && kv_width >= 1024 ? 20480 : 16384);
}

// Of all sets of sequences whose tables begin with the same pages, the one with most tokens to read once (members times common tokens) of those that pay.
// (kv_width: KV heads times their size.) Sequence i has n_pages[i] whole pages pages[i][..] behind which it writes. Tables that begin alike are the nodes of a tree: a node is the sequences that share its
// pages, it goes on as long as all of them do and then splits by their next page. Every page is looked at once for each table, as in comparing them with the
// first one's; a node whose sequences could not make a larger set is not looked into.
inline SharedGroup shared_group_of(const int32_t* const* pages, const int* n_pages, int n_all, int block_tokens, int heads_a_kv, int kv_width) {
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
            if (tokens * n > (long)best.n * best.tokens && shared_group_pays(n, n_all, tokens, heads_a_kv, kv_width)) { best.n = n; best.tokens = (int)tokens; best.members = with; }
            // (a part of them has fewer members and at most the longest one's pages)
            if (n > 2 && (long)(n - 1) * longest * block_tokens > (long)best.n * best.tokens) open[n_open++] = {with, shortest};
        }
    }
    return best;
}

}  // namespace b2

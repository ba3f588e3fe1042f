// Log probabilities of given tokens, the entropy of every row, and its most likely tokens, from one pass over the logits.
// With m the row's largest logit, L = log2 e, d_i = (x_i - m) L, S = sum 2^d_i, T = sum d_i 2^d_i:
//   logprob(t) = x_t - m - log2 S / L,   entropy = (log2 S - T / S) / L.
// Every thread keeps (m, S, T) of its entries, S and T against its own running maximum; they are joined over the CTA and, where a row has a cluster of CTAs, over
// the cluster. A masked entry (-infinity) adds nothing; a row of nothing else gets log probabilities of -infinity and entropy 0; a NaN makes the row's
// numbers NaN.
//
// The most likely tokens come from the same pass: a thread's running maximum bounds its entries. Of the maxima of 32 to 128 groups of threads (at least twice n)
// the n-th largest is reached by n entries at least, so that the n most likely are among the entries that reach it, which lie with the few threads whose maximum
// does; their entries are read once more (from L2) and ranked by (value, lower id). Where those are too many (thousands of equal entries, a row masked but for
// a few), the ones above the bound are ranked and the equal ones taken in the order of their ids; what that does not settle is searched n times.
//
// Bound by memory for many rows (each logit read once: 1024 rows of 128256 in 32 bits 93 us in a graph, 5.65 TB/s; 102 a call), by the latency of the phases behind the pass
// for few (32 rows 13 us, of which the pass is 4; one row of 32000 7.6; calls 14.3 and 9.1).
#include "device_ops.h"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <math.h>

namespace b2 {

namespace {
constexpr int LP_THREADS = 256, LP_WARPS = LP_THREADS / 32;
constexpr int LP_CAND = 1024;             // entries that may be ranked
constexpr float LP_LOG2E = 1.4426950408889634f, LP_LN2 = 0.6931471805599453f;
constexpr float LP_FLOOR = -200.f;        // 2^-200 is 0 in 32 bits: keeps d 2^d of a masked entry from being infinity times 0

__device__ __forceinline__ float lp_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ unsigned lp_key(float x) {      // larger float <-> larger key; NaN lowest, -0 like 0
    if (x != x) return 0u;
    const unsigned u = __float_as_uint(x + 0.f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

template <typename T> __device__ __forceinline__ float lp_float(T v);
template <> __device__ __forceinline__ float lp_float(float v) { return v; }
template <> __device__ __forceinline__ float lp_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float lp_float(__nv_bfloat16 v) { return __bfloat162float(v); }

struct Sums { float m, s, t; };           // largest entry; sum 2^d, sum d 2^d against it
__device__ __forceinline__ Sums lp_join(const Sums& a, const Sums& b) {
    const float m = fmaxf(a.m, b.m), ref = m == -INFINITY ? 0.f : m;
    const float da = fmaxf((a.m - ref) * LP_LOG2E, LP_FLOOR), db = fmaxf((b.m - ref) * LP_LOG2E, LP_FLOOR);
    const float ca = lp_exp2(da), cb = lp_exp2(db);
    return {m, ca * a.s + cb * b.s, ca * (a.t + da * a.s) + cb * (b.t + db * b.s)};
}
__device__ __forceinline__ Sums lp_join_warp(Sums v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        v = lp_join(v, Sums{__shfl_xor_sync(0xffffffffu, v.m, o), __shfl_xor_sync(0xffffffffu, v.s, o), __shfl_xor_sync(0xffffffffu, v.t, o)});
    return v;
}

// entries [begin, end) of a row in pieces of VEC that start at 16-byte boundaries: piece p holds entries base + p VEC .. + VEC - 1 of the row, of which the first and
// the last piece may have some outside
template <typename T, int VEC>
struct Pieces {
    const T* row;
    int base, begin, end, n;
    __device__ Pieces(const T* row_, int begin_, int end_) : row(row_), begin(begin_), end(end_) {
        const int off = (int)(((uintptr_t)(row + begin) & 15) / sizeof(T));      // entries between the boundary below and `begin`
        base = begin - off;
        n = end > begin ? (end - base + VEC - 1) / VEC : 0;
    }
    __device__ int first(int p) const { return base + p * VEC; }
    // entries outside come out as -infinity (they add nothing and are never ranked: see id_ok)
    __device__ uint4 load(int p) const {
        const int i0 = first(p);
        if (p < n && i0 >= begin && i0 + VEC <= end) return __ldg(reinterpret_cast<const uint4*>(row + i0));
        uint4 raw;
        T* v = reinterpret_cast<T*>(&raw);
#pragma unroll
        for (int e = 0; e < VEC; e++) v[e] = p < n && i0 + e >= begin && i0 + e < end ? row[i0 + e] : (T)(-INFINITY);
        return raw;
    }
    static __device__ __forceinline__ float at(const uint4& raw, int e) { return lp_float(reinterpret_cast<const T*>(&raw)[e]); }
    __device__ bool id_ok(int id) const { return id >= begin && id < end; }
};

struct LpShared {
    Sums sums[LP_WARPS], cta;
    alignas(16) unsigned group[128];
    unsigned bound;
    int n_sel, n_cand, n_own, sel[LP_THREADS], warp_ties[LP_WARPS];
    unsigned long long cand[LP_CAND], own[LOGPROB_MAX_TOP], wbest[LP_WARPS];
};

__device__ __forceinline__ float lp_value(unsigned long long key) {      // of the entry that a rank key was made of (-0 comes back as 0)
    const unsigned k = (unsigned)(key >> 32);
    return k == 0 ? __int_as_float(0x7fffffff) : __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
__device__ __forceinline__ unsigned long long lp_rank_key(float x, int id) { return ((unsigned long long)lp_key(x) << 32) | (unsigned)~id; }

// ranks n keys (all different) in `keys`, the first `want` go to `put(rank, key)`
template <typename Put>
__device__ __forceinline__ void lp_rank(const unsigned long long* keys, int n, int want, Put put) {
    for (int i = threadIdx.x; i < n; i += LP_THREADS) {
        const unsigned long long k = keys[i];
        int above = 0;
        for (int j = 0; j < n; j++) above += keys[j] > k;
        if (above < want) put(above, k);
    }
}
__device__ __forceinline__ unsigned long long lp_cluster_key(uint32_t address) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(address) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lp_cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
}  // namespace

// cluster of `parts` CTAs a row (1: none); LP_UNROLL 16-byte pieces a thread has under way
template <typename T, int LP_UNROLL, int CTAS>
__global__ void __launch_bounds__(LP_THREADS, CTAS) logprobs_kernel(const LogprobArgs a, const RowMap map, int parts) {
    constexpr int VEC = 16 / sizeof(T);
    __shared__ LpShared sh;
    __shared__ unsigned long long all[8 * LOGPROB_MAX_TOP];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    griddep_wait();                                               // (in the engines' chains: the logits, the sampled tokens)
    const int part = parts > 1 ? (int)lp_cluster_rank() : 0, r = blockIdx.x / parts;
    const int to = map.n ? map.out[r] : r;
    const T* row = (const T*)a.logits + (long)r * a.row_stride;
    const int chunk = ((a.n_vocab + parts - 1) / parts + VEC - 1) / VEC * VEC;
    const Pieces<T, VEC> pc(row, min(a.n_vocab, part * chunk), min(a.n_vocab, (part + 1) * chunk));
    const int top = min(a.n_top, pc.end - pc.begin);              // of this CTA's entries
    if (tid == 0) { sh.n_sel = sh.n_cand = sh.n_own = 0; }

    // (the asked token's logit, read ahead by the thread that will want it)
    const int token = part == 0 && tid == 0 && a.logprob ? a.tokens[map.n ? map.token[r] : r] : -1;
    const bool has_token = token >= 0 && token < a.n_vocab;
    const float token_logit = has_token ? lp_float(row[token]) : 0.f;

    // ---- the pass
    Sums v = {-INFINITY, 0.f, 0.f};
    for (int p0 = tid; p0 < pc.n; p0 += LP_UNROLL * LP_THREADS) {
        uint4 x[LP_UNROLL];
#pragma unroll
        for (int u = 0; u < LP_UNROLL; u++) x[u] = pc.load(p0 + u * LP_THREADS);
        float m = v.m;
#pragma unroll
        for (int u = 0; u < LP_UNROLL; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) m = fmaxf(m, pc.at(x[u], e));
        const float ref = m == -INFINITY ? 0.f : m;
        const float dm = fmaxf((v.m - ref) * LP_LOG2E, LP_FLOOR), c = lp_exp2(dm);
        float s = c * v.s, t = c * (v.t + dm * v.s);
#pragma unroll
        for (int u = 0; u < LP_UNROLL; u++)
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float d = (pc.at(x[u], e) - ref) * LP_LOG2E, w = lp_exp2(d);
                s += w;
                t = fmaf(fmaxf(d, LP_FLOOR), w, t);
            }
        v = {m, s, t};
    }
    const unsigned mine = pc.n > tid ? lp_key(v.m) : 0u;
    const int size = a.n_top <= 16 ? 8 : a.n_top <= 32 ? 4 : 2, n_groups = LP_THREADS / size;
    if (a.n_top > 0) {                                            // maxima of groups of `size` threads
        unsigned g = max(mine, __shfl_xor_sync(0xffffffffu, mine, 1));
        if (size >= 4) g = max(g, __shfl_xor_sync(0xffffffffu, g, 2));
        if (size >= 8) g = max(g, __shfl_xor_sync(0xffffffffu, g, 4));
        if (tid % size == 0) sh.group[tid / size] = g;
    }
    const Sums w = lp_join_warp(v);
    if (lane == 0) sh.sums[warp] = w;
    __syncthreads();
    if (warp == 1) {
        Sums j = lane < LP_WARPS ? sh.sums[lane] : Sums{-INFINITY, 0.f, 0.f};
        j = lp_join_warp(j);
        if (lane == 0) sh.cta = j;
    }
    if (a.n_top > 0 && top > 0) {
        // ---- the top-th largest of the groups' maxima (equal ones in the groups' order; 0 where fewer groups have entries)
        if (tid < n_groups) {
            const unsigned g = sh.group[tid];
            int above = 0;
            for (int i = 0; i < n_groups; i += 4) {
                const uint4 o = *reinterpret_cast<const uint4*>(&sh.group[i]);
                above += (o.x > g || (o.x == g && i < tid)) + (o.y > g || (o.y == g && i + 1 < tid)) + (o.z > g || (o.z == g && i + 2 < tid)) + (o.w > g || (o.w == g && i + 3 < tid));
            }
            if (above == top - 1) sh.bound = g;
        }
        __syncthreads();
        const unsigned bound = sh.bound;
        const int rounds = (pc.n + LP_THREADS - 1) / LP_THREADS;
        // the entries whose keys are `from` or larger, as far as there is room
        auto collect = [&](unsigned from) {
            if (mine >= from && pc.n > tid) sh.sel[atomicAdd(&sh.n_sel, 1)] = tid;
            __syncthreads();
            const int n_sel = sh.n_sel;
            for (int i = tid; i < n_sel * rounds; i += LP_THREADS) {
                const int p = sh.sel[i % n_sel] + i / n_sel * LP_THREADS;
                const uint4 x = pc.load(p);
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    const int id = pc.first(p) + e;
                    if (lp_key(pc.at(x, e)) >= from && pc.id_ok(id)) {
                        const int at = atomicAdd(&sh.n_cand, 1);
                        if (at < LP_CAND) sh.cand[at] = lp_rank_key(pc.at(x, e), id);
                    }
                }
            }
            __syncthreads();
        };
        auto rank = [&](int want) { lp_rank(sh.cand, sh.n_cand, want, [&](int place, unsigned long long k) { sh.own[place] = k; }); };
        collect(bound);
        bool found = sh.n_cand <= LP_CAND && sh.n_cand >= top;    // (fewer: NaNs, which reach no bound)
        if (found) rank(top);
        else if (bound < 0xffffffffu) {
            // too many equal entries: those above the bound, then the ones at it in the order of their ids
            __syncthreads();
            if (tid == 0) sh.n_sel = sh.n_cand = 0;
            __syncthreads();
            collect(bound + 1);
            int at = sh.n_cand;
            if (at <= LP_CAND) {
                rank(top);
                for (int p0 = 0; at < top && p0 < pc.n; p0 += LP_THREADS) {
                    const uint4 x = pc.load(p0 + tid);
                    int ties = 0;
#pragma unroll
                    for (int e = 0; e < VEC; e++) ties += lp_key(pc.at(x, e)) == bound && pc.id_ok(pc.first(p0 + tid) + e);
                    int before = ties;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) { const int up = __shfl_up_sync(0xffffffffu, before, o); if (lane >= o) before += up; }
                    if (lane == 31) sh.warp_ties[warp] = before;
                    __syncthreads();
                    before += at - ties;
                    for (int i = 0; i < LP_WARPS; i++) { if (i < warp) before += sh.warp_ties[i]; at += sh.warp_ties[i]; }
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const int id = pc.first(p0 + tid) + e;
                        if (before < top && lp_key(pc.at(x, e)) == bound && pc.id_ok(id)) sh.own[before++] = lp_rank_key(pc.at(x, e), id);
                    }
                    __syncthreads();
                }
                found = at >= top;
            }
        }
        if (!found) {
            __syncthreads();
            // many equal entries or NaNs: one search per place, below the key of the place before
            unsigned long long below = ~0ull;
            for (int place = 0; place < top; place++) {
                unsigned long long best = 0;
                for (int p = tid; p < pc.n; p += LP_THREADS) {
                    const uint4 x = pc.load(p);
#pragma unroll
                    for (int e = 0; e < VEC; e++) {
                        const int id = pc.first(p) + e;
                        const unsigned long long k = lp_rank_key(pc.at(x, e), id);
                        if (pc.id_ok(id) && k < below && k > best) best = k;
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
                if (lane == 0) sh.wbest[warp] = best;
                __syncthreads();
                for (int i = 0; i < LP_WARPS; i++) best = max(best, sh.wbest[i]);
                if (tid == 0) sh.own[place] = best;
                below = best;
                __syncthreads();
            }
        }
    }
    if (tid == 0) sh.n_own = a.n_top > 0 ? max(0, top) : 0;
    __syncthreads();

    // ---- the row's first CTA joins the parts and writes
    Sums total = sh.cta;
    const unsigned long long* keys = sh.own;
    int n_keys = sh.n_own;
    if (parts > 1) {
        cluster_sync();
        if (part != 0) { cluster_sync(); return; }                // (its shared memory is read until then)
        if (warp == 0) {                                          // (a lane a part)
            const uint32_t at = cluster_address(smem_u32(&sh.cta), min(lane, parts - 1));
            float f[3];
#pragma unroll
            for (int e = 0; e < 3; e++) asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f[e]) : "r"(at + 4 * e) : "memory");
            const Sums j = lp_join_warp(lane < parts ? Sums{f[0], f[1], f[2]} : Sums{-INFINITY, 0.f, 0.f});
            if (lane == 0) sh.sums[0] = j;
        }
        if (a.n_top > 0) {
            // part i has min(n_top, its entries) keys
            n_keys = 0;
            for (int i = 0; i < parts; i++) {
                const int have = min(a.n_top, max(0, min(a.n_vocab, (i + 1) * chunk) - min(a.n_vocab, i * chunk)));
                const uint32_t at = cluster_address(smem_u32(&sh.own[0]), i);
                for (int j = tid; j < have; j += LP_THREADS) all[n_keys + j] = lp_cluster_key(at + 8 * j);
                n_keys += have;
            }
            keys = all;
        }
        __syncthreads();
        total = sh.sums[0];
        cluster_sync();
    }
    const float log2_s = log2f(total.s), ref = total.m == -INFINITY ? 0.f : total.m;
    auto logprob = [&](float x) { return (x - ref) - log2_s * LP_LN2; };      // (not in powers of two: the type's lowest value stays finite)
    const bool none = total.s == 0.f;                              // every entry masked
    if (a.n_top > 0) {
        float* lp = a.top_logprob + (long)to * a.n_top;
        int* ids = a.top_id + (long)to * a.n_top;
        auto put = [&](int rank, unsigned long long k) {
            const int id = (int)~(unsigned)k;
            ids[rank] = id;
            lp[rank] = none ? -INFINITY : logprob(lp_value(k));
        };
        if (parts > 1) lp_rank(keys, n_keys, a.n_top, put);
        else for (int i = tid; i < n_keys; i += LP_THREADS) put(i, keys[i]);
        for (int i = min(a.n_top, a.n_vocab) + tid; i < a.n_top; i += LP_THREADS) { ids[i] = -1; lp[i] = -INFINITY; }
    }
    if (tid == 0) {
        if (a.entropy) a.entropy[to] = none ? 0.f : (log2_s - total.t / total.s) * LP_LN2;
        if (a.logprob) a.logprob[to] = !has_token || none ? -INFINITY : logprob(token_logit);
    }
}

template <typename T>
static cudaError_t logprobs_typed(const LogprobArgs& a, const RowMap& map, cudaStream_t s) {
    // few rows: up to eight CTAs a row, as long as four an SM hold them and a thread still has entries (rows of 128256, nothing in L2: with eight an SM 128 rows take
    // 30 us instead of 22, with two 256 rows 48 instead of 36)
    int parts = 1;
    while (parts < 8 && (long)a.n_rows * parts * 2 <= 4 * 148 && a.n_vocab / (parts * 2) >= 2 * LP_THREADS) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_rows * parts)); cfg.blockDim = dim3(LP_THREADS); cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = parts; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = parts > 1 ? 1 : 0;
    // Four CTAs an SM hold all of them: twice as many pieces under way a thread. 32 rows of 128256 14.3 -> 13.1 us, 128 25.7 -> 22.6, 500 of 32003 in bf16 15.1 ->
    // 14.4; more rows want the CTAs instead (1024 of 128256: 98 that way, 92 with eight CTAs an SM).
    if (cfg.gridDim.x <= 4 * 148) return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, 4, 4>, a, map, parts);
    return cudaLaunchKernelEx(&cfg, logprobs_kernel<T, 2, 8>, a, map, parts);
}

cudaError_t logprobs_launch(const LogprobArgs& a, cudaStream_t s, const RowMap* map) {
    if (a.n_rows == 0) return cudaSuccess;
    const RowMap none = {};
    switch (a.type) {
        case ELEM_F32: return logprobs_typed<float>(a, map ? *map : none, s);
        case ELEM_F16: return logprobs_typed<__half>(a, map ? *map : none, s);
        default: return logprobs_typed<__nv_bfloat16>(a, map ? *map : none, s);
    }
}

}  // namespace b2

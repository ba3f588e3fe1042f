// Attention of a batch over a paged cache whose first n_prefix tokens are the same pages for every sequence.
//   keys of row i of a sequence with n rows and c own tokens: the prefix, and own tokens 0 .. c - n + i;   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),
//   s_j = scale log2(e) q.k_j. No key: 0.
// Bound by the bytes of the cache: the prefix is read once for all rows, each sequence's own tokens once for its rows. With a prefix every pass leaves partial
// results (maximum, sum, weighted sum) of its keys in 32 bits, and a small kernel joins them; without one, the CTAs that share a tile's keys are a cluster and
// join through each other's shared memory.
//
// Three forms of a pass. A row of a tile is (token, head of the KV head's group).
//   up to 16 rows (single tokens): shared_prefix_step_kernel; the four computing warps share each tile of 64 keys. A CTA whose keys are done takes over the work
//     of one that has not started, so that copies of the next sequence are under way while this one ends.
//   up to 32 rows of the batch, or several tokens of a sequence: shared_prefix_rows_kernel; tiles of 64 rows, a warp has 16 of them and all keys.
//   more rows (the prefix of a batch): shared_prefix_tc.cu, on tensor memory.
// Both kernels here: mma.sync m16n8k16, keys and values by tensor copies (a warp of its own) in 128-byte-swizzled rows. They are bound by the copies, not by
// the products: 32 rows of 64 keys want 1 % of the tensor cores.
// The pass over single own tokens runs beside the prefix pass, on SMs that one leaves it (sp_share). With several rows a sequence behind a prefix on tensor memory it has
// the SMs that are left over, and else begins as CTAs of that pass end: no SM has registers for a CTA of each (320 and 160 threads of 168). Up to 16 rows of a KV
// head in the whole batch: one launch for both.
//
// Probabilities are rounded to the cache's type for the weighted sum (the other operand is the cache as it is); scores, maxima, sums, joins stay 32-bit.
#include "device_ops.h"
#include "ptx.cuh"
#include "tensor_map.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <limits.h>
#include <math.h>

namespace b2 {

namespace {
constexpr int SP_WARPS = 4, SP_THREADS = 32 * (SP_WARPS + 1);
constexpr int SP_TT = 64;            // keys of a tile
constexpr int sp_stages(int hd) { return hd == 64 ? 4 : 2; }             // tiles under way: 64 KB, three CTAs an SM

__device__ unsigned int sp_error[5];                             // see mbar_give_up
__device__ __forceinline__ unsigned int* sp_err(const SharedPrefixArgs& a) { return a.err ? a.err : sp_error; }

__device__ __forceinline__ float sp_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

template <typename E> struct SpType;
template <> struct SpType<__half> {
    static constexpr uint32_t EXP = 0x7c00u;                     // exponent bits: all set in an infinity or NaN
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ float value(uint16_t v) { return __half2float(*reinterpret_cast<const __half*>(&v)); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
template <> struct SpType<__nv_bfloat16> {
    static constexpr uint32_t EXP = 0x7f80u;
    static __device__ __forceinline__ uint32_t pack(float a, float b) { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    static __device__ __forceinline__ float value(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
    static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
};
__device__ __forceinline__ void sp_ldmatrix_x4(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ void sp_ldmatrix_x4_trans(uint32_t (&r)[4], const void* p) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(smem_u32(p)));
}
__device__ __forceinline__ uint32_t sp_cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float sp_cluster_load(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}
}  // namespace

struct SpPlan {
    int prefix_z;                // blockIdx.z that is the prefix for all rows (-1: none); the others are sequences
    int prefix_splits, splits;   // CTAs that share the keys of a tile of rows, of the prefix and of a sequence's own tokens
    int own_slot;                // >= 0: there is a prefix, and the own tokens' results are partial ones too, in slots from here on; -1: they are the output, and
                                 //   the CTAs that share a tile are a cluster
    int behind;                  // launched behind the prefix pass, which it runs beside
    int steal;                   // a CTA goes on with the work of CTAs that have not started (single-token form without clusters)
    int mrows;                   // rows of a tile that q is staged for (single-token form)
    int box_rows;                // keys of a copy: a page, or a power of two that divides it
    int slots;                   // joining: partial results of the prefix per row (< 0: as `cut` says)
    PrefixCut cut;
    size_t ml_at;                // where the (maximum, sum) of the partial results lie in the workspace
    PrefixShare share;           // adapt: the prefix pass has written down its cut
};

// partial results: [slot][row][head][head_dim] weighted sums, then [slot][row][head][2] (maximum in log2, sum)
__device__ __forceinline__ size_t sp_part(const SharedPrefixArgs& a, int slot, int row, int head) { return ((size_t)slot * a.r.n_rows + row) * a.n_head + head; }

// the rows and keys that a CTA works on
struct SpWork {
    int split, r0, n_tok, own;   // its number among the CTAs that share the tile's keys; first row of the sequence, its rows, its own tokens (prefix pass: 0, all rows, the prefix's tokens)
    const int* table;
    int f0, n_f;                 // rows (token, head) of the tile, numbered within the sequence
    int G, lim_lo, lim_hi, q0, q1, n_tiles;      // keys that the tile's first and last rows see; this CTA's share of them; its tiles of keys
    bool own_pass;
    // keys that token i of the sequence sees
    __device__ int limit(int i) const { return own_pass ? max(0, own - n_tok + i + 1) : own; }
    __device__ SpWork() {}
    // what a sequence's work is known from: its first row, the row behind it, its own tokens
    struct Read { int b, e, held; };
    static __device__ __forceinline__ Read read(const SharedPrefixArgs& a, int z) {
        if (a.tab) return {z, z + 1, a.tab[a.slots.slot[z]].ints[1] + 1 - a.n_prefix};
        return {a.r.row_start[z], a.r.row_start[z + 1], a.r.lengths[z]};
    }
    static __device__ __forceinline__ const int* table_of(const SharedPrefixArgs& a, int z) {
        return a.tab ? a.tab[a.slots.slot[z]].block_table + a.n_prefix / a.r.block_tokens : a.r.pages + z * a.r.table_stride;
    }
    __device__ SpWork(const SharedPrefixArgs& a, const SpPlan& p, int mt, int x, int z) : SpWork(a, p, mt, x, z, z == p.prefix_z ? Read{0, 0, 0} : read(a, z)) {}
    __device__ SpWork(const SharedPrefixArgs& a, const SpPlan& p, int mt, int x, int z, const Read& r) {
        G = a.n_head / a.n_kv; own_pass = z != p.prefix_z;
        const int splits = own_pass ? p.splits : p.prefix_splits, tile = x / splits;
        split = x % splits;
        r0 = 0; n_tok = a.r.n_rows; own = a.n_prefix; table = a.prefix_pages;
        if (own_pass) {
            // (whatever the arrays hold: limits and row numbers that wrapped would be followed)
            r0 = min(max(r.b, 0), a.r.n_rows); n_tok = min(max(r.e, 0), a.r.n_rows) - r0; table = table_of(a, z);
            own = min(max(r.held, 0), a.r.max_pages * a.r.block_tokens);
        }
        f0 = tile * mt; n_f = min(mt, (own_pass ? min(n_tok, a.max_rows) : n_tok) * G - f0);
        lim_lo = limit(f0 / G); lim_hi = limit((f0 + max(n_f, 1) - 1) / G);
        const int chunk = ((lim_hi + splits - 1) / splits + SP_TT - 1) / SP_TT * SP_TT;
        q0 = min(lim_hi, split * chunk); q1 = min(lim_hi, q0 + chunk);
        n_tiles = (q1 - q0 + SP_TT - 1) / SP_TT;
    }
};

// The copying warp: tiles ti .. to - 1 of one KV head's keys and values; `it` counts the CTA's tiles. A lane has a box of keys; page ids of 32 boxes are read at once
// (`ids`: those of the first, read by sp_first_ids).
template <int HD, int STAGES>
__device__ __forceinline__ void sp_copy(const SharedPrefixArgs& a, const SpPlan& p, const SpWork& w, const CUtensorMap* map_k, const CUtensorMap* map_v, int kvh, int ti, int to, int& it,
                                        int& ids, uint8_t* tiles_at, uint64_t* full, uint64_t* empty, int lane) {
    constexpr int PARTS = HD / 64, PART = SP_TT * 128;
    const int boxes = SP_TT / p.box_rows, ahead = 32 / boxes, bt = a.r.block_tokens;
    for (; ti < to; ti++, it++) {
        const int st = it % STAGES, t0 = w.q0 + ti * SP_TT, n_box = min(boxes, (w.q1 - t0 + p.box_rows - 1) / p.box_rows), j = t0 + lane * p.box_rows;
        if (ti && ti % ahead == 0) ids = j < w.q1 ? w.table[j / bt] : 0;
        const int id = __shfl_sync(0xffffffffu, ids, ti % ahead * boxes + lane % boxes);
        const int row = (int)(((long)min(max(id, 0), (int)a.r.n_pages - 1) * a.n_kv + kvh) * bt + j % bt);
        if (it >= STAGES) mbar_wait_warp(&empty[st], (it / STAGES - 1) & 1, sp_err(a), 0xa0001u, (unsigned)it);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(n_box * p.box_rows * 128 * PARTS * 2));
        __syncwarp();
        if (lane < n_box)
            for (int c = 0; c < PARTS; c++) {
                uint8_t* dst = tiles_at + (st * 2 * PARTS + c) * PART + lane * p.box_rows * 128;
                tma_load_3d(dst, map_k, c * 64, row, 0, &full[st]);
                tma_load_3d(dst + PARTS * PART, map_v, c * 64, row, 0, &full[st]);
            }
        __syncwarp();
    }
}
// this lane's page of the first 32 boxes from key q0 on (whatever the table holds behind the last token: it is not followed)
__device__ __forceinline__ int sp_first_ids(const SharedPrefixArgs& a, const SpPlan& p, const int* table, int q0, int most, int lane) {
    const long j = q0 + (long)lane * p.box_rows;
    return j < most ? table[j / a.r.block_tokens] : 0;
}

// Take over the work of a CTA of this grid that has not started: asked for by one thread, the answer (16 bytes) arrives on a barrier. After a refusal nothing more may be
// asked.
__device__ __forceinline__ void sp_ask_work(void* answer, uint64_t* bar) {
    mbar_arrive_expect_tx(bar, 16);
    asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ bool sp_answered_work(const uint64_t* answer, int& x, int& y, int& z) {
    uint32_t got, i, j, k;
    asm volatile("{\n\t.reg .pred p;\n\t.reg .b128 r;\n\tmov.b128 r, {%4, %5};\n\tclusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\tselp.u32 %0, 1, 0, p;\n\t"
                 "mov.u32 %1, 0;\n\tmov.u32 %2, 0;\n\tmov.u32 %3, 0;\n\t@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, r;\n\t}"
                 : "=&r"(got), "=&r"(i), "=&r"(j), "=&r"(k) : "l"(answer[0]), "l"(answer[1]) : "memory");
    x = (int)i; y = (int)j; z = (int)k;
    return got != 0;
}

// The tile's queries into shared memory, rows padded by 16 bytes, by `n` threads
template <typename E, int HD>
__device__ __forceinline__ void sp_stage_q(const SharedPrefixArgs& a, const SpWork& w, int kvh, uint16_t* q_s, int thread, int n) {
    for (int e = thread; e < w.n_f * (HD / 8); e += n) {
        const int row = e / (HD / 8), c8 = e % (HD / 8), f = w.f0 + row, i = f / w.G;
        const size_t at = (size_t)(w.r0 + i) * a.q_row + (size_t)(kvh * w.G + f - i * w.G) * a.q_head + c8 * 8;
        uint4 v;
        if (a.q_f32) {
            const float* q = (const float*)a.q + at;
            v = make_uint4(SpType<E>::pack(q[0], q[1]), SpType<E>::pack(q[2], q[3]), SpType<E>::pack(q[4], q[5]), SpType<E>::pack(q[6], q[7]));
        } else {
            const uint16_t* q = (const uint16_t*)a.q + at;
            if (((uintptr_t)q & 15) == 0) v = *reinterpret_cast<const uint4*>(q);
            else v = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
        }
        *reinterpret_cast<uint4*>(q_s + row * (HD + 8) + c8 * 8) = v;
    }
}

// q fragments of rows f and f + 8 (numbered within the sequence; `in`: they belong to the tile)
template <typename E, int HD>
__device__ __forceinline__ void sp_load_q(const SharedPrefixArgs& a, const SpWork& w, int kvh, int row, int tq, uint32_t (&qa)[HD / 16][4]) {
    using T = SpType<E>;
    const bool words = !a.q_f32 && (((uintptr_t)a.q | (a.q_row * 2) | (a.q_head * 2)) & 3) == 0;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const bool in = row + 8 * h < w.n_f;
        const int f = w.f0 + row + 8 * h, i = in ? f / w.G : 0, head = kvh * w.G + (in ? f - i * w.G : 0);
        const size_t at = (size_t)(w.r0 + i) * a.q_row + (size_t)head * a.q_head + 2 * tq;
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++)
#pragma unroll
            for (int part = 0; part < 2; part++) {
                uint32_t v = 0;
                const size_t d = at + kk * 16 + part * 8;
                if (in) {
                    if (words) v = __ldcg(reinterpret_cast<const uint32_t*>((const uint16_t*)a.q + d));
                    else if (a.q_f32) { const float* q = (const float*)a.q + d; v = T::pack(__ldcg(q), __ldcg(q + 1)); }
                    else { const uint16_t* q = (const uint16_t*)a.q + d; v = (uint32_t)__ldcg(q) | (uint32_t)__ldcg(q + 1) << 16; }
                }
                qa[kk][2 * part + h] = v;
            }
    }
}

// two neighbouring columns of a row's output
template <typename E, int HD>
__device__ __forceinline__ void sp_store_out(const SharedPrefixArgs& a, int t, int head, int d, float x, float y) {
    const uint32_t v = SpType<E>::pack(x, y);
    if (a.out_h) {
        const int col = head * HD + d;
        *reinterpret_cast<uint32_t*>(a.out_h + ((size_t)(col >> 3) * a.out_T_pad + t) * 8 + (col & 7)) = v;
    } else {
        uint16_t* dst = (uint16_t*)a.out + (size_t)t * a.out_row + (size_t)head * a.out_head + d;
        if (((uintptr_t)dst & 3) == 0) *reinterpret_cast<uint32_t*>(dst) = v;
        else { dst[0] = (uint16_t)v; dst[1] = (uint16_t)(v >> 16); }
    }
}

// What a thread's columns of a row (numbers col, col + 1, col + 8, ...) come to: partial results, this CTA's share of a cluster's, or output
template <typename E, int HD, int N>
__device__ __forceinline__ void sp_finish(const SharedPrefixArgs& a, const SpPlan& p, const SpWork& w, int kvh, int row, int col, float m, float l, const float (&o)[N][4], int h, float* acc,
                                          float* row_m, float* row_l) {
    const int f = w.f0 + row, i = f / w.G, head = kvh * w.G + f - i * w.G;
    if (p.own_slot >= 0) {
        const size_t at = sp_part(a, w.own_pass ? p.own_slot + w.split : w.split, w.r0 + i, head);
#pragma unroll
        for (int nt = 0; nt < N; nt++) *reinterpret_cast<float2*>(a.work + at * HD + col + nt * 8) = make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
        if (col == 0) *reinterpret_cast<float2*>(a.work + p.ml_at + at * 2) = make_float2(m, l);
    } else if (p.splits > 1) {
#pragma unroll
        for (int nt = 0; nt < N; nt++) *reinterpret_cast<float2*>(acc + row * HD + col + nt * 8) = make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
        if (col == 0) { row_m[row] = m; row_l[row] = l; }
    } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;              // (0: no keys. A NaN stays one.)
#pragma unroll
        for (int nt = 0; nt < N; nt++) sp_store_out<E, HD>(a, w.r0 + i, head, col + nt * 8, o[nt][2 * h] * inv, o[nt][2 * h + 1] * inv);
    }
}

// the cluster's CTAs joined; every CTA writes its share of the tile
template <typename E, int HD>
__device__ __forceinline__ void sp_join_cluster(const SharedPrefixArgs& a, const SpPlan& p, const SpWork& w, int kvh, const float* acc, const float* row_m, const float* row_l) {
    cluster_sync();
    for (int e = sp_cluster_rank() * SP_THREADS + threadIdx.x; e < w.n_f * (HD / 4); e += p.splits * SP_THREADS) {
        const int row = e / (HD / 4), d = e % (HD / 4) * 4, f = w.f0 + row, i = f / w.G, head = kvh * w.G + f - i * w.G;
        float m = -INFINITY, l = 0.f;
        for (int c = 0; c < p.splits; c++) m = fmaxf(m, sp_cluster_load(cluster_address(smem_u32(row_m + row), c)));
        const float ref = m == -INFINITY ? 0.f : m;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < p.splits; c++) {
            const float c1 = sp_exp2(sp_cluster_load(cluster_address(smem_u32(row_m + row), c)) - ref);
            const float4 v = cluster_load4(cluster_address(smem_u32(acc + row * HD + d), c));
            l = fmaf(c1, sp_cluster_load(cluster_address(smem_u32(row_l + row), c)), l);
            sum.x = fmaf(c1, v.x, sum.x); sum.y = fmaf(c1, v.y, sum.y); sum.z = fmaf(c1, v.z, sum.z); sum.w = fmaf(c1, v.w, sum.w);
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        sp_store_out<E, HD>(a, w.r0 + i, head, d, sum.x * inv, sum.y * inv);
        sp_store_out<E, HD>(a, w.r0 + i, head, d + 2, sum.z * inv, sum.w * inv);
    }
    cluster_sync();                                              // (the others may still read this one's results)
}

// 16 bytes at (key, eight dims) of a tile's keys or values in 128-byte-swizzled rows
__device__ __forceinline__ uint8_t* sp_piece(uint8_t* base, int key, int c8) { return base + (c8 >> 3) * (SP_TT * 128) + key * 128 + (((c8 ^ key) & 7) << 4); }

// Does a value of 16 keys from `ks` on, dims 8 c0 .. 8 (c0 + n) - 1, have all exponent bits set (infinity or NaN)?
template <typename E>
__device__ __forceinline__ bool sp_any_bad(uint8_t* vb, int ks, int c0, int n, int lane) {
    uint32_t bad = 0;
    for (int e = lane; e < 16 * n; e += 32) {
        const uint4 v4 = *reinterpret_cast<const uint4*>(sp_piece(vb, ks + e / n, c0 + e % n));
        const uint32_t v[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
        for (int w = 0; w < 4; w++) bad |= (v[w] & SpType<E>::EXP) == SpType<E>::EXP || (v[w] >> 16 & SpType<E>::EXP) == SpType<E>::EXP;
    }
    return __any_sync(0xffffffffu, bad);
}

// A pass that is the operator's first kernel waits for what the kernels before it wrote (q, this step's keys); one behind the prefix pass starts beside it, since that
// has waited, and does not end before it, so that what is behind this pass is behind both. The next kernel may start early, but not to sit on SMs beside
// a pass that is to run beside the prefix's.
__device__ __forceinline__ void sp_begin(const SpPlan& p) { if (!p.behind) { griddep_wait(); griddep_launch(); } }
__device__ __forceinline__ void sp_end(const SpPlan& p) { if (p.behind) { griddep_launch(); griddep_wait(); } }

// Single tokens: a tile of up to 16 rows (the group's heads, a few tokens), the four computing warps share a tile of keys. Scores: a warp has 16 keys; maxima and
// probabilities go through shared memory; weighted sums: a warp has a quarter of the dims and all 64 keys, so that nothing has to be merged at the end.
// What a CTA waits for before its first keys are here takes as long as the keys of some 100 tokens (3 us): CTAs that run go on with the work of those that have not
// started (p.steal), and their copies run ahead into it. 256 sequences, 8 KV heads of 128, no prefix: of 256 tokens 50 us (5.4 TB/s), of 512 85 us (6.35), of 64
// 24 us (2.8: nearly all of it what a CTA waits for, 3.8 us a sequence).
// grid: (tile * splits + split, KV head, sequence), the prefix's CTAs among them (p.prefix_z) where its rows are as few
template <typename E, int HD>
__global__ void __launch_bounds__(SP_THREADS, 3) shared_prefix_step_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedPrefixArgs a,
                                                                           const SpPlan p) {
    constexpr int PARTS = HD / 64, PART = SP_TT * 128, STAGES = sp_stages(HD), NT = HD / 32;
    using T = SpType<E>;
    extern __shared__ uint8_t sp_raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES], next_full[2], next_empty[2], answered;
    __shared__ alignas(16) uint64_t answer[2];
    __shared__ SpWork next[2];                                   // the work after the first, n_f < 0: no more
    __shared__ int next_kvh[2];
    __shared__ float wmax[2][SP_WARPS][16], wsum[2][SP_WARPS][16], row_m[16], row_l[16];
    __shared__ alignas(16) uint16_t prob[2][16][SP_TT + 8];
    uint8_t* tiles_at = reinterpret_cast<uint8_t*>(((uintptr_t)sp_raw + 1023) & ~(uintptr_t)1023);      // [stage][keys, values][part]
    float* acc = reinterpret_cast<float*>(tiles_at);             // [16][HD], behind the last tile of a CTA that shares its keys
    uint16_t* q_s = reinterpret_cast<uint16_t*>(tiles_at + STAGES * 2 * PARTS * PART);      // [2][mrows][HD + 8], by turns
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, tq = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], SP_WARPS); }
        for (int i = 0; i < 2; i++) { mbar_init(&next_full[i], 1); mbar_init(&next_empty[i], SP_WARPS); }
        mbar_init(&answered, 1);
        fence_mbar_init();
    }
    sp_begin(p);
    int kvh = blockIdx.y;
    SpWork w(a, p, 16, blockIdx.x, blockIdx.z);
    if (w.n_f <= 0 && !p.steal) { sp_end(p); return; }           // (all CTAs of the cluster)
    if (w.n_f <= 0) w.n_tiles = 0;
    __syncthreads();

    if (warp == SP_WARPS) {
        SpWork v = w;
        int v_kvh = kvh, ids = sp_first_ids(a, p, v.table, v.q0, v.q1, lane);
        for (int it = 0, n = 0, asked = 0;; n++) {
            if (p.steal && lane == 0) sp_ask_work(answer, &answered);
            // ahead of the last tile: which work is next, and what it is known from is asked for, to be here when the tile is on its way
            const int first = max(v.n_tiles - 1, min(1, v.n_tiles));
            sp_copy<HD, STAGES>(a, p, v, &map_k, &map_v, v_kvh, 0, first, it, ids, tiles_at, full, empty, lane);
            int x = 0, y = 0, z = 0, next_ids = 0;
            SpWork::Read read = {0, 0, 0};
            auto take = [&]() {
                mbar_wait_warp(&answered, asked++ & 1, sp_err(a), 0xa0004u, (unsigned)n);
                if (!sp_answered_work(answer, x, y, z) || x >= (int)gridDim.x || y >= (int)gridDim.y || z >= (int)gridDim.z) return false;      // (a wait that ran out leaves anything)
                if (z == p.prefix_z) return true;
                read = SpWork::read(a, z);
                if (p.splits == 1) next_ids = sp_first_ids(a, p, SpWork::table_of(a, z), 0, a.r.max_pages * a.r.block_tokens, lane);
                return true;
            };
            bool more = p.steal && take();
            sp_copy<HD, STAGES>(a, p, v, &map_k, &map_v, v_kvh, first, v.n_tiles, it, ids, tiles_at, full, empty, lane);
            while (more) {                                       // (work without rows is passed over)
                v = SpWork(a, p, 16, x, z, read);
                if (v.n_f > 0) break;
                __syncwarp();
                if (lane == 0) { fence_proxy_async(); sp_ask_work(answer, &answered); }
                more = take();
            }
            v_kvh = y;
            ids = !more || (p.splits == 1 && v.own_pass) ? next_ids : sp_first_ids(a, p, v.table, v.q0, v.q1, lane);
            // (work n + 1's place, and the queries of work n - 1, are free again)
            if (n >= 1) mbar_wait_warp(&next_empty[n & 1], ((n - 1) >> 1) & 1, sp_err(a), 0xa0005u, (unsigned)n);
            if (more) sp_stage_q<E, HD>(a, v, v_kvh, q_s + ((n + 1) & 1) * p.mrows * (HD + 8), lane, 32);
            __syncwarp();
            if (lane == 0) {
                if (!more) v.n_f = -1;
                next[n & 1] = v; next_kvh[n & 1] = v_kvh;
                mbar_arrive(&next_full[n & 1]);
                fence_proxy_async();                             // (the answer has been read, the next may replace it)
            }
            if (!more) break;
        }
    } else {
        const int k0 = 16 * warp, c0 = warp * (HD / 32), col = warp * (HD / 4) + 2 * tq;
        for (int hh = 0, it = 0;; hh++) {
            if (hh > 0) {
                const int i = (hh - 1) & 1;
                mbar_wait(&next_full[i], ((hh - 1) >> 1) & 1, sp_err(a), 0xa0006u, (unsigned)hh);
                if (next[i].n_f < 0) break;
                w = next[i]; kvh = next_kvh[i];
            } else {
                sp_stage_q<E, HD>(a, w, kvh, q_s, tid, SP_WARPS * 32);
                named_bar_sync(1, SP_WARPS * 32);
            }
            if (w.n_f <= 0) {                                    // (only the first work may have no rows)
                __syncwarp();
                if (lane == 0) mbar_arrive(&next_empty[1]);
                continue;
            }
            int lim[2];
#pragma unroll
            for (int h = 0; h < 2; h++) lim[h] = g + 8 * h < w.n_f ? min(w.q1, w.limit((w.f0 + g + 8 * h) / w.G)) : w.q1;
            uint32_t qa[HD / 16][4];                             // (rows past the staged ones repeat the last: nothing of them is kept)
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) sp_ldmatrix_x4(qa[kk], q_s + (hh & 1) * p.mrows * (HD + 8) + min(lane & 15, p.mrows - 1) * (HD + 8) + kk * 16 + (lane >> 4) * 8);
            __syncwarp();
            if (lane == 0) mbar_arrive(&next_empty[(hh + 1) & 1]);
            float o[NT][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};      // (l: this thread's columns of scores)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
            for (int ti = 0; ti < w.n_tiles; ti++, it++) {
                const int st = it % STAGES, buf = it & 1, t0 = w.q0 + ti * SP_TT, valid = min(SP_TT, w.q1 - t0);
                uint8_t *kb = tiles_at + st * 2 * PARTS * PART, *vb = kb + PARTS * PART;
                mbar_wait(&full[st], (it / STAGES) & 1, sp_err(a), 0xa0002u, (unsigned)it);
                __syncwarp();
                // ---- scores of this warp's keys, scaled, masked, and their maxima in rows g and g + 8; this thread's columns are 2 tq, 2 tq + 1 of every eight keys
                float sc[2][4], sd[2][4], mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int nt = 0; nt < 2; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sc[nt][e] = sd[nt][e] = 0.f;
                if (k0 < valid) {                                // (two sums, added up: shorter chains of dependent products)
#pragma unroll
                    for (int nt = 0; nt < 2; nt++)
#pragma unroll
                        for (int kk = 0; kk < HD / 16; kk += 2) {
                            uint32_t b4[4];                      // dims kk * 16 .. + 31 of eight keys
                            sp_ldmatrix_x4(b4, sp_piece(kb, k0 + nt * 8 + (lane & 7), kk * 2 + (lane >> 3)));
                            T::mma(sc[nt], qa[kk], b4[0], b4[1]);
                            T::mma(sd[nt], qa[kk + 1], b4[2], b4[3]);
                        }
                }
#pragma unroll
                for (int nt = 0; nt < 2; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = t0 + k0 + nt * 8 + 2 * tq + (e & 1);
                        sc[nt][e] = key < lim[e >> 1] ? (sc[nt][e] + sd[nt][e]) * a.scale_log2 : -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
                    }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                    if (tq == 0) wmax[buf][warp][g + 8 * h] = mx[h];
                }
                named_bar_sync(1, SP_WARPS * 32);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float m = m_run[h];
#pragma unroll
                    for (int i = 0; i < SP_WARPS; i++) m = fmaxf(m, wmax[buf][i][g + 8 * h]);
                    const float ref = m == -INFINITY ? 0.f : m, fall = sp_exp2(m_run[h] - ref);      // (nothing seen yet: every weight is 0)
                    m_run[h] = m;
                    l_run[h] *= fall;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) { o[nt][2 * h] *= fall; o[nt][2 * h + 1] *= fall; }
#pragma unroll
                    for (int nt = 0; nt < 2; nt++) {
                        const float e0 = sp_exp2(sc[nt][2 * h] - ref), e1 = sp_exp2(sc[nt][2 * h + 1] - ref);
                        l_run[h] += e0 + e1;
                        *reinterpret_cast<uint32_t*>(&prob[buf][g + 8 * h][k0 + nt * 8 + 2 * tq]) = T::pack(e0, e1);
                    }
                }
                if (valid & 15) {
                    // values past the last key up to the next 16: 0 * garbage must stay 0 in the weighted sum (every warp clears its dims)
                    const int n_bad = 16 - (valid & 15);
                    for (int e = lane; e < n_bad * NT; e += 32) *reinterpret_cast<uint4*>(sp_piece(vb, valid + e / NT, c0 + e % NT)) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();                         // (later copies may replace them)
                    __syncwarp();
                }
                named_bar_sync(1, SP_WARPS * 32);
#pragma unroll
                for (int s = 0; s < SP_TT / 16; s++) {
                    if (16 * s >= valid) break;
                    // keys that only later rows of the tile see: a value there that is no number must not reach the earlier rows through a weight of 0
                    if (w.lim_lo < w.lim_hi && t0 + 16 * s + 16 > w.lim_lo && sp_any_bad<E>(vb, 16 * s, c0, NT, lane)) {
#pragma unroll 1
                        for (int k = 16 * s; k < 16 * s + 16; k++)
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint32_t v = *reinterpret_cast<const uint32_t*>(sp_piece(vb, k, c0 + nt) + 4 * tq);
#pragma unroll
                                for (int e = 0; e < 4; e++) {
                                    const float weight = T::value(prob[buf][g + 8 * (e >> 1)][k]);
                                    if (weight != 0.f) o[nt][e] = fmaf(weight, T::value((uint16_t)(e & 1 ? v >> 16 : v)), o[nt][e]);
                                }
                            }
                        continue;
                    }
                    uint32_t pa[4];
                    sp_ldmatrix_x4(pa, &prob[buf][lane & 15][16 * s + (lane >> 4) * 8]);
#pragma unroll
                    for (int nt = 0; nt < NT; nt += 2) {
                        uint32_t b4[4];                          // 16 keys x 16 dims, transposed on load
                        sp_ldmatrix_x4_trans(b4, sp_piece(vb, 16 * s + (lane & 15), c0 + nt + (lane >> 4)));
                        T::mma(o[nt], pa, b4[0], b4[1]);
                        T::mma(o[nt + 1], pa, b4[2], b4[3]);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[st]);
            }
            // ---- sums over the warps' keys
#pragma unroll
            for (int h = 0; h < 2; h++) {
                l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
                l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
                if (tq == 0) wsum[hh & 1][warp][g + 8 * h] = l_run[h];
            }
            named_bar_sync(1, SP_WARPS * 32);                    // (and everyone is done with the tiles of this head)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int row = g + 8 * h;
                if (row >= w.n_f) continue;
                const float l = (wsum[hh & 1][0][row] + wsum[hh & 1][1][row]) + (wsum[hh & 1][2][row] + wsum[hh & 1][3][row]);
                sp_finish<E, HD, NT>(a, p, w, kvh, row, col, m_run[h], l, o, h, acc, row_m, row_l);
            }
        }
    }
    if (p.own_slot < 0 && p.splits > 1) sp_join_cluster<E, HD>(a, p, w, kvh, acc, row_m, row_l);
    sp_end(p);
}

// Several tokens of a sequence, or the prefix pass of up to 32 rows: a tile of 64 rows, a warp has 16 of them and all keys. Own tokens of 40 sequences of 3 to 33
// rows, 32 heads over 4 of 64: 13.5 us by themselves, behind a prefix most of them when its pass has ended.
// grid: (tile * splits + split, KV head, sequence, or prefix)
template <typename E, int HD>
__global__ void __launch_bounds__(SP_THREADS, 2) shared_prefix_rows_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const SharedPrefixArgs a,
                                                                           const SpPlan p) {
    constexpr int PARTS = HD / 64, PART = SP_TT * 128, STAGES = sp_stages(HD), MT = 64, KS = SP_TT / 16, NT = HD / 8;
    using T = SpType<E>;
    extern __shared__ uint8_t sp_raw[];
    __shared__ uint64_t full[STAGES], empty[STAGES];
    __shared__ float row_m[MT], row_l[MT];
    uint8_t* tiles_at = reinterpret_cast<uint8_t*>(((uintptr_t)sp_raw + 1023) & ~(uintptr_t)1023);      // [stage][keys, values][part]
    float* acc = reinterpret_cast<float*>(tiles_at);             // [MT][HD], behind the last tile of a CTA that shares its keys
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31, g = lane >> 2, tq = lane & 3;
    if (tid == 0) {
        for (int i = 0; i < STAGES; i++) { mbar_init(&full[i], 1); mbar_init(&empty[i], SP_WARPS); }
        fence_mbar_init();
    }
    sp_begin(p);
    const int kvh = blockIdx.y;
    const SpWork w(a, p, MT, blockIdx.x, blockIdx.z);
    if (w.n_f <= 0) { sp_end(p); return; }
    __syncthreads();

    if (warp == SP_WARPS) {
        int it = 0, ids = sp_first_ids(a, p, w.table, w.q0, w.q1, lane);
        sp_copy<HD, STAGES>(a, p, w, &map_k, &map_v, kvh, 0, w.n_tiles, it, ids, tiles_at, full, empty, lane);
    } else {
        const int row0 = 16 * warp + g;
        const bool idle = 16 * warp >= w.n_f;                    // this warp has no rows
        uint32_t qa[HD / 16][4];
        sp_load_q<E, HD>(a, w, kvh, row0, tq, qa);
        float o[NT][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};          // (l: this thread's columns of scores)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) o[nt][0] = o[nt][1] = o[nt][2] = o[nt][3] = 0.f;
        int lim[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const bool in = row0 + 8 * h < w.n_f;
            lim[h] = in ? min(w.q1, w.limit((w.f0 + row0 + 8 * h) / w.G)) : w.q1;
        }
        for (int ti = 0; ti < w.n_tiles; ti++) {
            const int st = ti % STAGES, t0 = w.q0 + ti * SP_TT, valid = min(SP_TT, w.q1 - t0);
            uint8_t *kb = tiles_at + st * 2 * PARTS * PART, *vb = kb + PARTS * PART;
            mbar_wait(&full[st], (ti / STAGES) & 1, sp_err(a), 0xa0003u, (unsigned)ti);
            __syncwarp();
            if (!idle) {
                if (valid & 15) {                                // (every warp clears what it reads)
                    const int n_bad = 16 - (valid & 15);
                    for (int e = lane; e < n_bad * (HD / 8); e += 32) *reinterpret_cast<uint4*>(sp_piece(vb, valid + e / (HD / 8), e % (HD / 8))) = make_uint4(0, 0, 0, 0);
                    __syncwarp();
                }
                float sc[2 * KS][4], mx[2] = {m_run[0], m_run[1]}, ref[2];
#pragma unroll
                for (int nt = 0; nt < 2 * KS; nt++) {
                    sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk += 2) {
                        uint32_t b4[4];
                        sp_ldmatrix_x4(b4, sp_piece(kb, nt * 8 + (lane & 7), kk * 2 + (lane >> 3)));
                        T::mma(sc[nt], qa[kk], b4[0], b4[1]);
                        T::mma(sc[nt], qa[kk + 1], b4[2], b4[3]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < 2 * KS; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int key = t0 + nt * 8 + 2 * tq + (e & 1);
                        sc[nt][e] = key < lim[e >> 1] ? sc[nt][e] * a.scale_log2 : -INFINITY;
                        mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
                    }
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
                    mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
                    ref[h] = mx[h] == -INFINITY ? 0.f : mx[h];
                    const float fall = sp_exp2(m_run[h] - ref[h]);
                    m_run[h] = mx[h];
                    l_run[h] *= fall;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) { o[nt][2 * h] *= fall; o[nt][2 * h + 1] *= fall; }
                }
#pragma unroll
                for (int nt = 0; nt < 2 * KS; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) { sc[nt][e] = sp_exp2(sc[nt][e] - ref[e >> 1]); l_run[e >> 1] += sc[nt][e]; }
#pragma unroll
                for (int s = 0; s < KS; s++) {
                    if (16 * s >= valid) break;
                    if (w.lim_lo < w.lim_hi && t0 + 16 * s + 16 > w.lim_lo && sp_any_bad<E>(vb, 16 * s, 0, HD / 8, lane)) {
#pragma unroll 1
                        for (int k = 0; k < 16; k++) {
                            const int from = (lane & ~3) | (k & 7) >> 1;
                            float weight[2];
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                float mine = 0.f;
#pragma unroll
                                for (int e = 0; e < 4; e++) if (e == (k >> 3) * 2 + (k & 1)) mine = sc[2 * s + (e >> 1)][2 * h + (e & 1)];
                                weight[h] = __shfl_sync(0xffffffffu, mine, from);
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                const uint32_t v = *reinterpret_cast<const uint32_t*>(sp_piece(vb, 16 * s + k, nt) + 4 * tq);
#pragma unroll
                                for (int e = 0; e < 4; e++)
                                    if (weight[e >> 1] != 0.f) o[nt][e] = fmaf(weight[e >> 1], T::value((uint16_t)(e & 1 ? v >> 16 : v)), o[nt][e]);
                            }
                        }
                        continue;
                    }
                    const uint32_t pa[4] = {T::pack(sc[2 * s][0], sc[2 * s][1]), T::pack(sc[2 * s][2], sc[2 * s][3]),
                                            T::pack(sc[2 * s + 1][0], sc[2 * s + 1][1]), T::pack(sc[2 * s + 1][2], sc[2 * s + 1][3])};
#pragma unroll
                    for (int nt = 0; nt < NT; nt += 2) {
                        uint32_t b4[4];
                        sp_ldmatrix_x4_trans(b4, sp_piece(vb, 16 * s + (lane & 15), nt + (lane >> 4)));
                        T::mma(o[nt], pa, b4[0], b4[1]);
                        T::mma(o[nt + 1], pa, b4[2], b4[3]);
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[st]);
        }
        named_bar_sync(1, SP_WARPS * 32);                        // everyone is done with the tiles
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
            l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
            if (row0 + 8 * h < w.n_f) sp_finish<E, HD, NT>(a, p, w, kvh, row0 + 8 * h, 2 * tq, m_run[h], l_run[h], o, h, acc, row_m, row_l);
        }
    }
    if (p.own_slot < 0 && p.splits > 1) sp_join_cluster<E, HD>(a, p, w, kvh, acc, row_m, row_l);
    sp_end(p);
}

// The partial results of the prefix and of the own tokens, joined: a thread four dims of a row and head, all of whose reads
// are under way at once (up to eight results; four CTAs' worth of one row in one CTA, three results at a time, took 12 us). 256 rows of 32 heads of 128 with
// three results each: 8 us, 64 rows with ten: 7.
constexpr int SP_JOIN = 128;
template <typename E, int HD>
__global__ void __launch_bounds__(SP_JOIN) shared_prefix_join_kernel(const SharedPrefixArgs a, const SpPlan p) {
    __shared__ int live;
    constexpr int B = 8;
    const int per_row = (a.n_head * (HD / 4) + SP_JOIN - 1) / SP_JOIN, t = blockIdx.x / per_row, e = blockIdx.x % per_row * SP_JOIN + threadIdx.x;
    const int G = a.n_head / a.n_kv, head = e / (HD / 4), d = e % (HD / 4) * 4, kvh = head / G;
    const bool in = head < a.n_head;
    const size_t at = sp_part(a, 0, t, head), step = (size_t)a.r.n_rows * a.n_head;
    const float* ml = a.work + p.ml_at + at * 2;
    const float* from = a.work + at * HD + d;
    // rows that no sequence has, or that are past a sequence's max_rows, have no result
    if (!a.tab && threadIdx.x < 32) {
        const int s = seq_of_row(a.r.row_start, a.r.n_seqs, t, threadIdx.x);
        if (threadIdx.x == 0) live = s < a.r.n_seqs && t >= a.r.row_start[0] && t - max(0, a.r.row_start[s]) < a.max_rows;
    }
    griddep_wait();
    griddep_launch();
    PrefixCut cut = p.cut;
    if (p.share.adapt) {
        const int2 took = *reinterpret_cast<const int2*>(a.work + p.share.cut_at);
        cut.run = took.x; cut.per_unit = took.y;
    }
    const int slots = !in ? 0 : p.slots >= 0 ? p.slots : cut.slots(kvh * cut.pairs + (t * G + head - kvh * G) / 256), all = slots + p.splits;
    float m = -INFINITY, l = 0.f;
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j0 = 0; j0 < all; j0 += B) {                        // (behind the prefix's: the own tokens')
        float2 one[B];
        float4 v[B];
#pragma unroll
        for (int j = 0; j < B; j++) {
            one[j] = make_float2(-INFINITY, 0.f); v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j0 + j >= all || !in) continue;
            const size_t off = (j0 + j < slots ? j0 + j : p.own_slot + j0 + j - slots) * step;
            one[j] = __ldcg(reinterpret_cast<const float2*>(ml + off * 2));
            v[j] = __ldcg(reinterpret_cast<const float4*>(from + off * HD));
        }
        float m2 = m;
#pragma unroll
        for (int j = 0; j < B; j++) m2 = fmaxf(m2, one[j].x);
        const float ref = m2 == -INFINITY ? 0.f : m2, fall = sp_exp2(m - ref);
        m = m2; l *= fall; sum.x *= fall; sum.y *= fall; sum.z *= fall; sum.w *= fall;
#pragma unroll
        for (int j = 0; j < B; j++) {
            const float c = sp_exp2(one[j].x - ref);
            l = fmaf(c, one[j].y, l);
            sum.x = fmaf(c, v[j].x, sum.x); sum.y = fmaf(c, v[j].y, sum.y); sum.z = fmaf(c, v[j].z, sum.z); sum.w = fmaf(c, v[j].w, sum.w);
        }
    }
    __syncthreads();
    if (!in || (!a.tab && !live)) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;                  // (0: no keys. A NaN stays one.)
    sp_store_out<E, HD>(a, t, head, d, sum.x * inv, sum.y * inv);
    sp_store_out<E, HD>(a, t, head, d + 2, sum.z * inv, sum.w * inv);
}

// ---------------------------------------------------------------- host side
namespace {
constexpr int SP_SMS = PREFIX_SMS;
constexpr size_t sp_smem(int hd, int mrows) { return (size_t)sp_stages(hd) * 2 * SP_TT * hd * 2 + 2 * mrows * (hd + 8) * 2 + 1024; }

template <typename E, int HD>
cudaError_t sp_rows(const SharedPrefixArgs& a, SpPlan p, bool single, dim3 grid, cudaStream_t s, bool pdl) {
    if (!(single ? allow_smem<shared_prefix_step_kernel<E, HD>>((int)sp_smem(HD, 16)) : allow_smem<shared_prefix_rows_kernel<E, HD>>((int)sp_smem(HD, 0)))) return cudaErrorInvalidValue;
    p.box_rows = SP_TT;
    while (a.r.block_tokens % p.box_rows) p.box_rows /= 2;
    const long rows = a.r.n_pages * a.n_kv * a.r.block_tokens;
    CUtensorMap mk, mv;                                          // (copies move 16-bit entries whatever their format)
    if (!bf16_rows_map(&mk, a.k_pool, HD, rows, HD, 1, 0, p.box_rows) || !bf16_rows_map(&mv, a.v_pool, HD, rows, HD, 1, 0, p.box_rows)) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(SP_THREADS); cfg.dynamicSmemBytes = sp_smem(HD, single ? p.mrows : 0); cfg.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (p.own_slot < 0 && p.splits > 1) {
        at[n].id = cudaLaunchAttributeClusterDimension;
        at[n].val.clusterDim.x = p.splits; at[n].val.clusterDim.y = 1; at[n].val.clusterDim.z = 1;
        n++;
    }
    if (pdl) {
        at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    cfg.attrs = at; cfg.numAttrs = n;
    return single ? cudaLaunchKernelEx(&cfg, shared_prefix_step_kernel<E, HD>, mk, mv, a, p) : cudaLaunchKernelEx(&cfg, shared_prefix_rows_kernel<E, HD>, mk, mv, a, p);
}
template <typename E, int HD>
cudaError_t sp_join(const SharedPrefixArgs& a, const SpPlan& p, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.n_head * (HD / 4) + SP_JOIN - 1) / SP_JOIN * a.r.n_rows)); cfg.blockDim = dim3(SP_JOIN); cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, shared_prefix_join_kernel<E, HD>, a, p);
}
// at most 16 rows a KV head of a sequence (prefix pass: of the batch): the single-token form
cudaError_t sp_rows_of(const SharedPrefixArgs& a, const SpPlan& p, bool single, dim3 grid, cudaStream_t s, bool pdl) {
    const bool h = a.type == ELEM_F16;
    if (a.head_dim == 64) return h ? sp_rows<__half, 64>(a, p, single, grid, s, pdl) : sp_rows<__nv_bfloat16, 64>(a, p, single, grid, s, pdl);
    return h ? sp_rows<__half, 128>(a, p, single, grid, s, pdl) : sp_rows<__nv_bfloat16, 128>(a, p, single, grid, s, pdl);
}
// CTAs that share a tile's keys: about two CTAs an SM in all, no fewer keys than a tile each, at most a portable cluster
int sp_splits(long tiles, long keys, int most) {
    int n = 1;
    while (2 * n <= most && tiles * n * 2 <= 2 * SP_SMS && keys / (2 * n) >= SP_TT) n *= 2;
    return n;
}
// Up to so many rows a KV head the prefix is read by the kernels above, more by the pass on tensor memory. 32 heads over 8 KV heads of 128, prefixes of 512, 2000
// and 8000, own tokens 20 to 500, these kernels / tensor memory: 20 rows 10.4 / 14.3, 17.7 / 18.6, 24.9 / 22.9 us; 32 rows 11.0 / 15.1, 18.0 / 19.5, 26.6 / 25.8;
// 64 rows 14.9 / 15.0, 22.0 / 18.6, 34.7 / 27.1. (The rule goes by rows alone, for a workspace that does not depend on the prefix: up to 2 us are lost behind 8000.)
constexpr int SP_PREFIX_ROWS = 32;
constexpr int SP_PREFIX_SPLITS = 32, SP_OWN_SPLITS = 8;
}  // namespace

// Runs of equal length over all units laid end to end, or over every unit by itself where that makes them no more than three blocks longer: a run that goes on
// into another unit loads queries, starts and ends its pipeline and writes its results twice, which takes as long as three blocks (6 us). For `sms` CTAs at most.
// (Units fit an int: every entry refuses n_rows * n_head of more than 31 bits.)
PrefixCut prefix_cut(long n_rows, int n_head, int n_kv, int n_prefix, int sms) {
    PrefixCut c = {};
    c.pairs = (int)((n_rows * (n_head / n_kv) + 255) / 256);
    c.units = n_kv * c.pairs;
    c.blocks = (n_prefix + 127) / 128;
    const unsigned total = (unsigned)c.units * (unsigned)c.blocks, s = (unsigned)sms;      // (31 bits: see PrefixCut)
    c.run = (int)((total + s - 1) / s);
    const int parts = c.units <= sms ? (int)(s / (unsigned)c.units) : 1, each = (c.blocks + parts - 1) / parts;
    c.per_unit = c.run && c.units <= sms && each <= c.run + 3;
    if (c.per_unit) c.run = each;
    c.ctas = c.run == 0 ? 0 : c.per_unit ? c.units * ((c.blocks + each - 1) / each) : (int)((total + (unsigned)c.run - 1) / (unsigned)c.run);
    return c;
}

// The cuts that bring the prefix pass and the pass over single own tokens to an end soonest. A run of blocks takes FIXED us and BLOCK a block (1.8
// by itself, 2.2 beside the other pass), NEXT more for every unit that it goes on into; a CTA of the other pass (three an SM) takes ITEM us for a sequence and KV head and BYTES a MB, all of them together no
// less than the memory gives. They have the SMs that the prefix pass leaves, and all from its end on.
// Measured (32 heads over 8 KV heads of 128; with all SMs for the prefix, as given here): 256 samples of 1 to 512 own tokens behind 8192 103 -> 87 us, on 64 SMs
// (on 96: 96, on 48: 119); 64 of 16 to 300 behind 8000 42 -> 34, on 88; behind 2000 35 -> 26, on 48; 64 of 16 to 1000 behind 8000 66 -> 50, on 56; 32 of 20 to
// 500 behind 1000 22.5 -> 19.5, on 32.
static void sp_share(const SharedPrefixArgs& a, PrefixShare& share) {
    constexpr float FIXED = 8.f, BLOCK = 2.2f, NEXT = 6.f, ITEM = 4.5f, BYTES = 35.f, MEMORY = 5.f;      // MEMORY: MB a us
    struct Choice { PrefixCut cut; float beside, ends; } c[16];
    int n = 0;
    for (int sms = PREFIX_SMS; sms > PREFIX_SMS - 8 * 16; sms -= 8) {
        const PrefixCut t = prefix_cut(a.r.n_rows, a.n_head, a.n_kv, a.n_prefix, sms);
        if (n && c[n - 1].cut.ctas == t.ctas && c[n - 1].cut.run == t.run) continue;
        c[n].cut = t;
        c[n].beside = 3.f * (PREFIX_SMS - t.ctas);
        c[n++].ends = FIXED + BLOCK * t.run + (t.per_unit ? 0.f : NEXT * (float)((t.run + t.blocks - 2) / t.blocks));
    }
    const float items = (float)a.r.n_seqs * a.n_kv;
    const long most = (long)a.r.max_pages * a.r.block_tokens;
    for (int l = 0; l < SHARE_LEVELS; l++) {
        const float mb = fmaxf(32.f, 0.72f * (16 << l)) * a.head_dim * 4e-6f, alone = ITEM + BYTES * mb;
        float least = INFINITY;
        int best = 0;
        if (l > 0 && most <= 16 << (l - 1)) {                    // (no sequence can hold as much)
            share.run[l] = share.run[l - 1]; share.ctas[l] = share.ctas[l - 1]; share.per_unit[l] = share.per_unit[l - 1];
            continue;
        }
        for (int i = 0; i < n; i++) {                            // (of equals the one with most SMs)
            const float item = fmaxf(alone, c[i].beside * (mb / MEMORY)), begun = c[i].beside * ceilf(c[i].ends / item);
            const float total = begun < items ? c[i].ends + fmaxf(ceilf((items - begun) * (1.f / (3.f * PREFIX_SMS))) * alone, (items - begun) * (mb / MEMORY))
                                              : fmaxf(c[i].ends, ceilf(items / c[i].beside) * item);
            if (total < least) { least = total; best = i; }
        }
        share.run[l] = c[best].cut.run; share.ctas[l] = (short)c[best].cut.ctas; share.per_unit[l] = (short)c[best].cut.per_unit;
    }
    share.adapt = 1;
}

// most partial results that a row's prefix can have: a unit of b blocks in runs of ceil(u b / 148) lies in at most ceil(148 / u) + 1 of them
static long sp_prefix_slots(long n_rows, int n_head, int n_kv) {
    if (n_rows * (n_head / n_kv) <= SP_PREFIX_ROWS) return SP_PREFIX_SPLITS;
    const PrefixCut c = prefix_cut(n_rows, n_head, n_kv, 1, SP_SMS);
    return (SP_SMS + c.units - 1) / c.units + 1;
}
// and its own tokens: the splits of the fewest CTAs that so many rows can be
static long sp_own_slots(long n_rows, int n_head, int n_kv) {
    return sp_splits((n_rows * (n_head / n_kv) + 63) / 64 * n_kv, LONG_MAX, SP_OWN_SPLITS);
}
size_t shared_prefix_work_floats(long n_rows, int n_head, int n_kv, int head_dim) {
    return (size_t)(sp_prefix_slots(n_rows, n_head, n_kv) + sp_own_slots(n_rows, n_head, n_kv)) * n_rows * n_head * (head_dim + 2) + 4;      // (and the cut that the prefix pass took)
}

// the prefix and the own tokens in one launch (grid.z: the sequences and the prefix)
static bool sp_one_launch(const SharedPrefixArgs& a) {
    const int G = a.n_head / a.n_kv;
    return (long)a.r.n_rows * G <= 16 && a.max_rows * G <= 16 && a.r.n_seqs < 65535;
}
int shared_prefix_launches(const SharedPrefixArgs& a) { return a.n_prefix == 0 ? 1 : sp_one_launch(a) ? 2 : 3; }

cudaError_t shared_prefix_error(unsigned int* code) {
    // (all streams: a copy on the default one does not wait for those that were made not to wait for it)
    cudaError_t e = cudaDeviceSynchronize();
    unsigned int more = 0;
    if (e == cudaSuccess) e = take_error_word(sp_error, code);
    if (e == cudaSuccess) e = shared_prefix_tc_error(&more);
    if (e == cudaSuccess && *code == 0) *code = more;
    return e;
}
__global__ void sp_give_up_kernel(unsigned int code) { mbar_give_up(0, sp_error, code, 0); }
cudaError_t shared_prefix_give_up(unsigned int code, bool tensor_memory, cudaStream_t s) {
    if (tensor_memory) return shared_prefix_tc_give_up(code, s);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = cfg.blockDim = dim3(1); cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, sp_give_up_kernel, code);
}

cudaError_t shared_prefix_launch(const SharedPrefixArgs& a, cudaStream_t s) {
    const int R = a.r.n_rows, G = a.n_head / a.n_kv, S = a.r.n_seqs;
    if (R == 0 || S == 0) return cudaSuccess;
    if ((long)prefix_cut(R, a.n_head, a.n_kv, 1, SP_SMS).units * ((a.n_prefix + 127) / 128) > INT_MAX / 2) return cudaErrorInvalidValue;
    cudaError_t e;
    const bool few = (long)R * G <= SP_PREFIX_ROWS, single = a.max_rows * G <= 16, h = a.type == ELEM_F16;
    const int mt = single ? 16 : 64, tiles = (a.max_rows * G + mt - 1) / mt;
    SpPlan own = {};
    own.prefix_z = own.own_slot = -1;
    own.splits = sp_splits((long)tiles * a.n_kv * S, (long)a.r.max_pages * a.r.block_tokens, SP_OWN_SPLITS);
    own.mrows = single ? a.max_rows * G : 0;
    if (a.n_prefix == 0) {
        own.steal = single && own.splits == 1;
        return sp_rows_of(a, own, single, dim3(tiles * own.splits, a.n_kv, S), s, g_chain_pdl);
    }
    const long slots = sp_prefix_slots(R, a.n_head, a.n_kv);
    own.own_slot = (int)slots;
    own.ml_at = (size_t)(slots + sp_own_slots(R, a.n_head, a.n_kv)) * R * a.n_head * a.head_dim;
    own.splits = std::min(own.splits, (int)sp_own_slots(R, a.n_head, a.n_kv));      // (fewer sequences than their rows need: max_rows was too small)
    own.steal = single;
    if (few) own.slots = own.prefix_splits = sp_splits((long)a.n_kv, a.n_prefix, SP_PREFIX_SPLITS);
    if (sp_one_launch(a)) {
        own.prefix_z = S;
        own.mrows = R * G;
        own.steal = 0;
        e = sp_rows_of(a, own, true, dim3(std::max(own.prefix_splits, own.splits), a.n_kv, S + 1), s, g_chain_pdl);
    } else {
        if (few) {
            SpPlan p = own;
            p.prefix_z = 0;
            p.steal = 0;
            e = sp_rows_of(a, p, false, dim3(p.prefix_splits, a.n_kv, 1), s, g_chain_pdl);
        } else {
            own.cut = prefix_cut(R, a.n_head, a.n_kv, a.n_prefix, SP_SMS);
            own.slots = -1;
            if (single) sp_share(a, own.share);
            own.share.cut_at = shared_prefix_work_floats(R, a.n_head, a.n_kv, a.head_dim) - 4;
            e = shared_prefix_tc_launch(a, own.cut, own.ml_at, own.share, s);
        }
        if (e != cudaSuccess) return e;
        own.behind = 1;
        e = sp_rows_of(a, own, single, dim3(tiles * own.splits, a.n_kv, S), s, true);
    }
    if (e != cudaSuccess) return e;
    if (a.head_dim == 64) return h ? sp_join<__half, 64>(a, own, s) : sp_join<__nv_bfloat16, 64>(a, own, s);
    return h ? sp_join<__half, 128>(a, own, s) : sp_join<__nv_bfloat16, 128>(a, own, s);
}

}  // namespace b2

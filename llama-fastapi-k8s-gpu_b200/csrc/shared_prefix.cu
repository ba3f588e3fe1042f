// Attention of a batch over a paged cache whose first n_prefix tokens are the same pages for every sequence.
//   keys of row i of a sequence with n rows and c own tokens: the prefix, and own tokens 0 .. c - n + i;   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),
//   s_j = scale log2(e) q.k_j. No key: 0.
// The prefix is read once for all rows: its pass leaves (m, sum, weighted sum) of every row in 32 bits, the pass over the sequences' own tokens joins them.
//
// The prefix pass is shared_prefix_tc.cu (tensor memory) or, where the rows of a KV head fill no more than one tile of 64, the kernel here over the same
// rows; the own pass is the kernel here. Here: mma.sync m16n8k16, tiles of 64 keys by cp.async in rows padded by 16 bytes, three buffers. A row of the
// tile is (token, head of the KV head's group). MT 16: a CTA's four warps take 16 keys of a tile each and are merged at the end, which is the form for single
// tokens, bound by the cache's bytes; MT 64: a warp has 16 rows and all keys. The keys of a tile of rows are split over a cluster of up to eight CTAs, which
// join through each other's shared memory.
// Probabilities are rounded to the cache's type for the weighted sum (the other operand is the cache as it is); scores, maxima, sums, joins stay 32-bit.
#include "device_ops.h"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

namespace b2 {

namespace {
constexpr int SP_THREADS = 128;
constexpr int SP_TT = 64;            // keys of a tile
constexpr int SP_STAGES = 3;

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
__device__ __forceinline__ void sp_cp16(void* dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void sp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void sp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint32_t sp_cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ float sp_cluster_load(uint32_t address) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(address) : "memory");
    return v;
}
}  // namespace

enum SpRole { SP_PREFIX = 0, SP_OWN = 1, SP_JOINED = 2 };      // the prefix for all rows; own tokens of a sequence; both, one after the other
struct SpPlan {
    int role, splits;            // CTAs that share the keys of a tile (a cluster, except for SP_PREFIX)
    int fixed_slots;             // SP_OWN: partial results of the prefix per row (0: none; < 0: as `cut` says)
    PrefixCut cut;
};

// partial results of the prefix: [slot][row][head][head_dim] weighted sums, then [slot][row][head][2] (maximum in log2, sum)
__device__ __forceinline__ size_t sp_part(const SharedPrefixArgs& a, int slot, int row, int head) { return ((size_t)slot * a.r.n_rows + row) * a.n_head + head; }

// grid: (tile * splits + split, KV head, sequence)
template <typename E, int HD, int MT>
__global__ void __launch_bounds__(SP_THREADS) shared_prefix_rows_kernel(const SharedPrefixArgs a, const SpPlan p, const size_t ml_at) {
    constexpr int LD = HD + 8;                                   // padded row (entries)
    constexpr int KS = MT == 16 ? 1 : 4;                         // 16-key steps of a tile that a warp takes
    using T = SpType<E>;
    extern __shared__ __align__(16) uint8_t sp_smem[];
    uint16_t* ks = reinterpret_cast<uint16_t*>(sp_smem);         // [SP_STAGES][SP_TT][LD]
    uint16_t* vs = ks + SP_STAGES * SP_TT * LD;
    __shared__ float row_m[MT], row_l[MT];
    // behind another kernel of the engine's chain: what it wrote (q, this step's keys). Behind the prefix pass that is long done, and only the joining waits.
    if (p.role != SP_OWN || p.fixed_slots == 0) griddep_wait();
    griddep_launch();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tq = lane & 3;
    const int split = blockIdx.x % p.splits, tile = blockIdx.x / p.splits, kvh = blockIdx.y, z = blockIdx.z;
    const int G = a.n_head / a.n_kv, bt = a.r.block_tokens;

    // ---- the rows and keys of this tile
    int r0 = 0, n_tok = a.r.n_rows, own = 0;
    const int* table = nullptr;
    const int lead = p.role == SP_OWN ? 0 : a.n_prefix;
    if (p.role != SP_PREFIX) {
        if (a.tab) {
            const SlotDev sd = a.tab[a.slots.slot[z]];
            r0 = z; n_tok = 1; own = sd.ints[1] + 1 - a.n_prefix; table = sd.block_table + a.n_prefix / bt;
        } else {
            const int b = a.r.row_start[z], e = a.r.row_start[z + 1];
            r0 = max(0, b); n_tok = min(e, a.r.n_rows) - r0;
            own = a.r.lengths[z]; table = a.r.pages + z * a.r.table_stride;
        }
    }
    const int f0 = tile * MT, n_f = min(MT, n_tok * G - f0);     // rows (token, head) of the tile, numbered within the sequence
    if (n_f <= 0) { griddep_wait(); return; }                    // (all CTAs of the cluster)
    const int cap = a.r.max_pages * bt;
    // keys that token i of the sequence sees
    auto limit = [&](int i) { return p.role == SP_PREFIX ? lead : lead + max(0, min(own - n_tok + i + 1, cap)); };
    const int lim_lo = limit(f0 / G), lim_hi = limit((f0 + n_f - 1) / G);
    const int chunk = ((lim_hi + p.splits - 1) / p.splits + 15) & ~15;
    const int q0 = min(lim_hi, split * chunk), q1 = min(lim_hi, q0 + chunk);
    const int n_tiles = (q1 - q0 + SP_TT - 1) / SP_TT;

    // ---- q fragments: rows g and g + 8 of this warp's 16
    const int w_row = MT == 16 ? 0 : 16 * warp;
    uint32_t qa[HD / 16][4];
    int lim[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int f = f0 + w_row + g + 8 * h;
        const bool in = w_row + g + 8 * h < n_f;
        const int i = in ? f / G : 0, head = kvh * G + (in ? f % G : 0);
        lim[h] = in ? limit(i) : lim_hi;
        const size_t at = (size_t)(r0 + i) * a.q_row + (size_t)head * a.q_head;
#pragma unroll
        for (int kk = 0; kk < HD / 16; kk++)
#pragma unroll
            for (int part = 0; part < 2; part++) {
                uint32_t v = 0;
                const size_t d = at + kk * 16 + part * 8 + 2 * tq;
                if (in) {
                    if (a.q_f32) { const float* q = (const float*)a.q + d; v = T::pack(__ldcg(q), __ldcg(q + 1)); }
                    else { const uint16_t* q = (const uint16_t*)a.q + d; v = (uint32_t)__ldcg(q) | (uint32_t)__ldcg(q + 1) << 16; }
                }
                qa[kk][2 * part + h] = v;
            }
    }
    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};          // (l: this thread's columns)

    // all threads: tile ti -> buffer ti % SP_STAGES. A thread copies one 16-byte piece of every eighth (sixteenth) row.
    constexpr int CPR = HD / 8, RPP = SP_THREADS / CPR;
    const int c8 = tid % CPR * 8;
    auto issue = [&](int ti) {
        const int st = ti % SP_STAGES, t0 = q0 + ti * SP_TT;
        uint16_t *kd = ks + st * SP_TT * LD + c8, *vd = vs + st * SP_TT * LD + c8;
        if (ti < n_tiles) {
            int page[SP_TT / RPP], off[SP_TT / RPP];
#pragma unroll
            for (int m = 0; m < SP_TT / RPP; m++) {
                int j = min(t0 + tid / CPR + m * RPP, q1 - 1);
                const int* from = j < lead ? a.prefix_pages : table;
                if (j >= lead) j -= lead;
                off[m] = j % bt;
                page[m] = min(max(from[j / bt], 0), (int)a.r.n_pages - 1);
            }
#pragma unroll
            for (int m = 0; m < SP_TT / RPP; m++) {
                const int j = tid / CPR + m * RPP;
                if (t0 + j < q1) {
                    const size_t at = (((size_t)page[m] * a.n_kv + kvh) * bt + off[m]) * HD + c8;
                    sp_cp16(kd + j * LD, (const uint16_t*)a.k_pool + at);
                    sp_cp16(vd + j * LD, (const uint16_t*)a.v_pool + at);
                } else {                                         // 0 * garbage must stay 0 in the weighted sum
                    *reinterpret_cast<uint4*>(kd + j * LD) = make_uint4(0, 0, 0, 0);
                    *reinterpret_cast<uint4*>(vd + j * LD) = make_uint4(0, 0, 0, 0);
                }
            }
        }
        sp_commit();
    };
    for (int i = 0; i < SP_STAGES - 1; i++) issue(i);
    for (int ti = 0; ti < n_tiles; ti++) {
        sp_wait<SP_STAGES - 2>();
        __syncthreads();                                         // tile ti is here for every warp, and every warp is done with the one before
        issue(ti + SP_STAGES - 1);
        const int st = ti % SP_STAGES, t0 = q0 + ti * SP_TT, k0 = MT == 16 ? 16 * warp : 0;      // this warp's first key of the tile
        if (t0 + k0 >= q1) continue;
        float sc[2 * KS][4];
#pragma unroll
        for (int nt = 0; nt < 2 * KS; nt++) {
            sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
            const uint16_t* kr = ks + (st * SP_TT + k0 + nt * 8 + (lane & 7)) * LD + (lane >> 3) * 8;
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk += 2) {
                uint32_t b4[4];                                  // dims kk * 16 .. + 31 of eight keys
                sp_ldmatrix_x4(b4, kr + kk * 16);
                T::mma(sc[nt], qa[kk], b4[0], b4[1]);
                T::mma(sc[nt], qa[kk + 1], b4[2], b4[3]);
            }
        }
        // ---- scale, mask, running maxima of rows g and g + 8; this thread's columns are 2 tq, 2 tq + 1 of every eight keys
        float mx[2] = {m_run[0], m_run[1]};
#pragma unroll
        for (int nt = 0; nt < 2 * KS; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = t0 + k0 + nt * 8 + 2 * tq + (e & 1);
                sc[nt][e] = key < min(lim[e >> 1], q1) ? sc[nt][e] * a.scale_log2 : -INFINITY;
                mx[e >> 1] = fmaxf(mx[e >> 1], sc[nt][e]);
            }
        float ref[2], fall[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
            mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
            ref[h] = mx[h] == -INFINITY ? 0.f : mx[h];           // nothing seen yet: every weight is 0
            fall[h] = sp_exp2(m_run[h] - ref[h]);
            m_run[h] = mx[h];
            l_run[h] *= fall[h];
        }
#pragma unroll
        for (int nt = 0; nt < 2 * KS; nt++)
#pragma unroll
            for (int e = 0; e < 4; e++) { sc[nt][e] = sp_exp2(sc[nt][e] - ref[e >> 1]); l_run[e >> 1] += sc[nt][e]; }
#pragma unroll
        for (int nt = 0; nt < HD / 8; nt++) { o[nt][0] *= fall[0]; o[nt][1] *= fall[0]; o[nt][2] *= fall[1]; o[nt][3] *= fall[1]; }
#pragma unroll
        for (int s = 0; s < KS; s++) {
            const uint32_t pa[4] = {T::pack(sc[2 * s][0], sc[2 * s][1]), T::pack(sc[2 * s][2], sc[2 * s][3]),
                                    T::pack(sc[2 * s + 1][0], sc[2 * s + 1][1]), T::pack(sc[2 * s + 1][2], sc[2 * s + 1][3])};
            const uint16_t* vb = vs + (st * SP_TT + k0 + 16 * s) * LD;
            // keys that only later rows of the tile see: a value there that is no number must not reach the earlier rows through a weight of 0
            if (t0 + k0 + 16 * s + 16 > lim_lo && lim_lo < lim_hi) {
                uint32_t bad = 0;
                for (int e = lane; e < 16 * (HD / 2); e += 32) {
                    const uint32_t v = *reinterpret_cast<const uint32_t*>(vb + e / (HD / 2) * LD + e % (HD / 2) * 2);
                    bad |= (v & T::EXP) == T::EXP || (v >> 16 & T::EXP) == T::EXP;
                }
                if (__any_sync(0xffffffffu, bad)) {
                    for (int k = 0; k < 16; k++) {
                        const int from = (lane & ~3) | (k & 7) >> 1;
                        float w[2];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            float mine = 0.f;
#pragma unroll
                            for (int e = 0; e < 4; e++) if (e == (k >> 3) * 2 + (k & 1)) mine = sc[2 * s + (e >> 1)][2 * h + (e & 1)];
                            w[h] = __shfl_sync(0xffffffffu, mine, from);
                        }
#pragma unroll
                        for (int nt = 0; nt < HD / 8; nt++)
#pragma unroll
                            for (int e = 0; e < 4; e++)
                                if (w[e >> 1] != 0.f) o[nt][e] = fmaf(w[e >> 1], T::value(vb[k * LD + nt * 8 + 2 * tq + (e & 1)]), o[nt][e]);
                    }
                    continue;
                }
            }
#pragma unroll
            for (int nt = 0; nt < HD / 8; nt += 2) {
                uint32_t b4[4];                                  // 16 keys x 16 dims, transposed on load
                sp_ldmatrix_x4_trans(b4, vb + (lane & 15) * LD + nt * 8 + (lane >> 4) * 8);
                T::mma(o[nt], pa, b4[0], b4[1]);
                T::mma(o[nt + 1], pa, b4[2], b4[3]);
            }
        }
    }
    sp_wait<0>();
    __syncthreads();                                             // everyone is done with the buffers

    // ---- this CTA's (maximum, sum, weighted sum) of every row: merged over the warps (MT 16) or as they are (MT 64)
    float* acc = reinterpret_cast<float*>(sp_smem);              // [MT][HD]
#pragma unroll
    for (int h = 0; h < 2; h++) {
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 1);
        l_run[h] += __shfl_xor_sync(0xffffffffu, l_run[h], 2);
    }
    if (MT == 16) {
        float* wo = acc + MT * HD;                               // [4][16][HD]
        float* wm = wo + 4 * MT * HD;                            // [4][16]
        float* wl = wm + 4 * MT;
#pragma unroll
        for (int h = 0; h < 2; h++) {
#pragma unroll
            for (int nt = 0; nt < HD / 8; nt++)
                *reinterpret_cast<float2*>(wo + (warp * MT + g + 8 * h) * HD + nt * 8 + 2 * tq) = make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
            if (tq == 0) { wm[warp * MT + g + 8 * h] = m_run[h]; wl[warp * MT + g + 8 * h] = l_run[h]; }
        }
        __syncthreads();
        for (int e = tid; e < n_f * (HD / 4); e += SP_THREADS) {
            const int row = e / (HD / 4), d = e % (HD / 4) * 4;
            float m = -INFINITY, l = 0.f;
#pragma unroll
            for (int w = 0; w < 4; w++) m = fmaxf(m, wm[w * MT + row]);
            const float ref = m == -INFINITY ? 0.f : m;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const float f = sp_exp2(wm[w * MT + row] - ref);
                const float4 v = *reinterpret_cast<const float4*>(wo + (w * MT + row) * HD + d);
                sum.x += f * v.x; sum.y += f * v.y; sum.z += f * v.z; sum.w += f * v.w;
                l += f * wl[w * MT + row];
            }
            *reinterpret_cast<float4*>(acc + row * HD + d) = sum;
            if (d == 0) { row_m[row] = m; row_l[row] = l; }
        }
    } else {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int row = w_row + g + 8 * h;
#pragma unroll
            for (int nt = 0; nt < HD / 8; nt++) *reinterpret_cast<float2*>(acc + row * HD + nt * 8 + 2 * tq) = make_float2(o[nt][2 * h], o[nt][2 * h + 1]);
            if (tq == 0) { row_m[row] = m_run[h]; row_l[row] = l_run[h]; }
        }
    }
    __syncthreads();
    float* ml = a.work + ml_at;
    if (p.role == SP_PREFIX) {
        for (int e = tid; e < n_f * (HD / 4); e += SP_THREADS) {
            const int f = f0 + e / (HD / 4), d = e % (HD / 4) * 4;
            const size_t at = sp_part(a, split, f / G, kvh * G + f % G);
            *reinterpret_cast<float4*>(a.work + at * HD + d) = *reinterpret_cast<const float4*>(acc + (f - f0) * HD + d);
            if (d == 0) *reinterpret_cast<float2*>(ml + at * 2) = make_float2(row_m[f - f0], row_l[f - f0]);
        }
        return;
    }
    // ---- join the cluster's CTAs and the prefix; this CTA writes its share of the tile
    if (p.splits > 1) cluster_sync();
    griddep_wait();                                              // the prefix's partial results are there
    const uint32_t rank = p.splits > 1 ? sp_cluster_rank() : 0;
    const int n_pieces = n_f * (HD / 4);
    for (int e = rank * SP_THREADS + tid; e < n_pieces; e += p.splits * SP_THREADS) {
        const int row = e / (HD / 4), d = e % (HD / 4) * 4, f = f0 + row, t = r0 + f / G, head = kvh * G + f % G;
        int slots = p.fixed_slots;
        if (slots < 0) slots = p.cut.slots(kvh * p.cut.pairs + (t * G + f % G) / 256);
        float m = -INFINITY, l = 0.f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](float m1, float l1, const float4& v) {
            const float m2 = fmaxf(m, m1), ref = m2 == -INFINITY ? 0.f : m2, c0 = sp_exp2(m - ref), c1 = sp_exp2(m1 - ref);
            l = c0 * l + c1 * l1;
            sum.x = c0 * sum.x + c1 * v.x; sum.y = c0 * sum.y + c1 * v.y; sum.z = c0 * sum.z + c1 * v.z; sum.w = c0 * sum.w + c1 * v.w;
            m = m2;
        };
#pragma unroll 4
        for (int i = 0; i < slots; i++) {
            const size_t at = sp_part(a, i, t, head);
            const float2 one = __ldcg(reinterpret_cast<const float2*>(ml + at * 2));
            add(one.x, one.y, __ldcg(reinterpret_cast<const float4*>(a.work + at * HD + d)));
        }
        if (p.splits > 1) {
#pragma unroll 2
            for (int c = 0; c < p.splits; c++)
                add(sp_cluster_load(cluster_address(smem_u32(row_m + row), c)), sp_cluster_load(cluster_address(smem_u32(row_l + row), c)),
                    cluster_load4(cluster_address(smem_u32(acc + row * HD + d), c)));
        } else {
            add(row_m[row], row_l[row], *reinterpret_cast<const float4*>(acc + row * HD + d));
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;              // (0: no keys. A NaN stays one.)
        sum.x *= inv; sum.y *= inv; sum.z *= inv; sum.w *= inv;
        const uint32_t lo = T::pack(sum.x, sum.y), hi = T::pack(sum.z, sum.w);
        if (a.out_h) {
            const int col = head * HD + d;
            *reinterpret_cast<uint2*>(a.out_h + ((size_t)(col >> 3) * a.out_T_pad + t) * 8 + (col & 7)) = make_uint2(lo, hi);
        } else {
            uint16_t* dst = (uint16_t*)a.out + (size_t)t * a.out_row + (size_t)head * a.out_head + d;
            if (((uintptr_t)dst & 7) == 0) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
            else { dst[0] = (uint16_t)lo; dst[1] = (uint16_t)(lo >> 16); dst[2] = (uint16_t)hi; dst[3] = (uint16_t)(hi >> 16); }
        }
    }
    if (p.splits > 1) cluster_sync();                            // (the others may still read this one's results)
}

// ---------------------------------------------------------------- host side
namespace {
constexpr int SP_SMS = 148;
constexpr size_t sp_smem(int hd) { return (size_t)SP_STAGES * 2 * SP_TT * (hd + 8) * 2; }

template <typename E, int HD, int MT>
cudaError_t sp_rows(const SharedPrefixArgs& a, const SpPlan& p, size_t ml_at, dim3 grid, cudaStream_t s, bool pdl) {
    const auto kernel = shared_prefix_rows_kernel<E, HD, MT>;
    if (!allow_smem<shared_prefix_rows_kernel<E, HD, MT>>((int)sp_smem(HD))) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid; cfg.blockDim = dim3(SP_THREADS); cfg.dynamicSmemBytes = sp_smem(HD); cfg.stream = s;
    cudaLaunchAttribute at[2];
    int n = 0;
    if (p.role != SP_PREFIX && p.splits > 1) {
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
    return cudaLaunchKernelEx(&cfg, kernel, a, p, ml_at);
}
template <int MT>
cudaError_t sp_rows_of(const SharedPrefixArgs& a, const SpPlan& p, size_t ml_at, dim3 grid, cudaStream_t s, bool pdl) {
    const bool h = a.type == ELEM_F16;
    if (a.head_dim == 64) return h ? sp_rows<__half, 64, MT>(a, p, ml_at, grid, s, pdl) : sp_rows<__nv_bfloat16, 64, MT>(a, p, ml_at, grid, s, pdl);
    return h ? sp_rows<__half, 128, MT>(a, p, ml_at, grid, s, pdl) : sp_rows<__nv_bfloat16, 128, MT>(a, p, ml_at, grid, s, pdl);
}
// CTAs that share a tile's keys: about two CTAs an SM in all, no fewer keys than a tile each, at most a portable cluster
int sp_splits(long tiles, long keys, int most) {
    int n = 1;
    while (2 * n <= most && tiles * n * 2 <= 2 * SP_SMS && keys / (2 * n) >= SP_TT) n *= 2;
    return n;
}
constexpr int SP_PREFIX_ROWS = 64;          // up to so many rows a KV head the prefix pass is the kernel above
constexpr int SP_PREFIX_SPLITS = 32;
}  // namespace

PrefixCut prefix_cut(long n_rows, int n_head, int n_kv, int n_prefix) {
    PrefixCut c = {};
    c.pairs = (int)((n_rows * (n_head / n_kv) + 255) / 256);
    c.units = n_kv * c.pairs;
    c.blocks = (n_prefix + 127) / 128;
    const long total = (long)c.units * c.blocks;
    c.run = (int)((total + SP_SMS - 1) / SP_SMS);
    c.ctas = c.run ? (int)((total + c.run - 1) / c.run) : 0;
    return c;
}

// most partial results a row can have: a unit of b blocks in runs of ceil(u b / 148) lies in at most ceil(148 / u) + 1 of them
static long sp_most_slots(long n_rows, int n_head, int n_kv) {
    if (n_rows * (n_head / n_kv) <= SP_PREFIX_ROWS) return SP_PREFIX_SPLITS;
    const PrefixCut c = prefix_cut(n_rows, n_head, n_kv, 1);
    return (SP_SMS + c.units - 1) / c.units + 1;
}
size_t shared_prefix_work_floats(long n_rows, int n_head, int n_kv, int head_dim) {
    return (size_t)sp_most_slots(n_rows, n_head, n_kv) * n_rows * n_head * (head_dim + 2);
}

cudaError_t shared_prefix_launch(const SharedPrefixArgs& a, cudaStream_t s) {
    const int R = a.r.n_rows, G = a.n_head / a.n_kv, S = a.r.n_seqs;
    if (R == 0 || S == 0) return cudaSuccess;
    cudaError_t e;
    SpPlan own = {};
    own.role = SP_OWN;
    size_t ml_at = 0;
    bool behind = false;
    if (a.n_prefix > 0) {
        int slots;
        if ((long)R * G <= SP_PREFIX_ROWS) {
            SpPlan p = {};
            p.role = SP_PREFIX;
            const int mt = R * G <= 16 ? 16 : 64;
            p.splits = sp_splits((long)a.n_kv, a.n_prefix, SP_PREFIX_SPLITS);
            slots = own.fixed_slots = p.splits;
            ml_at = (size_t)slots * R * a.n_head * a.head_dim;
            const dim3 grid(p.splits, a.n_kv, 1);
            e = mt == 16 ? sp_rows_of<16>(a, p, ml_at, grid, s, g_chain_pdl) : sp_rows_of<64>(a, p, ml_at, grid, s, g_chain_pdl);
        } else {
            own.cut = prefix_cut(R, a.n_head, a.n_kv, a.n_prefix);
            own.fixed_slots = -1;
            slots = (int)sp_most_slots(R, a.n_head, a.n_kv);
            ml_at = (size_t)slots * R * a.n_head * a.head_dim;
            e = shared_prefix_tc_launch(a, own.cut, s);
        }
        if (e != cudaSuccess) return e;
        behind = true;
    }
    const int mt = a.max_rows * G <= 16 ? 16 : 64, tiles = (a.max_rows * G + mt - 1) / mt;
    own.splits = sp_splits((long)tiles * a.n_kv * S, (long)a.r.max_pages * a.r.block_tokens, 8);
    const dim3 grid(tiles * own.splits, a.n_kv, S);
    return mt == 16 ? sp_rows_of<16>(a, own, ml_at, grid, s, behind || g_chain_pdl) : sp_rows_of<64>(a, own, ml_at, grid, s, behind || g_chain_pdl);
}

}  // namespace b2

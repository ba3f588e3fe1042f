// The prefix pass of shared_prefix.cu on the 5th-generation tensor cores: many query rows of a KV head over the keys that all sequences share.
//
// Rows are (row of the batch, head of the KV head's group); a unit is 256 of them, two tiles of 128. A CTA takes a run of key blocks of 128 (PrefixCut), which
// may end one unit and start the next. Keys and values come by tensor copies from their pages (64 columns a part in 128-byte-swizzled rows, two blocks under
// way) and serve both tiles. Tensor memory: two score tiles (2 x 128 columns, probabilities are written over them as the A operand of the second product) and
// two outputs. While one tile's softmax runs, the other's products do; the second product starts with the first half of the probabilities. Warps 0-3 and 4-7:
// softmax of a tile, a thread a row, scores read from tensor memory twice (maximum, then exponentials); 8: copies; 9: matrix instructions.
// The output is rescaled only where a row's maximum has grown by more than 2^8 (probabilities are then up to 2^8, sums stay 32-bit).
// Bound by the chain of a tile (scores, maximum, exponentials, second product: 1.8 us a block, of which the tensor cores take 1.1 with heads of 128 and the
// exponentials' unit 1.1), in which every instruction of the issuing warp counts. One pass over the scores with a vote every 32 whether the reference still
// serves took a fifth longer, a third score tile for heads of 64 a tenth.
#include "device_ops.h"
#include "ptx.cuh"
#include "tc05.cuh"
#include "tensor_map.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2 {

namespace {
constexpr int ST_ROWS = 128, ST_K = 128, ST_PART = 128 * 128;    // rows of a tile, keys of a block; bytes of a part (128 rows x 64 columns)
constexpr int ST_THREADS = 320;

__device__ unsigned int st_error[5];                             // see mbar_give_up

__device__ __forceinline__ float st_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <bool F16>
__device__ __forceinline__ uint32_t st_pack(float a, float b) {
    if constexpr (F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
}
// the sequences' own tokens on average, as a level of PrefixShare (of very many sequences a sample's)
__device__ __forceinline__ int st_level(const SharedPrefixArgs& a) {
    __shared__ float part[ST_THREADS / 32];
    const int n_seqs = a.r.n_seqs, step = (n_seqs + 1023) / 1024, most = a.r.max_pages * a.r.block_tokens;
    float own = 0.f;
#pragma unroll 1
    for (int z = threadIdx.x * step; z < n_seqs; z += ST_THREADS * step) {
        const int held = a.tab ? a.tab[a.slots.slot[z]].ints[1] + 1 - a.n_prefix : a.r.lengths[z];
        own += (float)min(max(held, 0), most);
    }
#pragma unroll 1
    for (int o = 16; o; o >>= 1) own += __shfl_xor_sync(0xffffffffu, own, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = own;
    __syncthreads();
    own = 0.f;
#pragma unroll 1
    for (int w = 0; w < ST_THREADS / 32; w++) own += part[w];
    const float mean = own * step / n_seqs;
    int level = 0;
    while (level < SHARE_LEVELS - 1 && mean > (float)(16 << level)) level++;
    return level;
}
}  // namespace

cudaError_t shared_prefix_tc_error(unsigned int* code) { return take_error_word(st_error, code); }
__global__ void st_give_up_kernel(unsigned int code) { mbar_give_up(0, st_error, code, 0); }
cudaError_t shared_prefix_tc_give_up(unsigned int code, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = cfg.blockDim = dim3(1); cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, st_give_up_kernel, code);
}

template <int HD, bool F16>
__global__ void __launch_bounds__(ST_THREADS, 1) shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                                         const SharedPrefixArgs a, const PrefixCut all_sms, const int box_rows, const size_t ml_at, const __grid_constant__ PrefixShare share) {
    constexpr int PARTS = HD / 64;
    extern __shared__ uint8_t st_smem[];
    __shared__ uint64_t q_full[2], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_half[2], p_full[2], pv_done[2];
    __shared__ uint32_t tmem_at;
    unsigned int* err = a.err ? a.err : st_error;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint8_t* qs = reinterpret_cast<uint8_t*>(((uintptr_t)st_smem + 1023) & ~(uintptr_t)1023);      // [tile][part]
    uint8_t* ks = qs + 2 * PARTS * ST_PART;                      // [stage][part]
    uint8_t* vs = ks + 2 * PARTS * ST_PART;
    griddep_wait();
    griddep_launch();
    PrefixCut cut = all_sms;
    if (share.adapt) {
        const int level = st_level(a);
        cut.run = share.run[level]; cut.per_unit = share.per_unit[level]; cut.ctas = share.ctas[level];
        if (blockIdx.x == 0 && threadIdx.x == 0) *reinterpret_cast<int2*>(a.work + share.cut_at) = make_int2(cut.run, cut.per_unit);
        if ((int)blockIdx.x >= cut.ctas) return;                 // (all threads alike)
    }
    if (warp == 9) {
        if (lane == 0) {
            for (int i = 0; i < 2; i++) {
                mbar_init(&q_full[i], 128); mbar_init(&k_full[i], 1); mbar_init(&k_empty[i], 1); mbar_init(&v_full[i], 1); mbar_init(&v_empty[i], 1);
                mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 128); mbar_init(&p_full[i], 128); mbar_init(&pv_done[i], 1);
            }
            fence_mbar_init();
        }
        __syncwarp();
        tc_alloc(&tmem_at, 512);
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t s_at = __shfl_sync(0xffffffffu, tmem_at, 0), o_at = s_at + 256;      // (known to be uniform)
    const int G = a.n_head / a.n_kv, M = a.r.n_rows * G, n_prefix = a.n_prefix;
    const int x0 = cut.begin(blockIdx.x), x1 = cut.end(blockIdx.x);

    // runs of blocks of one unit: every role walks them the same way
    struct Segment { int kvh, row0, b0, n; bool two; };
    auto segment = [&](int x) {
        Segment g;
        const int u = x / cut.blocks;
        g.b0 = x - u * cut.blocks;
        g.n = min(cut.blocks - g.b0, x1 - x);
        g.kvh = u / cut.pairs;
        g.row0 = u % cut.pairs * 2 * ST_ROWS;
        g.two = M - g.row0 > ST_ROWS;
        return g;
    };

    if (warp == 8) {
        // ================= copies: a lane has a box of keys (one page, or a part of one)
        const int bt = a.r.block_tokens, boxes = ST_K / box_rows;
        int it = 0;
        for (int x = x0; x < x1;) {
            const Segment g = segment(x);
            x += g.n;
            for (int i = 0; i < g.n; i++, it++) {
                const int j0 = (g.b0 + i) * ST_K, n_box = min(boxes, (n_prefix - j0 + box_rows - 1) / box_rows), st = it & 1;
                int row = 0;
                if (lane < n_box) {
                    const int j = j0 + lane * box_rows;
                    const int page = min(max(a.prefix_pages[j / bt], 0), (int)a.r.n_pages - 1);
                    row = (int)(((long)page * a.n_kv + g.kvh) * bt + j % bt);
                }
                for (int kv = 0; kv < 2; kv++) {
                    uint64_t *full = kv ? &v_full[st] : &k_full[st], *empty = kv ? &v_empty[st] : &k_empty[st];
                    uint8_t* dst = (kv ? vs : ks) + st * PARTS * ST_PART + lane * box_rows * 128;
                    if (it >= 2) mbar_wait_warp(empty, ((it >> 1) - 1) & 1, err, 0x90001u, (unsigned)it);
                    if (lane == 0) mbar_arrive_expect_tx(full, (uint32_t)(n_box * box_rows * 128 * PARTS));
                    __syncwarp();
                    if (lane < n_box)
                        for (int c = 0; c < PARTS; c++) tma_load_3d(dst + c * ST_PART, kv ? &map_v : &map_k, c * 64, row, 0, full);
                    __syncwarp();
                }
            }
        }
    } else if (warp == 9) {
        // ================= matrix instructions (all lanes run the loop, one issues)
        const uint32_t f16 = F16 ? ~((1u << 7) | (1u << 10)) : ~0u;      // (tc_idesc_bf16 without the bits that say bf16)
        const uint32_t id_s = tc_idesc_bf16(ST_ROWS, ST_K) & f16, id_o = tc_idesc_bf16(ST_ROWS, HD, true) & f16;
        const uint64_t dq0 = tc_desc(smem_u32(qs)), dk0 = tc_desc(smem_u32(ks)), dv0 = tc_desc(smem_u32(vs), ST_PART);
        int it = 0, segs[2] = {0, 0}, done[2] = {0, 0};          // blocks of the CTA, segments and blocks of each tile so far
        for (int x = x0; x < x1;) {
            const Segment g = segment(x);
            x += g.n;
            const int tiles = g.two ? 2 : 1;
            auto scores = [&](int t, int at) {
                const uint64_t dq = dq0 + t * (PARTS * ST_PART >> 4), dk = dk0 + (at & 1) * (PARTS * ST_PART >> 4);
#pragma unroll
                for (int c = 0; c < PARTS; c++) tc_mma4_one<2, 2>(s_at + t * ST_K, dq + c * (ST_PART >> 4), dk + c * (ST_PART >> 4), id_s, c ? 1u : 0u);
                tc_commit_one(&s_full[t]);
            };
            mbar_wait_warp(&k_full[it & 1], (it >> 1) & 1, err, 0x90002u, (unsigned)it);
#pragma unroll
            for (int t = 0; t < 2; t++) {                        // (unrolled: which tile it is costs no instructions)
                if (t == tiles) break;
                mbar_wait_warp(&q_full[t], segs[t]++ & 1, err, 0x90003u, (unsigned)it);
                tc_after_sync();
                scores(t, it);
            }
            tc_commit_one(&k_empty[it & 1]);
            for (int i = 0; i < g.n; i++) {
                const int at = it + i;
                mbar_wait_warp(&v_full[at & 1], (at >> 1) & 1, err, 0x90004u, (unsigned)at);
                const int valid = min(ST_K, n_prefix - (g.b0 + i) * ST_K), steps = (valid + 15) / 16;
                if (valid & 15) {
                    // keys past the prefix up to the next 16: whatever the page holds must not meet the zero weights as values
                    const int n_bad = 16 - (valid & 15);
                    for (int e = lane; e < PARTS * n_bad * 8; e += 32)
                        *reinterpret_cast<uint4*>(vs + ((at & 1) * PARTS + e / (n_bad * 8)) * ST_PART + (valid + e / 8 % n_bad) * 128 + (e & 7) * 16) = make_uint4(0, 0, 0, 0);
                    fence_proxy_async();
                    __syncwarp();
                }
                const uint64_t dv = dv0 + (at & 1) * (PARTS * ST_PART >> 4);
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    if (t == tiles) break;
                    auto sums = [&](int k0, int k1) {            // 16-key steps k0 .. k1 - 1 of the block
                        if (k1 - k0 == 4) tc_mma4_ts_one<8, 128>(o_at + t * HD, s_at + t * ST_K + k0 * 8, dv + k0 * 128, id_o, (i | k0) ? 1u : 0u);
                        else for (int k = k0; k < k1; k++) tc_mma_ts_one(o_at + t * HD, s_at + t * ST_K + k * 8, dv + k * 128, id_o, (i | k) ? 1u : 0u);
                    };
                    mbar_wait_warp(&p_half[t], done[t] & 1, err, 0x90005u, (unsigned)at);
                    tc_after_sync();
                    sums(0, min(steps, 4));
                    mbar_wait_warp(&p_full[t], done[t] & 1, err, 0x9000au, (unsigned)at);
                    done[t]++;
                    tc_after_sync();
                    sums(4, max(steps, 4));
                    tc_commit_one(&pv_done[t]);
                    if (t == tiles - 1) tc_commit_one(&v_empty[at & 1]);
                    if (i + 1 < g.n) {
                        // the next scores replace the probabilities that this product reads
                        mbar_wait_warp(&pv_done[t], (done[t] - 1) & 1, err, 0x90009u, (unsigned)at);
                        if (t == 0) { mbar_wait_warp(&k_full[(at + 1) & 1], ((at + 1) >> 1) & 1, err, 0x90002u, (unsigned)at); }
                        tc_after_sync();
                        scores(t, at + 1);
                        if (t == tiles - 1) tc_commit_one(&k_empty[(at + 1) & 1]);
                    }
                }
            }
            it += g.n;
        }
    } else {
        // ================= softmax: a thread a row of its tile
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_mine = s_at + t * ST_K + lanes, o_mine = o_at + t * HD + lanes;
        uint32_t done = 0;                                       // blocks of this tile so far
        for (int x = x0; x < x1;) {
            const Segment g = segment(x);
            const int unit = x / cut.blocks;
            x += g.n;
            if (t == 1 && !g.two) continue;
            // ---- the warp's 32 queries, into 128-byte-swizzled rows (rows past the end: zeros): neighbouring lanes have neighbouring pieces of a row
            const int f0 = g.row0 + t * ST_ROWS + (warp & 3) * 32, f = f0 + lane;
            const bool in = f < M;
            const int r = in ? f / G : 0, head = g.kvh * G + (in ? f - r * G : 0);
            const size_t q_mine = (size_t)r * a.q_row + (size_t)head * a.q_head;
            constexpr int LANES = HD / 8, ROWS = 32 / LANES;     // lanes a row, rows at once
            // (all of a batch's loads ahead of its stores: one after the other, they took 6 us)
            constexpr int BATCH = 8;
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += BATCH * ROWS) {
                uint4 v[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; b++) {
                    const int from = i0 + b * ROWS + lane / LANES;
                    const size_t at = __shfl_sync(0xffffffffu, q_mine, from) + lane % LANES * 8;
                    v[b] = make_uint4(0, 0, 0, 0);
                    if (f0 + from >= M) continue;
                    if (a.q_f32) {
                        const float* q = (const float*)a.q + at;
                        v[b] = make_uint4(st_pack<F16>(q[0], q[1]), st_pack<F16>(q[2], q[3]), st_pack<F16>(q[4], q[5]), st_pack<F16>(q[6], q[7]));
                    } else {
                        const uint16_t* q = (const uint16_t*)a.q + at;
                        if (((uintptr_t)q & 15) == 0) v[b] = *reinterpret_cast<const uint4*>(q);
                        else v[b] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
                    }
                }
#pragma unroll
                for (int b = 0; b < BATCH; b++) {
                    const int c8 = lane % LANES, row = (warp & 3) * 32 + i0 + b * ROWS + lane / LANES;
                    *reinterpret_cast<uint4*>(qs + (t * PARTS + (c8 >> 3)) * ST_PART + row * 128 + (((c8 & 7) ^ (row & 7)) << 4)) = v[b];
                }
            }
            fence_proxy_async();
            mbar_arrive(&q_full[t]);
            float m_ref = -INFINITY;
            uint64_t l2 = f2_pack(0.f, 0.f), l3 = l2;            // sums of even and odd entries, twice
            const uint64_t scale2 = f2_pack(a.scale_log2, a.scale_log2);
            for (int i = 0; i < g.n; i++, done++) {
                mbar_wait(&s_full[t], done & 1, err, 0x90006u, done);
                tc_after_sync();
                __syncwarp();
                const int valid = n_prefix - (g.b0 + i) * ST_K;
                // 32 scores at a time, the next ones on their way: the maximum, then the exponentials
                uint32_t raw[2][32];
                auto load = [&](int c) { tc_ld32(s_mine + c * 32, raw[c & 1]); };
                auto mask = [&](int c) {
                    if (valid < ST_K) {
#pragma unroll
                        for (int j = 0; j < 32; j++) if (c * 32 + j >= valid) raw[c & 1][j] = 0xff800000u;
                    }
                };
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                load(0);
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    tc_wait_ld(raw[c & 1]);
                    load((c + 1) & 3);                           // (the last of these: the first scores again)
                    mask(c);
#pragma unroll
                    for (int j = 0; j < 32; j++) mx4[j & 3] = fmaxf(mx4[j & 3], __uint_as_float(raw[c & 1][j]));
                }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * a.scale_log2;
                const bool grow = mx > m_ref + 8.f || (m_ref == -INFINITY && mx > -INFINITY);
                float fall = 1.f;
                if (grow) {
                    fall = st_exp2(m_ref - mx);                  // (0 the first time)
                    m_ref = mx;
                    const uint64_t fall2 = f2_pack(fall, fall);
                    l2 = f2_mul(l2, fall2); l3 = f2_mul(l3, fall2);
                }
                const float ref = m_ref > -INFINITY ? -m_ref : 0.f;
                const uint64_t ref2 = f2_pack(ref, ref);
                if (i > 0 && __any_sync(0xffffffffu, grow)) {    // the products so far must be in before they are rescaled
                    tc_wait_ld(raw[0]);
                    mbar_wait(&pv_done[t], (done - 1) & 1, err, 0x90007u, done);
                    tc_after_sync();
                    __syncwarp();
                    for (int c = 0; c < HD; c += 16) {
                        float o[16];
                        tc_ld16(o_mine + c, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] *= fall;
                        tc_st16(o_mine + c, o);
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    tc_wait_ld(raw[c & 1]);
                    if (c < 3) load(c + 1);
                    mask(c);
                    uint32_t p[16];
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float2 d = f2_unpack(f2_fma(f2_pack(__uint_as_float(raw[c & 1][j]), __uint_as_float(raw[c & 1][j + 1])), scale2, ref2));
                        const float e0 = st_exp2(d.x), e1 = st_exp2(d.y);
                        if (j & 2) l3 = f2_add(l3, f2_pack(e0, e1)); else l2 = f2_add(l2, f2_pack(e0, e1));
                        p[j >> 1] = st_pack<F16>(e0, e1);
                    }
                    tc_st16(s_mine + c * 16, p);                 // over scores that have been read
                    if (c == 1 || c == 3) {
                        tc_wait_st();
                        tc_before_sync();
                        mbar_arrive(c == 1 ? &p_half[t] : &p_full[t]);
                    }
                }
            }
            // ---- this segment's results of the row
            mbar_wait(&pv_done[t], (done - 1) & 1, err, 0x90008u, done);
            tc_after_sync();
            __syncwarp();
            const int slot = blockIdx.x - cut.first_cta(unit);
            const size_t at = ((size_t)slot * a.r.n_rows + r) * a.n_head + head;
            // 32 columns at a time through the part of shared memory that held the warp's queries (nothing reads them any more), so that a row's
            // columns leave side by side: straight from the registers, every lane's 16 bytes went to a row of their own and a run of 4 blocks took 20 us
            // longer than its blocks
            uint8_t* mine = qs + t * PARTS * ST_PART + (warp & 3) * 32 * 128;
            size_t to[8];
#pragma unroll
            for (int i = 0; i < 8; i++) to[i] = __shfl_sync(0xffffffffu, at, i * 4 + (lane >> 3)) * HD + (lane & 7) * 4;
#pragma unroll
            for (int c = 0; c < HD; c += 32) {
                uint32_t o[32];
                __syncwarp();
                tc_ld32(o_mine + c, o);
                tc_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(mine + lane * 128 + (((e >> 2) ^ (lane & 7)) << 4)) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                __syncwarp();
                uint4 v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = *reinterpret_cast<const uint4*>(mine + (i * 4 + (lane >> 3)) * 128 + (((lane & 7) ^ ((i * 4 + (lane >> 3)) & 7)) << 4));
#pragma unroll
                for (int i = 0; i < 8; i++) if (f0 + i * 4 + (lane >> 3) < M) *reinterpret_cast<uint4*>(a.work + to[i] + c) = v[i];
            }
            const float2 la = f2_unpack(l2), lb = f2_unpack(l3);
            if (in) *reinterpret_cast<float2*>(a.work + ml_at + at * 2) = make_float2(m_ref, (la.x + la.y) + (lb.x + lb.y));
            tc_before_sync();
        }
    }
    __syncthreads();
    if (warp == 9) tc_dealloc(tmem_at, 512);
}

// ---------------------------------------------------------------- host side
template <int HD, bool F16>
static cudaError_t st_launch(const SharedPrefixArgs& a, const PrefixCut& cut, size_t ml_at, const PrefixShare& share, cudaStream_t s) {
    constexpr int parts = HD / 64, smem = 6 * parts * ST_PART + 1024;
    if (!allow_smem<shared_prefix_tc_kernel<HD, F16>>(smem)) return cudaErrorInvalidValue;
    int box = ST_K;
    while (a.r.block_tokens % box) box /= 2;
    const long rows = a.r.n_pages * a.n_kv * a.r.block_tokens;
    CUtensorMap mk, mv;                                          // (copies move 16-bit entries whatever their format)
    if (!bf16_rows_map(&mk, a.k_pool, HD, rows, HD, 1, 0, box) || !bf16_rows_map(&mv, a.v_pool, HD, rows, HD, 1, 0, box)) return cudaErrorInvalidValue;
    return launch_chain(shared_prefix_tc_kernel<HD, F16>, dim3(share.adapt ? PREFIX_SMS : cut.ctas), dim3(ST_THREADS), smem, s, mk, mv, a, cut, box, ml_at, share);
}

cudaError_t shared_prefix_tc_launch(const SharedPrefixArgs& a, const PrefixCut& cut, size_t ml_at, const PrefixShare& share, cudaStream_t s) {
    if (a.r.block_tokens % 16 || cut.ctas < 1) return cudaErrorInvalidValue;
    if (a.head_dim == 64) return a.type == ELEM_F16 ? st_launch<64, true>(a, cut, ml_at, share, s) : st_launch<64, false>(a, cut, ml_at, share, s);
    if (a.head_dim == 128) return a.type == ELEM_F16 ? st_launch<128, true>(a, cut, ml_at, share, s) : st_launch<128, false>(a, cut, ml_at, share, s);
    return cudaErrorInvalidValue;
}

}  // namespace b2

// Attention over a paged cache in 4 bits for many rows of a sequence (prompts), on the 5th-generation tensor cores. What is computed: attention_4bit.cu.
//
// Rows are (token, head of the KV head's group), numbered within their sequence; a unit is 256 of them with a KV head, two tiles of 128 rows. The blocks of 128 keys of all units laid
// end to end are cut into equal runs, one a CTA; a run that begins or ends inside a unit leaves partial results in 32 bits, which a small kernel joins. A tile's last row says how many
// blocks its unit has, so that a prompt's later keys cost its first rows nothing.
// Warps 0-3 and 4-7: softmax of a tile, a thread a row, as in shared_prefix_tc.cu. 8-15: codes into operands. 16: copies of the cache's bytes. 17: matrix instructions. Tensor memory: two
// score tiles (probabilities are written over them) and two outputs.
//
// A value s (c - 8) has up to 14 bits, an f16 or bf16 operand 11 or 8. Rounded, keys would be off by 2^-12 each, and a score by more than all else together (relative error of the output
// 3.5e-4 from the keys alone, 1.8e-4 from the values, where the output's own rounding to f16 is 2.1e-4). So keys and values are two operands each, both exact: with the upper
// bits of the scale, and with the rest of it. That doubles the products, which then are what this is bound by: 2048 rows behind 6000 tokens, 32 heads over 8 of 128, 353 to 361 us, 650 to 670 TFLOP/s of
// what is asked for and twice as much of what is done. Probabilities are rounded to the queries' type.
#include "attention_4bit.cuh"
#include "kv_4bit.cuh"
#include "ptx.cuh"
#include "tc05.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <limits.h>
#include <math.h>

namespace b2 {

namespace {
constexpr int T4_ROWS = 128, T4_K = 128, T4_PART = 128 * 128;    // rows of a tile, keys of a block; bytes of a part (128 rows x 64 columns)
constexpr int T4_THREADS = 640, T4_RAW = 3;                      // copies under way: keys or values of a block
constexpr int T4_SMS = 148;
constexpr int t4_stages(int d) { return d == 64 ? 2 : 1; }       // blocks of operands

__device__ unsigned int t4_error[5];                             // see mbar_give_up

__device__ __forceinline__ float t4_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
template <bool F16>
__device__ __forceinline__ uint32_t t4_pack(float a, float b) {
    if constexpr (F16) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
}
template <int N> __device__ __forceinline__ void t4_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void t4_fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
// (groups of four warps: two of the first, two of the second, one of the third. They begin with 96 each.)
constexpr int T4_REG_SOFTMAX = 144, T4_REG_OPERANDS = 64, T4_REG_OTHERS = 56;
static_assert(2 * T4_REG_SOFTMAX + 2 * T4_REG_OPERANDS + T4_REG_OTHERS <= 5 * 96, "registers of a block");

// Four steps of K, each with two operands B whose products are added up: the queries are read once for both (the second takes them from where the first has left them). Shared memory
// is read at 96 bytes a cycle then instead of 128, all that it has, and the warps that make operands write there too.
template <int SA, int SB>
__device__ __forceinline__ void t4_mma8_one(uint32_t d, uint64_t a, uint64_t b, uint64_t c, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p, q, e;\n\t.reg .b64 a1, b1, c1, a2, b2, c2, a3, b3, c3;\n\tsetp.ne.b32 p, %5, 0;\n\tsetp.eq.b32 q, 0, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
                 "add.s64 a1, %1, %6;\n\tadd.s64 b1, %2, %7;\n\tadd.s64 c1, %3, %7;\n\tadd.s64 a2, a1, %6;\n\tadd.s64 b2, b1, %7;\n\tadd.s64 c2, c1, %7;\n\t"
                 "add.s64 a3, a2, %6;\n\tadd.s64 b3, b2, %7;\n\tadd.s64 c3, c2, %7;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], %1, %2, %4, p;\n\t@e tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], %1, %3, %4, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], a1, b1, %4, q;\n\t@e tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], a1, c1, %4, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], a2, b2, %4, q;\n\t@e tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], a2, c2, %4, q;\n\t"
                 "@e tcgen05.mma.cta_group::1.kind::f16.collector::a::fill [%0], a3, b3, %4, q;\n\t@e tcgen05.mma.cta_group::1.kind::f16.collector::a::lastuse [%0], a3, c3, %4, q;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "l"(c), "r"(idesc), "r"(accumulate), "n"(SA), "n"(SB) : "memory");
}

struct T4Seq {
    int r0, n, own, lim0, tiles;     // first row, rows that are computed, tokens, keys of the first row, units a KV head
    __device__ T4Seq() {}
    __device__ T4Seq(const Attention4Args& a, int z) {
        r0 = min(max(a.r.row_start[z], 0), a.r.n_rows);
        const int all = max(min(max(a.r.row_start[z + 1], 0), a.r.n_rows) - r0, 0);
        n = min(all, a.max_rows);
        own = min(max(a.r.lengths[z], 0), a.r.max_pages * a.r.block_tokens);
        lim0 = own - all + 1;
        tiles = (int)(((long)n * a.group + 2 * T4_ROWS - 1) / (2 * T4_ROWS));
    }
    __device__ int limit(int i) const { return max(0, lim0 + i); }
    // blocks of keys that the unit's last row sees
    __device__ int steps(int tile, const Attention4Args& a) const {
        const int last = min(n - 1, a4_row(a, (unsigned)tile * (2 * T4_ROWS) + 2 * T4_ROWS - 1));      // (below 2^31 + 256)
        return max(1, (min(limit(last), own) + T4_K - 1) / T4_K);
    }
    __device__ long all_steps(const Attention4Args& a) const { long s = 0; for (int t = 0; t < tiles; t++) s += steps(t, a); return s; }
};

// the runs of blocks of one unit: every role walks them the same way
struct T4Walk {
    int z, tile, kvh, block, left;   // left: blocks of the CTA's run that are not given out yet
    T4Seq s;
    int b0, n, steps;                // this segment: first block, blocks, blocks of its unit
    int seg_kvh, seg_f0, seg_z;
    __device__ bool next(const Attention4Args& a) {
        if (left <= 0) return false;
        steps = s.steps(tile, a);
        b0 = block; n = min(steps - block, left); seg_kvh = kvh; seg_f0 = tile * 2 * T4_ROWS; seg_z = z;
        return true;
    }
    __device__ void done(const Attention4Args& a) {
        left -= n; block = 0;
        if (left <= 0 || ++kvh < a.n_kv) return;
        kvh = 0;
        if (++tile < s.tiles) return;
        tile = 0;
        do { if (++z >= a.r.n_seqs) { left = 0; return; } s = T4Seq(a, z); } while (s.tiles == 0);
    }
};

// A group's scale in two parts of the operands' type, each twice, so that a code (3 bits, or a power of two) times either is exact. f16, 11 bits: the upper 7 of the scale's 11 bits, and the
// other 4. bf16, 8 bits: rounded to 5, and what is left: 32 of the scale's last place at most, 5 bits.
template <bool F16>
struct T4Scale {
    uint32_t hi, lo;
    __device__ __forceinline__ explicit T4Scale(uint32_t bits) {
        if constexpr (F16) {
            const uint32_t two = bits | bits << 16;
            hi = two & 0xfff0fff0u;
            const __half2 rest = __hsub2(*reinterpret_cast<const __half2*>(&two), *reinterpret_cast<const __half2*>(&hi));
            lo = *reinterpret_cast<const uint32_t*>(&rest);
        } else {
            // (a NaN may become a number in `up`; the rest is a NaN then)
            const float s = __half2float(__ushort_as_half((uint16_t)bits)), up = __uint_as_float((__float_as_uint(s) + 0x40000u) & 0xfff80000u);
            hi = __byte_perm(__float_as_uint(up), 0, 0x3232);
            lo = t4_pack<false>(s - up, s - up);
        }
    }
};
__device__ __forceinline__ uint32_t t4_fma(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
template <bool F16> __device__ __forceinline__ uint32_t t4_mul(uint32_t a, uint32_t b) {
    uint32_t r;
    if constexpr (F16) { const __half2 v = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b)); r = *reinterpret_cast<const uint32_t*>(&v); }
    else { const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b)); r = *reinterpret_cast<const uint32_t*>(&v); }
    return r;
}
// The codes of N words (the first lowest) less 8 and times a scale in two parts: 16 bytes of either operand each, codes in the order 0, 4, 1, 5, 2, 6, 3, 7, which a mask leaves them in
// (queries are put into the same order, outputs taken out of it). f16: 64 + c is a code shifted into the number 64; that times a part of the scale less 72 times it is exact, up to
// the scales whose 72-fold is past f16's range. bf16: 128 + c, less 136, times the parts.
template <bool F16, int N>
__device__ __forceinline__ void t4_operands(const uint32_t (&words)[N], uint32_t scale, uint4 (&hi)[N], uint4 (&lo)[N]) {
    const T4Scale<F16> s(scale);
    if (F16 && !__any_sync(0xffffffffu, (scale & 0x7fffu) >= 0x6000u)) {
        const uint32_t off_hi = t4_mul<F16>(s.hi, 0xd480d480u), off_lo = t4_mul<F16>(s.lo, 0xd480d480u);      // -72
#pragma unroll
        for (int n = 0; n < N; n++) {
            const uint32_t w = words[n], c0 = (w << 4 & 0x00f000f0u) | 0x54005400u, c1 = (w & 0x00f000f0u) | 0x54005400u, c2 = (w >> 4 & 0x00f000f0u) | 0x54005400u,
                           c3 = (w >> 8 & 0x00f000f0u) | 0x54005400u;
            hi[n] = make_uint4(t4_fma(c0, s.hi, off_hi), t4_fma(c1, s.hi, off_hi), t4_fma(c2, s.hi, off_hi), t4_fma(c3, s.hi, off_hi));
            lo[n] = make_uint4(t4_fma(c0, s.lo, off_lo), t4_fma(c1, s.lo, off_lo), t4_fma(c2, s.lo, off_lo), t4_fma(c3, s.lo, off_lo));
        }
        return;
    }
#pragma unroll
    for (int n = 0; n < N; n++) {
        uint32_t c[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t x = (words[n] >> (4 * i) & 0x000f000fu) | (F16 ? 0x64006400u : 0x43004300u), off = F16 ? 0x64086408u : 0x43084308u;
            if constexpr (F16) { const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&off)); c[i] = *reinterpret_cast<const uint32_t*>(&v); }
            else { const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&off)); c[i] = *reinterpret_cast<const uint32_t*>(&v); }
        }
        hi[n] = make_uint4(t4_mul<F16>(c[0], s.hi), t4_mul<F16>(c[1], s.hi), t4_mul<F16>(c[2], s.hi), t4_mul<F16>(c[3], s.hi));
        lo[n] = make_uint4(t4_mul<F16>(c[0], s.lo), t4_mul<F16>(c[1], s.lo), t4_mul<F16>(c[2], s.lo), t4_mul<F16>(c[3], s.lo));
    }
}
}  // namespace

template <int D, bool F16>
__global__ void __launch_bounds__(T4_THREADS, 1) attention_4bit_tc_kernel(const Attention4Args a) {
    constexpr int PARTS = D / 64, NG = D / Q4_GROUP, BLOCK = q4_block(D), RAW = T4_K / Q4_TOKENS * BLOCK, ST = t4_stages(D), OPERAND = 2 * PARTS * T4_PART;      // (both halves of K or V)
    constexpr int PART = 2 * T4_ROWS * (D + 2);                  // floats of a partial result
    extern __shared__ uint8_t t4_smem[];
    __shared__ uint64_t raw_full[T4_RAW], raw_empty[T4_RAW], q_full[2], k_full[ST][PARTS], k_empty[ST][PARTS], v_full[ST][2], v_empty[ST][2], s_full[2], p_half[2], p_full[2], pv_done[2], seg_done[2];
    __shared__ uint32_t tmem_at;
    __shared__ int first_bad[2][NG];                             // first key of the segment whose value's group is no number
    __shared__ T4Walk start;
    __shared__ long run_shared[2];                               // blocks a run, runs that have one more
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint8_t* qs = reinterpret_cast<uint8_t*>(((uintptr_t)t4_smem + 1023) & ~(uintptr_t)1023);      // [tile][part]
    uint8_t* ks = qs + 2 * PARTS * T4_PART;                      // [stage][upper, rest][part]
    uint8_t* vs = ks + ST * OPERAND;
    uint8_t* raw = vs + ST * OPERAND;                            // [T4_RAW]
    const int G = a.group;
    griddep_wait();
    griddep_launch();
    if (warp == 17) {
        if (lane == 0) {
            for (int i = 0; i < T4_RAW; i++) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 8); }
            for (int i = 0; i < 2; i++) {
                mbar_init(&q_full[i], 128); mbar_init(&s_full[i], 1); mbar_init(&p_half[i], 128); mbar_init(&p_full[i], 128); mbar_init(&pv_done[i], 1); mbar_init(&seg_done[i], 8);
            }
            for (int i = 0; i < ST; i++) {
                for (int c = 0; c < PARTS; c++) { mbar_init(&k_full[i][c], 8); mbar_init(&k_empty[i][c], 1); }
                for (int h = 0; h < 2; h++) { mbar_init(&v_full[i][h], 8); mbar_init(&v_empty[i][h], 1); }
            }
            fence_mbar_init();
        }
        __syncwarp();
        tc_alloc(&tmem_at, 512);
        // ---- all blocks, and where this CTA's run of them begins
        long total = 0, u0 = 0, before = 0;
        for (int pass = 0; pass < 2; pass++) {
            for (int z0 = 0; z0 < a.r.n_seqs; z0 += 32) {
                T4Seq s;
                long mine = 0;
                s.tiles = 0;
                if (z0 + lane < a.r.n_seqs) s = T4Seq(a, z0 + lane);
                // few units a sequence: a lane counts its own; else all lanes those of one after the other
                if (__any_sync(0xffffffffu, s.tiles > 4)) {
                    for (int l = 0; l < 32; l++) {
                        T4Seq one;
                        one.n = __shfl_sync(0xffffffffu, s.n, l); one.own = __shfl_sync(0xffffffffu, s.own, l); one.lim0 = __shfl_sync(0xffffffffu, s.lim0, l); one.tiles = __shfl_sync(0xffffffffu, s.tiles, l);
                        long sum = 0;
                        for (int t = lane; t < one.tiles; t += 32) sum += one.steps(t, a);
#pragma unroll
                        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                        if (lane == l) mine = sum;
                    }
                } else mine = s.all_steps(a);
                mine *= a.n_kv;
                long sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) { const long v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
                if (pass == 1) {
                    const unsigned past = __ballot_sync(0xffffffffu, before + sum > u0);
                    if (past) {
                        const int l = __ffs(past) - 1;
                        long rest = u0 - before - __shfl_sync(0xffffffffu, sum - mine, l);
                        if (lane == l) {
                            int tile = 0;
                            for (; tile + 1 < s.tiles; tile++) {
                                const long here = (long)s.steps(tile, a) * a.n_kv;
                                if (rest < here) break;
                                rest -= here;
                            }
                            const int each = s.steps(tile, a);
                            start.z = z0 + l; start.tile = tile; start.kvh = (int)(rest / each); start.block = (int)(rest % each); start.s = s;
                        }
                        break;
                    }
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
            if (pass == 0) {
                total = before; before = 0;
                const long ctas = min((long)gridDim.x, total), run = ctas ? total / ctas : 0, longer = total - run * ctas, me = blockIdx.x;
                u0 = run * me + min(me, longer);
                const long mine = me < ctas ? run + (me < longer) : 0;
                if (lane == 0) { start.left = (int)min(mine, (long)INT_MAX); run_shared[0] = run; run_shared[1] = longer; }
                if (mine == 0) break;
            }
        }
    }
    tc_before_sync();
    __syncthreads();
    tc_after_sync();
    const uint32_t s_at = __shfl_sync(0xffffffffu, tmem_at, 0), o_at = s_at + 256;
    T4Walk walk = start;

    if (warp >= 16) {
        t4_fewer_registers<T4_REG_OTHERS>();
        if (warp == 16) {
            // ================= copies: lane j has the block's 16-token block j, keys, then values
            const int blocks = a.r.block_tokens / Q4_TOKENS;
            int it = 0;
            for (; walk.next(a); walk.done(a)) {
                const long table = walk.seg_z * a.r.table_stride;
                const int own = walk.s.own;
                for (int i = 0; i < walk.n; i++) {
                    const int j0 = (walk.b0 + i) * T4_K, n = max(0, min(T4_K / Q4_TOKENS, (own - j0 + Q4_TOKENS - 1) / Q4_TOKENS));
                    long from = 0;
                    if (lane < n) {
                        const unsigned b = j0 / Q4_TOKENS + lane, page_no = b / (unsigned)blocks;
                        const int page = min(max(a.r.pages[table + page_no], 0), (int)a.r.n_pages - 1);
                        from = (((long)page * a.n_kv + walk.seg_kvh) * blocks + (b - page_no * blocks)) * BLOCK;
                    }
                    for (int kv = 0; kv < 2; kv++, it++) {
                        const int st = it % T4_RAW;
                        if (it >= T4_RAW) mbar_wait_warp(&raw_empty[st], (it / T4_RAW - 1) & 1, t4_error, 0xc0001u, (unsigned)it);
                        if (lane == 0) mbar_arrive_expect_tx(&raw_full[st], (uint32_t)(n * BLOCK));
                        __syncwarp();
                        if (lane < n) tma_load_1d(raw + st * RAW + lane * BLOCK, (const uint8_t*)(kv ? a.v_pool : a.k_pool) + from, BLOCK, &raw_full[st]);
                        __syncwarp();
                    }
                }
            }
        } else if (warp == 17) {
            // ================= matrix instructions (all lanes run the loop, one issues)
            const uint32_t f16 = F16 ? ~((1u << 7) | (1u << 10)) : ~0u;      // (tc_idesc_bf16 without the bits that say bf16)
            const uint32_t id_s = tc_idesc_bf16(T4_ROWS, T4_K) & f16, id_o = tc_idesc_bf16(T4_ROWS, D, true) & f16;
            const uint64_t dq0 = tc_desc(smem_u32(qs)), dk0 = tc_desc(smem_u32(ks)), dv0 = tc_desc(smem_u32(vs), T4_PART);
            int it = 0, segs[2] = {0, 0}, done[2] = {0, 0};      // blocks of the CTA, segments and blocks of each tile so far
            for (; walk.next(a); walk.done(a)) {
                const int n = walk.n, tiles = (long)walk.s.n * G - walk.seg_f0 > T4_ROWS ? 2 : 1;
                // (`first`: nobody has waited for these keys yet; `last`: nobody needs them any more)
                auto scores = [&](int t, int at, bool first, bool last) {
                    const int st = at % ST;
                    const uint64_t dq = dq0 + t * (PARTS * T4_PART >> 4), dk = dk0 + st * (OPERAND >> 4);
#pragma unroll
                    for (int c = 0; c < PARTS; c++) {
                        if (first) { mbar_wait_warp(&k_full[st][c], (at / ST) & 1, t4_error, 0xc0002u, (unsigned)at); tc_after_sync(); }
                        t4_mma8_one<2, 2>(s_at + t * T4_K, dq + c * (T4_PART >> 4), dk + c * (T4_PART >> 4), dk + (PARTS + c) * (T4_PART >> 4), id_s, c ? 1u : 0u);
                        if (last) tc_commit_one(&k_empty[st][c]);
                    }
                    tc_commit_one(&s_full[t]);
                };
#pragma unroll
                for (int t = 0; t < 2; t++) {                    // (unrolled: which tile it is costs no instructions)
                    if (t == tiles) break;
                    mbar_wait_warp(&q_full[t], segs[t]++ & 1, t4_error, 0xc0003u, (unsigned)it);
                    tc_after_sync();
                    scores(t, it, t == 0, t == tiles - 1);
                }
                for (int i = 0; i < n; i++) {
                    const int at = it + i, st = at % ST;
                    const uint32_t turn = (at / ST) & 1;
                    const uint64_t dv = dv0 + st * (OPERAND >> 4);
#pragma unroll
                    for (int t = 0; t < 2; t++) {
                        if (t == tiles) break;
                        auto sums = [&](int half) {              // 64 keys of the block
#pragma unroll
                            for (int h = 0; h < 2; h++)
                                tc_mma4_ts_one<8, 128>(o_at + t * D, s_at + t * T4_K + half * 32, dv + h * (PARTS * T4_PART >> 4) + half * 512, id_o, (i | half | h) ? 1u : 0u);
                        };
                        if (t == 0) mbar_wait_warp(&v_full[st][0], turn, t4_error, 0xc0004u, (unsigned)at);
                        mbar_wait_warp(&p_half[t], done[t] & 1, t4_error, 0xc0005u, (unsigned)at);
                        tc_after_sync();
                        sums(0);
                        if (t == tiles - 1) tc_commit_one(&v_empty[st][0]);
                        if (t == 0) mbar_wait_warp(&v_full[st][1], turn, t4_error, 0xc0004u, (unsigned)at);
                        mbar_wait_warp(&p_full[t], done[t] & 1, t4_error, 0xc000au, (unsigned)at);
                        done[t]++;
                        tc_after_sync();
                        sums(1);
                        tc_commit_one(&pv_done[t]);
                        if (t == tiles - 1) tc_commit_one(&v_empty[st][1]);
                        if (i + 1 < n) {
                            // the next scores replace the probabilities that this product reads
                            mbar_wait_warp(&pv_done[t], (done[t] - 1) & 1, t4_error, 0xc0009u, (unsigned)at);
                            tc_after_sync();
                            scores(t, at + 1, t == 0, t == tiles - 1);
                        }
                    }
                }
                it += n;
            }
        }
    } else if (warp >= 8) {
        // ================= codes into operands: keys 64 dims at a time, values 64 keys at a time, by all eight warps. What a warp is to write is ready before its place is free.
        // (The tensor cores take 70 % of the time, and reading operands beside the warps that write them makes their products a fifth longer. Neither warps of their own for keys and values nor
        // the second tile's product ahead of the first one's next scores where it is ready first made it faster: a hundredth slower for 2048 rows behind 6000.)
        t4_fewer_registers<T4_REG_OPERANDS>();
        const int dw = warp & 7, eight = lane & 7;               // (eight neighbouring lanes: keys that follow one another; a lane has the 32 dims of a group)
        auto put = [&](uint8_t* row, int key, int g, const uint4 (&hi)[4], const uint4 (&lo)[4]) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                uint8_t* at = row + (((w + 4 * (g & 1)) ^ (key & 7)) << 4);
                *reinterpret_cast<uint4*>(at) = hi[w];
                *reinterpret_cast<uint4*>(at + PARTS * T4_PART) = lo[w];
            }
        };
        const int k_token = (lane >> 4) * 8 + eight, k_g = lane >> 3 & 1;                                       // of block dw
        const int v_key = NG == 4 ? dw * 8 + eight : dw * 16 + k_token, v_g = NG == 4 ? lane >> 3 : k_g;       // of 64 keys (heads of 64: four warps' work)
        const int v_token = v_key % Q4_TOKENS, v_pair = v_token >> 1;
        // scales of groups that are no numbers: NaN and infinities; in f16 operands those too whose eightfold is past the type's range, which would be infinities there
        constexpr uint32_t NO_NUMBER = F16 ? 0x7000 : 0x7c00;
        int it = 0, seg = 0;
        for (; walk.next(a); walk.done(a), seg++) {
            if (seg >= 2) mbar_wait_warp(&seg_done[seg & 1], ((seg >> 1) - 1) & 1, t4_error, 0xc000bu, (unsigned)seg);
            if (dw == 0 && lane < NG) first_bad[seg & 1][lane] = INT_MAX;
            named_bar_sync(1, 256);
            for (int i = 0; i < walk.n; i++, it++) {
                const int j0 = (walk.b0 + i) * T4_K, st = it % ST;
                uint32_t words[4];
                uint4 hi[4], lo[4];
                int r = 2 * it;
                mbar_wait_warp(&raw_full[r % T4_RAW], (r / T4_RAW) & 1, t4_error, 0xc000cu, (unsigned)it);
                const uint8_t* p = raw + r % T4_RAW * RAW + dw * BLOCK;
#pragma unroll 1
                for (int c = 0; c < PARTS; c++) {
#pragma unroll
                    for (int w = 0; w < 4; w++) words[w] = *reinterpret_cast<const uint32_t*>(p + k_token * (D / 2) + (q4_key_chunk(D, k_token, w) * NG + 2 * c + k_g) * 4);
                    uint32_t scale = *reinterpret_cast<const uint16_t*>(p + q4_scale(D, k_token, 2 * c + k_g));
                    if ((scale & 0x7fffu) >= NO_NUMBER) scale = 0x7fff;
                    t4_operands<F16>(words, scale, hi, lo);
                    if (it >= ST) mbar_wait_warp(&k_empty[st][c], (it / ST - 1) & 1, t4_error, 0xc000du, (unsigned)it);
                    put(ks + st * OPERAND + c * T4_PART + (dw * Q4_TOKENS + k_token) * 128, k_token, k_g, hi, lo);
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&k_full[st][c]);
                }
                if (lane == 0) mbar_arrive(&raw_empty[r % T4_RAW]);
                r++;
                mbar_wait_warp(&raw_full[r % T4_RAW], (r / T4_RAW) & 1, t4_error, 0xc000cu, (unsigned)it);
#pragma unroll 1
                for (int half = 0; half < 2; half++) {
                    if (NG == 4 || dw < 4) {
                        const uint8_t* p = raw + r % T4_RAW * RAW + (half * 4 + v_key / Q4_TOKENS) * BLOCK;
                        const int k = half * 64 + v_key;
                        uint32_t scale = *reinterpret_cast<const uint16_t*>(p + q4_scale(D, v_token, v_g));
#pragma unroll
                        for (int w = 0; w < 4; w++)
                            words[w] = __byte_perm(*reinterpret_cast<const uint32_t*>(p + v_pair * D + (q4_value_chunk(D, v_pair, 2 * w) * NG + v_g) * 4),
                                                   *reinterpret_cast<const uint32_t*>(p + v_pair * D + (q4_value_chunk(D, v_pair, 2 * w + 1) * NG + v_g) * 4), v_token & 1 ? 0x7632u : 0x5410u);
                        // keys that nobody has: zeros. A value that is no number must not meet the zero weights of rows that do not see it: it is written down instead.
                        if (j0 + k >= walk.s.own) scale = 0;
                        if ((scale & 0x7fffu) >= NO_NUMBER) {
                            atomicMin(&first_bad[seg & 1][v_g], j0 + k);
                            scale = 0;
                        }
                        __syncwarp();
                        t4_operands<F16>(words, scale, hi, lo);
                        if (it >= ST) mbar_wait_warp(&v_empty[st][half], (it / ST - 1) & 1, t4_error, 0xc000eu, (unsigned)it);
                        put(vs + st * OPERAND + (v_g >> 1) * T4_PART + k * 128, k, v_g, hi, lo);
                    }
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&v_full[st][half]);
                }
                if (lane == 0) mbar_arrive(&raw_empty[r % T4_RAW]);
            }
        }
    } else {
        // ================= softmax: a thread a row of its tile
        t4_more_registers<T4_REG_SOFTMAX>();
        const int t = warp >> 2;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, s_mine = s_at + t * T4_K + lanes, o_mine = o_at + t * D + lanes;
        A4Desc* desc = a4_desc<PART>(a, gridDim.x) + blockIdx.x * 2;
        bool open[2] = {false, false};
        uint32_t done = 0;                                       // blocks of this tile so far
        int seg = 0;
        long given = run_shared[0] * blockIdx.x + min((long)blockIdx.x, run_shared[1]);      // the segment's first block among all
        for (; walk.next(a); given += walk.n, walk.done(a), seg++) {
            const int M = (int)min((long)INT_MAX, (long)walk.s.n * G), n_f = min(2 * T4_ROWS, M - walk.seg_f0), r0 = walk.s.r0, own = walk.s.own;
            const bool begins = walk.b0 == 0, ends = walk.b0 + walk.n == walk.steps;
            if (t == 1 && n_f <= T4_ROWS) {
                // No rows for these warps. They go no further than two segments ahead of the other tile: arrivals of a later segment would count as ones of this phase.
                if (seg >= 2) mbar_wait_warp(&seg_done[seg & 1], ((seg >> 1) - 1) & 1, t4_error, 0xc000fu, (unsigned)seg);
                if (lane == 0) mbar_arrive(&seg_done[seg & 1]);
                continue;
            }
            // ---- the warp's 32 queries, into 128-byte-swizzled rows (rows past the end: zeros): neighbouring lanes have neighbouring pieces of a row
            const int f0 = walk.seg_f0 + t * T4_ROWS + (warp & 3) * 32, f = f0 + lane;
            const bool in = f < M;
            const int i_mine = in ? a4_row(a, f) : 0, head = walk.seg_kvh * G + (in ? f - i_mine * G : 0), r = r0 + i_mine;
            const int lim = in ? min(walk.s.limit(i_mine), own) : 0;
            const size_t q_mine = (size_t)r * a.q_row + (size_t)head * a.q_head;
            constexpr int LANES = D / 8, ROWS = 32 / LANES, BATCH = 8;      // lanes a row, rows at once
#pragma unroll
            for (int i0 = 0; i0 < 32; i0 += BATCH * ROWS) {
                uint4 v[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; b++) {
                    const int from = i0 + b * ROWS + lane / LANES;
                    const uint16_t* q = (const uint16_t*)a.q + __shfl_sync(0xffffffffu, q_mine, from) + lane % LANES * 8;
                    v[b] = make_uint4(0, 0, 0, 0);
                    if (f0 + from >= M) continue;
                    if (((uintptr_t)q & 15) == 0) v[b] = *reinterpret_cast<const uint4*>(q);
                    else v[b] = make_uint4(q[0] | (uint32_t)q[1] << 16, q[2] | (uint32_t)q[3] << 16, q[4] | (uint32_t)q[5] << 16, q[6] | (uint32_t)q[7] << 16);
                }
#pragma unroll
                for (int b = 0; b < BATCH; b++) {
                    const int c8 = lane % LANES, row = (warp & 3) * 32 + i0 + b * ROWS + lane / LANES;
                    // (in the order of the keys' codes: 0, 4, 1, 5, ...)
                    *reinterpret_cast<uint4*>(qs + (t * PARTS + (c8 >> 3)) * T4_PART + row * 128 + (((c8 & 7) ^ (row & 7)) << 4)) =
                        make_uint4(__byte_perm(v[b].x, v[b].z, 0x5410), __byte_perm(v[b].x, v[b].z, 0x7632), __byte_perm(v[b].y, v[b].w, 0x5410), __byte_perm(v[b].y, v[b].w, 0x7632));
                }
            }
            fence_proxy_async();
            mbar_arrive(&q_full[t]);
            float m_ref = -INFINITY;
            uint64_t l2 = f2_pack(0.f, 0.f), l3 = l2;            // sums of even and odd entries, twice
            // Weights are held 2^7 times as large in f16, 2^15 at most (the reference lags by 2^8): the smallest f16 number is then 2^-31 of the weight at the reference, and many small ones that
            // count in the divisor count above it too. Sums and outputs have the same factor.
            constexpr float UP = F16 ? 7.f : 0.f;
            const uint64_t scale2 = f2_pack(a.scale_log2, a.scale_log2), up2 = f2_pack(UP, UP);
            for (int i = 0; i < walk.n; i++, done++) {
                mbar_wait(&s_full[t], done & 1, t4_error, 0xc0006u, done);
                tc_after_sync();
                __syncwarp();
                const int valid = lim - (walk.b0 + i) * T4_K;
                // 32 scores at a time, the next ones on their way: the maximum, then the exponentials
                uint32_t x[2][32];
                const bool partly = __any_sync(0xffffffffu, valid < T4_K);
                auto mask = [&](uint32_t (&v)[32], int left) {
                    if (partly) {
#pragma unroll
                        for (int j = 0; j < 32; j++) if (j >= left) v[j] = 0xff800000u;
                    }
                };
                float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tc_ld32(s_mine, x[0]);
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        tc_wait_ld(x[u]);
                        tc_ld32(s_mine + ((c + u + 1) & 3) * 32, x[u ^ 1]);      // (the last of these: the first scores again)
                        mask(x[u], valid - (c + u) * 32);
#pragma unroll
                        for (int j = 0; j < 32; j += 2) mx4[j >> 1 & 3] = fmaxf(fmaxf(mx4[j >> 1 & 3], __uint_as_float(x[u][j])), __uint_as_float(x[u][j + 1]));
                    }
                }
                const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
                const bool grow = (mx - m_ref) * a.scale_log2 > 8.f;      // (-inf less itself: no)
                float fall = 1.f;
                if (grow) {
                    fall = t4_exp2((m_ref - mx) * a.scale_log2);      // (0 the first time)
                    m_ref = mx;
                    const uint64_t fall2 = f2_pack(fall, fall);
                    l2 = f2_mul(l2, fall2); l3 = f2_mul(l3, fall2);
                }
                const float ref = m_ref > -INFINITY ? -m_ref : 0.f;
                const uint64_t ref2 = f2_pack(ref, ref);
                if (i > 0 && __any_sync(0xffffffffu, grow)) {    // the products so far must be in before they are rescaled
                    tc_wait_ld(x[0]);
                    mbar_wait(&pv_done[t], (done - 1) & 1, t4_error, 0xc0007u, done);
                    tc_after_sync();
                    __syncwarp();
                    for (int c = 0; c < D; c += 16) {
                        float o[16];
                        tc_ld16(o_mine + c, o);
#pragma unroll
                        for (int e = 0; e < 16; e++) o[e] *= fall;
                        tc_st16(o_mine + c, o);
                    }
                }
#pragma unroll 1
                for (int c = 0; c < 4; c += 2) {
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        tc_wait_ld(x[u]);
                        if (c + u < 3) tc_ld32(s_mine + (c + u + 1) * 32, x[u ^ 1]);
                        mask(x[u], valid - (c + u) * 32);
                        uint32_t p[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float2 d = f2_unpack(f2_fma(f2_add(f2_pack(__uint_as_float(x[u][j]), __uint_as_float(x[u][j + 1])), ref2), scale2, up2));
                            const float e0 = t4_exp2(d.x), e1 = t4_exp2(d.y);
                            if (j & 2) l3 = f2_add(l3, f2_pack(e0, e1)); else l2 = f2_add(l2, f2_pack(e0, e1));
                            p[j >> 1] = t4_pack<F16>(e0, e1);
                        }
                        tc_st16(s_mine + (c + u) * 16, p);       // over scores that have been read
                    }
                    tc_wait_st();
                    tc_before_sync();
                    mbar_arrive(c == 0 ? &p_half[t] : &p_full[t]);
                }
            }
            // ---- this segment's results of the row: output, or a part of it
            mbar_wait(&pv_done[t], (done - 1) & 1, t4_error, 0xc0008u, done);
            tc_after_sync();
            __syncwarp();
            const float2 la = f2_unpack(l2), lb = f2_unpack(l3);
            const float l = (la.x + la.y) + (lb.x + lb.y);
            const bool whole = begins && ends;
            const float scaled = m_ref * a.scale_log2, rest = t4_exp2(a4_rest(m_ref, a.scale_log2, scaled)), by = !whole ? rest : l == 0.f ? 0.f : 1.f / l;      // (0: no keys. A NaN stays one.)
            const int slot = begins ? 1 : 0;
            float* part = a.work + ((size_t)blockIdx.x * 2 + slot) * PART;
            // 32 columns at a time through the part of shared memory that held the warp's queries (nothing reads them any more), so that a row's columns leave side by side
            uint8_t* mine = qs + t * PARTS * T4_PART + (warp & 3) * 32 * 128;
#pragma unroll 1
            for (int g = 0; g < NG; g++) {
                uint32_t o[32];
                __syncwarp();
                tc_ld32(o_mine + g * 32, o);
                tc_wait_ld();
                const bool none = lim > first_bad[seg & 1][g];   // a value that the row sees is no number
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    const int f = (e & ~7) + (e >> 2 & 1);       // columns are in the order of the codes
                    float4 v = make_float4(__uint_as_float(o[f]) * by, __uint_as_float(o[f + 2]) * by, __uint_as_float(o[f + 4]) * by, __uint_as_float(o[f + 6]) * by);
                    if (l == 0.f) v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (none) v = make_float4(NAN, NAN, NAN, NAN);
                    *reinterpret_cast<float4*>(mine + lane * 128 + (((e >> 2) ^ (lane & 7)) << 4)) = v;
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int row = i * 4 + (lane >> 3), d = g * 32 + (lane & 7) * 4, to_r = __shfl_sync(0xffffffffu, r, row), to_h = __shfl_sync(0xffffffffu, head, row);
                    const float4 v = *reinterpret_cast<const float4*>(mine + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
                    if (f0 + row >= M) continue;
                    if (whole) a4_store_out(a, to_r, to_h, d, v.x, v.y, v.z, v.w);
                    else *reinterpret_cast<float4*>(part + (size_t)(t * T4_ROWS + (warp & 3) * 32 + row) * D + d) = v;
                }
            }
            if (!whole) {
                open[slot] = true;
                if (in) *reinterpret_cast<float2*>(part + 2 * T4_ROWS * D + (t * T4_ROWS + (warp & 3) * 32 + lane) * 2) = make_float2(scaled, l * rest);
                if (t == 0 && warp == 0 && lane == 0) {
                    const long last = given + walk.steps - walk.b0 - 1, run = run_shared[0], longer = run_shared[1], most = longer * (run + 1);
                    desc[slot] = {n_f, r0, walk.seg_f0, walk.seg_kvh, (int)(last < most ? last / (run + 1) : longer + (last - most) / run)};
                }
            }
            tc_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_done[seg & 1]);
        }
        if (warp == 0 && lane < 2 && !open[lane]) desc[lane].rows = 0;      // (whatever the workspace held)
    }
    __syncthreads();
    if (warp == 17) tc_dealloc(tmem_at, 512);
}

// ---------------------------------------------------------------- host side
template <int D, bool F16>
static cudaError_t t4_launch(const Attention4Args& a, cudaStream_t s) {
    constexpr int parts = D / 64, smem = (2 * parts + 2 * t4_stages(D) * 2 * parts) * T4_PART + T4_RAW * T4_K / Q4_TOKENS * q4_block(D) + 1024;
    static_assert(smem <= 227 * 1024 - 1024, "shared memory");
    if (!allow_smem<attention_4bit_tc_kernel<D, F16>>(smem)) return cudaErrorInvalidValue;
    cudaError_t e = launch_chain(attention_4bit_tc_kernel<D, F16>, dim3(T4_SMS), dim3(T4_THREADS), smem, s, a);
    return e != cudaSuccess ? e : attention_4bit_join(a, T4_SMS, 2 * T4_ROWS, s);
}
size_t attention_4bit_tc_work_bytes(int head_dim) { return (size_t)T4_SMS * 2 * (2 * T4_ROWS * (head_dim + 2) * 4 + sizeof(A4Desc)); }
cudaError_t attention_4bit_tc_launch(const Attention4Args& a, cudaStream_t s) {
    if (a.head_dim == 64) return a.type == ELEM_F16 ? t4_launch<64, true>(a, s) : t4_launch<64, false>(a, s);
    return a.type == ELEM_F16 ? t4_launch<128, true>(a, s) : t4_launch<128, false>(a, s);
}
namespace { __global__ void t4_give_up_kernel(unsigned int code) { mbar_give_up(0, t4_error, code, 0); } }
cudaError_t attention_4bit_tc_give_up(unsigned int code, cudaStream_t s) { return launch_chain(t4_give_up_kernel, dim3(1), dim3(1), 0, s, code); }
cudaError_t attention_4bit_tc_error(unsigned int* code) { return take_error_word(t4_error, code); }

}  // namespace b2

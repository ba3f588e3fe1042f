// Attention of a ragged batch over a paged cache in 4 bits (kv_4bit.cuh).
//   keys of row i of a sequence with n rows and c tokens: tokens 0 .. c - n + i;   out = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale log2(e) q.k_j. No key: 0.
// Bound by the bytes of the cache (9/16 of a byte an entry) and, close behind, by the instructions that turn codes into operands.
//
// A warp works by itself: it has its own ring of steps of 32 keys, its own copies, and keeps the weighted sums of all dims. The steps of all (sequence, KV head, tile of rows)
// laid end to end are cut into equal runs, one a warp; a run that begins or ends inside such a segment leaves a partial result (maximum, sum, weighted sum, 32 bits) there.
// The CTA's warps join theirs through shared memory at the end, a small kernel joins those of several CTAs. All joins have an order that the call's sizes and lengths give, so that the same
// call has the same bits.
//
// Products are transposed, keys (dims) times rows, so that eight rows fill an instruction: mma.sync m16n8k16.
//   scores: the operand of the keys is the codes c themselves as the subnormal f16 numbers c 2^-24 (c 2^-20 for every other one, where the query's entry is 1/16 of itself): a mask
//     and nothing else. Queries are held in f16 at a power of two that puts a row's largest entry near 2^10; the code's offset of 8 is the sum's initial value, -8 2^-24 sum q
//     over the group, and the group's scale multiplies the group's sum in 32 bits. No key is rounded.
//   weighted sums: the operand of the values is again their codes alone, c 2^-24 and c 2^-20. A probability times the scale of its key's value, group by group, is the other, rounded
//     to f16 once (2^-11), whatever the type of queries and output; the offset of 8 is a product of that operand and a constant. Scales are taken at a power of two that keeps the
//     operand in f16's range, found from the scales as they come. Score fragments become operands by movmatrix.
// The reference of a row's exponentials moves only where a score exceeds it by 2^6. It is a score before it is scaled, so that the largest one's difference is exact however large it is (one
// fused multiply-add with a scaled reference would save an instruction a score, and be off by as much as the reference's last place). Partial results have a scaled one, and what it is off by
// in their sums (a4_rest).
// Measured (32 heads over 8 of 128, f16): 256 chats of 16 to 4100 tokens 141 us, 4.4 TB/s of what has to be read, 0.66 of a copy's; 32 chats of 20 to 1500 16.5, one of 32000 18.6, of 700 8.5. A step is
// some 600 instructions, issued one in two cycles by the twelve warps that fit an SM: those of unpacking (160) and of the values' weights (100) are the most. More CTAs than fit were a fifth slower, four an
// SM with 128 registers a tenth, the next step's scores beside this one's values a tenth; products in other orders were the same, and so were larger shares for the CTAs that an SM serves first. A call
// begins with 2 us of finding a warp's place and 1 of its queries, beside the copies.
#include "attention_4bit.cuh"
#include "kv_4bit.cuh"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <float.h>
#include <math.h>
#include <type_traits>

namespace b2 {

namespace {
constexpr int A4_WARPS = 4, A4_THREADS = 32 * A4_WARPS;
constexpr int A4_BLOCKS = 2, A4_KEYS = A4_BLOCKS * Q4_TOKENS;      // blocks and keys of a step
constexpr int A4_STAGES = 2;         // steps under way
constexpr int A4_BEGIN = 2;          // units that a segment's beginning and end count as, beside its steps
constexpr int A4_SMS = 148;
// The join's CTAs. 148 tiles of 256 rows, us: a row a CTA 41 (CTAs start one in 1.1 ns), 16 rows 4. Tiles of 8 and 16 rows, a call of (8 sequences, 12 rows a KV head) and (1, 16, 20000 tokens): 1 row a
// CTA of 128 threads 19.4 and 18, 4 rows 16.3 and 18.0, 16 of 512 16.4 and 18.8; (1, 4, 4000 tokens) and (32, 4, 500): 1 row of 128 threads 13.1 and 18.1, 2 of 256 12.7 and 17.3.
constexpr int a4_join_threads(int mt) { return mt == 8 ? 256 : mt == 16 ? 128 : 512; }
constexpr int a4_join_rows(int mt) { return mt == 8 ? 2 : mt == 16 ? 4 : 16; }

__device__ unsigned int a4_error[5];                             // see mbar_give_up

__device__ __forceinline__ float a4_exp2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ __half2 a4_as_half2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ void a4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same, from other initial values
__device__ __forceinline__ void a4_mma_from(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}
__device__ __forceinline__ uint32_t a4_transpose(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// by one lane of the warp: keys and values to two places, told to the barrier (`EXPECT`: with all the bytes that it is to wait for); every operand the same in all lanes
template <bool EXPECT>
__device__ __forceinline__ void a4_copy(uint32_t bar, uint32_t all, uint32_t to_k, uint32_t to_v, const void* k, const void* v, uint32_t bytes) {
    if constexpr (EXPECT)
        asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t"
                     "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%2], [%4], %6, [%0];\n\t"
                     "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%3], [%5], %6, [%0];\n\t}"
                     ::"r"(bar), "r"(all), "r"(to_k), "r"(to_v), "l"(k), "l"(v), "r"(bytes) : "memory");
    else
        asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%1], [%3], %5, [%0];\n\t"
                     "@e cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%2], [%4], %5, [%0];\n\t}"
                     ::"r"(bar), "r"(to_k), "r"(to_v), "l"(k), "l"(v), "r"(bytes) : "memory");
}
__device__ __forceinline__ void a4_no_copy(uint32_t bar) {
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar) : "memory");
}
// chunks of a block's row: 16 bytes for heads of 128, 8 for heads of 64
template <int NG> __device__ __forceinline__ void a4_chunk(const uint8_t* p, uint32_t (&w)[NG]) {
    if constexpr (NG == 4) { const uint4 v = *reinterpret_cast<const uint4*>(p); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
}

// a token's scales, two a word
template <int NG> __device__ __forceinline__ void a4_scale_words(const uint8_t* p, uint32_t (&w)[NG / 2]) {
    if constexpr (NG == 4) { const uint2 v = *reinterpret_cast<const uint2*>(p); w[0] = v.x; w[1] = v.y; }
    else w[0] = *reinterpret_cast<const uint32_t*>(p);
}
template <int NG> __device__ __forceinline__ void a4_scales(const uint8_t* p, float (&s)[NG]) {
    uint32_t w[NG / 2];
    a4_scale_words<NG>(p, w);
#pragma unroll
    for (int gi = 0; gi < NG; gi += 2) {
        const float2 v = __half22float2(a4_as_half2(w[gi >> 1]));
        s[gi] = v.x; s[gi + 1] = v.y;
    }
}

// what is known of a sequence: its first row, its rows (those that are computed), its tokens, the keys that its first row sees, tiles of rows, steps
struct A4Seq {
    int r0, n, own, lim0, tiles, steps;
    __device__ A4Seq() {}
    __device__ A4Seq(const Attention4Args& a, int z, int mt) : A4Seq(a, a.r.row_start[z], a.r.row_start[z + 1], a.r.lengths[z], mt) {}
    __device__ A4Seq(const Attention4Args& a, int b, int e, int held, int mt) {
        r0 = min(max(b, 0), a.r.n_rows);
        const int all = max(min(max(e, 0), a.r.n_rows) - r0, 0);                         // (whatever the arrays hold)
        n = min(all, a.max_rows);
        own = min(max(held, 0), a.r.max_pages * a.r.block_tokens);
        lim0 = own - all + 1;
        tiles = (n * a.group + mt - 1) / mt;
        steps = n ? max(1, (own + A4_KEYS - 1) / A4_KEYS) : 0;
    }
    __device__ long units(int n_kv) const { return steps ? (long)(n_kv * tiles) * (steps + A4_BEGIN) : 0; }
    __device__ int limit(int i) const { return max(0, lim0 + i); }                      // keys that row i sees
};
// a place in the steps of all segments laid end to end, each behind its beginning's units
struct A4At {
    int z, kvh, tile, step;
    A4Seq s;
    // to the next segment
    __device__ void next(const Attention4Args& a, int mt) {
        step = 0;
        if (++tile < s.tiles) return;
        tile = 0;
        if (++kvh < a.n_kv) return;
        kvh = 0;
        do { if (++z >= a.r.n_seqs) return; s = A4Seq(a, z, mt); } while (s.steps == 0);
    }
};

// x / y for quotients below 2^20: an approximate one is off by at most one
__device__ __forceinline__ int a4_quotient(int x, int y) {
    const int q = (int)__fdividef((float)x, (float)y), r = x - q * y;
    return q + (r >= y) - (r < 0);
}

// All units cut into equal runs, one a warp (the first have a unit more). T: of numbers of units, int where all fit (64-bit products and quotients take a hundred instructions).
template <typename T>
struct A4Cut {
    T run, longer;                                               // units of a run, runs that have one more
    __device__ static T over(T x, T y) {
        if constexpr (sizeof(T) == 4) return a4_quotient(x, y);
        else return x / y;
    }
    __device__ A4Cut(T total, int warps) : run(over(total, warps)), longer(total - run * warps) {}
    __device__ T at(int i) const { return run * i + min((T)i, longer); }      // first unit of run i
    __device__ int owner(T u) const {                            // the run that has a unit
        const T most = longer * (run + 1);
        return (int)(u < most ? over(u, run + 1) : longer + over(u - most, run));
    }
};

// partial results in 32 bits: [rows of a tile][D] weighted sums, then [rows][2] (reference in log2, sum), see a4_rest
template <int D> __host__ __device__ constexpr int a4_part(int mt) { return mt * (D + 2); }

// results of the same row over different keys, added up
struct A4Sum {
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void most(float ref) { m = fmaxf(m, ref); }
    __device__ __forceinline__ float base() const { return m == -INFINITY ? 0.f : m; }
    __device__ __forceinline__ void fall(float before) {
        const float c = a4_exp2(before - base());
        l *= c; v.x *= c; v.y *= c; v.z *= c; v.w *= c;
    }
    __device__ __forceinline__ void add(float2 ml, float4 x) {
        const float c = a4_exp2(ml.x - base());
        l = fmaf(c, ml.y, l);
        v.x = fmaf(c, x.x, v.x); v.y = fmaf(c, x.y, v.y); v.z = fmaf(c, x.z, v.z); v.w = fmaf(c, x.w, v.w);
    }
    __device__ __forceinline__ void out(const Attention4Args& a, int t, int head, int d) const {
        const float inv = l == 0.f ? 0.f : 1.f / l;              // (0: no keys. A NaN stays one.)
        a4_store_out(a, t, head, d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
    }
};

constexpr int a4_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr int A4_MOST_CTAS = A4_SMS * 3;      // CTAs that run at once (of tiles of 8 and of 16 rows)
// units of work that a call can have at most
inline double a4_most_units(const Attention4Args& a, int mt) {
    const long steps = ((long)a.r.max_pages * a.r.block_tokens + A4_KEYS - 1) / A4_KEYS;
    return (double)a.r.n_seqs * a.n_kv * (((double)a.max_rows * (a.n_head / a.n_kv) + mt - 1) / mt) * (steps + A4_BEGIN);
}
}  // namespace

template <int D, int NT>
__global__ void __launch_bounds__(A4_THREADS, a4_per_sm(NT)) attention_4bit_step_kernel(const Attention4Args a) {
    constexpr int NG = D / Q4_GROUP, BLOCK = q4_block(D), KB = A4_BLOCKS, STAGE = 2 * KB * BLOCK, S = A4_STAGES, MT = 8 * NT, PART = a4_part<D>(MT);
    constexpr int REGION = S * STAGE > PART * 4 ? S * STAGE : PART * 4;
    extern __shared__ __align__(128) uint8_t a4_raw[];
    __shared__ uint64_t full[A4_WARPS][S];
    struct Held { int rows, r0, f0, kvh, ends, last; };          // rows 0: no result; `last`: the CTA where a segment that begins here ends
    __shared__ Held held[A4_WARPS][2];                           // of segments that began before the warp's run, and that go on behind it
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, tq = lane & 3;
    uint8_t* ring = a4_raw + warp * REGION;                      // behind the last step: the result of a segment that goes on
    float* const head_part = reinterpret_cast<float*>(a4_raw + A4_WARPS * REGION);      // [warp] results of segments that began before
    if (lane == 0) {
        for (int i = 0; i < S; i++) mbar_init(&full[warp][i], 1);
        held[warp][0].rows = held[warp][1].rows = 0;
        fence_mbar_init();
    }
    griddep_wait();
    griddep_launch();
    __syncwarp();
    const int n_kv = a.n_kv, G = a.group, blocks = a.r.block_tokens / Q4_TOKENS, last_page = (int)a.r.n_pages - 1;

    // ---- the units of all sequences, and this warp's run [u0, u1) of them. Up to 1024 sequences are read once a CTA and kept, the first 64 as they are.
    // (1000 of 200 tokens 90 us; read by every warp 97.)
    constexpr int KEPT = 1024, KEPT_WHOLE = 64;
    __shared__ int kept_units[KEPT];
    __shared__ A4Seq kept[KEPT_WHOLE];
    const int n_seqs = a.r.n_seqs;
    long total = 0;
    const bool keep = n_seqs <= KEPT && a.few_units;
    if (keep) {
        for (int z = threadIdx.x; z < n_seqs; z += A4_THREADS) {
            const A4Seq s(a, z, MT);
            kept_units[z] = (int)s.units(n_kv);
            if (z < KEPT_WHOLE) kept[z] = s;
        }
        __syncthreads();
        int sum = 0;
        for (int z = lane; z < n_seqs; z += 32) sum += kept_units[z];
        total = __reduce_add_sync(0xffffffffu, (unsigned)sum);
    } else {
        for (int z = lane; z < n_seqs; z += 32) total += A4Seq(a, z, MT).units(n_kv);
#pragma unroll
        for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
    }
    const int all_warps = gridDim.x * A4_WARPS, warps = (int)min((long)all_warps, total), me = blockIdx.x * A4_WARPS + warp;
    long u0 = 0, u1 = 0;
    if (me < warps) {
        auto run = [&](auto zero) {
            const A4Cut<decltype(zero)> cut((decltype(zero))total, warps);
            u0 = cut.at(me); u1 = cut.at(me + 1);
        };
        if (a.few_units) run(0);
        else run(0l);
    }
    __shared__ A4At places[A4_WARPS][2];                         // where the warp is, and where its copies are (few registers: they change once a segment)
    A4At& at = places[warp][0];
    A4At& ahead = places[warp][1];
    A4At start;
    start.z = n_seqs; start.kvh = start.tile = start.step = start.s.own = start.s.steps = start.s.tiles = 0;
    long first = u0;                                             // the first unit that is a step
    if (u0 < u1) {
        long rest = 0;
        if (keep) {
            int before = 0;
            for (int z0 = 0; z0 < n_seqs; z0 += 32) {
                const int mine = z0 + lane < n_seqs ? kept_units[z0 + lane] : 0;
                int sum = mine;                                  // of sequences z0 .. z0 + lane
#pragma unroll
                for (int o = 1; o < 32; o *= 2) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
                const unsigned past = __ballot_sync(0xffffffffu, before + sum > (int)u0);
                if (past) {
                    const int l = __ffs(past) - 1;
                    start.z = z0 + l;
                    start.s = start.z < KEPT_WHOLE ? kept[start.z] : A4Seq(a, start.z, MT);
                    rest = u0 - before - __shfl_sync(0xffffffffu, sum - mine, l);
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        } else {
            long before = 0;
            for (int z0 = 0; z0 < n_seqs; z0 += 32) {
                const long mine = z0 + lane < n_seqs ? A4Seq(a, z0 + lane, MT).units(n_kv) : 0;
                long sum = mine;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) { const long v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
                const unsigned past = __ballot_sync(0xffffffffu, before + sum > u0);
                if (past) {
                    const int l = __ffs(past) - 1;
                    start.z = z0 + l;
                    start.s = A4Seq(a, start.z, MT);
                    rest = u0 - before - __shfl_sync(0xffffffffu, sum - mine, l);
                    break;
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        const int each = start.s.steps + A4_BEGIN;
        if (a.few_units) {
            const int per = start.s.tiles * each;
            start.kvh = a4_quotient((int)rest, per);
            start.tile = a4_quotient((int)rest - start.kvh * per, each);
        } else {
            const long per = start.s.tiles * (long)each;
            start.kvh = (int)(rest / per);
            start.tile = (int)((rest - start.kvh * per) / each);
        }
        const int in = (int)(rest - ((long)start.kvh * start.s.tiles + start.tile) * each);
        first += max(A4_BEGIN - in, 0);
        start.step = max(in - A4_BEGIN, 0);
    }

    static_assert(KB == 2, "a page ends at most once in a step");
    // ---- copies: by one lane, a step's keys and its values (neighbours in their page; two copies each where a page ends between), the page's id read a step ahead. Everything they
    // need is the same in all lanes.
    if (lane == 0) { at = start; ahead = start; }
    int to_copy = (int)max(u1 - first, 0l), id = 0, id_2 = 0, in_page = 0, put = 0;      // units of the run from the next copy on; pages of the step's blocks
    int c_step = start.step, c_steps = start.s.steps, c_own = start.s.own;     // of the copies' segment
    const long per_head = (long)blocks * BLOCK, per_page = n_kv * per_head;
    long from_head = start.kvh * per_head;
    const int* table = a.r.pages + start.z * a.r.table_stride;
    // a segment's queries, on their way into the L1 cache
    auto fetch_queries = [&](const A4At& p) {
        const int f0 = p.tile * MT, row = lane >> 1;
        if (row >= min((long)MT, (long)p.s.n * G - f0)) return;
        const int f = f0 + row, i = a4_row(a, f);
        const uint16_t* q = (const uint16_t*)a.q + (size_t)(p.s.r0 + i) * a.q_row + (size_t)(p.kvh * G + f - i * G) * a.q_head + (lane & 1) * (D / 2);
        asm volatile("prefetch.global.L1 [%0];" ::"l"(q));
    };
    auto read_id = [&]() {
        const unsigned b = c_step * KB;                          // block of the sequence
        unsigned page = __umulhi(b, a.per_page);                 // the quotient by the page's blocks, or one less
        in_page = (int)(b - page * blocks);
        if (in_page >= blocks) { page++; in_page -= blocks; }
        if (to_copy <= 0 || (int)b * Q4_TOKENS >= c_own) return;
        id = table[page];
        if (in_page + 1 == blocks && (int)(b + 1) * Q4_TOKENS < c_own) id_2 = table[page + 1];
    };
    read_id();
    if (to_copy > 0) fetch_queries(start);
    __syncwarp();
    auto copy = [&]() {
        if (to_copy <= 0) return;
        const int n = min(KB, (c_own - c_step * A4_KEYS + Q4_TOKENS - 1) / Q4_TOKENS), here = in_page + 1 == blocks ? min(n, 1) : n;      // blocks, those of the first page
        const uint32_t bar = smem_u32(&full[warp][put]), to = smem_u32(ring + put * STAGE);
        if (n <= 0) a4_no_copy(bar);
        else {
            const long from = from_head + min(max(id, 0), last_page) * per_page + in_page * BLOCK;
            a4_copy<true>(bar, (uint32_t)(n * 2 * BLOCK), to, to + KB * BLOCK, (const uint8_t*)a.k_pool + from, (const uint8_t*)a.v_pool + from, (uint32_t)(here * BLOCK));
            if (here < n) {
                const long from_2 = from_head + min(max(id_2, 0), last_page) * per_page;
                a4_copy<false>(bar, 0, to + BLOCK, to + (KB + 1) * BLOCK, (const uint8_t*)a.k_pool + from_2, (const uint8_t*)a.v_pool + from_2, BLOCK);
            }
        }
        __syncwarp();
        put = put + 1 == S ? 0 : put + 1;
        to_copy--;
        if (++c_step == c_steps) {                               // the next segment
            to_copy -= A4_BEGIN;
            c_step = 0;
            if (lane == 0) ahead.next(a, MT);
            __syncwarp();
            c_steps = ahead.s.steps; c_own = ahead.s.own;
            from_head = ahead.kvh * per_head;
            table = a.r.pages + ahead.z * a.r.table_stride;
            if (to_copy > 0) fetch_queries(ahead);
            __syncwarp();
        }
        read_id();
    };
    for (int i = 0; i < S; i++) copy();

    // -8 2^-24 and -8 2^-20. Not as constants: fragments are neighbouring registers, and constants would be moved there anew for every product
    const uint32_t zero = (uint32_t)a.few_units >> 1, less[4] = {0x80088008u + zero, 0x80808080u + zero, 0x80088008u + 2 * zero, 0x80808080u + 2 * zero};
    // where a lane's chunks and scales lie in a step: key g of a block (the one 8 further on is turned alike), pair tq of the values
    const uint32_t k_from = (uint32_t)(g * (D / 2) + q4_key_chunk(D, g, tq) * NG * 4), k_scale = (uint32_t)q4_scale(D, g, 0);
    const uint32_t v_from = (uint32_t)(KB * BLOCK + tq * D + q4_value_chunk(D, tq, g) * NG * 4), v_scale = k_scale + KB * BLOCK;
    int st = 0;
    uint32_t parity = 0;
    for (long u = first; u < u1;) {
        // ================= a segment: queries, as the fragments of eight rows each; rows past the tile's are zeros
        const A4Seq s = at.s;
        const int kvh = at.kvh, f0 = at.tile * MT, n_f = (int)min((long)MT, (long)s.n * G - f0), r0 = s.r0;
        const long left = s.steps - at.step;
        const int n = (int)min(left, u1 - u), step0 = at.step;
        const bool begins = step0 == 0, ends = n == left;
        uint32_t qb[NT][NG][4];
        float off[NT][NG][4], by[NT][2];                         // of rows 2 tq and 2 tq + 1: the sums' initial values, and what a score is multiplied with
        int lim[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int f = f0 + nt * 8 + g;
            const bool in = nt * 8 + g < n_f;
            const int i = in ? a4_row(a, f) : 0;
            const size_t q_at = (size_t)(r0 + i) * a.q_row + (size_t)(kvh * G + (in ? f - i * G : 0)) * a.q_head + 8 * tq;
            const uint16_t* q = (const uint16_t*)a.q + q_at;
            uint4 raw[NG];
#pragma unroll
            for (int gi = 0; gi < NG; gi++) raw[gi] = make_uint4(0, 0, 0, 0);
            if (in && ((uintptr_t)q & 15) == 0) {
#pragma unroll
                for (int gi = 0; gi < NG; gi++) raw[gi] = *reinterpret_cast<const uint4*>(q + gi * Q4_GROUP);
            } else if (in) {
#pragma unroll
                for (int gi = 0; gi < NG; gi++) {
                    const uint16_t* p = q + gi * Q4_GROUP;
                    raw[gi] = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
                }
            }
            float value[NG][8], top = 0.f;
            auto as_floats = [&](auto f16) {
#pragma unroll
                for (int gi = 0; gi < NG; gi++)
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const uint32_t w = e < 2 ? raw[gi].x : e < 4 ? raw[gi].y : e < 6 ? raw[gi].z : raw[gi].w;
                        if constexpr (decltype(f16)::value) { const float2 v = __half22float2(a4_as_half2(w)); value[gi][e] = v.x; value[gi][e + 1] = v.y; }
                        else { value[gi][e] = __uint_as_float(w << 16); value[gi][e + 1] = __uint_as_float(w & 0xffff0000u); }
                    }
            };
            if (a.type == ELEM_F16) as_floats(std::true_type{});
            else as_floats(std::false_type{});
#pragma unroll
            for (int gi = 0; gi < NG; gi++)
#pragma unroll
                for (int e = 0; e < 8; e++) top = fmaxf(top, fabsf(value[gi][e]));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int ex = max((int)(__float_as_uint(top) >> 23) - 127, -100);
            const float up = __uint_as_float((uint32_t)(137 - ex) << 23);                // 2^(10 - ex)
            const int ex1 = (ex + 14) >> 1, ex2 = ex + 14 - ex1;                         // (2^24 of the codes, 2^(ex - 10) of the queries, in two steps: each is a normal number)
            // (held to the largest number: no difference times it then is still none, and any other one far past every exponent)
            const float mine = fminf(a.scale_log2 * __uint_as_float((uint32_t)(127 + ex1) << 23) * __uint_as_float((uint32_t)(127 + ex2) << 23), FLT_MAX);
#pragma unroll
            for (int j = 0; j < 2; j++) by[nt][j] = __shfl_sync(0xffffffffu, mine, (2 * tq + j) * 4);
#pragma unroll
            for (int gi = 0; gi < NG; gi++) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 4; e++) {                    // entries e and e + 4: the codes e and e + 4 of a word are masked out together
                    const float down = e & 1 ? 0.0625f : 1.f;
                    const uint32_t h = a4_half2(value[gi][e] * (up * down), value[gi][e + 4] * (up * down));
                    qb[nt][gi][e] = h;
                    const float2 back = __half22float2(a4_as_half2(h));
                    sum = fmaf(back.x + back.y, e & 1 ? 16.f : 1.f, sum);
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
                for (int e = 0; e < 4; e++) off[nt][gi][e] = __shfl_sync(0xffffffffu, sum, (2 * tq + (e & 1)) * 4 + (e >> 1)) * -0x1p-21f;      // 8 2^-24 (from different lanes, which have the same)
            }
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + 2 * tq + j;
                lim[nt][j] = row < n_f ? min(s.limit(a4_row(a, f0 + row)), s.own) : s.own;
            }
        }
        const int own = s.own, lim_lo = min(s.limit(a4_row(a, f0)), own);                       // keys that all rows of the tile see
        // weighted sums, 2^24 (even dims) and 2^20 (odd) times too small, and sums; both times 2^up_v, which goes down where a value's scale exceeds most_v, 2^(9 - up_v); references of the
        // exponentials
        float o[NT][NG][2][4], ref[NT][2], l[NT][2], up_v = 30.f, most_v = 0x1p-21f;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            ref[nt][0] = ref[nt][1] = -FLT_MAX; l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
            for (int gi = 0; gi < NG; gi++)
#pragma unroll
                for (int e = 0; e < 8; e++) o[nt][gi][e >> 2][e & 3] = 0.f;
        }

        // one step; `part`: not every row sees all of its keys
        auto step = [&](int t0, auto part) {
            constexpr bool PARTLY = decltype(part)::value;
            const uint8_t* stage = ring + st * STAGE;
            // ---- scores: keys g and g + 8 of a block, rows 2 tq and 2 tq + 1
            float sc[KB][NT][4];
#pragma unroll
            for (int b = 0; b < KB; b++) {
                uint32_t w[2][NG];
                float ks[2][NG];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    a4_chunk<NG>(stage + k_from + b * BLOCK + 8 * h * (D / 2), w[h]);
                    a4_scales<NG>(stage + k_scale + b * BLOCK + h * 8 * NG * 2, ks[h]);
                }
#pragma unroll
                for (int gi = 0; gi < NG; gi++) {
                    const uint32_t x = w[0][gi], y = w[1][gi], x8 = x >> 8, y8 = y >> 8;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float c[4];
                        a4_mma_from(c, off[nt][gi], x & 0x000f000fu, y & 0x000f000fu, x & 0x00f000f0u, y & 0x00f000f0u, qb[nt][gi][0], qb[nt][gi][1]);
                        a4_mma(c, x8 & 0x000f000fu, y8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x00f000f0u, qb[nt][gi][2], qb[nt][gi][3]);
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint64_t k2 = f2_pack(ks[h][gi], ks[h][gi]), c2 = f2_pack(c[2 * h], c[2 * h + 1]);
                            const float2 t = f2_unpack(gi ? f2_fma(k2, c2, f2_pack(sc[b][nt][2 * h], sc[b][nt][2 * h + 1])) : f2_mul(k2, c2));
                            sc[b][nt][2 * h] = t.x; sc[b][nt][2 * h + 1] = t.y;
                        }
                    }
                }
            }
            // ---- the largest of the values' scales
            __half2 most = a4_as_half2(0);                       // (read again below: few registers)
#pragma unroll
            for (int b = 0; b < KB; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint32_t two[NG / 2];
                    a4_scale_words<NG>(stage + v_scale + b * BLOCK + h * 8 * NG * 2, two);
#pragma unroll
                    for (int gi = 0; gi < NG; gi += 2) {
                        __half2 v = a4_as_half2(two[gi >> 1]);
                        if (PARTLY && t0 + b * 16 + g + 8 * h >= own) v = a4_as_half2(0);      // (whatever lies there)
                        most = __hmax2(most, __habs2(v));
                    }
                }
            const float2 most2 = __half22float2(most);
            const float top_v = fmaxf(most2.x, most2.y);
            // ---- differences to the references, which go up where a score is far above them (as the values' power of two goes down where a scale is)
            bool above = top_v > most_v;
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    float mx = -INFINITY;
#pragma unroll
                    for (int b = 0; b < KB; b++) {
                        if constexpr (PARTLY) {
#pragma unroll
                            for (int h = 0; h < 2; h++) if (t0 + b * 16 + g + 8 * h >= lim[nt][j]) sc[b][nt][j + 2 * h] = -INFINITY;
                        }
                        mx = fmaxf(fmaxf(mx, sc[b][nt][j]), sc[b][nt][j + 2]);
                    }
                    above |= (mx - ref[nt][j]) * by[nt][j] > 6.f;
                }
            if (__any_sync(0xffffffffu, above)) {
                float fall_v = 1.f;
                const float all_v = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top_v)));
                if (all_v > most_v) {
                    const int e = min((int)(__float_as_uint(all_v) >> 23) - 127, 16);    // all_v * 2^(6 - e) in [64, 128)
                    fall_v = a4_exp2(6 - e - up_v);
                    up_v = 6 - e;
                    most_v = __uint_as_float((uint32_t)(130 + e) << 23);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int j = 0; j < 2; j++) {
                        float mx = -INFINITY;
#pragma unroll
                        for (int b = 0; b < KB; b++) mx = fmaxf(fmaxf(mx, sc[b][nt][j]), sc[b][nt][j + 2]);
#pragma unroll
                        for (int d = 4; d < 32; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                        mx = fmaxf(mx, ref[nt][j]);
                        const float fall = a4_exp2((ref[nt][j] - mx) * by[nt][j]);
                        ref[nt][j] = mx;
                        l[nt][j] *= fall * fall_v;
#pragma unroll
                        for (int gi = 0; gi < NG; gi++)
#pragma unroll
                            for (int m = 0; m < 2; m++) { o[nt][gi][m][j] *= fall * fall_v; o[nt][gi][m][j + 2] *= fall * fall_v; }
                    }
            }
            // ---- probabilities; times the values' scales, as operands with keys in pairs; weighted sums: dims 32 gi + 4 g + 2 m and + 1
#pragma unroll
            for (int b = 0; b < KB; b++) {
                if (PARTLY && t0 + b * 16 >= own) break;
                float pr[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        pr[nt][e] = a4_exp2(fmaf(sc[b][nt][e] - ref[nt][e & 1], by[nt][e & 1], up_v));
                        l[nt][e & 1] += pr[nt][e];
                    }
                uint32_t w[2][NG];
                float vs[2][NG];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    a4_chunk<NG>(stage + v_from + b * BLOCK + 4 * h * D, w[h]);
                    a4_scales<NG>(stage + v_scale + b * BLOCK + h * 8 * NG * 2, vs[h]);
                }
#pragma unroll
                for (int gi = 0; gi < NG; gi++) {
                    const uint32_t x = w[0][gi], y = w[1][gi], x8 = x >> 8, y8 = y >> 8;
                    const float s0 = vs[0][gi], s1 = vs[1][gi];
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const float2 za = f2_unpack(f2_mul(f2_pack(pr[nt][0], pr[nt][1]), f2_pack(s0, s0))), zb = f2_unpack(f2_mul(f2_pack(pr[nt][2], pr[nt][3]), f2_pack(s1, s1)));
                        float z[4] = {za.x, za.y, zb.x, zb.y};
                        if constexpr (PARTLY) {                  // (a scale that is no number must not reach rows that do not see its key)
#pragma unroll
                            for (int e = 0; e < 4; e++) if (sc[b][nt][e] == -INFINITY) z[e] = 0.f;
                        }
                        const uint32_t b0 = a4_transpose(a4_half2(z[0], z[1])), b1 = a4_transpose(a4_half2(z[2], z[3]));
                        a4_mma(o[nt][gi][0], x & 0x000f000fu, x & 0x00f000f0u, y & 0x000f000fu, y & 0x00f000f0u, b0, b1);
                        a4_mma(o[nt][gi][1], x8 & 0x000f000fu, x8 & 0x00f000f0u, y8 & 0x000f000fu, y8 & 0x00f000f0u, b0, b1);
#pragma unroll
                        for (int m = 0; m < 2; m++) a4_mma(o[nt][gi][m], less[0], less[1], less[2], less[3], b0, b1);
                    }
                }
            }
        };
        for (int i = 0; i < n; i++) {
            const int t0 = (step0 + i) * A4_KEYS;
            mbar_wait_warp(&full[warp][st], parity, a4_error, 0xb0001u, (unsigned)i);
            if (t0 + A4_KEYS > lim_lo) step(t0, std::true_type{});
            else step(t0, std::false_type{});
            __syncwarp();                                        // the step's memory is free
            copy();
            if (++st == S) { st = 0; parity ^= 1; }
        }
        // the sums as they are, for the reference times `by` as it is rounded where they are a partial result's
        float scaled[NT][2], by_l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                scaled[nt][j] = ref[nt][j] * by[nt][j];
                by_l[nt][j] = a4_exp2(begins && ends ? -up_v : a4_rest(ref[nt][j], by[nt][j], scaled[nt][j]) - up_v);
            }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int gi = 0; gi < NG; gi++)
#pragma unroll
                for (int m = 0; m < 2; m++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[nt][gi][m][e] *= by_l[nt][e & 1] * (e & 2 ? 0x1p20f : 0x1p24f);
        u += n;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int d = 4; d < 32; d *= 2) l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], d);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) { l[nt][0] *= by_l[nt][0]; l[nt][1] *= by_l[nt][1]; }
        // ---- output, or a result for the joins
        const int slot = begins ? 1 : 0;
        float* part_at = begins ? reinterpret_cast<float*>(ring) : head_part + warp * PART;      // (a segment that goes on is the run's last: no copy is under way)
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const int row = nt * 8 + 2 * tq + j;
                if (row >= n_f) continue;
                if (begins && ends) {
                    const int f = f0 + row, i = a4_row(a, f);
                    const float inv = l[nt][j] == 0.f ? 0.f : 1.f / l[nt][j];            // (0: no keys. A NaN stays one.)
#pragma unroll
                    for (int gi = 0; gi < NG; gi++)
                        a4_store_out(a, r0 + i, kvh * G + f - i * G, gi * Q4_GROUP + 4 * g, o[nt][gi][0][j] * inv, o[nt][gi][0][j + 2] * inv, o[nt][gi][1][j] * inv,
                                     o[nt][gi][1][j + 2] * inv);
                } else {
#pragma unroll
                    for (int gi = 0; gi < NG; gi++)
                        *reinterpret_cast<float4*>(part_at + row * D + gi * Q4_GROUP + 4 * g) = make_float4(o[nt][gi][0][j], o[nt][gi][0][j + 2], o[nt][gi][1][j], o[nt][gi][1][j + 2]);
                    if (g == 0) *reinterpret_cast<float2*>(part_at + MT * D + row * 2) = make_float2(l[nt][j] == 0.f ? -INFINITY : scaled[nt][j], l[nt][j]);
                }
            }
        if (!(begins && ends) && lane == 0) {
            const long end = u - n + left - 1;                   // the segment's last unit
            auto owner = [&](auto zero) {
                using T = decltype(zero);
                return A4Cut<T>((T)total, warps).owner((T)end) / A4_WARPS;
            };
            held[warp][slot] = {n_f, r0, f0, kvh, ends ? 1 : 0, !begins ? 0 : a.few_units ? owner(0) : owner(0l)};
        }
        // the segment behind it (not the sequence's loads if there is none)
        u += A4_BEGIN;
        __syncwarp();
        if (u < u1 && lane == 0) at.next(a, MT);
        __syncwarp();
    }
    __syncthreads();

    // ================= what the CTA's warps have left, joined: from one warp's result on to where the segment ends. What an earlier CTA has begun, or a later one ends, goes to
    // the workspace.
    A4Desc* desc = a4_desc<PART>(a, gridDim.x) + blockIdx.x * 2;
    bool left_open[2] = {false, false};
    for (int w = 0; w < A4_WARPS; w++)
        for (int slot = w == 0 ? 0 : 1; slot < 2; slot++) {      // (slot 0 of a later warp: joined with what it goes on from)
            const Held h = held[w][slot];
            if (h.rows == 0) continue;
            int end = w;                                         // warps w .. end have results of this segment
            bool ends = h.ends;
            while (!ends && end + 1 < A4_WARPS) { end++; ends = held[end][0].ends; }
            auto part_of = [&](int v) { return v == w && slot == 1 ? reinterpret_cast<const float*>(a4_raw + v * REGION) : head_part + v * PART; };
            const bool finish = slot == 1 && ends;
            float* to = a.work + ((size_t)blockIdx.x * 2 + slot) * PART;
            for (int e = threadIdx.x; e < h.rows * (D / 4); e += A4_THREADS) {
                const int row = e / (D / 4), d = e % (D / 4) * 4;
                A4Sum sum;
                for (int v = w; v <= end; v++) sum.most(part_of(v)[MT * D + row * 2]);
                for (int v = w; v <= end; v++)
                    sum.add(*reinterpret_cast<const float2*>(part_of(v) + MT * D + row * 2), *reinterpret_cast<const float4*>(part_of(v) + row * D + d));
                if (finish) {
                    const int f = h.f0 + row, i = a4_row(a, f);
                    sum.out(a, h.r0 + i, h.kvh * G + f - i * G, d);
                } else {
                    *reinterpret_cast<float4*>(to + row * D + d) = sum.v;
                    if (d == 0) *reinterpret_cast<float2*>(to + MT * D + row * 2) = make_float2(sum.m, sum.l);
                }
            }
            if (!finish) {
                left_open[slot] = true;
                if (threadIdx.x == 0) desc[slot] = {h.rows, h.r0, h.f0, h.kvh, h.last};
            }
        }
    if (threadIdx.x < 2 && !left_open[threadIdx.x]) desc[threadIdx.x].rows = 0;      // (whatever the workspace held)
}

// The results of a segment that lies in several CTAs, from the one where it begins on: a CTA has up to 16 rows, a row the lanes of a warp (half of one for heads of 64), four dims each; where
// there are fewer rows, a row that many times, every so many-th of the segment's CTAs for each. (A row a CTA is bound by the start of CTAs, 1.1 ns each: 41 us for 148 tiles of 256 rows.)
template <int D, int MT>
__global__ void __launch_bounds__(a4_join_threads(MT), 1024 / a4_join_threads(MT)) attention_4bit_join_kernel(const Attention4Args a, const int ctas) {
    constexpr int PART = a4_part<D>(MT), LANES = D / 4, THREADS = a4_join_threads(MT), ROWS = a4_join_rows(MT), GROUPS = THREADS / LANES, B = MT > 16 ? 4 : 8;
    static_assert(ROWS <= GROUPS && MT % ROWS == 0, "lanes for every row of a CTA");
    __shared__ float4 sums[GROUPS][LANES];
    __shared__ float2 refs[GROUPS];
    const int c = blockIdx.x, row0 = blockIdx.y * ROWS, at = threadIdx.x / LANES, d = threadIdx.x % LANES * 4;
    griddep_wait();
    griddep_launch();
    const A4Desc h = a4_desc<PART>(a, ctas)[c * 2 + 1];
    const int rows = min(h.rows - row0, ROWS);
    if (rows <= 0) return;
    int per = GROUPS / ROWS;                                     // lanes of a row's dims: so many times, each for a share of the CTAs
    while (per * 2 * rows <= GROUPS) per *= 2;
    const int row = row0 + at / per, n = row < h.rows ? min(h.last, ctas - 1) - c + 1 : 0;
    A4Sum sum;
    for (int j0 = at % per; j0 < n; j0 += per * B) {
        float2 ml[B];
        float4 v[B];
#pragma unroll
        for (int j = 0; j < B; j++) {
            ml[j] = make_float2(-INFINITY, 0.f); v[j] = make_float4(0.f, 0.f, 0.f, 0.f);
            const int i = j0 + j * per;
            if (i >= n) continue;
            const float* from = a.work + ((size_t)(c + i) * 2 + (i == 0)) * PART;
            ml[j] = __ldcg(reinterpret_cast<const float2*>(from + MT * D + row * 2));
            v[j] = __ldcg(reinterpret_cast<const float4*>(from + row * D + d));
        }
        const float before = sum.m;
#pragma unroll
        for (int j = 0; j < B; j++) sum.most(ml[j].x);
        sum.fall(before);
#pragma unroll
        for (int j = 0; j < B; j++) sum.add(ml[j], v[j]);
    }
    A4Sum all = sum;
    if (per > 1) {
        sums[at][d / 4] = sum.v;
        if (d == 0) refs[at] = make_float2(sum.m, sum.l);
        __syncthreads();
        if (at % per) return;
        all = A4Sum();
        for (int j = at; j < at + per; j++) all.most(refs[j].x);
        for (int j = at; j < at + per; j++) all.add(refs[j], sums[j][d / 4]);
    }
    if (row >= h.rows) return;
    const int G = a.group, f = h.f0 + row, i = a4_row(a, f);
    all.out(a, h.r0 + i, h.kvh * G + f - i * G, d);
}

// ---------------------------------------------------------------- host side
namespace {
template <int D, int NT>
constexpr int a4_smem() {
    constexpr int ring = A4_STAGES * 2 * A4_BLOCKS * q4_block(D), part = a4_part<D>(8 * NT) * 4;
    return A4_WARPS * ((ring > part ? ring : part) + part);
}
template <int D, int MT>
cudaError_t a4_join(const Attention4Args& a, int ctas, cudaStream_t s) {
    return launch_chain(attention_4bit_join_kernel<D, MT>, dim3(ctas, MT / a4_join_rows(MT)), dim3(a4_join_threads(MT)), 0, s, a, ctas);
}
template <int D, int NT>
cudaError_t a4_step(Attention4Args a, cudaStream_t s) {
    constexpr int MT = 8 * NT, smem = a4_smem<D, NT>();
    if (!allow_smem<attention_4bit_step_kernel<D, NT>>(smem)) return cudaErrorInvalidValue;
    // as many CTAs as run at once, no more than there can be steps for
    const double units = a4_most_units(a, MT);
    const int ctas = (int)std::min<double>(A4_SMS * a4_per_sm(NT), std::ceil(units / A4_WARPS));
    a.few_units = units < 1e9 && a.n_kv < 1 << 20;               // (quotients: a4_quotient)
    const unsigned blocks = a.r.block_tokens / Q4_TOKENS;
    a.per_page = blocks == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / blocks);
    cudaError_t e = launch_chain(attention_4bit_step_kernel<D, NT>, dim3(ctas), dim3(A4_THREADS), smem, s, a);
    if (e != cudaSuccess) return e;
    return attention_4bit_join(a, ctas, MT, s);
}
}  // namespace

cudaError_t attention_4bit_join(const Attention4Args& a, int ctas, int rows, cudaStream_t s) {
    if (a.head_dim == 64) return rows == 8 ? a4_join<64, 8>(a, ctas, s) : rows == 16 ? a4_join<64, 16>(a, ctas, s) : a4_join<64, 256>(a, ctas, s);
    return rows == 8 ? a4_join<128, 8>(a, ctas, s) : rows == 16 ? a4_join<128, 16>(a, ctas, s) : a4_join<128, 256>(a, ctas, s);
}

namespace {
// Where no sequence may have more rows a KV head than this, this file's tiles of 16 rows; else the whole call on tensor memory, short sequences too (200 chats of 16 to 2000 tokens beside 512 rows behind
// 2000: 527 us, in two calls 141). us here and there (heads of 128, 8 KV heads): a sequence of 4000 tokens with 32 rows a KV head
// 17 and 23, 64 rows 18 and 24, 128 rows 24 and 25; 32 sequences of 1000 tokens with 32 rows 40 and 82, 64 rows 69 and 83, 68 rows 82 and 83, 256 rows 244 and 105.
constexpr long A4_TC_ROWS = 64;
bool a4_many(long rows, int n_head, int n_kv) { return rows * (n_head / n_kv) > A4_TC_ROWS; }
}  // namespace

size_t attention_4bit_work_bytes(long n_rows, int n_head, int n_kv, int head_dim) {
    const long rows = n_rows * (n_head / n_kv) <= 8 ? 8 : 16;
    const size_t step = (size_t)A4_MOST_CTAS * 2 * (rows * (head_dim + 2) * 4 + sizeof(A4Desc));
    return a4_many(n_rows, n_head, n_kv) ? std::max(step, attention_4bit_tc_work_bytes(head_dim)) : step;      // (all rows may be one sequence's)
}

cudaError_t attention_4bit_launch(const Attention4Args& args, cudaStream_t s) {
    Attention4Args a = args;
    if (a.r.n_rows == 0 || a.r.n_seqs == 0) return cudaSuccess;
    a.group = a.n_head / a.n_kv;
    a.per_group = a.group == 1 ? 0xffffffffu : (unsigned)((1ull << 32) / a.group);
    const DependentLaunch dependent;
    if (a4_many(a.max_rows, a.n_head, a.n_kv)) return attention_4bit_tc_launch(a, s);
    // tiles of 8 rows where all fit one, of 16 (with more registers and less running at once) where not: 4 rows a KV head in tiles of 8 and of 16, us: 32 sequences of 500 tokens 15.2 and 17.6,
    // 256 of 2000 138 and 206, one of 30000 18.4 and 24.2
    const bool few = (long)a.max_rows * (a.n_head / a.n_kv) <= 8;
    if (a.head_dim == 64) return few ? a4_step<64, 1>(a, s) : a4_step<64, 2>(a, s);
    return few ? a4_step<128, 1>(a, s) : a4_step<128, 2>(a, s);
}

namespace { __global__ void a4_give_up_kernel(unsigned int code) { mbar_give_up(0, a4_error, code, 0); } }
cudaError_t attention_4bit_give_up(unsigned int code, bool tensor_memory, cudaStream_t s) {
    return tensor_memory ? attention_4bit_tc_give_up(code, s) : launch_chain(a4_give_up_kernel, dim3(1), dim3(1), 0, s, code);
}
cudaError_t attention_4bit_error(unsigned int* code) {
    unsigned int more = 0;
    cudaError_t e = take_error_word(a4_error, code);
    if (e == cudaSuccess) e = attention_4bit_tc_error(&more);
    if (e == cudaSuccess && *code == 0) *code = more;
    return e;
}

}  // namespace b2

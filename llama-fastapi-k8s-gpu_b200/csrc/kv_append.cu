// Keys and values of new tokens into the paged cache, keys (and queries) rotated on the way.
//   angle = position * freq_i, the product and its reduction to a turn in 64 bits (at position 100000 a 32-bit product is off by up to 0.004 of a radian);
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos) for the entries 2i, 2i + 1 ("pairs") or i, i + rot_dims / 2 ("halves") below rot_dims, the others as
//   they are; one rounding to the cache's type at the end.
// The GGUF engine's own steps do this behind their projection (rope_store in prefill.cu, which also adds that product's K splits up); this one takes rows of any
// producer.
//
// Bound by memory: every entry is read once and written once. A CTA takes one row; a thread keeps one 16-byte piece of a head (both halves of a pair of pieces
// under "halves", so that q may be rotated in place) and has three heads at a time. Its loads are under way while the row's sequence, its page and the angles
// are found, a chain of two to three dependent reads; what hides that chain is other CTAs, so registers are few. Eight rows a CTA, which find all of that once, kept
// too few CTAs on an SM (16384 rows of 48 heads of 128: 107 us instead of 93 with five CTAs an SM). A row a CTA takes 70 us there in a graph, 5.75 TB/s, and 76 a call;
// 32 rows 4.0 and 10.1.
#include "device_ops.h"
#include "ptx.cuh"
#include <cuda_bf16.h>

namespace b2 {

namespace {
constexpr int KA_THREADS = 256;
constexpr int KA_MAX_PAIRS = 256;      // rot_dims <= 512

template <typename T> __device__ __forceinline__ float ka_float(T v);
template <> __device__ __forceinline__ float ka_float(float v) { return v; }
template <> __device__ __forceinline__ float ka_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float ka_float(__nv_bfloat16 v) { return __bfloat162float(v); }
// rounded in pairs: one instruction at full rate, where one entry goes through the unit of the transcendental functions
__device__ __forceinline__ void ka_round(float a, float b, __half& x, __half& y) { const __half2 v = __floats2half2_rn(a, b); x = __low2half(v); y = __high2half(v); }
__device__ __forceinline__ void ka_round(float a, float b, __nv_bfloat16& x, __nv_bfloat16& y) { const __nv_bfloat162 v = __floats2bfloat162_rn(a, b); x = __low2bfloat16(v); y = __high2bfloat16(v); }

// (two entries: as two loads, so that any row may start anywhere)
template <typename T, int VEC>
struct alignas(VEC == 8 ? 16 : sizeof(T)) Piece { T v[VEC]; };

}  // namespace

// blockDim.x = pieces of a head at once (`wide`) times heads at once
template <typename In, typename Out, int VEC, bool HALVES>
__global__ void __launch_bounds__(KA_THREADS, VEC == 8 && sizeof(In) * (HALVES ? 2 : 1) >= 4 ? 5 : 6) kv_append_kernel(const KvAppendArgs a, const int wide) {
    // heads that a thread has under way: about 16 registers
    constexpr int PER = HALVES ? 2 : 1, REGS = (int)sizeof(In) * VEC * PER / 4, UNROLL = VEC != 8 || REGS <= 4 ? 3 : REGS == 8 ? 2 : 1;
    extern __shared__ __align__(16) float2 ka_turn[];            // [rot_dims / 2]
    __shared__ long place;                                       // entry of the pools where KV head 0 of the row lies, or -1
    __shared__ long pos;                                         // position of the row
    __shared__ int live;                                         // the row belongs to a sequence
    using InPiece = Piece<In, VEC>;
    using OutPiece = Piece<Out, VEC>;
    const int tid = threadIdx.x, lane = tid & 31, n_threads = blockDim.x;
    const long row = blockIdx.x;
    const int D = a.head_dim, half = a.rot_dims >> 1, heads = 2 * a.n_kv + (a.q ? a.n_head : 0), at_once = n_threads / wide, h0 = tid / wide;
    // pieces of a head: two vectors half a rotation apart while they are rotated together, one otherwise
    const int turned = HALVES ? half / VEC : 0, pieces = turned + (D - turned * 2 * VEC) / VEC;
    bool ready = false;
    for (int p = tid % wide; p < pieces; p += wide) {            // (every thread has a first one)
        const bool two = HALVES && p < turned;
        const int d = two ? p * VEC : turned * 2 * VEC + (p - turned) * VEC;
        const bool rot = d < a.rot_dims;
        for (int hc = 0; hc < heads; hc += UNROLL * at_once) {
            InPiece x[UNROLL][PER];
            // key, value, query: 0, 1, 2, or 3: no head of this thread
            auto kind_of = [&](int h) { return h0 >= at_once || h >= heads ? 3 : h < a.n_kv ? 0 : h < 2 * a.n_kv ? 1 : 2; };
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int h = hc + h0 + u * at_once, kind = kind_of(h);
                if (kind == 3) continue;
                const In* from = (kind == 0 ? (const In*)a.k + row * a.k_row + h * a.k_head : kind == 1 ? (const In*)a.v + row * a.v_row + (h - a.n_kv) * a.v_head
                                                                                                     : (const In*)a.q + row * a.q_row + (h - 2 * a.n_kv) * a.q_head) + d;
                x[u][0] = *reinterpret_cast<const InPiece*>(from);
                if (two) x[u][PER - 1] = *reinterpret_cast<const InPiece*>(from + half);
            }
            if (!ready) {
                ready = true;
                if (tid < 32) {
                    int s, end = 0, held = 0, first;
                    if (a.r.n_seqs <= 32) {                      // all of it in one read
                        const bool one = lane < a.r.n_seqs;
                        const int e = one ? a.r.row_start[lane + 1] : 0, l = one ? a.r.lengths[lane] : 0;
                        first = a.r.row_start[0];
                        s = __popc(__ballot_sync(0xffffffffu, one && e <= row));
                        end = __shfl_sync(0xffffffffu, e, s & 31);
                        held = __shfl_sync(0xffffffffu, l, s & 31);
                    } else {
                        s = seq_of_row(a.r.row_start, a.r.n_seqs, (int)row, lane);
                        first = a.r.row_start[0];
                        if (s < a.r.n_seqs) { end = a.r.row_start[s + 1]; held = a.r.lengths[s]; }
                    }
                    if (lane == 0) {
                        const bool in = s < a.r.n_seqs && row >= first;
                        long where = -1, at = 0;
                        if (in) {
                            at = held - (end - row);
                            const long page_no = at >= 0 ? at / a.r.block_tokens : a.r.max_pages;
                            if (page_no < a.r.max_pages) {
                                const int page = a.r.pages[s * a.r.table_stride + page_no];
                                if (page >= 0 && page < a.r.n_pages) where = ((long)page * a.n_kv * a.r.block_tokens + at % a.r.block_tokens) * D;
                            }
                        }
                        place = where; live = in; pos = a.first_pos + at;
                    }
                }
                __syncthreads();
                for (int i = tid; i < half; i += n_threads) {
                    const double turns = (double)pos * (double)a.freqs[i] * 0.15915494309189533577;      // 1 / (2 pi)
                    float sn, cs;
                    sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
                    ka_turn[i] = make_float2(a.amplitude * cs, a.amplitude * sn);
                }
                __syncthreads();
                if (!live) return;                               // (all threads)
            }
            const float2* turn = ka_turn + (two ? d : d >> 1);
            const long where = place;
#pragma unroll
            for (int u = 0; u < UNROLL; u++) {
                const int h = hc + h0 + u * at_once, kind = kind_of(h);
                if (kind == 3 || (kind != 2 && where < 0)) continue;
                float z[2][VEC] = {};
#pragma unroll
                for (int e = 0; e < VEC; e++) {
                    z[0][e] = ka_float(x[u][0].v[e]);
                    if (two) z[1][e] = ka_float(x[u][PER - 1].v[e]);
                }
                if (rot && kind != 1) {
                    if constexpr (VEC == 8) {                    // cosines and sines 16 bytes at a time (halves of a rotation are multiples of 4 or 8 pairs)
#pragma unroll
                        for (int i = 0; i < VEC / 2; i++) {
                            if (two) {
                                const float4 c = *reinterpret_cast<const float4*>(turn + 2 * i);
                                const float v0 = z[0][2 * i], v1 = z[1][2 * i], v2 = z[0][2 * i + 1], v3 = z[1][2 * i + 1];
                                z[0][2 * i] = v0 * c.x - v1 * c.y; z[1][2 * i] = v0 * c.y + v1 * c.x;
                                z[0][2 * i + 1] = v2 * c.z - v3 * c.w; z[1][2 * i + 1] = v2 * c.w + v3 * c.z;
                            } else if (i < VEC / 4) {
                                const float4 c = *reinterpret_cast<const float4*>(turn + 2 * i);
                                const float v0 = z[0][4 * i], v1 = z[0][4 * i + 1], v2 = z[0][4 * i + 2], v3 = z[0][4 * i + 3];
                                z[0][4 * i] = v0 * c.x - v1 * c.y; z[0][4 * i + 1] = v0 * c.y + v1 * c.x;
                                z[0][4 * i + 2] = v2 * c.z - v3 * c.w; z[0][4 * i + 3] = v2 * c.w + v3 * c.z;
                            }
                        }
                    } else {
                        const float2 c = turn[0];
                        float& other = HALVES ? z[1][0] : z[0][VEC - 1];
                        const float v0 = z[0][0], v1 = other;
                        z[0][0] = v0 * c.x - v1 * c.y; other = v0 * c.y + v1 * c.x;
                    }
                }
                OutPiece y[2];
                if constexpr (VEC == 1) {
                    ka_round(z[0][0], z[1][0], y[0].v[0], y[1].v[0]);
                } else {
#pragma unroll
                    for (int e = 0; e < VEC; e += 2) {
                        ka_round(z[0][e], z[0][e + 1], y[0].v[e], y[0].v[e + 1]);
                        if (two) ka_round(z[1][e], z[1][e + 1], y[1].v[e], y[1].v[e + 1]);
                    }
                }
                Out* to = kind == 2 ? (Out*)a.q_out + row * a.qo_row + (h - 2 * a.n_kv) * a.qo_head
                                    : (kind == 0 ? (Out*)a.k_pool : (Out*)a.v_pool) + where + (long)(kind == 0 ? h : h - a.n_kv) * a.r.block_tokens * D;
                *reinterpret_cast<OutPiece*>(to + d) = y[0];
                if (two) *reinterpret_cast<OutPiece*>(to + d + half) = y[1];
            }
        }
    }
}

template <typename In, typename Out, int VEC, bool HALVES>
static cudaError_t kv_append_rows(const KvAppendArgs& a, cudaStream_t s) {
    const int turned = HALVES ? a.rot_dims / 2 / VEC : 0, pieces = turned + (a.head_dim - turned * 2 * VEC) / VEC, wide = pieces < KA_THREADS / 2 ? pieces : KA_THREADS / 2;
    // smaller CTAs, more of them at different points of their chains, once there are many rows: 16384 of 48 heads of 128 78 -> 70 us, 872 of 40 heads of 64 7.6 -> 8.3
    const int most = a.r.n_rows > 8 * 148 ? KA_THREADS / 2 : KA_THREADS, threads = (most / wide * wide + 31) / 32 * 32;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.r.n_rows); cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = sizeof(float2) * (a.rot_dims / 2); cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kv_append_kernel<In, Out, VEC, HALVES>, a, wide);      // (this launch's own status)
}

template <typename In, typename Out>
static cudaError_t kv_append_typed(const KvAppendArgs& a, cudaStream_t s) {
    // 16-byte pieces where every address allows them and a piece is rotated by one rule; else two entries ("pairs") or one at a time
    const long in_align = 16 / sizeof(In);
    auto ok = [](const void* p, long row, long head, long align) { return ((uintptr_t)p & 15) == 0 && row % align == 0 && head % align == 0; };
    const bool wide = a.head_dim % 8 == 0 && a.rot_dims % (a.halves ? 16 : 8) == 0 && ok(a.k, a.k_row, a.k_head, in_align) && ok(a.v, a.v_row, a.v_head, in_align) &&
                      ok(a.k_pool, 0, 0, 8) && ok(a.v_pool, 0, 0, 8) && (!a.q || (ok(a.q, a.q_row, a.q_head, in_align) && ok(a.q_out, a.qo_row, a.qo_head, 8)));
    if (a.halves) return wide ? kv_append_rows<In, Out, 8, true>(a, s) : kv_append_rows<In, Out, 1, true>(a, s);
    return wide ? kv_append_rows<In, Out, 8, false>(a, s) : kv_append_rows<In, Out, 2, false>(a, s);
}

cudaError_t kv_append_launch(const KvAppendArgs& a, cudaStream_t s) {
    if (a.r.n_rows == 0) return cudaSuccess;
    if (a.rot_dims / 2 > KA_MAX_PAIRS) return cudaErrorInvalidValue;
    const bool h = a.cache_type == ELEM_F16;
    switch (a.in_type) {
        case ELEM_F32: return h ? kv_append_typed<float, __half>(a, s) : kv_append_typed<float, __nv_bfloat16>(a, s);
        case ELEM_F16: return h ? kv_append_typed<__half, __half>(a, s) : kv_append_typed<__half, __nv_bfloat16>(a, s);
        default: return h ? kv_append_typed<__nv_bfloat16, __half>(a, s) : kv_append_typed<__nv_bfloat16, __nv_bfloat16>(a, s);
    }
}

}  // namespace b2

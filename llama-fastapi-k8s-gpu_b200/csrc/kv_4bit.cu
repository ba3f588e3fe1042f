// Keys and values of new tokens into the paged cache in 4 bits (kv_4bit.cuh), keys and queries rotated on the way; and rows of that cache back in 16 or 32 bits.
// The rotation is that of kv_append.cu, but sines and cosines too are computed in 64 bits and rounded once, and its products and sums are rounded one by one (no fused
// multiply-add): which code an entry gets is decided at borders, and so it follows from the definition alone, whatever rotates the keys.
//
// A warp takes a row, or a part of its heads where the rows are few, and finds its place by itself; a lane has a piece of eight entries of a head, 32 bits of codes, and four
// neighbouring lanes have a group.
// Reads are bound by memory and by the chain that each row begins with (sequence, page, codes), so as many warps as an SM holds have two turns of pieces each under way, at 32 registers, which
// spill 5 to 14 words a thread: 65536 rows of 2 x 8 heads of 128 to f16 66 us, 0.79 of the measured bandwidth (four turns and half the warps 78), to f32 135, 37000 ragged rows of 2 x 5 heads to bf16
// 29.6. A warp takes 16 of the 32 bits that a word of values has, its neighbour's token the others. (Two rows a warp, both places found at once: 29.3 for those 37000 rows, 144 to f32, 23.1
// instead of 22.5 for 20000 rows of 8 heads to f16.)
// Appends wait: 16384 rows of 32 + 2 x 8 heads of 128 take 93 us, 3500 instructions a row at 0.60 of the issue slots, 3.8 TB/s or 0.58 of the measured bandwidth, and the largest stall is that of
// entries on their way, with 27 warps of an SM under way at 64 registers. 32 rows 5.2 us: their chain, and the turns of a row one after the other. (More turns of queries under way, one CTA
// an SM more or fewer: 1 to 6 % slower.)
#include "device_ops.h"
#include "kv_4bit.cuh"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <type_traits>

namespace b2 {

namespace {
constexpr int K4_WARPS = 8, K4_THREADS = 32 * K4_WARPS;
// log2 of the warps a row, for up to four warps a scheduler, no more than leaves each a turn of 32 pieces of the keys
inline int k4_parts(long rows, int pieces) {
    int log = 0;
    while (rows << (log + 1) <= 148 * 16 && pieces >> (log + 1) >= 32) log++;
    return log;
}

template <typename T> __device__ __forceinline__ float k4_float(T v);
template <> __device__ __forceinline__ float k4_float(float v) { return v; }
template <> __device__ __forceinline__ float k4_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float k4_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> struct alignas(16) K4Piece { T v[8]; };

__device__ __forceinline__ void k4_store(__half* p, bool wide, const float (&x)[8]) {
    K4Piece<__half> t;
#pragma unroll
    for (int e = 0; e < 8; e += 2) { const __half2 h = __floats2half2_rn(x[e], x[e + 1]); t.v[e] = __low2half(h); t.v[e + 1] = __high2half(h); }
    if (wide) *reinterpret_cast<K4Piece<__half>*>(p) = t;
    else
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = t.v[e];
}
__device__ __forceinline__ void k4_store(__nv_bfloat16* p, bool wide, const float (&x)[8]) {
    K4Piece<__nv_bfloat16> t;
#pragma unroll
    for (int e = 0; e < 8; e += 2) { const __nv_bfloat162 h = __floats2bfloat162_rn(x[e], x[e + 1]); t.v[e] = __low2bfloat16(h); t.v[e + 1] = __high2bfloat16(h); }
    if (wide) *reinterpret_cast<K4Piece<__nv_bfloat16>*>(p) = t;
    else
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = t.v[e];
}
__device__ __forceinline__ void k4_store(float* p, bool wide, const float (&x)[8]) {
    if (wide) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = x[e];
}

// The place of a row: whether it belongs to a sequence, its token number there (its last 32 bits; `number`: all of it, which lengths near -2^31 need), and the first byte of KV head 0's block
// of 16 tokens, or -1; by a whole warp. Up to 32 sequences: their starts and lengths in one read.
struct K4Place { int live, token; long block; };
__device__ __forceinline__ K4Place k4_place(const RaggedPages& r, int n_kv, int dim, int row, int lane, long* number = nullptr) {
    int s, end = 0, held = 0;
    const int first = r.row_start[0];
    if (r.n_seqs <= 32) {
        const bool one = lane < r.n_seqs;
        const int e = one ? r.row_start[lane + 1] : 0, l = one ? r.lengths[lane] : 0;
        s = __popc(__ballot_sync(0xffffffffu, one && e <= row));
        end = __shfl_sync(0xffffffffu, e, s & 31);
        held = __shfl_sync(0xffffffffu, l, s & 31);
    } else {
        s = seq_of_row(r.row_start, r.n_seqs, row, lane);
        if (s < r.n_seqs) { end = r.row_start[s + 1]; held = r.lengths[s]; }
    }
    K4Place p = {s < r.n_seqs && row >= first, 0, -1};
    if (!p.live) return p;
    const long at = (long)held - ((long)end - row);
    p.token = (int)at;
    if (number) *number = at;
    if (at < 0 || at >= (long)r.max_pages * r.block_tokens) return p;      // (below 2^31)
    const unsigned block = (unsigned)at / Q4_TOKENS, blocks = (unsigned)r.block_tokens / Q4_TOKENS, page_no = block / blocks;
    const int page = r.pages[s * r.table_stride + page_no];
    if (page >= 0 && page < r.n_pages) p.block = ((long)page * n_kv * blocks + (block - page_no * blocks)) * q4_block(dim);
    return p;
}
}  // namespace

// the larger one, NaN if one is; the largest and the smallest of three
__device__ __forceinline__ float k4_max(float a, float b) { float m; asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b)); return m; }
__device__ __forceinline__ float k4_max(float a, float b, float c) { float m; asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c)); return m; }
__device__ __forceinline__ float k4_min(float a, float b, float c) { float m; asm("min.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c)); return m; }

// Scale and codes of a group that four neighbouring lanes have: eight entries each, the eight codes of this lane's as a word.
// A code is the low bits of entry * (1 / scale) + 8 + 1.5 2^23, whose last place is a whole number (ties to even). The reciprocal is off by 2^-23 of it at most, and the product by as
// much of the quotient (8.01), so that this is the quotient rounded unless the fraction is within 2^-18 of a half; those are divided, as are entries by scales that are so small or large that the quotient may lie outside.
__device__ __forceinline__ uint32_t k4_quantise(const float (&x)[8], __half& scale) {
    float hi = k4_max(x[0], x[1]), lo = fminf(x[0], x[1]);
#pragma unroll
    for (int e = 2; e < 8; e += 2) { hi = k4_max(hi, x[e], x[e + 1]); lo = k4_min(lo, x[e], x[e + 1]); }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) { hi = k4_max(hi, __shfl_xor_sync(0xffffffffu, hi, o)); lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)); }
    scale = __float2half_rn(fminf(fmaxf((hi > -lo ? hi : lo) * -0.125f, -65504.f), 65504.f));
    const float s = __half2float(scale);
    constexpr float BIAS = 12582912.f;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    uint32_t word = 0;
    float near = 0.f;
    const uint64_t r2 = f2_pack(r, r), bias2 = f2_pack(BIAS + 8.f, BIAS + 8.f), minus2 = f2_pack(-1.f, -1.f);
#pragma unroll
    for (int e = 6; e >= 0; e -= 2) {
        const uint64_t x2 = f2_pack(x[e], x[e + 1]), t2 = f2_fma(x2, r2, bias2);
        const float2 t = f2_unpack(t2), rest = f2_unpack(f2_fma(x2, r2, f2_fma(t2, minus2, bias2)));
        near = fmaxf(near, fmaxf(fabsf(rest.x), fabsf(rest.y)));
        word = (word * 16 + __float_as_uint(fminf(t.y, BIAS + 15.f))) * 16 + __float_as_uint(fminf(t.x, BIAS + 15.f));
    }
    word -= 0x3f400000u;                                         // (what the upper bits of eight such numbers add up to)
    if (!(near < 0.5f - 0x1p-18f) || !(fabsf(s) >= 0x1p-14f && fabsf(s) < 65504.f)) {
        word = 0;
#pragma unroll 1
        for (int e = 0; e < 8; e++) {
            float v = x[0];
#pragma unroll
            for (int i = 1; i < 8; i++) v = e == i ? x[i] : v;
            const float c = s == 0.f ? 8.f : fminf(fmaxf(rintf(__fdiv_rn(v, s)) + 8.f, 0.f), 15.f);
            word |= (uint32_t)c << (4 * e);
        }
    }
    if (s == 0.f) scale = __ushort_as_half(0);
    if (!(hi < INFINITY && lo > -INFINITY)) { scale = __ushort_as_half(0x7fff); word = 0x88888888u; }      // (NaN)
    return word;
}

__device__ __forceinline__ void k4_prefetch(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }
template <typename T> __device__ __forceinline__ void k4_fetch(const T* p, bool wide, K4Piece<T>& t) {
    if (wide) t = *reinterpret_cast<const K4Piece<T>*>(p);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) t.v[e] = p[e];
}

// How keys are rotated: entries of a piece with each other, a piece with another one, or any (halves that are no whole pieces, a rotation that ends inside one)
enum K4Turn { K4_PAIRS, K4_HALVES, K4_ANY };

// `wide`: bits 0 .. 3, whether pieces of k, v, q and q_out are 16 bytes at 16-byte addresses. `parts`: log2 of the warps a row
template <typename In, int D, int TURN>
__global__ void __launch_bounds__(K4_THREADS, 4) kv_append_4bit_kernel(const KvAppendArgs a, const int wide, const int parts) {
    constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES, UNROLL = sizeof(In) == 4 || TURN != K4_PAIRS ? 1 : 2;      // pieces of a head, heads of a turn, turns under way
    __shared__ alignas(16) float2 turns[K4_WARPS][D / 2];        // cosines and sines of the warp's row
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, half = a.rot_dims >> 1;
    const long item = (long)blockIdx.x * K4_WARPS + warp, row = item >> parts;
    griddep_wait();
    griddep_launch();
    if (row >= a.r.n_rows) return;
    const int part = (int)(item - (row << parts)), w = lane % PIECES, d = 8 * w, h0 = lane / PIECES;
    const bool rotates = d < a.rot_dims, left = d < half;
    K4Place place;
    bool ready = false;
    float2* turn = turns[warp];
    const long step = (long)(a.r.block_tokens / Q4_TOKENS) * q4_block(D);
    // KIND 0: keys, 1: values, 2: queries. Each warp of the row has a part of the heads of each. False: the row has no sequence.
    auto heads_of = [&](auto kind, const In* base, long head, int heads, int wide_in) {
        constexpr int KIND = decltype(kind)::value;
        const int all = (heads + AT_ONCE - 1) / AT_ONCE, last = all * (part + 1) >> parts, mine = min(last, (heads - h0 + AT_ONCE - 1) / AT_ONCE);      // (this lane's)
        int i = all * part >> parts;
        const In* from = base + (i * AT_ONCE + h0) * head;
        K4Piece<In> x[UNROLL] = {}, y[UNROLL] = {};              // (a lane without a head of its own goes on with zeros)
        int loaded = i;                                          // turns whose entries are under way or here
        auto load = [&](K4Piece<In>& p, K4Piece<In>& q) {
            if (loaded < mine) {
                k4_fetch(from, wide_in, p);
                if constexpr (KIND != 1 && TURN == K4_HALVES) { if (rotates) k4_fetch(left ? from + half : from - half, wide_in, q); }
                if constexpr (KIND != 1 && TURN == K4_ANY) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int at = d + e, other = a.halves ? (at < half ? at + half : at - half) : at ^ 1;
                        q.v[e] = at < a.rot_dims ? from[other - d] : p.v[e];
                    }
                }
            }
            from += AT_ONCE * head;
            loaded++;
        };
#pragma unroll
        for (int u = 0; u < UNROLL; u++) load(x[u], y[u]);
        if (!ready) {                                            // (the first entries are under way)
            ready = true;
            long number = 0;
            place = k4_place(a.r, a.n_kv, D, (int)row, lane, &number);
            if (!place.live) return false;
            const double pos = (double)(a.first_pos + number);
            for (int j = lane; j < half; j += 32) {
                const double t = pos * (double)a.freqs[j] * 0.15915494309189533577;      // 1 / (2 pi)
                double sn, cs;
                sincospi(2.0 * (t - rint(t)), &sn, &cs);
                turn[j] = make_float2((float)((double)a.amplitude * cs), (float)((double)a.amplitude * sn));
            }
            __syncwarp();
        }
        const int token = place.token & (Q4_TOKENS - 1);
        uint8_t* pool = (uint8_t*)(KIND == 0 ? a.k_pool : a.v_pool) + place.block + (i * AT_ONCE + h0) * step;
        uint16_t* to = KIND == 2 ? (uint16_t*)a.q_out + row * a.qo_row + d + (i * AT_ONCE + h0) * a.qo_head : nullptr;
        auto turns_of = [&](auto f16) {
#pragma unroll 1
            while (i < last) {
#pragma unroll
                for (int u = 0; u < UNROLL; u++) {
                    if (i >= last) break;
                    const bool in = i < mine;
                    float z[8];
#pragma unroll
                    for (int e = 0; e < 8; e++) z[e] = k4_float(x[u].v[e]);
                    if constexpr (KIND != 1) {
                        if (rotates) {
                            if constexpr (TURN == K4_PAIRS) {
#pragma unroll
                                for (int e = 0; e < 8; e += 4) {
                                    const float4 t = *reinterpret_cast<const float4*>(turn + (d + e) / 2);
                                    const float v0 = z[e], v1 = z[e + 1], v2 = z[e + 2], v3 = z[e + 3];
                                    z[e] = __fsub_rn(__fmul_rn(v0, t.x), __fmul_rn(v1, t.y)); z[e + 1] = __fadd_rn(__fmul_rn(v1, t.x), __fmul_rn(v0, t.y));
                                    z[e + 2] = __fsub_rn(__fmul_rn(v2, t.z), __fmul_rn(v3, t.w)); z[e + 3] = __fadd_rn(__fmul_rn(v3, t.z), __fmul_rn(v2, t.w));
                                }
                            } else if constexpr (TURN == K4_HALVES) {
                                const float2* with = turn + (left ? d : d - half);
                                const float sign = left ? -1.f : 1.f;
#pragma unroll
                                for (int e = 0; e < 8; e += 2) {
                                    const float4 t = *reinterpret_cast<const float4*>(with + e);
                                    z[e] = __fadd_rn(__fmul_rn(z[e], t.x), __fmul_rn(k4_float(y[u].v[e]), sign * t.y));
                                    z[e + 1] = __fadd_rn(__fmul_rn(z[e + 1], t.z), __fmul_rn(k4_float(y[u].v[e + 1]), sign * t.w));
                                }
                            } else {
#pragma unroll
                                for (int e = 0; e < 8; e++) {
                                    const int at = d + e;
                                    if (at >= a.rot_dims) continue;
                                    const bool one = a.halves ? at < half : (e & 1) == 0;
                                    const float2 t = turn[a.halves ? (one ? at : at - half) : at >> 1];
                                    z[e] = __fadd_rn(__fmul_rn(z[e], t.x), __fmul_rn(k4_float(y[u].v[e]), one ? -t.y : t.y));
                                }
                            }
                        }
                    }
                    if constexpr (KIND == 2) {
                        __syncwarp();                                // (a head's entries are read before they are replaced: q in place)
                        if (in) k4_store((std::conditional_t<decltype(f16)::value, __half, __nv_bfloat16>*)to, wide >> 3 & 1, z);
                        to += AT_ONCE * a.qo_head;
                        load(x[u], y[u]);
                    } else {
                        load(x[u], y[u]);
                        __half scale;
                        const uint32_t word = k4_quantise(z, scale);
                        if (in && place.block >= 0) {
                            if (KIND == 0) *reinterpret_cast<uint32_t*>(pool + q4_key(D, token, w)) = word;
                            else {
                                *reinterpret_cast<uint16_t*>(pool + q4_value(D, token, 2 * w)) = (uint16_t)word;
                                *reinterpret_cast<uint16_t*>(pool + q4_value(D, token, 2 * w + 1)) = (uint16_t)(word >> 16);
                            }
                            if ((w & 3) == 0) *reinterpret_cast<__half*>(pool + q4_scale(D, token, w >> 2)) = scale;
                        }
                        pool += AT_ONCE * step;
                    }
                    i++;
                }
            }
        };
        if (KIND != 2 || a.cache_type == ELEM_F16) turns_of(std::true_type{});
        else turns_of(std::false_type{});
        return true;
    };
    // the values and queries of a row that is one warp's alone: on their way into L2 while the keys are dealt with
    if (parts == 0) {
        constexpr int LINES = D * (int)sizeof(In) / 128;
        for (int i = lane; i < a.n_kv * LINES; i += 32) k4_prefetch((const In*)a.v + row * a.v_row + i / LINES * a.v_head + i % LINES * (128 / sizeof(In)));
        if (a.q) for (int i = lane; i < a.n_head * LINES; i += 32) k4_prefetch((const In*)a.q + row * a.q_row + i / LINES * a.q_head + i % LINES * (128 / sizeof(In)));
    }
    if (!heads_of(std::integral_constant<int, 0>{}, (const In*)a.k + row * a.k_row + d, a.k_head, a.n_kv, wide & 1)) return;
    heads_of(std::integral_constant<int, 1>{}, (const In*)a.v + row * a.v_row + d, a.v_head, a.n_kv, wide >> 1 & 1);
    if (a.q) heads_of(std::integral_constant<int, 2>{}, (const In*)a.q + row * a.q_row + d, a.q_head, a.n_head, wide >> 2 & 1);
}

// The eight codes of a word less 8, and those times their scale, rounded once
__device__ __forceinline__ void k4_codes(uint32_t word, __half2 (&v)[4]) {
    // byte i twice, its codes as 1024 + c and 1024 + 16 c, and those as c - 8, exact
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t two = (__byte_perm(word, 0, i | 0x40 | i << 8 | 0x4000) & 0x00f0000fu) | 0x64006400u;
        v[i] = __hfma2(*reinterpret_cast<const __half2*>(&two), __halves2half2(__ushort_as_half(0x3c00), __ushort_as_half(0x2c00)),
                       __halves2half2(__ushort_as_half(0xe408), __ushort_as_half(0xd480)));
    }
}
__device__ __forceinline__ void k4_put(__half* p, bool wide, const __half2 (&v)[4], __half scale) {
    K4Piece<__half> t;
    const __half2 s = __half2half2(scale);
#pragma unroll
    for (int i = 0; i < 4; i++) { const __half2 x = __hmul2(v[i], s); t.v[2 * i] = __low2half(x); t.v[2 * i + 1] = __high2half(x); }
    if (wide) *reinterpret_cast<K4Piece<__half>*>(p) = t;
    else
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = t.v[e];
}
template <typename Out>
__device__ __forceinline__ void k4_put(Out* p, bool wide, const __half2 (&v)[4], __half scale) {
    float x[8];
    const float s = __half2float(scale);
#pragma unroll
    for (int i = 0; i < 4; i++) { const float2 f = __half22float2(v[i]); x[2 * i] = s * f.x; x[2 * i + 1] = s * f.y; }
    k4_store(p, wide, x);
}

template <typename Out, int D>
__global__ void __launch_bounds__(K4_THREADS, 8) kv_read_4bit_kernel(const KvReadArgs a, const int wide, const int parts) {
    constexpr int PIECES = D / 8, AT_ONCE = 32 / PIECES, UNROLL = 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long item = (long)blockIdx.x * K4_WARPS + warp, row = item >> parts;
    griddep_wait();
    griddep_launch();
    if (row >= a.r.n_rows) return;
    const K4Place place = k4_place(a.r, a.n_kv, D, (int)row, lane);
    if (place.block < 0) return;
    const int part = (int)(item - (row << parts));
    const int token = place.token & (Q4_TOKENS - 1), w = lane % PIECES, h0 = lane / PIECES;
    const int all = (a.n_kv + AT_ONCE - 1) / AT_ONCE, first = all * part >> parts, last = all * (part + 1) >> parts;
    const long step = (long)(a.r.block_tokens / Q4_TOKENS) * q4_block(D), begin = place.block + (first * AT_ONCE + h0) * step;
    const uint8_t *kp = (const uint8_t*)a.k_pool + begin + q4_key(D, token, w), *vp = (const uint8_t*)a.v_pool + begin + q4_value(D, token, 2 * w);
    const int next = q4_value(D, token, 2 * w + 1) - q4_value(D, token, 2 * w), ks = q4_scale(D, token, w >> 2) - q4_key(D, token, w), vs = q4_scale(D, token, w >> 2) - q4_value(D, token, 2 * w);
    Out* k = (Out*)a.k + row * a.k_row + (first * AT_ONCE + h0) * a.k_head + 8 * w;
    Out* v = (Out*)a.v + row * a.v_row + (first * AT_ONCE + h0) * a.v_head + 8 * w;
    const int n = min(last - first, (a.n_kv - h0 + AT_ONCE - 1) / AT_ONCE - first);      // heads of this lane
    for (int i = 0; i < n; i += UNROLL) {
        uint32_t kw[UNROLL], vw[UNROLL];
        __half sk[UNROLL], sv[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (i + u >= n) break;
            if (a.k) { kw[u] = *reinterpret_cast<const uint32_t*>(kp); sk[u] = *reinterpret_cast<const __half*>(kp + ks); }
            if (a.v) {
                vw[u] = *reinterpret_cast<const uint16_t*>(vp) | (uint32_t)*reinterpret_cast<const uint16_t*>(vp + next) << 16;
                sv[u] = *reinterpret_cast<const __half*>(vp + vs);
            }
            kp += AT_ONCE * step; vp += AT_ONCE * step;
        }
#pragma unroll
        for (int u = 0; u < UNROLL; u++) {
            if (i + u >= n) break;
            __half2 c[4];
            if (a.k) { k4_codes(kw[u], c); k4_put(k, wide & 1, c, sk[u]); }
            if (a.v) { k4_codes(vw[u], c); k4_put(v, wide >> 1 & 1, c, sv[u]); }
            k += AT_ONCE * a.k_head; v += AT_ONCE * a.v_head;
        }
    }
}

// ---------------------------------------------------------------- host side
// 16 bytes at a time wherever eight entries of a row start
static int k4_wide(const void* p, long row, long head, int size) { return ((uintptr_t)p & 15) == 0 && row * size % 16 == 0 && head * size % 16 == 0; }

static unsigned k4_ctas(long rows, int parts) { return (unsigned)(((rows << parts) + K4_WARPS - 1) / K4_WARPS); }

template <typename In, int D>
static cudaError_t k4_append(const KvAppendArgs& a, cudaStream_t s) {
    const int size = sizeof(In), parts = k4_parts(a.r.n_rows, a.n_kv * D / 8);
    const int wide = k4_wide(a.k, a.k_row, a.k_head, size) | k4_wide(a.v, a.v_row, a.v_head, size) << 1 | k4_wide(a.q, a.q_row, a.q_head, size) << 2 | k4_wide(a.q_out, a.qo_row, a.qo_head, 2) << 3;
    auto* kernel = a.rot_dims % (a.halves ? 16 : 8) ? kv_append_4bit_kernel<In, D, K4_ANY> : a.halves ? kv_append_4bit_kernel<In, D, K4_HALVES> : kv_append_4bit_kernel<In, D, K4_PAIRS>;
    return launch_chain(kernel, dim3(k4_ctas(a.r.n_rows, parts)), dim3(K4_THREADS), 0, s, a, wide, parts);
}
template <typename In>
static cudaError_t k4_append_dim(const KvAppendArgs& a, cudaStream_t s) { return a.head_dim == 64 ? k4_append<In, 64>(a, s) : k4_append<In, 128>(a, s); }
cudaError_t kv_append_4bit_launch(const KvAppendArgs& a, cudaStream_t s) {
    if (a.r.n_rows == 0) return cudaSuccess;
    const DependentLaunch dependent;
    return a.in_type == ELEM_F32 ? k4_append_dim<float>(a, s) : a.in_type == ELEM_F16 ? k4_append_dim<__half>(a, s) : k4_append_dim<__nv_bfloat16>(a, s);
}

template <typename Out, int D>
static cudaError_t k4_read(const KvReadArgs& a, cudaStream_t s) {
    const int parts = k4_parts(a.r.n_rows, a.n_kv * D / 8), wide = k4_wide(a.k, a.k_row, a.k_head, sizeof(Out)) | k4_wide(a.v, a.v_row, a.v_head, sizeof(Out)) << 1;
    return launch_chain(kv_read_4bit_kernel<Out, D>, dim3(k4_ctas(a.r.n_rows, parts)), dim3(K4_THREADS), 0, s, a, wide, parts);
}
template <typename Out>
static cudaError_t k4_read_dim(const KvReadArgs& a, cudaStream_t s) { return a.head_dim == 64 ? k4_read<Out, 64>(a, s) : k4_read<Out, 128>(a, s); }
cudaError_t kv_read_4bit_launch(const KvReadArgs& a, cudaStream_t s) {
    if (a.r.n_rows == 0 || (!a.k && !a.v)) return cudaSuccess;
    const DependentLaunch dependent;
    return a.out_type == ELEM_F32 ? k4_read_dim<float>(a, s) : a.out_type == ELEM_F16 ? k4_read_dim<__half>(a, s) : k4_read_dim<__nv_bfloat16>(a, s);
}

}  // namespace b2

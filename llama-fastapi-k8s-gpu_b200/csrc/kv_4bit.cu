// Keys and values of new tokens into the paged cache in 4 bits (kv_4bit.cuh), keys and queries rotated on the way; and rows of that cache back in 16 or 32 bits.
// The rotation is that of kv_append.cu, but sines and cosines too are computed in 64 bits and rounded once, and its products and sums are rounded one by one (no fused
// multiply-add): which code an entry gets is decided at borders, and so it follows from the definition alone, whatever rotates the keys.
//
// Bound by memory. A CTA takes one row; a thread has a piece of eight entries of a head, one 32-bit word of codes, and four neighbouring lanes have a group.
#include "device_ops.h"
#include "kv_4bit.cuh"
#include "ptx.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2 {

namespace {
constexpr int K4_THREADS = 256;

template <typename T> __device__ __forceinline__ float k4_float(T v);
template <> __device__ __forceinline__ float k4_float(float v) { return v; }
template <> __device__ __forceinline__ float k4_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float k4_float(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> struct alignas(16) K4Piece { T v[8]; };

// eight entries from `p`
template <typename T>
__device__ __forceinline__ void k4_load(const T* p, bool wide, float (&x)[8]) {
    K4Piece<T> t;
    if (wide) t = *reinterpret_cast<const K4Piece<T>*>(p);
    else
#pragma unroll
        for (int e = 0; e < 8; e++) t.v[e] = p[e];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = k4_float(t.v[e]);
}
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

// the place of a row: whether it belongs to a sequence, its token number there, and the first byte of KV head 0's block of 16 tokens, or -1; by a whole warp
struct K4Place { int live; int token; long block; };
__device__ __forceinline__ K4Place k4_place(const RaggedPages& r, int n_kv, int dim, int row, int lane) {
    const int s = seq_of_row(r.row_start, r.n_seqs, row, lane);
    K4Place p = {s < r.n_seqs && row >= r.row_start[0], 0, -1};
    if (!p.live) return p;
    const long at = (long)r.lengths[s] - ((long)r.row_start[s + 1] - row);
    const long page_no = at >= 0 ? at / r.block_tokens : r.max_pages;
    p.token = (int)at;
    if (page_no < r.max_pages) {
        const int page = r.pages[s * r.table_stride + page_no], blocks = r.block_tokens / Q4_TOKENS;
        if (page >= 0 && page < r.n_pages) p.block = ((long)page * n_kv * blocks + at % r.block_tokens / Q4_TOKENS) * q4_block(dim);
    }
    return p;
}
}  // namespace

// Scale and codes of a group that four neighbouring lanes have: eight entries each, the eight codes of this lane's as a word
__device__ __forceinline__ uint32_t k4_quantise(const float (&x)[8], __half& scale) {
    float hi = x[0], lo = x[0], none = 0.f;                      // none: NaN if an entry is no finite number
#pragma unroll
    for (int e = 0; e < 8; e++) { hi = fmaxf(hi, x[e]); lo = fminf(lo, x[e]); none = fmaf(x[e], 0.f, none); }
#pragma unroll
    for (int o = 1; o < 4; o *= 2) {
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o)); lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        none += __shfl_xor_sync(0xffffffffu, none, o);
    }
    scale = __float2half_rn(fminf(fmaxf((hi > -lo ? hi : lo) * -0.125f, -65504.f), 65504.f));
    const float s = __half2float(scale);
    uint32_t word = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const float c = s == 0.f ? 8.f : fminf(fmaxf(rintf(__fdiv_rn(x[e], s)) + 8.f, 0.f), 15.f);
        word |= (uint32_t)c << (4 * e);
    }
    if (s == 0.f) scale = __ushort_as_half(0);
    if (none != 0.f) { scale = __ushort_as_half(0x7fff); word = 0x88888888u; }      // (NaN)
    return word;
}

template <typename In, typename Out>
__global__ void __launch_bounds__(K4_THREADS) kv_append_4bit_kernel(const KvAppendArgs a, const int wide_k, const int wide_v, const int wide_q, const int wide_o) {
    extern __shared__ float2 k4_turn[];                          // [rot_dims / 2] cosines and sines
    __shared__ K4Place place;
    const int tid = threadIdx.x, lane = tid & 31, D = a.head_dim, per_head = D / 8, half = a.rot_dims >> 1;
    const long row = blockIdx.x;
    if (tid < 32) {
        const K4Place p = k4_place(a.r, a.n_kv, D, (int)row, lane);
        if (lane == 0) place = p;
    }
    __syncthreads();
    if (!place.live) return;
    const double pos = (double)(a.first_pos + place.token);
    for (int i = tid; i < half; i += K4_THREADS) {
        const double turns = pos * (double)a.freqs[i] * 0.15915494309189533577;      // 1 / (2 pi)
        double sn, cs;
        sincospi(2.0 * (turns - rint(turns)), &sn, &cs);
        k4_turn[i] = make_float2((float)((double)a.amplitude * cs), (float)((double)a.amplitude * sn));
    }
    __syncthreads();
    const int blocks = a.r.block_tokens / Q4_TOKENS, token = place.token & (Q4_TOKENS - 1);
    const long block = place.block;
    const int pieces = (2 * a.n_kv + (a.q ? a.n_head : 0)) * per_head;
    for (int i = tid; i < (pieces + 31) / 32 * 32; i += K4_THREADS) {      // (whole warps: groups are shuffled together)
        const bool in = i < pieces;
        const int h = in ? i / per_head : 0, w = i - h * per_head, d = 8 * w, kind = h < a.n_kv ? 0 : h < 2 * a.n_kv ? 1 : 2;
        const In* from = kind == 0 ? (const In*)a.k + row * a.k_row + h * a.k_head : kind == 1 ? (const In*)a.v + row * a.v_row + (h - a.n_kv) * a.v_head
                                                                                              : (const In*)a.q + row * a.q_row + (h - 2 * a.n_kv) * a.q_head;
        const bool wide = kind == 0 ? wide_k : kind == 1 ? wide_v : wide_q;
        float x[8], y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = y[e] = 0.f;
        const bool turned = kind != 1 && d < a.rot_dims;
        if (in) {
            k4_load(from + d, wide, x);
            if (turned && a.halves) {                            // the entries that these are rotated with
                if (half % 8 == 0) k4_load(from + (d < half ? d + half : d - half), wide, y);
                else
#pragma unroll
                    for (int e = 0; e < 8; e++) y[e] = d + e < a.rot_dims ? k4_float(from[d + e < half ? d + e + half : d + e - half]) : 0.f;
            }
        }
        __syncwarp();                                            // a head's entries are read before they are replaced (q in place): a warp has whole heads
        if (turned) {
            float z[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int at = d + e;
                if (at >= a.rot_dims) { z[e] = x[e]; continue; }
                const bool first = a.halves ? at < half : (e & 1) == 0;
                const float2 t = k4_turn[a.halves ? (first ? at : at - half) : at >> 1];
                const float other = a.halves ? y[e] : x[e ^ 1];
                z[e] = first ? __fsub_rn(__fmul_rn(x[e], t.x), __fmul_rn(other, t.y)) : __fadd_rn(__fmul_rn(other, t.y), __fmul_rn(x[e], t.x));
            }
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = z[e];
        }
        if (kind == 2) {
            if (in) k4_store((Out*)a.q_out + row * a.qo_row + (h - 2 * a.n_kv) * a.qo_head + d, wide_o, x);
        }
        __half scale;
        const uint32_t word = k4_quantise(x, scale);
        if (in && kind != 2 && block >= 0) {
            uint8_t* to = (uint8_t*)(kind == 0 ? a.k_pool : a.v_pool) + block + (long)(kind == 0 ? h : h - a.n_kv) * blocks * q4_block(D);
            *reinterpret_cast<uint32_t*>(to + q4_word(D, token, w)) = word;
            if ((w & 3) == 0) *reinterpret_cast<__half*>(to + (kind == 0 ? q4_key_scale(D, token, w >> 2) : q4_value_scale(D, token, w >> 2))) = scale;
        }
    }
}

// a row a CTA
template <typename Out>
__global__ void __launch_bounds__(K4_THREADS) kv_read_4bit_kernel(const KvReadArgs a, const int wide_k, const int wide_v) {
    __shared__ K4Place place;
    const int tid = threadIdx.x, D = a.head_dim, per_head = D / 8;
    const long row = blockIdx.x;
    if (tid < 32) {
        const K4Place p = k4_place(a.r, a.n_kv, D, (int)row, tid);
        if (tid == 0) place = p;
    }
    __syncthreads();
    if (place.block < 0) return;
    const int blocks = a.r.block_tokens / Q4_TOKENS, token = place.token & (Q4_TOKENS - 1);
    const int first = a.k ? 0 : a.n_kv, last = a.v ? 2 * a.n_kv : a.n_kv;
    for (int i = first * per_head + tid; i < last * per_head; i += K4_THREADS) {
        const int h2 = i / per_head, w = i - h2 * per_head, h = h2 < a.n_kv ? h2 : h2 - a.n_kv;
        const bool key = h2 < a.n_kv;
        const uint8_t* from = (const uint8_t*)(key ? a.k_pool : a.v_pool) + place.block + (long)h * blocks * q4_block(D);
        const uint32_t word = *reinterpret_cast<const uint32_t*>(from + q4_word(D, token, w));
        const float s = __half2float(*reinterpret_cast<const __half*>(from + (key ? q4_key_scale(D, token, w >> 2) : q4_value_scale(D, token, w >> 2))));
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = s * (float)((int)(word >> (4 * e) & 15) - 8);
        k4_store((key ? (Out*)a.k + row * a.k_row + h * a.k_head : (Out*)a.v + row * a.v_row + h * a.v_head) + 8 * w, key ? wide_k : wide_v, x);
    }
}

// ---------------------------------------------------------------- host side
// 16 bytes at a time wherever eight entries of a row start
static int k4_wide(const void* p, long row, long head, int size) { return ((uintptr_t)p & 15) == 0 && row * size % 16 == 0 && head * size % 16 == 0; }

template <typename In, typename Out>
static cudaError_t k4_append(const KvAppendArgs& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.r.n_rows); cfg.blockDim = dim3(K4_THREADS); cfg.dynamicSmemBytes = sizeof(float2) * (a.rot_dims / 2); cfg.stream = s;
    const int size = sizeof(In);
    return cudaLaunchKernelEx(&cfg, kv_append_4bit_kernel<In, Out>, a, k4_wide(a.k, a.k_row, a.k_head, size), k4_wide(a.v, a.v_row, a.v_head, size), k4_wide(a.q, a.q_row, a.q_head, size),
                              k4_wide(a.q_out, a.qo_row, a.qo_head, 2));
}
cudaError_t kv_append_4bit_launch(const KvAppendArgs& a, cudaStream_t s) {
    if (a.r.n_rows == 0) return cudaSuccess;
    const bool h = a.cache_type == ELEM_F16;
    switch (a.in_type) {
        case ELEM_F32: return h ? k4_append<float, __half>(a, s) : k4_append<float, __nv_bfloat16>(a, s);
        case ELEM_F16: return h ? k4_append<__half, __half>(a, s) : k4_append<__half, __nv_bfloat16>(a, s);
        default: return h ? k4_append<__nv_bfloat16, __half>(a, s) : k4_append<__nv_bfloat16, __nv_bfloat16>(a, s);
    }
}

template <typename Out>
static cudaError_t k4_read(const KvReadArgs& a, cudaStream_t s) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.r.n_rows); cfg.blockDim = dim3(K4_THREADS); cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, kv_read_4bit_kernel<Out>, a, k4_wide(a.k, a.k_row, a.k_head, sizeof(Out)), k4_wide(a.v, a.v_row, a.v_head, sizeof(Out)));
}
cudaError_t kv_read_4bit_launch(const KvReadArgs& a, cudaStream_t s) {
    if (a.r.n_rows == 0 || (!a.k && !a.v)) return cudaSuccess;
    return a.out_type == ELEM_F32 ? k4_read<float>(a, s) : a.out_type == ELEM_F16 ? k4_read<__half>(a, s) : k4_read<__nv_bfloat16>(a, s);
}

}  // namespace b2

// What both kernels of attention over a cache in 4 bits share: storing outputs, and results of a segment of keys that several CTAs have.
#pragma once
#include "device_ops.h"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2 {

#ifdef __CUDACC__
__device__ __forceinline__ uint32_t a4_half2(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
// the row of its sequence that (row, head) f belongs to: f over the group's heads (the quotient by multiplication may be one less)
__device__ __forceinline__ int a4_row(const Attention4Args& a, unsigned f) {
    const unsigned i = __umulhi(f, a.per_group);
    return (int)(i + (f - i * (unsigned)a.group >= (unsigned)a.group));
}
// A partial result has its reference in log2, rounded: reference * by. What that is off by, in log2, goes into its sums, so that weights between partial results are those of the exact references.
// (Held to 2^60: scores of up to 2^84. A reference of none, less infinity or with sums that are NaN, gives some number.)
__device__ __forceinline__ float a4_rest(float ref, float by, float scaled) { return fminf(fmaxf(fmaf(ref, by, -scaled), -60.f), 60.f); }
// four neighbouring dims of a row's output
__device__ __forceinline__ void a4_store_out(const Attention4Args& a, int t, int head, int d, float x, float y, float z, float w) {
    uint32_t lo, hi;
    if (a.type == ELEM_F16) { lo = a4_half2(x, y); hi = a4_half2(z, w); }
    else {
        const __nv_bfloat162 l = __floats2bfloat162_rn(x, y), h = __floats2bfloat162_rn(z, w);
        lo = *reinterpret_cast<const uint32_t*>(&l); hi = *reinterpret_cast<const uint32_t*>(&h);
    }
    uint16_t* dst = (uint16_t*)a.out + (size_t)t * a.out_row + (size_t)head * a.out_head + d;
    if (((uintptr_t)dst & 7) == 0) *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
    else { dst[0] = (uint16_t)lo; dst[1] = (uint16_t)(lo >> 16); dst[2] = (uint16_t)hi; dst[3] = (uint16_t)(hi >> 16); }
}

#endif

// where a CTA's results of a segment that goes on in another CTA lie: the first, of one that began in an earlier CTA, and the last
struct A4Desc { int rows, r0, f0, kvh, last; };      // rows of the tile (0: no such result), first row of the sequence, first (row, head) of the tile, the CTA where the segment ends
#ifdef __CUDACC__
template <int PART> __device__ __forceinline__ A4Desc* a4_desc(const Attention4Args& a, int ctas) { return reinterpret_cast<A4Desc*>(a.work + (size_t)ctas * 2 * PART); }
#endif

// the results in the workspace, joined into outputs: rows of a tile, CTAs of the kernel that has left them
cudaError_t attention_4bit_join(const Attention4Args& a, int ctas, int rows, cudaStream_t s);

// attention_4bit_tc.cu: many rows of a sequence
size_t attention_4bit_tc_work_bytes(int head_dim);
cudaError_t attention_4bit_tc_launch(const Attention4Args& a, cudaStream_t s);
cudaError_t attention_4bit_tc_error(unsigned int* code);
cudaError_t attention_4bit_tc_give_up(unsigned int code, cudaStream_t s);

}  // namespace b2

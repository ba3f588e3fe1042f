// Keys and values of new tokens into the paged cache, keys (and queries) rotated on the way.
//   angle = position * freq_i, the product and its reduction to a turn in 64 bits (at position 100000 a 32-bit product is off by up to 0.004 of a radian);
//   (a, b) -> amplitude * (a cos - b sin, a sin + b cos) for the entries 2i, 2i + 1 ("pairs") or i, i + rot_dims / 2 ("halves") below rot_dims, the others as
//   they are; one rounding to the cache's type at the end.
// The GGUF engine's own steps do this behind their projection (rope_store in prefill.cu, which also adds that product's K splits up); this one takes rows of any
// producer.
//
// Bound by memory: every entry is read once and written once. A CTA takes one row (few rows) or four; a thread takes 16-byte pieces (both halves of a pair of
// pieces under "halves", so that q may be rotated in place), whose loads are under way while the row's sequence, its page and the angles are found: those are
// a chain of three dependent reads.
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
template <typename T> __device__ __forceinline__ T ka_round(float v);
template <> __device__ __forceinline__ __half ka_round(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 ka_round(float v) { return __float2bfloat16_rn(v); }

// (two entries: as two loads, so that any row may start anywhere)
template <typename T, int VEC>
struct alignas(VEC == 8 ? 16 : sizeof(T)) Piece { T v[VEC]; };

}  // namespace

template <typename In, typename Out, int VEC, int ROWS>
__global__ void __launch_bounds__(KA_THREADS) kv_append_kernel(const KvAppendArgs a) {
    constexpr int UNROLL = 3;
    extern __shared__ float2 ka_turn[];                          // [ROWS][rot_dims / 2]
    __shared__ long place[ROWS];                                 // entry of the pool where KV head 0 of the row lies, or -1
    __shared__ long pos[ROWS];                                   // position of the row
    __shared__ int live[ROWS];                                   // the row belongs to a sequence
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row0 = blockIdx.x * ROWS, rows = min(ROWS, a.r.n_rows - row0);
    const int D = a.head_dim, half = a.rot_dims >> 1, heads = 2 * a.n_kv + (a.q ? a.n_head : 0);
    // pieces of a head: two vectors half a rotation apart while they are rotated together, one otherwise
    const int turned = a.halves ? half / VEC : 0, pieces = turned + (D - turned * 2 * VEC) / VEC;
    const int n_items = rows * heads * pieces;
    struct Item { int row, kind, head, d; bool two, rot; };
    auto item_at = [&](int i) {
        Item it;
        const int p = i % pieces, h = i / pieces % heads;
        it.row = i / (pieces * heads);
        it.kind = h < a.n_kv ? 0 : h < 2 * a.n_kv ? 1 : 2;       // key, value, query
        it.head = it.kind == 0 ? h : it.kind == 1 ? h - a.n_kv : h - 2 * a.n_kv;
        it.two = p < turned;
        it.d = it.two ? p * VEC : turned * 2 * VEC + (p - turned) * VEC;
        it.rot = it.kind != 1 && it.d < a.rot_dims;
        return it;
    };
    using InPiece = Piece<In, VEC>;
    using OutPiece = Piece<Out, VEC>;
    InPiece x[UNROLL][2];
    auto load = [&](int u, int i) {
        if (i >= n_items) return;
        const Item it = item_at(i);
        const In* src = it.kind == 0 ? (const In*)a.k + (row0 + it.row) * a.k_row + it.head * a.k_head
                      : it.kind == 1 ? (const In*)a.v + (row0 + it.row) * a.v_row + it.head * a.v_head
                                     : (const In*)a.q + (row0 + it.row) * a.q_row + it.head * a.q_head;
        x[u][0] = *reinterpret_cast<const InPiece*>(src + it.d);
        if (it.two) x[u][1] = *reinterpret_cast<const InPiece*>(src + it.d + half);
    };
    auto store = [&](int u, int i) {
        if (i >= n_items) return;
        const Item it = item_at(i);
        if (!live[it.row] || (it.kind != 2 && place[it.row] < 0)) return;
        OutPiece y[2];
        const float2* turn = ka_turn + it.row * half;
        if (it.two && it.rot) {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                const float2 c = turn[it.d + e];
                const float p = ka_float(x[u][0].v[e]), r = ka_float(x[u][1].v[e]);
                y[0].v[e] = ka_round<Out>(p * c.x - r * c.y);
                y[1].v[e] = ka_round<Out>(p * c.y + r * c.x);
            }
        } else if (it.rot && !a.halves) {
#pragma unroll
            for (int e = 0; e + 1 < VEC; e += 2) {
                const float2 c = turn[(it.d + e) >> 1];
                const float p = ka_float(x[u][0].v[e]), r = ka_float(x[u][0].v[e + 1]);
                y[0].v[e] = ka_round<Out>(p * c.x - r * c.y);
                y[0].v[e + 1] = ka_round<Out>(p * c.y + r * c.x);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VEC; e++) {
                y[0].v[e] = ka_round<Out>(ka_float(x[u][0].v[e]));
                if (it.two) y[1].v[e] = ka_round<Out>(ka_float(x[u][1].v[e]));
            }
        }
        Out* dst = it.kind == 2 ? (Out*)a.q_out + (row0 + it.row) * a.qo_row + it.head * a.qo_head
                                : (it.kind == 0 ? (Out*)a.k_pool : (Out*)a.v_pool) + place[it.row] + (long)it.head * a.r.block_tokens * D;
        *reinterpret_cast<OutPiece*>(dst + it.d) = y[0];
        if (it.two) *reinterpret_cast<OutPiece*>(dst + it.d + half) = y[1];
    };
#pragma unroll
    for (int u = 0; u < UNROLL; u++) load(u, tid + u * KA_THREADS);
    if (warp < rows) {
        const int row = row0 + warp;
        const int s = seq_of_row(a.r.row_start, a.r.n_seqs, row, lane);
        if (lane == 0) {
            bool in = s < a.r.n_seqs && row >= a.r.row_start[0];
            long where = -1, at = 0;
            if (in) {
                at = (long)a.r.lengths[s] - (a.r.row_start[s + 1] - row);
                const long page_no = at >= 0 ? at / a.r.block_tokens : a.r.max_pages;
                if (page_no < a.r.max_pages) {
                    const int page = a.r.pages[s * a.r.table_stride + page_no];
                    if (page >= 0 && page < a.r.n_pages) where = ((long)page * a.n_kv * a.r.block_tokens + at % a.r.block_tokens) * D;
                }
            }
            place[warp] = where; live[warp] = in; pos[warp] = a.first_pos + at;
        }
    }
    __syncthreads();
    for (int i = tid; i < rows * half; i += KA_THREADS) {
        const int r = i / half;
        const double turns = (double)pos[r] * (double)a.freqs[i % half] * 0.15915494309189533577;      // 1 / (2 pi)
        float sn, cs;
        sincospif((float)(2.0 * (turns - rint(turns))), &sn, &cs);
        ka_turn[i] = make_float2(a.amplitude * cs, a.amplitude * sn);
    }
    __syncthreads();
    for (int i0 = tid; i0 < n_items; i0 += UNROLL * KA_THREADS) {
#pragma unroll
        for (int u = 0; u < UNROLL; u++) store(u, i0 + u * KA_THREADS);
#pragma unroll
        for (int u = 0; u < UNROLL; u++) load(u, i0 + (UNROLL + u) * KA_THREADS);
    }
}

template <typename In, typename Out, int VEC>
static cudaError_t kv_append_rows(const KvAppendArgs& a, cudaStream_t s) {
    const size_t turn = sizeof(float2) * (a.rot_dims / 2);
    // four rows a CTA share the set-up once there are enough rows to fill the SMs without (148 SMs, 8 CTAs of 256 threads each)
    if (a.r.n_rows <= 4 * 148) kv_append_kernel<In, Out, VEC, 1><<<a.r.n_rows, KA_THREADS, turn, s>>>(a);
    else kv_append_kernel<In, Out, VEC, 4><<<(a.r.n_rows + 3) / 4, KA_THREADS, 4 * turn, s>>>(a);
    return cudaGetLastError();
}

template <typename In, typename Out>
static cudaError_t kv_append_typed(const KvAppendArgs& a, cudaStream_t s) {
    // 16-byte pieces where every address allows them and a piece is rotated by one rule; else two entries ("pairs") or one at a time
    const long in_align = 16 / sizeof(In) > 8 ? 8 : 16 / sizeof(In);
    auto ok = [](const void* p, long row, long head, long align) { return ((uintptr_t)p & 15) == 0 && row % align == 0 && head % align == 0; };
    const bool wide = a.head_dim % 8 == 0 && a.rot_dims % (a.halves ? 16 : 8) == 0 && ok(a.k, a.k_row, a.k_head, in_align) && ok(a.v, a.v_row, a.v_head, in_align) &&
                      ok(a.k_pool, 0, 0, 8) && ok(a.v_pool, 0, 0, 8) && (!a.q || (ok(a.q, a.q_row, a.q_head, in_align) && ok(a.q_out, a.qo_row, a.qo_head, 8)));
    if (wide) return kv_append_rows<In, Out, 8>(a, s);
    if (a.halves) return kv_append_rows<In, Out, 1>(a, s);
    return kv_append_rows<In, Out, 2>(a, s);
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

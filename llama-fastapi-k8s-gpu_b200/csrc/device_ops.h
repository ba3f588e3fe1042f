// Launch interfaces of the operators over a caller's device memory (device_ops.cu checks their arguments and exports them).
#pragma once
#include "kernels.h"

namespace b2 {

enum ElemType { ELEM_F32 = 0, ELEM_F16 = 1, ELEM_BF16 = 2 };

// Which rows belong to which sequence, and where a sequence's own cached tokens lie. Row r belongs to sequence s when row_start[s] <= r < row_start[s + 1]; the
// rows of a sequence are the newest of its lengths[s] own tokens. All arrays are device memory.
struct RaggedPages {
    const int *row_start, *lengths;
    const int* pages;            // [n_seqs][table_stride], the first max_pages entries of each are read
    long table_stride;
    int max_pages, n_seqs, n_rows;
    int block_tokens;
    long n_pages;                // pages of the pools: ids outside are not followed
};

#ifdef __CUDACC__
// the sequence of row `row`: how many of row_start[1..n_seqs] are <= row, by the whole warp, 32 probes a round
__device__ __forceinline__ int seq_of_row(const int* row_start, int n_seqs, int row, int lane) {
    int lo = 0, n = n_seqs;                                      // the count lies in [lo, lo + n]
    while (n > 0) {
        const int step = (n + 31) / 32, at = lo + (lane + 1) * step - 1;        // probes entries lo + step - 1, lo + 2 step - 1, ...
        const bool below = at < lo + n && row_start[1 + at] <= row;
        const int passed = __popc(__ballot_sync(0xffffffffu, below));
        const int skip = min(passed * step, n);
        lo += skip;
        n = min(n - skip, step - 1);
    }
    return lo;
}
#endif

// Launches inside this scope may start while the kernel before them ends (launch_chain): they wait for it before they touch memory. Calls one after another, us each, with it and
// without: attention of 32 chats over a cache in 4 bits 19.5 and 21.2, of one chat 11.5 and 12.3.
struct DependentLaunch {
    bool prev;
    DependentLaunch() : prev(g_chain_pdl) { g_chain_pdl = true; }
    ~DependentLaunch() { g_chain_pdl = prev; }
};

// ---------------------------------------------------------------- kv_append.cu
struct KvAppendArgs {
    RaggedPages r;
    const void *k, *v, *q;       // rows x heads x head_dim, last dimension contiguous; q may be null
    long k_row, k_head, v_row, v_head, q_row, q_head, qo_row, qo_head;      // strides in elements
    void *k_pool, *v_pool;       // [n_pages][n_kv][block_tokens][head_dim]
    void* q_out;                 // cache type
    const float* freqs;          // [rot_dims / 2]
    long first_pos;
    int n_head, n_kv, head_dim, rot_dims, halves;
    float amplitude;
    int in_type, cache_type;
};
cudaError_t kv_append_launch(const KvAppendArgs& a, cudaStream_t s);

// ---------------------------------------------------------------- kv_4bit.cu: the same into a cache in 4 bits (kv_4bit.cuh; cache_type: q_out's), and out of it
cudaError_t kv_append_4bit_launch(const KvAppendArgs& a, cudaStream_t s);
struct KvReadArgs {
    RaggedPages r;
    const void *k_pool, *v_pool; // [n_pages][n_kv][block_tokens / 16][9 * head_dim] bytes
    void *k, *v;                 // [n_rows][n_kv][head_dim] of out_type, either may be null
    long k_row, k_head, v_row, v_head;
    int n_kv, head_dim, out_type;
};
cudaError_t kv_read_4bit_launch(const KvReadArgs& a, cudaStream_t s);

// ---------------------------------------------------------------- attention_4bit.cu
struct Attention4Args {
    RaggedPages r;
    const void* q;               // [n_rows][n_head][head_dim] of `type`
    long q_row, q_head;
    const void *k_pool, *v_pool; // as KvReadArgs
    void* out;                   // like q
    long out_row, out_head;
    float* work;                 // attention_4bit_work_bytes
    int max_rows;                // most rows of a sequence
    int n_head, n_kv, head_dim, type;
    float scale_log2;
    int group;                   // heads of a KV head, and 2^32 over them (both set by the launch)
    unsigned per_group;
    unsigned per_page;           // 2^32 over the blocks of a page (set by the launch)
    int few_units;               // units of work that tables and rows allow fit 31 bits (set by the launch)
};
size_t attention_4bit_work_bytes(long n_rows, int n_head, int n_kv, int head_dim);
cudaError_t attention_4bit_launch(const Attention4Args& a, cudaStream_t s);
cudaError_t attention_4bit_error(unsigned int* code);            // code of the first wait that ran out (does not wait), see shared_prefix_error
cudaError_t attention_4bit_give_up(unsigned int code, bool tensor_memory, cudaStream_t s);      // see shared_prefix_give_up

// ---------------------------------------------------------------- logprobs.cu
constexpr int LOGPROB_MAX_TOP = 64;
struct RowMap { int n; int token[BATCH_MAX], out[BATCH_MAX]; };      // row r's token is tokens[token[r]], its results go to row out[r] (n 0: to r, tokens[r])
struct LogprobArgs {
    const void* logits;          // [n_rows][n_vocab], rows row_stride elements apart
    long row_stride;
    const int* tokens;           // [n_rows] or null
    float *logprob, *entropy;    // [n_rows], either may be null
    float* top_logprob;          // [n_rows][n_top]
    int* top_id;
    int n_rows, n_vocab, n_top, type;
};
cudaError_t logprobs_launch(const LogprobArgs& a, cudaStream_t s, const RowMap* map = nullptr);

// ---------------------------------------------------------------- shared_prefix.cu, shared_prefix_tc.cu
struct SharedPrefixArgs {
    RaggedPages r;
    const void* q;               // [n_rows][n_head][head_dim] of the cache's type (q_f32: 32-bit, rounded to it)
    long q_row, q_head;
    int q_f32;
    const void *k_pool, *v_pool;
    const int* prefix_pages;
    int n_prefix;
    void* out;                   // like q, cache's type
    long out_row, out_head;
    float* work;                 // partial results of the prefix
    int max_rows;                // most rows of a sequence
    int n_head, n_kv, head_dim, type;
    float scale_log2;
    // batched steps of the engine: the slots' own page tables and positions instead of r's arrays, one row each; out in operand order
    const SlotDev* tab;
    BatchIdx slots;
    __half* out_h;
    int out_T_pad;
    unsigned int* err;           // where a wait that runs out is recorded (null: see shared_prefix_error)
};
size_t shared_prefix_work_floats(long n_rows, int n_head, int n_kv, int head_dim);
cudaError_t shared_prefix_launch(const SharedPrefixArgs& a, cudaStream_t s);
int shared_prefix_launches(const SharedPrefixArgs& a);

// Prefix pass on tensor memory: the key blocks of every (KV head, 256 query rows) cut into equal runs, one run a CTA. A unit's partial results are numbered by
// the CTAs that its blocks fall to.
struct PrefixCut {
    int units, pairs, blocks, run, ctas;      // units = n_kv * pairs; blocks of 128 keys a unit; blocks a CTA
    int per_unit;                             // != 0: every unit is cut by itself, else all of them laid end to end
    __host__ __device__ int runs() const { return (blocks + run - 1) / run; }      // (of a unit that is cut by itself)
    // (units * blocks fits 31 bits: shared_prefix_launch refuses more)
    __host__ __device__ int first_cta(int unit) const { return per_unit ? unit * runs() : (int)((unsigned)(unit * blocks) / (unsigned)run); }
    __host__ __device__ int slots(int unit) const {
        return per_unit ? runs() : (int)((unsigned)((unit + 1) * blocks - 1) / (unsigned)run) - first_cta(unit) + 1;
    }
    // the blocks [begin, end) of all units laid end to end that a CTA has
    __host__ __device__ int begin(int cta) const { return per_unit ? cta / runs() * blocks + cta % runs() * run : cta * run; }
    __host__ __device__ int end(int cta) const {
        const int e = begin(cta) + run, most = per_unit ? (cta / runs() + 1) * blocks : units * blocks;
        return e < most ? e : most;
    }
};
constexpr int PREFIX_SMS = 148;
PrefixCut prefix_cut(long n_rows, int n_head, int n_kv, int n_prefix, int sms);
// What the prefix pass leaves to a pass of single own tokens, which runs beside it and is bound by other things: which of the cuts it takes goes by the mean of
// the sequences' own tokens, 16 << level or fewer (the last: any). It writes {run, per_unit} into the workspace at cut_at.
constexpr int SHARE_LEVELS = 8;
struct PrefixShare { int adapt; size_t cut_at; int run[SHARE_LEVELS]; short ctas[SHARE_LEVELS], per_unit[SHARE_LEVELS]; };      // adapt 0: all SMs
cudaError_t shared_prefix_tc_launch(const SharedPrefixArgs& a, const PrefixCut& cut, size_t ml_at, const PrefixShare& share, cudaStream_t s);      // ml_at: see SpPlan

// code of the first wait of these kernels that ran out on the current device since the last call (0: none); waits for the device
cudaError_t shared_prefix_error(unsigned int* code);
cudaError_t shared_prefix_tc_error(unsigned int* code);      // (of that file; does not wait)
// enqueue: what a wait that ran out leaves behind, without the wait (for tests)
cudaError_t shared_prefix_give_up(unsigned int code, bool tensor_memory, cudaStream_t s);
cudaError_t shared_prefix_tc_give_up(unsigned int code, cudaStream_t s);
#ifdef __CUDACC__
// a file's error words (see mbar_give_up): the code, and none from here on, so that later calls can be told apart from earlier ones
template <size_t N>
cudaError_t take_error_word(const unsigned int (&symbol)[N], unsigned int* code) {
    const cudaError_t e = cudaMemcpyFromSymbol(code, symbol, sizeof(*code));
    const unsigned int none = 0;
    return e == cudaSuccess && *code ? cudaMemcpyToSymbol(symbol, &none, sizeof(none)) : e;
}
#endif

}  // namespace b2

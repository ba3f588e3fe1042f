// C entry points of the operators over a caller's device memory: argument checks (all before anything touches the device), then one or two launches on the
// caller's stream. Nothing is allocated, nothing waits, nothing is kept between calls; the caller's current device is left as it was.
#include "../../include/b200_gguf.h"
#include "device_ops.h"

#include <math.h>
#include <string>

using namespace b2;

int b2_fail(int code, const std::string& msg);

namespace {

int elem_type(int ggml) { return ggml == B2_TYPE_F32 ? ELEM_F32 : ggml == B2_TYPE_F16 ? ELEM_F16 : ggml == B2_TYPE_BF16 ? ELEM_BF16 : -1; }
size_t elem_size(int type) { return type == ELEM_F32 ? 4 : 2; }

struct OnDevice {
    int before = -1, device;
    cudaError_t status;
    explicit OnDevice(int d) : device(d) {
        status = cudaGetDevice(&before);
        if (status == cudaSuccess && before != device) status = cudaSetDevice(device);
    }
    ~OnDevice() { if (before >= 0 && before != device) cudaSetDevice(before); }
};

int bad(const char* what, const std::string& why) { return b2_fail(B2_ERR_ARG, std::string(what) + ": " + why); }
int done(const char* what, cudaError_t e) {
    if (e == cudaSuccess) return B2_OK;
    return b2_fail(B2_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

// 0, or the refusal; also fills `out`
int check_where(const char* what, const b2_ragged_pages& w, RaggedPages& out) {
    if (w.n_seqs < 0 || w.n_rows < 0) return bad(what, "negative number of sequences or rows");
    if (w.n_seqs > 65535) return bad(what, "at most 65535 sequences");
    if (w.block_tokens <= 0 || w.block_tokens % 16) return bad(what, "block_tokens must be a positive multiple of 16");
    if (w.max_pages <= 0 || w.n_pages <= 0) return bad(what, "max_pages and n_pages must be positive");
    // (kernels go on from the last token to the end of its tile and of a warp's page ids)
    if ((int64_t)w.max_pages * w.block_tokens > INT32_MAX - 4096) return bad(what, "max_pages * block_tokens must fit 32 bits, less 4096");
    if (w.n_pages > INT32_MAX) return bad(what, "n_pages must fit 32 bits");
    if (w.n_seqs > 1 && w.table_stride < w.max_pages) return bad(what, "table_stride is smaller than max_pages");
    if (w.n_rows && w.n_seqs && (!w.row_start || !w.lengths || !w.pages)) return bad(what, "null row_start, lengths or pages");
    if (((uintptr_t)w.row_start | (uintptr_t)w.lengths | (uintptr_t)w.pages) & 3) return bad(what, "integer arrays must be 4-byte aligned");
    out.row_start = w.row_start; out.lengths = w.lengths; out.pages = w.pages; out.table_stride = w.table_stride; out.max_pages = w.max_pages;
    out.n_seqs = w.n_seqs; out.n_rows = w.n_rows; out.block_tokens = w.block_tokens; out.n_pages = w.n_pages;
    return B2_OK;
}

}  // namespace

extern "C" int b2_kv_append(int device, const b2_ragged_pages* where, const b2_kv_append_args* x, void* stream) {
    const char* what = "b2_kv_append";
    if (!where || !x) return bad(what, "null arguments");
    KvAppendArgs a = {};
    if (int rc = check_where(what, *where, a.r)) return rc;
    a.in_type = elem_type(x->in_type); a.cache_type = elem_type(x->cache_type);
    if (a.in_type < 0) return b2_fail(B2_ERR_UNSUPPORTED, "b2_kv_append: rows must be f32, f16 or bf16");
    if (a.cache_type != ELEM_F16 && a.cache_type != ELEM_BF16) return b2_fail(B2_ERR_UNSUPPORTED, "b2_kv_append: the cache must be f16 or bf16");
    if (x->n_kv <= 0 || x->head_dim <= 0 || x->head_dim > 1024 || x->head_dim % 2) return bad(what, "n_kv must be positive, head_dim even and at most 1024");
    if (x->q && x->n_head <= 0) return bad(what, "n_head must be positive");
    if (x->rot_dims < 0 || x->rot_dims > x->head_dim || x->rot_dims > 512 || x->rot_dims % 2) return bad(what, "rot_dims must be even, at most head_dim and 512");
    if (x->layout != B2_ROTATE_PAIRS && x->layout != B2_ROTATE_HALVES) return bad(what, "unknown rotation layout");
    if (!isfinite(x->amplitude)) return bad(what, "amplitude must be finite");
    if (x->first_pos < 0 || x->first_pos > (int64_t)1 << 40) return bad(what, "first_pos out of range");
    if (where->n_rows == 0 || where->n_seqs == 0) return B2_OK;
    if (!x->k || !x->v || !x->k_pool || !x->v_pool || (x->q && !x->q_out) || (x->rot_dims && !x->freqs)) return bad(what, "null device pointer");
    if (((uintptr_t)x->k | (uintptr_t)x->v | (uintptr_t)x->q) % elem_size(a.in_type) || ((uintptr_t)x->k_pool | (uintptr_t)x->v_pool | (uintptr_t)x->q_out) & 1 ||
        (uintptr_t)x->freqs & 3) return bad(what, "pointers must be aligned to their elements");
    a.k = x->k; a.v = x->v; a.q = x->q; a.k_row = x->k_row; a.k_head = x->k_head; a.v_row = x->v_row; a.v_head = x->v_head; a.q_row = x->q_row; a.q_head = x->q_head;
    a.k_pool = x->k_pool; a.v_pool = x->v_pool; a.q_out = x->q_out; a.qo_row = x->q_out_row; a.qo_head = x->q_out_head;
    a.freqs = x->freqs; a.first_pos = x->first_pos; a.n_head = x->n_head; a.n_kv = x->n_kv; a.head_dim = x->head_dim; a.rot_dims = x->rot_dims;
    a.halves = x->layout == B2_ROTATE_HALVES; a.amplitude = x->amplitude;
    OnDevice on(device);
    return done(what, on.status != cudaSuccess ? on.status : kv_append_launch(a, (cudaStream_t)stream));
}

extern "C" int b2_token_logprobs(int device, const void* logits, int type, int64_t row_stride, int n_rows, int n_vocab, const int32_t* tokens, float* logprob,
                                 float* entropy, int n_top, float* top_logprob, int32_t* top_id, void* stream) {
    const char* what = "b2_token_logprobs";
    LogprobArgs a = {};
    a.type = elem_type(type);
    if (a.type < 0) return b2_fail(B2_ERR_UNSUPPORTED, "b2_token_logprobs: logits must be f32, f16 or bf16");
    if (n_rows < 0 || n_rows > (1 << 27) || n_vocab <= 0 || n_vocab > (1 << 30)) return bad(what, "n_rows must be in 0..2^27, n_vocab in 1..2^30");
    if (n_rows > 1 && row_stride < n_vocab) return bad(what, "row_stride is smaller than n_vocab");
    if (n_top < 0 || n_top > LOGPROB_MAX_TOP) return bad(what, "n_top must be in 0.." + std::to_string(LOGPROB_MAX_TOP));
    if (n_rows == 0) return B2_OK;
    if (!logits || (logprob && !tokens) || (n_top && (!top_logprob || !top_id))) return bad(what, "null device pointer");
    if ((uintptr_t)logits % elem_size(a.type) || ((uintptr_t)tokens | (uintptr_t)logprob | (uintptr_t)entropy | (uintptr_t)top_logprob | (uintptr_t)top_id) & 3)
        return bad(what, "pointers must be aligned to their elements");
    a.logits = logits; a.row_stride = row_stride; a.tokens = tokens; a.logprob = logprob; a.entropy = entropy; a.top_logprob = top_logprob; a.top_id = top_id;
    a.n_rows = n_rows; a.n_vocab = n_vocab; a.n_top = n_top;
    OnDevice on(device);
    return done(what, on.status != cudaSuccess ? on.status : logprobs_launch(a, (cudaStream_t)stream));
}

static int check_heads(const char* what, int n_head, int n_kv, int head_dim) {
    if (head_dim != 64 && head_dim != 128) return b2_fail(B2_ERR_UNSUPPORTED, std::string(what) + ": head_dim must be 64 or 128");
    if (n_kv <= 0 || n_kv > 65535 || n_head <= 0 || n_head % n_kv) return bad(what, "n_head must be a multiple of n_kv");
    if (n_head / n_kv > 64) return b2_fail(B2_ERR_UNSUPPORTED, std::string(what) + ": at most 64 heads a KV head");
    return B2_OK;
}

extern "C" int b2_attention_shared_prefix_workspace(int n_rows, int n_head, int n_kv, int head_dim, int64_t* bytes) {
    const char* what = "b2_attention_shared_prefix_workspace";
    if (int rc = check_heads(what, n_head, n_kv, head_dim)) return rc;
    if (!bytes || n_rows < 0) return bad(what, "null result or negative number of rows");
    if ((int64_t)n_rows * n_head > INT32_MAX) return bad(what, "rows * n_head must fit 32 bits");      // (as the call: prefix_cut counts units in an int)
    *bytes = n_rows ? (int64_t)shared_prefix_work_floats(n_rows, n_head, n_kv, head_dim) * 4 : 0;
    return B2_OK;
}

extern "C" int b2_attention_shared_prefix(int device, const b2_ragged_pages* where, const b2_shared_prefix_args* x, void* stream) {
    const char* what = "b2_attention_shared_prefix";
    if (!where || !x) return bad(what, "null arguments");
    SharedPrefixArgs a = {};
    if (int rc = check_where(what, *where, a.r)) return rc;
    if (int rc = check_heads(what, x->n_head, x->n_kv, x->head_dim)) return rc;
    a.type = elem_type(x->type);
    if (a.type != ELEM_F16 && a.type != ELEM_BF16) return b2_fail(B2_ERR_UNSUPPORTED, "b2_attention_shared_prefix: queries and cache must be f16 or bf16");
    if (x->n_prefix < 0 || x->n_prefix > (1 << 28)) return bad(what, "n_prefix out of range");
    if (x->max_rows <= 0) return bad(what, "max_rows must be positive");
    if ((int64_t)where->n_rows * x->n_head > INT32_MAX || (int64_t)x->max_rows * x->n_head > INT32_MAX) return bad(what, "rows * n_head must fit 32 bits");
    if (!(x->scale > 0.f) || !isfinite(x->scale)) return bad(what, "scale must be positive and finite");
    if (where->n_pages * where->block_tokens > INT32_MAX / x->n_kv) return bad(what, "n_pages * n_kv * block_tokens must fit 32 bits");
    if (where->n_rows == 0 || where->n_seqs == 0) return B2_OK;
    if (!x->q || !x->k_pool || !x->v_pool || !x->out || (x->n_prefix && (!x->prefix_pages || !x->workspace))) return bad(what, "null device pointer");
    if (((uintptr_t)x->k_pool | (uintptr_t)x->v_pool | (uintptr_t)x->workspace) & 15) return bad(what, "the pools and the workspace must be 16-byte aligned");
    if (((uintptr_t)x->q | (uintptr_t)x->out) & 1 || (uintptr_t)x->prefix_pages & 3) return bad(what, "pointers must be aligned to their elements");
    const int64_t need = x->n_prefix ? (int64_t)shared_prefix_work_floats(where->n_rows, x->n_head, x->n_kv, x->head_dim) * 4 : 0;
    if (x->workspace_bytes < need) return bad(what, "the workspace holds " + std::to_string(x->workspace_bytes) + " bytes, " + std::to_string(need) + " are needed");
    a.q = x->q; a.q_row = x->q_row; a.q_head = x->q_head; a.k_pool = x->k_pool; a.v_pool = x->v_pool; a.prefix_pages = x->prefix_pages; a.n_prefix = x->n_prefix;
    a.out = x->out; a.out_row = x->out_row; a.out_head = x->out_head; a.work = (float*)x->workspace;
    a.max_rows = x->max_rows < where->n_rows ? x->max_rows : where->n_rows;
    a.n_head = x->n_head; a.n_kv = x->n_kv; a.head_dim = x->head_dim; a.scale_log2 = x->scale * 1.4426950408889634f;
    OnDevice on(device);
    return done(what, on.status != cudaSuccess ? on.status : shared_prefix_launch(a, (cudaStream_t)stream));
}

extern "C" int b2_device_op_error(int device, uint32_t* code) {
    if (!code) return bad("b2_device_op_error", "null result");
    OnDevice on(device);
    if (on.status != cudaSuccess) return done("b2_device_op_error", on.status);
    return done("b2_device_op_error", shared_prefix_error(code));
}

extern "C" int b2_op_give_up(int device, int tensor_memory, uint32_t code, void* stream) {
    OnDevice on(device);
    return done("b2_op_give_up", on.status != cudaSuccess ? on.status : shared_prefix_give_up(code, tensor_memory != 0, (cudaStream_t)stream));
}

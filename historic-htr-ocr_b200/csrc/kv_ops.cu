// kv_ops.cu — the C ABI of the operators over a caller's KV cache (include/ocr_cuda.h): argument checks, workspaces and
// launches. The kernels are in k_kv_cache.cu, k_kv_attn.cu, k_kv_attn_one.cu and k_kv_attn_tc.cu.
#include "ctx.h"
#include "kv.cuh"

using namespace ocr;

namespace {

bool aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

ocr_status check_shape(const ocr_kv_cache* c) {
    if (!c) return fail(OCR_ERR_ARG, "null argument");
    if (c->type != OCR_KV_F16 && c->type != OCR_KV_Q8_0 && c->type != OCR_KV_Q4_0)
        return fail(OCR_ERR_ARG, "KV cache type " + std::to_string(c->type) + ": f16 (1), q4_0 (2) or q8_0 (8)");
    if (c->d_head != 64 && c->d_head != 128) return fail(OCR_ERR_ARG, "KV cache heads of 64 or 128 only");
    if (c->n_slot < 1 || c->n_slot > 65535 || c->n_kv < 1 || c->n_kv > 65535 || c->n_rows < 1)
        return fail(OCR_ERR_ARG, "KV cache shape out of range");
    if (c->window < 0 || c->sinks < 0) return fail(OCR_ERR_ARG, "KV cache window or sinks below 0");
    if (c->ring && (c->window < 1 || (long)c->sinks + c->window > c->n_rows))
        return fail(OCR_ERR_ARG, "a ring cache holds its sinks and its window: n_rows >= sinks + window, window >= 1");
    return OCR_OK;
}

ocr_status check_cache(const ocr_kv_cache* c) {
    OCR_TRY(check_shape(c));
    if (!c->k || !c->v || !aligned(c->k, 16) || !aligned(c->v, 16))
        return fail(OCR_ERR_ARG, "KV cache k and v must be 16-byte aligned device memory");
    if (c->type != OCR_KV_F16 && (!c->k_scale || !c->v_scale || !aligned(c->k_scale, 8) || !aligned(c->v_scale, 8)))
        return fail(OCR_ERR_ARG, "KV cache scales must be 8-byte aligned device memory");
    return OCR_OK;
}

ocr_status check_rows(const ocr_rows* r, const char* name) {
    if (!r || !r->data) return fail(OCR_ERR_ARG, std::string(name) + ": null argument");
    const size_t item = r->half ? 2 : 4;
    if (!aligned(r->data, 16) || (r->slot_stride * item) % 16 || (r->row_stride * item) % 16 ||
        (r->head_stride * item) % 16)
        return fail(OCR_ERR_ARG, std::string(name) + ": data and strides must be multiples of 16 bytes");
    return OCR_OK;
}

// (read: rows that the cache holds, which overwrites none)
ocr_status check_call(const ocr_kv_cache* c, int rows, const int32_t* d_pos, bool read = false) {
    if (!d_pos) return fail(OCR_ERR_ARG, "null argument");
    if (rows < 1) return fail(OCR_ERR_ARG, "rows must be at least 1");
    if (c->ring && !read ? rows > c->n_rows - c->sinks - c->window + 1 : rows > c->n_rows)
        return fail(OCR_ERR_ARG, "rows: more than the cache takes in one call");
    return OCR_OK;
}

KvView view(const ocr_kv_cache* c) {
    return {(uint8_t*)c->k, (uint8_t*)c->v, (__half*)c->k_scale, (__half*)c->v_scale, c->type, c->n_slot, c->n_kv,
            c->d_head, c->n_rows, c->window, c->sinks, c->ring ? 1 : 0};
}

ocr_status launched(cudaError_t e, const char* what) { return e == cudaSuccess ? OCR_OK : cuda_fail(e, what); }

ocr_status move(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* k, const ocr_rows* v, int rows,
                const int32_t* d_pos, const int32_t* d_n, bool write) {
    if (!ctx) return fail(OCR_ERR_ARG, "null argument");
    OCR_TRY(check_cache(c));
    OCR_TRY(check_rows(k, "k"));
    OCR_TRY(check_rows(v, "v"));
    if (!k->half != !v->half) return fail(OCR_ERR_ARG, "k and v must be of one type");
    OCR_TRY(check_call(c, rows, d_pos, !write));
    if ((double)rows * c->n_kv * (c->d_head / KV_BLOCK) * 8 > 4294967295.0)  // (the kernel counts a slot's threads in 32 bits)
        return fail(OCR_ERR_ARG, "rows: more than one launch takes");
    OCR_CUDA(cudaSetDevice(ctx->device));
    const KvMoveArgs a{view(c),       {d_pos, d_n, rows}, k->data,        v->data,       k->half ? 1 : 0, k->slot_stride,
                       k->row_stride, k->head_stride,     v->slot_stride, v->row_stride, v->head_stride,  ctx->d_err};
    return launched(write ? launch_kv_write(ctx->stream, a, ctx->pdl) : launch_kv_read(ctx->stream, a, ctx->pdl),
                    write ? "ocr_op_kv_write" : "ocr_op_kv_read");
}

// The attentions' workspace: made by a context's first such call, large enough for any, and kept as long as the context,
// since a captured step holds its address. Zero when it is made (the tickets count from zero, and each last arriver
// leaves zero).
ocr_status ensure_kv_work(ocr_ctx* ctx) {
    if (ctx->kv_work) return OCR_OK;
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    OCR_CUDA(cudaStreamIsCapturing(ctx->stream, &capture));
    if (capture != cudaStreamCaptureStatusNone)
        return fail(OCR_ERR_STATE, "a context's first attention over a KV cache makes its workspace: call one before capturing");
    const size_t n = kv_attention_work_bytes(ctx->num_sms);
    void* p = nullptr;
    const cudaError_t e = dalloc(&p, n, &ctx->mem_work);
    if (e != cudaSuccess) {
        if (p) dfree(p, n, &ctx->mem_work);
        return cuda_fail(e, "the KV attentions' workspace");
    }
    ctx->kv_work = p;
    return OCR_OK;
}

ocr_status attend(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* q, int n_head, int rows, const int32_t* d_pos,
                  const int32_t* d_n, const int32_t* d_parent, float scale, const ocr_rows* out, const char* what) {
    if (!ctx) return fail(OCR_ERR_ARG, "null argument");
    OCR_TRY(check_cache(c));
    OCR_TRY(check_rows(q, "q"));
    OCR_TRY(check_rows(out, "out"));
    if (!q->half != !out->half) return fail(OCR_ERR_ARG, "q and out must be of one type");
    OCR_TRY(check_call(c, rows, d_pos));
    if (n_head < 1 || n_head % c->n_kv) return fail(OCR_ERR_ARG, "n_head must be a multiple of n_kv");
    if (!(scale > 0.0f && scale <= 3.4e38f)) return fail(OCR_ERR_ARG, "scale must be positive and finite");
    if ((double)c->n_slot * rows * n_head > 1e9 || (double)rows * (n_head / c->n_kv) > (double)kv_attention_many_rows())
        return fail(OCR_ERR_ARG, "rows: more than one launch takes");
    KvAttnArgs a{view(c),        {d_pos, d_n, rows}, d_parent,         q->data,         out->data,
                 q->half ? 1 : 0, n_head,            q->slot_stride,   q->row_stride,   q->head_stride,
                 out->slot_stride, out->row_stride,  out->head_stride, scale,           nullptr,
                 ctx->num_sms,     ctx->d_err};
    if (kv_attention_many_slots(a) < 1) return fail(OCR_ERR_ARG, "rows: more than one launch takes");
    OCR_CUDA(cudaSetDevice(ctx->device));
    OCR_TRY(ensure_kv_work(ctx));
    a.work = ctx->kv_work;
    return launched(launch_kv_attention(ctx->stream, a, ctx->pdl), what);
}

}  // namespace

extern "C" {

ocr_status ocr_kv_cache_bytes(const ocr_kv_cache* c, size_t* quants, size_t* scales) {
    OCR_TRY(check_shape(c));
    if (!quants || !scales) return fail(OCR_ERR_ARG, "null argument");
    const size_t rows = (size_t)c->n_slot * c->n_kv * c->n_rows;
    *quants = rows * kv_row_bytes(c->type, c->d_head);
    *scales = c->type == OCR_KV_F16 ? 0 : rows * (c->d_head / KV_BLOCK) * 2;
    return OCR_OK;
}

ocr_status ocr_op_kv_write(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* k, const ocr_rows* v, int rows,
                           const int32_t* d_pos, const int32_t* d_n) {
    return move(ctx, c, k, v, rows, d_pos, d_n, true);
}

ocr_status ocr_op_kv_read(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* k, const ocr_rows* v, int rows,
                          const int32_t* d_pos, const int32_t* d_n) {
    return move(ctx, c, k, v, rows, d_pos, d_n, false);
}

ocr_status ocr_op_attention_window(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* q, int n_head, int rows,
                                   const int32_t* d_pos, const int32_t* d_n, float scale, const ocr_rows* out) {
    return attend(ctx, c, q, n_head, rows, d_pos, d_n, nullptr, scale, out, "ocr_op_attention_window");
}

ocr_status ocr_op_attention_tree(ocr_ctx* ctx, const ocr_kv_cache* c, const ocr_rows* q, int n_head, int rows,
                                 const int32_t* d_pos, const int32_t* d_n, const int32_t* d_parent, float scale,
                                 const ocr_rows* out) {
    if (!d_parent) return fail(OCR_ERR_ARG, "null argument");
    if (rows > KV_TREE_MAX) return fail(OCR_ERR_ARG, "a tree has at most 64 drafts");
    return attend(ctx, c, q, n_head, rows, d_pos, d_n, d_parent, scale, out, "ocr_op_attention_tree");
}

ocr_status ocr_op_kv_keep(ocr_ctx* ctx, const ocr_kv_cache* caches, int n_layer, int rows, const int32_t* d_pos,
                          const int32_t* d_path, const int32_t* d_n) {
    if (!ctx || !caches || !d_path || !d_n) return fail(OCR_ERR_ARG, "null argument");
    if (n_layer < 1 || n_layer > KV_KEEP_LAYERS) return fail(OCR_ERR_ARG, "n_layer must be 1 … 64");
    if (rows > KV_TREE_MAX) return fail(OCR_ERR_ARG, "a tree has at most 64 drafts");
    KvKeepArgs a{};
    for (int i = 0; i < n_layer; i++) {
        const ocr_kv_cache &c = caches[i], &f = caches[0];
        OCR_TRY(check_cache(&c));
        if (c.type != f.type || c.n_slot != f.n_slot || c.n_kv != f.n_kv || c.d_head != f.d_head ||
            c.n_rows != f.n_rows || c.sinks != f.sinks || !c.ring != !f.ring)
            return fail(OCR_ERR_ARG, "the layers' caches must be of one shape");
        OCR_TRY(check_call(&c, rows, d_pos));
        a.layer[i] = {(uint8_t*)c.k, (uint8_t*)c.v, (__half*)c.k_scale, (__half*)c.v_scale};
    }
    OCR_CUDA(cudaSetDevice(ctx->device));
    a.c = view(caches);
    a.n_layer = n_layer;
    a.T = rows;
    a.pos = d_pos;
    a.path = d_path;
    a.n = d_n;
    a.err = ctx->d_err;
    return launched(launch_kv_keep(ctx->stream, a, ctx->pdl), "ocr_op_kv_keep");
}

}  // extern "C"

// sp_fp8_runtime.cpp -- host side of the 8-bit block cache: its memory, the checks of a call's
// arguments, and the launches. No call but init and free allocates, copies or waits, so all of
// them may be captured into a graph.
#include "sp_block_runtime.h"

namespace {

using namespace sp_block;

SpFp8Side layer_side(const sp_hip_fp8_cache_t *c, int layer, bool v) {
    const size_t H = (size_t)c->config.n_heads_kv, at = (size_t)layer * c->n_blocks * H;
    SpFp8Side s;
    s.codes = (uint8_t *)(v ? c->d_v_codes : c->d_k_codes) + at * SP_FP8_BLOCK * c->config.head_dim;
    s.exps = (uint8_t *)(v ? c->d_v_exp : c->d_k_exp) + at;
    return s;
}

int copy_rows(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const void *k, const void *v,
              long long row_stride, int dtype, void *stream, bool write, const char *who) {
    SpFp8Copy A;
    memset(&A, 0, sizeof(A));
    const hipStream_t s = (hipStream_t)(stream || !c ? stream : c->stream);
    const int none = copy_ok(c, layer, b, k, v, row_stride, dtype, s, who, &A.s);
    if (none) return none < 0 ? -1 : 0;
    const OnDevice on(((const Priv *)c->priv)->device);
    if (!on.ok()) { sp_set_error("%s: the cache's device", who); return -1; }
    if (k) A.side[0] = layer_side(c, layer, false);
    if (v) A.side[1] = layer_side(c, layer, true);
    A.rows[0] = const_cast<void *>(k);
    A.rows[1] = const_cast<void *>(v);
    A.row_stride = row_stride;
    A.H = c->config.n_heads_kv;
    const int four = dtype == SP_DTYPE_F32 ? 16 : 8;
    A.aligned = row_stride % 4 == 0 && (uintptr_t)k % four == 0 && (uintptr_t)v % four == 0;
    return ok(write ? sp_fp8_launch_write(A, c->config.head_dim, dtype, s)
                    : sp_fp8_launch_read(A, c->config.head_dim, dtype, s), who) ? 0 : -1;
}

}  // namespace

extern "C" int sp_hip_fp8_cache_init(sp_hip_fp8_cache_t *c, const sp_config_t *cfg, int n_blocks, void *stream) {
    const char *who = "fp8_cache_init";
    const size_t nexp = init_ok(c, cfg, n_blocks, who);
    if (!nexp) return -1;
    const int hd = cfg->head_dim;
    Priv *pv = new (std::nothrow) Priv();
    if (!pv) { sp_set_error("%s: out of memory", who); return -1; }
    c->config = *cfg;
    c->n_blocks = n_blocks;
    c->stream = stream;
    c->priv = pv;
    const hipStream_t s = (hipStream_t)stream;
    bool good = ok(hipGetDevice(&pv->device), who) && stream_ok(c, s, who) &&
                ok(hipDeviceGetAttribute(&pv->cus, hipDeviceAttributeMultiprocessorCount, pv->device), who);
    const size_t ncode = nexp * SP_FP8_BLOCK * hd;
    pv->ws[0].rows = SP_FP8_DECODE_ROWS;
    pv->ws[1].rows = sp_fp8_prefill_rows(hd);
    Places at;
    // cleared to 0: codes and counters; to the least exponent: exponents; not cleared: partial results
    const size_t k_at = at.add(ncode), v_at = at.add(ncode), count_at = at.add(2 * SP_FP8_SLOTS * sizeof(int)),
                 ke_at = at.add(nexp), ve_at = at.add(nexp);
    const size_t p0_at = at.add((size_t)pv->ws[0].rows * (hd + 4) * sizeof(float));
    const size_t p1_at = at.add((size_t)pv->ws[1].rows * (hd + 4) * sizeof(float));
    good = good && ok(hipMalloc(&pv->memory, at.size), who) && ok(hipMemsetAsync(pv->memory, 0, ke_at, s), who) &&
           ok(hipMemsetAsync((char *)pv->memory + ke_at, 127 + SP_FP8_EMIN, p0_at - ke_at, s), who);
    if (good) {
        char *base = (char *)pv->memory;
        c->d_k_codes = base + k_at;
        c->d_v_codes = base + v_at;
        c->d_k_exp = base + ke_at;
        c->d_v_exp = base + ve_at;
        pv->ws[0].part = (float *)(base + p0_at);
        pv->ws[1].part = (float *)(base + p1_at);
        pv->ws[0].counters = (int *)(base + count_at);
        pv->ws[1].counters = pv->ws[0].counters + SP_FP8_SLOTS;
    }
    good = good && ok(hipStreamSynchronize(s), who);
    return good ? 0 : init_failed(c, sp_hip_fp8_cache_free);
}

extern "C" void sp_hip_fp8_cache_free(sp_hip_fp8_cache_t *c) { free_cache(c); }

extern "C" int sp_hip_fp8_write(sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch, const void *d_k,
                                const void *d_v, long long row_stride, int dtype, void *stream) {
    return copy_rows(c, layer, batch, d_k, d_v, row_stride, dtype, stream, true, "fp8_write");
}

extern "C" int sp_hip_fp8_read(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch, void *d_k,
                               void *d_v, long long row_stride, int dtype, void *stream) {
    return copy_rows(c, layer, batch, d_k, d_v, row_stride, dtype, stream, false, "fp8_read");
}

extern "C" int sp_hip_fp8_attn_decode(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch,
                                      const void *d_q, long long q_stride, int n_q, int dtype, float kq_scale,
                                      int window, void *d_out, long long out_stride, float *d_lse, void *stream) {
    if (batch && batch->d_row) {
        sp_set_error("fp8_attn_decode: one row per sequence (d_row NULL); fp8_attn_prefill takes more");
        return -1;
    }
    return attend(c, layer, batch, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, stream,
                  0, "fp8_attn_decode", layer_side, sp_fp8_launch_attn);
}

extern "C" int sp_hip_fp8_attn_prefill(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch,
                                       const void *d_q, long long q_stride, int n_q, int dtype, float kq_scale,
                                       int window, void *d_out, long long out_stride, float *d_lse, void *stream) {
    return attend(c, layer, batch, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, stream,
                  1, "fp8_attn_prefill", layer_side, sp_fp8_launch_attn);
}

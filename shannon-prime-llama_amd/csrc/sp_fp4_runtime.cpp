// sp_fp4_runtime.cpp -- host side of the 4-bit block cache: its memory, the checks of a call's
// arguments, and the launches. No call but init and free allocates, copies or waits, so all of
// them may be captured into a graph.
#include "sp_block_runtime.h"
#include "sp_fp4.h"

namespace {

using namespace sp_block;

// (layer, block, KV head) of a layer's first tile
size_t first_tile(const sp_hip_fp4_cache_t *c, int layer) {
    return (size_t)layer * c->n_blocks * c->config.n_heads_kv;
}

SpFp8Side layer_side(const sp_hip_fp4_cache_t *c, int layer, bool v) {
    const size_t at = first_tile(c, layer);
    SpFp8Side s;
    s.codes = (uint8_t *)(v ? c->d_v_codes : c->d_k_codes) + at * sp_fp4_tile(c->config.head_dim);
    s.exps = (uint8_t *)(v ? c->d_v_exp : c->d_k_exp) + at * sp_fp4_exps(c->config.head_dim);
    return s;
}

float *layer_weight(const sp_hip_fp4_cache_t *c, int layer) { return c->d_weight + first_tile(c, layer) * SP_FP4_BLOCK; }

int copy_rows(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const void *k, const void *v,
              long long row_stride, int dtype, void *stream, bool write, const char *who) {
    SpFp4Copy A;
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
    A.weight = layer_weight(c, layer);
    A.row_stride = row_stride;
    A.H = c->config.n_heads_kv;
    const uintptr_t at = (uintptr_t)k | (uintptr_t)v;
    const int esize = dtype == SP_DTYPE_F32 ? 4 : 2;
    A.aligned = row_stride % 8 == 0 && at % 16 == 0 ? 8 : row_stride % 4 == 0 && at % (4 * esize) == 0 ? 4 : 1;
    return ok(write ? sp_fp4_launch_write(A, c->config.head_dim, dtype, s)
                    : sp_fp4_launch_read(A, c->config.head_dim, dtype, s), who) ? 0 : -1;
}

}  // namespace

extern "C" int sp_hip_fp4_cache_init(sp_hip_fp4_cache_t *c, const sp_config_t *cfg, int n_blocks, void *stream) {
    const char *who = "fp4_cache_init";
    const size_t tiles = init_ok(c, cfg, n_blocks, who);
    if (!tiles) return -1;
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
    const size_t ncode = tiles * sp_fp4_tile(hd), nexp = tiles * sp_fp4_exps(hd);
    pv->ws[0].rows = SP_FP8_DECODE_ROWS;
    pv->ws[1].rows = sp_fp8_prefill_rows(hd);
    Places at;
    // cleared to 0: codes, weights and counters; to the least exponent: exponents; not cleared: partial results
    const size_t k_at = at.add(ncode), v_at = at.add(ncode),
                 w_at = at.add(tiles * SP_FP4_BLOCK * sizeof(float)), count_at = at.add(2 * SP_FP8_SLOTS * sizeof(int)),
                 ke_at = at.add(nexp), ve_at = at.add(nexp);
    const size_t p0_at = at.add((size_t)pv->ws[0].rows * (hd + 4) * sizeof(float));
    const size_t p1_at = at.add((size_t)pv->ws[1].rows * (hd + 4) * sizeof(float));
    good = good && ok(hipMalloc(&pv->memory, at.size), who) && ok(hipMemsetAsync(pv->memory, 0, ke_at, s), who) &&
           ok(hipMemsetAsync((char *)pv->memory + ke_at, SP_FP4_LEAST, p0_at - ke_at, s), who);
    if (good) {
        char *base = (char *)pv->memory;
        c->d_k_codes = base + k_at;
        c->d_v_codes = base + v_at;
        c->d_k_exp = base + ke_at;
        c->d_v_exp = base + ve_at;
        c->d_weight = (float *)(base + w_at);
        pv->ws[0].part = (float *)(base + p0_at);
        pv->ws[1].part = (float *)(base + p1_at);
        pv->ws[0].counters = (int *)(base + count_at);
        pv->ws[1].counters = pv->ws[0].counters + SP_FP8_SLOTS;
    }
    good = good && ok(hipStreamSynchronize(s), who);
    return good ? 0 : init_failed(c, sp_hip_fp4_cache_free);
}

extern "C" void sp_hip_fp4_cache_free(sp_hip_fp4_cache_t *c) { free_cache(c); }

extern "C" int sp_hip_fp4_write(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch, const void *d_k,
                                const void *d_v, long long row_stride, int dtype, void *stream) {
    return copy_rows(c, layer, batch, d_k, d_v, row_stride, dtype, stream, true, "fp4_write");
}

extern "C" int sp_hip_fp4_read(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch, void *d_k,
                               void *d_v, long long row_stride, int dtype, void *stream) {
    return copy_rows(c, layer, batch, d_k, d_v, row_stride, dtype, stream, false, "fp4_read");
}

extern "C" int sp_hip_fp4_attn_decode(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch,
                                      const void *d_q, long long q_stride, int n_q, int dtype, float kq_scale,
                                      int window, void *d_out, long long out_stride, float *d_lse, void *stream) {
    if (batch && batch->d_row) {
        sp_set_error("fp4_attn_decode: one row per sequence (d_row NULL); fp4_attn_prefill takes more");
        return -1;
    }
    return attend(c, layer, batch, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, stream,
                  0, "fp4_attn_decode", layer_side, sp_fp4_launch_attn);
}

extern "C" int sp_hip_fp4_attn_prefill(const sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch,
                                       const void *d_q, long long q_stride, int n_q, int dtype, float kq_scale,
                                       int window, void *d_out, long long out_stride, float *d_lse, void *stream) {
    return attend(c, layer, batch, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, stream,
                  1, "fp4_attn_prefill", layer_side, sp_fp4_launch_attn);
}

extern "C" int sp_hip_fp4_weigh(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const void *d_q,
                                long long q_stride, int n_q, int dtype, float kq_scale, int window,
                                const float *d_lse, void *stream) {
    const char *who = "fp4_weigh";
    SpFp4Weigh A;
    memset(&A, 0, sizeof(A));
    const hipStream_t s = (hipStream_t)(stream || !c ? stream : c->stream);
    const int none = query_ok(c, layer, b, d_q, q_stride, n_q, dtype, kq_scale, window, nullptr, q_stride, d_lse, s, who, &A.s);
    if (none) return none < 0 ? -1 : 0;
    if (!d_q || !d_lse) { sp_set_error("%s: q and lse", who); return -1; }
    const Priv *pv = (const Priv *)c->priv;
    const OnDevice on(pv->device);
    if (!on.ok()) { sp_set_error("%s: the cache's device", who); return -1; }
    A.k = layer_side(c, layer, false);
    A.q = d_q;
    A.lse = d_lse;
    A.weight = layer_weight(c, layer);
    A.q_stride = q_stride;
    A.H = c->config.n_heads_kv;
    A.G = n_q / A.H;
    A.window = window >= MAX_ROWS ? 0 : window;  // no position is that far
    const double log2e = 1.4426950408889634074, unit = fabs((double)kq_scale) * (log2e / 2);
    A.c = (float)unit;
    A.lost = (float)((A.c >= 0x1p-126f ? unit / A.c - 1.0 : 0.0) * log2e - (log2e - (float)log2e));
    A.negate = kq_scale < 0.0f;
    A.cus = pv->cus;
    return ok(sp_fp4_launch_weigh(A, c->config.head_dim, dtype, s), who) ? 0 : -1;
}

extern "C" int sp_hip_fp4_evict(sp_hip_fp4_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, int keep, int first,
                                int recent, int32_t *d_kept, void *stream) {
    const char *who = "fp4_evict";
    SpFp4Evict A;
    memset(&A, 0, sizeof(A));
    if (!batch_ok(c, layer, b, who, &A.s)) return -1;
    A.s.row = nullptr;
    if (keep < 1 || keep > MAX_ROWS || first < 0 || recent < 0 || first > keep || recent > keep - first) {
        sp_set_error("%s: keep %d with the first %d and the last %d", who, keep, first, recent);
        return -1;
    }
    if ((uintptr_t)d_kept % 4) { sp_set_error("%s: kept is an array of int32 at a multiple of 4 bytes", who); return -1; }
    const hipStream_t s = (hipStream_t)(stream ? stream : c->stream);
    if (!stream_ok(c, s, who)) return -1;
    if (b->n_seq == 0) return 0;
    if (!d_kept) { sp_set_error("%s: kept", who); return -1; }
    A.H = c->config.n_heads_kv;
    if ((long long)b->n_seq * A.H * SP_FP4_EVICT_THREADS > SP_FP8_MOST_THREADS) {
        sp_set_error("%s: too many sequences", who);
        return -1;
    }
    const OnDevice on(((const Priv *)c->priv)->device);
    if (!on.ok()) { sp_set_error("%s: the cache's device", who); return -1; }
    for (int v = 0; v < 2; v++) A.side[v] = layer_side(c, layer, v != 0);
    A.weight = layer_weight(c, layer);
    A.kept = d_kept;
    A.NC = c->config.head_dim / 32;
    A.keep = keep;
    A.first = first;
    A.recent = recent;
    return ok(sp_fp4_launch_evict(A, s), who) ? 0 : -1;
}

// sp_fp8_runtime.cpp -- host side of the 8-bit block cache: its memory, the checks of a call's
// arguments, and the launches. No call but init and free allocates, copies or waits, so all of
// them may be captured into a graph.
#include <hip/hip_runtime.h>

#include <math.h>
#include <string.h>

#include <new>

#include "sp_fp8.h"
#include "sp_internal.h"

namespace {

// Partial results of attention calls and the arrival counts of their shares: one for decode calls
// and one for prefill calls, so that one of each may be under way on two streams.
struct Workspace {
    float *part = nullptr;
    int *counters = nullptr;
    int rows = 0;
};

struct Fp8Priv {
    int device = 0, cus = 256;
    void *memory = nullptr;  // codes, exponents and workspaces: one allocation
    Workspace ws[2];
};

// The cache's device for the length of a call (the caller's current device may be another).
class OnDevice {
public:
    explicit OnDevice(int dev) {
        if (hipGetDevice(&before_) != hipSuccess) before_ = dev;
        if (before_ != dev) ok_ = hipSetDevice(dev) == hipSuccess;
        else before_ = -1;
    }
    ~OnDevice() {
        if (before_ >= 0) (void)hipSetDevice(before_);
    }
    bool ok() const { return ok_; }

private:
    int before_ = -1;
    bool ok_ = true;
};

bool ok(hipError_t e, const char *what) {
    if (e == hipSuccess) return true;
    sp_set_error("%s: %s", what, hipGetErrorString(e));
    (void)hipGetLastError();  // reported here: not left for the next reader of the device's last error
    return false;
}

bool dtype_ok(int dtype) { return dtype == SP_DTYPE_F32 || dtype == SP_DTYPE_F16 || dtype == SP_DTYPE_BF16; }

constexpr int MAX_ROWS = 1 << 30;    // positions and rows: differences of them stay in an int
constexpr int MAX_STRIDE = 1 << 24;  // table entries of a sequence, 64 positions each
constexpr long long MAX_ELEMS = 1ll << 62;

// The sequences of a call, checked as far as the host sees them.
bool batch_ok(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const char *who, SpFp8Seqs *S) {
    if (!c || !c->priv) { sp_set_error("%s: bad cache", who); return false; }
    if (layer < 0 || layer >= c->config.n_layers) {
        sp_set_error("%s: layer %d of %d", who, layer, c->config.n_layers);
        return false;
    }
    if (!b || b->n_seq < 0 || b->n_rows < 0 || b->n_rows > MAX_ROWS || b->n_seq > MAX_ROWS) {
        sp_set_error("%s: bad batch", who);
        return false;
    }
    if (!b->d_row && b->n_rows != b->n_seq) {
        sp_set_error("%s: without d_row there is one row per sequence (%d rows, %d sequences)", who, b->n_rows, b->n_seq);
        return false;
    }
    if (b->n_seq > 0 && (!b->d_table || !b->d_len || b->table_stride < 1 || b->table_stride > MAX_STRIDE)) {
        sp_set_error("%s: a batch needs d_table, d_len and 1 <= table_stride <= %d", who, MAX_STRIDE);
        return false;
    }
    if (((uintptr_t)b->d_table | (uintptr_t)b->d_len | (uintptr_t)b->d_row) % 4) {
        sp_set_error("%s: d_table, d_len and d_row are arrays of int32 at multiples of 4 bytes", who);
        return false;
    }
    S->table = b->d_table;
    S->len = b->d_len;
    S->row = b->d_row;
    S->n_seq = b->n_seq;
    S->stride = b->table_stride;
    S->n_rows = b->n_rows;
    S->n_blocks = c->n_blocks;
    return true;
}

bool stream_ok(const sp_hip_fp8_cache_t *c, hipStream_t s, const char *who) {
    const Fp8Priv *pv = (const Fp8Priv *)c->priv;
    if (!s) return true;
    hipDevice_t d = -1;
    if (!ok(hipStreamGetDevice(s, &d), who)) return false;
    if (d != pv->device) {
        sp_set_error("%s: the cache is on device %d, the stream on device %d", who, pv->device, (int)d);
        return false;
    }
    return true;
}

SpFp8Side layer_side(const sp_hip_fp8_cache_t *c, int layer, bool v) {
    const size_t H = (size_t)c->config.n_heads_kv, at = (size_t)layer * c->n_blocks * H;
    SpFp8Side s;
    s.codes = (uint8_t *)(v ? c->d_v_codes : c->d_k_codes) + at * SP_FP8_BLOCK * c->config.head_dim;
    s.exps = (uint8_t *)(v ? c->d_v_exp : c->d_k_exp) + at;
    return s;
}

// esize bytes per element: the pointer is a multiple of it
bool aligned_to(const void *p, int dtype) { return (uintptr_t)p % (dtype == SP_DTYPE_F32 ? 4 : 2) == 0; }

int copy_rows(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const void *k, const void *v,
              long long row_stride, int dtype, void *stream, bool write, const char *who) {
    SpFp8Copy A;
    memset(&A, 0, sizeof(A));
    if (!batch_ok(c, layer, b, who, &A.s)) return -1;
    if (!dtype_ok(dtype)) { sp_set_error("%s: dtype %d", who, dtype); return -1; }
    const int hd = c->config.head_dim, H = c->config.n_heads_kv;
    if (row_stride < (long long)H * hd || row_stride > MAX_ELEMS / MAX_ROWS) {
        sp_set_error("%s: row_stride %lld for %d heads of %d", who, row_stride, H, hd);
        return -1;
    }
    if (!aligned_to(k, dtype) || !aligned_to(v, dtype)) {
        sp_set_error("%s: rows are not at a multiple of their element's size", who);
        return -1;
    }
    const hipStream_t s = (hipStream_t)(stream ? stream : c->stream);
    if (!stream_ok(c, s, who)) return -1;
    if (b->n_rows == 0 || b->n_seq == 0 || (!k && !v)) return 0;
    if (((long long)b->n_rows / 64 + 2ll * b->n_seq) * SP_FP8_COPY_THREADS > SP_FP8_MOST_THREADS) {
        sp_set_error("%s: too many rows or sequences", who);
        return -1;
    }
    const OnDevice on(((const Fp8Priv *)c->priv)->device);
    if (!on.ok()) { sp_set_error("%s: the cache's device", who); return -1; }
    if (k) A.side[0] = layer_side(c, layer, false);
    if (v) A.side[1] = layer_side(c, layer, true);
    A.rows[0] = const_cast<void *>(k);
    A.rows[1] = const_cast<void *>(v);
    A.row_stride = row_stride;
    A.H = H;
    const int four = dtype == SP_DTYPE_F32 ? 16 : 8;
    A.aligned = row_stride % 4 == 0 && (uintptr_t)k % four == 0 && (uintptr_t)v % four == 0;
    return ok(write ? sp_fp8_launch_write(A, hd, dtype, s) : sp_fp8_launch_read(A, hd, dtype, s), who) ? 0 : -1;
}

int attend(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *b, const void *d_q, long long q_stride,
           int n_q, int dtype, float kq_scale, int window, void *d_out, long long out_stride, float *d_lse,
           void *stream, int which, const char *who) {
    SpFp8Attn A;
    memset(&A, 0, sizeof(A));
    if (!batch_ok(c, layer, b, who, &A.s)) return -1;
    if (!dtype_ok(dtype)) { sp_set_error("%s: dtype %d", who, dtype); return -1; }
    const int hd = c->config.head_dim, H = c->config.n_heads_kv;
    if (n_q <= 0 || n_q % H || (long long)n_q * hd > (1 << 30)) {
        sp_set_error("%s: n_q %d must be a positive multiple of n_heads_kv %d", who, n_q, H);
        return -1;
    }
    if (!isfinite(kq_scale)) { sp_set_error("%s: kq_scale is not finite", who); return -1; }
    if (window < 0) { sp_set_error("%s: window %d", who, window); return -1; }
    for (const long long st : {q_stride, out_stride})
        if (st < (long long)n_q * hd || st > MAX_ELEMS / MAX_ROWS) {
            sp_set_error("%s: row strides of q and out are at least n_q * head_dim", who);
            return -1;
        }
    if (!aligned_to(d_q, dtype) || !aligned_to(d_out, dtype) || (uintptr_t)d_lse % 4) {
        sp_set_error("%s: q, out or lse is not at a multiple of its element's size", who);
        return -1;
    }
    const hipStream_t s = (hipStream_t)(stream ? stream : c->stream);
    if (!stream_ok(c, s, who)) return -1;
    if (b->n_rows == 0 || b->n_seq == 0) return 0;
    if (!d_q || !d_out) { sp_set_error("%s: q and out", who); return -1; }
    if ((long long)b->n_rows * (n_q / H) > MAX_ROWS) { sp_set_error("%s: too many rows", who); return -1; }
    const Fp8Priv *pv = (const Fp8Priv *)c->priv;
    const OnDevice on(pv->device);
    if (!on.ok()) { sp_set_error("%s: the cache's device", who); return -1; }
    A.k = layer_side(c, layer, false);
    A.v = layer_side(c, layer, true);
    A.q = d_q;
    A.out = d_out;
    A.lse = d_lse;
    A.q_stride = q_stride;
    A.out_stride = out_stride;
    A.H = H;
    A.G = n_q / H;
    A.window = window >= MAX_ROWS ? 0 : window;  // no position is that far
    A.c = fabsf(kq_scale) * 0.72134752044448170f;
    A.negate = kq_scale < 0.0f;
    A.part = pv->ws[which].part;
    A.counters = pv->ws[which].counters;
    A.part_rows = pv->ws[which].rows;
    A.target = pv->cus;
    return ok(sp_fp8_launch_attn(A, hd, dtype, s), who) ? 0 : -1;
}

}  // namespace

extern "C" int sp_hip_fp8_cache_init(sp_hip_fp8_cache_t *c, const sp_config_t *cfg, int n_blocks, void *stream) {
    const char *who = "fp8_cache_init";
    if (!c) { sp_set_error("%s: no cache", who); return -1; }
    memset(c, 0, sizeof(*c));
    if (!cfg || cfg->n_layers <= 0 || cfg->n_heads_kv <= 0 || cfg->n_heads_kv > 65535 || n_blocks <= 0) {
        sp_set_error("%s: bad config", who);
        return -1;
    }
    const int hd = cfg->head_dim;
    if (hd != 64 && hd != 96 && hd != 128 && hd != 256) {
        sp_set_error("%s: head_dim %d (64, 96, 128 or 256)", who, hd);
        return -1;
    }
    // codes of one side: n_layers * n_blocks * n_heads_kv tiles
    const unsigned __int128 tiles = (unsigned __int128)cfg->n_layers * n_blocks * cfg->n_heads_kv;
    if (tiles * SP_FP8_BLOCK * hd > ((unsigned __int128)1 << 50)) { sp_set_error("%s: too large", who); return -1; }
    if (!sp_hip_available()) { sp_set_error("%s: no gfx950 device", who); return -1; }
    Fp8Priv *pv = new (std::nothrow) Fp8Priv();
    if (!pv) { sp_set_error("%s: out of memory", who); return -1; }
    c->config = *cfg;
    c->n_blocks = n_blocks;
    c->stream = stream;
    c->priv = pv;
    const hipStream_t s = (hipStream_t)stream;
    bool good = ok(hipGetDevice(&pv->device), who) && stream_ok(c, s, who) &&
                ok(hipDeviceGetAttribute(&pv->cus, hipDeviceAttributeMultiprocessorCount, pv->device), who);
    const size_t nexp = (size_t)tiles, ncode = nexp * SP_FP8_BLOCK * hd;
    pv->ws[0].rows = SP_FP8_DECODE_ROWS;
    pv->ws[1].rows = sp_fp8_prefill_rows(hd);
    size_t size = 0;
    const auto place = [&size](size_t bytes) {
        const size_t at = size;
        size += (bytes + 255) / 256 * 256;
        return at;
    };
    // cleared to 0: codes and counters; to the least exponent: exponents; not cleared: partial results
    const size_t k_at = place(ncode), v_at = place(ncode), count_at = place(2 * SP_FP8_SLOTS * sizeof(int)),
                 ke_at = place(nexp), ve_at = place(nexp);
    const size_t p0_at = place((size_t)pv->ws[0].rows * (hd + 4) * sizeof(float));
    const size_t p1_at = place((size_t)pv->ws[1].rows * (hd + 4) * sizeof(float));
    good = good && ok(hipMalloc(&pv->memory, size), who) && ok(hipMemsetAsync(pv->memory, 0, ke_at, s), who) &&
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
    if (!good) {
        char why[256];
        strncpy(why, sp_hip_last_error(), sizeof(why) - 1);
        why[sizeof(why) - 1] = 0;
        sp_hip_fp8_cache_free(c);
        sp_set_error("%s", why);
        return -1;
    }
    return 0;
}

extern "C" void sp_hip_fp8_cache_free(sp_hip_fp8_cache_t *c) {
    if (!c) return;
    Fp8Priv *pv = (Fp8Priv *)c->priv;
    if (pv) {
        const OnDevice on(pv->device);
        if (pv->memory) (void)hipFree(pv->memory);
        delete pv;
    }
    memset(c, 0, sizeof(*c));
}

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
                  0, "fp8_attn_decode");
}

extern "C" int sp_hip_fp8_attn_prefill(const sp_hip_fp8_cache_t *c, int layer, const sp_hip_fp8_batch_t *batch,
                                       const void *d_q, long long q_stride, int n_q, int dtype, float kq_scale,
                                       int window, void *d_out, long long out_stride, float *d_lse, void *stream) {
    return attend(c, layer, batch, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, stream,
                  1, "fp8_attn_prefill");
}

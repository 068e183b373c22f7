// sp_block_runtime.h -- what the host sides of the block caches (sp_fp8_runtime.cpp, sp_fp4_runtime.cpp)
// share: the checks of a call's arguments, the device of a call, and attention calls. A Cache is
// sp_hip_fp8_cache_t or sp_hip_fp4_cache_t.
#pragma once

#include <hip/hip_runtime.h>

#include <math.h>
#include <string.h>

#include <new>

#include "sp_fp8.h"
#include "sp_internal.h"

namespace sp_block {

// Partial results of attention calls and the arrival counts of their shares: one for decode calls
// and one for prefill calls, so that one of each may be under way on two streams.
struct Workspace {
    float *part = nullptr;
    int *counters = nullptr;
    int rows = 0;
};

struct Priv {
    int device = 0, cus = 256;
    void *memory = nullptr;  // what the cache holds and its workspaces: one allocation
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

inline bool ok(hipError_t e, const char *what) {
    if (e == hipSuccess) return true;
    sp_set_error("%s: %s", what, hipGetErrorString(e));
    (void)hipGetLastError();  // reported here: not left for the next reader of the device's last error
    return false;
}

inline bool dtype_ok(int dtype) { return dtype == SP_DTYPE_F32 || dtype == SP_DTYPE_F16 || dtype == SP_DTYPE_BF16; }

constexpr int MAX_ROWS = 1 << 30;    // positions and rows: differences of them stay in an int
constexpr int MAX_STRIDE = 1 << 24;  // table entries of a sequence, 64 positions each
constexpr long long MAX_ELEMS = 1ll << 62;

// The sequences of a call, checked as far as the host sees them.
template <class Cache>
bool batch_ok(const Cache *c, int layer, const sp_hip_fp8_batch_t *b, const char *who, SpFp8Seqs *S) {
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

template <class Cache>
bool stream_ok(const Cache *c, hipStream_t s, const char *who) {
    const Priv *pv = (const Priv *)c->priv;
    if (!s) return true;
    hipDevice_t d = -1;
    if (!ok(hipStreamGetDevice(s, &d), who)) return false;
    if (d != pv->device) {
        sp_set_error("%s: the cache is on device %d, the stream on device %d", who, pv->device, (int)d);
        return false;
    }
    return true;
}

// esize bytes per element: the pointer is a multiple of it
inline bool aligned_to(const void *p, int dtype) { return (uintptr_t)p % (dtype == SP_DTYPE_F32 ? 4 : 2) == 0; }

// The checks of write and read; 1: nothing to do.
template <class Cache>
int copy_ok(const Cache *c, int layer, const sp_hip_fp8_batch_t *b, const void *k, const void *v, long long row_stride,
            int dtype, hipStream_t s, const char *who, SpFp8Seqs *S) {
    if (!batch_ok(c, layer, b, who, S)) return -1;
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
    if (!stream_ok(c, s, who)) return -1;
    if (b->n_rows == 0 || b->n_seq == 0 || (!k && !v)) return 1;
    if (((long long)b->n_rows / 64 + 2ll * b->n_seq) * SP_FP8_COPY_THREADS > SP_FP8_MOST_THREADS) {
        sp_set_error("%s: too many rows or sequences", who);
        return -1;
    }
    return 0;
}

// The checks of calls with queries; 1: nothing to do. d_out NULL: the call has no output rows.
template <class Cache>
int query_ok(const Cache *c, int layer, const sp_hip_fp8_batch_t *b, const void *d_q, long long q_stride, int n_q,
             int dtype, float kq_scale, int window, const void *d_out, long long out_stride, const float *d_lse,
             hipStream_t s, const char *who, SpFp8Seqs *S) {
    if (!batch_ok(c, layer, b, who, S)) return -1;
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
    if (!stream_ok(c, s, who)) return -1;
    if (b->n_rows == 0 || b->n_seq == 0) return 1;
    if ((long long)b->n_rows * (n_q / H) > MAX_ROWS) { sp_set_error("%s: too many rows", who); return -1; }
    return 0;
}

// layer_side(c, layer, is_v): where a side of a layer lies; launch: the format's attention.
template <class Cache, class Side, class Launch>
int attend(const Cache *c, int layer, const sp_hip_fp8_batch_t *b, const void *d_q, long long q_stride,
           int n_q, int dtype, float kq_scale, int window, void *d_out, long long out_stride, float *d_lse,
           void *stream, int which, const char *who, Side layer_side, Launch launch) {
    SpFp8Attn A;
    memset(&A, 0, sizeof(A));
    const hipStream_t s = (hipStream_t)(stream || !c ? stream : c->stream);
    const int none = query_ok(c, layer, b, d_q, q_stride, n_q, dtype, kq_scale, window, d_out, out_stride, d_lse, s, who, &A.s);
    if (none) return none < 0 ? -1 : 0;
    if (!d_q || !d_out) { sp_set_error("%s: q and out", who); return -1; }
    const int hd = c->config.head_dim, H = c->config.n_heads_kv;
    const Priv *pv = (const Priv *)c->priv;
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
    return ok(launch(A, hd, dtype, s), who) ? 0 : -1;
}

// The checks of init, which leave `c` empty where they fail: the number of tiles of one side, or 0.
template <class Cache>
size_t init_ok(Cache *c, const sp_config_t *cfg, int n_blocks, const char *who) {
    if (!c) { sp_set_error("%s: no cache", who); return 0; }
    memset(c, 0, sizeof(*c));
    if (!cfg || cfg->n_layers <= 0 || cfg->n_heads_kv <= 0 || cfg->n_heads_kv > 65535 || n_blocks <= 0) {
        sp_set_error("%s: bad config", who);
        return 0;
    }
    const int hd = cfg->head_dim;
    if (hd != 64 && hd != 96 && hd != 128 && hd != 256) {
        sp_set_error("%s: head_dim %d (64, 96, 128 or 256)", who, hd);
        return 0;
    }
    const unsigned __int128 tiles = (unsigned __int128)cfg->n_layers * n_blocks * cfg->n_heads_kv;
    if (tiles * SP_FP8_BLOCK * hd > ((unsigned __int128)1 << 50)) { sp_set_error("%s: too large", who); return 0; }
    if (!sp_hip_available()) { sp_set_error("%s: no gfx950 device", who); return 0; }
    return (size_t)tiles;
}

// Places of a cache's parts in its one allocation.
struct Places {
    size_t size = 0;
    size_t add(size_t bytes) {
        const size_t at = size;
        size += (bytes + 255) / 256 * 256;
        return at;
    }
};

// Frees what a failed init has, and leaves its reason as the last error.
template <class Cache>
int init_failed(Cache *c, void (*free_cache)(Cache *)) {
    char why[256];
    strncpy(why, sp_hip_last_error(), sizeof(why) - 1);
    why[sizeof(why) - 1] = 0;
    free_cache(c);
    sp_set_error("%s", why);
    return -1;
}

template <class Cache>
void free_cache(Cache *c) {
    if (!c) return;
    Priv *pv = (Priv *)c->priv;
    if (pv) {
        const OnDevice on(pv->device);
        if (pv->memory) (void)hipFree(pv->memory);
        delete pv;
    }
    memset(c, 0, sizeof(*c));
}

}  // namespace sp_block

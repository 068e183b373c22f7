// sp_fp8_attn.hip -- attention over the 8-bit block cache, for one or more query tokens per
// sequence.
//
// For the row of query head n at position p of its sequence, over the positions t <= p (and
// t > p - window), with k_t = 2^ek(t) K_t and v_t = 2^ev(t) V_t the block's codes and scales:
//   s_t = kq_scale * q . k_t,   out = sum_t e^{s_t - m} v_t / sum_t e^{s_t - m},   lse = m + log(sum)
// in one pass over the blocks with the running maximum m and sum l.
//
// A wave holds 16 columns, each a (token, query head of the KV head's group) pair, and takes a
// block of 64 positions at a time: scores^T = K q^T with K as the row operand (four 16-position
// groups of v_mfma_f32_16x16x32_f16), then out^T += V^T p^T. The codes go from memory to
// registers in operand order (sp_fp8.h) and become fp16 there, exactly; the scores' layout is
// the weights' operand layout, so nothing passes through LDS inside the loop.
//
// Precision. q is scaled by a power of two that puts its row's largest entry in [2^14, 2^15)
// and rounded to fp16: exact for fp16 and bf16 rows (entries below 2^-39 of the row's largest
// lose bits). An fp32 row is split into two fp16 parts (22 bits). The weights are counted from
// 2^14 at the maximum, so that those of 2^-28 of it are still normal fp16 numbers, and rounded
// to fp16 (half a step, 2^-11, beside the 2^-11 and 2^-8 of an fp16 or bf16 result) or, for fp32
// results, split in two. Sums, maxima and the running output are fp32. The running output counts in
// units of the current V scale: when the scale or the maximum changes it is rescaled, and the
// exponents' range (-40 to 40) keeps it finite.
#include "sp_fp8.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float P_TOP = 14.0f;  // log2 of the largest weight

// Eight codes (two dwords) as fp16.
__device__ __forceinline__ h8 to_half(unsigned a, unsigned b) {
    const h2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    const h2 y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const h2 z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    const h2 w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return h8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}
__device__ __forceinline__ f4 mma(h8 a, h8 b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// maximum and sum over the four lanes that share a column (lane ^ 16, lane ^ 32)
__device__ __forceinline__ float column_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float column_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

__device__ __forceinline__ long long wave_sum(long long v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d, 64);
    return v;
}

// What one block of threads works on: `cols` columns from ct * cols of a sequence, one of
// n_split shares of the cache blocks that they see.
struct Share {
    int seq, r0, n_new, first;  // first: position of the sequence's first row
    int ct, split, n_split;
    int slot;  // of the partial result, in units of KV heads; group's first: slot - split
};

// The work is divided on the device, so that lengths may change under a captured call: with T
// the blocks that all column groups see and R = T / target, a column group of n blocks gets
// ceil(n / R) shares. Groups of two or more shares number at most 2 * target shares in all
// (n > R gives ceil(n / R) < 2 n / R), which bounds the partial results.
__device__ __forceinline__ bool find_share(const SpFp8Attn &A, int item, int lane, int cols, Share &out) {
    const SpFp8Seqs &S = A.s;
    long long total = 0, rows = 0;
    for (int i0 = 0; i0 < S.n_seq; i0 += 64) {
        const int i = i0 + lane;
        if (i < S.n_seq) {
            int a, b, len;
            sp_fp8_seq(S, i, a, b, len);
            const int lo = A.window > 0 ? max(len - (b - a) - A.window + 1, 0) >> 6 : 0;
            const int nb = max(min((len + 63) >> 6, S.stride) - lo, 0);
            const long long ct = ((long long)(b - a) * A.G + cols - 1) / cols;
            total += ct * nb;
            rows += b - a;
        }
    }
    total = wave_sum(total) * A.H;
    if (wave_sum(rows) > S.n_rows) return false;  // the array of rows is not ascending
    const int R = (int)max((total + A.target - 1) / A.target, 1ll);
    int slots = 0;
    for (int i0 = 0; i0 < S.n_seq; i0 += 64) {
        const int i = i0 + lane;
        int a = 0, b = 0, len = 0, ct = 0, ns = 1;
        if (i < S.n_seq) {
            sp_fp8_seq(S, i, a, b, len);
            const int lo = A.window > 0 ? max(len - (b - a) - A.window + 1, 0) >> 6 : 0;
            const int nb = max(min((len + 63) >> 6, S.stride) - lo, 0);
            ct = (int)(((long long)(b - a) * A.G + cols - 1) / cols);
            ns = max((nb + R - 1) / R, 1);
        }
        const int n = ct * ns, sum = sp_fp8_scan(n, lane);
        const int part = ns > 1 ? n : 0, psum = sp_fp8_scan(part, lane);
        const unsigned long long past = __ballot(sum > item);
        if (past) {
            const int l = __ffsll(past) - 1;
            out.seq = i0 + l;
            out.r0 = __shfl(a, l, 64);
            out.n_new = __shfl(b, l, 64) - out.r0;
            out.first = __shfl(len, l, 64) - out.n_new;
            out.n_split = __shfl(ns, l, 64);
            const int at = item - (__shfl(sum, l, 64) - __shfl(n, l, 64));
            out.ct = at / out.n_split;
            out.split = at - out.ct * out.n_split;
            out.slot = slots + __shfl(psum, l, 64) - __shfl(part, l, 64) + at;
            return true;
        }
        item -= __shfl(sum, 63, 64);
        slots += __shfl(psum, 63, 64);
    }
    return false;
}

template <int DT>
__device__ __forceinline__ void load8(const typename SpFp8Elem<DT>::T *p, bool aligned, float x[8]) {
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    if (aligned) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const T4 v = reinterpret_cast<const T4 *>(p)[k];
#pragma unroll
            for (int n = 0; n < 4; n++) x[4 * k + n] = SpFp8Elem<DT>::get(v[n]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = SpFp8Elem<DT>::get(p[k]);
    }
}

struct f2 {
    float x, y;
};
__device__ __forceinline__ void put_pair(float *p, float x, float y) {
    const f2 v{x, y};
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(p), __builtin_bit_cast(unsigned long long, v),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f2 get_pair(const float *p) {
    return __builtin_bit_cast(f2, __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED,
                                                    __HIP_MEMORY_SCOPE_AGENT));
}

// Weight of a partial result with maximum m in one with maximum M. One without a position
// (m = -inf) has sums of 0, or NaN where q has: kept as they are.
__device__ __forceinline__ float weight(float m, float M) {
    return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - M);
}

template <int DT>
__device__ __forceinline__ void finish(const SpFp8Attn &A, long long row, int head, int hd, int d, float m, float l,
                                       float o0, float o1) {
    typedef typename SpFp8Elem<DT>::T T;
    T *out = reinterpret_cast<T *>(A.out) + row * A.out_stride + (long long)head * hd + d;
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    out[0] = SpFp8Elem<DT>::put(l == 0.0f ? 0.0f : o0 * r);
    out[1] = SpFp8Elem<DT>::put(l == 0.0f ? 0.0f : o1 * r);
    if (A.lse && d == 0)
        A.lse[row * A.H * A.G + head] = l == 0.0f ? -INFINITY : (m - P_TOP + __log2f(l)) * 0.69314718055994531f;
}

template <int HD, int DT, int NW>
__global__ __launch_bounds__(NW * 64) void k_fp8_attn(SpFp8Attn A) {
    constexpr int COLS = 16, NC = HD / 32, ND = HD / 16, TILE = 64 * HD, ROW = HD + 2;
    constexpr bool SPLIT2 = DT == SP_DTYPE_F32;
    constexpr int NH = SPLIT2 ? 2 : 1;
    typedef typename SpFp8Elem<DT>::T T;
    extern __shared__ __align__(16) float smem[];  // [NW][columns][HD + 4]: o, m, l
    __shared__ int last_flag;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % A.H;
    Share sh;
    if (!find_share(A, blockIdx.x / A.H, lane, COLS, sh)) return;
    const int n_cols = min((int)min((long long)sh.n_new * A.G - (long long)sh.ct * COLS, (long long)COLS), COLS);
    const int col = lane & 15, g = lane >> 4;
    const long long c0 = (long long)sh.ct * COLS;
    const int tk0 = (int)(c0 / A.G), tk1 = (int)((c0 + n_cols - 1) / A.G);
    const int pos0 = sh.first + tk0, pos1 = sh.first + tk1;
    // the cache blocks that these columns see, and this share of them
    const int j0 = A.window > 0 ? max(pos0 - A.window + 1, 0) >> 6 : 0;
    const int j1 = min((pos1 >> 6) + 1, A.s.stride);  // pos1 < 0: 0
    const int per = max((j1 - j0 + sh.n_split - 1) / sh.n_split, 0);
    const int t0 = j0 + sh.split * per, t1 = min(t0 + per, j1);

    // ---- queries ----
    const bool active = col < n_cols;
    const long long cn = c0 + (active ? col : 0);
    const int tk = (int)(cn / A.G), head = h * A.G + (int)(cn % A.G);
    const int pos = active ? sh.first + tk : -1;
    const int from = A.window > 0 ? pos - A.window : -1;  // sees (from, pos]
    h8 q[NC][NH];
    float cscale;
    {
        float x[NC][8], top = 0.0f;
        const T *src = reinterpret_cast<const T *>(A.q) + (sh.r0 + tk) * A.q_stride + (long long)head * HD + g * 8;
        const bool aligned = ((uintptr_t)A.q % (4 * sizeof(T))) == 0 && A.q_stride % 4 == 0;
#pragma unroll
        for (int c = 0; c < NC; c++) {
            load8<DT>(src + c * 32, aligned, x[c]);
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[c][k]));
        }
        top = column_max(top);
        int e = (__float_as_int(top) >> 23) - 127 - 14;
        e = top == 0.0f || !(top < INFINITY) ? 0 : max(e, -126);
        const float down = A.negate ? -sp_fp8_pow2(-e) : sp_fp8_pow2(-e);
        cscale = A.c * sp_fp8_pow2(e);
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float y = active ? x[c][k] * down : 0.0f;
                const _Float16 hi = (_Float16)y;
                q[c][0][k] = hi;
                if (SPLIT2) q[c][NH - 1][k] = (_Float16)(y - (float)hi);
            }
    }

    // ---- this wave's blocks: t0 + w, t0 + w + NW, ... ----
    f4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;
    int ev_now = 0;
    const int mine = t1 > t0 + w ? (t1 - t0 - w + NW - 1) / NW : 0;
    for (int base = 0; base < mine; base += 64) {
        const int count = min(mine - base, 64);
        // lane k: block number and scales of the k-th block
        int blk = -1, ek = 0, ev = 0;
        if (lane < count) {
            blk = sp_fp8_block(A.s, sh.seq, t0 + w + NW * (base + lane));
            if (blk >= 0) {
                ek = sp_fp8_exponent(A.k.exps[(long long)blk * A.H + h]);
                ev = sp_fp8_exponent(A.v.exps[(long long)blk * A.H + h]);
            }
        }
        u4 kr[2 * NC], vr[ND];
        const auto load_k = [&](int k) {
            const int b = max(__builtin_amdgcn_readlane(blk, k), 0);  // none: read block 0, all masked
            const uint8_t *p = A.k.codes + ((long long)b * A.H + h) * TILE + lane * 16;
#pragma unroll
            for (int n = 0; n < 2 * NC; n++) kr[n] = *reinterpret_cast<const u4 *>(p + n * 1024);
        };
        const auto load_v = [&](int k) {
            const int b = max(__builtin_amdgcn_readlane(blk, k), 0);
            const uint8_t *p = A.v.codes + ((long long)b * A.H + h) * TILE + lane * 16;
#pragma unroll
            for (int n = 0; n < ND; n++) vr[n] = *reinterpret_cast<const u4 *>(p + n * 1024);
        };
        load_k(0);
        load_v(0);
        for (int k = 0; k < count; k++) {
            const int t = t0 + w + NW * (base + k);
            const bool none = __builtin_amdgcn_readlane(blk, k) < 0;
            const float cs = cscale * sp_fp8_pow2(__builtin_amdgcn_readlane(ek, k));
            f4 s[4];
#pragma unroll
            for (int n = 0; n < 4; n++) s[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u4 r = kr[u * NC + c];
                    const h8 a = to_half(r[0], r[1]), b = to_half(r[2], r[3]);
#pragma unroll
                    for (int n = 0; n < NH; n++) {
                        s[2 * u] = mma(a, q[c][n], s[2 * u]);
                        s[2 * u + 1] = mma(b, q[c][n], s[2 * u + 1]);
                    }
                }
            if (k + 1 < count) load_k(k + 1);
            const bool open = !none && t * 64 + 63 <= pos0 && (A.window <= 0 || t * 64 > pos1 - A.window);
            float top = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    float x = s[n][i] * cs;
                    if (!open) {
                        const int at = t * 64 + n * 16 + 4 * g + i;
                        x = !none && at <= pos && at > from ? x : -INFINITY;
                    }
                    s[n][i] = x;
                    top = fmaxf(top, x);
                }
            const float m_new = fmaxf(m, column_max(top));
            const float ref = m_new == -INFINITY ? 0.0f : m_new - P_TOP;
            const float alpha = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            float sum = 0.0f;
            h8 p[2][NH];
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float x = __builtin_amdgcn_exp2f(s[n][i] - ref);
                    sum += x;
                    const _Float16 hi = (_Float16)x;
                    p[n / 2][0][(n % 2) * 4 + i] = hi;
                    if (SPLIT2) p[n / 2][NH - 1][(n % 2) * 4 + i] = (_Float16)(x - (float)hi);
                }
            l = l * alpha + sum;
            m = m_new;
            const int ev_k = __builtin_amdgcn_readlane(ev, k);
            const float f = alpha * sp_fp8_pow2(ev_now - ev_k);
            ev_now = ev_k;
            if (__any(f != 1.0f)) {
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= f;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const h8 a = to_half(vr[d][0], vr[d][1]), b = to_half(vr[d][2], vr[d][3]);
#pragma unroll
                for (int n = 0; n < NH; n++) {
                    o[d] = mma(a, p[0][n], o[d]);
                    o[d] = mma(b, p[1][n], o[d]);
                }
            }
            if (k + 1 < count) load_v(k + 1);
        }
    }
    l = column_sum(l);

    // ---- the waves' results joined ----
    constexpr int LROW = HD + 4;
    const float unit = sp_fp8_pow2(ev_now);
    if (active) {
        float *rec = smem + (w * n_cols + col) * LROW;
#pragma unroll
        for (int d = 0; d < ND; d++) *reinterpret_cast<f4 *>(rec + d * 16 + g * 4) = o[d] * unit;
        if (g == 0) {
            rec[HD] = m;
            rec[HD + 1] = l;
        }
    }
    __syncthreads();
    const long long slot = (long long)sh.slot * A.H + h;
    for (int at = tid; at < n_cols * (HD / 2); at += NW * 64) {
        const int cc = at / (HD / 2), d = at % (HD / 2) * 2;
        float M = -INFINITY;
#pragma unroll
        for (int v = 0; v < NW; v++) M = fmaxf(M, smem[(v * n_cols + cc) * LROW + HD]);
        float L = 0.0f, x = 0.0f, y = 0.0f;
#pragma unroll
        for (int v = 0; v < NW; v++) {
            const float *rec = smem + (v * n_cols + cc) * LROW;
            const float f = weight(rec[HD], M);
            L += rec[HD + 1] * f;
            x += rec[d] * f;
            y += rec[d + 1] * f;
        }
        if (sh.n_split == 1) {
            const long long n = c0 + cc;
            finish<DT>(A, sh.r0 + n / A.G, h * A.G + (int)(n % A.G), HD, d, M, L, x, y);
        } else if (slot < SP_FP8_SLOTS) {
            float *dst = A.part + (slot * COLS + cc) * ROW;
            if (d == 0) put_pair(dst, M, L);
            put_pair(dst + 2 + d, x, y);
        }
    }
    if (sh.n_split == 1 || slot >= SP_FP8_SLOTS) return;

    // ---- the last of the column group's shares to arrive joins them all, in their order ----
    // each block's stores are complete before it counts itself
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const long long slot0 = (long long)(sh.slot - sh.split) * A.H + h;
    if (tid == 0) {
        int *cnt = A.counters + slot0;
        const int arrived = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last_flag = arrived == sh.n_split - 1;
        if (last_flag) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!last_flag) return;
    for (int at = tid; at < n_cols * (HD / 2); at += NW * 64) {
        const int cc = at / (HD / 2), d = at % (HD / 2) * 2;
        const float *src = A.part + (slot0 * COLS + cc) * ROW;
        const long long step = (long long)A.H * COLS * ROW;
        float M = -INFINITY, L = 0.0f, x = 0.0f, y = 0.0f;
        for (int v0 = 0; v0 < sh.n_split; v0 += 8) {
            f2 ml[8], xy[8];
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const float *rec = src + min(v0 + v, sh.n_split - 1) * step;
                ml[v] = get_pair(rec);
                xy[v] = get_pair(rec + 2 + d);
            }
            float Mn = M;
#pragma unroll
            for (int v = 0; v < 8; v++)
                if (v0 + v < sh.n_split) Mn = fmaxf(Mn, ml[v].x);
            const float f0 = weight(M, Mn);
            L *= f0;
            x *= f0;
            y *= f0;
#pragma unroll
            for (int v = 0; v < 8; v++) {
                const float f = v0 + v < sh.n_split ? weight(ml[v].x, Mn) : 0.0f;
                if (v0 + v < sh.n_split) {
                    L += ml[v].y * f;
                    x += xy[v].x * f;
                    y += xy[v].y * f;
                }
            }
            M = Mn;
        }
        const long long n = c0 + cc;
        finish<DT>(A, sh.r0 + n / A.G, h * A.G + (int)(n % A.G), HD, d, M, L, x, y);
    }
}

template <int HD, int DT, int NW>
hipError_t launch(const SpFp8Attn &A, hipStream_t s) {
    constexpr int COLS = 16;
    // column groups: each sequence's rows times G, in groups of COLS
    const long long groups = A.s.row ? ((long long)A.s.n_rows * A.G) / COLS + A.s.n_seq
                                     : (long long)A.s.n_seq * ((A.G + COLS - 1) / COLS);
    // shares: one per group, and at most target more over all KV heads
    const long long blocks = (groups + (A.target + A.H - 1) / A.H) * A.H;
    if (blocks > 0x7fffffffll) return hipErrorInvalidValue;
    const int cols = A.s.row ? COLS : (A.G < COLS ? A.G : COLS);
    const size_t lds = (size_t)NW * cols * (HD + 4) * sizeof(float);
    SpFp8Attn a = A;
    void *args[] = {&a};
    const void *f = (const void *)k_fp8_attn<HD, DT, NW>;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(NW * 64), args, lds, s);
}

template <int HD>
hipError_t launch_dt(const SpFp8Attn &A, int dtype, hipStream_t s) {
    switch (dtype) {
        case SP_DTYPE_F32: return launch<HD, SP_DTYPE_F32, 4>(A, s);
        case SP_DTYPE_F16: return launch<HD, SP_DTYPE_F16, 4>(A, s);
        case SP_DTYPE_BF16: return launch<HD, SP_DTYPE_BF16, 4>(A, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

size_t sp_fp8_workspace_floats(int hd) { return (size_t)SP_FP8_SLOTS * 32 * (hd + 2); }

hipError_t sp_fp8_launch_attn(const SpFp8Attn &A, int hd, int dtype, hipStream_t s) {
    switch (hd) {
        case 64: return launch_dt<64>(A, dtype, s);
        case 96: return launch_dt<96>(A, dtype, s);
        case 128: return launch_dt<128>(A, dtype, s);
        case 256: return launch_dt<256>(A, dtype, s);
    }
    return hipErrorInvalidValue;
}

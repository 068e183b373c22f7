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
// and rounded to fp16, whose last bit is 2^-24 or more, 2^-39 of the row's largest entry (2^-38 with one
// next to 2^15). A bf16 row is exact but for its entries below 2^-31 of the largest, which lose bits and
// vanish at 2^-39; an fp16 row is exact but, where its largest is 2^15 or more, for a last bit of 2^-24.
// An fp32 row is split into two fp16 parts (22 bits, of entries below 2^-17 of the largest fewer, down
// to the same last bit). The weights are counted from
// 2^14 at the maximum, so that those of 2^-28 of it are still normal fp16 numbers, and rounded
// to fp16 (half a step, 2^-11, beside the 2^-11 and 2^-8 of an fp16 or bf16 result) or, for fp32
// results, split in two. Sums, maxima and the running output are fp32. The running output counts in
// units of the current V scale: when the scale or the maximum changes it is rescaled, and the
// exponents' range (-40 to 40) keeps it finite.
#include <type_traits>

#include "sp_device.h"
#include "sp_fp8.h"

namespace {

using sp_fp8::f4;
using sp_fp8::u4;
using sp_fp8::store4;
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr float P_TOP = 14.0f;  // log2 of the largest weight

// A score further than this from 0 has the maximum taken off first, which is exact at the maximum, and
// P_TOP added then. Taken together they are rounded where a float counts in 4 or more (from 2^25 on):
// the largest weight becomes 2^16, which is no fp16 number. Below, rounding them costs less than the
// score's own last bit. (Always in two steps: 40.5 us for 39.7 with 32 rows of each of 12 sequences at
// head_dim 64, 32 / 8 heads.)
constexpr float FAR_SCORE = 0x1p18f;
__device__ __forceinline__ bool is_far(float m) { return fabsf(m) > FAR_SCORE && fabsf(m) < INFINITY; }

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

// A.c 2^e, at most the largest float. kq_scale, the query's exponent and the block's are put together in
// one step: two of them may multiply to more than a float holds where all three are an ordinary scale.
__device__ __forceinline__ float score_scale(const SpFp8Attn &A, int e) {
    return fminf(__builtin_amdgcn_ldexpf(A.c, e), 0x1.fffffep127f);
}

// Results that all lanes agree on are taken into scalar registers (readfirstlane, readlane), so
// that what follows from them is scalar too.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) { return __int_as_float(uniform(__float_as_int(v))); }

__device__ __forceinline__ float wave_sum(float v) { return uniform(sp_wave_sum_dpp(v)); }

// What one block of threads works on: `cols` columns from ct * cols of a sequence, one of
// n_split shares of the cache blocks that they see.
struct Share {
    int seq, r0, n_new, first;  // first: position of the sequence's first row
    int ct, split, n_split;
    int slot;  // of the partial result, in units of KV heads; group's first: slot - split
};

// A sequence's rows, length, column groups and the cache blocks that its rows see.
struct Extent {
    int a, b, len, ct, nb;
    bool bad;  // d_row does not ascend here, or leaves the call's rows
};
__device__ __forceinline__ Extent extent(const SpFp8Attn &A, int i, int cols) {
    Extent e{0, 0, 0, 0, 0, false};
    if (i < A.s.n_seq) {
        sp_fp8_seq(A.s, i, e.a, e.b, e.len);
        e.bad = A.s.row && (A.s.row[i] != e.a || A.s.row[i + 1] != e.b);
        const int lo = A.window > 0 ? max(e.len - (e.b - e.a) - A.window + 1, 0) >> 6 : 0;
        e.nb = max(min((e.len + 63) >> 6, A.s.stride) - lo, 0);
        e.ct = ((e.b - e.a) * A.G + cols - 1) / cols;
    }
    return e;
}
__device__ __forceinline__ int shares_of(int nb, int R, int alone) {
    return nb <= alone ? 1 : (nb + R - 1) / R;
}

// Fewest cache blocks of a share: what makes `target` of them, but where few groups are cut into
// many shares no less than costs least. n blocks in n / R shares take the time of R / 8 blocks, a wave
// each, and then of n / R shares' partial results, eight loaded at once, in A.join rounds: R is the
// root of n A.join (16 rows over 32000 positions of two heads of 128 take 36 us, where `target` shares
// took 50; four rows of one head 23 for 43). alone: blocks up to which a group is not shared out.
__device__ __forceinline__ int first_share(const SpFp8Attn &A, float T, float mean, int least, int &alone) {
    const float even = min(T / (float)A.target * 1.002f, 0x1p24f);  // (2^24 blocks: a whole table row)
    const int cheap = (int)__builtin_sqrtf(min(mean, 0x1p24f) * A.join);
    alone = max(4 * least, 2 * cheap);
    return max(max((int)even + 1, cheap), least);
}

// The work is divided on the device, so that lengths may change under a captured call. With T
// the blocks that all column groups see, a column group of n blocks gets ceil(n / R) shares,
// R the first of R0, 5/4 R0, 3/2 R0 and 2 R0, R0 > T / target, that makes at most `target`
// shares, if one does. R is at least `least`, and up to four times that (or `alone`) is not shared out:
// a share's own waves join their results in LDS, which costs less than the stores, the count and
// the loads (three memory latencies) that join shares. Groups of two or more shares (n > R, so
// ceil(n / R) < 2 n / R) have at most 2 T / R < 2 target shares, which bounds the partial
// results. by_group: `item` counts column groups, and their first shares are found.
__device__ __forceinline__ bool find_share(const SpFp8Attn &A, int item, int lane, int cols, int least, bool by_group,
                                           Share &out) {
    const int n_seq = A.s.n_seq;
    if (n_seq == 1) {  // nothing to search, and no exchange between lanes
        const Extent e = extent(A, 0, cols);
        const float T = (float)e.ct * (float)e.nb * (float)A.H;
        int alone;
        const int R0 = first_share(A, T, (float)e.nb, least, alone);
        int R = 2 * R0;
        for (int k = 2; k >= 0; k--) {
            const int r = R0 + k * R0 / 4;
            if ((float)shares_of(e.nb, r, alone) * (float)e.ct * (float)A.H <= (float)A.target) R = r;
        }
        const int ns = shares_of(e.nb, R, alone);
        if (by_group) item *= ns;
        out = Share{0, e.a, e.b - e.a, e.len - (e.b - e.a), e.ct - 1 - item / ns, item % ns, ns, item};
        return !e.bad && item < e.ct * ns;
    }
    const Extent e0 = extent(A, lane, cols);  // kept: up to 64 sequences are read once
    float T = (float)e0.ct * (float)e0.nb, groups = (float)e0.ct;
    bool bad = e0.bad;
    for (int i0 = 64; i0 < n_seq; i0 += 64) {
        const Extent e = extent(A, i0 + lane, cols);
        T += (float)e.ct * (float)e.nb;
        groups += (float)e.ct;
        bad = bad || e.bad;
    }
    if (__any(bad)) return false;  // the grid was made for rows that ascend
    T = wave_sum(T) * (float)A.H;
    int alone;
    const int R0 = first_share(A, T, T / fmaxf(wave_sum(groups) * (float)A.H, 1.0f), least, alone);
    float n[3] = {0.0f, 0.0f, 0.0f};
    for (int i0 = 0; i0 < n_seq; i0 += 64) {
        const Extent e = i0 ? extent(A, i0 + lane, cols) : e0;
#pragma unroll
        for (int k = 0; k < 3; k++) n[k] += (float)e.ct * (float)shares_of(e.nb, R0 + k * R0 / 4, alone);
    }
    int R = 2 * R0;
#pragma unroll
    for (int k = 2; k >= 0; k--)
        if (wave_sum(n[k]) * (float)A.H <= (float)A.target) R = R0 + k * R0 / 4;
    int slots = 0;
    for (int i0 = 0; i0 < n_seq; i0 += 64) {
        const Extent e = i0 ? extent(A, i0 + lane, cols) : e0;
        const int ns = shares_of(e.nb, R, alone), mine = by_group ? e.ct : e.ct * ns, sum = sp_fp8_scan(mine, lane);
        const int part = ns > 1 ? e.ct * ns : 0, psum = sp_fp8_scan(part, lane);
        const unsigned long long past = __ballot(sum > item);
        if (past) {
            const int l = __ffsll(past) - 1;
            const auto of = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
            out.seq = i0 + l;
            out.r0 = of(e.a);
            out.n_new = of(e.b) - out.r0;
            out.first = of(e.len) - out.n_new;
            out.n_split = of(ns);
            const int at = (item - (of(sum) - of(mine))) * (by_group ? out.n_split : 1);
            // the last column group first: under the causal mask it sees most
            out.ct = of(e.ct) - 1 - at / out.n_split;
            out.split = at % out.n_split;
            out.slot = slots + of(psum) - of(part) + at;
            return true;
        }
        item -= __builtin_amdgcn_readlane(sum, 63);
        slots += __builtin_amdgcn_readlane(psum, 63);
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

struct Two {
    float x, y;
};
__device__ __forceinline__ void put_pair(float *p, float x, float y) {
    const Two v{x, y};
    __hip_atomic_store(reinterpret_cast<unsigned long long *>(p), __builtin_bit_cast(unsigned long long, v),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Two get_pair(const float *p) {
    return __builtin_bit_cast(Two, __hip_atomic_load(reinterpret_cast<const unsigned long long *>(p), __ATOMIC_RELAXED,
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
        A.lse[row * A.H * A.G + head] = l == 0.0f ? -INFINITY : (m + (__log2f(l) - P_TOP)) * 0.69314718055994531f;
}

// Whether a partial result has its place (always: see find_share).
__device__ __forceinline__ bool slot_fits(const SpFp8Attn &A, long long slot, int cols) {
    return slot < SP_FP8_SLOTS && (slot + 1) * cols <= A.part_rows;
}

// Joins partial results (m, l, o pair) in order.
struct Acc {
    float M = -INFINITY, L = 0.0f, x = 0.0f, y = 0.0f;
    __device__ __forceinline__ void add(float m, float l, float px, float py) {
        const float Mn = fmaxf(M, m), f0 = weight(M, Mn), f = weight(m, Mn);
        L = L * f0 + l * f;
        x = x * f0 + px * f;
        y = y * f0 + py * f;
        M = Mn;
    }
};

// The last of a column group's shares to arrive joins them all, in their order. Every thread of
// the block calls it after its partial's stores. smem: at least NW * n_cols * HD floats.
template <int HD, int DT, int NW, int COLS>
__device__ __forceinline__ void join_shares(const SpFp8Attn &A, const Share &sh, int h, int c0, int n_cols,
                                            float *smem, int *last_flag) {
    constexpr int NT = NW * 64, ROW = HD + 2;
    const int tid = threadIdx.x, pairs = n_cols * (HD / 2);
    // each block's stores are complete before it counts itself
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const long long slot0 = (long long)(sh.slot - sh.split) * A.H + h;
    if (tid == 0) {
        int *cnt = A.counters + slot0;
        const int arrived = __hip_atomic_fetch_add(cnt, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last_flag = arrived == sh.n_split - 1;
        if (*last_flag) __hip_atomic_store(cnt, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);  // for the next call
    }
    __syncthreads();
    if (!*last_flag) return;
    // groups of threads take runs of shares, so that a run's loads are in flight together
    const int groups = pairs < NT ? min(NT / pairs, NW / 2) : 1, run = (sh.n_split + groups - 1) / groups;
    for (int i0 = 0; i0 < pairs; i0 += NT) {
        const int grp = groups == 1 ? 0 : tid / pairs, at = i0 + tid - grp * pairs;
        const bool here = grp < groups && at < pairs;
        const int cc = at / (HD / 2), d = at % (HD / 2) * 2;
        const int v1 = min((grp + 1) * run, sh.n_split);
        Acc acc;
        if (here) {
            const float *src = A.part + (slot0 * COLS + cc) * ROW;
            const long long step = (long long)A.H * COLS * ROW;
            for (int v0 = grp * run; v0 < v1; v0 += 8) {
                Two ml[8], xy[8];
#pragma unroll
                for (int v = 0; v < 8; v++) {
                    const float *rec = src + min(v0 + v, v1 - 1) * step;
                    ml[v] = get_pair(rec);
                    xy[v] = get_pair(rec + 2 + d);
                }
#pragma unroll
                for (int v = 0; v < 8; v++)
                    if (v0 + v < v1) acc.add(ml[v].x, ml[v].y, xy[v].x, xy[v].y);
            }
        }
        if (groups > 1) {  // pairs < NT: one round
            f4 *join = reinterpret_cast<f4 *>(smem);
            if (here && grp) join[(grp - 1) * pairs + at] = f4{acc.M, acc.L, acc.x, acc.y};
            __syncthreads();
            if (here && !grp)
                for (int v = 0; v < groups - 1; v++) {
                    const f4 r = join[v * pairs + at];
                    acc.add(r[0], r[1], r[2], r[3]);
                }
        }
        if (here && !grp) {
            const int n = c0 + cc;
            finish<DT>(A, sh.r0 + n / A.G, h * A.G + n % A.G, HD, d, acc.M, acc.L, acc.x, acc.y);
        }
    }
}

// Few rows: one token a sequence, or several. A block of NW waves takes a share of the cache
// blocks that its columns see, each wave every NW-th of them, and joins the waves' results in
// LDS; CG groups of 16 columns share a block's loads and conversions. It is bound by memory: a
// wave has 64 * head_dim codes of K and of V in flight and asks for the next as soon as the
// registers are free, which takes eight waves a CU (four at head_dim 256) to keep HBM busy.
// Measured: 2 x 131072 positions of 8 heads of 256 (1.07 GB) in 191 us, 5.6 TB/s; 16 sequences of 1 to 4K
// of 32 heads of 96 with float32 rows (261 MB) in 54 us, 4.8 TB/s; one of 32768 of 8 heads of 128
// (67 MB) in 18.2 us, of which the join of 32 shares takes 4 and an empty launch 4.2; 12 of 1 to
// 4.5K with two to five rows each (73 MB) in 20.9 us; 777 positions of 8 heads of 64 in 7.1 us. With 16
// waves of 128 registers the loop spills; four waves a block make more shares to join (22.0 us for
// the 32768 where eight took 20.1 beside them).
template <int HD, int DT, int NW, int CG>
__global__ __launch_bounds__(NW * 64) void k_fp8_attn(SpFp8Attn A) {
    constexpr int COLS = 16 * CG, NC = HD / 32, ND = HD / 16, TILE = 64 * HD, ROW = HD + 2, NT = NW * 64;
    constexpr bool SPLIT2 = DT == SP_DTYPE_F32;
    constexpr int NH = SPLIT2 ? 2 : 1;
    typedef typename SpFp8Elem<DT>::T T;
    extern __shared__ __align__(16) float smem[];  // [NW][columns][HD + 4]: o, m, l
    __shared__ int last_flag;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % A.H;
    Share sh;
    if (!find_share(A, blockIdx.x / A.H, lane, COLS, NW / 2, false, sh)) return;
    const int c0 = sh.ct * COLS, n_cols = min(sh.n_new * A.G - c0, COLS);
    const int col = lane & 15, g = lane >> 4;
    const int tk0 = c0 / A.G, tk1 = (c0 + n_cols - 1) / A.G;
    const int pos0 = sh.first + tk0, pos1 = sh.first + tk1;
    // the cache blocks that these columns see, and this share of them
    const int j0 = A.window > 0 ? max(pos0 - A.window + 1, 0) >> 6 : 0;
    const int j1 = min((pos1 >> 6) + 1, A.s.stride);  // pos1 < 0: 0
    const int per = max((j1 - j0 + sh.n_split - 1) / sh.n_split, 0);
    const int t0 = j0 + sh.split * per, t1 = min(t0 + per, j1);

    // ---- this wave's blocks: t0 + w, t0 + w + NW, ... ----
    // The chain of loads is length, table, codes: the table's and the first codes' loads are
    // issued before anything waits for the queries or the scales.
    const int mine = t1 > t0 + w ? (t1 - t0 - w + NW - 1) / NW : 0;
    int blk = -1, ekb = 0, evb = 0;  // lane k: block number and scale bytes of the k-th block
    const auto look_up = [&](int base) {
        blk = base + lane < mine ? sp_fp8_block(A.s, sh.seq, t0 + w + NW * (base + lane)) : -1;
    };
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
    const auto start = [&]() {
        const long long at = (long long)max(blk, 0) * A.H + h;
        ekb = A.k.exps[at];
        evb = A.v.exps[at];
        load_k(0);
        load_v(0);
    };
    if (mine > 0) look_up(0);

    // ---- queries ----
    bool active[CG];
    int pos[CG], from[CG];  // sees (from, pos]
    float x[CG][NC][8];
#pragma unroll
    for (int y = 0; y < CG; y++) {
        active[y] = y * 16 + col < n_cols;
        const int cn = c0 + (active[y] ? y * 16 + col : 0), tk = cn / A.G, head = h * A.G + cn % A.G;
        pos[y] = active[y] ? sh.first + tk : -1;
        from[y] = A.window > 0 ? pos[y] - A.window : -1;
        const T *src = reinterpret_cast<const T *>(A.q) + (long long)(sh.r0 + tk) * A.q_stride + (long long)head * HD + g * 8;
        const bool aligned = ((uintptr_t)A.q % (4 * sizeof(T))) == 0 && A.q_stride % 4 == 0;
#pragma unroll
        for (int c = 0; c < NC; c++) load8<DT>(src + c * 32, aligned, x[y][c]);
    }
    if (mine > 0) start();
    h8 q[CG][NC][NH];
    int qe[CG];  // scores count in 2^(qe + the block's exponent) * A.c
#pragma unroll
    for (int y = 0; y < CG; y++) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[y][c][k]));
        top = column_max(top);
        int e = (__float_as_int(top) >> 23) - 127 - 14;
        e = top == 0.0f || !(top < INFINITY) ? 0 : max(e, -126);
        const float down = A.negate ? -sp_fp8_pow2(-e) : sp_fp8_pow2(-e);
        qe[y] = e + 1;
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float v = active[y] ? x[y][c][k] * down : 0.0f;
                const _Float16 hi = (_Float16)v;
                q[y][c][0][k] = hi;
                if (SPLIT2) q[y][c][NH - 1][k] = (_Float16)(v - (float)hi);
            }
    }

    f4 o[CG][ND];
    float m[CG], l[CG];
#pragma unroll
    for (int y = 0; y < CG; y++) {
        m[y] = -INFINITY;
        l[y] = 0.0f;
#pragma unroll
        for (int d = 0; d < ND; d++) o[y][d] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    int ev_now = 0;
    for (int base = 0; base < mine; base += 64) {
        const int count = min(mine - base, 64);
        if (base) {
            look_up(base);
            start();
        }
        for (int k = 0; k < count; k++) {
            const int t = t0 + w + NW * (base + k);
            const bool none = __builtin_amdgcn_readlane(blk, k) < 0;
            const int ek = sp_fp8_exponent(__builtin_amdgcn_readlane(ekb, k));
            f4 s[CG][4];
#pragma unroll
            for (int y = 0; y < CG; y++)
#pragma unroll
                for (int n = 0; n < 4; n++) s[y][n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < NC; c++)
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const u4 r = kr[u * NC + c];
                    const h8 a = to_half(r[0], r[1]), b = to_half(r[2], r[3]);
#pragma unroll
                    for (int y = 0; y < CG; y++)
#pragma unroll
                        for (int n = 0; n < NH; n++) {
                            s[y][2 * u] = mma(a, q[y][c][n], s[y][2 * u]);
                            s[y][2 * u + 1] = mma(b, q[y][c][n], s[y][2 * u + 1]);
                        }
                }
            if (k + 1 < count) load_k(k + 1);
            const bool open = !none && t * 64 + 63 <= pos0 && (A.window <= 0 || t * 64 > pos1 - A.window);
            const int ev_k = sp_fp8_exponent(__builtin_amdgcn_readlane(evb, k));
            const float ev_step = sp_fp8_pow2(ev_now - ev_k);
            ev_now = ev_k;
            h8 p[CG][2][NH];
#pragma unroll
            for (int y = 0; y < CG; y++) {
                const float cs = score_scale(A, qe[y] + ek);
                float top = -INFINITY;
                // positions of this block that the column sees, counted from the lane's first: (before, upto]
                const int lane0 = t * 64 + 4 * g, upto = none ? -1 : pos[y] - lane0, before = from[y] - lane0;
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        float x = s[y][n][i] * cs;
                        if (!open) x = n * 16 + i <= upto && n * 16 + i > before ? x : -INFINITY;
                        s[y][n][i] = x;
                        top = fmaxf(top, x);
                    }
                const float m_new = fmaxf(m[y], column_max(top));
                float ref = m_new == -INFINITY ? 0.0f : m_new;
                const bool far = is_far(m_new);
                if (__any(far)) {  // (a column that is not stays as it is beside others)
                    const float first = far ? ref : 0.0f;
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[y][n][i] -= first;
                    ref -= first;
                }
                ref -= P_TOP;
                const float alpha = weight(m[y], m_new);
                float sum = 0.0f;
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float x = __builtin_amdgcn_exp2f(s[y][n][i] - ref);
                        sum += x;
                        const _Float16 hi = (_Float16)x;
                        p[y][n / 2][0][(n % 2) * 4 + i] = hi;
                        if (SPLIT2) p[y][n / 2][NH - 1][(n % 2) * 4 + i] = (_Float16)(x - (float)hi);
                    }
                l[y] = l[y] * alpha + sum;
                m[y] = m_new;
                const float f = alpha * ev_step;
                if (__any(f != 1.0f)) {
#pragma unroll
                    for (int d = 0; d < ND; d++) o[y][d] *= f;
                }
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const h8 a = to_half(vr[d][0], vr[d][1]), b = to_half(vr[d][2], vr[d][3]);
#pragma unroll
                for (int y = 0; y < CG; y++)
#pragma unroll
                    for (int n = 0; n < NH; n++) {
                        o[y][d] = mma(a, p[y][0][n], o[y][d]);
                        o[y][d] = mma(b, p[y][1][n], o[y][d]);
                    }
            }
            if (k + 1 < count) load_v(k + 1);
        }
    }

    // ---- the waves' results joined ----
    constexpr int LROW = HD + 4;
    const float unit = sp_fp8_pow2(ev_now);
#pragma unroll
    for (int y = 0; y < CG; y++) {
        const float sum = column_sum(l[y]);
        if (active[y]) {
            float *rec = smem + (w * n_cols + y * 16 + col) * LROW;
#pragma unroll
            for (int d = 0; d < ND; d++) *reinterpret_cast<f4 *>(rec + d * 16 + g * 4) = o[y][d] * unit;
            if (g == 0) {
                rec[HD] = m[y];
                rec[HD + 1] = sum;
            }
        }
    }
    __syncthreads();
    const long long slot = (long long)sh.slot * A.H + h;
    const bool alone = sh.n_split == 1;
    if (!alone && !slot_fits(A, slot, COLS)) return;
    const int pairs = n_cols * (HD / 2);
    for (int at = tid; at < pairs; at += NT) {
        const int cc = at / (HD / 2), d = at % (HD / 2) * 2;
        Acc acc;
#pragma unroll 4
        for (int v = 0; v < NW; v++) acc.M = fmaxf(acc.M, smem[(v * n_cols + cc) * LROW + HD]);
#pragma unroll 4
        for (int v = 0; v < NW; v++) {
            const float *rec = smem + (v * n_cols + cc) * LROW;
            const float f = weight(rec[HD], acc.M);
            acc.L += rec[HD + 1] * f;
            acc.x += rec[d] * f;
            acc.y += rec[d + 1] * f;
        }
        if (alone) {
            const int n = c0 + cc;
            finish<DT>(A, sh.r0 + n / A.G, h * A.G + n % A.G, HD, d, acc.M, acc.L, acc.x, acc.y);
        } else {
            float *dst = A.part + (slot * COLS + cc) * ROW;
            if (d == 0) put_pair(dst, acc.M, acc.L);
            put_pair(dst + 2 + d, acc.x, acc.y);
        }
    }
    if (alone) return;

    join_shares<HD, DT, NW, COLS>(A, sh, h, c0, n_cols, smem, &last_flag);
}

// ---------------------------------------------------------------------------
// many rows: prompts and their chunks
// ---------------------------------------------------------------------------
// A block of threads holds CW columns a wave and shares each cache block's conversion: the codes
// become fp16 once, in LDS, in the operand order of the matrix instructions, two places deep with
// one barrier a block. As above the scores are K q^T and the weights stay where they were made.
//   CW 32: v_mfma_f32_32x32x16_f16. Lane (column, sub of 2) has positions 8 (i / 4) + 4 sub + i % 4
//          of each 32; V's operand is laid out for that order.
//   CW 16: v_mfma_f32_16x16x32_f16. Lane (column, sub of 4) has positions 16 (i / 4) + 4 sub + i % 4.
// A wave of 32 columns reads LDS half as often a column; one of 16 needs half of the registers,
// which is what puts two waves on a SIMD at head_dim 256 (one of 32 columns takes 77 us where two of
// 16 take 60; with float32 rows 2048 over 8000, 32 / 8 heads, 1050 where they take 757). At head_dim
// 128 both fit, and 32 columns win: 907 us against 1190. With float32 rows there, which take twice
// the queries and weights, 16 win up to 8K (2048 rows 86 us for 106, 12 sequences of 256 rows 242
// for 271, 512 rows over 8000 134 for 135), 32 beyond (2048 over 32000 1516 for 1653): 16 it is.
//
// The loop is pipelined by one cache block: the next block's scores go through the matrix cores
// among this one's weights and its product with V, so that neither unit waits for the other.
//
// The running maximum is a reference that is raised only when a score passes it by W_SLACK
// (the weights, 2^W_TOP at the reference, then still fit fp16), so that the output is rescaled
// a few times in a whole sequence and no exchange between lanes is needed in the others. The
// output counts in units of the strongest V scale of late; a block whose scale is up to
// 2^W_FOLD below has the difference taken off its weights' exponents, for nothing, and only
// others rescale the output. In such a block weights below 2^-18 of the reference are subnormal
// fp16 numbers, rounded at 2^-29 of it. Split weights (fp32 results) count from 2^14, their reference follows
// within a factor of two and their unit always, so that the second part keeps its bits.
//
// Bound by the matrix cores and, beside them, by power: 2048 rows over 32768 positions, 32 / 8 heads
// of 128, take 886 to 935 us by card in a row of calls (1.14 to 1.20 PFLOP/s; a large bf16 matrix product reaches 1.19 to
// 1.24) and 930 to 960 alone, the matrix cores busy 51% of the cycles; the same loop with nothing but its matrix
// instructions takes 595 us at a clock of 1.7 GHz. 2048 rows in a window of 1024, 16 / 8 heads of
// 256: 59 us under the tracer, 52 in a run of calls (0.66 PFLOP/s), 18 blocks a column group with
// 11 us before the first; LDS reads, the codes' conversion and the weights each hide a fifth of the rest.
typedef float f16x __attribute__((ext_vector_type(16)));
template <int DT>
constexpr float WIDE_TOP = DT == SP_DTYPE_F32 ? 14.0f : 12.0f;  // W_TOP

// LDS written before is seen after, by the whole block; loads from memory stay in flight.
__device__ __forceinline__ void lds_barrier() {
    __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int CW>
struct Tile;
template <>
struct Tile<32> {
    typedef f16x V;
    static __device__ __forceinline__ V mma(h8 a, h8 b, V c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Tile<16> {
    typedef f4 V;
    static __device__ __forceinline__ V mma(h8 a, h8 b, V c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

// Place of a row's 16-byte piece s in the row of column c (HD / 8 pieces a row in LDS): the
// pieces that 16 neighbouring columns read at once are in 16 different groups of four banks.
template <int HD>
__device__ __forceinline__ int turned(int c, int s) {
    if (HD % 128 == 0) return s ^ (c & 15);
    if (HD == 64) return s ^ ((c >> 1) & 7);
    const int t = s + ((c >> 2) & 3);  // HD 96: rows of 12 pieces start at every fourth group
    return t >= HD / 8 ? t - HD / 8 : t;
}

template <int HD, int DT, int NW, int CW>
__global__ __launch_bounds__(NW * 64) void k_fp8_attn_wide(SpFp8Attn A) {
    typedef Tile<CW> M;
    typedef typename M::V V;
    constexpr int COLS = CW * NW, TILE = 64 * HD, NT = NW * 64, HT = NT / 2, ROW = HD + 4;
    constexpr int VL = CW == 32 ? 16 : 4;   // values of a lane in a matrix instruction's result
    constexpr int RB = 64 / CW;             // row blocks of a cache block's 64 positions
    constexpr int NE = RB * VL;             // scores of a lane
    constexpr int NP = NE / 8;              // steps of the product with V, eight weights of a lane each
    constexpr int NS = CW == 32 ? HD / 16 : HD / 32;  // steps of the scores
    constexpr int ND = HD / CW;             // row blocks of the output
    constexpr int KE = CW == 32 ? 16 : 32;  // channels of a score step
    constexpr bool SPLIT2 = DT == SP_DTYPE_F32;
    constexpr int NH = SPLIT2 ? 2 : 1;
    constexpr float W_TOP = WIDE_TOP<DT>, W_SLACK = SPLIT2 ? 1.0f : 3.0f;
    constexpr int W_FOLD = SPLIT2 ? 0 : 8;
    constexpr int KP = (HD * 4 + HT - 1) / HT;  // K pieces of 16 codes a thread (half the threads)
    constexpr int VP = (HD * 2 + HT - 1) / HT;  // pairs of V pieces (the other half)
    constexpr int RAW = KP > 2 * VP ? KP : 2 * VP;
    typedef typename SpFp8Elem<DT>::T T;
    extern __shared__ __align__(16) float smem[];  // K, K, V, V: two places each, 64 * HD fp16
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int h = blockIdx.x % A.H;
    Share sh;
    if (!find_share(A, blockIdx.x / A.H, lane, COLS, A.least, false, sh)) return;
    const int c0 = sh.ct * COLS, n_cols = min(sh.n_new * A.G - c0, COLS);
    const int col = lane & (CW - 1), sub = lane / CW;
    const int pos0 = sh.first + c0 / A.G, pos1 = sh.first + (c0 + n_cols - 1) / A.G;
    const int j0 = A.window > 0 ? max(pos0 - A.window + 1, 0) >> 6 : 0;
    const int j1 = min((pos1 >> 6) + 1, A.s.stride);
    const int per = max((j1 - j0 + sh.n_split - 1) / sh.n_split, 0);
    const int t0 = j0 + sh.split * per, n = max(min(t0 + per, j1) - t0, 0);

    // ---- where the blocks are: lane k of a window of 64 ----
    int blk = -1, ekb = 0, evb = 0;
    struct Facts {
        int b;  // block number, -1: none
        int ek, ev;
    };
    const auto facts = [&](int k) __attribute__((always_inline)) {  // called with k = 0, 1, 2, ...
        if ((k & 63) == 0) {
            blk = k + lane < n ? sp_fp8_block(A.s, sh.seq, t0 + k + lane) : -1;
            const long long at = (long long)max(blk, 0) * A.H + h;
            ekb = A.k.exps[at];
            evb = A.v.exps[at];
        }
        return Facts{__builtin_amdgcn_readlane(blk, k & 63), sp_fp8_exponent(__builtin_amdgcn_readlane(ekb, k & 63)),
                     sp_fp8_exponent(__builtin_amdgcn_readlane(evb, k & 63))};
    };
    // ---- staging: half of the waves bring K, half V ----
    // K's piece (uc, g, r), uc = u * HD/32 + c. V's pieces in pairs: CW 32 takes g and g + 2 of a
    // channel, which its operand has side by side; CW 16 two channel groups.
    const bool stage_v = w >= NW / 2;
    const int st = stage_v ? tid - HT : tid;
    u4 raw[RAW];
    const auto fetch = [&](int block) __attribute__((always_inline)) {
        const long long b = (long long)max(block, 0) * A.H + h;  // none: block 0, masked
        if (!stage_v) {
            const uint8_t *p = A.k.codes + b * TILE;
#pragma unroll
            for (int i = 0; i < KP; i++)
                if (KP * HT == HD * 4 || st + i * HT < HD * 4) raw[i] = *reinterpret_cast<const u4 *>(p + (st + i * HT) * 16);
        } else {
            const uint8_t *p = A.v.codes + b * TILE;
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const int x = st + i * HT;
                if (VP * HT == HD * 2 || x < HD * 2) {
                    // CW 32: x = (dg / 2, g % 2, dg % 2, r); CW 16: x = (dg / 2, g, r)
                    const uint8_t *s = CW == 32 ? p + ((x >> 6) * 2 + ((x >> 4) & 1)) * 1024 + ((x >> 5) & 1) * 256 + (x & 15) * 16
                                                : p + (x >> 6) * 2048 + (x & 63) * 16;
                    raw[2 * i] = *reinterpret_cast<const u4 *>(s);
                    raw[2 * i + 1] = *reinterpret_cast<const u4 *>(s + (CW == 32 ? 512 : 1024));
                }
            }
        }
    };
    h8 *const kbuf = reinterpret_cast<h8 *>(smem), *const vbuf = kbuf + 2 * TILE / 8;
    const auto stage = [&](int kb, int vb) __attribute__((always_inline)) {
        if (!stage_v) {
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const int x = st + i * HT, g = (x >> 4) & 3, r = x & 15, uc = x >> 6;
                if (KP * HT == HD * 4 || x < HD * 4) {
                    // row block and step of the operand, lane in it: CW 32 holds positions r and 16 + r of a
                    // 32 in one row block, CW 16 in two
                    h8 *d = kbuf + kb * (TILE / 8) +
                            (CW == 32 ? (uc * 2 + (g >> 1)) * 64 + (g & 1) * 32 + r
                                      : ((uc / (HD / 32)) * 2 * NS + uc % (HD / 32)) * 64 + (x & 63));
                    d[0] = to_half(raw[i][0], raw[i][1]);
                    d[CW == 32 ? 16 : NS * 64] = to_half(raw[i][2], raw[i][3]);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const int x = st + i * HT;
                if (VP * HT == HD * 2 || x < HD * 2) {
                    // (opaque: else the conversions are shared with K's, and moved to where V's go)
                    __asm__("" : "+v"(raw[2 * i]), "+v"(raw[2 * i + 1]));
                    h8 *d = vbuf + vb * (TILE / 8) + (x >> 6) * 256 + (x & 63);
                    if (CW == 32) {
#pragma unroll
                        for (int t4 = 0; t4 < 4; t4++) d[t4 * 64] = to_half(raw[2 * i][t4], raw[2 * i + 1][t4]);
                    } else {
#pragma unroll
                        for (int t4 = 0; t4 < 4; t4++)
                            d[t4 * 64] = to_half(raw[2 * i + t4 / 2][t4 % 2 * 2], raw[2 * i + t4 / 2][t4 % 2 * 2 + 1]);
                    }
                }
            }
        }
    };
    Facts f0{-1, 0, 0}, f1{-1, 0, 0}, f2{-1, 0, 0};  // of blocks k, k + 1, k + 2
    if (n > 0) {
        f0 = facts(0);
        fetch(f0.b);
    }

    // ---- queries ----
    const int mycol = w * CW + col;
    const bool active = mycol < n_cols;
    const int cn = c0 + (active ? mycol : 0), tk = cn / A.G, head = h * A.G + cn % A.G;
    const long long row = (long long)sh.r0 + tk;
    const int pos = active ? sh.first + tk : -1;
    const int from = A.window > 0 ? pos - A.window : -1;  // sees (from, pos]
    // of this wave's columns: whether there are any, and their first and last position
    const bool busy = w * CW < n_cols;
    const int wlast = min(w * CW + CW - 1, n_cols - 1);
    const int wpos0 = sh.first + (c0 + w * CW) / A.G, wpos1 = sh.first + (c0 + wlast) / A.G;
    h8 q[NS][NH];
    int qe;  // scores count in 2^(qe + the block's exponent) * A.c
    {
        // Rows of 16-bit types go through LDS, in 16-byte pieces: loaded as they lie, and read
        // back by column with a row's pieces turned around so that 16 columns' reads meet no bank
        // twice. (Loaded by column, a wave's 16 bytes are in 16 or 32 rows at a time.)
        const T *src = reinterpret_cast<const T *>(A.q) + row * A.q_stride + (long long)head * HD + sub * 8;
        const bool aligned = (uintptr_t)A.q % (4 * sizeof(T)) == 0 && A.q_stride % 4 == 0;
        const bool pieces = !SPLIT2 && (uintptr_t)A.q % 16 == 0 && A.q_stride % 8 == 0;
        const auto piece = [&](int c, int s) {
            return reinterpret_cast<u4 *>(smem) + c * (HD / 8) + turned<HD>(c, s);
        };
        if (pieces) {
            u4 got[COLS * HD / 8 / NT];
#pragma unroll
            for (int i = 0; i < COLS * HD / 8 / NT; i++) {
                const int at = tid + i * NT, nn = c0 + min(at / (HD / 8), n_cols - 1);
                got[i] = *reinterpret_cast<const u4 *>(reinterpret_cast<const T *>(A.q) + (long long)(sh.r0 + nn / A.G) * A.q_stride +
                                                       (long long)(h * A.G + nn % A.G) * HD + at % (HD / 8) * 8);
            }
#pragma unroll
            for (int i = 0; i < COLS * HD / 8 / NT; i++) *piece((tid + i * NT) / (HD / 8), (tid + i * NT) % (HD / 8)) = got[i];
            lds_barrier();
        }
        const auto eight = [&](int s, float x[8]) __attribute__((always_inline)) {
            if (pieces) load8<DT>(reinterpret_cast<const T *>(piece(mycol, s * (KE / 8) + sub)), true, x);
            else load8<DT>(src + s * KE, aligned, x);
        };
        float top = 0.0f;
        float x[8];
#pragma unroll
        for (int s = 0; s < NS; s++) {
            eight(s, x);
#pragma unroll
            for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(x[k]));
        }
        if (CW == 16) top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        int e = (__float_as_int(top) >> 23) - 127 - 14;
        e = top == 0.0f || !(top < INFINITY) ? 0 : max(e, -126);
        const float down = A.negate ? -sp_fp8_pow2(-e) : sp_fp8_pow2(-e);
        qe = e + 1;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            eight(s, x);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float v = active ? x[k] * down : 0.0f;
                const _Float16 hi = (_Float16)v;
                q[s][0][k] = hi;
                if (SPLIT2) q[s][NH - 1][k] = (_Float16)(v - (float)hi);
            }
        }
    }
    lds_barrier();  // the queries are in registers: LDS is for the blocks

    V o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = V{};
    // m: the reference; off = W_TOP - m (far: -m), 0 while m is -inf; most: what a score and off
    // may come to before the reference is raised; the output's unit is 2^ev_now
    float m = -INFINITY, off = 0.0f, most = -INFINITY, l = 0.0f;
    int ev_now = 0;
    // the column's reference is past FAR_SCORE: the fused difference of a score and the reference would not
    // be 0 where they are equal, and the constants added to the reference would be rounded
    bool far = false;
    // of the block whose weights come next: score scale, exponent offset, its part in l
    float cs = 0.0f, shift = 0.0f, lmul = 1.0f;
    h8 p[NP][NH];

    // out^T += V^T p^T for one of the NP steps
    const auto product = [&](auto step, const h8 *vd) __attribute__((always_inline)) {
        constexpr int t = decltype(step)::value;
        constexpr int AT_ONCE = ND % 4 == 0 ? 4 : ND % 3 == 0 ? 3 : 2;  // operands read before the first is used
#pragma unroll
        for (int d0 = 0; d0 < ND; d0 += AT_ONCE) {
            h8 a[AT_ONCE];
#pragma unroll
            for (int d = 0; d < AT_ONCE; d++) a[d] = vd[((d0 + d) * NP + t) * 64];
#pragma unroll
            for (int d = 0; d < AT_ONCE; d++)
#pragma unroll
                for (int x = 0; x < NH; x++) o[d0 + d] = M::mma(a[d], p[t][x], o[d0 + d]);
        }
    };
    // next = K q^T of one block; of the one before, the weights from its scores and all but the
    // last step of the product with V
    const auto blend = [&](auto with_scores, auto with_weights, const h8 *kd, const h8 *vd, V(&next)[RB],
                           const V(&s)[RB]) __attribute__((always_inline)) {
        float sum = 0.0f;
        // K's operands are read two steps ahead (one at CW 16, whose steps are twice as many reads)
        constexpr int AHEAD = CW == 32 ? 2 : 1;
        h8 ka[AHEAD + 1][RB];
        if constexpr (decltype(with_scores)::value) {
#pragma unroll
            for (int c = 0; c < AHEAD; c++)
#pragma unroll
                for (int b = 0; b < RB; b++) ka[c][b] = kd[(b * NS + c) * 64];
        }
#pragma unroll
        for (int c = 0; c < NS; c++) {
            if constexpr (decltype(with_scores)::value) {
                if (c + AHEAD < NS) {
#pragma unroll
                    for (int b = 0; b < RB; b++) ka[(c + AHEAD) % (AHEAD + 1)][b] = kd[(b * NS + c + AHEAD) * 64];
                }
#pragma unroll
                for (int x = 0; x < NH; x++)
#pragma unroll
                    for (int b = 0; b < RB; b++) next[b] = M::mma(ka[c % (AHEAD + 1)][b], q[c][x], c || x ? next[b] : V{});
            }
            if constexpr (decltype(with_weights)::value) {
#pragma unroll
                for (int i = c * (NE / 2) / NS * 2; i < (c + 1) * (NE / 2) / NS * 2; i++) {
                    const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / VL][i % VL], cs, shift));
                    sum += x;
                    const _Float16 hi = (_Float16)x;
                    p[i >> 3][0][i & 7] = hi;
                    if (SPLIT2) p[i >> 3][NH - 1][i & 7] = (_Float16)(x - (float)hi);
                }
                // the steps whose weights were complete before this one
                const int done = c * (NE / 2) / NS * 2 / 8, before = c ? (c - 1) * (NE / 2) / NS * 2 / 8 : 0;
                if (done > before) {
                    if (done == 1) product(std::integral_constant<int, 0>(), vd);
                    if constexpr (NP == 4) {
                        if (done == 2) product(std::integral_constant<int, 1>(), vd);
                        if (done == 3) product(std::integral_constant<int, 2>(), vd);
                    }
                }
            }
        }
        if constexpr (decltype(with_weights)::value) l += sum * lmul;
    };
    const auto mask = [&](const Facts &f, int k, V(&s)[RB]) __attribute__((always_inline)) {
        const int t = t0 + k;
        if (f.b >= 0 && t * 64 + 63 <= wpos0 && (A.window <= 0 || t * 64 > wpos1 - A.window)) return;
        const int lane0 = t * 64 + 4 * sub, upto = f.b < 0 ? -1 : pos - lane0, before = from - lane0;
#pragma unroll
        for (int i = 0; i < NE; i++) {
            const int at = CW == 32 ? (i >> 2) * 8 + (i & 3) : (i >> 2) * 16 + (i & 3);
            s[i / VL][i % VL] = at <= upto && at > before ? s[i / VL][i % VL] : -INFINITY;
        }
    };
    const auto largest = [&](const V(&s)[RB]) __attribute__((always_inline)) {
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < NE; i++) top = fmaxf(top, s[i / VL][i % VL]);
        return top;
    };
    // the reference and the output's unit for a block with largest score `top` (this lane's)
    const auto settle = [&](const Facts &f, float top, V(&s)[RB]) __attribute__((always_inline)) {
        // never 0: a masked score stays -inf when it is multiplied
        cs = fmaxf(score_scale(A, qe + f.ek), 0x1p-126f);
        const bool raise = __builtin_fmaf(top, cs, off) > most;
        float scale = 1.0f;
        bool rescale = false;
        if (f.ev > ev_now || f.ev < ev_now - W_FOLD) {
            scale = sp_fp8_pow2(ev_now - f.ev);
            ev_now = f.ev;
            rescale = true;
        }
        if (__any(raise)) {
            if (CW == 16) top = fmaxf(top, __shfl_xor(top, 16, 64));
            const float mx = fmaxf(top, __shfl_xor(top, 32, 64)) * cs, m_new = fmaxf(m, mx);
            const float alpha = weight(m, m_new);
            l *= alpha;
            scale *= alpha;
            m = m_new;
            rescale = true;
            far = is_far(m);
            off = m == -INFINITY ? 0.0f : (far ? 0.0f : W_TOP) - m;
            // (far: whatever is past the reference raises it, since what is less than half a float's step past
            // it may be rounded to a whole one)
            most = m == -INFINITY ? -INFINITY : far ? 0.0f : W_TOP + W_SLACK;
        }
        shift = off;
        if (far) {  // the reference was rounded: round the scores as it was, and take it off first
#pragma unroll
            for (int i = 0; i < NE; i++) s[i / VL][i % VL] = s[i / VL][i % VL] * cs + off;
            cs = 1.0f;
            shift = W_TOP;
        }
        if (rescale) {
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= scale;
        }
        shift += (float)(f.ev - ev_now);
        lmul = sp_fp8_pow2(ev_now - f.ev);
    };
    const std::true_type yes;
    const std::false_type no;
    const std::integral_constant<int, NP - 1> last_step;

    // ---- block 0's scores; K one block ahead of V from here ----
    // Blocks past the last are fetched as block 0 and never used: no turn asks for its place.
    constexpr int STEP = TILE / 8;
    V sa[RB], sb[RB];
    if (n > 0) {
        stage(0, 0);
        f1 = facts(1);
        f2 = facts(2);
        fetch(f1.b);
    }
    lds_barrier();
    if (n > 0) {
        if (busy) {
            blend(yes, no, kbuf + lane, nullptr, sa, sa);
            mask(f0, 0, sa);
            ev_now = f0.ev;
            settle(f0, largest(sa), sa);
        }
        if (!stage_v) {
            stage(1, 0);
            fetch(f2.b);
        }
    }
    lds_barrier();
    // at turn k: K of block k + 1 and V of block k are in LDS, registers hold K of k + 2 or V of k + 1
    const auto bring = [&](int k) __attribute__((always_inline)) {
        stage(k & 1, 1 - (k & 1));
        const Facts f3 = facts(k + 3);
        fetch(stage_v ? f2.b : f3.b);
        f1 = f2;
        f2 = f3;
    };
    const auto turn = [&](int k, V(&s)[RB], V(&next)[RB]) __attribute__((always_inline)) {
        const Facts f = f1;
        const h8 *vd = vbuf + (k & 1) * STEP + lane;
        // The conversion comes first, and the stretch that keeps the matrix cores fed has the wave's
        // priority over the other one's conversion and maximum: 955 us without both, 903 with them
        // (2048 rows over 32768, heads of 128).
        bring(k);
        __builtin_amdgcn_s_setprio(1);
        blend(yes, yes, kbuf + (1 - (k & 1)) * STEP + lane, vd, next, s);
        __builtin_amdgcn_s_setprio(0);
        product(last_step, vd);
        mask(f, k + 1, next);
        settle(f, largest(next), next);
        lds_barrier();
    };
    if (busy) {
        int k = 0;
        for (; k + 2 < n; k += 2) {
            turn(k, sa, sb);
            turn(k + 1, sb, sa);
        }
        if (k + 1 < n) {
            turn(k, sa, sb);
#pragma unroll
            for (int b = 0; b < RB; b++) sa[b] = sb[b];
            k++;
        }
        if (k < n) {  // the last one: no more scores
            const h8 *vd = vbuf + (k & 1) * STEP + lane;
            blend(no, yes, nullptr, vd, sa, sa);
            product(last_step, vd);
        }
    } else {  // no columns: bring blocks for the other waves
        for (int k = 0; k + 1 < n; k++) {
            bring(k);
            lds_barrier();
        }
    }
    lds_barrier();
    if (CW == 16) l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // ---- results ----
    // of lane values i .. i + 3 of row block d: channels from
    const auto channel = [&](int d, int i) { return d * CW + i * 2 + 4 * sub; };
    const float unit = sp_fp8_pow2(ev_now);
    if (sh.n_split > 1) {  // joined by k_fp8_attn_join
        const long long slot = (long long)sh.slot * A.H + h;
        if (active && slot_fits(A, slot, COLS)) {
            float *dst = A.part + (slot * COLS + mycol) * ROW;
            if (sub == 0) *reinterpret_cast<Two *>(dst + HD) = Two{m, l};
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int i = 0; i < VL; i += 4)
                    *reinterpret_cast<f4 *>(dst + channel(d, i)) =
                        f4{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]} * unit;
        }
        return;
    }
    // as the queries came: by column into LDS, in rows to memory
    const bool through = !SPLIT2 && (uintptr_t)A.out % 16 == 0 && A.out_stride % 8 == 0;
    if (active) {
        const float r = l == 0.0f ? 0.0f : unit / l;
        const bool aligned = (uintptr_t)A.out % (4 * sizeof(T)) == 0 && A.out_stride % 4 == 0;
        T *out = through ? reinterpret_cast<T *>(smem) : reinterpret_cast<T *>(A.out) + row * A.out_stride + (long long)head * HD;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < VL; i += 4) {
                f4 x;
#pragma unroll
                for (int j = 0; j < 4; j++) x[j] = l == 0.0f ? 0.0f : o[d][i + j] * r;
                const int ch = channel(d, i);
                if (through) store4<DT>(out, (mycol * (HD / 8) + turned<HD>(mycol, ch >> 3)) * 8 + (ch & 4), x, true);
                else store4<DT>(out, ch, x, aligned);
            }
        if (A.lse && sub == 0)
            A.lse[row * A.H * A.G + head] = l == 0.0f ? -INFINITY : (m + (__log2f(l) - W_TOP)) * 0.69314718055994531f;
    }
    if (!through) return;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < COLS * HD / 8 / NT; i++) {
        const int at = tid + i * NT, c = at / (HD / 8), nn = c0 + c;
        if (c < n_cols)
            *reinterpret_cast<u4 *>(reinterpret_cast<T *>(A.out) + (long long)(sh.r0 + nn / A.G) * A.out_stride +
                                    (long long)(h * A.G + nn % A.G) * HD + at % (HD / 8) * 8) =
                reinterpret_cast<const u4 *>(smem)[c * (HD / 8) + turned<HD>(c, at % (HD / 8))];
    }
}

// Joins the shares of the column groups that have more than one, in their order. A launch of its
// own: a group's partial results are 64 to 128 KB a share, too many for the last block to
// arrive alone. Blocks of threads: (KV head, column group) by as many columns as 256 threads take
// at once, four channels each (with 32 columns a block, four to eight rounds of dependent loads:
// 1250 rows over 8930 positions of one head of 256 took 67 us, not 39).
template <int HD>
constexpr int JOIN_COLS = HD == 64 ? 16 : HD == 256 ? 4 : 8;

template <int HD, int DT, int COLS>
__global__ __launch_bounds__(256) void k_fp8_attn_join(SpFp8Attn A) {
    constexpr int ROW = HD + 4, PER = HD / 4;
    static_assert(JOIN_COLS<HD> * PER <= 256 && COLS % JOIN_COLS<HD> == 0);
    typedef typename SpFp8Elem<DT>::T T;
    const int h = blockIdx.x % A.H;
    Share sh;
    if (!find_share(A, blockIdx.x / A.H, threadIdx.x & 63, COLS, A.least, true, sh) || sh.n_split == 1) return;
    const long long slot0 = (long long)sh.slot * A.H + h;
    if (!slot_fits(A, slot0 + (long long)(sh.n_split - 1) * A.H, COLS)) return;
    const int c0 = sh.ct * COLS, n_cols = min(sh.n_new * A.G - c0, COLS);
    const bool aligned = (uintptr_t)A.out % (4 * sizeof(T)) == 0 && A.out_stride % 4 == 0;
    const int c = blockIdx.y * JOIN_COLS<HD> + threadIdx.x / PER, d = threadIdx.x % PER * 4;
    if ((int)threadIdx.x >= JOIN_COLS<HD> * PER || c >= n_cols) return;
    const float *src = A.part + (slot0 * COLS + c) * ROW;
    const long long step = (long long)A.H * COLS * ROW;
    float M = -INFINITY, L = 0.0f;
    f4 x = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int v0 = 0; v0 < sh.n_split; v0 += 8) {
        Two ml[8];
        f4 part[8];
#pragma unroll
        for (int v = 0; v < 8; v++) {
            const float *rec = src + min(v0 + v, sh.n_split - 1) * step;
            ml[v] = *reinterpret_cast<const Two *>(rec + HD);
            part[v] = *reinterpret_cast<const f4 *>(rec + d);
        }
#pragma unroll
        for (int v = 0; v < 8; v++)
            if (v0 + v < sh.n_split) {
                const float Mn = fmaxf(M, ml[v].x), a = weight(M, Mn), b = weight(ml[v].x, Mn);
                L = L * a + ml[v].y * b;
                x = x * a + part[v] * b;
                M = Mn;
            }
    }
    const int nn = c0 + c, head = h * A.G + nn % A.G;
    const long long row = (long long)sh.r0 + nn / A.G;
    const float r = L == 0.0f ? 0.0f : 1.0f / L;
#pragma unroll
    for (int j = 0; j < 4; j++) x[j] = L == 0.0f ? 0.0f : x[j] * r;
    store4<DT>(A.out, row * A.out_stride + (long long)head * HD + d, x, aligned);
    if (A.lse && d == 0)
        A.lse[row * A.H * A.G + head] = L == 0.0f ? -INFINITY : (M + (__log2f(L) - WIDE_TOP<DT>)) * 0.69314718055994531f;
}

template <int HD, int DT, int NW, int CG>
hipError_t launch(const SpFp8Attn &A, hipStream_t s) {
    constexpr int COLS = 16 * CG;
    SpFp8Attn a = A;
    a.target = min(A.target, 256);
    // column groups: each sequence's rows times G, in groups of COLS
    const long long groups = A.s.row ? ((long long)A.s.n_rows * A.G) / COLS + A.s.n_seq
                                     : (long long)A.s.n_seq * ((A.G + COLS - 1) / COLS);
    // shares: one per group, and at most target more over all KV heads
    const long long blocks = (groups + (a.target + A.H - 1) / A.H) * A.H;
    if (blocks * (NW * 64) > SP_FP8_MOST_THREADS) return hipErrorInvalidValue;
    const int cols = A.s.row ? COLS : (A.G < COLS ? A.G : COLS);
    const size_t lds = (size_t)NW * cols * (HD + 4) * sizeof(float);
    const long long each = A.s.row ? ((long long)A.s.n_rows * A.G + A.s.n_seq - 1) / A.s.n_seq : A.G;
    a.join = (float)min(each, (long long)COLS) * (HD / 2) / (NW * 64);
    void *args[] = {&a};
    const void *f = (const void *)k_fp8_attn<HD, DT, NW, CG>;
    return hipLaunchKernel(f, dim3((unsigned)blocks), dim3(NW * 64), args, lds, s);
}

template <int HD, int DT>
hipError_t launch_wide(const SpFp8Attn &A, hipStream_t s) {
    constexpr int CW = HD == 256 || (HD == 128 && DT == SP_DTYPE_F32) ? 16 : 32, NW = 8;
    constexpr int COLS = CW * NW;
    SpFp8Attn a = A;
    a.target = min(A.target, 256);
    const long long groups = (long long)A.s.n_rows * A.G / COLS + A.s.n_seq;
    // With a block for each CU sharing gains nothing. Below that a group is shared out where the
    // others leave CUs idle, and a second launch joins the shares.
    // (No sequence's rows see more than `most` cache blocks; up to 4 * LEAST are not shared out. Waves
    // of 16 columns take two blocks a share: 512 rows over 768 positions of one head of 256 20 us for 34;
    // of 32 they are the slower ones, 1024 rows from position 0 of 8 heads of 128 44 us for 40.)
    constexpr int LEAST = CW == 16 ? 2 : 4;
    const long long most = A.window > 0 ? min((long long)A.s.stride, ((long long)A.s.n_rows + A.window + 126) / 64) : A.s.stride;
    const bool share = groups * A.H < a.target && most > 4 * LEAST;
    a.least = share ? LEAST : 1 << 28;
    a.join = 0.0f;
    const long long blocks = (groups + (share ? (a.target + A.H - 1) / A.H : 0)) * A.H;
    if (blocks * (NW * 64) > SP_FP8_MOST_THREADS) return hipErrorInvalidValue;
    void *args[] = {&a};
    const hipError_t e = hipLaunchKernel((const void *)k_fp8_attn_wide<HD, DT, NW, CW>, dim3((unsigned)blocks), dim3(NW * 64),
                                         args, (size_t)HD * 512, s);
    if (e != hipSuccess || !share) return e;
    return hipLaunchKernel((const void *)k_fp8_attn_join<HD, DT, COLS>, dim3((unsigned)(groups * A.H), COLS / JOIN_COLS<HD>),
                           dim3(256), args, 0, s);
}

template <int HD, int DT>
hipError_t launch_dt(const SpFp8Attn &A, hipStream_t s) {
    constexpr int NW = HD == 256 ? 4 : 8;
    // 32 columns a wave where their output, queries and weights fit its registers (12 sequences of 1 to
    // 4.5K, 32 columns each: head_dim 256 48 us with 16 and 80 with 32, fp32 rows at 128 26 and 45).
    constexpr int CG = HD == 256 || DT == SP_DTYPE_F32 ? 1 : 2;
    const long long columns = (long long)A.s.n_rows * A.G;  // of each KV head
    // The kernel for many rows takes a cache block over 256 columns at once (128 in waves of 16), this
    // one over 32 or 16 and reads it again for the next. What decides is how many columns there are over
    // all KV heads (a few blocks of threads with many columns each leave the chip idle) and how many a
    // sequence has (columns that none has are worked through). The longer the context the better for
    // the other, but the host does not know it. Measured, few rows / many in us, one sequence:
    //   columns x heads              4096        8192        16384       32768
    //   head_dim 64     from 0       8 / 10      9 / 13      16 / 18     33 / 28
    //                   over 8K      31 / 32     46 / 43     86 / 65
    //     float32 rows  from 0       7 / 13      11 / 17     23 / 24     51 / 41
    //                   over 8K      36 / 40     67 / 58     126 / 89
    //   head_dim 96     from 0       9 / 12      10 / 16     20 / 22     43 / 37
    //                   over 8K      37 / 39     53 / 54     100 / 81
    //     float32 rows  from 0       9 / 17      15 / 22     30 / 33     66 / 53
    //                   over 8K      45 / 50     83 / 72     157 / 117
    //   head_dim 128    from 0       11 / 14     12 / 18     24 / 25     52 / 40
    //                   over 8K      43 / 44     62 / 60     114 / 90
    //                   over 32K     118 / 96    194 / 160
    //     one head, two from 0       15 / 22     23 / 32
    //     one head, two over 8K      42 / 43     59 / 56
    //     float32 rows  from 0       10 / 14     17 / 18     35 / 26     76 / 43
    //                   over 8K      52 / 52     100 / 83    180 / 145
    //   head_dim 256    from 0       11 / 15     21 / 20     44 / 30     102 / 49
    //                   over 8K      76 / 61     141 / 100   268 / 171
    //     one head, two over 8K      74 / 60     130 / 93
    //     float32 rows  from 0       13 / 22     25 / 31     52 / 46     120 / 75
    //                   over 8K      94 / 91     178 / 149   326 / 252
    // Twelve sequences of 1 to 4.5K, 8 heads, 42 / 84 / 168 columns each: head_dim 64 22 / 35, 39 / 37,
    // 52 / 48; 128 32 / 47, 53 / 51, 74 / 69, float32 rows -, 62 / 61, 104 / 101; 256 68 / 58, 92 / 74,
    // 149 / 119; 24 and 40 sequences of 256 with 42 columns 102 / 131, 122 / 137.
    constexpr bool F32 = DT == SP_DTYPE_F32;
    // Up to a column group of this kernel's on each CU (8192 columns; 4096 in waves of 16) it is the
    // better one over short contexts and within 7% of the other over 8K; past that it takes a second turn
    // (300 rows over 16000, head_dim 128: 188 / 116), and the other is taken, though it is up to 2 us slower
    // (7 with float32 rows) where such a call starts at position 0: it saves 9 to 40 over 8K. At head_dim
    // 256, where this one reads more, the other from 4096 on: 4 us slower from 0 (float32 rows 9), 15 (3)
    // faster over 8K.
    constexpr int MANY = 256 * 16 * CG + (HD == 256 ? 0 : 1), EACH = F32 ? 128 : 64;
    if (A.s.row && columns * A.H >= MANY && columns >= EACH * (long long)A.s.n_seq) return launch_wide<HD, DT>(A, s);
    if (columns > 16ll * A.s.n_seq) return launch<HD, DT, NW, CG>(A, s);
    return launch<HD, DT, NW, 1>(A, s);
}

template <int HD>
hipError_t launch_hd(const SpFp8Attn &A, int dtype, hipStream_t s) {
    switch (dtype) {
        case SP_DTYPE_F32: return launch_dt<HD, SP_DTYPE_F32>(A, s);
        case SP_DTYPE_F16: return launch_dt<HD, SP_DTYPE_F16>(A, s);
        case SP_DTYPE_BF16: return launch_dt<HD, SP_DTYPE_BF16>(A, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t sp_fp8_launch_attn(const SpFp8Attn &A, int hd, int dtype, hipStream_t s) {
    switch (hd) {
        case 64: return launch_hd<64>(A, dtype, s);
        case 96: return launch_hd<96>(A, dtype, s);
        case 128: return launch_hd<128>(A, dtype, s);
        case 256: return launch_hd<256>(A, dtype, s);
    }
    return hipErrorInvalidValue;
}

// sp_fp4_evict.hip -- attention weights added to the positions of the 4-bit block cache, and eviction by
// them.
//
// Weigh: for each position t and KV head, w_t += sum over the call's rows and the query heads of that
// KV head of e^{s_t - lse}, with the scores of the attention that gave lse. The sums are fp32.
#include "sp_block_attn.h"
#include "sp_fp4.h"

namespace {

using namespace sp_block;
using sp_fp4::eight;
using sp_fp4::Largest;
using sp_fp4::relative;

// The float with exponent byte b of rel.
__device__ __forceinline__ float power(unsigned rel, int b) {
    return __int_as_float((b == 3 ? rel >> 1 : rel << (23 - 8 * b)) & 0x7f800000);
}

// ---------------------------------------------------------------------------
// weigh
// ---------------------------------------------------------------------------
// A wave holds one block's K as operands, converted once, and the eight waves of a block of threads take
// eight consecutive blocks of a sequence, or fewer and part of the columns each. Columns (row, query head) pass by in stages: the block of
// threads brings them into LDS as operands, and each wave takes them 16 at a time. The weights are
// summed over columns in the registers that the scores come in, and over the 16 lanes at the end.
//
// Queries of 16-bit types are operands as they are, with K in their type: no maximum to look for, no
// conversion. K counts relative to the block's largest exponent and is what attention sees of it: an fp16 number. As
// bf16 that is the same number wherever no exponent is more than 23 below the largest; of other blocks (empty
// rows among them) the fp16 numbers are made first (see Operand). fp32 queries are scaled by a power of two and
// split in two fp16 parts, as in attention.
//
// Bound for many columns by the matrix cores and the exponentials (for 64 positions of 16 columns 16 and 16
// instructions of 16 and 8 cycles at head_dim 128, beside two multiply-adds a weight): 64 rows over 32768
// positions, 32 / 8 heads, bf16, 26.5 us, 0.65 PFLOP/s. For few by latencies: one row of 12 sequences of 1 to 4.5K
// 10.8 us (21 MB of K), of which an empty launch is 4.
constexpr int WN = 512;  // threads
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// Four or sixteen bytes a lane from memory to LDS: lane l's to the l-th place from `to`. The wave waits for
// them as for loads.
typedef __attribute__((address_space(1))) void Global;
typedef __attribute__((address_space(3))) void Shared;
__device__ __forceinline__ void to_lds16(const void *from, void *to) { __builtin_amdgcn_global_load_lds((Global *)from, (Shared *)to, 16, 0, 0); }
__device__ __forceinline__ void to_lds4(const void *from, void *to) { __builtin_amdgcn_global_load_lds((Global *)from, (Shared *)to, 4, 0, 0); }

template <int DT>
struct Operand {
    typedef h8 V;
    // K counts in 2^-down(c, top) of the block's largest scale.
    static __device__ __forceinline__ int down(float, int) { return 0; }
    static __device__ __forceinline__ V codes(unsigned w, float scale) { return eight(w, scale); }
    static __device__ __forceinline__ V seen(unsigned w, float scale, int) { return eight(w, scale); }
    static __device__ __forceinline__ f4 mma(V a, V b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Operand<SP_DTYPE_BF16> {
    typedef b8 V;
    // bf16 queries may be as large or small as a float, where kq_scale makes up for it: a product of a query's entry
    // and a K that counts relative to its block alone may leave a float's range though the score is ordinary. So K
    // counts in 2^-60 of what it adds to a score in powers of two. Sums of finite queries stay finite (but
    // where a score's terms pass 2^188), and what vanishes below a float is less than 2^-66 of a power of two. At most 2^-100
    // of the block's scale, where the least that is seen is still a normal bf16 number (such terms vanish below 2^-66 too).
    static __device__ __forceinline__ int down(float c, int top) {
        const int unit = (__float_as_int(c) >> 23) - 127 + 1 + top - 127;  // of scores, in log2
        return min(60 - unit, 100);
    }
    static __device__ __forceinline__ V codes(unsigned w, float scale) {
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 0), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 2), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, 3);
        return b8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
    // Eight codes as attention sees them: multiples of 2^-24 of the block's largest scale. (At most two bits of an
    // fp16 number that small are left, or the code's own: exact in bf16.)
    static __device__ __forceinline__ V seen(unsigned w, float scale, int down) {
        const float unit = sp_fp8_pow2(-down);
        const h8 x = eight(w, scale);
        V v;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = (__bf16)((float)x[k] * unit);
        return v;
    }
    static __device__ __forceinline__ f4 mma(V a, V b, f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};

// DIRECT (16-bit rows at multiples of 16 bytes): a stage's pieces go from memory to LDS past the registers,
// a wave's 16 bytes a lane as one operand, while the stage before is worked on.
// SHARED: a block of threads takes 2^A.blocks blocks, and its waves share the columns; else eight. (The shared one
// takes 11.6 us where the other takes 10.5 for the step of 12 sequences below.)
template <int HD, int DT, bool DIRECT, bool SHARED>
__global__ __launch_bounds__(WN, HD == 256 || (!DIRECT && (HD == 128 || (HD == 96 && SHARED))) ? 2 : 4) void k_fp4_weigh(SpFp4Weigh A, int items) {
    typedef Operand<DT> Op;
    typedef typename Op::V V;
    constexpr int NC = HD / 32, NW = WN / 64;
    constexpr int LP = HD == 64 ? 8 : HD == 256 ? 32 : 16;  // threads of a column (96: twelve of them have a part)
    constexpr bool SPLIT2 = DT == SP_DTYPE_F32;
    constexpr int NH = SPLIT2 ? 2 : 1;
    // Columns of a stage. (Staged by way of registers, 128 of them leave room for half of the waves at head_dim 96: 20 us
    // for 13 in a step of 12 sequences of 1 to 4.5K; but waves that share them want a part each: 79 us for 114 with
    // 512 rows over 2048 positions, 32 / 8 heads of 128.)
    constexpr int CS = DIRECT || SHARED ? (HD == 256 ? 64 : 128) : HD == 64 ? 128 : WN / LP;
    constexpr int PER = CS * LP / WN;            // of a thread
    constexpr int BUF = CS / 16 * NC * NH * 64;  // eights of a stage
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T8 __attribute__((ext_vector_type(8)));
    struct Column {
        float lse;  // +inf: adds nothing
        int qe;     // scores count in 2^(qe + the block's exponent) * A.c
    };
    __shared__ __align__(16) V qs[(DIRECT ? 2 : 1) * BUF];
    __shared__ Column col_of[DIRECT ? 1 : CS];
    __shared__ float lse_of[DIRECT ? 2 * CS : 1];
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int h = blockIdx.y, r = lane & 15, g = lane >> 4;
    const int two = SHARED ? A.blocks : 3;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        // ---- the sequence, and 2^two blocks of those that its rows see ----
        int seq = -1, r0 = 0, n_new = 0, first = 0, j0 = 0, left = item;
        for (int i0 = 0; i0 < A.s.n_seq && seq < 0; i0 += 64) {
            int a = 0, b = 0, len = 0, lo = 0, n = 0;
            if (i0 + lane < A.s.n_seq) {
                sp_fp8_seq(A.s, i0 + lane, a, b, len);
                lo = A.window > 0 ? max(len - (b - a) - A.window + 1, 0) >> 6 : 0;
                if (b > a) n = (max(min((len + 63) >> 6, A.s.stride) - lo, 0) + (1 << two) - 1) >> two;
            }
            const int sum = sp_fp8_scan(n, lane);
            const unsigned long long past = __ballot(sum > left);
            if (past) {
                const int l = __ffsll(past) - 1;
                const auto of = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
                seq = i0 + l;
                r0 = of(a);
                n_new = of(b) - r0;
                first = of(len) - n_new;
                j0 = of(lo) + ((left - (of(sum) - of(n))) << two);
            } else {
                left -= __builtin_amdgcn_readlane(sum, 63);
            }
        }
        if (seq < 0) return;
        const int t = j0 + (w & ((1 << two) - 1)), n_cols = n_new * A.G;
        const int blk = uniform(t <= (first + n_new - 1) >> 6 ? sp_fp8_block(A.s, seq, t) : -1);
        const long long tile = (long long)max(blk, 0) * A.H + h;
        // ---- columns: this thread's eight entries of some, into LDS (staged: one by one, which takes no longer
        // than in vectors of four: 64 rows over 32768 positions, 32 / 8 heads of 128, 54.7 and 55.3 us with float32 rows) ----
        const auto direct = [&](int c0, int buf) __attribute__((always_inline)) {
            const int here = min(n_cols - c0, CS);
            for (int f = w; f < (here + 15) / 16 * NC; f += NW) {  // fragments: 16 columns, 32 channels
                const int n = c0 + min(f / NC * 16 + r, here - 1);
                const T *src = reinterpret_cast<const T *>(A.q) + (long long)(r0 + n / A.G) * A.q_stride +
                               (long long)(h * A.G + n % A.G) * HD + f % NC * 32 + g * 8;
                to_lds16(src, qs + buf * BUF + f * 64);
            }
            for (int c = w * 64; c < here; c += WN) {
                const int n = c0 + min(c + lane, here - 1);
                to_lds4(A.lse + (long long)(r0 + n / A.G) * A.H * A.G + h * A.G + n % A.G, lse_of + buf * CS + c);
            }
        };
        const int mine = tid / LP, part = tid % LP;
        const auto stage = [&](int c0) __attribute__((always_inline)) {
            T8 raw[PER];
            float lse[PER];
#pragma unroll
            for (int y = 0; y < PER; y++) {
                const int n = c0 + y * (WN / LP) + mine;
                raw[y] = T8{};
                lse[y] = INFINITY;
                if (n >= n_cols) continue;
                const int row = r0 + n / A.G, head = h * A.G + n % A.G;
                lse[y] = A.lse[(long long)row * A.H * A.G + head];
                if (part >= HD / 8) continue;
                const T *src = reinterpret_cast<const T *>(A.q) + (long long)row * A.q_stride + (long long)head * HD + part * 8;
#pragma unroll
                for (int k = 0; k < 8; k++) raw[y][k] = src[k];
            }
#pragma unroll
            for (int y = 0; y < PER; y++) {
                if (c0 + y * (WN / LP) >= n_cols) break;
                const int c = y * (WN / LP) + mine;
                // not: rows that see nothing, and those whose scores are no numbers
                bool finite = true;
#pragma unroll
                for (int k = 0; k < 8; k++) finite = finite && fabsf(SpFp8Elem<DT>::get(raw[y][k])) < INFINITY;
                const unsigned long long odd = __ballot(!finite) >> (lane & ~(LP - 1));
                const bool active = fabsf(lse[y]) < INFINITY && (odd & ((1ull << LP) - 1)) == 0;
                V q[NH];
                int qe = 1;
                if constexpr (!SPLIT2) {
#pragma unroll
                    for (int k = 0; k < 8; k++) q[0][k] = active ? raw[y][k] : (T)0.0f;
                } else {
                    float top = 0.0f;
#pragma unroll
                    for (int k = 0; k < 8; k++) top = fmaxf(top, fabsf(raw[y][k]));
#pragma unroll
                    for (int s = LP / 2; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
                    int e = (__float_as_int(top) >> 23) - 127 - 14;
                    e = top == 0.0f || !active ? 0 : max(e, -126);
                    const float down = sp_fp8_pow2(-e);
                    qe = e + 1;
#pragma unroll
                    for (int k = 0; k < 8; k++) {
                        const float v = active ? raw[y][k] * down : 0.0f;
                        const _Float16 hi = (_Float16)v;
                        q[0][k] = hi;
                        q[NH - 1][k] = (_Float16)(v - (float)hi);
                    }
                }
                if (part < HD / 8) {
                    V *d = qs + ((c >> 4) * NC + (part >> 2)) * NH * 64 + (part & 3) * 16 + (c & 15);
#pragma unroll
                    for (int k = 0; k < NH; k++) d[k * 64] = q[k];
                }
                if (part == 0) {
                    Column to;
                    to.lse = active ? lse[y] : INFINITY;
                    to.qe = qe;
                    col_of[c] = to;
                }
            }
        };
        // ---- K of this wave's block, relative to its largest exponent, as in attention ----
        int top, down;
        V ka[NC][4];
        {
            u4 kr[NC];
            unsigned ks[NC];
            const uint8_t *p = A.k.codes + tile * sp_fp4_tile(HD) + g * 256 + (4 * (r & 3) + (r >> 2)) * 16;
            const uint8_t *e = A.k.exps + tile * sp_fp4_exps(HD) + r * 4;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kr[c] = *reinterpret_cast<const u4 *>(p + c * 1024);
                ks[c] = *reinterpret_cast<const unsigned *>(e + c * 64);
            }
            if constexpr (DIRECT) direct(0, 0);
            else stage(0);
            Largest m;
#pragma unroll
            for (int c = 0; c < NC; c++) m.add(ks[c]);
            top = uniform(sp_fp4::row_max(m.get()));
            down = Op::down(A.c, top);
            unsigned near = 0x80808080u;  // a byte's highest bit: its exponents are at most 23 below
            if constexpr (DT == SP_DTYPE_BF16) {
#pragma unroll
                for (int c = 0; c < NC; c++) near &= (relative(ks[c], top) | 0x80808080u) - (127 - 23) * 0x01010101u;
            }
            if (DT != SP_DTYPE_BF16 || __all(near == 0x80808080u)) {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const unsigned rel = relative(ks[c], top + down);
#pragma unroll
                    for (int n = 0; n < 4; n++) ka[c][n] = Op::codes(kr[c][n], power(rel, n));
                }
            } else {
#pragma unroll
                for (int c = 0; c < NC; c++) {
                    const unsigned rel = relative(ks[c], top);
#pragma unroll
                    for (int n = 0; n < 4; n++) ka[c][n] = Op::seen(kr[c][n], power(rel, n), down);
                }
            }
        }
        f4 acc[4];
#pragma unroll
        for (int n = 0; n < 4; n++) acc[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        // whether every column sees all of this block: nothing then depends on a column's position
        const bool all = t * 64 + 63 <= first && (A.window <= 0 || t * 64 > first + n_new - 1 - A.window);
        const auto units = [&](int qe) {  // of the scores, times log2 e
            const float up = fminf(__builtin_amdgcn_ldexpf(A.c, qe + top + down - 127), 0x1.fffffep127f);
            return A.negate ? -up : up;
        };
        const float cs1 = units(1);
        int buf = 0;
        for (int c0 = 0; c0 < n_cols; c0 += CS) {
            if constexpr (DIRECT) {
                // this stage is there, and all have read the one that the next goes over
                __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
                lds_barrier();
                buf = c0 / CS & 1;
                if (c0 + CS < n_cols) direct(c0 + CS, buf ^ 1);
            } else {
                if (c0) {
                    lds_barrier();  // all have read the stage before
                    stage(c0);
                }
                lds_barrier();
            }
            if (blk < 0) continue;
#pragma unroll 1
            for (int y = w >> two; y < CS / 16 && c0 + y * 16 < n_cols; y += NW >> two) {
                const int n0 = c0 + y * 16;
                bool open = all;
                if (!all) {
                    const int pos0 = first + n0 / A.G, pos1 = first + min(n0 + 15, n_cols - 1) / A.G;
                    if (t * 64 > pos1 || (A.window > 0 && t * 64 + 63 <= pos0 - A.window)) continue;
                    open = t * 64 + 63 <= pos0 && (A.window <= 0 || t * 64 > pos1 - A.window);
                }
                const V *qy = qs + buf * BUF + y * NC * NH * 64 + lane;
                f4 s[4];
#pragma unroll
                for (int n = 0; n < 4; n++) s[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int k = 0; k < NH; k++) {
                        const V q = qy[(c * NH + k) * 64];
#pragma unroll
                        for (int n = 0; n < 4; n++) s[n] = Op::mma(ka[c][n], q, s[n]);
                    }
                float lse, cs = cs1;
                if constexpr (DIRECT) {
                    lse = lse_of[buf * CS + y * 16 + r];
                    lse = n0 + r < n_cols && fabsf(lse) < INFINITY ? lse : INFINITY;
                    // a query that is not finite has no finite score: one of them tells (finite ones have: see Operand)
                    const bool odd = !(fabsf(s[0][0]) < INFINITY);
                    if (__any(odd)) {
                        lse = odd ? INFINITY : lse;
#pragma unroll
                        for (int n = 0; n < 4; n++) s[n] = odd ? f4{0.0f, 0.0f, 0.0f, 0.0f} : s[n];
                    }
                } else {
                    const Column col = col_of[y * 16 + r];
                    lse = col.lse;
                    cs = units(col.qe);
                }
                // In powers of two a weight's exponent is s cs - lse log2 e, both products near lse where weights count, and the
                // difference is rounded once. What the second one's rounding, log2 e's and that of kq_scale log2 e lose of a
                // weight near 1 is a factor of the column's (of a smaller one it is that but for 2^-25 of its exponent).
                // Without it weights near lse 60 are off by up to 2^-18. (Past 2^20 a score has lost more itself.)
                const float of_lse = lse * 1.44269504088896341f, low = __builtin_fmaf(lse, 1.44269504088896341f, -of_lse);
                const float more = __builtin_fmaf(lse, A.lost, -low);
                const float factor = __builtin_amdgcn_exp2f(fabsf(of_lse) < 0x1p20f ? more : 0.0f);
                lse = of_lse;
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) s[n][i] = __builtin_fmaf(s[n][i], cs, -lse);
                if (__builtin_expect(!open, 0)) {
                    const int pos = first + (n0 + r) / A.G, lane0 = t * 64 + 4 * g;
                    const int upto = pos - lane0, before = (A.window > 0 ? pos - A.window : -1) - lane0;
#pragma unroll
                    for (int n = 0; n < 4; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[n][i] = 16 * i + n <= upto && 16 * i + n > before ? s[n][i] : -INFINITY;
                    __asm__ volatile("" ::: "memory");  // (a branch: else the comparisons are made for every block)
                }
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) acc[n][i] = __builtin_fmaf(__builtin_amdgcn_exp2f(s[n][i]), factor, acc[n][i]);
            }
        }
        // ---- over the columns' lanes: lane r of a row keeps value i = r / 4 of row block n = r % 4 ----
        float sum = 0.0f;
#pragma unroll
        for (int n = 0; n < 4; n++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                float v = acc[n][i];
#define SP_ROR(ctrl) __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, 0xf, 0xf, true))
                v += SP_ROR(0x128);
                v += SP_ROR(0x124);
                v += SP_ROR(0x122);
                v += SP_ROR(0x121);
#undef SP_ROR
                if (r == i * 4 + n) sum = v;
            }
        lds_barrier();  // the next item's first stage, or the shares' sums
        if (SHARED) {
            float *sums = reinterpret_cast<float *>(qs);
            sums[tid] = sum;
            lds_barrier();
            for (int k = tid + (64 << two); k < WN; k += 64 << two) sum += sums[k];
            lds_barrier();
            if (w >> two) continue;
        }
        if (blk < 0) continue;
        // position 16 i + 4 g + n. An atomic: two sequences of the call may share the block.
        if (sum != 0.0f) unsafeAtomicAdd(A.weight + tile * 64 + (r >> 2) * 16 + 4 * g + (r & 3), sum);
    }
}

template <int HD>
hipError_t launch_weigh(const SpFp4Weigh &A, int dtype, hipStream_t s) {
    // A block of threads takes eight blocks of a sequence, or fewer and shares the columns out to its waves where
    // eight would leave CUs idle and each share has 16 columns to work on (32 / 8 heads of 128, bf16, 128 rows over 2048 / 8192
    // positions: 11.4 / 22.9 us, with eight 33.1 / 33.0; 32 rows over 2048 8.5 and 11.7; float32, 512 over 2048: 79 and 200).
    // That goes by the blocks that a table row, or a window, has room for: the lengths are on the device. With a table much wider
    // than the sequence the columns are not shared out (128 / 512 rows over 2048 in one of 512 blocks: 43 / 151 us, in one of 32 12 /
    // 29), nor in a batch with one long sequence.
    SpFp4Weigh a = A;
    const long long columns = (long long)A.s.n_rows * A.G / A.s.n_seq, all = ((long long)A.s.n_rows + A.window + 126) / 64;
    const long long seen = A.window > 0 && all < A.s.stride ? all : A.s.stride;  // no sequence has more blocks
    const auto count = [&](int blocks) { return (long long)A.s.n_seq * ((seen + (1 << blocks) - 1) >> blocks); };
    a.blocks = 3;
    while (a.blocks && count(a.blocks) * A.H < A.cus && columns >= 16 << (4 - a.blocks)) a.blocks--;
    // 16-bit rows that cannot go straight into LDS take the shared form always. With eight blocks the other one is ahead in
    // steps (12 sequences of 1 to 4.5K, head_dim 64 / 96 / 128 / 256: 9.5 / 11.2 / 13.8 / 17.9 us for 10.0 / 14.7 / 15.5 / 19.3)
    // and behind with more columns (64 rows over 32768: 22.8 / 28.8 / 42.5 / 63 for 23.5 / 39 / 40.5 / 59.5).
    // The grid is a few blocks of threads for each CU, which take what there is in turn.
    const long long most = count(a.blocks);
    int items = (int)(most < (1ll << 30) ? most : 1ll << 30);
    const int wide = (4 * A.cus + A.H - 1) / A.H;
    const bool direct = dtype != SP_DTYPE_F32 && (uintptr_t)A.q % 16 == 0 && A.q_stride % 8 == 0;
    const auto pick = [&](auto whole, auto shared) { return a.blocks < 3 ? (const void *)shared : (const void *)whole; };
    const void *f = dtype == SP_DTYPE_F32 ? pick(k_fp4_weigh<HD, SP_DTYPE_F32, false, false>, k_fp4_weigh<HD, SP_DTYPE_F32, false, true>)
                  : dtype == SP_DTYPE_F16 ? (direct ? pick(k_fp4_weigh<HD, SP_DTYPE_F16, true, false>, k_fp4_weigh<HD, SP_DTYPE_F16, true, true>)
                                                    : (const void *)k_fp4_weigh<HD, SP_DTYPE_F16, false, true>)
                                          : (direct ? pick(k_fp4_weigh<HD, SP_DTYPE_BF16, true, false>, k_fp4_weigh<HD, SP_DTYPE_BF16, true, true>)
                                                    : (const void *)k_fp4_weigh<HD, SP_DTYPE_BF16, false, true>);
    void *args[] = {&a, &items};
    return hipLaunchKernel(f, dim3((unsigned)(items < wide ? items : wide), (unsigned)A.H), dim3(WN), args, 0, s);
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
// Which positions stay: one block of threads for each (sequence, KV head) finds the last one that stays, by its
// key (the weight's bits, in order) and position. Counts of eleven of the keys' bits, from the top of the range that
// they have, find a bin (attention weights span few of a float's octaves: bits above the range would
// put them into few bins, where lanes that meet take turns: 13 us for 2 with 32768 positions); when it holds
// no more than MOST_FEW of them, these are listed and compared with each other. Then the kept positions are
// written in order: each wave counts its run of the positions, and with the counts of the waves before it
// knows where its own go.
//
// A wave's run is consecutive, and a lane has four neighbours of each 256 positions. K of these fours stay in registers
// from the first pass on (K 0, longer sequences: they are made again for each).
//
// Bound by latencies: with 32768 positions of 8 KV heads 16 us, 6 of them for the weights, whose 1024 lines
// are as many as a CU has in flight in that time, 4 for the counts, 4 to list and compare 80 keys and 3 to write 8192
// positions; with 1064 positions of 12 x 8 5 us, 2 of them for lengths, table and weights. Keys in LDS and counts
// down to the last bit took 20 us of the first and the same of the second.
constexpr int SN = SP_FP4_EVICT_THREADS;

// Order of weights as unsigned numbers: NaN below all, -0 as 0.
constexpr unsigned NO_PLACE = 0, NAN_KEY = 1, NO_KEY = 0xffffffffu;  // NO_KEY: stays whatever its weight
__device__ __forceinline__ unsigned key_of(float w) {
    const unsigned u = __float_as_uint(w + 0.0f);
    return w != w ? NAN_KEY : (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#define SP_MAX(ctrl) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xf, 0xf, true))
    SP_MAX(0x128);  // row_ror 8, 4, 2, 1
    SP_MAX(0x124);
    SP_MAX(0x122);
    SP_MAX(0x121);
#undef SP_MAX
    return max(max((unsigned)__builtin_amdgcn_readlane((int)v, 0), (unsigned)__builtin_amdgcn_readlane((int)v, 16)),
               max((unsigned)__builtin_amdgcn_readlane((int)v, 32), (unsigned)__builtin_amdgcn_readlane((int)v, 48)));
}

template <int K>
__global__ __launch_bounds__(SN) void k_fp4_select(SpFp4Evict A) {
    constexpr int NW = SN / 64, BITS = 11, BINS = 1 << BITS, STEP = K ? K : 4;
    constexpr int MOST_FEW = 256;
    typedef unsigned long long u64;
    __shared__ int bins[BINS];
    __shared__ __align__(16) u64 few[MOST_FEW];
    __shared__ int wave_n[NW], wave_more[NW];
    __shared__ unsigned wave_hi[NW], wave_lo[NW];
    __shared__ int found_bin, found_above, found_here, n_few;
    __shared__ unsigned last_key;
    __shared__ int last_pos;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int h = blockIdx.x % A.H, seq = blockIdx.x / A.H;
    int a, b, n;
    sp_fp8_seq(A.s, seq, a, b, n);
    n = uniform(n);
    int *kept = A.kept + ((long long)seq * A.H + h) * A.keep;
    if (n <= A.keep) {
        for (int j = tid; j < A.keep; j += SN) kept[j] = j < n ? j : -1;
        return;
    }
    if (n > (long long)A.s.stride * 64) {
        for (int j = tid; j < A.keep; j += SN) kept[j] = -1;
        return;
    }
    // wave w has positions [p0, p1), a lane the p0 + 256 i + 4 lane + (0 .. 3)
    const int run = ((n + 4 * SN - 1) / (4 * SN)) * 256, p0 = min(w * run, n), p1 = min(p0 + run, n);
    const int *table = A.s.table + (long long)seq * A.s.stride;
    const int last = ((n + 63) >> 6) - 1, behind = n - A.recent;
    int bad = 0;  // a block that is missing
    uint4 key[STEP];
    // keys from memory: of positions p + 256 i + 4 lane + (0 .. 3)
    const auto make = [&](int p) __attribute__((always_inline)) {
        int blk[STEP];
        float4 weight[STEP];
#pragma unroll
        for (int i = 0; i < STEP; i++) blk[i] = table[min((p + i * 256 + 4 * lane) >> 6, last)];
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            bad |= blk[i] < 0 || blk[i] >= A.s.n_blocks;
            weight[i] = *reinterpret_cast<const float4 *>(
                A.weight + ((long long)min(max(blk[i], 0), A.s.n_blocks - 1) * A.H + h) * 64 + (4 * lane & 63));
        }
#pragma unroll
        for (int i = 0; i < STEP; i++) {
            const int at = p + i * 256 + 4 * lane;
            const auto one = [&](int k, float x) {
                return at + k >= p1 ? NO_PLACE : at + k < A.first || at + k >= behind ? NO_KEY : key_of(x);
            };
            key[i] = uint4{one(0, weight[i].x), one(1, weight[i].y), one(2, weight[i].z), one(3, weight[i].w)};
        }
    };
    // f(p, i): key[i] has the keys of positions p + (0 .. 3)
    const auto each = [&](auto f) __attribute__((always_inline)) {
        for (int p = p0; p < p1; p += 256 * STEP) {
            if (K == 0) make(p);
#pragma unroll
            for (int i = 0; i < STEP; i++)
                if (p + i * 256 < p1) f(p + i * 256 + 4 * lane, i);
        }
    };
    // ---- the keys' range ----
    unsigned hi = 0, lo = 0;  // largest key + 1, the least one's negative
    if (K) make(p0);
    each([&](int, int i) __attribute__((always_inline)) {
        const uint4 k = key[i];
        hi = max(max(hi, max(k.x + 1, k.y + 1)), max(k.z + 1, k.w + 1));
        lo = max(max(lo, max(0 - k.x, 0 - k.y)), max(0 - k.z, 0 - k.w));
    });
    hi = wave_umax(hi);
    lo = wave_umax(lo);
    for (int k = tid; k < BINS; k += SN) bins[k] = 0;
    if (tid < MOST_FEW) few[tid] = 0;
    if (tid == 0) n_few = 0;
    if (lane == 0) {
        wave_hi[w] = hi;
        wave_lo[w] = lo;
        wave_more[w] = 0;
    }
    if (__syncthreads_or(bad)) {
        for (int j = tid; j < A.keep; j += SN) kept[j] = -1;
        return;
    }
    hi = wave_umax(lane < NW ? wave_hi[lane] : 0u);
    lo = wave_umax(lane < NW ? wave_lo[lane] : 0u);
    const unsigned least = 0 - lo;
    // ---- the bin of the last that stays: of the `here` keys in [limit, limit + 2^shift) `want` stay ----
    int want = A.keep - A.first - A.recent, here = n - A.first - A.recent;
    unsigned limit = least;
    int shift = hi > least + 1 ? 32 - __clz(hi - 1 - least) : 0;
    // (it ends before NO_KEY)
    const auto span = [&]() { return shift == 32 ? NO_KEY - limit : min(1u << shift, NO_KEY - limit); };
    for (bool fresh = true; want && shift > 0 && here > want && here > MOST_FEW; fresh = false) {
        const int down = max(shift - BITS, 0);
        if (!fresh) {
            for (int k = tid; k < BINS; k += SN) bins[k] = 0;
            __syncthreads();
        }
        const unsigned size = span();
        const auto count = [&](unsigned k) __attribute__((always_inline)) {
            if (k - limit < size) atomicAdd(&bins[(k - limit) >> down], 1);
        };
        each([&](int, int i) __attribute__((always_inline)) {
            count(key[i].x);
            count(key[i].y);
            count(key[i].z);
            count(key[i].w);
        });
        __syncthreads();
        // sums from the top: thread 0 has the two highest bins
        const int top = BINS - 1 - 2 * tid, c1 = bins[top], c0 = bins[top - 1];
        const int sum = sp_fp8_scan(c0 + c1, lane);
        if (lane == 63) wave_n[w] = sum;
        __syncthreads();
        int before = sum - c0 - c1;
        for (int k = 0; k < w; k++) before += wave_n[k];
        if (before < want && before + c0 + c1 >= want) {
            const bool second = before + c1 < want;
            found_bin = second ? top - 1 : top;
            found_above = second ? before + c1 : before;
            found_here = second ? c0 : c1;
        }
        __syncthreads();
        limit += (unsigned)found_bin << down;
        want -= found_above;
        here = found_here;
        shift = down;
    }
    // ---- the last that stays: a position stays if its key is larger, or the same and it is no later ----
    unsigned end = want ? limit : NO_KEY;
    int end_pos = 0x7fffffff;
    const bool compare = want && here > want && here <= MOST_FEW;
    const auto stays = [&](unsigned k, int p) { return k > end - (p <= end_pos); };
    int n_stay = 0;  // of this lane, then of the wave
    if (compare) {
        const unsigned size = span();
        each([&](int p, int i) __attribute__((always_inline)) {
            const unsigned k[4] = {key[i].x, key[i].y, key[i].z, key[i].w};
#pragma unroll
            for (int x = 0; x < 4; x++)
                if (k[x] - limit < size) {
                    const int at = atomicAdd(&n_few, 1);  // (`here` of them, unless weights change meanwhile)
                    if (at < MOST_FEW) few[at] = (u64)k[x] << 32 | (unsigned)~(p + x);
                } else {
                    n_stay += k[x] >= limit;
                }
        });
        __syncthreads();
        if (tid < here) {
            const u64 mine = few[tid];
            int above = 0;
            for (int k = 0; k < here; k += 4)  // (behind them are zeros)
#pragma unroll
                for (int x = 0; x < 4; x++) above += few[k + x] > mine;
            const int p = ~(unsigned)mine;
            if (above < want) atomicAdd(&wave_more[p / run], 1);
            if (above == want - 1) {
                last_key = (unsigned)(mine >> 32);
                last_pos = p;
            }
        }
    } else {
        if (want && here > want) {  // all the same: the first `want` of them
            int ties = 0;
            each([&](int, int i) __attribute__((always_inline)) {
                ties += (key[i].x == end) + (key[i].y == end) + (key[i].z == end) + (key[i].w == end);
            });
            ties = sp_fp8_scan(ties, lane);
            if (lane == 63) wave_n[w] = ties;
            __syncthreads();
            int met = 0;
            for (int k = 0; k < w; k++) met += wave_n[k];
            if (met < want && met + wave_n[w] >= want)
                each([&](int p, int i) __attribute__((always_inline)) {
                    const unsigned k[4] = {key[i].x, key[i].y, key[i].z, key[i].w};
                    const int mine = (k[0] == end) + (k[1] == end) + (k[2] == end) + (k[3] == end), sum = sp_fp8_scan(mine, lane);
                    int t = met + sum - mine;
#pragma unroll
                    for (int x = 0; x < 4; x++)
                        if (k[x] == end && ++t == want) last_pos = p + x;
                    met += __builtin_amdgcn_readlane(sum, 63);
                });
            __syncthreads();
            end_pos = last_pos;
        }
        each([&](int p, int i) __attribute__((always_inline)) {
            n_stay += stays(key[i].x, p) + stays(key[i].y, p + 1) + stays(key[i].z, p + 2) + stays(key[i].w, p + 3);
        });
    }
    n_stay = sp_fp8_scan(n_stay, lane);
    if (lane == 63) wave_n[w] = n_stay;
    __syncthreads();
    if (compare) {
        end = last_key;
        end_pos = last_pos;
    }
    int at = 0;  // kept before this wave's run
    for (int k = 0; k < w; k++) at += wave_n[k] + wave_more[k];
    each([&](int p, int i) __attribute__((always_inline)) {
        const bool stay[4] = {stays(key[i].x, p), stays(key[i].y, p + 1), stays(key[i].z, p + 2), stays(key[i].w, p + 3)};
        const int mine = stay[0] + stay[1] + stay[2] + stay[3], sum = sp_fp8_scan(mine, lane);
        int j = at + sum - mine;
#pragma unroll
        for (int x = 0; x < 4; x++) {
            if (stay[x] && j < A.keep) kept[j] = p + x;
            j += stay[x];
        }
        at += __builtin_amdgcn_readlane(sum, 63);
    });
}

// Rows to their new places: a block of threads for each (sequence, KV head, side) and PLANES planes of
// eight channels goes up the places. A row never moves up, so a place's row lies at or behind it:
// a round that has loaded its rows may store them, whatever the rounds before and behind do. A
// round is so large (NT places, ROUND of a thread) that most calls take one. It is a chain of three loads (position,
// block, row): each round's are in flight together, and the first's with the sequence's length.
template <int NT, int PLANES, int ROUND>
__global__ __launch_bounds__(NT) void k_fp4_move(SpFp4Evict A) {
    constexpr int PLACES = NT * ROUND;
    const int tid = threadIdx.x;
    const int h = blockIdx.x % A.H, seq = blockIdx.x / A.H, is_v = blockIdx.y & 1, n0 = (blockIdx.y >> 1) * PLANES;
    const int *kept = A.kept + ((long long)seq * A.H + h) * A.keep;
    const int *table = A.s.table + (long long)seq * A.s.stride;
    int p[ROUND], dst[ROUND];  // positions, blocks of the places
    const auto fetch = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < ROUND; k++) {
            const int j = min(j0 + k * NT + tid, A.keep - 1);
            p[k] = kept[j];
            dst[k] = table[min(j >> 6, A.s.stride - 1)];
        }
    };
    // the first round's are on their way together with what tells whether there is one
    fetch(0);
    int a, b, n;
    sp_fp8_seq(A.s, seq, a, b, n);
    const int head = kept[0];
#pragma unroll
    for (int k = 0; k < ROUND; k++) __asm__ volatile("" : "+v"(p[k]), "+v"(dst[k]));
    if (n <= A.keep || head < 0) return;  // head: a block is missing
    const SpFp8Side side = A.side[is_v];
    const int tile = A.NC * 256, exps = A.NC * 64;  // dwords of codes, bytes of exponents
    const bool with_exp = n0 % 4 == 0, with_weight = is_v == 0 && n0 == 0;
    unsigned *codes = reinterpret_cast<unsigned *>(side.codes) + n0 * 64;
    uint8_t *exp_plane = side.exps + n0 / 4 * 64;
    for (int j0 = 0; j0 < A.keep; j0 += PLACES) {
        int src[ROUND];  // blocks of the positions
        if (j0) fetch(j0);
#pragma unroll
        for (int k = 0; k < ROUND; k++) {
            const int j = j0 + k * NT + tid;
            p[k] = j < A.keep ? max(min(p[k], n - 1), j) : j;  // (where they are, whatever kept holds)
            src[k] = table[min(p[k], n - 1) >> 6];
        }
        unsigned code[ROUND][PLANES];
        uint8_t e[ROUND];
        float weight[ROUND];
#pragma unroll
        for (int k = 0; k < ROUND; k++) {
            const int j = j0 + k * NT + tid;
            if (p[k] == j) continue;
            const long long from = (long long)src[k] * A.H + h;  // tile
#pragma unroll
            for (int x = 0; x < PLANES; x++) code[k][x] = codes[from * tile + x * 64 + (p[k] & 63)];
            if (with_exp) e[k] = exp_plane[from * exps + sp_fp4_place(p[k] & 63)];
            if (with_weight) weight[k] = A.weight[from * 64 + (p[k] & 63)];
        }
        // what the loop has loaded is in registers before any of it is stored over
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int k = 0; k < ROUND; k++) {
            const int j = j0 + k * NT + tid;
            if (p[k] == j) continue;
            const long long to = (long long)dst[k] * A.H + h;
#pragma unroll
            for (int x = 0; x < PLANES; x++) codes[to * tile + x * 64 + (j & 63)] = code[k][x];
            if (with_exp) exp_plane[to * exps + sp_fp4_place(j & 63)] = e[k];
            if (with_weight) A.weight[to * 64 + (j & 63)] = weight[k];
        }
    }
    // behind the last place nothing counts in its block's largest exponent
    const int tail = A.keep & 63;
    if (tail == 0 || !with_exp) return;
    const int t = tail + tid;
    if (t < 64) exp_plane[((long long)table[A.keep >> 6] * A.H + h) * exps + sp_fp4_place(t)] = SP_FP4_LEAST;
}

template <int NT, int PLANES, int ROUND>
hipError_t launch_move(const SpFp4Evict &A, hipStream_t s) {
    void *args[] = {const_cast<SpFp4Evict *>(&A)};
    return hipLaunchKernel((const void *)k_fp4_move<NT, PLANES, ROUND>, dim3((unsigned)(A.H * A.s.n_seq), (unsigned)(2 * A.NC * 4 / PLANES)),
                           dim3(NT), args, 0, s);
}

}  // namespace

hipError_t sp_fp4_launch_weigh(const SpFp4Weigh &A, int hd, int dtype, hipStream_t s) {
    switch (hd) {
        case 64: return launch_weigh<64>(A, dtype, s);
        case 96: return launch_weigh<96>(A, dtype, s);
        case 128: return launch_weigh<128>(A, dtype, s);
        case 256: return launch_weigh<256>(A, dtype, s);
    }
    return hipErrorInvalidValue;
}

hipError_t sp_fp4_launch_evict(const SpFp4Evict &A, hipStream_t s) {
    void *args[] = {const_cast<SpFp4Evict *>(&A)};
    // No sequence is longer than its table row, and shorter ones in a wide one take the form of the longest: of 12 x 1064
    // positions both kernels take 16.6 us with 17 blocks to a row, 19.3 with 512 or more; of 32768 36 and (2048 blocks) 45.
    const long long most = (long long)A.s.stride * 64;
    const void *select = most <= 2 * 4 * SN ? (const void *)k_fp4_select<2>
                       : most <= 8 * 4 * SN ? (const void *)k_fp4_select<8> : (const void *)k_fp4_select<0>;
    const hipError_t e = hipLaunchKernel(select, dim3((unsigned)(A.H * A.s.n_seq)), dim3(SN), args, 0, s);
    if (e != hipSuccess) return e;
    // Many sequences and KV heads: blocks of 256 threads with four planes and 1024 places a round. Few, with more
    // places: blocks of 1024 threads with one plane and 8192 places. (1000 places of 12 x 8: 6.4 us, the other way 27.8;
    // 8192 of 1 x 8: 24.6, the other way 9.8.)
    const long long groups = (long long)A.H * A.s.n_seq * 2 * A.NC;
    return groups < 256 && A.keep > 1024 ? launch_move<1024, 1, 8>(A, s) : launch_move<256, 4, 4>(A, s);
}

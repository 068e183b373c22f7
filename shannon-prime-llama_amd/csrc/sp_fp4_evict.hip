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

__device__ __forceinline__ float power(unsigned rel, int b) {
    return __int_as_float((b == 3 ? rel >> 1 : rel << (23 - 8 * b)) & 0x7f800000);
}

// ---------------------------------------------------------------------------
// weigh
// ---------------------------------------------------------------------------
// A wave holds one block's K as operands, converted once, and eight waves of a block of threads take
// eight consecutive blocks of a sequence. Columns (row, query head) pass by in stages: the block of
// threads brings them into LDS as operands, and each wave takes them 16 at a time. The weights are
// summed over columns in the registers that the scores come in, and over the 16 lanes at the end.
constexpr int WN = 512;  // threads

template <int HD, int DT>
__global__ __launch_bounds__(WN) void k_fp4_weigh(SpFp4Weigh A, int items) {
    constexpr int NC = HD / 32, NW = WN / 64;
    constexpr int LP = HD == 64 ? 8 : HD == 256 ? 32 : 16;  // threads of a column (96: twelve of them have a part)
    constexpr int CS = WN / LP, CG = CS / 16;               // columns of a stage, groups of 16
    constexpr bool SPLIT2 = DT == SP_DTYPE_F32;
    constexpr int NH = SPLIT2 ? 2 : 1;
    typedef typename SpFp8Elem<DT>::T T;
    struct Column {
        float lse;  // +inf: adds nothing
        int qe;     // scores count in 2^(qe + the block's exponent) * A.c
        int pos, from;
    };
    __shared__ __align__(16) h8 qs[2][CG * NC * NH * 64];
    __shared__ Column col_of[2][CS];
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int h = blockIdx.y, r = lane & 15, g = lane >> 4;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        // ---- the sequence, and eight blocks of those that its rows see ----
        int seq = -1, r0 = 0, n_new = 0, first = 0, j0 = 0, left = item;
        for (int i0 = 0; i0 < A.s.n_seq && seq < 0; i0 += 64) {
            int a = 0, b = 0, len = 0, lo = 0, n = 0;
            if (i0 + lane < A.s.n_seq) {
                sp_fp8_seq(A.s, i0 + lane, a, b, len);
                lo = A.window > 0 ? max(len - (b - a) - A.window + 1, 0) >> 6 : 0;
                if (b > a) n = (max(min((len + 63) >> 6, A.s.stride) - lo, 0) + NW - 1) / NW;
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
                j0 = of(lo) + (left - (of(sum) - of(n))) * NW;
            } else {
                left -= __builtin_amdgcn_readlane(sum, 63);
            }
        }
        if (seq < 0) return;
        const int t = j0 + w, n_cols = n_new * A.G;
        const int blk = uniform(t <= (first + n_new - 1) >> 6 ? sp_fp8_block(A.s, seq, t) : -1);
        const long long tile = (long long)max(blk, 0) * A.H + h;
        // ---- K of this wave's block ----
        u4 kr[NC];
        unsigned ks[NC];
        {
            const uint8_t *p = A.k.codes + tile * sp_fp4_tile(HD) + g * 256 + (4 * (r & 3) + (r >> 2)) * 16;
            const uint8_t *e = A.k.exps + tile * sp_fp4_exps(HD) + r * 4;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kr[c] = *reinterpret_cast<const u4 *>(p + c * 1024);
                ks[c] = *reinterpret_cast<const unsigned *>(e + c * 64);
            }
        }
        // ---- columns: this thread's eight entries of one ----
        const int mine = tid / LP, part = tid % LP;
        float x[8];
        const auto load = [&](int c0) __attribute__((always_inline)) {
            const int n = c0 + mine;
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = 0.0f;
            if (n < n_cols && part < HD / 8) {
                const bool aligned = (uintptr_t)A.q % (4 * sizeof(T)) == 0 && A.q_stride % 4 == 0;
                load8<DT>(reinterpret_cast<const T *>(A.q) + (long long)(r0 + n / A.G) * A.q_stride +
                              (long long)(h * A.G + n % A.G) * HD + part * 8, aligned, x);
            }
        };
        const auto put = [&](int c0, int to) __attribute__((always_inline)) {
            const int n = c0 + mine, tk = n / A.G;
            float top = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) top = x[k] != x[k] ? INFINITY : fmaxf(top, fabsf(x[k]));
#pragma unroll
            for (int s = LP / 2; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
            float lse = INFINITY;
            if (n < n_cols) lse = A.lse[(long long)(r0 + tk) * A.H * A.G + h * A.G + n % A.G];
            // rows that see nothing, and those whose scores are no numbers
            const bool active = n < n_cols && fabsf(lse) < INFINITY && top < INFINITY;
            int e = (__float_as_int(top) >> 23) - 127 - 14;
            e = top == 0.0f || !active ? 0 : max(e, -126);
            const float down = A.negate ? -sp_fp8_pow2(-e) : sp_fp8_pow2(-e);
            h8 q[NH];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float v = active ? x[k] * down : 0.0f;
                const _Float16 hi = (_Float16)v;
                q[0][k] = hi;
                if (SPLIT2) q[NH - 1][k] = (_Float16)(v - (float)hi);
            }
            if (part < HD / 8) {
                h8 *d = qs[to] + ((mine >> 4) * NC + (part >> 2)) * NH * 64 + (part & 3) * 16 + (mine & 15);
#pragma unroll
                for (int k = 0; k < NH; k++) d[k * 64] = q[k];
            }
            if (part == 0) {
                Column c;
                c.lse = active ? lse : INFINITY;
                c.qe = e + 1;
                c.pos = active ? first + tk : -1;
                c.from = A.window > 0 ? c.pos - A.window : -1;
                col_of[to][mine] = c;
            }
        };
        load(0);
        // relative to the block's largest exponent, as in attention
        Largest m;
#pragma unroll
        for (int c = 0; c < NC; c++) m.add(ks[c]);
        const int top = uniform(sp_fp4::row_max(m.get()));
#pragma unroll
        for (int c = 0; c < NC; c++) ks[c] = relative(ks[c], top);
        h8 ka[NC][4];
#pragma unroll
        for (int c = 0; c < NC; c++)
#pragma unroll
            for (int n = 0; n < 4; n++) ka[c][n] = eight(kr[c][n], power(ks[c], n));
        f4 acc[4];
#pragma unroll
        for (int n = 0; n < 4; n++) acc[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        int at = 0;
        for (int c0 = 0; c0 < n_cols; c0 += CS, at ^= 1) {
            put(c0, at);
            lds_barrier();  // (two places: a stage is written after all have read the one before the last)
            if (c0 + CS < n_cols) load(c0 + CS);
            if (blk < 0) continue;
            for (int y = 0; y < CG && c0 + y * 16 < n_cols; y++) {
                const int n0 = c0 + y * 16, n1 = min(n0 + 15, n_cols - 1);
                const int pos0 = first + n0 / A.G, pos1 = first + n1 / A.G;
                if (t * 64 > pos1 || (A.window > 0 && t * 64 + 63 <= pos0 - A.window)) continue;
                const Column col = col_of[at][y * 16 + r];
                const h8 *qy = qs[at] + y * NC * NH * 64 + lane;
                f4 s[4];
#pragma unroll
                for (int n = 0; n < 4; n++) s[n] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < NC; c++)
#pragma unroll
                    for (int k = 0; k < NH; k++) {
                        const h8 q = qy[(c * NH + k) * 64];
#pragma unroll
                        for (int n = 0; n < 4; n++) s[n] = mma(ka[c][n], q, s[n]);
                    }
                const float cs = fminf(__builtin_amdgcn_ldexpf(A.c, col.qe + top - 127), 0x1.fffffep127f);
                const bool open = t * 64 + 63 <= pos0 && (A.window <= 0 || t * 64 > pos1 - A.window);
                const int lane0 = t * 64 + 4 * g, upto = col.pos - lane0, before = col.from - lane0;
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        // the score less lse, rounded once
                        float d = __builtin_fmaf(s[n][i], cs, -col.lse);
                        if (!open) d = 16 * i + n <= upto && 16 * i + n > before ? d : -INFINITY;
                        acc[n][i] += __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
                    }
            }
        }
        lds_barrier();  // the next item's first stage
        if (blk < 0) continue;
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
        // position 16 i + 4 g + n. An atomic: two sequences of the call may share the block.
        if (sum != 0.0f) unsafeAtomicAdd(A.weight + tile * 64 + (r >> 2) * 16 + 4 * g + (r & 3), sum);
    }
}

template <int HD>
hipError_t launch_weigh(const SpFp4Weigh &A, int dtype, hipStream_t s) {
    // Eights of blocks: no sequence has more than its table row. The grid is a few blocks of threads
    // for each CU, which take what there is in turn.
    const long long most = (long long)A.s.n_seq * ((A.s.stride + 7) / 8);
    int items = (int)(most < (1ll << 30) ? most : 1ll << 30);
    const int wide = (4 * A.cus + A.H - 1) / A.H;
    const void *f = dtype == SP_DTYPE_F32 ? (const void *)k_fp4_weigh<HD, SP_DTYPE_F32>
                  : dtype == SP_DTYPE_F16 ? (const void *)k_fp4_weigh<HD, SP_DTYPE_F16>
                                          : (const void *)k_fp4_weigh<HD, SP_DTYPE_BF16>;
    void *args[] = {const_cast<SpFp4Weigh *>(&A), &items};
    return hipLaunchKernel(f, dim3((unsigned)(items < wide ? items : wide), (unsigned)A.H), dim3(WN), args, 0, s);
}

// ---------------------------------------------------------------------------
// evict
// ---------------------------------------------------------------------------
// Which positions stay: one block of threads for each (sequence, KV head) finds the weight of the last
// one that stays by three counts of its bits from the top (11, 11 and 10), then writes the kept
// positions in order: each wave counts its run of the positions, and with the counts of the
// waves before it knows where its own go.
constexpr int SN = SP_FP4_EVICT_THREADS;

// Order of weights as unsigned numbers: NaN below all, -0 as 0.
__device__ __forceinline__ unsigned key_of(float w) {
    const unsigned u = __float_as_uint(w + 0.0f);
    return w != w ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}

__global__ __launch_bounds__(SN) void k_fp4_select(SpFp4Evict A) {
    constexpr int NW = SN / 64, BINS = 2048;
    __shared__ int bins[BINS];
    __shared__ int wave_n[NW], wave_t[NW];
    __shared__ int found_bin, found_above;
    const int tid = threadIdx.x, lane = tid & 63, w = uniform(tid >> 6);
    const int h = blockIdx.x % A.H, seq = blockIdx.x / A.H;
    int a, b, n;
    sp_fp8_seq(A.s, seq, a, b, n);
    int *kept = A.kept + ((long long)seq * A.H + h) * A.keep;
    if (n <= A.keep) {
        for (int j = tid; j < A.keep; j += SN) kept[j] = j < n ? j : -1;
        return;
    }
    int bad = 0;
    for (int j = tid; j < (n + 63) >> 6; j += SN) bad |= sp_fp8_block(A.s, seq, j) < 0;
    if (__syncthreads_or(bad)) {
        for (int j = tid; j < A.keep; j += SN) kept[j] = -1;
        return;
    }
    const int lo = A.first, hi = n - A.recent;  // of these `need` stay
    const int need = A.keep - A.first - A.recent;
    const int *table = A.s.table + (long long)seq * A.s.stride;
    const auto key_at = [&](int p) { return key_of(A.weight[((long long)table[p >> 6] * A.H + h) * 64 + (p & 63)]); };
    // keys of `limit` and more stay, of those that equal it `ties` if exact
    unsigned limit = 0xffffffffu;
    int ties = 0;
    bool exact = true;
    if (need > 0) {
        int want = need;  // of the keys that agree with `limit` in the bits above `shift`
        unsigned prefix = 0;
        int shift = 32;
        for (int pass = 0; pass < 3; pass++) {
            const int bits = pass < 2 ? 11 : 10, down = shift - bits;
            for (int k = tid; k < BINS; k += SN) bins[k] = 0;
            __syncthreads();
            for (int p = lo + tid; p < hi; p += SN) {
                const unsigned key = key_at(p);
                if (pass == 0 || key >> shift == prefix) atomicAdd(&bins[(key >> down) & ((1 << bits) - 1)], 1);
            }
            __syncthreads();
            // sums from the top: thread 0 has the two highest bins
            const int top = (1 << bits) - 1 - 2 * tid;
            const int c1 = top >= 0 ? bins[top] : 0, c0 = top >= 1 ? bins[top - 1] : 0;
            const int sum = sp_fp8_scan(c0 + c1, lane);
            if (lane == 63) wave_n[w] = sum;
            __syncthreads();
            int before = sum - c0 - c1;
            for (int k = 0; k < w; k++) before += wave_n[k];
            if (before < want && before + c0 + c1 >= want) {
                const bool second = before + c1 < want;
                found_bin = second ? top - 1 : top;
                found_above = second ? before + c1 : before;
            }
            __syncthreads();
            prefix = prefix << bits | (unsigned)found_bin;
            want -= found_above;
            shift = down;
            const int here = bins[found_bin];
            __syncthreads();
            if (here == want) {  // all of them stay
                exact = false;
                break;
            }
        }
        limit = prefix << shift;
        ties = exact ? want : 0;
    }
    // ---- in order: wave w has positions [w * run, (w + 1) * run) ----
    const int run = ((n + SN - 1) / SN) * 64, p0 = w * run, p1 = min(p0 + run, n);
    // 2: stays, 1: equals the limit, 0: goes
    const auto verdict = [&](int p) {
        if (p < lo || p >= hi) return 2;
        if (need == 0) return 0;
        const unsigned key = key_at(p);
        return key > limit || (!exact && key == limit) ? 2 : key == limit ? 1 : 0;
    };
    int n_stay = 0, n_tie = 0;
    for (int p = p0; p < p1; p += 64) {
        const int v = p + lane < p1 ? verdict(p + lane) : 0;
        n_stay += __popcll(__ballot(v == 2));
        n_tie += __popcll(__ballot(v == 1));
    }
    __syncthreads();
    if (lane == 0) {
        wave_n[w] = n_stay;
        wave_t[w] = n_tie;
    }
    __syncthreads();
    int at = 0, tied = 0;  // kept before this wave's run, and ties met
    for (int k = 0; k < w; k++) {
        at += wave_n[k] + max(min(wave_t[k], ties - tied), 0);
        tied += wave_t[k];
    }
    const unsigned long long below = (1ull << lane) - 1;
    for (int p = p0; p < p1; p += 64) {
        const int v = p + lane < p1 ? verdict(p + lane) : 0;
        const unsigned long long t = __ballot(v == 1);
        const bool stays = v == 2 || (v == 1 && tied + __popcll(t & below) < ties);
        const unsigned long long s = __ballot(stays);
        const int j = at + __popcll(s & below);
        if (stays && j < A.keep) kept[j] = p + lane;
        at += __popcll(s);
        tied += __popcll(t);
    }
}

// Rows to their new places: one block of threads for each (sequence, KV head, side, 32 channels) goes up
// the places. A row never moves up, so a place's row lies at or behind it: a round that
// has loaded its rows may store them, whatever the rounds before and behind do.
constexpr int MN = SP_FP4_EVICT_THREADS;
constexpr int MOVES = 8;  // dwords of a thread a round: 2048 places

__global__ __launch_bounds__(MN) void k_fp4_move(SpFp4Evict A) {
    constexpr int ROUND = MN / 4 * MOVES;
    const int tid = threadIdx.x, plane = tid >> 8, lane = tid & 255;
    const int h = blockIdx.x % A.H, seq = blockIdx.x / A.H, is_v = blockIdx.y & 1, G = blockIdx.y >> 1;
    int a, b, n;
    sp_fp8_seq(A.s, seq, a, b, n);
    if (n <= A.keep) return;
    const int *kept = A.kept + ((long long)seq * A.H + h) * A.keep;
    if (kept[0] < 0) return;  // a block is missing
    const SpFp8Side side = A.side[is_v];
    const int *table = A.s.table + (long long)seq * A.s.stride;
    const int tile = A.NC * 1024, exps = A.NC * 64;
    const bool with_exp = plane == 0, with_weight = plane == 1 && is_v == 0 && G == 0;
    for (int j0 = 0; j0 < A.keep; j0 += ROUND) {
        unsigned code[MOVES];
        int exp[MOVES];
        float weight[MOVES];
        bool moves[MOVES];
#pragma unroll
        for (int k = 0; k < MOVES; k++) {
            const int j = j0 + k * (MN / 4) + lane;
            const int p = j < A.keep ? kept[j] : j;
            moves[k] = p != j;
            if (!moves[k]) continue;
            const long long at = (long long)table[p >> 6] * A.H + h;
            code[k] = reinterpret_cast<const unsigned *>(side.codes + at * tile)[(G * 4 + plane) * 64 + (p & 63)];
            if (with_exp) exp[k] = side.exps[at * exps + G * 64 + sp_fp4_place(p & 63)];
            if (with_weight) weight[k] = A.weight[at * 64 + (p & 63)];
        }
        // what this round loads is in registers before any of it is stored over
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int k = 0; k < MOVES; k++) {
            if (!moves[k]) continue;
            const int j = j0 + k * (MN / 4) + lane;
            const long long at = (long long)table[j >> 6] * A.H + h;
            reinterpret_cast<unsigned *>(side.codes + at * tile)[(G * 4 + plane) * 64 + (j & 63)] = code[k];
            if (with_exp) side.exps[at * exps + G * 64 + sp_fp4_place(j & 63)] = (uint8_t)exp[k];
            if (with_weight) A.weight[at * 64 + (j & 63)] = weight[k];
        }
    }
    // behind the last place nothing counts in its block's largest exponent
    const int tail = A.keep & 63;
    if (tail == 0) return;
    const int t = tail + tid;
    if (t < 64) side.exps[((long long)table[A.keep >> 6] * A.H + h) * exps + G * 64 + sp_fp4_place(t)] = SP_FP4_LEAST;
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
    const hipError_t e = hipLaunchKernel((const void *)k_fp4_select, dim3((unsigned)(A.H * A.s.n_seq)), dim3(SN), args, 0, s);
    if (e != hipSuccess) return e;
    return hipLaunchKernel((const void *)k_fp4_move, dim3((unsigned)(A.H * A.s.n_seq), (unsigned)(2 * A.NC)), dim3(MN), args, 0, s);
}

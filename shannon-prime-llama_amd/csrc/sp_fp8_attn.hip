// sp_fp8_attn.hip -- attention over the 8-bit block cache (sp_block_attn.h): its codes as operands, and
// which kernel a call takes.
#include "sp_block_attn.h"

namespace {

using namespace sp_block;

// Eight codes (two dwords) as fp16.
__device__ __forceinline__ h8 to_half(unsigned a, unsigned b) {
    const h2 x = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, false);
    const h2 y = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(a, 1.0f, true);
    const h2 z = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, false);
    const h2 w = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(b, 1.0f, true);
    return h8{x[0], x[1], y[0], y[1], z[0], z[1], w[0], w[1]};
}

struct Fp8 {
    // A block in a wave's registers, in the order it is held in.
    template <int HD>
    struct Few {
        static constexpr int NC = HD / 32, ND = HD / 16, TILE = 64 * HD, AT_ONCE = 1;
        u4 kr[2 * NC], vr[ND];
        int ekb, evb;  // lane k: scale bytes of the k-th block
        __device__ __forceinline__ void look_up(const SpFp8Attn &A, long long at) {
            ekb = A.k.exps[at];
            evb = A.v.exps[at];
        }
        __device__ __forceinline__ void load_k(const SpFp8Side &S, long long tile, int lane) {
            const uint8_t *p = S.codes + tile * TILE + lane * 16;
#pragma unroll
            for (int n = 0; n < 2 * NC; n++) kr[n] = *reinterpret_cast<const u4 *>(p + n * 1024);
        }
        __device__ __forceinline__ void load_v(const SpFp8Side &S, long long tile, int lane) {
            const uint8_t *p = S.codes + tile * TILE + lane * 16;
#pragma unroll
            for (int n = 0; n < ND; n++) vr[n] = *reinterpret_cast<const u4 *>(p + n * 1024);
        }
        __device__ __forceinline__ int k_exponent(int k) { return sp_fp8_exponent(__builtin_amdgcn_readlane(ekb, k)); }
        __device__ __forceinline__ int v_exponent(int k) { return sp_fp8_exponent(__builtin_amdgcn_readlane(evb, k)); }
        // row blocks 2 u and 2 u + 1 of step c
        __device__ __forceinline__ void k_rows(int c, int u, h8 &a, h8 &b) const {
            const u4 r = kr[u * NC + c];
            a = to_half(r[0], r[1]);
            b = to_half(r[2], r[3]);
        }
        __device__ __forceinline__ void v_rows(int d, h8 (&a)[AT_ONCE][2]) const {
            a[0][0] = to_half(vr[d][0], vr[d][1]);
            a[0][1] = to_half(vr[d][2], vr[d][3]);
        }
        // position of value i of row block n, from the lane's first; its step and place among V's operands
        static constexpr __device__ __forceinline__ int at(int n, int i) { return n * 16 + i; }
        static constexpr __device__ __forceinline__ int step(int n, int) { return n / 2; }
        static constexpr __device__ __forceinline__ int place(int n, int i) { return n % 2 * 4 + i; }
        static __device__ __forceinline__ void put(float *rec, const f4 (&o)[ND], int g, float unit) {
#pragma unroll
            for (int d = 0; d < ND; d++) *reinterpret_cast<f4 *>(rec + d * 16 + g * 4) = o[d] * unit;
        }
    };

    // A block on its way into LDS: half of the threads bring K, half V.
    // K's piece (uc, g, r), uc = u * HD/32 + c. V's pieces in pairs: CW 32 takes g and g + 2 of a
    // channel, which its operand has side by side; CW 16 two channel groups.
    template <int HD, int NT, int CW>
    struct Wide {
        static constexpr int TILE = 64 * HD, HT = NT / 2;
        static constexpr int NS = CW == 32 ? HD / 16 : HD / 32, NP = CW == 32 ? 4 : 2;
        static constexpr int KP = (HD * 4 + HT - 1) / HT;  // K pieces of 16 codes a thread (half the threads)
        static constexpr int VP = (HD * 2 + HT - 1) / HT;  // pairs of V pieces (the other half)
        // fp16 eights: of a block's place in LDS, of a row block of it, of a step of V
        static constexpr int K_PLACE = TILE / 8, V_PLACE = TILE / 8, K_ROW = NS * 64, V_ROW = NP * 64, V_STEP = 64;
        static constexpr int LDS = HD * 512, BYTES = LDS;
        struct Raw {
            u4 x[KP > 2 * VP ? KP : 2 * VP];
        };
        static constexpr __device__ __forceinline__ int at(int lane) { return lane; }
        static constexpr __device__ __forceinline__ int v_at(int lane) { return lane; }
        static __device__ __forceinline__ void look_up(const SpFp8Attn &A, int h, int blk, int, int, int *, int &ekb, int &evb) {
            const long long at = (long long)max(blk, 0) * A.H + h;
            ekb = A.k.exps[at];
            evb = A.v.exps[at];
        }
        static __device__ __forceinline__ void fetch_k(const SpFp8Side &S, long long tile, int st, Raw &raw) {
            const uint8_t *p = S.codes + tile * TILE;
#pragma unroll
            for (int i = 0; i < KP; i++)
                if (KP * HT == HD * 4 || st + i * HT < HD * 4) raw.x[i] = *reinterpret_cast<const u4 *>(p + (st + i * HT) * 16);
        }
        static __device__ __forceinline__ void fetch_v(const SpFp8Side &S, long long tile, int st, Raw &raw) {
            const uint8_t *p = S.codes + tile * TILE;
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const int x = st + i * HT;
                if (VP * HT == HD * 2 || x < HD * 2) {
                    // CW 32: x = (dg / 2, g % 2, dg % 2, r); CW 16: x = (dg / 2, g, r)
                    const uint8_t *s = CW == 32 ? p + ((x >> 6) * 2 + ((x >> 4) & 1)) * 1024 + ((x >> 5) & 1) * 256 + (x & 15) * 16
                                                : p + (x >> 6) * 2048 + (x & 63) * 16;
                    raw.x[2 * i] = *reinterpret_cast<const u4 *>(s);
                    raw.x[2 * i + 1] = *reinterpret_cast<const u4 *>(s + (CW == 32 ? 512 : 1024));
                }
            }
        }
        static __device__ __forceinline__ void stage_k(Raw &raw, int st, int, h8 *to) {
#pragma unroll
            for (int i = 0; i < KP; i++) {
                const int x = st + i * HT, g = (x >> 4) & 3, r = x & 15, uc = x >> 6;
                if (KP * HT == HD * 4 || x < HD * 4) {
                    // row block and step of the operand, lane in it: CW 32 holds positions r and 16 + r of a
                    // 32 in one row block, CW 16 in two
                    h8 *d = to + (CW == 32 ? (uc * 2 + (g >> 1)) * 64 + (g & 1) * 32 + r
                                           : ((uc / (HD / 32)) * 2 * NS + uc % (HD / 32)) * 64 + (x & 63));
                    d[0] = to_half(raw.x[i][0], raw.x[i][1]);
                    d[CW == 32 ? 16 : NS * 64] = to_half(raw.x[i][2], raw.x[i][3]);
                }
            }
        }
        static __device__ __forceinline__ void stage_v(Raw &raw, int st, int, h8 *to) {
#pragma unroll
            for (int i = 0; i < VP; i++) {
                const int x = st + i * HT;
                if (VP * HT == HD * 2 || x < HD * 2) {
                    // (opaque: else the conversions are shared with K's, and moved to where V's go)
                    __asm__("" : "+v"(raw.x[2 * i]), "+v"(raw.x[2 * i + 1]));
                    h8 *d = to + (x >> 6) * 256 + (x & 63);
                    if (CW == 32) {
#pragma unroll
                        for (int t4 = 0; t4 < 4; t4++) d[t4 * 64] = to_half(raw.x[2 * i][t4], raw.x[2 * i + 1][t4]);
                    } else {
#pragma unroll
                        for (int t4 = 0; t4 < 4; t4++)
                            d[t4 * 64] = to_half(raw.x[2 * i + t4 / 2][t4 % 2 * 2], raw.x[2 * i + t4 / 2][t4 % 2 * 2 + 1]);
                    }
                }
            }
        }
    };
};

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
    if (A.s.row && columns * A.H >= MANY && columns >= EACH * (long long)A.s.n_seq) return launch_wide<Fp8, HD, DT>(A, s);
    if (columns > 16ll * A.s.n_seq) return launch<Fp8, HD, DT, NW, CG>(A, s);
    return launch<Fp8, HD, DT, NW, 1>(A, s);
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
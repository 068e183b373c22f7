// sp_fp4_attn.hip -- attention over the 4-bit block cache (sp_block_attn.h): its codes as operands, and
// which kernel a call takes.
//
// E2M1 codes times a power of two are exact in fp16 as long as the power stays in its range. A
// block's codes are converted relative to its largest exponent, which is then the block's scale
// for the loop (that of the 8-bit cache): exact for values down to 2^-23 of the block's largest
// scale, below that rounded at 2^-24 of it.
//
// Half of the 8-bit cache's bytes, and twice its conversions: a pair of codes takes one instruction, and with the
// scale in it none more, but V's pairs are neighbours in channels where the operand wants positions, a
// permutation each. Few rows are then bound by the vector unit as much as by memory: one sequence of 32768 positions of 8 heads
// of 128 (36 MB) 17.8 us, where 256 blocks of threads hold two blocks a wave: 2 us to the first codes, 9.5 in the loop (5
// of them issue vector instructions), 5 for the join of 32 shares; 16 sequences of 1 to 4K of 32 heads of 96, float32
// rows (139 MB) 45.4 us, 3.1 TB/s; 12 of 1 to 4.5K with up to five rows (38 MB) 22.4 us. Half blocks (32 positions a wave
// at a time, 137 registers for 179) took 18.6, 65 and 25.5 us where whole ones took 17.8, 56 (that case now has two
// shares a CU, the longest first) and 22.5; the next block's codes two blocks ahead 19.0 for the
// first; scaled matrix instructions, which take the codes as they are, sum 32 products with 15 bits.
// Many rows differ by the conversion alone (LDS holds fp16 in both): 2048 rows over 32768 positions, 32 / 8 heads of
// 128, 880 to 905 us by card (1.18 to 1.21 PFLOP/s; the 8-bit cache 887 to 904); 2048 rows in a window of 1024, 16 / 8 heads of
// 256, 56 us (51), the matrix cores busy 28% of the cycles, the vector unit 43, LDS 37.
#include "sp_block_attn.h"
#include "sp_fp4.h"

namespace {

using namespace sp_block;
using sp_fp4::eight;
using sp_fp4::Largest;
using sp_fp4::relative;

// The float with exponent byte b of e (b known where this is expanded): the byte, moved, in one instruction.
__device__ __forceinline__ float byte_power(unsigned e, int b) {
    float r;
    const int by = 23;
    if (b == 0) __asm__("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_0" : "=v"(r) : "v"(by), "v"(e));
    else if (b == 1) __asm__("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_1" : "=v"(r) : "v"(by), "v"(e));
    else if (b == 2) __asm__("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_2" : "=v"(r) : "v"(by), "v"(e));
    else __asm__("v_lshlrev_b32_sdwa %0, %1, %2 dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:DWORD src1_sel:BYTE_3" : "=v"(r) : "v"(by), "v"(e));
    return r;
}
// Two codes: byte b of w.
__device__ __forceinline__ h2 two(unsigned w, float scale, int b) {
    return b == 0 ? sp_fp4::two<0>(w, scale) : b == 1 ? sp_fp4::two<1>(w, scale) : b == 2 ? sp_fp4::two<2>(w, scale)
                                                                                          : sp_fp4::two<3>(w, scale);
}

struct Fp4 {
    // A block in a wave's registers. K: lane (r, g) has plane 4 c + g of quad Q(r). V: lane (r, g) has
    // quads 4 i + g of plane r (head_dim 64: half of plane r / 2; 96: lanes past plane 11 repeat it, and
    // their rows of the output are dropped; 256: planes r and 16 + r).
    template <int HD>
    struct Few {
        static constexpr int NC = HD / 32, PV = HD == 256 ? 2 : 1, CH = HD == 64 ? 4 : 8, ND = PV * CH, AT_ONCE = 2;
        u4 kr[NC], vr[PV][4], vs[PV];
        unsigned ks[NC];
        static __device__ __forceinline__ int plane(int r, int x) { return HD == 64 ? r >> 1 : HD == 96 ? min(r, 11) : 16 * x + r; }
        __device__ __forceinline__ void look_up(const SpFp8Attn &, long long) {}
        __device__ __forceinline__ void load_k(const SpFp8Side &S, long long tile, int lane) {
            const int r = lane & 15, g = lane >> 4;
            const uint8_t *p = S.codes + tile * sp_fp4_tile(HD) + g * 256 + (4 * (r & 3) + (r >> 2)) * 16;
            const uint8_t *e = S.exps + tile * sp_fp4_exps(HD) + r * 4;
#pragma unroll
            for (int c = 0; c < NC; c++) {
                kr[c] = *reinterpret_cast<const u4 *>(p + c * 1024);
                ks[c] = *reinterpret_cast<const unsigned *>(e + c * 64);
            }
        }
        __device__ __forceinline__ void load_v(const SpFp8Side &S, long long tile, int lane) {
            const int r = lane & 15, g = lane >> 4;
            const uint8_t *p = S.codes + tile * sp_fp4_tile(HD) + g * 16, *e = S.exps + tile * sp_fp4_exps(HD) + g * 16;
#pragma unroll
            for (int x = 0; x < PV; x++) {
                const int n = plane(r, x);
#pragma unroll
                for (int i = 0; i < 4; i++) vr[x][i] = *reinterpret_cast<const u4 *>(p + n * 256 + i * 64);
                vs[x] = *reinterpret_cast<const u4 *>(e + (n >> 2) * 64);
            }
        }
        // the block's largest exponent; from here on ks and vs are relative to it
        __device__ __forceinline__ int k_exponent(int) {
            Largest m;
#pragma unroll
            for (int c = 0; c < NC; c++) m.add(ks[c]);
            const int top = uniform(sp_fp4::row_max(m.get()));  // the same in all four rows
#pragma unroll
            for (int c = 0; c < NC; c++) ks[c] = relative(ks[c], top);
            return top - 127;
        }
        __device__ __forceinline__ int v_exponent(int) {
            Largest m;
#pragma unroll
            for (int x = 0; x < PV; x++)
#pragma unroll
                for (int i = 0; i < 4; i++) m.add(vs[x][i]);
            const int top = sp_fp4::wave_max(m.get());
#pragma unroll
            for (int x = 0; x < PV; x++)
#pragma unroll
                for (int i = 0; i < 4; i++) vs[x][i] = relative(vs[x][i], top);
            if (HD == 64) {
                const int half = (threadIdx.x & 1) * 16;
#pragma unroll
                for (int i = 0; i < 4; i++) vr[0][i] >>= half;
            }
            return top - 127;
        }
        // row blocks 2 u and 2 u + 1 of step c
        __device__ __forceinline__ void k_rows(int c, int u, h8 &a, h8 &b) const {
            a = eight(kr[c][2 * u], byte_power(ks[c], 2 * u));
            b = eight(kr[c][2 * u + 1], byte_power(ks[c], 2 * u + 1));
        }
        // channels d and d + 1: one byte of each of the lane's sixteen positions, turned
        __device__ __forceinline__ void v_rows(int d, h8 (&a)[AT_ONCE][2]) const {
            const int x = d / CH, byte = d % CH / 2;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                h2 c[8];
#pragma unroll
                for (int k = 0; k < 8; k++) c[k] = two(vr[x][2 * s + k / 4][k % 4], byte_power(vs[x][2 * s + k / 4], k % 4), byte);
#pragma unroll
                for (int o = 0; o < 2; o++)
                    a[o][s] = h8{c[0][o], c[1][o], c[2][o], c[3][o], c[4][o], c[5][o], c[6][o], c[7][o]};
            }
        }
        // position of value i of row block n, from the lane's first; its step and place among V's operands
        static constexpr __device__ __forceinline__ int at(int n, int i) { return 16 * i + n; }
        static constexpr __device__ __forceinline__ int step(int, int i) { return i / 2; }
        static constexpr __device__ __forceinline__ int place(int n, int i) { return i % 2 * 4 + n; }
        static __device__ __forceinline__ void put(float *rec, const f4 (&o)[ND], int g, float unit) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int r = 4 * g + i;
                if (HD == 96 && r >= 12) break;
#pragma unroll
                for (int d = 0; d < ND; d += 4)
                    *reinterpret_cast<f4 *>(rec + d / CH * 128 + r * CH + d % CH) =
                        f4{o[d][i], o[d + 1][i], o[d + 2][i], o[d + 3][i]} * unit;
            }
        }
    };

    // A block on its way into LDS: half of the threads bring K, half V, in pieces of a quad of a plane. Of K
    // that is an operand row of eight channels for each of four positions (16 bytes each); of V, half of an operand
    // row of eight positions for each of eight channels (8 bytes each). Rows are put where the lanes
    // that write at once meet no bank twice, nor those that read (of a read of 16 bytes a lane these are lanes 0 to 3,
    // 12 to 15, 20 to 23 and 24 to 27 of each 32, and the others): of K a row's place is turned by other bits of
    // it, of V steps, upper lanes and row blocks lie apart by what keeps them in different banks.
    template <int HD, int NT, int CW>
    struct Wide {
        static constexpr int HT = NT / 2, NW = NT / 64;
        static constexpr int NS = CW == 32 ? HD / 16 : HD / 32, NP = CW == 32 ? 4 : 2, PAD = CW == 32 ? 0 : 2;
        static constexpr int PIECES = 2 * HD, PER = (PIECES + HT - 1) / HT;
        // fp16 eights: of a block's place in LDS, of a row block of it, of a step of V
        static constexpr int K_ROW = NS * 64 + PAD, K_PLACE = 64 / CW * K_ROW;
        static constexpr int V_STEP = CW == 32 ? 66 : 73, V_ROW = CW == 32 ? 264 : 148, V_PLACE = HD / CW * V_ROW;
        static constexpr int LDS = 2 * (K_PLACE + V_PLACE) * 16, BYTES = LDS + 64 * 4;
        static_assert(64 % NW == 0);
        struct Raw {
            u4 x[PER];
            unsigned e[PER];
        };
        // place of lane `lane` of an operand of K, and of one of V
        static constexpr __device__ __forceinline__ int at(int lane) { return lane ^ ((lane >> 3) & (CW == 32 ? 3 : 1)); }
        static constexpr __device__ __forceinline__ int v_at(int lane) { return lane + (lane >> 5) * (CW == 32 ? 1 : 2); }
        static __device__ __forceinline__ bool mine(int x) { return PER * HT == PIECES || x < PIECES; }
        // The largest exponents of the 64 blocks that the lanes have: each wave finds those of its share
        // of them, coalesced, and all meet in LDS.
        static __device__ __forceinline__ void look_up(const SpFp8Attn &A, int h, int blk, int w, int lane, int *area, int &ekb,
                                                       int &evb) {
            constexpr int EACH = 64 / NW, DW = sp_fp4_exps(HD) / 4, TWICE = DW > 64 ? 2 : 1, SOME = EACH / TWICE;
#pragma unroll 1
            for (int i0 = 0; i0 < EACH; i0 += SOME) {  // (as many loads together as the loop's registers leave room for)
                unsigned ke[SOME][TWICE], ve[SOME][TWICE];
#pragma unroll
                for (int i = 0; i < SOME; i++) {
                    const int b = max(__builtin_amdgcn_readlane(blk, w * EACH + i0 + i), 0);
                    const long long tile = ((long long)b * A.H + h) * DW;
#pragma unroll
                    for (int t = 0; t < TWICE; t++) {
                        const int x = min(lane + t * 64, DW - 1);
                        ke[i][t] = reinterpret_cast<const unsigned *>(A.k.exps)[tile + x];
                        ve[i][t] = reinterpret_cast<const unsigned *>(A.v.exps)[tile + x];
                    }
                }
#pragma unroll
                for (int i = 0; i < SOME; i++) {
                    Largest k, v;
#pragma unroll
                    for (int t = 0; t < TWICE; t++) {
                        k.add(ke[i][t]);
                        v.add(ve[i][t]);
                    }
                    const int both = sp_fp4::wave_max(k.get()) | sp_fp4::wave_max(v.get()) << 8;
                    if (lane == 0) area[w * EACH + i0 + i] = both;
                }
            }
            lds_barrier();
            // A block that is missing is masked, and what is staged in its place (block 0, which another stream may be writing)
            // meets weights of 0: relative to the largest exponent there is it is finite whatever it is.
            ekb = blk < 0 ? SP_FP4_MOST : area[lane] & 255;
            evb = blk < 0 ? SP_FP4_MOST : area[lane] >> 8;
        }
        static __device__ __forceinline__ void fetch_k(const SpFp8Side &S, long long tile, int st, Raw &raw) {
            const uint8_t *p = S.codes + tile * sp_fp4_tile(HD), *e = S.exps + tile * sp_fp4_exps(HD);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int x = st + i * HT, q = x & 15;  // x = (plane, quad)
                if (!mine(x)) continue;
                raw.x[i] = *reinterpret_cast<const u4 *>(p + x * 16);
                raw.e[i] = *reinterpret_cast<const unsigned *>(e + (x >> 6) * 64 + (q & 3) * 16 + (q >> 2) * 4);
            }
        }
        // A V piece: its plane and quad; which step of the product, group of lanes and half of an eight that quad is.
        struct Piece {
            int n, quad, step, sub, half;
        };
        static __device__ __forceinline__ Piece piece(int x) {
            Piece p;
            if (CW == 32) {  // x = (plane, quad)
                p.n = x >> 4;
                p.quad = x & 15;
                p.step = p.quad >> 2;
                p.half = p.quad >> 1 & 1;
                p.sub = p.quad & 1;
            } else {  // x = (plane / 4, sub % 2, plane % 2, plane / 2 % 2, sub / 2, step, half)
                p.n = (x >> 6) * 4 + (x >> 3 & 1) * 2 + (x >> 4 & 1);
                p.half = x & 1;
                p.step = x >> 1 & 1;
                p.sub = (x >> 2 & 1) * 2 + (x >> 5 & 1);
                p.quad = p.step * 8 + p.half * 4 + p.sub;
            }
            return p;
        }
        static __device__ __forceinline__ void fetch_v(const SpFp8Side &S, long long tile, int st, Raw &raw) {
            const uint8_t *p = S.codes + tile * sp_fp4_tile(HD), *e = S.exps + tile * sp_fp4_exps(HD);
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int x = st + i * HT;
                if (!mine(x)) continue;
                const Piece v = piece(x);
                raw.x[i] = *reinterpret_cast<const u4 *>(p + v.n * 256 + v.quad * 16);
                raw.e[i] = *reinterpret_cast<const unsigned *>(e + (v.n >> 2) * 64 + (v.quad & 3) * 16 + (v.quad >> 2) * 4);
            }
        }
        static __device__ __forceinline__ void stage_k(Raw &raw, int st, int top, h8 *to) {
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int x = st + i * HT, q = x & 15, n = x >> 4;
                if (!mine(x)) continue;
                const unsigned rel = relative(raw.e[i], top + 127);
                // its first position's lane and row block
                const int lane = CW == 32 ? (n & 1) * 32 + 4 * (q & 7) : (n & 3) * 16 + 4 * (q & 3);
                h8 *d = to + (CW == 32 ? (q >> 3) * K_ROW + (n >> 1) * 64 : (q >> 2) * K_ROW + (n >> 2) * 64);
#pragma unroll
                for (int b = 0; b < 4; b++) d[at(lane + b)] = eight(raw.x[i][b], byte_power(rel, b));
            }
        }
        static __device__ __forceinline__ void stage_v(Raw &raw, int st, int top, h8 *to) {
            typedef _Float16 h4 __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int i = 0; i < PER; i++) {
                const int x = st + i * HT;
                if (!mine(x)) continue;
                const Piece v = piece(x);
                const unsigned rel = relative(raw.e[i], top + 127);
                float scale[4];
#pragma unroll
                for (int b = 0; b < 4; b++) scale[b] = byte_power(rel, b);
                const int lane = v.sub * CW + v.n * 8 % CW;  // of its first channel
                h4 *d = reinterpret_cast<h4 *>(to + v.n * 8 / CW * V_ROW + v.step * V_STEP + v_at(lane)) + v.half;
#pragma unroll
                for (int byte = 0; byte < 4; byte++) {
                    h2 c[4];
#pragma unroll
                    for (int b = 0; b < 4; b++) c[b] = two(raw.x[i][b], scale[b], byte);
#pragma unroll
                    for (int o = 0; o < 2; o++) d[2 * (2 * byte + o)] = h4{c[0][o], c[1][o], c[2][o], c[3][o]};
                }
            }
        }
    };
};

// Which kernel. All figures are of 8 KV heads, in us; rows are 16-bit and head_dim is 128 where not said.
//   Many rows (MANY columns over all KV heads) go to the kernel that converts a block once, in LDS: 512 rows of 32 heads over
//   2048 positions take it 40 and the few-row kernel 46, 256 rows 34 and 26; with float32 rows 256 take 36 and 40,
//   128 28 and 23; at head_dim 256 256 take 45 and 59, 128 37 and 31. Behind a long cache the conversions outweigh that kernel's
//   slower start and its second launch, and half as many columns suffice: 128 rows over 4096 / 8192 / 16000 positions take
//   34 / 43 / 57 and 30 / 44 / 71, with float32 rows 36 / 50 / 78 and 33 / 54 / 100, at head_dim 256 45 / 60 / 93 and
//   53 / 98 / 181 (3000 positions 41 and 43).
//   The table's width stands for the cache's length, which only the device knows: in a table of 96 blocks (48 with 16-bit
//   rows of 256) and more short sequences take that kernel too, and lose: 256 rows over 1024 / 2048 positions take 42 / 34 where
//   a table as wide as the sequence gives them 19 / 27, 128 over 2048 28 for 23, 64 of each of 12 over 1000 51 for 42. Without the rule
//   long ones would lose as the figures before say.
//   Sequences of few rows each leave most of its columns idle (EACH): 32 sequences of 16 rows of 16 heads take 53 and 31,
//   of 32 heads 54 and 54, 16 of 64 rows of 32 heads 69 and 99; float32 rows 52 and 46, 56 and 82, 74 and 156.
//   Few rows: past a group for each CU half the waves a block leave a CU two blocks out of step, and two shares a CU
//   even out unequal lengths, beside the order in which they are begun: 40 sequences of 1 to 4K 35 us, with one share a
//   CU 51 (head_dim 256: 78 and 95). Decode at 4000
//   positions of 32 / 40 / 64 sequences takes 41 / 56 / 59 with four waves and 33 / 58 / 64 with eight, at 600 positions
//   12.7 / 16.6 / 17.1 and 12.5 / 19.5 / 21.4. With two column groups a wave eight stay ahead (64 sequences of 5 rows of
//   32 heads 85, with four 116).
template <int HD, int DT>
hipError_t launch_dt(const SpFp8Attn &A, hipStream_t s) {
    constexpr int NW = HD == 256 ? 4 : 8;
    constexpr int CG = HD == 256 || DT == SP_DTYPE_F32 ? 1 : 2;
    constexpr int MANY = 256 * 16 * CG + 1, EACH = 64, LONG = HD == 256 && DT != SP_DTYPE_F32 ? 48 : 96;
    const long long columns = (long long)A.s.n_rows * A.G;  // of each KV head
    if (A.s.row && columns >= EACH * (long long)A.s.n_seq &&
        (columns * A.H >= MANY || (columns * A.H >= MANY / 2 && most_blocks(A) >= LONG)))
        return launch_wide<Fp4, HD, DT>(A, s);
    if (CG == 2 && columns > 16ll * A.s.n_seq) return launch<Fp4, HD, DT, NW, CG>(A, s);
    if (few_groups(A, 16) * A.H > 256) return launch<Fp4, HD, DT, 4, 1>(A, s, 2);
    return launch<Fp4, HD, DT, NW, 1>(A, s);
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

hipError_t sp_fp4_launch_attn(const SpFp8Attn &A, int hd, int dtype, hipStream_t s) {
    switch (hd) {
        case 64: return launch_hd<64>(A, dtype, s);
        case 96: return launch_hd<96>(A, dtype, s);
        case 128: return launch_hd<128>(A, dtype, s);
        case 256: return launch_hd<256>(A, dtype, s);
    }
    return hipErrorInvalidValue;
}

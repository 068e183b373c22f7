// sp_fp4.h -- the 4-bit block cache: layout and argument blocks of its kernels.
//
// A block is 64 positions of one layer. For each KV head it holds a tile of 64 * head_dim OCP
// E2M1 codes for K, one for V, and for each position and 32 channels a biased exponent byte b:
// the codes count in units of 2^(b - 127) (the OCP MXFP4 format). Tiles lie in planes of eight
// channels, a dword for each position with the lowest channel in the lowest four bits:
//   byte (n * 64 + p) * 4 + j / 2 holds position p, channel 8 n + j;
// so 16 bytes are eight channels of four positions, a quad. Exponents lie in planes of 32
// channels, the quads of one turned (a 4 x 4 transpose):
//   byte G * 64 + (q % 4) * 16 + (q / 4) * 4 + p % 4 with q = p / 4 belongs to channels 32 G on.
//
// The scale belongs to a position because rows are then written and moved alone, with nothing
// around them rounded again. One loop reads K and V in this order without an exchange between
// lanes: K's row operand r takes position 4 Q(r) + b in row block b, Q(r) = 4 (r % 4) + r / 4, so a
// lane's 16 bytes are its rows of four row blocks; the scores of lane (g, column) are then
// positions 16 i + 4 g + b, and V's lane (r, g) needs quads 4 i + g of plane r, whose exponents the
// turn puts side by side.
#pragma once

#include "../../include/sp_hip_fp4.h"
#include "sp_fp8.h"

#define SP_FP4_MAX 6.0f
#define SP_FP4_EVICT_THREADS 1024  // of a block of eviction's kernels
#define SP_FP4_LEAST (127 + SP_FP8_EMIN)  // exponent byte of what no row was written to
#define SP_FP4_MOST (127 + SP_FP8_EMAX)   // and the largest

__host__ __device__ constexpr int sp_fp4_tile(int hd) { return 32 * hd; }  // bytes of codes
__host__ __device__ constexpr int sp_fp4_exps(int hd) { return 2 * hd; }   // and of exponents

// Place of position p's exponent in its plane.
__device__ __forceinline__ int sp_fp4_place(int p) { return (p >> 2 & 3) * 16 + (p >> 4) * 4 + (p & 3); }

struct SpFp4Copy {
    SpFp8Seqs s;
    SpFp8Side side[2];  // codes NULL: this side is skipped
    void *rows[2];
    float *weight;  // of the positions: [n_blocks][H][64]
    long long row_stride;
    int H;
    int aligned;  // elements of a row that may be read and written at a time: 8, 4 or 1
};

struct SpFp4Weigh {
    SpFp8Seqs s;
    SpFp8Side k;
    const void *q;
    const float *lse;
    float *weight;
    long long q_stride;
    int H, G;
    int window;
    float c;  // |kq_scale| * log2(e) / 2
    float lost;  // of an lse: what c and log2(e) lose in 32 bits, in powers of two (see weigh)
    int negate;
    int cus;
    int blocks;  // log2 of the blocks that a block of threads takes at a time
};

struct SpFp4Evict {
    SpFp8Seqs s;
    SpFp8Side side[2];
    float *weight;
    int *kept;  // [n_seq][H][keep]
    int H, NC;
    int keep, first, recent;
};

hipError_t sp_fp4_launch_write(const SpFp4Copy &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp4_launch_read(const SpFp4Copy &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp4_launch_attn(const SpFp8Attn &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp4_launch_weigh(const SpFp4Weigh &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp4_launch_evict(const SpFp4Evict &A, hipStream_t s);

namespace sp_fp4 {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

// Two codes, those of byte `B` of a dword, times a power of two, as fp16.
template <int B>
__device__ __forceinline__ h2 two(unsigned w, float scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, scale, B);
}
// A dword's eight codes.
__device__ __forceinline__ h8 eight(unsigned w, float scale) {
    const h2 a = two<0>(w, scale), b = two<1>(w, scale), c = two<2>(w, scale), d = two<3>(w, scale);
    return h8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Exponent bytes e of four positions relative to the block's largest, `top`: bytes of 2^(e - top) as
// floats have them. No byte borrows from its neighbour: they are within 87 and 167 and at most top.
__device__ __forceinline__ unsigned relative(unsigned e, int top) { return e - (unsigned)(top - 127) * 0x01010101u; }

// Largest bytes: of dwords, gathered in pairs of 16 bits.
typedef unsigned short s2 __attribute__((ext_vector_type(2)));
struct Largest {
    s2 odd = {0, 0}, even = {0, 0};  // in the upper bytes
    __device__ __forceinline__ void add(unsigned w) {
        odd = __builtin_elementwise_max(odd, __builtin_bit_cast(s2, w));
        even = __builtin_elementwise_max(even, __builtin_bit_cast(s2, w << 8));
    }
    __device__ __forceinline__ int get() const {
        const s2 m = __builtin_elementwise_max(odd, even);
        return (m[0] > m[1] ? m[0] : m[1]) >> 8;
    }
};
// Largest value (not negative) of each 16 lanes of a row.
__device__ __forceinline__ int row_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x128, 0xf, 0xf, true));  // row_ror 8, 4, 2, 1
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x124, 0xf, 0xf, true));
    v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x122, 0xf, 0xf, true));
    return max(v, __builtin_amdgcn_update_dpp(0, v, 0x121, 0xf, 0xf, true));
}
// And of a wave, in a scalar register.
__device__ __forceinline__ int wave_max(int v) {
    v = row_max(v);
    return __builtin_amdgcn_readfirstlane(max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
                                              max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48))));
}

}  // namespace sp_fp4

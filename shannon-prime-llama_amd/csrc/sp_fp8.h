// sp_fp8.h -- the 8-bit block cache: layout, argument blocks and the device helpers that its
// write, read and attention kernels share.
//
// A block is 64 positions of one layer. For each KV head it holds a tile of 64 * head_dim
// OCP E4M3 codes for K, one for V, and for each a biased exponent byte b: the codes count
// in units of 2^(b - 127). The order inside a tile is that of the matrix instructions'
// operands, so that a wave's 16-byte loads of a tile are contiguous and need no exchange:
//   K: 16 bytes are eight channels of position r and of position r + 16,
//      byte ((u * hd/32 + c) * 64 + g * 16 + r) * 16 + half * 8 + j holds
//      position 32 u + 16 half + r, channel 32 c + 8 g + j;
//   V: 16 bytes are one channel of sixteen positions,
//      byte (dg * 64 + g * 16 + r) * 16 + 4 t + i holds position 16 t + 4 g + i, channel 16 dg + r.
// With K as the row operand the scores of lane (g, column) are positions 16 t + 4 g + i,
// which is how V's bytes are grouped: the weights go into the second product from the
// registers they were made in.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/shannon_prime.h"
#include "../../include/sp_hip.h"

#define SP_FP8_EMIN (-40)
#define SP_FP8_EMAX 40
#define SP_FP8_MAX 448.0f

// Sequences of a call as the kernels take them.
struct SpFp8Seqs {
    const int *table;  // [n_seq][stride] block numbers
    const int *len;    // [n_seq] positions, the call's rows included
    const int *row;    // [n_seq + 1] first rows, or NULL: row i is sequence i's
    int n_seq, stride, n_rows, n_blocks;
};

// One side (K or V) of a layer.
struct SpFp8Side {
    uint8_t *codes;  // [n_blocks][H][64 * hd]
    uint8_t *exps;   // [n_blocks][H]
};

struct SpFp8Copy {
    SpFp8Seqs s;
    SpFp8Side side[2];  // codes NULL: this side is skipped
    void *rows[2];
    long long row_stride;
    int H;
    int aligned;  // rows may be read and written four elements at a time
};

struct SpFp8Attn {
    SpFp8Seqs s;
    SpFp8Side k, v;
    const void *q;
    void *out;
    float *lse;
    long long q_stride, out_stride;
    int H, G;  // KV heads, query heads per KV head
    int window;
    float c;   // kq_scale * log2(e) / 2, not negative (half: a float whatever kq_scale is)
    int negate;
    float *part;    // partial results: part_rows rows of hd + 4 floats
    int part_rows;
    int *counters;  // SP_FP8_SLOTS, one per partial result, zero between calls
    int target;     // CUs; the launch makes it the blocks that fill them
    int least;      // fewest cache blocks of a share (the launch's choice)
    float join;     // rounds in which a block of threads joins shares (the launch's)
};

hipError_t sp_fp8_launch_write(const SpFp8Copy &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp8_launch_read(const SpFp8Copy &A, int hd, int dtype, hipStream_t s);
hipError_t sp_fp8_launch_attn(const SpFp8Attn &A, int hd, int dtype, hipStream_t s);
// Rows of partial results. Shares number at most 512 (twice 256 CUs): of 32 columns in the kernel
// for few rows, of at most 256 (128 at head_dim 256) in the one for many, which only prefill calls use.
#define SP_FP8_DECODE_ROWS (512 * 32)
inline int sp_fp8_prefill_rows(int hd) { return 512 * (hd == 256 ? 128 : 256); }

#define SP_FP8_SLOTS 1024

// A launch's threads along its first axis are counted in 32 bits.
#define SP_FP8_MOST_THREADS 0xffffffffll
#define SP_FP8_COPY_THREADS 256  // of a block of write or read

__device__ __forceinline__ int sp_fp8_floor64(int x) { return x >> 6; }  // arithmetic: toward -inf

// Rows and length of sequence i, whatever the arrays hold: 0 <= r0 <= r1 <= n_rows,
// 0 <= len <= 2^30 (what the longest table row covers).
__device__ __forceinline__ void sp_fp8_seq(const SpFp8Seqs &S, int i, int &r0, int &r1, int &len) {
    len = min(max(S.len[i], 0), 1 << 30);
    if (S.row) {
        r0 = min(max(S.row[i], 0), S.n_rows);
        r1 = min(max(S.row[i + 1], r0), S.n_rows);
    } else {
        r0 = i;
        r1 = i + 1;
    }
}

// Block number of a sequence's positions [64 j, 64 j + 64), or -1 where there is none.
__device__ __forceinline__ int sp_fp8_block(const SpFp8Seqs &S, int seq, int j) {
    if (j < 0 || j >= S.stride) return -1;
    const int b = S.table[(long long)seq * S.stride + j];
    return b >= 0 && b < S.n_blocks ? b : -1;
}

// The exponent that a byte of the cache stands for; one that no write made counts as the nearest.
__device__ __forceinline__ int sp_fp8_exponent(int b) { return min(max(b - 127, SP_FP8_EMIN), SP_FP8_EMAX); }

// Inclusive sum over the lanes of a wave (every lane active): shifts inside the rows of 16, then
// the rows' sums through scalar registers.
__device__ __forceinline__ int sp_fp8_scan(int v, int lane) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    const int a = __builtin_amdgcn_readlane(v, 15), b = a + __builtin_amdgcn_readlane(v, 31),
              c = b + __builtin_amdgcn_readlane(v, 47);
    return v + (lane < 16 ? 0 : lane < 32 ? a : lane < 48 ? b : c);
}

template <int DT>
struct SpFp8Elem;
template <>
struct SpFp8Elem<SP_DTYPE_F32> {
    typedef float T;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct SpFp8Elem<SP_DTYPE_F16> {
    typedef _Float16 T;
    static __device__ __forceinline__ float get(_Float16 x) { return (float)x; }
    static __device__ __forceinline__ _Float16 put(float x) { return (_Float16)x; }
};
template <>
struct SpFp8Elem<SP_DTYPE_BF16> {
    typedef __bf16 T;
    static __device__ __forceinline__ float get(__bf16 x) { return (float)x; }
    static __device__ __forceinline__ __bf16 put(float x) { return (__bf16)x; }
};

// 2^e for e in [-126, 127]
__device__ __forceinline__ float sp_fp8_pow2(int e) { return __int_as_float((e + 127) << 23); }

namespace sp_fp8 {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef unsigned int u4 __attribute__((ext_vector_type(4)));

// Four elements of a row; `aligned`: at an address that a vector load takes.
template <int DT>
__device__ __forceinline__ f4 load4(const void *base, long long off, bool aligned) {
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const T *p = reinterpret_cast<const T *>(base) + off;
    f4 x;
    if (aligned) {
        const T4 v = *reinterpret_cast<const T4 *>(p);
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = SpFp8Elem<DT>::get(v[k]);
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = SpFp8Elem<DT>::get(p[k]);
    }
    return x;
}

template <int DT>
__device__ __forceinline__ void store4(void *base, long long off, f4 x, bool aligned) {
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T4 __attribute__((ext_vector_type(4)));
    T *p = reinterpret_cast<T *>(base) + off;
    T4 v;
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = SpFp8Elem<DT>::put(x[k]);
    if (aligned) {
        *reinterpret_cast<T4 *>(p) = v;
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = v[k];
    }
}

}  // namespace sp_fp8

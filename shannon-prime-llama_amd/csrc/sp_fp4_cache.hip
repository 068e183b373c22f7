// sp_fp4_cache.hip -- writing rows into the 4-bit block cache and reading them back.
//
// The scale of 32 channels is 2^e with the least e in [-40, 40] for which their largest magnitude
// is at most 6 * 2^e: nothing is clipped, and every code is within half a step of its value. A
// power of two makes quantising a multiplication without error, followed by one rounding.
//
// One block of threads serves one (cache block, KV head, side). A thread takes eight channels of a
// position (16 bytes of a 16-bit row, so a wave's loads are whole lines), which are a dword of
// codes; four neighbours share a scale and agree on it in two exchanges inside the wave. A whole
// block's codes and exponents go through LDS and out in 16-byte stores; of a part of one each
// dword and byte is stored alone, and no other position's is touched.
#include "sp_fp4.h"

namespace {

using namespace sp_fp4;
using sp_fp8::f4;
using sp_fp8::u4;
using sp_fp8::load4;
using sp_fp8::store4;

constexpr int NT = SP_FP8_COPY_THREADS;
// A plane of codes in LDS: 64 dwords and four spare ones, which put the planes that a wave writes at
// once into different banks.
constexpr int PLANE = 68;

// Eight elements of a row; `aligned`: how many may be read at a time.
template <int DT>
__device__ __forceinline__ void row8(const void *base, long long off, int aligned, float (&x)[8]) {
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T8 __attribute__((ext_vector_type(8)));
    if (sizeof(T) == 2 && aligned == 8) {
        const T8 v = *reinterpret_cast<const T8 *>(reinterpret_cast<const T *>(base) + off);
#pragma unroll
        for (int k = 0; k < 8; k++) x[k] = SpFp8Elem<DT>::get(v[k]);
        return;
    }
    const f4 a = load4<DT>(base, off, aligned >= 4), b = load4<DT>(base, off + 4, aligned >= 4);
#pragma unroll
    for (int k = 0; k < 4; k++) {
        x[k] = a[k];
        x[4 + k] = b[k];
    }
}

template <int DT>
__device__ __forceinline__ void put8(void *base, long long off, int aligned, const float (&x)[8]) {
    typedef typename SpFp8Elem<DT>::T T;
    typedef T T8 __attribute__((ext_vector_type(8)));
    if (sizeof(T) == 2 && aligned == 8) {
        T8 v;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = SpFp8Elem<DT>::put(x[k]);
        *reinterpret_cast<T8 *>(reinterpret_cast<T *>(base) + off) = v;
        return;
    }
    store4<DT>(base, off, f4{x[0], x[1], x[2], x[3]}, aligned >= 4);
    store4<DT>(base, off + 4, f4{x[4], x[5], x[6], x[7]}, aligned >= 4);
}

// Largest of four neighbouring lanes (none negative).
__device__ __forceinline__ float four_max(float v) {
    int b = __float_as_int(v);
    b = max(b, __builtin_amdgcn_update_dpp(0, b, 0xb1, 0xf, 0xf, true));  // lanes 1 0 3 2
    b = max(b, __builtin_amdgcn_update_dpp(0, b, 0x4e, 0xf, 0xf, true));  // lanes 2 3 0 1
    return __int_as_float(b);
}

template <int HD, int DT>
__global__ __launch_bounds__(NT) void k_fp4_write(SpFp4Copy A) {
    constexpr int NP = HD / 8, PER = 64 * NP / NT, TILE = sp_fp4_tile(HD), EXPS = sp_fp4_exps(HD);
    static_assert(PER * NT == 64 * NP && NP % 4 == 0 && NT % 4 == 0);
    __shared__ __align__(16) unsigned tile[NP * PLANE];
    __shared__ __align__(16) unsigned char exps[EXPS];
    const int tid = threadIdx.x, h = blockIdx.y, is_v = blockIdx.z;
    const SpFp8Side side = A.side[is_v];
    if (!side.codes) return;
    int seq, j, r0, first, last;
    if (!sp_fp8_pair(A.s, blockIdx.x, tid & 63, seq, j, r0, first, last)) return;
    // the call's positions in this cache block: [lo, hi) of its 64
    const int lo = max(first - j * 64, 0), hi = min(last + 1 - j * 64, 64);
    const long long row0 = (long long)r0 + ((long long)j * 64 - first);  // row of position 0 of the block
    float x[PER][8];
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int it = tid + k * NT, t = it / NP, n = it % NP;
        if (t >= lo && t < hi)
            row8<DT>(A.rows[is_v], (row0 + t) * A.row_stride + (long long)h * HD + n * 8, A.aligned, x[k]);
    }
    const int blk = sp_fp8_block(A.s, seq, j);  // while the rows are on their way
    if (blk < 0) return;
    const long long at = (long long)blk * A.H + h;
    uint8_t *dst = side.codes + at * TILE, *edst = side.exps + at * EXPS;
    const bool whole = lo == 0 && hi == 64;
    const float most = SP_FP4_MAX * 0x1p40f;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int it = tid + k * NT, t = it / NP, n = it % NP, eplace = (n >> 2) * 64 + sp_fp4_place(t);
        if (t < lo || t >= hi) {
            // a block that starts anew: what lies behind its rows counts as nothing in its largest exponent
            if (lo == 0 && n % 4 == 0) edst[eplace] = SP_FP4_LEAST;
            continue;
        }
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float v = x[k][i];
            x[k][i] = v != v ? 0.0f : fminf(fmaxf(v, -most), most);
            m = fmaxf(m, fabsf(x[k][i]));
        }
        // 6 = 1.5 * 2^2: one more than the exponent less 2 where the fraction is past 1.5
        int e = ((__float_as_int(four_max(m)) + 0x3fffff) >> 23) - 129;
        e = min(max(e, SP_FP8_EMIN), SP_FP8_EMAX);
        const float down = sp_fp8_pow2(-e);
#pragma unroll
        for (int i = 0; i < 8; i++) x[k][i] *= down;
        unsigned w = 0;
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][0], x[k][1], 1.0f, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][2], x[k][3], 1.0f, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][4], x[k][5], 1.0f, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[k][6], x[k][7], 1.0f, 3);
        if (whole) {
            tile[n * PLANE + t] = w;
            if (n % 4 == 0) exps[eplace] = (uint8_t)(e + 127);
        } else {
            *reinterpret_cast<unsigned *>(dst + (n * 64 + t) * 4) = w;
            if (n % 4 == 0) edst[eplace] = (uint8_t)(e + 127);
        }
    }
    if (!is_v)  // no attention yet
        for (int t = lo + tid; t < hi; t += NT) A.weight[at * 64 + t] = 0.0f;
    if (!whole) return;
    __syncthreads();
    for (int p = tid; p < NP * 16; p += NT)
        *reinterpret_cast<u4 *>(dst + p * 16) = *reinterpret_cast<const u4 *>(tile + (p >> 4) * PLANE + (p & 15) * 4);
    for (int p = tid; p < EXPS / 16; p += NT)
        *reinterpret_cast<u4 *>(edst + p * 16) = *reinterpret_cast<const u4 *>(exps + p * 16);
}

template <int HD, int DT>
__global__ __launch_bounds__(NT) void k_fp4_read(SpFp4Copy A) {
    constexpr int NP = HD / 8, PER = 64 * NP / NT, TILE = sp_fp4_tile(HD), EXPS = sp_fp4_exps(HD);
    __shared__ __align__(16) unsigned tile[NP * PLANE];
    __shared__ __align__(16) unsigned char exps[EXPS];
    const int tid = threadIdx.x, h = blockIdx.y, is_v = blockIdx.z;
    const SpFp8Side side = A.side[is_v];
    if (!side.codes) return;
    int seq, j, r0, first, last;
    if (!sp_fp8_pair(A.s, blockIdx.x, tid & 63, seq, j, r0, first, last)) return;
    const int blk = sp_fp8_block(A.s, seq, j);
    const int lo = max(first - j * 64, 0), hi = min(last + 1 - j * 64, 64);
    const long long row0 = (long long)r0 + ((long long)j * 64 - first);
    const long long at = (long long)max(blk, 0) * A.H + h;
    const uint8_t *src = side.codes + at * TILE, *esrc = side.exps + at * EXPS;
    // few rows: their dwords alone; more: the tile through LDS, in 16-byte loads (256 sequences of 1 / 8 / 16 / 64 rows
    // of 8 heads of 128, bf16: 10.8 / 12.3 / 14.8 / 24.2 us alone, 11.6 / 12.7 / 14.9 / 22.5 through LDS)
    const bool few = hi - lo < 16;
    if (!few) {
        for (int p = tid; p < NP * 16; p += NT)
            *reinterpret_cast<u4 *>(tile + (p >> 4) * PLANE + (p & 15) * 4) = *reinterpret_cast<const u4 *>(src + p * 16);
        for (int p = tid; p < EXPS / 16; p += NT)
            *reinterpret_cast<u4 *>(exps + p * 16) = *reinterpret_cast<const u4 *>(esrc + p * 16);
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int it = tid + k * NT, t = it / NP, n = it % NP;
        if (t < lo || t >= hi) continue;
        const int eplace = (n >> 2) * 64 + sp_fp4_place(t);
        unsigned w = few ? *reinterpret_cast<const unsigned *>(src + (n * 64 + t) * 4) : tile[n * PLANE + t];
        const int e = few ? esrc[eplace] : exps[eplace];
        if (blk < 0) w = 0;  // no block: zeros
        const float up = sp_fp8_pow2(sp_fp8_exponent(e));
        const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 0), b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 1),
                   c = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 2), d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.0f, 3);
        const float x[8] = {a[0] * up, a[1] * up, b[0] * up, b[1] * up, c[0] * up, c[1] * up, d[0] * up, d[1] * up};
        put8<DT>(A.rows[is_v], (row0 + t) * A.row_stride + (long long)h * HD + n * 8, A.aligned, x);
    }
}

template <int HD>
hipError_t launch(const SpFp4Copy &A, int dtype, bool write, hipStream_t s) {
    // a sequence of n rows touches at most n / 64 + 2 blocks (one without an array of rows)
    const long long pairs = A.s.row ? (long long)A.s.n_rows / 64 + 2ll * A.s.n_seq : A.s.n_seq;
    const dim3 grid((unsigned)pairs, (unsigned)A.H, 2);
    const void *f = nullptr;
    if (write)
        f = dtype == SP_DTYPE_F32 ? (const void *)k_fp4_write<HD, SP_DTYPE_F32>
          : dtype == SP_DTYPE_F16 ? (const void *)k_fp4_write<HD, SP_DTYPE_F16>
                                  : (const void *)k_fp4_write<HD, SP_DTYPE_BF16>;
    else
        f = dtype == SP_DTYPE_F32 ? (const void *)k_fp4_read<HD, SP_DTYPE_F32>
          : dtype == SP_DTYPE_F16 ? (const void *)k_fp4_read<HD, SP_DTYPE_F16>
                                  : (const void *)k_fp4_read<HD, SP_DTYPE_BF16>;
    void *args[] = {const_cast<SpFp4Copy *>(&A)};
    return hipLaunchKernel(f, grid, dim3(NT), args, 0, s);
}

hipError_t launch_hd(const SpFp4Copy &A, int hd, int dtype, bool write, hipStream_t s) {
    switch (hd) {
        case 64: return launch<64>(A, dtype, write, s);
        case 96: return launch<96>(A, dtype, write, s);
        case 128: return launch<128>(A, dtype, write, s);
        case 256: return launch<256>(A, dtype, write, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t sp_fp4_launch_write(const SpFp4Copy &A, int hd, int dtype, hipStream_t s) {
    return launch_hd(A, hd, dtype, true, s);
}
hipError_t sp_fp4_launch_read(const SpFp4Copy &A, int hd, int dtype, hipStream_t s) {
    return launch_hd(A, hd, dtype, false, s);
}

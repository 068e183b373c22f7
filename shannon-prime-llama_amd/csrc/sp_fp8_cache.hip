// sp_fp8_cache.hip -- writing rows into the 8-bit block cache and reading them back.
//
// The scale of a block is 2^e with the least e in [-40, 40] for which the block's largest
// magnitude is at most 448 * 2^e. A power of two costs E4M3 no precision (its numbers have
// the same relative step in every octave), lets a block grow its scale without rounding its
// normal codes again, and makes quantising a multiplication without error.
//
// One block of threads serves one (cache block, KV head, side): the positions of a cache
// block are one sequence's consecutive rows, so the block's maximum, the old scale and the
// codes belong to one block of threads and no atomic is needed. Thread items are four
// positions by four channels: a load of four elements per position (rows stay coalesced:
// 64 lanes cover two rows of head_dim 128), and four codes make a dword of either order
// (K: four channels of a position, V: four positions of a channel). A whole block's codes go
// through LDS and out in 16-byte stores; a part of one is stored in dwords, and in bytes where
// a dword of V has older positions.
//
// Both are bound by memory: each reads and writes what it has to once. Measured (one launch, K
// and V): six prompts of head_dim 64, 86 MB with their float32 rows, written in 18.0 us
// (4.8 TB/s, the rate of a large device copy); a 32K context of 8 heads of 128 read back as fp16,
// 201 MB, in 36.2 us (5.6 TB/s); 2048 rows appended inside a block, 12.6 MB, in 7.6 us and one
// row to each of 12 sequences in 4.9 us, where an empty launch takes 4.2.
#include "sp_fp8.h"

namespace {

using sp_fp8::f4;
using sp_fp8::u4;
using sp_fp8::load4;
using sp_fp8::store4;

// The (sequence, cache block) pair of a grid index: sequence, block index in the sequence and
// the call's rows of it. False: no such pair. Every lane of a wave agrees, in scalar registers.
__device__ __forceinline__ bool pair_of(const SpFp8Seqs &S, int p, int lane, int &seq, int &j, int &r0, int &first,
                                        int &last) {
    if (!S.row || S.n_seq == 1) {  // nothing to search
        seq = S.row ? 0 : p;
        int r1, len;
        sp_fp8_seq(S, seq, r0, r1, len);
        first = len - (r1 - r0);
        last = len - 1;
        j = sp_fp8_floor64(first) + (S.row ? p : 0);
        return r1 > r0 && j <= sp_fp8_floor64(last);
    }
    for (int i0 = 0; i0 < S.n_seq; i0 += 64) {
        const int i = i0 + lane;
        int a = 0, b = 0, len = 0, n = 0;
        if (i < S.n_seq) {
            sp_fp8_seq(S, i, a, b, len);
            if (b > a) n = sp_fp8_floor64(len - 1) - sp_fp8_floor64(len - (b - a)) + 1;
        }
        const int sum = sp_fp8_scan(n, lane);
        const unsigned long long past = __ballot(sum > p);
        if (past) {
            const int l = __ffsll(past) - 1;
            const auto of = [l](int v) { return __builtin_amdgcn_readlane(v, l); };
            seq = i0 + l;
            r0 = of(a);
            first = of(len) - (of(b) - r0);
            last = of(len) - 1;
            j = sp_fp8_floor64(first) + p - (of(sum) - of(n));
            return true;
        }
        p -= __builtin_amdgcn_readlane(sum, 63);
    }
    return false;
}

// Byte of (position t, channel d) in a tile; t and d multiples of 4 give a dword's first byte
// for K (channels d..d+3 of t) and, with t the quad's first position, for V (d's positions).
template <int HD>
__device__ __forceinline__ int k_byte(int t, int d) {
    return (((t >> 5) * (HD / 32) + (d >> 5)) * 64 + ((d >> 3) & 3) * 16 + (t & 15)) * 16 + ((t >> 4) & 1) * 8 + (d & 7);
}
__device__ __forceinline__ int v_byte(int t, int d) {
    return ((d >> 4) * 64 + ((t >> 2) & 3) * 16 + (d & 15)) * 16 + (t >> 4) * 4 + (t & 3);
}
// The tile in LDS has 16 spare bytes after each 256 (K) or 1024 (V), which spreads the
// dwords that a wave writes or reads at once over the banks.
__device__ __forceinline__ int k_pad(int b) { return b + (b >> 8) * 16; }
__device__ __forceinline__ int v_pad(int b) { return b + (b >> 10) * 16; }

__device__ __forceinline__ unsigned pack4(float a, float b, float c, float d) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
__device__ __forceinline__ f4 unpack4(unsigned w) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return f4{lo[0], lo[1], hi[0], hi[1]};
}

// The codes of word w at a scale 2^-d times as fine, rounded once more.
__device__ __forceinline__ unsigned recode(unsigned w, float down) {
    const f4 x = unpack4(w) * down;
    return pack4(x[0], x[1], x[2], x[3]);
}

constexpr int NT = SP_FP8_COPY_THREADS;

template <int HD, int DT>
__global__ __launch_bounds__(NT) void k_fp8_write(SpFp8Copy A) {
    constexpr int ITEMS = 16 * (HD / 4), PER = (ITEMS + NT - 1) / NT, TILE = 64 * HD;
    __shared__ __align__(16) unsigned char tile[TILE + TILE / 16];
    __shared__ float wmax[NT / 64];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y, is_v = blockIdx.z;
    const SpFp8Side side = A.side[is_v];
    if (!side.codes) return;
    int seq, j, r0, first, last;
    if (!pair_of(A.s, blockIdx.x, lane, seq, j, r0, first, last)) return;
    // the call's positions in this cache block: [lo, hi) of its 64
    const int lo = max(first - j * 64, 0), hi = min(last + 1 - j * 64, 64);
    const void *rows = A.rows[is_v];
    // row of position 0 of the block
    const long long row0 = (long long)r0 + ((long long)j * 64 - first);
    f4 x[PER][4];
    float m = 0.0f;
    const float top = SP_FP8_MAX * 0x1p40f;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int it = tid + k * NT, quad = it / (HD / 4), d = it % (HD / 4) * 4;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = quad * 4 + i;
            x[k][i] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (it < ITEMS && t >= lo && t < hi)
                x[k][i] = load4<DT>(rows, (row0 + t) * A.row_stride + (long long)h * HD + d, A.aligned);
        }
    }
    const int blk = sp_fp8_block(A.s, seq, j);  // while the rows are on their way
    if (blk < 0) return;
    uint8_t *exp_at = side.exps + (long long)blk * A.H + h;
    const int e_old = lo > 0 ? sp_fp8_exponent(*exp_at) : SP_FP8_EMIN;
#pragma unroll
    for (int k = 0; k < PER; k++)
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < 4; n++) {
                float v = x[k][i][n];
                v = v != v ? 0.0f : fminf(fmaxf(v, -top), top);
                x[k][i][n] = v;
                m = fmaxf(m, fabsf(v));
            }
#pragma unroll
    for (int s = 32; s; s >>= 1) m = fmaxf(m, __shfl_xor(m, s, 64));
    if (lane == 0) wmax[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(wmax[0], wmax[1]), fmaxf(wmax[2], wmax[3]));
    // 448 = 1.75 * 2^8: one more than the exponent less 8 where the fraction is past 1.75
    int e = ((__float_as_int(m) + 0x1fffff) >> 23) - 135;
    e = min(max(e, SP_FP8_EMIN), SP_FP8_EMAX);
    e = max(e, e_old);
    const float down = sp_fp8_pow2(-e);
    uint8_t *dst = side.codes + ((long long)blk * A.H + h) * TILE;
    if (lo > 0 && e > e_old) {
        // the older positions' codes, at the larger scale; the bytes of positions that hold
        // nothing yet stay as they are
        const float shift = sp_fp8_pow2(e_old - e);
        for (int p = tid; p < TILE / 16; p += NT) {
            u4 w = *reinterpret_cast<const u4 *>(dst + p * 16);
            if (is_v) {
                const int g = (p >> 4) & 3;
#pragma unroll
                for (int t4 = 0; t4 < 4; t4++) {
                    const int n = min(max(lo - (16 * t4 + 4 * g), 0), 4);  // old positions of this dword
                    const unsigned keep = n == 4 ? 0u : 0xffffffffu << (8 * n);
                    w[t4] = (w[t4] & keep) | (recode(w[t4], shift) & ~keep);
                }
            } else {
                const int t = (p / (HD / 32 * 64)) * 32 + (p & 15);
#pragma unroll
                for (int n = 0; n < 4; n++)
                    if (t + 16 * (n >> 1) < lo) w[n] = recode(w[n], shift);
            }
            *reinterpret_cast<u4 *>(dst + p * 16) = w;
        }
        // complete before the new positions' stores, which may share these 16 bytes
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }
    if (tid == 0) *exp_at = (uint8_t)(e + 127);
    const bool whole = lo == 0 && hi == 64;
#pragma unroll
    for (int k = 0; k < PER; k++) {
        const int it = tid + k * NT, quad = it / (HD / 4), d = it % (HD / 4) * 4;
        if (it >= ITEMS) break;
        unsigned w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) x[k][i] *= down;
        if (is_v) {
#pragma unroll
            for (int n = 0; n < 4; n++) w[n] = pack4(x[k][0][n], x[k][1][n], x[k][2][n], x[k][3][n]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = pack4(x[k][i][0], x[k][i][1], x[k][i][2], x[k][i][3]);
        }
        if (whole) {
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const int at = is_v ? v_pad(v_byte(quad * 4, d + n)) : k_pad(k_byte<HD>(quad * 4 + n, d));
                *reinterpret_cast<unsigned *>(tile + at) = w[n];
            }
        } else if (!is_v) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int t = quad * 4 + i;
                if (t >= lo && t < hi) *reinterpret_cast<unsigned *>(dst + k_byte<HD>(t, d)) = w[i];
            }
        } else if (quad * 4 >= lo && quad * 4 + 4 <= hi) {
#pragma unroll
            for (int n = 0; n < 4; n++) *reinterpret_cast<unsigned *>(dst + v_byte(quad * 4, d + n)) = w[n];
        } else {
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int t = quad * 4 + i;
                    if (t >= lo && t < hi) dst[v_byte(t, d + n)] = (uint8_t)(w[n] >> (8 * i));
                }
        }
    }
    if (!whole) return;
    __syncthreads();
    for (int p = tid; p < TILE / 16; p += NT)
        *reinterpret_cast<u4 *>(dst + p * 16) =
            *reinterpret_cast<const u4 *>(tile + (is_v ? v_pad(p * 16) : k_pad(p * 16)));
}

template <int HD, int DT>
__global__ __launch_bounds__(NT) void k_fp8_read(SpFp8Copy A) {
    constexpr int ITEMS = 16 * (HD / 4), TILE = 64 * HD;
    __shared__ __align__(16) unsigned char tile[TILE + TILE / 16];
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y, is_v = blockIdx.z;
    const SpFp8Side side = A.side[is_v];
    if (!side.codes) return;
    int seq, j, r0, first, last;
    if (!pair_of(A.s, blockIdx.x, lane, seq, j, r0, first, last)) return;
    const int blk = sp_fp8_block(A.s, seq, j);
    const int lo = max(first - j * 64, 0), hi = min(last + 1 - j * 64, 64);
    const long long row0 = (long long)r0 + ((long long)j * 64 - first);
    float up = 0.0f;
    if (blk >= 0) {
        up = sp_fp8_pow2(sp_fp8_exponent(side.exps[(long long)blk * A.H + h]));
        const uint8_t *src = side.codes + ((long long)blk * A.H + h) * TILE;
        for (int p = tid; p < TILE / 16; p += NT)
            *reinterpret_cast<u4 *>(tile + (is_v ? v_pad(p * 16) : k_pad(p * 16))) =
                *reinterpret_cast<const u4 *>(src + p * 16);
    }
    __syncthreads();
    for (int it = tid; it < ITEMS; it += NT) {
        const int quad = it / (HD / 4), d = it % (HD / 4) * 4;
        if (quad * 4 + 4 <= lo || quad * 4 >= hi) continue;
        f4 x[4];
        if (blk < 0) {
            x[0] = x[1] = x[2] = x[3] = f4{0.0f, 0.0f, 0.0f, 0.0f};  // no block: zeros
        } else if (is_v) {
            f4 c[4];
#pragma unroll
            for (int n = 0; n < 4; n++)
                c[n] = unpack4(*reinterpret_cast<const unsigned *>(tile + v_pad(v_byte(quad * 4, d + n)))) * up;
#pragma unroll
            for (int i = 0; i < 4; i++) x[i] = f4{c[0][i], c[1][i], c[2][i], c[3][i]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                x[i] = unpack4(*reinterpret_cast<const unsigned *>(tile + k_pad(k_byte<HD>(quad * 4 + i, d)))) * up;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = quad * 4 + i;
            if (t >= lo && t < hi)
                store4<DT>(A.rows[is_v], (row0 + t) * A.row_stride + (long long)h * HD + d, x[i], A.aligned);
        }
    }
}

template <int HD>
hipError_t launch(const SpFp8Copy &A, int dtype, bool write, hipStream_t s) {
    // a sequence of n rows touches at most n / 64 + 2 blocks (one without an array of rows)
    const long long pairs = A.s.row ? (long long)A.s.n_rows / 64 + 2ll * A.s.n_seq : A.s.n_seq;
    const dim3 grid((unsigned)pairs, (unsigned)A.H, 2);
    const void *f = nullptr;
    if (write)
        f = dtype == SP_DTYPE_F32 ? (const void *)k_fp8_write<HD, SP_DTYPE_F32>
          : dtype == SP_DTYPE_F16 ? (const void *)k_fp8_write<HD, SP_DTYPE_F16>
                                  : (const void *)k_fp8_write<HD, SP_DTYPE_BF16>;
    else
        f = dtype == SP_DTYPE_F32 ? (const void *)k_fp8_read<HD, SP_DTYPE_F32>
          : dtype == SP_DTYPE_F16 ? (const void *)k_fp8_read<HD, SP_DTYPE_F16>
                                  : (const void *)k_fp8_read<HD, SP_DTYPE_BF16>;
    void *args[] = {const_cast<SpFp8Copy *>(&A)};
    return hipLaunchKernel(f, grid, dim3(NT), args, 0, s);
}

hipError_t launch_hd(const SpFp8Copy &A, int hd, int dtype, bool write, hipStream_t s) {
    switch (hd) {
        case 64: return launch<64>(A, dtype, write, s);
        case 96: return launch<96>(A, dtype, write, s);
        case 128: return launch<128>(A, dtype, write, s);
        case 256: return launch<256>(A, dtype, write, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace

hipError_t sp_fp8_launch_write(const SpFp8Copy &A, int hd, int dtype, hipStream_t s) {
    return launch_hd(A, hd, dtype, true, s);
}
hipError_t sp_fp8_launch_read(const SpFp8Copy &A, int hd, int dtype, hipStream_t s) {
    return launch_hd(A, hd, dtype, false, s);
}

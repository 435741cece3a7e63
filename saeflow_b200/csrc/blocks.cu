// Block-scaled 8-bit matrices: e4m3 numbers with one power-of-two scale per 128 columns of a row
// ("row blocks") or per 128 x 128 tile. Quantising, scattering into and gathering out of a store.
//
//   s  = max(0, ((bits(amax) + 0x1FFFFF) >> 23) - 8)        amax over the block's finite elements
//   q  = e4m3_rn(x * 2^(127 - s))                           x ~ q * 2^(s - 127)
//
// 448 (the largest e4m3) is 1.75 * 2^8, so the scale exponent is amax's less 8, one more where its
// mantissa exceeds 1.75 (the carry of the addition). The product with a power of two is exact, so
// an element is rounded once, and dequantising is exact in every output type that has the range.
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "sf_common.cuh"
#include "sf_internal.h"

namespace sf {

namespace {

constexpr int kBlk = SF_BLOCK;

__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const int s = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
    return (uint32_t)max(s, 0);
}
// 2^(127 - s) for s <= 247 (scale_byte's range), and 2^(s - 127), a subnormal for s = 0.
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float scale_value(uint32_t s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

__device__ __forceinline__ void unpack_e4m3(uint32_t w, float *v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
        const float2 f = __half22float2(__half2(r));
        v[2 * h] = f.x;
        v[2 * h + 1] = f.y;
    }
}

// The aligned word of a row's e4m3 bytes at column k, a multiple of 4; 0 outside the K columns. A word that
// holds a column may also hold bytes past the last, which no one uses.
template <typename I>
__device__ __forceinline__ uint32_t load_word(const uint8_t *row, I k, I K) {
    return k >= 0 && k < K ? __ldg(reinterpret_cast<const uint32_t *>(row + k)) : 0u;
}

// Eight e4m3 bytes at column k of a row of `limit` columns; nothing past them is written.
__device__ __forceinline__ void store8(uint8_t *row, int64_t k, int64_t limit, uint2 w) {
    if (k + 8 <= limit) {
        *reinterpret_cast<uint2 *>(row + k) = w;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (k + j < limit) row[k + j] = (uint8_t)((j < 4 ? w.x : w.y) >> (8 * (j & 3)));
    }
}

// Sixteen of them, at a 16-byte aligned column.
__device__ __forceinline__ void store16(uint8_t *row, int64_t k, int64_t limit, uint4 w) {
    if (k + 16 <= limit) {
        *reinterpret_cast<uint4 *>(row + k) = w;
    } else {
        store8(row, k, limit, make_uint2(w.x, w.y));
        store8(row, k + 8, limit, make_uint2(w.z, w.w));
    }
}

// Sixteen elements as a thread holds them: 16-bit types as eight words of two, fp32
// as sixteen. Magnitudes compare as integers, two at a time in the 16-bit types.
template <typename XT>
struct Held {
    static constexpr bool HALF = sizeof(XT) == 2;
    static constexpr int WORDS = HALF ? 8 : 16;
    static constexpr uint32_t ABS = HALF ? 0x7fff7fffu : 0x7fffffffu;
    static __device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return HALF ? __vmaxu2(a, b) : max(a, b); }
    // fp32 value of element j of the words
    static __device__ __forceinline__ float value(const uint32_t *w, int j) {
        if constexpr (!HALF) {
            return __uint_as_float(w[j]);
        } else if constexpr (std::is_same_v<XT, __nv_bfloat16>) {
            return __uint_as_float((j & 1) ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        } else {
            const __half2 h = *reinterpret_cast<const __half2 *>(&w[j >> 1]);
            return (j & 1) ? __high2float(h) : __low2float(h);
        }
    }
    // fp32 magnitude bits of half `j` of a word of magnitudes
    static __device__ __forceinline__ uint32_t bits(uint32_t w, int j) { return __float_as_uint(value(&w, j)); }
    static __device__ __forceinline__ uint32_t bits(uint32_t w) { return HALF ? max(bits(w, 0), bits(w, 1)) : w; }
    // a word's magnitudes, 0 where they are not finite
    static __device__ __forceinline__ uint32_t finite(uint32_t w) {
        w &= ABS;
        if constexpr (HALF) {
            const uint32_t inf = std::is_same_v<XT, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
            return ((w & 0xffffu) < inf ? w & 0xffffu : 0u) | ((w >> 16) < inf ? w & 0xffff0000u : 0u);
        } else {
            return w < 0x7f800000u ? w : 0u;
        }
    }
    // NaN in place of what is not finite
    static __device__ __forceinline__ uint32_t nan_for_inf(uint32_t w) {
        if constexpr (HALF) {
            const uint32_t inf = std::is_same_v<XT, __nv_bfloat16> ? 0x7f80u : 0x7c00u;
            return w | ((w & 0x7fffu) >= inf ? 0x7fffu : 0u) | (((w >> 16) & 0x7fffu) >= inf ? 0x7fff0000u : 0u);
        } else {
            return (w & 0x7fffffffu) >= 0x7f800000u ? 0x7fffffffu : w;
        }
    }
};

__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}

// The 16 elements from column k of a row, zeros past K, in two steps so that several rows' loads can be under
// way before the first is used. `base` is the row's first element. Rows with a unit column stride are read in
// aligned 16-byte pieces and shifted into place, so any alignment of the element type costs one more piece
// and a few selects.
template <typename XT>
struct Fetched {
    uint32_t w[Held<XT>::WORDS + 4];
    unsigned off;  // bytes of the first piece before the first element
};

template <typename XT>
__device__ __forceinline__ void fetch16(const XT *base, int64_t k, int64_t K, int64_t sxk, Fetched<XT> &f) {
    using H = Held<XT>;
    constexpr int W = H::WORDS, PER = 16 / W;
    f.off = 0;
    if (sxk == 1 && k + 16 <= K) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(base + k);
        const uint4 *p = reinterpret_cast<const uint4 *>(at & ~uintptr_t(15));
        f.off = (unsigned)at & 15u;
#pragma unroll
        for (int j = 0; j < W + 4; j += 4) {
            if (j == W && f.off == 0) break;  // with off > 0 the last piece holds the last element
            const uint4 a = __ldg(p + j / 4);
            f.w[j] = a.x, f.w[j + 1] = a.y, f.w[j + 2] = a.z, f.w[j + 3] = a.w;
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < W; ++j) {
        XT e[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i)
            e[i] = k + j * PER + i < K ? __ldg(base + (k + j * PER + i) * sxk) : from_f32<XT>(0.f);
        if constexpr (PER == 1)
            f.w[j] = __float_as_uint(to_f32(e[0]));
        else
            f.w[j] = (uint32_t)*reinterpret_cast<const uint16_t *>(&e[0]) |
                     (uint32_t)*reinterpret_cast<const uint16_t *>(&e[1]) << 16;
    }
}

template <typename XT>
__device__ __forceinline__ void place16(Fetched<XT> &f, uint32_t *v) {
    using H = Held<XT>;
    constexpr int W = H::WORDS;
    if (f.off) {
#pragma unroll
        for (int j = 0; j < W + 2; ++j) f.w[j] = (f.off & 8) ? f.w[j + 2] : f.w[j];
#pragma unroll
        for (int j = 0; j < W + 1; ++j) f.w[j] = (f.off & 4) ? f.w[j + 1] : f.w[j];
        if (H::HALF && (f.off & 2)) {
#pragma unroll
            for (int j = 0; j < W; ++j) f.w[j] = __funnelshift_r(f.w[j], f.w[j + 1], 16);
        }
    }
#pragma unroll
    for (int j = 0; j < W; ++j) v[j] = f.w[j];
}

// Aligned and inside the matrix: the words as they lie.
template <typename XT>
__device__ __forceinline__ void load16_aligned(const XT *src, uint32_t *v) {
#pragma unroll
    for (int j = 0; j < Held<XT>::WORDS; j += 4) {
        const uint4 a = __ldg(reinterpret_cast<const uint4 *>(src) + j / 4);
        v[j] = a.x, v[j + 1] = a.y, v[j + 2] = a.z, v[j + 3] = a.w;
    }
}

// Sixteen held elements times a scale, as e4m3.
template <typename XT>
__device__ __forceinline__ uint4 pack16(const uint32_t *v, float inv) {
    using H = Held<XT>;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        w[j] = e4m3x2(H::value(v, 4 * j) * inv, H::value(v, 4 * j + 1) * inv) |
               e4m3x2(H::value(v, 4 * j + 2) * inv, H::value(v, 4 * j + 3) * inv) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Row blocks: eight lanes to a block of 128, sixteen elements each; a group takes two blocks of a row
// (`by` divides by the pairs of a row), so that enough bytes are on their way. Aligned fp32 rows are read as
// four neighbours from 4l of each 32, which puts a group's loads side by side (134 -> 115 us).
// Bound by HBM: 8192 x 16384 bf16 in 62.3 us, 65536 x 2304 fp32 in 115 us, 6.5 TB/s both, the rate of a copy;
// a few thousand rows by launch and latency (4095 x 2304 bf16 5.6 us, of which a launch is 2.2).
template <typename XT>
__global__ void __launch_bounds__(256) quant_rows_kernel(const XT *__restrict__ x, int64_t n, int64_t K, int64_t sxm,
                                                         int64_t sxk, bool vec, const int64_t *__restrict__ slots,
                                                         uint8_t *__restrict__ q, int64_t q_pitch,
                                                         uint8_t *__restrict__ s, int64_t s_pitch, int64_t cap,
                                                         Divisor by, unsigned *err) {
    using H = Held<XT>;
    const int l = threadIdx.x & 7;
    const int64_t item = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const int64_t row = by.div(item);
    if (row >= n) return;  // whole groups leave together
    const unsigned group = 0xffu << (threadIdx.x & 24);
    const int64_t pair = item - row * by.d;
    int64_t slot = row;
    if (slots) {
        slot = __ldg(slots + row);
        if (slot >= cap && l == 0 && pair == 0) atomicOr(err, kErrIndex);
        if (slot < 0 || slot >= cap) return;
    }
    // Sixteen columns from 16l; of aligned fp32 rows four from 4l of each 32, so that the group's 16-byte loads
    // are side by side.
    const XT *src = x + row * sxm;
    uint32_t v[2][H::WORDS];
    const bool whole = vec && (2 * pair + 2) * kBlk <= K;
    const bool quads = !H::HALF && whole;
    if (quads) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
#pragma unroll
            for (int j = 0; j < H::WORDS / 4; ++j) {
                const uint4 a = __ldg(reinterpret_cast<const uint4 *>(src + (2 * pair + b) * kBlk) + 8 * j + l);
                v[b][4 * j] = a.x, v[b][4 * j + 1] = a.y, v[b][4 * j + 2] = a.z, v[b][4 * j + 3] = a.w;
            }
        }
    } else if (whole) {
#pragma unroll
        for (int b = 0; b < 2; ++b) load16_aligned(src + (2 * pair + b) * kBlk + 16 * l, v[b]);
    } else {
        Fetched<XT> f[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) fetch16(src, (2 * pair + b) * kBlk + 16 * l, K, sxk, f[b]);
#pragma unroll
        for (int b = 0; b < 2; ++b) place16(f[b], v[b]);
    }
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const int64_t blk = 2 * pair + b;
        if (blk * kBlk >= K) break;
        uint32_t m = v[b][0] & H::ABS;
#pragma unroll
        for (int j = 1; j < H::WORDS; ++j) m = H::umax(m, v[b][j] & H::ABS);
#pragma unroll
        for (int d = 4; d; d >>= 1) m = H::umax(m, __shfl_xor_sync(group, m, d));
        uint32_t bits = H::bits(m);
        if (bits >= 0x7f800000u) {  // the group's: look at each element
            m = 0;
#pragma unroll
            for (int j = 0; j < H::WORDS; ++j) {
                m = H::umax(m, H::finite(v[b][j]));
                v[b][j] = H::nan_for_inf(v[b][j]);
            }
#pragma unroll
            for (int d = 4; d; d >>= 1) m = H::umax(m, __shfl_xor_sync(group, m, d));
            bits = H::bits(m);
        }
        const uint32_t sb = scale_byte(bits);
        uint8_t *dst = q + slot * q_pitch;
        const uint4 w = pack16<XT>(v[b], inverse_scale(sb));
        if (!H::HALF && quads) {
            uint32_t *to = reinterpret_cast<uint32_t *>(dst + blk * kBlk) + l;
            to[0] = w.x, to[8] = w.y, to[16] = w.z, to[24] = w.w;
        } else {
            store16(dst, blk * kBlk + 16 * l, K, w);
        }
        if (l == 0) s[slot * s_pitch + blk] = (uint8_t)sb;
    }
}

// Output elements of a thread of read_rows_kernel, eight to a piece. 16-bit outputs, 16384 rows of 2304 from a
// store of 262144: 22.5 us with 16, 19.9 with 32, 21.9 with 64; fp32, 65536 rows: 147, 141 and 145 us with 8,
// 16 and 32.
template <typename OT>
constexpr int kReadElements = sizeof(OT) == 4 ? 16 : 32;

// Two neighbours in the output type (16-bit conversions run at four times the rate in pairs).
__device__ __forceinline__ void store_pair(float *o, float a, float b) { o[0] = a, o[1] = b; }
__device__ __forceinline__ void store_pair(__nv_bfloat16 *o, float a, float b) {
    *reinterpret_cast<__nv_bfloat162 *>(o) = __floats2bfloat162_rn(a, b);
}
__device__ __forceinline__ void store_pair(__half *o, float a, float b) {
    *reinterpret_cast<__half2 *>(o) = __floats2half2_rn(a, b);
}

// Dequantising gather. A piece is eight numbers on their way to an aligned place of an output row (16 bytes of a
// 16-bit type, 32 of fp32 by two stores): `shift` elements of the row lie before its first 16-byte boundary,
// so piece c covers columns 8c - shift ... With shift = 0 a piece lies in one block; otherwise it may span
// two, with two scales. Eight lanes take eight neighbouring pieces at a time and several times over, so
// that enough bytes are on their way. `tile_shift` is 7 where a scale row serves 128 rows.
// Bound by HBM: 16384 of 262144 rows of 2304 as bf16 in 18.5 us, 6.1 TB/s, with some of them still in L2, 22.0 us
// with none; as fp32 (four bytes written for one read) 65536 rows in 140 us, 5.4 TB/s. Rows that start between
// boundaries: 20000 x 777 bf16 17.8 us, 2.6 TB/s. Walking the rows with a grid that stays, each row's index
// loaded a step ahead, was no faster (22.4 to 25.7 us).
template <typename OT, bool ALIGNED>
__global__ void __launch_bounds__(256, 4) read_rows_kernel(const uint8_t *__restrict__ q, int64_t q_pitch,
                                                        const uint8_t *__restrict__ s, int64_t s_pitch,
                                                        int64_t src_rows, int K, int tile_shift,
                                                        const int64_t *__restrict__ rows, OT *__restrict__ out,
                                                        int64_t n, int64_t out_pitch, Divisor by, unsigned *err) {
    constexpr int PIECES = kReadElements<OT> / 8;
    const int64_t group = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const int64_t i = by.div(group);
    if (i >= n) return;
    const int c = (int)(group - i * by.d) * 8 * PIECES + (threadIdx.x & 7);
    int64_t row = i;
    if (rows) {
        row = __ldg(rows + i);
        if (row >= src_rows && c == 0) atomicOr(err, kErrIndex);
    }
    const bool have = row >= 0 && row < src_rows;
    const uint8_t *src = q + row * q_pitch, *sc = s + (row >> tile_shift) * s_pitch;
    OT *dst = out + i * out_pitch;
    const int shift = ALIGNED ? 0 : (int)((reinterpret_cast<uintptr_t>(dst) & 15u) / sizeof(OT));
    uint2 w[PIECES];
    uint32_t sb[PIECES][2];
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int k = (c + 8 * p) * 8 - shift;  // may start before the row, or end past it
        w[p] = make_uint2(0u, 0u);
        sb[p][0] = sb[p][1] = 0;
        if (!have || k >= K || k + 8 <= 0) continue;
        sb[p][0] = __ldg(sc + (max(k, 0) >> 7));
        if (!ALIGNED) sb[p][1] = __ldg(sc + ((min(k + 8, K) - 1) >> 7));
        if (ALIGNED && k + 8 <= K) {
            w[p] = __ldg(reinterpret_cast<const uint2 *>(src + k));
        } else if (ALIGNED) {
            w[p] = make_uint2(load_word(src, k, K), load_word(src, k + 4, K));
        } else {
            const int k4 = k & ~3;
            const uint32_t a0 = load_word(src, k4, K), a1 = load_word(src, k4 + 4, K), a2 = load_word(src, k4 + 8, K);
            const int bits = 8 * (k & 3);
            w[p] = make_uint2(__funnelshift_r(a0, a1, bits), __funnelshift_r(a1, a2, bits));
        }
    }
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
        const int k = (c + 8 * p) * 8 - shift;
        if (k >= K) break;
        float v[8];
        unpack_e4m3(w[p].x, v);
        unpack_e4m3(w[p].y, v + 4);
        const float s0 = have ? scale_value(sb[p][0]) : 0.f, s1 = ALIGNED ? s0 : have ? scale_value(sb[p][1]) : 0.f;
        const int turn = (k + 7) & ~(kBlk - 1);  // columns from here have the second scale
        alignas(16) OT o[8];
#pragma unroll
        for (int j = 0; j < 8; j += 2)
            store_pair(o + j, v[j] * (ALIGNED || k + j < turn ? s0 : s1), v[j + 1] * (ALIGNED || k + j + 1 < turn ? s0 : s1));
        if (k >= 0 && k + 8 <= K) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(OT) / 2; ++j)  // streaming: 21.1 -> 19.9 us at the sizes above
                __stcs(reinterpret_cast<uint4 *>(dst + k) + j, reinterpret_cast<const uint4 *>(o)[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j >= 0 && k + j < K) dst[k + j] = o[j];
        }
    }
}

// Gather of rows as they are held: one warp per row, two 4-byte loads to each 8-byte store. 16384 rows of 2304 in
// 13.7 us, 5.5 TB/s, part of them in L2; 65536 in 67 us, 4.5 TB/s, 0.68 of the copy rate: bound by its loads in flight.
__global__ void __launch_bounds__(256) take_rows_kernel(const uint8_t *__restrict__ q, int64_t q_pitch,
                                                        const uint8_t *__restrict__ s, int64_t s_pitch,
                                                        int64_t src_rows, int64_t K, unsigned nb,
                                                        const int64_t *__restrict__ rows, uint8_t *__restrict__ oq,
                                                        int64_t oq_pitch, uint8_t *__restrict__ os, int64_t os_pitch,
                                                        int64_t n, unsigned *err) {
    const int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    const int lane = threadIdx.x & 31;
    if (i >= n) return;
    const int64_t row = rows ? __ldg(rows + i) : i;
    if (row >= src_rows && lane == 0) atomicOr(err, kErrIndex);
    const bool have = row >= 0 && row < src_rows;
    for (int64_t k = 8 * lane; k < K; k += 256) {
        const uint8_t *src = q + row * q_pitch;
        const uint2 w = have ? make_uint2(load_word(src, k, K), load_word(src, k + 4, K)) : make_uint2(0u, 0u);
        store8(oq + i * oq_pitch, k, K, w);
    }
    for (unsigned b = lane; b < nb; b += 32) os[i * os_pitch + b] = have ? __ldg(s + row * s_pitch + b) : (uint8_t)0;
}

// One 128 x 128 tile of x per block, read once, for both orientations. Thread t of warp w holds rows
// 16w + 4(lane / 8) + 0..3 and columns 16(lane % 8) + 0..15, in the input's type: a row's 16 results are
// one 16-byte store, and four rows of a column make one word of the transpose, which goes through shared
// memory (16-byte chunks swizzled by the column) to be written by rows. The elements are looked at in
// pairs for the maxima; only a tile that holds an infinity or NaN looks at each of them.
// Bound by HBM for tiles (8192 x 16384 bf16 in 88.8 us, 6.0 TB/s) and by its instructions and four barriers a
// tile for row blocks both ways (105.5 us, 5.1 TB/s; with column sums 117 us; fp32 16384 x 16384 374 us,
// 4.3 TB/s). Held as 64 fp32 values a thread, one block fitted an SM and the same took 560 us.
template <typename XT, bool TILE>
__global__ void __launch_bounds__(256, sizeof(XT) == 4 ? 2 : TILE ? 4 : 3)
    quant_tile_kernel(const XT *__restrict__ x, int64_t R, int64_t C, int64_t sxm, int64_t sxk, bool vec, uint8_t *__restrict__ q,
                      int64_t q_pitch, uint8_t *__restrict__ qs, int64_t qs_pitch,
                      uint8_t *__restrict__ t, int64_t t_pitch, uint8_t *__restrict__ ts, int64_t ts_pitch,
                      float *__restrict__ sums) {
    using H = Held<XT>;
    constexpr int W = H::WORDS, PER = 16 / W;  // words of 16 elements, elements of a word
    __shared__ __align__(16) uint32_t trans[kBlk * 32];  // first the column sums of 32 groups of four rows
    float *scratch = reinterpret_cast<float *>(trans);
    __shared__ __align__(16) float col_inv[kBlk];
    __shared__ uint32_t col_max[8][kBlk / PER];
    __shared__ uint32_t warp_max[8];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7;
    const int64_t rb = blockIdx.y + (int64_t)gridDim.y * blockIdx.z, cb = blockIdx.x;
    if (rb * kBlk >= R) return;
    const int rl = 16 * warp + 4 * (lane >> 3);
    const int64_t r0 = rb * kBlk + rl, c0 = cb * kBlk + 16 * l;

    uint32_t v[4][W];
    if (vec && r0 + 4 <= R && c0 + 16 <= C) {
#pragma unroll
        for (int i = 0; i < 4; ++i) load16_aligned(x + (r0 + i) * sxm + c0, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            Fetched<XT> f[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) fetch16(x + (r0 + i + h) * sxm, c0, r0 + i + h < R ? C : 0, sxk, f[h]);
#pragma unroll
            for (int h = 0; h < 2; ++h) place16(f[h], v[i + h]);
        }
    }
    if (sums) {  // each thread's four rows; quad j of lane l at quad 4l + (j + l / 2) % 4, without bank conflicts
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
            float a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a[e] = (H::value(v[0], j + e) + H::value(v[1], j + e)) + (H::value(v[2], j + e) + H::value(v[3], j + e));
            *reinterpret_cast<float4 *>(&scratch[(rl >> 2) * kBlk + 16 * l + 4 * (((j >> 2) + (l >> 1)) & 3)]) =
                make_float4(a[0], a[1], a[2], a[3]);
        }
    }
    uint32_t rm[4];  // fp32 magnitude bits of each row's maximum
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t m = v[i][0] & H::ABS;
#pragma unroll
        for (int j = 1; j < W; ++j) m = H::umax(m, v[i][j] & H::ABS);
#pragma unroll
        for (int d = 4; d; d >>= 1) m = H::umax(m, __shfl_xor_sync(0xffffffffu, m, d));
        rm[i] = H::bits(m);
        odd |= rm[i] >= 0x7f800000u;
    }
    const bool not_finite = __syncthreads_or(odd);
    uint32_t cm[W];  // magnitudes of each column's maximum over this thread's rows
    if (not_finite) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < W; ++j) m = H::umax(m, H::finite(v[i][j]));
#pragma unroll
            for (int d = 4; d; d >>= 1) m = H::umax(m, __shfl_xor_sync(0xffffffffu, m, d));
            rm[i] = H::bits(m);
        }
#pragma unroll
        for (int j = 0; j < W; ++j) {
            cm[j] = H::umax(H::umax(H::finite(v[0][j]), H::finite(v[1][j])),
                            H::umax(H::finite(v[2][j]), H::finite(v[3][j])));
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i][j] = H::nan_for_inf(v[i][j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < W; ++j)
            cm[j] = H::umax(H::umax(v[0][j] & H::ABS, v[1][j] & H::ABS), H::umax(v[2][j] & H::ABS, v[3][j] & H::ABS));
    }
    if (TILE) {
        uint32_t m = max(max(rm[0], rm[1]), max(rm[2], rm[3]));
        m = __reduce_max_sync(0xffffffffu, m);
        if (lane == 0) warp_max[warp] = m;
    } else if (t) {
#pragma unroll
        for (int j = 0; j < W; ++j) {
            uint32_t m = H::umax(cm[j], __shfl_xor_sync(0xffffffffu, cm[j], 8));
            m = H::umax(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (lane < 8) col_max[warp][W * l + j] = m;
        }
    }
    __syncthreads();
    uint32_t tile_byte = 0;
    if (TILE) {
        uint32_t m = warp_max[0];
#pragma unroll
        for (int w = 1; w < 8; ++w) m = max(m, warp_max[w]);
        tile_byte = scale_byte(m);
    }
    if (threadIdx.x < kBlk) {
        const int c = threadIdx.x;
        const int64_t col = cb * kBlk + c;
        if (!TILE && t) {
            uint32_t m = col_max[0][c / PER];
#pragma unroll
            for (int w = 1; w < 8; ++w) m = H::umax(m, col_max[w][c / PER]);
            const uint32_t sb = scale_byte(H::bits(m, PER == 1 ? 0 : c & 1));
            col_inv[c] = inverse_scale(sb);
            if (col < C) ts[col * ts_pitch + rb] = (uint8_t)sb;
        }
        if (sums && col < C) {
            const int at = (c & ~15) + 4 * (((c >> 2) + (c >> 5)) & 3) + (c & 3);
            float a = 0.f;
#pragma unroll
            for (int g = 0; g < 32; ++g) a += scratch[g * kBlk + at];
            sums[rb * C + col] = a;
        }
    }
    if (TILE && threadIdx.x == 0) {
        if (q) qs[rb * qs_pitch + cb] = (uint8_t)tile_byte;
        if (t) ts[cb * ts_pitch + rb] = (uint8_t)tile_byte;
    }
    if (q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r0 + i >= R) break;
            const uint32_t sb = TILE ? tile_byte : scale_byte(rm[i]);
            store16(q + (r0 + i) * q_pitch, c0, C, pack16<XT>(v[i], inverse_scale(sb)));
            if (!TILE && l == 0) qs[(r0 + i) * qs_pitch + cb] = (uint8_t)sb;
        }
    }
    if (!t) return;
    if (!TILE || sums) __syncthreads();  // col_inv is written, scratch has been read
    const float tile_inv = inverse_scale(tile_byte);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int c = 16 * l + j;
        const float inv = TILE ? tile_inv : col_inv[c];
        trans[c * 32 + ((warp ^ l) << 2 | (lane >> 3))] =
            e4m3x2(H::value(v[0], j) * inv, H::value(v[1], j) * inv) |
            e4m3x2(H::value(v[2], j) * inv, H::value(v[3], j) * inv) << 16;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = 32 * i + 4 * warp + (lane >> 3);
        if (cb * kBlk + c >= C) break;
        const uint4 w = *reinterpret_cast<const uint4 *>(&trans[c * 32 + ((l ^ (c >> 4)) << 2)]);
        store16(t + (cb * kBlk + c) * t_pitch, rb * kBlk + 16 * l, R, w);
    }
}

// col_sums[c] = the partial sums of the row blocks: 32 columns a block, eight ranges of row blocks summed in
// order, then the ranges in order.
__global__ void __launch_bounds__(256) join_sums_kernel(const float *__restrict__ part, int64_t nrb, int64_t C,
                                                        float *__restrict__ out) {
    __shared__ float range[8][32];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane, each = (nrb + 7) / 8;
    float a = 0.f;
    if (c < C) {
#pragma unroll 8
        for (int64_t r = w * each; r < min(nrb, (w + 1) * each); ++r) a += __ldg(part + r * C + c);
    }
    range[w][lane] = a;
    __syncthreads();
    if (w == 0 && c < C) {
        a = range[0][lane];
#pragma unroll
        for (int i = 1; i < 8; ++i) a += range[i][lane];
        out[c] = a;
    }
}

bool aligned_to(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

template <typename F>
int with_type(int dtype, F f) {
    if (dtype == SF_F32) return f(float{});
    if (dtype == SF_BF16) return f(__nv_bfloat16{});
    return f(__half{});
}

int check_strided(const sf_matrix *m, const char *name) {
    if (!m) return set_error(SF_ERR_INVALID, "%s is NULL", name);
    if (!valid_dtype(m->dtype)) return set_error(SF_ERR_INVALID, "%s has unsupported dtype code %d", name, m->dtype);
    if (m->rows < 0 || m->cols < 0) return set_error(SF_ERR_INVALID, "%s has a negative extent", name);
    if (m->rows > 0 && m->cols > 0 && !m->data) return set_error(SF_ERR_INVALID, "%s has a NULL data pointer", name);
    return SF_OK;
}

// 16-byte loads or stores of rows: unit column stride, aligned base and pitch.
bool vector_rows(const sf_matrix &m) {
    return m.stride_col == 1 && aligned_to(m.data, 16) && (m.stride_row * (int64_t)dtype_size(m.dtype)) % 16 == 0;
}

// Threads of 256-wide blocks for `items` groups of `width` threads; 0 and an error where it is too many.
int grid_for(uint64_t items, int width, unsigned *grid) {
    const uint64_t blocks = (items * (uint64_t)width + 255) / 256;
    if (blocks > 0x7fffffffull) return set_error(SF_ERR_UNSUPPORTED, "too many rows for one call");
    *grid = (unsigned)blocks;
    return SF_OK;
}

}  // namespace

int check_blocks(const sf_blocks *b, const char *name) {
    if (!b) return set_error(SF_ERR_INVALID, "%s is NULL", name);
    if (b->rows < 0 || b->cols < 0) return set_error(SF_ERR_INVALID, "%s has a negative extent", name);
    if (b->tile != 0 && b->tile != 1) return set_error(SF_ERR_INVALID, "%s: tile must be 0 or 1", name);
    if (b->rows == 0 || b->cols == 0) return SF_OK;
    if (!b->data || !b->scales) return set_error(SF_ERR_INVALID, "%s has a NULL pointer", name);
    if (!aligned_to(b->data, 16) || b->data_pitch % 16 || b->data_pitch < b->cols)
        return set_error(SF_ERR_INVALID, "%s: data needs a 16-byte aligned base and a row pitch that is a multiple of "
                         "16 bytes and covers a row (pitch %lld, %lld columns)", name, (long long)b->data_pitch,
                         (long long)b->cols);
    if (!aligned_to(b->scales, 4) || b->scale_pitch % 4 || b->scale_pitch < (b->cols + kBlk - 1) / kBlk)
        return set_error(SF_ERR_INVALID, "%s: scales need a 4-byte aligned base and a row pitch that is a multiple of "
                         "4 bytes and covers a row (pitch %lld)", name, (long long)b->scale_pitch);
    return SF_OK;
}

}  // namespace sf

using namespace sf;

extern "C" {

int sf_blocks_write(const sf_matrix *x, const int64_t *slots, const sf_blocks *dst, sf_stream stream) {
    int st = check_strided(x, "x");
    if (st) return st;
    if ((st = check_blocks(dst, "dst"))) return st;
    if (dst->tile) return set_error(SF_ERR_INVALID, "dst must be in row blocks");
    if (x->cols != dst->cols)
        return set_error(SF_ERR_INVALID, "x has %lld columns but the store has %lld", (long long)x->cols,
                         (long long)dst->cols);
    if (!slots && x->rows > dst->rows) return set_error(SF_ERR_INVALID, "x has more rows than dst");
    if (x->rows == 0 || x->cols == 0) return SF_OK;
    const Divisor by = Divisor::of((x->cols + 2 * kBlk - 1) / (2 * kBlk));
    unsigned grid = 0;
    if ((st = grid_for((uint64_t)x->rows * by.d, 8, &grid))) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_type(x->dtype, [&](auto tag) {
        using T = decltype(tag);
        quant_rows_kernel<T><<<grid, 256, 0, s>>>(
            reinterpret_cast<const T *>(x->data), x->rows, x->cols, x->stride_row, x->stride_col, vector_rows(*x),
            slots, static_cast<uint8_t *>(dst->data), dst->data_pitch, static_cast<uint8_t *>(dst->scales), dst->scale_pitch,
            dst->rows, by, device_error_word());
        return check_cuda(cudaGetLastError(), "quant_rows launch");
    });
}

int sf_blocks_read(const sf_blocks *src, const int64_t *rows, const sf_matrix *out, sf_stream stream) {
    int st = check_blocks(src, "src");
    if (st) return st;
    if ((st = check_strided(out, "out"))) return st;
    if (out->cols != src->cols) return set_error(SF_ERR_INVALID, "out and src differ in columns");
    if (!rows && out->rows > src->rows) return set_error(SF_ERR_INVALID, "out has more rows than src");
    if (out->rows == 0 || out->cols == 0) return SF_OK;
    if (out->cols > 1 && out->stride_col != 1) return set_error(SF_ERR_UNSUPPORTED, "out needs a unit column stride");
    if (out->cols > INT32_MAX - 4096) return set_error(SF_ERR_UNSUPPORTED, "too many columns");
    const bool aligned = vector_rows(*out);
    // a row's pieces of eight, one more where rows start between boundaries
    const int64_t pieces = (out->cols + 7) / 8 + (aligned ? 0 : 1);
    const int64_t each = out->dtype == SF_F32 ? kReadElements<float> : kReadElements<__half>;  // 8 lanes, 8 a piece
    const Divisor by = Divisor::of((pieces + each - 1) / each);
    unsigned grid = 0;
    if ((st = grid_for((uint64_t)out->rows * by.d, 8, &grid))) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_type(out->dtype, [&](auto tag) {
        using T = decltype(tag);
        auto kern = aligned ? read_rows_kernel<T, true> : read_rows_kernel<T, false>;
        kern<<<grid, 256, 0, s>>>(
            static_cast<const uint8_t *>(src->data), src->data_pitch, static_cast<const uint8_t *>(src->scales),
            src->scale_pitch, src->rows, (int)src->cols, src->tile ? 7 : 0, rows,
            reinterpret_cast<T *>(const_cast<void *>(out->data)), out->rows, out->stride_row, by, device_error_word());
        return check_cuda(cudaGetLastError(), "read_rows launch");
    });
}

int sf_blocks_take(const sf_blocks *src, const int64_t *rows, const sf_blocks *dst, sf_stream stream) {
    int st = check_blocks(src, "src");
    if (st) return st;
    if ((st = check_blocks(dst, "dst"))) return st;
    if (src->tile || dst->tile) return set_error(SF_ERR_INVALID, "src and dst must be in row blocks");
    if (dst->cols != src->cols) return set_error(SF_ERR_INVALID, "dst and src differ in columns");
    if (!rows && dst->rows > src->rows) return set_error(SF_ERR_INVALID, "dst has more rows than src");
    if (dst->rows == 0 || dst->cols == 0) return SF_OK;
    const unsigned nb = (unsigned)((src->cols + kBlk - 1) / kBlk);
    unsigned grid = 0;
    if ((st = grid_for((uint64_t)dst->rows, 32, &grid))) return st;
    take_rows_kernel<<<grid, 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t *>(src->data), src->data_pitch, static_cast<const uint8_t *>(src->scales),
        src->scale_pitch, src->rows, src->cols, nb, rows, static_cast<uint8_t *>(dst->data), dst->data_pitch,
        static_cast<uint8_t *>(dst->scales), dst->scale_pitch, dst->rows, device_error_word());
    return check_cuda(cudaGetLastError(), "take_rows launch");
}

int sf_blocks_quantize_workspace(const sf_matrix *x, int col_sums, size_t *bytes) {
    const int st = check_strided(x, "x");
    if (st) return st;
    if (!bytes) return set_error(SF_ERR_INVALID, "bytes is NULL");
    *bytes = col_sums ? (size_t)((x->rows + kBlk - 1) / kBlk) * (size_t)x->cols * sizeof(float) : 0;
    return SF_OK;
}

int sf_blocks_quantize(const sf_matrix *x, const sf_blocks *q, const sf_blocks *qt, float *col_sums, void *workspace,
                       size_t workspace_bytes, sf_stream stream) {
    int st = check_strided(x, "x");
    if (st) return st;
    if (!q && !qt) return set_error(SF_ERR_INVALID, "q and qt are both NULL");
    if (q && (st = check_blocks(q, "q"))) return st;
    if (qt && (st = check_blocks(qt, "qt"))) return st;
    if (q && (q->rows != x->rows || q->cols != x->cols)) return set_error(SF_ERR_INVALID, "q must have x's shape");
    if (qt && (qt->rows != x->cols || qt->cols != x->rows))
        return set_error(SF_ERR_INVALID, "qt must have the shape of x's transpose");
    if (q && qt && q->tile != qt->tile)
        return set_error(SF_ERR_INVALID, "q and qt must both be in row blocks or both in tiles");
    size_t need = 0;
    if ((st = sf_blocks_quantize_workspace(x, col_sums != nullptr, &need))) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (x->rows == 0 || x->cols == 0) {
        if (col_sums && x->cols > 0)
            return check_cuda(cudaMemsetAsync(col_sums, 0, (size_t)x->cols * sizeof(float), s), "column sums");
        return SF_OK;
    }
    if (need && (!workspace || workspace_bytes < need))
        return set_error(SF_ERR_WORKSPACE, "workspace of %zu bytes needed", need);
    const int64_t nrb = (x->rows + kBlk - 1) / kBlk, ncb = (x->cols + kBlk - 1) / kBlk;
    // row blocks along y and z, at most 65535 either way; blocks past the last leave at once
    const int64_t ny = std::min<int64_t>(nrb, 32768), nz = (nrb + ny - 1) / ny;
    if (nz > 65535 || ncb > INT32_MAX) return set_error(SF_ERR_UNSUPPORTED, "too many rows or columns for one call");
    const bool tile = (q ? q : qt)->tile != 0;
    float *part = col_sums ? static_cast<float *>(workspace) : nullptr;
    const sf_blocks none = {};
    const sf_blocks a = q ? *q : none, b = qt ? *qt : none;
    st = with_type(x->dtype, [&](auto tag) {
        using T = decltype(tag);
        auto kern = tile ? quant_tile_kernel<T, true> : quant_tile_kernel<T, false>;
        kern<<<dim3((unsigned)ncb, (unsigned)ny, (unsigned)nz), 256, 0, s>>>(
            reinterpret_cast<const T *>(x->data), x->rows, x->cols, x->stride_row, x->stride_col, vector_rows(*x),
            static_cast<uint8_t *>(a.data), a.data_pitch, static_cast<uint8_t *>(a.scales), a.scale_pitch,
            static_cast<uint8_t *>(b.data), b.data_pitch, static_cast<uint8_t *>(b.scales), b.scale_pitch, part);
        return check_cuda(cudaGetLastError(), "quant_tile launch");
    });
    if (st || !col_sums) return st;
    join_sums_kernel<<<(unsigned)((x->cols + 31) / 32), 256, 0, s>>>(part, nrb, x->cols, col_sums);
    return check_cuda(cudaGetLastError(), "join_sums launch");
}

}  // extern "C"

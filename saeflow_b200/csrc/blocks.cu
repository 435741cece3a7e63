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

#include "sf_common.cuh"
#include "sf_internal.h"

namespace sf {

namespace {

constexpr int kBlk = SF_BLOCK;

// Magnitude bits of v where v is finite, else 0: ordered as integers like the magnitudes.
__device__ __forceinline__ uint32_t finite_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    const int s = (int)((amax_bits + 0x1FFFFFu) >> 23) - 8;
    return (uint32_t)max(s, 0);
}
// 2^(127 - s) for s <= 247 (scale_byte's range), and 2^(s - 127), a subnormal for s = 0.
__device__ __forceinline__ float inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }
__device__ __forceinline__ float scale_value(uint32_t s) { return __uint_as_float(s ? s << 23 : 0x00400000u); }

// Four fp32 -> four e4m3 in one word. The conversion saturates, which in-range quotients never
// meet; an infinity would become 448, so non-finite elements go in as NaN.
__device__ __forceinline__ uint32_t pack_e4m3(const float *v, float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float2 f;
        f.x = v[2 * h] * inv;
        f.y = v[2 * h + 1] * inv;
        if ((__float_as_uint(v[2 * h]) & 0x7f800000u) == 0x7f800000u) f.x = __int_as_float(0x7fffffff);
        if ((__float_as_uint(v[2 * h + 1]) & 0x7f800000u) == 0x7f800000u) f.y = __int_as_float(0x7fffffff);
        w |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (16 * h);
    }
    return w;
}
__device__ __forceinline__ void unpack_e4m3(uint32_t w, float *v) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * h)), __NV_E4M3);
        const float2 f = __half22float2(__half2(r));
        v[2 * h] = f.x;
        v[2 * h + 1] = f.y;
    }
}

// Eight consecutive elements from column k of a row, zeros past K.
template <typename XT>
__device__ __forceinline__ void load8(const XT *row, int64_t k, int64_t K, int64_t sxk, bool vec, float (&v)[8]) {
    if (vec && k + 8 <= K) {
        uint4 q[sizeof(XT) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(XT) / 2; ++i) q[i] = __ldg(reinterpret_cast<const uint4 *>(row + k) + i);
        const XT *e = reinterpret_cast<const XT *>(q);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = to_f32(e[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = k + j < K ? to_f32(__ldg(row + (k + j) * sxk)) : 0.f;
    }
}

// Eight e4m3 bytes from column k of a row of K columns; nothing past them is read.
__device__ __forceinline__ uint2 load8_e4m3(const uint8_t *row, int64_t k, int64_t K) {
    if (k + 8 <= K) return __ldg(reinterpret_cast<const uint2 *>(row + k));
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k + j < K) w[j >> 2] |= (uint32_t)__ldg(row + k + j) << (8 * (j & 3));
    return make_uint2(w[0], w[1]);
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

// Row blocks: eight lanes to a block of 128, each with columns 8l..8l+7 and 64+8l..64+8l+7, so that
// every load and store of the group is one contiguous run.
template <typename XT>
__global__ void __launch_bounds__(256) quant_rows_kernel(const XT *__restrict__ x, int64_t n, int64_t K, int64_t sxm,
                                                         int64_t sxk, bool vec, const int64_t *__restrict__ slots,
                                                         uint8_t *__restrict__ q, int64_t q_pitch,
                                                         uint8_t *__restrict__ s, int64_t s_pitch, int64_t cap,
                                                         unsigned nb, unsigned *err) {
    const int l = threadIdx.x & 7;
    const uint64_t item = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    if (item >= (uint64_t)n * nb) return;  // whole groups leave together
    const unsigned group = 0xffu << (threadIdx.x & 24);
    const int64_t row = (int64_t)(item / nb);
    const unsigned blk = (unsigned)(item - (uint64_t)row * nb);
    int64_t slot = row;
    if (slots) {
        slot = __ldg(slots + row);
        if (slot >= cap && l == 0 && blk == 0) atomicOr(err, kErrIndex);
        if (slot < 0 || slot >= cap) return;
    }
    const int64_t k0 = (int64_t)blk * kBlk + 8 * l;
    float a[8], b[8];
    load8(x + row * sxm, k0, K, sxk, vec, a);
    load8(x + row * sxm, k0 + 64, K, sxk, vec, b);
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, max(finite_bits(a[j]), finite_bits(b[j])));
#pragma unroll
    for (int d = 4; d; d >>= 1) m = max(m, __shfl_xor_sync(group, m, d));
    const uint32_t sb = scale_byte(m);
    const float inv = inverse_scale(sb);
    uint8_t *dst = q + slot * q_pitch;
    store8(dst, k0, K, make_uint2(pack_e4m3(a, inv), pack_e4m3(a + 4, inv)));
    store8(dst, k0 + 64, K, make_uint2(pack_e4m3(b, inv), pack_e4m3(b + 4, inv)));
    if (l == 0) s[slot * s_pitch + blk] = (uint8_t)sb;
}

// Dequantising gather: the same lanes as above; `tile_shift` is 7 where a scale row serves 128 rows.
template <typename OT>
__global__ void __launch_bounds__(256) read_rows_kernel(const uint8_t *__restrict__ q, int64_t q_pitch,
                                                        const uint8_t *__restrict__ s, int64_t s_pitch,
                                                        int64_t src_rows, int64_t K, int tile_shift,
                                                        const int64_t *__restrict__ rows, OT *__restrict__ out,
                                                        int64_t n, int64_t out_pitch, bool vec, unsigned nb,
                                                        unsigned *err) {
    const int l = threadIdx.x & 7;
    const uint64_t item = ((uint64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    if (item >= (uint64_t)n * nb) return;
    const int64_t i = (int64_t)(item / nb);
    const unsigned blk = (unsigned)(item - (uint64_t)i * nb);
    int64_t row = i;
    if (rows) {
        row = __ldg(rows + i);
        if (row >= src_rows && l == 0 && blk == 0) atomicOr(err, kErrIndex);
    }
    const bool have = row >= 0 && row < src_rows;
    const float scale = have ? scale_value(__ldg(s + (row >> tile_shift) * s_pitch + blk)) : 0.f;
    OT *dst = out + i * out_pitch;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int64_t k = (int64_t)blk * kBlk + 64 * h + 8 * l;
        if (k >= K) break;
        const uint2 w = have ? load8_e4m3(q + row * q_pitch, k, K) : make_uint2(0u, 0u);
        float v[8];
        unpack_e4m3(w.x, v);
        unpack_e4m3(w.y, v + 4);
        OT o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = from_f32<OT>(have ? v[j] * scale : 0.f);
        if (vec && k + 8 <= K) {
            const uint4 *src = reinterpret_cast<const uint4 *>(o);
#pragma unroll
            for (int j = 0; j < (int)sizeof(OT) / 2; ++j) reinterpret_cast<uint4 *>(dst + k)[j] = src[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < K) dst[k + j] = o[j];
        }
    }
}

// Gather of rows as they are held: one warp per row.
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
        const uint2 w = have ? load8_e4m3(q + row * q_pitch, k, K) : make_uint2(0u, 0u);
        store8(oq + i * oq_pitch, k, K, w);
    }
    for (unsigned b = lane; b < nb; b += 32) os[i * os_pitch + b] = have ? __ldg(s + row * s_pitch + b) : (uint8_t)0;
}

// One 128 x 128 tile of x per block, read once, for both orientations. Thread t of warp w holds rows
// 16w + 4(lane / 8) + 0..3 and columns 8(lane % 8) + 0..7 (and + 64): four rows of a column make one
// word of the transpose, which goes through shared memory (pitch 33 words) to be written by rows.
template <typename XT, bool TILE>
__global__ void __launch_bounds__(256) quant_tile_kernel(const XT *__restrict__ x, int64_t R, int64_t C, int64_t sxm,
                                                         int64_t sxk, bool vec, uint8_t *__restrict__ q,
                                                         int64_t q_pitch, uint8_t *__restrict__ qs, int64_t qs_pitch,
                                                         uint8_t *__restrict__ t, int64_t t_pitch,
                                                         uint8_t *__restrict__ ts, int64_t ts_pitch,
                                                         float *__restrict__ sums) {
    __shared__ uint32_t trans[kBlk * 33];
    __shared__ uint32_t col_max[kBlk];
    __shared__ float col_sum[8][kBlk];
    __shared__ uint32_t tile_max;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane & 7;
    const int64_t rb = blockIdx.y, cb = blockIdx.x;
    const int rl = 16 * warp + 4 * (lane >> 3);
    const int64_t r0 = rb * kBlk + rl, c0 = cb * kBlk + 8 * l;
    if (threadIdx.x < kBlk) col_max[threadIdx.x] = 0;
    if (threadIdx.x == 0) tile_max = 0;
    __syncthreads();
    float v[4][16];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float(&lo)[8] = *reinterpret_cast<float(*)[8]>(&v[i][0]);
        float(&hi)[8] = *reinterpret_cast<float(*)[8]>(&v[i][8]);
        if (r0 + i < R) {
            load8(x + (r0 + i) * sxm, c0, C, sxk, vec, lo);
            load8(x + (r0 + i) * sxm, c0 + 64, C, sxk, vec, hi);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[i][j] = 0.f;
        }
    }
    uint32_t rm[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        rm[i] = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j) rm[i] = max(rm[i], finite_bits(v[i][j]));
#pragma unroll
        for (int d = 4; d; d >>= 1) rm[i] = max(rm[i], __shfl_xor_sync(0xffffffffu, rm[i], d));
    }
    if (TILE) {
        if (l == 0) atomicMax(&tile_max, max(max(rm[0], rm[1]), max(rm[2], rm[3])));
    } else if (t) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            uint32_t m = max(max(finite_bits(v[0][j]), finite_bits(v[1][j])),
                             max(finite_bits(v[2][j]), finite_bits(v[3][j])));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = max(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (lane < 8) atomicMax(&col_max[8 * l + (j & 7) + 64 * (j >> 3)], m);
        }
    }
    if (sums) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            float a = (v[0][j] + v[1][j]) + (v[2][j] + v[3][j]);
            a += __shfl_xor_sync(0xffffffffu, a, 8);
            a += __shfl_xor_sync(0xffffffffu, a, 16);
            if (lane < 8) col_sum[warp][8 * l + (j & 7) + 64 * (j >> 3)] = a;
        }
    }
    __syncthreads();
    if (q) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (r0 + i >= R) break;
            const uint32_t sb = scale_byte(TILE ? tile_max : rm[i]);
            const float inv = inverse_scale(sb);
            uint8_t *dst = q + (r0 + i) * q_pitch;
            store8(dst, c0, C, make_uint2(pack_e4m3(&v[i][0], inv), pack_e4m3(&v[i][4], inv)));
            store8(dst, c0 + 64, C, make_uint2(pack_e4m3(&v[i][8], inv), pack_e4m3(&v[i][12], inv)));
            if (!TILE && l == 0) qs[(r0 + i) * qs_pitch + cb] = (uint8_t)sb;
        }
        if (TILE && threadIdx.x == 0) qs[rb * qs_pitch + cb] = (uint8_t)scale_byte(tile_max);
    }
    if (sums && threadIdx.x < kBlk && cb * kBlk + threadIdx.x < C) {
        float a = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) a += col_sum[w][threadIdx.x];
        sums[rb * C + cb * kBlk + threadIdx.x] = a;
    }
    if (!t) return;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int c = 8 * l + (j & 7) + 64 * (j >> 3);
        const float inv = inverse_scale(scale_byte(TILE ? tile_max : col_max[c]));
        const float col[4] = {v[0][j], v[1][j], v[2][j], v[3][j]};
        trans[c * 33 + (rl >> 2)] = pack_e4m3(col, inv);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = 32 * i + 4 * warp + (lane >> 3);
        if (cb * kBlk + c >= C) break;
        const uint32_t *src = &trans[c * 33 + 4 * l];
        uint8_t *dst = t + (cb * kBlk + c) * t_pitch;
        store8(dst, rb * kBlk + 16 * l, R, make_uint2(src[0], src[1]));
        store8(dst, rb * kBlk + 16 * l + 8, R, make_uint2(src[2], src[3]));
        if (!TILE && l == 0) ts[(cb * kBlk + c) * ts_pitch + rb] = (uint8_t)scale_byte(col_max[c]);
    }
    if (TILE && threadIdx.x == 0) ts[cb * ts_pitch + rb] = (uint8_t)scale_byte(tile_max);
}

// col_sums[c] = the partial sums of the row blocks, in order.
__global__ void __launch_bounds__(256) join_sums_kernel(const float *__restrict__ part, int64_t nrb, int64_t C,
                                                        float *__restrict__ out) {
    const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= C) return;
    float a = 0.f;
#pragma unroll 8
    for (int64_t r = 0; r < nrb; ++r) a += __ldg(part + r * C + c);
    out[c] = a;
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
    const unsigned nb = (unsigned)((x->cols + kBlk - 1) / kBlk);
    unsigned grid = 0;
    if ((st = grid_for((uint64_t)x->rows * nb, 8, &grid))) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_type(x->dtype, [&](auto tag) {
        using T = decltype(tag);
        quant_rows_kernel<T><<<grid, 256, 0, s>>>(
            reinterpret_cast<const T *>(x->data), x->rows, x->cols, x->stride_row, x->stride_col, vector_rows(*x),
            slots, static_cast<uint8_t *>(dst->data), dst->data_pitch, static_cast<uint8_t *>(dst->scales),
            dst->scale_pitch, dst->rows, nb, device_error_word());
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
    if (out->stride_col != 1) return set_error(SF_ERR_UNSUPPORTED, "out needs a unit column stride");
    const unsigned nb = (unsigned)((src->cols + kBlk - 1) / kBlk);
    unsigned grid = 0;
    if ((st = grid_for((uint64_t)out->rows * nb, 8, &grid))) return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_type(out->dtype, [&](auto tag) {
        using T = decltype(tag);
        read_rows_kernel<T><<<grid, 256, 0, s>>>(
            static_cast<const uint8_t *>(src->data), src->data_pitch, static_cast<const uint8_t *>(src->scales),
            src->scale_pitch, src->rows, src->cols, src->tile ? 7 : 0, rows,
            reinterpret_cast<T *>(const_cast<void *>(out->data)), out->rows, out->stride_row, vector_rows(*out), nb,
            device_error_word());
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
    if (nrb > 65535) return set_error(SF_ERR_UNSUPPORTED, "too many rows for one call");
    const bool tile = (q ? q : qt)->tile != 0;
    float *part = col_sums ? static_cast<float *>(workspace) : nullptr;
    const sf_blocks none = {};
    const sf_blocks a = q ? *q : none, b = qt ? *qt : none;
    st = with_type(x->dtype, [&](auto tag) {
        using T = decltype(tag);
        auto kern = tile ? quant_tile_kernel<T, true> : quant_tile_kernel<T, false>;
        kern<<<dim3((unsigned)ncb, (unsigned)nrb), 256, 0, s>>>(
            reinterpret_cast<const T *>(x->data), x->rows, x->cols, x->stride_row, x->stride_col, vector_rows(*x),
            static_cast<uint8_t *>(a.data), a.data_pitch, static_cast<uint8_t *>(a.scales), a.scale_pitch,
            static_cast<uint8_t *>(b.data), b.data_pitch, static_cast<uint8_t *>(b.scales), b.scale_pitch, part);
        return check_cuda(cudaGetLastError(), "quant_tile launch");
    });
    if (st || !col_sums) return st;
    join_sums_kernel<<<(unsigned)((x->cols + 255) / 256), 256, 0, s>>>(part, nrb, x->cols, col_sums);
    return check_cuda(cudaGetLastError(), "join_sums launch");
}

}  // extern "C"

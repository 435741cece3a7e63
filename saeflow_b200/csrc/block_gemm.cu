// Product of two block-scaled 8-bit matrices on the 5th-generation tensor cores, sm_100a.
//
//   out[m, n] = act(sum_k a[m, k] 2^(sa - 127) b[n, k] 2^(sb - 127) + bias[n])
//
// tcgen05.mma kind::mxf8f6f4 multiplies each 32 elements of K by one power-of-two scale per row of
// either operand before they enter the fp32 accumulator in TMEM. A block here spans 128 elements of K,
// so its byte serves four instructions, and one 32-bit word of a row's scale bytes serves 512 elements:
// the instruction descriptor says which byte of the word applies. Tiles (one scale per 128 x 128) are
// the same words read once per 128 rows.
//
// Persistent kernel, one CTA per SM, 128 x 128 tiles, 224 threads:
//   warp 0      TMA producer: 128 rows x 128 bytes of a and of b per stage, SWIZZLE_128B, mbarrier ring
//   warp 1      TMEM allocator and MMA issuer; two accumulators of 128 columns
//   warps 2-5   epilogue: bias, activation, rounding, stores
//   warp 6      scale words of both operands for 512 elements of K into shared memory, in the order that
//               tcgen05.cp spreads over TMEM (row r at byte 16 (r % 32) + 4 (r / 32))
#include <algorithm>

#include "sf_common.cuh"
#include "sf_internal.h"

namespace sf {

namespace {

constexpr int kTile = 128;
constexpr int kKBytes = 128;                  // elements (bytes) of K per stage
constexpr int kStages = 6;
constexpr int kScaleSlots = 4;                // scale words of 512 elements of K each
constexpr int kThreads = 224;
constexpr int kTileBytes = kTile * kKBytes;   // one operand of one stage
constexpr int kTmemCols = 512;
constexpr int kScaleCol = 256;                // TMEM columns of the scales, behind the accumulators

struct GemmParams {
    int M, N, nkb;
    int m_tiles, n_tiles;
    int group_m;  // m-tiles that run side by side over each n-tile
    const uint8_t *a_scales, *b_scales;
    int64_t a_scale_pitch, b_scale_pitch;
    int a_shift, b_shift;  // log2 of the rows a scale row serves: 0 row blocks, 7 tiles
    const float *bias, *thr;
    int activation;  // enum sf_activation, -1 none
    void *out;
    int64_t out_pitch;
    int out_vec;
    unsigned *err;
};

struct __align__(16) Shared {
    uint64_t full[kStages], empty[kStages];
    uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
    uint64_t tmem_full[2], tmem_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float bias[2][kTile];
    alignas(16) float thr[2][kTile];
};

__device__ __forceinline__ void tile_coords(const GemmParams &p, int u, int &m_blk, int &n_blk) {
    const int per_group = p.group_m * p.n_tiles;
    const int g = u / per_group;
    const int first = g * p.group_m;
    const int gm = min(p.m_tiles - first, p.group_m);
    const int local = u - g * per_group;
    m_blk = first + local % gm;
    n_blk = local / gm;
}

// The scale words of 128 rows from `first` for K blocks 4 g .. 4 g + 3: lane i gets rows i, 32 + i, 64 + i,
// 96 + i. Rows past the end take the last row's: their products are of zeros.
__device__ __forceinline__ uint4 scale_words(const uint8_t *s, int64_t pitch, int shift, int first, int rows, int g,
                                             int lane) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t r = min(first + 32 * i + lane, rows - 1) >> shift;
        w[i] = __ldg(reinterpret_cast<const uint32_t *>(s + r * pitch) + g);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ float activate(float v, float t, int activation) {
    if (activation == SF_ACT_RELU) return v < 0.f ? 0.f : v;  // fmaxf would turn a NaN into 0
    if (activation == SF_ACT_JUMPRELU) return v > t && v > 0.f ? v : 0.f;
    return v;
}

template <typename OT>
__device__ __forceinline__ void store_chunk(const GemmParams &p, const float (&v)[32], int row, int col0,
                                            uint64_t policy) {
    if (row >= p.M) return;
    OT *dst = reinterpret_cast<OT *>(p.out) + (int64_t)row * p.out_pitch + col0;
    if (p.out_vec && col0 + 32 <= p.N) {
        alignas(16) OT o[32];
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = from_f32<OT>(v[j]);
        const uint4 *src = reinterpret_cast<const uint4 *>(o);
#pragma unroll
        for (int j = 0; j < (int)(2 * sizeof(OT)); ++j)
            st_global_v4_hint(reinterpret_cast<uint4 *>(dst) + j, src[j], policy);
    } else {
#pragma unroll
        for (int j = 0; j < 32; ++j)
            if (col0 + j < p.N) dst[j] = from_f32<OT>(v[j]);
    }
}

template <typename OT>
__global__ void __launch_bounds__(kThreads, 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                      const GemmParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sA = smem;
    uint8_t *sB = sA + kStages * kTileBytes;
    uint8_t *sScale = sB + kStages * kTileBytes;  // per slot: 512 bytes of a's words, 512 of b's
    Shared *sh = reinterpret_cast<Shared *>(sScale + kScaleSlots * 1024);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int units = p.m_tiles * p.n_tiles;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh->full[s], 1);
            mbar_init(&sh->empty[s], 1);
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(&sh->scale_full[s], 1);
            mbar_init(&sh->scale_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh->tmem_full[b], 1);
            mbar_init(&sh->tmem_empty[b], 4);
        }
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
    }
    if (warp == 1) {
        tmem_alloc(&sh->tmem_base, kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    volatile int *abort_flag = &sh->abort_flag;
    auto wait = [&](uint64_t *bar, uint32_t parity) { return mbar_wait(bar, parity, abort_flag, p.err); };

    if (warp == 0) {
        if (lane == 0) {
            const uint64_t pol_a = l2_policy_evict_last(), pol_b = l2_policy_evict_normal();
            int stage = 0;
            uint32_t phase = 0, armed = 0, armed_parity = 0;
            bool ok = true;
            for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
                int m_blk, n_blk;
                tile_coords(p, u, m_blk, n_blk);
                for (int kb = 0; kb < p.nkb; ++kb) {
                    if (!(ok = wait(&sh->empty[stage], phase ^ 1u))) break;
                    mbar_arrive_expect_tx(&sh->full[stage], 2 * kTileBytes);
                    armed |= 1u << stage;
                    armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                    tma_load_2d(sA + stage * kTileBytes, &tmA, &sh->full[stage], kb * kKBytes, m_blk * kTile, pol_a);
                    tma_load_2d(sB + stage * kTileBytes, &tmB, &sh->full[stage], kb * kKBytes, n_blk * kTile, pol_b);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (*abort_flag)  // copies in flight must land before the CTA leaves
                for (int s = 0; s < kStages; ++s)
                    if (armed & (1u << s)) mbar_wait_drain(&sh->full[s], (armed_parity >> s) & 1u, p.err);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, slot = 0, acc = 0;
            uint32_t phase = 0, slot_phase = 0, acc_phase = 0;
            bool ok = true;
            for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
                if (!(ok = wait(&sh->tmem_empty[acc], acc_phase ^ 1u))) break;
                tc_fence_after();
                const uint32_t d = tmem + acc * kTile;
                uint32_t scales = 0;
                for (int kb = 0; kb < p.nkb; ++kb) {
                    if ((kb & 3) == 0) {
                        if (!(ok = wait(&sh->scale_full[slot], slot_phase))) break;
                        tc_fence_after();
                        // Slot by slot: a slot's TMEM columns are written again four slots (16 stages)
                        // later, when the stages that read them have long been released.
                        scales = tmem + kScaleCol + slot * 8;
                        const uint32_t src = smem_u32(sScale + slot * 1024);
                        tmem_copy_32x128b(scales, smem_desc_rows16(src));
                        tmem_copy_32x128b(scales + 4, smem_desc_rows16(src + 512));
                        umma_commit(&sh->scale_empty[slot]);
                        if (++slot == kScaleSlots) {
                            slot = 0;
                            slot_phase ^= 1u;
                        }
                    }
                    if (!(ok = wait(&sh->full[stage], phase))) break;
                    tc_fence_after();
                    const uint32_t a = smem_u32(sA + stage * kTileBytes), b = smem_u32(sB + stage * kTileBytes);
                    const uint32_t idesc = make_idesc_e4m3_scaled(kTile, kTile, kb & 3);
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        umma_e4m3_scaled(d, smem_desc_sw128(a + ks * 32, 16, 1024),
                                         smem_desc_sw128(b + ks * 32, 16, 1024), idesc, scales, scales + 4,
                                         (kb | ks) ? 1u : 0u);
                    umma_commit(&sh->empty[stage]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                umma_commit(&sh->tmem_full[acc]);
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            umma_commit(&sh->drain);
            mbar_wait_drain(&sh->drain, 0, p.err);
        }
    } else if (warp < 6) {
        const int et = threadIdx.x - 64;
        const int quad = warp & 3;
        const uint64_t pol = l2_policy_evict_first();
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int u = blockIdx.x; u < units; u += gridDim.x) {
            int m_blk, n_blk;
            tile_coords(p, u, m_blk, n_blk);
            const int col = n_blk * kTile + et;
            sh->bias[acc][et] = p.bias && col < p.N ? __ldg(p.bias + col) : 0.f;
            sh->thr[acc][et] = p.thr && col < p.N ? __ldg(p.thr + col) : 0.f;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            if (!wait(&sh->tmem_full[acc], acc_phase)) break;
            tc_fence_after();
            const int row = m_blk * kTile + quad * 32 + lane;
#pragma unroll 1
            for (int c = 0; c < kTile; c += 32) {
                uint32_t r[32];
                tmem_ld_32x32b_x32(tmem + (static_cast<uint32_t>(quad * 32) << 16) + acc * kTile + c, r);
                tmem_ld_wait();
                if (c + 32 == kTile) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh->tmem_empty[acc]);
                }
                float v[32];
#pragma unroll
                for (int j = 0; j < 32; ++j)
                    v[j] = activate(__uint_as_float(r[j]) + sh->bias[acc][c + j], sh->thr[acc][c + j], p.activation);
                store_chunk<OT>(p, v, row, n_blk * kTile + c, pol);
            }
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
    } else {
        int slot = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < units; u += gridDim.x) {
            int m_blk, n_blk;
            tile_coords(p, u, m_blk, n_blk);
            for (int g = 0; 4 * g < p.nkb; ++g) {
                const uint4 a = scale_words(p.a_scales, p.a_scale_pitch, p.a_shift, m_blk * kTile, p.M, g, lane);
                const uint4 b = scale_words(p.b_scales, p.b_scale_pitch, p.b_shift, n_blk * kTile, p.N, g, lane);
                if (!(ok = wait(&sh->scale_empty[slot], phase ^ 1u))) break;
                uint8_t *dst = sScale + slot * 1024 + lane * 16;
                *reinterpret_cast<uint4 *>(dst) = a;
                *reinterpret_cast<uint4 *>(dst + 512) = b;
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh->scale_full[slot]);
                if (++slot == kScaleSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem, kTmemCols);
    }
}

template <typename OT>
int launch(const CUtensorMap &tmA, const CUtensorMap &tmB, const GemmParams &p, cudaStream_t stream) {
    auto kern = block_gemm_kernel<OT>;
    const size_t smem = 1024 + 2 * kStages * kTileBytes + kScaleSlots * 1024 + sizeof(Shared);
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(block_gemm)");
    kern<<<std::min(p.m_tiles * p.n_tiles, num_sms()), kThreads, smem, stream>>>(tmA, tmB, p);
    return check_cuda(cudaGetLastError(), "block_gemm launch");
}

int check_product(const sf_blocks *a, const sf_blocks *b, const sf_matrix *out) {
    int st = check_blocks(a, "a");
    if (st) return st;
    if ((st = check_blocks(b, "b"))) return st;
    if (a->cols != b->cols)
        return set_error(SF_ERR_INVALID, "a has %lld columns but b has %lld", (long long)a->cols, (long long)b->cols);
    if (a->cols == 0) return set_error(SF_ERR_INVALID, "a and b have no columns");
    if (!out || !valid_dtype(out->dtype)) return set_error(SF_ERR_INVALID, "out is NULL or of an unsupported dtype");
    if (out->rows != a->rows || out->cols != b->rows) return set_error(SF_ERR_INVALID, "out must be [a rows, b rows]");
    if (out->rows > 0 && out->cols > 0 && !out->data) return set_error(SF_ERR_INVALID, "out has a NULL data pointer");
    if (out->cols > 1 && out->stride_col != 1) return set_error(SF_ERR_UNSUPPORTED, "out needs a unit column stride");
    // int coordinates, up to a tile past the end
    constexpr int64_t most = INT32_MAX - 4096;
    if (a->rows > most || b->rows > most || a->cols > most) return set_error(SF_ERR_UNSUPPORTED, "extent too large");
    return SF_OK;
}

}  // namespace

}  // namespace sf

using namespace sf;

extern "C" {

int sf_block_matmul_workspace(const sf_blocks *a, const sf_blocks *b, const sf_matrix *out, size_t *bytes) {
    const int st = check_product(a, b, out);
    if (st) return st;
    if (!bytes) return set_error(SF_ERR_INVALID, "bytes is NULL");
    *bytes = 0;
    return SF_OK;
}

int sf_block_matmul(const sf_blocks *a, const sf_blocks *b, const float *bias, const float *threshold, int activation,
                    const sf_matrix *out, void *workspace, size_t workspace_bytes, sf_stream stream) {
    int st = check_product(a, b, out);
    if (st) return st;
    if (activation != -1 && activation != SF_ACT_RELU && activation != SF_ACT_JUMPRELU)
        return set_error(SF_ERR_INVALID, "unknown activation %d", activation);
    if (activation == SF_ACT_JUMPRELU && !threshold) return set_error(SF_ERR_INVALID, "jumprelu needs a threshold");
    if (out->rows == 0 || out->cols == 0) return SF_OK;
    (void)workspace;
    (void)workspace_bytes;
    GemmParams p{};
    p.M = (int)a->rows;
    p.N = (int)b->rows;
    p.nkb = (int)((a->cols + kKBytes - 1) / kKBytes);
    p.m_tiles = (p.M + kTile - 1) / kTile;
    p.n_tiles = (p.N + kTile - 1) / kTile;
    if ((int64_t)p.m_tiles * p.n_tiles > INT32_MAX / 2) return set_error(SF_ERR_UNSUPPORTED, "too many output tiles");
    // A group of m-tiles runs side by side over each n-tile: b is read from HBM once per group, while
    // the group's 32 MB of a stay in L2.
    p.group_m = (int)std::max<int64_t>(1, std::min<int64_t>(p.m_tiles, (int64_t(32) << 20) / (kTile * a->cols)));
    p.a_scales = static_cast<const uint8_t *>(a->scales);
    p.b_scales = static_cast<const uint8_t *>(b->scales);
    p.a_scale_pitch = a->scale_pitch;
    p.b_scale_pitch = b->scale_pitch;
    p.a_shift = a->tile ? 7 : 0;
    p.b_shift = b->tile ? 7 : 0;
    p.bias = bias;
    p.thr = activation == SF_ACT_JUMPRELU ? threshold : nullptr;
    p.activation = activation;
    p.out = const_cast<void *>(out->data);
    p.out_pitch = out->stride_row;
    p.out_vec = (reinterpret_cast<uintptr_t>(out->data) % 16 == 0 &&
                 (out->stride_row * (int64_t)dtype_size(out->dtype)) % 16 == 0)
                    ? 1
                    : 0;
    p.err = device_error_word();
    CUtensorMap tmA, tmB;
    if ((st = make_map_e4m3(&tmA, a->data, (uint64_t)a->cols, (uint64_t)a->rows, (uint64_t)a->data_pitch, kTile)))
        return st;
    if ((st = make_map_e4m3(&tmB, b->data, (uint64_t)b->cols, (uint64_t)b->rows, (uint64_t)b->data_pitch, kTile)))
        return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (out->dtype == SF_BF16) return launch<__nv_bfloat16>(tmA, tmB, p, s);
    if (out->dtype == SF_F16) return launch<__half>(tmA, tmB, p, s);
    return launch<float>(tmA, tmB, p, s);
}

}  // extern "C"

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
// Persistent kernel, one CTA per SM, warp-specialised (352 threads; 384 for long sums):
//   warp 0      TMA producer: 128-byte rows of both operands, SWIZZLE_128B, mbarrier ring
//   warp 1      TMEM allocator and MMA issuer
//   8 warps     epilogue: bias, activation, rounding, stores; two warps to 32 rows, half the columns each
//   1 warp      scale words of both operands for 512 elements of K into shared memory, in the order that
//               tcgen05.cp spreads over TMEM (row r at byte 16 (r % 32) + 4 (r / 32))
//
// Long sums (RANGES). The tensor cores add 32 products at a time to the sum in TMEM and round it toward zero, a
// bias that grows with the number of additions. So a sum stays in TMEM for a range of K, at most 1024 for fp32
// outputs and 2560 for 16-bit ones, and the epilogue warps add the ranges in registers, rounding to nearest.
// Error against 64 bits (relative, 4096 x K x 4096; one range / these / an fp32 FMA chain): operands of both signs
// K = 2304 1.2e-7 / 6.4e-8 / 6.2e-8, 8192 4.9e-7 / 8.1e-8 / 1.3e-7; of one sign 2304 6.1e-7 / 1.7e-7 / 1.3e-7, 8192
// 3.9e-6 / 1.9e-7 / 4.3e-7. Of 16-bit outputs (bf16, K = 2304 to 16384) one number in ten thousand rounds to the
// neighbour of the exact one's, as with an fp32 chain; ranges of 1024 would halve that. A handoff between two ranges
// takes about 1000 clocks (a range of 1024 about 5000): 4096 x 2304 x 16384 fp32 154 -> 175 us, 2304 x 8192 x 16384
// bf16 246 -> 281 us, 8192 x 16384 x 2304 bf16 279 -> 276 us, against one range each.
//
// Two sizes. PAIR: a CTA pair (cta_group::2) computes 256 x 256, each CTA loading 128 rows of either
// operand; both CTAs' loads complete on the leader's barriers. Single: one CTA computes 128 x COLS.
// A pair's tile has rows of `a` for its rows (TMEM lanes); a single CTA's has rows of `b`, so that few rows of
// `a` make a narrow tile (COLS = 32) beside 128 rows of weights.
//
// What bounds it. A pair reads 64 KB of operands from L2 per K block; all 148 SMs together get about 6 KB a
// clock, 700 to 780 clocks a block, where the MMAs take 512 (530 measured with the loads left out): large
// products are bound by operand delivery, and in a steady loop by the 1000 W power cap (SM clock near
// 1.4 GHz). Few rows of `a` are bound by the bytes of `b`; K below some 1500 by the handoff of tiles: the epilogue
// takes about 3300 clocks a tile, and at K = 768 waits another 1050 to 1440 for the next one's sums while the MMA
// warp waits about 3000 for its accumulator. Two accumulators of 256 columns and the scales exceed TMEM, so the accumulators overlap;
// 224-column tiles, whose accumulators do not, move 7% more bytes and were slower at every K from 128 up.
// Measured on a B200, bf16 outputs (M x K x N): 16384 x 2304 x 65536 1.95 ms, 2.5 PFLOP/s (in a steady loop 2.3 ms,
// 2.15 PFLOP/s, 0.92 of the library's 8-bit product with one scale per tensor); 4096 x 8192 x 16384 395 us, 2.8
// PFLOP/s, tensor pipe 77%; 16384 x 768 x 65536 985 us, 1.7 PFLOP/s; 4096 x 768 x 16384 58 to 69 us, box to box;
// 1 x 2304 x 65536 31 us, 4.9 TB/s of weights.
#include <algorithm>
#include <type_traits>

#include "sf_common.cuh"
#include "sf_internal.h"

namespace sf {

namespace {

constexpr int kKBytes = 128;                   // elements (bytes) of K per stage
constexpr int kScaleSlots = 3;                 // scale words of 512 elements of K each
constexpr int kEpilogueWarps = 8;              // two for each quarter of the TMEM lanes
// Long sums (RANGES) keep 128 more registers in each epilogue thread, which the four warps before them give up:
// 128 x 56 + 256 x 224 = 384 x 168, what the block is launched with.
constexpr int threads_of(bool ranges) { return 32 * ((ranges ? 4 : 3) + kEpilogueWarps); }
constexpr int kControlRegs = 56, kEpilogueRegs = 224, kLaunchRegs = 168;
static_assert(128 * kControlRegs + 32 * kEpilogueWarps * kEpilogueRegs == threads_of(true) * kLaunchRegs, "registers");
constexpr int kTmemCols = 512;
constexpr int kPairCols = 256;                 // columns of a pair's tile
constexpr int kRowTile = 128;                  // rows (TMEM lanes) per CTA

struct GemmParams {
    int rows, cols;            // of the tile grid: a's and b's, or b's and a's (kSwapped)
    int nkb, groups;           // K blocks of 128, and groups of four of them
    int splits, split_groups;  // ranges of K: split z takes groups [z split_groups, (z + 1) split_groups)
    int range_groups;          // groups whose sum the tensor cores keep; ranges are added in fp32 registers (RANGES)
    int row_tiles, col_tiles;
    int col_bytes;             // the columns' operand per CTA and stage, as its TMA box is cut
    int group_rows;            // row tiles that run side by side over each column tile
    Divisor32 by_tiles, by_group, by_rows, by_last_rows;  // tiles, tiles of a group, rows of a group, of the last
    const uint8_t *r_scales, *c_scales;  // of the rows' and the columns' operand
    int64_t r_pitch, c_pitch;
    int r_shift, c_shift;      // log2 of the rows a scale row serves: 0 row blocks, 7 tiles
    const float *bias, *thr;
    int activation;            // enum sf_activation, -1 none
    void *out;                 // of plain stores
    int64_t out_pitch;
    int64_t out_split;         // elements between the splits' outputs
    unsigned *err;
};

// Compile-time shape of a kernel.
template <bool PAIR_, int COLS_, int STAGES_>
struct Shape {
    static constexpr bool PAIR = PAIR_;
    static constexpr int COLS = COLS_;                          // columns of a tile
    static constexpr int ROWS = PAIR ? 256 : 128;               // rows of a tile
    static constexpr int COLS_HERE = PAIR ? COLS / 2 : COLS;    // rows of the columns' operand loaded per CTA
    static constexpr int STAGES = STAGES_;
    static constexpr int R_BYTES = kRowTile * kKBytes, C_BYTES = COLS_HERE * kKBytes;
    static constexpr int COL_WORDS = COLS <= 128 ? 4 : 8;  // TMEM columns of the columns' scales
    static constexpr int SLOT_COLS = 4 + COL_WORDS;
    static constexpr int SLOT_BYTES = 512 + COL_WORDS / 4 * 512;
    // Two accumulators and the scales in 512 columns of TMEM: at 256 columns the accumulators overlap by 40.
    static constexpr int ACC1 = COLS == 256 ? 216 : COLS;
    static constexpr bool OVERLAP = ACC1 < COLS;
    static constexpr int SCALE_COL = ACC1 + COLS;
    static_assert(SCALE_COL + kScaleSlots * SLOT_COLS <= kTmemCols, "TMEM columns");
};

// How a tile's sums reach the output. kTma: boxes of 32 rows x 128 bytes, for rows that start on 16-byte boundaries. kRows:
// 256-byte runs of a row through shared memory, shifted to the output's own 16-byte boundaries. kSwapped: the
// rows of the tile are the columns of the output, and a warp stores 32 neighbours of one row at a time.
enum Store { kTma = 0, kRows = 1, kSwapped = 2 };

constexpr int out_bytes(int store) {  // of shared memory per epilogue warp
    return store == kTma ? 32 * 128 : store == kRows ? 32 * 256 : 0;
}

struct __align__(16) Shared {
    uint64_t full[12], empty[12];
    uint64_t scale_full[kScaleSlots], scale_empty[kScaleSlots];
    uint64_t tmem_full[2], tmem_empty[2];
    uint64_t drain;
    uint32_t tmem_base;
    int abort_flag;
    alignas(16) float bias[kEpilogueWarps][128];
    alignas(16) float thr[kEpilogueWarps][128];
};

struct Unit {
    int row0, col0, split, kb0, kb1;
};

template <typename S>
__device__ __forceinline__ Unit unit_of(const GemmParams &p, int u) {
    Unit r;
    r.split = p.by_tiles.div(u);
    u -= r.split * (int)p.by_tiles.d;
    const int g = p.by_group.div(u);
    const int first = g * p.group_rows;
    const bool last = p.row_tiles - first < p.group_rows;
    const Divisor32 by = last ? p.by_last_rows : p.by_rows;
    const int local = u - g * (int)p.by_group.d;
    const int col = by.div(local);
    r.row0 = (first + local - col * (int)by.d) * S::ROWS;
    r.col0 = col * S::COLS;
    r.kb0 = 4 * r.split * p.split_groups;
    r.kb1 = min(p.nkb, r.kb0 + 4 * p.split_groups);
    return r;
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

// max(v, floor) that keeps a NaN (fmaxf would drop it): ReLU with floor 0, nothing with floor -inf.
__device__ __forceinline__ float at_least(float v, float floor) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(v), "f"(floor));
    return r;
}
__device__ __forceinline__ float jump(float v, float t) { return v > t && v > 0.f ? v : 0.f; }
__device__ __forceinline__ float floor_of(int activation) {
    return activation == SF_ACT_RELU ? 0.f : __int_as_float(0xff800000);
}

// max of two 16-bit floats each and zero, keeping NaN.
template <typename OT>
__device__ __forceinline__ uint32_t relu2(uint32_t w) {
    uint32_t r;
    if constexpr (std::is_same_v<OT, __nv_bfloat16>)
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    else
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0u));
    return r;
}

// Two neighbours in a 16-bit output type (converted one by one they run at a quarter of the rate).
template <typename OT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (std::is_same_v<OT, __nv_bfloat16>) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Bias, activation and rounding of 32 sums: the words of the output. `bias(j)` gives four at a time, `thr(j)` one.
// The activation is uniform: tested once, not per element (which took 1350 clocks). ReLU of a 16-bit output
// comes after its rounding, two at a time; both are monotone, so their order does not matter.
template <typename OT, typename Bias, typename Thr>
__device__ __forceinline__ void finish32(uint32_t (&r)[32], int activation, Bias bias, Thr thr,
                                         uint32_t (&o)[8 * sizeof(OT)]) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
        const float4 b = bias(j);
        r[j] = __float_as_uint(__uint_as_float(r[j]) + b.x);
        r[j + 1] = __float_as_uint(__uint_as_float(r[j + 1]) + b.y);
        r[j + 2] = __float_as_uint(__uint_as_float(r[j + 2]) + b.z);
        r[j + 3] = __float_as_uint(__uint_as_float(r[j + 3]) + b.w);
    }
    if (activation == SF_ACT_JUMPRELU) {
#pragma unroll
        for (int j = 0; j < 32; ++j) r[j] = __float_as_uint(jump(__uint_as_float(r[j]), thr(j)));
    }
    if constexpr (sizeof(OT) == 4) {
#pragma unroll
        for (int j = 0; j < 32; ++j) o[j] = r[j];
        if (activation == SF_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(at_least(__uint_as_float(o[j]), 0.f));
        }
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j] = pack2<OT>(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
        if (activation == SF_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < 16; ++j) o[j] = relu2<OT>(o[j]);
        }
    }
}

// Eight words shifted right by `bytes` < 16, a multiple of 2 (of 4 where ES is 4): the first four.
template <int ES>
__device__ __forceinline__ void shift_words(uint32_t (&w)[8], int bytes) {
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = (bytes & 8) ? w[j + 2] : w[j];
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = (bytes & 4) ? w[j + 1] : w[j];
    if (ES == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = (bytes & 2) ? __funnelshift_r(w[j], w[j + 1], 16) : w[j];
    }
}

// 256 bytes of each of 32 output rows from a warp's buffer (16-byte chunk j of row r at chunk j ^ r % 16) to
// `out`, the first row's run; the runs start between 16-byte boundaries, each at its own place. A half warp
// takes a row: the aligned chunks by shifting two of the buffer's into one, then the elements before the
// first and after the last boundary, a lane to a row. `rows` and `cols` of them exist.
template <typename OT>
__device__ __forceinline__ void store_runs(const uint8_t *buf, OT *out, int64_t pitch, int rows, int cols, int lane) {
    constexpr int E = 16 / sizeof(OT), ES = sizeof(OT);
    const int limit = min(cols, 16 * E);
    auto lead_of = [&](int r) {  // elements before the first boundary
        return (int)((0u - (uint32_t)reinterpret_cast<uintptr_t>(out + r * pitch)) & 15u) / ES;
    };
#pragma unroll 4
    for (int it = 0; it < 16; ++it) {
        const int r = 2 * it + (lane >> 4), d = lane & 15;
        const int lead = lead_of(r);
        if (r >= rows || lead + E * (d + 1) > limit) continue;
        const uint4 a = *reinterpret_cast<const uint4 *>(buf + r * 256 + ((d ^ (r & 15)) << 4));
        uint4 b = a;
        if (lead) b = *reinterpret_cast<const uint4 *>(buf + r * 256 + (((d + 1) ^ (r & 15)) << 4));
        uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        shift_words<ES>(w, lead * ES);
        *reinterpret_cast<uint4 *>(out + r * pitch + lead + E * d) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (lane >= rows) return;
    const int lead = lead_of(lane);
    OT *dst = out + lane * pitch;
    if (limit == 16 * E) {
        // Whole runs: the first `lead` elements and the last E - lead, as pieces of 2, 4 and 8 bytes that end and
        // start at a boundary (element by element they took longer than all the rest).
        if (lead == 0) return;
        const uint4 a = *reinterpret_cast<const uint4 *>(buf + lane * 256 + ((lane & 15) << 4));
        const uint4 b = *reinterpret_cast<const uint4 *>(buf + lane * 256 + ((15 ^ (lane & 15)) << 4));
        uint32_t w[8] = {a.x, a.y, a.z, a.w, 0u, 0u, 0u, 0u}, t[8] = {b.x, b.y, b.z, b.w, 0u, 0u, 0u, 0u};
        uint8_t *to = reinterpret_cast<uint8_t *>(dst);
        int bytes = lead * ES;
        if (ES == 2 && (bytes & 2)) {
            *reinterpret_cast<uint16_t *>(to) = (uint16_t)w[0];
            to += 2;
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
        }
        if (bytes & 4) {
            *reinterpret_cast<uint32_t *>(to) = w[0];
            to += 4;
            w[0] = w[1];
            w[1] = w[2];
        }
        if (bytes & 8) *reinterpret_cast<uint2 *>(to) = make_uint2(w[0], w[1]);
        shift_words<ES>(t, bytes);
        to = reinterpret_cast<uint8_t *>(dst + 15 * E + lead);
        bytes = 16 - bytes;
        if (bytes & 8) {
            *reinterpret_cast<uint2 *>(to) = make_uint2(t[0], t[1]);
            to += 8;
            t[0] = t[2];
            t[1] = t[3];
        }
        if (bytes & 4) {
            *reinterpret_cast<uint32_t *>(to) = t[0];
            to += 4;
            t[0] = t[1];
        }
        if (ES == 2 && (bytes & 2)) *reinterpret_cast<uint16_t *>(to) = (uint16_t)t[0];
        return;
    }
    const int tail = lead + max(0, limit - lead) / E * E;  // the first element after the last boundary
    auto one = [&](int j) {
        const int at = j * ES;
        dst[j] = *reinterpret_cast<const OT *>(buf + lane * 256 + (((at >> 4) ^ (lane & 15)) << 4) + (at & 15));
    };
#pragma unroll
    for (int j = 0; j < E - 1; ++j) {
        if (j < min(lead, limit)) one(j);
        if (tail + j < limit) one(tail + j);
    }
}

template <typename OT, typename S, int STORE, bool RANGES>
__global__ void __launch_bounds__(threads_of(RANGES), 1)
    block_gemm_kernel(const __grid_constant__ CUtensorMap tmR, const __grid_constant__ CUtensorMap tmC,
                      const __grid_constant__ CUtensorMap tmOut, const GemmParams p) {
    constexpr bool PAIR = S::PAIR, SWAP = STORE == kSwapped;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *sR = smem;
    uint8_t *sC = sR + S::STAGES * S::R_BYTES;
    constexpr int OUT_BYTES = out_bytes(STORE);
    uint8_t *sOut = sC + S::STAGES * S::C_BYTES;  // one buffer per epilogue warp
    uint8_t *sScale = sOut + kEpilogueWarps * OUT_BYTES;
    Shared *sh = reinterpret_cast<Shared *>(sScale + kScaleSlots * S::SLOT_BYTES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int EPI = RANGES ? 4 : 2;  // the first epilogue warp; the scales' is the last, or (RANGES) the third
    const uint32_t rank = PAIR ? cluster_ctarank() : 0u;
    const bool leader = rank == 0;
    const int first_unit = PAIR ? (int)cluster_id_x() : (int)blockIdx.x;
    const int step_units = PAIR ? (int)num_clusters_x() : (int)gridDim.x;
    const int units = p.row_tiles * p.col_tiles * p.splits;
    constexpr int kCtas = PAIR ? 2 : 1;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) {
            mbar_init(&sh->full[s], 1);   // leader's: its expect_tx arrive + both CTAs' bytes
            mbar_init(&sh->empty[s], 1);  // one commit of the leader's MMA thread
        }
        for (int s = 0; s < kScaleSlots; ++s) {
            mbar_init(&sh->scale_full[s], kCtas);  // leader's: one arrive per CTA's scale warp
            mbar_init(&sh->scale_empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh->tmem_full[b], 1);
            mbar_init(&sh->tmem_empty[b], kEpilogueWarps * kCtas);  // leader's: one arrive per epilogue warp
        }
        mbar_init(&sh->drain, 1);
        sh->abort_flag = 0;
        fence_mbar_init();
        tma_prefetch_desc(&tmR);
        tma_prefetch_desc(&tmC);
        if (STORE == kTma) tma_prefetch_desc(&tmOut);
    }
    if (warp == 1) {
        if (PAIR) {
            tmem_alloc_pair(&sh->tmem_base, kTmemCols);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(&sh->tmem_base, kTmemCols);
            tmem_relinquish();
        }
    }
    tc_fence_before();
    if (PAIR)
        cluster_sync();
    else
        __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh->tmem_base;
    volatile int *abort_flag = &sh->abort_flag;
    const uint32_t peer_abort = PAIR ? map_to_rank(smem_u32(&sh->abort_flag), rank ^ 1u) : 0u;
    // A wait that runs out (or sees the abort flag) also raises the other CTA's flag.
    auto wait = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (mbar_wait(bar, parity, abort_flag, p.err)) return true;
        if (PAIR) st_remote_u32(peer_abort, 1u);
        return false;
    };
    // The same with cluster-scope acquire, for phases that the peer's threads complete.
    auto wait_cluster = [&](uint64_t *bar, uint32_t parity) -> bool {
        if (!PAIR) return wait(bar, parity);
        if (mbar_wait_cluster(bar, parity, abort_flag, p.err)) return true;
        st_remote_u32(peer_abort, 1u);
        return false;
    };
    // A whole warp waits: every lane sees the phase, and all of them agree on whether it came, so that a wait that
    // ran out does not split the warp before an instruction that needs all of it (at most 1% of the time; one
    // polling lane that the others follow cost 5 to 25%).
    auto wait_warp = [&](uint64_t *bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)) != 0; };
    auto wait_warp_cluster = [&](uint64_t *bar, uint32_t parity) {
        return __all_sync(0xffffffffu, wait_cluster(bar, parity)) != 0;
    };
    auto arrive_leader = [&](uint64_t *bar) {
        if (PAIR)
            mbar_arrive_remote(map_to_rank(smem_u32(bar), 0));
        else
            mbar_arrive(bar);
    };
    // For TMEM that has been read.
    auto release_leader = [&](uint64_t *bar) {
        if (PAIR)
            mbar_arrive_remote_cta(map_to_rank(smem_u32(bar), 0));
        else
            mbar_arrive(bar);
    };
    // Completion of the MMA thread's work so far, on this barrier of every CTA.
    auto commit = [&](uint64_t *bar) {
        if (PAIR) {
            umma_commit_pair(map_to_rank(smem_u32(bar), 0));
            umma_commit_pair(map_to_rank(smem_u32(bar), 1));
        } else {
            umma_commit(bar);
        }
    };

    if (warp >= EPI && warp < EPI + kEpilogueWarps) {
        if (RANGES) set_registers_up<kEpilogueRegs>();
        // ---------------------------------------------------------------- epilogue
        const int quad = warp & 3;
        // This warp's columns: a half of the tile's, or the first warp all 32 of the narrowest.
        constexpr int HALF = S::COLS < 64 ? S::COLS : S::COLS / 2;
        constexpr int STEP = HALF < 64 ? HALF : 64;  // columns loaded at a time
        constexpr int STEPS = HALF / STEP;
        static_assert(STEPS <= 2, "at most two steps a tile");
        static_assert(S::OVERLAP || STEPS == 1, "released after the first step");
        const int half = (warp - EPI) >> 2;
        const bool mine = half * HALF < S::COLS;
        int acc = 0;
        uint32_t acc_phase = 0;
        // Bias and threshold of the coming tile, loaded a tile ahead: this thread's row's (kSwapped), else those of
        // this warp's columns, passed through the warp's own shared memory (no barrier between warps).
        constexpr int OWN = SWAP ? 1 : HALF / 32;
        float next_bias[OWN], next_thr[OWN];
        float *my_bias = sh->bias[warp - EPI], *my_thr = sh->thr[warp - EPI];
        auto load_vectors = [&](const Unit &un) {
#pragma unroll
            for (int j = 0; j < OWN; ++j) {
                const int at = SWAP ? un.row0 + (int)rank * kRowTile + quad * 32 + lane
                                    : un.col0 + half * HALF + 32 * j + lane;
                const bool have = at < (SWAP ? p.rows : p.cols);
                next_bias[j] = p.bias && have ? __ldg(p.bias + at) : 0.f;
                next_thr[j] = p.thr && have ? __ldg(p.thr + at) : 0.f;
            }
        };
        Unit next = unit_of<S>(p, min(first_unit, units - 1));
        load_vectors(next);
        for (int u = first_unit; u < units; u += step_units) {
            const Unit un = next;
            const int row = un.row0 + (int)rank * kRowTile + quad * 32 + lane;
            const float row_bias = next_bias[0], row_thr = next_thr[0];
            if (!SWAP) {
#pragma unroll
                for (int j = 0; j < OWN; ++j) {
                    my_bias[32 * j + lane] = next_bias[j];
                    my_thr[32 * j + lane] = next_thr[j];
                }
                __syncwarp();
            }
            next = unit_of<S>(p, min(u + step_units, units - 1));
            load_vectors(next);
            if (!RANGES && !wait_warp(&sh->tmem_full[acc], acc_phase)) break;
            tc_fence_after();
            const uint32_t lanes = tmem + (static_cast<uint32_t>(quad * 32) << 16) + half * HALF;
            // Overlapping accumulators: the shared columns (the first's last 40, the second's first 40) are
            // read first and released to the next tile's MMAs. A warp whose half has none of them releases at
            // once: what it still had to read of the tile before, in the accumulator that those MMAs take, it has.
            auto release = [&]() {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) release_leader(&sh->tmem_empty[acc]);
            };
            auto advance = [&]() {
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            };

            // Columns [c0, c0 + STEP) of this warp's half, from r to the output.
            auto put = [&](uint32_t (&r)[STEP / 32][32], int c0, bool last) {
#pragma unroll
                for (int h = 0; h < STEP / 32; ++h) {
                    const int c = c0 + 32 * h;
                    const int col = un.col0 + half * HALF + c;
                    uint32_t o[8 * sizeof(OT)];
                    if constexpr (SWAP) {
                        finish32<OT>(
                            r[h], p.activation, [&](int) { return make_float4(row_bias, row_bias, row_bias, row_bias); },
                            [&](int) { return row_thr; }, o);
                        if (row < p.rows) {
                            OT *dst = reinterpret_cast<OT *>(p.out) + un.split * p.out_split +
                                      (int64_t)col * p.out_pitch + row;
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (col + j < p.cols) dst[j * p.out_pitch] = reinterpret_cast<const OT *>(o)[j];
                        }
                    } else {
                        finish32<OT>(
                            r[h], p.activation, [&](int j) { return *reinterpret_cast<const float4 *>(my_bias + c + j); },
                            [&](int j) { return my_thr[c + j]; }, o);
                        uint8_t *buf = sOut + (warp - EPI) * OUT_BYTES;
                        const int row_w = un.row0 + (int)rank * kRowTile + quad * 32;
                        constexpr int CHUNKS = 2 * sizeof(OT);
                        if constexpr (STORE == kTma) {
                            // 32 rows of 128 bytes (64 columns of 16 bits, 32 of fp32), 16-byte chunk j of row r at
                            // chunk j ^ r % 8 as the tensor map says
                            if (h == 0 || sizeof(OT) == 4) {
                                tma_store_wait_read<0>();  // the last store has read the buffer
                                __syncwarp();
                            }
#pragma unroll
                            for (int j = 0; j < CHUNKS; ++j) {
                                const int chunk = (sizeof(OT) == 4 ? 0 : CHUNKS * h) + j;
                                *reinterpret_cast<uint4 *>(buf + lane * 128 + ((chunk ^ (lane & 7)) << 4)) =
                                    make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                            }
                            if (h == STEP / 32 - 1 || sizeof(OT) == 4) {
                                fence_proxy_async_smem();
                                __syncwarp();
                                const int col_w = sizeof(OT) == 4 ? col : col - 32 * h;
                                if (lane == 0) {
                                    if (row_w < p.rows && col_w < p.cols)
                                        tma_store_3d(&tmOut, buf, col_w, row_w, un.split);
                                    tma_store_commit();
                                }
                            }
                        } else {
                            // 256 bytes of a row: this warp's 128 columns of 16 bits, or 64 of fp32
                            constexpr int RUN = 256 / sizeof(OT);
                            const int c_run = c / RUN * RUN;
#pragma unroll
                            for (int j = 0; j < CHUNKS; ++j) {
                                const int chunk = (c - c_run) * (int)sizeof(OT) / 16 + j;
                                *reinterpret_cast<uint4 *>(buf + lane * 256 + ((chunk ^ (lane & 15)) << 4)) =
                                    make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
                            }
                            if (h == STEP / 32 - 1 && (sizeof(OT) == 4 || last)) {
                                __syncwarp();
                                const int col_w = un.col0 + half * HALF + c_run;
                                if (col_w < p.cols && row_w < p.rows)
                                    store_runs<OT>(buf,
                                                   reinterpret_cast<OT *>(p.out) + un.split * p.out_split +
                                                       (int64_t)row_w * p.out_pitch + col_w,
                                                   p.out_pitch, p.rows - row_w, p.cols - col_w, lane);
                                __syncwarp();
                            }
                        }
                    }
                }
            };
            if constexpr (RANGES) {
                // Long K: the sums of its ranges, added here in their order with rounding to nearest.
                float sums[STEPS][STEP / 32][32];
#pragma unroll
                for (int i = 0; i < STEPS * STEP; ++i) sums[i / STEP][i % STEP / 32][i % 32] = 0.f;
                bool ok = true;
                for (int kb0 = un.kb0; kb0 < un.kb1; kb0 += 4 * p.range_groups) {
                    if (!(ok = wait_warp(&sh->tmem_full[acc], acc_phase))) break;
                    tc_fence_after();
                    const bool shares = !S::OVERLAP || half == (acc ^ 1);
                    if (!shares || !mine) release();
                    uint32_t r[STEP / 32][32];
                    auto load = [&](int i) {
#pragma unroll
                        for (int h = 0; h < STEP / 32; ++h)
                            tmem_ld_32x32b_x32(lanes + acc * S::ACC1 + i * STEP + 32 * h, r[h]);
                        tmem_ld_wait();
                    };
                    auto add = [&](int i) {
#pragma unroll
                        for (int j = 0; j < STEP; ++j) {
                            sums[i][j / 32][j % 32] += __uint_as_float(r[j / 32][j % 32]);
                            asm volatile("" : "+f"(sums[i][j / 32][j % 32]));  // before the next load: else both are held
                        }
                    };
                    if (mine) {
                        if (STEPS == 2 && acc == 0) {
                            load(STEPS - 1);
                            if (shares) release();
                            add(STEPS - 1);
                            load(0);
                            add(0);
                        } else {
                            load(0);
                            if (shares) release();
                            add(0);
                            if (STEPS == 2) {
                                load(STEPS - 1);
                                add(STEPS - 1);
                            }
                        }
                    }
                    advance();
                }
                if (!ok) break;
                if (mine) {
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                        uint32_t r[STEP / 32][32];
#pragma unroll
                        for (int j = 0; j < STEP; ++j) r[j / 32][j % 32] = __float_as_uint(sums[i][j / 32][j % 32]);
                        put(r, i * STEP, i == STEPS - 1);
                    }
                }
            } else {
                const bool shares = !S::OVERLAP || half == (acc ^ 1);
                const uint32_t taddr = lanes + acc * S::ACC1;
                if (!shares || !mine) release();
                // One step's sums at a time: loading the second while the first is finished spilled registers, and
                // was slower at every size measured (16384 x 256 x 65536: 773 against 638 us).
                const int c_first = STEPS == 2 && acc == 0 ? STEP : 0;
#pragma unroll 1
                for (int i = 0; mine && i < STEPS; ++i) {
                    const int c0 = i == 0 ? c_first : STEP - c_first;
                    uint32_t r[STEP / 32][32];
#pragma unroll
                    for (int h = 0; h < STEP / 32; ++h) tmem_ld_32x32b_x32(taddr + c0 + 32 * h, r[h]);
                    tmem_ld_wait();
                    if (shares && i == (S::OVERLAP ? 0 : STEPS - 1)) release();
                    put(r, c0, i == STEPS - 1);
                }
                advance();
            }
        }
        if (STORE == kTma) tma_store_wait_read<0>();  // the buffers go with the CTA
    } else {
        if (RANGES) set_registers_down<kControlRegs>();
        if (warp == 0) {
            // ---------------------------------------------------------------- TMA producer
            if (lane == 0) {
                // a group's row tiles are read again for each of its column tiles
                const uint64_t pol_c = l2_policy_evict_normal();
                const uint64_t pol_r = p.col_tiles > 1 ? l2_policy_evict_last() : pol_c;
                int stage = 0;
                uint32_t phase = 0, armed = 0, armed_parity = 0;
                bool ok = true;
                for (int u = first_unit; ok && u < units; u += step_units) {
                    const Unit un = unit_of<S>(p, u);
                    const int row0 = un.row0 + (int)rank * kRowTile, col0 = un.col0 + (int)rank * S::COLS_HERE;
                    for (int kb = un.kb0; kb < un.kb1; ++kb) {
                        if (!(ok = wait(&sh->empty[stage], phase ^ 1u))) break;
                        if (leader) {
                            mbar_arrive_expect_tx(&sh->full[stage], kCtas * (S::R_BYTES + p.col_bytes));
                            armed |= 1u << stage;
                            armed_parity = (armed_parity & ~(1u << stage)) | (phase << stage);
                        }
                        uint8_t *dr = sR + stage * S::R_BYTES, *dc = sC + stage * S::C_BYTES;
                        if (PAIR) {
                            const uint32_t full = map_to_rank(smem_u32(&sh->full[stage]), 0);
                            tma_load_2d_pair(dr, &tmR, full, kb * kKBytes, row0, pol_r);
                            tma_load_2d_pair(dc, &tmC, full, kb * kKBytes, col0, pol_c);
                        } else {
                            tma_load_2d(dr, &tmR, &sh->full[stage], kb * kKBytes, row0, pol_r);
                            tma_load_2d(dc, &tmC, &sh->full[stage], kb * kKBytes, col0, pol_c);
                        }
                        if (++stage == S::STAGES) {
                            stage = 0;
                            phase ^= 1u;
                        }
                    }
                }
                if (*abort_flag) {  // copies in flight must land before the CTA leaves
                    if (leader) {
                        for (int s = 0; s < S::STAGES; ++s)
                            if (armed & (1u << s)) mbar_wait_drain(&sh->full[s], (armed_parity >> s) & 1u, p.err);
                    } else {
                        const unsigned long long t0 = global_timer_ns();
                        while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
                    }
                }
            }
        } else if (warp == 1) {
            // ---------------------------------------------------------------- MMA issuer (the leader's)
            // The whole warp walks the loop, so that addresses and descriptors stay in uniform registers, and
            // one elected lane issues: with the loop inside a one-lane branch each instruction's operands were
            // moved there one by one (some 140 clocks an MMA, more than a 256 x 256 x 32 one takes).
            if (leader) {
                const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
                const uint64_t desc_r = smem_desc_sw128(smem_u32(sR), 16, 1024);
                const uint64_t desc_c = smem_desc_sw128(smem_u32(sC), 16, 1024);
                const uint64_t desc_s = smem_desc_rows16(smem_u32(sScale));
                int stage = 0, slot = 0, acc = 0;
                uint32_t phase = 0, slot_phase = 0, acc_phase = 0;
                bool ok = true, first = true;
                for (int u = first_unit; ok && u < units; u += step_units) {
                    const Unit un = unit_of<S>(p, u);
                    // A sum in TMEM runs over a range of K, the whole of the unit's unless it is long (RANGES).
                    for (int kb0 = un.kb0; ok && kb0 < un.kb1; kb0 += RANGES ? 4 * p.range_groups : un.kb1) {
                        const int kb1 = RANGES ? min(un.kb1, kb0 + 4 * p.range_groups) : un.kb1;
                        // Accumulators that overlap: the previous sum's epilogue must have read the columns that
                        // this one shares with it (and so has finished the sum before that).
                        if (S::OVERLAP) {
                            if (!first && !(ok = wait_warp(&sh->tmem_empty[acc ^ 1], acc ? acc_phase : acc_phase ^ 1u))) break;
                            first = false;
                        } else if (!(ok = wait_warp(&sh->tmem_empty[acc], acc_phase ^ 1u))) {
                            break;
                        }
                        tc_fence_after();
                        const uint32_t d = tmem_u + acc * S::ACC1;
                        for (int kb4 = kb0; ok && kb4 < kb1; kb4 += 4) {
                            if (!(ok = wait_warp_cluster(&sh->scale_full[slot], slot_phase))) break;
                            tc_fence_after();
                            const uint32_t scales = tmem_u + S::SCALE_COL + slot * S::SLOT_COLS;
                            if (elect_one()) {
                                const uint64_t src = desc_s + slot * (S::SLOT_BYTES >> 4);
#pragma unroll
                                for (int i = 0; i < S::SLOT_COLS / 4; ++i) {
                                    if (PAIR)
                                        tmem_copy_32x128b_pair(scales + 4 * i, src + 32 * i);
                                    else
                                        tmem_copy_32x128b(scales + 4 * i, src + 32 * i);
                                }
                            }
                            __syncwarp();
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (kb4 + j >= kb1) break;
                                if (!(ok = wait_warp(&sh->full[stage], phase))) break;
                                tc_fence_after();
                                const uint64_t rd = desc_r + stage * (S::R_BYTES >> 4), cd = desc_c + stage * (S::C_BYTES >> 4);
                                constexpr uint32_t IDESC0 = make_idesc_e4m3_scaled(S::ROWS, S::COLS, 0);
                                const uint32_t idesc = IDESC0 | (j << 4) | (j << 29);
                                if (elect_one()) {
#pragma unroll
                                    for (int ks = 0; ks < 4; ++ks) {
                                        const uint32_t accumulate = (kb4 > kb0 || j || ks) ? 1u : 0u;
                                        if (PAIR)
                                            umma_e4m3_scaled_pair(d, rd + 2 * ks, cd + 2 * ks, idesc, scales, scales + 4,
                                                                  accumulate);
                                        else
                                            umma_e4m3_scaled(d, rd + 2 * ks, cd + 2 * ks, idesc, scales, scales + 4, accumulate);
                                    }
                                    commit(&sh->empty[stage]);
                                    // Released with the group's last MMA: a slot is filled again, in shared memory and
                                    // then in TMEM, only after the MMAs that read it.
                                    if (j == 3 || kb4 + j + 1 == kb1) commit(&sh->scale_empty[slot]);
                                    if (kb4 + j + 1 == kb1) commit(&sh->tmem_full[acc]);
                                }
                                __syncwarp();
                                if (++stage == S::STAGES) {
                                    stage = 0;
                                    phase ^= 1u;
                                }
                            }
                            if (++slot == kScaleSlots) {
                                slot = 0;
                                slot_phase ^= 1u;
                            }
                        }
                        if (++acc == 2) {
                            acc = 0;
                            acc_phase ^= 1u;
                        }
                    }
                }
                if (elect_one()) {
                    if (PAIR)
                        umma_commit_pair(map_to_rank(smem_u32(&sh->drain), 0));
                    else
                        umma_commit(&sh->drain);
                }
                __syncwarp();
                mbar_wait_drain(&sh->drain, 0, p.err);
            }
        } else if (!RANGES || warp == 2) {
            // ---------------------------------------------------------------- scales (both CTAs)
            // A group's words are loaded while the one before waits for its slot: a load from HBM takes as long
            // as the MMAs of a group.
            constexpr int WORDS = 1 + S::COL_WORDS / 4;
            int u = first_unit, g = 0;
            Unit un = unit_of<S>(p, u < units ? u : 0);
            g = un.kb0 / 4;
            uint4 w[WORDS];
            auto load = [&]() {
                w[0] = scale_words(p.r_scales, p.r_pitch, p.r_shift, un.row0 + (int)rank * kRowTile, p.rows, g, lane);
#pragma unroll
                for (int i = 1; i < WORDS; ++i)
                    w[i] = scale_words(p.c_scales, p.c_pitch, p.c_shift, un.col0 + 128 * (i - 1), p.cols, g, lane);
            };
            int slot = 0;
            uint32_t phase = 0;
            if (u < units) load();
            while (u < units) {
                uint4 now[WORDS];
#pragma unroll
                for (int i = 0; i < WORDS; ++i) now[i] = w[i];
                if (4 * ++g >= un.kb1) {
                    u += step_units;
                    if (u < units) {
                        un = unit_of<S>(p, u);
                        g = un.kb0 / 4;
                    }
                }
                if (u < units) load();
                if (!wait_warp(&sh->scale_empty[slot], phase ^ 1u)) break;
                uint8_t *dst = sScale + slot * S::SLOT_BYTES + lane * 16;
#pragma unroll
                for (int i = 0; i < WORDS; ++i) *reinterpret_cast<uint4 *>(dst + 512 * i) = now[i];
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) arrive_leader(&sh->scale_full[slot]);
                if (++slot == kScaleSlots) {
                    slot = 0;
                    phase ^= 1u;
                }
            }
        }
    }

    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();  // the leader's MMAs no longer read this CTA's shared memory
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        if (PAIR)
            tmem_dealloc_pair(tmem, kTmemCols);
        else
            tmem_dealloc(tmem, kTmemCols);
    }
}

// out = act(sum of the splits' partial sums, in order, + bias): four columns a thread.
template <typename OT>
__global__ void __launch_bounds__(256) join_splits_kernel(const float *__restrict__ part, int64_t split_stride,
                                                          int64_t pitch, int splits, int M, int N,
                                                          const float *__restrict__ bias,
                                                          const float *__restrict__ thr, int activation,
                                                          OT *__restrict__ out, int64_t out_pitch) {
    const int n = (int)(blockIdx.x * blockDim.x + threadIdx.x) * 4;
    if (n >= N) return;
    for (int m = blockIdx.y; m < M; m += gridDim.y) {
        const float *src = part + (int64_t)m * pitch + n;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int z = 0; z < splits; ++z) {
            const float4 v = __ldg(reinterpret_cast<const float4 *>(src + z * split_stride));
            s.x += v.x;
            s.y += v.y;
            s.z += v.z;
            s.w += v.w;
        }
        const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (n + j >= N) break;
            float t = at_least(v[j] + (bias ? __ldg(bias + n + j) : 0.f), floor_of(activation));
            if (thr) t = jump(t, __ldg(thr + n + j));
            out[(int64_t)m * out_pitch + n + j] = from_f32<OT>(t);
        }
    }
}

// ------------------------------------------------------------------------------- host side

template <typename OT, typename S, int STORE>
int launch(const CUtensorMap &tmR, const CUtensorMap &tmC, const CUtensorMap &tmOut, const GemmParams &p,
           cudaStream_t stream) {
    const bool ranges = p.range_groups < p.split_groups;
    auto kern = ranges ? block_gemm_kernel<OT, S, STORE, true> : block_gemm_kernel<OT, S, STORE, false>;
    constexpr size_t smem = 1024 + S::STAGES * (S::R_BYTES + S::C_BYTES) + kEpilogueWarps * out_bytes(STORE) +
                            kScaleSlots * S::SLOT_BYTES + sizeof(Shared);
    static_assert(smem <= 232448, "shared memory per block");
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return check_cuda(e, "cudaFuncSetAttribute(block_gemm)");
    const int units = p.row_tiles * p.col_tiles * p.splits;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.blockDim = dim3(threads_of(ranges));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    if (S::PAIR) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.numAttrs = 1;
        cfg.gridDim = dim3(2 * std::max(1, num_sms() / 2));
        cfg.gridDim = dim3(2 * std::min(units, pair_slots(reinterpret_cast<const void *>(kern), cfg)));
    } else {
        cfg.gridDim = dim3(std::min(units, num_sms()));
    }
    e = cudaLaunchKernelEx(&cfg, kern, tmR, tmC, tmOut, p);
    if (e != cudaSuccess) return check_cuda(e, "block_gemm launch");
    return check_cuda(cudaGetLastError(), "block_gemm launch");
}

// Operand stages: what the store buffers leave of shared memory.
template <int STORE>
using Pair = Shape<true, kPairCols, STORE == kRows ? 4 : 5>;
using One32 = Shape<false, 32, 10>;
using One64 = Shape<false, 64, 8>;
using One128 = Shape<false, 128, 6>;

// What a call does, from its sizes alone.
struct Plan {
    bool pair;   // CTA pairs on 256 x 256 tiles; else single CTAs on 128 rows of b x `cols` rows of a (kSwapped)
    int cols;
    int splits;  // of K, among SMs and into a workspace
    int range_groups;  // groups of 512 of K to a sum in TMEM
};

int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }
int cdiv(int64_t a, int64_t b) { return (int)cdiv64(a, b); }

Plan make_plan(int64_t M, int64_t N, int64_t K, int out_dtype) {
    Plan pl{};
    const int sms = num_sms();
    const int groups = cdiv(K, 4 * kKBytes);
    // Either kernel is paced by its operand loads: 128 + cols rows per K block for a single CTA, 256 for a CTA of
    // a pair, whose tile is twice the work. Waves times that predict the faster one; measured (us, pair against
    // single): 256 x 768 x 16384 11.8 / 16.8, 512 x 512 x 5000 8.7 / 13.7, 2048 x 1024 x 2048 11.3 / 16.0, and
    // about even where both fit one wave (200 x 768 x 5000: 9.6 / 9.7).
    const int cols = M <= 32 ? 32 : M <= 64 ? 64 : 128;
    const int64_t one_tiles = cdiv64(N, 128) * cdiv64(M, cols);
    const int64_t pair_tiles = cdiv64(N, 256) * cdiv64(M, 256);
    const int64_t one_cost = cdiv64(one_tiles, sms) * (128 + cols), pair_cost = cdiv64(pair_tiles, sms / 2) * 256;
    pl.pair = M > 128 && pair_cost < one_cost;
    pl.cols = pl.pair ? kPairCols : cols;
    const int64_t tiles = pl.pair ? pair_tiles : one_tiles;
    const int slots = pl.pair ? sms / 2 : sms;
    // Few tiles: K is split among the idle SMs, at least 2048 of it to each, and the partial sums joined by a
    // second kernel. Measured (us, split against whole): K = 768 12.7 / 9.5 (512 x 2048), 2304 13.0 / 12.4
    // (256 x 2048), 5000 19.3 / 23.6 (1000 x 768), 8192 16.1 / 24.4 (640 x 640), 13558 23.5 / 35.1 (636 x 1094).
    pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(groups / 4, slots / tiles));
    // fp32 outputs: splits of at most 8192, whatever the number of tiles, which is what the workspace query has
    // always asked for. Their exactness comes from the ranges below.
    if (out_dtype == SF_F32) pl.splits = std::max(pl.splits, cdiv(K, 8192));
    // whole splits: none without a group
    const int split_groups = cdiv(groups, pl.splits);
    pl.splits = cdiv(groups, split_groups);
    const int most = out_dtype == SF_F32 ? 2 : 5;  // 1024 or 2560 of K: the errors are at the top of this file
    pl.range_groups = cdiv(split_groups, cdiv(split_groups, most));
    return pl;
}

int64_t partial_pitch(int64_t N) { return (N + 3) / 4 * 4; }

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

// Checks a product of which something is asked for and plans it. Its tiles, over all splits, are numbered in 32
// bits, and a step of the grid past the last.
int plan_product(const sf_blocks *a, const sf_blocks *b, const sf_matrix *out, Plan *pl) {
    *pl = make_plan(a->rows, b->rows, a->cols, out->dtype);
    const int64_t tiles = pl->pair ? cdiv64(b->rows, kPairCols) * cdiv64(a->rows, 256)
                                   : cdiv64(b->rows, kRowTile) * cdiv64(a->rows, pl->cols);
    if (tiles * pl->splits > INT32_MAX - 65536) return set_error(SF_ERR_UNSUPPORTED, "too many output tiles");
    return SF_OK;
}

// Rows that TMA can write: 16-byte aligned base, pitch and length. A store of a row that ends between boundaries
// writes up to the next one (measured: zeros beside the output, in every type).
bool tma_rows(const sf_matrix &out) {
    const int64_t es = (int64_t)dtype_size(out.dtype);
    return reinterpret_cast<uintptr_t>(out.data) % 16 == 0 && out.stride_row >= out.cols &&
           (out.stride_row * es) % 16 == 0 && (out.cols * es) % 16 == 0;
}

template <typename OT>
int run_plan(const Plan &pl, int store, const CUtensorMap &r, const CUtensorMap &c, const CUtensorMap &o, const GemmParams &p,
             cudaStream_t s) {
    if (pl.pair)
        return store == kTma ? launch<OT, Pair<kTma>, kTma>(r, c, o, p, s)
                             : launch<OT, Pair<kRows>, kRows>(r, c, o, p, s);
    if (pl.cols == 32) return launch<OT, One32, kSwapped>(r, c, o, p, s);
    if (pl.cols == 64) return launch<OT, One64, kSwapped>(r, c, o, p, s);
    return launch<OT, One128, kSwapped>(r, c, o, p, s);
}

}  // namespace

}  // namespace sf

using namespace sf;

extern "C" {

int sf_block_matmul_workspace(const sf_blocks *a, const sf_blocks *b, const sf_matrix *out, size_t *bytes) {
    int st = check_product(a, b, out);
    if (st) return st;
    if (!bytes) return set_error(SF_ERR_INVALID, "bytes is NULL");
    *bytes = 0;
    if (out->rows == 0 || out->cols == 0) return SF_OK;
    Plan pl;
    if ((st = plan_product(a, b, out, &pl))) return st;
    if (pl.splits > 1) *bytes = (size_t)pl.splits * out->rows * partial_pitch(out->cols) * sizeof(float);
    return SF_OK;
}

int sf_block_matmul_plan(const sf_blocks *a, const sf_blocks *b, const sf_matrix *out, sf_block_plan *plan) {
    int st = check_product(a, b, out);
    if (st) return st;
    if (!plan) return set_error(SF_ERR_INVALID, "plan is NULL");
    *plan = sf_block_plan{};
    if (out->rows == 0 || out->cols == 0) return SF_OK;
    Plan pl;
    if ((st = plan_product(a, b, out, &pl))) return st;
    plan->tile_rows = pl.pair ? 256 : pl.cols;
    plan->tile_cols = pl.pair ? kPairCols : kRowTile;
    plan->splits = pl.splits;
    plan->range = (int)std::min<int64_t>(a->cols, (int64_t)pl.range_groups * 4 * kKBytes);
    return SF_OK;
}

int sf_block_matmul(const sf_blocks *a, const sf_blocks *b, const float *bias, const float *threshold, int activation,
                    const sf_matrix *out, void *workspace, size_t workspace_bytes, sf_stream stream) {
    size_t need = 0;
    int st = sf_block_matmul_workspace(a, b, out, &need);
    if (st) return st;
    if (activation != -1 && activation != SF_ACT_RELU && activation != SF_ACT_JUMPRELU)
        return set_error(SF_ERR_INVALID, "unknown activation %d", activation);
    if (activation == SF_ACT_JUMPRELU && !threshold) return set_error(SF_ERR_INVALID, "jumprelu needs a threshold");
    if (out->rows == 0 || out->cols == 0) return SF_OK;
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16))
        return set_error(SF_ERR_WORKSPACE, "16-byte aligned workspace of %zu bytes needed", need);
    const int M = (int)a->rows, N = (int)b->rows;
    Plan pl;
    if ((st = plan_product(a, b, out, &pl))) return st;
    // Partial sums go to the workspace in fp32, without bias or activation, and are joined after.
    const bool partial = pl.splits > 1;
    sf_matrix dst = *out;
    if (partial) {
        dst.data = workspace;
        dst.dtype = SF_F32;
        dst.stride_row = dst.cols = partial_pitch(N);  // whole 16-byte units: what is past column N is not read
    }
    const int store = !pl.pair ? kSwapped : tma_rows(dst) ? kTma : kRows;
    const sf_blocks *R = pl.pair ? a : b, *C = pl.pair ? b : a;
    const int row_tile = pl.pair ? 256 : 128;
    GemmParams p{};
    p.rows = (int)R->rows;
    p.cols = (int)C->rows;
    p.nkb = cdiv(a->cols, kKBytes);
    p.groups = cdiv(p.nkb, 4);
    p.splits = pl.splits;
    p.split_groups = cdiv(p.groups, pl.splits);
    p.range_groups = pl.range_groups;
    p.row_tiles = cdiv(p.rows, row_tile);
    p.col_tiles = cdiv(p.cols, pl.cols);
    // A group of row tiles runs side by side over each column tile: the columns' operand is read from HBM
    // once per group, while the group's 32 MB stay in L2.
    p.group_rows = (int)std::max<int64_t>(1, std::min<int64_t>(p.row_tiles, (int64_t(32) << 20) / (row_tile * a->cols)));
    p.by_tiles = Divisor32::of(p.row_tiles * p.col_tiles);
    p.by_group = Divisor32::of(p.group_rows * p.col_tiles);
    p.by_rows = Divisor32::of(p.group_rows);
    p.by_last_rows = Divisor32::of(p.row_tiles % p.group_rows ? p.row_tiles % p.group_rows : p.group_rows);
    p.r_scales = static_cast<const uint8_t *>(R->scales);
    p.c_scales = static_cast<const uint8_t *>(C->scales);
    p.r_pitch = R->scale_pitch;
    p.c_pitch = C->scale_pitch;
    p.r_shift = R->tile ? 7 : 0;
    p.c_shift = C->tile ? 7 : 0;
    p.bias = partial ? nullptr : bias;
    p.thr = partial || activation != SF_ACT_JUMPRELU ? nullptr : threshold;
    p.activation = partial ? -1 : activation;
    p.out = const_cast<void *>(dst.data);
    p.out_pitch = dst.stride_row;
    p.out_split = (int64_t)M * dst.stride_row;
    p.err = device_error_word();
    CUtensorMap tmR, tmC, tmOut = {};
    if ((st = make_map_e4m3(&tmR, R->data, (uint64_t)R->cols, (uint64_t)R->rows, (uint64_t)R->data_pitch, kRowTile)))
        return st;
    // A tile with fewer columns than its width loads only those (rows past a matrix cost TMA as much as rows
    // of it); the rest of the stage holds anything, for sums that are never stored.
    const int box = pl.pair ? kPairCols / 2 : std::min(pl.cols, cdiv(p.cols, 8) * 8);
    p.col_bytes = box * kKBytes;
    if ((st = make_map_e4m3(&tmC, C->data, (uint64_t)C->cols, (uint64_t)C->rows, (uint64_t)C->data_pitch, box)))
        return st;
    const int64_t es = (int64_t)dtype_size(dst.dtype);
    if (store == kTma &&
        (st = make_map_out(&tmOut, dst.data, dst.dtype, (uint64_t)dst.cols, (uint64_t)M, (uint64_t)pl.splits,
                           (uint64_t)(dst.stride_row * es), (uint64_t)(p.out_split * es))))
        return st;
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    if (dst.dtype == SF_BF16)
        st = run_plan<__nv_bfloat16>(pl, store, tmR, tmC, tmOut, p, s);
    else if (dst.dtype == SF_F16)
        st = run_plan<__half>(pl, store, tmR, tmC, tmOut, p, s);
    else
        st = run_plan<float>(pl, store, tmR, tmC, tmOut, p, s);
    if (st || !partial) return st;
    const dim3 grid(cdiv(N, 1024), std::min(M, 65535));
    const float *part = static_cast<const float *>(workspace);
    const float *thr = activation == SF_ACT_JUMPRELU ? threshold : nullptr;
    void *o = const_cast<void *>(out->data);
#define SF_JOIN(T)                                                                                                 \
    join_splits_kernel<T><<<grid, 256, 0, s>>>(part, p.out_split, p.out_pitch, pl.splits, M, N, bias, thr, activation, \
                                               static_cast<T *>(o), out->stride_row)
    if (out->dtype == SF_BF16)
        SF_JOIN(__nv_bfloat16);
    else if (out->dtype == SF_F16)
        SF_JOIN(__half);
    else
        SF_JOIN(float);
#undef SF_JOIN
    return check_cuda(cudaGetLastError(), "join_splits launch");
}

}  // extern "C"

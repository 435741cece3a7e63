// The 8-bit linear step and its gradients: quantising passes (blocks.cu) and products (block_gemm.cu) over
// operands laid out in two buffers, one that the backward keeps and one per call.
#include <algorithm>

#include "sf_common.cuh"
#include "sf_internal.h"

namespace {

constexpr int kNeedX = 1, kNeedW = 2, kNeedB = 4;

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// Hands out parts of a buffer in order; with a NULL buffer it only counts.
struct Carver {
    char *base;
    size_t used = 0;

    void *take(size_t n) {
        void *p = base + used;
        used += up256(n);
        return p;
    }
    sf_blocks blocks(int64_t rows, int64_t cols, bool tile) {
        sf_blocks b{};
        b.rows = rows;
        b.cols = cols;
        b.data_pitch = (cols + 15) / 16 * 16;
        b.scale_pitch = (cols + 4 * SF_BLOCK - 1) / (4 * SF_BLOCK) * 4;
        b.tile = tile ? 1 : 0;
        b.data = take((size_t)rows * b.data_pitch);
        b.scales = take((size_t)(tile ? (rows + SF_BLOCK - 1) / SF_BLOCK : rows) * b.scale_pitch);
        return b;
    }
};

struct Kept {
    sf_blocks xt, wq;
};

Kept lay_out_keep(Carver &c, int64_t M, int64_t K, int64_t N, int needs) {
    Kept k{};
    if (needs & kNeedW) k.xt = c.blocks(K, M, false);
    if (needs & kNeedX) k.wq = c.blocks(K, N, true);
    return k;
}

sf_matrix like(int64_t rows, int64_t cols, int dtype) { return sf_matrix{nullptr, dtype, 0, rows, cols, cols, 1}; }

// Scratch of a product; a placeholder address stands for the output where only its shape is known.
int product_bytes(const sf_blocks &a, const sf_blocks &b, sf_matrix out, size_t *bytes) {
    if (!out.data) out.data = reinterpret_cast<const void *>(uintptr_t(256));
    return sf_block_matmul_workspace(&a, &b, &out, bytes);
}

int product(const sf_blocks &a, const sf_blocks &b, const float *bias, const sf_matrix *out, void *ws, size_t ws_bytes,
            sf_stream stream) {
    return sf_block_matmul(&a, &b, bias, nullptr, -1, out, ws, ws_bytes, stream);
}

int check_step(int64_t M, int64_t K, int64_t N) {
    if (M < 0 || K <= 0 || N < 0) return sf::set_error(SF_ERR_INVALID, "linear8 takes x [M, K] and W [K, N] with K > 0");
    return SF_OK;
}

}  // namespace

using sf::set_error;

extern "C" {

int sf_linear8_bytes(int64_t M, int64_t K, int64_t N, int x_dtype, int W_dtype, int needs, size_t *keep,
                     size_t *forward_temp, size_t *backward_temp) {
    int st = check_step(M, K, N);
    if (st) return st;
    if (!keep || !forward_temp || !backward_temp) return set_error(SF_ERR_INVALID, "NULL pointer");
    char *const nowhere = reinterpret_cast<char *>(uintptr_t(256));  // placed like a real buffer, never read
    Carver kc{nowhere}, fc{nowhere}, bc{nowhere};
    const Kept k = lay_out_keep(kc, M, K, N, needs);
    *keep = kc.used;
    const sf_blocks xq = fc.blocks(M, K, false), wt = fc.blocks(N, K, true);
    size_t ws = 0;
    if ((st = product_bytes(xq, wt, like(M, N, x_dtype), &ws))) return st;
    *forward_temp = fc.used + up256(ws);
    *backward_temp = 0;
    if (M == 0 || N == 0) return SF_OK;
    size_t wx = 0, ww = 0;
    const sf_blocks dyq = bc.blocks(M, N, false);
    if ((needs & kNeedX) && (st = product_bytes(dyq, k.wq, like(M, K, x_dtype), &wx))) return st;
    if (needs & kNeedW) {
        const sf_blocks dyt = bc.blocks(N, M, false);
        if ((st = product_bytes(k.xt, dyt, like(K, N, W_dtype), &ww))) return st;
    }
    if (needs & kNeedB) bc.take((size_t)((M + SF_BLOCK - 1) / SF_BLOCK) * N * sizeof(float));
    *backward_temp = bc.used + up256(std::max(wx, ww));
    return SF_OK;
}

int sf_linear8_forward(const sf_matrix *x, const sf_matrix *W, const float *bias, const sf_matrix *y, int needs,
                       void *keep, void *temp, size_t temp_bytes, sf_stream stream) {
    if (!x || !W || !y) return set_error(SF_ERR_INVALID, "x, W and y are required");
    const int64_t M = x->rows, K = x->cols, N = W->cols;
    int st = check_step(M, K, N);
    if (st) return st;
    if (W->rows != K) return set_error(SF_ERR_INVALID, "x has %lld columns but W has %lld rows", (long long)K, (long long)W->rows);
    if (y->rows != M || y->cols != N) return set_error(SF_ERR_INVALID, "y must be [M, N]");
    Carver kc{static_cast<char *>(keep)}, tc{static_cast<char *>(temp)};
    const Kept k = lay_out_keep(kc, M, K, N, needs);
    if (kc.used && !keep) return set_error(SF_ERR_WORKSPACE, "keep of %zu bytes needed", kc.used);
    const sf_blocks xq = tc.blocks(M, K, false), wt = tc.blocks(N, K, true);
    if (tc.used && (!temp || temp_bytes < tc.used)) return set_error(SF_ERR_WORKSPACE, "temp of %zu bytes needed", tc.used);
    if ((st = sf_blocks_quantize(x, &xq, (needs & kNeedW) ? &k.xt : nullptr, nullptr, nullptr, 0, stream))) return st;
    if ((st = sf_blocks_quantize(W, (needs & kNeedX) ? &k.wq : nullptr, &wt, nullptr, nullptr, 0, stream))) return st;
    return product(xq, wt, bias, y, tc.base + tc.used, temp_bytes - tc.used, stream);
}

int sf_linear8_backward(const sf_matrix *dy, const void *keep, int64_t K, int needs, const sf_matrix *dx,
                        const sf_matrix *dW, float *db, void *temp, size_t temp_bytes, sf_stream stream) {
    if (!dy) return set_error(SF_ERR_INVALID, "dy is NULL");
    const int64_t M = dy->rows, N = dy->cols;
    int st = check_step(M, K, N);
    if (st) return st;
    if (M == 0) return set_error(SF_ERR_INVALID, "dy has no rows");
    if ((dx && !(needs & kNeedX)) || (dW && !(needs & kNeedW)))
        return set_error(SF_ERR_INVALID, "a gradient that the forward kept nothing for");
    if (N == 0) {  // no features: dx is zeros, dW and db are empty
        if (!dx) return SF_OK;
        if (dx->rows != M || dx->cols != K || !dx->data || !sf::valid_dtype(dx->dtype))
            return set_error(SF_ERR_INVALID, "dx must be [M, K]");
        if (dx->stride_col != 1 || dx->stride_row < K) return set_error(SF_ERR_UNSUPPORTED, "dx needs a unit column stride");
        const size_t es = sf::dtype_size(dx->dtype);
        return sf::check_cuda(cudaMemset2DAsync(const_cast<void *>(dx->data), (size_t)dx->stride_row * es, 0, (size_t)K * es,
                                                (size_t)M, reinterpret_cast<cudaStream_t>(stream)),
                              "dx of no features");
    }
    Carver kc{static_cast<char *>(const_cast<void *>(keep))}, tc{static_cast<char *>(temp)};
    const Kept k = lay_out_keep(kc, M, K, N, needs);
    if (kc.used && !keep) return set_error(SF_ERR_INVALID, "keep is NULL");
    const sf_blocks dyq = tc.blocks(M, N, false);
    sf_blocks dyt{};
    if (dW) dyt = tc.blocks(N, M, false);
    const size_t sums = db ? (size_t)((M + SF_BLOCK - 1) / SF_BLOCK) * N * sizeof(float) : 0;
    void *const sums_at = tc.take(sums);
    if (!temp || temp_bytes < tc.used) return set_error(SF_ERR_WORKSPACE, "temp of %zu bytes needed", tc.used);
    void *const ws = tc.base + tc.used;
    const size_t ws_bytes = temp_bytes - tc.used;
    if ((st = sf_blocks_quantize(dy, dx || !dW ? &dyq : nullptr, dW ? &dyt : nullptr, db, sums_at, sums, stream))) return st;
    if (dx && (st = product(dyq, k.wq, nullptr, dx, ws, ws_bytes, stream))) return st;
    if (dW && (st = product(k.xt, dyt, nullptr, dW, ws, ws_bytes, stream))) return st;
    return SF_OK;
}

}  // extern "C"

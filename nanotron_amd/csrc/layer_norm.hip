// Layer normalisation over rows, forward and backward.
//
// Both passes are bound by memory: forward reads x and writes y, backward reads x and dy and writes dx.  A row lives in
// the registers of the threads that read it (a 16-byte piece a thread up to 1024 threads), so that the mean
// and then the variance about it, a sum of squared differences and not a difference of squares, cost no second read, nor does
// what the mean was off by.
// 16384 rows of 8192 bf16: forward 105 to 116 us, 537 MB at 4.6 to 5.1 TB/s, backward 159 to 168 us, 823 MB at 4.9 to 5.2; 4096 rows of
// 4096 16 and 21 us; one row of 4096 2.5 us.
#include "ops_common.h"

namespace ntfp8 {
namespace {

// threads of a block.  Forward: 256, or those of a row; backward: rows enough to fill a CU
constexpr int forward_block(int tpr) { return tpr < 256 ? 256 : tpr; }
constexpr int backward_block(int tpr) { return tpr <= 128 ? 512 : 1024; }
constexpr int kMostPieces = 4;   // 16-byte pieces of a row that a thread of the widest kernels holds

struct Norm {
    const void* x;
    const void* dy;
    const void* weight;
    const void* bias;
    void* out;           // y or dx
    float* mean;
    float* rstd;
    float* partial;      // backward: [grid][2][cols] sums for dweight and dbias, or NULL
    int64_t x_stride, dy_stride;
    int64_t rows;
    int cols;
    float eps;
};

// Sums of a and b over the `TPR` threads of a row, in every one of them.  `at`: [2][waves] of the block, turned over from
// call to call, so that one barrier suffices.
template <int TPR>
__device__ __forceinline__ void row_sums(float& a, float& b, float2* at) {
    a = wave_sum(a);
    b = wave_sum(b);
    if constexpr (TPR > 64) {
        constexpr int kWaves = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / kWaves * kWaves;
        if ((threadIdx.x & 63) == 0) at[wave] = make_float2(a, b);
        __syncthreads();
        a = b = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float2 o = at[first + w];
            a += o.x;
            b += o.y;
        }
    }
}

template <int D, int W, int TPR, int VPT>
__global__ __launch_bounds__(forward_block(TPR)) void layer_norm_forward_kernel(const Norm n) {
    constexpr int kBlock = forward_block(TPR), VE = 16 / size_of(D);
    __shared__ float2 sums[3][kBlock / 64];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
    const bool live = row < n.rows;   // (rows that share a block share its barriers)
    const int64_t x0 = row * n.x_stride;
    float v[VPT][VE], sum = 0.0f, none = 0.0f;
    Piece<D, VE> raw[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (t + k * TPR) * VE;
        raw[k] = load_piece<D, VE>(n.x, x0 + c, live && c < n.cols ? n.cols - c : 0);
    }
    // weight and bias are asked for before the row's sums are waited for, unless a row takes 1024 threads: held that long they
    // leave registers for one block a CU only, 8192 rows of 16384 168 us instead of 117
    constexpr bool kEarly = TPR < 1024;
    float w[VPT][VE], b[VPT][VE];
    auto affine = [&](int k) {
        const int c = (t + k * TPR) * VE, left = c < n.cols ? n.cols - c : 0;
        if (n.weight) unpack<W, VE>(load_piece<W, VE>(n.weight, c, left), w[k]);
        if (n.bias) unpack<W, VE>(load_piece<W, VE>(n.bias, c, left), b[k]);
    };
#pragma unroll
    for (int k = 0; k < VPT; ++k)
        if constexpr (kEarly) affine(k);
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        unpack<D, VE>(raw[k], v[k]);
#pragma unroll
        for (int e = 0; e < VE; ++e) sum += v[k][e];   // (zeros behind the row's end)
    }
    row_sums<TPR>(sum, none, sums[0]);
    const float over = 1.0f / (float)n.cols;
    float mean = sum * over, var = 0.0f;
    none = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (t + k * TPR) * VE;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            const float d = c + e < n.cols ? v[k][e] - mean : 0.0f;
            v[k][e] = d;
            var += d * d;
        }
    }
    row_sums<TPR>(var, none, sums[1]);
    var *= over;
    // The mean may be an ulp or two off, of which rstd makes 0.02 in a row of 1000.1s.  In rows whose mean is more than 16 deviations
    // it is corrected by the differences' own mean, divided and not multiplied, so that equal differences leave nothing; in others it
    // is good to 2^-15 of a deviation.  (For every row, beside the squares, it took 109 us instead of 105 for 16384 rows of 8192, and
    // 280 instead of 214 for 8192 of 32768, whose registers it overran; so, 112 and 218 where all rows are such, 105 and 214 where none is.)
    bool far = mean * mean > 256.0f * var;
    if constexpr (TPR > 64 && kBlock > TPR) far = __syncthreads_or(far);   // (rows that share barriers take them together)
    if (far) {
        float rest = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) rest += v[k][e];   // (zeros behind the row's end)
        row_sums<TPR>(rest, none, sums[2]);
        rest /= (float)n.cols;
        mean += rest;
        var -= rest * rest;
        var = var < 0.0f ? 0.0f : var;
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) v[k][e] -= rest;
    }
    const float rstd = 1.0f / sqrtf(var + n.eps);
    if (!live) return;
    if (t == 0 && n.mean) {
        n.mean[row] = mean;
        n.rstd[row] = rstd;
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (t + k * TPR) * VE;
        if (c >= n.cols) continue;
        if constexpr (!kEarly) affine(k);
        float y[VE];
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            y[e] = v[k][e] * rstd;
            if (n.weight) y[e] *= w[k][e];
            if (n.bias) y[e] += b[k][e];
        }
        store_piece<D, VE>(n.out, row * n.cols + c, y, n.cols - c);
    }
}

// dx = rstd (g - mean(g) - xhat mean(g xhat)) with g = dy weight; dweight = sum over rows of dy xhat, dbias of dy.
// A thread owns the same columns in every row that its group of TPR threads takes, and sums their share of dweight and
// dbias in registers; the groups of a block are added through LDS, and each block leaves one row of partial sums for
// column_sums_kernel.  One block of 1024 threads per CU: with blocks of 256 the partial sums would be a third of what the
// pass moves at 4096 columns.  Between the row's sums and dx the row is kept as it was read, and unpacked again: half the
// registers for 16-bit rows.  The next row is read while this one's sums go round, and the weight kept, where there are
// registers for it (kAhead, kHold).
template <int D, int W, int TPR, int VPT>
__global__ __launch_bounds__(backward_block(TPR)) void layer_norm_backward_kernel(const Norm n) {
    constexpr int kBlock = backward_block(TPR), kGroups = kBlock / TPR, VE = 16 / size_of(D);
    constexpr bool kHold = VPT * VE <= 8, kAhead = VPT * VE <= 16;
    __shared__ float2 sums[2][kBlock / 64];
    // [threads of the upper half of the groups][element], for one of dweight and dbias at a time
    __shared__ float other[kGroups > 1 ? kBlock / 2 * VPT * VE : 1];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float wh[VPT][VE], dw[VPT][VE], db[VPT][VE];
    auto weight = [&](int k, float (&w)[VE]) {
        const int c = (t + k * TPR) * VE;
        if (n.weight) {
            unpack<W, VE>(load_piece<W, VE>(n.weight, c, c < n.cols ? n.cols - c : 0), w);
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) w[e] = 1.0f;
        }
    };
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        if constexpr (kHold) weight(k, wh[k]);
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[k][e] = db[k][e] = 0.0f;
    }
    const float over = 1.0f / (float)n.cols;
    struct Row {
        Piece<D, VE> x[VPT], g[VPT];
        float mean, rstd;
    };
    auto read = [&](Row& r, int64_t row) {
        const bool live = row < n.rows;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (t + k * TPR) * VE, left = live && c < n.cols ? n.cols - c : 0;
            r.x[k] = load_piece<D, VE>(n.x, row * n.x_stride + c, left);
            r.g[k] = load_piece<D, VE>(n.dy, row * n.dy_stride + c, left);
        }
        r.mean = live ? n.mean[row] : 0.0f;
        r.rstd = live ? n.rstd[row] : 0.0f;
    };
    // xhat and g of a piece
    auto open = [&](const Row& r, int k, float (&x)[VE], float (&g)[VE]) {
        unpack<D, VE>(r.x[k], x);
        unpack<D, VE>(r.g[k], g);
#pragma unroll
        for (int e = 0; e < VE; ++e) x[e] = (x[e] - r.mean) * r.rstd;
    };
    const int64_t step = (int64_t)gridDim.x * kGroups;
    int64_t row = (int64_t)blockIdx.x * kGroups + group;
    Row now, next;
    if constexpr (kAhead) read(next, row);
    // (the same number of turns for every group: the barriers are the block's)
    int turn = 0;
    for (int64_t first = (int64_t)blockIdx.x * kGroups; first < n.rows; first += step, row += step, turn ^= 1) {
        if constexpr (kAhead) now = next;
        else read(now, row);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float x[VE], g[VE], w[VE];
            open(now, k, x, g);
            if constexpr (!kHold) weight(k, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                db[k][e] += g[e];
                dw[k][e] += g[e] * x[e];
                g[e] *= kHold ? wh[k][e] : w[e];
                s1 += g[e];
                s2 += g[e] * x[e];
            }
        }
        if constexpr (kAhead) read(next, row + step);
        row_sums<TPR>(s1, s2, sums[turn]);
        s1 *= over;
        s2 *= over;
        if (n.out && row < n.rows) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = (t + k * TPR) * VE;
                if (c >= n.cols) continue;
                float x[VE], g[VE], w[VE], d[VE];
                open(now, k, x, g);
                if constexpr (!kHold) weight(k, w);
#pragma unroll
                for (int e = 0; e < VE; ++e) d[e] = now.rstd * (g[e] * (kHold ? wh[k][e] : w[e]) - s1 - x[e] * s2);
                store_piece<D, VE>(n.out, row * n.cols + c, d, n.cols - c);
            }
        }
    }
    if (!n.partial) return;
    if constexpr (kGroups > 1) {
        auto add_up = [&](float (&d)[VPT][VE]) {
#pragma unroll
            for (int half = kGroups / 2; half >= 1; half /= 2) {
                __syncthreads();
                if (group >= half && group < 2 * half) {
#pragma unroll
                    for (int k = 0; k < VPT; ++k)
#pragma unroll
                        for (int e = 0; e < VE; ++e) other[((k * VE + e) * half + group - half) * TPR + t] = d[k][e];
                }
                __syncthreads();
                if (group < half) {
#pragma unroll
                    for (int k = 0; k < VPT; ++k)
#pragma unroll
                        for (int e = 0; e < VE; ++e) d[k][e] += other[((k * VE + e) * half + group) * TPR + t];
                }
            }
        };
        add_up(dw);
        add_up(db);
    }
    if (group == 0) {
        float* const p = n.partial + (int64_t)blockIdx.x * 2 * n.cols;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (t + k * TPR) * VE;
            if (c >= n.cols) continue;
            store_piece<NTFP8_F32, VE>(p, c, dw[k], n.cols - c);
            store_piece<NTFP8_F32, VE>(p, n.cols + c, db[k], n.cols - c);
        }
    }
}

// dweight and dbias from the blocks' partial sums [blocks][2][cols]: 32 columns a block of 256 threads, 8 runs of blocks.  Summed in
// 64 bits: one after another in 32 they brought most of the error of a weight's gradient
constexpr int kSumColumns = 32, kSumRuns = 8;
template <int W>
__global__ __launch_bounds__(kSumColumns * kSumRuns) void column_sums_kernel(const float* __restrict__ partial, int blocks, int cols,
                                                                             void* dweight, void* dbias) {
    __shared__ double part[kSumRuns][kSumColumns];
    const int c = threadIdx.x % kSumColumns, run = threadIdx.x / kSumColumns;
    const int64_t at = (int64_t)blockIdx.x * kSumColumns + c;   // of 2 cols
    double s = 0.0;
    if (at < 2 * (int64_t)cols) {
#pragma unroll 8
        for (int b = run; b < blocks; b += kSumRuns) s += (double)partial[(int64_t)b * 2 * cols + at];
    }
    part[run][c] = s;
    __syncthreads();
    if (run == 0 && at < 2 * (int64_t)cols) {
#pragma unroll
        for (int r = 1; r < kSumRuns; ++r) s += part[r][c];
        if (at < cols) {
            if (dweight) store_one<W>(dweight, at, (float)s);
        } else if (dbias) {
            store_one<W>(dbias, at - cols, (float)s);
        }
    }
}

// Threads of a row and pieces a thread, by the row's length in 16-byte pieces.  Forward: two pieces a thread, requested together
template <typename F>
int by_width_forward(int pieces, F&& f) {
    using std::integral_constant;
    if (pieces <= 64) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (pieces <= 128) return f(integral_constant<int, 64>{}, integral_constant<int, 2>{});
    if (pieces <= 256) return f(integral_constant<int, 128>{}, integral_constant<int, 2>{});
    if (pieces <= 512) return f(integral_constant<int, 256>{}, integral_constant<int, 2>{});
    if (pieces <= 1024) return f(integral_constant<int, 512>{}, integral_constant<int, 2>{});
    if (pieces <= 2048) return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    return f(integral_constant<int, 1024>{}, integral_constant<int, kMostPieces>{});
}
// backward: one, whose sums for weight and bias take the registers
template <typename F>
int by_width(int pieces, F&& f) {
    using std::integral_constant;
    if (pieces <= 64) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (pieces <= 128) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    if (pieces <= 256) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (pieces <= 512) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{});
    if (pieces <= 1024) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
    if (pieces <= 2048) return f(integral_constant<int, 1024>{}, integral_constant<int, 2>{});
    return f(integral_constant<int, 1024>{}, integral_constant<int, kMostPieces>{});
}
// weight and bias are fp32, or of the type of x
template <int D, typename F>
int with_weight(int w_dtype, F&& f) {
    if (w_dtype == NTFP8_F32) return f(std::integral_constant<int, NTFP8_F32>{});
    return f(std::integral_constant<int, D>{});
}
int pieces_of(int dtype, int64_t cols) { return (int)((cols * size_of(dtype) + 15) / 16); }

}  // namespace

int64_t layer_norm_most_cols(int dtype) { return 1024 * kMostPieces * 16 / size_of(dtype); }

// blocks of the backward kernel: one per CU of 1024 threads, two of 512
int layer_norm_blocks(int dtype, int64_t rows, int64_t cols) {
    return by_width(pieces_of(dtype, cols), [&](auto tpr, auto) {
        constexpr int kBlock = backward_block(decltype(tpr)::value), kGroups = kBlock / decltype(tpr)::value;
        return (int)std::min<int64_t>((rows + kGroups - 1) / kGroups, (int64_t)cu_count() * (1024 / kBlock));
    });
}

int run_layer_norm_forward(const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride, const void* weight, const void* bias,
                           int w_dtype, float eps, void* y, float* mean, float* rstd, hipStream_t st) {
    return with_dtype(x_dtype, [&](auto d) {
        return with_weight<decltype(d)::value>(w_dtype, [&](auto w) {
            return by_width_forward(pieces_of(x_dtype, cols), [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value, kBlock = forward_block(TPR), kRows = kBlock / TPR;
                // (a launch takes fewer than 2^32 threads)
                constexpr int64_t kMost = (int64_t)kRows << 21;
                for (int64_t row = 0; row < rows; row += kMost) {
                    const int64_t some = std::min(kMost, rows - row);
                    const Norm n = {static_cast<const char*>(x) + row * x_stride * size_of(x_dtype), nullptr, weight, bias, static_cast<char*>(y) + row * cols * size_of(x_dtype),
                                    mean ? mean + row : nullptr, mean ? rstd + row : nullptr, nullptr, x_stride, 0, some, (int)cols, eps};
                    layer_norm_forward_kernel<decltype(d)::value, decltype(w)::value, TPR, decltype(vpt)::value><<<(unsigned)((some + kRows - 1) / kRows), kBlock, 0, st>>>(n);
                    if (const int rc = launch_status(); rc != NTFP8_OK) return rc;
                }
                return (int)NTFP8_OK;
            });
        });
    });
}

int run_layer_norm_backward(const void* dy, int64_t dy_stride, const void* x, int x_dtype, int64_t rows, int64_t cols, int64_t x_stride,
                            const void* weight, int w_dtype, const float* mean, const float* rstd, void* dx, void* dweight, void* dbias,
                            float* scratch, hipStream_t st) {
    const bool sums = dweight || dbias;
    const int blocks = layer_norm_blocks(x_dtype, rows, cols);
    Norm n = {x, dy, weight, nullptr, dx, const_cast<float*>(mean), const_cast<float*>(rstd), sums ? scratch : nullptr, x_stride, dy_stride, rows, (int)cols, 0.0f};
    const int rc = with_dtype(x_dtype, [&](auto d) {
        return with_weight<decltype(d)::value>(w_dtype, [&](auto w) {
            return by_width(pieces_of(x_dtype, cols), [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value;
                layer_norm_backward_kernel<decltype(d)::value, decltype(w)::value, TPR, decltype(vpt)::value><<<blocks, backward_block(TPR), 0, st>>>(n);
                return launch_status();
            });
        });
    });
    if (rc != NTFP8_OK || !sums) return rc;
    return with_dtype(w_dtype, [&](auto w) {
        column_sums_kernel<decltype(w)::value><<<(unsigned)((2 * cols + kSumColumns - 1) / kSumColumns), kSumColumns * kSumRuns, 0, st>>>(scratch, blocks, (int)cols, dweight, dbias);
        return launch_status();
    });
}

}  // namespace ntfp8

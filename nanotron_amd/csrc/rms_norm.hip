// Root-mean-square norms around a block of a residual stream, forward and backward, each in one pass:
//   p = x / rms(x) * post_weight (or x),  h = residual_scale residual + gate p,  y = h / rms(h) * weight
// and, without a residual, the norm alone: h = x.  rms(x) = root(mean(x^2) + eps).
//
// Bound by memory.  A row lives in the registers of the threads that read it, so that both norms cost one read; h is rounded to the type of
// the residual stream before the second norm reads it, as the backward pass does, which has it from memory.
// 16384 rows of 4096, bf16 with an fp32 residual stream, both norms and a gate: 805 MB forward in 153 us, 1208 MB backward in 229, 5.3 TB/s.  Backward with a norm behind the block or
// a gate over more than 8192 elements of 16 bits holds two pieces of every row and vector a thread, of which 105 to 110 registers are spilled: 4096 rows of 16384, both norms and a
// gate, 574 us, 2.1 TB/s (without them 215, 5.0; forward 176, 4.6).
#include "ops_common.h"

namespace ntfp8 {
namespace {

constexpr int forward_block(int tpr) { return tpr < 256 ? 256 : tpr; }
// backward: rows enough to fill a CU; with a norm behind the block or a gate half the threads, which then have registers for its vectors (both norms
// and a gate, 16384 x 4096, forward and backward: 404 us, 431 with 1024 threads that read the vectors for every row)
constexpr int backward_block(int tpr, bool full) { return tpr == 1024 || (tpr >= 256 && !full) ? 1024 : 512; }
constexpr int kMostPieces = 2;   // 16-byte pieces of a row of x that a thread holds
enum Gate { kNoGate = 0, kChannelGate = 1, kElementGate = 2 };
constexpr int kVectors = 3;      // gradients that are summed over rows: weight, post_weight, a channel's gate

struct Norms {
    const void *x, *residual, *gate, *weight, *post_weight;
    const void *h, *dy, *dh;          // backward: h as the forward pass left it
    void *y, *h_out;
    void *dx, *dresidual, *dgate;
    float *first, *second;            // [rows] 1 / rms of x and of h
    float* partial;                   // backward: [grid][kVectors][cols]
    int64_t x_stride, residual_stride, gate_stride, dy_stride, dh_stride;   // (backward: residual_stride is that of h)
    int64_t rows;
    int cols, w_dtype, gate_kind;
    float eps, scale;
};

// Sum of a over the TPR threads of a row, in every one of them.  `at`: [waves] of the block, another for every call in a row
template <int TPR>
__device__ __forceinline__ float row_sum(float a, float* at) {
    a = wave_sum(a);
    if constexpr (TPR > 64) {
        constexpr int kWaves = TPR / 64;
        const int wave = threadIdx.x >> 6, first = wave / kWaves * kWaves;
        if ((threadIdx.x & 63) == 0) at[wave] = a;
        __syncthreads();
        a = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) a += at[first + w];
    }
    return a;
}
// a weight's piece, of fp32 or the type of x
template <int D, int VE>
__device__ __forceinline__ void vector_piece(const void* p, int w_dtype, int c, int cols, float (&w)[VE]) {
    const int left = c < cols ? cols - c : 0;
    if (w_dtype == NTFP8_F32) unpack<NTFP8_F32, VE>(load_piece<NTFP8_F32, VE>(p, c, left), w);
    else unpack<D, VE>(load_piece<D, VE>(p, c, left), w);
}

template <int D, int R, int TPR, int VPT>
__global__ __launch_bounds__(forward_block(TPR)) void rms_norm_forward_kernel(const Norms n) {
    constexpr int kBlock = forward_block(TPR), VE = 16 / size_of(D);
    __shared__ float sums[2][kBlock / 64];
    const int t = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kBlock / TPR) + threadIdx.x / TPR;
    const bool live = row < n.rows;   // (rows that share a block share its barriers)
    const float over = 1.0f / (float)n.cols;
    Piece<D, VE> raw[VPT], raw_gate[VPT];
    Piece<R, VE> raw_residual[VPT];
    float v[VPT][VE];
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (t + k * TPR) * VE, left = live && c < n.cols ? n.cols - c : 0;
        raw[k] = load_piece<D, VE>(n.x, row * n.x_stride + c, left);
        if (n.residual) raw_residual[k] = load_piece<R, VE>(n.residual, row * n.residual_stride + c, left);
        if (n.gate_kind == kElementGate) raw_gate[k] = load_piece<D, VE>(n.gate, row * n.gate_stride + c, left);
    }
#pragma unroll
    for (int k = 0; k < VPT; ++k) unpack<D, VE>(raw[k], v[k]);
    if (n.post_weight) {
        float s = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) s += v[k][e] * v[k][e];   // (zeros behind the row's end)
        s = row_sum<TPR>(s, sums[0]);
        const float first = 1.0f / sqrtf(s * over + n.eps);
        if (t == 0 && live && n.first) n.first[row] = first;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float w[VE];
            vector_piece<D, VE>(n.post_weight, n.w_dtype, (t + k * TPR) * VE, n.cols, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[k][e] = v[k][e] * first * w[e];
        }
    }
    if (n.residual) {
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (t + k * TPR) * VE;
            if (n.gate_kind != kNoGate) {
                float g[VE];
                if (n.gate_kind == kElementGate) unpack<D, VE>(raw_gate[k], g);
                else vector_piece<D, VE>(n.gate, n.w_dtype, c, n.cols, g);
#pragma unroll
                for (int e = 0; e < VE; ++e) v[k][e] *= g[e];
            }
            float r[VE];
            unpack<R, VE>(raw_residual[k], r);
#pragma unroll
            for (int e = 0; e < VE; ++e) v[k][e] = fmaf(n.scale, r[e], v[k][e]);
            if constexpr (R != NTFP8_F32) {
#pragma unroll
                for (int e = 0; e < VE; e += 2) {
                    const uint32_t w = pack_pair<R>(v[k][e], v[k][e + 1]);
                    unpack_pair<R>(w, v[k][e], v[k][e + 1]);
                }
            }
            if (live && c < n.cols) store_piece<R, VE>(n.h_out, row * n.cols + c, v[k], n.cols - c);
        }
    }
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < VPT; ++k)
#pragma unroll
        for (int e = 0; e < VE; ++e) s += v[k][e] * v[k][e];
    s = row_sum<TPR>(s, sums[1]);
    const float second = 1.0f / sqrtf(s * over + n.eps);
    if (!live) return;
    if (t == 0 && n.second) n.second[row] = second;
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        const int c = (t + k * TPR) * VE;
        if (c >= n.cols) continue;
        float w[VE], y[VE];
        if (n.weight) vector_piece<D, VE>(n.weight, n.w_dtype, c, n.cols, w);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            y[e] = v[k][e] * second;
            if (n.weight) y[e] *= w[e];
        }
        store_piece<D, VE>(n.y, row * n.cols + c, y, n.cols - c);
    }
}

// With n = h second, g = dy weight:  dh = dh_out + second (g - n mean(g n)), dweight = sum over rows of dy n, dresidual = scale dh,
// dgate = dh p, d = gate dh;  with u = x first, q = d post_weight:  dpost_weight = sum of d u, dx = first (q - u mean(q u)); without that norm
// dx = d.  A thread owns the same columns in all rows of its group and sums their share of the vectors' gradients in registers; the
// groups of a block are added through LDS, and each block leaves one row of sums a vector for vector_sums_kernel.
// kFull: there is a norm behind the block, or a gate.
template <int D, int R, bool kFull, int TPR, int VPT>
__global__ __launch_bounds__(backward_block(TPR, kFull)) void rms_norm_backward_kernel(const Norms n) {
    constexpr int kBlock = backward_block(TPR, kFull), kGroups = kBlock / TPR, VE = 16 / size_of(D), kSums = kFull ? kVectors : 1;
    constexpr bool kHold = VPT == 1;
    __shared__ float sums[2][2][kBlock / 64];
    __shared__ float other[kGroups > 1 ? kBlock / 2 * VPT * VE : 1];
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    const float over = 1.0f / (float)n.cols;
    float total[kSums][VPT][VE];
#pragma unroll
    for (int s = 0; s < kSums; ++s)
#pragma unroll
        for (int k = 0; k < VPT; ++k)
#pragma unroll
            for (int e = 0; e < VE; ++e) total[s][k][e] = 0.0f;
    // the vectors, kept where there are registers for them
    float held[kHold ? kSums : 1][VE];
    if constexpr (kHold) {
        if (n.weight) vector_piece<D, VE>(n.weight, n.w_dtype, t * VE, n.cols, held[0]);
        if constexpr (kFull) {
            if (n.post_weight) vector_piece<D, VE>(n.post_weight, n.w_dtype, t * VE, n.cols, held[1]);
            if (n.gate_kind == kChannelGate) vector_piece<D, VE>(n.gate, n.w_dtype, t * VE, n.cols, held[2]);
        }
    }
    auto vector = [&](int which, const void* p, int k, float (&w)[VE]) {
        if constexpr (kHold) {
#pragma unroll
            for (int e = 0; e < VE; ++e) w[e] = held[kFull ? which : 0][e];
        } else {
            vector_piece<D, VE>(p, n.w_dtype, (t + k * TPR) * VE, n.cols, w);
        }
    };
    struct Row {
        Piece<D, VE> dy[VPT], x[VPT], gate[VPT];
        Piece<R, VE> h[VPT], dh[VPT];
        float first, second;
    };
    auto read = [&](Row& r, int64_t row) {
        const bool live = row < n.rows;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (t + k * TPR) * VE, left = live && c < n.cols ? n.cols - c : 0;
            r.h[k] = load_piece<R, VE>(n.h, row * n.residual_stride + c, left);
            r.dy[k] = load_piece<D, VE>(n.dy, row * n.dy_stride + c, n.dy ? left : 0);
            r.dh[k] = load_piece<R, VE>(n.dh, row * n.dh_stride + c, n.dh ? left : 0);
            if constexpr (kFull) {
                r.x[k] = load_piece<D, VE>(n.x, row * n.x_stride + c, left);
                if (n.gate_kind == kElementGate) r.gate[k] = load_piece<D, VE>(n.gate, row * n.gate_stride + c, left);
            }
        }
        r.second = live ? n.second[row] : 0.0f;
        r.first = kFull && live && n.post_weight ? n.first[row] : 0.0f;
    };
    const int64_t step = (int64_t)gridDim.x * kGroups;
    int64_t row = (int64_t)blockIdx.x * kGroups + group;
    Row now;
    int turn = 0;
    // (the same number of turns for every group: the barriers are the block's)
    for (int64_t at = (int64_t)blockIdx.x * kGroups; at < n.rows; at += step, row += step, turn ^= 1) {
        const bool live = row < n.rows;
        read(now, row);
        const Piece<D, VE>(&dy)[VPT] = now.dy, (&x)[VPT] = now.x, (&gate)[VPT] = now.gate;
        const Piece<R, VE>(&h)[VPT] = now.h, (&dh)[VPT] = now.dh;
        const float first = now.first, second = now.second;
        float a[VPT][VE], s = 0.0f;   // g
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            float hv[VE], w[VE];
            unpack<R, VE>(h[k], hv);
            unpack<D, VE>(dy[k], a[k]);
            if (n.weight) vector(0, n.weight, k, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float nv = hv[e] * second;
                total[0][k][e] += a[k][e] * nv;
                if (n.weight) a[k][e] *= w[e];
                s += a[k][e] * nv;
            }
        }
        s = row_sum<TPR>(s, sums[turn][0]) * over;
        float q = 0.0f;
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            const int c = (t + k * TPR) * VE, left = live && c < n.cols ? n.cols - c : 0;
            float hv[VE], d[VE], o[VE];
            unpack<R, VE>(h[k], hv);
            unpack<R, VE>(dh[k], d);
#pragma unroll
            for (int e = 0; e < VE; ++e) a[k][e] = d[e] + second * (a[k][e] - hv[e] * second * s);   // dh
            if (n.dresidual) {
#pragma unroll
                for (int e = 0; e < VE; ++e) o[e] = n.scale * a[k][e];
                if (left) store_piece<R, VE>(n.dresidual, row * n.cols + c, o, left);
            }
            if constexpr (kFull) {
                float u[VE], pw[VE], g[VE];
                unpack<D, VE>(x[k], u);
                if (n.post_weight) {
                    vector(1, n.post_weight, k, pw);
#pragma unroll
                    for (int e = 0; e < VE; ++e) u[e] *= first;
                }
                if (n.gate_kind != kNoGate) {
                    if (n.gate_kind == kElementGate) unpack<D, VE>(gate[k], g);
                    else vector(2, n.gate, k, g);
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        o[e] = a[k][e] * (n.post_weight ? u[e] * pw[e] : u[e]);
                        total[2][k][e] += o[e];
                        a[k][e] *= g[e];
                    }
                    if (n.gate_kind == kElementGate && n.dgate && left) store_piece<D, VE>(n.dgate, row * n.cols + c, o, left);
                }
                if (n.post_weight) {
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        total[1][k][e] += a[k][e] * u[e];
                        a[k][e] *= pw[e];
                        q += a[k][e] * u[e];
                    }
                }
            }
        }
        if constexpr (kFull) {
            if (n.post_weight) q = row_sum<TPR>(q, sums[turn][1]) * over;   // (uniform)
        }
        if (n.dx) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = (t + k * TPR) * VE;
                if constexpr (kFull) {
                    if (n.post_weight) {
                        float u[VE];
                        unpack<D, VE>(x[k], u);
#pragma unroll
                        for (int e = 0; e < VE; ++e) a[k][e] = first * (a[k][e] - u[e] * first * q);
                    }
                }
                if (live && c < n.cols) store_piece<D, VE>(n.dx, row * n.cols + c, a[k], n.cols - c);
            }
        }
    }
    if (!n.partial) return;
    if constexpr (kGroups > 1) {
#pragma unroll
        for (int s = 0; s < kSums; ++s) {
#pragma unroll
            for (int half = kGroups / 2; half >= 1; half /= 2) {
                __syncthreads();
                if (group >= half && group < 2 * half) {
#pragma unroll
                    for (int k = 0; k < VPT; ++k)
#pragma unroll
                        for (int e = 0; e < VE; ++e) other[((k * VE + e) * half + group - half) * TPR + t] = total[s][k][e];
                }
                __syncthreads();
                if (group < half) {
#pragma unroll
                    for (int k = 0; k < VPT; ++k)
#pragma unroll
                        for (int e = 0; e < VE; ++e) total[s][k][e] += other[((k * VE + e) * half + group) * TPR + t];
                }
            }
        }
    }
    if (group == 0) {
        float* const p = n.partial + (int64_t)blockIdx.x * kSums * n.cols;
#pragma unroll
        for (int s = 0; s < kSums; ++s)
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                const int c = (t + k * TPR) * VE;
                if (c < n.cols) store_piece<NTFP8_F32, VE>(p, (int64_t)s * n.cols + c, total[s][k], n.cols - c);
            }
    }
}

// The vectors' gradients from the blocks' sums [blocks][vectors][cols], in 64 bits: 32 columns a block of 256 threads, 8 runs of blocks
constexpr int kSumColumns = 32, kSumRuns = 8;
struct Vectors {
    void* out[kVectors];
};
template <int W>
__global__ __launch_bounds__(kSumColumns * kSumRuns) void vector_sums_kernel(const float* __restrict__ partial, int blocks, int vectors, int cols, const Vectors v) {
    __shared__ double part[kSumRuns][kSumColumns];
    const int c = threadIdx.x % kSumColumns, run = threadIdx.x / kSumColumns, col = blockIdx.x * kSumColumns + c;
    void* const out = v.out[blockIdx.y];
    if (!out) return;
    double s = 0.0;
    if (col < cols) {
#pragma unroll 8
        for (int b = run; b < blocks; b += kSumRuns) s += (double)partial[((int64_t)b * vectors + blockIdx.y) * cols + col];
    }
    part[run][c] = s;
    __syncthreads();
    if (run == 0 && col < cols) {
#pragma unroll
        for (int r = 1; r < kSumRuns; ++r) s += part[r][c];
        store_one<W>(out, col, (float)s);
    }
}

// Threads of a row and pieces a thread, by the row's length in 16-byte pieces
template <typename F>
int by_width(int pieces, F&& f) {
    using std::integral_constant;
    if (pieces <= 64) return f(integral_constant<int, 64>{}, integral_constant<int, 1>{});
    if (pieces <= 128) return f(integral_constant<int, 128>{}, integral_constant<int, 1>{});
    if (pieces <= 256) return f(integral_constant<int, 256>{}, integral_constant<int, 1>{});
    if (pieces <= 512) return f(integral_constant<int, 512>{}, integral_constant<int, 1>{});
    if (pieces <= 1024) return f(integral_constant<int, 1024>{}, integral_constant<int, 1>{});
    return f(integral_constant<int, 1024>{}, integral_constant<int, kMostPieces>{});
}
// the residual stream is fp32, or of the type of x
template <int D, typename F>
int with_residual(int r_dtype, F&& f) {
    if (r_dtype == NTFP8_F32) return f(std::integral_constant<int, NTFP8_F32>{});
    return f(std::integral_constant<int, D>{});
}
int pieces_of(int dtype, int64_t cols) { return (int)((cols * size_of(dtype) + 15) / 16); }

}  // namespace

int64_t rms_norm_most_cols(int dtype) { return 1024 * kMostPieces * 16 / size_of(dtype); }

int rms_norm_blocks(int dtype, int64_t rows, int64_t cols, bool full) {
    return by_width(pieces_of(dtype, cols), [&](auto tpr, auto) {
        const int block = backward_block(decltype(tpr)::value, full), groups = block / decltype(tpr)::value;
        return (int)std::min<int64_t>((rows + groups - 1) / groups, (int64_t)cu_count() * (full ? 1 : 1024 / block));
    });
}

int run_rms_norm_forward(const ntops_rms_norm_desc& d, hipStream_t st) {
    return with_dtype(d.x_dtype, [&](auto t) {
        return with_residual<decltype(t)::value>(d.residual_dtype, [&](auto r) {
            return by_width(pieces_of(d.x_dtype, d.cols), [&](auto tpr, auto vpt) {
                constexpr int TPR = decltype(tpr)::value, kBlock = forward_block(TPR), kRows = kBlock / TPR;
                const int64_t xs = size_of(d.x_dtype), rs = size_of(d.residual_dtype);
                // (a launch takes fewer than 2^32 threads)
                constexpr int64_t kMost = (int64_t)kRows << 21;
                auto at = [](const void* p, int64_t bytes) -> void* { return p ? const_cast<char*>(static_cast<const char*>(p)) + bytes : nullptr; };
                for (int64_t row = 0; row < d.rows; row += kMost) {
                    Norms n = {};
                    n.rows = std::min(kMost, d.rows - row), n.cols = (int)d.cols, n.w_dtype = d.w_dtype, n.eps = d.eps, n.scale = d.residual_scale;
                    n.x = at(d.x, row * d.x_stride * xs), n.x_stride = d.x_stride;
                    n.residual = at(d.residual, row * d.residual_stride * rs), n.residual_stride = d.residual_stride;
                    n.gate_kind = d.gate_kind, n.gate_stride = d.gate_stride;
                    n.gate = d.gate_kind == kElementGate ? at(d.gate, row * d.gate_stride * xs) : const_cast<void*>(d.gate);
                    n.weight = d.weight, n.post_weight = d.post_weight;
                    n.y = at(d.y, row * d.cols * xs), n.h_out = at(d.h, row * d.cols * rs);
                    n.first = static_cast<float*>(at(d.first, row * 4)), n.second = static_cast<float*>(at(d.second, row * 4));
                    rms_norm_forward_kernel<decltype(t)::value, decltype(r)::value, TPR, decltype(vpt)::value><<<(unsigned)((n.rows + kRows - 1) / kRows), kBlock, 0, st>>>(n);
                    if (const int rc = launch_status(); rc != NTFP8_OK) return rc;
                }
                return (int)NTFP8_OK;
            });
        });
    });
}

int run_rms_norm_backward(const ntops_rms_norm_desc& d, const ntops_rms_norm_grads& g, hipStream_t st) {
    const bool full = d.post_weight || d.gate_kind != kNoGate;
    const bool vectors = g.dweight || g.dpost_weight || (g.dgate && d.gate_kind == kChannelGate);
    const int blocks = rms_norm_blocks(d.x_dtype, d.rows, d.cols, full);
    Norms n = {};
    n.rows = d.rows, n.cols = (int)d.cols, n.w_dtype = d.w_dtype, n.eps = d.eps, n.scale = d.residual_scale;
    n.x = d.x, n.x_stride = d.x_stride, n.gate = d.gate, n.gate_kind = d.gate_kind, n.gate_stride = d.gate_stride;
    // (without a residual h is x)
    n.h = d.h ? d.h : d.x, n.residual_stride = d.h ? d.cols : d.x_stride;
    n.weight = d.weight, n.post_weight = d.post_weight, n.first = d.first, n.second = d.second;
    n.dy = g.dy, n.dy_stride = g.dy_stride, n.dh = g.dh, n.dh_stride = g.dh_stride;
    n.dx = g.dx, n.dresidual = g.dresidual, n.dgate = d.gate_kind == kElementGate ? g.dgate : nullptr;
    n.partial = vectors ? static_cast<float*>(g.scratch) : nullptr;
    const int rc = with_dtype(d.x_dtype, [&](auto t) {
        return with_residual<decltype(t)::value>(d.residual_dtype, [&](auto r) {
            return by_width(pieces_of(d.x_dtype, d.cols), [&](auto tpr, auto vpt) {
                constexpr int D = decltype(t)::value, R = decltype(r)::value, TPR = decltype(tpr)::value, VPT = decltype(vpt)::value;
                if (full) rms_norm_backward_kernel<D, R, true, TPR, VPT><<<blocks, backward_block(TPR, true), 0, st>>>(n);
                else rms_norm_backward_kernel<D, R, false, TPR, VPT><<<blocks, backward_block(TPR, false), 0, st>>>(n);
                return launch_status();
            });
        });
    });
    if (rc != NTFP8_OK || !vectors) return rc;
    const Vectors v = {{g.dweight, g.dpost_weight, d.gate_kind == kChannelGate ? g.dgate : nullptr}};
    return with_dtype(d.w_dtype, [&](auto w) {
        const int count = full ? kVectors : 1;
        vector_sums_kernel<decltype(w)::value><<<dim3((unsigned)((d.cols + kSumColumns - 1) / kSumColumns), count), kSumColumns * kSumRuns, 0, st>>>(
            static_cast<const float*>(g.scratch), blocks, count, (int)d.cols, v);
        return launch_status();
    });
}

}  // namespace ntfp8

// Softmax cross entropy of a projection, without the logits: launches and the small kernels around the matrix products of
// head_gemm.h.
//
// With P = softmax(x W^T) and dl = P - onehot(labels): loss = mean or sum of logsumexp - logit of the label, dx = dl W,
// dW = dl^T x, three products of 2 tokens hidden vocab operations each.  The first one's epilogue turns a piece of 128 logits into
// its maximum, its sum and (where gradients are wanted) its exponentials below that maximum, rounded once to fp16, 2 bytes
// a logit that hold the softmax up to one factor a row and piece.  softmax_rows_kernel knows the whole row and makes dl of
// them in place, 16 bits again, as the matrix cores take it.  Nothing is computed twice and nothing of 4 bytes a logit exists; what
// there is of 2 bytes a logit is bounded by taking the tokens in pieces (head_piece).
#include "head_gemm.h"

namespace ntfp8 {
namespace {

constexpr int64_t kMostHeld = (int64_t)1 << 31;   // bytes of exponentials at a time, and of sums of dx
// elements between rows of the products' operands: 256 of them are within reach of 32-bit offsets.  Rows further apart are copied, as
// unaligned ones are
constexpr int64_t kMostStride = (int64_t)1 << 22;

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
int64_t held_cols(int64_t vocab) { return up(vocab, kHeadK); }

// What the products need, in one launch: how many labels count and 1 / that (or 1) as the factor of loss and gradients; with
// `place`, the tokens that count numbered in their order: place[token] = number or -1, token_of and kept (its label) the other way round,
// losses of the others 0; no label found yet: label_logit = NaN; x gathered by those numbers, and x and weight with rows padded with
// zeros to 16-byte boundaries.
struct HeadBegin {
    const int64_t* labels;
    int64_t tokens, ignore;
    int mean;
    float lift;
    float *label_logit, *factors, *losses;
    int *rows, *place, *token_of;
    int64_t* kept;
    int each, blocks;             // tokens of a workgroup, and how many workgroups have tokens; the others have rows of weight
    const uint16_t *x, *w;
    int64_t ldx, ldw, vocab;
    int cols, padded;
    uint16_t *x_to, *w_to;        // NULL: read where it is
};
__device__ __forceinline__ void pad_row(const uint16_t* __restrict__ from, int cols, int padded, uint16_t* __restrict__ to) {   // a wave
#pragma unroll 8
    for (int k = (threadIdx.x & 63) * 8; k < padded; k += 64 * 8) {
        const Piece<NTFP8_BF16, 8> v = load_piece<NTFP8_BF16, 8>(from, k, cols - k);
        *reinterpret_cast<v4i*>(to + k) = (v4i){(int)v.w[0], (int)v.w[1], (int)v.w[2], (int)v.w[3]};
    }
}
// Every workgroup counts the labels in front of its own by itself: one after another, a launch that numbers the tokens and one that
// gathers them, took 12 us of a step of 333 tokens and 21 of 4096, this 6 and 17.
__global__ __launch_bounds__(256) void head_begin_kernel(const HeadBegin h) {
    __shared__ uint32_t part[4];
    __shared__ int spot[256];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((int)blockIdx.x >= h.blocks) {   // uniform
        const int64_t step = (int64_t)(gridDim.x - h.blocks) * 4;
        for (int64_t r = (int64_t)(blockIdx.x - h.blocks) * 4 + wave; r < h.vocab; r += step) pad_row(h.w + r * h.ldw, h.cols, h.padded, h.w_to + r * h.padded);
        return;
    }
    const int64_t first = (int64_t)blockIdx.x * h.each, last = std::min(first + h.each, h.tokens);
    const bool gather = h.place != nullptr;
    int64_t before = first;
    if (gather || blockIdx.x == 0) {   // uniform
        // (the first workgroup has none before it, and counts all)
        const int64_t n = blockIdx.x == 0 ? h.tokens : first;
        uint32_t count = 0;
#pragma unroll 8
        for (int64_t i = threadIdx.x; i < n; i += 256) count += h.labels[i] != h.ignore;
        count = wave_fold(count, [](uint32_t a, uint32_t b) { return a + b; });
        if ((threadIdx.x & 63) == 0) part[wave] = count;
        __syncthreads();
        count = part[0] + part[1] + part[2] + part[3];
        __syncthreads();
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            const float f = !h.mean ? 1.0f : count ? 1.0f / (float)count : 0.0f;
            h.factors[0] = f;
            h.factors[1] = f * h.lift;   // of the gradients: dl is kept times 1 / lift
            *h.rows = (int)count;
        }
        before = blockIdx.x == 0 ? 0 : count;
    }
    for (int64_t base = first; base < last; base += 256) {
        const int64_t i = base + threadIdx.x;
        const int64_t label = i < last ? h.labels[i] : h.ignore;
        const bool keep = gather ? label != h.ignore : i < last;
        const uint64_t kept = __ballot(keep);
        if ((threadIdx.x & 63) == 0) part[wave] = __popcll(kept);
        __syncthreads();
        int64_t at = before + __popcll(kept & (((uint64_t)1 << (threadIdx.x & 63)) - 1));
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (w < wave) at += part[w];
            before += part[w];
        }
        spot[threadIdx.x] = keep ? (int)at : -1;
        if (i < last) {
            h.label_logit[i] = __uint_as_float(kNanBits);
            if (gather) {
                h.place[i] = keep ? (int)at : -1;
                if (keep) {
                    h.token_of[at] = (int)i;
                    h.kept[at] = label;
                } else {
                    h.losses[i] = 0.0f;
                }
            }
        }
        __syncthreads();
        if (h.x_to) {
            const int rows = (int)std::min<int64_t>(256, last - base);
            for (int r = wave; r < rows; r += 4) {
                const int to = __builtin_amdgcn_readfirstlane(spot[r]);
                if (to >= 0) pad_row(h.x + (base + r) * h.ldx, h.cols, h.padded, h.x_to + (int64_t)to * h.padded);
            }
        }
        __syncthreads();
    }
}

// A row to a block: its maximum and sum from its pieces, its loss, and dl in the place of its exponentials (rows beyond those
// that count have neither).
// dl = e 2^(piece's maximum - logsumexp) and, at the label, softmax - 1 from the fp32 logit.  T = bf16: the one rounding that
// counts is that of dl to 8 bits of significand, e has 11.  T = fp16: dl is kept times 2^15, as its smallest values
// would fall below fp16's normal numbers.  Bound by memory: 4096 rows of 128000 are read and written in 410 us, 5.1 TB/s.
template <int T, bool kGradient>
__global__ __launch_bounds__(256) void softmax_rows_kernel(const float2* __restrict__ stats, int pieces, const int64_t* __restrict__ labels, int64_t ignore,
                                                           const float* __restrict__ label_logit, float* __restrict__ losses, const int* __restrict__ rows, int row0,
                                                           const int* __restrict__ token_of, uint16_t* held, int64_t ldd) {
    const int64_t row = blockIdx.x;
    if (kGradient && row0 + row >= *rows) return;   // uniform
    const int64_t label = labels[row];
    uint16_t* const d = held + row * ldd;
    float* const own = losses + (kGradient ? token_of[row] : row);
    if (!kGradient && label == ignore) {   // uniform
        if (threadIdx.x == 0) *own = 0.0f;
        return;
    }
    __shared__ float part[4];
    const float2* const p = stats + row * pieces;
    float top = -__builtin_inff();
    for (int i = threadIdx.x; i < pieces; i += 256) top = __builtin_elementwise_maximum(top, p[i].x);
    auto over_waves = [&](float v, auto f) {
        v = __uint_as_float(wave_fold(__float_as_uint(v), [&](uint32_t a, uint32_t b) { return __float_as_uint(f(__uint_as_float(a), __uint_as_float(b))); }));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
        __syncthreads();
        return f(f(part[0], part[1]), f(part[2], part[3]));
    };
    top = over_waves(top, [](float a, float b) { return __builtin_elementwise_maximum(a, b); });
    float sum = 0.0f;
    for (int i = threadIdx.x; i < pieces; i += 256) sum += p[i].y * __builtin_amdgcn_exp2f(p[i].x - top);   // (top -inf or inf: NaN, as the softmax is)
    sum = over_waves(sum, [](float a, float b) { return a + b; });
    const float log_sum = __builtin_amdgcn_logf(sum);   // (base 2; sum >= 1)
    // in base 2, from the maximum down: the logit's product is exact inside the fma
    const float loss = __builtin_fmaf(-label_logit[row], kLog2e, top) + log_sum;
    if (threadIdx.x == 0) *own = loss * 0.693147180559945309417f;
    if constexpr (kGradient) {
        constexpr float kScale = T == NTFP8_BF16 ? 1.0f : 32768.0f;
        const bool bad = loss != loss;   // no such label, or logits that are not numbers: the row says so
        const float lse = bad ? loss : top + log_sum;
        const float at_label = (__builtin_amdgcn_exp2f(-loss) - 1.0f) * kScale;
        for (int64_t c = threadIdx.x * 8; c < ldd; c += 256 * 8) {
            const v4i raw = *reinterpret_cast<const v4i*>(d + c);
            const float f = __builtin_amdgcn_exp2f(p[c / kPieceCols].x - lse) * (kScale * 0x1p-15f);
            v4i out;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float a, b;
                unpack_pair<NTFP8_F16>((uint32_t)raw[k], a, b);
                a *= f;
                b *= f;
                if (c + 2 * k == label) a = at_label;
                if (c + 2 * k + 1 == label) b = at_label;
                out[k] = (int)pack_pair<T>(a, b);
            }
            *reinterpret_cast<v4i*>(d + c) = out;
        }
    }
}

// one workgroup: the losses' sum times the factor
template <int kThreads>
__device__ __forceinline__ void sum_losses(const float* __restrict__ losses, int64_t tokens, const float* __restrict__ factors, float* __restrict__ loss) {
    __shared__ float part[kThreads / 64];
    float s = 0.0f;
#pragma unroll 8
    for (int64_t i = threadIdx.x; i < tokens; i += kThreads) s += losses[i];
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0f;
        for (int w = 0; w < kThreads / 64; ++w) s += part[w];
        *loss = factors[0] == 0.0f ? 0.0f : s * factors[0];
    }
}
__global__ __launch_bounds__(1024) void head_end_kernel(const float* __restrict__ losses, int64_t tokens, const float* __restrict__ factors, float* __restrict__ loss) {
    sum_losses<1024>(losses, tokens, factors, loss);
}

// dx: row place[token] - row0 of what was computed for the tokens that count, zeros for the others (if row0 is 0; the other
// launches of a call leave rows that are not theirs alone).  Computed is the row itself or, with K cut into runs
// (`groups` workgroups, tiles of tile_rows, tiles_n of them across, kt_all K-tiles), the sum of the runs in fp32 times alpha.  With `loss`, one more workgroup sums the losses.
template <int D>
__global__ __launch_bounds__(256) void put_rows_kernel(const void* __restrict__ from, int groups, int tile_rows, int tiles_n, int kt_all, const int* __restrict__ rows,
                                                       const float* __restrict__ factors,
                                                       const int* __restrict__ place, int64_t tokens, int row0, int count, int cols, void* __restrict__ out,
                                                       const float* __restrict__ losses, float* __restrict__ loss) {
    if (loss && blockIdx.x == gridDim.x - 1) {   // uniform
        sum_losses<256>(losses, tokens, factors, loss);
        return;
    }
    const float a = factors[1];
    const int live = max(0, min(*rows - row0, count)), splits = runs_of(groups, (live + tile_rows - 1) / tile_rows * tiles_n, kt_all).splits;
    const int64_t split_stride = (int64_t)live * cols;
    const int chunks = (cols + 7) / 8;
    const int64_t all = tokens * chunks, step = (int64_t)(gridDim.x - (loss ? 1 : 0)) * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
        const int64_t t = i / chunks;
        const int c = (int)(i - t * chunks) * 8, left = cols - c, at = place[t];
        const int64_t r = at - row0;
        if (at < 0 ? row0 != 0 : r < 0 || r >= count) continue;
        float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (at >= 0) {
            if (splits == 1) {
                unpack<D, 8>(load_piece<D, 8>(from, r * cols + c, left), s);
            } else {
#pragma unroll 8
                for (int k = 0; k < splits; ++k) {
                    float v[8];
                    unpack<NTFP8_F32, 8>(load_piece<NTFP8_F32, 8>(from, k * split_stride + r * cols + c, left), v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) s[e] += v[e];
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] *= a;
            }
        }
        store_piece<D, 8>(out, t * cols + c, s, left);
    }
}

struct Scaled {
    const void* x[2];
    void* out[2];
    int64_t n[2];
};
// (as few workgroups as can keep the memory busy: where the factor is 1 the launch is nothing but their coming and going)
template <int S, int D>
__global__ __launch_bounds__(1024) void scale_kernel(const Scaled t, const float* __restrict__ factor) {
    const float f = *factor;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int64_t n = t.n[k];
        if (t.x[k] == t.out[k] && f == 1.0f) continue;
#pragma unroll 4
        for (int64_t i = ((int64_t)blockIdx.x * 1024 + threadIdx.x) * 8; i < n; i += (int64_t)gridDim.x * 8192) {
            const int left = (int)std::min<int64_t>(8, n - i);
            float v[8];
            unpack<S, 8>(load_piece<S, 8>(t.x[k], i, left), v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
            store_piece<D, 8>(t.out[k], i, v, left);
        }
    }
}

template <int T, bool kAT, bool kBT, int EPI>
int launch_gemm(HeadGemm g, int mi, hipStream_t st) {
    g.tiles_n = (int)(((softmax_of(EPI) ? g.ldd : g.N) + kBigN - 1) / kBigN);
    g.magic = magic_of((uint32_t)(kGroupM * g.tiles_n));
    const int64_t tiles = (g.M + 32 * (int64_t)mi - 1) / (32 * mi) * g.tiles_n;
    // (with 256-row tiles up to 128 more, for those of a last round that go in halves; how many is known to the device)
    const unsigned blocks = (unsigned)((EPI == kPartial ? g.groups : tiles) + (mi == 8 ? 128 : 0));
    if constexpr (kAT) {
        head_gemm_kernel<T, kAT, kBT, 8, EPI><<<blocks, kBigThreads, 0, st>>>(g);
    } else {
        if constexpr (EPI == kSoftmax) {
            if (mi == 8 && g.K <= (kLongK - 1) * kHeadK && g.M * g.ldd * 2 > kFoundBytes) {
                head_gemm_kernel<T, kAT, kBT, 8, kSoftmaxThrough><<<blocks, kBigThreads, 0, st>>>(g);
                return launch_status();
            }
        }
        if (mi == 8) head_gemm_kernel<T, kAT, kBT, 8, EPI><<<blocks, kBigThreads, 0, st>>>(g);
        else if (mi == 4) head_gemm_kernel<T, kAT, kBT, 4, EPI><<<blocks, kBigThreads, 0, st>>>(g);
        else if (mi == 2) head_gemm_kernel<T, kAT, kBT, 2, EPI><<<blocks, kBigThreads, 0, st>>>(g);
        else head_gemm_kernel<T, kAT, kBT, 1, EPI><<<blocks, kBigThreads, 0, st>>>(g);
    }
    return launch_status();
}

// What a launch of `tiles` workgroups takes, us, each of `kts` K-tiles of (32 mi) x 256 outputs: rounds of one workgroup a CU, a
// K-tile's time and what a workgroup takes besides.  A K-tile of fewer rows takes more of their share, since the 256 columns
// are the larger part of what it loads.  (Measured at 64 to 2048 tokens, 512 to 4096 hidden, vocabularies of 6 to 50 thousand; with a
// transposed operand a K-tile takes a tenth more.)  A last round of up to 128 tiles of 256 rows goes in halves, a little slower
// than a launch of such tiles (dx of 766 x 1024 from 50001 labels, all of it in halves 80, in tiles of 128 rows 73).
float launch_us(int mi, int64_t tiles, int64_t kts, bool transposed) {
    constexpr float kTile[4] = {0.48f, 0.62f, 0.72f, 1.37f}, kRest[4] = {4.0f, 5.0f, 6.0f, 9.0f};
    auto round = [&](int at) { return (float)kts * kTile[at] * (transposed ? 1.1f : 1.0f) + kRest[at]; };
    const int at = mi == 1 ? 0 : mi == 2 ? 1 : mi == 4 ? 2 : 3;
    const int64_t rest = tiles % 256;
    return (float)(tiles / 256) * round(at) + (rest == 0 ? 0.0f : mi == 8 && rest <= 128 ? 1.08f * round(2) : round(at));
}
int64_t tiles_of(int64_t rows, int64_t cols, int mi) { return (rows + 32 * mi - 1) / (32 * mi) * ((cols + kBigN - 1) / kBigN); }

// Rows of a tile / 32, and runs that K is cut into if all tokens count, for the products with an untransposed A
struct Tiling {
    int mi, splits;
};
// logits: 333 tokens against 6001 rows of 512, us with 256 / 128 / 64 / 32 rows a tile: 21.4, 13.6, 11.6, 16.2; 512 tokens, 32000 rows of 2048: 53.3,
// 58.8, 99.6, 156.9
Tiling tiling_of_logits(int64_t rows, int64_t cols, int64_t kts) {
    Tiling best = {8, 1};
    float least = 1e30f;
    for (int mi = 8; mi >= 1; mi /= 2) {
        const float us = launch_us(mi, tiles_of(rows, cols, mi), kts, false);
        if (us < least) least = us, best.mi = mi;
    }
    return best;
}
// dx: K is the vocabulary, and there are few tiles; runs of K fill the chip, for their fp32 sums' way to memory and back
Tiling tiling_of_dx(int64_t rows, int64_t cols, int64_t kts) {
    Tiling best = {8, 1};
    float least = 1e30f;
    for (int mi = 8; mi >= 1; mi /= 2) {
        const int64_t tiles = tiles_of(rows, cols, mi);
        for (int64_t want = 1; want <= 64 && want <= std::max<int64_t>(1, kts / 4); ++want) {
            const int64_t each = (kts + want - 1) / want, splits = (kts + each - 1) / each;
            if (splits > 1 && tiles * splits > 1024) break;
            float us = launch_us(mi, tiles * splits, each, true);
            if (splits > 1) us += (float)(rows * cols) * (float)splits * 8.0f / 4.5e6f;
            if (us < least) least = us, best = {mi, (int)splits};
        }
    }
    return best;
}

struct Plan {
    int64_t piece;            // tokens at a time
    int64_t ldd, pieces;
    bool pad_x, pad_w;
    int64_t padded;           // hidden, up to a multiple of 8
    Tiling logits, dx;
    int64_t dx_rows;          // tokens at a time of dx's product: with few labels a piece has so many that its sums are the larger part
    int64_t at_factors, at_label, at_place, at_token, at_kept, at_stats, at_held, at_x, at_w, at_dx, bytes;
};
// tokens at a time that `each` bytes of a token allow (and a launch with a row to a block, of fewer than 2^32 threads)
int64_t piece_with(int64_t each) { return std::min<int64_t>(1 << 23, std::max<int64_t>(256, kMostHeld / each / 256 * 256)); }
int64_t piece_of(int64_t vocab) { return piece_with(2 * held_cols(vocab)); }

Plan plan_of(const ntops_linear_cross_entropy_desc& d) {
    Plan p = {};
    const bool gradient = d.dx || d.dweight;
    p.ldd = held_cols(d.vocab);
    p.pieces = (p.ldd + kPieceCols - 1) / kPieceCols;
    // (without gradients nothing is held but 8 bytes for 128 logits)
    p.piece = std::min(d.tokens, gradient ? piece_of(d.vocab) : piece_with(8 * p.pieces));
    p.padded = up(d.hidden, 8);
    // (with gradients the tokens that count are gathered: those that are ignored cost nothing, and what is in them, NaN say, is
    // seen by nobody)
    p.pad_x = gradient || d.hidden % 8 || d.x_stride % 8 || d.x_stride > kMostStride || reinterpret_cast<uintptr_t>(d.x) % 16;
    p.pad_w = d.hidden % 8 || d.weight_stride % 8 || d.weight_stride > kMostStride || reinterpret_cast<uintptr_t>(d.weight) % 16;
    p.logits = tiling_of_logits(p.piece, p.ldd, (p.padded + kHeadK - 1) / kHeadK);
    p.dx_rows = std::min(p.piece, std::max<int64_t>(256, kMostHeld / (4 * d.hidden) / 256 * 256));
    if (d.dx) p.dx = tiling_of_dx(p.dx_rows, d.hidden, p.ldd / kHeadK);
    int64_t at = 0;
    auto room = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 256);
        return here;
    };
    p.at_factors = room(256);
    p.at_label = room(d.tokens * 4);
    if (gradient) {
        p.at_place = room(d.tokens * 4);
        p.at_token = room(d.tokens * 4);
        p.at_kept = room(d.tokens * 8);
    }
    p.at_stats = room(p.piece * p.pieces * 8);
    p.at_held = gradient ? room(p.piece * p.ldd * 2) : 0;
    p.at_x = p.pad_x ? room(d.tokens * p.padded * 2) : 0;
    p.at_w = p.pad_w ? room(d.vocab * p.padded * 2) : 0;
    p.at_dx = d.dx ? room(up(p.dx_rows, 32 * p.dx.mi) * d.hidden * 4 * p.dx.splits) : 0;
    p.bytes = at;
    return p;
}

template <int T>
int run(const ntops_linear_cross_entropy_desc& d, hipStream_t st) {
    const Plan p = plan_of(d);
    char* const ws = static_cast<char*>(d.workspace);
    float* const factors = reinterpret_cast<float*>(ws + p.at_factors);
    float* const label_logit = reinterpret_cast<float*>(ws + p.at_label);
    float2* const stats = reinterpret_cast<float2*>(ws + p.at_stats);
    uint16_t* const held = reinterpret_cast<uint16_t*>(ws + p.at_held);
    const bool gradient = d.dx || d.dweight;
    const char* x = static_cast<const char*>(d.x);
    const char* w = static_cast<const char*>(d.weight);
    int64_t ldx = d.x_stride, ldw = d.weight_stride;
    auto status = [](int rc) { return rc != NTFP8_OK; };
    int* const count = reinterpret_cast<int*>(factors + 2);
    int* const place = gradient ? reinterpret_cast<int*>(ws + p.at_place) : nullptr;
    int* const token_of = gradient ? reinterpret_cast<int*>(ws + p.at_token) : nullptr;
    int64_t* const kept = gradient ? reinterpret_cast<int64_t*>(ws + p.at_kept) : nullptr;
    const int64_t* const labels = gradient ? kept : d.labels;
    HeadBegin b = {};
    b.labels = d.labels, b.tokens = d.tokens, b.ignore = d.ignore_index, b.mean = d.mean, b.lift = T == NTFP8_F16 ? 0x1p-15f : 1.0f;
    b.label_logit = label_logit, b.factors = factors, b.losses = d.losses, b.rows = count, b.place = place, b.token_of = token_of, b.kept = kept;
    b.each = (int)up((d.tokens + 1023) / 1024, 4), b.blocks = (int)((d.tokens + b.each - 1) / b.each);
    b.cols = (int)d.hidden, b.padded = (int)p.padded;
    if (p.pad_x) {
        b.x = reinterpret_cast<const uint16_t*>(x), b.ldx = ldx, b.x_to = reinterpret_cast<uint16_t*>(ws + p.at_x);
        x = ws + p.at_x, ldx = p.padded;
    }
    if (p.pad_w) {
        b.w = reinterpret_cast<const uint16_t*>(w), b.ldw = ldw, b.vocab = d.vocab, b.w_to = reinterpret_cast<uint16_t*>(ws + p.at_w);
        w = ws + p.at_w, ldw = p.padded;
    }
    head_begin_kernel<<<(unsigned)(b.blocks + std::min<int64_t>((b.vocab + 3) / 4, 4096)), 256, 0, st>>>(b);
    if (status(launch_status())) return NTFP8_ERR_LAUNCH;
    for (int64_t row = 0; row < d.tokens; row += p.piece) {
        const int64_t rows = std::min(p.piece, d.tokens - row);
        HeadGemm g = {};
        g.A = x + row * ldx * 2, g.lda = ldx, g.a_cols = (int)p.padded;
        g.B = w, g.ldb = ldw, g.b_cols = (int)p.padded, g.b_rows = 0;
        g.M = (int)rows, g.N = (int)d.vocab, g.K = (int)p.padded;
        g.rows = gradient ? count : nullptr, g.row0 = (int)row;
        g.D = held, g.ldd = p.ldd, g.stats = stats, g.pieces = (int)p.pieces;
        g.labels = labels + row, g.label_logit = label_logit + row;
        if (status(gradient ? launch_gemm<T, false, false, kSoftmax>(g, p.logits.mi, st) : launch_gemm<T, false, false, kLosses>(g, p.logits.mi, st))) return NTFP8_ERR_LAUNCH;
        auto rows_kernel = gradient ? softmax_rows_kernel<T, true> : softmax_rows_kernel<T, false>;
        rows_kernel<<<(unsigned)rows, 256, 0, st>>>(stats, (int)p.pieces, labels + row, d.ignore_index, label_logit + row, gradient ? d.losses : d.losses + row, count, (int)row,
                                                    gradient ? token_of + row : nullptr, held, p.ldd);
        if (status(launch_status())) return NTFP8_ERR_LAUNCH;
        for (int64_t at = 0; d.dx && at < rows; at += p.dx_rows) {
            const int64_t some = std::min(p.dx_rows, rows - at), row0 = row + at;
            float* const loss = row0 + some == d.tokens ? d.loss : nullptr;
            HeadGemm h = {};
            h.A = held + at * p.ldd, h.lda = p.ldd, h.a_cols = (int)p.ldd;
            h.B = w, h.ldb = ldw, h.b_cols = (int)p.padded, h.b_rows = (int)d.vocab;
            h.M = (int)some, h.N = (int)d.hidden, h.K = (int)p.ldd;
            h.rows = count, h.row0 = (int)row0;
            h.D = ws + p.at_dx, h.d_dtype = d.grad_dtype, h.alpha = factors + 1;
            h.groups = (int)tiles_of(some, d.hidden, p.dx.mi) * p.dx.splits;
            if (status(launch_gemm<T, false, true, kPartial>(h, p.dx.mi, st))) return NTFP8_ERR_LAUNCH;
            auto put = d.grad_dtype == T ? put_rows_kernel<T> : put_rows_kernel<NTFP8_F32>;
            const int64_t n = d.tokens * ((d.hidden + 7) / 8);
            put<<<(unsigned)std::min<int64_t>((n + 255) / 256, 8192) + (loss ? 1 : 0), 256, 0, st>>>(
                ws + p.at_dx, h.groups, 32 * p.dx.mi, (int)((d.hidden + kBigN - 1) / kBigN), (int)(p.ldd / kHeadK), count, factors, place, d.tokens, (int)row0, (int)some, (int)d.hidden, d.dx, d.losses, loss);
            if (status(launch_status())) return NTFP8_ERR_LAUNCH;
        }
        if (d.dweight) {
            HeadGemm h = {};
            h.A = held, h.lda = p.ldd, h.a_cols = (int)p.ldd;
            h.B = x + row * ldx * 2, h.ldb = ldx, h.b_cols = (int)p.padded, h.b_rows = (int)rows;
            h.M = (int)d.vocab, h.N = (int)d.hidden, h.K = (int)rows;
            h.rows = count, h.row0 = (int)row;
            h.D = d.dweight, h.d_dtype = d.grad_dtype, h.accumulate = row > 0, h.alpha = factors + 1;
            if (status(launch_gemm<T, true, true, kStore>(h, 8, st))) return NTFP8_ERR_LAUNCH;
        }
    }
    if (d.loss && !d.dx) {
        head_end_kernel<<<1, 1024, 0, st>>>(d.losses, d.tokens, factors, d.loss);
        return launch_status();
    }
    return NTFP8_OK;
}

}  // namespace

int64_t head_piece(int64_t vocab) { return piece_of(vocab); }
int64_t head_workspace(const ntops_linear_cross_entropy_desc& d) { return plan_of(d).bytes; }
int run_head(const ntops_linear_cross_entropy_desc& d, hipStream_t st) { return d.x_dtype == NTFP8_BF16 ? run<NTFP8_BF16>(d, st) : run<NTFP8_F16>(d, st); }

int run_scale(const ntops_scale_tensor* t, int count, int x_dtype, const float* factor, int out_dtype, hipStream_t st) {
    for (int i = 0; i < count; i += 2) {
        Scaled g = {};
        int64_t most = 0;
        for (int k = 0; k < 2 && i + k < count; ++k) {
            g.x[k] = t[i + k].x, g.out[k] = t[i + k].out, g.n[k] = t[i + k].n;
            most = std::max(most, t[i + k].n);
        }
        const unsigned blocks = (unsigned)std::min<int64_t>((most + 8191) / 8192, 2 * cu_count());
        const int rc = with_dtype(x_dtype, [&](auto s) {
            return with_dtype(out_dtype, [&](auto d) {
                scale_kernel<decltype(s)::value, decltype(d)::value><<<blocks, 1024, 0, st>>>(g, factor);
                return launch_status();
            });
        });
        if (rc != NTFP8_OK) return rc;
    }
    return NTFP8_OK;
}

}  // namespace ntfp8

// Matrix products of 16-bit operands for gfx950, in the forms that a projection with a softmax cross entropy needs:
//   logits   A [M, K] rows, B [N, K] rows            x . weight^T, with the softmax's maxima and sums in the epilogue
//   dx       A [M, K] rows, B [K, N] (transposed)    dl . weight
//   dweight  A [K, M] and B [K, N] (transposed)      dl^T . x
//
// Block tile (32 MI) x 256 x 64 (128 bytes of K), four waves in a 2 x 2 arrangement, a wave owning (16 MI) x 128 outputs as MI x 8
// accumulator blocks of V_MFMA_F32_16X16X32.  Tiles travel from memory straight into LDS, 16 bytes a lane, and lie there as
// those of the fp8 GEMM do: rows of 128 bytes with their 16-byte chunks swizzled; a transposed operand as 64 rows of k with 512
// bytes of n (or m) each, its 32-byte pieces swizzled, gathered with the transposing 64-bit LDS read.
//
// bf16, 4096 tokens, 4096 hidden, 128000 labels: logits with their exponentials 3030 us (1.42 PFLOP/s), dx 2920 (1.47), dweight 3220 (1.33);
// by card up to 3 % more.  Bound by energy: the clock falls to 1.77 GHz while 72, 77 and 67 % of the MFMA slots are used, with 8 to 11 % of the
// waves' time spent waiting.  Of 766 tokens, 1024 hidden, 50001 labels 100, 73 and 90 us: 12 to 16 K-tiles a tile, whose first loads and stores nothing hides.
#pragma once
#include "gemm_common.h"
#include "gemm_big.h"
#include "ops_common.h"

namespace ntfp8 {

constexpr int kHeadK = kBK / 2;   // elements of K per LDS stage
constexpr int kPieceCols = 128;   // columns of logits that share a maximum: those of a wave

typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <int T>
__device__ __forceinline__ v4f mfma_16x16x32(v4i b_frag, v4i a_frag, v4f c) {
    // B first: a lane owns 4 consecutive n (n = 4 (lane / 16) + r) of one output row m = lane % 16
    if constexpr (T == NTFP8_BF16) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, b_frag), __builtin_bit_cast(v8bf, a_frag), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, b_frag), __builtin_bit_cast(v8h, a_frag), c, 0, 0, 0);
}

enum HeadEpilogue {
    kStore,     // D = alpha * sums, rounded to d_dtype (fp32: optionally added to D)
    kPartial,   // with K cut into runs, the sums of a run in fp32, D[run][M][N]; of all of K as kStore
    kLosses,    // per row and 128 columns: the largest logit and the sum of exponentials below it; the labels' logits
    kSoftmax,   // the same, and the exponentials themselves in fp16
    kSoftmaxThrough,   // the same, written through to memory
};
constexpr bool softmax_of(int epilogue) { return epilogue >= kLosses; }
constexpr bool keeps(int epilogue) { return epilogue >= kSoftmax; }

// Written through, or left in the L2.  A tile's 128 KB of 16-bit outputs a CU, left in the L2s, are written back while the next round
// of tiles computes; if that takes less time than the memory needs, they are in the way of its loads, and those of the last round
// are at the cost of the kernels behind.  So they are left there where K is long, or where the kernel behind finds them there.  us, through / left:
//   logits, with the pass over their rows: 4096 tokens, 4096 hidden, 128000 labels 3535 / 3475; 2048, 4096, 32000 452 / 440; 4096, 2048,
//   50000 810 / 832; 766, 1024, 50001 133 / 130 and 4 more in the product behind; a step of 256, 2048, 50000 294 / 285
//   logits of 4096 tokens, 50000 labels at 40, 50, 56 and 64 K-tiles 949 / 980, 1121 / 1115, 1209 / 1204, 1357 / 1340; of 128000 at 56 3190 / 3100
//   weight gradients: 128000 x 4096 of 4096 tokens 3294 / 3212; 50001 x 1024 of 766 93 / 93 and 10 more in the kernels behind
//   50000 x 4096 at 24, 40, 56 and 64 K-tiles 528 / 543, 825 / 837, 1088 / 1106, 1262 / 1274; 128000 x 3584 at 64 2815 / 2792
// So logits turn at about 48 K-tiles, weight gradients at 64 or behind, by their size; one bound for both costs either 3 % at most.
constexpr int kLongK = 64;                                // K-tiles
constexpr int64_t kFoundBytes = (int64_t)64 << 20;        // exponentials

struct HeadGemm {
    const void* A;
    const void* B;
    int64_t lda, ldb;            // elements between rows, a multiple of 8; both operands on 16-byte boundaries
    int M, N, K;                 // K: a multiple of 8 unless both operands are transposed
    const int* rows;             // NULL, or how many of the tokens count, known to the device alone, ...
    int row0;                    // ... of which this launch has those from row0 on: M is at most that many, K where A is transposed
    int a_cols, b_cols;          // columns of a row that may be read, a multiple of 8
    int b_rows;                  // rows of a transposed B (K or fewer; those behind count as zeros)
    int tiles_n;
    uint32_t magic;              // magic_of(kGroupM tiles_n)
    int groups;                  // kPartial: workgroups (tiles times runs of K)
    void* D;
    int d_dtype, accumulate;
    const float* alpha;
    // logits
    int64_t ldd;                 // elements between rows of the exponentials, N of them or more (a multiple of 8)
    float2* stats;               // [M][pieces]: base-2 maximum, sum
    int pieces;
    const int64_t* labels;
    float* label_logit;
};

// What a workgroup needs behind its K loop, read in front of it: a launch's arguments are in no cache, and one trip after
// another to them and to what they point to, between the last product and the first store, was a quarter of a small product's time
struct HeadOutput {
    void* D;
    int64_t ldd;
    float2* stats;
    const int64_t* labels;
    float* label_logit;
    float alpha;
    int N, pieces, d_dtype, accumulate;
};
template <int EPI>
__device__ __forceinline__ HeadOutput head_output(const HeadGemm& G) {
    HeadOutput o = {G.D, G.ldd, G.stats, G.labels, G.label_logit, 1.0f, G.N, G.pieces, G.d_dtype, G.accumulate};
    if constexpr (softmax_of(EPI)) {
        asm volatile("" ::"s"(o.D), "s"(o.ldd), "s"(o.stats), "s"(o.labels), "s"(o.label_logit), "s"(o.N), "s"(o.pieces));
    } else {
        o.alpha = *G.alpha;
        asm volatile("" ::"s"(o.D), "s"(o.N), "s"(o.d_dtype), "s"(o.accumulate) : "memory");
    }
    return o;
}

// Runs that K is cut into where there are fewer tiles than workgroups, and K-tiles of each.  The device does it, who knows how many
// tokens count.  us of a step, three of four tokens ignored, with the runs that all tokens would have / so: 2048 tokens, 2048 hidden,
// 32000 labels 357 / 274; 4096, 2048, 50000 1036 / 650; where all count, 4096, 4096, 128000 9935 / 9950 (dx's kernel takes either).
struct HeadRuns {
    int splits, kts;
};
__host__ __device__ __forceinline__ HeadRuns runs_of(int groups, int tiles, int kt_all) {
    if (tiles <= 0 || kt_all <= 0) return {1, kt_all};
    const int most = groups / tiles, want = kt_all / 4 < most ? kt_all / 4 : most, kts = (kt_all + (want > 1 ? want : 1) - 1) / (want > 1 ? want : 1);
    return {(kt_all + kts - 1) / kts, kts};
}

// LDS stages: what fits beside each other in 160 KB
template <int MI>
constexpr int head_stages() { return MI == 8 ? 2 : MI == 1 ? 4 : 3; }

// One operand's loads: `kRows` rows of 128 bytes (or 64 rows of 2 kRows bytes of a transposed one) a K-tile
template <bool kT, int kRows>
struct HeadOperand {
    static constexpr int kLoads = kRows * kBK / 1024 / kBigWaves;   // 1 KB wave-level loads per wave
    static_assert(!kT || kRows == 256 || kRows == 128, "");
    const char* base;
    int64_t step;        // bytes from K-tile to K-tile
    int64_t row_bytes;
    int rows, cols;      // that may be read from base on (transposed: of all of K, from the first column of the matrix on)
    uint32_t off[kLoads];

    __device__ __forceinline__ void init(const void* p, int64_t ld, int first, int count, int readable, int k_rows, int wave, int lane) {
        row_bytes = ld * 2;
        cols = readable;
        if constexpr (kT) {
            base = static_cast<const char*>(p);
            step = kHeadK * row_bytes;
            rows = k_rows;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                // 2 rows of k a wave-level load (4 of a 128-column operand), in chunks of 16 bytes; 32-byte piece c of row k is
                // stored at piece c ^ ((k mod 4) | 4 (k / 16 mod 2)): the 4 rows that one transposing read of 16 lanes touches, and
                // the two groups of 16 lanes that go through LDS together, then use different banks
                constexpr int kChunks = kRows / 8;
                const int k = (wave + kBigWaves * i) * (64 / kChunks) + lane / kChunks;
                const int piece = (lane % kChunks >> 1) ^ ((k & 3) | (((k >> 4) & 1) << 2));
                off[i] = (uint32_t)k * (uint32_t)row_bytes + (uint32_t)first * 2u + (uint32_t)(piece * 32 + (lane & 1) * 16);
            }
        } else {
            base = static_cast<const char*>(p) + (int64_t)first * row_bytes;
            step = kBK;
            rows = min(count, kRows);
            const int chunk = ((lane & 7) ^ (lane >> 3) ^ (wave & 1)) << 4;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) off[i] = (uint32_t)((wave + kBigWaves * i) * 8 + (lane >> 3)) * (uint32_t)row_bytes + chunk;
        }
    }
    // the descriptor of a K-tile; one past the last has no bytes
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t at(int ktile, bool live) const {
        int r = rows;
        if constexpr (kT) r = max(0, min(rows - ktile * kHeadK, kHeadK));
        const uint32_t bytes = live && r > 0 ? (uint32_t)(r - 1) * (uint32_t)row_bytes + (uint32_t)cols * 2u : 0u;
        const char* p = base;
        if constexpr (kT) p += (int64_t)ktile * step;
        return make_rsrc(p, (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes));
    }
    __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, uint8_t* stage, int l, int ktile, int wave) const {
        lds_load16(r, (lds_ptr)(uintptr_t)(stage + (wave + kBigWaves * l) * 1024), off[l], kT ? 0 : ktile * kBK);
    }
    // lanes whose chunk of the last K-tile lies behind K: nothing is read there, zeros instead
    __device__ __forceinline__ void poison() {
        if constexpr (!kT) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) off[i] = kDropped;
        }
    }
};

// Fragment reads.  Plain: block i is 16 rows, 2048 bytes, further on.  Transposed: lane u of a group of 16 (k 16 g .. + 15) addresses
// row k0 + u / 4, columns 4 (u mod 4) .. + 3 of the block's 32-byte piece, and receives rows k0 .. k0 + 3 of column u.
template <bool kT, int kCols>
struct HeadFragment {
    static constexpr int kPitch = 2 * kCols;   // bytes of a row of k of a transposed operand
    int at[2];
    int turn;
    __device__ __forceinline__ void init(int first, int lane) {   // first: row (column) of the wave's block 0 within the tile
        const int g = lane >> 4, u = lane & 15;
        if constexpr (kT) {
            // (a wave's blocks are pieces 0 .. 7 or 8 .. 15 of 16, or 0 .. 3 or 4 .. 7 of 8: the swizzle reaches over 8)
            at[0] = (16 * g + (u >> 2)) * kPitch + (first >> 7) * 256 + (u & 3) * 8;
            at[1] = at[0];
            turn = (((u >> 2) | ((g & 1) << 2)) << 5) ^ (first << 1 & 128);
        } else {
            at[0] = lds_off16(first + u, 2 * g);
            at[1] = lds_off16(first + u, 2 * g + 1);
            turn = 0;
        }
    }
    // half h of block i: k 8 h .. + 7 of the lane group's 16
    __device__ __forceinline__ v4i read(uint8_t* stage, int i, int h) const {
        if constexpr (kT) {
            typedef short v4s __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4s* tr_ptr;
            typedef int v2i __attribute__((ext_vector_type(2)));
            // (one index each: the compiler follows a pointer back to its array over few steps only, and where it does not, it
            // waits for every direct-to-LDS load in flight before the read)
            int off = at[0] + ((i << 5) ^ turn);
            asm("" : "+v"(off));
            const v2i lo = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&stage[off + h * (8 * kPitch)]));
            const v2i hi = __builtin_bit_cast(v2i, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&stage[off + h * (8 * kPitch) + 4 * kPitch]));
            return (v4i){lo.x, lo.y, hi.x, hi.y};
        } else {
            return *reinterpret_cast<const v4i*>(stage + at[h] + i * 2048);
        }
    }
};

__device__ __forceinline__ float lanes_over_rows_max(float v) {   // over lanes l, l ^ 16, l ^ 32, l ^ 48
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __builtin_elementwise_maximum(__uint_as_float(r.x), __uint_as_float(r.y));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(r.x), __uint_as_float(r.y));
}
__device__ __forceinline__ float lanes_over_rows_sum(float v) {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r.x) + __uint_as_float(r.y);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r.x) + __uint_as_float(r.y);
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLift = 15.0f;   // exponentials are kept in fp16 as 2^15 e, 1 at the maximum: 29 binades below it are normal numbers

// Logits of a wave, MI x 8 blocks at rows m_base, columns n_base (a piece of kPieceCols columns).  For each row the largest
// logit (NaN if one is) and the sum of exponentials below it, both in base 2 and fp32; with kKeep the exponentials as well,
// once rounded, which the gradient is later made of by one multiplication a row and piece.
template <int MI, bool kKeep, bool kThrough>
__device__ __forceinline__ void softmax_epilogue(v4f (&acc)[MI][kBigNJ], const HeadOutput& G, int M, int m_base, int n_base, int lane) {
    if (n_base >= (int)G.ldd) return;   // uniform
    const int mrow = lane & 15, q = lane >> 4;
    const float none = -__builtin_inff();
    if (n_base + kPieceCols > G.N) {   // uniform: columns behind the vocabulary count for nothing
#pragma unroll
        for (int j = 0; j < kBigNJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool out = n_base + 16 * j + 4 * q + e >= G.N;
#pragma unroll
                for (int i = 0; i < MI; ++i) acc[i][j][e] = out ? none : acc[i][j][e];
            }
    }
    uint16_t* const D = static_cast<uint16_t*>(G.D);
    const int piece = n_base / kPieceCols;
    // the label's column within this piece, -1 for none; all rows' are asked for at once
    int64_t label[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) label[i] = m_base + 16 * i + mrow < M ? G.labels[m_base + 16 * i + mrow] : -1;
    int rel[MI];
#pragma unroll
    for (int i = 0; i < MI; ++i) rel[i] = label[i] >= n_base && label[i] < min(n_base + kPieceCols, G.N) ? (int)(label[i] - n_base) : -1;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = m_base + 16 * i + mrow;
        float top = acc[i][0][0];
#pragma unroll
        for (int j = 0; j < kBigNJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = __builtin_elementwise_maximum(top, acc[i][j][e]);
        top = lanes_over_rows_max(top);
        if (__any(rel[i] >= 0)) {   // the label's logit
#pragma unroll
            for (int j = 0; j < kBigNJ; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (rel[i] == 16 * j + 4 * q + e) G.label_logit[m] = acc[i][j][e];
        }
        const float base = top == none ? 0.0f : top * kLog2e;
        const float lift = (kKeep ? kLift : 0.0f) - base;
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < kBigNJ; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, lift));
                acc[i][j][e] = p;
                sum += p;
            }
        sum = lanes_over_rows_sum(sum);
        if (q == 0 && m < M) G.stats[(int64_t)m * G.pieces + piece] = make_float2(top == none ? none : base, kKeep ? sum * 0x1p-15f : sum);
        if constexpr (kKeep) {
#pragma unroll
            for (int j = 0; j < kBigNJ; j += 2) {
                // (as 16-bit outputs of the fp8 GEMM: 16 bytes a lane, a full 32-byte sector per row)
                uint32_t x0 = OutT<NTFP8_F16>::pack2(acc[i][j][0], acc[i][j][1]);
                uint32_t x1 = OutT<NTFP8_F16>::pack2(acc[i][j][2], acc[i][j][3]);
                uint32_t y0 = OutT<NTFP8_F16>::pack2(acc[i][j + 1][0], acc[i][j + 1][1]);
                uint32_t y1 = OutT<NTFP8_F16>::pack2(acc[i][j + 1][2], acc[i][j + 1][3]);
                swap_rows16(x0, y0);
                swap_rows16(x1, y1);
                const int n = n_base + (j + (q & 1)) * 16 + (q >> 1) * 8;
                const v4i out = {(int)x0, (int)x1, (int)y0, (int)y1};
                if (m < M && n < (int)G.ldd) {
                    if constexpr (kThrough) store16_through(D + (int64_t)m * G.ldd + n, out);
                    else *reinterpret_cast<v4i*>(D + (int64_t)m * G.ldd + n) = out;
                }
            }
        }
        sched_fence();
    }
}

// Stores of a wave's tile.  Rows of whole pieces go as those of the fp8 GEMM do; others, whose rows begin anywhere, a lane's
// 4 consecutive outputs at a time at whatever address they have (element by element, the weight's gradient of 6001 x 515 in fp32 took
// twice as long).  `stay`: 16-bit outputs are left in the L2.
template <int DT, bool kAcc, int MI>
__device__ __forceinline__ void store_tile(const v4f (&acc)[MI][kBigNJ], void* D, float alpha, int M, int N, int m_base, int n_base, int lane, bool stay = false) {
    if ((N & 7) == 0) {
        // (16 rows at a time: the compiler would have the values of all of them at once, and no registers for them)
        auto rows = [&](auto through, int i) __attribute__((always_inline)) {
            const v4f (&part)[1][kBigNJ] = reinterpret_cast<const v4f (&)[1][kBigNJ]>(acc[i]);
            store_wave_tile16<DT, kAcc, 1, kBigNJ, false, decltype(through)::value>(part, D, alpha, M, N, m_base + 16 * i, n_base, lane);
            sched_fence();
        };
        if (stay) {
#pragma unroll
            for (int i = 0; i < MI; ++i) rows(std::false_type{}, i);
        } else {
#pragma unroll
            for (int i = 0; i < MI; ++i) rows(std::true_type{}, i);
        }
        return;
    }
    const int mrow = lane & 15, q = lane >> 4;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        const int m = m_base + 16 * i + mrow;
        if (m >= M) continue;
#pragma unroll
        for (int j = 0; j < kBigNJ; ++j) {
            const int n = n_base + 16 * j + 4 * q, left = N - n;
            if (left <= 0) continue;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e] * alpha;
            if constexpr (kAcc) {
                float old[4];
                unpack<DT, 4>(load_piece<DT, 4>(D, (int64_t)m * N + n, left), old);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += old[e];
            }
            store_piece<DT, 4>(D, (int64_t)m * N + n, v, left);
        }
        sched_fence();
    }
}

// What the launch's arguments say of sizes, or less of them where the device knows better
struct HeadSizes {
    int M, K, b_rows;
};
template <bool kAT>
__device__ __forceinline__ HeadSizes head_sizes(const HeadGemm& G) {
    HeadSizes z = {G.M, G.K, G.b_rows};
    if (G.rows) {   // uniform
        const int live = __builtin_amdgcn_readfirstlane(max(0, *G.rows - G.row0));   // (loaded by vector: sizes, tiles and descriptors are scalars)
        if constexpr (kAT) {
            z.K = min(z.K, live);
            z.b_rows = min(z.b_rows, live);
        } else {
            z.M = min(z.M, live);
        }
    }
    return z;
}

// The tile of 32 MI x 256 outputs at (m0, n0), K-tiles kt0 .. kt1 - 1 of kt_all.  sA, sB: the LDS stages.
template <int T, bool kAT, bool kBT, int MI, int EPI>
__device__ __forceinline__ void head_tile(const HeadGemm& G, const HeadSizes& z, int m0, int n0, int split, int kt0, int kt1, int kt_all, uint8_t* sA, uint8_t* sB) {
    constexpr int NS = head_stages<MI>(), kStageA = 32 * MI * kBK, kStageB = kBigN * kBK;
    const int M = z.M, K = z.K, b_rows = z.b_rows;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave >> 1) * (MI * 16), wn = (wave & 1) * 128;

    HeadOperand<kAT, 32 * MI> a;
    HeadOperand<kBT, kBigN> b;
    a.init(G.A, G.lda, m0, M - m0, G.a_cols, K, wave, lane);
    b.init(G.B, G.ldb, n0, G.N - n0, G.b_cols, b_rows, wave, lane);
    constexpr int NL = HeadOperand<kAT, 32 * MI>::kLoads + HeadOperand<kBT, kBigN>::kLoads;
    HeadFragment<kAT, 32 * MI> ra;
    HeadFragment<kBT, kBigN> rb;
    ra.init(wm, lane);
    rb.init(wn, lane);
    // chunks of the last K-tile behind K read as zeros, not as the start of the next row
    const bool dead = (kt_all - 1) * kHeadK + (((lane & 7) ^ (lane >> 3) ^ (wave & 1)) << 3) >= K;
    auto poison = [&]() {
        if (dead) {
            a.poison();
            b.poison();
        }
    };
    auto issue = [&](int kt) {   // one K-tile into its stage; tiles behind the last are empty, so that every tile is NL loads
        const bool live = kt < kt1;
        const int s = kt % NS;
        const __amdgpu_buffer_rsrc_t r0 = a.at(kt, live), r1 = b.at(kt, live);
#pragma unroll
        for (int l = 0; l < a.kLoads; ++l) a.load(r0, sA + (s) * kStageA, l, kt, wave);
#pragma unroll
        for (int l = 0; l < b.kLoads; ++l) b.load(r1, sB + (s) * kStageB, l, kt, wave);
    };

    const HeadOutput out = head_output<EPI>(G);
    v4f acc[MI][kBigNJ];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < kBigNJ; ++j) acc[i][j] = (v4f){0.f, 0.f, 0.f, 0.f};
    if constexpr (MI == 8) {
        // Whole tiles: the schedule of the fp8 GEMM's (gemm_big.h), a slot being two MFMAs of 16 cycles where it has one of
        // 32, ordered so that no MFMA waits for the accumulator of the one before it.  front(f), groups 0-5 of K-tile f: the B
        // fragments 2-7 are read behind every other one of the first 24 slots, a barrier releases the stage, and the loads of tile
        // f + 2 go into it, behind every third slot up to the end of back(f); a second barrier publishes tile f + 1.  back(f): groups 6
        // and 7, interleaved per A fragment, which is dead after them and refilled from tile f + 1.
        constexpr int kRelease = 25, kEvery = 3, kFront = (MI * 6 - 1 - kRelease) / kEvery;
        const int n = kt1 - kt0;
        v4i fa[MI][2], fw[kBigNJ][2];
        __amdgpu_buffer_rsrc_t r0, r1;
        auto load = [&](int f, int l) {
            if (l < a.kLoads) a.load(r0, sA + (f & 1) * kStageA, l, kt0 + f, wave);
            else b.load(r1, sB + (f & 1) * kStageB, l - a.kLoads, kt0 + f, wave);
        };
        auto ready = [&](int f) {   // for the loads of tile f
            if (kt0 + f == kt_all - 1) poison();
            r0 = a.at(kt0 + f, f < n);
            r1 = b.at(kt0 + f, f < n);
        };
#pragma unroll
        for (int f = 0; f < 2; ++f) {
            ready(f);
#pragma unroll
            for (int l = 0; l < NL; ++l) load(f, l);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");
        wg_barrier();
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            fa[i][0] = ra.read(sA + (0) * kStageA, i, 0);
            fa[i][1] = ra.read(sA + (0) * kStageA, i, 1);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) fw[h >> 1][h & 1] = rb.read(sB + (0) * kStageB, h >> 1, h & 1);
        for (int f = 0; f < n; ++f) {
            const int s = f & 1;
            ready(f + 2);
            sched_fence();
#pragma unroll
            for (int x = 0; x < MI * 6; ++x) {
                const int j = x / MI, h = x % MI / (MI / 2), i = x % (MI / 2) * 2;
                acc[i][j] = mfma_16x16x32<T>(fw[j][h], fa[i][h], acc[i][j]);
                acc[i + 1][j] = mfma_16x16x32<T>(fw[j][h], fa[i + 1][h], acc[i + 1][j]);
                if (x < 24 && x % 2 == 0) fw[2 + x / 4][x / 2 % 2] = rb.read(sB + (s) * kStageB, 2 + x / 4, x / 2 % 2);
                if (x == kRelease) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // every fragment of tile f is in registers
                    wg_barrier();
                }
                if (x > kRelease && (x - kRelease) % kEvery == 0) load(f + 2, (x - kRelease) / kEvery - 1);
                sched_fence();
            }
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kFront) : "memory");   // all but tile f + 2's
            wg_barrier();
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                acc[i][6] = mfma_16x16x32<T>(fw[6][0], fa[i][0], acc[i][6]);
                acc[i][7] = mfma_16x16x32<T>(fw[7][0], fa[i][0], acc[i][7]);
                if (i > 0) {
                    fa[i - 1][0] = ra.read(sA + (s ^ 1) * kStageA, i - 1, 0);
                    fa[i - 1][1] = ra.read(sA + (s ^ 1) * kStageA, i - 1, 1);
                }
                sched_fence();
                acc[i][6] = mfma_16x16x32<T>(fw[6][1], fa[i][1], acc[i][6]);
                acc[i][7] = mfma_16x16x32<T>(fw[7][1], fa[i][1], acc[i][7]);
                if (i < 4) fw[i >> 1][i & 1] = rb.read(sB + (s ^ 1) * kStageB, i >> 1, i & 1);
#pragma unroll
                for (int l = kFront + i * (NL - kFront) / MI; l < kFront + (i + 1) * (NL - kFront) / MI; ++l) load(f + 2, l);
                sched_fence();
            }
            fa[MI - 1][0] = ra.read(sA + (s ^ 1) * kStageA, MI - 1, 0);
            fa[MI - 1][1] = ra.read(sA + (s ^ 1) * kStageA, MI - 1, 1);
            sched_fence();
        }
    } else if constexpr (MI == 4) {
        // Half tiles: the schedule of the fp8 GEMM's, three stages and one barrier a K-tile.  front: groups 0-5, the B fragments
        // read three groups ahead; the barrier behind it releases this K-tile's stage and publishes the next one.  back: groups
        // 6 and 7, whose A fragments are refilled from the next K-tile.  The loads of the K-tile after next but one go into the
        // released stage, a third during back, the others during the next front.
        constexpr int kBackLoads = NL / 3, kFrontLoads = NL - kBackLoads, kSlots = 5 * (MI / 2);
        const int n = kt1 - kt0;
        v4i fa[MI][2], fb[4][2];
        __amdgpu_buffer_rsrc_t r0, r1;
        int coming = 0, to = 0;   // the K-tile being loaded, and its stage
        auto ready = [&](int f) {
            if (kt0 + f == kt_all - 1) poison();
            coming = kt0 + f;
            to = f % NS;
            r0 = a.at(kt0 + f, f < n);
            r1 = b.at(kt0 + f, f < n);
        };
        auto load = [&](int l) {
            if (l < a.kLoads) a.load(r0, sA + (to) * kStageA, l, coming, wave);
            else b.load(r1, sB + (to) * kStageB, l - a.kLoads, coming, wave);
        };
#pragma unroll
        for (int f = 0; f < NS; ++f) {
            ready(f);
#pragma unroll
            for (int l = 0; l < NL; ++l) load(l);
        }
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * NL) : "memory");
        wg_barrier();
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            fa[i][0] = ra.read(sA + (0) * kStageA, i, 0);
            fa[i][1] = ra.read(sA + (0) * kStageA, i, 1);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) fb[h >> 1][h & 1] = rb.read(sB + (0) * kStageB, h >> 1, h & 1);
        auto front = [&](auto loads_tag, int s) __attribute__((always_inline)) {
            constexpr bool loads = decltype(loads_tag)::value;
            sched_fence();
#pragma unroll
            for (int j = 0; j < 6; ++j) {
#pragma unroll
                for (int x = 0; x < MI; ++x) {   // two MFMAs each, neither on the accumulator of the one before
                    const int h = x / (MI / 2), i = x % (MI / 2) * 2;
                    acc[i][j] = mfma_16x16x32<T>(fb[j & 3][h], fa[i][h], acc[i][j]);
                    acc[i + 1][j] = mfma_16x16x32<T>(fb[j & 3][h], fa[i + 1][h], acc[i + 1][j]);
                    // B fragment j + 3 (behind group 0 fragments 2 and 3), so that none is on its way at the barrier
                    if (x < 2 && j < 5) fb[(j + (j ? 3 : 2)) & 3][x] = rb.read(sB + (s) * kStageB, j + (j ? 3 : 2), x);
                    else if (j == 0) fb[3][x - 2] = rb.read(sB + (s) * kStageB, 3, x - 2);
                    if (loads && j > 0 && x >= 2) {
                        const int y = (j - 1) * (MI - 2) + x - 2;
#pragma unroll
                        for (int l = kBackLoads + y * kFrontLoads / kSlots; l < kBackLoads + (y + 1) * kFrontLoads / kSlots; ++l) load(l);
                    }
                    sched_fence();
                }
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NL) : "memory");   // all but the newest K-tile
            wg_barrier();
        };
        auto back = [&](int next) __attribute__((always_inline)) {   // next: stage of the K-tile behind this one
            sched_fence();
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                acc[i][6] = mfma_16x16x32<T>(fb[2][0], fa[i][0], acc[i][6]);
                acc[i][7] = mfma_16x16x32<T>(fb[3][0], fa[i][0], acc[i][7]);
                if (i > 0) {
                    fa[i - 1][0] = ra.read(sA + (next) * kStageA, i - 1, 0);
                    fa[i - 1][1] = ra.read(sA + (next) * kStageA, i - 1, 1);
                }
                sched_fence();
                acc[i][6] = mfma_16x16x32<T>(fb[2][1], fa[i][1], acc[i][6]);
                acc[i][7] = mfma_16x16x32<T>(fb[3][1], fa[i][1], acc[i][7]);
#pragma unroll
                for (int l = i * kBackLoads / MI; l < (i + 1) * kBackLoads / MI; ++l) load(l);
                fb[i >> 1][i & 1] = rb.read(sB + (next) * kStageB, i >> 1, i & 1);
                sched_fence();
            }
            fa[MI - 1][0] = ra.read(sA + (next) * kStageA, MI - 1, 0);
            fa[MI - 1][1] = ra.read(sA + (next) * kStageA, MI - 1, 1);
            sched_fence();
        };
        front(std::false_type{}, 0);   // (K-tile 3 goes into the stage that it still reads)
        int s = 0;
        for (int f = 1; f < n; ++f) {
            const int next = s == NS - 1 ? 0 : s + 1;
            ready(f + 2);
            back(next);
            front(std::true_type{}, next);
            s = next;
        }
        back(s == NS - 1 ? 0 : s + 1);   // (loads nothing more: the last of them are those of an empty K-tile again)
    } else {
#pragma unroll
        for (int l = 0; l < NS - 1; ++l) {
            if (kt0 + l == kt_all - 1) poison();
            issue(kt0 + l);
        }
        for (int kt = kt0; kt < kt1; ++kt) {
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 2) * NL) : "memory");   // this tile has landed ...
            wg_barrier();                                                          // ... for every wave, and all are done with the one before
            if (kt + NS - 1 == kt_all - 1) poison();
            issue(kt + NS - 1);
            const int s = kt % NS;
            v4i fa[MI][2], fb[2];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                fa[i][0] = ra.read(sA + (s) * kStageA, i, 0);
                fa[i][1] = ra.read(sA + (s) * kStageA, i, 1);
            }
#pragma unroll
            for (int j = 0; j < kBigNJ; ++j) {
                fb[0] = rb.read(sB + (s) * kStageB, j, 0);
                fb[1] = rb.read(sB + (s) * kStageB, j, 1);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int i = 0; i < MI; ++i) acc[i][j] = mfma_16x16x32<T>(fb[h], fa[i][h], acc[i][j]);
            }
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the empty tiles too: nothing may land in LDS behind the workgroup)

    if constexpr (softmax_of(EPI)) {
        softmax_epilogue<MI, keeps(EPI), EPI == kSoftmaxThrough>(acc, out, M, m0 + wm, n0 + wn, lane);
    } else {
        const bool part = EPI == kPartial && kt1 - kt0 < kt_all;
        void* const D = part ? static_cast<float*>(out.D) + (int64_t)split * M * out.N : out.D;
        const float alpha = part ? 1.0f : out.alpha;
        if (!part && out.d_dtype == T) store_tile<T, false, MI>(acc, D, alpha, M, out.N, m0 + wm, n0 + wn, lane, EPI == kPartial || kt_all >= kLongK);   // (dx: put_rows_kernel reads it next)
        else if (EPI == kStore && out.accumulate) store_tile<NTFP8_F32, true, MI>(acc, D, alpha, M, out.N, m0 + wm, n0 + wn, lane);
        else store_tile<NTFP8_F32, false, MI>(acc, D, alpha, M, out.N, m0 + wm, n0 + wn, lane);
    }
}

template <int T, bool kAT, bool kBT, int MI, int EPI>
__global__ __launch_bounds__(kBigThreads) void head_gemm_kernel(const HeadGemm G) {
    // 256-row tiles that do not fill a last round (kTail): its tiles in halves of 128 rows, twice the workgroups for half as long.
    // us, whole / so: weight gradients of 6001 x 515 from 333 tokens 18.3 / 13.1, of 50001 x 1024 from 766 101 / 95, of 128000 x 4096 from 4096 3404 / 3300
    constexpr bool kTail = MI == 8;
    constexpr int kBytesA = head_stages<MI>() * 32 * MI * kBK, kBytesB = head_stages<kTail ? 4 : MI>() * kBigN * kBK;
    __shared__ __attribute__((aligned(1024))) uint8_t sA[kBytesA];
    __shared__ __attribute__((aligned(1024))) uint8_t sB[kBytesB];
    static_assert(!kTail || kBytesA >= head_stages<4>() * 128 * kBK, "half tiles use the same arrays");
    const HeadSizes z = head_sizes<kAT>(G);
    if (kAT && G.accumulate && z.K == 0) return;
    const int tiles_m = (z.M + 32 * MI - 1) / (32 * MI), tiles = tiles_m * G.tiles_n;
    const int kt_all = (z.K + kHeadK - 1) / kHeadK;
    HeadRuns runs = {1, kt_all};
    if constexpr (EPI == kPartial) {   // (quotients are vector arithmetic: what descriptors are made of is scalar)
        runs = runs_of(G.groups, tiles, kt_all);
        runs.splits = __builtin_amdgcn_readfirstlane(runs.splits);
        runs.kts = __builtin_amdgcn_readfirstlane(runs.kts);
    }
    const int total = tiles * runs.splits;
    int pid = blockIdx.x, pid_m, pid_n;
    auto place = [&](int tile) {   // -> its run of K
        const int split = EPI == kPartial ? __builtin_amdgcn_readfirstlane(tile / tiles) : 0;
        tile_in_group(EPI == kPartial ? tile - split * tiles : tile, tiles_m, G.tiles_n, G.magic, pid_m, pid_n);
        return split;
    };
    if constexpr (kTail) {
        const int rest = total & 255, whole = rest > 128 ? total : total - rest;
        if (pid >= whole) {
            const int half = pid - whole;
            if (rest > 128 || half >= 2 * rest) return;
            const int at = run_of_xcd(half, 2 * rest), split = place(whole + (at >> 1)), kt0 = split * runs.kts;
            const int m0 = pid_m * 256 + (at & 1) * 128;
            if (m0 < z.M) head_tile<T, kAT, kBT, 4, EPI>(G, z, m0, pid_n * kBigN, split, kt0, min(kt_all, kt0 + runs.kts), kt_all, sA, sB);
            return;
        }
    }
    // Within each round of 256 workgroups an XCD takes a contiguous run of the tiles
    if (pid >= total) return;
    const int round0 = pid & ~255, split = place(round0 + run_of_xcd(pid - round0, min(256, total - round0))), kt0 = split * runs.kts;
    head_tile<T, kAT, kBT, MI, EPI>(G, z, pid_m * 32 * MI, pid_n * kBigN, split, kt0, min(kt_all, kt0 + runs.kts), kt_all, sA, sB);
}

}  // namespace ntfp8

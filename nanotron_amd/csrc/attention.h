// What the attention kernels share: the spans that workgroups serve, tiles of rows in LDS and their fragments, products and stores.
//
// Every product is taken so that the 32 rows that a wave owns (queries, or keys in the pass for dk and dv) are the columns of
// V_MFMA_F32_32X32X16's result, one a lane: a row's maximum, sum, logsumexp and limit of a mask are then one register, its
// scores lie in that lane and lane ^ 32, and the scores, rounded to 16 bits, are the second operand of the next product as they
// lie: its 16 places of k are taken in the order in which the result registers hold them, 4 h + j and 8 + 4 h + j of half
// wave h, and the other operand, transposed out of LDS four rows at a time, is read in that order too.
#pragma once
#include "gemm_common.h"
#include "ops_common.h"

namespace ntfp8 {

typedef __bf16 v8bf_attn __attribute__((ext_vector_type(8)));
typedef _Float16 v8h_attn __attribute__((ext_vector_type(8)));
typedef int v2i_attn __attribute__((ext_vector_type(2)));

constexpr int kAttnStep = 64;               // rows of a tile in LDS
constexpr int kAttnWaves = 4, kAttnQueries = 32 * kAttnWaves;   // of the kernels that own queries
constexpr int kAttnKeyWaves = 4, kAttnKeyStep = 32;   // of the kernel that owns keys: its waves, the rows of its tiles of queries, and its keys
constexpr int kAttnKeys = 32 * kAttnKeyWaves;
// Workgroups of both that a CU holds: three of short heads, whose sums take half the registers (168 of each lane; 16 heads of 64, forward, 4 sequences of
// 4096 in bf16 341 us for 362 with two, backward 4 of 4096 in fp16 590 us for 640), two of the others
constexpr int attn_workgroups(int padded_dim) { return padded_dim <= 64 ? 3 : 2; }
constexpr uint32_t kNowhere = 0xfffffff0u;  // past every descriptor: reads as zeros
constexpr int kAttnMost = 1024;             // workgroups that look for the largest magnitudes, of dout and of v
constexpr float kLog2E = 1.44269504088896340736f;

// A run of rows of one sequence that a workgroup owns, and the other side's rows that belong to it
struct AttnTask {
    int own, rows;     // first row (counted over all sequences), and how many
    int other, len;    // first row of the other side's sequence, and its length
    int at, seq;       // first row within its sequence
    int shift;         // own queries: row i sees the keys 0 .. shift + i; own keys: key i is seen by the queries shift + i and behind
    int pad;
};

struct AttnArgs {
    const void *q, *k, *v, *dout;
    int64_t q_stride, k_stride, v_stride, do_stride;   // elements between rows,
    int64_t q_head, k_head, v_head, do_head;           // heads
    int64_t q_batch, k_batch, v_batch, do_batch;       // and sequences of equal lengths
    const AttnTask* tasks;                             // or NULL: `sequences` of q_len and k_len rows
    int64_t tiles;
    int tile_heads;   // heads of a group that the waves of a workgroup take (of 32 queries), 1: all its waves take one (of 128)
    int sequences, q_len, k_len;
    int64_t q_rows, k_rows;
    int heads, kv_heads, group, dim, causal;
    float c;           // scale * log2(e)
    float scale;
    void* out;
    const void* o;     // backward: the output of the forward pass
    uint8_t* low;      // of every element of out the 8 bits behind those that its rounding kept, where a backward pass follows (or NULL)
    float* lse;        // [heads][q_rows] minus the logarithm of a row's sum of exponentials, in units of q k^T; minus infinity for a row that sees nothing
    float* delta;      // [heads][q_rows] minus the sum of dout out
    uint32_t* most;    // fp16 gradients: bits of the largest magnitudes in dout and v, of each workgroup that looked, [2][kAttnMost]
    int most_q, most_v;   // and how many looked
    void *dq, *dk, *dv;
    int splits;        // runs that the keys of a tile are cut into ...
    float* part;       // ... and their results before they are joined: [split][q_rows][heads][dim], then
    float2* part_ml;   // [split][q_rows][heads] maximum (base 2) and sum
    // dk and dv: runs that the queries of a tile of keys are cut into, and their sums before they are added up: [split][dk, dv][k_rows][kv_heads][dim]
    int k_splits;
    float* k_part;
};

// workgroups that the heads of a group are
__host__ __device__ constexpr int attn_chunks(int group, int tile_heads) { return (group + tile_heads - 1) / tile_heads; }
// The task of tile `t`.  Under a causal mask the longest come first; else those of a sequence one behind the other, while its keys are in the L2 (16 sequences
// of 1024, 16 heads of 128, forward 192 -> 168 us; causal 64 sequences of 512, both passes, would lose 2 %)
__device__ __forceinline__ AttnTask attn_task(const AttnArgs& A, int t, int tile_rows, bool keys) {
    if (A.tasks) {
        AttnTask r = A.tasks[t];
        r.rows = __builtin_amdgcn_readfirstlane(r.rows);
        r.own = __builtin_amdgcn_readfirstlane(r.own);
        r.other = __builtin_amdgcn_readfirstlane(r.other);
        r.len = __builtin_amdgcn_readfirstlane(r.len);
        r.at = __builtin_amdgcn_readfirstlane(r.at);
        r.seq = __builtin_amdgcn_readfirstlane(r.seq);
        r.shift = __builtin_amdgcn_readfirstlane(r.shift);
        return r;
    }
    const int own_len = keys ? A.k_len : A.q_len, len = keys ? A.q_len : A.k_len;
    const int per = (own_len + tile_rows - 1) / tile_rows, seq = A.causal ? t % A.sequences : t / per, rank = A.causal ? t / A.sequences : t % per;
    const int at = (keys ? rank : per - 1 - rank) * tile_rows;
    return {seq * own_len + at, min(tile_rows, own_len - at), seq * len, len, at, seq, keys ? at - (A.k_len - A.q_len) : at + A.k_len - A.q_len, 0};
}
// What a wave of the kernels that own queries has: tile, head of keys, head inside its group, first row in the tile.  Either its workgroup's waves share a head
// and take 32 of 128 rows each, or the same 32 rows of heads of their own (the last ones may have none).  Heads that share keys go to one XCD:
// workgroups are dealt to the eight in turn.
struct AttnOwn {
    int tile, kv, inside, row;
};
__device__ __forceinline__ AttnOwn attn_own(const AttnArgs& A, int group, int wave) {
    const bool shared = A.tile_heads > 1;
    const int picks = A.kv_heads * attn_chunks(A.group, A.tile_heads), tile = group / picks, pick = group - tile * picks, chunk = pick / A.kv_heads;
    return {tile, pick - chunk * A.kv_heads, chunk * A.tile_heads + (shared ? wave : 0), shared ? 0 : wave * 32};
}
// element offset of a run of rows: packed ones are counted over all sequences, others within theirs
__device__ __forceinline__ int64_t attn_rows(const AttnArgs& A, int64_t packed, int seq, int at, int64_t stride, int64_t batch) {
    return A.tasks ? packed * stride : seq * batch + at * stride;
}

template <int T>
__device__ __forceinline__ v16f mfma_attn(v4i rows, v4i cols, v16f c) {   // result: row (register) of `rows`, column (lane) of `cols`
    if constexpr (T == NTFP8_BF16) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf_attn, rows), __builtin_bit_cast(v8bf_attn, cols), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h_attn, rows), __builtin_bit_cast(v8h_attn, cols), c, 0, 0, 0);
}
__device__ __forceinline__ v16f zeros16() { return (v16f){0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0}; }
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// kRows rows of DP elements in LDS, 16-byte chunks swizzled so that neither 8 rows' reads of one chunk nor the transposing reads of 4
// rows' 64 bytes meet in a bank
template <int DP, int kRows = kAttnStep>
struct AttnTile {
    static constexpr int kPitch = DP <= 64 ? 128 : 256, kBytes = kRows * kPitch;
    static __device__ __forceinline__ int swizzle(int row) {
        if constexpr (kPitch == 128) return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
        else return (row & 3) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1);
    }
    // loads: 1 KB a wave each, straight into LDS, by kWaves waves
    template <int kWaves = kAttnWaves>
    struct Source {
        static constexpr int kLoads = kBytes / 1024 / kWaves;
        const char* base;
        uint32_t row_bytes;   // (2^25 at most)
        uint32_t off[kLoads];
        int dim;
        __device__ __forceinline__ void init(const void* p, int64_t elements, int64_t stride, int dim_, int wave, int lane) {
            base = static_cast<const char*>(p) + 2 * elements;
            row_bytes = (uint32_t)(2 * stride);
            dim = dim_;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int byte = ((i * kWaves + wave) * 64 + lane) * 16, row = byte / kPitch, chunk = (byte % kPitch >> 4) ^ swizzle(row);
                off[i] = chunk * 8 < dim ? (uint32_t)row * row_bytes + chunk * 16 : kNowhere;
            }
        }
        // rows first .. of `len`, those behind it as zeros
        __device__ __forceinline__ void load(uint8_t* stage, int first, int len, int wave) const {
            const int rows = min(kRows, len - first);
            const uint32_t bytes = rows > 0 ? (uint32_t)(rows - 1) * row_bytes + 2u * dim : 0u;
            const __amdgpu_buffer_rsrc_t r = make_rsrc(base + (uint64_t)(uint32_t)first * row_bytes, (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes));
#pragma unroll
            for (int i = 0; i < kLoads; ++i) lds_load16(r, (lds_ptr)(uintptr_t)(stage + (i * kWaves + wave) * 1024), off[i], 0);
        }
    };
    // fragments: 32 rows by 16 elements as they lie, and 16 rows by 32 elements transposed
    int plain, plain_turn, across, across_turn;
    __device__ __forceinline__ void init(int lane) {
        const int row = lane & 31, h = lane >> 5, u = lane & 15, first = 4 * h + (u >> 2);
        plain = row * kPitch;
        plain_turn = (h ^ swizzle(row)) << 4;
        across = first * kPitch + (u & 1) * 8;
        across_turn = ((((lane >> 4) & 1) * 2 + ((u & 3) >> 1)) ^ swizzle(first)) << 4;
    }
    // rows 32 b .., elements 16 k ..
    __device__ __forceinline__ v4i rows(const uint8_t* stage, int b, int k) const {
        return *reinterpret_cast<const v4i*>(stage + plain + ((k << 5) ^ plain_turn) + b * 32 * kPitch);
    }
    // elements 32 e .. of the rows 16 s .., in the order of the result registers
    __device__ __forceinline__ v4i columns(uint8_t* stage, int s, int e) const {
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4s* tr_ptr;
        const int lo = across + ((e << 6) ^ across_turn) + s * 16 * kPitch, hi = (across + ((e << 6) ^ across_turn ^ 16)) + (s * 16 + 8) * kPitch;
        const v2i_attn a = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&stage[lo]));
        const v2i_attn b = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&stage[hi]));
        return (v4i){a.x, a.y, b.x, b.y};
    }
    // The same of the stage that begins at byte `at` of an array, for kernels without registers to keep each fragment's address in: an
    // exclusive or and an addition a read, which the compiler is kept from doing once and for all
    __device__ __forceinline__ v4i rows_anew(const uint8_t* array, int at, int b, int k) const {
        int off = (plain + plain_turn) ^ (k << 5);
        asm volatile("" : "+v"(off));
        off += at;
        return *reinterpret_cast<const v4i*>(array + off + b * 32 * kPitch);
    }
    __device__ __forceinline__ v4i columns_anew(uint8_t* array, int at, int s, int e) const {
        typedef short v4s __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) v4s* tr_ptr;
        int lo = (across + across_turn) ^ (e << 6);
        asm volatile("" : "+v"(lo));
        lo += at;
        int hi = lo ^ 16;
        asm volatile("" : "+v"(hi));
        const v2i_attn a = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&array[lo + s * 16 * kPitch]));
        const v2i_attn b = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)&array[hi + (s * 16 + 8) * kPitch]));
        return (v4i){a.x, a.y, b.x, b.y};
    }
};

// 32 rows of global memory as the second operand: row `row` of each lane, 16 elements a fragment.  `live`: the row exists
template <int DP>
__device__ __forceinline__ void load_own(v4i (&f)[DP / 16], const void* p, int64_t element, int dim, bool live, int lane) {
    const char* const at = static_cast<const char*>(p) + 2 * element;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
        const int e = 16 * k + 8 * (lane >> 5);
        f[k] = live && e < dim ? *reinterpret_cast<const v4i*>(at + 2 * e) : (v4i){0, 0, 0, 0};
    }
}
// 8 result registers (16 places of k) as a fragment of the second operand
template <int T>
__device__ __forceinline__ v4i pack_scores(const v16f& s, int first) {
    return (v4i){(int)pack_pair<T>(s[first], s[first + 1]), (int)pack_pair<T>(s[first + 2], s[first + 3]), (int)pack_pair<T>(s[first + 4], s[first + 5]),
                 (int)pack_pair<T>(s[first + 6], s[first + 7])};
}
// the place in its block of 32 of a result register
__device__ __forceinline__ int place_of(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }
// and what is left of it without the lane's share, for comparisons with a bound that holds that share, once a tile: sixteen places made in front
// of a loop are spilled, and waited for behind the loads of the next tile
__device__ __forceinline__ constexpr int place_in_half(int r) { return 8 * (r >> 2) + (r & 3); }

// Whether what a wave loaded of a stage (its pieces of 1 KB, see Source; all of them where kWaves is 1) holds a value that is not finite: the
// largest magnitude of the pairs of 16 bits, in integers.  Where waves share a stage each looks at its own part, which its own wait has brought, and
// leaves the answer in front of the barrier: every wave looking at the whole stage took three times as long as its products.
template <int T, int DP, int kRows, int kWaves>
__device__ __forceinline__ bool attn_not_finite(const uint8_t* stage, int wave, int lane) {
    typedef unsigned short v2us __attribute__((ext_vector_type(2)));
    constexpr int kLoads = AttnTile<DP, kRows>::kBytes / 1024 / kWaves;
    v2us most = {0, 0};
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const v4i x = *reinterpret_cast<const v4i*>(stage + (i * kWaves + wave) * 1024 + lane * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) most = __builtin_elementwise_max(most, __builtin_bit_cast(v2us, x[w] & 0x7fff7fff));
    }
    constexpr unsigned short kInf = T == NTFP8_BF16 ? 0x7f80 : 0x7c00;
    return __any(most.x >= kInf || most.y >= kInf);
}
// A wave's answer for all of them, behind the next barrier, and theirs
__device__ __forceinline__ void attn_tell(int (&odd)[kAttnWaves], int wave, bool mine) {
    odd[wave] = mine;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
}
__device__ __forceinline__ bool attn_any_wave(const int (&odd)[kAttnWaves]) {
    int any = 0;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) any |= odd[w];
    return __builtin_amdgcn_readfirstlane(any);
}
// acc (elements by own rows) += columns of a stage's rows 16 s .. * scores
template <int T, int DP>
__device__ __forceinline__ void add_columns(v16f (&acc)[DP / 32], const AttnTile<DP>& tile, uint8_t* stage, int s, v4i scores) {
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) acc[e] = mfma_attn<T>(tile.columns(stage, s, e), scores, acc[e]);
}
// The same over the 16 kScores rows of a stage that holds values which are not finite, under a mask: a score of zero times such a value would
// reach the rows that do not count it (a padded row, a token to come), so the stage's rows go one at a time, and only into the
// rows that count them: this lane's row counts the rows from .. to - 1.  A function of its own, which finds the sums in memory: beside the loops of
// the kernels it would take the registers that they live from (240 of 256 in the forward pass with it, 102 spilled, 450 TFLOP/s for 990).
template <int DP, int kScores>
struct AttnSingly {
    v16f acc[DP / 32];
    v4i scores[kScores];
};
template <int T, int DP, int kScores, int kRows>
__device__ __attribute__((noinline)) void attn_add_singly(AttnSingly<DP, kScores>* w, uint32_t stage, int from, int to) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s* tr_ptr;
    typedef AttnTile<DP, kRows> Tile;
    const int lane = threadIdx.x & 63;
    Tile tile;
    tile.init(lane);
#pragma unroll 1
    for (int e = 0; e < DP / 32; ++e) {
        v16f acc = w->acc[e];
#pragma unroll 1
        for (int i = 0; i < 16 * kScores; ++i) {
            const int s = i >> 4, j = (i & 3) + ((i >> 3) & 1) * 4;   // its place in the fragments of half wave (i >> 2) & 1
            const bool mine = (lane >> 5) == ((i >> 2) & 1), take = i >= from && i < to;
            const uint32_t lo = stage + ((tile.across + tile.across_turn) ^ (e << 6)) + s * 16 * Tile::kPitch;
            const uint32_t hi = stage + ((tile.across + tile.across_turn) ^ (e << 6) ^ 16) + (s * 16 + 8) * Tile::kPitch;
            const v2i_attn a = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(uintptr_t)lo));
            const v2i_attn b = __builtin_bit_cast(v2i_attn, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr_ptr)(uintptr_t)hi));
            v4i f = {a.x, a.y, b.x, b.y};
#pragma unroll
            for (int k = 0; k < 4; ++k) f[k] = mine && (j >> 1) == k ? (j & 1 ? f[k] & (int)0xffff0000 : f[k] & 0xffff) : 0;
            const v16f d = mfma_attn<T>(f, w->scores[s], zeros16());
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[r] += take ? d[r] : 0.0f;
        }
        w->acc[e] = acc;
    }
}
template <int T, int DP, int kScores, typename Tile>
__device__ __forceinline__ void add_columns_singly(v16f (&acc)[DP / 32], const Tile&, uint8_t* stage, const v4i (&scores)[kScores], int from, int to) {
    AttnSingly<DP, kScores> w;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) w.acc[e] = acc[e];
#pragma unroll
    for (int k = 0; k < kScores; ++k) w.scores[k] = scores[k];
    attn_add_singly<T, DP, kScores, Tile::kBytes / Tile::kPitch>(&w, (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)stage, from, to);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) acc[e] = w.acc[e];
}

// What rounding x to T left out, as 8 more bits of significand: the difference of their bit patterns as fp32, in steps of 2^-8 of one of T's.
// The backward pass subtracts the sum of dout out from every dout v^T; made of the rounded out alone it brings a fifth of dq's and dk's error.
template <int T>
constexpr int kLowShift = T == NTFP8_BF16 ? 8 : 5;
template <int T>
__device__ __forceinline__ uint32_t low_bits(float x, float rounded) {
    const int r = (int)(__float_as_uint(x) - __float_as_uint(rounded));
    const int code = max(-128, min(127, (r + (1 << (kLowShift<T> - 1))) >> kLowShift<T>));
    return (__float_as_uint(rounded) & 0x7fffffffu) < kInfBits ? (uint32_t)code & 0xffu : 0u;
}
template <int T>
__device__ __forceinline__ float with_low(float rounded, uint32_t code) {
    return __uint_as_float(__float_as_uint(rounded) + (uint32_t)((int)(code << 24) >> 24 << kLowShift<T>));
}
// of 8 consecutive elements
template <int T>
__device__ __forceinline__ void store_low(uint8_t* low, int64_t element, const float (&x)[8]) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float a, b;
        unpack_pair<T>(pack_pair<T>(x[i], x[i + 1]), a, b);
        w[i / 4] |= (low_bits<T>(x[i], a) | low_bits<T>(x[i + 1], b) << 8) << (i % 4 * 8);
    }
    *reinterpret_cast<v2i_attn*>(low + element) = (v2i_attn){(int)w[0], (int)w[1]};
}

// acc * factor as one row a lane, rounded to T: 16 bytes a lane and store.  p: the row's first element
template <int T, int DP>
__device__ __forceinline__ void store_rows(const v16f (&acc)[DP / 32], float factor, void* p, int64_t element, int dim, bool live, int lane, uint8_t* low = nullptr) {
    char* const at = static_cast<char*>(p) + 2 * element;
    const int h = lane >> 5;
#pragma unroll
    for (int e = 0; e < DP / 32; ++e)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float v[8];
#pragma unroll
            for (int r = 0; r < 8; ++r) v[r] = acc[e][8 * s + r] * factor;
            // 8 elements in a row: the second four of this half wave for the first four of the other
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                uint32_t x = __float_as_uint(v[r]), y = __float_as_uint(v[4 + r]);
                swap_halves(x, y);
                v[r] = __uint_as_float(x);
                v[4 + r] = __uint_as_float(y);
            }
            const int first = 32 * e + 16 * s + 8 * h;
            if (live && first < dim) {
                *reinterpret_cast<v4i*>(at + 2 * first) =
                    (v4i){(int)pack_pair<T>(v[0], v[1]), (int)pack_pair<T>(v[2], v[3]), (int)pack_pair<T>(v[4], v[5]), (int)pack_pair<T>(v[6], v[7])};
                if (low) store_low<T>(low, element + first, v);
            }
        }
}

// the lane's number, made anew where a register kept for it would be spilled
__device__ __forceinline__ uint32_t lane_anew() {
    uint32_t none = 0;
    asm volatile("" : "+v"(none));
    return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none));
}

// max of a lane and its counterpart of the other half wave
__device__ __forceinline__ float both_max(float v) {
    uint32_t x = __float_as_uint(v), y = x;
    swap_halves(x, y);
    return fmaxf(__uint_as_float(x), __uint_as_float(y));
}
__device__ __forceinline__ float both_sum(float v) {
    uint32_t x = __float_as_uint(v), y = x;
    swap_halves(x, y);
    return __uint_as_float(x) + __uint_as_float(y);
}

// The maximum (base 2) of a row is minus infinity where it sees no key.  Where it sees some that all score minus infinity (an infinity in the query, a
// product beyond fp32) or NaN it is this instead, so that the row's sum, 0, makes the 0 / 0 that its softmax is, while beside a run of keys with
// scores it counts nothing: exp2(this - their maximum) is 0
constexpr float kAttnLowest = -3.4028234663852886e38f;
__device__ __forceinline__ float attn_top(float top, bool sees) { return sees && top == -__builtin_inff() ? kAttnLowest : top; }
// what a row's outputs are multiplied by, and what is kept of its maximum and sum for the backward pass
__device__ __forceinline__ float attn_over(float top, float sum) { return top == -__builtin_inff() ? 0.0f : 1.0f / sum; }
__device__ __forceinline__ float attn_lse(const AttnArgs& A, float top, float sum) {
    return top == -__builtin_inff() ? top : sum == 0.0f ? __builtin_nanf("") : -(top + log2f(sum)) / A.c;
}

// calls f with the type and the head's size rounded up to what the kernels are built for
template <typename F>
int with_attn(int dtype, int dim, F&& f) {
    using std::integral_constant;
    auto by_dim = [&](auto t) { 
        if (dim <= 64) return f(t, integral_constant<int, 64>{});
        return dim <= 96 ? f(t, integral_constant<int, 96>{}) : f(t, integral_constant<int, 128>{});
    };
    return dtype == NTFP8_BF16 ? by_dim(integral_constant<int, NTFP8_BF16>{}) : by_dim(integral_constant<int, NTFP8_F16>{});
}

}  // namespace ntfp8

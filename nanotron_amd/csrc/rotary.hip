// Rotary positions: pairs (a, b) of every query and key head turned by position * frequency, (a cos - b sin, b cos + a sin) scale.
//
// Bound by memory: x is read and written once, queries and keys in one launch.  The angles are those of a token and serve all its heads:
// a workgroup makes the sines and cosines of its tokens in LDS, in turns (position * frequency / 2 pi) in 64 bits, of which the whole ones
// are dropped before anything is rounded to 32, so far positions lose nothing and no table bounds them.
// 16381 tokens of 32 + 8 heads of 128 in bf16: 168 MB each way in 73 us, 4.6 TB/s, with one 16-byte piece at a time a thread (two 82, four 88; loads and stores
// past the caches 92).  One token: 3.4 us, a launch.
#include "ops_common.h"

namespace ntfp8 {
namespace {

constexpr int kThreads = 256, kTurns = 4;   // threads of a workgroup, and pieces of work of each, about
constexpr int kMostPairs = 1024;            // sines and cosines in LDS

struct Rotary {
    const void* in[2];        // queries and keys
    void* out[2];
    int64_t stride[2], head[2];
    int heads[2];
    int64_t tokens;
    int dim, pairs, tokens_a_block;
    int units, turning;       // a head's: of all, and those that turn
    uint32_t magic_heads, magic_units, magic_pairs;   // ceil(2^32 / n)
    const void* positions;
    int64_t position_count, first_token;
    int position_bits;
    const double* frequencies;
    int interleaved, inverse;
    float scale;
};

// x / n for x n < 2^32
__device__ __forceinline__ int over(int x, int n, uint32_t magic) { return n == 1 ? x : (int)__umulhi((uint32_t)x, magic); }

template <int D, bool kInterleaved>
__global__ __launch_bounds__(kThreads) void rotary_kernel(const Rotary R) {
    constexpr int VE = 16 / size_of(D);   // a unit: two pieces of VE elements, VE pairs
    __shared__ float2 turn[kMostPairs];
    const int64_t token0 = (int64_t)blockIdx.x * R.tokens_a_block;
    const int tokens = (int)min((int64_t)R.tokens_a_block, R.tokens - token0);
    const int all_heads = R.heads[0] + R.heads[1], total = tokens * all_heads * R.units;
    struct Unit {
        Piece<D, VE> a, b;
        int64_t from, to;   // elements
        int first, second;  // counts of the pieces
        int at;             // its first sine, -1 where nothing turns
        int which;
    };
    auto read = [&](Unit& u, int i) {
        const int unit_row = over(i, R.units, R.magic_units), unit = i - unit_row * R.units;
        const int token = over(unit_row, all_heads, R.magic_heads);
        int head = unit_row - token * all_heads;
        u.which = head >= R.heads[0];
        head -= u.which ? R.heads[0] : 0;
        u.from = (token0 + token) * R.stride[u.which] + head * R.head[u.which];
        u.to = ((token0 + token) * R.heads[u.which] + head) * R.dim;
        int a, b;
        if (unit >= R.turning) {   // behind what turns: 2 VE elements in a row
            a = 2 * R.pairs + (unit - R.turning) * 2 * VE;
            b = a + VE;
            u.first = max(0, min(VE, R.dim - a));
            u.second = max(0, min(VE, R.dim - b));
            u.at = -1;
        } else if (kInterleaved) {
            a = unit * 2 * VE;
            b = a + VE;
            u.first = max(0, min(VE, 2 * R.pairs - a));
            u.second = max(0, min(VE, 2 * R.pairs - b));
            u.at = token * R.pairs + unit * VE;
        } else {
            a = unit * VE;
            b = R.pairs + a;
            u.first = u.second = min(VE, R.pairs - a);
            u.at = token * R.pairs + a;
        }
        u.a = load_piece<D, VE>(R.in[u.which], u.from + a, u.first);
        u.b = load_piece<D, VE>(R.in[u.which], u.from + b, u.second);
        u.from = u.to + a;
        u.to += b;
    };
    // What is read first is asked for before the angles are worked out.  One piece of work at a time: the registers of two or four
    // halve or quarter the waves on a CU, whose loads overlap (16381 tokens, 40 heads of 128: 73, 82, 88 us)
    Unit unit;
    if ((int)threadIdx.x < total) read(unit, threadIdx.x);
    for (int i = threadIdx.x; i < tokens * R.pairs; i += kThreads) {
        const int token = over(i, R.pairs, R.magic_pairs);
        int64_t p = R.first_token + token0 + token;
        if (p >= R.position_count) p %= R.position_count;
        const double position = R.position_bits == 64 ? (double)static_cast<const int64_t*>(R.positions)[p] : (double)static_cast<const int32_t*>(R.positions)[p];
        const double turns = position * (R.frequencies[i - token * R.pairs] * 0.15915494309189533577);
        float sine, cosine;
        sincospif((float)(2.0 * (turns - rint(turns))), &sine, &cosine);
        turn[i] = make_float2(cosine * R.scale, (R.inverse ? -sine : sine) * R.scale);
    }
    __syncthreads();
    auto write = [&](const Unit& u) {
        float x[VE], y[VE], p[VE], q[VE];
        unpack<D, VE>(u.a, x);
        unpack<D, VE>(u.b, y);
        if (u.at < 0) {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                p[e] = x[e];
                q[e] = y[e];
            }
        } else if constexpr (kInterleaved) {
#pragma unroll
            for (int e = 0; e < VE / 2; ++e) {
                const float2 s = 2 * e < u.first ? turn[u.at + e] : make_float2(0, 0), t = 2 * e < u.second ? turn[u.at + VE / 2 + e] : make_float2(0, 0);
                p[2 * e] = fmaf(x[2 * e], s.x, -(x[2 * e + 1] * s.y));
                p[2 * e + 1] = fmaf(x[2 * e + 1], s.x, x[2 * e] * s.y);
                q[2 * e] = fmaf(y[2 * e], t.x, -(y[2 * e + 1] * t.y));
                q[2 * e + 1] = fmaf(y[2 * e + 1], t.x, y[2 * e] * t.y);
            }
        } else {
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float2 s = e < u.first ? turn[u.at + e] : make_float2(0, 0);
                p[e] = fmaf(x[e], s.x, -(y[e] * s.y));
                q[e] = fmaf(y[e], s.x, x[e] * s.y);
            }
        }
        store_piece<D, VE>(R.out[u.which], u.from, p, u.first);
        store_piece<D, VE>(R.out[u.which], u.to, q, u.second);
    };
    for (int i = threadIdx.x; i < total; i += kThreads) {
        if (i != (int)threadIdx.x) read(unit, i);
        write(unit);
    }
}

uint32_t magic_of_count(int n) { return (uint32_t)(((1ull << 32) + n - 1) / n); }

}  // namespace

int run_rotary(const ntops_rotary_desc& d, hipStream_t st) {
    const int ve = 16 / size_of(d.dtype);
    Rotary r = {};
    r.in[0] = d.q, r.in[1] = d.k, r.out[0] = d.q_out, r.out[1] = d.k_out;
    r.stride[0] = d.q_stride, r.stride[1] = d.k_stride, r.head[0] = d.q_head, r.head[1] = d.k_head;
    r.heads[0] = d.heads, r.heads[1] = d.kv_heads;
    r.dim = d.head_dim, r.pairs = d.pairs;
    r.turning = d.interleaved ? (2 * d.pairs + 2 * ve - 1) / (2 * ve) : (d.pairs + ve - 1) / ve;
    r.units = r.turning + (d.head_dim - 2 * d.pairs + 2 * ve - 1) / (2 * ve);
    r.positions = d.positions, r.position_count = d.position_count, r.position_bits = d.position_bits;
    r.frequencies = d.frequencies, r.interleaved = d.interleaved, r.inverse = d.inverse, r.scale = d.scale;
    const int heads = d.heads + d.kv_heads;
    // a workgroup's tokens: about kTurns pieces of work a thread, and no more angles than LDS has room for
    r.tokens_a_block = std::max(1, std::min(kTurns * kThreads / (heads * r.units), kMostPairs / d.pairs));
    r.magic_heads = magic_of_count(heads), r.magic_units = magic_of_count(r.units), r.magic_pairs = magic_of_count(d.pairs);
    // (a launch takes fewer than 2^32 threads)
    const int64_t most = (int64_t)r.tokens_a_block << 23;
    for (int64_t token = 0; token < d.tokens; token += most) {
        r.tokens = std::min(most, d.tokens - token), r.first_token = token;
        if (token) {
            const int64_t bytes = size_of(d.dtype);
            r.in[0] = static_cast<const char*>(d.q) + token * d.q_stride * bytes;
            r.out[0] = static_cast<char*>(d.q_out) + token * d.heads * d.head_dim * bytes;
            if (d.k) {
                r.in[1] = static_cast<const char*>(d.k) + token * d.k_stride * bytes;
                r.out[1] = static_cast<char*>(d.k_out) + token * d.kv_heads * d.head_dim * bytes;
            }
        }
        const unsigned grid = (unsigned)((r.tokens + r.tokens_a_block - 1) / r.tokens_a_block);
        const int rc = with_dtype(d.dtype, [&](auto t) {
            if (d.interleaved) rotary_kernel<decltype(t)::value, true><<<grid, kThreads, 0, st>>>(r);
            else rotary_kernel<decltype(t)::value, false><<<grid, kThreads, 0, st>>>(r);
            return launch_status();
        });
        if (rc != NTFP8_OK) return rc;
    }
    return NTFP8_OK;
}

}  // namespace ntfp8

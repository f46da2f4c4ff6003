// Attention, backward.  With p = exp2(c q k^T - lse) and delta = sum over elements of dout out, a row each:
//   dv = p^T dout,  ds = p (dout v^T - delta),  dq = scale ds k,  dk = scale ds^T q
// One kernel owns queries and makes dq, one owns keys and makes dk and dv; both make the scores again, seven products where five
// would do, so that every sum is made in one place and order: no atomics, the same bits for the same inputs.
//
// Bound by the products: 16384 causal tokens, 32 heads of 128 over 8, in bf16 take 6.4 to 6.8 ms, 0.86 PFLOP/s of the five products and 1.2 of the seven that are
// made, 70 % of the matrix instructions' slots at the 1.4 to 1.5 GHz that the power limit leaves; 4096 tokens 431 to 438 us.  delta is memory, 4.8 TB/s.
//
// fp16: ds is a gradient and may be smaller than that type's normal numbers, and p in a long row is.  p is kept times 2^8, ds
// times the power of two that the largest magnitudes of dout and v allow it without overflow.  That one serves the call: what is 2^28 below 2 dim |dout| |v|
// of the largest of all its sequences goes into that type's subnormals.
#include "attention.h"

namespace ntfp8 {
namespace {

constexpr float kLiftP = 8.0f;
// what ds is multiplied by beyond p's lift: |dout v^T - delta| is at most 2 dim |dout| |v|, brought to 2^15 with the lift
template <int T>
__device__ __forceinline__ float gradient_lift(const AttnArgs& A) {
    if constexpr (T == NTFP8_BF16) return 1.0f;
    uint32_t q = 0, v = 0;
    // (one trip to memory, not one for every 64)
#pragma unroll
    for (int n = 0; n < kAttnMost; n += 64) {
        const int i = n + (threadIdx.x & 63);
        const uint32_t x = i < A.most_q ? A.most[i] : 0u, y = i < A.most_v ? A.most[kAttnMost + i] : 0u;
        q = max(q, x);
        v = max(v, y);
    }
    const float most = 2.0f * A.dim * __uint_as_float(wave_most(q)) * __uint_as_float(wave_most(v));
    if (!(most > 0.0f) || most > 1e30f || most < 1e-30f) return 1.0f;
    const int e = (int)(__float_as_uint(most) >> 23) - 127;   // 2^e <= most < 2^(e + 1)
    return __uint_as_float((uint32_t)(127 + 14 - e) << 23);
}

// delta, 16 lanes a row; the workgroups behind the first q_groups read v, for its largest magnitude.  Each leaves what it found in a place of
// its own: no atomics, and nothing to clear before
template <int T>
__global__ __launch_bounds__(256) void attention_delta_kernel(const AttnArgs A, const int* cu_q, const int* cu_k, int q_groups) {
    __shared__ uint32_t found[4];
    const bool values = (int)blockIdx.x >= q_groups;
    const int own = values ? blockIdx.x - q_groups : blockIdx.x, groups = values ? gridDim.x - q_groups : q_groups;
    const int heads = values ? A.kv_heads : A.heads, own_len = values ? A.k_len : A.q_len;
    const uint32_t items = (uint32_t)((values ? A.k_rows : A.q_rows) * heads);   // (2^27 at most)
    const int d = (threadIdx.x & 15) * 8;
    const int* const cu = values ? cu_k : cu_q;
    const int begin = cu ? cu[0] : 0, end = cu ? cu[A.sequences] : 0;
    uint32_t most = 0;
    for (uint32_t item = (uint32_t)own * 16 + (threadIdx.x >> 4); item < items; item += (uint32_t)groups * 16) {
        const int row = (int)(item / (uint32_t)heads), head = (int)(item - (uint32_t)row * (uint32_t)heads);
        const bool live = !cu || (row >= begin && row < end);   // rows of no sequence may hold anything
        float x[8] = {}, y[8] = {}, sum = 0.0f;
        if (live && d < A.dim) {
            const int seq = A.tasks ? 0 : row / own_len;
            const int64_t at = A.tasks ? row : row - seq * own_len;
            const int64_t stride = values ? A.v_stride : A.do_stride, batch = values ? A.v_batch : A.do_batch, apart = values ? A.v_head : A.do_head;
            unpack<T, 8>(load_piece<T, 8>(values ? A.v : A.dout, seq * batch + at * stride + head * apart + d), x);
            if (!values) {
                const int64_t at_out = (int64_t)item * A.dim + d;
                unpack<T, 8>(load_piece<T, 8>(A.o, at_out), y);
                if (A.low) {
                    const v2i_attn low = *reinterpret_cast<const v2i_attn*>(A.low + at_out);
#pragma unroll
                    for (int i = 0; i < 8; ++i) y[i] = with_low<T>(y[i], (uint32_t)low[i / 4] >> (i % 4 * 8));
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sum += x[i] * y[i];
            const uint32_t size = __float_as_uint(x[i]) & 0x7fffffffu;
            most = max(most, size < kInfBits ? size : 0u);   // (what is not finite spoils its own sequence, whatever the others are lifted by)
        }
#pragma unroll
        for (int m = 1; m < 16; m *= 2) sum += __shfl_xor(sum, m);
        if (!values && d == 0) A.delta[head * A.q_rows + row] = live ? -sum : 0.0f;
    }
    if constexpr (T == NTFP8_F16) {
        most = wave_most(most);
        if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = most;
        __syncthreads();
        if (threadIdx.x == 0) A.most[(values ? kAttnMost : 0) + own] = max(max(found[0], found[1]), max(found[2], found[3]));
    }
}

// How a tile is taken: all its rows and keys see each other, or some do not, or these hold values that are not finite
constexpr int kWhole = 0, kMasked = 1, kSingly = 2;

// dq of 128 queries of one head, 32 a wave, or of 32 of four heads
template <int T, int DP>
__device__ __forceinline__ void attention_dq(const AttnArgs& A, int group, uint8_t* lds) {
    typedef AttnTile<DP> Tile;
    uint8_t *const sk = lds, *const sv = lds + 2 * Tile::kBytes;
    int(*const odd)[kAttnWaves] = reinterpret_cast<int(*)[kAttnWaves]>(lds + 4 * Tile::kBytes);   // [stage]: a wave's part of the keys is not finite throughout
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttnOwn own = attn_own(A, group, wave);
    const int kv = own.kv, head = kv * A.group + own.inside;
    const AttnTask task = attn_task(A, own.tile, A.tile_heads > 1 ? 32 : kAttnQueries, false);
    if (task.rows <= 0) return;
    const int64_t k0 = attn_rows(A, task.other, task.seq, 0, A.k_stride, A.k_batch) + kv * A.k_head;
    const int64_t v0 = attn_rows(A, task.other, task.seq, 0, A.v_stride, A.v_batch) + kv * A.v_head;
    const int end = A.causal ? min(max(task.shift + task.rows, 0), task.len) : task.len, steps = (end + kAttnStep - 1) / kAttnStep;
    Tile tile;
    tile.init(lane);
    typename Tile::template Source<> ks, vs;
    ks.init(A.k, k0, A.k_stride, A.dim, wave, lane);
    vs.init(A.v, v0, A.v_stride, A.dim, wave, lane);
    if (steps > 0) {
        ks.load(sk, 0, task.len, wave);
        vs.load(sv, 0, task.len, wave);
    }
    const int row = own.row + (lane & 31);
    const bool live = row < task.rows && own.inside < A.group;
    v4i q[DP / 16], g[DP / 16];
    load_own<DP>(q, A.q, attn_rows(A, task.own, task.seq, task.at, A.q_stride, A.q_batch) + head * A.q_head + row * A.q_stride, A.dim, live, lane);
    load_own<DP>(g, A.dout, attn_rows(A, task.own, task.seq, task.at, A.do_stride, A.do_batch) + head * A.do_head + row * A.do_stride, A.dim, live, lane);
    const int64_t at = (int64_t)task.own + row;
    const float lse = live ? A.lse[head * A.q_rows + at] * A.c : -__builtin_inff(), delta = live ? A.delta[head * A.q_rows + at] : 0.0f;
    const float lift = gradient_lift<T>(A);
    v16f dq[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) dq[e] = zeros16();
    // One tile of keys.  kMasked: some rows of the workgroup may not see all of them.  One of those with keys which are not finite is left for
    // later, see the forward pass, and then fetched by itself
    bool left = false;
    auto step = [&](int j, auto how_) __attribute__((always_inline)) {
        constexpr int kHow = decltype(how_)::value;
        constexpr bool kMask = kHow != kWhole;
        const int key0 = j * kAttnStep, stage = kHow == kSingly ? 0 : (j & 1) * Tile::kBytes;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (kHow == kSingly) {
            wg_barrier();
            ks.load(sk, key0, task.len, wave);
            vs.load(sv, key0, task.len, wave);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if constexpr (kMask) attn_tell(odd[j & 1], wave, attn_not_finite<T, DP, kAttnStep, kAttnWaves>(sk + stage, wave, lane));
        wg_barrier();
        if (kHow != kSingly && j + 1 < steps) {
            ks.load(sk + Tile::kBytes - stage, key0 + kAttnStep, task.len, wave);
            vs.load(sv + Tile::kBytes - stage, key0 + kAttnStep, task.len, wave);
        }
        if constexpr (kMask) {
            const bool not_finite = attn_any_wave(odd[j & 1]);
            left |= not_finite;
            if (not_finite != (kHow == kSingly)) return;
        }
        if (own.row >= task.rows || own.inside >= A.group) return;   // (without rows, it brings its part of the tiles)
        const int lead = task.shift + own.row;   // the last key that the wave's first row sees
        if (kMask && A.causal && key0 > lead + 31) return;   // (uniform in the wave)
        const int last = (A.causal ? min(task.len - 1, lead + (lane & 31)) : task.len - 1) - key0, last_half = last - 4 * (lane >> 5);
        // Runs of products, of two blocks of 32 keys: scores and dout v^T of the one, of the other, then dq; beside each the arithmetic of the run
        // before.  Fragments are read two products ahead.
        constexpr int kProducts = DP / 16;   // of a run
        v16f s[2], d[2];
        v4i p[4], f[3];
        // fragment x of the runs: keys, values, keys, values of the two blocks, then columns of the keys
        auto fetch = [&](int x) __attribute__((always_inline)) {
            const int run = x / kProducts, i = x % kProducts;
            if (run < 4) f[x % 3] = tile.rows(run & 1 ? sv + stage : sk + stage, run >> 1, i);
            else f[x % 3] = tile.columns(sk + stage, (x - 4 * kProducts) / (DP / 32), (x - 4 * kProducts) % (DP / 32));
        };
        auto run = [&](int which, auto&& beside) __attribute__((always_inline)) {
            const int b = which >> 1;
            v16f& to = which & 1 ? d[b] : s[b];
            to = zeros16();
#pragma unroll
            for (int i = 0; i < kProducts; ++i) {
                const int x = which * kProducts + i;
                if (!kMask || x + 2 < 4 * kProducts) fetch(x + 2);
                to = mfma_attn<T>(f[x % 3], which & 1 ? g[i] : q[i], to);
#pragma unroll
                for (int r = i * 16 / kProducts; r < (i + 1) * 16 / kProducts; ++r) beside(r);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto exponential = [&](int b, int r) __attribute__((always_inline)) { s[b][r] = exp2_fast(__builtin_fmaf(s[b][r], A.c, lse)); };
        auto gradient = [&](int b, int r) __attribute__((always_inline)) {
            d[b][r] = s[b][r] * ((d[b][r] + delta) * lift);
            if (kMask && 32 * b + place_in_half(r) > last_half) d[b][r] = 0.0f;
            if (r % 8 == 7) p[2 * b + r / 8] = pack_scores<T>(d[b], r - 7);
        };
        fetch(0);
        fetch(1);
        run(0, [](int) {});
        run(1, [&](int r) __attribute__((always_inline)) { exponential(0, r); });
        run(2, [&](int r) __attribute__((always_inline)) { gradient(0, r); });
        run(3, [&](int r) __attribute__((always_inline)) { exponential(1, r); });
        if constexpr (kMask) {
#pragma unroll
            for (int r = 0; r < 16; ++r) gradient(1, r);
            if constexpr (kHow == kSingly) {
                add_columns_singly<T, DP, 4>(dq, tile, sk + stage, p, 0, last + 1);
                return;
            }
            fetch(4 * kProducts);
            fetch(4 * kProducts + 1);
        }
#pragma unroll
        for (int i = 0; i < 2 * kProducts; ++i) {
            const int x = 4 * kProducts + i;
            if (i + 2 < 2 * kProducts) fetch(x + 2);
            dq[i % (DP / 32)] = mfma_attn<T>(f[x % 3], p[i / (DP / 32)], dq[i % (DP / 32)]);
            if constexpr (!kMask) {
                if (i < kProducts) {
#pragma unroll
                    for (int r = i * 16 / kProducts; r < (i + 1) * 16 / kProducts; ++r) gradient(1, r);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // tiles that every row sees whole, then the others
    const int clear = max(0, min(min(task.len, A.causal ? task.shift + 1 : task.len) / kAttnStep, steps));
    int j = 0;
    for (; j < clear; ++j) step(j, std::integral_constant<int, kWhole>{});
    for (; j < steps; ++j) step(j, std::integral_constant<int, kMasked>{});
    if (__builtin_expect(left, 0))
        for (j = clear; j < steps; ++j) step(j, std::integral_constant<int, kSingly>{});
    store_rows<T, DP>(dq, A.scale / lift, A.dq, (at * A.heads + head) * A.dim, A.dim, live, lane);
}

// dk and dv of 128 keys of one head of keys, 32 a wave: over the heads of queries that share it, and their queries 32 at a time.  A wave holds
// its keys and both sums in registers, 160 of the 256 that two waves a SIMD have; its values stay in LDS.  Tried: 256 keys of eight waves, three and four
// tiles ahead, fragments read further ahead (nothing, or spilled registers).
template <int T, int DP>
__device__ __forceinline__ void attention_dkv(const AttnArgs& A, int group, uint8_t* lds) {
    typedef AttnTile<DP, kAttnKeyStep> Tile;
    uint8_t *const sq = lds, *const sg = lds + 2 * Tile::kBytes, *const sv = lds + 4 * Tile::kBytes;
    float(*const rows_of)[2][64] = reinterpret_cast<float(*)[2][64]>(sv + kAttnKeys / kAttnKeyStep * Tile::kBytes);   // [stage]: lse and delta (a wave loads 64)
    int(*const odd)[kAttnKeyWaves] = reinterpret_cast<int(*)[kAttnKeyWaves]>(rows_of + 2);   // [stage]: a wave's part of the queries or gradients is not finite throughout
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int run = group / A.kv_heads, kv = group - run * A.kv_heads, t = run / A.k_splits, split = run - t * A.k_splits;
    const AttnTask task = attn_task(A, t, kAttnKeys, true);
    if (task.rows <= 0) return;
    const int begin = A.causal ? max(0, task.shift) / kAttnKeyStep : 0, per = max(0, (task.len + kAttnKeyStep - 1) / kAttnKeyStep - begin);
    const int each = (per * A.group + A.k_splits - 1) / A.k_splits, step0 = min(split * each, per * A.group), steps = min(step0 + each, per * A.group);
    Tile tile;
    tile.init(lane);
    typename Tile::template Source<kAttnKeyWaves> qs, gs, vs;
    qs.init(A.q, 0, A.q_stride, A.dim, wave, lane);
    gs.init(A.dout, 0, A.do_stride, A.dim, wave, lane);
    // Tiles of a head's queries: first those whose rows all see all keys of the workgroup, then the ones in front of and behind these
    const int front = A.causal ? min(max(0, (task.shift + task.rows - 1 + kAttnKeyStep - 1) / kAttnKeyStep - begin), per) : 0;
    const int whole = max(0, min(task.len / kAttnKeyStep - begin, per) - front);
    auto row_of = [&](int i) { return (begin + (i < whole ? front + i : i < whole + front ? i - whole : i)) * kAttnKeyStep; };
    // The tile that is loaded next, and its head's first rows: counted along, a division a step is as long as three of its products
    int next_tile = 0, next_row = 0;
    const int64_t q_apart = 2 * A.q_head, g_apart = 2 * A.do_head;
    const float* stats = nullptr;
    auto seek = [&](int j) __attribute__((always_inline)) {
        const int in = per > 0 ? j / per : 0, head = kv * A.group + in;
        next_tile = j - in * per;
        qs.base = static_cast<const char*>(A.q) + 2 * (attn_rows(A, task.other, task.seq, 0, A.q_stride, A.q_batch) + head * A.q_head);
        gs.base = static_cast<const char*>(A.dout) + 2 * (attn_rows(A, task.other, task.seq, 0, A.do_stride, A.do_batch) + head * A.do_head);
        stats = (wave == 0 ? A.lse : A.delta) + head * A.q_rows + task.other;
    };
    seek(step0);
    auto load = [&](int stage) __attribute__((always_inline)) {
        const int first = next_row = row_of(next_tile);
        qs.load(sq + stage * Tile::kBytes, first, task.len, wave);
        gs.load(sg + stage * Tile::kBytes, first, task.len, wave);
        if (wave < 2) {
            const __amdgpu_buffer_rsrc_t r = make_rsrc(stats + first, (uint32_t)__builtin_amdgcn_readfirstlane(min(kAttnKeyStep, task.len - first) * 4));
            // (a lane's offset from memory would be waited for behind the loads above, 800 cycles a step)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(uintptr_t)&rows_of[stage][wave][0], 4, lane_anew() * 4, 0, 0, 0);
        }
        if (++next_tile == per) {
            next_tile = 0;
            qs.base += q_apart;
            gs.base += g_apart;
            stats += A.q_rows;
        }
    };
    vs.init(A.v, attn_rows(A, task.own, task.seq, task.at, A.v_stride, A.v_batch) + kv * A.v_head, A.v_stride, A.dim, wave, lane);
    if (step0 < steps) {
#pragma unroll
        for (int i = 0; i < kAttnKeys / kAttnKeyStep; ++i) vs.load(sv + i * Tile::kBytes, i * kAttnKeyStep, task.rows, wave);
        load(step0 & 1);
    }
    const int mine = wave * 32 * Tile::kPitch;
    const int row = wave * 32 + (lane & 31);
    const bool live = row < task.rows;
    v4i k[DP / 16];
    load_own<DP>(k, A.k, attn_rows(A, task.own, task.seq, task.at, A.k_stride, A.k_batch) + kv * A.k_head + row * A.k_stride, A.dim, live, lane);
    constexpr float kDown = T == NTFP8_F16 ? 1.0f / 256.0f : 1.0f;   // 2^-kLiftP
    const float lift = gradient_lift<T>(A), down = lift * kDown, up = kLiftP / A.c;
    v16f dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) dk[e] = dv[e] = zeros16();
    // One tile of queries of one head.  kMasked: some of its rows may not see all the workgroup's keys, and where it is not finite it is left for later
    bool left = false;
    auto step = [&](int j, auto how_) __attribute__((always_inline)) {
        constexpr int kHow = decltype(how_)::value;
        constexpr bool kMask = kHow != kWhole;
        if constexpr (kHow == kSingly) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            wg_barrier();
            seek(j);
            load(j & 1);
        }
        const int row0 = next_row, stage = j & 1, at = stage * Tile::kBytes;   // (its load was the last)
        uint8_t *const qa = sq + stage * Tile::kBytes, *const ga = sg + stage * Tile::kBytes;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (kMask)
            attn_tell(odd[stage], wave, attn_not_finite<T, DP, kAttnKeyStep, kAttnKeyWaves>(qa, wave, lane) || attn_not_finite<T, DP, kAttnKeyStep, kAttnKeyWaves>(ga, wave, lane));
        wg_barrier();
        if (kHow != kSingly && j + 1 < steps) load(stage ^ 1);
        if constexpr (kMask) {
            const bool not_finite = attn_any_wave(odd[stage]);
            left |= not_finite;
            if (not_finite != (kHow == kSingly)) return;
        }
        if (wave * 32 >= task.rows) return;
        const int lead = task.shift + wave * 32;   // the first query that sees the wave's first key
        if (kMask && A.causal && row0 + kAttnKeyStep - 1 < lead) return;
        const int from = A.causal ? lead + (lane & 31) - row0 : 0, to = task.len - row0, half = 4 * (lane_anew() >> 5);   // rows of the tile that see this lane's key
        // s and d begin at what is subtracted from them
        v16f s, d;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const v4f x = *reinterpret_cast<const v4f*>(&rows_of[stage][0][8 * n + 4 * (lane >> 5)]), y = *reinterpret_cast<const v4f*>(&rows_of[stage][1][8 * n + 4 * (lane >> 5)]);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[4 * n + i] = T == NTFP8_F16 ? x[i] + up : x[i];
                d[4 * n + i] = y[i];
            }
        }
        // Four runs of products: scores, dout v^T, dv and dk.  Beside the second go the exponentials, beside the third what ds is made of; the
        // fragments are read two products ahead.  A wave issues one instruction after another, so their order is set here.
        constexpr int kProducts = DP / 16;   // of a run
        v4i fq[3], fg[2], fv[2], p[2], ds[2];
        // (short heads have registers for the fragments' addresses: 8192 causal tokens, 16 heads of 64, both passes 805 -> 768 us)
        auto rows = [&](uint8_t* array, int begin, int i) __attribute__((always_inline)) { return DP == 64 ? tile.rows(array + begin, 0, i) : tile.rows_anew(array, begin, 0, i); };
        auto fetch_q = [&](int i) __attribute__((always_inline)) { fq[i % 3] = rows(sq, at, i); };
        auto fetch_g = [&](int i) __attribute__((always_inline)) {
            fg[i & 1] = rows(sg, at, i);
            fv[i & 1] = rows(sv, mine, i);
        };
        fetch_q(0);
        fetch_q(1);
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            if (i + 2 < kProducts) fetch_q(i + 2);
            if (i + 1 == kProducts) fetch_g(0);
            s = mfma_attn<T>(fq[i % 3], k[i], s);
            __builtin_amdgcn_sched_barrier(0);
        }
        auto counted = [&](float x, int r) __attribute__((always_inline)) {
            if constexpr (!kMask) return x;
            return place_in_half(r) >= from - half && place_in_half(r) < to - half ? x : 0.0f;
        };
        v4i fa[3];
        // fragment x of the products for dv, and those for dk behind them
        auto fetch_a = [&](int x) __attribute__((always_inline)) {
            uint8_t* const from = x < kProducts ? sg : sq;
            const int block = x % kProducts / (DP / 32), e = x % (DP / 32);
            fa[x % 3] = DP == 64 ? tile.columns(from + at, block, e) : tile.columns_anew(from, at, block, e);
        };
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            if (i + 1 < kProducts) fetch_g(i + 1);
            if (i + 2 >= kProducts) fetch_a(i + 2 - kProducts);
            d = mfma_attn<T>(fg[i & 1], fv[i & 1], d);
#pragma unroll
            for (int r = i * 16 / kProducts; r < (i + 1) * 16 / kProducts; ++r) {
                s[r] = counted(exp2_fast(s[r] * A.c), r);
                if (r % 8 == 7) p[r / 8] = pack_scores<T>(s, r - 7);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        auto gradient = [&](int r) __attribute__((always_inline)) {
            d[r] = counted(T == NTFP8_F16 ? s[r] * (d[r] * down) : s[r] * d[r], r);
            if (r % 8 == 7) ds[r / 8] = pack_scores<T>(d, r - 7);
        };
        if constexpr (kMask) {
#pragma unroll
            for (int r = 0; r < 16; ++r) gradient(r);
            if constexpr (kHow == kSingly) {
                add_columns_singly<T, DP, 2>(dv, tile, ga, p, from, to);
                add_columns_singly<T, DP, 2>(dk, tile, qa, ds, from, to);
                return;
            }
        }
#pragma unroll
        for (int x = 0; x < kProducts; ++x) {
            fetch_a(x + 2);
            dv[x % (DP / 32)] = mfma_attn<T>(fa[x % 3], p[x / (DP / 32)], dv[x % (DP / 32)]);
            if constexpr (!kMask) {
#pragma unroll
                for (int r = x * 16 / kProducts; r < (x + 1) * 16 / kProducts; ++r) gradient(r);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int x = 0; x < kProducts; ++x) {
            if (x + 2 < kProducts) fetch_a(kProducts + x + 2);
            dk[x % (DP / 32)] = mfma_attn<T>(fa[(kProducts + x) % 3], ds[x / (DP / 32)], dk[x % (DP / 32)]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    for (int j = step0; j < steps;) {
        const int i = j % per;
        for (const int end = min(steps, j + whole - i); j < end; ++j) step(j, std::integral_constant<int, kWhole>{});
        for (const int end = min(steps, j + per - max(i, whole)); j < end; ++j) step(j, std::integral_constant<int, kMasked>{});
    }
    if (__builtin_expect(left, 0))
        for (int j = step0; j < steps; ++j)
            if (j % per >= whole) step(j, std::integral_constant<int, kSingly>{});
    const int64_t to = (((int64_t)task.own + row) * A.kv_heads + kv) * A.dim;
    const float dk_by = A.scale / lift;
    if (A.k_splits > 1) {
        if (!live) return;
        const int64_t all = A.k_rows * A.kv_heads * A.dim;
        float* const part = A.k_part + 2 * split * all + to;
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * e + 8 * g + 4 * (lane >> 5);
                if (d >= A.dim) continue;
                v4f x, y;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = dk[e][4 * g + i] * dk_by;
                    y[i] = dv[e][4 * g + i] * kDown;
                }
                *reinterpret_cast<v4f*>(part + d) = x;
                *reinterpret_cast<v4f*>(part + all + d) = y;
            }
        return;
    }
    if (A.dv) store_rows<T, DP>(dv, kDown, A.dv, to, A.dim, live, lane);
    if (A.dk) store_rows<T, DP>(dk, dk_by, A.dk, to, A.dim, live, lane);
}

// Both in one launch, the workgroups of keys first: they have more to do each, and those of queries fill what they leave of the chip
template <int T, int DP>
__global__ __launch_bounds__(64 * kAttnWaves, attn_workgroups(DP)) void attention_backward_kernel(const AttnArgs A, const AttnTask* k_tasks, int k_groups) {
    static_assert(kAttnWaves == kAttnKeyWaves, "");
    constexpr int kKeys = (4 + kAttnKeys / kAttnKeyStep) * AttnTile<DP, kAttnKeyStep>::kBytes + 1024 + 8 * kAttnKeyWaves, kQueries = 4 * AttnTile<DP>::kBytes + 8 * kAttnWaves;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[kKeys > kQueries ? kKeys : kQueries];
    if ((int)blockIdx.x < k_groups) {
        AttnArgs K = A;
        K.tasks = k_tasks;
        attention_dkv<T, DP>(K, blockIdx.x, lds);
    } else {
        attention_dq<T, DP>(A, blockIdx.x - k_groups, lds);
    }
}

// The runs' sums added up, in their order: 8 elements a thread, dk and dv side by side
template <int T>
__global__ __launch_bounds__(256) void attention_add_kernel(const AttnArgs A) {
    const int64_t at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8, all = A.k_rows * A.kv_heads * A.dim;
    void* const out = blockIdx.y ? A.dv : A.dk;
    if (at >= all || !out) return;
    float x[8] = {};
    const float* p = A.k_part + blockIdx.y * all + at;
    for (int s = 0; s < A.k_splits; ++s, p += 2 * all) {
        const v4f a = *reinterpret_cast<const v4f*>(p), b = *reinterpret_cast<const v4f*>(p + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] += a[i];
            x[4 + i] += b[i];
        }
    }
    store_piece<T, 8>(out, at, x);
}

}  // namespace

int run_attention_backward_kernels(const AttnArgs& A, const AttnTask* k_tasks, int64_t k_tiles, const int* cu_q, const int* cu_k, int dtype, hipStream_t st) {
    return with_attn(dtype, A.dim, [&](auto t, auto d) {
        constexpr int T = decltype(t)::value, DP = decltype(d)::value;
        AttnArgs B = A;
        const int64_t q_groups = (A.q_rows * A.heads + 15) / 16, v_groups = (A.k_rows * A.kv_heads + 15) / 16;
        if (T == NTFP8_F16) B.most_q = (int)std::min<int64_t>(q_groups, kAttnMost), B.most_v = (int)std::min<int64_t>(v_groups, kAttnMost);
        const int first = T == NTFP8_F16 ? B.most_q : (int)q_groups;
        attention_delta_kernel<T><<<(unsigned)(first + B.most_v), 256, 0, st>>>(B, cu_q, cu_k, first);
        if (const int rc = launch_status(); rc != NTFP8_OK) return rc;
        const bool keys = A.dk || A.dv;
        const int64_t k_groups = keys ? k_tiles * A.kv_heads * A.k_splits : 0;
        const int64_t groups = k_groups + (A.dq ? A.tiles * A.kv_heads * attn_chunks(A.group, A.tile_heads) : 0);
        if (groups == 0) return (int)NTFP8_OK;   // (no keys, and dq not asked for)
        attention_backward_kernel<T, DP><<<(unsigned)groups, 64 * kAttnWaves, 0, st>>>(B, k_tasks, (int)k_groups);
        if (const int rc = launch_status(); rc != NTFP8_OK) return rc;
        if (keys && A.k_splits > 1) {
            attention_add_kernel<T><<<dim3((unsigned)((A.k_rows * A.kv_heads * A.dim + 2047) / 2048), 2), 256, 0, st>>>(A);
            if (const int rc = launch_status(); rc != NTFP8_OK) return rc;
        }
        return (int)NTFP8_OK;
    });
}

}  // namespace ntfp8

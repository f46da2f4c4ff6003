// Attention, forward: out = softmax(scale q k^T) v over sequences of any lengths, heads of queries sharing heads of keys.
//
// A row's softmax is one pass over its keys: with m the running maximum and l the running sum of exp(s - m), a tile of keys with maximum m' adds
// its exp(s - max(m, m')) after the sums so far are multiplied by exp(m - max(m, m')); out is the products' sum over l, lse = m + log l is kept for
// the backward pass.  All in units of log 2, so that an exponential is one instruction.
#include "attention.h"

namespace ntfp8 {
namespace {

// ------------------------------------------------------------------------------------------------ tasks
// The tiles of packed sequences, heaviest first: two lists, of queries (block 0) and of keys (block 1, where asked for).  Offsets are clamped to
// the rows that there are, so that none of them, whatever it holds, leads out of a tensor; rows before the first sequence and
// behind the last one get tasks that see nothing, which write zeros.
constexpr int kPlanThreads = 1024, kBuckets = 256;
struct Plan {
    const int* cu_q;
    const int* cu_k;
    int sequences;
    int q_rows, k_rows, causal;
    int q_tile, k_tile, q_tasks, k_tasks;   // rows a tile, tasks there is room for
    AttnTask* q_list;
    AttnTask* k_list;
};

__global__ __launch_bounds__(kPlanThreads) void attention_plan_kernel(const Plan P) {
    __shared__ int count[kBuckets], total;
    const bool keys = blockIdx.x == 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tile = keys ? P.k_tile : P.q_tile, own_rows = keys ? P.k_rows : P.q_rows, most = keys ? P.k_tasks : P.q_tasks;
    const int* const own_cu = keys ? P.cu_k : P.cu_q;
    const int* const other_cu = keys ? P.cu_q : P.cu_k;
    const int other_rows = keys ? P.q_rows : P.k_rows;
    AttnTask* const list = keys ? P.k_list : P.q_list;
    int unit = 1;   // of cost, so that the longest possible one falls into the last bucket
    while (other_rows / unit >= kBuckets) unit *= 2;
    for (int i = threadIdx.x; i < kBuckets; i += kPlanThreads) count[i] = 0;
    if (threadIdx.x == 0) total = 0;
    __syncthreads();
    auto clamped = [](int v, int most_) { return min(max(v, 0), most_); };
    // A lane reads a sequence, and makes its task where it is of one tile; the lanes share the tiles of a longer one.  (A wave for each sequence: 3000 of 8 rows
    // 185 us, 10 so; 256 of 64 rows 20 and 5)
    auto each = [&](auto&& f) {
        constexpr int kWaves = kPlanThreads / 64;
        for (int base = 0; base < P.sequences + 2; base += kPlanThreads) {
            const int own = base + lane * kWaves + wave;
            int a = 0, len = 0, b = 0, seen = 0;
            if (own < P.sequences) {
                a = clamped(own_cu[own], own_rows);
                len = max(0, clamped(own_cu[own + 1], own_rows) - a);
                b = clamped(other_cu[own], other_rows);
                seen = max(0, clamped(other_cu[own + 1], other_rows) - b);
            } else if (own == P.sequences) {
                len = clamped(own_cu[0], own_rows);
            } else if (own == P.sequences + 1) {
                a = clamped(own_cu[P.sequences], own_rows);
                len = own_rows - a;
            }
            auto put = [&](int s, int first, int rows, int other, int keys_of, int at) __attribute__((always_inline)) {
                const AttnTask t = {first + at, min(tile, rows - at), other, keys_of, at, s, keys ? at - (rows - keys_of) : at + keys_of - rows, 0};
                int cost = keys_of;
                if (P.causal) cost = keys ? keys_of - max(0, t.shift) : t.shift + t.rows;
                f(t, min(max(cost, 0) / unit, kBuckets - 1));
            };
            if (len > 0 && len <= tile) put(own, a, len, b, seen, 0);
            for (uint64_t longer = __ballot(len > tile); longer; longer &= longer - 1) {
                const int from = __ffsll((unsigned long long)longer) - 1;
                const int first = __shfl(a, from), rows = __shfl(len, from), other = __shfl(b, from), seen_there = __shfl(seen, from);
                for (int at = lane * tile; at < rows; at += 64 * tile) put(base + from * kWaves + wave, first, rows, other, seen_there, at);
            }
        }
    };
    each([&](const AttnTask&, int bucket) { atomicAdd(&count[bucket], 1); });
    __syncthreads();
    // where each bucket begins, the heaviest in front
    if (wave == 0) {
        int held[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            held[i] = count[kBuckets - 1 - (4 * lane + i)];
            sum += held[i];
        }
        int before = sum;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int o = __shfl_up(before, d);
            if (lane >= d) before += o;
        }
        if (lane == 63) total = before;
        before -= sum;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            count[kBuckets - 1 - (4 * lane + i)] = before;
            before += held[i];
        }
    }
    __syncthreads();
    each([&](const AttnTask& t, int bucket) {
        const int at = atomicAdd(&count[bucket], 1);   // (the order within a bucket reaches no result)
        if (at < most) list[at] = t;
    });
    for (int i = total + threadIdx.x; i < most; i += kPlanThreads) list[i] = {0, 0, 0, 0, 0, 0, 0, 0};
}

// ------------------------------------------------------------------------------------------------ prompts
// A workgroup owns 128 queries of one head, a wave 32 of them (or 32 queries of four heads, a wave each: AttnOwn), and walks their keys 64 at a time: scores of 64 keys by 32
// queries, the running maximum and sum, and the product with the values, into out^T [elements][queries]: the queries are the columns of both products,
// one a lane, so a row's maximum and sum stay in a lane (and its twin of the other half) and the scores are the second operand of the next product as
// they come.  Tiles of keys and values travel straight into LDS.  The scores of the next tile are made while the exponentials of this one are: products
// and arithmetic then share a wave's time.
//
// Bound by the products: 16384 causal tokens, 32 heads of 128 over 8, in bf16 take 2.0 to 2.1 ms, 1.1 PFLOP/s, with 63 to 65 % of the matrix instructions' slots taken at
// the 1.5 to 1.6 GHz that the power limit leaves (all-zero operands, the same instructions: 1.48 PFLOP/s); 4096 tokens 152 to 156 us.  Tried: 64 queries a
// wave, which halves the reads of LDS but moves sums between register files (slower); three and four tiles ahead, and waves of raised priority (nothing).
template <int T, int DP>
__global__ __launch_bounds__(64 * kAttnWaves, attn_workgroups(DP)) void attention_forward_kernel(const AttnArgs A) {
    typedef AttnTile<DP> Tile;
    __shared__ __attribute__((aligned(1024))) uint8_t sk[2 * Tile::kBytes];
    __shared__ __attribute__((aligned(1024))) uint8_t sv[2 * Tile::kBytes];
    __shared__ __attribute__((aligned(16))) int odd[2][kAttnWaves];   // [stage]: a wave's part of the values is not finite throughout
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttnOwn own = attn_own(A, blockIdx.x, wave);
    const int kv = own.kv, inside = own.inside, head = kv * A.group + inside, wave_row = own.row;
    const AttnTask task = attn_task(A, own.tile, A.tile_heads > 1 ? 32 : kAttnQueries, false);
    if (task.rows <= 0) return;
    const int64_t q0 = attn_rows(A, task.own, task.seq, task.at, A.q_stride, A.q_batch) + head * A.q_head;
    const int64_t k0 = attn_rows(A, task.other, task.seq, 0, A.k_stride, A.k_batch) + kv * A.k_head;
    const int64_t v0 = attn_rows(A, task.other, task.seq, 0, A.v_stride, A.v_batch) + kv * A.v_head;
    const int end = A.causal ? min(max(task.shift + task.rows, 0), task.len) : task.len;
    int first = 0, steps = (end + kAttnStep - 1) / kAttnStep;
    if (A.splits > 1) {
        const int each = (steps + A.splits - 1) / A.splits;
        first = blockIdx.y * each;
        steps = max(0, min(steps - first, each));
    }
    Tile tile;
    tile.init(lane);
    typename Tile::template Source<> ks, vs;
    ks.init(A.k, k0, A.k_stride, A.dim, wave, lane);
    vs.init(A.v, v0, A.v_stride, A.dim, wave, lane);
    if (steps > 0) ks.load(sk, first * kAttnStep, task.len, wave);
    const int row = wave_row + (lane & 31);
    const bool live = row < task.rows && inside < A.group;
    v4i q[DP / 16];
    load_own<DP>(q, A.q, q0 + row * A.q_stride, A.dim, live, lane);
    v16f out[DP / 32], s[2];
    float top = -__builtin_inff(), sum = 0.0f;   // maximum (of scores times c) and this half wave's sum
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) out[e] = zeros16();
    auto scores = [&](const uint8_t* keys, v16f (&to)[2]) __attribute__((always_inline)) {
        to[0] = to[1] = zeros16();
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
            to[0] = mfma_attn<T>(tile.rows(keys, 0, k), q[k], to[0]);
            to[1] = mfma_attn<T>(tile.rows(keys, 1, k), q[k], to[1]);
        }
    };
    if (steps > 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        wg_barrier();
        ks.load(sk + Tile::kBytes, (first + 1) * kAttnStep, task.len, wave);   // (behind the last key: zeros)
        vs.load(sv, first * kAttnStep, task.len, wave);
        scores(sk, s);
    }
    const bool idle = wave_row >= task.rows || inside >= A.group;   // a wave without rows brings its part of the tiles
    const int lead = task.shift + wave_row;                                             // the last key that the wave's first row sees
    const int last_key = A.causal ? min(task.len - 1, lead + (lane & 31)) : task.len - 1;   // and that this lane's does
    // a row's maximum of a tile's scores, in two chains
    auto largest = [&]() __attribute__((always_inline)) {
        float x = s[0][0], y = s[1][0];
#pragma unroll
        for (int r = 1; r < 16; ++r) {
            x = fmaxf(x, s[0][r]);
            y = fmaxf(y, s[1][r]);
        }
        return both_max(fmaxf(x, y)) * A.c;
    };
    // The exponentials are taken below a maximum that is raised only once a row's has grown by more than 2^8 (what is
    // kept in 16 bits loses nothing by that): rescaling the outputs is 64 multiplications a lane
    auto raise = [&](float most) __attribute__((always_inline)) {
        if (__any(most > top + 8.0f)) {
            const float now = fmaxf(top, most);
            const float by = now == top ? 1.0f : exp2_fast(top - now);
            sum *= by;
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) out[e] *= by;
            top = now;
        }
        return top == -__builtin_inff() ? 0.0f : top;
    };
    // exponentials of 4 scores, from register r of block g on
    auto exponentials = [&](int g, int r, float below) __attribute__((always_inline)) {
        float x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = s[g][r + i] = exp2_fast(__builtin_fmaf(s[g][r + i], A.c, -below));
        sum += (x[0] + x[1]) + (x[2] + x[3]);
    };
    // One tile of keys that every row of the workgroup sees whole.  A wave issues one instruction after another, so their
    // order is set here: between two products of 32 cycles each what is done beside them, and fragments read two pairs of products ahead.
    float most = steps > 0 ? largest() : 0.0f;
    auto whole_step = [&](int j) __attribute__((always_inline)) {
        const int key0 = (first + j) * kAttnStep, stage = (j & 1) * Tile::kBytes, other = Tile::kBytes - stage;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        wg_barrier();
        ks.load(sk + stage, key0 + 2 * kAttnStep, task.len, wave);
        vs.load(sv + other, key0 + kAttnStep, task.len, wave);
        if (idle) return;
        const float below = raise(most);
        constexpr int kPairs = DP / 16;   // of products of the next scores
        v4i fk[3][2], p[4];
        v16f next[2] = {zeros16(), zeros16()};
        auto fetch = [&](int k) __attribute__((always_inline)) {
            fk[k % 3][0] = tile.rows(sk + other, 0, k);
            fk[k % 3][1] = tile.rows(sk + other, 1, k);
        };
        v4i fv[4];
        auto fetch_v = [&](int x) __attribute__((always_inline)) { fv[x & 3] = tile.columns(sv + stage, x / (DP / 32), x % (DP / 32)); };
        fetch(0);
        fetch(1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            next[0] = mfma_attn<T>(fk[k % 3][0], q[k], next[0]);
            if (k + 2 < kPairs) fetch(k + 2);
            else fetch_v(k + 2 - kPairs);
            // the k-th share of 8 quadruples of exponentials
#pragma unroll
            for (int n = k * 8 / kPairs; n < (k + 1) * 8 / kPairs; ++n) exponentials(n / 4, n % 4 * 4, below);
            __builtin_amdgcn_sched_barrier(0);
            next[1] = mfma_attn<T>(fk[k % 3][1], q[k], next[1]);
#pragma unroll
            for (int n = k * 8 / kPairs; n < (k + 1) * 8 / kPairs; ++n)
                if (n % 2 == 1) p[n / 2] = pack_scores<T>(s[n / 4], n % 4 == 1 ? 0 : 8);
            __builtin_amdgcn_sched_barrier(0);
        }
        s[0] = next[0];
        s[1] = next[1];
#pragma unroll
        for (int x = 0; x < DP / 8; ++x) {
            if (x + 2 < DP / 8) fetch_v(x + 2);
            out[x % (DP / 32)] = mfma_attn<T>(fv[x & 3], p[x / (DP / 32)], out[x % (DP / 32)]);
            __builtin_amdgcn_sched_barrier(0);
        }
        most = largest();
    };
    // The scores' tile under its mask, into the sums.  kSingly: it holds values which are not finite
    auto masked = [&](int key0, uint8_t* values, auto singly_) __attribute__((always_inline)) {
        const int last = last_key - key0, last_half = last - 4 * (lane >> 5);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (32 * g + place_in_half(r) > last_half) s[g][r] = -__builtin_inff();
        const float below = raise(largest());
        v4i p[4];   // of 16 keys each
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int r = 0; r < 16; r += 4) exponentials(g, r, below);
            p[2 * g] = pack_scores<T>(s[g], 0);
            p[2 * g + 1] = pack_scores<T>(s[g], 8);
        }
        if constexpr (decltype(singly_)::value) {
            add_columns_singly<T, DP, 4>(out, tile, values, p, 0, last + 1);
        } else {
#pragma unroll
            for (int g = 0; g < 4; ++g) add_columns<T, DP>(out, tile, values, g, p[g]);
        }
    };
    // Any tile: rows that do not see all of it.  One with values which are not finite is left for later (of the same tiles, for
    // every wave): what such a tile needs would take registers from this loop
    bool left = false;
    auto step = [&](int j) __attribute__((always_inline)) {
        const int key0 = (first + j) * kAttnStep, stage = (j & 1) * Tile::kBytes, other = Tile::kBytes - stage;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        attn_tell(odd[j & 1], wave, attn_not_finite<T, DP, kAttnStep, kAttnWaves>(sv + stage, wave, lane));
        wg_barrier();
        if (j + 1 < steps) {
            ks.load(sk + stage, key0 + 2 * kAttnStep, task.len, wave);
            vs.load(sv + other, key0 + kAttnStep, task.len, wave);
        }
        const bool later = attn_any_wave(odd[j & 1]);
        left |= later;
        if (idle || (A.causal && key0 > lead + 31)) return;   // (uniform in the wave; so are the tiles behind this one)
        if (!later) masked(key0, sv + stage, std::false_type{});
        if (j + 1 < steps) scores(sk + other, s);
    };
    // tiles that every row sees whole (behind the last the next scores are made of zeros, beside its exponentials: less than a tile of its own kind), then the others
    const int whole = min(task.len, A.causal ? task.shift + 1 : task.len) / kAttnStep, clear = min(whole - first, steps);
    int j = 0;
    for (; j < clear; ++j) whole_step(j);
    for (; j < steps; ++j) step(j);
    if (__builtin_expect(left, 0)) {
        for (j = max(0, clear); j < steps; ++j) {
            const int key0 = (first + j) * kAttnStep;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            wg_barrier();
            ks.load(sk, key0, task.len, wave);
            vs.load(sv, key0, task.len, wave);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            attn_tell(odd[j & 1], wave, attn_not_finite<T, DP, kAttnStep, kAttnWaves>(sv, wave, lane));
            wg_barrier();
            if (!attn_any_wave(odd[j & 1]) || (A.causal && key0 > lead + 31)) continue;
            scores(sk, s);
            masked(key0, sv, std::true_type{});
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (what was requested behind the last tile lands in this workgroup's LDS)
    const float all = both_sum(sum);
    top = attn_top(top, first * kAttnStep <= last_key);   // (of this run's keys)
    const int64_t at = (int64_t)task.own + row;
    if (A.splits > 1) {
        if (!live) return;
        const int64_t to = ((int64_t)blockIdx.y * A.q_rows + at) * A.heads + head;
        if (lane < 32) A.part_ml[to] = make_float2(top, all);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * e + 8 * g + 4 * (lane >> 5);
                if (d < A.dim) *reinterpret_cast<v4f*>(A.part + to * A.dim + d) = (v4f){out[e][4 * g], out[e][4 * g + 1], out[e][4 * g + 2], out[e][4 * g + 3]};
            }
        return;
    }
    store_rows<T, DP>(out, attn_over(top, all), A.out, (at * A.heads + head) * A.dim, A.dim, live, lane, A.low);
    if (A.lse && live && lane < 32) A.lse[head * A.q_rows + at] = attn_lse(A, top, all);
}

// ------------------------------------------------------------------------------------------------ few queries
// Where the queries of a group of heads are 32 rows or fewer (a token, or a few, of every sequence) the keys are the work: the rows
// (head in its group, query) share them, every wave takes keys of its own, 32 at a time through LDS of its own without a
// barrier, and the waves' results are joined at the end; workgroups' (`splits` of a sequence) by a second launch.
// Bound by memory: 32 tokens over caches of 8192, 8 heads of 128 in bf16, are 1.07 GB in 190 us, 5.7 TB/s.  One token over 4096 keys is latency, 8.2 to
// 8.6 us here (a launch, the trip for keys and values, 8 products in a row, the waves' join) and 3.5 to 3.9 for the second launch.
constexpr int kFewStep = 32, kFewRows = 32;
template <int T, int DP>
__global__ __launch_bounds__(64 * kAttnWaves, 1) void attention_few_kernel(const AttnArgs A) {
    typedef AttnTile<DP> Tile;
    constexpr int kBytes = Tile::kBytes / 2, kLoads = kBytes / 1024, kStages = 2;
    __shared__ __attribute__((aligned(1024))) uint8_t sk[kAttnWaves][kStages * kBytes];
    __shared__ __attribute__((aligned(1024))) uint8_t sv[kAttnWaves][kStages * kBytes];
    __shared__ float2 ml[kAttnWaves][kFewRows];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int seq = blockIdx.x / A.kv_heads, kv = blockIdx.x - seq * A.kv_heads;
    const int n = A.q_len, rows = A.group * n;
    // this lane's row: query `token` of head `head`
    const int row = lane & 31, inside = row / n, token = row - inside * n, head = kv * A.group + inside;
    const bool live = row < rows;
    const int64_t q0 = seq * A.q_batch + token * A.q_stride + head * A.q_head;
    const int len = A.k_len, steps_all = (len + kFewStep - 1) / kFewStep, runs = A.splits * kAttnWaves, run = blockIdx.y * kAttnWaves + wave;
    const int each = (steps_all + runs - 1) / runs, first = run * each, steps = max(0, min(steps_all - first, each));
    const int last_row = A.causal ? len - n + token : len - 1;   // the last key that this row sees
    const int first_last = A.causal ? len - n : len - 1;         // and the row that sees least
    Tile tile;
    tile.init(lane);
    const char* const kp = static_cast<const char*>(A.k) + 2 * (seq * A.k_batch + kv * A.k_head);
    const char* const vp = static_cast<const char*>(A.v) + 2 * (seq * A.v_batch + kv * A.v_head);
    const int64_t kb = 2 * A.k_stride, vb = 2 * A.v_stride;
    uint32_t koff[kLoads], voff[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int byte = (i * 64 + lane) * 16, r = byte / Tile::kPitch, chunk = (byte % Tile::kPitch >> 4) ^ Tile::swizzle(r);
        koff[i] = chunk * 8 < A.dim ? (uint32_t)r * (uint32_t)kb + chunk * 16 : kNowhere;
        voff[i] = chunk * 8 < A.dim ? (uint32_t)r * (uint32_t)vb + chunk * 16 : kNowhere;
    }
    // (a step behind the last is all zeros: every step is the same number of loads)
    auto load = [&](int j) {
        const int key = (first + j) * kFewStep, count = j < steps ? min(kFewStep, len - key) : 0;
        const uint32_t kbytes = count > 0 ? (uint32_t)(count - 1) * (uint32_t)kb + 2u * A.dim : 0u, vbytes = count > 0 ? (uint32_t)(count - 1) * (uint32_t)vb + 2u * A.dim : 0u;
        const __amdgpu_buffer_rsrc_t rk = make_rsrc(kp + (count > 0 ? key * kb : 0), (uint32_t)__builtin_amdgcn_readfirstlane((int)kbytes));
        const __amdgpu_buffer_rsrc_t rv = make_rsrc(vp + (count > 0 ? key * vb : 0), (uint32_t)__builtin_amdgcn_readfirstlane((int)vbytes));
        uint8_t* const k = sk[wave] + (j & 1) * kBytes;
        uint8_t* const v = sv[wave] + (j & 1) * kBytes;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) lds_load16(rk, (lds_ptr)(uintptr_t)(k + i * 1024), koff[i], 0);
#pragma unroll
        for (int i = 0; i < kLoads; ++i) lds_load16(rv, (lds_ptr)(uintptr_t)(v + i * 1024), voff[i], 0);
    };
    if (steps > 0) {
        load(0);
        load(1);
    }
    v4i q[DP / 16];   // (behind the first keys and values: what waits for it, waits for one trip to memory and not for two)
    load_own<DP>(q, A.q, q0, A.dim, live, lane);
    v16f out[DP / 32];
#pragma unroll
    for (int e = 0; e < DP / 32; ++e) out[e] = zeros16();
    float top = -__builtin_inff(), sum = 0.0f;
    // A step's scores and values into the sums.  kSingly: some rows do not see all of its values, which are not finite throughout
    auto add = [&](int j, bool masked, auto singly_) __attribute__((always_inline)) {
        uint8_t* const k = sk[wave] + (j & 1) * kBytes;
        uint8_t* const v = sv[wave] + (j & 1) * kBytes;
        v16f s = zeros16();
#pragma unroll
        for (int i = 0; i < DP / 16; ++i) s = mfma_attn<T>(tile.rows(k, 0, i), q[i], s);
        const int last = min(len - 1, last_row) - (first + j) * kFewStep, last_half = last - 4 * (lane >> 5);
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (place_in_half(r) > last_half) s[r] = -__builtin_inff();
        }
        float most = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) most = fmaxf(most, s[r]);
        most = both_max(most) * A.c;
        if (__any(most > top + 8.0f)) {
            const float now = fmaxf(top, most), by = now == top ? 1.0f : exp2_fast(top - now);
            sum *= by;
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) out[e] *= by;
            top = now;
        }
        const float below = top == -__builtin_inff() ? 0.0f : top;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(__builtin_fmaf(s[r], A.c, -below));
            sum += s[r];
        }
        const v4i p[2] = {pack_scores<T>(s, 0), pack_scores<T>(s, 8)};
        if constexpr (decltype(singly_)::value) {
            add_columns_singly<T, DP, 2>(out, tile, v, p, 0, last + 1);
        } else {
            add_columns<T, DP>(out, tile, v, 0, p[0]);
            add_columns<T, DP>(out, tile, v, 1, p[1]);
        }
    };
    auto masked_at = [&](int j) { return (first + j) * kFewStep + kFewStep - 1 > min(len - 1, first_last); };
    bool left = false;   // a step for later, see above
    for (int j = 0; j < steps; ++j) {
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");   // all but the step requested since
        const bool masked = masked_at(j);
        if (masked && attn_not_finite<T, DP, kFewStep, 1>(sv[wave] + (j & 1) * kBytes, 0, lane)) left = true;
        else add(j, masked, std::false_type{});
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the stage has been read
        __builtin_amdgcn_sched_barrier(0);
        load(j + 2);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (the last requests write zeros into stages nobody reads again)
    if (__builtin_expect(left, 0)) {
        for (int j = 0; j < steps; ++j) {
            if (!masked_at(j)) continue;
            load(j);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            if (attn_not_finite<T, DP, kFewStep, 1>(sv[wave] + (j & 1) * kBytes, 0, lane)) add(j, true, std::true_type{});
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
    }
    sum = both_sum(sum);
    top = attn_top(top, first * kFewStep <= min(len - 1, last_row));   // (of this wave's keys)
    if (lane < kFewRows) ml[wave][lane] = make_float2(top, sum);
    __syncthreads();
    float all_top = -__builtin_inff(), all_sum = 0.0f;
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) all_top = fmaxf(all_top, ml[w][row].x);
#pragma unroll
    for (int w = 0; w < kAttnWaves; ++w) {
        const float2 o = ml[w][row];
        if (o.x != -__builtin_inff()) all_sum += o.y * (o.x == all_top ? 1.0f : exp2_fast(o.x - all_top));
    }
    const float mine = top == -__builtin_inff() ? 0.0f : top == all_top ? 1.0f : exp2_fast(top - all_top);
    // the waves' outputs, [wave][element][row] in the stages that they no longer need, added up in the order of the waves
    float* const at = reinterpret_cast<float*>(&sk[0][0]);
    static_assert(sizeof(sk[0]) >= sizeof(float) * 64 * kFewRows && sizeof(sk) + sizeof(sv) >= sizeof(float) * kAttnWaves * DP * kFewRows, "");
    // (64 elements a wave in the stages of keys, the others in those of values)
    float* const over = reinterpret_cast<float*>(&sv[0][0]);
#pragma unroll
    for (int e = 0; e < DP / 32; ++e)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float* const to = e < 2 ? at : over;
            to[(wave * 64 + 32 * (e & 1) + place_of(r, lane)) * kFewRows + row] = out[e][r] * mine;   // (0 times what is not finite is NaN, as within a wave)
        }
    __syncthreads();
    // 8 threads a row, 8 elements at a time
    const int r = threadIdx.x & 31;
    if (r < rows) {
        const int in = r / n, tok = r - in * n, hd = kv * A.group + in;
        const int64_t out_row = (int64_t)seq * n + tok;
        const int64_t to = ((int64_t)blockIdx.y * A.q_rows + out_row) * A.heads + hd;
        const float by = A.splits > 1 ? 1.0f : attn_over(all_top, all_sum);
        for (int d = (threadIdx.x >> 5) * 8; d < A.dim; d += 64) {
            const float* const from = d < 64 ? at : over;
            float x[8] = {};
#pragma unroll
            for (int w = 0; w < kAttnWaves; ++w)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] += from[(w * 64 + (d & 63) + i) * kFewRows + r];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= by;
            if (A.splits > 1) store_piece<NTFP8_F32, 8>(A.part, to * A.dim + d, x);
            else {
                store_piece<T, 8>(A.out, (out_row * A.heads + hd) * A.dim + d, x);
                if (A.low) store_low<T>(A.low, (out_row * A.heads + hd) * A.dim + d, x);
            }
        }
        if (threadIdx.x < kFewRows) {
            if (A.splits > 1) A.part_ml[to] = make_float2(all_top, all_sum);
            else if (A.lse) A.lse[hd * A.q_rows + out_row] = attn_lse(A, all_top, all_sum);
        }
    }
}

// The splits' results joined: a row of one head is a wave's, 16 lanes of 8 elements by four runs of splits
template <int T, int kAhead>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttnArgs A) {
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), pitch = A.q_rows * A.heads;
    if (row >= pitch) return;   // (whole waves)
    const int lane = threadIdx.x & 63, d = (lane & 15) * 8, run = lane >> 4;
    // the first splits are asked for before the largest maximum is known: one trip to memory for two (a token over 4096 keys, 32 splits, 12.7 -> 11.1 us;
    // 4 times as many as there are cost 512 tokens over 8192 keys 4 us of 84)
    float2 ml[kAhead];
    v4f part[kAhead][2];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
        const int s = run + 4 * i;
        ml[i] = make_float2(-__builtin_inff(), 0.0f);
        part[i][0] = part[i][1] = (v4f){0, 0, 0, 0};
        if (s >= A.splits) continue;
        ml[i] = A.part_ml[s * pitch + row];
        if (d >= A.dim) continue;
        const v4f* const p = reinterpret_cast<const v4f*>(A.part + (s * pitch + row) * A.dim + d);
        part[i][0] = p[0], part[i][1] = p[1];
    }
    // every lane's splits, one after another: their largest maximum
    float top = -__builtin_inff();
    for (int s = lane; s < A.splits; s += 64) top = fmaxf(top, A.part_ml[s * pitch + row].x);
#pragma unroll
    for (int m = 32; m >= 1; m /= 2) top = fmaxf(top, __shfl_xor(top, m));
    float sum = 0.0f, x[8] = {};
    auto add = [&](float2 o, v4f a, v4f b) __attribute__((always_inline)) {
        // (of a split of which the row sees nothing, nothing counts)
        const float by = o.x == -__builtin_inff() ? 0.0f : o.x == top ? 1.0f : exp2_fast(o.x - top);
        sum += o.y * by;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] += a[i] * by;
            x[4 + i] += b[i] * by;
        }
    };
#pragma unroll
    for (int i = 0; i < kAhead; ++i) add(ml[i], part[i][0], part[i][1]);
    for (int s = run + 4 * kAhead; s < A.splits; s += 4) {
        const v4f* const p = reinterpret_cast<const v4f*>(A.part + (s * pitch + row) * A.dim + d);
        if (d < A.dim) add(A.part_ml[s * pitch + row], p[0], p[1]);
        else add(A.part_ml[s * pitch + row], (v4f){0, 0, 0, 0}, (v4f){0, 0, 0, 0});
    }
#pragma unroll
    for (int m = 16; m <= 32; m *= 2) {
        sum += __shfl_xor(sum, m);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] += __shfl_xor(x[i], m);
    }
    if (run != 0) return;
    if (d < A.dim) {
        const float over = attn_over(top, sum);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] *= over;
        store_piece<T, 8>(A.out, row * A.dim + d, x);
        if (A.low) store_low<T>(A.low, row * A.dim + d, x);
    }
    if (A.lse && d == 0) A.lse[(row % A.heads) * A.q_rows + row / A.heads] = attn_lse(A, top, sum);
}

}  // namespace

// ------------------------------------------------------------------------------------------------ launches
int run_attention_plan(const int* cu_q, const int* cu_k, int sequences, int q_rows, int k_rows, int causal, int q_tile, int k_tile, int q_tasks, int k_tasks,
                       AttnTask* q_list, AttnTask* k_list, hipStream_t st) {
    const Plan p = {cu_q, cu_k, sequences, q_rows, k_rows, causal, q_tile, k_tile, q_tasks, k_tasks, q_list, k_list};
    attention_plan_kernel<<<k_list ? 2 : 1, kPlanThreads, 0, st>>>(p);
    return launch_status();
}

int run_attention_forward_kernels(const AttnArgs& A, int dtype, bool few, hipStream_t st) {
    return with_attn(dtype, A.dim, [&](auto t, auto d) {
        constexpr int T = decltype(t)::value, DP = decltype(d)::value;
        const dim3 grid((unsigned)(few ? (int64_t)A.sequences * A.kv_heads : A.tiles * A.kv_heads * attn_chunks(A.group, A.tile_heads)), (unsigned)A.splits);
        if (few) attention_few_kernel<T, DP><<<grid, 64 * kAttnWaves, 0, st>>>(A);
        else attention_forward_kernel<T, DP><<<grid, 64 * kAttnWaves, 0, st>>>(A);
        if (const int rc = launch_status(); rc != NTFP8_OK || A.splits <= 1) return rc;
        const unsigned rows = (unsigned)((A.q_rows * A.heads + 3) / 4);
        if (A.splits <= 4) attention_join_kernel<T, 1><<<rows, 256, 0, st>>>(A);
        else attention_join_kernel<T, 8><<<rows, 256, 0, st>>>(A);
        return launch_status();
    });
}

}  // namespace ntfp8

// Attention: which kernels a call takes, how the work is cut, and what lies where in the workspace.
#include "attention.h"

namespace ntfp8 {

int run_attention_plan(const int* cu_q, const int* cu_k, int sequences, int q_rows, int k_rows, int causal, int q_tile, int k_tile, int q_tasks, int k_tasks,
                       AttnTask* q_list, AttnTask* k_list, hipStream_t st);
int run_attention_forward_kernels(const AttnArgs& A, int dtype, bool few, hipStream_t st);
int run_attention_backward_kernels(const AttnArgs& A, const AttnTask* k_tasks, int64_t k_tiles, const int* cu_q, const int* cu_k, int dtype, hipStream_t st);

namespace {

int64_t up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }
// tiles of `tile` rows: exactly of equal sequences, at most of packed ones (each may end in part of one, and so may the rows of none)
int64_t tiles_of(const ntops_attention_desc& d, int64_t rows, int64_t tile) {
    if (d.cu_q) return rows / tile + d.sequences + 2;
    return d.sequences * ((rows / d.sequences + tile - 1) / tile);
}

// Heads of a group whose 32 queries a workgroup's waves take, or 1, and 128 queries of that one: what leaves fewer waves without rows; of packed sequences,
// whose tiles end anywhere, also where that is equal, up to a length that makes no difference.  (us: a token of 32 sequences over 8192 keys each, packed, 32
// heads of 128 over 8, 204 to 214 and 385 by one head; 64 causal sequences of 16384 tokens, forward 131 and 147, both passes 525 and 560; 4 sequences of 64
// over 2000 keys 31 and 36.  64 causal sequences of a batch of 512, equal waves: 302 and 290.)
constexpr int64_t kSharedRows = 1024;
int tile_heads_of(const ntops_attention_desc& d) {
    const int64_t rows = std::max<int64_t>(1, d.q_rows / d.sequences);   // (of packed ones, on average)
    const int group = d.heads / d.kv_heads;
    const int64_t apart = (rows + 31) / 32 * attn_chunks(group, kAttnWaves), one = (rows + kAttnQueries - 1) / kAttnQueries * group;
    return group > 1 && rows <= kSharedRows && (apart < one || (d.cu_q && apart == one)) ? kAttnWaves : 1;
}
int queries_of(const ntops_attention_desc& d) { return tile_heads_of(d) > 1 ? 32 : kAttnQueries; }

struct Choice {
    bool few;
    int splits;
    int64_t tiles;
};
// Rows of a group's heads that a wave's products have columns for, 32, are the few kernel's (us, for it and for the other: a token over 4096 keys, 32
// heads of 128 over 8, 11.1 and 17.4; 32 such tokens over 8192 191 and 458; 32 tokens of 8 heads over 4096 14.2 and 17.2).  Both cut the keys where
// there are fewer workgroups than the chip holds.  Few rows, into 128 keys at least, a step of each of four waves, and only beyond 512, which four steps
// take as long as the launch that joins (uncut and cut, over 256 keys 8.4 and 10.4, 512 10.2 and 10.4, 640 11.1 and 10.4; into 128 and 256, 4096
// keys 11.1 and 11.7).  More rows, into 512 keys at least (512 tokens over 8192 keys 85, 130 uncut, 95 with twice as many runs; of
// 512 and 256 at least: 512 tokens of 32 heads of 128 24 and 34, 1500 of 2 heads 33 and 30).  Packed sequences are cut by their average length, which is all that the
// host knows: a token each, 32 heads of 128 over 8, over 32 caches of 260 to 16380 keys in even steps 319 us for 213 at the copy's rate, of 128 to 32768 evenly in their
// logarithm 515 for 145, over one of 32768 and 31 of 100, uncut, 511 for 29.
Choice choose(const ntops_attention_desc& d) {
    const int64_t cus = cu_count(), q_len = d.q_rows / d.sequences, k_len = d.k_rows / d.sequences;   // (of packed ones, on average)
    Choice c = {};
    c.splits = 1;
    c.few = !d.cu_q && d.heads / d.kv_heads * q_len <= 32 && d.sequences * d.kv_heads <= ((int64_t)1 << 22);
    if (c.few) {
        const int64_t units = d.sequences * d.kv_heads;
        c.splits = (int)std::max<int64_t>(1, std::min((cus + units - 1) / units, k_len <= 512 ? 1 : k_len / 128));
        return c;
    }
    c.tiles = tiles_of(d, d.q_rows, queries_of(d));
    const int64_t groups = c.tiles * d.kv_heads * attn_chunks(d.heads / d.kv_heads, tile_heads_of(d)), room = 2 * cus;
    if (groups < room) c.splits = (int)std::max<int64_t>(1, std::min(room / groups, k_len / 512));
    return c;
}

// Runs that the queries of a tile of keys are cut into, so that there are workgroups of keys for two and a half a CU (two or three have room, those of queries
// fill in), but none of less than 10 steps where it is longest (of packed sequences, where one is twice as long as their average).  Backward, us, 32 heads
// of 128 over 8, for two, two and a half, three and four a CU: 1024 tokens 64, 65, 73, 91; 2048 160, 153, 161, 173; 4096 648, 474, 473, 485.  For
// 8, 10 and 16 steps at least: 512 tokens of these heads 38, 40, 45; 1500 of 2 heads of 128 47, 45, 41; 1000 of 4 of 64 over one 29, 27, 27.
int key_splits(const ntops_attention_desc& d) {
    if (d.k_rows == 0) return 1;   // (nothing to add up: a launch of no workgroups is an error)
    const int64_t rows = std::min(d.q_rows, d.q_rows / d.sequences * (d.cu_q && d.sequences > 1 ? 2 : 1));
    const int64_t units = std::max<int64_t>(1, tiles_of(d, d.k_rows, kAttnKeys) * d.kv_heads), steps = (rows + kAttnKeyStep - 1) / kAttnKeyStep * (d.heads / d.kv_heads);
    return (int)std::max<int64_t>(1, std::min(5 * cu_count() / 2 / units, steps / 10));
}

// Tasks of packed sequences: those of queries, and behind them those of keys
struct Plan {
    int64_t q_tiles, k_tiles, keys_at, bytes;
};
Plan plan_of(const ntops_attention_desc& d) {
    Plan p = {tiles_of(d, d.q_rows, queries_of(d)), tiles_of(d, d.k_rows, kAttnKeys), 0, 0};
    p.keys_at = up(p.q_tiles * (int64_t)sizeof(AttnTask), 256);
    p.bytes = p.keys_at + up(p.k_tiles * (int64_t)sizeof(AttnTask), 256);
    return p;
}

struct Layout {
    int64_t plan, part, part_ml, delta, most, k_part, bytes;
};
Layout layout_of(const ntops_attention_desc& d, bool backward, const Choice& c) {
    Layout l = {};
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        const int64_t here = at;
        at += up(bytes, 256);
        return here;
    };
    l.plan = take(d.cu_q && !d.plan ? plan_of(d).bytes : 0);
    if (backward) {
        l.delta = take(d.q_rows * d.heads * 4);
        l.most = take(d.dtype == NTFP8_F16 ? 2 * kAttnMost * 4 : 0);
        const int splits = key_splits(d);
        if (splits > 1) l.k_part = take(2 * splits * d.k_rows * d.kv_heads * d.head_dim * 4);
    } else if (c.splits > 1) {
        l.part = take(c.splits * d.q_rows * d.heads * d.head_dim * 4);
        l.part_ml = take(c.splits * d.q_rows * d.heads * 8);
    }
    l.bytes = at;
    return l;
}

AttnArgs args_of(const ntops_attention_desc& d) {
    AttnArgs a = {};
    a.q = d.q, a.k = d.k, a.v = d.v, a.dout = d.dout;
    a.q_stride = d.q_stride, a.k_stride = d.k_stride, a.v_stride = d.v_stride, a.do_stride = d.do_stride;
    a.q_head = d.q_head, a.k_head = d.k_head, a.v_head = d.v_head, a.do_head = d.do_head;
    a.q_batch = d.q_batch, a.k_batch = d.k_batch, a.v_batch = d.v_batch, a.do_batch = d.do_batch;
    a.sequences = (int)d.sequences, a.q_len = (int)(d.q_rows / d.sequences), a.k_len = (int)(d.k_rows / d.sequences);
    a.q_rows = d.q_rows, a.k_rows = d.k_rows;
    a.tile_heads = tile_heads_of(d), a.heads = d.heads, a.kv_heads = d.kv_heads, a.group = d.heads / d.kv_heads, a.dim = d.head_dim, a.causal = d.causal;
    a.c = d.scale * kLog2E, a.scale = d.scale;
    a.out = d.out, a.o = d.out, a.low = d.out_low, a.lse = d.lse, a.dq = d.dq, a.dk = d.dk, a.dv = d.dv, a.splits = 1;
    return a;
}

}  // namespace

// What a launch has to hold: workgroups, and threads, in 32 bits
bool attention_fits(const ntops_attention_desc& d) {
    constexpr int64_t kMost = (int64_t)1 << 22;
    return tiles_of(d, d.q_rows, queries_of(d)) * d.kv_heads * attn_chunks(d.heads / d.kv_heads, tile_heads_of(d)) <= kMost && tiles_of(d, d.q_rows, kAttnQueries) * d.heads <= kMost && tiles_of(d, d.k_rows, kAttnKeys) * d.kv_heads <= kMost;
}

int64_t attention_plan(const ntops_attention_desc& d) { return d.cu_q ? plan_of(d).bytes : 0; }

int64_t attention_workspace(const ntops_attention_desc& d, bool backward) {
    return layout_of(d, backward, choose(d)).bytes;
}

namespace {
// the tasks of a call's sequences at `at`; those of keys where a backward pass reads them
int make_plan(const ntops_attention_desc& d, char* at, bool keys, hipStream_t st) {
    const Plan p = plan_of(d);
    return run_attention_plan(d.cu_q, d.cu_k, (int)d.sequences, (int)d.q_rows, (int)d.k_rows, d.causal, queries_of(d), kAttnKeys, (int)p.q_tiles, (int)p.k_tiles,
                              reinterpret_cast<AttnTask*>(at), keys ? reinterpret_cast<AttnTask*>(at + p.keys_at) : nullptr, st);
}
}  // namespace

int run_attention_forward(const ntops_attention_desc& d, hipStream_t st) {
    const Choice c = choose(d);
    const Layout l = layout_of(d, false, c);
    char* const ws = static_cast<char*>(d.workspace);
    AttnArgs a = args_of(d);
    a.tiles = c.tiles, a.splits = c.splits;
    if (c.splits > 1) a.part = reinterpret_cast<float*>(ws + l.part), a.part_ml = reinterpret_cast<float2*>(ws + l.part_ml);
    if (d.cu_q) {
        char* const plan = d.plan ? static_cast<char*>(d.plan) : ws + l.plan;
        a.tasks = reinterpret_cast<AttnTask*>(plan);
        if (const int rc = make_plan(d, plan, d.plan != nullptr, st)) return rc;
    }
    return run_attention_forward_kernels(a, d.dtype, c.few, st);
}

int run_attention_backward(const ntops_attention_desc& d, hipStream_t st) {
    AttnArgs a = args_of(d);
    const Plan p = plan_of(d);
    a.tiles = p.q_tiles;
    const Layout l = layout_of(d, true, {});
    char* const ws = static_cast<char*>(d.workspace);
    a.delta = reinterpret_cast<float*>(ws + l.delta), a.most = reinterpret_cast<uint32_t*>(ws + l.most);
    a.k_splits = key_splits(d), a.k_part = reinterpret_cast<float*>(ws + l.k_part);
    const AttnTask* k_list = nullptr;
    if (d.cu_q) {
        char* const plan = d.plan ? static_cast<char*>(d.plan) : ws + l.plan;
        a.tasks = reinterpret_cast<AttnTask*>(plan);
        k_list = reinterpret_cast<AttnTask*>(plan + p.keys_at);
        if (!d.plan)
            if (const int rc = make_plan(d, plan, true, st)) return rc;
    }
    return run_attention_backward_kernels(a, k_list, p.k_tiles, d.cu_q, d.cu_k, d.dtype, st);
}

}  // namespace ntfp8

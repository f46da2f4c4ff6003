// AdamW over many tensors, moments in fp32 or in 8 bits.
//
// Bound by memory: an fp32 parameter with a 16-bit gradient moves 26 bytes with fp32 moments, 14 with 8-bit ones.  One launch
// takes as many tensors as its arguments hold (59 to 122), their pointers and sizes among them, so that nothing has
// to be copied to the device first; a workgroup takes a run of elements of one tensor.  A decoder layer of 218 million fp32
// parameters with fp32 moments, 16-bit gradients and copies: 1030 us, 28 bytes each at 5.9 TB/s; with 8-bit moments and fp32
// gradients 555 us, 16.3 bytes at 6.4 TB/s.
//
// 8-bit moments.  The first moment m and the root r of the second are kept as E4M3 codes, blocks of 256 elements with a
// power-of-two scale each, found from the new values: a wave holds a block, four elements a lane, so that the block's
// largest magnitude is a fold over the lanes and the codes never exist anywhere but in registers and the state.
//   * r and not r^2: the format's 17 binades then span 34 of the second moment.
//   * Stochastic rounding: beta2 = 0.95 moves r by at most 2.5 % a step downwards, less than half a step of the format (3 to
//     6 %); rounded to nearest it would never fall.  The 16 bits are hashed from the element's place and the caller's seed,
//     and both moments of an element use the same ones, so that their errors partly cancel in m / r.
//   * r above zero keeps the smallest code: a root of zero under a first moment that is not would divide by eps.
//   * What is not finite becomes NaN by itself: the scale is found from the block's finite values.  (A scale that made room for an
//     infinity would leave its neighbours the smallest code alone, 2^111, whose square is infinite in the next step.)
#include "ops_common.h"

namespace ntfp8 {
namespace {

constexpr int kThreads = 256, kEach = 4;
constexpr int kBlock = NTOPS_ADAMW_BLOCK;
static_assert(kBlock == 64 * kEach, "a wave holds a block of 8-bit moments");
constexpr int kChunk = kThreads * kEach;   // elements of a workgroup

// What a launch knows of a tensor: as little as its kind needs, the arguments of a launch being 4 KB, and addresses in the 48
// bits that they have.  (200 tensors of up to 20 000 elements go in two launches instead of three, 18.9 us instead of 20.7.)
template <int N>
struct Addresses {
    uint32_t low[N];
    uint16_t high[N];
    __device__ __forceinline__ void* operator[](int i) const {
        typedef void __attribute__((address_space(1)))* global;   // (said, so that the compiler knows it of a number)
        return (void*)(global)((uint64_t)high[i] << 32 | low[i]);
    }
    void set(int i, const void* p) {
        low[i] = (uint32_t)reinterpret_cast<uintptr_t>(p);
        high[i] = (uint16_t)(reinterpret_cast<uintptr_t>(p) >> 32);
    }
};
// (whole addresses: a step of 5 million parameters with 8-bit moments takes 14.5 us, 14.9 if it puts them together)
template <int N>
struct WholeAddresses {
    void* p[N];
    __device__ __forceinline__ void* operator[](int i) const { return p[i]; }
    void set(int i, const void* q) { p[i] = const_cast<void*>(q); }
};
template <bool k8>
struct Entry {
    Addresses<4> at;   // parameter, gradient, moments
    int n;
};
template <>
struct Entry<true> {
    WholeAddresses<6> at;   // and the scales of both moments
    int n;
    uint32_t pair;          // number of the first pair of elements in its tensor, which may have several entries
};
template <bool k8, bool kCopy>
struct Step {
    static constexpr int kMost = (3968 - 64) / (int)(sizeof(Entry<k8>) + 4 + (kCopy ? sizeof(Addresses<2>) / 2 : 0));
    Entry<k8> t[kMost];
    int first[kMost];              // first workgroup of the launch for each tensor; 2^31 - 1 behind the last
    Addresses<kCopy ? kMost : 1> copy;
    const float* grad_scale;
    float beta1, rest1, beta2, rest2, keep, to, root, eps;
    uint32_t seed;
    int copy_dtype;
};
static_assert(sizeof(Step<false, false>) <= 4096 && sizeof(Step<true, true>) <= 4096 && Step<false, false>::kMost <= 128, "");

// 16 bits for each of the two elements of a pair, the even one's in the low half
__device__ __forceinline__ uint32_t dither_of(uint32_t pair, uint32_t seed) {
    uint32_t x = pair * 0x9E3779B1u + seed;   // (seed times an odd constant, from the host)
    x = (x ^ (x >> 15)) * 0x6A09E667u;
    x = (x ^ (x >> 13)) * 0x3C6EF373u;
    return x ^ (x >> 16);
}

// exponent k of the block scale 2^k from the bits of its largest magnitude: 2^k times it lies in (224, 448]
__device__ __forceinline__ int scale_exponent(uint32_t top) {
    const int k = 135 - (int)(top >> 23) - ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return top == 0u ? 0 : min(max(k, -126), 126);
}

// |value| times the scale (at most 448) plus its dither -> code without sign.  Below 2^-6 codes are 2^-9 apart, as they are
// from 2^-6 to 2^-5: moved up by 2^-6 a value is rounded like one of those, 8 codes further on.
__device__ __forceinline__ uint32_t encode(float a, float scale, uint32_t dither) {
    const float y = a * scale;
    const bool small = y < 0x1p-6f;
    return ((__float_as_uint(y + (small ? 0x1p-6f : 0.0f)) + (dither << 4)) >> 20) - (small ? 968u : 960u);
}

template <int N>
__device__ __forceinline__ void decode(uint32_t w, float inverse, float (&v)[N]) {
    static_assert(N == 4, "");
    typedef float v2 __attribute__((ext_vector_type(2)));
    const v2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    v[0] = lo.x * inverse, v[1] = lo.y * inverse, v[2] = hi.x * inverse, v[3] = hi.y * inverse;
}

// Four elements a thread and no loop: with four such pieces a thread, all requested before the first was used, steps were
// as fast from 4 million elements on with fp32 moments, slower with 8-bit ones (12.7 million bf16 parameters 35.5 / 40.2 us) and
// below (0.9 million fp32 ones 6.0 / 8.0).
// kStream: what a step moves does not fit the memory-side cache (256 MB) and is read and written past the caches.  us, with /
// without: a decoder layer of 218 million fp32 parameters with fp32 moments 1016 / 1130, with 8-bit ones 554 / 596; 12.7 million,
// which fit, 54 / 49 where the same ones were stepped just before.
template <int P, int G, bool k8, bool kCopy, bool kStream>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Step<k8, kCopy> s) {
    // The last tensor whose first workgroup is not behind this one: every lane compares one, so that the arguments are read
    // in one trip (looked up by halves they are seven dependent ones, 3 us in front of a workgroup's first load)
    const int lane = threadIdx.x & 63;
    int which = __popcll(__ballot(lane < s.kMost && s.first[lane] <= (int)blockIdx.x));
    if constexpr (s.kMost > 64) which += __popcll(__ballot(lane + 64 < s.kMost && s.first[min(lane + 64, s.kMost - 1)] <= (int)blockIdx.x));
    which = __builtin_amdgcn_readfirstlane(which - 1);
    const Entry<k8> entry = s.t[which];
    const struct {
        void *p, *g, *m, *v;
    } T = {entry.at[0], entry.at[1], entry.at[2], entry.at[3]};
    const int64_t n = entry.n, i = (int64_t)((int)blockIdx.x - s.first[which]) * kChunk + threadIdx.x * kEach;
    const int left = i < n ? (int)min((int64_t)kEach, n - i) : 0;
    float* const scale_m = static_cast<float*>(entry.at[k8 ? 4 : 0]);
    float* const scale_v = static_cast<float*>(entry.at[k8 ? 5 : 0]);
    void* const copy = s.copy[kCopy ? which : 0];
    float p[kEach], g[kEach], m[kEach], v[kEach], r[kEach];
    const Piece<P, kEach> pr = load_piece<P, kEach, kStream>(T.p, i, left);
    const Piece<G, kEach> gr = load_piece<G, kEach, kStream>(T.g, i, left);
    if constexpr (k8) {
        uint32_t mc = 0, vc = 0;
        float ms = 1.0f, vs = 1.0f;
        if (left == kEach) {
            mc = reinterpret_cast<const Word*>(static_cast<const uint8_t*>(T.m) + i)->w;
            vc = reinterpret_cast<const Word*>(static_cast<const uint8_t*>(T.v) + i)->w;
        } else {
            for (int e = 0; e < left; ++e) {
                mc |= (uint32_t)static_cast<const uint8_t*>(T.m)[i + e] << (8 * e);
                vc |= (uint32_t)static_cast<const uint8_t*>(T.v)[i + e] << (8 * e);
            }
        }
        if (left) {
            ms = scale_m[i / kBlock];
            vs = scale_v[i / kBlock];
        }
        decode(mc, __builtin_amdgcn_rcpf(ms), m);   // (exact: powers of two)
        decode(vc, __builtin_amdgcn_rcpf(vs), v);
    } else {
        unpack<NTFP8_F32, kEach>(load_piece<NTFP8_F32, kEach, kStream>(T.m, i, left), m);
        unpack<NTFP8_F32, kEach>(load_piece<NTFP8_F32, kEach, kStream>(T.v, i, left), v);
    }
    const float factor = s.grad_scale ? *s.grad_scale : 1.0f;
    unpack<P, kEach>(pr, p);
    unpack<G, kEach>(gr, g);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        g[e] *= factor;
        m[e] = s.beta1 * m[e] + s.rest1 * g[e];
        if constexpr (k8) v[e] *= v[e];
        v[e] = s.beta2 * v[e] + s.rest2 * (g[e] * g[e]);
        if constexpr (k8) {
            // (to the last bit but one: with 8-bit moments the arithmetic bounds the step, and correctly rounded roots and
            // quotients are a fifth of it)
            r[e] = __builtin_amdgcn_sqrtf(v[e]);
            p[e] = p[e] * s.keep - s.to * (m[e] * __builtin_amdgcn_rcpf(r[e] * s.root + s.eps));
        } else {
            p[e] = p[e] * s.keep - s.to * (m[e] / (sqrtf(v[e]) * s.root + s.eps));
        }
    }
    store_piece<P, kEach, kStream>(T.p, i, p, left);
    if (kCopy && copy) {
        if (s.copy_dtype == NTFP8_BF16) store_piece<NTFP8_BF16, kEach, kStream>(copy, i, p, left);
        else if (s.copy_dtype == NTFP8_F16) store_piece<NTFP8_F16, kEach, kStream>(copy, i, p, left);
        else store_piece<NTFP8_F32, kEach, kStream>(copy, i, p, left);
    }
    if constexpr (k8) {
        uint32_t mt = 0, rt = 0;
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            mt = max(mt, __float_as_uint(m[e]) & 0x7fffffffu);   // (NaN lies above all others)
            rt = max(rt, __float_as_uint(r[e]) & 0x7fffffffu);
        }
        mt = wave_most(mt);
        rt = wave_most(rt);
        uint32_t mbad = 0, rbad = 0;   // 0x7f in the byte of an element that is not finite, NaN whatever its sign
        if (max(mt, rt) >= kInfBits) {   // uniform: a block with such an element in it, of which only the others count
            mt = rt = 0;
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const uint32_t mb = __float_as_uint(m[e]) & 0x7fffffffu, rb = __float_as_uint(r[e]) & 0x7fffffffu;
                if (mb >= kInfBits) mbad |= 0x7fu << (8 * e), m[e] = 0.0f;   // (whose code keeps to its byte)
                else mt = max(mt, mb);
                if (rb >= kInfBits) rbad |= 0x7fu << (8 * e), r[e] = 0.0f;
                else rt = max(rt, rb);
            }
            mt = wave_most(mt);
            rt = wave_most(rt);
        }
        const int mk = scale_exponent(mt), rk = scale_exponent(rt);
        const float mf = __uint_as_float((uint32_t)(mk + 127) << 23), rf = __uint_as_float((uint32_t)(rk + 127) << 23);
        uint32_t mw = mbad, rw = rbad;
#pragma unroll
        for (int e = 0; e < kEach; e += 2) {
            const uint32_t d = dither_of(entry.pair + (uint32_t)(i >> 1) + e / 2, s.seed);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t d16 = h ? d >> 16 : d & 0xffffu, bits = __float_as_uint(m[e + h]);
                mw |= (encode(__builtin_fabsf(m[e + h]), mf, d16) | ((bits >> 24) & 0x80u)) << (8 * (e + h));
                rw |= max(encode(r[e + h], rf, d16), min(__float_as_uint(r[e + h]), 1u)) << (8 * (e + h));
            }
        }
        if (left == kEach) {
            reinterpret_cast<Word*>(static_cast<uint8_t*>(T.m) + i)->w = mw;
            reinterpret_cast<Word*>(static_cast<uint8_t*>(T.v) + i)->w = rw;
        } else {
            for (int e = 0; e < left; ++e) {
                static_cast<uint8_t*>(T.m)[i + e] = (uint8_t)(mw >> (8 * e));
                static_cast<uint8_t*>(T.v)[i + e] = (uint8_t)(rw >> (8 * e));
            }
        }
        if ((threadIdx.x & 63) == 0 && left) {
            scale_m[i / kBlock] = mf;
            scale_v[i / kBlock] = rf;
        }
    } else {
        store_piece<NTFP8_F32, kEach, kStream>(T.m, i, m, left);
        store_piece<NTFP8_F32, kEach, kStream>(T.v, i, v, left);
    }
}

__global__ __launch_bounds__(256) void adamw_unpack_kernel(const uint8_t* __restrict__ codes, const float* __restrict__ scale, int64_t n,
                                                           float* __restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
        out[i] = __builtin_amdgcn_cvt_f32_fp8((int)codes[i], 0) / scale[i / kBlock];
}

}  // namespace

namespace {

bool within_reach(const void* p) { return reinterpret_cast<uintptr_t>(p) >> 48 == 0; }

template <int P, int G, bool k8, bool kCopy>
int run(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options& o, hipStream_t st) {
    using S = Step<k8, kCopy>;
    S s = {};
    s.copy_dtype = o.copy_dtype;
    s.grad_scale = o.grad_scale;
    s.beta1 = (float)o.beta1, s.rest1 = (float)(1.0 - o.beta1);
    s.beta2 = (float)o.beta2, s.rest2 = (float)(1.0 - o.beta2);
    s.keep = (float)(1.0 - o.lr * o.weight_decay);
    s.to = (float)(o.lr / (1.0 - pow(o.beta1, (double)o.step)));
    s.root = (float)(1.0 / sqrt(1.0 - pow(o.beta2, (double)o.step)));
    s.eps = (float)o.eps;
    s.seed = o.seed * 0xBB67AE85u;
    int64_t all = 0;
    for (int i = 0; i < count; ++i) all += tensors[i].n;
    const bool stream = all * (2 * size_of(P) + size_of(G) + (k8 ? 4 : 16) + (kCopy ? 2 : 0)) > ((int64_t)256 << 20);
    constexpr int64_t part = (int64_t)kChunk << 20;   // a tensor of more workgroups than a launch should have is split
    int used = 0, blocks = 0;
    auto launch = [&]() {
        if (used == 0) return (int)NTFP8_OK;
        for (int i = used; i < S::kMost; ++i) s.first[i] = 0x7fffffff;
        if (stream) adamw_kernel<P, G, k8, kCopy, true><<<(unsigned)blocks, kThreads, 0, st>>>(s);
        else adamw_kernel<P, G, k8, kCopy, false><<<(unsigned)blocks, kThreads, 0, st>>>(s);
        used = blocks = 0;
        return launch_status();
    };
    constexpr int kState = k8 ? 1 : 4;
    for (int i = 0; i < count; ++i) {
        const ntops_adamw_tensor& t = tensors[i];
        for (int64_t at = 0; at < t.n; at += part) {
            const int64_t n = std::min(part, t.n - at);
            const int more = (int)((n + kChunk - 1) / kChunk);
            if (used == S::kMost || blocks + more > (1 << 23))   // (a launch takes fewer than 2^32 threads)
                if (const int rc = launch(); rc != NTFP8_OK) return rc;
            s.t[used].at.set(0, static_cast<char*>(t.param) + at * size_of(P));
            s.t[used].at.set(1, static_cast<const char*>(t.grad) + at * size_of(G));
            s.t[used].at.set(2, static_cast<char*>(t.exp_avg) + at * kState);
            s.t[used].at.set(3, static_cast<char*>(t.exp_avg_sq) + at * kState);
            s.t[used].n = (int)n;
            s.first[used] = blocks;
            if constexpr (k8) {
                s.t[used].pair = (uint32_t)(at >> 1);
                s.t[used].at.set(4, t.exp_avg_scale + at / kBlock);
                s.t[used].at.set(5, t.exp_avg_sq_scale + at / kBlock);
            }
            if constexpr (kCopy) s.copy.set(used, t.copy ? static_cast<char*>(t.copy) + at * size_of(o.copy_dtype) : nullptr);
            blocks += more;
            ++used;
        }
    }
    return launch();
}

}  // namespace

bool adamw_within_reach(const ntops_adamw_tensor* tensors, int count) {
    for (int i = 0; i < count; ++i) {
        const ntops_adamw_tensor& t = tensors[i];
        for (const void* p : {(const void*)t.param, t.grad, (const void*)t.exp_avg, (const void*)t.exp_avg_sq, (const void*)t.exp_avg_scale, (const void*)t.exp_avg_sq_scale, (const void*)t.copy})
            if (!within_reach(p)) return false;
    }
    return true;
}

int run_adamw(const ntops_adamw_tensor* tensors, int count, const ntops_adamw_options& o, hipStream_t st) {
    bool copies = false;
    for (int i = 0; i < count; ++i) copies = copies || tensors[i].copy;
    return with_dtype(o.param_dtype, [&](auto p) {
        constexpr int P = decltype(p)::value;
        return with_dtype(o.grad_dtype, [&](auto g) {
            constexpr int G = decltype(g)::value;
            if (o.bits == 8) return copies ? run<P, G, true, true>(tensors, count, o, st) : run<P, G, true, false>(tensors, count, o, st);
            return copies ? run<P, G, false, true>(tensors, count, o, st) : run<P, G, false, false>(tensors, count, o, st);
        });
    });
}

int run_adamw_unpack(const void* codes, const float* scale, int64_t n, float* out, hipStream_t st) {
    adamw_unpack_kernel<<<(unsigned)std::min<int64_t>((n + 255) / 256, 1 << 16), 256, 0, st>>>(static_cast<const uint8_t*>(codes), scale, n, out);
    return launch_status();
}

}  // namespace ntfp8

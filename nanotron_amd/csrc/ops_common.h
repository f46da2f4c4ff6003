// Device helpers shared by the operators of ntops.h: rows of any alignment in 16-byte pieces, sums over a wave.
#pragma once
#include <algorithm>
#include <type_traits>

#include "../../include/ntops.h"
#include "common.h"

namespace ntfp8 {

constexpr int size_of(int dtype) { return dtype == NTFP8_F32 ? 4 : 2; }

typedef float v2f_ops __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf_ops __attribute__((ext_vector_type(2)));
typedef _Float16 v2h_ops __attribute__((ext_vector_type(2)));

// Two fp32 values rounded to nearest even into one word of D (16-bit types)
template <int D>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
    if constexpr (D == NTFP8_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f_ops){a, b}, v2bf_ops));
    else return __builtin_bit_cast(uint32_t, __builtin_convertvector((v2f_ops){a, b}, v2h_ops));
}
template <int D>
__device__ __forceinline__ void unpack_pair(uint32_t w, float& a, float& b) {
    if constexpr (D == NTFP8_BF16) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
    } else {
        a = half_bits_to_float(w & 0xffffu);
        b = half_bits_to_float(w >> 16);
    }
}

template <int D>
__device__ __forceinline__ void store_one(void* p, int64_t i, float v) {
    if constexpr (D == NTFP8_F32) static_cast<float*>(p)[i] = v;
    else static_cast<uint16_t*>(p)[i] = (uint16_t)pack_pair<D>(v, v);
}

// N consecutive elements as words.  Rows may begin on any element: the hardware takes wide accesses of any alignment, and a
// row of odd length costs a second line at its ends instead of an access per element.
template <int D, int N>
struct __attribute__((packed, aligned(D == NTFP8_F32 ? 4 : 2))) Piece {
    static constexpr int kWords = N * size_of(D) / 4;
    uint32_t w[kWords];
};
// the same words as the vector that a non-temporal access takes
template <int D, int N>
struct PieceVector {
    typedef uint32_t type __attribute__((ext_vector_type(Piece<D, N>::kWords), aligned(D == NTFP8_F32 ? 4 : 2)));
};
// kStream: read or written once, not kept in the caches
template <int D, int N, bool kStream = false>
__device__ __forceinline__ Piece<D, N> load_piece(const void* p, int64_t i) {
    const char* const at = static_cast<const char*>(p) + i * size_of(D);
    if constexpr (kStream) return __builtin_bit_cast(Piece<D, N>, __builtin_nontemporal_load(reinterpret_cast<const typename PieceVector<D, N>::type*>(at)));
    else return *reinterpret_cast<const Piece<D, N>*>(at);
}
// the first `count` elements, zeros behind them
template <int D, int N, bool kStream = false>
__device__ __forceinline__ Piece<D, N> load_piece(const void* p, int64_t i, int count) {
    if (count >= N) return load_piece<D, N, kStream>(p, i);
    Piece<D, N> r;
#pragma unroll
    for (int k = 0; k < Piece<D, N>::kWords; ++k) {
        if constexpr (D == NTFP8_F32) {
            r.w[k] = k < count ? static_cast<const uint32_t*>(p)[i + k] : 0u;
        } else {
            const uint32_t lo = 2 * k < count ? static_cast<const uint16_t*>(p)[i + 2 * k] : 0u;
            const uint32_t hi = 2 * k + 1 < count ? static_cast<const uint16_t*>(p)[i + 2 * k + 1] : 0u;
            r.w[k] = lo | (hi << 16);
        }
    }
    return r;
}
template <int D, int N>
__device__ __forceinline__ void unpack(const Piece<D, N>& r, float (&v)[N]) {
    if constexpr (D == NTFP8_F32) {
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] = __uint_as_float(r.w[k]);
    } else {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) unpack_pair<D>(r.w[k], v[2 * k], v[2 * k + 1]);
    }
}
template <int D, int N, bool kStream = false>
__device__ __forceinline__ void store_piece(void* p, int64_t i, const float (&v)[N], int count = N) {
    if (count >= N) {
        Piece<D, N> r;
        if constexpr (D == NTFP8_F32) {
#pragma unroll
            for (int k = 0; k < N; ++k) r.w[k] = __float_as_uint(v[k]);
        } else {
#pragma unroll
            for (int k = 0; k < N / 2; ++k) r.w[k] = pack_pair<D>(v[2 * k], v[2 * k + 1]);
        }
        char* const at = static_cast<char*>(p) + i * size_of(D);
        if constexpr (kStream) __builtin_nontemporal_store(__builtin_bit_cast(typename PieceVector<D, N>::type, r), reinterpret_cast<typename PieceVector<D, N>::type*>(at));
        else *reinterpret_cast<Piece<D, N>*>(at) = r;
    } else {
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (k < count) store_one<D>(p, i + k, v[k]);
    }
}

// four bytes at any address
struct __attribute__((packed, aligned(1))) Word {
    uint32_t w;
};

// the value of another lane: `kCtrl` as V_MOV_DPP takes it (0x120 + n: n lanes to the right, turning inside rows of 16)
template <int kCtrl>
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, kCtrl, 0xf, 0xf, true);
}
// folds the words of the 64 lanes with f, the result in every lane: inside rows of 16 lanes, then over rows and halves
template <typename F>
__device__ __forceinline__ uint32_t wave_fold(uint32_t v, F&& f) {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    v = f(v, turned<0x128>(v));
    v = f(v, turned<0x124>(v));
    v = f(v, turned<0x122>(v));
    v = f(v, turned<0x121>(v));
    v2u r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(r.x, r.y);
    r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(r.x, r.y);
}
__device__ __forceinline__ float wave_sum(float v) {
    return __uint_as_float(wave_fold(__float_as_uint(v), [](uint32_t a, uint32_t b) { return __float_as_uint(__uint_as_float(a) + __uint_as_float(b)); }));
}
__device__ __forceinline__ uint32_t wave_most(uint32_t v) {
    return wave_fold(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// calls f with an integral constant for the type code
template <typename F>
int with_dtype(int dtype, F&& f) {
    switch (dtype) {
        case NTFP8_F32: return f(std::integral_constant<int, NTFP8_F32>{});
        case NTFP8_F16: return f(std::integral_constant<int, NTFP8_F16>{});
        default: return f(std::integral_constant<int, NTFP8_BF16>{});
    }
}
inline int launch_status() { return hipGetLastError() == hipSuccess ? NTFP8_OK : NTFP8_ERR_LAUNCH; }

}  // namespace ntfp8

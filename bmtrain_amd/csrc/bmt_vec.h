// Device-side helpers of the kernels that take fp32, fp16 and bf16 alike: 16-byte vectors at any element alignment,
// conversion to and from fp32, and the reductions they share.
#pragma once
#include "bmt_device.h"
#include "bmt_host.h"
#include <cstdio>

namespace bmt {

enum : int32_t { kFp32 = 0, kFp16 = 1, kBf16 = 2 };   // type codes of the C entries

struct Single {};                                      // the fp32 tag beside Half and BFloat16

// 16- / 8- / 4-byte accesses whose address is a multiple of the element size only.  gfx950 takes them in one
// instruction; an access off its natural grid touches one more 128-byte line per wave.
typedef u32x4 u32x4_any2 __attribute__((aligned(2)));
typedef u32x2 u32x2_any2 __attribute__((aligned(2)));
typedef u32x4 u32x4_any4 __attribute__((aligned(4)));

// Bits: storage of one element; kVec: elements of a 16-byte vector.
template <typename T>
struct Elem {                                          // Half, BFloat16
    typedef uint16_t Bits;
    typedef u32x4_any2 Vec;
    static constexpr int kVec = 8;
    static __device__ __forceinline__ float get(Bits b) { return T::to_f32(b); }
    static __device__ __forceinline__ Bits put(float f) { return T::from_f32(f); }
    static __device__ __forceinline__ void unpack(const u32x4 &w, float *x) {
#pragma unroll
        for (int k = 0; k < 4; k++) x[2 * k] = lo_f32<T>(w[k]), x[2 * k + 1] = hi_f32<T>(w[k]);
    }
    static __device__ __forceinline__ u32x4 pack(const float *x) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = pack2<T>(x[2 * k], x[2 * k + 1]);
        return w;
    }
};
template <>
struct Elem<Single> {
    typedef uint32_t Bits;
    typedef u32x4_any4 Vec;
    static constexpr int kVec = 4;
    static __device__ __forceinline__ float get(Bits b) { return __builtin_bit_cast(float, b); }
    static __device__ __forceinline__ Bits put(float f) { return __builtin_bit_cast(uint32_t, f); }
    static __device__ __forceinline__ void unpack(const u32x4 &w, float *x) {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = get(w[k]);       // by value: a bit cast of w[k] itself reads element 0
    }
    static __device__ __forceinline__ u32x4 pack(const float *x) {
        u32x4 w;
#pragma unroll
        for (int k = 0; k < 4; k++) w[k] = put(x[k]);
        return w;
    }
};

// Elements in front of the first 16-byte boundary at or behind p, at most n.
template <typename T>
__device__ __forceinline__ int head_elements(const typename Elem<T>::Bits *p, int n) {
    const int h = (int)((16u - ((uint32_t)(uintptr_t)p & 15u)) & 15u) / (int)sizeof(typename Elem<T>::Bits);
    return h < n ? h : n;
}

// Four consecutive elements as floats (`count` of them exist; the others read as 0).
template <typename T>
__device__ __forceinline__ void load4(const typename Elem<T>::Bits *p, int count, float *x) {
    if (count >= 4) {
        if (sizeof(typename Elem<T>::Bits) == 2) {
            const u32x2 w = *(const u32x2_any2 *)p;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                x[2 * k] = Elem<T>::get((typename Elem<T>::Bits)(w[k] & 0xFFFFu));
                x[2 * k + 1] = Elem<T>::get((typename Elem<T>::Bits)(w[k] >> 16));
            }
        } else {
            const u32x4 w = *(const u32x4_any4 *)p;
#pragma unroll
            for (int k = 0; k < 4; k++) x[k] = Elem<T>::get((typename Elem<T>::Bits)w[k]);
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = k < count ? Elem<T>::get(p[k]) : 0.f;
    }
}
template <typename T>
__device__ __forceinline__ void store4(typename Elem<T>::Bits *p, int count, const float *x) {
    if (count >= 4) {
        if (sizeof(typename Elem<T>::Bits) == 2) {
            u32x2 w;
#pragma unroll
            for (int k = 0; k < 2; k++)
                w[k] = (uint32_t)Elem<T>::put(x[2 * k]) | ((uint32_t)Elem<T>::put(x[2 * k + 1]) << 16);
            *(u32x2_any2 *)p = w;
        } else {
            u32x4 w;
#pragma unroll
            for (int k = 0; k < 4; k++) w[k] = (uint32_t)Elem<T>::put(x[k]);
            *(u32x4_any4 *)p = w;
        }
    } else {
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (k < count) p[k] = Elem<T>::put(x[k]);
    }
}
// Four consecutive elements as raw bits, to be converted later: loads of several arrays can be on their way before the
// first value is needed.  load: all four exist (PAST: read past the caches); load_some: the first `count` do, the others read as 0.
template <typename T>
struct Raw4 {
    uint32_t w[sizeof(typename Elem<T>::Bits)];        // 2 dwords of 16-bit elements, 4 of 32-bit ones
    template <bool PAST = false>
    __device__ __forceinline__ void load(const typename Elem<T>::Bits *p) {
        if (sizeof(typename Elem<T>::Bits) == 2) {
            const u32x2_any2 *at = (const u32x2_any2 *)p;
            const u32x2 v = PAST ? __builtin_nontemporal_load(at) : *at;
            w[0] = v[0], w[1] = v[1];
        } else {
            const u32x4_any4 *at = (const u32x4_any4 *)p;
            const u32x4 v = PAST ? __builtin_nontemporal_load(at) : *at;
#pragma unroll
            for (int k = 0; k < (int)sizeof(typename Elem<T>::Bits); k++) w[k] = v[k];
        }
    }
    __device__ __forceinline__ void load_some(const typename Elem<T>::Bits *p, int count) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const typename Elem<T>::Bits b = k < count ? p[k] : 0;
            if (sizeof(b) == 4) w[k] = b;
            else w[k / 2] = k % 2 ? (w[k / 2] & 0xFFFFu) | ((uint32_t)b << 16) : (uint32_t)b;
        }
    }
    __device__ __forceinline__ float get(int k) const {
        if (sizeof(typename Elem<T>::Bits) == 4) return Elem<T>::get((typename Elem<T>::Bits)w[k]);
        return Elem<T>::get((typename Elem<T>::Bits)(w[k / 2] >> (16 * (k % 2))));
    }
};

// Four mask bytes, one to each byte of a dword (absent mask: all set); bytes behind `count` read as unset.
typedef uint32_t u32_any1 __attribute__((aligned(1)));
__device__ __forceinline__ uint32_t load_mask4(const uint8_t *p, int count) {
    if (!p) return count >= 4 ? 0x01010101u : 0x01010101u >> (8 * (4 - count));
    if (count >= 4) return *(const u32_any1 *)p;
    uint32_t w = 0;
#pragma unroll
    for (int k = 0; k < 4; k++)
        if (k < count) w |= (uint32_t)p[k] << (8 * k);
    return w;
}
__device__ __forceinline__ bool mask_set(uint32_t w, int k) { return (w >> (8 * k) & 0xFFu) != 0; }
__device__ __forceinline__ int mask_count(uint32_t w) {
    int n = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) n += mask_set(w, k) ? 1 : 0;
    return n;
}

// Sums of eight values over a wave: lane 8 j ends with the sum of v[j].  Every step halves the values a lane carries
// (it hands one half to its partner and takes the other), so eight values cost ten exchanges instead of 48.
template <typename V>
__device__ __forceinline__ V wave_sum8(V *v) {
    const int lane = threadIdx.x % kWave;
#pragma unroll
    for (int half = 4; half > 0; half >>= 1) {
        const bool upper = (lane & (8 * half)) != 0;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j >= half) break;
            const V keep = upper ? v[j + half] : v[j], give = upper ? v[j] : v[j + half];
            v[j] = keep + __shfl_xor(give, 8 * half, kWave);
        }
    }
    V sum = v[0];
#pragma unroll
    for (int off = 4; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
    return sum;
}

// Workgroups are dealt to the eight XCDs in turn.  This numbering gives every XCD runs of RUN consecutive units of work
// instead (the last incomplete round of 8 * RUN units keeps the plain order), so that what one XCD's L2 and its share of
// the memory channels see is consecutive.
template <uint32_t RUN>
__device__ __forceinline__ uint32_t xcd_run(uint32_t id, uint32_t count) {
    constexpr uint32_t kXcds = 8, kRound = kXcds * RUN;
    const uint32_t base = id / kRound * kRound, k = id - base;
    return base + kRound <= count ? base + (k % kXcds) * RUN + k / kXcds : id;
}

// Sum over groups of `lanes` neighbouring lanes (a power of two up to 64); every lane ends with its group's sum.
template <typename V>
__device__ __forceinline__ V lanes_sum(V v, int lanes) {
    for (int off = lanes >> 1; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// Host side: whether a launch of `grid` workgroups of `threads` is within the 2^32 threads that a dispatch can count.
inline bool launch_fits(int64_t grid, int64_t threads) { return grid * threads < ((int64_t)1 << 32); }

// Host side: refuses a call of C entry `who` because of `why`.
inline int refuse(const char *who, const char *why) {
    char text[200];
    snprintf(text, sizeof(text), "%s: %s", who, why);
    return fail(-1, text);
}

}  // namespace bmt

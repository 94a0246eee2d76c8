// One row of logits (float32, bf16 or f16, any length) worked on by one workgroup: how the operators that filter,
// rank and distil a row read it.  Device code for gfx950.
#pragma once
#include "icrl_common.h"

namespace icrl {

typedef unsigned long long u64;

template <typename T>
struct Elem;   // how many fit 16 bytes, and their value in float32 (exact for all three types)
template <>
struct Elem<float> {
    static constexpr int VEC = 4;
    using Raw = unsigned;
    static __device__ __forceinline__ float value(Raw r) { return __uint_as_float(r); }
};
template <>
struct Elem<__bf16> {
    static constexpr int VEC = 8;
    using Raw = unsigned short;
    static __device__ __forceinline__ float value(Raw r) { return __uint_as_float((unsigned)r << 16); }
};
template <>
struct Elem<_Float16> {
    static constexpr int VEC = 8;
    using Raw = unsigned short;
    static __device__ __forceinline__ float value(Raw r) { return (float)__builtin_bit_cast(_Float16, r); }
};

// Where a row's entries are between the passes over it.  PLACE > 0: in registers, at most PLACE vectors of 16 bytes a
// thread (every pass is unrolled, so passes have to be short).  IN_MEMORY: every pass reads the row again, from the caches
// where it fits them.
constexpr int IN_MEMORY = 0;

// A row is cut into one contiguous piece per wave, a multiple of 64 x 16 bytes, and a piece into wave-wide vectors of
// 16 bytes a lane: reads are 1 KB of consecutive bytes, and (wave, vector, lane, element) is the order of the indices,
// which the draw and the ranking of ties need.  Rows need no alignment beyond their element's: gfx950 reads 16 bytes
// from any address.  Places past the row's end hold -inf, or (CANON) a NaN of their own that orders below every entry,
// the canonical NaN included; CANON also turns every NaN into one and -0 into +0, so that equal entries have equal keys.
template <typename T, int NT, int PLACE, bool CANON>
struct Row {
    using Type = T;
    static constexpr int VEC = Elem<T>::VEC;
    using Raw = typename Elem<T>::Raw;
    static constexpr Raw kNan = sizeof(T) == 4 ? (Raw)0xFFC00000u : (__is_same(T, __bf16) ? (Raw)0xFFC0u : (Raw)0xFE00u);
    static constexpr Raw kMinusInf = sizeof(T) == 4 ? (Raw)0xFF800000u : (__is_same(T, __bf16) ? (Raw)0xFF80u : (Raw)0xFC00u);
    static constexpr Raw kFill = CANON ? (Raw)~0u : kMinusInf;
    struct alignas(16) Pack { Raw e[VEC]; };
    typedef unsigned Words __attribute__((ext_vector_type(4), aligned(2), may_alias));   // one 16-byte access
    const T* src;
    int V, vectors;      // vectors: how many per thread
    int first;           // index of the thread's first entry
    int wave_first;      // of the wave's
    Pack end;            // the entries of the row's last vector, if it is not whole
    Pack keep[PLACE > 0 ? PLACE : 1];

    // Vector i, 16 bytes where the row has them.  Rows in memory: the one vector that the row ends inside of is read when
    // the row is opened, entry by entry, and handed out by the thread that owns it (nothing of that is left in the passes).
    __device__ __forceinline__ Words read(int i) const {
        const int at = first + i * 64 * VEC;
        if constexpr (PLACE == IN_MEMORY) {
            if (wave_first + (i + 1) * 64 * VEC <= V) return *reinterpret_cast<const Words*>(src + at);
            Words w = at < V ? __builtin_bit_cast(Words, end) : __builtin_bit_cast(Words, fill());
            if (at + VEC <= V) w = *reinterpret_cast<const Words*>(src + at);
            return w;
        } else {
            if (at + VEC <= V) return *reinterpret_cast<const Words*>(src + at);
            Pack p = fill();
            read_end(p, at);
            return __builtin_bit_cast(Words, p);
        }
    }
    __device__ __forceinline__ void read_end(Pack& p, int at) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
            if (at + j < V) __builtin_memcpy(&p.e[j], src + at + j, sizeof(Raw));
    }
    static __device__ __forceinline__ Pack fill() {
        Pack p;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p.e[j] = kFill;
        return p;
    }
    __device__ __forceinline__ Pack canonical(Words w, int i) const { return canonical_at(w, first + i * 64 * VEC); }
    __device__ __forceinline__ Pack canonical_at(Words w, int at) const {
        Pack p = __builtin_bit_cast(Pack, w);
        if (CANON) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float x = Elem<T>::value(p.e[j]);
                p.e[j] = x != x && at + j < V ? kNan : p.e[j];
            }
        }
        return p;
    }
    __device__ __forceinline__ Pack fetch(int i) const {
        return canonical(read(i), i);
    }
    // the vector of any thread: 16 bytes from entry `at` on
    __device__ __forceinline__ Pack fetch_at(int at) const {
        Words w;
        if (at + VEC <= V) {
            w = *reinterpret_cast<const Words*>(src + at);
        } else {
            Pack p = fill();
            read_end(p, at);
            w = __builtin_bit_cast(Words, p);
        }
        return canonical_at(w, at);
    }

    __device__ __forceinline__ void open(const T* row, int count) {
        src = row;
        V = count;
        vectors = (count + NT * VEC - 1) / (NT * VEC);
        first = ((int)(threadIdx.x >> 6) * vectors * 64 + (int)(threadIdx.x & 63)) * VEC;
        if constexpr (PLACE == IN_MEMORY) {
            wave_first = __builtin_amdgcn_readfirstlane(first);
            end = fill();
            const int whole = count / VEC * VEC;
            if (first <= whole && (whole - first) % (64 * VEC) == 0 && whole - first < vectors * 64 * VEC)   // one thread, or none
                read_end(end, whole);
        }
        if constexpr (PLACE > 0) {
#pragma unroll
            for (int i = 0; i < PLACE; ++i)
                if (i < vectors) keep[i] = canonical(read(i), i);
        }
    }

    // A vector as a pass sees it.  16-bit entries are widened anew in every pass: the compiler, which would otherwise widen
    // the row once for all of them and then has twice its registers to keep, is told that they may have changed.
    static __device__ __forceinline__ Pack pass(const Pack& p) {
        Words w = __builtin_bit_cast(Words, p);
        if (sizeof(T) == 2) asm("" : "+v"(w));
        return __builtin_bit_cast(Pack, w);
    }
    // entry i < V, from memory
    __device__ __forceinline__ float entry(int i) const {
        const float x = Elem<T>::value(__builtin_bit_cast(Raw, src[i]));
        return CANON && x != x ? Elem<T>::value(kNan) : x;
    }
    // f(vector, index of its first entry) for each of the thread's vectors
    template <typename F>
    __device__ __forceinline__ void each_pack(F&& f) const {
        if constexpr (PLACE > 0) {
#pragma unroll
            for (int i = 0; i < PLACE; ++i)
                if (i < vectors) f(pass(keep[i]), first + i * 64 * VEC);
        } else {
            constexpr int AHEAD = 4;   // reads in flight: a queue in registers
            Words p[AHEAD];            // (as words: packs of 16-bit entries are taken apart on arrival, which waits for them)
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (q < vectors) p[q] = read(q);
#pragma unroll 1
            for (int i = 0; i < vectors; ++i) {
                const Words now = p[0];
#pragma unroll
                for (int q = 0; q + 1 < AHEAD; ++q) p[q] = p[q + 1];
                if (i + AHEAD < vectors) p[AHEAD - 1] = read(i + AHEAD);
                f(canonical(now, i), first + i * 64 * VEC);
            }
        }
    }
    // The same for an f of few instructions, which leaves a pass waiting for its reads: four vectors are always on their
    // way, at the price of f's code five times.  (The queue above moves what it has just asked for and so waits for it one
    // vector later; gradient of 512 x 131072 bf16 50.4 against 45.7 us.)  Places past the end are handed out in the row's
    // last vector only.
    template <typename F>
    __device__ __forceinline__ void sweep(F&& f) const {
        if constexpr (PLACE > 0) {
            each_pack(f);
        } else {
            constexpr int AHEAD = 4, STEP = 64 * VEC;
            const int left = V - wave_first, live = min(vectors, left > 0 ? (left + STEP - 1) / STEP : 0);
            const int whole = left > 0 ? min(vectors, left / STEP) : 0;
            int i = 0;
            if (whole >= AHEAD) {
                Words p[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) p[q] = *reinterpret_cast<const Words*>(src + first + q * STEP);
#pragma unroll 1
                for (; i + AHEAD <= whole; i += AHEAD) {
#pragma unroll
                    for (int q = 0; q < AHEAD; ++q) {
                        const Words now = p[q];
                        p[q] = *reinterpret_cast<const Words*>(src + first + min(i + AHEAD + q, whole - 1) * STEP);
                        f(canonical(now, i + q), first + (i + q) * STEP);
                    }
                }
            }
            Words p[AHEAD];   // at most three whole ones and the last
#pragma unroll
            for (int q = 0; q < AHEAD; ++q)
                if (i + q < live) p[q] = read(i + q);
#pragma unroll 1
            for (; i < live; ++i) {
                const Words now = p[0];
#pragma unroll
                for (int q = 0; q + 1 < AHEAD; ++q) p[q] = p[q + 1];
                f(canonical(now, i), first + i * STEP);
            }
        }
    }
    // f(value, index) for every place of a vector, or of all of them (places past the end included)
    template <typename F>
    __device__ __forceinline__ void vector(const Pack& p, int at, F&& f) const {
#pragma unroll
        for (int j = 0; j < VEC; ++j) f(Elem<T>::value(p.e[j]), at + j);
    }
    template <typename F>
    __device__ __forceinline__ void each(F&& f) const {
        each_pack([&](const Pack& p, int at) { vector(p, at, f); });
    }
    template <typename F>
    __device__ __forceinline__ void sweep_each(F&& f) const {
        sweep([&](const Pack& p, int at) { vector(p, at, f); });
    }
};

// Unsigned keys in the order of the values.  -inf: 0x007FFFFF; the canonical NaN below it, places past the end below that.
constexpr unsigned kKeyNan = 0x003FFFFFu, kKeyMinusInf = 0x007FFFFFu, kKeyFinite = 0x00800000u, kKeyPlusInf = 0xFF800000u;
__device__ __forceinline__ unsigned order_key(float x) {
    int b = __float_as_int(x);
    b = b == (int)0x80000000 ? 0 : b;   // -0 and +0 are equal
    return (unsigned)(b ^ ((b >> 31) | (int)0x80000000));
}

// 2^r in float64 for |r| <= 1/2, by the Taylor series of e^(r ln 2): nine terms leave 0.3466^10 / 10! = 7e-12 of the
// result.  (The library's exp2 spends several times the instructions on bits that no sum here can show.)
__device__ __forceinline__ double exp2_fraction(double r) {
    constexpr double L = 0.69314718055994530942, L2 = L * L, L3 = L2 * L, L4 = L2 * L2, L5 = L4 * L;
    double p = L4 * L5 / 362880.0;
    p = fma(p, r, L4 * L4 / 40320.0);
    p = fma(p, r, L4 * L3 / 5040.0);
    p = fma(p, r, L3 * L3 / 720.0);
    p = fma(p, r, L5 / 120.0);
    p = fma(p, r, L4 / 24.0);
    p = fma(p, r, L3 / 6.0);
    p = fma(p, r, L2 / 2.0);
    p = fma(p, r, L);
    return fma(p, r, 1.0);
}
// 2^t 2^scale where the result is a normal number, |t| < 2^30: the nearest integer is read off the sum with 1.5 2^52 and
// added to the exponent's bits (rounding, conversion and ldexp instructions run at a quarter of the rate)
__device__ __forceinline__ double exp2_normal(double t, int scale) {
    const double shifted = t + 0x1.8p52, r = t - (shifted - 0x1.8p52);
    const int n = (int)__double_as_longlong(shifted);
    return __longlong_as_double(__double_as_longlong(exp2_fraction(r)) + ((long long)(n + scale) << 52));
}

__device__ __forceinline__ u64 wave_sum_u64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

}  // namespace icrl

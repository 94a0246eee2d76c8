// Distillation of a policy from the k largest logits that a teacher kept for each position: loss and gradient.
//
// With z = x / T, p = softmax(z) over the row's V words and q_j the teacher's probability of listed word j, the words
// outside the list count as one more word whose teacher probability q_r is what the list leaves over:
//   loss = sum_j q_j (log q_j - log p_j) + q_r (log q_r - log p_r),   p_r = sum of p outside the list,
//   dloss/dx_i = (p_i W - q_i) / T for listed words, p_i (W - q_r / p_r) / T for the others,   W = sum_j q_j + q_r.
// Without the teacher's log-normaliser q is the softmax over the list and q_r = 0.
//
// Bound by memory: the forward pass reads the row once, the gradient writes it once; rows up to 32768 (65536) entries
// of 4 (2) bytes stay in registers in between, longer ones are read again.  Measured: loss and gradient of 9728 x 10000
// float32, k = 64, a fifth of the rows idle: 176 us for 700 MB, 4.0 TB/s (a plain copy reaches 4.8); 512 x 131072 bf16,
// k = 128, in two calls, 5% idle: 103 us for 383 MB (the rows' sums take one CU each about as long as their reads).
// p_r is summed directly over the words outside (a bitmap of the list in LDS tells them apart): as 1 - sum it would lose
// all its digits where the policy is sure.  Row sums are float32 per
// thread (at most a few hundred terms each) and float64 from there on; the handful of numbers per row and the list's
// terms are float64 throughout, since the loss is a difference of nearly equal ones.
#include <math.h>

#include "vocab_row.h"

namespace {
using namespace icrl;

constexpr int MAX_K = 1024, MAX_V = 1 << 18;   // the bitmap of a row of 2^18 words is 32 KB of LDS
constexpr double LOG2E = 1.4426950408889634074;

// e^x in float64 to 7e-12 of itself (any x: infinite above 1e4, zero below -1e4, NaN for NaN)
__device__ __forceinline__ double exp_of(double x) {
    const double t = fmin(fmax(x, -1e4), 1e4) * LOG2E, n = rint(t);
    return x != x ? x : ldexp(exp2_fraction(t - n), (int)n);
}

template <typename T>
__device__ __forceinline__ T from_float(float x) { return (T)x; }   // round to nearest even

template <int NT, int COUNT>
__device__ __forceinline__ void block_sums(double (&v)[COUNT], double* lds) {
#pragma unroll
    for (int c = 0; c < COUNT; ++c) v[c] = wave_sum_d(v[c]);
    __syncthreads();
    if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int c = 0; c < COUNT; ++c) lds[(threadIdx.x >> 6) * COUNT + c] = v[c];
    __syncthreads();
#pragma unroll
    for (int c = 0; c < COUNT; ++c) {
        v[c] = 0.0;
        for (int w = 0; w < NT / 64; ++w) v[c] += lds[w * COUNT + c];
    }
}

template <typename T, int VEC>
struct alignas(16) Out { T e[VEC]; };

// Writes f(value) over the row (same vectors as the row's reads; the places need the element's alignment only).
template <typename T, int NT, int NV, typename F>
__device__ __forceinline__ void write_row(const Row<T, NT, NV, false>& row, T* dst, F&& f) {
    constexpr int VEC = Elem<T>::VEC;
    row.sweep([&](const typename Row<T, NT, NV, false>::Pack& p, int at) {
        Out<T, VEC> o;
#pragma unroll
        for (int j = 0; j < VEC; ++j) o.e[j] = from_float<T>(f(Elem<T>::value(p.e[j])));
        if (at + VEC <= row.V) {
            __builtin_nontemporal_store(__builtin_bit_cast(typename Row<T, NT, NV, false>::Words, o),
                                        reinterpret_cast<typename Row<T, NT, NV, false>::Words*>(dst + at));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j)
                if (at + j < row.V) dst[at + j] = o.e[j];
        }
    });
}

// A whole row of one value (rows of weight zero, rows without a defined gradient).
template <typename T, int NT>
__device__ __forceinline__ void fill_row(T* dst, int V, float x) {
    constexpr int VEC = Elem<T>::VEC;
    using Words = typename Row<T, NT, IN_MEMORY, false>::Words;
    Out<T, VEC> o;
#pragma unroll
    for (int j = 0; j < VEC; ++j) o.e[j] = from_float<T>(x);
    for (int at = threadIdx.x * VEC; at < V; at += NT * VEC) {
        if (at + VEC <= V) __builtin_nontemporal_store(__builtin_bit_cast(Words, o), reinterpret_cast<Words*>(dst + at));
        else
            for (int j = at; j < V; ++j) dst[j] = o.e[0];
    }
}

// stats of a row: log-normaliser of z, the teacher's log-normaliser, W, and W - q_r / p_r.  Float64: a log-normaliser
// of some hundreds rounded to float32 would be off by more than float32 rounding in every probability made from it.
__device__ __forceinline__ void put_stats(double* stats, int r, double a, double b, double c, double d) {
    double* at = stats + 4 * (int64_t)r;
    at[0] = a; at[1] = b; at[2] = c; at[3] = d;
}

template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT, 4) void distill_kernel(const T* logits, int64_t ld, int V,
                                                     const float* __restrict__ t_values, const int64_t* __restrict__ t_indices,
                                                     int k, const float* __restrict__ t_lse, double per_t,
                                                     const float* __restrict__ row_weight, float* __restrict__ row_loss,
                                                     double* __restrict__ stats, T* dlogits, int64_t ldd) {
    extern __shared__ unsigned bits[];   // (V + 31) / 32 words: which words are listed
    __shared__ double sums[NT / 64 * 4];
    __shared__ float red[NT / 64][2];
    __shared__ int bad;
    const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T* src = logits + (int64_t)r * ld;
    const float* tv = t_values + (int64_t)r * k;
    const int64_t* ti = t_indices + (int64_t)r * k;
    T* dst = dlogits ? dlogits + (int64_t)r * ldd : nullptr;
    const float weight = row_weight ? row_weight[r] : 1.f;
    if (weight == 0.f) {   // an idle row: nothing of it is read
        if (tid == 0) {
            row_loss[r] = 0.f;
            if (stats) put_stats(stats, r, 0.0, 0.0, 0.0, 0.0);
        }
        if (dst) fill_row<T, NT>(dst, V, 0.f);
        return;
    }
    // this thread's entries of the list (their logits gathered while the row is on its way)
    constexpr int MINE = MAX_K / NT;
    int index[MINE];   // -1: none, or absent; -2: past the vocabulary
    float value[MINE], logit[MINE];
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
        const int j = tid + q * NT;
        const int64_t i = j < k ? ti[j] : -1;
        index[q] = i < 0 ? -1 : i < V ? (int)i : -2;
        value[q] = index[q] >= 0 ? tv[j] : -INFINITY;
    }
    Row<T, NT, NV, false> row;
    row.open(src, V);
#pragma unroll
    for (int q = 0; q < MINE; ++q)
        logit[q] = index[q] >= 0 ? Elem<T>::value(__builtin_bit_cast(typename Elem<T>::Raw, src[index[q]])) : 0.f;
    const int words = (V + 31) / 32;
    for (int w = tid; w < words; w += NT) bits[w] = 0;
    if (tid == 0) bad = 0;
    __syncthreads();
    // a negative index is an absent entry; one past the vocabulary, or the same one twice, is an error that makes the
    // row's results NaN
    float t_top = -INFINITY;
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
        if (index[q] == -2) bad = 1;
        if (index[q] >= 0) {
            if (atomicOr(&bits[index[q] >> 5], 1u << (index[q] & 31)) >> (index[q] & 31) & 1u) bad = 1;
            t_top = fmaxf(t_top, value[q]);
        }
    }
    // the sum outside the list.  A row in registers: its largest entry first.  A row that is read again by every pass: in
    // one pass, every thread's sum relative to its own largest entry so far
    constexpr bool ONLINE = NV == IN_MEMORY;
    const float c = (float)(per_t * LOG2E);
    float best = -INFINITY, part = 0.f;
    auto outside_sum = [&](const auto& p, int at, float top) {   // a vector's entries share a word of the bitmap
        const unsigned listed = at < V ? bits[at >> 5] >> (at & 31) : 0u;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < Elem<T>::VEC; ++j) {
            const float e = __builtin_amdgcn_exp2f((Elem<T>::value(p.e[j]) - top) * c);
            s += listed >> j & 1u ? 0.f : e;
        }
        return s;
    };
    if constexpr (ONLINE) {
        __syncthreads();   // the bitmap is whole
        row.sweep([&](const auto& p, int at) {
            float top = best;
#pragma unroll
            for (int j = 0; j < Elem<T>::VEC; ++j) top = fmaxf(top, Elem<T>::value(p.e[j]));
            if (top == -INFINITY) {   // nothing yet but -inf, or NaN, which fmaxf passes over
#pragma unroll
                for (int j = 0; j < Elem<T>::VEC; ++j)
                    if (Elem<T>::value(p.e[j]) != Elem<T>::value(p.e[j])) part = NAN;
                return;
            }
            part = part * (best == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((best - top) * c)) + outside_sum(p, at, top);
            best = top;
        });
    } else {
        row.each([&](float x, int) { best = fmaxf(best, x); });
    }
    float own = best;
    t_top = wave_max(t_top);
    best = wave_max(best);
    if (lane == 0) { red[wave][0] = t_top; red[wave][1] = best; }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) { t_top = fmaxf(t_top, red[w][0]); best = fmaxf(best, red[w][1]); }
    if (bad) {
        if (tid == 0) {
            row_loss[r] = NAN;
            if (stats) put_stats(stats, r, NAN, NAN, NAN, NAN);
        }
        if (dst) fill_row<T, NT>(dst, V, NAN);
        return;
    }
    if constexpr (ONLINE) {
        if (own > -INFINITY) part *= __builtin_amdgcn_exp2f((own - best) * c);
    } else {
        row.each_pack([&](const auto& p, int at) { part += outside_sum(p, at, best); });
    }
    // sums over the list: its part of Z, u_j = e^(t_j / T - t_ref), u_j (log u_j - z_j)
    const bool tail = t_lse != nullptr;
    const double t_ref = tail ? (double)t_lse[r] : (double)t_top * per_t;
    double s[4] = {(double)part, 0.0, 0.0, 0.0}, e_listed[MINE], u_listed[MINE];
#pragma unroll
    for (int q = 0; q < MINE; ++q) {
        const double z = ((double)logit[q] - (double)best) * per_t, d = (double)value[q] * per_t - t_ref;
        e_listed[q] = index[q] >= 0 ? exp_of(z) : 0.0;
        u_listed[q] = index[q] >= 0 ? exp_of(d) : 0.0;
        s[1] += e_listed[q];
        s[2] += u_listed[q];
        if (u_listed[q] != 0.0) s[3] += u_listed[q] * (d - z);
    }
    block_sums<NT, 4>(s, sums);
    const double Z = s[0] + s[1], log_z = log(Z), U = s[2];
    double loss, q_scale, W, ratio = 0.0, teacher = t_ref;   // q_j = u_j q_scale
    if (tail) {
        q_scale = 1.0;
        W = U;
        loss = s[3] + U * log_z;
        // Where the policy has no mass outside the list the last word is left out: whether the teacher's is zero there
        // is for its rounding to say, and the term would be 0 or infinite by that.
        const double left = 1.0 - U;
        if (left > 0.0 && s[0] > 0.0) {
            const double p_r = s[0] / Z;
            loss += left * (log(left) - log(p_r));
            W += left;
            ratio = left / p_r;
        }
    } else {
        // no entries, or none with mass: nothing to learn from this row
        const bool any = U != 0.0 && t_top != -INFINITY;
        q_scale = any ? 1.0 / U : 0.0;
        W = any ? 1.0 : 0.0;
        loss = any ? s[3] / U - log(U) + log_z : 0.0;
        teacher = any ? t_ref + log(U) : 0.0;
    }
    if (tid == 0) {
        row_loss[r] = (float)((double)weight * loss);
        if (stats) put_stats(stats, r, (double)best * per_t + log_z, teacher, W, W - ratio);
    }
    if (!dst) return;
    if (W == 0.0) {
        fill_row<T, NT>(dst, V, 0.f);
        return;
    }
    const double g = (double)weight * per_t;
    __syncthreads();   // dlogits may be the logits themselves: every gathered logit is in its thread's hands
    const float outside = (float)(g * (W - ratio) / Z);
    write_row<T, NT, NV>(row, dst, [&](float x) { return outside * __builtin_amdgcn_exp2f((x - best) * c); });
    __syncthreads();   // the row's writes come before those at the listed words
#pragma unroll
    for (int q = 0; q < MINE; ++q)
        if (index[q] >= 0)
            dst[index[q]] = from_float<T>((float)(g * (e_listed[q] / Z * W - u_listed[q] * q_scale)));
}

// The gradient alone, from the forward pass's stats.
template <typename T, int NT, int NV>
__global__ __launch_bounds__(NT) void distill_grad_kernel(const T* logits, int64_t ld, int V,
                                                          const float* __restrict__ t_values,
                                                          const int64_t* __restrict__ t_indices, int k, double per_t,
                                                          const double* __restrict__ stats,
                                                          const float* __restrict__ row_weight, T* dlogits, int64_t ldd) {
    __shared__ float at_listed[MAX_K];
    const int r = blockIdx.x, tid = threadIdx.x;
    const T* src = logits + (int64_t)r * ld;
    const float* tv = t_values + (int64_t)r * k;
    const int64_t* ti = t_indices + (int64_t)r * k;
    T* dst = dlogits + (int64_t)r * ldd;
    const float weight = row_weight ? row_weight[r] : 1.f;
    const double log_z = stats[4 * (int64_t)r], teacher = stats[4 * (int64_t)r + 1], W = stats[4 * (int64_t)r + 2],
                 W_out = stats[4 * (int64_t)r + 3];
    if (weight == 0.f || W == 0.0) {   // W = 0: nothing to learn from this row, or idle in the forward pass
        fill_row<T, NT>(dst, V, 0.f);
        return;
    }
    Row<T, NT, NV, false> row;
    row.open(src, V);
    const double g = (double)weight * per_t;
    for (int j = tid; j < k; j += NT) {
        const int64_t i = ti[j];
        if (i < 0 || i >= V) continue;   // past the vocabulary: the stats are NaN already
        const float x = Elem<T>::value(__builtin_bit_cast(typename Elem<T>::Raw, src[i]));
        const double p = exp_of((double)x * per_t - log_z), q = exp_of((double)tv[j] * per_t - teacher);
        at_listed[j] = (float)(g * (p * W - q));
    }
    __syncthreads();
    // p = 2^((x - base) c), base the x that would have p = 1; its float32 rounding goes into the factor
    const float base = (float)(log_z / per_t), c = (float)(per_t * LOG2E);
    const float outside = (float)(g * W_out * exp((double)base * per_t - log_z));
    write_row<T, NT, NV>(row, dst, [&](float x) { return outside * __builtin_amdgcn_exp2f((x - base) * c); });
    __syncthreads();
    for (int j = tid; j < k; j += NT) {
        const int64_t i = ti[j];
        if (i >= 0 && i < V) dst[i] = from_float<T>(at_listed[j]);
    }
}

#define ICRL_ROW_DISPATCH(T, V, CALL)                                              \
    do {                                                                           \
        constexpr int vec_ = icrl::Elem<T>::VEC;                                   \
        if ((V) <= 256 * 4 * vec_) { CALL(T, 256, 4); }                            \
        else if ((V) <= 512 * 8 * vec_) { CALL(T, 512, 8); }                       \
        else if ((V) <= 1024 * 8 * vec_) { CALL(T, 1024, 8); }                     \
        else { CALL(T, 1024, IN_MEMORY); }                                         \
    } while (0)

int check(const char* who, const void* logits, int64_t ld, int N, int V, const void* tv, const void* ti, int k, double temperature) {
    ICRL_REQUIRE(logits && tv && ti && N > 0 && V > 0, "%s: null pointer or empty shape", who);
    ICRL_REQUIRE(ld >= V, "%s: ld_logits < V", who);
    ICRL_REQUIRE(V <= MAX_V, "%s: vocabulary %d exceeds %d entries", who, V, MAX_V);
    ICRL_REQUIRE(k >= 1 && k <= V && k <= MAX_K, "%s: k must be in [1, min(%d, V)] (got %d)", who, MAX_K, k);
    ICRL_REQUIRE(temperature > 0.0 && isfinite(temperature), "%s: temperature must be positive and finite", who);
    return ICRL_OK;
}

// The gradient's rows are the logits' own places, or share none with them: a row may be written while others are read.
bool same_or_apart(const void* logits, int64_t ld, const void* dlogits, int64_t ldd, int N, int V, int64_t size) {
    const intptr_t a = reinterpret_cast<intptr_t>(logits), b = reinterpret_cast<intptr_t>(dlogits);
    if (a == b && (ld == ldd || N == 1)) return true;
    if (a + ((N - 1) * ld + V) * size <= b || b + ((N - 1) * ldd + V) * size <= a) return true;
    if (ld != ldd || N == 1) return false;
    const int64_t row = ld * size, shift = (((b - a) % row) + row) % row;   // side by side in the rows of one matrix
    return shift >= V * size && row - shift >= V * size;
}
#define ICRL_REQUIRE_PLACES(who)                                                                                    \
    ICRL_REQUIRE(!dlogits || dtype < ICRL_F32 || dtype > ICRL_F16 ||                                                \
                     same_or_apart(logits, ld_logits, dlogits, ld_dlogits, N, V, dtype == ICRL_F32 ? 4 : 2),        \
                 who ": dlogits overlaps the logits without being them")
}  // namespace

extern "C" int icrl_distill_loss(const void* logits, int dtype, int64_t ld_logits, int N, int V, const float* teacher_values,
                                 const int64_t* teacher_indices, int k, const float* teacher_lse, double temperature,
                                 const float* row_weight, float* row_loss, double* stats, void* dlogits, int64_t ld_dlogits,
                                 icrl_stream_t stream) {
    if (int rc = check("icrl_distill_loss", logits, ld_logits, N, V, teacher_values, teacher_indices, k, temperature)) return rc;
    ICRL_REQUIRE(row_loss, "icrl_distill_loss: null pointer or empty shape");
    ICRL_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, "icrl_distill_loss: stats must be 8-byte aligned");
    ICRL_REQUIRE(!dlogits || ld_dlogits >= V, "icrl_distill_loss: ld_dlogits < V");
    ICRL_REQUIRE_PLACES("icrl_distill_loss");
    const size_t lds = (size_t)((V + 31) / 32) * 4;
#define ICRL_CALL(T, NT, NV)                                                                                            \
    hipLaunchKernelGGL((distill_kernel<T, NT, NV>), dim3(N), dim3(NT), lds, icrl::as_stream(stream),                    \
                       static_cast<const T*>(logits), ld_logits, V, teacher_values, teacher_indices, k, teacher_lse,    \
                       1.0 / temperature, row_weight, row_loss, stats, static_cast<T*>(dlogits), ld_dlogits)
    switch (dtype) {
        case ICRL_F32: ICRL_ROW_DISPATCH(float, V, ICRL_CALL); break;
        case ICRL_BF16: ICRL_ROW_DISPATCH(__bf16, V, ICRL_CALL); break;
        case ICRL_F16: ICRL_ROW_DISPATCH(_Float16, V, ICRL_CALL); break;
        default: icrl::set_error("icrl_distill_loss: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
#undef ICRL_CALL
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

extern "C" int icrl_distill_grad(const void* logits, int dtype, int64_t ld_logits, int N, int V, const float* teacher_values,
                                 const int64_t* teacher_indices, int k, double temperature, const double* stats,
                                 const float* row_weight, void* dlogits, int64_t ld_dlogits, icrl_stream_t stream) {
    if (int rc = check("icrl_distill_grad", logits, ld_logits, N, V, teacher_values, teacher_indices, k, temperature)) return rc;
    ICRL_REQUIRE(stats && dlogits, "icrl_distill_grad: null pointer or empty shape");
    ICRL_REQUIRE(reinterpret_cast<uintptr_t>(stats) % 8 == 0, "icrl_distill_grad: stats must be 8-byte aligned");
    ICRL_REQUIRE(ld_dlogits >= V, "icrl_distill_grad: ld_dlogits < V");
    ICRL_REQUIRE_PLACES("icrl_distill_grad");
#define ICRL_CALL(T, NT, NV)                                                                                           \
    hipLaunchKernelGGL((distill_grad_kernel<T, NT, NV>), dim3(N), dim3(NT), 0, icrl::as_stream(stream),                \
                       static_cast<const T*>(logits), ld_logits, V, teacher_values, teacher_indices, k,                \
                       1.0 / temperature, stats, row_weight, static_cast<T*>(dlogits), ld_dlogits)
    switch (dtype) {
        case ICRL_F32: ICRL_ROW_DISPATCH(float, V, ICRL_CALL); break;
        case ICRL_BF16: ICRL_ROW_DISPATCH(__bf16, V, ICRL_CALL); break;
        case ICRL_F16: ICRL_ROW_DISPATCH(_Float16, V, ICRL_CALL); break;
        default: icrl::set_error("icrl_distill_grad: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
#undef ICRL_CALL
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

// Rows of logits ranked and filtered: token sampling with temperature, top-k, top-p and min-p, and the k largest
// entries of a row with its log-normaliser.  One workgroup per row; few long rows are shared by several.
//
// A row's order is: larger value first, ties by lowest index.  An entry's place in it is its composite, (order key of the
// value) << 32 | ~index, and what a filter keeps is always a beginning of the order, composite >= cut.
//
// What bounds these operators is not memory but how often a row's entries pass through the one CU that works on it (a
// row of 10 000 costs 0.07 us for every instruction per entry), so passes are few and short, and everything else is done
// on lists of at most a thread per entry:
//   - The k-th largest of the threads' own maxima is a lower bound of the k-th largest entry, and hardly more than k
//     entries reach it.  They are collected and ranked; filters that start from a top-k never look at the row again.
//   - min-p is a bound itself.
//   - top-p alone: a histogram of the masses of 2048 value ranges names the range that the cut falls into, and only that
//     range is ranked.  Where a list gets longer than the threads (ties), or top-k is large, the same is done with exact
//     sums, and a range that is too long even so is refined by radix passes over its keys.
//
// Masses are 64-bit integers, multiples of 2^-S of the row's largest weight with S = 62 - ceil(log2 V) (at most 51):
// integer sums have no order, so atomics and any split of the row give the same bits, and 2^-45 of the largest weight
// at V = 131072 is finer than float32 by six orders of magnitude: a draw falls on the side of a border that exact
// arithmetic gives unless it is that close.
#include <algorithm>
#include <math.h>

#include "vocab_row.h"

namespace {
using namespace icrl;

constexpr int BINS = 2048;

template <int NT>
struct Shared {
    u64 hist[BINS];           // histogram; afterwards, or instead, the list of entries that is ranked
    u64 part[NT / 64 + 1];    // per-wave sums
    unsigned key_lo, key_hi;
    int count, bin, index;
    u64 above, cut, total;
    float red[NT / 64];
    int flag;
};

__device__ __forceinline__ u64 composite(unsigned key, int index) { return (u64)key << 32 | (unsigned)~index; }
__device__ __forceinline__ float value_of(u64 c) {
    const unsigned key = (unsigned)(c >> 32);
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ int index_of(u64 c) { return (int)~(unsigned)c; }

// Weights of one row: e^((x - top) / T) as multiples of 2^-S.  An infinite top counts as the largest finite number (as do
// the entries equal to it; the callers see to it that no others are kept then).
struct Weights {
    double top, per_unit;   // per_unit = log2(e) / T
    int S;
    __device__ __forceinline__ double units(float x) const {   // before rounding
        const double t = ((double)fminf(x, 3.402823466e38f) - top) * per_unit;
        return exp2_normal(fmax(t, -(double)(S + 2)), S);       // at least 1/4, which rounds to nothing; at most 2^51
    }
    static __device__ __forceinline__ u64 rounded(double units) {   // the sum's low 52 bits: units to the nearest integer
        return (u64)__double_as_longlong(units + 0x1p52) & ((1ull << 52) - 1);
    }
    __device__ __forceinline__ u64 operator()(float x) const { return rounded(units(x)); }
};
__device__ __forceinline__ Weights weights_of(float best, double temp, int S) {
    return Weights{(double)fminf(best, 3.402823466e38f), 1.4426950408889634074 / temp, S};
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float m = red[0];
#pragma unroll
    for (int w = 1; w < NT / 64; ++w) m = fmaxf(m, red[w]);
    return m;
}

// Exclusive prefix of v over the workgroup's threads (and the total in sm.total); every thread calls it.
template <int NT>
__device__ __forceinline__ u64 block_prefix(u64 v, Shared<NT>& sm) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 inc = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const u64 up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
    }
    __syncthreads();
    if (lane == 63) sm.part[wave] = inc;
    __syncthreads();
    u64 before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) {
        const u64 p = sm.part[w];
        if (w < wave) before += p;
        total += p;
    }
    sm.total = total;   // every thread writes the same value
    return before + inc - v;
}

// Descending sort of one u64 per thread: bitonic, exchanges inside a wave by shuffles, across waves through LDS.
template <int NT>
__device__ __forceinline__ u64 block_sort(u64 v, u64* lds) {
    const int tid = threadIdx.x;
#pragma unroll
    for (int size = 2; size <= NT; size <<= 1) {
        const bool down = (tid & size) == 0 || size == NT;
#pragma unroll
        for (int stride = size >> 1; stride > 0; stride >>= 1) {
            u64 other;
            if (stride >= 64) {
                __syncthreads();
                lds[tid] = v;
                __syncthreads();
                other = lds[tid ^ stride];
            } else {
                other = __shfl_xor(v, stride, 64);
            }
            const bool lower = (tid & stride) == 0;
            const bool take_larger = lower == down;
            v = (other > v) == take_larger ? other : v;
        }
    }
    return v;
}

// Per-wave sums of f(value, index) into sm.part; the total is returned to every thread.
template <int NT, typename R, typename F>
__device__ __forceinline__ u64 wave_totals(const R& row, Shared<NT>& sm, F&& f) {
    u64 mine = 0;
    row.each([&](float x, int i) { mine += f(x, i); });
    mine = wave_sum_u64(mine);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sm.part[threadIdx.x >> 6] = mine;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) total += sm.part[w];
    return total;
}

// The index at which the running sum of f in index order first exceeds `target` (< the total that wave_totals has just
// left per wave).  One wave owns that place; it walks its piece vector by vector.
template <int NT, typename R, typename F>
__device__ __forceinline__ int locate(const R& row, Shared<NT>& sm, u64 target, F&& f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 before = 0;
    for (int w = 0; w < wave; ++w) before += sm.part[w];
    if (target >= before && target - before < sm.part[wave]) {
        u64 left = target - before;
        bool found = false;
        for (int i = 0; i < row.vectors && !found; ++i) {
            const auto p = row.fetch(i);
            const int at0 = row.first + i * 64 * R::VEC;
            u64 own = 0;
            row.vector(p, at0, [&](float x, int at) { own += f(x, at); });
            u64 inc = own;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 up = __shfl_up(inc, o, 64);
                if (lane >= o) inc += up;
            }
            const u64 all = __shfl(inc, 63, 64);
            if (left >= all) {
                left -= all;
                continue;
            }
            found = true;
            if (left >= inc - own && left < inc) {
                u64 run = inc - own;
                bool done = false;
                row.vector(p, at0, [&](float x, int at) {
                    run += f(x, at);
                    if (!done && run > left) { sm.index = at; done = true; }
                });
            }
        }
    }
    __syncthreads();
    return sm.index;
}

// The same with the vectors of the piece summed side by side, one a wave, where f is long (512 rows of 10 000, top-p 0.9:
// 33.3 against 31.7 us, 64 rows of 131072 without filters on a workgroup each 71 against 57; in the kernel that records rows
// its registers would cost more: 44 against 55 us for 4096 x 10000).  sm.hist is free.
template <int NT, typename R, typename F>
__device__ __forceinline__ int locate_wide(const R& row, Shared<NT>& sm, u64 target, F&& f) {
    constexpr int WAVES = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int piece = 0;
    u64 left = target;
#pragma unroll 1
    while (piece < WAVES - 1 && left >= sm.part[piece]) left -= sm.part[piece++];
    __syncthreads();   // (the histogram's last readers are done)
#pragma unroll 1
    for (int base = 0; base < row.vectors; base += WAVES) {
        const int i = base + wave, at0 = ((piece * row.vectors + i) * 64 + lane) * R::VEC;
        u64 own = 0;
        typename R::Pack p = R::fill();
        if (i < row.vectors) {
            p = row.fetch_at(at0);
            row.vector(p, at0, [&](float x, int at) { own += f(x, at); });
        }
        u64 inc = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64 up = __shfl_up(inc, o, 64);
            if (lane >= o) inc += up;
        }
        if (lane == 63) sm.hist[wave] = inc;
        __syncthreads();
        u64 before = 0, all = 0;
#pragma unroll 1
        for (int w = 0; w < WAVES; ++w) {
            const u64 s = sm.hist[w];
            before += w < wave ? s : 0;
            all += s;
        }
        if (left >= before + inc - own && left < before + inc) {   // one thread, if it is here at all
            u64 run = before + inc - own;
            bool done = false;
            row.vector(p, at0, [&](float x, int at) {
                run += f(x, at);
                if (!done && run > left) { sm.index = at; done = true; }
            });
        }
        if (left < all) break;
        left -= all;
        __syncthreads();
    }
    __syncthreads();
    return sm.index;
}

// Where the running sum of the bins (bin_at(0) first) reaches `need` (which need_of makes from the total): bin in sm.bin, the
// sum of the bins before it in sm.above.  Returns need.
template <int NT, typename H, typename G>
__device__ __forceinline__ u64 find_bin(Shared<NT>& sm, H&& bin_at, G&& need_of) {
    constexpr int PER = BINS / NT;
    u64 own[PER], sum = 0;
#pragma unroll
    for (int b = 0; b < PER; ++b) {
        own[b] = bin_at(threadIdx.x * PER + b);
        sum += own[b];
    }
    u64 run = block_prefix<NT>(sum, sm);
    const u64 need = need_of(sm.total);
    if (run < need && run + sum >= need) {
        bool done = false;
#pragma unroll
        for (int b = 0; b < PER; ++b) {
            if (!done && run + own[b] >= need) { sm.bin = threadIdx.x * PER + b; sm.above = run; done = true; }
            run += own[b];
        }
    }
    __syncthreads();
    return need;
}

template <int NT>
__device__ __forceinline__ void clear_hist(Shared<NT>& sm) {
    __syncthreads();
    for (int b = threadIdx.x; b < BINS; b += NT) sm.hist[b] = 0;
    __syncthreads();
}

// Sorts the n <= NT composites in sm.hist: thread i gets the i-th of the order (0 past the end).  Short lists are ranked
// by comparing all with all (n / 2 reads of two entries each, 0.5 us at n = 100 against 2.8 us for the sort).
template <int NT>
__device__ __forceinline__ u64 ranked(int n, Shared<NT>& sm) {
    const int tid = threadIdx.x;
    if (n <= 256 && n < BINS / 2) {
        u64* out = sm.hist + BINS / 2;
        if (tid == 0) sm.hist[n] = 0;   // an even number of entries to read
        __syncthreads();
        if (tid < n) {
            const u64 mine = sm.hist[tid];
            const ulonglong2* two = reinterpret_cast<const ulonglong2*>(sm.hist);
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < (n + 1) / 2; ++j) {
                const ulonglong2 o = two[j];
                rank += (o.x > mine) + (o.y > mine);
            }
            out[rank] = mine;
        }
        __syncthreads();
        return tid < n ? out[tid] : 0;
    }
    const u64 c = tid < n ? sm.hist[tid] : 0;
    return block_sort<NT>(c, sm.hist);
}

// Equal value ranges counted from the top: monotone in the row's order; what is far below the top, NaN included, is the
// last one, and +inf, which lies above a finite top, the first.
struct RangeBins {
    float top, per;
    __device__ __forceinline__ int operator()(float x) const {
        const float at = (top - x) * per;
        return at < (float)(BINS - 1) ? (int)fmaxf(at, 0.f) : BINS - 1;
    }
};

// The cut after the shortest prefix (in the row's order, among the entries with composite >= `from`) whose amounts -
// by_mass: weights, else 1 each - reach need_of(total).  width: the value range that the first histogram spreads over its
// bins, counted from the top; any positive width gives the same cut, a good one makes the second step short.
// Weights are computed for a whole vector before anything depends on one of them: a weight is a chain of some 20 float64
// instructions, and only side by side do they hide each other's latency.
// Returns with the kept masses of the waves' pieces in sm.part and their total in `mass_kept` if by_mass and the second
// step was the short one; otherwise mass_kept is 0.
template <int NT, typename R, typename G>
__device__ __forceinline__ u64 find_cut(const R& row, Shared<NT>& sm, bool by_mass, u64 from, const Weights& weight, float width,
                                        G&& need_of, u64& mass_kept) {
    constexpr int VEC = R::VEC;
    // with values, not keys (a few instructions an entry less); NaN, which no comparison keeps, belongs to a whole row
    const float from_x = value_of(from);
    const unsigned from_index = ~(unsigned)from;
    const bool whole = from_x != from_x;
    auto kept = [&](float x, int i) {
        return whole ? i < row.V : (x > from_x) | ((x == from_x) & ((unsigned)i <= from_index));
    };
    auto amount = [&](float x) { return by_mass ? weight(x) : (u64)1; };
    const RangeBins bin{(float)weight.top, (float)BINS / width};
    auto amounts = [&](const typename R::Pack& p, u64 (&a)[VEC]) {
        if (by_mass) {
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = weight(Elem<typename R::Type>::value(p.e[j]));
        } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = 1;
        }
    };
    mass_kept = 0;
    clear_hist<NT>(sm);
    if (threadIdx.x == 0) { sm.count = 0; sm.key_lo = ~0u; sm.key_hi = 0; }
    u64 rest = 0;   // the last bin, which may hold most of the row, is summed in registers
    row.each_pack([&](const typename R::Pack& p, int at) {
        u64 a[VEC];
        amounts(p, a);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float x = Elem<typename R::Type>::value(p.e[j]);
            const int b = bin(x);
            const bool in = kept(x, at + j);
            rest += in && b == BINS - 1 ? a[j] : 0;
            if (in && b < BINS - 1) atomicAdd(&sm.hist[b], a[j]);
        }
    });
    rest = wave_sum_u64(rest);
    if ((threadIdx.x & 63) == 0 && rest) atomicAdd(&sm.hist[BINS - 1], rest);
    __syncthreads();
    auto counted = [&](int b) { return sm.hist[b]; };
    u64 need = find_bin<NT>(sm, counted, need_of);
    const int b0 = sm.bin;
    const u64 above = sm.above;
    need -= above;
    __syncthreads();   // the histogram's place now takes the entries of that bin
    u64 sure = 0;      // this thread's share of the mass above it
    row.each_pack([&](const typename R::Pack& p, int at) {
        u64 a[VEC];
        amounts(p, a);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float x = Elem<typename R::Type>::value(p.e[j]);
            const int b = bin(x);
            const bool in = kept(x, at + j);
            sure += in && b < b0 ? a[j] : 0;
            if (in && b == b0) {
                const int to = atomicAdd(&sm.count, 1);
                if (to < NT) sm.hist[to] = composite(order_key(x), at + j);
            }
        }
    });
    sure = wave_sum_u64(sure);
    __syncthreads();
    const int members = sm.count;
    if (members <= NT) {
        const u64 c = ranked<NT>(members, sm);
        const u64 a = c ? amount(value_of(c)) : 0;
        const u64 before = block_prefix<NT>(a, sm);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sm.part[threadIdx.x >> 6] = sure;
        if (before < need && before + a >= need) { sm.cut = c; sm.total = before + a; }
        __syncthreads();
        if (by_mass) {
            mass_kept = above + sm.total;
            if (a && before < need) atomicAdd(&sm.part[index_of(c) / (row.vectors * 64 * VEC)], a);
            __syncthreads();
        }
        return sm.cut;
    }
    // many entries in one range: radix over the keys that occur in it, 11 bits a pass
    unsigned lo = ~0u, hi = 0;
    row.each([&](float x, int i) {
        const unsigned key = order_key(x);
        if (kept(x, i) && bin(x) == b0) { lo = min(lo, key); hi = max(hi, key); }
    });
    atomicMin(&sm.key_lo, lo);
    atomicMax(&sm.key_hi, hi);
    __syncthreads();
    lo = sm.key_lo;
    hi = sm.key_hi;
    while (lo < hi) {
        const int bits = 32 - __clz((int)(hi - lo)), shift = bits > 11 ? bits - 11 : 0;
        clear_hist<NT>(sm);
        row.each([&](float x, int i) {
            const unsigned key = order_key(x);
            if (key >= lo && key <= hi && kept(x, i) && bin(x) == b0) {
                const u64 a = amount(x);
                if (a) atomicAdd(&sm.hist[(hi - key) >> shift], a);
            }
        });
        __syncthreads();
        const u64 want = need;
        find_bin<NT>(sm, counted, [&](u64) { return want; });
        need -= sm.above;
        const unsigned upper = hi - ((unsigned)sm.bin << shift);
        const unsigned span = (1u << shift) - 1u;
        lo = upper - lo > span ? upper - span : lo;
        hi = upper;
        __syncthreads();
    }
    // the entries with this key, in index order, until they reach what is left
    const u64 each = amount(value_of((u64)lo << 32));
    auto tie = [&](float y, int i) { return (u64)(order_key(y) == lo && kept(y, i)); };
    wave_totals<NT>(row, sm, tie);
    const int last = locate<NT>(row, sm, (need + each - 1) / each - 1, tie);
    __syncthreads();
    return composite(lo, last);
}

// A value that at least k entries of the row reach (k <= NT), not far below the k-th largest: the k-th largest of the
// threads' own maxima, cut to its key's upper 16 bits.  Four bits a step: the waves share out the 16 continuations of
// what is known (0.5 us; a single wave, bit by bit, takes 1.9).  -inf: fewer than k threads hold an entry above it.
template <int NT>
__device__ __forceinline__ float bound_of(float own_max, int k, Shared<NT>& sm) {
    constexpr int WAVES = NT / 64, PER = 16 / WAVES;   // continuations a wave counts
    unsigned* keys = reinterpret_cast<unsigned*>(sm.hist);
    int* reached = reinterpret_cast<int*>(sm.hist + BINS / 2);   // 16 counts a step
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();
    keys[threadIdx.x] = order_key(own_max) >> 16;
    __syncthreads();
    unsigned key[WAVES], t = 0;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) key[i] = keys[lane + 64 * i];
#pragma unroll
    for (int step = 0; step < 4; ++step) {
        const int shift = 12 - 4 * step;
#pragma unroll
        for (int c = 0; c < PER; ++c) {
            const unsigned at_least = t | (unsigned)(wave * PER + c) << shift;
            int n = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) n += __popcll(__ballot(key[i] >= at_least));
            if (lane == 0) reached[16 * step + wave * PER + c] = n;
        }
        __syncthreads();
        // counts fall as the continuation rises: the last that k maxima reach
        const int n = lane < 16 ? reached[16 * step + lane] : 0;
        const int last = __popcll(__ballot(lane < 16 && n >= k)) - 1;
        t |= (unsigned)max(last, 0) << shift;   // (none: fewer than k maxima, which only step 0 can say; t stays 0)
    }
    t <<= 16;
    // between two upper halves lies -inf's: what rounds down to it or below says nothing
    return t <= kKeyMinusInf ? -INFINITY : value_of((u64)t << 32);
}

// Composites of the entries >= bound (> -inf) into sm.hist, at most `room` of them; returns how many there are.  A thread
// keeps its first two to itself, so that nothing waits for the shared counter while it reads; only what a thread finds
// beyond them goes through it one by one.  FEW: hardly a vector holds any (the lists of a top-k; 64 rows of 131072 bf16 with
// settings of their own, first launch: 25 us, 30 without).  Otherwise a wave goes through one find of every
// lane at a time, as often as its busiest lane has finds, once or twice, and not once for each place of a vector (333 rows
// of 50257 f16 with some 600 finds: 47 against 38 us; a record's 64 of 10000, 512 threads: 44.2 against 45.3, of 30000, 1024
// threads: 82.8 against 74.5).
template <int NT, bool FEW, typename R>
__device__ __forceinline__ int collect(const R& row, Shared<NT>& sm, float bound, int room) {
    const int lane = threadIdx.x & 63;
    __syncthreads();
    if (threadIdx.x == 0) sm.count = 0;
    __syncthreads();
    u64 mine[2] = {0, 0};
    int n = 0;
    row.sweep([&](const typename R::Pack& p, int at) {
        float most = -INFINITY;
#pragma unroll
        for (int j = 0; j < R::VEC; ++j) most = fmaxf(most, Elem<typename R::Type>::value(p.e[j]));
        if (!(most >= bound)) return;
        auto keep = [&](float x, int i) {
            const u64 c = composite(order_key(x), i);
            if (n >= 2) {
                const int to = atomicAdd(&sm.count, 1);
                if (to < room) sm.hist[to] = c;
            }
            mine[1] = n == 1 ? c : mine[1];
            mine[0] = n == 0 ? c : mine[0];
            ++n;
        };
        if (FEW) {
#pragma unroll
            for (int j = 0; j < R::VEC; ++j) {
                const float x = Elem<typename R::Type>::value(p.e[j]);
                if (x >= bound) keep(x, at + j);
            }
            return;
        }
        unsigned found = 0;
#pragma unroll
        for (int j = 0; j < R::VEC; ++j) found |= (unsigned)(Elem<typename R::Type>::value(p.e[j]) >= bound) << j;
#pragma unroll 1
        while (found) {
            const int at_j = __ffs((int)found) - 1;
            found &= found - 1;
            float x = 0.f;
#pragma unroll
            for (int j = 0; j < R::VEC; ++j) x = at_j == j ? Elem<typename R::Type>::value(p.e[j]) : x;
            keep(x, at + at_j);
        }
    });
    n = min(n, 2);
    const u64 one = __ballot(n >= 1), two = __ballot(n == 2), below = (1ull << lane) - 1;
    int base = 0;
    if (lane == 0) base = atomicAdd(&sm.count, __popcll(one) + __popcll(two));
    base = __shfl(base, 0, 64) + __popcll(one & below) + __popcll(two & below);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (i < n && base + i < room) sm.hist[base + i] = mine[i];
    __syncthreads();
    return sm.count;
}

// ---------------------------------------------------------------------------------------------- sampling
struct Setting {   // one filter setting: a value for each row, or one for all of them
    const float* rows;
    double all;
    __device__ __forceinline__ double at(int r) const { return rows ? (double)rows[r] : all; }
};

struct Requests {
    const double* uniforms;
    Setting temperature, top_p, min_p;
    const int* top_k_rows;
    int top_k_all;
};
struct Results {
    int64_t* tokens;
    int64_t token_stride;
    float* log_prob;
    int64_t lp_stride;
};

// One row's settings, and what follows from them.
struct Request {
    double temp, top_p, min_p, u, floor_z;   // w >= min_p as x - best >= floor_z = T log(min_p)
    int top_k;
    __device__ __forceinline__ Request(const Requests& all, int r)
        : temp(all.temperature.at(r)), top_p(all.top_p.at(r)), min_p(all.min_p.at(r)), u(all.uniforms[r]), floor_z(-INFINITY),
          top_k(all.top_k_rows ? all.top_k_rows[r] : all.top_k_all) {
        if (min_p > 0.0) floor_z = log(min_p) * temp;
    }
    __device__ __forceinline__ bool fine() const {
        return temp >= 0.0 && temp < INFINITY && top_k >= 0 && top_p >= 0.0 && top_p <= 1.0 && min_p >= 0.0 && min_p <= 1.0 && u == u;
    }
    __device__ __forceinline__ u64 prefix_mass(u64 total) const {   // what top_p asks for
        const double w = ceil(top_p * (double)total);
        const u64 want = w < 1.0 ? 1 : (u64)w;
        return want < total ? want : total;
    }
    __device__ __forceinline__ u64 target(u64 total) const {
        const double want = u * (double)total;
        const u64 t = want > 0.0 ? (u64)fmin(want, 0x1p63) : 0;
        return t < total ? t : total - 1;
    }
    // value range that holds every entry with weight: entries further below the top have none
    __device__ __forceinline__ float reach(int S) const { return fmaxf((float)(S * 0.6931471805599453 * temp), 1e-30f); }
    // value range below which lies less than e^-7 of the top's weight, V entries taken together: up to top_p = 0.999 no
    // cut lies there, and the bins over it are half as wide
    __device__ __forceinline__ float span(int V, int S) const {
        return fmaxf(fminf((float)temp * (__logf((float)V) + 7.f), reach(S)), 1e-30f);
    }
    __device__ __forceinline__ void write(const Results& out, int r, int token, float x, float best, u64 total, int S) const {
        out.tokens[r * out.token_stride] = token;
        if (out.log_prob) {
            const double z = x == best ? 0.0 : ((double)x - (double)best) / temp;
            out.log_prob[r * out.lp_stride] = (float)(z - log(ldexp((double)total, -S)));
        }
    }
};

// What of a row remains after the cut and min-p: the weight of entry i, value x, or 0.
struct Mass {
    Weights weight;
    float best, cut_x;
    unsigned cut_index;
    double floor_z;
    __device__ __forceinline__ u64 operator()(float x, int i) const {
        const u64 w = weight(x);
        const bool in = (x > cut_x) | ((x == cut_x) & ((unsigned)i <= cut_index));
        const bool low = (x != best) & ((double)x - (double)best < floor_z);
        return (in & !low) ? w : 0;
    }
};

// Rows too long for one CU (split calls, see sample_chunk_mass): what the first launch leaves of a row, and where the
// workgroups on its chunks meet.  8-byte words per row: the state, the pieces' masses, a list of entries, the histogram.
struct RowState {
    float best, per;    // per: bins per unit of value, computed once for both launches
    int pending;        // 0: drawn; 1: top-p over the whole row; 2: no prefix to find
    unsigned listed, ticket;
};
constexpr int CHUNK_NT = 512, MAX_PIECES = 512, ROOM = 512;
constexpr int STATE_WORDS = 8, WORK_WORDS = STATE_WORDS + MAX_PIECES + ROOM + BINS;
static_assert(ROOM <= CHUNK_NT && MAX_PIECES <= CHUNK_NT, "a thread ranks one entry and adds up one piece");
struct Work {
    u64* rows;
    __device__ __forceinline__ RowState* state(int r) const { return reinterpret_cast<RowState*>(rows + (int64_t)r * WORK_WORDS); }
    __device__ __forceinline__ u64* pieces(int r) const { return rows + (int64_t)r * WORK_WORDS + STATE_WORDS; }
    __device__ __forceinline__ u64* list(int r) const { return pieces(r) + MAX_PIECES; }
    __device__ __forceinline__ u64* hist(int r) const { return list(r) + ROOM; }
};

struct Kept { u64 w; unsigned index; float x; };

// w_i = e^((x_i - best) / T); keep the first top_k of the row's order, of those the shortest prefix with top_p of their mass,
// of those w_i >= min_p; the token is the first kept one, by index, at which the running mass exceeds u times the total.
// Bound by the arithmetic of the passes that weigh entries (about 45 instructions an entry, 20 of them float64; a top-p
// over the whole row weighs it twice) and, with a list, by two reads of the row on one CU.  Measured (us a call): 1 row of
// 10 000, top-k 50 and top-p 0.95: 10.4; 512 rows of 10 000, top-p 0.9: 31-33 (the rows' bytes alone take 5, the vector
// instructions, 144 an entry altogether, 20); 333 rows of 50 257 f16, min-p 0.05: 27; 64 rows of 131 072 bf16, settings of
// their own, with the launches below: 54-61.
// split.rows not null: rows that need the weights of all their entries are left to the launches that follow.
template <typename T, int NT>
__global__ __launch_bounds__(NT, 4) void sample_filtered_kernel(const T* __restrict__ logits, int64_t ld, int V, int S, Requests all,
                                                                Results out, Work split) {
    __shared__ Shared<NT> sm;
    const int r = blockIdx.x, tid = threadIdx.x;
    // Read again by every pass: the passes that weigh entries, unrolled over a row in registers, would be far longer than
    // the instruction cache, and with registers to spare two workgroups fit a CU (512 rows of 10 000: 33 against 36 us)
    Row<T, NT, IN_MEMORY, false> row;
    row.open(logits + (int64_t)r * ld, V);
    const Request q(all, r);
    const int top_k = q.top_k;
    const double floor_z = q.floor_z;
    if (tid == 0) {
        sm.flag = 0;
        if (split.rows) split.state(r)->pending = 0;
    }
    float best = -INFINITY;
    u64 nan = 0;                                     // the wave's lanes
    row.sweep([&](const auto& p, int) {
#pragma unroll
        for (int j = 0; j < Elem<T>::VEC; j += 2) {
            const float x = Elem<T>::value(p.e[j]), y = Elem<T>::value(p.e[j + 1]);
            best = fmaxf(best, fmaxf(x, y));         // fmaxf passes over NaN
            nan |= __ballot(__builtin_isunordered(x, y));
        }
    });
    const float own = best;
    best = block_max<NT>(best, sm.red);
    if (nan) sm.flag = 1;
    __syncthreads();
    if (!q.fine() || sm.flag || best == -INFINITY) {
        if (tid == 0) {
            out.tokens[r * out.token_stride] = -1;
            if (out.log_prob) out.log_prob[r * out.lp_stride] = NAN;
        }
        return;
    }
    if (q.temp == 0.0 || top_k == 1 || q.top_p == 0.0) {   // the first largest entry
        if (tid == 0) sm.index = V;
        __syncthreads();
        if (own == best) {
            int first = V;
            row.sweep_each([&](float x, int i) { first = x == best ? min(first, i) : first; });
            atomicMin(&sm.index, first);
        }
        __syncthreads();
        if (tid == 0) {
            out.tokens[r * out.token_stride] = sm.index;
            if (out.log_prob) out.log_prob[r * out.lp_stride] = 0.f;
        }
        return;
    }
    const Weights weight = weights_of(best, q.temp, S);
    const bool by_k = top_k > 0 && top_k < V, by_p = q.top_p < 1.0;
    const bool leave = split.rows && !by_k;   // to the launches on the row's chunks, unless a list settles it

    // ---- the short list: entries no smaller than a bound that everything kept reaches
    float bound = -INFINITY;
    if (by_k) {
        if (top_k <= NT / 2) bound = bound_of<NT>(own, top_k, sm);
    } else if (q.min_p > 0.0 && best < INFINITY && !(leave && by_p)) {
        const double z = (double)best + floor_z;
        bound = (float)z;
        if ((double)bound > z) bound = nextafterf(bound, -INFINITY);
    }
    if (bound > -INFINITY) {
        constexpr int ITEMS = NT >= 1024 ? 2 : 4;   // entries a thread may hold; lists that are ranked have one each
        const bool rank = by_k || by_p;
        const int room = rank ? NT : NT * ITEMS, n = by_k ? collect<NT, true>(row, sm, bound, room) : collect<NT, false>(row, sm, bound, room);
        bool listed = n <= room;
        if (listed) {
            u64 c[ITEMS], w[ITEMS];
            if (rank) {
                c[0] = ranked<NT>(n, sm);
                if (by_k && tid >= top_k) c[0] = 0;
#pragma unroll
                for (int e = 1; e < ITEMS; ++e) c[e] = 0;
            } else {
#pragma unroll
                for (int e = 0; e < ITEMS; ++e) c[e] = tid + e * NT < n ? sm.hist[tid + e * NT] : 0;
            }
#pragma unroll
            for (int e = 0; e < ITEMS; ++e) {
                const float x = value_of(c[e]);
                w[e] = c[e] && (best < INFINITY || x == best) ? weight(x) : 0;
            }
            if (by_p) {
                const u64 before = block_prefix<NT>(w[0], sm);
                const u64 mass_listed = sm.total;
                const u64 from = by_k ? mass_listed : wave_totals<NT>(row, sm, [&](float y, int) { return y > -INFINITY ? weight(y) : 0; });
                if (before >= q.prefix_mass(from)) w[0] = 0;
            }
            // the masses of the waves' pieces name the piece that the draw falls into, and its kept entries settle it among
            // themselves: each adds up the weights of those that come no later in the vocabulary
            const int piece = row.vectors * 64 * Elem<T>::VEC;
            Kept* kept = reinterpret_cast<Kept*>(sm.hist);
            constexpr int KEPT = BINS / 2;   // as many as fit the histogram's place
            static_assert(sizeof(Kept) * KEPT <= sizeof(sm.hist), "the kept list fits");
            __syncthreads();
            if (tid == 0) sm.count = 0;
            if (tid < NT / 64) sm.part[tid] = 0;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < ITEMS; ++e) {
                const float x = value_of(c[e]);
                if (x != best && (double)x - (double)best < floor_z) w[e] = 0;
                if (w[e]) atomicAdd(&sm.part[index_of(c[e]) / piece], w[e]);
            }
            __syncthreads();
            u64 total = 0;
#pragma unroll
            for (int p = 0; p < NT / 64; ++p) total += sm.part[p];
            const u64 target = q.target(total);
            u64 before = 0;
            int at = 0;
            while (before + sm.part[at] <= target) before += sm.part[at++];
#pragma unroll
            for (int e = 0; e < ITEMS; ++e) {
                if (w[e] && index_of(c[e]) / piece != at) w[e] = 0;   // not in that piece
                if (w[e]) {
                    const int to = atomicAdd(&sm.count, 1);
                    if (to < KEPT) kept[to] = Kept{w[e], (unsigned)index_of(c[e]), value_of(c[e])};
                }
            }
            __syncthreads();
            const int m = sm.count;
            listed = m <= KEPT;
            if (listed) {
                for (int e = tid; e < m; e += NT) {   // (an entry a thread again: as few waves as the list takes)
                    const Kept mine = kept[e];
                    u64 upto = before;
#pragma unroll 4
                    for (int j = 0; j < m; ++j) {
                        const Kept o = kept[j];
                        upto += o.index <= mine.index ? o.w : 0;
                    }
                    if (upto > target && upto - mine.w <= target) q.write(out, r, (int)mine.index, mine.x, best, total, S);
                }
                return;
            }
        }
    }

    if (leave) {
        u64* hist = split.hist(r);
        for (int b = tid; b < BINS; b += NT) hist[b] = 0;
        if (tid == 0) *split.state(r) = RowState{best, (float)BINS / q.span(V, S), by_p ? 1 : 2, 0u, 0u};
        return;
    }

    // ---- the whole row
    // with an entry of +inf only the entries of +inf have weight (all the same)
    u64 cut = (u64)(best == INFINITY ? kKeyPlusInf : kKeyFinite) << 32, total = 0;
    for (int filter = 0; filter < 2; ++filter) {   // top-k, then top-p: one copy of the code
        const bool by_mass = filter == 1;
        if (!(by_mass ? by_p : by_k)) continue;
        const u64 k = (u64)top_k;
        cut = find_cut<NT>(row, sm, by_mass, cut, weight, by_mass ? q.span(V, S) : q.reach(S),
                           [&](u64 of) { return by_mass ? q.prefix_mass(of) : k < of ? k : of; }, total);
    }
    const Mass mass{weight, best, value_of(cut), ~(unsigned)cut, floor_z};
    if (total == 0 || q.min_p > 0.0) total = wave_totals<NT>(row, sm, mass);
    const int token = locate_wide<NT>(row, sm, q.target(total), mass);
    if (tid == 0) q.write(out, r, token, row.entry(token), best, total, S);
}

// ---- rows split over workgroups
// A row's weights cost some 45 instructions an entry, twice (40 us a pass for 131072 entries on one CU), so where rows are
// long and few their chunks are weighed side by side: one launch adds the chunks' histograms up (integers: any order
// gives the same), the next collects the range of the cut and the masses above it, and the workgroup that finishes last
// with a row draws.  No workgroup waits for another.
template <typename T>
__global__ __launch_bounds__(CHUNK_NT, 4) void sample_chunk_mass(const T* __restrict__ logits, int64_t ld, int V, int chunk, int S,
                                                                 Requests all, Work split) {
    constexpr int NT = CHUNK_NT;
    __shared__ Shared<NT> sm;
    const int r = blockIdx.y, tid = threadIdx.x, first = blockIdx.x * chunk;
    const RowState state = *split.state(r);
    if (state.pending != 1) return;
    const Request q(all, r);
    const Weights weight = weights_of(state.best, q.temp, S);
    const RangeBins bin{(float)weight.top, state.per};
    const float from = state.best == INFINITY ? INFINITY : -3.402823466e38f;
    Row<T, NT, IN_MEMORY, false> row;
    row.open(logits + (int64_t)r * ld + first, min(chunk, V - first));
    clear_hist<NT>(sm);
    u64 rest = 0;
    row.each_pack([&](const auto& p, int) {
        constexpr int VEC = Elem<T>::VEC;
        u64 a[VEC];
#pragma unroll
        for (int j = 0; j < VEC; ++j) a[j] = weight(Elem<T>::value(p.e[j]));
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            const float x = Elem<T>::value(p.e[j]);
            const int b = bin(x);
            rest += x >= from && b == BINS - 1 ? a[j] : 0;
            if (x >= from && b < BINS - 1) atomicAdd(&sm.hist[b], a[j]);
        }
    });
    rest = wave_sum_u64(rest);
    if ((tid & 63) == 0 && rest) atomicAdd(&sm.hist[BINS - 1], rest);
    __syncthreads();
    u64* hist = split.hist(r);
    for (int b = tid; b < BINS; b += NT)
        if (sm.hist[b]) atomicAdd(&hist[b], sm.hist[b]);
}

template <typename T>
__global__ __launch_bounds__(CHUNK_NT, 4) void sample_chunk_draw(const T* __restrict__ logits, int64_t ld, int V, int chunk, int S,
                                                                 Requests all, Results out, Work split) {
    constexpr int NT = CHUNK_NT, WAVES = NT / 64;
    __shared__ Shared<NT> sm;
    __shared__ u64 pieces[MAX_PIECES];
    const int r = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, first = blockIdx.x * chunk;
    const RowState state = *split.state(r);
    if (state.pending == 0) return;
    const Request q(all, r);
    const float best = state.best;
    const Weights weight = weights_of(best, q.temp, S);
    const RangeBins bin{(float)weight.top, state.per};
    const float from = best == INFINITY ? INFINITY : -3.402823466e38f;
    Row<T, NT, IN_MEMORY, false> row;
    row.open(logits + (int64_t)r * ld + first, min(chunk, V - first));
    Mass mass{weight, best, from, ~0u, q.floor_z};
    int b0 = 0;
    u64 need = 0, sum = 0;
    if (state.pending == 1) {
        const u64* hist = split.hist(r);
        need = find_bin<NT>(sm, [&](int b) { return hist[b]; }, [&](u64 of) { return q.prefix_mass(of); });
        b0 = sm.bin;
        need -= sm.above;
        if (tid == 0) sm.count = 0;
        __syncthreads();
        row.each_pack([&](const auto& p, int at) {
            constexpr int VEC = Elem<T>::VEC;
            u64 a[VEC];
#pragma unroll
            for (int j = 0; j < VEC; ++j) a[j] = weight(Elem<T>::value(p.e[j]));
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                const float x = Elem<T>::value(p.e[j]);
                const int b = bin(x);
                const bool low = (x != best) & ((double)x - (double)best < q.floor_z);
                sum += x >= from && b < b0 && !low ? a[j] : 0;
                if (x >= from && b == b0) {
                    const int to = atomicAdd(&sm.count, 1);
                    if (to < ROOM) sm.hist[to] = composite(order_key(x), first + at + j);
                }
            }
        });
    } else {
        row.each_pack([&](const auto& p, int at) {
#pragma unroll
            for (int j = 0; j < Elem<T>::VEC; ++j) sum += mass(Elem<T>::value(p.e[j]), at + j);
        });
    }
    sum = wave_sum_u64(sum);
    if (lane == 0) __hip_atomic_store(&split.pieces(r)[blockIdx.x * WAVES + wave], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (state.pending == 1) {   // this chunk's entries of the range, behind those of the chunks before
        const int n = sm.count;
        if (tid == 0) sm.index = (int)atomicAdd(&split.state(r)->listed, (unsigned)n);
        __syncthreads();
        const int to = sm.index + tid;
        if (tid < min(n, ROOM) && to < ROOM)
            __hip_atomic_store(&split.list(r)[to], sm.hist[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    // The last workgroup to get here draws.  What it reads of the others they have stored at agent scope (past their XCD's
    // cache), every wave has waited for its stores when one thread counts the workgroup in, and it is loaded at agent
    // scope: no fence, which would write the XCD's whole cache back (64 rows of 131072 took 92 us in this launch with one
    // in every wave).
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (tid == 0)
        sm.flag = __hip_atomic_fetch_add(&split.state(r)->ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
    __syncthreads();
    if (!sm.flag) return;
    const int count = (int)gridDim.x * WAVES;
    for (int p = tid; p < count; p += NT) pieces[p] = __hip_atomic_load(&split.pieces(r)[p], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // entries of a wave's piece of chunk c, as Row::open cuts it (the last chunk may be shorter than the others)
    auto piece_of = [&](int c) {
        constexpr int VEC = Elem<T>::VEC;
        return (min(chunk, V - c * chunk) + NT * VEC - 1) / (NT * VEC) * 64 * VEC;
    };
    __syncthreads();
    if (state.pending == 1) {
        const int n = (int)__hip_atomic_load(&split.state(r)->listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (n > ROOM) {   // more equal values than that: the whole row on this workgroup
            Row<T, NT, IN_MEMORY, false> long_row;
            long_row.open(logits + (int64_t)r * ld, V);
            u64 total = 0;
            const u64 cut = find_cut<NT>(long_row, sm, true, (u64)(best == INFINITY ? kKeyPlusInf : kKeyFinite) << 32, weight,
                                         q.span(V, S), [&](u64 of) { return q.prefix_mass(of); }, total);
            const Mass kept{weight, best, value_of(cut), ~(unsigned)cut, q.floor_z};
            total = wave_totals<NT>(long_row, sm, kept);
            const int token = locate_wide<NT>(long_row, sm, q.target(total), kept);
            if (tid == 0) q.write(out, r, token, long_row.entry(token), best, total, S);
            return;
        }
        if (tid < n) sm.hist[tid] = __hip_atomic_load(&split.list(r)[tid], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        const u64 c = ranked<NT>(n, sm);
        const float x = value_of(c);
        const u64 w = c ? weight(x) : 0;
        const u64 before = block_prefix<NT>(w, sm);
        if (c && before < need) {
            const int i = index_of(c);
            if (before + w >= need) sm.cut = c;
            if (!((x != best) & ((double)x - (double)best < q.floor_z))) atomicAdd(&pieces[i / chunk * WAVES + i % chunk / piece_of(i / chunk)], w);
        }
        __syncthreads();
        mass.cut_x = value_of(sm.cut);
        mass.cut_index = ~(unsigned)sm.cut;
    }
    const u64 mine = tid < count ? pieces[tid] : 0, before = block_prefix<NT>(mine, sm), total = sm.total, target = q.target(total);
    if (target >= before && target - before < mine) {   // the piece that the draw falls into
        sm.index = tid;
        sm.above = target - before;
    }
    __syncthreads();
    // within it: as locate() does, on a row of one wave that begins there
    const int at = sm.index, c = at / WAVES, piece = piece_of(c), offset = at % WAVES * piece, begin = c * chunk + offset;
    u64 left = sm.above;
    if (wave == 0) {
        Row<T, 64, IN_MEMORY, false> part;
        part.open(logits + (int64_t)r * ld + begin, min(piece, min(chunk - offset, V - begin)));
        bool found = false;
        for (int i = 0; i < part.vectors && !found; ++i) {
            const auto p = part.fetch(i);
            const int at0 = begin + part.first + i * 64 * part.VEC;
            u64 own = 0;
            part.vector(p, at0, [&](float y, int e) { own += mass(y, e); });
            u64 inc = own;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const u64 up = __shfl_up(inc, o, 64);
                if (lane >= o) inc += up;
            }
            const u64 sum_all = __shfl(inc, 63, 64);
            if (left >= sum_all) {
                left -= sum_all;
                continue;
            }
            found = true;
            if (left >= inc - own && left < inc) {
                u64 run = inc - own;
                bool done = false;
                part.vector(p, at0, [&](float y, int e) {
                    run += mass(y, e);
                    if (!done && run > left) { q.write(out, r, e, y, best, total, S); done = true; }
                });
            }
        }
    }
}

// ---------------------------------------------------------------------------------------------- top-k and log-normaliser
// values, indices: the first k of the row's order; lse = log sum e^(x / T) = max / T + log sum e^((x - max) / T), whose sum
// is float32 within a thread (some tens of terms) and float64 across them.  Bound by the one read of the row, which then
// stays in registers: 9728 rows of 10 000 (389 MB), k = 64: 101-103 us, 3.8 TB/s, against 4.0 of a plain sum.  Eight waves a
// SIMD, four workgroups a CU, so that one row's ranking runs under the others' reads.
template <typename T, int NT, int PLACE>
__global__ __launch_bounds__(NT, 8) void topk_lse_kernel(const T* __restrict__ logits, int64_t ld, int V, int k, double per_t,
                                                      float* __restrict__ values, int64_t* __restrict__ indices,
                                                      float* __restrict__ lse) {
    __shared__ Shared<NT> sm;
    __shared__ double sums[NT / 64];
    const int r = blockIdx.x, tid = threadIdx.x;
    Row<T, NT, PLACE, false> row;
    row.open(logits + (int64_t)r * ld, V);
    float best = -INFINITY;
    bool nan = false;
    if (tid == 0) sm.flag = 0;
    row.sweep_each([&](float x, int) {
        best = fmaxf(best, x);
        nan |= x != x;
    });
    const float own = best;
    best = block_max<NT>(best, sm.red);
    if (nan) sm.flag = 1;
    if (lse) {
        const bool some = best > -INFINITY && best < INFINITY;
        float part = 0.f;
        if (some) {
            const float c = (float)(per_t * 1.4426950408889634074);
            row.sweep_each([&](float x, int) { part += __builtin_amdgcn_exp2f((x - best) * c); });
        }
        double s = wave_sum_d((double)part);
        if ((tid & 63) == 0) sums[tid >> 6] = s;
        __syncthreads();
        if (tid == 0) {
            s = 0.0;
            for (int w = 0; w < NT / 64; ++w) s += sums[w];
            lse[r] = sm.flag ? NAN : some ? (float)((double)best * per_t + log(s)) : best;
        }
    }
    const float bound = k <= NT / 2 ? bound_of<NT>(own, k, sm) : -INFINITY;
    int n = NT + 1;
    if (bound > -INFINITY) n = collect<NT, NT <= 512>(row, sm, bound, NT);
    if (n > NT) {   // more ties than threads, a long list, or a row with fewer than k entries above -inf
        Row<T, NT, IN_MEMORY, true> again;
        again.open(logits + (int64_t)r * ld, V);
        const Weights weight = weights_of(best, INFINITY, 0);   // its top alone is used
        const float lowest = -block_max<NT>(-own, sm.red);   // the NT-th largest entry is no lower than the lowest thread's
        const float width = lowest > -INFINITY && best < INFINITY ? fmaxf((best - lowest) * 1.001f, 1e-30f) : 64.f;
        const u64 want = (u64)k;
        u64 none;
        const u64 cut = find_cut<NT>(again, sm, false, (u64)kKeyNan << 32, weight, width, [&](u64) { return want; }, none);
        __syncthreads();
        if (tid == 0) sm.count = 0;
        __syncthreads();
        again.each([&](float x, int i) {
            const u64 c = composite(order_key(x), i);
            if (c >= cut) sm.hist[atomicAdd(&sm.count, 1)] = c;   // exactly k entries, k <= NT
        });
        __syncthreads();
        n = k;
    }
    const u64 c = ranked<NT>(n, sm);
    if (tid < k) {
        values[(int64_t)r * k + tid] = value_of(c);
        indices[(int64_t)r * k + tid] = index_of(c);
    }
}

constexpr int MAX_K = 1024, MAX_V = 1 << 22;

// Workgroup size and vectors per thread in registers for rows of V entries of which `list` are to be ranked.
#define ICRL_ROW_DISPATCH(T, V, list, CALL)                                          \
    do {                                                                             \
        constexpr int vec_ = icrl::Elem<T>::VEC;                                     \
        if ((V) <= 256 * 4 * vec_ && (list) <= 256) { CALL(T, 256, 4); }             \
        else if ((V) <= 512 * 8 * vec_ && (list) <= 512) { CALL(T, 512, 8); }        \
        else if ((V) <= 1024 * 8 * vec_) { CALL(T, 1024, 8); }                       \
        else { CALL(T, 1024, IN_MEMORY); }                                           \
    } while (0)
}  // namespace

namespace {
// Entries per workgroup where rows are split (a multiple of what its threads read at once), or 0: not split.  Where two
// workgroups a CU are reached they get at least 8192 entries, up to four a CU, since rows that a list has settled leave
// theirs idle.  32 bit, top-p 0.9, one workgroup a row against split (us a call):
//   V        1 row          16             64             128
//   32768    38.8 / 21.3    39.9 / 26.4    40.4 / 29.4    43.5 / 38.4
//   50257    52.9 / 22.8    54.9 / 28.3    55.4 / 37.1    58.0 / 55.0
//   131072    108 / 27.4     113 / 34.7     115 / 65.5     120 / 97.7
// Shorter rows and more of them gain nothing.  Settings per row that leave no row to split cost 4 us (64 rows of 50257,
// top-k 50: 14.6 against 18.8).
int chunk_entries(int N, int V) {
    if (V < 32768 || N > 128) return 0;
    const int unit = CHUNK_NT * 8;
    const int chunks = std::min(MAX_PIECES / (CHUNK_NT / 64), std::max(2, 1024 / N));
    const int64_t even = ((int64_t)V + chunks - 1) / chunks, per = chunks * N > 512 ? std::max<int64_t>(even, 8192) : even;
    return (int)((per + unit - 1) / unit * unit);
}
}  // namespace

extern "C" int64_t icrl_sample_filtered_work_bytes(int N, int V) {
    return N > 0 && V > 0 && chunk_entries(N, V) ? (int64_t)N * WORK_WORDS * 8 : 0;
}

extern "C" int icrl_sample_tokens_filtered(const void* logits, int dtype, int64_t ld_logits, int N, int V,
                                           const double* uniforms, const float* temperature_rows, double temperature,
                                           const int32_t* top_k_rows, int top_k, const float* top_p_rows, double top_p,
                                           const float* min_p_rows, double min_p, int64_t* tokens_out,
                                           int64_t token_stride, float* log_prob, int64_t log_prob_stride, void* work,
                                           int64_t work_bytes, icrl_stream_t stream) {
    ICRL_REQUIRE(logits && uniforms && tokens_out && N > 0 && V > 0, "icrl_sample_tokens_filtered: null pointer or empty shape");
    ICRL_REQUIRE(ld_logits >= V, "icrl_sample_tokens_filtered: ld_logits < V");
    ICRL_REQUIRE(V <= MAX_V, "icrl_sample_tokens_filtered: vocabulary %d exceeds %d entries", V, MAX_V);
    ICRL_REQUIRE(temperature_rows || (temperature >= 0.0 && isfinite(temperature)), "icrl_sample_tokens_filtered: temperature must be finite and not negative");
    ICRL_REQUIRE(top_k_rows || top_k >= 0, "icrl_sample_tokens_filtered: top_k must not be negative (0: off)");
    ICRL_REQUIRE(top_p_rows || (top_p >= 0.0 && top_p <= 1.0), "icrl_sample_tokens_filtered: top_p must be in [0, 1]");
    ICRL_REQUIRE(min_p_rows || (min_p >= 0.0 && min_p <= 1.0), "icrl_sample_tokens_filtered: min_p must be in [0, 1]");
    ICRL_REQUIRE(!work || (reinterpret_cast<uintptr_t>(work) % 8 == 0 && work_bytes >= icrl_sample_filtered_work_bytes(N, V)),
                 "icrl_sample_tokens_filtered: work must be 8-byte aligned and hold icrl_sample_filtered_work_bytes(N, V) bytes");
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    const int S = std::min(51, 62 - bits);
    const Requests all{uniforms, {temperature_rows, temperature}, {top_p_rows, top_p}, {min_p_rows, min_p}, top_k_rows, top_k};
    const Results out{tokens_out, token_stride, log_prob, log_prob_stride};
    // settings given once for all rows may say that a list settles every row: no launches for what would be left
    const bool lists = (!top_k_rows && top_k > 0 && top_k < V) || (!temperature_rows && temperature == 0.0) ||
                       (!top_p_rows && top_p == 1.0 && !min_p_rows && min_p > 0.0);
    const int chunk = work && !lists ? chunk_entries(N, V) : 0;
    const Work split{chunk ? static_cast<u64*>(work) : nullptr};
    hipStream_t st = icrl::as_stream(stream);
#define ICRL_CALL(T, NT) \
    hipLaunchKernelGGL((sample_filtered_kernel<T, NT>), dim3(N), dim3(NT), 0, st, static_cast<const T*>(logits), ld_logits, V, S, all, out, split)
    // Two workgroups of 512 share a CU, one of 1024 has it to itself: wide ones pay where rows are long and there is a
    // CU for each of them, with more rows than CUs the narrow ones (333 rows of 50257, min-p 0.05: 34 against 56 us).
#define ICRL_WIDTHS(T)                                                                                                       \
    if (V <= 4096) { ICRL_CALL(T, 256); }                                                                                    \
    else if (V <= 16384 || N > 256) { ICRL_CALL(T, 512); }                                                                   \
    else { ICRL_CALL(T, 1024); }                                                                                             \
    if (chunk) {                                                                                                            \
        const dim3 grid((V + chunk - 1) / chunk, N);                                                                         \
        hipLaunchKernelGGL(sample_chunk_mass<T>, grid, dim3(CHUNK_NT), 0, st, static_cast<const T*>(logits), ld_logits, V, chunk, S, \
                           all, split);                                                                                      \
        hipLaunchKernelGGL(sample_chunk_draw<T>, grid, dim3(CHUNK_NT), 0, st, static_cast<const T*>(logits), ld_logits, V, chunk, S, \
                           all, out, split);                                                                                 \
    }
    switch (dtype) {
        case ICRL_F32: ICRL_WIDTHS(float); break;
        case ICRL_BF16: ICRL_WIDTHS(__bf16); break;
        case ICRL_F16: ICRL_WIDTHS(_Float16); break;
        default: icrl::set_error("icrl_sample_tokens_filtered: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
#undef ICRL_WIDTHS
#undef ICRL_CALL
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

extern "C" int icrl_topk_lse_rows(const void* logits, int dtype, int64_t ld_logits, int N, int V, int k, double temperature,
                                  float* values, int64_t* indices, float* lse, icrl_stream_t stream) {
    ICRL_REQUIRE(logits && values && indices && N > 0 && V > 0, "icrl_topk_lse_rows: null pointer or empty shape");
    ICRL_REQUIRE(ld_logits >= V, "icrl_topk_lse_rows: ld_logits < V");
    ICRL_REQUIRE(V <= MAX_V, "icrl_topk_lse_rows: vocabulary %d exceeds %d entries", V, MAX_V);
    ICRL_REQUIRE(k >= 1 && k <= V && k <= MAX_K, "icrl_topk_lse_rows: k must be in [1, min(%d, V)] (got %d)", MAX_K, k);
    ICRL_REQUIRE(temperature > 0.0 && isfinite(temperature), "icrl_topk_lse_rows: temperature must be positive and finite");
#define ICRL_CALL(T, NT, PLACE)                                                                                     \
    hipLaunchKernelGGL((topk_lse_kernel<T, NT, PLACE>), dim3(N), dim3(NT), 0, icrl::as_stream(stream),              \
                       static_cast<const T*>(logits), ld_logits, V, k, 1.0 / temperature, values, indices, lse)
    switch (dtype) {
        case ICRL_F32: ICRL_ROW_DISPATCH(float, V, k, ICRL_CALL); break;
        case ICRL_BF16: ICRL_ROW_DISPATCH(__bf16, V, k, ICRL_CALL); break;
        case ICRL_F16: ICRL_ROW_DISPATCH(_Float16, V, k, ICRL_CALL); break;
        default: icrl::set_error("icrl_topk_lse_rows: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
#undef ICRL_CALL
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

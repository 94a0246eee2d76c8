// Products of 8-bit operands (e4m3) with one power-of-two scale for each row and block of 128 along k, in two ways:
//
// 16-bit outputs run on the scaled matrix instruction v_mfma_scale_f32_32x32x64_f8f6f4, which multiplies each lane's 32
// products by the two scales (bytes holding the exponent + 127) as it adds them up: a scale costs no instruction.  It
// does not keep every bit: of each 8 products in a row it drops what lies more than 13 binary places below the largest
// one's 2^(exponent a + exponent b) (found with sums of one large and one small product), which leaves sums of random
// terms off by 8e-6 of their size - far below a 16-bit output's rounding, but not below float32's.
//
// float32 outputs therefore turn the codes, scale included, into bf16 (v_cvt_scalef32_pk_bf16_fp8: exact, four
// significant bits of eight) and multiply those at half the rate, with exact products and float32 sums (3e-8).
//
// Operands are cut once by icrl_cut_fp8 into the instruction's fragment order (rows and k padded with zeros), like
// icrl_cut_f16x2's: rows in blocks of 32, k in blocks of 64; a block is 2048 bytes, lane l = row % 32 + 32 (k % 64 / 32)
// holding 32 codes as two 16-byte halves, half h of all lanes before half h + 1.  Any 1 KB of it is one wave's 16-byte
// load, into registers or straight into LDS, and a fragment's reads from LDS have no bank conflicts.  Scales: one byte
// per row and block of 128; four blocks of a row to a 32-bit word, words of a 32-row block side by side.
#include <algorithm>
#include <type_traits>

#include "vocab_row.h"

namespace {
using namespace icrl;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int BLOCK = 128;
inline int blocks128(int K) { return (K + BLOCK - 1) / BLOCK; }
inline int scale_words(int K) { return (blocks128(K) + 3) / 4; }   // 32-bit words of scales per row

// scale = the smallest power of two 2^e with max |x| <= 448 2^e over a row's block of 128, code = x / scale rounded once.
// Bound by memory: 32000 x 2048 float32 98 us, 4096 x 2048 bf16 12-15 us; small operands by the launch (512 x 512: 2.6-4 us).
// Eight lanes cut one row's block of 128: 16 entries a lane, which are one 16-byte half of the fragment's lane.
template <typename T>
__global__ __launch_bounds__(64) void cut_kernel(const T* __restrict__ x, int64_t ld, int rows, int K, int nblocks, int words,
                                                  unsigned char* __restrict__ pieces, unsigned char* __restrict__ scales) {
    const int lane8 = threadIdx.x & 7;
    const int64_t unit = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 3);   // (row, group of four blocks' block)
    const int padded = words * 4;
    const int row = (int)(unit / padded), b = (int)(unit % padded);
    if (row >= (rows + 31) / 32 * 32) return;
    const int k0 = b * BLOCK + lane8 * 16;
    float v[16];
    unsigned top = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.f;
    if (row < rows && k0 < K) {
        const T* src = x + (int64_t)row * ld + k0;
        if (k0 + 16 <= K) {
            constexpr int VEC = Elem<T>::VEC;
#pragma unroll
            for (int q = 0; q < 16 / VEC; ++q) {
                typename Elem<T>::Raw raw[VEC];
                __builtin_memcpy(raw, src + q * VEC, 16);
#pragma unroll
                for (int j = 0; j < VEC; ++j) v[q * VEC + j] = Elem<T>::value(raw[j]);
            }
        } else {
            for (int j = 0; j < 16; ++j)
                if (k0 + j < K) v[j] = (float)src[j];
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) top = max(top, (unsigned)__shfl_xor((int)top, o, 64));
    // the smallest power of two 2^e with top <= 448 2^e (448 = 1.75 2^8 is the type's largest value)
    int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    e = top == 0 ? 0 : max(e, -127);
    const bool finite = top < 0x7F800000u;   // a block with an infinity or a NaN: the scale is NaN
    if (lane8 == 0) scales[(((int64_t)(row >> 5) * words + (b >> 2)) * 32 + (row & 31)) * 4 + (b & 3)] = finite ? (unsigned char)(e + 127) : 255;
    if (b >= nblocks) return;
    const float inv = finite ? ldexpf(1.f, -e) : 0.f;
    i32x4 out;
#pragma unroll
    for (int q = 0; q < 4; ++q) {   // exact scaling, then one rounding to nearest even
        int w = 0;
        w = __builtin_amdgcn_cvt_pk_fp8_f32(finite ? v[4 * q] * inv : 0.f, finite ? v[4 * q + 1] * inv : 0.f, w, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(finite ? v[4 * q + 2] * inv : 0.f, finite ? v[4 * q + 3] * inv : 0.f, w, true);
        out[q] = w;
    }
    const int kb = 2 * b + (lane8 >> 2), half = lane8 & 1, group = lane8 >> 1 & 1;
    unsigned char* dst = pieces + ((((int64_t)(row >> 5) * (2 * nblocks) + kb) * 2 + half) * 64 + (row & 31) + 32 * group) * 16;
    *reinterpret_cast<i32x4*>(dst) = out;
}

template <typename T>
__device__ __forceinline__ void store_out(T* p, float x) { *p = (T)x; }

struct Operand {
    const unsigned char* pieces;
    const unsigned* scales;
    int row_blocks;
};

__device__ __forceinline__ i32x8 join(i32x4 a, i32x4 b) {
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A lane's 32 codes of a block of 64, as the multiplication takes them, with their scale (its byte in the low 8 bits).
struct ScaledFragment {
    i32x8 codes;
    unsigned scale;
    ScaledFragment() = default;
    __device__ __forceinline__ ScaledFragment(i32x4 lo, i32x4 hi, unsigned s) : codes(join(lo, hi)), scale(s) {}
};
__device__ __forceinline__ void multiply(const ScaledFragment& a, const ScaledFragment& b, f32x16& acc) {
    acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a.codes, b.codes, acc, 0, 0, 0, (int)a.scale, 0, (int)b.scale);
}

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct ExactFragment {
    bf16x8 part[4];   // 8 codes each: which k they are does not matter as long as both operands agree
    ExactFragment() = default;
    __device__ __forceinline__ ExactFragment(i32x4 lo, i32x4 hi, unsigned s) {
        const unsigned byte = s & 255u;
        const float scale = __uint_as_float(byte == 255u ? 0x7FC00000u : byte << 23);
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                const unsigned codes = (unsigned)(q < 2 ? lo[2 * q + w] : hi[2 * q - 4 + w]);
                const bf16x2 l = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, false);
                const bf16x2 h = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(codes, scale, true);
                part[q][4 * w] = l[0]; part[q][4 * w + 1] = l[1];
                part[q][4 * w + 2] = h[0]; part[q][4 * w + 3] = h[1];
            }
    }
};
__device__ __forceinline__ void multiply(const ExactFragment& a, const ExactFragment& b, f32x16& acc) {
#pragma unroll
    for (int q = 0; q < 4; ++q) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.part[q], b.part[q], acc, 0, 0, 0);
}
template <typename T>
using Fragment = std::conditional_t<sizeof(T) == 4, ExactFragment, ScaledFragment>;

// ---- few rows: one 32 x 32 tile of the output per workgroup, k cut over its waves, fragments straight from memory
// Bound by the launch and one trip to memory: 1 x 10000 x 512 takes 3.7 us for 5 MB.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void gemm_fp8_rows(Operand a, Operand b, T* __restrict__ out, int64_t ldo, int M, int N,
                                                            int nblocks, int words, const float* __restrict__ bias) {
    __shared__ float part[WAVES][16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int rb_n = blockIdx.x, rb_m = blockIdx.y;
    const i32x4* pa = reinterpret_cast<const i32x4*>(a.pieces) + (int64_t)rb_m * nblocks * 256 + lane;
    const i32x4* pb = reinterpret_cast<const i32x4*>(b.pieces) + (int64_t)rb_n * nblocks * 256 + lane;
    const unsigned* sa = a.scales + (int64_t)rb_m * words * 32 + (lane & 31);
    const unsigned* sb = b.scales + (int64_t)rb_n * words * 32 + (lane & 31);
    f32x16 acc = {};
    for (int blk = wave; blk < nblocks; blk += WAVES) {
        i32x4 fa[4], fb[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) { fb[q] = pb[(int64_t)blk * 256 + q * 64]; fa[q] = pa[(int64_t)blk * 256 + q * 64]; }
        const unsigned ea = sa[(blk >> 2) * 32] >> (8 * (blk & 3)), eb = sb[(blk >> 2) * 32] >> (8 * (blk & 3));
#pragma unroll
        for (int q = 0; q < 2; ++q)
            multiply(Fragment<T>(fa[2 * q], fa[2 * q + 1], ea), Fragment<T>(fb[2 * q], fb[2 * q + 1], eb), acc);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) part[wave][i][lane] = acc[i];
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += WAVES * 64) {
        const int i = e >> 6, l = e & 63;
        const int m = rb_m * 32 + 8 * (i >> 2) + 4 * (l >> 5) + (i & 3), n = rb_n * 32 + (l & 31);
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += part[w][i][l];
        if (m < M && n < N) store_out(out + (int64_t)m * ldo + n, s + (bias ? bias[n] : 0.f));
    }
}

// ---- tiles of (64 WM) x (64 WN) per workgroup of 2 x 2 waves
// Operands are staged through LDS 64 of k at a time in four buffers, copied there without passing registers: three stages
// (of 1024 clocks of matrix instructions on 256 x 256 tiles) are in flight while one is multiplied, which covers the
// latency of the caches behind the L2.  The fragments of the next stage are read from LDS into registers while the
// current ones are multiplied, so one wave per SIMD keeps the matrix cores busy.
// Measured: 4096 x 32000 x 2048 into bf16 324 us, 1650 TFLOP/s (a library product of 8192 cubed reaches 2740): the matrix
// cores are busy 36% of the CUs' time, and a quarter of a wave's is spent in waits.  512 x 10000 x 512 into float32 13.5 us,
// of which 20 MB of output take 3 and bf16's rate 4: workgroups of eight stages, bound by their beginnings and ends.
template <typename T, int WM, int WN>
__global__ __launch_bounds__(256) void gemm_fp8_tiles(Operand a, Operand b, T* __restrict__ out, int64_t ldo, int M, int N,
                                                      int nblocks, int words, const float* __restrict__ bias, int tiles_m,
                                                      int tiles_n) {
    constexpr int RA = 2 * WM, RB = 2 * WN;                 // 32-row blocks per tile
    constexpr int STAGE = (RA + RB) * 2048, DEPTH = 4;      // bytes of one stage of 64; buffers
    constexpr int COPIES = (RA + RB) / 2;                   // 16-byte copies per thread and stage
    constexpr bool WIDE = sizeof(T) == 2;                   // the products' tiles are transposed (see the end)
    constexpr int SCALE_WAVES = (RA + RB + 7) / 8;           // waves that copy scales
    constexpr int BUFFERS = DEPTH * STAGE, SCALES = SCALE_WAVES * 1024;   // scales: a word per row for 512 of k, in two buffers
    __shared__ __attribute__((aligned(16))) unsigned char lds[BUFFERS + 2 * SCALES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
    // workgroups go round the 8 XCDs: give each XCD a contiguous run of tiles, in bands of 8 tile rows, so that what
    // its L2 holds is shared by the tiles it works on
    const int total = tiles_m * tiles_n;
    int t = blockIdx.x;
    {
        const int per = total / 8, extra = total % 8, xcd = t % 8, at = t / 8;
        t = xcd * per + min(xcd, extra) + at;
    }
    const int band = t / (8 * tiles_n), in_band = t % (8 * tiles_n), rows_in_band = min(8, tiles_m - 8 * band);
    const int tm = 8 * band + in_band % rows_in_band, tn = in_band / rows_in_band;
    // a stage is RA + RB pieces of 2 KB; wave w copies the (w & 1)-th KB of every second piece
    const unsigned char* from[COPIES];
#pragma unroll
    for (int q = 0; q < COPIES; ++q) {
        const int piece = 2 * q + (wave >> 1);
        const bool is_a = piece < RA;
        const Operand& o = is_a ? a : b;
        const int rb = min(is_a ? tm * RA + piece : tn * RB + (piece - RA), o.row_blocks - 1);   // past the end: any rows, never stored
        from[q] = o.pieces + (int64_t)rb * nblocks * 4096 + (wave & 1) * 1024 + lane * 16;
    }
    const int stages = 2 * nblocks;
    auto stage = [&](int s) {
        unsigned char* base = lds + (s % DEPTH) * STAGE + (wave >> 1) * 2048 + (wave & 1) * 1024;
#pragma unroll
        for (int q = 0; q < COPIES; ++q)
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const __attribute__((address_space(1))) unsigned*>(reinterpret_cast<uintptr_t>(from[q] + (int64_t)s * 2048)),
                (__attribute__((address_space(3))) unsigned*)(base + q * 4096), 16, 0, 0);
    };
    // scale words of one 512 of k: 128 bytes a row block, eight row blocks a wave
    const unsigned char* scales_from;
    {
        const int piece = min(8 * wave + lane / 8, RA + RB - 1);
        const bool is_a = piece < RA;
        const Operand& o = is_a ? a : b;
        const int rb = min(is_a ? tm * RA + piece : tn * RB + (piece - RA), o.row_blocks - 1);
        scales_from = reinterpret_cast<const unsigned char*>(o.scales) + (int64_t)rb * words * 128 + (lane & 7) * 16;
    }
    auto stage_scales = [&](int word) {
        if (wave < SCALE_WAVES)
            __builtin_amdgcn_global_load_lds(
                reinterpret_cast<const __attribute__((address_space(1))) unsigned*>(reinterpret_cast<uintptr_t>(scales_from + (int64_t)word * 128)),
                (__attribute__((address_space(3))) unsigned*)(lds + BUFFERS + (word & 1) * SCALES + wave * 1024), 16, 0, 0);
    };
    f32x16 acc[WM][WN] = {};
    struct Raw { i32x4 a[WM][2], b[WN][2]; } raw[2];
    auto fetch = [&](int s, Raw& r) {
        const unsigned char* base = lds + (s % DEPTH) * STAGE + lane * 16;
#pragma unroll
        for (int i = 0; i < WM; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) r.a[i][h] = *reinterpret_cast<const i32x4*>(base + (wm * WM + i) * 2048 + h * 1024);
#pragma unroll
        for (int i = 0; i < WN; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h) r.b[i][h] = *reinterpret_cast<const i32x4*>(base + (RA + wn * WN + i) * 2048 + h * 1024);
    };
    unsigned ea[WM], eb[WN];
    // this wave's copies up to a stage have landed (all but the `later` newest stages' copies; scales among them only make
    // it wait for more), its reads too, and then everyone's
    auto landed = [&](int later) {
        if (later >= 2) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(2 * COPIES) : "memory");
        else if (later == 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"i"(COPIES) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        asm volatile("s_barrier" ::: "memory");
    };
    stage_scales(0);
    for (int s = 0; s < DEPTH - 1 && s < stages; ++s) stage(s);
    landed(min(DEPTH - 2, stages - 1));
    fetch(0, raw[0]);
    auto step = [&](int s, const Raw& now, Raw& then) {
        if ((s & 7) == 0) {
            const unsigned* e = reinterpret_cast<const unsigned*>(lds + BUFFERS + (s >> 3 & 1) * SCALES) + (lane & 31);
#pragma unroll
            for (int i = 0; i < WM; ++i) ea[i] = e[(wm * WM + i) * 32];
#pragma unroll
            for (int i = 0; i < WN; ++i) eb[i] = e[(RA + wn * WN + i) * 32];
        }
        if (s + 1 < stages) {
            landed(min(DEPTH - 3, stages - 2 - s));   // stages s + 2 .. are newer than s + 1
            // the buffer of stage s + DEPTH - 1 held stage s - 1, and the next scales' buffer the words before these: every wave
            // had read them before this barrier
            if (s + DEPTH - 1 < stages) stage(s + DEPTH - 1);
            if ((s & 7) == 1 && s + 7 < stages) stage_scales((s >> 3) + 1);
            fetch(s + 1, then);
        }
        Fragment<T> fb[WN];
#pragma unroll
        for (int j = 0; j < WN; ++j) fb[j] = Fragment<T>(now.b[j][0], now.b[j][1], eb[j]);
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const Fragment<T> fa(now.a[i][0], now.a[i][1], ea[i]);
#pragma unroll
            for (int j = 0; j < WN; ++j) {
                if (WIDE) multiply(fb[j], fa, acc[i][j]);
                else multiply(fa, fb[j], acc[i][j]);
            }
        }
        if (s & 1) {   // the next block of 128: the next byte of the words
#pragma unroll
            for (int i = 0; i < WM; ++i) ea[i] >>= 8;
#pragma unroll
            for (int i = 0; i < WN; ++i) eb[i] >>= 8;
        }
    };
    for (int s = 0; s < stages; s += 2) {   // stages come in pairs: k is padded to 128
        step(s, raw[0], raw[1]);
        step(s + 1, raw[1], raw[0]);
    }
    if constexpr (WIDE) {
        // 16-bit outputs: a lane holds four neighbouring columns of a row at a time (the transposed product's rows), which
        // go through LDS, so that a store writes 16 bytes a lane and whole lines of a row; one by one they would be written
        // in 64-byte pieces (4096 x 32000 x 2048: 356 us so, 330 through LDS).  Rows are 8 bytes apart from a multiple of
        // the banks.
        constexpr int COLS = 32 * WN, PITCH = COLS * 2 + 8;
        static_assert(4 * 32 * WM * PITCH <= (int)sizeof(lds), "the waves' tiles fit the stages' place");
        unsigned char* mine = lds + wave * (32 * WM * PITCH);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();   // every wave has read its last stage
#pragma unroll
        for (int j = 0; j < WN; ++j) {
            float add[4][4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = (tn * RB + wn * WN + j) * 32 + 8 * q + 4 * (lane >> 5) + e;
                    add[q][e] = bias && n < N ? bias[n] : 0.f;
                }
#pragma unroll
            for (int i = 0; i < WM; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    struct alignas(8) Four { T e[4]; } four;
#pragma unroll
                    for (int e = 0; e < 4; ++e) four.e[e] = (T)(acc[i][j][4 * q + e] + add[q][e]);
                    *reinterpret_cast<Four*>(mine + (32 * i + (lane & 31)) * PITCH + (32 * j + 8 * q + 4 * (lane >> 5)) * 2) = four;
                }
        }
        // (a wave reads back its own tile only: no barrier)
        constexpr int PER_ROW = COLS / 8, ROWS = 64 / PER_ROW;   // lanes per row, rows per store
        const int m0 = (tm * RA + wm * WM) * 32, n0 = (tn * RB + wn * WN) * 32 + lane % PER_ROW * 8;
        typedef unsigned Words __attribute__((ext_vector_type(4), aligned(2), may_alias));
        typedef unsigned Pair __attribute__((ext_vector_type(2), may_alias));
#pragma unroll 4
        for (int row = lane / PER_ROW; row < 32 * WM; row += ROWS) {
            const Pair* from = reinterpret_cast<const Pair*>(mine + row * PITCH + lane % PER_ROW * 16);
            const Pair lo = from[0], hi = from[1];
            Words w = {lo[0], lo[1], hi[0], hi[1]};
            T* to = out + (int64_t)(m0 + row) * ldo + n0;
            if (m0 + row < M) {
                if (n0 + 8 <= N) {
                    *reinterpret_cast<Words*>(to) = w;
                } else {
                    struct Eight { T e[8]; };
                    const Eight v = __builtin_bit_cast(Eight, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (n0 + e < N) to[e] = v.e[e];
                }
            }
        }
        return;
    }
    // float32 outputs: a lane holds 16 rows of one column of each 32 x 32 tile: a store writes two whole lines
#pragma unroll
    for (int j = 0; j < WN; ++j) {
        const int n = (tn * RB + wn * WN + j) * 32 + (lane & 31);
        if (n >= N) continue;
        const float add = bias ? bias[n] : 0.f;
#pragma unroll
        for (int i = 0; i < WM; ++i) {
            const int m0 = (tm * RA + wm * WM + i) * 32, mine = m0 + 4 * (lane >> 5);
            T* p = out + (int64_t)mine * ldo + n;
            if (m0 + 32 <= M) {
#pragma unroll
                for (int q = 0; q < 16; ++q) store_out(p + (8 * (q >> 2) + (q & 3)) * ldo, acc[i][j][q] + add);
            } else {
#pragma unroll
                for (int q = 0; q < 16; ++q) {
                    const int d = 8 * (q >> 2) + (q & 3);
                    if (mine + d < M) store_out(p + d * ldo, acc[i][j][q] + add);
                }
            }
        }
    }
}
}  // namespace

extern "C" int64_t icrl_fp8_piece_bytes(int rows, int K) {
    return rows > 0 && K > 0 ? (int64_t)((rows + 31) / 32 * 32) * blocks128(K) * BLOCK : 0;
}
extern "C" int64_t icrl_fp8_scale_bytes(int rows, int K) {
    return rows > 0 && K > 0 ? (int64_t)((rows + 31) / 32 * 32) * scale_words(K) * 4 : 0;
}

extern "C" int icrl_cut_fp8(const void* x, int dtype, int64_t ld, int rows, int K, void* pieces, void* scales, icrl_stream_t stream) {
    ICRL_REQUIRE(x && pieces && scales && rows > 0 && K > 0, "icrl_cut_fp8: null pointer or empty shape");
    ICRL_REQUIRE(ld >= K, "icrl_cut_fp8: row stride < K");
    ICRL_REQUIRE(reinterpret_cast<uintptr_t>(pieces) % 16 == 0 && reinterpret_cast<uintptr_t>(scales) % 4 == 0,
                 "icrl_cut_fp8: pieces must be 16-byte aligned, scales 4-byte");
    const int words = scale_words(K), nb = blocks128(K);
    const int64_t units = (int64_t)((rows + 31) / 32 * 32) * words * 4, grid = units / 8;
    ICRL_REQUIRE(grid <= 0x7FFFFFFF, "icrl_cut_fp8: operand too large");
#define ICRL_CALL(T)                                                                                              \
    hipLaunchKernelGGL((cut_kernel<T>), dim3((unsigned)grid), dim3(64), 0, icrl::as_stream(stream),               \
                       static_cast<const T*>(x), ld, rows, K, nb, words, static_cast<unsigned char*>(pieces),     \
                       static_cast<unsigned char*>(scales))
    switch (dtype) {
        case ICRL_F32: ICRL_CALL(float); break;
        case ICRL_BF16: ICRL_CALL(__bf16); break;
        case ICRL_F16: ICRL_CALL(_Float16); break;
        default: icrl::set_error("icrl_cut_fp8: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
#undef ICRL_CALL
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

namespace {
template <typename T>
void launch_gemm(const Operand& a, const Operand& b, T* out, int64_t ldo, int M, int N, int K, const float* bias, hipStream_t st) {
    const int nb = blocks128(K), words = scale_words(K);
    if (M <= 64) {
        hipLaunchKernelGGL((gemm_fp8_rows<T, 4>), dim3(b.row_blocks, a.row_blocks), dim3(256), 0, st, a, b, out, ldo, M, N, nb,
                           words, bias);
        return;
    }
#define ICRL_TILES(WM, WN)                                                                                                     \
    do {                                                                                                                       \
        const int tm = (M + 64 * WM - 1) / (64 * WM), tn = (N + 64 * WN - 1) / (64 * WN);                                      \
        hipLaunchKernelGGL((gemm_fp8_tiles<T, WM, WN>), dim3(tm * tn), dim3(256), 0, st, a, b, out, ldo, M, N, nb, words, bias, \
                           tm, tn);                                                                                            \
    } while (0)
    // Measured (us; 256 x 256, 128 x 128 and 64 x 128 tiles): 4096 x 32000 x 2048 330 / 340 / 380, the same at k = 128
    // 98 / 86 / 89, 2048 x 10000 x 2048 80 / 57 / 65, 512 x 10000 x 512 (float32 out) 23 / 13.5 / 12, 1024 x 4096 x 4096
    // 69 / 32 / 30.  The largest tiles have one workgroup per CU and need many rounds of a long k to make up for their
    // ends; the smallest ones spread better when there are fewer than three of the middle ones per CU.
    const int64_t tiles256 = (int64_t)((M + 255) / 256) * ((N + 255) / 256), tiles128 = (int64_t)((M + 127) / 128) * ((N + 127) / 128);
    if (tiles256 >= 1024 && K >= 2048) ICRL_TILES(4, 4);
    else if (tiles128 >= 768) ICRL_TILES(2, 2);
    else ICRL_TILES(1, 2);
#undef ICRL_TILES
}
}  // namespace

extern "C" int icrl_gemm_fp8(const void* a_pieces, const void* a_scales, const void* b_pieces, const void* b_scales, void* C,
                             int dtype, int64_t ldc, int M, int N, int K, const float* bias, icrl_stream_t stream) {
    ICRL_REQUIRE(a_pieces && a_scales && b_pieces && b_scales && C && M > 0 && N > 0 && K > 0, "icrl_gemm_fp8: null operand or empty shape");
    ICRL_REQUIRE(ldc >= N, "icrl_gemm_fp8: leading dimension ldc < N");
    ICRL_REQUIRE((reinterpret_cast<uintptr_t>(a_pieces) | reinterpret_cast<uintptr_t>(b_pieces)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) % 4 == 0,
                 "icrl_gemm_fp8: pieces must be 16-byte aligned, scales 4-byte");
    ICRL_REQUIRE((int64_t)((M + 127) / 128) * ((N + 127) / 128) <= 0x7FFFFFFF, "icrl_gemm_fp8: output too large");
    const Operand a{static_cast<const unsigned char*>(a_pieces), static_cast<const unsigned*>(a_scales), (M + 31) / 32};
    const Operand b{static_cast<const unsigned char*>(b_pieces), static_cast<const unsigned*>(b_scales), (N + 31) / 32};
    hipStream_t st = icrl::as_stream(stream);
    switch (dtype) {
        case ICRL_F32: launch_gemm(a, b, static_cast<float*>(C), ldc, M, N, K, bias, st); break;
        case ICRL_BF16: launch_gemm(a, b, static_cast<__bf16*>(C), ldc, M, N, K, bias, st); break;
        case ICRL_F16: launch_gemm(a, b, static_cast<_Float16*>(C), ldc, M, N, K, bias, st); break;
        default: icrl::set_error("icrl_gemm_fp8: unknown dtype %d", dtype); return ICRL_ERR_ARG;
    }
    ICRL_LAUNCH_CHECK();
    return ICRL_OK;
}

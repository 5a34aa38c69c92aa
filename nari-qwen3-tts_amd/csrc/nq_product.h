// Products of rows, out = residual + act(x w^T * scales + bias), for operands of 8-bit integers or bf16: the kernels that
// nq_int8.hip and nq_linear_act.hip instantiate.  Both types meet the matrix units in the same bytes: an operand of
// 32 rows is 32 bytes of K (32 integers, 16 bf16), one of 16 rows 64 bytes, 16 bytes a lane.
//
// Few rows: a workgroup owns 16 output channels and all of K, its waves interleave K in
// pieces of 128 bytes, each through LDS of its own, and add their sums at the end, in the order of the waves.
// Many rows: (32 TM WM) x (32 TN WN) tiles, K staged 128 bytes at a
// time through three or four LDS buffers, the next stages' loads in flight.
#pragma once

#include <type_traits>

#include "nq_common.h"
#include "nq_internal.h"

namespace nq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

struct ProductArgs {
    const char *x;
    int64_t x_s0;  // row strides of the operands and K in bytes
    const float *sx;
    const char *w;
    int64_t w_s0;
    const float *sw;
    int M, N, K;
    uint16_t *out;
    int64_t o_s0;
    int wide;  // out rows take 16-byte stores, residual's 16-byte loads
    const uint16_t *bias;  // the epilogue's: null where there is none
    const uint16_t *residual;
    int64_t r_s0;
    int act;
};

// |sum| <= 2^31, so that sum * sx stays inside fp32 up to sx = 2^96; a larger sx comes last, when a model's weights have
// made sum * sw small enough for the result, where that fits.
__device__ __forceinline__ float scaled(int sum, float sx, float sw) {
    const bool far = sx > 0x1p96f;
    return static_cast<float>(sum) * (far ? sw : sx) * (far ? sx : sw);
}

struct Int8Op {
    typedef i32x4 Acc4;
    typedef i32x16 Acc16;
    static constexpr bool kScales = true;
    static __device__ __forceinline__ Acc4 mfma(i32x4 a, i32x4 b, Acc4 c) {
        return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ Acc16 mfma(i32x4 a, i32x4 b, Acc16 c) {
        return __builtin_amdgcn_mfma_i32_32x32x32_i8(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float value(int sum, float sx, float sw) { return scaled(sum, sx, sw); }
};

struct Bf16Op {
    typedef f32x4 Acc4;
    typedef f32x16 Acc16;
    static constexpr bool kScales = false;
    static __device__ __forceinline__ Acc4 mfma(i32x4 a, i32x4 b, Acc4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ Acc16 mfma(i32x4 a, i32x4 b, Acc16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    static __device__ __forceinline__ float value(float sum, float, float) { return sum; }
};

// The activations in fp32, by the hardware's exponential and reciprocal (an ulp each); the bf16 result's half step is far
// above their roundings.  y / (1 + exp(-z)) with z = y (silu) or 2 sqrt(2 / pi) (y + 0.044715 y^3) (gelu_tanh, since (1 + tanh(z /
// 2)) / 2 is that factor); at the ends the exponential is infinite or 0.  gelu is max(y, 0) - |y| erfc(|y| / sqrt 2) / 2, which
// does not cancel in its tail as 1 + erf would: erfc(a) = k 2^(q(k) - a^2 log2 e) with k = 1 / (1 + 0.3 a), and q a polynomial
// fitted to log2(erfc(a) exp(a^2) / k) at Chebyshev nodes for a up to 10.5, 8e-7 off there; behind it the exponential is 0, and k is
// not: |y| is held to 16 on the positive side, so that plus infinity stays.  Minus infinity times 0 is NaN, as in the formulas of
// the three.
template <int kAct>
__device__ __forceinline__ float activate(float y) {
    if constexpr (kAct == NQ_ACT_RELU) return y < 0.f ? 0.f : y;
    if constexpr (kAct == NQ_ACT_SILU) return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * y));
    if constexpr (kAct == NQ_ACT_GELU_TANH) {
        const float z = y * fmaf(-0.10294324f, y * y, -2.3022082f);  // -2 sqrt(2 / pi) log2 e (0.044715 y^3 + y)
        return y * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z));
    }
    if constexpr (kAct == NQ_ACT_GELU) {
        const float m = fabsf(fminf(y, 16.0f)), k = __builtin_amdgcn_rcpf(fmaf(0.21213203f, m, 1.0f));
        float q = fmaf(0.6919735f, k, -2.821275f);
        q = fmaf(q, k, 4.1087608f);
        q = fmaf(q, k, -2.9656343f);
        q = fmaf(q, k, 1.7799832f);
        q = fmaf(q, k, 0.27396405f);
        q = fmaf(q, k, 1.4983267f);
        q = fmaf(q, k, -2.5660994f);
        return fmaf(-0.5f * m * k, __builtin_amdgcn_exp2f(fmaf(-0.72134752f * y, y, q)), y < 0.f ? 0.f : y);  // NaN stays
    }
    return y;
}

// N values' activation
template <int N>
__device__ __forceinline__ void activate_all(float (&v)[N], int act) {
    switch (act) {  // once for all of them: straight code for every one costs its fetch
        case NQ_ACT_RELU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = activate<NQ_ACT_RELU>(v[e]);
            break;
        case NQ_ACT_GELU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = activate<NQ_ACT_GELU>(v[e]);
            break;
        case NQ_ACT_GELU_TANH:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = activate<NQ_ACT_GELU_TANH>(v[e]);
            break;
        case NQ_ACT_SILU:
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] = activate<NQ_ACT_SILU>(v[e]);
            break;
        default: break;
    }
}

constexpr int kBand = 8;            // tiles in m of a band
constexpr int kStage = 128;         // bytes of K a stage
constexpr int kChunks = kStage / 16;

// LDS place of 16-byte chunk c of row r: measured free of conflicts for the operand reads (32 rows and two chunks, 16
// rows and four) and for the writes (eight rows).
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kChunks + (c ^ ((r >> 1) & 7)); }

__device__ const i32x4 kZero16 = {0, 0, 0, 0};  // what a chunk behind K is read from

// Waits until at most N of the wave's loads are under way (and all its LDS reads are back), then the barrier: what those
// loads wrote to LDS is there for every wave, and what they read there may be overwritten.
constexpr int wait_for(int vm, int lgkm) { return (vm & 15) | (vm >> 4) << 14 | 7 << 4 | lgkm << 8; }  // s_waitcnt's operand
template <int N>
__device__ __forceinline__ void arrive() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(wait_for(N, 0));
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 16 MT rows of x against 16 weight rows, the waves splitting K: wave w takes the 128-byte pieces w, w + kRowWaves, ..,
// each into one of its own two LDS buffers, and the eight sums meet in LDS at the end; nobody waits for another wave
// before that.  The loads write LDS themselves, eight lanes a row, so that each covers whole lines: operands loaded straight
// into registers have neighbouring lanes in different rows, four times the line look-ups, and took 16.1 us instead of
// 6.5 at 64 x 2048 (K 6144).  Two buffers of eight waves against one of sixteen and three of eight: 5.9, 6.6 and 6.4 us
// at 32 rows of that product.
constexpr int kRowWaves = 8;

template <typename Op, bool kEpi, int MT>
__global__ void __launch_bounds__(kRowWaves * kWave)
product_rows_kernel(ProductArgs a) {
    constexpr int NW = kRowWaves, V = 2 * (MT + 1);  // loads of 1 KB (eight rows) a piece: the weights', then x's
    constexpr int kBuf = 1024 * V;
    constexpr int kPart = MT * 256;  // sums of a wave
    static_assert(kPart * 4 <= 2 * kBuf, "the sums fit where the operands were");
    __shared__ __attribute__((aligned(16))) char lds[NW * 2 * kBuf];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    // load v writes rows 8 v .. + 7 of a piece, lane l place l % 8 of row l / 8
    const char *from[V];
    int col[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool x = v >= 2;
        const int rr = 8 * (x ? v - 2 : v) + lane / 8, g = (x ? m0 : n0) + rr, n = x ? a.M : a.N;
        col[v] = wave * kStage + 16 * ((lane & 7) ^ ((rr >> 1) & 7));
        from[v] = (x ? a.x : a.w) + (g < n ? g : n - 1) * (x ? a.x_s0 : a.w_s0) + col[v];
    }
    char *mine = lds + wave * 2 * kBuf;
    auto load = [&](int piece, int buf) __attribute__((always_inline)) {
        const int at = piece * NW * kStage;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const char *p = at + col[v] < a.K ? from[v] + at : reinterpret_cast<const char *>(&kZero16);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)p,
                (__attribute__((address_space(3))) void *)(mine + buf * kBuf + 1024 * v), 16, 0, 0);
        }
    };
    // operand h: lane l holds row l % 16, bytes 64 h + 16 (l / 16) .. + 15 of the piece, the same order in both
    int get[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) get[h] = 16 * chunk_at(lane & 15, 4 * h + (lane >> 4));
    typename Op::Acc4 acc[MT] = {};
    const int pieces = (a.K + NW * kStage - 1) / (NW * kStage);
    load(0, 0);
    load(1, 1);
    for (int p = 0; p < pieces; p += 2) {
#pragma unroll
        for (int d = 0; d < 2; ++d) {  // pieces behind the last read zeros, so that the waits can count
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(V) : "memory");
            i32x4 w[2], x[2][MT];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char *src = mine + d * kBuf + get[h];
                w[h] = *reinterpret_cast<const i32x4 *>(src);
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    x[h][m] = *reinterpret_cast<const i32x4 *>(src + 2048 * (m + 1));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // read before the buffer is written again
            load(p + d + 2, d);
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int m = 0; m < MT; ++m)
                    acc[m] = Op::mfma(w[h], x[h][m], acc[m]);
        }
    }
    arrive<0>();  // every wave's loads and reads are done
    typedef typename std::remove_reference<decltype(acc[0][0])>::type Sum;
    Sum *part = reinterpret_cast<Sum *>(lds);
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<typename Op::Acc4 *>(part + wave * kPart + m * 256 + lane * 4) = acc[m];
    __syncthreads();
    // element e of tile m: lane e / 4, weight row 4 (lane / 16) + e % 4, x row lane % 16; threads along weight rows
    for (int i = threadIdx.x; i < kPart; i += NW * kWave) {
        const int m = i / 256, row = (i & 255) >> 4, n = i & 15;
        const int e = m * 256 + ((n >> 2) * 16 + row) * 4 + (n & 3);
        Sum sum = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += part[w * kPart + e];
        const int r = m0 + 16 * m + row;
        if (r >= a.M || n0 + n >= a.N) continue;
        float v = Op::kScales ? Op::value(sum, a.sx[r], a.sw[n0 + n]) : Op::value(sum, 0.f, 0.f);
        if constexpr (kEpi) {
            if (a.bias) v += bf16_to_f32(a.bias[n0 + n]);
            float one[1] = {v};
            activate_all(one, a.act);
            v = one[0];
            if (a.residual) v += bf16_to_f32(a.residual[r * a.r_s0 + n0 + n]);
        }
        a.out[r * a.o_s0 + n0 + n] = f32_to_bf16(v);
    }
}

// WM x WN waves, each TM x TN parts of 32 x 32.  K goes through NB LDS buffers, 128 bytes a stage, written by the
// loads themselves (a register on the way would cost its write to LDS: 0.14 us a stage of 128 x 256).  Step k: stage k
// has arrived, the loads of stage k + NB - 1 are issued; the operands of each 32 bytes are read while the MFMAs of the 32
// before run, also across the barrier.  The results cross LDS once more, so that they leave in whole lines.
// 4001 x 2048 (K 6144) bf16 94 us = 1070 TFLOP/s, int8 55.5 us = 1810 TOP/s; 4096^3 124 us = 1105 TFLOP/s and 73 us = 1880
// TOP/s (a library's bf16: 86 and 92 us).  No unit is full: the MFMAs run in half of the clocks, of the eight waves of a
// CU's one workgroup (its buffers take the LDS) two share a matrix unit and all meet at every stage's barrier.  Without the
// stages' loads it would be 84 us at 4096^3, with loads of one and the same cached tile 119: their way into LDS beside the
// operand reads costs, not the memory behind them.  Waiting for operands before the next are asked for gave 7 %, bands of
// tiles 3 %, an MFMA ahead of the reads and the loads between MFMAs 6 %.  Other tiles and depths at 4096^3, us: 256 x 256 in
// two buffers 118, but 137 where that leaves CUs idle (4001 x 2048); in four buffers of 64 bytes 124; four waves 129 to 150; waves
// in two groups, one reading operands while the other multiplies, 129.
template <typename Op, bool kEpi, int WM, int WN, int TM, int TN, int NB>
__global__ void __launch_bounds__(WM * WN * kWave)
product_tile_kernel(ProductArgs a, int tiles_m, int tiles_n) {
    constexpr int NW = WM * WN, T = NW * kWave, BM = 32 * TM * WM, BN = 32 * TN * WN;
    constexpr int V = (BM + BN) / 8 / NW;  // loads of 1 KB (eight rows) a wave and stage
    constexpr int STEPS = kStage / 32;
    static_assert(V * NW * 8 == BM + BN && STEPS == 4, "a stage splits evenly over the waves");
    constexpr int kBuf = (BM + BN) * kStage;     // bytes of a stage: weights, then x
    constexpr int kOutPitch = BN * (kEpi ? 4 : 2) + 16;  // bytes of a result row, fp32 where a residual may follow
    constexpr int kOut = BM * kOutPitch;
    constexpr int kScales = NB * kBuf > kOut ? NB * kBuf : kOut;  // behind the buffers: the tile's scales, there when the sums are
    // one array: with a second one the compiler waits for every load in flight before it reads LDS (57 us become 87)
    __shared__ __attribute__((aligned(16))) char lds[kScales + 4 * (BM + 2 * BN)];
    float *const s_w = reinterpret_cast<float *>(lds + kScales), *const s_x = s_w + BN, *const s_b = s_x + BM;
    // XCD b % 8 takes tiles (b % 8) per .., in bands of kBand tiles in m: those under way at a time share rows and weights in
    // one L2
    const int tiles = tiles_m * tiles_n, per = (tiles + 7) / 8;
    const int t = static_cast<int>(blockIdx.x % 8) * per + static_cast<int>(blockIdx.x / 8);
    if (t >= tiles) return;
    const int band = t / (kBand * tiles_n), high = min(kBand, tiles_m - band * kBand), inside = t - band * kBand * tiles_n;
    const int m0 = (band * kBand + inside % high) * BM, n0 = inside / high * BN;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r32 = lane & 31, half = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;
    if constexpr (Op::kScales) {
        for (int i = threadIdx.x; i < BN; i += T) s_w[i] = n0 + i < a.N ? a.sw[n0 + i] : 0.f;
        for (int i = threadIdx.x; i < BM; i += T) s_x[i] = m0 + i < a.M ? a.sx[m0 + i] : 0.f;
    }
    if constexpr (kEpi) {
        // without a bias -0, which changes no value: with 0 a -0 would lose its sign here and not where rows are few
        for (int i = threadIdx.x; i < BN; i += T) s_b[i] = a.bias && n0 + i < a.N ? bf16_to_f32(a.bias[n0 + i]) : -0.f;
    }

    // load v writes rows 8 (wave V + v) .. + 7 of a stage, lane l place l % 8 of row l / 8
    const char *from[V];
    int col[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int r = 8 * (wave * V + v) + lane / 8;
        const bool x = r >= BN;
        const int rr = x ? r - BN : r, g = (x ? m0 : n0) + rr, n = x ? a.M : a.N;
        col[v] = 16 * ((lane & 7) ^ ((rr >> 1) & 7));
        from[v] = (x ? a.x : a.w) + (g < n ? g : n - 1) * (x ? a.x_s0 : a.w_s0) + col[v];
    }
    int get[STEPS];  // chunk 2 j + half of row r32: the parts are constants away (32 rows keep the exclusive-or)
#pragma unroll
    for (int j = 0; j < STEPS; ++j) get[j] = 16 * chunk_at(r32, 2 * j + half);
    const int w_part = wn * TN * 32 * kStage, x_part = BN * kStage + wm * TM * 32 * kStage;

    typename Op::Acc16 acc[TM][TN] = {};

    const int stages = (a.K + kStage - 1) / kStage;
    auto load = [&](auto whole, int k, int buf, int v) __attribute__((always_inline)) {
        const char *p = from[v];
        if constexpr (!whole) p = k * kStage + col[v] < a.K ? p : reinterpret_cast<const char *>(&kZero16);
        from[v] += kStage;
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void *)p,
            (__attribute__((address_space(3))) void *)(lds + buf + 1024 * (wave * V + v)), 16, 0, 0);
    };
    i32x4 wf[2][TN], xf[2][TM];
    auto read = [&](int buf, int j) __attribute__((always_inline)) {
#pragma unroll
        for (int n = 0; n < TN; ++n)
            wf[j & 1][n] = *reinterpret_cast<const i32x4 *>(lds + buf + w_part + get[j] + n * 32 * kStage);
#pragma unroll
        for (int m = 0; m < TM; ++m)
            xf[j & 1][m] = *reinterpret_cast<const i32x4 *>(lds + buf + x_part + get[j] + m * 32 * kStage);
    };
    auto multiply = [&](int j) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < TM; ++m)
#pragma unroll
            for (int n = 0; n < TN; ++n)
                acc[m][n] = Op::mfma(wf[j & 1][n], xf[j & 1][m], acc[m][n]);
    };
    int b0 = 0, bl = (NB - 1) * kBuf;      // the buffers of stage k and of stage k + NB - 1, whose loads step k issues
    constexpr std::true_type whole{};      // stages inside K: no look at the chunks, 14 vector instructions instead of 40
    constexpr std::false_type part{};
#pragma unroll
    for (int i = 0; i < NB - 1; ++i)
#pragma unroll
        for (int v = 0; v < V; ++v) load(part, i, i * kBuf, v);
    auto step = [&](auto next, int k) __attribute__((always_inline)) {
        arrive<(NB - 2) * V>();  // stage k is there; those behind it may be under way
        read(b0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (k > 0) multiply(STEPS - 1);  // the last operands of stage k - 1
#pragma unroll
        for (int j = 0; j + 1 < STEPS; ++j) {
            // operands j, before the next are asked for: the compiler's own wait, behind that, would be for all, since a load
            // that writes LDS is under way
            __builtin_amdgcn_s_waitcnt(wait_for(63, 0));
            __builtin_amdgcn_sched_barrier(0);
            read(b0, j + 1);
            // into the buffer that the barrier freed; stages behind the last read zeros, so that the waits can count
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (v * (STEPS - 1) / V == j) load(next, k + NB - 1, bl, v);
            multiply(j);
            // an MFMA, the reads, then a load behind each of the other MFMAs: the matrix unit has work at once
            __builtin_amdgcn_sched_group_barrier(8, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, TM + TN, 0);
#pragma unroll
            for (int i = 1; i < TM * TN; ++i) {
                __builtin_amdgcn_sched_group_barrier(8, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x20, 1, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        bl = b0;
        b0 = b0 == (NB - 1) * kBuf ? 0 : b0 + kBuf;
    };
    int k = 0;
    for (; (k + NB) * kStage <= a.K; ++k) step(whole, k);
    for (; k < stages; ++k) step(part, k);
    multiply(STEPS - 1);
    arrive<0>();  // no load is left that would write over the results

    // the lane holds x row r32, weight rows 8 (i / 4) + 4 half + i % 4 of each part
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int r = (wm * TM + m) * 32 + r32;
        const float sx = Op::kScales ? s_x[r] : 0.f;
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int c = (wn * TN + n) * 32 + 2 * i + 4 * half;
                const float4 sw = Op::kScales ? *reinterpret_cast<const float4 *>(s_w + c) : make_float4(0.f, 0.f, 0.f, 0.f);
                float4 v = make_float4(Op::value(acc[m][n][i], sx, sw.x), Op::value(acc[m][n][i + 1], sx, sw.y),
                                       Op::value(acc[m][n][i + 2], sx, sw.z), Op::value(acc[m][n][i + 3], sx, sw.w));
                if constexpr (kEpi) {
                    *reinterpret_cast<float4 *>(lds + r * kOutPitch + 4 * c) = v;
                } else {
                    *reinterpret_cast<uint2 *>(lds + r * kOutPitch + 2 * c) =
                        make_uint2(pack2_bf16(v.x, v.y), pack2_bf16(v.z, v.w));
                }
            }
    }
    __syncthreads();
#pragma unroll 1
    for (int i = threadIdx.x; i < BM * BN / 8; i += T) {
        const int r = i / (BN / 8), c = i % (BN / 8) * 8;
        if (m0 + r >= a.M || n0 + c >= a.N) continue;
        const char *src = lds + r * kOutPitch + (kEpi ? 4 : 2) * c;
        uint16_t *dst = a.out + (m0 + r) * a.o_s0 + n0 + c;
        const bool whole = a.wide && n0 + c + 8 <= a.N;
        if constexpr (kEpi) {
            const float4 lo = *reinterpret_cast<const float4 *>(src), hi = *reinterpret_cast<const float4 *>(src + 16);
            const float4 bl = *reinterpret_cast<const float4 *>(s_b + c), bh = *reinterpret_cast<const float4 *>(s_b + c + 4);
            float v[8] = {lo.x + bl.x, lo.y + bl.y, lo.z + bl.z, lo.w + bl.w, hi.x + bh.x, hi.y + bh.y, hi.z + bh.z, hi.w + bh.w};
            activate_all(v, a.act);
            const uint16_t *res = a.residual + (m0 + r) * a.r_s0 + n0 + c;
            if (whole) {
                if (a.residual) {
                    float f[8];
                    unpack8(*reinterpret_cast<const uint4 *>(res), f);
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] += f[e];
                }
                *reinterpret_cast<uint4 *>(dst) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]),
                                                             pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (n0 + c + e < a.N) dst[e] = f32_to_bf16(a.residual ? v[e] + bf16_to_f32(res[e]) : v[e]);
            }
        } else if (whole) {
            *reinterpret_cast<i32x4 *>(dst) = *reinterpret_cast<const i32x4 *>(src);
        } else {
            for (int e = 0; e < 8 && n0 + c + e < a.N; ++e) dst[e] = reinterpret_cast<const uint16_t *>(src)[e];
        }
    }
}

bool al(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <typename Op, bool kEpi, int MT>
void launch_rows(const ProductArgs &a, hipStream_t st) {
    hipLaunchKernelGGL((product_rows_kernel<Op, kEpi, MT>), dim3((a.N + 15) / 16, (a.M + 16 * MT - 1) / (16 * MT)),
                       dim3(kRowWaves * kWave), 0, st, a);
}

template <typename Op, bool kEpi, int WM, int WN, int TM, int TN, int NB>
void launch_tiles(const ProductArgs &a, hipStream_t st) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    const int tiles_m = (a.M + BM - 1) / BM, tiles_n = (a.N + BN - 1) / BN;
    hipLaunchKernelGGL((product_tile_kernel<Op, kEpi, WM, WN, TM, TN, NB>), dim3((tiles_m * tiles_n + 7) / 8 * 8),
                       dim3(WM * WN * kWave), 0, st, a, tiles_m, tiles_n);
}

// Rows and columns of out a workgroup takes.  Few tiles: the waves split K.  Otherwise the largest tile that still gives every
// CU one.
// Measured, K 2048, us (the rule's own first):
//   M 16  N 4096:  16-row pieces 3.1, 32-row 3.6;                 N 12288: 7.3, 64 x 64 tiles 7.4
//   M 32  N 6144:  32-row pieces 7.1, 64 x 64 tiles 7.2;          N 12288: 64 x 64 tiles 7.5, 32-row pieces 10.2
//   M 64  N 4096:  64-row pieces 5.2, 32-row 6.2, 64 x 64 6.4;    N 6144: 64 x 64 tiles 7.4, 64-row pieces 9.9
//   M 77  N 2048 (K 6144): 48-row pieces int8 8.2, bf16 12.5, 64-row 9.5, 14.3; M 48 N 4096: 5.2, 8.7 and 5.9, 9.1: pieces of 48
//   rows where they are no more than pieces of 64, since each reads its rows of x again
//   M 256 N 4096:  64 x 64 tiles 7.6, 64 x 128 8.7;               N 6144: 64 x 128 tiles 8.9, 64 x 64 9.6, 128 x 256 17.5
//   M 640 N 6144:  64 x 128 tiles 15.0, 128 x 256 18.5;           N 12288: 128 x 256 tiles 21.9, 64 x 128 26.8
//   M 1000 N 12288: 128 x 256 tiles 37.4, 64 x 128 39.0
// With an epilogue also 128 x 128, where those are one round of the CUs and 64 x 128 are two (not in the plain product, whose
// tiles nq_linear_int8_tile tells), 128 x 128 before what the rule would take:
//   M 500 N 6144:  bf16 19.1 and 23.3, int8 13.6 and 15.2;        M 640 N 6144: 24.3 and 29.3, 16.8 and 17.8
//   M 1500 N 2048: 21.1 and 23.1, 14.5 and 15.5;                  M 2000 N 2048, K 6144: 57.7 and 66.6, 33.1 and 36.9
//   one round of 64 x 128 (M 500 N 4096): 18.1 and 15.5, 12.5 and 10.8; two of 128 x 128 (M 800 N 6144): 37.6 and 30.0
constexpr int tile_id(int rows, int columns) { return rows << 16 | columns; }
int tile_for(int M, int N, bool epilogue = false) {
    auto count = [&](int bm, int bn) { return static_cast<int64_t>((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    auto rounds = [](int64_t tiles) { return (tiles + 255) / 256; };
    if (M <= 16) return tile_id(16, 16);
    if (count(32, 16) <= (M <= 32 ? 512 : 256)) return tile_id(32, 16);
    if (count(64, 16) <= 256) return (M + 47) / 48 == (M + 63) / 64 ? tile_id(48, 16) : tile_id(64, 16);
    if (count(64, 64) <= 256) return tile_id(64, 64);
    if (epilogue && count(64, 128) > 256 && count(128, 128) <= 256) return tile_id(128, 128);
    if (3 * rounds(count(128, 256)) > rounds(count(64, 128))) return tile_id(64, 128);
    return tile_id(128, 256);
}

bool one_round(int M, int N, int bm, int bn) {
    return static_cast<int64_t>((M + bm - 1) / bm) * ((N + bn - 1) / bn) <= 256;
}

// Four stages in LDS where a CU has one workgroup of a small tile: three are 48 KB on their way at most, less than the time of a
// load asks for.  us with four and three, K 2048 unless said, bf16 then int8: M 200 N 4096 10.9 and 11.9, 8.5 and 8.9; M 300 N 2048
// (K 6144) 22.9 and 27.5, 14.3 and 16.6; M 640 N 2048 (K 6144; 64 x 128) 32.4 and 35.1, 19.1 and 20.7; five to eight
// no better.  Tiles of 64 x 128 in several rounds keep two workgroups a CU with three (M 1500 N 6144: 56.4 and, with four, 66.5).
template <typename Op, bool kEpi>
int launch_product(const ProductArgs &a, hipStream_t st) {
    const int tile = tile_for(a.M, a.N, kEpi);
    if constexpr (kEpi) {
        if (tile == tile_id(128, 128)) {
            launch_tiles<Op, kEpi, 2, 4, 2, 1, 3>(a, st);
            return NQ_LAUNCH_STATUS();
        }
    }
    switch (tile) {
        case tile_id(16, 16): launch_rows<Op, kEpi, 1>(a, st); break;
        case tile_id(32, 16): launch_rows<Op, kEpi, 2>(a, st); break;
        case tile_id(48, 16): launch_rows<Op, kEpi, 3>(a, st); break;
        case tile_id(64, 16): launch_rows<Op, kEpi, 4>(a, st); break;
        case tile_id(64, 64): launch_tiles<Op, kEpi, 2, 2, 1, 1, 4>(a, st); break;
        case tile_id(64, 128):
            if (one_round(a.M, a.N, 64, 128)) launch_tiles<Op, kEpi, 2, 4, 1, 1, 4>(a, st);
            else launch_tiles<Op, kEpi, 2, 4, 1, 1, 3>(a, st);
            break;
        default: launch_tiles<Op, kEpi, 2, 4, 2, 2, 3>(a, st);  // 128 x 256
    }
    return NQ_LAUNCH_STATUS();
}

// Grid sizes and the kernels' 32-bit row and column numbers.
bool product_fits(int M, int N) {
    return static_cast<int64_t>((M + 31) / 32) * ((N + 31) / 32) <= 0x3fffffff && N <= 0x7fffff00 && M <= 0x7fffff00;
}

}  // namespace
}  // namespace nq

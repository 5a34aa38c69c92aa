// Products of 8-bit integers with a scale for each token and output channel:
//   out[m, n] = bf16(float(sum_k cx[m, k] cw[n, k]) * sx[m] * sw[n])
// with the sum in int32 (exact for K <= 2^17), and the quantisation of rows that
// makes both operands: s = max |x| / 127, c = rint(127 x / max |x|).  127 x is exact
// in fp32 for a bf16 x.  With significands a of x and b of max |x| (integers below
// 256) and 2^k between their exponents a quotient is 127 a / (b 2^k); from a tie,
// (2n + 1) / 2, it differs by |254 a - (2n + 1) b 2^k| / (b 2^(k + 1)), whose
// numerator is an integer: by nothing, or by at least 1 / (254 a) > 2^-16 of the
// quotient itself.  The computed one is within 2^-23 of itself, and a tie, a float,
// comes out as it is; so the codes are those of exact arithmetic.
//
// Few rows: a workgroup owns 16 output channels and all of K, its waves interleave K in
// pieces of 128 bytes, each through LDS of its own, and add their int32 sums at the end.
// Integer sums are exact in any order, so cutting K costs no determinism.
// Many rows: (32 TM WM) x (32 TN WN) tiles of mfma_i32_32x32x32_i8, K staged 128 bytes at a
// time through three LDS buffers, the next two stages' loads in flight.
#include <type_traits>

#include "nq_common.h"
#include "nq_int8_codes.h"
#include "nq_internal.h"

namespace nq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kQThreads = 256;
constexpr int kQVec = 4;  // 8-value vectors a thread keeps; longer rows are read twice

// A workgroup a row, which stays in registers between the maximum and the codes up to 8192 values.  Bound by HBM:
// 4001 rows of 6144 (74 MB) 14.6 us, 5.1 TB/s; by its launch and one round trip at 1 row of 2048, 2.4 us.
__global__ void __launch_bounds__(kQThreads)
quantize_int8_rows_kernel(const uint16_t *__restrict__ x, int64_t x_s0, int K, int8_t *__restrict__ q, int64_t q_s0,
                          float *__restrict__ scales) {
    __shared__ float s_max[kQThreads / kWave];
    __shared__ int s_odd[kQThreads / kWave];
    const int64_t row = blockIdx.x;
    const int nvec = K / 8;
    const uint16_t *xr = x + row * x_s0;
    uint4 held[kQVec];
    float amax = 0.f;
    bool odd = false;
    auto look = [&](const uint4 &v) {
        float f[8];
        unpack8(v, f);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            amax = fmaxf(amax, fabsf(f[e]));
            odd |= !(fabsf(f[e]) < __builtin_inff());
        }
    };
#pragma unroll
    for (int i = 0; i < kQVec; ++i) {
        const int vi = threadIdx.x + i * kQThreads;
        held[i] = vi < nvec ? *reinterpret_cast<const uint4 *>(xr + vi * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kQVec; ++i) look(held[i]);
    for (int vi = threadIdx.x + kQVec * kQThreads; vi < nvec; vi += kQThreads)
        look(*reinterpret_cast<const uint4 *>(xr + vi * 8));
    amax = group_max<kWave>(amax);
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const bool any = __any(odd);
    if (lane == 0) {
        s_max[wave] = amax;
        s_odd[wave] = any;
    }
    __syncthreads();
    int bad = 0;
#pragma unroll
    for (int w = 0; w < kQThreads / kWave; ++w) {
        amax = fmaxf(amax, s_max[w]);
        bad |= s_odd[w];
    }
    // very large and very small rows are scaled by a power of two first: 127 x and 1 / top stay normal
    const float scale = amax > 1.8446744073709552e19f ? 5.421010862427522e-20f
                        : amax < 5.421010862427522e-20f ? 1.8446744073709552e19f : 1.0f;
    const bool zero = bad || amax == 0.f;
    const float top = zero ? 1.0f : amax * scale;
    const float inv = 1.0f / top;
    auto put = [&](int vi, const uint4 &v) __attribute__((always_inline)) {
        float f[8];
        unpack8(v, f);
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = code_bits(zero ? 0.f : f[e] * scale, top, inv);
        *reinterpret_cast<uint2 *>(q + row * q_s0 + vi * 8) =
            make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
    };
#pragma unroll
    for (int i = 0; i < kQVec; ++i) {
        const int vi = threadIdx.x + i * kQThreads;
        if (vi < nvec) put(vi, held[i]);
    }
    for (int vi = threadIdx.x + kQVec * kQThreads; vi < nvec; vi += kQThreads)
        put(vi, *reinterpret_cast<const uint4 *>(xr + vi * 8));
    // a row with NaN or infinity: its product is NaN
    if (threadIdx.x == 0) scales[row] = bad ? __builtin_nanf("") : (amax == 0.f ? 1.0f : amax / 127.0f);
}

struct Int8Args {
    const int8_t *x;
    int64_t x_s0;
    const float *sx;
    const int8_t *w;
    int64_t w_s0;
    const float *sw;
    int M, N, K;
    uint16_t *out;
    int64_t o_s0;
    int wide;  // out rows take 16-byte stores
};

// |sum| <= 2^31, so that sum * sx stays inside fp32 up to sx = 2^96; a larger sx comes last, when a model's weights have
// made sum * sw small enough for the result, where that fits.
__device__ __forceinline__ float scaled(int sum, float sx, float sw) {
    const bool far = sx > 0x1p96f;
    return static_cast<float>(sum) * (far ? sw : sx) * (far ? sx : sw);
}

constexpr int kStage = 128;         // bytes of K a stage
constexpr int kChunks = kStage / 16;

// LDS place of 16-byte chunk c of row r: measured free of conflicts for the operand reads (32 rows and two chunks, 16
// rows and four) and for the writes (eight rows).
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kChunks + (c ^ ((r >> 1) & 7)); }

__device__ const i32x4 kZero16 = {0, 0, 0, 0};  // what a chunk behind K is read from

// Waits until at most N of the wave's loads are under way (and all its LDS reads are back), then the barrier: what those
// loads wrote to LDS is there for every wave, and what they read there may be overwritten.
template <int N>
__device__ __forceinline__ void arrive() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
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

template <int MT>
__global__ void __launch_bounds__(kRowWaves * kWave)
int8_rows_kernel(Int8Args a) {
    constexpr int NW = kRowWaves, V = 2 * (MT + 1);  // loads of 1 KB (eight rows) a piece: the weights', then x's
    constexpr int kBuf = 1024 * V;
    constexpr int kPart = MT * 256;  // sums of a wave
    static_assert(kPart * 4 <= 2 * kBuf, "the sums fit where the operands were");
    __shared__ __attribute__((aligned(16))) char lds[NW * 2 * kBuf];
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    // load v writes rows 8 v .. + 7 of a piece, lane l place l % 8 of row l / 8
    const int8_t *from[V];
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
            const int8_t *p = at + col[v] < a.K ? from[v] + at : reinterpret_cast<const int8_t *>(&kZero16);
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void *)p,
                (__attribute__((address_space(3))) void *)(mine + buf * kBuf + 1024 * v), 16, 0, 0);
        }
    };
    // operand h: lane l holds row l % 16, bytes 64 h + 16 (l / 16) .. + 15 of the piece, the same order in both
    int get[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) get[h] = 16 * chunk_at(lane & 15, 4 * h + (lane >> 4));
    i32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
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
                    acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[h], x[h][m], acc[m], 0, 0, 0);
        }
    }
    arrive<0>();  // every wave's loads and reads are done
    int *part = reinterpret_cast<int *>(lds);
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<i32x4 *>(part + wave * kPart + m * 256 + lane * 4) = acc[m];
    __syncthreads();
    // element e of tile m: lane e / 4, weight row 4 (lane / 16) + e % 4, x row lane % 16; threads along weight rows
    for (int i = threadIdx.x; i < kPart; i += NW * kWave) {
        const int m = i / 256, row = (i & 255) >> 4, n = i & 15;
        const int e = m * 256 + ((n >> 2) * 16 + row) * 4 + (n & 3);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += part[w * kPart + e];
        const int r = m0 + 16 * m + row;
        if (r < a.M && n0 + n < a.N)
            a.out[r * a.o_s0 + n0 + n] = f32_to_bf16(scaled(sum, a.sx[r], a.sw[n0 + n]));
    }
}

// WM x WN waves, each TM x TN parts of 32 x 32.  K goes through three LDS buffers, 128 bytes a stage, written by the
// loads themselves (a register on the way would cost its write to LDS: 0.14 us a stage of 128 x 256).  Step k: stage k
// has arrived, the loads of stage k + 2 are issued; the operands of each 32 bytes are read while the MFMAs of the 32
// before run, also across the barrier.  The results cross LDS once more, so that they leave in whole lines.
// No unit is full: at 4001 x 2048 (K 6144) the MFMAs run in 38 % of the clocks and LDS in 21 % (128 KB read a stage, at 256
// bytes a clock), while the waves wait to issue in 54 % of theirs: the eight waves of a CU's one workgroup (its buffers
// take the LDS) meet at every stage's barrier.  A stage takes 1.0 us with every CU busy, launch, first loads and results
// 9 us.  640 x 12288 (K 2048) 22.5 us = 1430 TOP/s, 4001 x 2048 (K 6144) 56.6 us = 1780 TOP/s (2496 is what a library's
// 8192^3 reaches).  Other waves for that tile at the same sizes: 2 x 2 of 64 x 128 33 and 69 us, 1 x 4 of 128 x 64 32 and
// 68, 4 x 2 of 32 x 64 (128 x 128) 30 and 70 (24.4 and 67.9 since).
template <int WM, int WN, int TM, int TN>
__global__ void __launch_bounds__(WM * WN * kWave)
int8_tile_kernel(Int8Args a, int tiles_m, int tiles) {
    constexpr int NW = WM * WN, T = NW * kWave, BM = 32 * TM * WM, BN = 32 * TN * WN;
    constexpr int V = (BM + BN) / 8 / NW;  // loads of 1 KB (eight rows) a wave and stage
    constexpr int STEPS = kStage / 32;
    static_assert(V * NW * 8 == BM + BN && STEPS == 4, "a stage splits evenly over the waves");
    constexpr int kBuf = (BM + BN) * kStage;     // bytes of a stage: weights, then x
    constexpr int kOutPitch = BN * 2 + 16;       // bytes of a result row
    constexpr int kOut = BM * kOutPitch;
    constexpr int kScales = 3 * kBuf > kOut ? 3 * kBuf : kOut;  // behind the buffers: the tile's scales, there when the sums are
    // one array: with a second one the compiler waits for every load in flight before it reads LDS (57 us become 87)
    __shared__ __attribute__((aligned(16))) char lds[kScales + 4 * (BM + BN)];
    float *const s_w = reinterpret_cast<float *>(lds + kScales), *const s_x = s_w + BN;
    // XCD b % 8 takes tiles (b % 8) per ..: neighbours in m share their weights in one L2
    const int per = (tiles + 7) / 8;
    const int t = static_cast<int>(blockIdx.x % 8) * per + static_cast<int>(blockIdx.x / 8);
    if (t >= tiles) return;
    const int m0 = t % tiles_m * BM, n0 = t / tiles_m * BN;
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int r32 = lane & 31, half = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;
    for (int i = threadIdx.x; i < BN; i += T) s_w[i] = n0 + i < a.N ? a.sw[n0 + i] : 0.f;
    for (int i = threadIdx.x; i < BM; i += T) s_x[i] = m0 + i < a.M ? a.sx[m0 + i] : 0.f;

    // load v writes rows 8 (wave V + v) .. + 7 of a stage, lane l place l % 8 of row l / 8
    const int8_t *from[V];
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

    i32x16 acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0;

    const int stages = (a.K + kStage - 1) / kStage;
    auto load = [&](auto whole, int k, int buf, int v) __attribute__((always_inline)) {
        const int8_t *p = from[v];
        if constexpr (!whole) p = k * kStage + col[v] < a.K ? p : reinterpret_cast<const int8_t *>(&kZero16);
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
                acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j & 1][n], xf[j & 1][m], acc[m][n], 0, 0, 0);
    };
    int b0 = 0, b1 = kBuf, b2 = 2 * kBuf;  // buffers of stages k, k + 1, k + 2
    constexpr std::true_type whole{};      // stages inside K: no look at the chunks, 14 vector instructions instead of 40
    constexpr std::false_type part{};
#pragma unroll
    for (int v = 0; v < V; ++v) load(part, 0, b0, v);
#pragma unroll
    for (int v = 0; v < V; ++v) load(part, 1, b1, v);
    auto step = [&](auto next, int k) __attribute__((always_inline)) {
        arrive<V>();  // stage k is there; stage k + 1 may be under way
        read(b0, 0);
        __builtin_amdgcn_sched_barrier(0);
        if (k > 0) multiply(STEPS - 1);  // the last operands of stage k - 1
#pragma unroll
        for (int j = 0; j < STEPS; ++j) {
            // into the buffer that the barrier freed; stages behind the last read zeros, so that the waits can count
#pragma unroll
            for (int v = V * j / STEPS; v < V * (j + 1) / STEPS; ++v) load(next, k + 2, b2, v);
            __builtin_amdgcn_sched_barrier(0);
            if (j + 1 < STEPS) {
                read(b0, j + 1);
                __builtin_amdgcn_sched_barrier(0);
                multiply(j);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        const int b = b0;
        b0 = b1;
        b1 = b2;
        b2 = b;
    };
    int k = 0;
    for (; (k + 3) * kStage <= a.K; ++k) step(whole, k);
    for (; k < stages; ++k) step(part, k);
    multiply(STEPS - 1);
    arrive<0>();  // no load is left that would write over the results

    // the lane holds x row r32, weight rows 8 (i / 4) + 4 half + i % 4 of each part
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int r = (wm * TM + m) * 32 + r32;
        const float sx = s_x[r];
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int c = (wn * TN + n) * 32 + 2 * i + 4 * half;
                const float4 sw = *reinterpret_cast<const float4 *>(s_w + c);
                *reinterpret_cast<uint2 *>(lds + r * kOutPitch + 2 * c) =
                    make_uint2(pack2_bf16(scaled(acc[m][n][i], sx, sw.x), scaled(acc[m][n][i + 1], sx, sw.y)),
                               pack2_bf16(scaled(acc[m][n][i + 2], sx, sw.z), scaled(acc[m][n][i + 3], sx, sw.w)));
            }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < BM * BN / 8; i += T) {
        const int r = i / (BN / 8), c = i % (BN / 8) * 8;
        if (m0 + r >= a.M || n0 + c >= a.N) continue;
        const char *src = lds + r * kOutPitch + 2 * c;
        uint16_t *dst = a.out + (m0 + r) * a.o_s0 + n0 + c;
        if (a.wide && n0 + c + 8 <= a.N) {
            *reinterpret_cast<i32x4 *>(dst) = *reinterpret_cast<const i32x4 *>(src);
        } else {
            for (int e = 0; e < 8 && n0 + c + e < a.N; ++e) dst[e] = reinterpret_cast<const uint16_t *>(src)[e];
        }
    }
}

bool al(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int MT>
void launch_rows(const Int8Args &a, hipStream_t st) {
    hipLaunchKernelGGL(int8_rows_kernel<MT>, dim3((a.N + 15) / 16, (a.M + 16 * MT - 1) / (16 * MT)),
                       dim3(kRowWaves * kWave), 0, st, a);
}

template <int WM, int WN, int TM, int TN>
void launch_tiles(const Int8Args &a, hipStream_t st) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    const int tiles_m = (a.M + BM - 1) / BM, tiles = tiles_m * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL((int8_tile_kernel<WM, WN, TM, TN>), dim3((tiles + 7) / 8 * 8), dim3(WM * WN * kWave), 0, st, a,
                       tiles_m, tiles);
}

// Rows and columns of out a workgroup takes.  Few tiles: the waves split K.  Otherwise the largest tile that still gives every
// CU one: a stage of 128 bytes takes 0.28, 0.34 and 0.72 us at 64 x 64, 64 x 128 and 128 x 256 (1.0 with every CU busy).
// Measured, K 2048, us (the rule's own first):
//   M 16  N 4096:  16-row pieces 3.1, 32-row 3.6;                 N 12288: 7.3, 64 x 64 tiles 7.4
//   M 32  N 6144:  32-row pieces 7.1, 64 x 64 tiles 7.2;          N 12288: 64 x 64 tiles 7.5, 32-row pieces 10.2
//   M 64  N 4096:  64-row pieces 5.2, 32-row 6.2, 64 x 64 6.4;    N 6144: 64 x 64 tiles 7.4, 64-row pieces 9.9
//   M 256 N 4096:  64 x 64 tiles 7.6, 64 x 128 8.7;               N 6144: 64 x 128 tiles 8.9, 64 x 64 9.6, 128 x 256 17.5
//   M 640 N 6144:  64 x 128 tiles 15.0, 128 x 256 18.5;           N 12288: 128 x 256 tiles 21.9, 64 x 128 26.8
//   M 1000 N 12288: 128 x 256 tiles 37.4, 64 x 128 39.0 (128 x 128, which is not kept, 35.6; at 640 x 6144 13.6)
constexpr int tile_id(int rows, int columns) { return rows << 16 | columns; }
int tile_for(int M, int N) {
    auto count = [&](int bm, int bn) { return static_cast<int64_t>((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
    auto rounds = [](int64_t tiles) { return (tiles + 255) / 256; };
    if (M <= 16) return tile_id(16, 16);
    if (count(32, 16) <= (M <= 32 ? 512 : 256)) return tile_id(32, 16);
    if (count(64, 16) <= 256) return tile_id(64, 16);
    if (count(64, 64) <= 256) return tile_id(64, 64);
    if (3 * rounds(count(128, 256)) > rounds(count(64, 128))) return tile_id(64, 128);
    return tile_id(128, 256);
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_quantize_int8_rows(const uint16_t *x, int64_t x_s0, int M, int K, int8_t *q, int64_t q_s0,
                                     float *scales, void *stream) {
    NQ_CHECK_ARG(M >= 0 && K >= 0);
    if (M == 0) return NQ_OK;
    NQ_CHECK_ARG(x && q && scales && K >= 16 && x_s0 >= 0 && (M == 1 || q_s0 >= K));
    if (K % 16 || (M > 1 && (x_s0 % 8 || q_s0 % 8)) || !al(x, 16) || !al(q, 8)) return NQ_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(quantize_int8_rows_kernel, dim3(M), dim3(kQThreads), 0, static_cast<hipStream_t>(stream), x,
                       x_s0, K, q, q_s0, scales);
    return NQ_LAUNCH_STATUS();
}

extern "C" int nq_linear_int8_tile(int M, int N) {
    return M < 1 || N < 1 || M > 0x7fffff00 || N > 0x7fffff00 ? -1 : tile_for(M, N);
}

extern "C" int nq_linear_int8(const int8_t *xq, int64_t x_s0, const float *sx, const int8_t *wq, int64_t w_s0,
                              const float *sw, int M, int N, int K, uint16_t *out, int64_t o_s0, void *stream) {
    NQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0);
    if (M == 0 || N == 0) return NQ_OK;
    NQ_CHECK_ARG(xq && sx && wq && sw && out && K >= 16 && x_s0 >= 0 && w_s0 >= 0 && (M == 1 || o_s0 >= N));
    if (K % 16 || K > (1 << 17) || (M > 1 && x_s0 % 16) || (N > 1 && w_s0 % 16) || !al(xq, 16) || !al(wq, 16) ||
        !al(sx, 4) || !al(sw, 4))
        return NQ_ERR_UNSUPPORTED;
    if (static_cast<int64_t>((M + 31) / 32) * ((N + 31) / 32) > 0x3fffffff || N > 0x7fffff00 || M > 0x7fffff00)
        return NQ_ERR_UNSUPPORTED;
    const Int8Args a = {xq,  x_s0, sx,   wq, w_s0, sw, M, N, K, out, o_s0,
                        (M == 1 || o_s0 % 8 == 0) && al(out, 16)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    switch (tile_for(M, N)) {
        case tile_id(16, 16): launch_rows<1>(a, st); break;
        case tile_id(32, 16): launch_rows<2>(a, st); break;
        case tile_id(64, 16): launch_rows<4>(a, st); break;
        case tile_id(64, 64): launch_tiles<2, 2, 1, 1>(a, st); break;
        case tile_id(64, 128): launch_tiles<2, 4, 1, 1>(a, st); break;
        default: launch_tiles<2, 4, 2, 2>(a, st);  // 128 x 256
    }
    return NQ_LAUNCH_STATUS();
}

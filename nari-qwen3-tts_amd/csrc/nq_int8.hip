// Products of 8-bit integers with a scale for each token and output channel:
//   out[m, n] = bf16(float(sum_k cx[m, k] cw[n, k]) * sx[m] * sw[n])
// with the sum in int32 (exact for K <= 2^17), and the quantisation of rows that
// makes both operands: s = max |x| / 127, c = rint(127 x / max |x|).  127 x is exact
// in fp32 for a bf16 x and the quotient correctly rounded, and a quotient that is
// no tie lies at least 1 / 512 from one, so the codes are those of exact arithmetic.
//
// Few rows: a workgroup owns 16 output channels and all of K, its waves
// interleave K in pieces of 128 and add their int32 sums through LDS; weights and
// rows go straight from memory into mfma_i32_16x16x64_i8 operands.  Integer sums are exact in
// any order, so cutting K costs no determinism.
// Many rows: (32 TM WM) x (32 TN WN) tiles of mfma_i32_32x32x32_i8, K staged 128 bytes at a
// time through LDS, double buffered, the next stages' loads in flight.
#include "nq_common.h"
#include "nq_internal.h"

namespace nq {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

constexpr int kQThreads = 256;
constexpr int kQVec = 4;  // 8-value vectors a thread keeps; longer rows are read twice

// 127 x / amax; above 2^64 both are scaled down first (by a power of two), so that 127 x stays finite.
__device__ __forceinline__ int code_of(float x, float amax, float down) {
    return static_cast<int>(rintf((x * down * 127.0f) / amax));
}

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
    const float down = amax > 1.8446744073709552e19f ? 5.421010862427522e-20f : 1.0f;
    const float top = amax * down;
    const bool zero = bad || amax == 0.f;
    auto put = [&](int vi, const uint4 &v) {
        float f[8];
        unpack8(v, f);
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            w[e / 4] |= static_cast<uint32_t>((zero ? 0 : code_of(f[e], top, down)) & 0xff) << (8 * (e % 4));
        *reinterpret_cast<uint2 *>(q + row * q_s0 + vi * 8) = make_uint2(w[0], w[1]);
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
    int wide;  // out rows take 8-byte stores
};

__device__ __forceinline__ float scaled(int sum, float sx, float sw) { return static_cast<float>(sum) * sx * sw; }

// MT 16-row tiles of x against 16 weight rows.  Lane l holds row l % 16 of either operand, bytes
// 32 (l / 16) .. + 31 of a 128-byte piece of K, the same order in both; it ends with weight rows 4 (l / 16) .. + 3
// of x row l % 16.
template <int MT, int NW>
__global__ void __launch_bounds__(NW * kWave)
int8_rows_kernel(Int8Args a) {
    __shared__ __attribute__((aligned(16))) int part[NW][MT][kWave * 4];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int r16 = lane & 15, kq = lane >> 4;
    const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MT;
    const int wn = n0 + r16 < a.N ? n0 + r16 : a.N - 1;
    const int8_t *wp = a.w + wn * a.w_s0 + 32 * kq;
    const int8_t *xp[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const int r = m0 + 16 * m + r16;
        xp[m] = a.x + (r < a.M ? r : a.M - 1) * a.x_s0 + 32 * kq;
    }
    i32x4 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
    const i32x4 none = {0, 0, 0, 0};
#pragma unroll 2
    for (int k = wave * 128; k < a.K; k += NW * 128) {
        const int at = k + 32 * kq;
        i32x4 wv[2], xv[MT][2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const bool in = at + 16 * h < a.K;  // K is a multiple of 16
            wv[h] = in ? *reinterpret_cast<const i32x4 *>(wp + k + 16 * h) : none;
#pragma unroll
            for (int m = 0; m < MT; ++m)
                xv[m][h] = in ? *reinterpret_cast<const i32x4 *>(xp[m] + k + 16 * h) : none;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int m = 0; m < MT; ++m)
                acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv[h], xv[m][h], acc[m], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) *reinterpret_cast<i32x4 *>(&part[wave][m][lane * 4]) = acc[m];
    __syncthreads();
    // element e of tile m: lane e / 4, weight row 4 (lane / 16) + e % 4, x row lane % 16; threads along weight rows
    for (int i = threadIdx.x; i < MT * 256; i += NW * kWave) {
        const int m = i / 256, row = (i & 255) >> 4, n = i & 15;
        const int e = ((n >> 2) * 16 + row) * 4 + (n & 3);
        int sum = 0;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += part[w][m][e];
        const int r = m0 + 16 * m + row;
        if (r < a.M && n0 + n < a.N)
            a.out[r * a.o_s0 + n0 + n] = f32_to_bf16(scaled(sum, a.sx[r], a.sw[n0 + n]));
    }
}

constexpr int kStage = 128;         // bytes of K a stage
constexpr int kChunks = kStage / 16;

// LDS place of 16-byte chunk c of row r: eight neighbouring rows read at one c, and a row's eight chunks written
// together, touch all banks.
__device__ __forceinline__ int chunk_at(int r, int c) { return r * kChunks + (c ^ (r & 7)); }

template <int WM, int WN, int TM, int TN>
__global__ void __launch_bounds__(WM * WN * kWave)
int8_tile_kernel(Int8Args a, int tiles_m, int tiles) {
    constexpr int T = WM * WN * kWave, BM = 32 * TM * WM, BN = 32 * TN * WN;
    constexpr int XV = BM * kChunks / T, WV = BN * kChunks / T;
    static_assert(XV * T == BM * kChunks && WV * T == BN * kChunks, "stage splits evenly over the threads");
    __shared__ i32x4 xs[2][BM * kChunks];
    __shared__ i32x4 ws[2][BN * kChunks];
    // XCD b % 8 takes tiles (b % 8) per ..: neighbours in m share their weights in one L2
    const int per = (tiles + 7) / 8;
    const int t = static_cast<int>(blockIdx.x % 8) * per + static_cast<int>(blockIdx.x / 8);
    if (t >= tiles) return;
    const int m0 = t % tiles_m * BM, n0 = t / tiles_m * BN;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int r32 = lane & 31, half = lane >> 5;
    const int wm = wave / WN, wn = wave % WN;

    const int chunk = threadIdx.x % kChunks;
    const int8_t *xp[XV], *wp[WV];
#pragma unroll
    for (int v = 0; v < XV; ++v) {
        const int r = m0 + (threadIdx.x + v * T) / kChunks;
        xp[v] = a.x + (r < a.M ? r : a.M - 1) * a.x_s0 + 16 * chunk;
    }
#pragma unroll
    for (int v = 0; v < WV; ++v) {
        const int r = n0 + (threadIdx.x + v * T) / kChunks;
        wp[v] = a.w + (r < a.N ? r : a.N - 1) * a.w_s0 + 16 * chunk;
    }
    i32x16 acc[TM][TN];
#pragma unroll
    for (int m = 0; m < TM; ++m)
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[m][n][i] = 0;

    i32x4 xr[XV], wr[WV];
    const i32x4 none = {0, 0, 0, 0};
    auto load = [&](int k) {
        const bool in = k + 16 * chunk < a.K;
#pragma unroll
        for (int v = 0; v < WV; ++v) wr[v] = in ? *reinterpret_cast<const i32x4 *>(wp[v] + k) : none;
#pragma unroll
        for (int v = 0; v < XV; ++v) xr[v] = in ? *reinterpret_cast<const i32x4 *>(xp[v] + k) : none;
    };
    auto store = [&](int buf) {
#pragma unroll
        for (int v = 0; v < XV; ++v) xs[buf][chunk_at((threadIdx.x + v * T) / kChunks, chunk)] = xr[v];
#pragma unroll
        for (int v = 0; v < WV; ++v) ws[buf][chunk_at((threadIdx.x + v * T) / kChunks, chunk)] = wr[v];
    };
    load(0);
    store(0);
    if (kStage < a.K) load(kStage);
    int buf = 0;
    for (int k = 0; k < a.K; k += kStage, buf ^= 1) {
        __syncthreads();
        if (k + kStage < a.K) {
            store(buf ^ 1);
            if (k + 2 * kStage < a.K) load(k + 2 * kStage);
        }
#pragma unroll
        for (int s = 0; s < kStage / 32; ++s) {
            i32x4 wf[TN], xf[TM];
#pragma unroll
            for (int n = 0; n < TN; ++n) wf[n] = ws[buf][chunk_at((wn * TN + n) * 32 + r32, 2 * s + half)];
#pragma unroll
            for (int m = 0; m < TM; ++m) xf[m] = xs[buf][chunk_at((wm * TM + m) * 32 + r32, 2 * s + half)];
#pragma unroll
            for (int m = 0; m < TM; ++m)
#pragma unroll
                for (int n = 0; n < TN; ++n)
                    acc[m][n] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[n], xf[m], acc[m][n], 0, 0, 0);
        }
    }
    // the lane holds x row r32, weight rows 8 (i / 4) + 4 half + i % 4 of a 32 x 32 part
#pragma unroll
    for (int m = 0; m < TM; ++m) {
        const int row = m0 + (wm * TM + m) * 32 + r32;
        if (row >= a.M) continue;
        const float sx = a.sx[row];
        uint16_t *orow = a.out + row * a.o_s0;
#pragma unroll
        for (int n = 0; n < TN; ++n)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int col = n0 + (wn * TN + n) * 32 + 2 * i + 4 * half;
                if (a.wide && col + 3 < a.N) {
                    const float4 sw = *reinterpret_cast<const float4 *>(a.sw + col);
                    *reinterpret_cast<uint2 *>(orow + col) =
                        make_uint2(pack2_bf16(scaled(acc[m][n][i], sx, sw.x), scaled(acc[m][n][i + 1], sx, sw.y)),
                                   pack2_bf16(scaled(acc[m][n][i + 2], sx, sw.z), scaled(acc[m][n][i + 3], sx, sw.w)));
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col + e < a.N) orow[col + e] = f32_to_bf16(scaled(acc[m][n][i + e], sx, a.sw[col + e]));
                }
            }
    }
}

bool al(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <int MT, int NW>
void launch_rows(const Int8Args &a, hipStream_t st) {
    hipLaunchKernelGGL((int8_rows_kernel<MT, NW>), dim3((a.N + 15) / 16, (a.M + 16 * MT - 1) / (16 * MT)),
                       dim3(NW * kWave), 0, st, a);
}

template <int WM, int WN, int TM, int TN>
void launch_tiles(const Int8Args &a, hipStream_t st) {
    constexpr int BM = 32 * TM * WM, BN = 32 * TN * WN;
    const int tiles_m = (a.M + BM - 1) / BM, tiles = tiles_m * ((a.N + BN - 1) / BN);
    hipLaunchKernelGGL((int8_tile_kernel<WM, WN, TM, TN>), dim3((tiles + 7) / 8 * 8), dim3(WM * WN * kWave), 0, st, a,
                       tiles_m, tiles);
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

extern "C" int nq_linear_int8(const int8_t *xq, int64_t x_s0, const float *sx, const int8_t *wq, int64_t w_s0,
                              const float *sw, int M, int N, int K, uint16_t *out, int64_t o_s0, void *stream) {
    NQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0);
    if (M == 0 || N == 0) return NQ_OK;
    NQ_CHECK_ARG(xq && sx && wq && sw && out && K >= 16 && x_s0 >= 0 && w_s0 >= 0 && (M == 1 || o_s0 >= N));
    if (K % 16 || K > (1 << 17) || (M > 1 && x_s0 % 16) || (N > 1 && w_s0 % 16) || !al(xq, 16) || !al(wq, 16) || !al(sx, 4) || !al(sw, 4))
        return NQ_ERR_UNSUPPORTED;
    if (static_cast<int64_t>((M + 31) / 32) * ((N + 31) / 32) > 0x3fffffff || N > 0x7fffff00 || M > 0x7fffff00)
        return NQ_ERR_UNSUPPORTED;
    const Int8Args a = {xq,  x_s0, sx,   wq, w_s0, sw, M, N, K, out, o_s0,
                        (M == 1 || o_s0 % 4 == 0) && al(out, 8) && al(sw, 16)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (M <= 16) launch_rows<1, 16>(a, st);
    else if (M <= 32) launch_rows<2, 16>(a, st);
    else if (M <= 64) launch_rows<4, 16>(a, st);
    else if (static_cast<int64_t>((M + 127) / 128) * ((N + 127) / 128) >= 256) launch_tiles<2, 2, 2, 2>(a, st);
    else launch_tiles<2, 2, 1, 1>(a, st);
    return NQ_LAUNCH_STATUS();
}

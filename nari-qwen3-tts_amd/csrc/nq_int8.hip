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
// The product's kernels are in nq_product.h; integer sums are exact in any order, so cutting K costs no determinism.
#include "nq_common.h"
#include "nq_int8_codes.h"
#include "nq_internal.h"
#include "nq_product.h"

namespace nq {
namespace {

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
    if (!product_fits(M, N)) return NQ_ERR_UNSUPPORTED;
    ProductArgs a = {reinterpret_cast<const char *>(xq), x_s0, sx, reinterpret_cast<const char *>(wq), w_s0, sw, M, N, K,
                     out, o_s0, (M == 1 || o_s0 % 8 == 0) && al(out, 16), nullptr, nullptr, 0, NQ_ACT_NONE};
    return launch_product<Int8Op, false>(a, static_cast<hipStream_t>(stream));
}

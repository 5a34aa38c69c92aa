// RMS norm of rows, the residual's addition before it, answered as int8 codes with one scale a row, the operand of the
// int8 product:
//   x = bf16(residual + hidden), stored;  y_i = x_i w_i / sqrt(mean x^2 + eps);  scale = max |y| / 127;
//   code_i = rint(y_i / scale) = rint(127 p_i / max |p|),  p_i = x_i w_i
// The root is the row's own and leaves the codes: a product of two bf16 values has 16 significant bits, so p, 127 p and
// the quotient's side of every tie are exact in fp32 and the codes are those of exact arithmetic, whatever the order of the
// sum of squares.  (Through a bf16 row and its quantisation the codes would carry that row's rounding, half a step at
// the largest values.)
#include "nq_common.h"
#include "nq_int8_codes.h"
#include "nq_internal.h"

namespace nq {
namespace {

struct NormInt8Args {
    const uint16_t *hidden;  // null: nothing is added, nothing stored
    int64_t h_s0;
    uint16_t *residual;
    int64_t r_s0;
    const uint16_t *weight;
    int rows, width;
    float eps;
    int8_t *q;
    int64_t q_s0;
    float *scales;
};

// Rows whose sums or products leave fp32's comfort (values beyond 2^60 or all below 2^-30, NaN, infinities, zeros) are
// worked in double, which holds every product and square of bf16 values: a second look at the row, from what its own
// kWaves waves stored.
template <int kWaves>
__device__ __forceinline__ void norm_int8_row_wide(const NormInt8Args &a, int64_t row) {
    __shared__ double s_ss[kWaves], s_top[kWaves];
    constexpr int T = kWaves * kWave;
    const int tid = threadIdx.x;
    const uint16_t *x = a.residual + row * a.r_s0;
    double ss = 0.0, top = 0.0;
    int odd = 0;
    if constexpr (kWaves > 1) __syncthreads();  // the row's stores, by other waves too
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    for (int i = tid; i < a.width; i += T) {
        const double v = bf16_to_f32(x[i]), p = v * bf16_to_f32(a.weight[i]);
        ss += v * v;
        top = fmax(top, fabs(p));
        odd |= !(fabs(p) < __builtin_inf());
    }
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        ss += __shfl_xor(ss, m, kWave);
        top = fmax(top, __shfl_xor(top, m, kWave));
    }
    odd = __any(odd);
    if constexpr (kWaves > 1) {
        odd = __syncthreads_or(odd);
        if (tid % kWave == 0) {
            s_ss[tid / kWave] = ss;
            s_top[tid / kWave] = top;
        }
        __syncthreads();
        ss = 0.0;
        for (int w = 0; w < kWaves; ++w) {
            ss += s_ss[w];
            top = fmax(top, s_top[w]);
        }
    }
    const bool zero = odd || top == 0.0;
    for (int i = tid; i < a.width; i += T) {
        const double p = static_cast<double>(bf16_to_f32(x[i])) * bf16_to_f32(a.weight[i]);
        a.q[row * a.q_s0 + i] = zero ? 0 : static_cast<int8_t>(static_cast<int>(rint(127.0 * p / top)));
    }
    if (tid == 0)
        a.scales[row] = odd ? __builtin_nanf("")
                            : zero ? 1.0f : static_cast<float>(top / (127.0 * sqrt(ss / a.width + a.eps)));
}

// A workgroup of kWaves waves a row, which stays in registers between the sums and the codes up to 512 kWaves kVec
// values; what is longer is read twice.  Bound by HBM where rows are many: 4001 x 2048 (57 MB) 11.8 us, 4.9 TB/s, 5000 x
// 6144 39.7 us, 5.4 TB/s; by its launch and one round trip where they are few: 1 x 2048 2.7 us, replayed.
template <bool kAdd, int kWaves, int kVec>
__global__ void __launch_bounds__(kWaves * kWave)
norm_int8_kernel(NormInt8Args a) {
    constexpr int T = kWaves * kWave;
    __shared__ float s_ss[kWaves], s_top[kWaves];
    __shared__ int s_odd[kWaves];
    const int tid = threadIdx.x;
    const int64_t row = blockIdx.x;
    const int nvec = a.width / 8;
    const uint16_t *h = a.hidden + row * a.h_s0;
    uint16_t *r = a.residual + row * a.r_s0;
    float p[kVec][8];
    float ss = 0.f, top = 0.f;
    bool odd = false;
    // the new residual (stored) and its products with the weight
    auto sum = [&](uint4 rv, const uint4 &hv, const uint4 &wv, uint16_t *to, float (&out)[8]) __attribute__((always_inline)) {
        float x[8], w[8];
        if constexpr (kAdd) {
            float y[8];
            unpack8(rv, x);
            unpack8(hv, y);
            rv = make_uint4(pack2_bf16(x[0] + y[0], x[1] + y[1]), pack2_bf16(x[2] + y[2], x[3] + y[3]),
                            pack2_bf16(x[4] + y[4], x[5] + y[5]), pack2_bf16(x[6] + y[6], x[7] + y[7]));
            *reinterpret_cast<uint4 *>(to) = rv;
        }
        unpack8(rv, x);
        unpack8(wv, w);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            ss = fmaf(x[e], x[e], ss);
            out[e] = x[e] * w[e];
            top = fmaxf(top, fabsf(out[e]));
            odd |= !(fabsf(out[e]) < __builtin_inff());
        }
    };
    uint4 rv[kVec], hv[kVec], wv[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int vi = tid + i * T;
        const bool in = vi < nvec;
        rv[i] = in ? *reinterpret_cast<const uint4 *>(r + vi * 8) : make_uint4(0, 0, 0, 0);
        hv[i] = kAdd && in ? *reinterpret_cast<const uint4 *>(h + vi * 8) : make_uint4(0, 0, 0, 0);
        wv[i] = in ? *reinterpret_cast<const uint4 *>(a.weight + vi * 8) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int vi = tid + i * T;
        if (vi < nvec) sum(rv[i], hv[i], wv[i], r + vi * 8, p[i]);
    }
    for (int vi = tid + kVec * T; vi < nvec; vi += T) {
        float out[8];
        sum(*reinterpret_cast<const uint4 *>(r + vi * 8),
            kAdd ? *reinterpret_cast<const uint4 *>(h + vi * 8) : make_uint4(0, 0, 0, 0),
            *reinterpret_cast<const uint4 *>(a.weight + vi * 8), r + vi * 8, out);
    }
    ss = group_sum<kWave>(ss);
    top = group_max<kWave>(top);
    odd = __any(odd);
    if constexpr (kWaves > 1) {
        const int lane = tid & (kWave - 1), wave = tid / kWave;
        if (lane == 0) {
            s_ss[wave] = ss;
            s_top[wave] = top;
            s_odd[wave] = odd;
        }
        __syncthreads();
        ss = 0.f;
        int bad = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            ss += s_ss[w];
            top = fmaxf(top, s_top[w]);
            bad |= s_odd[w];
        }
        odd = bad;
    }
    // 127 p, 1 / top and the products that decide a code are normal between these; so is the sum of squares
    if (odd || !(top > 0x1p-100f && top < 0x1p100f) || !(ss > 0x1p-60f && ss < 0x1p120f)) {
        norm_int8_row_wide<kWaves>(a, row);  // the row's every thread: the tests are of its sums
        return;
    }
    const float inv = 1.0f / top;
    auto put = [&](int vi, const float (&v)[8]) __attribute__((always_inline)) {
        uint32_t c[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) c[e] = code_bits(v[e], top, inv);
        *reinterpret_cast<uint2 *>(a.q + row * a.q_s0 + vi * 8) =
            make_uint2(low_bytes(c[0], c[1], c[2], c[3]), low_bytes(c[4], c[5], c[6], c[7]));
    };
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
        const int vi = tid + i * T;
        if (vi < nvec) put(vi, p[i]);
    }
    for (int vi = tid + kVec * T; vi < nvec; vi += T) {
        float x[8], w[8], v[8];
        unpack8(*reinterpret_cast<const uint4 *>(r + vi * 8), x);  // this thread's own store
        unpack8(*reinterpret_cast<const uint4 *>(a.weight + vi * 8), w);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = x[e] * w[e];
        put(vi, v);
    }
    if (tid == 0) a.scales[row] = top / (127.0f * sqrtf(ss / static_cast<float>(a.width) + a.eps));
}

bool al(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

template <bool kAdd, int kWaves, int kVec>
int launch_as(const NormInt8Args &a, void *stream) {
    hipLaunchKernelGGL((norm_int8_kernel<kAdd, kWaves, kVec>), dim3(a.rows), dim3(kWaves * kWave), 0,
                       static_cast<hipStream_t>(stream), a);
    return NQ_LAUNCH_STATUS();
}

template <bool kAdd>
int launch(const NormInt8Args &a, void *stream) {
    const int rows = a.rows;
    NQ_CHECK_ARG(rows >= 0 && a.width >= 0);
    if (rows == 0) return NQ_OK;
    NQ_CHECK_ARG(a.residual && a.weight && a.q && a.scales && a.width >= 16 && a.eps >= 0.f);
    NQ_CHECK_ARG(a.r_s0 >= 0 && (rows == 1 || (a.q_s0 >= a.width && (!kAdd || a.r_s0 >= a.width))));
    if (a.width % 16 || !al(a.residual, 16) || !al(a.weight, 16) || !al(a.q, 8) || !al(a.scales, 4) ||
        (rows > 1 && (a.r_s0 % 8 || a.q_s0 % 8)))
        return NQ_ERR_UNSUPPORTED;
    if constexpr (kAdd) {
        NQ_CHECK_ARG(a.hidden && a.h_s0 >= 0);
        if (!al(a.hidden, 16) || (rows > 1 && a.h_s0 % 8)) return NQ_ERR_UNSUPPORTED;
    }
    // One vector of 8 a thread while that fills whole waves, up to four of them: a round trip less than with more a
    // thread, and fewer idle or waiting waves than with more threads.  Measured, us, replayed, with 1, 2 and 4 waves of one
    // vector: 100 x 512 2.76, 2.86, 2.93; 5000 x 512 5.3, 6.2, 7.9; 500 x 1024 3.67, 3.27, 3.35; 8000 x 1024 12.0, 11.9,
    // 13.2; 64 x 2048 with 1, 2, 4 waves of one and 8 of two 4.9, -, 3.0, 3.0; 4001 x 2048 12.3, -, 11.8, 15.1.  Longer
    // rows with 4 of one, 4 of four, 8 of two and 16 of one: 1 x 6144 4.0, 3.3, 3.0, 3.0; 5000 x 6144 41.5, 42.3, 39.7, 40.9.
    if (a.width <= 512) return launch_as<kAdd, 1, 1>(a, stream);
    if (a.width <= 1024) return launch_as<kAdd, 2, 1>(a, stream);
    if (a.width <= 2048) return launch_as<kAdd, 4, 1>(a, stream);
    return launch_as<kAdd, 8, 2>(a, stream);
}

}  // namespace
}  // namespace nq

extern "C" int nq_add_rmsnorm_int8(const uint16_t *hidden, int64_t h_s0, uint16_t *residual, int64_t r_s0,
                                   const uint16_t *weight, int rows, int width, float eps, int8_t *q, int64_t q_s0,
                                   float *scales, void *stream) {
    return nq::launch<true>({hidden, h_s0, residual, r_s0, weight, rows, width, eps, q, q_s0, scales}, stream);
}

extern "C" int nq_rmsnorm_int8(const uint16_t *x, int64_t x_s0, const uint16_t *weight, int rows, int width, float eps,
                               int8_t *q, int64_t q_s0, float *scales, void *stream) {
    // the rows are read alone: the kernel without the addition stores none
    return nq::launch<false>({nullptr, 0, const_cast<uint16_t *>(x), x_s0, weight, rows, width, eps, q, q_s0, scales}, stream);
}

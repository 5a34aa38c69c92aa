// Matrix products with an epilogue, for any number of rows:
//   out[m, n] = bf16(residual[m, n] + act(sum_k x[m, k] w[n, k] (* sx[m] * sw[n]) + bias[n]))
// bf16 operands with fp32 sums, or int8 codes with exact int32 sums and a scale for each row of both.  The bias, the
// activation and the residual are applied to the fp32 value, which is rounded once.
#include "nq_common.h"
#include "nq_internal.h"
#include "nq_product.h"

namespace nq {
namespace {

// The arguments that both products share.
int with_epilogue(ProductArgs &a, const uint16_t *bias, int act, const uint16_t *residual, int64_t r_s0) {
    NQ_CHECK_ARG(act >= NQ_ACT_NONE && act <= NQ_ACT_SILU);
    NQ_CHECK_ARG(!residual || r_s0 >= 0);
    NQ_CHECK_ARG(a.M == 1 || a.o_s0 >= a.N);
    if (!product_fits(a.M, a.N) || !al(a.out, 2) || !al(bias, 2) || !al(residual, 2)) return NQ_ERR_UNSUPPORTED;
    a.bias = bias;
    a.act = act;
    a.residual = residual;
    a.r_s0 = residual ? r_s0 : 0;
    a.wide = (a.M == 1 || (a.o_s0 % 8 == 0 && a.r_s0 % 8 == 0)) && al(a.out, 16) && al(residual, 16);
    return NQ_OK;
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_linear_act(const uint16_t *x, int64_t x_s0, const uint16_t *w, int64_t w_s0, int M, int N, int K,
                             const uint16_t *bias, int act, const uint16_t *residual, int64_t r_s0, uint16_t *out,
                             int64_t o_s0, void *stream) {
    NQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0);
    if (M == 0 || N == 0) return NQ_OK;
    NQ_CHECK_ARG(x && w && out && K >= 8 && x_s0 >= 0 && w_s0 >= 0);
    if (K % 8 || K > (1 << 24) || (M > 1 && x_s0 % 8) || (N > 1 && w_s0 % 8) || !al(x, 16) || !al(w, 16))
        return NQ_ERR_UNSUPPORTED;
    ProductArgs a = {reinterpret_cast<const char *>(x), 2 * x_s0, nullptr, reinterpret_cast<const char *>(w), 2 * w_s0,
                     nullptr, M, N, 2 * K, out, o_s0, 0, nullptr, nullptr, 0, 0};
    const int status = with_epilogue(a, bias, act, residual, r_s0);
    return status != NQ_OK ? status : launch_product<Bf16Op, true>(a, static_cast<hipStream_t>(stream));
}

extern "C" int nq_linear_int8_act(const int8_t *xq, int64_t x_s0, const float *sx, const int8_t *wq, int64_t w_s0,
                                  const float *sw, int M, int N, int K, const uint16_t *bias, int act,
                                  const uint16_t *residual, int64_t r_s0, uint16_t *out, int64_t o_s0, void *stream) {
    NQ_CHECK_ARG(M >= 0 && N >= 0 && K >= 0);
    if (M == 0 || N == 0) return NQ_OK;
    NQ_CHECK_ARG(xq && sx && wq && sw && out && K >= 16 && x_s0 >= 0 && w_s0 >= 0);
    if (K % 16 || K > (1 << 17) || (M > 1 && x_s0 % 16) || (N > 1 && w_s0 % 16) || !al(xq, 16) || !al(wq, 16) ||
        !al(sx, 4) || !al(sw, 4))
        return NQ_ERR_UNSUPPORTED;
    ProductArgs a = {reinterpret_cast<const char *>(xq), x_s0, sx, reinterpret_cast<const char *>(wq), w_s0, sw, M, N, K,
                     out, o_s0, 0, nullptr, nullptr, 0, 0};
    const int status = with_epilogue(a, bias, act, residual, r_s0);
    return status != NQ_OK ? status : launch_product<Int8Op, true>(a, static_cast<hipStream_t>(stream));
}

// A token a row from logits over a vocabulary of any size up to 2^20: temperature, min-p, top-k, top-p and the draw for a
// given uniform number.
//   e_i   = exp((x_i - max x) / T)          in double;  NaN logits count as -inf, -0 as 0
//   w_i   = rint(2^42 e_i), 0 where e_i < min_p: an integer, so that every sum is exact in any order and the token does
//           not depend on how the work is cut; 2^20 of them stay below 2^62
//   order : by (x desc, id asc); F(r) = sum of w over the ranks 0 .. r
//   total = F(min(k, V) - 1), k = top_k > 0 ? top_k : V
//   kept  = the ranks up to the first with F(r) >= p total (min-p and top-k leave a prefix too)
//   token = id of the first rank with F(r) >= u F(last kept)
// T not above zero: the first rank.  All three cuts and the draw are the same question, the first rank whose count or
// mass reaches a target, so a row is asked it up to three times and never sorted whole.
//
// A workgroup a row.  The logits that can have a weight (by their distance from the maximum) usually fit a list in
// LDS, which is sorted and summed there.  Where they do not, a radix descent finds the digits of the rank in question from
// histograms of counts and masses, until the ranks that share those digits fit the list.
#include "nq_common.h"
#include "nq_internal.h"

namespace nq {
namespace {

constexpr int kMinPThreads = 1024;
constexpr int kMinPWaves = kMinPThreads / kWave;
constexpr int kMinPList = 4096;           // entries of the list
constexpr int kMinPBins = 2048;
constexpr int kMinPVocab = 1 << 20;
constexpr double kMinPOne = 4398046511104.0;  // 2^42

struct MinPArgs {
    const void *logits;
    int64_t s0;
    int vocab;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p;
    const float *min_p;
    const float *uniforms;
    int64_t *tokens;
};

__device__ __forceinline__ uint64_t min_p_entry(float x, int id) {  // larger: earlier in the order
    const uint32_t u = __float_as_uint(x);
    const uint32_t key = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
    return (static_cast<uint64_t>(key) << 32) | (0xffffffffu - static_cast<uint32_t>(id));
}
__device__ __forceinline__ float entry_value(uint64_t e) {
    const uint32_t k = static_cast<uint32_t>(e >> 32);
    return __uint_as_float((k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}
__device__ __forceinline__ int entry_id(uint64_t e) {
    return static_cast<int>(0xffffffffu - static_cast<uint32_t>(e));
}
// NaN as -inf, -0 as 0
__device__ __forceinline__ float plain_logit(float x) { return x == x ? x + 0.0f : -__builtin_inff(); }

__device__ __forceinline__ uint64_t shfl_up64(uint64_t v, int d) {
    const uint32_t lo = __shfl_up(static_cast<uint32_t>(v), d, kWave);
    const uint32_t hi = __shfl_up(static_cast<uint32_t>(v >> 32), d, kWave);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t shfl64(uint64_t v, int lane) {
    const uint32_t lo = __shfl(static_cast<uint32_t>(v), lane, kWave);
    const uint32_t hi = __shfl(static_cast<uint32_t>(v >> 32), lane, kWave);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int m) {
    const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), m, kWave);
    const uint32_t hi = __shfl_xor(static_cast<uint32_t>(v >> 32), m, kWave);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {  // inclusive
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const uint64_t o = shfl_up64(v, d);
        if (lane >= d) v += o;
    }
    return v;
}

struct MinPShared {
    uint64_t list[kMinPList];
    uint64_t mass[2][kMinPBins];
    uint32_t count[2][kMinPBins];
    uint64_t part[2][kMinPWaves];
    uint64_t found_mass;
    uint64_t above_mass;
    uint32_t above_count, bin, bin_count, n;
    int found_id;
};

// Sums over the workgroup of the threads before this one; two barriers.
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t *part) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const uint64_t incl = wave_scan64(v);
    if (lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    uint64_t before = incl - v;
    for (int w = 0; w < wave; ++w) before += part[w];
    __syncthreads();
    return before;
}

// What a row's weights follow from.
struct RowRule {
    float max, least;  // least: no logit below it has a weight (a bound)
    double inv_t, min_p;
    __device__ __forceinline__ uint64_t weight(float x) const {
        if (x == max) return static_cast<uint64_t>(kMinPOne);  // an infinite one too
        const double e = exp((static_cast<double>(x) - static_cast<double>(max)) * inv_t);
        return e >= min_p ? static_cast<uint64_t>(rint(e * kMinPOne)) : 0;
    }
};

// f(id, logit) for every logit of the row, 16 bytes a load where the row's alignment allows.
template <typename InT, typename F>
__device__ __forceinline__ void each_logit(const InT *row, int vocab, F f) {
    constexpr int V = 16 / sizeof(InT), U = 4;
    const int tid = threadIdx.x;
    const int head = min(vocab, static_cast<int>((16 - reinterpret_cast<uintptr_t>(row) % 16) % 16 / sizeof(InT)));
    const int nv = (vocab - head) / V;
    auto one = [&](int id) __attribute__((always_inline)) {
        if constexpr (sizeof(InT) == 2) f(id, plain_logit(bf16_to_f32(row[id])));
        else f(id, plain_logit(row[id]));
    };
    if (tid < head) one(tid);
    const uint4 *body = reinterpret_cast<const uint4 *>(row + head);
    for (int j0 = tid; j0 < nv; j0 += U * kMinPThreads) {
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * kMinPThreads;
            v[u] = j < nv ? body[j] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u * kMinPThreads;
            if (j >= nv) break;
            const int id = head + j * V;
            if constexpr (sizeof(InT) == 2) {
                float x[8];
                unpack8(v[u], x);
#pragma unroll
                for (int e = 0; e < 8; ++e) f(id + e, plain_logit(x[e]));
            } else {
                f(id, plain_logit(__uint_as_float(v[u].x)));
                f(id + 1, plain_logit(__uint_as_float(v[u].y)));
                f(id + 2, plain_logit(__uint_as_float(v[u].z)));
                f(id + 3, plain_logit(__uint_as_float(v[u].w)));
            }
        }
    }
    const int tail = head + nv * V + tid;
    if (tail < vocab) one(tail);
}

// Sorts the list's n entries in descending order (all threads).
__device__ __forceinline__ void sort_list(MinPShared &s, int n) {
    int n2 = 2;
    while (n2 < n) n2 <<= 1;
    for (int i = n + threadIdx.x; i < n2; i += kMinPThreads) s.list[i] = 0;
    __syncthreads();
    for (int kk = 2; kk <= n2; kk <<= 1)
        for (int j = kk >> 1; j > 0; j >>= 1) {
            for (int i = threadIdx.x; i < n2 / 2; i += kMinPThreads) {
                const int lo = 2 * j * (i / j) + i % j;
                const uint64_t a = s.list[lo], b = s.list[lo + j];
                if (((lo & kk) == 0) == (a < b)) {
                    s.list[lo] = b;
                    s.list[lo + j] = a;
                }
            }
            __syncthreads();
        }
}

constexpr int kMinPEach = kMinPList / kMinPThreads;

// The sums of a sorted list: thread t has the ranks t E .. t E + E - 1, E = ceil(n / threads).
struct ListSums {
    uint64_t cum[kMinPEach];
    uint64_t before;
    int first, end;
};
__device__ __forceinline__ ListSums sum_list(MinPShared &s, int n, uint64_t above, const RowRule &rule) {
    ListSums r;
    const int each = (n + kMinPThreads - 1) / kMinPThreads;
    r.first = min(n, static_cast<int>(threadIdx.x) * each);
    r.end = min(n, r.first + each);
    uint64_t own = 0;
#pragma unroll
    for (int i = 0; i < kMinPEach; ++i) {
        if (r.first + i < r.end) own += rule.weight(entry_value(s.list[r.first + i]));
        r.cum[i] = own;
    }
    r.before = above + block_before(own, s.part[0]);
#pragma unroll
    for (int i = 0; i < kMinPEach; ++i) r.cum[i] += r.before;
    return r;
}
// The first rank whose mass reaches the target (which the list's last does): its mass and id, for every thread.
__device__ __forceinline__ void find_mass(MinPShared &s, const ListSums &r, uint64_t target) {
    uint64_t last = r.before;
#pragma unroll
    for (int i = 0; i < kMinPEach; ++i) {
        if (r.first + i < r.end && last < target && target <= r.cum[i]) {
            s.found_mass = r.cum[i];
            s.found_id = entry_id(s.list[r.first + i]);
        }
        last = r.cum[i];
    }
    __syncthreads();
}
__device__ __forceinline__ void find_rank(MinPShared &s, const ListSums &r, int rank) {
#pragma unroll
    for (int i = 0; i < kMinPEach; ++i)
        if (r.first + i < r.end && r.first + i == rank) s.found_mass = r.cum[i];
    __syncthreads();
}

// least integer target that p (in [0, 1]) of a mass asks for, at least 1
__device__ __forceinline__ uint64_t share(double p, uint64_t mass) {
    const uint64_t t = static_cast<uint64_t>(ceil(p * static_cast<double>(mass)));
    return t < 1 ? 1 : t > mass ? mass : t;
}

template <typename InT>
__global__ void __launch_bounds__(kMinPThreads)
min_p_kernel(MinPArgs a) {
    __shared__ MinPShared s;
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const InT *x = static_cast<const InT *>(a.logits) + row * a.s0;

    // 1. the first of the order
    uint64_t best = 0;
    each_logit(x, a.vocab, [&](int id, float v) {
        const uint64_t e = min_p_entry(v, id);
        best = e > best ? e : best;
    });
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
        const uint64_t o = shfl_xor64(best, m);
        best = o > best ? o : best;
    }
    if (lane == 0) s.part[0][wave] = best;
    if (tid == 0) s.n = 0;
    __syncthreads();
    best = s.part[0][0];
#pragma unroll
    for (int w = 1; w < kMinPWaves; ++w) best = s.part[0][w] > best ? s.part[0][w] : best;
    const float temperature = a.temperature[row];
    RowRule rule;
    rule.max = entry_value(best);
    if (!(temperature > 0.f) || rule.max == -__builtin_inff()) {
        if (tid == 0) a.tokens[row] = entry_id(best);
        return;
    }
    rule.inv_t = 1.0 / temperature;
    const float mp = a.min_p[row];
    rule.min_p = mp > 0.f ? (mp < 1.f ? mp : 1.0) : 0.0;
    const int kq = a.top_k[row];
    const int k = kq > 0 && kq < a.vocab ? kq : a.vocab;
    const float pq = a.top_p[row];
    const double p = pq < 1.f ? (pq > 0.f ? pq : 0.0) : 1.0;
    const float uq = a.uniforms[row];
    const double u = uq > 0.f ? (uq < 1.f ? uq : 1.0) : 0.0;
    // w >= 1 needs e >= 2^-43; the margin covers the roundings of this bound many times over
    const double reach = temperature * log(fmax(rule.min_p, 0x1p-43));
    rule.least = rule.max == __builtin_inff()
                     ? rule.max
                     : static_cast<float>(rule.max + reach - 1e-6 * (fabs(static_cast<double>(rule.max)) - reach));

    // 2. the list of those
    each_logit(x, a.vocab, [&](int id, float v) {
        if (v >= rule.least) {
            const uint32_t at = atomicAdd(&s.n, 1u);
            if (at < kMinPList) s.list[at] = min_p_entry(v, id);
        }
    });
    __syncthreads();
    const int n = static_cast<int>(s.n);
    if (n <= kMinPList) {
        sort_list(s, n);
        const ListSums sums = sum_list(s, n, 0, rule);
        find_rank(s, sums, min(k, n) - 1);
        uint64_t kept = s.found_mass;
        __syncthreads();
        if (p < 1.0) {
            find_mass(s, sums, share(p, kept));
            kept = s.found_mass;
            __syncthreads();
        }
        find_mass(s, sums, share(u, kept));
        if (tid == 0) a.tokens[row] = s.found_id;
        return;
    }

    // 3. too many: histograms of the order's digits, first of its top 11 bits
    for (int i = tid; i < kMinPBins; i += kMinPThreads) {
        s.mass[0][i] = 0;
        s.count[0][i] = 0;
    }
    __syncthreads();
    each_logit(x, a.vocab, [&](int id, float v) {
        if (v >= rule.least) {
            const uint64_t w = rule.weight(v);
            if (w) {
                const int bin = static_cast<int>(min_p_entry(v, id) >> 53);
                atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[0][bin]), w);
                atomicAdd(&s.count[0][bin], 1u);
            }
        }
    });
    __syncthreads();

    // The first rank whose count (by_mass false) or mass reaches the target, which all of them reach: s.found_mass its mass,
    // s.found_id its id.  Digits of an entry: 11, 11 and 10 bits of the logit, 10 and 10 of the id (below 2^20).
    auto locate = [&](uint64_t target, bool by_mass) {
        uint64_t prefix = 0xfff00000ull, mask = 0xfff00000ull, above_mass = 0;
        uint32_t above_count = 0;
        int shift = 64, level = 0;
        for (;; ++level) {
            const int bits = level < 2 ? 11 : 10;
            shift = level == 3 ? 10 : shift - bits;
            const int bins = 1 << bits, h = level > 0;
            if (level > 0) {
                for (int i = tid; i < bins; i += kMinPThreads) {
                    s.mass[1][i] = 0;
                    s.count[1][i] = 0;
                }
                __syncthreads();
                each_logit(x, a.vocab, [&](int id, float v) {
                    const uint64_t e = min_p_entry(v, id);
                    if (v >= rule.least && (e & mask) == prefix) {
                        const uint64_t w = rule.weight(v);
                        if (w) {
                            const int bin = static_cast<int>(e >> shift) & (bins - 1);
                            atomicAdd(reinterpret_cast<unsigned long long *>(&s.mass[1][bin]), w);
                            atomicAdd(&s.count[1][bin], 1u);
                        }
                    }
                });
                __syncthreads();
            }
            // thread t: the digits bins - 1 - 2 t and the next below
            uint64_t m[2] = {0, 0};
            uint32_t c[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int bin = bins - 1 - 2 * tid - i;
                if (bin >= 0) {
                    m[i] = s.mass[h][bin];
                    c[i] = s.count[h][bin];
                }
            }
            uint64_t bm = above_mass + block_before(m[0] + m[1], s.part[0]);
            uint32_t bc = above_count + static_cast<uint32_t>(block_before(c[0] + c[1], s.part[1]));
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint64_t from = by_mass ? bm : bc, to = from + (by_mass ? m[i] : c[i]);
                if (from < target && target <= to) {
                    s.bin = static_cast<uint32_t>(bins - 1 - 2 * tid - i);
                    s.bin_count = c[i];
                    s.above_mass = bm;
                    s.above_count = bc;
                }
                bm += m[i];
                bc += c[i];
            }
            if (tid == 0) s.n = 0;
            __syncthreads();
            above_mass = s.above_mass;
            above_count = s.above_count;
            prefix |= static_cast<uint64_t>(s.bin) << shift;
            mask |= static_cast<uint64_t>(bins - 1) << shift;
            const bool fits = s.bin_count <= kMinPList;
            __syncthreads();
            if (fits) break;  // at the last level: one entry
        }
        each_logit(x, a.vocab, [&](int id, float v) {
            const uint64_t e = min_p_entry(v, id);
            if (v >= rule.least && (e & mask) == prefix && rule.weight(v)) {
                const uint32_t at = atomicAdd(&s.n, 1u);
                if (at < kMinPList) s.list[at] = e;
            }
        });
        __syncthreads();
        const int m = min(static_cast<int>(s.n), kMinPList);
        sort_list(s, m);
        const ListSums sums = sum_list(s, m, above_mass, rule);
        if (by_mass) find_mass(s, sums, target);
        else find_rank(s, sums, static_cast<int>(target - above_count) - 1);
        const uint64_t mass = s.found_mass;
        __syncthreads();
        return mass;
    };
    // all of them, from the histogram
    uint64_t m = 0, c = 0;
    for (int i = tid; i < kMinPBins; i += kMinPThreads) {
        m += s.mass[0][i];
        c += s.count[0][i];
    }
    const uint64_t m0 = block_before(m, s.part[0]), c0 = block_before(c, s.part[1]);
    if (tid == kMinPThreads - 1) {
        s.found_mass = m0 + m;
        s.above_mass = c0 + c;
    }
    __syncthreads();
    uint64_t total = s.found_mass;
    const uint64_t weighted = s.above_mass;
    __syncthreads();
    if (static_cast<uint64_t>(k) < weighted) total = locate(k, false);
    const uint64_t kept = p < 1.0 ? locate(share(p, total), true) : total;
    locate(share(u, kept), true);
    if (tid == 0) a.tokens[row] = s.found_id;
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_sample_min_p(const void *logits, int logits_dtype, int64_t logits_s0, int rows, int vocab,
                               const float *temperature, const int32_t *top_k, const float *top_p, const float *min_p,
                               const float *uniforms, int64_t *tokens, void *stream) {
    NQ_CHECK_ARG(rows >= 0 && vocab >= 0);
    if (rows == 0) return NQ_OK;
    NQ_CHECK_ARG(logits && temperature && top_k && top_p && min_p && uniforms && tokens && vocab >= 1 && logits_s0 >= 0);
    if (vocab > kMinPVocab || (logits_dtype != NQ_F32 && logits_dtype != NQ_BF16)) return NQ_ERR_UNSUPPORTED;
    if (reinterpret_cast<uintptr_t>(logits) % (logits_dtype == NQ_F32 ? 4 : 2)) return NQ_ERR_UNSUPPORTED;
    const MinPArgs a = {logits, logits_s0, vocab, temperature, top_k, top_p, min_p, uniforms, tokens};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (logits_dtype == NQ_F32)
        hipLaunchKernelGGL(min_p_kernel<float>, dim3(rows), dim3(kMinPThreads), 0, st, a);
    else
        hipLaunchKernelGGL(min_p_kernel<uint16_t>, dim3(rows), dim3(kMinPThreads), 0, st, a);
    return NQ_LAUNCH_STATUS();
}

// The paged K/V cache in 8 bits: int8 codes in the pages' own layout
// [pages, 2, page_size, Hkv, D] and one fp32 scale for each block of 16 slots,
// kind (K, V) and kv head; its write, its read back, and the attention over it.
//
// Write.  A block's scale is a power of two, the least s with max |x| / s <= 127
// over the tokens it holds, so x / s and a rescale of the codes by old / new are
// exact up to the one rounding (ties to even): the codes do not depend on how the
// arithmetic is carried out, a block is rescaled only when its range grows by a
// factor of two, and the roundings of all its rescales add up to less than one
// step (1/2 + 1/4 + ...).  The price is a step of up to twice max |x| / 127.
//
// Attention.  S = q . c_K with the codes widened to bf16 (exact), each block's
// scale applied to its 16 columns of fp32 scores.  P V in bf16 with fp32 sums: in
// decode V's scale multiplies P before it is rounded to bf16 and V's codes are
// widened as they are; in prefill P is rounded alone (2^-8 of a weight either way, as
// the bf16 cache's attention rounds it) and V's codes are widened times their scale.
// So the cache moves half the bytes of a bf16 one and is never written out wider.
#include <stddef.h>

#include <type_traits>

#include "nq_common.h"
#include "nq_internal.h"

namespace nq {
namespace {

constexpr int kBlk = 16;  // slots that share a scale
constexpr int kKv8Threads = 256;
constexpr int kKv8Waves = kKv8Threads / kWave;
constexpr float kMinScale = 1.1754943508222875e-38f;  // 2^-126

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
typedef float floatx16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));  // plain vectors stay in registers
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

struct Pool8 {
    int8_t *codes;
    int64_t c_page, c_kind, c_slot, c_head;
    float *scales;
    int64_t s_page, s_kind, s_block, s_head;
    int num_pages, page_size;
};

// Least power of two s >= 2^-126 with amax / s <= 127 (amax finite, >= 0): amax = m 2^E, 1 <= m < 2,
// gives 2^(E - 6) where m <= 127 / 64, else 2^(E - 5).
__device__ __forceinline__ float scale_for(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 6 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return e < 1 ? kMinScale : __uint_as_float(static_cast<uint32_t>(e) << 23);
}

// What scales are: anything else (NaN, an infinity, a negative number) makes the queries that see its block NaN.
__device__ __forceinline__ bool is_scale(float s) { return s >= 0.f && s < __builtin_inff(); }

__device__ __forceinline__ uint32_t pack4_i8(float a, float b, float c, float d) {
    const int ia = static_cast<int>(rintf(a)), ib = static_cast<int>(rintf(b)), ic = static_cast<int>(rintf(c)),
              id = static_cast<int>(rintf(d));
    return (ia & 0xff) | ((ib & 0xff) << 8) | ((ic & 0xff) << 16) | (static_cast<uint32_t>(id) << 24);
}

template <int B>
__device__ __forceinline__ float byte_f32(uint32_t w) {
    return static_cast<float>(static_cast<int8_t>(w >> (8 * B)));
}

__device__ __forceinline__ float byte_of(uint32_t w, int j) { return static_cast<float>(static_cast<int8_t>(w >> (8 * j))); }

// Eight codes widened to bf16: integers of at most 8 bits, so the upper half of the float is exact.
__device__ __forceinline__ uint32_t pair_bf16(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ bf16x8_t widen8(uint32_t a, uint32_t b) {
    const u32x4 r = {pair_bf16(byte_f32<0>(a), byte_f32<1>(a)), pair_bf16(byte_f32<2>(a), byte_f32<3>(a)),
                     pair_bf16(byte_f32<0>(b), byte_f32<1>(b)), pair_bf16(byte_f32<2>(b), byte_f32<3>(b))};
    return __builtin_bit_cast(bf16x8_t, r);
}
// ---------------------------------------------------------------------------------------------
// Write: a wave takes the leaders among `group` consecutive tokens for one (kind, head).  A leader is a
// token that does not continue its predecessor's block (same page, next slot, same block of 16); its run
// are the tokens behind it that do.  So the slot map alone says who owns a block, a run's tokens are
// quantised with one scale, and a block's earlier slots are read only by the wave that may rescale them.
// Lane l holds slots l / (D/8) + i * (512/D), values 8 (l % (D/8)) .. + 7.
// Bound by its chain of loads (slots, then the block's scale and tokens) where tokens are few: 64 single tokens 4.5 us,
// 4 of them the launch and the chain.  Where they are many, 7677 tokens of 8 heads of 128 (47 MB) 14.8 us, 3.2 TB/s: 95 VGPRs
// hold five waves a SIMD, so its 7680 waves are a round and a half, each of which loads first and stores last (they wait in 51 %
// of their clocks, the vector units run in 31 %).
template <int D>
__global__ void __launch_bounds__(kKv8Threads)
kv8_write_kernel(const uint16_t *__restrict__ key, int64_t k_s0, int64_t k_s1, const uint16_t *__restrict__ value,
                 int64_t v_s0, int64_t v_s1, const int64_t *__restrict__ pages, const int64_t *__restrict__ offsets,
                 int tokens, int heads, int group, Pool8 pool, int32_t *__restrict__ status) {
    constexpr int LPT = D / 8, SPI = kWave / LPT, ITERS = kBlk / SPI;
    const int lane = threadIdx.x & (kWave - 1);
    const int which = blockIdx.y * kKv8Waves + threadIdx.x / kWave;
    if (which >= 2 * heads) return;
    const int kind = which >= heads ? 1 : 0, head = which - kind * heads;
    const int base = blockIdx.x * group;

    // lane i: token base - 1 + i and whether it continues token base - 2 + i
    const int t = base - 1 + lane;
    const bool in = lane < 33 && t >= 0 && t < tokens;
    const int64_t page = in ? pages[t] : -1, off = in ? offsets[t] : -1;
    const bool ok = in && page >= 0 && page < pool.num_pages && off >= 0 && off < pool.page_size;
    if (in && !ok && lane >= 1 && lane <= group && which == 0 && status) *status = NQ_ERR_INVALID_ARGUMENT;
    const int ipage = ok ? static_cast<int>(page) : -1, ioff = ok ? static_cast<int>(off) : -1;
    const int p_page = __shfl_up(ipage, 1, kWave), p_off = __shfl_up(ioff, 1, kWave);
    const bool cont = ok && lane >= 1 && p_page == ipage && ioff == p_off + 1 && (ioff & (kBlk - 1)) != 0;
    const uint64_t follows = __ballot(cont), valid = __ballot(ok);

    const uint16_t *src = kind ? value : key;
    const int64_t s0 = kind ? v_s0 : k_s0, s1 = kind ? v_s1 : k_s1;
    const int part = lane % LPT, slot0 = lane / LPT;
    for (int i = 1; i <= group; ++i) {
        if (!((valid >> i) & 1) || ((follows >> i) & 1)) continue;
        const uint64_t behind = ~(follows >> (i + 1));
        const int run = 1 + __builtin_ctzll(behind);  // at most 16: a block's first slot never follows
        const int pg = __builtin_amdgcn_readlane(ipage, i), of = __builtin_amdgcn_readlane(ioff, i);
        const int first = of & (kBlk - 1);
        int8_t *dst = pool.codes + pg * pool.c_page + kind * pool.c_kind + (of - first) * pool.c_slot +
                      head * pool.c_head + part * 8;
        float *sp = pool.scales + pg * pool.s_page + kind * pool.s_kind + (of / kBlk) * pool.s_block +
                    head * pool.s_head;
        const uint16_t *row = src + (base + i - 1) * s0 + head * s1 + part * 8;
        const float old = first ? *sp : 0.f;
        uint4 x[ITERS];
        uint2 held[ITERS];
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int slot = slot0 + k * SPI;
            const bool fresh = slot >= first && slot < first + run;
            x[k] = fresh ? *reinterpret_cast<const uint4 *>(row + (slot - first) * s0) : make_uint4(0, 0, 0, 0);
            held[k] = slot < first ? *reinterpret_cast<const uint2 *>(dst + slot * pool.c_slot) : make_uint2(0, 0);
        }
        float amax = 0.f;
        bool odd = false;  // NaN or infinity among the new values
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            float f[8];
            unpack8(x[k], f);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                amax = fmaxf(amax, fabsf(f[e]));
                odd |= !(fabsf(f[e]) < __builtin_inff());
            }
        }
        amax = group_max<kWave>(amax);
        // what was no scale becomes NaN and stays: every query that reads the block answers NaN
        const bool bad = __any(odd) || !is_scale(old);
        const float own = scale_for(amax);
        const float s = bad ? __builtin_nanf("") : (first && old > own ? old : own);
        const float inv = bad ? 0.f : 1.0f / s;  // exact: s is a power of two, at most 2^122
        const float shrink = bad ? 1.f : old / s;
#pragma unroll
        for (int k = 0; k < ITERS; ++k) {
            const int slot = slot0 + k * SPI;
            if (slot >= first && slot < first + run) {
                float f[8];
                unpack8(x[k], f);
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = bad ? 0.f : f[e] * inv;
                *reinterpret_cast<uint2 *>(dst + slot * pool.c_slot) =
                    make_uint2(pack4_i8(f[0], f[1], f[2], f[3]), pack4_i8(f[4], f[5], f[6], f[7]));
            } else if (slot < first && shrink != 1.f) {
                const uint32_t a = held[k].x, b = held[k].y;
                *reinterpret_cast<uint2 *>(dst + slot * pool.c_slot) = make_uint2(
                    pack4_i8(byte_f32<0>(a) * shrink, byte_f32<1>(a) * shrink, byte_f32<2>(a) * shrink,
                             byte_f32<3>(a) * shrink),
                    pack4_i8(byte_f32<0>(b) * shrink, byte_f32<1>(b) * shrink, byte_f32<2>(b) * shrink,
                             byte_f32<3>(b) * shrink));
            }
        }
        if (lane == 0) *sp = s;
    }
}

// ---------------------------------------------------------------------------------------------
// Read back: thread per 16 codes of one (token, kind, head).  Bound by HBM: 7677 tokens of 8 heads of 128 (47 MB) 10.7 us,
// 4.4 TB/s.
template <int D>
__global__ void __launch_bounds__(kKv8Threads)
kv8_read_kernel(Pool8 pool, const int64_t *__restrict__ pages, const int64_t *__restrict__ offsets, int tokens,
                int heads, uint16_t *__restrict__ key, int64_t k_s0, int64_t k_s1, uint16_t *__restrict__ value,
                int64_t v_s0, int64_t v_s1, int32_t *__restrict__ status) {
    constexpr int VEC = D / 16;
    const int64_t at = static_cast<int64_t>(blockIdx.x) * kKv8Threads + threadIdx.x;
    const int per = 2 * heads * VEC;
    const int64_t t = at / per;
    if (t >= tokens) return;
    int rest = static_cast<int>(at - t * per);
    const int vec = rest % VEC;
    rest /= VEC;
    const int head = rest % heads, kind = rest / heads;
    const int64_t page = pages[t], off = offsets[t];
    uint16_t *dst = kind ? value + t * v_s0 + head * v_s1 : key + t * k_s0 + head * k_s1;
    uint4 *o = reinterpret_cast<uint4 *>(dst + vec * 16);
    if (page < 0 || page >= pool.num_pages || off < 0 || off >= pool.page_size) {
        if (status) *status = NQ_ERR_INVALID_ARGUMENT;
        o[0] = o[1] = make_uint4(0, 0, 0, 0);
        return;
    }
    const uint4 c = *reinterpret_cast<const uint4 *>(pool.codes + page * pool.c_page + kind * pool.c_kind +
                                                     off * pool.c_slot + head * pool.c_head + vec * 16);
    const float s = pool.scales[page * pool.s_page + kind * pool.s_kind + (off / kBlk) * pool.s_block +
                                head * pool.s_head];
    auto four = [&](uint32_t w) {
        return make_uint2(pack2_bf16(byte_f32<0>(w) * s, byte_f32<1>(w) * s),
                          pack2_bf16(byte_f32<2>(w) * s, byte_f32<3>(w) * s));
    };
    const uint2 a = four(c.x), b = four(c.y), d = four(c.z), e = four(c.w);
    o[0] = make_uint4(a.x, a.y, b.x, b.y);
    o[1] = make_uint4(d.x, d.y, e.x, e.y);
}

// ---------------------------------------------------------------------------------------------
// Attention.
constexpr float kLog2e8 = 1.4426950408889634f;

struct Attend8 {
    const uint16_t *q;
    int64_t q_s0, q_s1;
    uint16_t *out;
    int64_t o_s0, o_s1;
    const int32_t *qo_indptr, *kv_indptr, *kv_indices, *last_page_len;
    int rows, tokens, n_indices, group, heads;  // group: query heads per kv head
    int bpp_log2;                               // blocks of 16 per page
    float scale;                                // |sm_scale| log2(e), above 0
    uint32_t flip;                              // sign bits of a bf16 pair where sm_scale is negative
    int32_t *status;
};

// The larger (the sum) of a lane's value and that of the lane 32 on or back.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float halves_sum(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// The same over lanes 16, 32 and 48 on.
__device__ __forceinline__ float quarters_max(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return halves_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// Largest r in [0, n) with f(r) <= x for a non-decreasing f with f(0) <= x, found by the whole wave: 64
// probes at once, so one round of loads up to 64 rows and two up to 4096.
template <typename F>
__device__ __forceinline__ int wave_find_le(int n, int x, F f) {
    const int lane = threadIdx.x & (kWave - 1);
    int lo = 0, count = n;
    while (count > 1) {
        const int step = (count + kWave - 1) / kWave;
        const int at = lane * step;
        const bool le = at < count && f(lo + at) <= x;
        const uint64_t m = __ballot(le);
        const int hit = m ? 63 - __builtin_clzll(m) : 0;
        lo += hit * step;
        count = step < count - hit * step ? step : count - hit * step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

// The ragged metadata, copied to LDS at entry (one round trip, then searches and row changes cost LDS reads);
// read in place beyond kMetaRows rows.
constexpr int kMetaRows = 512;
struct Meta8 {
    int32_t kv[kMetaRows + 1], qo[kMetaRows + 1], last[kMetaRows];
};
struct Rows8 {
    const Attend8 &a;
    const Meta8 &m;
    __device__ __forceinline__ bool held() const { return a.rows <= kMetaRows; }
    __device__ __forceinline__ int kv(int i) const { return held() ? m.kv[i] : a.kv_indptr[i]; }
    __device__ __forceinline__ int qo(int i) const {
        if (!a.qo_indptr) return i;
        return held() ? m.qo[i] : a.qo_indptr[i];
    }
    __device__ __forceinline__ int last(int i) const { return held() ? m.last[i] : a.last_page_len[i]; }
};
struct InPlace8 {  // the same without the copy, for kernels that look at one row
    const Attend8 &a;
    __device__ __forceinline__ int kv(int i) const { return a.kv_indptr[i]; }
    __device__ __forceinline__ int qo(int i) const { return a.qo_indptr ? a.qo_indptr[i] : i; }
    __device__ __forceinline__ int last(int i) const { return a.last_page_len[i]; }
};
__device__ __forceinline__ void load_meta(const Attend8 &a, Meta8 &m) {
    if (a.rows <= kMetaRows) {
        for (int i = threadIdx.x; i <= a.rows; i += blockDim.x) {
            m.kv[i] = a.kv_indptr[i];
            if (a.qo_indptr) m.qo[i] = a.qo_indptr[i];
            if (i < a.rows) m.last[i] = a.last_page_len[i];
        }
    }
    __syncthreads();
}

// What a row asks for.
struct Row8 {
    int first_page, n_pages, kv_len, q0, q_len;
};
template <typename R>
__device__ __forceinline__ Row8 row_of(const Attend8 &a, const R &rows, int r) {
    Row8 w;
    const int first = __builtin_amdgcn_readfirstlane(rows.kv(r)), end = __builtin_amdgcn_readfirstlane(rows.kv(r + 1));
    const int b = first < 0 ? 0 : (first > a.n_indices ? a.n_indices : first);
    const int e = end < b ? b : (end > a.n_indices ? a.n_indices : end);
    if ((b != first || e != end) && a.status) *a.status = NQ_ERR_INVALID_ARGUMENT;
    w.first_page = b;
    w.n_pages = e - b;
    const int ps = kBlk << a.bpp_log2;
    int last = __builtin_amdgcn_readfirstlane(rows.last(r));
    last = last < 1 ? 1 : (last > ps ? ps : last);
    w.kv_len = w.n_pages > 0 ? (w.n_pages - 1) * ps + last : 0;
    w.q0 = __builtin_amdgcn_readfirstlane(rows.qo(r));
    w.q_len = __builtin_amdgcn_readfirstlane(rows.qo(r + 1)) - w.q0;
    if (w.q0 < 0 || w.q_len < 0 || w.q0 > a.tokens - w.q_len) w.q_len = 0;  // not this call's queries
    return w;
}

__device__ __forceinline__ bf16x8_t load_q(const uint16_t *p, bool on, uint32_t flip) {
    u32x4 v = {0, 0, 0, 0};
    if (on) v = *reinterpret_cast<const u32x4 *>(p) ^ flip;
    return __builtin_bit_cast(bf16x8_t, v);
}

// Decode rows.  The blocks of all rows, in kv_indices order, are cut into equal spans, one a wave of every
// kv head; kv_indptr itself is the prefix sum that says whose a block is, so there is no plan launch.
// A row inside one span is finished by its wave; a row over several leaves (m, l, o) partials, which
// kv8_merge_kernel joins in order.
struct Spans {
    int64_t blocks;
    int waves;
};
template <typename R>
__device__ __forceinline__ Spans spans_of(const Attend8 &a, const R &rows, int waves) {
    int p = __builtin_amdgcn_readfirstlane(rows.kv(a.rows));
    p = p < 0 ? 0 : (p > a.n_indices ? a.n_indices : p);
    Spans s;
    s.blocks = static_cast<int64_t>(p) << a.bpp_log2;
    const int64_t most = (s.blocks + 1) / 2;  // a wave's step is two blocks
    s.waves = static_cast<int>(most < waves ? (most < 1 ? 1 : most) : waves);
    return s;
}
__device__ __forceinline__ int64_t span_start(const Spans &s, int64_t i) { return i * s.blocks / s.waves; }
// the span that holds block b: the largest i with span_start(i) <= b
__device__ __forceinline__ int span_of(const Spans &s, int64_t b) {
    return static_cast<int>(((b + 1) * s.waves + s.blocks - 1) / s.blocks) - 1;
}

// A step: 32 keys (two blocks).  S^T = K Q^T with mfma_16x16x32: lane l loads token l % 16 of each block, values
// (D/4)(l / 16) .. of K, and holds the scores of query slot l % 16 against tokens 4 (l / 16) + i.  Those are, in
// that order, the 8 keys of the lane's group in out^T = V^T P^T, so P needs no exchange between lanes; V is loaded
// as (D/16) values of each of the 8 tokens, and the byte a conversion picks does the transposition.
// K of the next step is asked for as soon as this one's is multiplied, V likewise: one set of registers, and loads always
// in flight.  Each byte is read once, so the loads are non-temporal: 64 rows of 66 to 2047 keys (135 MB) take 31.8 us
// instead of 34.4, 3 rows of about 50000 (308 MB) 56.3 instead of 60.0, 5.5 TB/s.  Two waves a SIMD: with plain
// loads three took as long and four (registers spilled) 49.6 and 81.7 us.
template <int D>
__global__ void __launch_bounds__(kKv8Threads, 2)
kv8_decode_kernel(Attend8 a, Pool8 pool, int waves, float2 *__restrict__ part_ml, float *__restrict__ part_o) {
    constexpr int W = D / 64;  // 16-byte loads of K, dwords of V
    __shared__ Meta8 meta;
    load_meta(a, meta);
    const Rows8 rows{a, meta};
    const int lane = threadIdx.x & (kWave - 1);
    // XCD x (workgroups x, x + 8, ..) takes spans x, x + 8, .. of every head: the heads of a span read the same
    // token rows at about the same time, from one L2
    const int unit = __builtin_amdgcn_readfirstlane((blockIdx.x / 8) * kKv8Waves + threadIdx.x / kWave);
    const int head = unit % a.heads;
    const int wi = unit / a.heads * 8 + static_cast<int>(blockIdx.x % 8);
    const Spans sp = spans_of(a, rows, waves);
    if (wi >= sp.waves) return;
    const int b0 = static_cast<int>(span_start(sp, wi)), b1 = static_cast<int>(span_start(sp, wi + 1));
    if (b0 >= b1) return;
    const int c = lane & 15, grp = lane >> 4;

    const int8_t *kbase = pool.codes + head * pool.c_head;
    const int8_t *vbase = kbase + pool.c_kind;
    const int c_slot = static_cast<int>(pool.c_slot);
    const int k_lane = c * c_slot + grp * (D / 4);
    const int v_lane = 4 * grp * c_slot + c * (D / 16);
    const int in_page = (1 << a.bpp_log2) - 1;

    // a window of 64 blocks' pages and scales, one a lane
    int wbase = b0;
    int w_pid = 0;
    float w_ks = 0.f, w_vs = 0.f;
    auto open_window = [&](int b) __attribute__((always_inline)) {
        wbase = b;
        const int mine = b + lane;
        w_pid = -1;
        w_ks = w_vs = 0.f;
        if (mine < b1) {
            const int pid = a.kv_indices[mine >> a.bpp_log2];
            if (pid >= 0 && pid < pool.num_pages) {
                const float *s = pool.scales + pid * pool.s_page + (mine & in_page) * pool.s_block + head * pool.s_head;
                // What is no scale, K's or V's, answers through the scores of the rows that see the block: as a V factor
                // it would be lost where a probability vanishes, and infinite K factors can drop a block's keys.
                const float ks = s[0], vs = s[pool.s_kind];
                const bool fine = is_scale(ks) && is_scale(vs);
                w_pid = pid;
                w_ks = fine ? ks : __builtin_nanf("");
                w_vs = fine ? vs : 0.f;
            } else if (a.status) {
                *a.status = NQ_ERR_INVALID_ARGUMENT;
            }
        }
    };
    struct Blocks {  // the two blocks of a step (the second repeats the first at the span's end)
        int at;
        int64_t off[2];
        float ks[2], vs[2];
        bool on[2];
    };
    auto look = [&](int b) __attribute__((always_inline)) {
        if (b + 1 >= wbase + kWave) open_window(b);
        Blocks n;
        n.at = b;
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const int blk = m && b + 1 < b1 ? b + 1 : b;
            const int pid = __builtin_amdgcn_readlane(w_pid, blk - wbase);
            n.on[m] = pid >= 0;
            n.ks[m] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w_ks), blk - wbase));
            n.vs[m] = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w_vs), blk - wbase));
            n.off[m] = (pid < 0 ? 0 : pid) * pool.c_page + (blk & in_page) * (kBlk * pool.c_slot);
        }
        return n;
    };
    u32x4 k[2][W];
    u32x2 v[8];
    auto load_k = [&](const Blocks &n) __attribute__((always_inline)) {
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int w = 0; w < W; ++w)
                k[m][w] =
                    __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kbase + n.off[m] + (k_lane + 16 * w)));
    };
    auto load_v = [&](const Blocks &n) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int8_t *p = vbase + n.off[e / 4] + (v_lane + (e % 4) * c_slot);
            if constexpr (W == 2) v[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p));
            else v[e].x = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p));
        }
    };

    open_window(b0);
    Blocks cur = look(b0);
    load_k(cur);
    load_v(cur);
    // the row of the first block
    int r = wave_find_le(a.rows, b0 >> a.bpp_log2, [&](int i) { return rows.kv(i); });
    int b = b0;
    while (b < b1 && r < a.rows) {
        const Row8 row = row_of(a, rows, r);
        const int rs = row.first_page << a.bpp_log2, re = (row.first_page + row.n_pages) << a.bpp_log2;
        if (re <= b) {
            ++r;
            continue;
        }
        if (rs > b) {  // pages of no row
            b = rs < b1 ? rs : b1;
            continue;
        }
        const int stop = re < b1 ? re : b1;
        if (row.q_len != 1) {
            b = stop;
            ++r;
            continue;
        }
        bf16x8_t qf[D / 32];
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
            qf[s] = load_q(a.q + row.q0 * a.q_s0 + (head * a.group + c) * a.q_s1 + grp * (D / 4) + 8 * s, c < a.group,
                           a.flip);
        if (cur.at != b) {  // behind pages that are not this launch's
            cur = look(b);
            load_k(cur);
            load_v(cur);
        }
        floatx4_t acc[D / 16];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) acc[j] = floatx4_t{0.f, 0.f, 0.f, 0.f};
        float m_run = -__builtin_inff(), l_run = 0.f;
        bool any = false;
        for (; b < stop; b += 2) {
            int nv[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int left = row.kv_len - (b + m - rs) * kBlk;
                nv[m] = b + m < stop && cur.on[m] && left > 0 ? (left < kBlk ? left : kBlk) : 0;
            }
            any |= nv[0] + nv[1] > 0;
            float p[8];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                floatx4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = 0; w < W; ++w) {
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(k[m][w].x, k[m][w].y), qf[2 * w], s, 0, 0, 0);
                    s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen8(k[m][w].z, k[m][w].w), qf[2 * w + 1], s, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) p[4 * m + i] = s[i];
                __builtin_amdgcn_sched_barrier(0);
            }
            const float f[2] = {cur.ks[0] * a.scale, cur.ks[1] * a.scale}, vs[2] = {cur.vs[0], cur.vs[1]};
            const int ahead = b + 2 < stop ? b + 2 : stop;
            if (ahead < b1) {
                cur = look(ahead);
                load_k(cur);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i)
                p[i] = 4 * grp + (i & 3) < nv[i / 4] ? p[i] * f[i / 4] : -__builtin_inff();
            float top = fmaxf(fmaxf(fmaxf(p[0], p[1]), fmaxf(p[2], p[3])), fmaxf(fmaxf(p[4], p[5]), fmaxf(p[6], p[7])));
            top = quarters_max(top);
            const float m_new = fmaxf(m_run, top);
            if (__any(m_new != m_run)) {
                const float alpha = m_run == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
                l_run *= alpha;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) acc[j] *= alpha;
                m_run = m_new;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                p[i] = 4 * grp + (i & 3) < nv[i / 4] ? __builtin_amdgcn_exp2f(p[i] - m_run) : 0.f;
                l_run += p[i];
                p[i] *= vs[i / 4];
            }
            const u32x4 pw = {pack2_bf16(p[0], p[1]), pack2_bf16(p[2], p[3]), pack2_bf16(p[4], p[5]),
                              pack2_bf16(p[6], p[7])};
            const bf16x8_t pf = __builtin_bit_cast(bf16x8_t, pw);
#pragma unroll
            for (int w = 0; w < W; ++w) {
#define NQ_V_FRAG(J)                                                                                                   \
    {                                                                                                                  \
        const u32x4 vw = {                                                                                             \
            pair_bf16(byte_f32<J>(v[0][w]), byte_f32<J>(v[1][w])), pair_bf16(byte_f32<J>(v[2][w]), byte_f32<J>(v[3][w])), \
            pair_bf16(byte_f32<J>(v[4][w]), byte_f32<J>(v[5][w])), pair_bf16(byte_f32<J>(v[6][w]), byte_f32<J>(v[7][w]))}; \
        acc[4 * w + J] =                                                                                               \
            __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, vw), pf, acc[4 * w + J], 0, 0, 0);    \
    }
                NQ_V_FRAG(0)
                NQ_V_FRAG(1)
                __builtin_amdgcn_sched_barrier(0);
                NQ_V_FRAG(2)
                NQ_V_FRAG(3)
                __builtin_amdgcn_sched_barrier(0);
#undef NQ_V_FRAG
            }
            if (ahead < b1) load_v(cur);
        }
        b = stop;
        l_run += __shfl_xor(l_run, 16, kWave);
        l_run += __shfl_xor(l_run, 32, kWave);
        // the lane holds out[slot c][(D/4) grp + (D/16) i + j] in acc[j][i]
        if (c < a.group) {
            if (rs >= b0 && re <= b1) {
                const float inv = any ? 1.0f / l_run : 0.f;
                uint16_t *o = a.out + row.q0 * a.o_s0 + (head * a.group + c) * a.o_s1 + grp * (D / 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[D / 32];
#pragma unroll
                    for (int j = 0; j < D / 32; ++j) w[j] = pack2_bf16(acc[2 * j][i] * inv, acc[2 * j + 1][i] * inv);
                    if constexpr (D == 128)
                        *reinterpret_cast<u32x4 *>(o + 8 * i) = u32x4{w[0], w[1], w[2], w[3]};
                    else
                        *reinterpret_cast<u32x2 *>(o + 4 * i) = u32x2{w[0], w[1]};
                }
            } else {
                const int64_t slot = ((static_cast<int64_t>(head) * waves + wi) * 2 + (rs >= b0 ? 1 : 0)) * a.group + c;
                if (grp == 0) part_ml[slot] = make_float2(m_run, l_run);
                float *o = part_o + slot * D + grp * (D / 4);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < D / 16; j += 4)
                        *reinterpret_cast<float4 *>(o + (D / 16) * i + j) =
                            make_float4(acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]);
            }
        }
        if (re <= b1) ++r;
    }
}

// Joins a decode row's partials: span i0, where the row begins, left its slot 1, the spans behind it slot 0.
// Weights 2^(m_i - m), in span order.  A row without pages gets zeros.  A workgroup takes one query head:
// D/4 threads a partial, 1024 / D partials at a time, four rounds of loads in flight.  Bound by its launch and two
// dependent loads: 4.2 us for 64 rows of 16 heads, 5.6 us where 3 rows left 2048 partials.
template <int D>
__global__ void __launch_bounds__(kKv8Threads)
kv8_merge_kernel(Attend8 a, int waves, const float2 *__restrict__ part_ml, const float *__restrict__ part_o) {
    constexpr int TP = D / 4, AT = kKv8Threads / TP;  // threads a partial, partials at a time
    __shared__ float s_red[2][kKv8Waves];
    __shared__ float4 s_o[AT][TP];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int r = blockIdx.x, head = blockIdx.y / a.group, g = blockIdx.y % a.group;
    const InPlace8 rows{a};
    const Spans sp = spans_of(a, rows, waves);
    const Row8 row = row_of(a, rows, r);
    if (row.q_len != 1) return;
    uint16_t *out = a.out + row.q0 * a.o_s0 + (head * a.group + g) * a.o_s1;
    // a row behind the batch's last page (a kv_indptr that decreases) was in no span
    const bool outside = (static_cast<int64_t>(row.first_page + row.n_pages) << a.bpp_log2) > sp.blocks;
    if (row.n_pages == 0 || outside) {
        if (threadIdx.x < TP) *reinterpret_cast<u32x2 *>(out + 4 * threadIdx.x) = u32x2{0, 0};
        return;
    }
    const int64_t rs = static_cast<int64_t>(row.first_page) << a.bpp_log2;
    const int64_t re = static_cast<int64_t>(row.first_page + row.n_pages) << a.bpp_log2;
    const int i0 = span_of(sp, rs), n = span_of(sp, re - 1) - i0 + 1;
    if (n == 1) return;
    const int64_t base = static_cast<int64_t>(head) * waves + i0;
    auto slot = [&](int i) __attribute__((always_inline)) { return ((base + i) * 2 + (i == 0 ? 1 : 0)) * a.group + g; };
    float m = -__builtin_inff();
    for (int i = threadIdx.x; i < n; i += kKv8Threads) m = fmaxf(m, part_ml[slot(i)].x);
    m = group_max<kWave>(m);
    if (lane == 0) s_red[0][wave] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kKv8Waves; ++w) m = fmaxf(m, s_red[0][w]);

    const int at = threadIdx.x / TP, v = threadIdx.x % TP;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
    for (int i = at; i < n; i += 4 * AT) {
        float2 ml[4];
        float4 x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int64_t p = slot(i + k * AT < n ? i + k * AT : i);
            ml[k] = part_ml[p];
            x[k] = *reinterpret_cast<const float4 *>(part_o + p * D + 4 * v);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (i + k * AT >= n) continue;
            const float w = ml[k].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[k].x - m);
            l += w * ml[k].y;
            o.x += w * x[k].x;
            o.y += w * x[k].y;
            o.z += w * x[k].z;
            o.w += w * x[k].w;
        }
    }
    s_o[at][v] = o;
    __shared__ float s_l[AT];
    if (v == 0) s_l[at] = l;
    __syncthreads();
    if (threadIdx.x >= TP) return;
    l = 0.f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < AT; ++k) {
        const float4 x = s_o[k][v];
        l += s_l[k];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
    }
    const float inv = l == 0.f && m == -__builtin_inff() ? 0.f : 1.0f / l;  // 0: no page of the row is in the pool
    *reinterpret_cast<u32x2 *>(out + 4 * v) = u32x2{pack2_bf16(o.x * inv, o.y * inv), pack2_bf16(o.z * inv, o.w * inv)};
}

// Rows of several queries.  A workgroup of NW waves takes 32 NW columns (queries times the G query heads of one kv
// head) against 32-key tiles, a wave 32 columns with mfma_32x32x16: S^T = K Q^T, out^T = V^T P^T, so a column's
// scores, maximum and output stay in two lanes and P needs no exchange.  K and V are widened to bf16, V times its
// scale, once a workgroup on their way to LDS (V transposed, keys in the order in which a lane holds P); a
// tile's loads are in flight while the one before it is multiplied.  Sums are rescaled only when a maximum has grown
// by more than 2^8 (P stays below that, and bf16 and fp32 lose nothing by it).  With few tiles the key range is
// cut into pieces, joined by kv8_join_kernel.
// 1856 queries of 16 heads over 6001 keys (77 GFLOP): 108 us and 10 for the join, 716 TFLOP/s at the clocks of a steady
// load (124 us in the first milliseconds of one); 64 rows of 128 queries over 512 keys 60 us.  No unit is full: the vector
// units run in 42 % of the clocks, the MFMAs in 29 %, LDS in 27 % (a fifth of that the conflicts of V's writes); they overlap
// in part only, around one barrier a step.  The loads' issue takes 0.17 us of a step of 1.25 (at the first milliseconds'
// clocks).  With uniform pieces the longest one takes 94 tiles where 79 is the mean.
// 64-key tiles take 1 to 10 % less where one long prompt fills the card and up to 1.6 times as long for batches
// (registers spill, one workgroup a CU).  Tried and no faster (against 127 us): 64 columns a wave at one wave a SIMD (156
// us), spans that cross tiles for even work (143 us), staging two steps ahead.
constexpr int kKeys = 32;
constexpr float kLag = 8.0f;

struct Tile8 {
    int q0, n_q, limit0;  // first query token, queries, keys the first of them sees
    int n_keys;           // keys the last of them sees
};
// The launch's tiles, counted from the last one of the last row (a row's last tile sees the most keys) down to the first of
// row 0; found by the whole wave, which sums the rows' tiles 64 at a time.  So workgroups without a tile come
// last: between the others they would hold back the ones behind them, 51 us instead of 35 for 16 rows of 256 queries.
template <typename R>
__device__ __forceinline__ bool tile_of(const Attend8 &a, const R &rows, int nq, int index, int skip_single, Row8 &row,
                                        Tile8 &t) {
    const int lane = threadIdx.x & (kWave - 1);
    int before = 0;
    for (int top = a.rows - 1; top >= 0; top -= kWave) {
        const int r = top - lane;
        int n = 0;
        if (r >= 0) {
            const int q0 = rows.qo(r), len = rows.qo(r + 1) - q0;
            const bool mine = q0 >= 0 && len > 0 && q0 <= a.tokens - len && !(skip_single && len == 1);
            n = mine ? (len + nq - 1) / nq : 0;
        }
        for (int d = 1; d < kWave && d < a.rows; d *= 2) {  // lanes behind row 0 hold none
            const int x = __shfl_up(n, d, kWave);
            if (lane >= d) n += x;
        }
        const uint64_t past = __ballot(before + n > index);
        if (past) {
            const int at = __builtin_ctzll(past);
            row = row_of(a, rows, top - at);
            const int first = (before + __builtin_amdgcn_readlane(n, at) - 1 - index) * nq;
            t.q0 = row.q0 + first;
            t.n_q = row.q_len - first < nq ? row.q_len - first : nq;
            t.limit0 = row.kv_len - row.q_len + first + 1;
            const int last = t.limit0 + t.n_q - 1;
            t.n_keys = last < 0 ? 0 : last;
            return true;
        }
        before += __builtin_amdgcn_readlane(n, kWave - 1);
    }
    return false;
}
__device__ __forceinline__ int pieces_of(const Tile8 &t, int splits) {
    const int n = (t.n_keys + kKeys - 1) / kKeys / 4;  // at least four key tiles a piece
    return n < 1 ? 1 : (n < splits ? n : splits);
}

template <int D>
struct Smem8 {
    u32x4 k[2][kKeys * (D / 8 + 1)];
    u32x4 v[2][D * (kKeys / 8)];
    float ks[2][kKeys / kBlk];     // K scales of the tile's blocks times sm_scale log2(e), 1 where one is none
    int odd[2][kKeys / kBlk];      // kAbsent: the block's page is not in the pool; kPoison: a scale is none
    Meta8 meta;
};
constexpr int kAbsent = 1, kPoison = 2;
// Places of 16-byte chunks, free of conflicts for the operand reads (32 rows, two chunks each) and for K's writes: rows of K
// one chunk longer than their values, V's chunks exclusive-ored with bits of their row.  V's writes, eight bytes in each of
// 16 rows and four quads, take 16 clocks for the 4 of neighbouring ones.
template <int D>
__device__ __forceinline__ int k_chunk(int key, int chunk) {
    return key * (D / 8 + 1) + chunk;
}
__device__ __forceinline__ int v_chunk(int d, int chunk) { return d * (kKeys / 8) + (chunk ^ ((d >> 2) & 3)); }

template <int D, int NW>
__global__ void __launch_bounds__(NW * kWave, 2)
kv8_prefill_kernel(Attend8 a, Pool8 pool, int splits, int skip_single, float2 *__restrict__ part_ml,
                   float *__restrict__ part_o) {
    constexpr int T = NW * kWave, COLS = 32 * NW, NB = kKeys / kBlk;
    // K: a thread stages KP pieces of eight values of one key; V: VB values of each of four keys
    constexpr int KT = T / kKeys, KP = D / 8 / KT;  // KT threads a key
    constexpr int VB = kKeys * D / 4 / T;           // 2 or 4
    static_assert(KP >= 1 && KP * KT * 8 == D && (VB == 2 || VB == 4), "a tile stages evenly");
    using Smem = Smem8<D>;
    __shared__ Smem sm;
    load_meta(a, sm.meta);
    const Rows8 rows{a, sm.meta};
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
    const int head = blockIdx.x % a.heads, slot = static_cast<int>(blockIdx.x) / a.heads;
    Row8 row;
    Tile8 t;
    if (!tile_of(a, rows, COLS / a.group, slot, skip_single, row, t)) return;
    const int pieces = pieces_of(t, splits);
    const int piece = blockIdx.y;
    if (piece >= pieces) return;
    const int n_kt = (t.n_keys + kKeys - 1) / kKeys;
    const int kt0 = static_cast<int>(static_cast<int64_t>(n_kt) * piece / pieces),
              kt1 = static_cast<int>(static_cast<int64_t>(n_kt) * (piece + 1) / pieces);

    constexpr int kBufK = 16 * kKeys * (D / 8 + 1), kBufV = 16 * D * (kKeys / 8);
    // Staging: a wave holds keys of one block, so its page, its scales and their addresses are uniform: 32 / NW keys of K;
    // of V the four quads of keys and 16 VB values, so that its writes (eight bytes a row of V and quad) spread over the banks.
    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    const int sk_key = threadIdx.x / KT, sk_piece = threadIdx.x % KT;
    const int quad = lane >> 4, sv_part = uwave % (NW / NB) * 16 + (lane & 15);
    const int c_slot = static_cast<int>(pool.c_slot);
    const int k_off = sk_key % kBlk * c_slot + 8 * sk_piece;
    const int v_off = 4 * quad * c_slot + VB * sv_part;
    const int8_t *base = pool.codes + head * pool.c_head;
    const float *s_base = pool.scales + head * pool.s_head;
    const int n_blocks = (row.kv_len + kBlk - 1) / kBlk;
    const int in_page = (1 << a.bpp_log2) - 1;
    // Pages and scales are uniform, but fetched as vectors: a scalar load outstanding would make every wait for an LDS
    // read in the loop a wait for that load too.
    uint32_t zero = 0;
    asm volatile("" : "+v"(zero));
    // the wave's block of tile kt, held to the row's: what lies beyond its keys is masked, a tile beyond the last never used
    auto block_of = [&](int kt) __attribute__((always_inline)) {
        const int blk = kt * NB + uwave * NB / NW;
        return blk < n_blocks ? blk : n_blocks - 1;
    };
    auto page_of = [&](int kt) __attribute__((always_inline)) {
        return (a.kv_indices + row.first_page + (block_of(kt) >> a.bpp_log2))[zero];
    };
    // The staging registers: K of one tile and V of the tile before it, with what their block needs.
    struct Stage {
        u32x2 k[KP];
        uint32_t v[4];
        float ks, vs, next_vs, v_vs;  // scales of K's block, V scales of the block before it and of V's
        bool on;                      // K's page is in the pool
    };
    const int8_t *v_from = base, *v_next = base;  // V of the tile whose K was asked for last, and of the one before
    auto load_v = [&](Stage &r) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int8_t *p = v_next + static_cast<uint32_t>(v_off + e * c_slot);
            if constexpr (VB == 4) r.v[e] = *reinterpret_cast<const uint32_t *>(p);
            else r.v[e] = *reinterpret_cast<const uint16_t *>(p);
        }
        r.v_vs = r.next_vs;
    };
    auto load_k = [&](int kt, int found, Stage &r) __attribute__((always_inline)) {
        v_next = v_from;
        r.next_vs = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(r.vs)));
        const int page = __builtin_amdgcn_readfirstlane(found);
        r.on = page >= 0 && page < pool.num_pages;
        const int64_t pid = r.on ? page : 0;
        const int blk = block_of(kt) & in_page;
        const int8_t *kp = base + pid * pool.c_page + blk * (kBlk * pool.c_slot);
#pragma unroll
        for (int e = 0; e < KP; ++e)
            r.k[e] = *reinterpret_cast<const u32x2 *>(kp + static_cast<uint32_t>(k_off) + 8 * KT * e);
        const float *sc = s_base + pid * pool.s_page + blk * pool.s_block;
        r.ks = sc[zero];
        r.vs = (sc + pool.s_kind)[zero];
        v_from = kp + pool.c_kind;
    };
    // First places of what a thread stages.  Key 8 a + 4 b + i of a block sits at position 8 b + 4 a + i of V's rows.
    char *stage = reinterpret_cast<char *>(&sm);
    const int put_k0 = static_cast<int>(offsetof(Smem, k)) + 16 * k_chunk<D>(sk_key, sk_piece);
    const int put_v0 = static_cast<int>(offsetof(Smem, v)) +
                       16 * v_chunk(sv_part * VB, 2 * (uwave * NB / NW) + (quad & 1)) + 8 * (quad >> 1);
    auto put_k = [&](const Stage &r, int e, int buf) __attribute__((always_inline)) {
        *reinterpret_cast<bf16x8_t *>(stage + put_k0 + 16 * KT * e + buf * kBufK) = widen8(r.k[e].x, r.k[e].y);
    };
    auto put_scales = [&](const Stage &r, int buf) __attribute__((always_inline)) {
        // What is no scale, K's or V's, answers through the scores of the queries that see the block, not through
        // 0 * NaN in those that do not.
        const bool fine = is_scale(r.ks) && is_scale(r.vs);
        const int blk = uwave * NB / NW;
        // above zero, also for a block that was never written: a masked score, minus infinity, stays that
        sm.ks[buf][blk] = r.on && fine ? fmaxf(r.ks * a.scale, kMinScale) : 1.0f;
        sm.odd[buf][blk] = !r.on ? kAbsent : fine ? 0 : kPoison;
    };
    auto put_v = [&](const Stage &r, int col, int buf) __attribute__((always_inline)) {
        const float vs = is_scale(r.v_vs) ? r.v_vs : 0.f;
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = r.v[e];
            asm("" : "+v"(x[e]));  // any 32 bits: one conversion picks a byte, where 16 known ones are shifted first
        }
        // value VB part + col: the same bits 2 and 3 of the row as part's first
        *reinterpret_cast<u32x2 *>(stage + put_v0 + buf * kBufV + 16 * (kKeys / 8) * col) =
            u32x2{pack2_bf16(byte_of(x[0], col) * vs, byte_of(x[1], col) * vs),
                  pack2_bf16(byte_of(x[2], col) * vs, byte_of(x[3], col) * vs)};
    };
    int found0 = 0, found1 = 0;
    if (kt0 < kt1) {
        found0 = page_of(kt0);
        found1 = page_of(kt0 + 1);
    }

    const int c = lane & 31, half = lane >> 5;
    const int col = wave * 32 + c;
    const int qi = col / a.group, g = col - qi * a.group;
    const bool live = qi < t.n_q;
    const int limit = live ? t.limit0 + qi : 0;
    bf16x8_t qf[D / 16];
#pragma unroll
    for (int s = 0; s < D / 16; ++s)
        qf[s] = load_q(a.q + (t.q0 + qi) * a.q_s0 + (head * a.group + g) * a.q_s1 + 16 * s + 8 * half, live, a.flip);

    // Where the lane reads, in bytes: chunk half of K row c and of V row c.  The other operands are constants away, V's
    // after an exclusive-or of the chunk (rows 32 j on keep it).
    const char *lds = reinterpret_cast<const char *>(&sm);
    const int at_k = static_cast<int>(offsetof(Smem, k)) + 16 * k_chunk<D>(c, half);
    const int at_v = static_cast<int>(offsetof(Smem, v)) + 16 * v_chunk(c, half);
    auto operand = [&](int at) __attribute__((always_inline)) {
        return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const u32x4 *>(lds + at));
    };
    floatx16_t acc[D / 32];
#pragma unroll
    for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] = 0.f;
    float m_run = -__builtin_inff(), l_run = 0.f, top = -__builtin_inff();
    bool any = false;  // whether the column has seen a key
    float f_k[NB] = {};
    Stage st;

    // Keys that a column does not see, in tiles that hold any such key.
    auto mask = [&](int kt, const int (&odd)[NB], floatx16_t &s) __attribute__((always_inline)) {
        const int key0 = kt * kKeys;
        const int some = __builtin_amdgcn_readfirstlane(odd[0] | odd[1]);
        if (key0 + kKeys <= t.limit0 && !some) {
            any = true;
            return;
        }
        if ((some & kAbsent) && a.status) *a.status = NQ_ERR_INVALID_ARGUMENT;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            // the lane's element i: key 8 (i / 4) + 4 half + i % 4
            const bool see = key0 + 8 * (i / 4) + 4 * half + (i & 3) < limit && odd[i / 8] != kAbsent;
            any |= see;
            const float v = odd[i / 8] == kPoison ? __builtin_nanf("") : s[i];
            s[i] = see ? v : -__builtin_inff();
        }
    };
    // A block's largest score; times its factor (positive) it counts for the maximum.
    auto block_top = [&](const floatx16_t &s, int k) __attribute__((always_inline)) {
        float m = s[8 * k];
#pragma unroll
        for (int i = 1; i < 8; ++i) m = fmaxf(m, s[8 * k + i]);
        return m;
    };
    // Tile kt: its scores are in `s` and their maximum in `top`; the next tile's go to `next`.  Two blocks of
    // independent work each, interleaved chunk by chunk (the fences hold the order): the next scores beside this
    // tile's exponentials and the staging of K two tiles ahead, then P V beside the next maximum and the staging of V
    // one tile ahead.  Operands are read AHEAD MFMAs before their own, the next tile's first ones too.  The one barrier
    // stands between the last read of K of tile kt + 1 and the first of V of tile kt: K of kt + 2 is staged before
    // it, where K of kt was, last read before the barrier of kt - 1; V of kt + 1 behind it, where V of kt - 1 was.
    constexpr int NK = D / 16, NV = NB * (D / 32);  // operands of a tile's scores and of its P V
    constexpr int PER = 16 / NK, STEPS = NK / 2;    // score elements beside each of the first; chunks that stage K
    constexpr int AHEAD = D == 128 ? 3 : 2;
    static_assert(NK % 4 == 0 && NV % 4 == 0 && NK - AHEAD >= STEPS, "the ring's places and the barrier's");
    bf16x8_t ring[4];
    auto read_k = [&](int n, int buf) __attribute__((always_inline)) {
        ring[n & 3] = operand(at_k + buf * kBufK + 32 * n);
    };
    auto read_v = [&](int n, int base) __attribute__((always_inline)) {
        ring[n & 3] = operand((base ^ (32 * (n / (D / 32)))) + 16 * (kKeys / 8) * 32 * (n % (D / 32)));
    };
    auto step = [&](auto last, auto buf, int kt, floatx16_t &s, floatx16_t &next) __attribute__((always_inline)) {
        constexpr int B = buf, N = 1 - B;  // tile kt's buffer, the next one's
        if (__any(top > m_run + kLag)) {
            const float m_new = fmaxf(m_run, top);
            const float alpha = m_run == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
            l_run *= alpha;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) acc[j] *= alpha;
            m_run = m_new;
        }
        const float m_use = m_run == -__builtin_inff() ? 0.f : m_run;  // no key yet: 2^(-inf) for all
        int v_base = at_v + B * kBufV;
        asm volatile("" : "+v"(v_base));  // places are made from it where they are used, not kept
        int n_odd[NB] = {};
        float n_f[NB] = {};
        uint32_t pw[8];
        float sum[2] = {0.f, 0.f};
        if constexpr (!last) {
#pragma unroll
            for (int i = 0; i < 16; ++i) next[i] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < NK; ++n) {
            if constexpr (!last)
                if (n == STEPS - 1) {
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        n_odd[b] = sm.odd[N][b];
                        n_f[b] = sm.ks[N][b];
                    }
                }
            if (n + AHEAD == NK) __syncthreads();
            if (n + AHEAD >= NK) read_v(n + AHEAD - NK, v_base);
            else if constexpr (!last) read_k(n + AHEAD, N);
            if constexpr (!last) next = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[n & 3], qf[n], next, 0, 0, 0);
#pragma unroll
            for (int i = PER * n; i < PER * (n + 1); i += 2) {
                const float x = __builtin_amdgcn_exp2f(fmaf(s[i], f_k[i / 8], -m_use));
                const float y = __builtin_amdgcn_exp2f(fmaf(s[i + 1], f_k[i / 8], -m_use));
                pw[i / 2] = pack2_bf16(x, y);
                float &l = sum[i / 2 % 2];
                l += x + y;
                asm volatile("" : "+v"(pw[i / 2]), "+v"(l));  // made here, not where they are used
            }
            if constexpr (!last) {  // K of tile kt + 2, or of one that is never used
                if (n < STEPS) {
#pragma unroll
                    for (int e = KP * n / STEPS; e < KP * (n + 1) / STEPS; ++e) put_k(st, e, B);
                }
                if (n == STEPS - 1) {  // then its registers are free for the tile behind
                    put_scales(st, B);
                    load_k(kt + 3, found0, st);
                    found0 = page_of(kt + 4);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l_run += sum[0] + sum[1];
        if constexpr (!last) {
            mask(kt + 1, n_odd, next);
#pragma unroll
            for (int b = 0; b < NB; ++b) f_k[b] = n_f[b];
        }
        float high = -__builtin_inff();
#pragma unroll
        for (int ch = 0; ch < NV / 2; ++ch) {
#pragma unroll
            for (int n = 2 * ch; n < 2 * ch + 2; ++n) {
                if (n + AHEAD < NV) read_v(n + AHEAD, v_base);
                else if constexpr (!last) read_k(n + AHEAD - NV, B);  // of tile kt + 2
                const int k = n / (D / 32), j = n % (D / 32);
                const bf16x8_t pf =
                    __builtin_bit_cast(bf16x8_t, u32x4{pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]});
                acc[j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(ring[n & 3], pf, acc[j], 0, 0, 0);
            }
            if constexpr (!last) {
                constexpr int PCH = NV / 2;
                if (ch % (PCH / NB) == 0) high = fmaxf(high, block_top(next, ch * NB / PCH) * f_k[ch * NB / PCH]);
#pragma unroll
                for (int e = VB * ch / PCH; e < VB * (ch + 1) / PCH; ++e) put_v(st, e, N);
                if (ch == PCH - 1) load_v(st);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!last) top = halves_max(high);
    };
    if (kt0 < kt1) {
        Stage first;
        first.vs = 0.f;
        load_k(kt0, found0, first);
        st.vs = first.vs;
        load_k(kt0 + 1, found1, st);
        load_v(st);
        found1 = page_of(kt0 + 2);
        found0 = page_of(kt0 + 3);
#pragma unroll
        for (int e = 0; e < KP; ++e) {
            put_k(first, e, 0);
            put_k(st, e, 1);
        }
        put_scales(first, 0);
        put_scales(st, 1);
#pragma unroll
        for (int e = 0; e < VB; ++e) put_v(st, e, 0);
        load_k(kt0 + 2, found1, st);
        load_v(st);
        __syncthreads();
        floatx16_t s0, s1;
#pragma unroll
        for (int i = 0; i < 16; ++i) s0[i] = 0.f;
#pragma unroll
        for (int n = 0; n < NK; ++n)
            s0 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(operand(at_k + 32 * n), qf[n], s0, 0, 0, 0);
        mask(kt0, sm.odd[0], s0);
#pragma unroll
        for (int b = 0; b < NB; ++b) f_k[b] = sm.ks[0][b];
#pragma unroll
        for (int k = 0; k < NB; ++k) top = fmaxf(top, block_top(s0, k) * f_k[k]);
        top = halves_max(top);
        __syncthreads();  // the first step stages over the first tile's K
        if (kt0 + 1 < kt1) {
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) read_k(n, 1);
        }
        constexpr std::integral_constant<int, 0> b0{};
        constexpr std::integral_constant<int, 1> b1{};
        int kt = kt0;
        for (; kt + 2 < kt1; kt += 2) {
            step(std::false_type{}, b0, kt, s0, s1);
            step(std::false_type{}, b1, kt + 1, s1, s0);
        }
        if (kt + 1 < kt1) {
            step(std::false_type{}, b0, kt, s0, s1);
            step(std::true_type{}, b1, kt + 1, s1, s0);
        } else {
            step(std::true_type{}, b0, kt, s0, s1);
        }
    }
    l_run = halves_sum(l_run);
    any = any | static_cast<bool>(__shfl_xor(static_cast<int>(any), 32, kWave));
    if (!live) return;
    // the lane holds out[col][32 j + 8 (i / 4) + 4 half + i % 4] in acc[j][i]
    if (pieces == 1) {
        const float inv = any ? 1.0f / l_run : 0.f;
        uint16_t *o = a.out + (t.q0 + qi) * a.o_s0 + (head * a.group + g) * a.o_s1 + 4 * half;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<u32x2 *>(o + 32 * j + 2 * i) =
                    u32x2{pack2_bf16(acc[j][i] * inv, acc[j][i + 1] * inv),
                          pack2_bf16(acc[j][i + 2] * inv, acc[j][i + 3] * inv)};
    } else {
        const int64_t at = ((static_cast<int64_t>(slot) * a.heads + head) * splits + piece) * COLS + col;
        // Minus infinity says that the piece saw no key.  One whose scores are all minus infinity has no weight beside
        // other pieces, and if there are no others the sum of 0 makes the row NaN.
        if (half == 0) part_ml[at] = make_float2(any ? fmaxf(m_run, -__FLT_MAX__) : -__builtin_inff(), l_run);
        float *o = part_o + at * D + 4 * half;
#pragma unroll
        for (int j = 0; j < D / 32; ++j)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4 *>(o + 32 * j + 2 * i) =
                    make_float4(acc[j][i], acc[j][i + 1], acc[j][i + 2], acc[j][i + 3]);
    }
}

// Joins the pieces of a tile, in order: D/8 threads a column, every piece's values in flight at once.  Bound by its reads:
// 31 MB of partials 10 us.
constexpr int kMaxPieces = 8;
template <int D>
__global__ void __launch_bounds__(kKv8Threads)
kv8_join_kernel(Attend8 a, int cols, int splits, int skip_single, const float2 *__restrict__ part_ml,
                const float *__restrict__ part_o) {
    constexpr int TP = D / 8;
    __shared__ Meta8 meta;
    load_meta(a, meta);
    const int head = blockIdx.x % a.heads, slot = static_cast<int>(blockIdx.x) / a.heads;
    Row8 row;
    Tile8 t;
    if (!tile_of(a, Rows8{a, meta}, cols / a.group, slot, skip_single, row, t)) return;
    const int pieces = pieces_of(t, splits);
    const int col = blockIdx.y * (kKv8Threads / TP) + threadIdx.x / TP, v = threadIdx.x % TP;
    if (pieces == 1 || col >= t.n_q * a.group) return;
    const int64_t base = (static_cast<int64_t>(slot) * a.heads + head) * splits * cols + col;
    float2 ml[kMaxPieces];
    float4 x[kMaxPieces][2];
#pragma unroll
    for (int i = 0; i < kMaxPieces; ++i) {
        if (i < pieces) {
            ml[i] = part_ml[base + static_cast<int64_t>(i) * cols];
            const float4 *p = reinterpret_cast<const float4 *>(part_o + (base + static_cast<int64_t>(i) * cols) * D + 8 * v);
            x[i][0] = p[0];
            x[i][1] = p[1];
        }
    }
    float m = -__builtin_inff(), l = 0.f, o[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < kMaxPieces; ++i)
        if (i < pieces) m = fmaxf(m, ml[i].x);
#pragma unroll
    for (int i = 0; i < kMaxPieces; ++i) {
        if (i < pieces) {
            const float w = ml[i].y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml[i].x - m);
            l += w * ml[i].y;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                o[4 * h] += w * x[i][h].x;
                o[4 * h + 1] += w * x[i][h].y;
                o[4 * h + 2] += w * x[i][h].z;
                o[4 * h + 3] += w * x[i][h].w;
            }
        }
    }
    const float inv = l == 0.f && m == -__builtin_inff() ? 0.f : 1.0f / l;
    const int qi = col / a.group, g = col - qi * a.group;
    *reinterpret_cast<u32x4 *>(a.out + (t.q0 + qi) * a.o_s0 + (head * a.group + g) * a.o_s1 + 8 * v) =
        u32x4{pack2_bf16(o[0] * inv, o[1] * inv), pack2_bf16(o[2] * inv, o[3] * inv), pack2_bf16(o[4] * inv, o[5] * inv),
              pack2_bf16(o[6] * inv, o[7] * inv)};
}

// Waves of the decode launch per kv head: eight a CU.
int decode_waves(int heads) {
    const int groups = 512 / heads;  // workgroups of four waves
    return (groups < 1 ? 1 : groups) * kKv8Waves;
}
struct Prefill8 {
    int waves, cols, slots, splits;
};
// Four waves, two workgroups a CU: their starts, barriers and ends overlap.  Eight (one a CU) stage each tile half as often
// per column, which counts where few tiles have long key ranges, of heads of 128: rows of 2000 columns and more that still
// leave two pieces a workgroup.  Measured with four and eight waves, us, 16 query heads of 128 on 8:
//   1 row of 1800 queries over 6001 keys 129, 117;  1 of 2000 over 2000 56, 52;  1 of 1000 over 12000 137, 123
//   1 of 4000 over 4000 117, 129;  4 of 2000 over 2000 115, 126;  64 of 128 over 512 60, 68;  1 of 300 over 300 15.3, 18.6
// (past what two pieces tell, where the rule takes four: 2 of 2000 over 4000 161, 139;  1 of 8000 over 8000 348, 302)
// Pieces: as many as fit the CUs at once, up to kMaxPieces.
Prefill8 prefill_plan(int tokens, int rows, int group, int heads, int D) {
    const int64_t columns = static_cast<int64_t>(tokens) * group;
    auto pieces = [&](int cols, int room) {
        const int64_t wgs = (columns / cols + (rows + 1) / 2) * heads, n = room / wgs;  // rows' last tiles: half a tile each
        return static_cast<int>(n < 1 ? 1 : n < kMaxPieces ? n : kMaxPieces);
    };
    Prefill8 p = {4, 128, 0, pieces(128, 512)};
    if (D == 128 && columns >= 2000ll * rows && pieces(256, 256) > 1) p = {8, 256, 0, pieces(256, 256)};
    p.slots = tokens / (p.cols / group) + rows;  // no batch has more tiles
    return p;
}
struct Layout8 {
    int64_t d_ml, d_o, p_ml, p_o, total;
};
int64_t up256(int64_t x) { return (x + 255) & ~int64_t(255); }
Layout8 layout8(int tokens, int rows, int qo_heads, int heads, int D, int parts) {
    const int group = qo_heads / heads;
    Layout8 L = {0, 0, 0, 0, 0};
    int64_t off = 0;
    if (parts & NQ_ATTN_DECODE) {
        const int64_t n = 2ll * decode_waves(heads) * qo_heads;
        L.d_ml = off;
        off = up256(off + n * 8);
        L.d_o = off;
        off = up256(off + n * D * 4);
    }
    if (parts & NQ_ATTN_PREFILL) {
        const Prefill8 p = prefill_plan(tokens, rows, group, heads, D);
        const int64_t n = p.splits > 1 ? static_cast<int64_t>(p.slots) * heads * p.splits * p.cols : 0;
        L.p_ml = off;
        off = up256(off + n * 8);
        L.p_o = off;
        off = up256(off + n * D * 4);
    }
    L.total = off;
    return L;
}

bool al(const void *p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A stride that breaks the alignment of what lies behind it (that of a dimension of one is never used).
bool odd_stride(int n, int64_t stride, int multiple) { return n > 1 && stride % multiple; }

int check_pool(const Pool8 &p, int heads, int head_dim) {
    NQ_CHECK_ARG(p.codes && p.scales && p.num_pages >= 1 && heads >= 1);
    NQ_CHECK_ARG(p.page_size >= 1 && (p.page_size & (p.page_size - 1)) == 0);
    NQ_CHECK_ARG(p.c_page >= 0 && p.c_kind >= 0 && p.c_slot >= 0 && p.c_head >= 0);
    NQ_CHECK_ARG(p.s_page >= 0 && p.s_kind >= 0 && p.s_block >= 0 && p.s_head >= 0);
    if ((head_dim != 64 && head_dim != 128) || p.page_size < kBlk) return NQ_ERR_UNSUPPORTED;
    if (!al(p.codes, 16) || odd_stride(p.num_pages, p.c_page, 16) || p.c_kind % 16 || p.c_slot % 16 ||
        odd_stride(heads, p.c_head, 16) || !al(p.scales, 4))
        return NQ_ERR_UNSUPPORTED;
    if (p.c_slot >= (1 << 26)) return NQ_ERR_UNSUPPORTED;  // 16 slots of a block stay within 32-bit offsets
    return NQ_OK;
}

}  // namespace
}  // namespace nq

using namespace nq;

extern "C" int nq_kv_int8_write(const uint16_t *key, int64_t k_s0, int64_t k_s1, const uint16_t *value, int64_t v_s0,
                                int64_t v_s1, int tokens, int num_kv_heads, int head_dim, int8_t *codes,
                                int64_t c_page, int64_t c_kind, int64_t c_slot, int64_t c_head, float *scales,
                                int64_t s_page, int64_t s_kind, int64_t s_block, int64_t s_head, int num_pages,
                                int page_size, const int64_t *write_pages, const int64_t *write_offsets,
                                int32_t *status, void *stream) {
    NQ_CHECK_ARG(tokens >= 0);
    const Pool8 pool = {codes, c_page, c_kind, c_slot, c_head, scales, s_page, s_kind, s_block, s_head, num_pages,
                        page_size};
    const int rc = check_pool(pool, num_kv_heads, head_dim);
    if (rc != NQ_OK) return rc;
    if (tokens == 0) return NQ_OK;
    NQ_CHECK_ARG(key && value && write_pages && write_offsets);
    if (!al(key, 16) || !al(value, 16) || odd_stride(tokens, k_s0, 8) || odd_stride(num_kv_heads, k_s1, 8) ||
        odd_stride(tokens, v_s0, 8) || odd_stride(num_kv_heads, v_s1, 8))
        return NQ_ERR_UNSUPPORTED;
    // A wave takes its leaders one after another, about 2 us each, so many short runs want small groups and a long prompt
    // large ones.  Measured with groups of 1, 4, 8, 16, us, 8 heads: 64 runs of 1 token 5.0, 11.4, 19.6, 35.9; 1024 of 1
    // 18.0, 15.4, 22.2, 36.8; 8 of 80 13.2, 7.5, 6.6, 8.8; 8 of 300 23.9, 10.4, 9.6, 12.3; 1 of 8191 63, 41.5, 25.5, 18.9.
    const int64_t units = 2ll * tokens * num_kv_heads;
    const int group = units <= 4096 ? 1 : units <= 24576 ? 4 : units <= 65536 ? 8 : 16;
    const dim3 grid((tokens + group - 1) / group, (2 * num_kv_heads + kKv8Waves - 1) / kKv8Waves);
    const auto kernel = head_dim == 128 ? kv8_write_kernel<128> : kv8_write_kernel<64>;
    hipLaunchKernelGGL(kernel, grid, dim3(kKv8Threads), 0, static_cast<hipStream_t>(stream), key, k_s0, k_s1, value,
                       v_s0, v_s1, write_pages, write_offsets, tokens, num_kv_heads, group, pool, status);
    return NQ_LAUNCH_STATUS();
}

extern "C" int nq_kv_int8_read(const int8_t *codes, int64_t c_page, int64_t c_kind, int64_t c_slot, int64_t c_head,
                               const float *scales, int64_t s_page, int64_t s_kind, int64_t s_block, int64_t s_head,
                               int num_pages, int page_size, const int64_t *pages, const int64_t *offsets, int tokens,
                               int num_kv_heads, int head_dim, uint16_t *key, int64_t k_s0, int64_t k_s1,
                               uint16_t *value, int64_t v_s0, int64_t v_s1, int32_t *status, void *stream) {
    NQ_CHECK_ARG(tokens >= 0);
    const Pool8 pool = {const_cast<int8_t *>(codes), c_page, c_kind, c_slot, c_head, const_cast<float *>(scales),
                        s_page, s_kind, s_block, s_head, num_pages, page_size};
    const int rc = check_pool(pool, num_kv_heads, head_dim);
    if (rc != NQ_OK) return rc;
    if (tokens == 0) return NQ_OK;
    NQ_CHECK_ARG(key && value && pages && offsets);
    if (!al(key, 16) || !al(value, 16) || odd_stride(tokens, k_s0, 8) || odd_stride(num_kv_heads, k_s1, 8) ||
        odd_stride(tokens, v_s0, 8) || odd_stride(num_kv_heads, v_s1, 8))
        return NQ_ERR_UNSUPPORTED;
    const int64_t threads = static_cast<int64_t>(tokens) * 2 * num_kv_heads * (head_dim / 16);
    const int64_t groups = (threads + kKv8Threads - 1) / kKv8Threads;
    if (groups > 0x7fffffffll) return NQ_ERR_UNSUPPORTED;
    const auto kernel = head_dim == 128 ? kv8_read_kernel<128> : kv8_read_kernel<64>;
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(groups)), dim3(kKv8Threads), 0,
                       static_cast<hipStream_t>(stream), pool, pages, offsets, tokens, num_kv_heads, key, k_s0, k_s1,
                       value, v_s0, v_s1, status);
    return NQ_LAUNCH_STATUS();
}

extern "C" int64_t nq_paged_attention_int8_workspace_bytes(int tokens, int rows, int num_qo_heads, int num_kv_heads,
                                                           int head_dim, int parts) {
    if (tokens < 1 || rows < 1 || num_kv_heads < 1 || num_kv_heads > 512 || num_qo_heads < num_kv_heads ||
        num_qo_heads % num_kv_heads || num_qo_heads / num_kv_heads > 16 || (head_dim != 64 && head_dim != 128) ||
        parts < 1 || parts > (NQ_ATTN_DECODE | NQ_ATTN_PREFILL))
        return -1;
    return layout8(tokens, rows, num_qo_heads, num_kv_heads, head_dim, parts).total;
}

namespace {

template <int D>
int launch_attention8(const Attend8 &a, const Pool8 &pool, int parts, char *ws, const Layout8 &L, hipStream_t st) {
    if (parts & NQ_ATTN_DECODE) {
        const int waves = decode_waves(a.heads);
        float2 *ml = reinterpret_cast<float2 *>(ws + L.d_ml);
        float *o = reinterpret_cast<float *>(ws + L.d_o);
        hipLaunchKernelGGL((kv8_decode_kernel<D>), dim3(((waves + 7) / 8 * a.heads + kKv8Waves - 1) / kKv8Waves * 8),
                           dim3(kKv8Threads), 0, st, a, pool, waves, ml, o);
        hipLaunchKernelGGL((kv8_merge_kernel<D>), dim3(a.rows, a.heads * a.group), dim3(kKv8Threads), 0, st, a, waves, ml, o);
    }
    if (parts & NQ_ATTN_PREFILL) {
        const Prefill8 p = prefill_plan(a.tokens, a.rows, a.group, a.heads, D);
        const int skip = (parts & NQ_ATTN_DECODE) ? 1 : 0;
        float2 *ml = reinterpret_cast<float2 *>(ws + L.p_ml);
        float *o = reinterpret_cast<float *>(ws + L.p_o);
        const dim3 grid(p.slots * a.heads, p.splits);
        const auto kernel = p.waves == 4 ? kv8_prefill_kernel<D, 4> : kv8_prefill_kernel<128, 8>;  // eight: D is 128
        hipLaunchKernelGGL(kernel, grid, dim3(p.waves * kWave), 0, st, a, pool, p.splits, skip, ml, o);
        if (p.splits > 1)
            hipLaunchKernelGGL((kv8_join_kernel<D>), dim3(p.slots * a.heads, p.cols * (D / 8) / kKv8Threads),
                               dim3(kKv8Threads), 0, st, a, p.cols, p.splits, skip, ml, o);
    }
    return NQ_LAUNCH_STATUS();
}

}  // namespace

extern "C" int nq_paged_attention_int8(const int32_t *qo_indptr, const int32_t *kv_indptr,
                                       const int32_t *last_page_len, const int32_t *kv_indices, int n_rows,
                                       int num_indices, const uint16_t *q, int64_t q_s0, int64_t q_s1, int tokens,
                                       const int8_t *codes, int64_t c_page, int64_t c_kind, int64_t c_slot,
                                       int64_t c_head, const float *scales, int64_t s_page, int64_t s_kind,
                                       int64_t s_block, int64_t s_head, int num_pages, int page_size,
                                       int num_qo_heads, int num_kv_heads, int head_dim, float sm_scale,
                                       uint16_t *out, int64_t o_s0, int64_t o_s1, int parts, void *workspace,
                                       int64_t workspace_bytes, int32_t *status, void *stream) {
    NQ_CHECK_ARG(n_rows >= 0 && tokens >= 0 && num_indices >= 0 && num_kv_heads >= 1);
    NQ_CHECK_ARG(num_qo_heads >= num_kv_heads && num_qo_heads % num_kv_heads == 0);
    NQ_CHECK_ARG(parts >= 1 && parts <= (NQ_ATTN_DECODE | NQ_ATTN_PREFILL));
    NQ_CHECK_ARG(qo_indptr || parts == NQ_ATTN_DECODE);
    NQ_CHECK_ARG(fabsf(sm_scale) * kLog2e8 <= __FLT_MAX__);  // not NaN either
    const Pool8 pool = {const_cast<int8_t *>(codes), c_page, c_kind, c_slot, c_head, const_cast<float *>(scales),
                        s_page, s_kind, s_block, s_head, num_pages, page_size};
    const int rc = check_pool(pool, num_kv_heads, head_dim);
    if (rc != NQ_OK) return rc;
    if (n_rows == 0 || tokens == 0) return NQ_OK;
    const int64_t need =
        nq_paged_attention_int8_workspace_bytes(tokens, n_rows, num_qo_heads, num_kv_heads, head_dim, parts);
    if (need < 0) return NQ_ERR_UNSUPPORTED;
    NQ_CHECK_ARG(q && out && kv_indptr && last_page_len && (kv_indices || num_indices == 0));
    NQ_CHECK_ARG(qo_indptr || n_rows <= tokens);
    NQ_CHECK_ARG(need == 0 || (workspace && workspace_bytes >= need && al(workspace, 16)));
    if (!al(q, 16) || odd_stride(tokens, q_s0, 8) || odd_stride(num_qo_heads, q_s1, 8) || !al(out, 16) ||
        odd_stride(tokens, o_s0, 8) || odd_stride(num_qo_heads, o_s1, 8))
        return NQ_ERR_UNSUPPORTED;
    int bpp = 0;
    while ((kBlk << bpp) < page_size) ++bpp;
    const Prefill8 p = prefill_plan(tokens, n_rows, num_qo_heads / num_kv_heads, num_kv_heads, head_dim);
    if (static_cast<int64_t>(p.slots) * num_kv_heads > 0x3fffffff || num_kv_heads > 65535 ||
        (static_cast<int64_t>(num_indices) * page_size) > 0x7fff0000ll)  // a tile behind the last key is still an int
        return NQ_ERR_UNSUPPORTED;
    const Attend8 a = {q,     q_s0,        q_s1,   out,         o_s0,
                       o_s1,  qo_indptr,   kv_indptr, kv_indices,  last_page_len,
                       n_rows, tokens,     num_indices, num_qo_heads / num_kv_heads, num_kv_heads,
                       bpp,   fmaxf(fabsf(sm_scale) * kLog2e8, kMinScale), sm_scale < 0.f ? 0x80008000u : 0u, status};
    char *ws = static_cast<char *>(workspace);
    const Layout8 L = layout8(tokens, n_rows, num_qo_heads, num_kv_heads, head_dim, parts);
    hipStream_t st = static_cast<hipStream_t>(stream);
    return head_dim == 128 ? launch_attention8<128>(a, pool, parts, ws, L, st)
                           : launch_attention8<64>(a, pool, parts, ws, L, st);
}

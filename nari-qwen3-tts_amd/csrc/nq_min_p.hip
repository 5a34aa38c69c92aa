// A token a row from logits over a vocabulary of any size up to 2^20: temperature, min-p, top-k, top-p and the draw for a
// given uniform number.
//   e_i   = exp((x_i - max x) / T)          in double;  NaN logits count as -inf, -0 as 0
//   w_i   = rint(2^42 e_i), or 0 where that is below 2^42 min_p: an integer, so that every sum is exact in any order and the token does
//           not depend on how the work is cut; 2^20 of them stay below 2^62
//   order : by (x desc, id asc); F(r) = sum of w over the ranks 0 .. r
//   total = F(min(k, V) - 1), k = top_k > 0 ? top_k : V
//   kept  = the ranks up to the first with F(r) >= p total (min-p and top-k leave a prefix too)
//   token = the first id at which the sum of w over the kept ids up to it reaches u of its whole
// T not above zero: the first rank.  Top-k and top-p are the same question, the first rank whose count or mass reaches a
// target, so a row is asked it up to twice and never sorted whole.
//
// A workgroup a row.  Where min-p leaves few logits, one pass collects them in LDS, by the maximum so far (what a later
// one drops is dropped behind the pass), and they are sorted and summed there.  Otherwise a histogram over the distance
// from the maximum, of counts for top-k and of masses for top-p, says which bin the last rank lies in, and that bin's
// logits alone are collected and sorted; a bin too full for the list (equal logits) is cut by the digits of its entries.
// The draw sums what is kept over cells of consecutive ids, and looks at the logits of the one cell that it falls into.
//
// Bound by the slowest row's passes.  64 x 65537 bf16 (us, replayed): the first rank 7, min-p .05 15, top-k 50 17, no cut 25,
// top-p .95 41; 256 x 131072 fp32, whose reading takes 26: 29, 34, 51, 63, 115.  The maximum takes a pass (2.4 and 17 us), the cells'
// masses another (15 and 34: some 27 vector instructions a logit where most are kept, in double), top-p before it a third for
// the bins' masses (8 and 32) and a fourth for the cut bin's logits (6 and 17).  A top-p row that keeps few: 28 and 93.
#include <type_traits>

#include "nq_common.h"
#include "nq_internal.h"

namespace nq {
namespace {

constexpr int kMinPDigits = 2048; // values of a digit that cuts a bin
constexpr int kMinPHeld = 8;     // logits a thread keeps in registers where the row fits
constexpr int kMinPVocab = 1 << 20;

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

// An entry of the order: the larger the earlier.
__device__ __forceinline__ uint64_t min_p_entry(float x, int id) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // -0 as 0
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
constexpr float kLargest = 3.4028234663852886e38f;

// The larger of the two; b where a is NaN (fmaxf answers NaN to a signalling one).
__device__ __forceinline__ float larger(float a, float b) { return a > b ? a : b; }

// v of lanes moved by a DPP control word, 0 where none comes from
template <int Ctrl, int Rows>
__device__ __forceinline__ uint64_t dpp64(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v)), Ctrl, Rows, 0xF, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(static_cast<uint32_t>(v >> 32)), Ctrl, Rows, 0xF, false);
    return (static_cast<uint64_t>(hi) << 32) | lo;
}
// Inclusive sums over the 64 lanes: wave_incl_scan's steps.
__device__ __forceinline__ uint64_t wave_scan64(uint64_t v) {
    v += dpp64<0x111, 0xF>(v);
    v += dpp64<0x112, 0xF>(v);
    v += dpp64<0x114, 0xF>(v);
    v += dpp64<0x118, 0xF>(v);
    v += dpp64<0x142, 0xA>(v);
    v += dpp64<0x143, 0xC>(v);
    return v;
}

// Two bounds of a logit, itself within them.  NaN is in none.
struct Span {
    float from, to;
    __device__ __forceinline__ bool has(float x) const { return x >= from && x <= to; }
};

// The same for two bf16 values in a word: with their bits made unsigned integers in the values' order (negative ones
// inverted, the others' first bit set; -0 before 0), a span is [low, low + size).
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
struct ShortSpan {
    u16x2 low, size;
    __device__ __forceinline__ ShortSpan(const Span &s) {
        auto key = [](float x) {
            const uint32_t u = __float_as_uint(x);
            return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
        };
        // a bf16 value's own 32-bit key ends in zeros, a negative one's in ones: the bounds are rounded inwards
        const uint32_t f = s.from == 0.f ? key(-0.f) : key(s.from), t = s.to == 0.f ? key(0.f) : key(s.to);
        const int lo = static_cast<int>(f >= 0x80000000u ? (f - 1 >> 16) + 1 : f >> 16);
        const int hi = static_cast<int>(t >= 0x80000000u ? t >> 16 : t + 1 >> 16) - (t >= 0x80000000u ? 0 : 1);
        low = static_cast<uint16_t>(lo);
        size = static_cast<uint16_t>(s.from <= s.to && hi >= lo ? hi - lo + 1 : 0);
    }
    static __device__ __forceinline__ u16x2 keys(uint32_t w) {
        typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(u16x2, w ^ (__builtin_bit_cast(uint32_t, __builtin_bit_cast(i16x2, w) >> 15) | 0x80008000u));
    }
    // 1 or more where a key is inside
    __device__ __forceinline__ u16x2 inside(u16x2 key) const { return __builtin_elementwise_sub_sat(size, static_cast<u16x2>(key - low)); }
};

// Which logits of four vectors a span holds, a bit a logit, added to a mask a vector at a time: fp32 word w in bit w, bf16's
// halves of word w in bits 15 - w and 31 - w.
struct WordMarks {
    Span in;
    __device__ __forceinline__ WordMarks(const Span &of) : in(of) {}
    __device__ __forceinline__ uint32_t add(uint32_t mask, const uint4 &v, int u) const {
        const float x[4] = {__uint_as_float(v.x), __uint_as_float(v.y), __uint_as_float(v.z), __uint_as_float(v.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e) mask |= in.has(x[e]) ? 1u << (4 * u + e) : 0u;
        return mask;
    }
    static __device__ __forceinline__ uint32_t first(int vectors) { return (1u << (4 * vectors)) - 1; }
};
struct HalfMarks {
    ShortSpan in;
    __device__ __forceinline__ HalfMarks(const Span &of) : in(of) {}
    __device__ __forceinline__ uint32_t add(uint32_t mask, const uint4 &v, int) const {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const u16x2 is = in.inside(ShortSpan::keys(w[e]));
            mask = mask << 1 | __builtin_bit_cast(uint32_t, __builtin_elementwise_min(is, static_cast<u16x2>(1)));
        }
        return mask;
    }
    static __device__ __forceinline__ uint32_t first(int vectors) { return (0xffffu << (16 - 4 * vectors) & 0xffffu) * 0x10001u; }
};

// Sizes by the threads of a row: 1024, or 256 for what they hold in registers.
template <int T>
struct MinPSizes {
    static constexpr int kList = T == 1024 ? 4096 : T * kMinPHeld;  // entries of the list
    static constexpr int kSorted = T / 2 < 256 ? 256 : T / 2;        // entries that are rather sorted, by counting those above each, than cut
    static constexpr int kShift = T == 1024 ? 0 : 3;                // the row's histogram has 128 bins an octave, or 16
    static constexpr int kLast = 45 * (128 >> kShift);
    static constexpr int kEach = kLast / T + 1, kBins = kEach * T;  // bins a thread, and of them all
};

template <int T>
struct MinPShared {
    static constexpr int kWaves = T / kWave;
    alignas(16) uint64_t list[MinPSizes<T>::kList];
    uint64_t hist[MinPSizes<T>::kBins];  // of the row
    uint64_t digits[T == 1024 ? kMinPDigits : 1];
    uint64_t cells[T];  // masses of consecutive ids
    double table[128];
    uint64_t part[kWaves];
    float max[2][kWaves];
    uint64_t found_mass, found, above;
    uint32_t rank[MinPSizes<T>::kSorted];
    uint32_t bin, n;
    int id;
};

// Appends a logit to the list (past its end it is counted alone) as it is: the entry is made when it is read.
template <int T>
__device__ __forceinline__ void append(MinPShared<T> &s, int id, float x) {
    const uint32_t at = __hip_atomic_fetch_add(&s.n, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
    if (at < MinPSizes<T>::kList) s.list[at] = (static_cast<uint64_t>(__float_as_uint(x)) << 32) | static_cast<uint32_t>(id);
}

__device__ __forceinline__ uint64_t listed_entry(uint64_t v) {
    return min_p_entry(__uint_as_float(static_cast<uint32_t>(v >> 32)), static_cast<int>(static_cast<uint32_t>(v)));
}

// Sums over the workgroup of the threads before this one, and of all; two barriers.
template <int T>
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t *part, uint64_t &total) {
    const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    const uint64_t incl = wave_scan64(v);
    if (lane == kWave - 1) part[wave] = incl;
    __syncthreads();
    uint64_t before = incl - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < T / kWave; ++w) {
        before += w < wave ? part[w] : 0;
        total += part[w];
    }
    __syncthreads();
    return before;
}

// 2^(42 + i / 128)
__device__ const double kExp2Table[128] = {
    4398046511104.0, 4421927468748.802, 4445938097632.095, 4470079101855.88,
    4494351189345.363, 4518755071869.717, 4543291465062.945, 4567961088444.878,
    4592764665442.265, 4617702923409.991, 4642776593652.408, 4667986411444.776,
    4693333116054.829, 4718817450764.449, 4744440162891.469, 4770202003811.579,
    4796103728980.37, 4822146097955.479, 4848329874418.864, 4874655826199.207,
    4901124725294.416, 4927737347894.278, 4954494474403.209, 4981396889463.146,
    5008445381976.555, 5035640745129.562, 5062983776415.216, 5090475277656.876,
    5118116055031.72, 5145906919094.391, 5173848684800.761, 5201942171531.834,
    5230188203117.7705, 5258587607862.048, 5287141218565.749, 5315849872551.985,
    5344714411690.448, 5373735682422.1, 5402914535783.991, 5432251827434.224,
    5461748417677.033, 5491405171488.027, 5521222958539.541, 5551202653226.147,
    5581345134690.294, 5611651286848.085, 5642121998415.203, 5672758162932.967,
    5703560678794.538, 5734530449271.263, 5765668382539.163, 5796975391705.564,
    5828452394835.877, 5860100314980.515, 5891920080201.963, 5923912623601.997,
    5956078883349.04, 5988419802705.679, 6020936330056.32, 6053629418935.009,
    6086500028053.38, 6119549121328.781, 6152777667912.536, 6186186642218.362,
    6219777023950.95, 6253549798134.687, 6287505955142.546, 6321646490725.129,
    6355972406039.863, 6390484707680.363, 6425184407705.946, 6460072523671.312,
    6495150078656.382, 6530418101296.299, 6565877625811.596, 6601529692038.518,
    6637375345459.519, 6673415637233.919, 6709651624228.731, 6746084369049.649,
    6782714940072.214, 6819544411473.137, 6856573863261.803, 6893804381311.943,
    6931237057393.474, 6968872989204.515, 7006713280403.578, 7044759040641.932,
    7083011385596.141, 7121471437000.784, 7160140322681.349, 7199019176587.3,
    7238109138825.341, 7277411355692.836, 7316926979711.437, 7356657169660.869,
    7396603090612.919, 7436765913965.6, 7477146817477.495, 7517746985302.307,
    7558567608023.569, 7599609882689.572, 7640875012848.455, 7682364208583.509,
    7724078686548.652, 7766019670004.119, 7808188388852.323, 7850586079673.927,
    7893213985764.103, 7936073357168.994, 7979165450722.371, 8022491530082.486,
    8066052865769.132, 8109850735200.898, 8153886422732.63, 8198161219693.094,
    8242676424422.843, 8287433342312.29, 8332433285839.99, 8377677574611.128,
    8423167535396.213, 8468904502169.985, 8514889816150.538, 8561124825838.647,
    8607610887057.3125, 8654349362991.52, 8701341624228.211, 8748589048796.485,
};

// What a row's weights follow from.  With t = 128 log2(e) (x - max) / T and i = rint(t), e = 2^(i / 128) 2^((t - i) / 128): a
// table, the Taylor series of 2^f for |f| <= 1 / 256 to its fourth power, whose rest is below 2e-15 of it, and an
// exponent; and -i, or -i / 8, is the logit's bin in the row's histogram.  A weight of 1 needs e >= 2^-43, so t is held to
// 45 octaves.
// Every pass gives a logit the same weight, to the last unit, since a target taken from one pass's sums is looked for in
// another's: so this file is built without contraction, and each fma is written out (contracted, t - i took the product
// unrounded in one pass and rounded in another).
template <int kShift>
struct RowRule {
    static constexpr int kPer = 128, kLast = 45 * (kPer >> kShift);
    const double *table;  // in LDS
    double max, turns;    // turns: 128 log2(e) / T
    double lowest;        // of t: -45 octaves
    uint64_t least_weight;  // a smaller one is none (min-p)
    float least;          // no logit below it has a weight (a bound, or the last one kept); NaN and -inf never reach it
    float tie;            // of the logits that equal it (NaN: none do) those with ids behind tie_id have none either
    int tie_id;
    bool bare;            // t keeps above its bound by itself, and least_weight drops no logit
    __device__ __forceinline__ double turn(float x) const {
        // beside an infinite maximum max, turns and lowest are 0 and infinite logits alone count: NaN becomes 0
        return fmax((static_cast<double>(x) - max) * turns, lowest);
    }
    __device__ __forceinline__ int bin(float x) const {  // does not decrease as x falls
        return -static_cast<int>(rint(turn(x))) >> kShift;
    }
    // The bin's logits lie between these two, with room for their roundings; the last bin's reach down to any that counts.
    __device__ __forceinline__ float bin_from(int bin) const {
        const double at = (((bin + 1) << kShift) - 0.5) / turns;
        return bin == kLast ? least : larger(static_cast<float>(max - at - 1e-6 * (fabs(max) + at)), least);
    }
    __device__ __forceinline__ float bin_to(int bin) const {
        const double at = ((bin << kShift) - 0.5) / turns;
        return static_cast<float>(max - at + 1e-6 * (fabs(max) + fabs(at)));
    }
    // The weight by t, whether or not the logit counts.
    __device__ __forceinline__ uint64_t weight(double t, int &bin) const {
        const double n = rint(t), f = t - n;
        const int i = static_cast<int>(n);
        double p = fma(3.583199206380349e-11, f, 2.6466421444330903e-08);  // (ln 2 / 128)^4 / 4!, and so on
        p = fma(p, f, 1.4662262387640426e-05);
        p = fma(p, f, 0.005415212348124573);
        p = fma(p, f, 1.0);
        const uint64_t e = __double_as_longlong(table[i & (kPer - 1)]);
        const uint32_t high = static_cast<uint32_t>(e >> 32) + (static_cast<uint32_t>(i & -kPer) << 13);  // its exponent + i / 128
        // behind 2^52 the integer is in the low bits, rounded
        const double w = fma(p, __longlong_as_double((static_cast<uint64_t>(high) << 32) | static_cast<uint32_t>(e)), 4503599627370496.0);
        bin = -i >> kShift;
        return static_cast<uint64_t>(__double_as_longlong(w)) & 0xfffffffffffffull;
    }
    __device__ __forceinline__ uint64_t weight(float x, int &bin) const {
        const uint64_t w = weight(turn(x), bin);
        return w >= least_weight ? w : 0;
    }
    __device__ __forceinline__ uint64_t bare_weight(float x, int &bin) const {
        return weight((static_cast<double>(x) - max) * turns, bin);
    }
    __device__ __forceinline__ uint64_t weight(uint64_t entry) const {
        int bin;
        const float x = entry_value(entry);
        const uint64_t w = weight(x, bin);
        return counts(x, entry_id(entry)) ? w : 0;
    }
    __device__ __forceinline__ bool counts(float x, int id) const { return x >= least && !(x == tie && id > tie_id); }
    __device__ __forceinline__ bool tied() const { return tie == tie; }
    __device__ __forceinline__ void end_at(uint64_t entry) {  // an entry that counts: none behind it does
        least = tie = entry_value(entry);
        tie_id = entry_id(entry);
    }
};
template <int T>
using Rule = RowRule<MinPSizes<T>::kShift>;

template <typename InT>
__device__ __forceinline__ float logit_at(const InT *row, int id) {
    if constexpr (sizeof(InT) == 2) return bf16_to_f32(row[id]);
    else return row[id];
}

// The ids of a cell, from .. to - 1, at most 2 T of them; a row has T cells at most.
struct Ids {
    int from, to;
};

// A row in registers, thread t the ids t, t + T, ..
template <typename InT, int T>
struct HeldRow {
    static constexpr bool kShort = false, kMemory = false;  // whether its logits are bf16 and many, and in memory
    float x[kMinPHeld];
    int vocab;
    __device__ __forceinline__ HeldRow(const InT *row, int v) : vocab(v) {
#pragma unroll
        for (int i = 0; i < kMinPHeld; ++i) {
            const int id = static_cast<int>(threadIdx.x) + i * T;
            x[i] = id < v ? logit_at(row, id) : -__builtin_inff();
        }
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < kMinPHeld; ++i) {
            const int id = static_cast<int>(threadIdx.x) + i * T;
            if (id < vocab) f(id, x[i]);
        }
    }
    // f for the logits of a span
    template <typename F>
    __device__ __forceinline__ void each_in(const Span &in, F f) const {
        each([&](int id, float v) {
            if (in.has(v)) f(id, v);
        });
    }
    // f for several logits at once: an id, the step to the next, and the logits, NaN where there is none
    template <typename F>
    __device__ __forceinline__ void several(F f) const {
#pragma unroll 1
        for (int i = 0; i < kMinPHeld; i += 4) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = static_cast<int>(threadIdx.x) + (i + e) * T < vocab ? (i ? x[e + 4] : x[e]) : __builtin_nanf("");
            f(static_cast<int>(threadIdx.x) + i * T, T, v);
        }
    }
    // The masses of the cells, 64 ids each.
    template <typename W>
    __device__ __forceinline__ void cells(uint64_t *sum, int, W weigh) const {
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll 1
        for (int i = 0; i < kMinPHeld; i += 4)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float v[1] = {i ? x[e + 4] : x[e]};  // behind the row's end -inf, which does not count
                const uint64_t m = wave_scan64(weigh(static_cast<int>(threadIdx.x) + (i + e) * T, v));
                if (lane == kWave - 1) sum[(i + e) * (T / kWave) + wave] = m;
            }
    }
    __device__ __forceinline__ Ids cell_ids(int cell, int) const { return {cell * kWave, min(vocab, cell * kWave + kWave)}; }
};
static_assert(kMinPHeld == 8, "two groups of four");

// What is left of a row, the n <= kMost logits of a list as append() left them, in registers: the list is free for others behind
// the constructor.  No entry is 0.
template <int T, int kMost = MinPSizes<T>::kList>
struct HeldList {
    static constexpr bool kShort = false, kMemory = false;
    static constexpr int kEach = kMost / T;
    uint64_t e[kEach];
    __device__ __forceinline__ HeldList(const MinPShared<T> &s, int n) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int at = static_cast<int>(threadIdx.x) + i * T;
            e[i] = at < n ? listed_entry(s.list[at]) : 0;
        }
        __syncthreads();
    }
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (e[i]) f(entry_id(e[i]), entry_value(e[i]));
    }
    template <typename F>
    __device__ __forceinline__ void entries(F f) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (e[i]) f(e[i]);
    }
    template <typename F>
    __device__ __forceinline__ void each_in(const Span &in, F f) const {
        each([&](int id, float v) {
            if (in.has(v)) f(id, v);
        });
    }
    template <typename F>
    __device__ __forceinline__ void several(F f) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const float v[1] = {e[i] ? entry_value(e[i]) : __builtin_nanf("")};
            f(entry_id(e[i]), 1, v);
        }
    }
    // The masses of the cells, as many ids each, a power of two, as make them T at most.
    static __device__ __forceinline__ int cell_bits(int vocab) {
        constexpr int kBits = T == 1024 ? 10 : 8;
        static_assert(1 << kBits == T && (T < 1024 || kMinPVocab <= T * 2 * T));
        return max(0, 32 - kBits - __clz(max(1, vocab - 1)));
    }
    template <typename W>
    __device__ __forceinline__ void cells(uint64_t *sum, int vocab, W weigh) const {
        const int bits = cell_bits(vocab);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (!e[i]) continue;
            const float v[1] = {entry_value(e[i])};
            atomicAdd(reinterpret_cast<unsigned long long *>(&sum[entry_id(e[i]) >> bits]), weigh(entry_id(e[i]), v));
        }
    }
    __device__ __forceinline__ Ids cell_ids(int cell, int vocab) const {
        const int bits = cell_bits(vocab);
        return {cell << bits, min(vocab, (cell + 1) << bits)};
    }
};

// A row in memory: 16 bytes a load from the first address that allows them, head logits before and some behind.
template <typename InT, int T>
struct FarRow {
    const InT *row;
    int vocab, head, nv;
    static constexpr int V = 16 / sizeof(InT);
    static constexpr bool kShort = sizeof(InT) == 2, kMemory = true;
    __device__ __forceinline__ FarRow(const InT *r, int v) : row(r), vocab(v) {
        head = min(v, static_cast<int>((16 - reinterpret_cast<uintptr_t>(r) % 16) % 16 / sizeof(InT)));
        nv = (v - head) / V;
    }
    __device__ __forceinline__ uint4 load(int j) const {
        return j < nv ? reinterpret_cast<const uint4 *>(row + head)[j] : make_uint4(0, 0, 0, 0);
    }
    static __device__ __forceinline__ void unpack(const uint4 &v, float (&x)[V]) {
        if constexpr (V == 8) {
            unpack8(v, x);
        } else {
            x[0] = __uint_as_float(v.x);
            x[1] = __uint_as_float(v.y);
            x[2] = __uint_as_float(v.z);
            x[3] = __uint_as_float(v.w);
        }
    }
    // f for the logits outside the whole vectors (fewer than T)
    template <typename F>
    __device__ __forceinline__ void few(F f) const {
        const int i = threadIdx.x, id = i < head ? i : i + nv * V;
        if (id < vocab) f(id, logit_at(row, id));
    }
    // f for each whole vector and its number, one for the logits outside them.  Four vectors of a thread are in flight.
    template <typename F, typename G>
    __device__ __forceinline__ void vectors(F f, G one) const {
        constexpr int U = 4;
        const int tid = threadIdx.x;
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(tid + u * T);
        few(one);
#pragma unroll 1
        for (int j = tid; j < nv; j += U * T) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (j + u * T >= nv) break;
                const uint4 r = v[u];
                v[u] = load(j + (u + U) * T);
                f(j + u * T, r);
            }
        }
    }
    // The masses of the cells: the logits before the vectors, those of 256 vectors each (fp32: 512), those behind.  A wave takes 256
    // vectors, so that its lanes' sums meet once in as many logits; four vectors of a thread are in flight.
    static constexpr int kPart = 4 * kWave, kCell = kPart * 8 / V;  // vectors
    template <typename W>
    __device__ __forceinline__ void cells(uint64_t *sum, int, W weigh) const {
        constexpr int U = kPart / kWave, kWaves = T / kWave;
        static_assert(kMinPVocab / V / kCell + 2 <= T && kCell * V <= 2 * T);
        const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(wave * kPart + u * kWave + lane);
        few([&](int id, float x) {
            const float one[1] = {x};
            atomicAdd(reinterpret_cast<unsigned long long *>(&sum[cell_of(id)]), weigh(id, one));
        });
#pragma unroll 1
        for (int c = wave; c * kPart < nv; c += kWaves) {
            uint64_t m = 0;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int j = c * kPart + u * kWave + lane;
                const uint4 r = v[u];
                v[u] = load(j + kWaves * kPart);
                if (j >= nv) continue;
                float x[V];
                unpack(r, x);
                m += weigh(head + j * V, x);
            }
            m = wave_scan64(m);
            if (lane == kWave - 1) atomicAdd(reinterpret_cast<unsigned long long *>(&sum[1 + c * kPart / kCell]), m);
        }
    }
    __device__ __forceinline__ int cell_of(int id) const {
        const int n = (nv + kCell - 1) / kCell;
        return id < head ? 0 : id >= head + nv * V ? n + 1 : 1 + (id - head) / (kCell * V);
    }
    __device__ __forceinline__ Ids cell_ids(int cell, int) const {
        const int end = head + nv * V, at = head + (cell - 1) * kCell * V;
        return cell == 0 ? Ids{0, head} : at >= end ? Ids{end, vocab} : Ids{at, min(end, at + kCell * V)};
    }
    // f for several logits at once: an id, the step to the next, and the logits
    template <typename F>
    __device__ __forceinline__ void several(F f) const {
        vectors(
            [&](int j, const uint4 &r) {
                float x[V];
                unpack(r, x);
                f(head + j * V, 1, x);
            },
            [&](int id, float x) {
                const float v[1] = {x};
                f(id, 1, v);
            });
    }
    // f for the logits of four vectors, the thread's j, j + T, .., whose bits are set.  A lane's logits come one after the
    // other, picked out of its registers: f is there once, where a copy behind a test of each logit costs the tests of all and the
    // fetch of 32 copies.
    template <typename F>
    __device__ __forceinline__ void marked(const uint4 (&r)[4], uint32_t mask, int j, F f) const {
        while (mask) {
            const int at = __builtin_ctz(mask), w = V == 8 ? 15 - (at & 15) : at;
            mask &= mask - 1;
            uint32_t q[8];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                q[2 * u] = w & 1 ? r[u].y : r[u].x;
                q[2 * u + 1] = w & 1 ? r[u].w : r[u].z;
            }
#pragma unroll
            for (int n = 4, bit = 2; n > 0; n >>= 1, bit <<= 1)
#pragma unroll
                for (int i = 0; i < n; ++i) q[i] = w & bit ? q[2 * i + 1] : q[2 * i];
            const int id = head + (j + (w >> 2) * T) * V + (w & 3) * (V / 4);
            if constexpr (V == 4) f(id, __uint_as_float(q[0]));
            else f(id + (at >> 4), __uint_as_float(at >= 16 ? q[0] & 0xffff0000u : q[0] << 16));
        }
    }
    // f for the logits of a span, which are few.  64 x 65537 bf16, a pass 4 us where a test in every logit's place took 6 to 8;
    // 131072 fp32 logits 10 us alone, 18 beside 255 other rows, which is the memory's rate.
    template <typename F>
    __device__ __forceinline__ void each_in(const Span &in, F f) const {
        each_in(in, f, f);
    }
    // the same with a function of its own for the logits outside whole vectors
    template <typename F, typename G>
    __device__ __forceinline__ void each_in(const Span &in, F f, G one) const {
        constexpr int U = 4;
        const int tid = threadIdx.x;
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(tid + u * T);
        few([&](int id, float x) {
            if (in.has(x)) one(id, x);
        });
        const typename std::conditional<V == 8, HalfMarks, WordMarks>::type marks(in);
#pragma unroll 1
        for (int j = tid; j < nv; j += U * T) {
            uint32_t mask = 0;
            uint4 r[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                mask = marks.add(mask, v[u], u);
                r[u] = v[u];
                v[u] = load(j + (u + U) * T);
            }
            const int whole = min(U, (nv - j + T - 1) / T);  // vectors that are there
            marked(r, mask & marks.first(whole), j, f);
        }
    }
    // The largest logit of this thread's part, and in `where` the first vector that holds its vectors' largest (-1: none).
    __device__ __forceinline__ float first_pass(int &where) const {
        float top = -__builtin_inff();
        where = -1;
        several([&](int id, int, const auto &x) {
            constexpr int N = sizeof(x) / sizeof(float);
            float high = larger(x[0], -__builtin_inff());
#pragma unroll
            for (int e = 1; e < N; ++e) high = larger(x[e], high);
            if (N == V) where = high > top ? (id - head) / V : where;
            if (N == V) top = larger(high, top);
        });
        few([&](int, float x) { top = larger(x, top); });
        return top;
    }
    // The same without `where`, and after each batch of loads: the largest so far of all threads goes through least(), and put takes
    // every logit of the batch from that on.
    template <typename L, typename P>
    __device__ __forceinline__ float first_pass(MinPShared<T> &s, L least, P put) const {
        constexpr int U = 8;
        const int tid = threadIdx.x;
        float top = -__builtin_inff();
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load(tid + u * T);
#pragma unroll 1
        for (int b = 0, turn = 0; b < nv; b += U * T, turn ^= 1) {
            float high[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float x[V];
                unpack(v[u], x);
                high[u] = larger(x[0], -__builtin_inff());
#pragma unroll
                for (int e = 1; e < V; ++e) high[u] = larger(x[e], high[u]);
                high[u] = b + tid + u * T < nv ? high[u] : -__builtin_inff();
                top = larger(high[u], top);
            }
            const float m = group_max<kWave>(top);
            if (tid % kWave == 0) s.max[turn][tid / kWave] = m;
            __syncthreads();
            float all = s.max[turn][0];
#pragma unroll
            for (int w = 1; w < T / kWave; ++w) all = fmaxf(all, s.max[turn][w]);
            const float from = least(all);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                uint4 r = v[u];
                v[u] = load(b + tid + (u + U) * T);
                if (!(high[u] >= from)) continue;
                const int id = head + (b + tid + u * T) * V;
#pragma unroll 1
                for (int e = 0; e < V; ++e) {
                    const float x = __uint_as_float(V == 8 ? r.x << 16 : r.x);
                    if (V == 8) {
                        r.x = __builtin_amdgcn_alignbit(r.y, r.x, 16);
                        r.y = __builtin_amdgcn_alignbit(r.z, r.y, 16);
                        r.z = __builtin_amdgcn_alignbit(r.w, r.z, 16);
                        r.w >>= 16;
                    } else {
                        r = make_uint4(r.y, r.z, r.w, 0);
                    }
                    put(id + e, x, from);
                }
            }
        }
        few([&](int id, float x) {
            top = larger(x, top);
            put(id, x, -3.4028234663852886e38f);
        });
        return top;
    }
    // f for this thread's logits outside whole vectors and those of one
    template <typename F>
    __device__ __forceinline__ void vector(int j, F f) const {
        few(f);
        if (j < 0) return;
#pragma unroll 1
        for (int e = 0; e < V; ++e) f(head + j * V + e, logit_at(row, head + j * V + e));
    }
};

// Sorts the list's n entries in descending order (all threads): a few by counting those above each, several threads a
// counted entry; more by a network.
template <int T>
__device__ __forceinline__ void sort_list(MinPShared<T> &s, int n) {
    const int tid = threadIdx.x;
    if (n <= MinPSizes<T>::kSorted) {
        const int span = n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512, parts = T / span;
        static_assert(MinPSizes<T>::kSorted <= T, "a thread an entry at least");
        const int i = tid & (span - 1), each = ((n + parts - 1) / parts + 1) & ~1;
        const int from = min(n, tid / span * each), to = min(n, from + each);
        for (int j = tid; j < span; j += T) s.rank[j] = 0;
        const uint64_t mine = i < n ? s.list[i] : 0;
        if (tid == 0 && n % 2) s.list[n] = 0;  // entries are read in pairs
        __syncthreads();
        uint32_t above = 0;
#pragma unroll 4
        for (int j = from; j < to; j += 2) {
            const ulonglong2 e = *reinterpret_cast<const ulonglong2 *>(s.list + j);
            above += (e.x > mine ? 1u : 0u) + (e.y > mine ? 1u : 0u);
        }
        if (i < n && above) atomicAdd(&s.rank[i], above);
        __syncthreads();
        if (tid < n) s.list[s.rank[tid]] = mine;  // thread tid < span holds entry tid
        __syncthreads();
        return;
    }
    int n2 = 2;
    while (n2 < n) n2 <<= 1;
    for (int i = n + tid; i < n2; i += T) s.list[i] = 0;
    __syncthreads();
    for (int kk = 2; kk <= n2; kk <<= 1)
        for (int j = kk >> 1; j > 0; j >>= 1) {
            for (int i = tid; i < n2 / 2; i += T) {
                const int lo = 2 * i - (i & (j - 1));
                const uint64_t a = s.list[lo], b = s.list[lo + j];
                if (((lo & kk) == 0) == (a < b)) {
                    s.list[lo] = b;
                    s.list[lo + j] = a;
                }
            }
            __syncthreads();
        }
}

// The sums of a sorted list: thread t has the ranks t E .. t E + E - 1, E = ceil(n / T).
template <int T>
struct ListSums {
    static constexpr int kEach = MinPSizes<T>::kList / T;
    uint64_t cum[kEach];
    uint64_t before;
    int first, end;
    __device__ __forceinline__ ListSums(MinPShared<T> &s, int n, uint64_t above, const Rule<T> &rule) {
        const int each = (n + T - 1) / T;
        first = min(n, static_cast<int>(threadIdx.x) * each);
        end = min(n, first + each);
        uint64_t own = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (first + i < end) own += rule.weight(s.list[first + i]);
            cum[i] = own;
        }
        uint64_t total;
        before = above + block_before<T>(own, s.part, total);
#pragma unroll
        for (int i = 0; i < kEach; ++i) cum[i] += before;
    }
    // The first rank whose mass reaches the target, which the list's last does: its entry, s.found, and the mass through it, s.found_mass.
    __device__ __forceinline__ void find_mass(MinPShared<T> &s, uint64_t target) const {
        uint64_t last = before;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (first + i < end && last < target && target <= cum[i]) {
                s.found_mass = cum[i];
                s.found = s.list[first + i];
            }
            last = cum[i];
        }
        __syncthreads();
    }
    __device__ __forceinline__ void find_rank(MinPShared<T> &s, int rank) const {
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (first + i < end && first + i == rank) s.found_mass = cum[i];
        __syncthreads();
    }
};

// The least integer that p (in [0, 1]) of a mass asks for, at least 1.
__device__ __forceinline__ uint64_t share(double p, uint64_t mass) {
    const uint64_t t = static_cast<uint64_t>(ceil(p * static_cast<double>(mass)));
    return t < 1 ? 1 : t > mass ? mass : t;
}

struct RowCuts {
    int k;
    double p, u;
};

// The token of a row whose weights are all among the list's n <= 64 logits, by one wave, a logit a lane: each counts the logits
// and the ids before its own, and the weights are summed in either order.
template <int T>
__device__ __forceinline__ int draw_from_few(const MinPShared<T> &s, int n, const Rule<T> &rule, const RowCuts &c) {
    const int lane = threadIdx.x & (kWave - 1);
    const uint64_t mine = lane < n ? listed_entry(s.list[lane]) : 0;
    uint64_t own = lane < n ? rule.weight(mine) : 0;
    int rank = 0, place = 0;
    for (int j = 0; j < n; ++j) {
        const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(mine)), j);
        const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(static_cast<uint32_t>(mine >> 32)), j);
        rank += ((static_cast<uint64_t>(hi) << 32) | lo) > mine ? 1 : 0;
        place += lo > static_cast<uint32_t>(mine) ? 1 : 0;  // a smaller id's lower half is larger
    }
    if (lane >= n) rank = place = lane;
    auto sums = [&](int to) {  // of the weights, lane r's first moved to lane `to`
        const uint32_t lo = __builtin_amdgcn_ds_permute(4 * to, static_cast<int>(static_cast<uint32_t>(own)));
        const uint32_t hi = __builtin_amdgcn_ds_permute(4 * to, static_cast<int>(static_cast<uint32_t>(own >> 32)));
        return wave_scan64((static_cast<uint64_t>(hi) << 32) | lo);
    };
    auto at = [](uint64_t v, int j) { return static_cast<uint64_t>(__shfl(static_cast<unsigned long long>(v), j, kWave)); };
    auto first = [](bool reached) { return __ffsll(static_cast<long long>(__ballot(reached))) - 1; };
    if (c.k < n || c.p < 1.0) {
        const uint64_t cum = sums(rank), mass = at(cum, min(c.k, n) - 1);
        if (rank > first(cum >= (c.p < 1.0 ? share(c.p, mass) : mass))) own = 0;
    }
    const uint64_t cum = sums(place);
    const int id = __builtin_amdgcn_ds_permute(4 * place, entry_id(mine));
    return __shfl(id, first(cum >= share(c.u, at(cum, kWave - 1))), kWave);
}

// A histogram's sums: thread t has the bins t E .. t E + E - 1.
template <int T, int kEach = MinPSizes<T>::kEach>
struct BinSums {
    uint64_t h[kEach], before, total;
    __device__ __forceinline__ BinSums(MinPShared<T> &s, const uint64_t *hist, uint64_t above) {
        uint64_t own = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int bin = kEach * threadIdx.x + i;
            h[i] = hist[bin];
            own += h[i];
        }
        before = above + block_before<T>(own, s.part, total);
    }
    // The first bin at which the sum reaches the target (the last does): s.bin, s.above before it, s.found_mass through it.
    __device__ __forceinline__ void find(MinPShared<T> &s, uint64_t target) const {
        uint64_t at = before;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (at < target && target <= at + h[i]) {
                s.bin = kEach * threadIdx.x + i;
                s.above = at;
                s.found_mass = at + h[i];
            }
            at += h[i];
        }
        __syncthreads();
    }
};

// The token of a row by what is kept of it: the first id at which the sum of the masses reaches u of the whole.  The cells'
// masses say in which one, and its logits are read again, two a thread.
template <int T, typename Row, typename InT>
__device__ __forceinline__ int draw_by_ids(MinPShared<T> &s, const Row &row, const InT *logits, const Rule<T> &rule,
                                           double u, int vocab) {
    s.cells[threadIdx.x] = 0;
    __syncthreads();
    auto weigh = [&](int id, const auto &x) {
        constexpr int N = sizeof(x) / sizeof(float);
        uint64_t sum = 0;
        int bin;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint64_t w = rule.weight(x[e], bin);
            sum += rule.counts(x[e], id + e) ? w : 0;
        }
        return sum;
    };
    auto weigh_bare = [&](int id, const auto &x) {
        constexpr int N = sizeof(x) / sizeof(float);
        uint64_t sum = 0;
        int bin;
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const uint64_t w = rule.bare_weight(x[e], bin);
            sum += rule.counts(x[e], id + e) ? w : 0;
        }
        return sum;
    };
    if (Row::kMemory && rule.bare) row.cells(s.cells, vocab, weigh_bare);
    else row.cells(s.cells, vocab, weigh);
    __syncthreads();
    const BinSums<T, 1> sums(s, s.cells, 0);
    const uint64_t target = share(u, sums.total);
    sums.find(s, target);
    const Ids ids = row.cell_ids(static_cast<int>(s.bin), vocab);
    const int id = ids.from + 2 * static_cast<int>(threadIdx.x);
    uint64_t w[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const float x[1] = {id + e < ids.to ? logit_at(logits, id + e) : -__builtin_inff()};
        w[e] = weigh(id + e, x);
    }
    uint64_t all;
    const uint64_t before = s.above + block_before<T>(w[0] + w[1], s.part, all);
    if (before < target && target <= before + w[0] + w[1]) s.id = target <= before + w[0] ? id : id + 1;
    __syncthreads();
    return s.id;
}

// The token of a row whose kept logits are all in the list, n <= MinPSizes<T>::kSorted, and, where top-k keeps the whole list, none but
// them (for thread 0).
template <int T, typename InT>
__device__ __forceinline__ int draw_from_list(MinPShared<T> &s, int n, const InT *logits, Rule<T> &rule, const RowCuts &c,
                                              int vocab) {
    if (n <= kWave) return threadIdx.x < kWave ? draw_from_few<T>(s, n, rule, c) : 0;
    const HeldList<T, (MinPSizes<T>::kSorted > T ? MinPSizes<T>::kSorted : T)> listed(s, n);
    if ((c.k < vocab && c.k <= n) || c.p < 1.0) {
        const int k = min(c.k, n);
        if (static_cast<int>(threadIdx.x) < n) s.list[threadIdx.x] = listed.e[0];
        __syncthreads();
        sort_list<T>(s, n);
        if (c.p < 1.0) {
            const ListSums<T> sums(s, n, 0, rule);
            sums.find_rank(s, k - 1);
            const uint64_t mass = s.found_mass;
            __syncthreads();
            sums.find_mass(s, share(c.p, mass));
            rule.end_at(s.found);
        } else {
            rule.end_at(s.list[k - 1]);
        }
    }
    return draw_by_ids<T>(s, listed, logits, rule, c.u, vocab);
}

// The row's histogram: of counts (kMass false) or of masses.  The list's counter is cleared besides.
template <bool kMass, int T, typename Row>
__device__ __forceinline__ void row_histogram(MinPShared<T> &s, const Row &row, const Rule<T> &rule) {
    for (int i = threadIdx.x; i < MinPSizes<T>::kBins; i += T) s.hist[i] = 0;
    if (threadIdx.x == 0) s.n = 0;
    auto weigh = [&](int id, int step, const auto &x) {
        constexpr int N = sizeof(x) / sizeof(float);
        int bin[N];
        uint64_t w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = rule.weight(x[e], bin[e]);
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (rule.counts(x[e], id + e * step)) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[bin[e]]), w[e]);
    };
    // A pass is bound by its vector instructions: without what a row does not need they are 21 a logit instead of 31.
    auto weigh_bare = [&](int, int, const auto &x) {
        constexpr int N = sizeof(x) / sizeof(float);
        int bin[N];
        uint64_t w[N];
#pragma unroll
        for (int e = 0; e < N; ++e) w[e] = rule.bare_weight(x[e], bin[e]);
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (x[e] >= rule.least) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[bin[e]]), w[e]);
    };
    if constexpr (!kMass) {
        __syncthreads();
        row.several([&](int id, int step, const auto &x) {
            constexpr int N = sizeof(x) / sizeof(float);
#pragma unroll
            for (int e = 0; e < N; ++e)
                if (rule.counts(x[e], id + e * step)) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[rule.bin(x[e])]), 1ull);
        });
    } else if (!rule.bare || rule.tied()) {
        __syncthreads();
        row.several(weigh);
    } else if constexpr (!Row::kShort) {
        __syncthreads();
        row.several(weigh_bare);
    } else {
        // A bf16 row repeats its values: they are counted where the list will be, 32 binades of either sign down from the
        // largest that counts, and each is weighed once, 5 instructions a logit instead of 21 (65537 logits 8 us).  Counter 0 of a
        // sign has what is smaller and zero, the last one what is larger (NaN, and what is too far below the maximum to count).
        constexpr int kHalf = MinPSizes<T>::kList;  // 32-bit counters of a sign
        static_assert(kHalf == 4096, "the sign's bit, moved by three, and the numbers share 16 bits");
        uint32_t *const count = reinterpret_cast<uint32_t *>(s.list);
        for (int i = threadIdx.x; i < 2 * kHalf; i += T) count[i] = 0;
        __syncthreads();
        const float high = fmaxf(fabsf(static_cast<float>(rule.max)), fabsf(rule.least));
        const int base = max(0, static_cast<int>((__float_as_uint(high) >> 16) & 0x7f80u) + 128 + 1 - kHalf);
        auto one = [&](int id, float x) {
            const float v[1] = {x};
            weigh(id, 1, v);
        };
        row.vectors(
            [&](int, const uint4 &r) {
                const uint32_t w[4] = {r.x, r.y, r.z, r.w};
                const u16x2 low = static_cast<uint16_t>(base), last = static_cast<uint16_t>(kHalf - 1);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const u16x2 size = __builtin_bit_cast(u16x2, w[e] & 0x7fff7fffu);
                    const u16x2 at = __builtin_elementwise_min(__builtin_elementwise_sub_sat(size, low), last);
                    const uint32_t both = __builtin_bit_cast(uint32_t, at) | (w[e] >> 3 & 0x10001000u);
                    atomicAdd(&count[both & 0xffffu], 1u);
                    atomicAdd(&count[both >> 16], 1u);
                }
            },
            one);
        __syncthreads();
        const bool small = base > 0 && count[0] + count[kHalf] > 0;
#pragma unroll 1
        for (int i = threadIdx.x; i < 2 * kHalf; i += T) {
            const uint32_t c = count[i], at = i % kHalf;
            const float x = __uint_as_float(((at + base) << 16) | (i >= kHalf ? 0x80000000u : 0u));
            if (c == 0 || at == kHalf - 1 || (at == 0 && base > 0) || !(x >= rule.least)) continue;
            int bin;
            const uint64_t w = rule.weight(x, bin);
            atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[bin]), c * w);
        }
        if (small) {
            const float most = __uint_as_float(static_cast<uint32_t>(base) << 16);
            row.each_in({-most, most}, one, [](int, float) {});  // those outside whole vectors are weighed
        }
    }
    __syncthreads();
}

// Of the listed logits those in question, in order, and the first at which the sum of counts or masses reaches the target
// (the last does): s.found, and the mass through it, s.found_mass.
template <int T, typename Q>
__device__ __forceinline__ void pick(MinPShared<T> &s, const HeldList<T> &listed, const Rule<T> &rule, uint64_t above,
                                     uint64_t target, bool mass, Q in_question) {
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    listed.entries([&](uint64_t e) {
        if (in_question(e)) s.list[atomicAdd(&s.n, 1u)] = e;
    });
    __syncthreads();
    const int n = static_cast<int>(s.n);
    sort_list<T>(s, n);
    if (mass) {
        ListSums<T>(s, n, above, rule).find_mass(s, target);
    } else {
        if (threadIdx.x == 0) s.found = s.list[target - above - 1];
        __syncthreads();
    }
    if (threadIdx.x == 0) s.n = 0;
}

// The entry at which the sum of counts or masses reaches the target, s.found, and the mass through it, s.found_mass, from the
// row's histogram of that kind, whose whole sum reaches it.  A bin that overflows the list is cut by the digits of an
// entry, ten or eleven bits at a time (32 of the logit, 20 of the id), until one does not; the last digits leave one entry.
template <int T, typename Row>
__device__ __forceinline__ void locate(MinPShared<T> &s, const Row &row, const Rule<T> &rule, const BinSums<T> &sums,
                                       uint64_t target, bool mass) {
    uint64_t prefix = 0, mask = 0;
    sums.find(s, target);
    const int bin = static_cast<int>(s.bin);
    uint64_t above = s.above;
    const Span in = {rule.bin_from(bin), rule.bin_to(bin)};
    auto in_question = [&](uint64_t e) {
        const float v = entry_value(e);
        return rule.bin(v) == bin && rule.counts(v, entry_id(e)) && (e & mask) == prefix;
    };
    constexpr int kBits = 11;
    static_assert(1 << kBits == kMinPDigits, "a digit fills the histogram");
    int shift = 64, bins = 0;  // the digits down to bit `shift` are known
    for (bool list = true;; list = !list) {
        if (!list) {
            if (shift == 32) {  // bits 20 .. 31 are ones in every entry
                shift = 20;
                mask |= 0xfff00000ull;
                prefix |= 0xfff00000ull;
            }
            const int bits = min(kBits, shift > 32 ? shift - 32 : shift);
            shift -= bits;
            bins = 1 << bits;
            for (int i = threadIdx.x; i < kMinPDigits && T == 1024; i += T) s.digits[i] = 0;
            if (threadIdx.x == 0) s.n = 0;
            __syncthreads();
        }
        if (list) {
            // a few logits beside the bin's own come along at first: the look at them waits until they are listed
            if (mask == 0) {
                row.each_in(in, [&](int id, float v) { append<T>(s, id, v); });
            } else {
                row.each_in(in, [&](int id, float v) {
                    if (in_question(min_p_entry(v, id))) append<T>(s, id, v);
                });
            }
        } else {
            row.each_in(in, [&](int id, float v) {
                const uint64_t e = min_p_entry(v, id);
                const int at = bins - 1 - (static_cast<int>(e >> shift) & (bins - 1));
                if (in_question(e)) atomicAdd(reinterpret_cast<unsigned long long *>(&s.digits[at]), mass ? rule.weight(e) : 1);
            });
        }
        __syncthreads();
        if (list) {
            if (T < 1024 || s.n <= MinPSizes<T>::kList) break;
            __syncthreads();  // all have read the count that the next pass clears
        } else {
            BinSums<T, T == 1024 ? kMinPDigits / T : 1>(s, s.digits, above).find(s, target);
            above = s.above;
            prefix |= static_cast<uint64_t>(bins - 1 - s.bin) << shift;
            mask |= static_cast<uint64_t>(bins - 1) << shift;
        }
    }
    pick<T>(s, HeldList<T>(s, static_cast<int>(s.n)), rule, above, target, mass, in_question);
}

// The token of a row by its histograms.
template <int T, typename Row, typename InT>
__device__ __forceinline__ int draw_by_bins(MinPShared<T> &s, const Row &row, const InT *logits, Rule<T> &rule,
                                            const RowCuts &c, int vocab) {
    // top-k: its last entry, or, where few are before it, those
    if (c.k < vocab) {
        row_histogram<false, T>(s, row, rule);
        const BinSums<T> sums(s, s.hist, 0);
        if (sums.total > static_cast<uint64_t>(c.k)) {
            if (c.k <= MinPSizes<T>::kSorted) {
                sums.find(s, c.k);
                const int bin = static_cast<int>(s.bin);
                if (s.found_mass <= MinPSizes<T>::kSorted) {
                    row.each_in({rule.bin_from(bin), __builtin_inff()}, [&](int id, float v) {
                        if (rule.counts(v, id) && rule.bin(v) <= bin) append<T>(s, id, v);
                    });  // at most MinPSizes<T>::kSorted
                    __syncthreads();
                    return draw_from_list<T>(s, static_cast<int>(s.n), logits, rule, c, vocab);
                }
                __syncthreads();
            }
            locate<T>(s, row, rule, sums, c.k, false);
            rule.end_at(s.found);
            __syncthreads();
        }
    }
    // top-p: its last entry, by the masses
    if (c.p < 1.0) {
        row_histogram<true, T>(s, row, rule);
        const BinSums<T> sums(s, s.hist, 0);
        locate<T>(s, row, rule, sums, share(c.p, sums.total), true);
        rule.end_at(s.found);
        __syncthreads();
    }
    return draw_by_ids<T>(s, row, logits, rule, c.u, vocab);
}

template <typename InT, int T, bool kHeld>
__global__ void __launch_bounds__(T)
min_p_kernel(MinPArgs a) {
    __shared__ MinPShared<T> s;
    typedef typename std::conditional<kHeld, HeldRow<InT, T>, FarRow<InT, T>>::type Row;
    const int64_t r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const InT *const logits = static_cast<const InT *>(a.logits) + r * a.s0;
    const Row row(logits, a.vocab);
    const float temperature = a.temperature[r], mp = a.min_p[r], pq = a.top_p[r], uq = a.uniforms[r];
    const int kq = a.top_k[r];
    const bool greedy = !(temperature > 0.f);
    const double min_p = mp > 0.f ? (mp < 1.f ? mp : 1.0) : 0.0;
    const RowCuts cuts = {kq > 0 && kq < a.vocab ? kq : a.vocab, pq < 1.f ? (pq > 0.f ? pq : 0.0) : 1.0,
                          uq > 0.f ? (uq < 1.f ? uq : 1.0) : 0.0};
    const double reach = temperature * log(fmax(min_p, 0x1p-43));
    // The least logit that can have a weight beside a maximum; the margins cover the roundings many times over.
    auto least = [&](float max) {
        return max > kLargest ? max
                              : larger(static_cast<float>(max + reach - 1e-6 * (fabs(static_cast<double>(max)) - reach)), -kLargest);
    };
    if (tid < 128) s.table[tid] = kExp2Table[tid];
    if (tid == 0) {
        s.n = 0;
        s.id = a.vocab;
    }
    __syncthreads();

    // 1. the maximum, and, where min-p may leave few, the list of what it leaves
    float top = -__builtin_inff();
    int where = -1;
    if constexpr (kHeld) {
        row.each([&](int, float v) { top = larger(v, top); });
    } else {
        if (!greedy && min_p > 0.0) {
            top = row.first_pass(s, least, [&](int id, float v, float from) {
                if (v >= from) append<T>(s, id, v);
            });
            __syncthreads();  // the batches' maxima are read
        } else {
            top = row.first_pass(where);
        }
    }
    const float own = top;
    top = group_max<kWave>(top);
    if (lane == 0) s.max[0][wave] = top;
    __syncthreads();
    top = s.max[0][0];
#pragma unroll
    for (int w = 1; w < T / kWave; ++w) top = fmaxf(top, s.max[0][w]);
    if (greedy || top == -__builtin_inff()) {
        if (own == top) {
            auto first = [&](int id, float v) {
                if (v == top) atomicMin(&s.id, id);
            };
            if constexpr (kHeld) row.each(first);
            else row.vector(where, first);
        }
        __syncthreads();
        if (tid == 0) a.tokens[r] = top == -__builtin_inff() ? 0 : s.id;
        return;
    }
    Rule<T> rule;
    rule.table = s.table;
    rule.max = top > kLargest ? 0.0 : top;
    rule.turns = top > kLargest ? 0.0 : 128.0 * 1.4426950408889634 / temperature;
    rule.lowest = top > kLargest ? 0.0 : -45.0 * 128.0;
    rule.least_weight = static_cast<uint64_t>(ceil(min_p * 4398046511104.0));
    rule.least = least(top);
    rule.bare = rule.least_weight == 0 && top <= kLargest && (rule.least - rule.max) * rule.turns >= rule.lowest;
    rule.tie = __builtin_nanf("");
    rule.tie_id = 0;
    const int found = static_cast<int>(s.n);
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    if constexpr (kHeld) {
        row.each([&](int id, float v) {
            if (rule.counts(v, id)) append<T>(s, id, v);
        });
    } else if (found > 0 && found <= MinPSizes<T>::kList) {
        const HeldList<T> list(s, found);
        list.each([&](int id, float v) {
            if (rule.counts(v, id)) append<T>(s, id, v);
        });
    } else if (cuts.k <= T / 2) {
        // the k-th largest of the threads' own maxima, or its bin: as many logits reach it, and few more
        for (int i = tid; i < MinPSizes<T>::kBins; i += T) s.hist[i] = 0;
        __syncthreads();
        if (own >= rule.least) atomicAdd(reinterpret_cast<unsigned long long *>(&s.hist[rule.bin(own)]), 1ull);
        __syncthreads();
        const BinSums<T> sums(s, s.hist, 0);
        if (sums.total >= static_cast<uint64_t>(cuts.k)) {
            sums.find(s, cuts.k);
            rule.least = rule.bin_from(static_cast<int>(s.bin));  // nothing below it is kept
            row.each_in({rule.least, __builtin_inff()}, [&](int id, float v) { append<T>(s, id, v); });
        }
    }
    __syncthreads();
    const int n = static_cast<int>(s.n);
    int token;
    if (n > 0 && n <= MinPSizes<T>::kSorted) {
        token = draw_from_list<T>(s, n, logits, rule, cuts, a.vocab);
    } else {
        __syncthreads();
        if constexpr (kHeld) {
            token = draw_by_bins<T>(s, row, logits, rule, cuts, a.vocab);
        } else if (n > 0 && n <= MinPSizes<T>::kList) {
            const HeldList<T> list(s, n);
            token = draw_by_bins<T>(s, list, logits, rule, cuts, a.vocab);
        } else {
            token = draw_by_bins<T>(s, row, logits, rule, cuts, a.vocab);
        }
    }
    if (tid == 0) a.tokens[r] = token;
}

// Threads a row: enough to hold it, or to keep a CU's loads in flight.
template <typename InT>
void launch_min_p(const MinPArgs &a, int rows, hipStream_t st) {
    if (a.vocab <= 256 * kMinPHeld)
        hipLaunchKernelGGL((min_p_kernel<InT, 256, true>), dim3(rows), dim3(256), 0, st, a);
    else if (a.vocab <= 1024 * kMinPHeld)
        hipLaunchKernelGGL((min_p_kernel<InT, 1024, true>), dim3(rows), dim3(1024), 0, st, a);
    else
        hipLaunchKernelGGL((min_p_kernel<InT, 1024, false>), dim3(rows), dim3(1024), 0, st, a);
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
    if (logits_dtype == NQ_F32) launch_min_p<float>(a, rows, st);
    else launch_min_p<uint16_t>(a, rows, st);
    return NQ_LAUNCH_STATUS();
}

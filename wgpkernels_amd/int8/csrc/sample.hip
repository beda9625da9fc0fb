// A token of every row of logits by given random numbers, with temperature, top-k, top-p and min-p, on gfx950. No reference counterpart.
//
// A token's weight is exp((logit - largest) / temperature) in FP64, held as a whole number of units: sums of weights are then the same in whatever
// order they are taken, so a row may be spread over workgroups and added up by atomics. A unit is 2^-44 of the heaviest weight in vocabularies of up
// to 2^18 tokens, whose sums then fit 62 bits; above, a row's own (row_scale). Each weight is off by half a unit, all of a row's together by at most
// 2^-27 of their sum (2^18 2^-45; above less than 2^-28): the token drawn is the 64-bit definition's wherever the draw, a number of 24 bits, is further from
// a border between two tokens, or top-p's from one between two keys. Tokens stand in the order of (logit, lowest index first), a 64-bit key: top-k and top-p
// each keep the keys down to a last one, `cut`.
//
// Four launches, a row over up to 64 workgroups in the first three: the largest logit; a histogram over (largest - logit) / temperature (of counts
// for top-k, of weights for top-p); the keys of the histogram's bins in which the cuts lie, and the weights of what certainly stays; then a
// workgroup a row finds the cut among those keys, and the token whose running weight, in vocabulary order, passes draw * (weight kept). A top-k of at most
// SMALL_K lists all of its keys: then no weight is taken of the rest of the row. Vocabularies above 2^18 take a launch more, for their units.
#include "wq8_common.h"
#include "wq8_abi.h"

namespace wq8 {

constexpr int SAMPLE_BINS = 1024, SAMPLE_SPLITS = 64, SAMPLE_PARTS = 256, SAMPLE_LIST = 2048, SAMPLE_PIECE = 2048, SHORT_LIST = 256;
// Keys listed in memory, all of sample over 8 rows of 262144 BF16, top-p 0.95 at temperature 1.5: 69 us with 16384 of them or 131072, 739 with 2048 (the row is
// read again); 64 flat rows of 131072 FP32, top-k 30000: 111 and 550 (2048); where 16384 are too few too, 4 flatter rows: 571, and 963 with 131072, which one
// workgroup goes through in memory.
constexpr int MOST_LISTED_KEYS = 16384;
// A small top-k takes no weight of what it leaves out but orders all of its keys in one workgroup. All of sample, us, (small, as a large one) for top-k 50,
// 200, 512, 1000 and top-p 0.9: 64 rows of 131072 BF16 30, 55; 34, 56; 46, 57; 58, 60. 32 rows: 27, 41; 31, 42; 41, 43; 49, 45. One of FP32: 21, 27; 25, 27; 34, 28;
// 41, 29: the border is that of many rows, few would have it at 256.
constexpr int SMALL_K = 1024;
// The last bin begins at 31.97: weights below 2^-46, less than half of any unit. With units of a row's own, which are 2^-52 at least, at 37.9: below 2^-54.
constexpr float BINS_PER_UNIT = 32.0f, LARGE_BINS_PER_UNIT = 27.0f;
constexpr int UNIT_BITS = 44, MOST_UNIT_BITS = 52, UNIT_VOCABULARY_BITS = 18;  // 2^52: what FP64's sum with 2^52 holds

struct SampleRow {  // a row's workspace
    uint64_t largest[SAMPLE_SPLITS];
    uint64_t kept[SAMPLE_PARTS];  // the weight kept of each part
    uint64_t mass[SAMPLE_BINS];
    uint32_t count[SAMPLE_BINS];
    uint64_t weighed;  // of large vocabularies: the row's weights in parts of 2^-20, each rounded up
    uint32_t listed, unused;
};

struct SampleArgs {
    const void* logits;
    int64_t ld;
    const float* draws;
    const float* temperature;  // per row, or null: the value below
    const int32_t* top_k;
    const float* top_p;
    const float* min_p;
    SampleRow* rows;
    uint64_t* lists;   // `capacity` keys a row
    int64_t* tokens;
    float temperature0, top_p0, min_p0, bins_per_unit;
    int top_k0;
    int vocabulary, capacity, bits, part, parts, split, splits, shift;  // indices have `bits`; parts of `part` tokens, splits of `split`, a multiple of that; units of 2^-shift, 0: row_scale()
};

// The order of a logit: larger numbers for larger logits, 0 for NaN; both zeros alike.
WQ8_DEVICE uint32_t logit_order(float l) {
    const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.0f);
    return l != l ? 0u : b >> 31 ? ~b : b | 0x80000000u;
}
WQ8_DEVICE float order_logit(uint32_t o) { return __builtin_bit_cast(float, o >> 31 ? o & 0x7fffffffu : ~o); }
// A token's key: its logit's order without the bits that 16-bit logits do not have (all 0, or all 1 below zero), then its index upside down.
template <int DT> struct Key {
    static constexpr int SPARE = DT == DT_BF16 ? 16 : DT == DT_F16 ? 13 : 0;
    int bits;  // of an index
    WQ8_DEVICE uint64_t of(float l, int index) const { return uint64_t(logit_order(l) >> SPARE) << bits | uint32_t((1 << bits) - 1 - index); }
    WQ8_DEVICE int index(uint64_t key) const { return (1 << bits) - 1 - int(uint32_t(key) & ((1u << bits) - 1)); }
    WQ8_DEVICE float logit(uint64_t key) const {
        const uint32_t o = uint32_t(key >> bits) << SPARE;
        return order_logit(o >> 31 ? o : o | ((1u << SPARE) - 1));
    }
};

// 2^t for t <= 0, 0 below -72 (and for NaN): t = n + f, |f| <= 1/2, 2^f by the series of exp(f ln 2) up to its 12th power, whose rest is below 2^-51
// of it (2.4e-16 at f = -1/2). The sum with 1.5 2^52 holds n in its low bits, which are added to the exponent of 2^f.
WQ8_DEVICE double power_of_2(double t) {
    const double shifted = t + 0x1.8p52, f = t - (shifted - 0x1.8p52);
    // ln(2)^i / i!, i = 12 .. 0
    constexpr double LN2 = 0x1.62e42fefa39efp-1;
    constexpr double POWER[13] = {1.0, LN2, LN2 * LN2, LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2 * LN2 * LN2,
                                  LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2,
                                  LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2,
                                  LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2, LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2 * LN2};
    constexpr double FACTORIAL[13] = {1, 1, 2, 6, 24, 120, 720, 5040, 40320, 362880, 3628800, 39916800, 479001600};
    double e = POWER[12] / FACTORIAL[12];
#pragma unroll
    for (int i = 11; i >= 0; --i) e = __builtin_fma(e, f, POWER[i] / FACTORIAL[i]);
    const uint64_t bits = __builtin_bit_cast(uint64_t, e);
    const uint32_t high = uint32_t(bits >> 32) + (uint32_t(__builtin_bit_cast(uint64_t, shifted)) << 20);
    const double power = __builtin_bit_cast(double, uint64_t(high) << 32 | uint32_t(bits));
    return t > -72.0 ? power : 0.0;
}

// What a row is sampled by.
struct Row {
    float top;         // its largest logit
    int first;         // the first token that has it
    double inverse;    // of the temperature, times log2(e)
    float half;        // 1/2 where distances from the largest logit may pass FP32, else 1
    float half_top, bins;  // half * top; bins a unit of half * logit
    double scale, min_p;
    float top_p;
    int top_k;
    bool greedy, nothing, infinite, by_p, by_k, small_k;

    WQ8_DEVICE double finite_weight(float l) const { return power_of_2((double(l) - double(top)) * inverse); }  // of a row whose largest logit is finite
    WQ8_DEVICE double weight(float l) const {
        return infinite ? l == top ? 1.0 : 0.0 : finite_weight(l);
    }
    // the nearest whole number of w * scale <= 2^52, from the low bits of its sum with 2^52
    WQ8_DEVICE uint64_t units(double w) const { return __builtin_bit_cast(uint64_t, __builtin_fma(w, scale, 0x1p52)) - 0x4330000000000000ull; }
    WQ8_DEVICE int bin(float l) const {
        if (l == top) return 0;
        const float b = __builtin_fmaf(-half, l, half_top) * bins;
        return b < float(SAMPLE_BINS - 1) ? int(b) : SAMPLE_BINS - 1;
    }
};

WQ8_DEVICE uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
// The sum over the wave
WQ8_DEVICE uint64_t sum64(uint64_t v) {
    return over_wave(v, [](uint64_t a, uint64_t b) { return a + b; });
}

// The largest of the wave's values
WQ8_DEVICE uint64_t wave_most(uint64_t v) {
    return over_wave(v, [](uint64_t a, uint64_t b) { return max64(a, b); });
}

// Units a weight of 1 of a row over a large vocabulary: as many as keep the row's sum below 2^62, the weights' rounding aside (an upper bound of the sum
// is known), and 2^52 at most. All of a row's weights together are then off by less than 2^24 2^-53 of the heaviest, or by 2^23 units of less than 2^-60 of
// their sum (sum < 2^(c - 20) < 2 (sum + 25) and sum > 2^8 there, a unit is 2^(c - 82)).
WQ8_DEVICE double row_scale(uint64_t weighed) {
    const int c = 64 - __builtin_clzll((weighed - 1) | 1);  // weighed <= 2^c
    const int shift = min(MOST_UNIT_BITS, 82 - c);
    return double(uint64_t(1) << shift);
}

WQ8_DEVICE Row read_row(const SampleArgs& p, const SampleRow& state, int row) {
    Row r;
    const int lane = threadIdx.x & 63;
    const uint64_t best = wave_most(lane < p.splits ? state.largest[lane] : 0);  // order, and the index upside down
    r.first = int(0xffffffffu - uint32_t(best));
    r.top = order_logit(uint32_t(best >> 32));
    r.infinite = r.top == __builtin_inff();
    const float t = p.temperature ? p.temperature[row] : p.temperature0;
    r.greedy = !(t > 0.0f);
    r.nothing = uint32_t(best >> 32) <= logit_order(-__builtin_inff());
    r.inverse = 0x1.71547652b82fep+0 / double(t);
    r.half = r.top >= 0x1p103f ? 0.5f : 1.0f;  // (2^103 above the lowest FP32: half a step past the largest)
    r.half_top = r.half * r.top;
    r.bins = fminf(float(double(p.bins_per_unit / r.half) / double(t)), 0x1.fffffep127f);  // (an infinity would part equal logits from others beside them)
    r.scale = p.shift ? double(uint64_t(1) << p.shift) : row_scale(state.weighed);
    r.min_p = fmin(double(p.min_p ? p.min_p[row] : p.min_p0), 1.0);
    r.top_p = p.top_p ? p.top_p[row] : p.top_p0;
    r.top_k = p.top_k ? p.top_k[row] : p.top_k0;
    r.by_p = r.top_p < 1.0f;
    r.by_k = r.top_k > 0 && r.top_k < p.vocabulary;
    r.small_k = r.by_k && r.top_k <= SMALL_K;
    return r;
}

// f(logit, index) for the row's values from begin to end, 8 neighbouring ones a thread at a time, four times that asked for together; after(i) behind
// every 2048, i the first of them. Past the end f has NaN. Rows may begin at any value: the loads of 16 bytes are as unaligned as the row is.
template <int DT, typename F, typename After> WQ8_DEVICE void each_logit(const SampleArgs& p, int row, int begin, int end, const F& f, const After& after) {
    using raw = typename Elem<DT>::raw;
    constexpr int AHEAD = 4;
    const raw* values = static_cast<const raw*>(p.logits) + row * p.ld;
    raw none;
    if constexpr (DT == DT_F32) none = __builtin_nanf("");
    else none = 0x7fff;
    for (int first = begin; first < end; first += AHEAD * SAMPLE_PIECE) {
        raw v[AHEAD][8];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = first + u * SAMPLE_PIECE + 8 * int(threadIdx.x);
            if (i + 8 <= end) __builtin_memcpy(v[u], values + i, sizeof(v[u]));
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) v[u][j] = i + j < end ? values[i + j] : none;
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int i = first + u * SAMPLE_PIECE + 8 * int(threadIdx.x);
            if (first + u * SAMPLE_PIECE >= end) break;
#pragma unroll
            for (int j = 0; j < 8; ++j) f(Elem<DT>::to_f(v[u][j]), i + j);
            after(first + u * SAMPLE_PIECE);
        }
    }
}
template <int DT, typename F> WQ8_DEVICE void each_logit(const SampleArgs& p, int row, int begin, int end, const F& f) {
    each_logit<DT>(p, row, begin, end, f, [](int) {});
}

// ---- 1: the largest logit of every part of a row -----------------------------------------------------------------------------
// HBM and the launch: 64 rows of 131072 BF16 5.8 us (2.9 TB/s), one row of FP32 3.3.
template <int DT> __global__ void __launch_bounds__(256) sample_largest(SampleArgs p) {
    __shared__ uint64_t best4[4];
    const int row = blockIdx.x / p.splits, s = blockIdx.x % p.splits;
    SampleRow& state = p.rows[row];
    for (int b = s * 256 + threadIdx.x; b < SAMPLE_BINS; b += 256 * p.splits) state.mass[b] = 0, state.count[b] = 0;
    if (!s && !threadIdx.x) state.listed = 0, state.weighed = 0;
    uint32_t most = 0;
    int at = 0;
    each_logit<DT>(p, row, s * p.split, min(p.vocabulary, (s + 1) * p.split), [&](float l, int i) {
        const uint32_t o = logit_order(l);
        if (o > most) most = o, at = i;  // (a thread's indices rise: the first of equal ones stays)
    });
    uint64_t best = uint64_t(most) << 32 | (0xffffffffu - uint32_t(at));
    best = wave_most(best);
    if (!(threadIdx.x & 63)) best4[threadIdx.x >> 6] = best;
    __syncthreads();
    if (!threadIdx.x) state.largest[s] = max64(max64(best4[0], best4[1]), max64(best4[2], best4[3]));
}

// ---- of large vocabularies: an upper bound of a row's weights ---------------------------------------------------------------------
// Bound by the exponentials: 16 rows of 1000000 BF16 21 us, one of FP32 9.5.
template <int DT> __global__ void __launch_bounds__(256) sample_weigh(SampleArgs p) {
    const int row = blockIdx.x / p.splits, s = blockIdx.x % p.splits;
    SampleRow& state = p.rows[row];
    const Row r = read_row(p, state, row);  // (its scale is not known yet)
    if (r.greedy || r.nothing) return;
    const int begin = s * p.split, end = min(p.vocabulary, begin + p.split);
    uint64_t sum = 0;
    // (rounded, and one more: also for what weighs nothing, fewer than 2^25 of those)
    auto add = [&](double w) { sum += __builtin_bit_cast(uint64_t, __builtin_fma(w, 0x1p20, 0x1p52 + 1.0)) - 0x4330000000000000ull; };
    if (r.infinite) each_logit<DT>(p, row, begin, end, [&](float l, int) { add(l == r.top ? 1.0 : 0.0); });
    else each_logit<DT>(p, row, begin, end, [&](float l, int) { add(r.finite_weight(l)); });
    sum = sum64(sum);
    if (!(threadIdx.x & 63)) atomicAdd(reinterpret_cast<unsigned long long*>(&state.weighed), (unsigned long long)sum);
}

// ---- 2: counts and weights over (largest - logit) / temperature ------------------------------------------------------------------
// Bound by the additions in LDS and the exponentials: the same 64 rows, of options of their own, 11 us; one row 4.8.
template <int DT> __global__ void __launch_bounds__(256) sample_bins(SampleArgs p) {
    __shared__ unsigned long long mass[SAMPLE_BINS];
    __shared__ uint32_t count[SAMPLE_BINS];
    const int row = blockIdx.x / p.splits, s = blockIdx.x % p.splits;
    SampleRow& state = p.rows[row];
    const Row r = read_row(p, state, row);
    if (r.greedy || r.nothing || !(r.by_k || r.by_p)) return;
    for (int b = threadIdx.x; b < SAMPLE_BINS; b += 256) mass[b] = 0, count[b] = 0;
    __syncthreads();
    const int begin = s * p.split, end = min(p.vocabulary, begin + p.split);
    // (the last bin, NaN's too, weighs nothing and is not counted)
    if (r.small_k)
        each_logit<DT>(p, row, begin, end, [&](float l, int) {
            const int b = r.bin(l);
            if (b < SAMPLE_BINS - 1) atomicAdd(&count[b], 1u);
        });
    else
        each_logit<DT>(p, row, begin, end, [&](float l, int) {
            const int b = r.bin(l);
            const uint64_t units = r.units(r.infinite ? 1.0 : r.finite_weight(l));
            if (b < SAMPLE_BINS - 1) {
                if (r.by_k) atomicAdd(&count[b], 1u);
                atomicAdd(&mass[b], (unsigned long long)units);
            }
        });
    __syncthreads();
    for (int b = threadIdx.x; b < SAMPLE_BINS; b += 256) {
        if (count[b]) atomicAdd(&state.count[b], count[b]);
        if (mass[b]) atomicAdd(reinterpret_cast<unsigned long long*>(&state.mass[b]), mass[b]);
    }
}

// ---- the bins in which a row's cuts lie --------------------------------------------------------------------------------------
// ceil(f * total) and floor(f * total) for 0 <= f < 1, exactly
WQ8_DEVICE uint64_t share_of(float f, uint64_t total, bool up) {
    const uint32_t b = __builtin_bit_cast(uint32_t, f);
    const uint32_t exponent = b >> 23 & 255;
    const uint64_t mantissa = exponent ? (b & 0x7fffff) | 0x800000 : b & 0x7fffff;
    const int shift = 150 - int(exponent ? exponent : 1);  // f = mantissa / 2^shift, shift >= 24
    const uint64_t high = __umul64hi(mantissa, total), low = mantissa * total;
    if (shift >= 128) return up && (high | low) ? 1 : 0;
    const uint64_t whole = shift >= 64 ? high >> (shift - 64) : shift ? high << (64 - shift) | low >> shift : low;
    const bool rest = shift >= 64 ? (low | (shift > 64 ? high << (128 - shift) : 0)) != 0 : (low << (64 - shift)) != 0;
    return whole + (up && rest ? 1 : 0);
}
// The weight that top-p wants: a key stays while the weight before it is less. At least 1, so that the first one stays.
WQ8_DEVICE uint64_t wanted_mass(float top_p, uint64_t total) {
    const uint64_t m = top_p > 0.0f ? share_of(top_p, total, true) : 0;
    return m ? m : 1;
}

struct Cut {
    int k_bin;                      // the bin of top-k's last key, or SAMPLE_BINS: every weight is among the k
    uint32_t k_left;                // how many of that bin's keys stay
    uint64_t k_before;              // the weight before it
    int low, high;                  // the bins of top-p's last key (low > high: no top-p)
    uint64_t low_before;            // the weight before them
    int certain;                    // bins below it stay whole (0 for a small k, whose bins are all listed); at most the last one, which weighs nothing
    WQ8_DEVICE bool listed(int bin) const { return bin == k_bin || (bin >= low && bin <= high); }
};

// Exclusive sums over the workgroup's 256 threads, and their total.
template <typename T> WQ8_DEVICE T scan256(T v, T* waves, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const T upto = T(wave_upto(v));
    __syncthreads();
    if (lane == 63) waves[wave] = upto;
    __syncthreads();
    T before = upto - v;
    total = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        if (w < wave) before += waves[w];
        total += waves[w];
    }
    return before;
}

struct CutScratch {
    uint64_t waves64[4];
    uint32_t waves32[4];
    uint64_t k_before, k_mass, low_before;
    uint32_t k_left;
    int k_bin, low, high;
};

WQ8_DEVICE Cut find_cut(const Row& r, const SampleRow& state, CutScratch& sc) {
    constexpr int EACH = SAMPLE_BINS / 256;
    uint64_t mass[EACH], masses = 0, total;
    uint32_t count[EACH], counts = 0, all;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        mass[i] = state.mass[EACH * threadIdx.x + i];
        count[i] = state.count[EACH * threadIdx.x + i];
        masses += mass[i];
        counts += count[i];
    }
    if (!threadIdx.x) sc.k_bin = SAMPLE_BINS, sc.low = 1, sc.high = 0, sc.low_before = 0;
    const uint64_t mass_before = scan256(masses, sc.waves64, total);
    const uint32_t count_before = scan256(counts, sc.waves32, all);
    Cut c;
    if (r.by_k) {
        uint32_t n = count_before;
        uint64_t m = mass_before;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            // (the last bin's weights are 0 and it is not counted: a k that reaches it leaves nothing out)
            if (n < uint32_t(r.top_k) && n + count[i] >= uint32_t(r.top_k)) {
                sc.k_bin = EACH * threadIdx.x + i;
                sc.k_left = r.top_k - n;
                sc.k_before = m;
                sc.k_mass = mass[i];
            }
            n += count[i];
            m += mass[i];
        }
        __syncthreads();
    }
    c.k_bin = sc.k_bin;
    c.k_left = c.k_bin < SAMPLE_BINS ? sc.k_left : ~0u;
    c.k_before = sc.k_before;
    if (r.small_k) {  // all up to the k's bin is listed; where the k reach the last bin, all but that
        c.low = c.certain = 0;
        c.high = min(c.k_bin, SAMPLE_BINS - 2);
        c.low_before = c.k_before = 0;
        c.k_left = r.top_k;
        __syncthreads();
        return c;
    }
    if (r.by_p) {
        // the k's weight is known up to its bin: top-p's last key lies between those of the least and the most that it can be
        const bool some = c.k_bin < SAMPLE_BINS;
        const uint64_t least = wanted_mass(r.top_p, some ? c.k_before : total), most = wanted_mass(r.top_p, some ? c.k_before + sc.k_mass : total);
        uint64_t m = mass_before;
#pragma unroll
        for (int i = 0; i < EACH; ++i) {
            if (m < least && m + mass[i] >= least) {
                sc.low = EACH * threadIdx.x + i;
                sc.low_before = m;
            }
            if (m < most && m + mass[i] >= most) sc.high = EACH * threadIdx.x + i;
            m += mass[i];
        }
        __syncthreads();
    }
    c.low = sc.low;
    c.high = sc.high;
    c.low_before = sc.low_before;
    c.certain = r.by_p ? c.low : min(c.k_bin, SAMPLE_BINS - 1);
    __syncthreads();
    return c;
}

// ---- 3: the keys of those bins, and the weights that certainly stay ------------------------------------------------------------
// Bound by the exponentials (45 instructions a value, most of them FP64): 200 rows of 50001 FP16 17 us, the 64 rows 21; one row 5.7.
template <int DT> __global__ void __launch_bounds__(256) sample_list(SampleArgs p) {
    __shared__ CutScratch scratch;
    __shared__ unsigned long long kept[SAMPLE_PARTS];
    const int row = blockIdx.x / p.splits, s = blockIdx.x % p.splits;
    SampleRow& state = p.rows[row];
    const Row r = read_row(p, state, row);
    if (r.greedy || r.nothing) return;
    const bool cutting = r.by_k || r.by_p;
    Cut c{};
    if (cutting) c = find_cut(r, state, scratch);
    if (c.certain || !cutting)
        for (int i = threadIdx.x; i < SAMPLE_PARTS; i += 256) kept[i] = 0;
    __syncthreads();
    const int begin = s * p.split, end = min(p.vocabulary, begin + p.split);
    auto list = [&](float l, int i) {
        const uint32_t at = atomicAdd(&state.listed, 1u);
        if (at < uint32_t(p.capacity)) p.lists[int64_t(row) * p.capacity + at] = Key<DT>{p.bits}.of(l, i);
    };
    uint64_t sum = 0;
    auto kept_of = [&](double w) { return w >= r.min_p ? r.units(w) : 0; };
    auto after = [&](int i) {
        sum = sum64(sum);
        if (!(threadIdx.x & 63)) atomicAdd(&kept[i / p.part], (unsigned long long)sum);
        sum = 0;
    };
    // a loop for each of what rows need, so that nothing parts the weights of one thread's values (each is a chain of 20 operations)
    if (cutting && !c.certain)
        each_logit<DT>(p, row, begin, end, [&](float l, int i) {
            if (c.listed(r.bin(l)) && l == l) list(l, i);
        });
    else if (cutting)
        each_logit<DT>(
            p, row, begin, end,
            [&](float l, int i) {
                const int b = r.bin(l);
                const uint64_t units = kept_of(r.infinite ? 1.0 : r.finite_weight(l));
                sum += b < c.certain ? units : 0;  // (an infinite row has its infinities in the first bin, all else in the last one, which stays out)
                if (c.listed(b) && l == l) list(l, i);
            },
            after);
    else if (r.infinite)
        each_logit<DT>(p, row, begin, end, [&](float l, int) { sum += l == r.top ? kept_of(1.0) : 0; }, after);
    else
        each_logit<DT>(p, row, begin, end, [&](float l, int) { sum += kept_of(r.finite_weight(l)); }, after);
    __syncthreads();
    const int first = s * (p.split / p.part), last = min(p.parts, first + p.split / p.part);
    for (int i = first + threadIdx.x; i < last; i += 256) state.kept[i] = cutting && !c.certain ? 0 : kept[i];
}

// ---- 4: the cut among the listed keys, and the token ---------------------------------------------------------------------------
// One workgroup a row, a chain of short steps: up to 256 keys (SHORT_LIST) each against all others, 7.8 us a row of top-k 50; more of them digit by digit, 22 the 64 rows.
// 200 keys in 32 rows (all of sample): 29.7 us compared, 33.0 by digits; 100 in one row 24.9 and 27.7.
struct __attribute__((aligned(16))) Listed {
    uint64_t key, units;
};
struct PickScratch {
    CutScratch cut;
    Listed list[SAMPLE_LIST];
    unsigned long long mass[256];
    uint32_t count[256];
    unsigned long long kept[SAMPLE_PARTS];
    unsigned long long lowest, highest, found, need;
    uint32_t in_digit;
    int digit, part;
    uint64_t part_target;
    uint64_t waves64[4];
    uint32_t waves32[4];
};

// The key at which the running count (by_count) or weight of `each`'s keys, from the largest on, reaches `need` (at least 1, at most their sum): digits of 8
// bits from the first in which they differ, counts and weights of each digit's values. 
template <bool BY_COUNT, typename Each> WQ8_DEVICE uint64_t select_key(PickScratch& sc, const Each& each, uint64_t need) {
    const int tid = threadIdx.x;
    if (!tid) sc.lowest = ~0ull, sc.highest = 0;
    __syncthreads();
    uint64_t low = ~uint64_t(0), high = 0;
    each([&](uint64_t key, uint64_t) {
        low = key < low ? key : low;
        high = max64(high, key);
    });
    low = ~wave_most(~low);
    high = wave_most(high);
    if (!(tid & 63) && low <= high) {
        atomicMin(&sc.lowest, (unsigned long long)low);
        atomicMax(&sc.highest, (unsigned long long)high);
    }
    __syncthreads();
    const uint64_t differ = sc.lowest ^ sc.highest;
    uint64_t key = sc.highest;
    int width = differ ? 64 - __builtin_clzll(differ) : 0;  // the bits above are settled
    while (width) {
        const int shift = max(0, width - 8);
        const uint64_t settled = width < 64 ? key >> width : 0;
        sc.mass[tid] = 0;
        sc.count[tid] = 0;
        __syncthreads();
        each([&](uint64_t k, uint64_t units) {
            if ((width < 64 ? k >> width : 0) != settled) return;
            const int d = int(k >> shift) & ((1 << (width - shift)) - 1);
            atomicAdd(&sc.count[d], 1u);
            if (!BY_COUNT) atomicAdd(&sc.mass[d], (unsigned long long)units);
        });
        __syncthreads();
        const int d = 255 - tid;
        const uint32_t n = sc.count[d];
        uint64_t before, here;
        if (BY_COUNT) {
            uint32_t all;
            before = scan256(n, sc.waves32, all);
            here = n;
        } else {
            uint64_t all;
            here = sc.mass[d];
            before = scan256(here, sc.waves64, all);
        }
        if (before < need && before + here >= need) {
            sc.digit = d;
            sc.in_digit = n;
            sc.need = need - before;
        }
        __syncthreads();
        need = sc.need;
        key = (settled << (width - shift) | uint64_t(sc.digit)) << shift;
        if (sc.in_digit == 1 && shift) {  // one key left: find it
            each([&](uint64_t k, uint64_t) {
                if (k >> shift == key >> shift) sc.found = k;
            });
            __syncthreads();
            key = sc.found;
            break;
        }
        __syncthreads();
        width = shift;
    }
    __syncthreads();
    return key;
}

template <int DT> __global__ void __launch_bounds__(256) sample_pick(SampleArgs p) {
    __shared__ PickScratch sc;
    const int row = blockIdx.x, tid = threadIdx.x;
    SampleRow& state = p.rows[row];
    const Row r = read_row(p, state, row);
    if (r.greedy || r.nothing) {
        if (!tid) p.tokens[row] = r.nothing ? -1 : r.first;
        return;
    }
    sc.kept[tid] = tid < p.parts ? state.kept[tid] : 0;
    const float u = p.draws[row];
    // the kept weight that the token's running weight has to pass
    auto drawn = [&](uint64_t total) {
        const uint64_t target = u > 0.0f ? u < 1.0f ? share_of(u, total, false) : total - 1 : 0;
        return target < total ? target : total - 1;
    };
    const Key<DT> keys{p.bits};
    auto sum_of = [&](uint64_t v) {  // over the workgroup
        v = sum64(v);
        __syncthreads();
        if (!(tid & 63)) sc.waves64[tid >> 6] = v;
        __syncthreads();
        return sc.waves64[0] + sc.waves64[1] + sc.waves64[2] + sc.waves64[3];
    };
    uint64_t cut = 0;  // keys from it on stay
    if (r.by_k || r.by_p) {
        const Cut c = find_cut(r, state, sc.cut);
        const uint32_t listed = state.listed;
        const bool whole = listed <= uint32_t(SAMPLE_LIST);  // they fit into LDS
        const uint64_t* keys_listed = p.lists + int64_t(row) * p.capacity;
        if (whole)
            for (int i = tid; i < int(listed); i += 256) {
                const uint64_t key = keys_listed[i];
                sc.list[i] = {key, r.units(r.weight(keys.logit(key)))};
            }
        uint64_t total = 0;  // of what top-p is taken
        if (r.by_p && !r.by_k || r.by_p && !r.small_k && c.k_bin == SAMPLE_BINS) {
            uint64_t mass = 0;
            for (int b = tid; b < SAMPLE_BINS; b += 256) mass += state.mass[b];
            total = sum_of(mass);
        }
        const int from = c.certain, to = r.by_p || r.small_k ? c.high : c.k_bin;  // the bins of the keys that may stay and are not certain to
        if (c.k_bin == SAMPLE_BINS && !r.by_p && !r.small_k) {
            // a k that leaves nothing out
        } else if (whole && listed <= uint32_t(SHORT_LIST) && (r.small_k || c.k_bin == SAMPLE_BINS || !r.by_p)) {
            // few keys, of one run of bins: each against all others, for its place and the weight before it
            const int n = int(listed), padded = (n + 7) / 8 * 8;
            if (tid >= n && tid < padded) sc.list[tid] = {0, 0};
            __syncthreads();
            const Listed mine = tid < n ? sc.list[tid] : Listed{0, 0};
            uint32_t place = 0;
            uint64_t before = 0;
            for (int j = 0; j < padded; j += 8)
#pragma unroll
                for (int u = 0; u < 8; ++u) {
                    const Listed other = sc.list[j + u];
                    const bool ahead = other.key > mine.key;
                    place += ahead;
                    before += ahead ? other.units : 0;
                }
            bool stays = tid < n && (!r.by_k || place < c.k_left);
            if (r.by_p) {
                if (r.small_k) total = sum_of(stays ? mine.units : 0);
                stays = stays && c.low_before + before < wanted_mass(r.top_p, total);
            }
            uint64_t last = stays ? ~mine.key : 0;  // the largest of these is the smallest key
            last = wave_most(last);
            __syncthreads();
            if (!(tid & 63)) sc.waves64[tid >> 6] = last;
            __syncthreads();
            cut = ~max64(max64(sc.waves64[0], sc.waves64[1]), max64(sc.waves64[2], sc.waves64[3]));
            __syncthreads();
            if (stays && r.weight(keys.logit(mine.key)) >= r.min_p) atomicAdd(&sc.kept[keys.index(mine.key) / p.part], (unsigned long long)mine.units);
        } else {
            __syncthreads();
            // the listed keys of some of the bins, from LDS or from memory; where they are too many for the list (logits that are alike), the row is read
            // again instead
            auto each = [&](int low, int high, const auto& f) {
                if (whole) {
                    for (int i = tid; i < int(listed); i += 256) {
                        const Listed one = sc.list[i];
                        const int b = r.bin(keys.logit(one.key));
                        if (b >= low && b <= high) f(one.key, one.units);
                    }
                } else if (listed <= uint32_t(p.capacity)) {
                    for (int i = tid; i < int(listed); i += 256) {
                        const uint64_t key = keys_listed[i];
                        const float l = keys.logit(key);
                        const int b = r.bin(l);
                        if (b >= low && b <= high) f(key, r.units(r.weight(l)));
                    }
                } else {
                    each_logit<DT>(p, row, 0, p.vocabulary, [&](float l, int i) {
                        const int b = r.bin(l);
                        if (l == l && b >= low && b <= high) f(keys.of(l, i), r.units(r.weight(l)));
                    });
                }
            };
            if (c.k_bin < SAMPLE_BINS) {
                const int low = r.small_k ? 0 : c.k_bin;
                cut = select_key<true>(sc, [&](const auto& f) { each(low, c.k_bin, f); }, c.k_left);
                uint64_t upto = 0;
                each(low, c.k_bin, [&](uint64_t key, uint64_t units) { upto += key >= cut ? units : 0; });
                total = c.k_before + sum_of(upto);
            } else if (r.small_k) {  // fewer than k weigh anything: all of them stay
                uint64_t all = 0;
                each(c.low, c.high, [&](uint64_t, uint64_t units) { all += units; });
                total = sum_of(all);
            }
            if (r.by_p) cut = select_key<false>(sc, [&](const auto& f) { each(c.low, c.high, f); }, wanted_mass(r.top_p, total) - c.low_before);
            each(from, to, [&](uint64_t key, uint64_t units) {
                if (key >= cut && r.weight(keys.logit(key)) >= r.min_p) atomicAdd(&sc.kept[keys.index(key) / p.part], (unsigned long long)units);
            });
        }
    }
    __syncthreads();
    // the part of the row in which the running weight passes the drawn one
    uint64_t total;
    const uint64_t here = sc.kept[tid], upto = scan256(here, sc.waves64, total), passes = drawn(total);
    if (upto <= passes && passes < upto + here) {
        sc.part = tid;
        sc.part_target = passes - upto;
    }
    __syncthreads();
    uint64_t target = sc.part_target;
    const int s = sc.part;
    // in it, 8 neighbouring tokens a thread at a time
    using raw = typename Elem<DT>::raw;
    const raw* values = static_cast<const raw*>(p.logits) + row * p.ld;
    const int end = min(p.vocabulary, (s + 1) * p.part);
    for (int begin = s * p.part; begin < end; begin += 8 * 256) {
        uint64_t units[8], mine = 0, piece;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = begin + 8 * tid + j;
            const float l = Elem<DT>::to_f(values[min(i, end - 1)]);
            const double w = i < end && l == l && keys.of(l, i) >= cut ? r.weight(l) : 0.0;
            units[j] = w >= r.min_p ? r.units(w) : 0;
            mine += units[j];
        }
        uint64_t before = scan256(mine, sc.waves64, piece);
        if (before <= target && target < before + mine) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if (before <= target && target < before + units[j]) p.tokens[row] = begin + 8 * tid + j;
                before += units[j];
            }
        }
        if (target < piece) break;
        target -= piece;
    }
}

}  // namespace wq8

using namespace wq8;

// Keys listed a row: as many as LDS holds, and more of few rows (1 GiB of lists in all, 2 GiB for 2^17 rows), but no more than there are tokens
static int list_capacity(int rows, int vocabulary) {
    const int64_t fit = (int64_t(1) << 27) / (rows > 0 ? rows : 1);
    const int most = int(fit < SAMPLE_LIST ? SAMPLE_LIST : fit > MOST_LISTED_KEYS ? MOST_LISTED_KEYS : fit);
    return most < vocabulary ? most : vocabulary;
}

template <int DT> static int launch_sample(const SampleArgs& p, int rows, hipStream_t stream) {
    sample_largest<DT><<<rows * p.splits, 256, 0, stream>>>(p);
    if (const int rc = int(hipGetLastError())) return rc;
    if (!p.shift) sample_weigh<DT><<<rows * p.splits, 256, 0, stream>>>(p);
    if (const int rc = int(hipGetLastError())) return rc;
    sample_bins<DT><<<rows * p.splits, 256, 0, stream>>>(p);
    if (const int rc = int(hipGetLastError())) return rc;
    sample_list<DT><<<rows * p.splits, 256, 0, stream>>>(p);
    if (const int rc = int(hipGetLastError())) return rc;
    sample_pick<DT><<<rows, 256, 0, stream>>>(p);
    return int(hipGetLastError());
}

WQ8_API int wq8_sample(const void* logits, int64_t ld, int dtype, const float* draws, const float* temperature, float temperature0, const void* top_k, int top_k0,
                       const float* top_p, float top_p0, const float* min_p, float min_p0, int rows, int vocabulary, int64_t* tokens, void* workspace,
                       hipStream_t stream) {
    if (!rows) return 0;
    if (dtype < 0 || dtype > 2) return -1;
    if (rows < 0 || rows > (1 << 17) || vocabulary < 1 || vocabulary > (1 << 24)) return -2;
    // up to 256 parts of 2048 tokens or a multiple; splits of whole parts, a thousand workgroups or so
    const int pieces = (vocabulary + SAMPLE_PIECE - 1) / SAMPLE_PIECE, part = (pieces + SAMPLE_PARTS - 1) / SAMPLE_PARTS * SAMPLE_PIECE;
    const int parts = (vocabulary + part - 1) / part;
    int splits = (1023 + rows) / rows;
    splits = splits < SAMPLE_SPLITS ? splits : SAMPLE_SPLITS;
    splits = splits < parts ? splits : parts;
    const int split = (parts + splits - 1) / splits * part;
    splits = (vocabulary + split - 1) / split;
    int bits = 0;
    while ((1 << bits) < vocabulary) ++bits;
    const SampleArgs p{logits, ld, draws, temperature, static_cast<const int32_t*>(top_k), top_p, min_p, static_cast<SampleRow*>(workspace),
                       reinterpret_cast<uint64_t*>(static_cast<SampleRow*>(workspace) + rows), tokens,
                       temperature0, top_p0, min_p0, bits <= UNIT_VOCABULARY_BITS ? BINS_PER_UNIT : LARGE_BINS_PER_UNIT, top_k0, vocabulary,
                       list_capacity(rows, vocabulary),
                       bits, part, parts, split, splits, bits <= UNIT_VOCABULARY_BITS ? UNIT_BITS : 0};
    if (dtype == DT_F16) return launch_sample<DT_F16>(p, rows, stream);
    if (dtype == DT_BF16) return launch_sample<DT_BF16>(p, rows, stream);
    return launch_sample<DT_F32>(p, rows, stream);
}

WQ8_API void wq8_sample_workspace(int rows, int64_t* sizes) {
    sizes[0] = int64_t(rows) * (int64_t(sizeof(SampleRow)) + int64_t(list_capacity(rows, 1 << 24)) * 8);
    sizes[1] = 0;
}

WQ8_API void wq8_sample_workspace_for(int rows, int vocabulary, int64_t* sizes) {
    sizes[1] = rows > 0 && vocabulary > 0 ? int64_t(rows) * int64_t(sizeof(SampleRow)) : 0;
    sizes[0] = sizes[1] ? sizes[1] + int64_t(rows) * list_capacity(rows, vocabulary) * 8 : 0;
}

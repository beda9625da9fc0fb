// A mixture-of-experts layer of INT8 weights for a few tokens on gfx950: the router (its product in 64 bits, and its choice) and the chosen
// experts' gated feed-forward blocks,
//     y[t] = residual[t] + rscale * sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),   e = ids[t, j],
// a chosen expert's weights read from memory once for up to 64 of its tokens (once for 8 choices in the form for the fewest tokens). No reference
// counterpart. Times below are with the weights in the Infinity Cache where they fit it; cold ones are of copies of the weights taken in turn.
#include "gemm_common.h"
#include "wq8_abi.h"

namespace wq8 {

typedef double v4d __attribute__((ext_vector_type(4)));

// ---- the router ---------------------------------------------------------------------------------------------------------
struct RouteArgs {
    const void* x;
    const void* router;
    const float* bias;
    double* logits;
    int32_t* ids;
    float* weights;
    int64_t ldx;
    int tokens, experts, k, top, score, normalise, parts, part;  // parts of `part` values of k
    float factor;
};

// 8 consecutive values as they are in memory, one of them as FP64; zeros when !valid.
template <int DT> struct Eight {
    u32x4 held[DT == DT_F32 ? 2 : 1];
    WQ8_DEVICE void load(const void* base, int64_t at, bool valid) {
        const u32x4* from = reinterpret_cast<const u32x4*>(static_cast<const typename Elem<DT>::raw*>(base) + at);
#pragma unroll
        for (int i = 0; i < (DT == DT_F32 ? 2 : 1); ++i) held[i] = valid ? from[i] : u32x4{0, 0, 0, 0};
    }
    WQ8_DEVICE double value(int j) const {
        const uint32_t word = DT == DT_F32 ? held[j >> 2][j & 3] : held[0][j >> 1];  // (a bit cast takes a vector's element only by way of a number)
        if constexpr (DT == DT_F32) return double(__builtin_bit_cast(float, word));
        else return double(Elem<DT>::to_f(uint16_t(word >> (16 * (j & 1)))));
    }
};

// Logits of 16 tokens x 16 experts over a part of K, in FP64 (the choice between near experts is a whole number: in FP32 one in some 10^4 tokens
// would go by the order of the sum). 8 waves take 32 values of every row in turn; their sums are added in order, the parts by route_choose. Matrix
// instructions of FP64 set the time (64 cycles for 4 values): parts short enough to fill the CUs (64 experts over 2048
// values 3.1 us, 7.3 with whole rows a workgroup).
constexpr int ROUTE_WAVES = 8, ROUTE_STEP = 32 * ROUTE_WAVES;
template <int XT, int RT>
__global__ void __launch_bounds__(64 * ROUTE_WAVES) route_logits(RouteArgs p) {
    __shared__ double sums[ROUTE_WAVES][4][64];
    // (the wave's number in a scalar: matrix instructions do not heed the lanes' mask, so no branch around them may go by one)
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int expert = blockIdx.x * 16 + (lane & 15), token = blockIdx.y * 16 + (lane & 15), end = min(p.k, int(blockIdx.z + 1) * p.part);
    const bool has_expert = expert < p.experts, has_token = token < p.tokens;
    v4d acc = {0, 0, 0, 0};
    for (int begin = blockIdx.z * p.part + 32 * wave; begin < end; begin += ROUTE_STEP) {
        const int k = begin + 8 * (lane >> 4);
        Eight<XT> a;
        Eight<RT> b;
        a.load(p.x, token * p.ldx + k, has_token && k < p.k);
        b.load(p.router, int64_t(expert) * p.k + k, has_expert && k < p.k);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a.value(j), b.value(j), acc, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    if (threadIdx.x >= 256) return;
    const int i = threadIdx.x >> 6;
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < ROUTE_WAVES; ++w) total += sums[w][i][lane];
    // element i of lane l is token 4 i + l / 16, expert l % 16
    const int t = blockIdx.y * 16 + 4 * i + (lane >> 4);
    if (has_expert && t < p.tokens) p.logits[(int64_t(blockIdx.z) * p.tokens + t) * p.experts + expert] = total;
}

// A double's order as an unsigned number above 1; 1 for NaN.
WQ8_DEVICE uint64_t order_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v != v ? 1 : b >> 63 ? ~b : b | (uint64_t(1) << 63);
}
WQ8_DEVICE uint64_t wave_max64(uint64_t v) {
    return over_wave(v, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
}
WQ8_DEVICE double wave_sum64(double v) {
    return __builtin_bit_cast(double, over_wave(__builtin_bit_cast(uint64_t, v), [](uint64_t a, uint64_t b) {
        return __builtin_bit_cast(uint64_t, __builtin_bit_cast(double, a) + __builtin_bit_cast(double, b));
    }));
}
WQ8_DEVICE double lane_value(double v, int lane) {  // lane the same for all
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, uint64_t(uint32_t(__builtin_amdgcn_readlane(int(b >> 32), lane))) << 32 |
                                          uint32_t(__builtin_amdgcn_readlane(int(uint32_t(b)), lane)));
}

// Scores, choice and weights of a token a wave; a lane holds NE neighbouring experts. Bound by its chain of operations: 8 of 64 experts 3.7 us (6 with
// exchanges through LDS).
template <int NE>
__global__ void __launch_bounds__(256) route_choose(RouteArgs p) {
    const int lane = threadIdx.x & 63, token = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= p.tokens) return;
    const double* logits = p.logits + int64_t(token) * p.experts;
    double score[NE];
    uint64_t wanted[NE];
    double top = -__builtin_inf();
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane * NE + i;
        score[i] = e < p.experts ? logits[e] : -__builtin_inf();
    }
    constexpr int TOGETHER = NE <= 4 ? 8 : 2;  // parts whose loads are asked for at once
    for (int first = 1; first < p.parts; first += TOGETHER) {
        double more[TOGETHER][NE];
#pragma unroll
        for (int s = 0; s < TOGETHER; ++s)
#pragma unroll
            for (int i = 0; i < NE; ++i)
                more[s][i] = logits[int64_t(min(first + s, p.parts - 1)) * p.tokens * p.experts + min(lane * NE + i, p.experts - 1)];
#pragma unroll
        for (int s = 0; s < TOGETHER; ++s)
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (first + s < p.parts) score[i] += more[s][i];
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) top = __builtin_fmax(top, score[i]);
    if (p.score == 0) {
        top = __builtin_bit_cast(double, over_wave(__builtin_bit_cast(uint64_t, top), [](uint64_t a, uint64_t b) {
            return __builtin_bit_cast(uint64_t, __builtin_fmax(__builtin_bit_cast(double, a), __builtin_bit_cast(double, b)));
        }));
        double sum = 0.0;
#pragma unroll
        for (int i = 0; i < NE; ++i) {
            score[i] = lane * NE + i < p.experts ? exp(score[i] - top) : 0.0;
            sum += score[i];
        }
        sum = wave_sum64(sum);
#pragma unroll
        for (int i = 0; i < NE; ++i) score[i] /= sum;
    } else {
#pragma unroll
        for (int i = 0; i < NE; ++i) score[i] = 1.0 / (1.0 + exp(-score[i]));
    }
#pragma unroll
    for (int i = 0; i < NE; ++i) {
        const int e = lane * NE + i;
        wanted[i] = e < p.experts ? order_of(p.bias ? score[i] + double(p.bias[e]) : score[i]) : 0;  // 0: no expert, or chosen already
    }
    double mine = 0.0, total = 0.0;
    int chosen = 0;
    for (int j = 0; j < p.top; ++j) {
        uint64_t best = 0;
#pragma unroll
        for (int i = 0; i < NE; ++i) best = wanted[i] > best ? wanted[i] : best;
        const uint64_t most = wave_max64(best);
        const int from = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(best == most)));  // neighbouring experts a lane: the lowest lane has the lowest index
        double value = 0.0;
        int e = 0;
        if (lane == from) {
            bool taken = false;
#pragma unroll
            for (int i = 0; i < NE; ++i)
                if (!taken && wanted[i] == most) {
                    taken = true;
                    value = score[i];
                    e = lane * NE + i;
                    wanted[i] = 0;
                }
        }
        value = lane_value(value, from);
        e = __builtin_amdgcn_readlane(e, from);
        total += value;
        if (lane == j) {
            mine = value;
            chosen = e;
        }
    }
    if (lane < p.top) {
        const int64_t at = int64_t(token) * p.top + lane;
        p.ids[at] = chosen;
        p.weights[at] = float((p.normalise ? mine / total : mine) * double(p.factor));
    }
}

// ---- the experts ----------------------------------------------------------------------------------------------------------
struct ExpertsArgs {
    const void* x;
    const int32_t* ids;     // (tokens, top); those outside the experts are left out
    const float* weights;
    const int8_t* gate_up;  // (experts, 2 hidden, k)
    const float* gate_up_scale;
    const int8_t* down;     // (experts, k, hidden)
    const float* down_scale;
    uint16_t* h;            // (2, tokens top, hidden): the hidden values as a BF16 and the rest as another
    float* part;            // (tokens top, k)
    const void* residual;
    const void* rscale;
    void* out;
    int64_t ldx, ldr, ldo;
    int tokens, top, experts, k, hidden;
};
constexpr int MOST_PAIRS = 4096, MOST_ONE = 64;  // choices of a call; of a token whose second product is experts_down_one

template <int DT> struct ExpertOp;
template <> struct ExpertOp<DT_BF16> {
    using frag = bf16x8;
    static WQ8_DEVICE v4f run(frag a, frag b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static WQ8_DEVICE __bf16 cvt(float f) { return static_cast<__bf16>(f); }
};
template <> struct ExpertOp<DT_F16> {
    using frag = f16x8;
    static WQ8_DEVICE v4f run(frag a, frag b, v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static WQ8_DEVICE _Float16 cvt(float f) { return static_cast<_Float16>(f); }
};
// 8 codes, exact in BF16 and FP16
template <int DT> WQ8_DEVICE typename ExpertOp<DT>::frag codes8(uint32_t lo, uint32_t hi) {
    typename ExpertOp<DT>::frag f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f[j] = ExpertOp<DT>::cvt(float(int8_t(lo >> (8 * j))));
        f[j + 4] = ExpertOp<DT>::cvt(float(int8_t(hi >> (8 * j))));
    }
    return f;
}

// Which of the choices a workgroup row `slot` serves: those of its expert, in order. Fewer choices than experts: a slot is a choice, and the first
// one of an expert serves all of them; else it is an expert.
WQ8_DEVICE bool slot_is_choice(const ExpertsArgs& p) { return p.tokens * p.top <= p.experts; }
WQ8_DEVICE int slot_expert(const ExpertsArgs& p, int slot) { return slot_is_choice(p) ? p.ids[slot] : slot; }
// Their number (0: another slot has them), and those from `first` on, up to MOST_LISTED, in LDS; every wave counts, the first one writes. A lane
// looks at 4 neighbouring choices at a time.
constexpr int MOST_LISTED = 64;
WQ8_DEVICE int find_choices(const ExpertsArgs& p, int slot, int expert, int first, uint16_t* list) {
    const int pairs = p.tokens * p.top, lane = threadIdx.x & 63;
    const bool by_choice = slot_is_choice(p);
    const uint64_t lower = (uint64_t(1) << lane) - 1;
    int count = 0;
    for (int base = 0; base < pairs; base += 256) {
        const int at = base + 4 * lane;
        int id[4];
        if (at + 4 <= pairs) __builtin_memcpy(id, p.ids + at, 16);
        else
#pragma unroll
            for (int j = 0; j < 4; ++j) id[j] = at + j < pairs ? p.ids[at + j] : -1;  // (no expert is -1)
        uint64_t mask[4];
        int before = 0, here = 0, earliest = 1 << 30;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mask[j] = __ballot(id[j] == expert);
            before += __popcll(mask[j] & lower);
            here += __popcll(mask[j]);
            if (mask[j]) earliest = min(earliest, 4 * __builtin_ctzll(mask[j]) + j);
        }
        if (!here) continue;
        if (by_choice && !count && base + earliest != slot) return 0;
        if (threadIdx.x < 64) {
            int place = count + before - first;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (id[j] == expert) {
                    if (place >= 0 && place < MOST_LISTED) list[place] = uint16_t(at + j);
                    ++place;
                }
        }
        count += here;
    }
    return count;
}

// Two tiles of 16 weight rows on up to CAP tokens (PLANES rows each). The four waves of a workgroup take slices of SLICE values of the width in
// turn, each through a ring of its own in LDS, filled by copies that pass the registers by: no wave waits for another one until the
// end, where the four sums of every output are added in order. HBM bounds it, and at these sizes the latency of a workgroup's beginning: one token, 8 of 64 experts of
// 2048 x 1024, gate and up 9.9 us for 33.6 MB (3.4 TB/s; cold 11.1). 16-byte chunks are placed by their row so that the 16 lanes that read one chunk of
// 16 rows meet different banks.
constexpr int RING = 19 * 1024;  // a wave's: two workgroups a CU
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;
template <int DT, int SLICE, int CAP, int PLANES, typename Source, typename Done>
WQ8_DEVICE void ring_rows(sgpr4 rw, int row0, int row1, int width, sgpr4 rx, uint32_t plane_bytes, int count, uint8_t* rings, const Source& source,
                          const Done& done) {
    constexpr int W_BYTES = 32 * SLICE, X_BYTES = CAP * PLANES * SLICE * 2, STAGE = W_BYTES + X_BYTES, STAGES = RING / STAGE < 8 ? RING / STAGE : 8;
    constexpr int W_COPIES = W_BYTES / 1024, X_COPIES = X_BYTES / 1024, COPIES = W_COPIES + X_COPIES;
    constexpr int W_CHUNKS = SLICE / 16, X_CHUNKS = SLICE / 8;  // of a row in a stage
    static_assert(STAGES >= 2 && X_BYTES % 1024 == 0 && (STAGES - 1) * COPIES < 64, "a ring of stages of whole copies");
    using frag = typename ExpertOp<DT>::frag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, sub = lane >> 4;
    uint8_t* ring = rings + wave * RING;
    auto w_turn = [](int r) { return SLICE == 128 ? r >> 1 & 7 : r >> 2 & 3; };
    auto x_turn = [](int q) { return SLICE == 128 ? q & 15 : q >> 1 & 7; };
    uint32_t w_from[W_COPIES], x_from[X_COPIES];
    int w_k[W_COPIES], x_k[X_COPIES];
#pragma unroll
    for (int j = 0; j < W_COPIES; ++j) {
        const int r = j * (64 / W_CHUNKS) + lane / W_CHUNKS, chunk = lane % W_CHUNKS ^ w_turn(r);
        w_k[j] = 16 * chunk;
        w_from[j] = uint32_t(r < 16 ? row0 + r : row1 + r - 16) * uint32_t(width) + 16u * chunk;  // rows past the matrix read zeros
    }
#pragma unroll
    for (int j = 0; j < X_COPIES; ++j) {
        const int q = j * (64 / X_CHUNKS) + lane / X_CHUNKS, chunk = lane % X_CHUNKS ^ x_turn(q);
        x_k[j] = 8 * chunk;
        x_from[j] = source(min(q % CAP, count - 1)) + (PLANES > 1 && q >= CAP ? plane_bytes : 0u) + 16u * chunk;
    }
    auto issue = [&](int i, uint8_t* stage) {
        const int k0 = (wave + 4 * i) * SLICE;
#pragma unroll
        for (int j = 0; j < W_COPIES; ++j) bdma16_nt(rw, k0 + w_k[j] < width ? w_from[j] + uint32_t(k0) : OUT_OF_RANGE, stage + 1024 * j);
#pragma unroll
        for (int j = 0; j < X_COPIES; ++j) bdma16(rx, k0 + x_k[j] < width ? x_from[j] + 2u * uint32_t(k0) : OUT_OF_RANGE, stage + W_BYTES + 1024 * j);
    };
    v4f a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
    const int slices = (width + SLICE - 1) / SLICE, mine = (slices - wave + 3) / 4;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i, ring + i * STAGE);
    int at = 0, free = STAGES - 1;
    for (int i = 0; i < mine; ++i) {
        wait_vmcnt<(STAGES - 2) * COPIES>();  // this slice's copies have landed
        wait_lgkm0();                         // and the last slice's reads are done: its stage is free
        asm volatile("" ::: "memory");
        issue(i + STAGES - 1, ring + free * STAGE);  // past the width: zeros (the same count every time)
        const uint8_t* ws = ring + at * STAGE;
        const uint8_t* xs = ws + W_BYTES;
        free = at;
        at = at + 1 == STAGES ? 0 : at + 1;
#pragma unroll
        for (int h = 0; h < SLICE / 64; ++h) {
            const int chunk = (4 * h + sub) ^ w_turn(r16);
            static_assert(SLICE == 64 || SLICE == 128, "turns repeat after 16 rows");
            const u32x4 c0 = *reinterpret_cast<const u32x4*>(ws + r16 * SLICE + 16 * chunk);
            const u32x4 c1 = *reinterpret_cast<const u32x4*>(ws + (16 + r16) * SLICE + 16 * chunk);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const frag f0 = codes8<DT>(c0[2 * e], c0[2 * e + 1]), f1 = codes8<DT>(c1[2 * e], c1[2 * e + 1]);
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    const int t = q * CAP + (r16 & (CAP - 1));
                    const frag x = *reinterpret_cast<const frag*>(xs + t * 2 * SLICE + 16 * ((8 * h + 2 * sub + e) ^ x_turn(t)));
                    a0 = ExpertOp<DT>::run(f0, x, a0);
                    a1 = ExpertOp<DT>::run(f1, x, a1);
                }
            }
        }
    }
    wait_vmcnt<0>();
    __syncthreads();
    v4f* red = reinterpret_cast<v4f*>(rings) + lane;  // of waves 1 to 3, two tiles each
    if (wave) red[(wave - 1) * 128] = a0, red[(wave - 1) * 128 + 64] = a1;
    __syncthreads();
    if (!wave) done(((a0 + red[0]) + red[128]) + red[256], ((a1 + red[64]) + red[192]) + red[320]);
}

// More tokens or tiles: 128 rows a workgroup, two runs of 64 of which each wave has a tile of 16, and the tokens' slices in LDS once for all of them. HBM: 32
// tokens, 8 of 128 experts of 2048 x 768 (78 chosen, up to 11 tokens each), gate and up 47 us for 245 MB (5.2 TB/s; cold 50), down 30 for 123 MB (4.1 TB/s: short rows; cold 31); 25
// tokens on each of 16 experts of 5120 x 1536 58 and 48 (4.3 and 2.6 TB/s: copies of tokens beside the codes').
// done(m, values of both tiles): element i is row 16 wave + 4 (lane / 16) + i of each run, token 16 m + lane % 16.
template <int DT, int SLICE, int MT, int PLANES, typename Source, typename Done>
WQ8_DEVICE void shared_rows(sgpr4 rw, int row0, int row1, int width, sgpr4 rx, uint32_t plane_bytes, int count, uint8_t* ring, const Source& source,
                            const Done& done) {
    constexpr int CAP = 16 * MT, W_BYTES = 128 * SLICE, X_BYTES = CAP * PLANES * SLICE * 2, STAGE = W_BYTES + X_BYTES;
    constexpr int W_CHUNKS = SLICE / 16, X_CHUNKS = SLICE / 8, W_COPIES = W_BYTES / 4096, X_ALL = X_BYTES / 1024, X_COPIES = (X_ALL + 3) / 4;
    constexpr int STAGES = 4 * RING / STAGE < 8 ? 4 * RING / STAGE : 8, COPIES = W_COPIES + X_COPIES;
    static_assert(STAGES >= 3 && (STAGES - 1) * COPIES < 64, "a ring of stages");
    using frag = typename ExpertOp<DT>::frag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, sub = lane >> 4;
    auto w_turn = [](int r) { return SLICE == 128 ? r >> 1 & 7 : r >> 2 & 3; };
    auto x_turn = [](int q) { return SLICE == 128 ? q & 15 : q >> 1 & 7; };
    uint32_t w_from[W_COPIES], x_from[X_COPIES];
    int w_k[W_COPIES], x_k[X_COPIES];
#pragma unroll
    for (int j = 0; j < W_COPIES; ++j) {
        const int r = (wave + 4 * j) * (64 / W_CHUNKS) + lane / W_CHUNKS, chunk = lane % W_CHUNKS ^ w_turn(r);
        w_k[j] = 16 * chunk;
        w_from[j] = uint32_t(r < 64 ? row0 + r : row1 + r - 64) * uint32_t(width) + 16u * chunk;  // rows past the matrix read zeros
    }
#pragma unroll
    for (int j = 0; j < X_COPIES; ++j) {
        const int q = (wave + 4 * j) % X_ALL * (64 / X_CHUNKS) + lane / X_CHUNKS, chunk = lane % X_CHUNKS ^ x_turn(q);  // (of two copies, two waves bring each)
        x_k[j] = 8 * chunk;
        x_from[j] = source(min(q % CAP, count - 1)) + (PLANES > 1 && q >= CAP ? plane_bytes : 0u) + 16u * chunk;
    }
    auto issue = [&](int k0, uint8_t* stage) {
#pragma unroll
        for (int j = 0; j < W_COPIES; ++j)
            bdma16_nt(rw, k0 + w_k[j] < width ? w_from[j] + uint32_t(k0) : OUT_OF_RANGE, stage + 1024 * (wave + 4 * j));
#pragma unroll
        for (int j = 0; j < X_COPIES; ++j)
            bdma16(rx, k0 + x_k[j] < width ? x_from[j] + 2u * uint32_t(k0) : OUT_OF_RANGE, stage + W_BYTES + 1024 * ((wave + 4 * j) % X_ALL));
    };
    v4f a0[MT], a1[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) a0[m] = a1[m] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i * SLICE, ring + i * STAGE);
    int at = 0, free = STAGES - 1;
    const int r = 16 * wave + r16;
    for (int k = 0; k < width; k += SLICE) {
        wait_vmcnt<(STAGES - 2) * COPIES>();  // this wave's copies of the slice have landed
        wait_lgkm0();                         // and its reads of the last one are done
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();         // every wave's
        issue(k + (STAGES - 1) * SLICE, ring + free * STAGE);
        const uint8_t* ws = ring + at * STAGE;
        const uint8_t* xs = ws + W_BYTES;
        free = at;
        at = at + 1 == STAGES ? 0 : at + 1;
#pragma unroll
        for (int h = 0; h < SLICE / 64; ++h) {
            const int w_at = r * SLICE + 16 * ((4 * h + sub) ^ w_turn(r));
            const u32x4 c0 = *reinterpret_cast<const u32x4*>(ws + w_at), c1 = *reinterpret_cast<const u32x4*>(ws + 64 * SLICE + w_at);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const frag f0 = codes8<DT>(c0[2 * e], c0[2 * e + 1]), f1 = codes8<DT>(c1[2 * e], c1[2 * e + 1]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        const int t = q * CAP + 16 * m + r16;
                        const frag x = *reinterpret_cast<const frag*>(xs + t * 2 * SLICE + 16 * ((8 * h + 2 * sub + e) ^ x_turn(r16)));
                        a0[m] = ExpertOp<DT>::run(f0, x, a0[m]);
                        a1[m] = ExpertOp<DT>::run(f1, x, a1[m]);
                    }
            }
        }
    }
    wait_vmcnt<0>();
#pragma unroll
    for (int m = 0; m < MT; ++m) done(m, a0[m], a1[m]);
}

// Hidden values are held as the sum of two BF16: FP16 would overflow where FP32 does not, and one rounding to 16 bits would add as much again to
// the output's error as the output's own.
WQ8_DEVICE void split_hidden(float h, uint32_t& hi, uint32_t& lo) {
    hi = Elem<DT_BF16>::from_f(h);
    const float back = Elem<DT_BF16>::to_f(uint16_t(hi));
    lo = __builtin_isfinite(back) ? Elem<DT_BF16>::from_f(h - back) : 0u;
}

// 4 neighbouring scales, from `rows` on zeros (a multiple of 4)
WQ8_DEVICE v4f scales4(const float* scale, int at, int rows) {
    v4f v = {0, 0, 0, 0};
    if (at < rows) __builtin_memcpy(&v, scale + at, 16);
    return v;
}

// gate and up of hidden channels of an expert, and their product: 16 channels a workgroup, whose waves share them (!own), or 64. Workgroups of
// `pass` n take the choices from 64 n (8 n) on, then those `passes` further.
template <int DT>
__global__ void __launch_bounds__(256, 2) experts_up(ExpertsArgs p, int own, int passes) {
    __shared__ __attribute__((aligned(1024))) uint8_t rings[4 * RING];
    __shared__ uint16_t list[MOST_LISTED];
    const int channels = own ? 64 : 16, groups = (p.hidden + channels - 1) / channels;
    const int tiles = gridDim.x / passes, tile = blockIdx.x % tiles, pass = blockIdx.x / tiles;
    const int slot = tile / groups, f0 = tile % groups * channels, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int expert = slot_expert(p, slot);
    if (uint32_t(expert) >= uint32_t(p.experts)) return;
    const float* scale = p.gate_up_scale + int64_t(expert) * 2 * p.hidden;
    const int64_t plane = int64_t(p.tokens) * p.top * p.hidden;
    const sgpr4 rw = buffer_rsrc(p.gate_up + int64_t(expert) * 2 * p.hidden * p.k, uint32_t(2 * p.hidden) * uint32_t(p.k));
    const sgpr4 rx = buffer_rsrc(p.x, uint32_t((p.tokens - 1) * p.ldx + p.k) * 2u);
    auto source = [&](int i) { return uint32_t(list[i] / p.top) * uint32_t(p.ldx) * 2u; };
    const int f = f0 + (own ? 16 * wave : 0) + 4 * (lane >> 4);  // the channels of this lane's sums
    const v4f gate_scale = scales4(scale, f, p.hidden), up_scale = scales4(scale + p.hidden, f, p.hidden);
    auto store4 = [&](int i, v4f gate, v4f up) {
        u32x2 hi, lo;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t h0, l0, h1, l1;
            split_hidden(wq_swiglu(gate[2 * j] * gate_scale[2 * j], up[2 * j] * up_scale[2 * j]), h0, l0);
            split_hidden(wq_swiglu(gate[2 * j + 1] * gate_scale[2 * j + 1], up[2 * j + 1] * up_scale[2 * j + 1]), h1, l1);
            hi[j] = h0 | h1 << 16;
            lo[j] = l0 | l1 << 16;
        }
        uint16_t* to = p.h + int64_t(list[i]) * p.hidden + f;
        *reinterpret_cast<u32x2*>(to) = hi;
        *reinterpret_cast<u32x2*>(to + plane) = lo;
    };
    const int most = own ? 64 : 8;
    for (int first = pass * most;; first += passes * most) {
        const int rest = find_choices(p, slot, expert, first, list) - first, left = min(rest, most);
        if (left <= 0) return;
        __syncthreads();
        auto done = [&](v4f gate, v4f up) {
            if ((lane & 15) < left && f < p.hidden) store4(lane & 15, gate, up);
        };
        if (!own) {
            if (left <= 4) ring_rows<DT, 128, 4, 1>(rw, f0, p.hidden + f0, p.k, rx, 0, left, rings, source, done);
            else ring_rows<DT, 128, 8, 1>(rw, f0, p.hidden + f0, p.k, rx, 0, left, rings, source, done);
        } else {
            auto done_at = [&](int m, v4f gate, v4f up) {
                if (16 * m + (lane & 15) < left && f < p.hidden) store4(16 * m + (lane & 15), gate, up);
            };
            if (left <= 16) shared_rows<DT, 128, 1, 1>(rw, f0, p.hidden + f0, p.k, rx, 0, left, rings, source, done_at);
            else if (left <= 32) shared_rows<DT, 128, 2, 1>(rw, f0, p.hidden + f0, p.k, rx, 0, left, rings, source, done_at);
            else shared_rows<DT, 64, 4, 1>(rw, f0, p.hidden + f0, p.k, rx, 0, left, rings, source, done_at);
        }
        if (rest <= passes * most) return;
        __syncthreads();
    }
}

// Output channels of an expert for its choices: 32 a workgroup, whose waves share them (!own), or 128.
__global__ void __launch_bounds__(256, 2) experts_down(ExpertsArgs p, int own, int passes) {
    __shared__ __attribute__((aligned(1024))) uint8_t rings[4 * RING];
    __shared__ uint16_t list[MOST_LISTED];
    const int channels = own ? 128 : 32, groups = (p.k + channels - 1) / channels;
    const int tiles = gridDim.x / passes, tile = blockIdx.x % tiles, pass = blockIdx.x / tiles;
    const int slot = tile / groups, n0 = tile % groups * channels, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int expert = slot_expert(p, slot);
    if (uint32_t(expert) >= uint32_t(p.experts)) return;
    const uint32_t plane = uint32_t(p.tokens) * uint32_t(p.top) * uint32_t(p.hidden) * 2u;
    const sgpr4 rw = buffer_rsrc(p.down + int64_t(expert) * p.k * p.hidden, uint32_t(p.k) * uint32_t(p.hidden));
    const sgpr4 rx = buffer_rsrc(p.h, 2u * plane);
    auto source = [&](int i) { return uint32_t(list[i]) * uint32_t(p.hidden) * 2u; };
    const float* scale = p.down_scale + int64_t(expert) * p.k;
    // the channels of this lane's sums: tiles of 16 in two runs, next to each other (!own) or 64 apart
    const int n = n0 + (own ? 16 * wave : 0) + 4 * (lane >> 4), apart = own ? 64 : 16;
    const v4f scale0 = scales4(scale, n, p.k), scale1 = scales4(scale, n + apart, p.k);
    auto store4 = [&](int i, v4f a, v4f b) {
        float* to = p.part + int64_t(list[i]) * p.k + n;
        if (n < p.k) *reinterpret_cast<v4f*>(to) = a * scale0;
        if (n + apart < p.k) *reinterpret_cast<v4f*>(to + apart) = b * scale1;
    };
    const int most = own ? 64 : 8;
    for (int first = pass * most;; first += passes * most) {
        const int rest = find_choices(p, slot, expert, first, list) - first, left = min(rest, most);
        if (left <= 0) return;
        __syncthreads();
        auto done = [&](v4f a, v4f b) {
            if ((lane & 15) < left) store4(lane & 15, a, b);
        };
        if (!own) {
            if (left <= 4) ring_rows<DT_BF16, 128, 4, 2>(rw, n0, n0 + 16, p.hidden, rx, plane, left, rings, source, done);
            else ring_rows<DT_BF16, 64, 8, 2>(rw, n0, n0 + 16, p.hidden, rx, plane, left, rings, source, done);
        } else {
            auto done_at = [&](int m, v4f a, v4f b) {
                if (16 * m + (lane & 15) < left) store4(16 * m + (lane & 15), a, b);
            };
            if (left <= 16) shared_rows<DT_BF16, 128, 1, 2>(rw, n0, n0 + 64, p.hidden, rx, plane, left, rings, source, done_at);
            else if (left <= 32) shared_rows<DT_BF16, 64, 2, 2>(rw, n0, n0 + 64, p.hidden, rx, plane, left, rings, source, done_at);
            else shared_rows<DT_BF16, 64, 4, 2>(rw, n0, n0 + 64, p.hidden, rx, plane, left, rings, source, done_at);
        }
        if (rest <= passes * most) return;
        __syncthreads();
    }
}

// residual + rscale * v, rounded once
template <int DT> WQ8_DEVICE float with_residual(const ExpertsArgs& p, int t, int n, float v) {
    using raw = typename Elem<DT>::raw;
    if (!p.residual) return v;
    const float scale = p.rscale ? Elem<DT>::to_f(static_cast<const raw*>(p.rscale)[n]) : 1.0f;
    return __builtin_fmaf(v, scale, Elem<DT>::to_f(static_cast<const raw*>(p.residual)[t * p.ldr + n]));
}

// A token's parts, weighted and added in the order of its choices: 5.0 us for 32 tokens x 8 x 2048, the length of its loads' chain.
template <int DT>
__global__ void __launch_bounds__(256) experts_join(ExpertsArgs p) {
    using raw = typename Elem<DT>::raw;
    const int quads = p.k / 4, at = blockIdx.x * 256 + threadIdx.x;
    if (at >= p.tokens * quads) return;
    const int t = at / quads, n = at % quads * 4;
    v4f sum = {0, 0, 0, 0};
    for (int j0 = 0; j0 < p.top; j0 += 8) {
        v4f part[8];
        float weight[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int pair = t * p.top + min(j0 + j, p.top - 1);
            const bool held = j0 + j < p.top && uint32_t(p.ids[pair]) < uint32_t(p.experts);  // the others' parts were not written
            part[j] = *reinterpret_cast<const v4f*>(p.part + int64_t(pair) * p.k + n);
            weight[j] = p.weights[pair];
            if (!held) part[j] = v4f{0, 0, 0, 0}, weight[j] = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) sum[i] = __builtin_fmaf(weight[j], part[j][i], sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) static_cast<raw*>(p.out)[t * p.ldo + n + i] = Elem<DT>::from_f(with_residual<DT>(p, t, n + i, sum[i]));
}

// Orders a wave's LDS accesses, its lanes' to each other (they run in step and in order: nothing is waited for).
WQ8_DEVICE void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One token: the second product and the sum over its choices in one launch (8 of 64 experts of 2048 x 1024: 6.6 us for 16.8 MB, cold 7.1; by
// ring_rows and experts_join 6.8 + 4.8). A workgroup has 8 output channels, a wave every eighth choice of the
// token: 8 rows of 128 neighbouring bytes a load, 8 loads ahead, so that an expert's 8 x 1024 codes are asked for at once. One token leaves nothing
// to share, and 16 rows of a matrix instruction would leave half the CUs idle: the products are FP32 on the vector unit, hidden values as FP32.
template <int DT>
__global__ void __launch_bounds__(512) experts_down_one(ExpertsArgs p) {
    using raw = typename Elem<DT>::raw;
    constexpr int STEP = 1024;
    __shared__ __attribute__((aligned(16))) float hidden[8][STEP];
    __shared__ float part[MOST_ONE][8];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n0 = blockIdx.x * 8, row = n0 + (lane >> 3), chunk = lane & 7;
    for (int j = wave; j < p.top; j += 8) {
        const int expert = p.ids[j];
        float sum = 0.0f;
        if (uint32_t(expert) < uint32_t(p.experts)) {
            const int8_t* codes = p.down + (int64_t(expert) * p.k + row) * p.hidden;
            const uint16_t* h = p.h + int64_t(j) * p.hidden;
            const int64_t plane = int64_t(p.top) * p.hidden;
            const float scale = p.down_scale[int64_t(expert) * p.k + row];
            for (int begin = 0; begin < p.hidden; begin += STEP) {
                u32x4 x[2][2], w[8];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int k = begin + 8 * (lane + 64 * i);
#pragma unroll
                    for (int q = 0; q < 2; ++q) x[i][q] = k < p.hidden ? *reinterpret_cast<const u32x4*>(h + q * plane + k) : u32x4{0, 0, 0, 0};
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int k = begin + 128 * i + 16 * chunk;
                    w[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(codes + (k < p.hidden ? k : 0)));  // past the row: against zeros
                }
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        v4f v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int word = 2 * half + (e >> 1), shift = 16 * (e & 1);
                            v[e] = Elem<DT_BF16>::to_f(uint16_t(x[i][0][word] >> shift)) + Elem<DT_BF16>::to_f(uint16_t(x[i][1][word] >> shift));
                        }
                        *reinterpret_cast<v4f*>(&hidden[wave][8 * (lane + 64 * i) + 4 * half]) = v;
                    }
                wave_fence();  // every lane reads what others wrote
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (begin + 128 * i >= p.hidden) break;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const v4f v = *reinterpret_cast<const v4f*>(&hidden[wave][128 * i + 16 * chunk + 4 * c]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum = __builtin_fmaf(float(int8_t(w[i][c] >> (8 * e))), v[e], sum);
                    }
                }
                wave_fence();  // and has read before they write again
            }
            sum += lane_xor<1>(sum);
            sum += lane_xor<2>(sum);
            sum += lane_xor<4>(sum);
            sum *= scale;
        }
        if (!chunk) part[j][lane >> 3] = sum;
    }
    __syncthreads();
    if (threadIdx.x >= 8) return;
    float total = 0.0f;
    for (int j = 0; j < p.top; ++j)
        if (uint32_t(p.ids[j]) < uint32_t(p.experts)) total = __builtin_fmaf(p.weights[j], part[j][threadIdx.x], total);
    static_cast<raw*>(p.out)[n0 + threadIdx.x] = Elem<DT>::from_f(with_residual<DT>(p, 0, n0 + threadIdx.x, total));
}

}  // namespace wq8

using namespace wq8;

// Parts of K: as many as fill the CUs, of whole steps
static int route_parts(int tokens, int experts, int k) {
    const int64_t tiles = int64_t((experts + 15) / 16) * ((tokens + 15) / 16), steps = (k + ROUTE_STEP - 1) / ROUTE_STEP, fill = 512 / tiles;
    return int(fill < 1 ? 1 : fill < steps ? fill : steps);
}

template <int XT>
static void launch_logits(const RouteArgs& p, int router_dtype, hipStream_t stream) {
    const dim3 grid((p.experts + 15) / 16, (p.tokens + 15) / 16, p.parts);
    if (router_dtype == DT_F16) route_logits<XT, DT_F16><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
    else if (router_dtype == DT_BF16) route_logits<XT, DT_BF16><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
    else route_logits<XT, DT_F32><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
}

WQ8_API int wq8_route(const void* x, int64_t ldx, int dtype, const void* router, int router_dtype, const float* bias, int tokens, int experts, int k, int top,
                      int score, int normalise, float factor, void* logits, int32_t* ids, float* weights, hipStream_t stream) {
    if (!tokens) return 0;
    if (dtype < 0 || dtype > 2 || router_dtype < 0 || router_dtype > 2 || score < 0 || score > 1) return -1;
    if (tokens < 0 || tokens > 65535 * 16 || experts < 1 || experts > 1024 || k < 8 || k % 8 || top < 1 || top > 64 || top > experts) return -2;
    const int wanted = route_parts(tokens, experts, k), steps = (k + ROUTE_STEP - 1) / ROUTE_STEP, part = (steps + wanted - 1) / wanted * ROUTE_STEP;
    const RouteArgs p{x, router, bias, static_cast<double*>(logits), ids, weights, ldx, tokens, experts, k, top, score, normalise, (k + part - 1) / part, part,
                      factor};
    if (dtype == DT_F16) launch_logits<DT_F16>(p, router_dtype, stream);
    else if (dtype == DT_BF16) launch_logits<DT_BF16>(p, router_dtype, stream);
    else launch_logits<DT_F32>(p, router_dtype, stream);
    if (const int rc = int(hipGetLastError())) return rc;
    const int groups = (tokens + 3) / 4;
    if (experts <= 64) route_choose<1><<<groups, 256, 0, stream>>>(p);
    else if (experts <= 128) route_choose<2><<<groups, 256, 0, stream>>>(p);
    else if (experts <= 256) route_choose<4><<<groups, 256, 0, stream>>>(p);
    else route_choose<16><<<groups, 256, 0, stream>>>(p);
    return int(hipGetLastError());
}

WQ8_API void wq8_route_workspace(int tokens, int experts, int k, int64_t* sizes) {
    sizes[0] = tokens > 0 && experts > 0 ? int64_t(route_parts(tokens, experts, k)) * tokens * experts * 8 : 0;
    sizes[1] = 0;
}

WQ8_API int wq8_experts(const void* x, int64_t ldx, int dtype, const void* ids, const float* weights, const int8_t* gate_up, const float* gate_up_scale,
                        const int8_t* down, const float* down_scale, const void* residual, int64_t ldr, const void* rscale, void* out, int64_t ldo, int tokens,
                        int top, int experts, int k, int hidden, void* workspace, hipStream_t stream) {
    if (!tokens) return 0;
    if (dtype != DT_F16 && dtype != DT_BF16) return -1;
    if (tokens < 0 || top < 1 || int64_t(tokens) * top > MOST_PAIRS || experts < 1 || k < 16 || k % 16 || hidden < 16 || hidden % 16) return -2;
    // an expert's matrix, the rows and the hidden values are each read through a buffer descriptor: less than 2 GiB
    if (int64_t(2) * hidden * k >= 1ll << 31 || ((tokens - 1) * ldx + k) * 2 >= 1ll << 31 || int64_t(tokens) * top * hidden * 4 >= 1ll << 31) return -2;
    const int pairs = tokens * top, slots = pairs <= experts ? pairs : experts;
    const int64_t h_bytes = (int64_t(pairs) * hidden * 4 + 255) / 256 * 256;
    const ExpertsArgs p{x, static_cast<const int32_t*>(ids), weights, gate_up, gate_up_scale, down, down_scale, static_cast<uint16_t*>(workspace),
                        reinterpret_cast<float*>(static_cast<char*>(workspace) + h_bytes), residual, rscale, out, ldx, ldr, ldo, tokens, top, experts, k, hidden};
    // Waves share tiles (ring_rows) in calls of up to 8 tokens with fewer than 1024 of them, of which the other form would make fewer workgroups than there
    // are CUs, or 2048 where a tile is long, whose beginning weighs less. Both products, us (ring_rows, shared_rows), tokens x channels x hidden, experts, choices:
    // 1 x 2048 x 1024, 64, 8 (512 tiles) 18.2, 21.6; 5 x 1552 x 592, 21, 3 (555, gate and up alone) 9.4, 12.2; 2 x 2048 x 1024, 64, 8 (1024) 32.1, 28.3; 8 x 1024 x 512, 32,
    // 4 (1024) 22.4, 18.2; 4 x 2048 x 1024, 64, 8 (2048) 48.2, 38.6; 2 x 5120 x 1536, 16, 2 (384) 29.7, 39.3; 4 x 5120 x 1536, 16, 4 (1536, of 5120) 49, 62.
    const auto shares = [&](int64_t tiles, int width) { return tokens <= 8 && slots * tiles < (width >= 4096 ? 2048 : 1024); };
    const int up = !shares(hidden / 16, k), down_own = !shares((k + 31) / 32, hidden);
    const int up_groups = up ? (hidden + 63) / 64 : hidden / 16, down_groups = down_own ? (k + 127) / 128 : (k + 31) / 32;
    // an expert of more tokens than a workgroup takes at once: other workgroups take the next ones
    const auto passes = [&](int most) { return tokens <= most ? 1 : tokens <= 2 * most ? 2 : 4; };
    const int up_passes = up ? passes(64) : 1, down_passes = down_own ? passes(64) : 1;
    if (int64_t(slots) * up_groups * up_passes > MAX_BLOCKS_256 || int64_t(slots) * down_groups * down_passes > MAX_BLOCKS_256 ||
        int64_t(tokens) * (k / 4) > 1ll << 30)
        return -2;
    if (dtype == DT_F16) experts_up<DT_F16><<<slots * up_groups * up_passes, 256, 0, stream>>>(p, up, up_passes);
    else experts_up<DT_BF16><<<slots * up_groups * up_passes, 256, 0, stream>>>(p, up, up_passes);
    if (const int rc = int(hipGetLastError())) return rc;
    if (tokens == 1 && top <= MOST_ONE) {
        if (dtype == DT_F16) experts_down_one<DT_F16><<<k / 8, 512, 0, stream>>>(p);
        else experts_down_one<DT_BF16><<<k / 8, 512, 0, stream>>>(p);
        return int(hipGetLastError());
    }
    experts_down<<<slots * down_groups * down_passes, 256, 0, stream>>>(p, down_own, down_passes);
    if (const int rc = int(hipGetLastError())) return rc;
    const int groups = (tokens * (k / 4) + 255) / 256;
    if (dtype == DT_F16) experts_join<DT_F16><<<groups, 256, 0, stream>>>(p);
    else experts_join<DT_BF16><<<groups, 256, 0, stream>>>(p);
    return int(hipGetLastError());
}

WQ8_API void wq8_experts_workspace(int tokens, int top, int k, int hidden, int64_t* sizes) {
    const int64_t pairs = int64_t(tokens) * top;
    sizes[0] = (pairs * hidden * 4 + 255) / 256 * 256 + pairs * k * 4;
    sizes[1] = 0;
}

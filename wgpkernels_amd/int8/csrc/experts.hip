// A mixture-of-experts layer of INT8 weights for a few tokens on gfx950: the router (its product in 64 bits, and its choice) and the chosen
// experts' gated feed-forward blocks,
//     y[t] = residual[t] + rscale * sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),   e = ids[t, j],
// every chosen expert's weights read once from HBM for all of its tokens. No reference counterpart.
#include "gemm_common.h"
#include "wq8_abi.h"
#include <type_traits>

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
    int tokens, experts, k, top, score, normalise;
    float factor;
};

// 8 consecutive values as FP64; zeros when !valid.
template <int DT> WQ8_DEVICE void load8d(const void* base, int64_t at, bool valid, double* v) {
    float f[8];
    load8<DT>(static_cast<const typename Elem<DT>::raw*>(base) + at, f, valid);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = double(f[j]);
}

// Logits of 16 tokens x 16 experts in FP64 (the choice between near experts is a whole number: in FP32 one in some 10^4 tokens would go by the
// order of the sum). 16 waves share K, 32 values of every row a step; their sums are added in order.
constexpr int ROUTE_WAVES = 16;
template <int XT, int RT>
__global__ void __launch_bounds__(64 * ROUTE_WAVES) route_logits(RouteArgs p) {
    __shared__ double sums[ROUTE_WAVES][4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int expert = blockIdx.x * 16 + (lane & 15), token = blockIdx.y * 16 + (lane & 15);
    const bool has_expert = expert < p.experts, has_token = token < p.tokens;
    v4d acc = {0, 0, 0, 0};
    for (int k = 8 * (lane >> 4) + 32 * wave; k - 8 * (lane >> 4) < p.k; k += 32 * ROUTE_WAVES) {
        double a[8], b[8];
        load8d<XT>(p.x, token * p.ldx + k, has_token && k < p.k, a);
        load8d<RT>(p.router, int64_t(expert) * p.k + k, has_expert && k < p.k, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc = __builtin_amdgcn_mfma_f64_16x16x4f64(a[j], b[j], acc, 0, 0, 0);
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
    if (has_expert && t < p.tokens) p.logits[int64_t(t) * p.experts + expert] = total;
}

// A double's order as an unsigned number above 1; 1 for NaN.
WQ8_DEVICE uint64_t order_of(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v);
    return v != v ? 1 : b >> 63 ? ~b : b | (uint64_t(1) << 63);
}
WQ8_DEVICE uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) {
        const uint64_t other = __shfl_xor(v, step);
        v = other > v ? other : v;
    }
    return v;
}
WQ8_DEVICE double wave_sum64(double v) {
#pragma unroll
    for (int step = 32; step; step >>= 1) v += __shfl_xor(v, step);
    return v;
}

// Scores, choice and weights of a token a wave; a lane holds NE neighbouring experts.
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
        top = __builtin_fmax(top, score[i]);
    }
    if (p.score == 0) {
#pragma unroll
        for (int step = 32; step; step >>= 1) top = __builtin_fmax(top, __shfl_xor(top, step));
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
        const int from = __builtin_ctzll(__ballot(best == most));  // neighbouring experts a lane: the lowest lane has the lowest index
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
        value = __shfl(value, from);
        e = __shfl(e, from);
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
constexpr int MOST_PAIRS = 4096;

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
// Their number (0: another slot has them), and those from `first` on, up to MOST_LISTED, in LDS; every wave counts, the first one writes.
constexpr int MOST_LISTED = 64;
WQ8_DEVICE int find_choices(const ExpertsArgs& p, int slot, int expert, int first, uint16_t* list) {
    const int pairs = p.tokens * p.top, lane = threadIdx.x & 63;
    const bool by_choice = slot_is_choice(p);
    int count = 0;
    for (int base = 0; base < pairs; base += 64) {
        const bool mine = base + lane < pairs && p.ids[base + lane] == expert;
        const uint64_t mask = __ballot(mine);
        if (!mask) continue;
        if (by_choice && !count && base + __builtin_ctzll(mask) != slot) return 0;
        const int at = count + __popcll(mask & ((uint64_t(1) << lane) - 1)) - first;
        if (threadIdx.x < 64 && mine && at >= 0 && at < MOST_LISTED) list[at] = uint16_t(base + lane);
        count += __popcll(mask);
    }
    return count;
}

// Two tiles of 16 weight rows on up to CAP tokens (PLANES rows each). The four waves of a workgroup take slices of SLICE values of the width in
// turn, each through a ring of its own in LDS, filled by copies that pass the registers by: no wave waits for another one until the
// end, where the four sums of every output are added in order. 16-byte chunks are placed by their row so that the 16 lanes that read one chunk of
// 16 rows meet different banks.
constexpr int RING = 19 * 1024;  // a wave's: two workgroups a CU
constexpr uint32_t OUT_OF_RANGE = 0x80000000u;
template <int DT, int SLICE, int CAP, int PLANES, typename Source, typename Store>
WQ8_DEVICE void ring_rows(sgpr4 rw, int row0, int row1, int rows, int width, sgpr4 rx, uint32_t plane_bytes, int count, uint8_t* rings, const Source& source,
                          const Store& store) {
    constexpr int W_BYTES = 32 * SLICE, X_BYTES = CAP * PLANES * SLICE * 2, STAGE = W_BYTES + X_BYTES, STAGES = RING / STAGE < 8 ? RING / STAGE : 8;
    constexpr int W_COPIES = W_BYTES / 1024, X_COPIES = X_BYTES / 1024, COPIES = W_COPIES + X_COPIES, MT = (CAP + 15) / 16;
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
        w_from[j] = uint32_t(min(r < 16 ? row0 + r : row1 + r - 16, rows - 1)) * uint32_t(width) + 16u * chunk;
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
    v4f a0[MT], a1[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) a0[m] = a1[m] = v4f{0, 0, 0, 0};
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
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        const int t = q * CAP + (CAP < 16 ? r16 & (CAP - 1) : 16 * m + r16);
                        const frag x = *reinterpret_cast<const frag*>(xs + t * 2 * SLICE + 16 * ((8 * h + 2 * sub + e) ^ x_turn(t)));
                        a0[m] = ExpertOp<DT>::run(f0, x, a0[m]);
                        a1[m] = ExpertOp<DT>::run(f1, x, a1[m]);
                    }
            }
        }
    }
    wait_vmcnt<0>();
    float (&red)[4][8][64] = *reinterpret_cast<float (*)[4][8][64]>(rings);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            red[wave][i][lane] = a0[m][i];
            red[wave][4 + i][lane] = a1[m][i];
        }
        __syncthreads();
        // element i of lane l is row 4 (l / 16) + i, token l % 16
        const int r = threadIdx.x & 15, t = threadIdx.x >> 4, l = 16 * (r >> 2) + t, i = r & 3;
        if (t < CAP && 16 * m + t < count)
            store(16 * m + t, r, ((red[0][i][l] + red[1][i][l]) + red[2][i][l]) + red[3][i][l],
                  ((red[0][4 + i][l] + red[1][4 + i][l]) + red[2][4 + i][l]) + red[3][4 + i][l]);
    }
}

// The same tiles, every wave with tiles of its own over the whole width: `blocks` of them one after another, `step` rows apart, without a pause in the copies
// between them. A workgroup of tiles this small would mostly begin and end. done(block, row's values of both tiles): element i is row
// 4 (lane / 16) + i, token lane % 16.
template <int DT, int SLICE, int CAP, int PLANES, typename Source, typename Done>
WQ8_DEVICE void ring_blocks(sgpr4 rw, int row0, int row1, int step, int blocks, int width, sgpr4 rx, uint32_t plane_bytes, int count, uint8_t* rings,
                            const Source& source, const Done& done) {
    constexpr int W_BYTES = 32 * SLICE, X_BYTES = CAP * PLANES * SLICE * 2, STAGE = W_BYTES + X_BYTES, STAGES = RING / STAGE < 8 ? RING / STAGE : 8;
    constexpr int W_COPIES = W_BYTES / 1024, X_COPIES = X_BYTES / 1024, COPIES = W_COPIES + X_COPIES;
    constexpr int W_CHUNKS = SLICE / 16, X_CHUNKS = SLICE / 8;
    static_assert(STAGES >= 3 && X_BYTES % 1024 == 0 && (STAGES - 1) * COPIES < 64 && CAP <= 16, "a ring of stages of whole copies");
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
    int next_k = 0, to_issue = blocks;
    uint32_t next_rows = 0;
    auto issue = [&](uint8_t* stage) {
        const int end = to_issue > 0 ? width : 0;
#pragma unroll
        for (int j = 0; j < W_COPIES; ++j) bdma16_nt(rw, next_k + w_k[j] < end ? w_from[j] + next_rows + uint32_t(next_k) : OUT_OF_RANGE, stage + 1024 * j);
#pragma unroll
        for (int j = 0; j < X_COPIES; ++j) bdma16(rx, next_k + x_k[j] < end ? x_from[j] + 2u * uint32_t(next_k) : OUT_OF_RANGE, stage + W_BYTES + 1024 * j);
        next_k += SLICE;
        if (next_k >= width) {
            next_k = 0;
            next_rows += uint32_t(step) * uint32_t(width);
            --to_issue;
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(ring + i * STAGE);
    int at = 0, free = STAGES - 1;
    for (int block = 0; block < blocks; ++block) {
        v4f a0 = {0, 0, 0, 0}, a1 = {0, 0, 0, 0};
        for (int k = 0; k < width; k += SLICE) {
            wait_vmcnt<(STAGES - 2) * COPIES>();
            wait_lgkm0();
            asm volatile("" ::: "memory");
            issue(ring + free * STAGE);
            const uint8_t* ws = ring + at * STAGE;
            const uint8_t* xs = ws + W_BYTES;
            free = at;
            at = at + 1 == STAGES ? 0 : at + 1;
#pragma unroll
            for (int h = 0; h < SLICE / 64; ++h) {
                const int chunk = (4 * h + sub) ^ w_turn(r16);
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
        done(block, a0, a1);
    }
    wait_vmcnt<0>();
}

// More tokens: 64 rows a workgroup (tile c of each of two runs of 32 rows, c = 0 and 1, for waves c and c + 2, which take alternate halves of a
// slice), and the tokens' slices in LDS once for all of them. done(m, c, both tiles' values) of waves 0 and 1: element i is row 16 c + 4 (lane / 16) + i of each
// run, token 16 m + lane % 16.
template <int DT, int MT, int PLANES, typename Source, typename Done>
WQ8_DEVICE void shared_rows(sgpr4 rw, int row0, int row1, int width, sgpr4 rx, uint32_t plane_bytes, int count, uint8_t* ring, const Source& source,
                            const Done& done) {
    constexpr int SLICE = 128, CAP = 16 * MT, W_BYTES = 64 * SLICE, X_BYTES = CAP * PLANES * SLICE * 2, STAGE = W_BYTES + X_BYTES;
    constexpr int STAGES = 4 * RING / STAGE < 8 ? 4 * RING / STAGE : 8, W_COPIES = W_BYTES / 4096, X_COPIES = X_BYTES / 4096, COPIES = W_COPIES + X_COPIES;
    static_assert(STAGES >= 3 && (STAGES - 1) * COPIES < 64, "a ring of stages");
    using frag = typename ExpertOp<DT>::frag;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, sub = lane >> 4;
    const int c = wave & 1, half = wave >> 1;
    uint32_t w_from[W_COPIES], x_from[X_COPIES];
    int w_k[W_COPIES], x_k[X_COPIES];
#pragma unroll
    for (int j = 0; j < W_COPIES; ++j) {
        const int r = (wave + 4 * j) * 8 + lane / 8, chunk = lane % 8 ^ (r >> 1 & 7);  // LDS row r: run r / 32, row r % 32 of it
        w_k[j] = 16 * chunk;
        w_from[j] = uint32_t(r < 32 ? row0 + r : row1 + r - 32) * uint32_t(width) + 16u * chunk;
    }
#pragma unroll
    for (int j = 0; j < X_COPIES; ++j) {
        const int q = (wave + 4 * j) * 4 + lane / 16, chunk = lane % 16 ^ (q & 15);
        x_k[j] = 8 * chunk;
        x_from[j] = source(min(q % CAP, count - 1)) + (PLANES > 1 && q >= CAP ? plane_bytes : 0u) + 16u * chunk;
    }
    auto issue = [&](int k0, uint8_t* stage) {
#pragma unroll
        for (int j = 0; j < W_COPIES; ++j)
            bdma16_nt(rw, k0 + w_k[j] < width ? w_from[j] + uint32_t(k0) : OUT_OF_RANGE, stage + 1024 * (wave + 4 * j));
#pragma unroll
        for (int j = 0; j < X_COPIES; ++j)
            bdma16(rx, k0 + x_k[j] < width ? x_from[j] + 2u * uint32_t(k0) : OUT_OF_RANGE, stage + W_BYTES + 1024 * (wave + 4 * j));
    };
    v4f a0[MT], a1[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) a0[m] = a1[m] = v4f{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i * SLICE, ring + i * STAGE);
    int at = 0, free = STAGES - 1;
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
        const int r = 16 * c + r16, chunk = (4 * half + sub) ^ (r >> 1 & 7);
        const u32x4 c0 = *reinterpret_cast<const u32x4*>(ws + r * SLICE + 16 * chunk);
        const u32x4 c1 = *reinterpret_cast<const u32x4*>(ws + (32 + r) * SLICE + 16 * chunk);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const frag f0 = codes8<DT>(c0[2 * e], c0[2 * e + 1]), f1 = codes8<DT>(c1[2 * e], c1[2 * e + 1]);
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    const int t = q * CAP + 16 * m + r16;
                    const frag x = *reinterpret_cast<const frag*>(xs + t * 2 * SLICE + 16 * ((8 * half + 2 * sub + e) ^ r16));
                    a0[m] = ExpertOp<DT>::run(f0, x, a0[m]);
                    a1[m] = ExpertOp<DT>::run(f1, x, a1[m]);
                }
        }
    }
    wait_vmcnt<0>();
    __syncthreads();
    // the second waves hand their sums over
    v4f* red = reinterpret_cast<v4f*>(ring) + c * MT * 2 * 64 + lane;
    if (half)
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            red[m * 128] = a0[m];
            red[m * 128 + 64] = a1[m];
        }
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int m = 0; m < MT; ++m) done(m, c, a0[m] + red[m * 128], a1[m] + red[m * 128 + 64]);
}

// Hidden values are held as the sum of two BF16: FP16 would overflow where FP32 does not, and one rounding to 16 bits would add as much again to
// the output's error as the output's own.
WQ8_DEVICE void split_hidden(float h, uint32_t& hi, uint32_t& lo) {
    hi = Elem<DT_BF16>::from_f(h);
    const float back = Elem<DT_BF16>::to_f(uint16_t(hi));
    lo = __builtin_isfinite(back) ? Elem<DT_BF16>::from_f(h - back) : 0u;
}

constexpr int MOST_BLOCKS = 4;  // tiles a wave, one after another

// gate and up of hidden channels of an expert, and their product: 16 channels a workgroup (own 0), or 64 `own` of them.
template <int DT>
__global__ void __launch_bounds__(256, 2) experts_up(ExpertsArgs p, int own) {
    __shared__ __attribute__((aligned(1024))) uint8_t rings[4 * RING];
    __shared__ float scales[2][64 * MOST_BLOCKS];
    __shared__ uint16_t list[MOST_LISTED];
    const int channels = own ? 64 * own : 16, groups = (p.hidden + channels - 1) / channels;
    const int slot = blockIdx.x / groups, f0 = (blockIdx.x % groups) * channels, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int expert = slot_expert(p, slot), here = min(channels, p.hidden - f0);
    if (uint32_t(expert) >= uint32_t(p.experts)) return;
    const float* scale = p.gate_up_scale + int64_t(expert) * 2 * p.hidden + f0;
    const int64_t plane = int64_t(p.tokens) * p.top * p.hidden;
    const sgpr4 rw = buffer_rsrc(p.gate_up + int64_t(expert) * 2 * p.hidden * p.k, uint32_t(2 * p.hidden) * uint32_t(p.k));
    const sgpr4 rx = buffer_rsrc(p.x, uint32_t((p.tokens - 1) * p.ldx + p.k) * 2u);
    auto source = [&](int i) { return uint32_t(list[i] / p.top) * uint32_t(p.ldx) * 2u; };
    // channels f0 + f .. + 3 of choice i
    auto store4 = [&](int i, int f, v4f gate, v4f up) {
        u32x2 hi, lo;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            uint32_t h0, l0, h1, l1;
            split_hidden(wq_swiglu(gate[2 * j] * scales[0][f + 2 * j], up[2 * j] * scales[1][f + 2 * j]), h0, l0);
            split_hidden(wq_swiglu(gate[2 * j + 1] * scales[0][f + 2 * j + 1], up[2 * j + 1] * scales[1][f + 2 * j + 1]), h1, l1);
            hi[j] = h0 | h1 << 16;
            lo[j] = l0 | l1 << 16;
        }
        uint16_t* to = p.h + int64_t(list[i]) * p.hidden + f0 + f;
        *reinterpret_cast<u32x2*>(to) = hi;
        *reinterpret_cast<u32x2*>(to + plane) = lo;
    };
    for (int f = threadIdx.x; f < here; f += 256) scales[0][f] = scale[f], scales[1][f] = scale[p.hidden + f];
    const int lane = threadIdx.x & 63;
    const int most = own ? 64 : 8;
    for (int first = 0;; first += most) {
        const int rest = find_choices(p, slot, expert, first, list) - first, left = min(rest, most);
        if (left <= 0) return;
        __syncthreads();
        if (!own) {
            auto store = [&](int i, int r, float gate, float up) {
                uint32_t hi, lo;
                split_hidden(wq_swiglu(gate * scales[0][r], up * scales[1][r]), hi, lo);
                const int64_t at = int64_t(list[i]) * p.hidden + f0 + r;
                p.h[at] = uint16_t(hi);
                p.h[at + plane] = uint16_t(lo);
            };
            if (left <= 4) ring_rows<DT, 128, 4, 1>(rw, f0, p.hidden + f0, 2 * p.hidden, p.k, rx, 0, left, rings, source, store);
            else ring_rows<DT, 128, 8, 1>(rw, f0, p.hidden + f0, 2 * p.hidden, p.k, rx, 0, left, rings, source, store);
        } else if (left <= 8) {
            const int mine = (here / 16 - wave + 3) / 4;
            auto done = [&](int block, v4f gate, v4f up) {
                const int f = 16 * (wave + 4 * block) + 4 * (lane >> 4);
                if ((lane & 15) < left) store4(lane & 15, f, gate, up);
            };
            if (left <= 4) ring_blocks<DT, 128, 4, 1>(rw, f0 + 16 * wave, p.hidden + f0 + 16 * wave, 64, mine, p.k, rx, 0, left, rings, source, done);
            else ring_blocks<DT, 128, 8, 1>(rw, f0 + 16 * wave, p.hidden + f0 + 16 * wave, 64, mine, p.k, rx, 0, left, rings, source, done);
        } else {
            for (int f = 0; f < here; f += 32) {
                auto done = [&](int m, int c, v4f gate, v4f up) {
                    const int i = 16 * m + (lane & 15), at = f + 16 * c;
                    if (i < left && at < here) store4(i, at + 4 * (lane >> 4), gate, up);
                };
                if (f) __syncthreads();
                if (left <= 16) shared_rows<DT, 1, 1>(rw, f0 + f, p.hidden + f0 + f, p.k, rx, 0, left, rings, source, done);
                else if (left <= 32) shared_rows<DT, 2, 1>(rw, f0 + f, p.hidden + f0 + f, p.k, rx, 0, left, rings, source, done);
                else shared_rows<DT, 4, 1>(rw, f0 + f, p.hidden + f0 + f, p.k, rx, 0, left, rings, source, done);
            }
        }
        if (rest <= most) return;
        __syncthreads();
    }
}

// Output channels of an expert for its choices, weighted: 32 a workgroup (own 0), or 128 `own`.
__global__ void __launch_bounds__(256, 2) experts_down(ExpertsArgs p, int own) {
    __shared__ __attribute__((aligned(1024))) uint8_t rings[4 * RING];
    __shared__ float scales[128 * MOST_BLOCKS], weights[MOST_LISTED];
    __shared__ uint16_t list[MOST_LISTED];
    const int channels = own ? 128 * own : 32, groups = (p.k + channels - 1) / channels;
    const int slot = blockIdx.x / groups, n0 = (blockIdx.x % groups) * channels, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int expert = slot_expert(p, slot), here = min(channels, p.k - n0);
    if (uint32_t(expert) >= uint32_t(p.experts)) return;
    const uint32_t plane = uint32_t(p.tokens) * uint32_t(p.top) * uint32_t(p.hidden) * 2u;
    const sgpr4 rw = buffer_rsrc(p.down + int64_t(expert) * p.k * p.hidden, uint32_t(p.k) * uint32_t(p.hidden));
    const sgpr4 rx = buffer_rsrc(p.h, 2u * plane);
    auto source = [&](int i) { return uint32_t(list[i]) * uint32_t(p.hidden) * 2u; };
    // channels n0 + n .. + 3 of choice i
    auto store4 = [&](int i, int n, v4f v) {
        if (n >= here) return;
        const float weight = weights[i];
        v4f out;
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = v[j] * scales[n + j] * weight;
        *reinterpret_cast<v4f*>(p.part + int64_t(list[i]) * p.k + n0 + n) = out;
    };
    for (int n = threadIdx.x; n < here; n += 256) scales[n] = p.down_scale[int64_t(expert) * p.k + n0 + n];
    const int lane = threadIdx.x & 63;
    const int most = own ? 32 : 8;
    for (int first = 0;; first += most) {
        const int rest = find_choices(p, slot, expert, first, list) - first, left = min(rest, most);
        if (left <= 0) return;
        __syncthreads();
        if (threadIdx.x < left) weights[threadIdx.x] = p.weights[list[threadIdx.x]];
        __syncthreads();
        if (!own) {
            auto store = [&](int i, int r, float a, float b) {
                float* to = p.part + int64_t(list[i]) * p.k + n0 + r;
                if (r < here) to[0] = a * scales[r] * weights[i];
                if (16 + r < here) to[16] = b * scales[16 + r] * weights[i];
            };
            if (left <= 4) ring_rows<DT_BF16, 128, 4, 2>(rw, n0, n0 + 16, p.k, p.hidden, rx, plane, left, rings, source, store);
            else ring_rows<DT_BF16, 64, 8, 2>(rw, n0, n0 + 16, p.k, p.hidden, rx, plane, left, rings, source, store);
        } else if (left <= 8) {
            const int mine = ((here + 31) / 32 - wave + 3) / 4;
            auto done = [&](int block, v4f a, v4f b) {
                const int n = 32 * (wave + 4 * block) + 4 * (lane >> 4);
                if ((lane & 15) < left) store4(lane & 15, n, a), store4(lane & 15, n + 16, b);
            };
            if (left <= 4) ring_blocks<DT_BF16, 64, 4, 2>(rw, n0 + 32 * wave, n0 + 32 * wave + 16, 128, mine, p.hidden, rx, plane, left, rings, source, done);
            else ring_blocks<DT_BF16, 64, 8, 2>(rw, n0 + 32 * wave, n0 + 32 * wave + 16, 128, mine, p.hidden, rx, plane, left, rings, source, done);
        } else {
            for (int n = 0; n < here; n += 64) {
                auto done = [&](int m, int c, v4f a, v4f b) {
                    const int i = 16 * m + (lane & 15), at = n + 16 * c + 4 * (lane >> 4);
                    if (i < left) store4(i, at, a), store4(i, at + 32, b);
                };
                if (n) __syncthreads();
                if (left <= 16) shared_rows<DT_BF16, 1, 2>(rw, n0 + n, n0 + n + 32, p.hidden, rx, plane, left, rings, source, done);
                else shared_rows<DT_BF16, 2, 2>(rw, n0 + n, n0 + n + 32, p.hidden, rx, plane, left, rings, source, done);
            }
        }
        if (rest <= most) return;
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

// A token's parts, added in the order of its choices.
template <int DT>
__global__ void __launch_bounds__(256) experts_join(ExpertsArgs p) {
    using raw = typename Elem<DT>::raw;
    const int quads = p.k / 4, at = blockIdx.x * 256 + threadIdx.x;
    if (at >= p.tokens * quads) return;
    const int t = at / quads, n = at % quads * 4;
    v4f sum = {0, 0, 0, 0};
    for (int j = 0; j < p.top; ++j) {
        const int pair = t * p.top + j;
        if (uint32_t(p.ids[pair]) >= uint32_t(p.experts)) continue;
        sum += *reinterpret_cast<const v4f*>(p.part + int64_t(pair) * p.k + n);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) static_cast<raw*>(p.out)[t * p.ldo + n + i] = Elem<DT>::from_f(with_residual<DT>(p, t, n + i, sum[i]));
}

}  // namespace wq8

using namespace wq8;

template <int XT>
static void launch_logits(const RouteArgs& p, int router_dtype, hipStream_t stream) {
    const dim3 grid((p.experts + 15) / 16, (p.tokens + 15) / 16);
    if (router_dtype == DT_F16) route_logits<XT, DT_F16><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
    else if (router_dtype == DT_BF16) route_logits<XT, DT_BF16><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
    else route_logits<XT, DT_F32><<<grid, 64 * ROUTE_WAVES, 0, stream>>>(p);
}

WQ8_API int wq8_route(const void* x, int64_t ldx, int dtype, const void* router, int router_dtype, const float* bias, int tokens, int experts, int k, int top,
                      int score, int normalise, float factor, void* logits, int32_t* ids, float* weights, hipStream_t stream) {
    if (!tokens) return 0;
    if (dtype < 0 || dtype > 2 || router_dtype < 0 || router_dtype > 2 || score < 0 || score > 1) return -1;
    if (tokens < 0 || tokens > 65535 * 16 || experts < 1 || experts > 1024 || k < 8 || k % 8 || top < 1 || top > 64 || top > experts) return -2;
    const RouteArgs p{x, router, bias, static_cast<double*>(logits), ids, weights, ldx, tokens, experts, k, top, score, normalise, factor};
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
    if (int64_t(slots) * (hidden / 16) > MAX_BLOCKS_256 || int64_t(slots) * ((k + 31) / 32) > MAX_BLOCKS_256 || int64_t(tokens) * (k / 4) > MAX_BLOCKS_256 * 64) return -2;
    const ExpertsArgs p{x, static_cast<const int32_t*>(ids), weights, gate_up, gate_up_scale, down, down_scale, static_cast<uint16_t*>(workspace),
                        reinterpret_cast<float*>(static_cast<char*>(workspace) + h_bytes), residual, rscale, out, ldx, ldr, ldo, tokens, top, experts, k, hidden};
    // tiles that waves share only where there are few, of 8 tokens at most
    const auto own = [&](int64_t tiles, int waves) { return tokens <= 8 && slots * tiles <= 1024 ? 0 : slots * tiles <= 4096 ? 1 : slots * tiles <= 8192 ? 2 : MOST_BLOCKS; };
    const int up = own(hidden / 16, 4), down_own = own((k + 31) / 32, 4);
    const int up_groups = up ? (hidden + 64 * up - 1) / (64 * up) : hidden / 16, down_groups = down_own ? (k + 128 * down_own - 1) / (128 * down_own) : (k + 31) / 32;
    if (dtype == DT_F16) experts_up<DT_F16><<<slots * up_groups, 256, 0, stream>>>(p, up);
    else experts_up<DT_BF16><<<slots * up_groups, 256, 0, stream>>>(p, up);
    if (const int rc = int(hipGetLastError())) return rc;
    experts_down<<<slots * down_groups, 256, 0, stream>>>(p, down_own);
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

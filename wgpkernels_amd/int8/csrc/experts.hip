// A mixture-of-experts layer of INT8 weights for a few tokens on gfx950: the router (its product in 64 bits, and its choice) and the chosen
// experts' gated feed-forward blocks,
//     y[t] = residual[t] + rscale * sum_j weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),   e = ids[t, j],
// every chosen expert's weights read once from HBM for all of its tokens. No reference counterpart.
#include "wq8_common.h"
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

// Where lanes past a row's end read their activations
__device__ const uint32_t zero_values[8] = {0, 0, 0, 0, 0, 0, 0, 0};

// Two tiles of weight rows on up to MT x 16 / P tokens. A matrix instruction takes 16 rows and 16 columns; here its rows are 16 / P weight
// rows, each P times over with another part of its values, and its columns 16 / P tokens likewise, so that a load of 16 bytes a lane covers 64 P
// neighbouring bytes of a row (few tokens: wide pieces of few rows, which HBM serves faster) and the products of one part with
// another's are not used. Lane l is row l % 16 of the operands: w0, w1 its weight rows, x its tokens' rows (`plane` values apart where there
// are two), `at` its first value; steps of 64 P values up to `end`, U of them asked for ahead.
template <int DT, int P, int MT, int PLANES, int U>
WQ8_DEVICE void stream_tiles(const int8_t* w0, const int8_t* w1, const uint16_t* const (&x)[MT], int64_t plane, int at, int end, int steps, v4f (&a0)[MT],
                             v4f (&a1)[MT]) {
    const int groups = (steps + U - 1) / U;
    u32x4 w[2][U][2], v[2][U][MT][PLANES][2];
    auto load = [&](auto buffer, int g) {
        constexpr int B = decltype(buffer)::value;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = at + (g * U + u) * 64 * P;
            const bool inside = k < end;
            const int from = inside ? k : 0;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int q = 0; q < PLANES; ++q) {
                    const u32x4* s = inside ? reinterpret_cast<const u32x4*>(x[m] + q * plane + k) : reinterpret_cast<const u32x4*>(zero_values);
                    v[B][u][m][q][0] = s[0];
                    v[B][u][m][q][1] = s[1];
                }
            w[B][u][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w0 + from));
            w[B][u][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(w1 + from));
        }
    };
    auto multiply = [&](auto buffer) {
        constexpr int B = decltype(buffer)::value;
        using frag = typename ExpertOp<DT>::frag;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const frag f0 = codes8<DT>(w[B][u][0][2 * half], w[B][u][0][2 * half + 1]);
                const frag f1 = codes8<DT>(w[B][u][1][2 * half], w[B][u][1][2 * half + 1]);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int q = 0; q < PLANES; ++q) {
                        const frag b = __builtin_bit_cast(frag, v[B][u][m][q][half]);
                        a0[m] = ExpertOp<DT>::run(f0, b, a0[m]);
                        a1[m] = ExpertOp<DT>::run(f1, b, a1[m]);
                    }
            }
    };
    using First = std::integral_constant<int, 0>;
    using Second = std::integral_constant<int, 1>;
    if (groups > 0) load(First{}, 0);
    for (int g = 0; g < groups; g += 2) {
        if (g + 1 < groups) load(Second{}, g + 1);
        multiply(First{});
        if (g + 2 < groups) load(First{}, g + 2);
        if (g + 1 < groups) multiply(Second{});
    }
}

// The choices of the expert that workgroup row `slot` has, in order; how many (0: none, or another slot has them).
WQ8_DEVICE int find_pairs(const ExpertsArgs& p, int slot, uint16_t* list, int& expert) {
    const int pairs = p.tokens * p.top, lane = threadIdx.x & 63;
    const bool by_pair = pairs <= p.experts;  // fewer choices than experts: a slot a choice, the first of its expert serving all
    expert = by_pair ? p.ids[slot] : slot;
    if (uint32_t(expert) >= uint32_t(p.experts)) return 0;
    int count = 0;
    for (int base = 0; base < pairs; base += 64) {
        const bool mine = base + lane < pairs && p.ids[base + lane] == expert;
        const uint64_t mask = __ballot(mine);
        if (!mask) continue;
        if (by_pair && !count && base + __builtin_ctzll(mask) != slot) return 0;
        if (threadIdx.x < 64 && mine) list[count + __popcll(mask & ((uint64_t(1) << lane) - 1))] = uint16_t(base + lane);
        count += __popcll(mask);
    }
    return count;
}

// Four waves over two tiles of 16 rows: P tiles of 16 / P rows, 4 / P parts of the values, so that every output is a sum of four. red holds
// the waves' results of 16 / P tokens; the sum of row r, token t of the tile that begins at register `first` (0 or 4):
template <int P> WQ8_DEVICE float add_parts(const float (&red)[4][8][64], int r, int t, int first) {
    if constexpr (P == 1) {
        const int i = first + (r & 3), l = 16 * (r >> 2) + t;
        return ((red[0][i][l] + red[1][i][l]) + red[2][i][l]) + red[3][i][l];
    } else if constexpr (P == 2) {
        const int tile = r >> 3, i = first + (r & 3), l = 16 * ((r >> 2) & 1) + t;
        return ((red[tile][i][l] + red[tile][i][l + 40]) + red[tile + 2][i][l]) + red[tile + 2][i][l + 40];
    } else {
        const int tile = r >> 2, i = first + (r & 3);
        return ((red[tile][i][t] + red[tile][i][t + 20]) + red[tile][i][t + 40]) + red[tile][i][t + 60];
    }
}

// Rows row0 .. row0 + 15 and row1 .. row1 + 15 (none past `rows`) of an expert's weights on the tokens of `count` choices from `first` on;
// store(choice, r, sum of row0 + r, sum of row1 + r).
template <int DT, int P, int MT, int PLANES, typename Row, typename Store>
WQ8_DEVICE void expert_rows(const int8_t* weights, int row0, int row1, int rows, int width, int64_t plane, int first, int count, float (&red)[4][8][64],
                            const Row& token_row, const Store& store) {
    constexpr int R = 16 / P, STEP = 64 * P;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int tile = wave % P, part = wave / P, line = lane & 15;
    const int r = tile * R + line % R;
    const int8_t* w0 = weights + int64_t(min(row0 + r, rows - 1)) * width;
    const int8_t* w1 = weights + int64_t(min(row1 + r, rows - 1)) * width;
    const uint16_t* x[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) x[m] = token_row(min(first + 16 * m + line % R, count - 1));
    const int each = ((width + STEP - 1) / STEP + 4 / P - 1) / (4 / P);
    const int begin = part * each * STEP, end = min(width, begin + each * STEP);
    const int steps = end > begin ? (end - begin + STEP - 1) / STEP : 0;
    v4f a0[MT], a1[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) a0[m] = a1[m] = v4f{0, 0, 0, 0};
    constexpr int U = MT * PLANES == 1 ? 4 : MT * PLANES == 2 ? 2 : 1;
    stream_tiles<DT, P, MT, PLANES, U>(w0, w1, x, plane, begin + 16 * ((lane >> 4) + 4 * (line / R)), end, steps, a0, a1);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            red[wave][i][lane] = a0[m][i];
            red[wave][4 + i][lane] = a1[m][i];
        }
        __syncthreads();
        const int row = threadIdx.x & 15, t = threadIdx.x >> 4;
        if (t < R && first + 16 * m + t < count) store(first + 16 * m + t, row, add_parts<P>(red, row, t, 0), add_parts<P>(red, row, t, 4));
    }
}

template <int DT, int PLANES, typename Row, typename Store>
WQ8_DEVICE void expert_tokens(const int8_t* weights, int row0, int row1, int rows, int width, int64_t plane, int count, float (&red)[4][8][64], const Row& row,
                              const Store& store) {
    if (count <= 4) expert_rows<DT, 4, 1, PLANES>(weights, row0, row1, rows, width, plane, 0, count, red, row, store);
    else if (count <= 8) expert_rows<DT, 2, 1, PLANES>(weights, row0, row1, rows, width, plane, 0, count, red, row, store);
    else if (count <= 16) expert_rows<DT, 1, 1, PLANES>(weights, row0, row1, rows, width, plane, 0, count, red, row, store);
    else if (count <= 32) expert_rows<DT, 1, 2, PLANES>(weights, row0, row1, rows, width, plane, 0, count, red, row, store);
    else
        for (int first = 0; first < count; first += 64) expert_rows<DT, 1, 4, PLANES>(weights, row0, row1, rows, width, plane, first, count, red, row, store);
}

// gate and up of 16 hidden channels of an expert, and their product. Held as the sum of two BF16 values: FP16 would overflow where FP32 does
// not, and one rounding to 16 bits would add as much again to the output's error as the output's own.
template <int DT>
__global__ void __launch_bounds__(256, 2) experts_up(ExpertsArgs p) {
    __shared__ uint16_t list[MOST_PAIRS];
    __shared__ float red[4][8][64];
    const int blocks = p.hidden / 16, slot = blockIdx.x / blocks, f0 = (blockIdx.x % blocks) * 16;
    int expert;
    const int count = find_pairs(p, slot, list, expert);
    if (!count) return;
    __syncthreads();
    const float* scale = p.gate_up_scale + int64_t(expert) * 2 * p.hidden + f0;
    const int64_t plane = int64_t(p.tokens) * p.top * p.hidden;
    auto row = [&](int i) { return static_cast<const uint16_t*>(p.x) + int64_t(list[i] / p.top) * p.ldx; };
    auto store = [&](int i, int r, float gate, float up) {
        const float h = wq_swiglu(gate * scale[r], up * scale[p.hidden + r]);
        const uint16_t hi = Elem<DT_BF16>::from_f(h);
        const float back = Elem<DT_BF16>::to_f(hi);
        const int64_t at = int64_t(list[i]) * p.hidden + f0 + r;
        p.h[at] = hi;
        p.h[at + plane] = __builtin_isfinite(back) ? Elem<DT_BF16>::from_f(h - back) : uint16_t(0);
    };
    expert_tokens<DT, 1>(p.gate_up + int64_t(expert) * 2 * p.hidden * p.k, f0, p.hidden + f0, 2 * p.hidden, p.k, 0, count, red, row, store);
}

// 32 output channels of an expert for its choices, weighted.
__global__ void __launch_bounds__(256, 2) experts_down(ExpertsArgs p) {
    __shared__ uint16_t list[MOST_PAIRS];
    __shared__ float red[4][8][64];
    const int blocks = (p.k + 31) / 32, slot = blockIdx.x / blocks, n0 = (blockIdx.x % blocks) * 32;
    int expert;
    const int count = find_pairs(p, slot, list, expert);
    if (!count) return;
    __syncthreads();
    const float* scale = p.down_scale + int64_t(expert) * p.k + n0;
    const int64_t plane = int64_t(p.tokens) * p.top * p.hidden;
    auto row = [&](int i) { return p.h + int64_t(list[i]) * p.hidden; };
    auto store = [&](int i, int r, float a, float b) {
        const float weight = p.weights[list[i]];
        float* to = p.part + int64_t(list[i]) * p.k + n0 + r;
        to[0] = a * scale[r] * weight;
        if (n0 + 16 + r < p.k) to[16] = b * scale[16 + r] * weight;
    };
    expert_tokens<DT_BF16, 2>(p.down + int64_t(expert) * p.k * p.hidden, n0, n0 + 16, p.k, p.hidden, plane, count, red, row, store);
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
    const int pairs = tokens * top, slots = pairs <= experts ? pairs : experts;
    const int64_t h_bytes = (int64_t(pairs) * hidden * 4 + 255) / 256 * 256;
    if (int64_t(slots) * (hidden / 16) > MAX_BLOCKS_256 || int64_t(slots) * ((k + 31) / 32) > MAX_BLOCKS_256 || int64_t(tokens) * (k / 4) > MAX_BLOCKS_256 * 64) return -2;
    const ExpertsArgs p{x, static_cast<const int32_t*>(ids), weights, gate_up, gate_up_scale, down, down_scale, static_cast<uint16_t*>(workspace),
                        reinterpret_cast<float*>(static_cast<char*>(workspace) + h_bytes), residual, rscale, out, ldx, ldr, ldo, tokens, top, experts, k, hidden};
    if (dtype == DT_F16) experts_up<DT_F16><<<slots * (hidden / 16), 256, 0, stream>>>(p);
    else experts_up<DT_BF16><<<slots * (hidden / 16), 256, 0, stream>>>(p);
    if (const int rc = int(hipGetLastError())) return rc;
    experts_down<<<slots * ((k + 31) / 32), 256, 0, stream>>>(p);
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

// Rotary positions with one or several axes (time, height, width) on gfx950, for the rows of one projection in one launch.
//
// Pair i of a head turns by the angle 2 pi p u_i, p the token's position on the pair's axis, u_i = frequency_i / 2 pi turns:
//     (a, b) -> (a cos - b sin, a sin + b cos); the inverse (and the gradient) turns the other way.
// u_i comes as a 64-bit fixed-point fraction, the nearest to frequency_i / 2 pi, so p u_i modulo one turn is one wrapping integer
// product: within |p| 2^-65 turns, where a product in FP32 has lost the angle at p = 10^5 and one in FP64 costs a
// reduction. The top 32 bits give the quadrant and the rest of the turn, |r| <= 1/8, for two short polynomials.
#include "wq8_common.h"
#include "wq8_abi.h"
#include <algorithm>

namespace wq8 {

enum { ROTARY_MAX_TENSORS = 4, ROTARY_PAIRS = 0, ROTARY_HALVES = 1 };

struct RotaryTensor { const void* x; void* y; int64_t x_token, x_head, y_token, y_head; int first_head; };
struct RotaryArgs {
    RotaryTensor t[ROTARY_MAX_TENSORS];
    const void* positions;
    const uint64_t* turns;  // per pair: frequency / 2 pi, as a fraction of 2^64, modulo one
    const int* axis;        // per pair: its column of positions
    int64_t tokens, pos_token, pos_axis;
    int count, heads, pairs, head_dim, wide, inverse, heads_per_thread;
};

// sin and cos of 2 pi phase / 2^32. Polynomials in r^2 fitted for least maximum error on |r| <= 1/8 turn: with the coefficients in FP32
// off by 2.4e-8 (the rounding of 2 pi, half a step of FP32 of the sine) and 6.7e-9, evaluated in FP32 by 8.6e-8 and 5.8e-8.
WQ8_DEVICE void turn_sincos(uint32_t phase, float& s, float& c) {
    const uint32_t quadrant = (phase + 0x20000000u) >> 30;
    const float r = float(int32_t(phase - (quadrant << 30))) * 0x1p-32f, z = r * r;
    float ps = -0x1.2d9bb8p+6f;
    ps = __builtin_fmaf(ps, z, 0x1.465ec6p+6f);
    ps = __builtin_fmaf(ps, z, -0x1.4abbbap+5f);
    ps = __builtin_fmaf(ps, z, 0x1.921fb6p+2f);
    ps *= r;
    float pc = 0x1.d9c366p+5f;
    pc = __builtin_fmaf(pc, z, -0x1.55c57cp+6f);
    pc = __builtin_fmaf(pc, z, 0x1.03c1dcp+6f);
    pc = __builtin_fmaf(pc, z, -0x1.3bd3ccp+4f);
    pc = __builtin_fmaf(pc, z, 1.0f);
    const float a = quadrant & 1 ? pc : ps, b = quadrant & 1 ? ps : pc;
    s = quadrant & 2 ? -a : a;
    c = (quadrant + 1) & 2 ? -b : b;
}

template <typename T, int N> struct alignas(N * sizeof(T) > 16 ? 16 : N * sizeof(T)) Pack { T v[N]; };

// A unit is PP pairs: 2 PP consecutive channels (pairs style), or PP of each half (halves style); units past the rotated
// channels hold 2 PP channels that are copied. A thread computes its unit's angles once and applies them to
// heads_per_thread heads. Bound by HBM: 403 MB of a 32760-token latent in 82 us, 4.9 TB/s, a copy's rate; few tokens by three
// loads one after another (axis, position, and the frequency beside it: 4.8 us).
template <int DT, int STYLE, int PP>
__global__ void __launch_bounds__(256) rotary_rows(RotaryArgs p) {
    using raw = typename Elem<DT>::raw;
    using Side = Pack<raw, PP>;
    touch_arguments<RotaryArgs>();
    const int units = p.head_dim / (2 * PP), turning = p.pairs / PP;
    const int64_t index = blockIdx.x * int64_t(256) + threadIdx.x;
    const int64_t token = index / units;
    if (token >= p.tokens) return;
    const int unit = int(index - token * units);
    const bool turns = unit < turning;
    const int a0 = turns && STYLE == ROTARY_HALVES ? unit * PP : unit * 2 * PP;
    const int b0 = turns && STYLE == ROTARY_HALVES ? p.pairs + unit * PP : a0 + PP;
    const int first = blockIdx.y * p.heads_per_thread, last = min(p.heads, first + p.heads_per_thread);
    // a few heads at a time, their loads first; the first ones' before the angles
    constexpr int TOGETHER = 4;
    Side a[TOGETHER], b[TOGETHER];
    raw* y[TOGETHER];
    const auto load = [&](int h0) {
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) {
            const int h = min(h0 + n, last - 1);
            int which = 0;
            for (int t = 1; t < p.count; ++t) which = h >= p.t[t].first_head ? t : which;
            const RotaryTensor& t = p.t[which];
            const raw* x = static_cast<const raw*>(t.x) + token * t.x_token + (h - t.first_head) * t.x_head;
            y[n] = static_cast<raw*>(t.y) + token * t.y_token + (h - t.first_head) * t.y_head;
            a[n] = *reinterpret_cast<const Side*>(x + a0);
            b[n] = *reinterpret_cast<const Side*>(x + b0);
        }
    };
    load(first);
    float s[PP], c[PP];
    if (turns) {
#pragma unroll
        for (int j = 0; j < PP; ++j) {
            const int pair = unit * PP + j;
            const int64_t at = token * p.pos_token + p.axis[pair] * p.pos_axis;
            const int64_t position = p.wide ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
            turn_sincos(uint32_t((uint64_t(position) * p.turns[pair]) >> 32), s[j], c[j]);
            if (p.inverse) s[j] = -s[j];
        }
    }
    for (int h0 = first;;) {
#pragma unroll
        for (int n = 0; n < TOGETHER; ++n) {
            if (h0 + n >= last) break;
            if (turns) {
                raw in[2 * PP], out[2 * PP];
#pragma unroll
                for (int j = 0; j < PP; ++j) { in[j] = a[n].v[j]; in[PP + j] = b[n].v[j]; }
#pragma unroll
                for (int j = 0; j < PP; ++j) {
                    const int ia = STYLE == ROTARY_PAIRS ? 2 * j : j, ib = STYLE == ROTARY_PAIRS ? 2 * j + 1 : PP + j;
                    const float u = Elem<DT>::to_f(in[ia]), v = Elem<DT>::to_f(in[ib]);
                    out[ia] = Elem<DT>::from_f(__builtin_fmaf(u, c[j], -(v * s[j])));
                    out[ib] = Elem<DT>::from_f(__builtin_fmaf(u, s[j], v * c[j]));
                }
#pragma unroll
                for (int j = 0; j < PP; ++j) { a[n].v[j] = out[j]; b[n].v[j] = out[PP + j]; }
            }
            *reinterpret_cast<Side*>(y[n] + a0) = a[n];
            *reinterpret_cast<Side*>(y[n] + b0) = b[n];
        }
        h0 += TOGETHER;
        if (h0 >= last) break;
        load(h0);
    }
}

template <int DT, int STYLE> static int launch_rotary(RotaryArgs& p, hipStream_t stream) {
    // the widest unit that divides the rotated and the copied channels
    const int rest = p.head_dim - 2 * p.pairs;
    const auto fits = [&](int pp) { return p.pairs % pp == 0 && rest % (2 * pp) == 0; };
    const int pp = DT != DT_F32 && STYLE == ROTARY_HALVES && fits(8) ? 8 : fits(4) ? 4 : 1;
    const int64_t threads = p.tokens * (p.head_dim / (2 * pp));
    const int64_t blocks = (threads + 255) / 256;
    if (blocks > MAX_BLOCKS_256) return -2;
    // heads per thread: up to 24, while 2^17 threads remain (a 32760-token latent of 24 heads: 82 us with all of them in a thread, 86.5 with 8: the
    // angles are made once)
    p.heads_per_thread = int(std::min<int64_t>(24, std::max<int64_t>(1, threads * p.heads >> 17)));
    const dim3 grid(static_cast<unsigned>(blocks), (p.heads + p.heads_per_thread - 1) / p.heads_per_thread);
    if (pp == 8) {
        if constexpr (DT != DT_F32 && STYLE == ROTARY_HALVES) rotary_rows<DT, STYLE, 8><<<grid, 256, 0, stream>>>(p);
    } else if (pp == 4) {
        rotary_rows<DT, STYLE, 4><<<grid, 256, 0, stream>>>(p);
    } else {
        rotary_rows<DT, STYLE, 1><<<grid, 256, 0, stream>>>(p);
    }
    return int(hipGetLastError());
}

}  // namespace wq8

using namespace wq8;

WQ8_API int wq8_rotary(const void* const* xs, void* const* ys, const long long* shapes, int count, const void* positions, int64_t pos_token,
                       int64_t pos_axis, int wide, int64_t tokens, const long long* turns, const void* axis, int pairs, int head_dim, int style,
                       int inverse, int dtype, hipStream_t stream) {
    if (dtype < 0 || dtype > 2 || style < 0 || style > 1) return -1;
    if (count < 1 || count > ROTARY_MAX_TENSORS || tokens < 0 || pairs < 0 || head_dim < 8 || head_dim % 8 || 2 * pairs > head_dim) return -2;
    RotaryArgs p = {};
    for (int i = 0; i < count; ++i) {
        const long long* s = shapes + 5 * i;
        if (s[0] < 0 || s[0] > (1 << 20)) return -2;
        p.t[i] = {xs[i], ys[i], s[1], s[2], s[3], s[4], p.heads};
        p.heads += int(s[0]);
    }
    p.positions = positions; p.pos_token = pos_token; p.pos_axis = pos_axis; p.wide = wide;
    p.turns = reinterpret_cast<const uint64_t*>(turns); p.axis = static_cast<const int*>(axis);
    p.tokens = tokens; p.count = count; p.pairs = pairs; p.head_dim = head_dim; p.inverse = inverse;
    if (!tokens || !p.heads) return 0;
    if (style == ROTARY_PAIRS)
        return dtype == DT_F16 ? launch_rotary<DT_F16, ROTARY_PAIRS>(p, stream) : dtype == DT_BF16 ? launch_rotary<DT_BF16, ROTARY_PAIRS>(p, stream)
                                                                               : launch_rotary<DT_F32, ROTARY_PAIRS>(p, stream);
    return dtype == DT_F16 ? launch_rotary<DT_F16, ROTARY_HALVES>(p, stream) : dtype == DT_BF16 ? launch_rotary<DT_BF16, ROTARY_HALVES>(p, stream)
                                                                            : launch_rotary<DT_F32, ROTARY_HALVES>(p, stream);
}

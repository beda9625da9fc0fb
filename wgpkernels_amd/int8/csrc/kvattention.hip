// Attention over the paged 8-bit key/value cache on gfx950.
//
// Row (token t of request r, query head h) of D channels, on key/value head h / group:
//     s_j = scale q . k_j,   p_j = exp(s_j - max s) over the keys j that the row sees,   out = sum p_j v_j / sum p_j.
// The row stands at position lens[r] - new[r] + t; it sees the keys up to its own position (causal) or every key of the
// request, and with a window w those after position - w alone. A row that sees no key is zero; keys on pages outside the cache
// are hidden.
//
// Arithmetic. INT8 codes are exact in FP16, so both products run on the FP16 matrix cores with FP32 sums, and the pages' scales
// never touch a code:
// - Queries are FP16; BF16 ones are first scaled by a power of two of their row's largest value, which keeps their 8 bits exact down to
//   2^-32 of it.
// - t_j = log2(e) scale ks q . k_j + log2(vs), ks and vs the scales of j's page; w_j = 2^(t_j - m) is the row's weight times its value
//   scale, rounded once to FP16 for the second product; the sum of weights takes w_j / vs, in FP32 (a page of small values has weights
//   that FP16 does not hold), 16 keys of one page at a time. So weights are relative to the largest product of weight and scale, and one
//   page of large values does not cost the others. Where w_j may be below FP32's range and 2^(t_j - m) / vs is not, beside
//   a page whose values are 2^40 times as large, the sum takes exponentials of its own.
// - m follows the running maximum, and is left alone until a t_j would leave FP16's range, so that sums are rarely scaled again.
// - A value scale is taken as at least 2^-90: sums of weights, of up to 2^LAG 2^90 a key, stay in range over 2^22 keys of zeros. Pages of smaller
//   scales that are not zero count as that large: off by less than 2^-83.
//
// Work. A tile is ROWS rows (token, query head) of one request and key/value head, over the keys that they see together. The tiles of
// a launch stand in one line (request, head, tile), each as long as its keys (a window without causality apart, see span_of), and the
// workgroups, as many as the GPU holds at once, take equal lengths of it: whole tiles, and parts of the two at a share's ends, whose results
// kv_attention_join adds. So requests of any lengths fill the GPU evenly; and nothing is read on the host, each workgroup finds its share
// from the lengths on the GPU.
#include "wq8_common.h"
#include "wq8_abi.h"
#include <algorithm>
#include <type_traits>

namespace wq8 {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int FEW_ROWS = 16;  // rows of a tile of kv_attention_few

struct AttentionArgs {
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int *tables, *lens, *starts;
    int64_t table_stride, pages;
    int width, tokens, requests, heads, group, block_log2, causal, window;
    unsigned group_inverse;   // 2^32 / group, rounded down
    int few_rows, many_rows;  // the rows of a request that this launch serves: more than few_rows, up to many_rows
    int shares;               // workgroups that take a share (a multiple of 8)
    float scale;
    // workspace: per share the split tile that begins in it, {parts, first row, rows, first token} and its head; two partial results a share
    v4i* split_tiles;
    int* split_heads;
    float* slots;
};

// ---- shares --------------------------------------------------------------------------------------------------------
// A request's part of the line: tiles of length first + more * i, i = 0 to tiles - 1, for each head.
struct Span {
    int rows, tiles, first_token, past, total;
    int64_t first, more;
    WQ8_DEVICE int64_t upto(int64_t i) const { return first * i + more * (i * (i - 1) / 2); }
};

// What a tile costs besides its keys, in keys (six prompts of up to 1000 tokens: 84 us at 128, 79 at 256, 80 at 512).
constexpr int TILE_KEYS_OVERHEAD = 256;
// The line's units a key: shares are whole units, so that the ends of many drift from the tiles' by up to one each (one token over 8192 keys, 8
// heads: 17.5 us at 1, 14.9 at 16).
constexpr int UNITS = 16;

template <typename T> WQ8_DEVICE T scalar_load(const T* p) { return *(const __attribute__((address_space(4))) T*)(uint64_t)p; }

// UNIFORM: r is the same in every lane (scalar loads and arithmetic).
template <int ROWS, bool UNIFORM> WQ8_DEVICE Span span_of(const AttentionArgs& p, int r) {
    Span s = {};
    if (r >= p.requests) return s;
    const auto load = [](const int* at) { return UNIFORM ? scalar_load(at) : *at; };
    const int begin = min(max(load(p.starts + r), 0), p.tokens), end = min(max(load(p.starts + r + 1), begin), p.tokens);
    const int len = max(0, load(p.lens + r));
    const int64_t rows = int64_t(end - begin) * p.group;
    if (rows <= p.few_rows || rows > p.many_rows) return s;
    s.rows = int(rows);
    s.tiles = (s.rows + ROWS - 1) / ROWS;
    s.first_token = begin;
    s.past = len - (end - begin);  // a length below zero counts as zero keys: positions stay in range
    s.total = p.pages ? max(0, min(len, p.width << p.block_log2)) : 0;
    // lengths in keys * group * UNITS: a causal tile's rows see ROWS / group keys more than those of the tile before
    // With a window every tile counts as the window's keys. Without causality a tile sees to the request's end as well, and the shares of a request's
    // first tiles take longest (32760 rows over themselves, 8 heads of 128, a window of 1000: 3990 us, 4120 without the window; causal: 210).
    const bool grows = p.causal && !p.window;
    const int seen = p.window ? min(s.total, p.window) : p.causal ? min(s.total, max(0, s.past)) : s.total;
    s.first = (int64_t(seen + TILE_KEYS_OVERHEAD) * p.group + ROWS) * UNITS;
    s.more = grows ? ROWS * UNITS : 0;
    return s;
}

WQ8_DEVICE int by_group(const AttentionArgs& p, int row) {  // row / group
    const unsigned q = __umulhi(unsigned(row), p.group_inverse);
    return int(unsigned(row) - q * unsigned(p.group) >= unsigned(p.group) ? q + 1 : q);
}
// a / b to about 2^-22 of itself; a starting point for counting, the same in every workgroup
WQ8_DEVICE float ratio(int64_t a, int64_t b) { return float(a) * __builtin_amdgcn_rcpf(float(b)); }

// a / b, no less but by rounding up
WQ8_DEVICE int64_t no_less(int64_t a, int b) { return int64_t(float(a) * 0x1.00002p0f * __builtin_amdgcn_rcpf(float(b))) + 1; }

WQ8_DEVICE int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
WQ8_DEVICE int64_t uniform(int64_t v) { return int64_t(uint64_t(uint32_t(uniform(int(v >> 32)))) << 32 | uint32_t(uniform(int(v)))); }

// Over the first 256 threads.
WQ8_DEVICE int64_t scan256(int64_t v, int64_t* lds4, int64_t& total) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(v, d);
        if (int(threadIdx.x & 63) >= d) v += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63 && threadIdx.x < 256) lds4[threadIdx.x >> 6] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < int(threadIdx.x >> 6)) before += lds4[w];
        total += lds4[w];
    }
    return v + before;
}

// A workgroup's share [at, end) of the line, and the tile that stands at `at`.
struct Item { int request, row0, rows, first_token, head, past, total; int64_t line_begin, line_end; };
template <int ROWS> struct Share {
    const AttentionArgs& p;
    int64_t* lds4;
    int64_t* ends;     // where each of 256 requests ends in the line
    int64_t at, end, share, line;
    int64_t base_at;
    int base, index;
    bool rounded = false;  // tiles are whole shares long
    int64_t mine = 0;      // strip(): the length of a head of this thread's request
    int mine_tiles = 0;
    // where item() stands
    Span span;
    int64_t head_at;   // where the head's tiles begin
    int request, head, tile;
    bool found = false;

    // 256 requests from `first` on: spans a thread each, their ends in LDS
    WQ8_DEVICE int64_t strip(int first, int64_t before) {
        base = first;
        base_at = before;
        const Span s = span_of<ROWS, false>(p, threadIdx.x < 256 ? first + int(threadIdx.x) : p.requests);
        mine = s.upto(s.tiles);
        mine_tiles = s.tiles;
        int64_t total;
        const int64_t e = before + scan256(mine * p.heads, lds4, total);
        if (threadIdx.x < 256) ends[threadIdx.x] = e;
        __syncthreads();
        return before + total;
    }
    // Consecutive workgroups go round the 8 XCDs: each XCD takes a contiguous length of the line, whose tiles share keys and
    // values in its L2. A share is at least `least` keys.
    WQ8_DEVICE Share(const AttentionArgs& args, int64_t* scan, int64_t* request_ends, int least) : p(args), lds4(scan), ends(request_ends) {
        if (p.requests == 1) {
            span = span_of<ROWS, true>(p, 0);
            line = span.upto(span.tiles) * p.heads;
            base = 0;
            base_at = 0;
        } else {
            line = 0;
            for (int r = 0; r < p.requests; r += 256) line = strip(r, line);
            line = uniform(line);
        }
        // no less than line / shares
        const int64_t shortest = int64_t(least) * p.group * UNITS;
        share = uniform(max(no_less(line, p.shares), shortest));
        // One request: as many parts as that gives a tile (but for rounding), of equal length, so that no workgroup has parts of two (1 token over
        // 1000 keys: 16.4 us without, 13.3 with).
        if (p.requests == 1 && span.tiles == 1) {
            const int parts = min(int(ratio(span.first, share) + 0x1p-4f), int(unsigned(p.shares) / unsigned(p.heads)));
            if (parts > 0) share = uniform(no_less(span.first, parts));
        }
        // Few tiles of few rows, one a head: none shares a workgroup with another's part, as beginning a tile takes about as long as a share. Of three lengths
        // of a share, between those that suffice without and with a part more for each tile, the shortest that does. (16 requests of up to 2048
        // keys, 8 heads: 22 us without, 19 with; 8 of up to 5000: 24.2 and 21.6; 3 of up to 30000, 4 heads: 27.6 and 24.6; 32 of up to 3000, 8
        // heads: 32.4 and 29.1; four equal ones: 19.2 both. Tiles of many rows: 5-8% faster for 20 to 60 rows a request, 5-9% slower for 80 to 128, and so not done.)
        if (ROWS == FEW_ROWS && p.requests > 1 && p.requests <= 256 && p.requests * p.heads <= p.shares >> 1 && p.shares < 1 << 14) {
            const int tiles = p.requests * p.heads;
            int64_t lengths[3], counts = int64_t(mine_tiles > 1) << 48, total;
#pragma unroll
            for (int i = 0; i < 3; ++i) {
                lengths[i] = uniform(max(no_less(line, p.shares - tiles * i / 2), shortest));
                if (mine_tiles == 1) counts += int64_t(parts_of(mine, lengths[i]) * p.heads) << (16 * i);  // at most twice the shares in all
            }
            scan256(counts, lds4, total);
            total = uniform(total);
            if (!(total >> 48)) {
                rounded = true;
                share = int(total & 0xffff) <= p.shares ? lengths[0] : int(total >> 16 & 0xffff) <= p.shares ? lengths[1] : lengths[2];
                const int64_t e = scan256(mine_tiles ? parts_of(mine, share) * share * p.heads : 0, lds4, line);
                line = uniform(line);
                if (threadIdx.x < 256) ends[threadIdx.x] = e;
                __syncthreads();
            }
        }
        index = int(blockIdx.x & 7) * (p.shares >> 3) + int(blockIdx.x >> 3);
        at = index * share;
        end = min(line, at + share);
    }
    WQ8_DEVICE int parts_of(int64_t length, int64_t of) const { return max(1, int(ratio(length, of) + 0.9375f)); }
    // The tile at `at`: looked up the first time, and where a request ends; else the next tile.
    WQ8_DEVICE Item item() {
        if (found && ++tile == span.tiles) {
            tile = 0;
            head_at += span.upto(span.tiles);
            found = ++head < p.heads;
        }
        if (!found) look_up();
        found = true;
        return {request, tile * ROWS, span.rows, span.first_token, head, span.past, span.total, head_at + span.upto(tile), head_at + span.upto(tile + 1)};
    }
    WQ8_DEVICE void look_up() {
        int a = 0;
        int64_t begin = 0;
        if (p.requests > 1) {
            if (p.requests > 256) {
                int64_t upto = 0;
                for (int r = 0; r < p.requests; r += 256) {
                    __syncthreads();
                    upto = uniform(strip(r, upto));
                    if (at < upto) break;
                }
            }
            int b = min(256, p.requests - base) - 1;  // the first request that ends past `at`
            while (a < b) {
                const int m = (a + b) >> 1;
                if (uniform(ends[m]) > at) b = m; else a = m + 1;
            }
            begin = a ? uniform(ends[a - 1]) : base_at;
            span = span_of<ROWS, true>(p, uniform(base + a));
            if (rounded) span.first = uniform(parts_of(span.first, share)) * share;
        }
        request = uniform(base + a);
        const int64_t per_head = span.upto(span.tiles);
        int64_t in = at - begin;
        head = uniform(int(ratio(in, per_head)));
        while (head > 0 && in < head * per_head) --head;
        while (head + 1 < p.heads && in >= (head + 1) * per_head) ++head;
        in -= head * per_head;
        head_at = uniform(begin + head * per_head);
        tile = 0;
        if (span.tiles > 1) {
            if (span.more) {  // first i + more i (i - 1) / 2 <= in
                const float h = float(span.first) - 0.5f * float(span.more), m = float(span.more);
                tile = int((__builtin_amdgcn_sqrtf(__builtin_fmaf(h, h, 2.0f * m * float(in))) - h) * __builtin_amdgcn_rcpf(m));
            } else {
                tile = int(ratio(in, span.first));
            }
            tile = uniform(min(max(tile, 0), span.tiles - 1));
            while (tile > 0 && span.upto(tile) > in) --tile;
            while (tile + 1 < span.tiles && span.upto(tile + 1) <= in) ++tile;
        }
    }
    // Where this share's part of the item begins and ends in the line. A piece shorter than what beginning a tile costs, and than a sixteenth of
    // the tile and the share, is left to the share on the other side of its boundary, which finds the same (six prompts of up to 1000
    // tokens: 84 us with 1 / 128 of the tile and the share, 81 with this).
    WQ8_DEVICE int64_t snapped(const Item& it, int64_t x) const {
        const int64_t least = min(min(it.line_end - it.line_begin, share) >> 4, int64_t(TILE_KEYS_OVERHEAD) * p.group * UNITS);
        return x - it.line_begin < least ? it.line_begin : it.line_end - x < least ? it.line_end : x;
    }
    // Of `steps` steps of the item's keys, the ones before place x of the line: the same for the shares on both sides of x.
    WQ8_DEVICE int step_of(const Item& it, int64_t x, int steps) const {
        if (x <= it.line_begin) return 0;
        if (x >= it.line_end) return steps;
        return uniform(min(int(ratio(x - it.line_begin, it.line_end - it.line_begin) * float(steps)), steps));
    }
};

// Keys that the rows of tokens [first, last] see together: [low, high).
struct Keys { int low, high; };
WQ8_DEVICE Keys keys_of(const AttentionArgs& p, const Item& it, int first, int last) {
    Keys k;
    k.high = p.causal ? min(it.total, it.past + last + 1) : it.total;
    const int at = it.past + first;
    k.low = p.window && at >= p.window ? at - p.window + 1 : 0;
    k.high = max(k.high, 0);
    k.low = min(k.low, k.high);
    return k;
}

// ---- codes to FP16 -------------------------------------------------------------------------------------------------
// FP16 1024 + u has u in its low bits: a code's byte with its sign bit turned is u = code + 128; minus 1152.
WQ8_DEVICE uint32_t minus1152(uint32_t v) {
    const f16x2 r = __builtin_bit_cast(f16x2, v) + f16x2{_Float16(-1152.0f), _Float16(-1152.0f)};
    return __builtin_bit_cast(uint32_t, r);
}
// The four codes of a dword as FP16: .x codes 0, 1, .y codes 2, 3.
WQ8_DEVICE u32x2 codes4(uint32_t w) {
    w ^= 0x80808080u;
    return u32x2{minus1152(__builtin_amdgcn_perm(0x64646464u, w, 0x07010700u)), minus1152(__builtin_amdgcn_perm(0x64646464u, w, 0x07030702u))};
}
// Two dwords of four channels of keys a and b: per channel (a, b) as FP16.
WQ8_DEVICE void code_pairs(uint32_t a, uint32_t b, uint32_t* out) {
    const uint32_t low = __builtin_amdgcn_perm(b, a, 0x05040100u) ^ 0x80808080u, high = __builtin_amdgcn_perm(b, a, 0x07060302u) ^ 0x80808080u;
    out[0] = minus1152(low & 0x00ff00ffu | 0x64006400u);
    out[1] = minus1152(__builtin_amdgcn_perm(0x64646464u, low, 0x07030701u));
    out[2] = minus1152(high & 0x00ff00ffu | 0x64006400u);
    out[3] = minus1152(__builtin_amdgcn_perm(0x64646464u, high, 0x07030701u));
}

// ---- queries -------------------------------------------------------------------------------------------------------
// N vectors of 8 channels of a row: as they are in memory, and in FP16; the latter returns what a product with them is multiplied by. A
// lane holds part of a row: `most` gives the largest of its magnitudes over the row's lanes. A negative scale's sign goes to the queries, as
// the largest of scores is looked for before their product with the scale.
template <int N> WQ8_DEVICE void fetch_query(const uint16_t* row, int stride, bool live, u32x4* raw) {
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = live ? *reinterpret_cast<const u32x4*>(row + i * stride) : u32x4{0, 0, 0, 0};
}
template <int DT, int N, typename Most> WQ8_DEVICE float use_query(u32x4* raw, f16x8* out, float scale, Most most) {
    const uint32_t flip = scale < 0.0f ? 0x80008000u : 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] ^= u32x4{flip, flip, flip, flip};
    const float by = __builtin_fabsf(scale) * 0x1.715476p+0f;  // log2(e)
    if constexpr (DT == DT_F16) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __builtin_bit_cast(f16x8, raw[i]);
        return by;
    } else {
        uint32_t top = 0;  // magnitudes order as their bits do
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) top = max(top, max(raw[i][j] << 16 & 0x7fff0000u, raw[i][j] & 0x7fff0000u));
        top = most(top);
        // the largest magnitude to [2^14, 2^15); rows below 2^-112 keep that factor
        const uint32_t e = max(top >> 23, 15u);
        const float up = __builtin_bit_cast(float, (268u - e) << 23), down = __builtin_bit_cast(float, (e - 14u) << 23);
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                out[i][2 * j] = static_cast<_Float16>(__builtin_bit_cast(float, raw[i][j] << 16) * up);
                out[i][2 * j + 1] = static_cast<_Float16>(__builtin_bit_cast(float, raw[i][j] & 0xffff0000u) * up);
            }
        return down * by;
    }
}

// A page's scales as the weights take them.
struct PageScales { float k, log_v, inv_v; };
constexpr float LEAST_V = 0x1p-90f, FAR = 0x1p-40f;  // values this much smaller than others are far from them
WQ8_DEVICE PageScales page_scales(float ks, float vs, bool live) {
    const float v = fmaxf(vs, LEAST_V);
    return {live ? ks : 0.0f, live ? __builtin_amdgcn_logf(v) : -__builtin_inff(), 1.0f / v};
}

// Sums go from one maximum to a larger one by 2^down: in two steps, as a sum of weights may stay in range where 2^down does not.
struct Keep {
    float half;
    WQ8_DEVICE explicit Keep(float down) : half(__builtin_amdgcn_exp2f(0.5f * down)) {}
    template <typename T> WQ8_DEVICE T operator()(T v) const { return v * half * half; }
};

constexpr float LOWEST = -0x1p+120f;  // the running maximum before any key: below every t, and -inf - LOWEST = -inf
// Weights are taken relative to 2^-HEAD of the largest, and to that until one passes it by 2^LAG (FP16 ends at 2^16): small weights keep
// their bits down to 2^-21 of the largest.
constexpr float HEAD = 7.0f, LAG = 15.0f;

WQ8_DEVICE f16x8 weights8(const float* w) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = static_cast<_Float16>(w[j]);
    return r;
}

WQ8_DEVICE float finish(float acc, float mass) { return mass > 0.0f ? acc / mass : mass == 0.0f ? 0.0f : mass; }

// A tile's partial result: rows x D sums, then rows pairs (maximum, sum of weights).
// A share has two: 2 i for a tile that began in an earlier share, 2 i + 1 for one that goes on in a later one.
template <int ROWS, int D> WQ8_DEVICE float* slot_of(const AttentionArgs& p, int slot) { return p.slots + int64_t(slot) * (ROWS * (D + 2)); }

// A tile that begins in this share and goes on in later ones, for kv_attention_join.
template <int ROWS> WQ8_DEVICE void note_split(const AttentionArgs& p, const Share<ROWS>& share, const Item& it) {
    if (threadIdx.x) return;
    int last = int(ratio(it.line_end - 1, share.share));  // the share that its end is in
    while (int64_t(last) * share.share > it.line_end - 1) --last;
    while (int64_t(last + 1) * share.share <= it.line_end - 1) ++last;
    if (share.snapped(it, int64_t(last) * share.share) == it.line_end) --last;
    p.split_tiles[share.index] = v4i{last - share.index + 1, it.row0, it.rows, it.first_token};
    p.split_heads[share.index] = it.head;
}

// ---- tiles of many rows --------------------------------------------------------------------------------------------
// 32 rows a wave, 64 keys a step. S^T = K Q^T and O^T = V^T P^T on 32x32x16: a lane holds one row (lane % 32) and, of S^T, the keys
// 8 (i / 4) + 4 (lane / 32) + i % 4. With the second product's keys in that order a lane's weights are its operand as they are. The
// workgroup converts each step's codes once, into LDS in the operands' order (1 KB a fragment, 16 bytes a lane, swizzled so that the
// writes spread over the banks), in two buffers: while one is used, the next step's codes are on their way in registers. Wave w
// converts the 16 keys (of one page) 16 (w % 4) of every 64: with 8 waves the first four the values, the others the keys; with 4 waves
// each does both. The second four waves convert before their products, the first four after them, so that of a SIMD's two waves one mostly feeds
// the matrix cores while the other converts.
//
// What bounds it: the power limit, with the matrix cores busy 49% of 1.99 GHz (32760 rows over as many keys, 12 heads of 128: 6.2-6.7 ms,
// 980-1060 TFLOP/s, where a library product of 8192^3 reaches 1220-1270; a form before it was busy 45% of 2.12 GHz). A SIMD's vector work overlaps
// its matrix work by half (4 products and 32 FMAs on two waves: 66 and 72 ns alone, 104 together; exponentials fully), and 64 keys of 32 rows
// take 32 products, about 240 vector instructions and 32 exponentials. Tried and not faster: the first product of the next keys beside this
// softmax (in whole steps, and in halves of 32 keys), the two waves of a SIMD a barrier apart, wave priorities, accumulators in AGPRs, two waves
// for the rows of a tile that has at most half of them; slower: 64 rows a wave with one wave a SIMD (24%), codes converted between the first
// product's instructions (5-9%). Steps of 64 keys are equal but where the keys come from far (a frame of 1560 rows over 32760
// keys: 4% slower). Heads of 64 have half the products for the same vector work: 64 keys of 32 rows take as long.

WQ8_DEVICE float max3(float a, float b, float c) {  // without the quieting moves of fmaxf
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

template <int DT, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES, D == 256 ? 1 : 2) kv_attention_tiles(AttentionArgs p) {
    constexpr int ROWS = 32 * WAVES, KF = D / 16, KI = D / 64, VI = D == 256 ? 2 : 1, RAW = 8 * VI > 4 * KI ? 8 * VI : 4 * KI, SWZ = 256 / D;
    constexpr int SUBS = D == 128 ? 2 : 1, STEP_KEYS = 64 * SUBS, K_SUB = 2 * KF * 64, V_SUB = 4 * (D / 32) * 64;
    __shared__ u32x4 k_lds[2][SUBS * K_SUB];
    __shared__ u32x4 v_lds[2][SUBS * V_SUB];
    __shared__ v4f page_k[2][SUBS], page_log_v[2][SUBS], page_inv_v[2][SUBS];
    __shared__ float page_far[2][SUBS];
    __shared__ int64_t scan[4], ends[256];
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, half = lane >> 5, granule = wave & 3;
    const bool does_v = WAVES == 4 || wave < 4, does_k = WAVES == 4 || wave >= 4;
    touch_arguments<AttentionArgs>();
    Share<ROWS> share(p, scan, ends, 256);
    if (!tid) p.split_tiles[share.index][0] = 0;
    // lane constants: places of the codes in memory and LDS, of the operands
    const int v_half = D == 64 ? lane >> 4 : D == 128 ? lane >> 5 : 0, v_dw = D == 64 ? lane & 15 : D == 128 ? lane & 31 : lane;
    const int v_at = 4 * v_half * D + 4 * v_dw;
    const int v_entry = lane ^ (lane >> 3 & 3);
    const int block_mask = (1 << p.block_log2) - 1;
    const int64_t page_bytes = (int64_t(p.heads) << p.block_log2) * D;

    for (; share.at < share.end; __syncthreads()) {
        const Item it = share.item();
        const int64_t part0 = share.snapped(it, share.at), part1 = share.snapped(it, min(share.end, it.line_end));
        share.at = it.line_end;
        if (part0 >= part1) continue;
        // this lane's row
        const int row = it.row0 + 32 * wave + (lane & 31);
        const bool live_row = row < it.rows;
        const int token = by_group(p, min(row, it.rows - 1)), member = min(row, it.rows - 1) - token * p.group;
        u32x4 query_raw[KF];
        fetch_query<KF>(static_cast<const uint16_t*>(p.q) + (it.first_token + token) * p.q_token + (it.head * p.group + member) * p.q_head + 8 * half, 16,
                        live_row, query_raw);
        f16x8 query[KF];
        const float query_scale = use_query<DT, KF>(query_raw, query, p.scale, [](uint32_t t) {
            const LanePair o = swap32(__builtin_bit_cast(float, t));
            return max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
        });

        // keys: of the tile, of the part, and from the part's first on those of the wave and of the row
        Keys tile = keys_of(p, it, by_group(p, it.row0), by_group(p, min(it.row0 + ROWS, it.rows) - 1));
        tile.low &= ~(STEP_KEYS - 1);
        const int all_steps = (tile.high - tile.low + STEP_KEYS - 1) / STEP_KEYS, step0 = share.step_of(it, part0, all_steps);
        const int steps = share.step_of(it, part1, all_steps) - step0;
        const int key0 = tile.low + step0 * STEP_KEYS, key1 = min(tile.high, key0 + steps * STEP_KEYS);
        const bool began = part0 > it.line_begin, goes_on = part1 < it.line_end;
        const int wave_first = it.row0 + 32 * wave, wave_last = min(wave_first + 31, it.rows - 1);
        const Keys own = keys_of(p, it, token, token);
        const int first_at = by_group(p, min(wave_first, it.rows - 1)), last_at = by_group(p, wave_last);
        const Keys first = keys_of(p, it, first_at, first_at), last = keys_of(p, it, last_at, last_at);
        const int own_low = (own.low - key0) - 4 * half, own_high = (own.high - key0) - 4 * half;
        const int some_low = (first.low - key0), some_high = wave_first < it.rows ? (last.high - key0) : -(1 << 30);
        const int all_low = (last.low - key0), all_high = (first.high - key0);

        // This wave's 16 keys of every 64: their pages and scales come 64 at a time, one a lane (vector loads: scalar ones would be waited for
        // with every LDS read).
        const int* table = p.tables + it.request * p.table_stride;
        const int64_t head_bytes = (int64_t(it.head) << p.block_log2) * D;
        int page = 0;
        float seen = 0.0f;  // the largest value scale so far
        bool far = false;   // these 64 keys have a page far from it
        PageScales lane_scales = {};
        const auto load_pages = [&](int first) {  // of the 64 keys first, first + 1, ... of the part
            const int key = key0 + 64 * (first + lane) + 16 * granule;
            page = key < key1 ? table[key >> p.block_log2] : -1;
            const bool live = page >= 0 && page < p.pages;
            if (!live) page = 0;
            if (does_v) {
                const int64_t at = int64_t(page) * p.heads + it.head;
                const float ks = p.k_scales[at], vs = p.v_scales[at];
                float least = live ? vs : __builtin_inff(), most = live ? vs : 0.0f;
                if (p.block_log2 < 6) {  // the other waves' pages of the 64 keys too
                    int other[4];
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int at = key - 16 * granule + 16 * g;
                        other[g] = at < key1 ? table[at >> p.block_log2] : -1;
                    }
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const bool there = other[g] >= 0 && other[g] < p.pages;
                        const float v = p.v_scales[int64_t(there ? other[g] : 0) * p.heads + it.head];
                        least = fminf(least, there ? v : __builtin_inff());
                        most = fmaxf(most, there ? v : 0.0f);
                    }
                }
                seen = fmaxf(seen, wave_max(most));
                far = fmaxf(least, LEAST_V) < seen * FAR;
                lane_scales = page_scales(ks, vs, live);
            }
        };
        // codes on their way: with 8 waves a wave has keys or values, in the same registers
        constexpr bool BOTH = WAVES == 4;
        uint32_t v_raw[SUBS][RAW], own_k_raw[BOTH ? SUBS : 1][BOTH ? 4 * KI : 1];
        const auto k_raw = [&](int u, int i) -> uint32_t& {
            if constexpr (BOTH) return own_k_raw[u][i];
            else return v_raw[u][i];
        };
        const auto load_codes = [&](int step) {
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                const int n = step * SUBS + u;
                const int64_t at = __builtin_amdgcn_readlane(page, n & 63) * page_bytes + head_bytes + ((key0 + 64 * n + 16 * granule) & block_mask) * D;
                if (does_v) {
#pragma unroll
                    for (int i = 0; i < VI; ++i)
                        if (D > 64 || lane < 32)
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                v_raw[u][8 * i + j] = *reinterpret_cast<const uint32_t*>(p.v_codes + at + (v_at + 4 * i * D + (j < 4 ? j : j + 4) * D));
                }
                if (does_k) {
#pragma unroll
                    for (int i = 0; i < KI; ++i) {
                        const u32x4 raw = *reinterpret_cast<const u32x4*>(p.k_codes + at + (16 * lane + 1024 * i));
#pragma unroll
                        for (int j = 0; j < 4; ++j) k_raw(u, 4 * i + j) = raw[j];
                    }
                }
            }
        };
        const auto store_codes = [&](int step) {
            const int buffer = step & 1;
#pragma unroll
            for (int u = 0; u < SUBS; ++u) {
                if (does_v) {
#pragma unroll
                    for (int i = 0; i < VI; ++i) {
                        uint32_t pairs[4][4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) code_pairs(v_raw[u][8 * i + 2 * j], v_raw[u][8 * i + 2 * j + 1], pairs[j]);
                        u32x4* at = v_lds[buffer] + u * V_SUB + ((v_dw >> 3) * 4 + granule) * 64;
                        if (D > 64 || lane < 32)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                const int entry = 4 * (v_dw & 7) + c + 32 * (v_half + i);
                                at[entry ^ (entry >> 3 & 3) ^ (v_dw & 8)] = u32x4{pairs[0][c], pairs[1][c], pairs[2][c], pairs[3][c]};
                            }
                    }
                    if (lane == ((step * SUBS + u) & 63)) {
                        reinterpret_cast<float*>(&page_k[buffer][u])[granule] = lane_scales.k;
                        reinterpret_cast<float*>(&page_log_v[buffer][u])[granule] = lane_scales.log_v;
                        reinterpret_cast<float*>(&page_inv_v[buffer][u])[granule] = lane_scales.inv_v;
                        if (!granule) page_far[buffer][u] = far ? __builtin_inff() : LOWEST;
                    }
                }
                if (does_k) {
#pragma unroll
                    for (int i = 0; i < KI; ++i) {
                        const int unit = lane + 64 * i, key = unit / KF, chunk = unit % KF;
                        u32x4* at = k_lds[buffer] + u * K_SUB + ((granule >> 1) * KF + chunk) * 64;
                        const u32x2 a = codes4(k_raw(u, 4 * i)), b = codes4(k_raw(u, 4 * i + 1)), c = codes4(k_raw(u, 4 * i + 2)), d = codes4(k_raw(u, 4 * i + 3));
                        const int entry = (16 * (granule & 1) + key) ^ (SWZ * chunk & 15);
                        at[entry] = u32x4{a[0], a[1], b[0], b[1]};
                        at[entry + 32] = u32x4{c[0], c[1], d[0], d[1]};
                    }
                }
            }
        };

        float top = LOWEST, mass = 0.0f;
        v16f acc[D / 32];
#pragma unroll
        for (int i = 0; i < D / 32; ++i) acc[i] = v16f{};

        if (steps > 0) {
            load_pages(0);
            load_codes(0);
            store_codes(0);
            if (steps > 1) load_codes(1);
            __syncthreads();
        }
        for (int step = 0; step < steps; ++step) {
            const int buffer = step & 1;
            const auto next = [&] {
                if (step + 1 < steps) {
                    store_codes(step + 1);
                    if ((step + 2) * SUBS % 64 == 0) load_pages((step + 2) * SUBS);
                    if (step + 2 < steps) load_codes(step + 2);
                }
            };
            if (wave >= 4) next();
#pragma unroll 1
            for (int u = 0; u < SUBS; ++u) {
                const int base = step * STEP_KEYS + 64 * u;
                if (base >= some_high || base + 64 <= some_low) continue;
                // Stages of four matrix instructions, whose operands were read two stages before (an LDS read takes longer than four of
                // them): what is between two sched_barriers stays there.
                v16f s[2] = {};
                constexpr int FIRST = KF / 2, STAGES = FIRST + D / 32;
                f16x8 operands[3][4];
                const auto read = [&](int stage) {
                    if (stage >= STAGES) return;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (stage < FIRST) {
                            const int f = 2 * stage + i / 2, h = i % 2;
                            operands[stage % 3][i] = __builtin_bit_cast(f16x8, k_lds[buffer][u * K_SUB + (h * KF + f) * 64 + (lane ^ (SWZ * f & 15))]);
                        } else {
                            const int c = (4 * (stage - FIRST) + i) % (D / 32), g = (4 * (stage - FIRST) + i) / (D / 32);
                            operands[stage % 3][i] = __builtin_bit_cast(f16x8, v_lds[buffer][u * V_SUB + (c * 4 + g) * 64 + (v_entry ^ (8 * (c & 1)))]);
                        }
                    }
                };
                read(0);
                read(1);
#pragma unroll
                for (int stage = 0; stage < FIRST; ++stage) {
                    read(stage + 2);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        s[i % 2] = __builtin_amdgcn_mfma_f32_32x32x16_f16(operands[stage % 3][i], query[2 * stage + i / 2], s[i % 2], 0, 0, 0);
                }
                // t = a s + b of the 16 keys of a page
                v4f a = page_k[buffer][u] * query_scale, b = page_log_v[buffer][u];
                v4f inv_v = page_inv_v[buffer][u];
                const float some_far = page_far[buffer][u];
                if (base + 64 > all_high || base < all_low) {  // some row does not see every key of the step
                    const int high = own_high - base, low = own_low - base;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int key = 32 * h + 8 * (i / 4) + i % 4, g = 2 * h + i / 8;
                            s[h][i] = key >= high || key < low ? -__builtin_inff() : __builtin_fmaf(s[h][i], a[g], b[g]);
                        }
                    a = v4f{1.0f, 1.0f, 1.0f, 1.0f};
                    b = v4f{};
                }
                float high = LOWEST;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const v16f& t = s[g >> 1];
                    const int i = 8 * (g & 1);
                    const float m = max3(max3(t[i], t[i + 1], t[i + 2]), max3(t[i + 3], t[i + 4], t[i + 5]), max3(t[i + 6], t[i + 7], t[i + 7]));
                    high = fmaxf(high, __builtin_fmaf(m, a[g], b[g]));
                }
                if (__ballot(fmaxf(high, some_far) > top + LAG)) {
                    const LanePair o = swap32(high);
                    const float next_top = fmaxf(top, fmaxf(o.a, o.b) - HEAD);
                    const Keep keep(top - next_top);
                    top = next_top;
                    mass = keep(mass);
#pragma unroll
                    for (int i = 0; i < D / 32; ++i) acc[i] = keep(acc[i]);
                    if (some_far > 0.0f) {
#pragma unroll
                        for (int g = 0; g < 4; ++g) {
                            const float up = b[g] - top + __builtin_amdgcn_logf(inv_v[g]);
#pragma unroll
                            for (int i = 0; i < 8; ++i) mass += __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + i], a[g], up));
                        }
                        inv_v = v4f{};
                    }
                }
                b -= top;
                const auto weights_of = [&](int g) {
                    float w[8], sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        w[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[g >> 1][8 * (g & 1) + i], a[g], b[g]));
                        sum += w[i];
                    }
                    mass = __builtin_fmaf(sum, inv_v[g], mass);
                    return weights8(w);
                };
                constexpr int PER = D / 128 ? D / 128 : 1, WIDE = 4 / (D / 32) ? 4 / (D / 32) : 1;  // stages a page, pages a stage
                f16x8 weights[WIDE], next_weights[WIDE];
#pragma unroll
                for (int i = 0; i < WIDE; ++i) weights[i] = weights_of(i);
#pragma unroll
                for (int stage = FIRST; stage < STAGES; ++stage) {
                    read(stage + 2);
                    __builtin_amdgcn_sched_barrier(0);
                    const int done = stage - FIRST + 1;
                    const bool turn = done % PER == 0 && done < D / 32;  // the next stage takes other pages' weights
                    if (turn)
#pragma unroll
                        for (int i = 0; i < WIDE; ++i) next_weights[i] = weights_of(done / PER * WIDE + i);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int c = (4 * (done - 1) + i) % (D / 32), g = (4 * (done - 1) + i) / (D / 32);
                        acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(operands[stage % 3][i], weights[g % WIDE], acc[c], 0, 0, 0);
                    }
                    if (turn)
#pragma unroll
                        for (int i = 0; i < WIDE; ++i) weights[i] = next_weights[i];
                }
            }
            if (wave < 4) next();
            __syncthreads();
        }

        const LanePair both = swap32(mass);
        mass = both.a + both.b;
        if (began || goes_on) {
            float* slot = slot_of<ROWS, D>(p, 2 * share.index + !began);
            const int r = 32 * wave + (lane & 31);
            if (live_row) {
#pragma unroll
                for (int c = 0; c < D / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        *reinterpret_cast<v4f*>(slot + r * D + 32 * c + 8 * i + 4 * half) = v4f{acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]};
                if (!half) {
                    slot[ROWS * D + 2 * r] = top;
                    slot[ROWS * D + 2 * r + 1] = mass;
                }
            }
            if (!began) note_split(p, share, it);
        } else if (live_row) {
            uint16_t* out = static_cast<uint16_t*>(p.out) + (it.first_token + token) * p.out_token + (it.head * p.group + member) * p.out_head;
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint16_t o[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[j] = Elem<DT>::from_f(finish(acc[c][4 * i + j], mass));
                    *reinterpret_cast<u32x2*>(out + 32 * c + 8 * i + 4 * half) = u32x2{o[0] | uint32_t(o[1]) << 16, o[2] | uint32_t(o[3]) << 16};
                }
        }
    }
}

// ---- tiles of few rows ---------------------------------------------------------------------------------------------
// 16 rows; each of the 4 waves takes every fourth step of 32 keys by itself, straight from memory to registers, on 16x16x32: a lane
// holds one row (lane % 16). Keys: a lane loads D / 4 consecutive channels of key lane % 16 (the product's channels in that
// order for keys and queries alike). Values: a lane loads D / 16 channels of the 8 keys that the weights' layout gives it,
// 16 b + 4 (lane / 16) + i, and transposes them in registers. Pages and scales come 64 granules of 16 keys at a time, one a
// lane. The waves' sums are joined in LDS.
// What bounds it: HBM (64 requests of up to 8192 keys, 545 MB of codes: 110 us, 4.95 TB/s, a 1 GiB copy's rate); for one request the time
// besides its keys (32760 keys, 8 heads: 17.4 us, of which the codes take 9 to 10; finding the share, the first loads and the join of the
// waves are about 8).
constexpr int FEW_KEYS = 32;

template <int DT, int D>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) kv_attention_few(AttentionArgs p) {
    constexpr int KF = D / 32, KV = D / 64, VF = D / 16, VW = D / 64;  // fragments; 16-byte loads of K a lane; dwords of V a key
    __shared__ __align__(16) float sums[4][FEW_ROWS][D + 4];
    __shared__ float tops[4][FEW_ROWS], masses[4][FEW_ROWS];
    __shared__ int64_t scan[4], ends[256];
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, quarter = lane >> 4;
    touch_arguments<AttentionArgs>();
    Share<FEW_ROWS> share(p, scan, ends, 8 * FEW_KEYS);
    if (!tid) p.split_tiles[share.index][0] = 0;
    for (; share.at < share.end; __syncthreads()) {
    const Item it = share.item();
    const int64_t part0 = share.snapped(it, share.at), part1 = share.snapped(it, min(share.end, it.line_end));
    share.at = it.line_end;
    if (part0 >= part1) continue;
    const int row = it.row0 + (lane & 15);
    const bool live_row = row < it.rows;
    const int token = by_group(p, min(row, it.rows - 1)), member = min(row, it.rows - 1) - token * p.group;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + (it.first_token + token) * p.q_token + (it.head * p.group + member) * p.q_head;
    u32x4 query_raw[KF];  // on their way while the first codes are asked for
    fetch_query<KF>(q + D / 4 * quarter, 8, live_row, query_raw);

    const int last_row = min(it.row0 + FEW_ROWS, it.rows) - 1;
    const int first_token = by_group(p, it.row0), last_token = by_group(p, last_row);
    Keys tile = keys_of(p, it, first_token, last_token);
    tile.low &= ~(FEW_KEYS - 1);
    const int all_steps = (tile.high - tile.low + FEW_KEYS - 1) / FEW_KEYS, step0 = share.step_of(it, part0, all_steps);
    const int key0 = tile.low + step0 * FEW_KEYS, key1 = min(tile.high, tile.low + share.step_of(it, part1, all_steps) * FEW_KEYS);
    const bool began = part0 > it.line_begin, goes_on = part1 < it.line_end;
    const Keys own = keys_of(p, it, token, token);
    const Keys first = keys_of(p, it, first_token, first_token), last = keys_of(p, it, last_token, last_token);

    const int* table = p.tables + it.request * p.table_stride;
    const int block_mask = (1 << p.block_log2) - 1;
    const int64_t page_bytes = (int64_t(p.heads) << p.block_log2) * D, head_bytes = (int64_t(it.head) << p.block_log2) * D;
    const int wave_key0 = key0 + wave * FEW_KEYS;
    const int steps = key1 > wave_key0 ? (key1 - wave_key0 + 4 * FEW_KEYS - 1) / (4 * FEW_KEYS) : 0;

    // granule i of the wave: keys wave_key0 + 128 (i / 2) + 16 (i % 2); a lane holds granule 64 n + lane
    int page = 0;
    bool live_page = false;
    float ks = 0.0f, vs = 0.0f, log_v = 0.0f, inv_v = 0.0f, seen = 0.0f;
    int far = 0;
    const auto load_granules = [&](int step) {
        const int key = wave_key0 + 4 * FEW_KEYS * (step + (lane >> 1)) + 16 * (lane & 1);
        page = key < key1 ? table[key >> p.block_log2] : -1;
        live_page = page >= 0 && page < p.pages;
        if (!live_page) page = 0;
        const int64_t at = int64_t(page) * p.heads + it.head;
        ks = p.k_scales[at];
        vs = p.v_scales[at];
    };
    const auto use_granules = [&] {
        seen = fmaxf(seen, wave_max(live_page ? vs : 0.0f));
        far = live_page && fmaxf(vs, LEAST_V) < seen * FAR;
        far |= __shfl_xor(far, 1);  // of the step's two granules
        const PageScales s = page_scales(ks, vs, live_page);
        ks = s.k;
        log_v = s.log_v;
        inv_v = s.inv_v;
    };
    const auto from_lane = [](float v, int from) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), from)); };

    struct Raw {  // a step on its way: its codes, and its pages' scales
        u32x4 k[2][KV];
        uint32_t v[8][VW];
        float scale[2], log_v[2], inv_v[2];
        int far;
    };
    const auto take_scales = [&](Raw& raw, int step) {
        raw.far = __builtin_amdgcn_readlane(far, 2 * (step & 31));
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int from = 2 * (step & 31) + b;
            raw.scale[b] = from_lane(ks, from);
            raw.log_v[b] = from_lane(log_v, from);
            raw.inv_v[b] = from_lane(inv_v, from);
        }
    };
    const auto load_codes = [&](Raw& raw, int step) {
        const int key = wave_key0 + 4 * FEW_KEYS * step;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t at = __builtin_amdgcn_readlane(page, 2 * (step & 31) + b) * page_bytes + head_bytes + ((key + 16 * b) & block_mask) * D;
            const int8_t* k = p.k_codes + at + (lane & 15) * D + D / 4 * quarter;
#pragma unroll
            for (int i = 0; i < KV; ++i) raw.k[b][i] = reinterpret_cast<const u32x4*>(k)[i];
            const int8_t* v = p.v_codes + at + 4 * quarter * D + D / 16 * (lane & 15);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < VW; ++j) raw.v[4 * b + i][j] = reinterpret_cast<const uint32_t*>(v + i * D)[j];
        }
    };

    float top = LOWEST, mass = 0.0f;
    v4f acc[VF];
#pragma unroll
    for (int i = 0; i < VF; ++i) acc[i] = v4f{};
    f16x8 query[KF];
    float query_scale = 0.0f;
    const auto take_step = [&](Raw& raw, int step) {
        const int key = wave_key0 + 4 * FEW_KEYS * step;
        // this step's operands out of the raw registers, then the loads of the step after the next
        f16x8 k[2][KF], v[VF];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int f = 0; f < KF; ++f) {
                const u32x2 a = codes4(raw.k[b][f >> 1][2 * (f & 1)]), c = codes4(raw.k[b][f >> 1][2 * (f & 1) + 1]);
                k[b][f] = __builtin_bit_cast(f16x8, u32x4{a[0], a[1], c[0], c[1]});
            }
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            uint32_t pairs[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) code_pairs(raw.v[2 * i][j], raw.v[2 * i + 1][j], pairs[i]);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * j + c] = __builtin_bit_cast(f16x8, u32x4{pairs[0][c], pairs[1][c], pairs[2][c], pairs[3][c]});
        }
        const float scale[2] = {raw.scale[0], raw.scale[1]}, page_log_v[2] = {raw.log_v[0], raw.log_v[1]};
        float page_inv_v[2] = {raw.inv_v[0], raw.inv_v[1]};
        const int some_far = raw.far;
        if (step + 2 < steps) {
            const bool turn = ((step + 2) & 31) == 0;
            if (turn) load_granules(step + 2);
            load_codes(raw, step + 2);
            if (turn) use_granules();
            take_scales(raw, step + 2);
        }
        float t[8];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            v4f s = {};
#pragma unroll
            for (int f = 0; f < KF; ++f) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b][f], query[f], s, 0, 0, 0);
            const float m = scale[b] * query_scale;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[4 * b + i] = __builtin_fmaf(s[i], m, page_log_v[b]);
        }
        if (key + FEW_KEYS > first.high || key + FEW_KEYS > key1 || key < last.low) {
            const int high = min(own.high, key1) - key - 4 * quarter, low = own.low - key - 4 * quarter;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = 16 * (i >> 2) + (i & 3);
                if (at >= high || at < low) t[i] = -__builtin_inff();
            }
        }
        float high = t[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) high = fmaxf(high, t[i]);
        if (__ballot(high > top + LAG) || some_far) {
            LanePair o = swap16(high);
            o = swap32(fmaxf(o.a, o.b));
            const float next = fmaxf(top, fmaxf(o.a, o.b) - HEAD);
            const Keep keep(top - next);
            top = next;
            mass = keep(mass);
#pragma unroll
            for (int i = 0; i < VF; ++i) acc[i] = keep(acc[i]);
            if (some_far) {
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const float up = __builtin_amdgcn_logf(page_inv_v[b]) - top;
#pragma unroll
                    for (int i = 0; i < 4; ++i) mass += __builtin_amdgcn_exp2f(t[4 * b + i] + up);
                    page_inv_v[b] = 0.0f;
                }
            }
        }
        float w[8];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                w[4 * b + i] = __builtin_amdgcn_exp2f(t[4 * b + i] - top);
                sum += w[4 * b + i];
            }
            mass = __builtin_fmaf(sum, page_inv_v[b], mass);
        }
        const f16x8 weights = weights8(w);
#pragma unroll
        for (int i = 0; i < VF; ++i) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[i], weights, acc[i], 0, 0, 0);
    };
    Raw even, odd;
    if (steps) {
        load_granules(0);
        load_codes(even, 0);
        if (steps > 1) load_codes(odd, 1);
        query_scale = use_query<DT, KF>(query_raw, query, p.scale, [](uint32_t t) {
            LanePair o = swap16(__builtin_bit_cast(float, t));
            t = max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
            o = swap32(__builtin_bit_cast(float, t));
            return max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
        });
        use_granules();
        take_scales(even, 0);
        take_scales(odd, 1);
    }
    for (int step = 0; step < steps; step += 2) {
        take_step(even, step);
        if (step + 1 < steps) take_step(odd, step + 1);
    }
    mass = add_xor32(add_xor16(mass));
    // a lane's sums: channels D / 4 * quarter + D / 16 * i + j of its row, i = 0-3, j = fragment
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < VF; j += 4)
            *reinterpret_cast<v4f*>(&sums[wave][lane & 15][D / 4 * quarter + VF * i + j]) = v4f{acc[j][i], acc[j + 1][i], acc[j + 2][i], acc[j + 3][i]};
    if (!quarter) {
        tops[wave][lane] = top;
        masses[wave][lane] = mass;
    }
    __syncthreads();
    // 16 threads a row, D / 16 channels each
    const int r = tid >> 4, c0 = (tid & 15) * (D / 16);
    const float most = fmaxf(fmaxf(tops[0][r], tops[1][r]), fmaxf(tops[2][r], tops[3][r]));
    float total = 0.0f, o[D / 16] = {};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const Keep keep(tops[w][r] - most);
        total += keep(masses[w][r]);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[j] = __builtin_fmaf(sums[w][r][c0 + j], keep(1.0f), o[j]);
    }
    const int out_row = it.row0 + r;
    if (began || goes_on) {
        float* slot = slot_of<FEW_ROWS, D>(p, 2 * share.index + !began);
        if (out_row < it.rows) {
#pragma unroll
            for (int j = 0; j < D / 16; j += 4) *reinterpret_cast<v4f*>(slot + r * D + c0 + j) = v4f{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if (!(tid & 15)) {
                slot[FEW_ROWS * D + 2 * r] = most;
                slot[FEW_ROWS * D + 2 * r + 1] = total;
            }
        }
        if (!began) note_split(p, share, it);
    } else if (out_row < it.rows) {
    const int out_token = by_group(p, out_row), out_member = out_row - out_token * p.group;
    uint16_t* out = static_cast<uint16_t*>(p.out) + (it.first_token + out_token) * p.out_token + (it.head * p.group + out_member) * p.out_head + c0;
#pragma unroll
    for (int j = 0; j < D / 16; j += 4) {
        uint16_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = Elem<DT>::from_f(finish(o[j + i], total));
        *reinterpret_cast<u32x2*>(out + j) = u32x2{e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16};
    }
    }
    }
}

// ---- parts joined --------------------------------------------------------------------------------------------------
// Adds the parts of a split tile: D / 4 lanes a row, GROUPS of them that each take every GROUPS-th part, with the loads of several parts on
// their way at a time; the groups' sums are added in an order of their own, the same every time. A workgroup has as many rows as that
// takes of 256 lanes (at 32 parts of 80 rows 63 us became 58 for the whole call with this many workgroups and 16 parts at a time; most
// tiles come apart into two or three, for which four at a time are faster, 77 us against 82 for six prompts of up to 1000 tokens).
template <int DT, int ROWS, int D, int GROUPS>
__global__ void __launch_bounds__(256) kv_attention_join(AttentionArgs p) {
    constexpr int LANES = D / 4, AT_ONCE = 256 / (LANES * GROUPS);
    touch_arguments<AttentionArgs>();
    const v4i tile = scalar_load(p.split_tiles + blockIdx.x);
    const int head = scalar_load(p.split_heads + blockIdx.x), parts = tile[0];
    const int c = 4 * (threadIdx.x % LANES), group = threadIdx.x / LANES % GROUPS;
    const int r = blockIdx.y * AT_ONCE + threadIdx.x / (LANES * GROUPS), row = tile[1] + r;
    if (parts < 2 || r >= ROWS || row >= tile[2]) return;  // whole waves
    float top = LOWEST, mass = 0.0f;
    v4f acc = {};
    const auto add = [&](auto at_a_time) {
        constexpr int U = decltype(at_a_time)::value;
        for (int base = group; base < parts; base += GROUPS * U) {
            v4f x[U];
            float t[U], m[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int part = min(base + u * GROUPS, parts - 1);
                const float* slot = slot_of<ROWS, D>(p, 2 * (int(blockIdx.x) + part) + !part);
                x[u] = *reinterpret_cast<const v4f*>(slot + r * D + c);
                t[u] = slot[ROWS * D + 2 * r];
                m[u] = slot[ROWS * D + 2 * r + 1];
            }
            float next = top;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (base + u * GROUPS >= parts) t[u] = -__builtin_inff();
                next = fmaxf(next, t[u]);
            }
            const Keep keep(top - next);
            top = next;
            mass = keep(mass);
            acc = keep(acc);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const Keep part(t[u] - next);
                mass += part(m[u]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(x[u][j], part(1.0f), acc[j]);
            }
        }
    };
    if (parts <= 4) add(std::integral_constant<int, 4 / GROUPS ? 4 / GROUPS : 1>());
    else add(std::integral_constant<int, 16>());
#pragma unroll
    for (int d = LANES; d < LANES * GROUPS; d <<= 1) {
        const float other = __shfl_xor(top, d), next = fmaxf(top, other);
        const Keep keep(top - next), take(other - next);
        mass = keep(mass) + take(__shfl_xor(mass, d));
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = __builtin_fmaf(acc[j], keep(1.0f), __shfl_xor(acc[j], d) * take(1.0f));
        top = next;
    }
    if (group) return;
    const int token = by_group(p, row), member = row - token * p.group;
    uint16_t* out = static_cast<uint16_t*>(p.out) + (tile[3] + token) * p.out_token + (head * p.group + member) * p.out_head + c;
    uint16_t o[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) o[j] = Elem<DT>::from_f(finish(acc[j], mass));
    *reinterpret_cast<u32x2*>(out) = u32x2{o[0] | uint32_t(o[1]) << 16, o[2] | uint32_t(o[3]) << 16};
}

// ---- launches ------------------------------------------------------------------------------------------------------
// Which launches serve a call, and their workspaces: [0] requests of up to `limit` rows on tiles of 16, [1] the others on tiles of 32 rows
// a wave.
struct Launches {
    bool used[2];
    int limit, shares[2], waves, few_rows;
    int64_t bytes[2];
};

static int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

static Launches plan_launches(int64_t tokens, int64_t requests, int64_t heads, int64_t group, int head_dim, int sms) {
    Launches l = {};
    const int64_t rows = tokens * group;
    // A request's rows are known on the GPU alone. On average up to 16 a request: all on the tiles of few rows; more than 64: all on
    // the others (each launch is about 5 us, used or not); between, each request by its rows. The average is right for requests alike; beside a
    // prompt, single tokens take a tile of 256 rows each: 63 of them over up to 8192 keys (8 heads of 128, group 8) 132 us, a prompt of 4096
    // tokens 349, all in one call 674; with one of 1000 tokens 126, 65 and 386. 255 single tokens over up to 4096 keys (group 1) 222, a prompt
    // of 3000 83, both on the tiles of few rows 278.
    l.limit = 32;
    l.used[1] = requests == 1 ? rows > l.limit : rows > FEW_ROWS * requests;
    l.used[0] = !l.used[1] || (requests > 1 && rows <= 64 * requests);
    if (!l.used[1]) l.limit = 0x7fffffff;
    if (!l.used[0]) l.limit = 0;
    l.few_rows = int(std::min<int64_t>(rows, FEW_ROWS));
    l.waves = head_dim == 256 ? 4 : 8;
    // Two workgroups a CU on the tiles of few rows hide more of the time that a tile takes besides its keys, where there are as many tiles as CUs (64
    // requests of up to 8192 keys, 8 heads: 119.5 us against 122.6); with fewer they are twice the parts to begin and to join (1 token over
    // 32760 keys, 8 heads: 28 us against 22; 16 requests of up to 2048: 21.1 and 19.1; but 8 of up to 30000: 58.4 and 60.2).
    const int64_t few_tiles = (rows / FEW_ROWS + std::min(tokens, requests)) * heads;
    const int per_cu[2] = {few_tiles >= sms ? 2 : 1, 1}, tile_rows[2] = {FEW_ROWS, 32 * l.waves};
    for (int i = 0; i < 2; ++i) {
        l.shares[i] = (per_cu[i] * sms + 7) & ~7;
        if (l.used[i]) l.bytes[i] = align256(int64_t(l.shares[i]) * 20) + align256(int64_t(l.shares[i]) * 2 * tile_rows[i] * (head_dim + 2) * 4);
    }
    return l;
}

template <int DT, int D> static int launch_attention(AttentionArgs p, const Launches& l, char* workspace, hipStream_t stream) {
    for (int i = 0; i < 2; ++i) {
        if (!l.used[i]) continue;
        p.few_rows = i ? l.limit : 0;
        p.many_rows = i ? 0x7fffffff : l.limit;
        p.shares = l.shares[i];
        char* at = workspace + (i ? l.bytes[0] : 0);
        p.split_tiles = reinterpret_cast<v4i*>(at);
        p.split_heads = reinterpret_cast<int*>(p.split_tiles + p.shares);
        p.slots = reinterpret_cast<float*>(at + align256(int64_t(p.shares) * 20));
        if (i) {
            constexpr int WAVES = D == 256 ? 4 : 8;
            kv_attention_tiles<DT, D, WAVES><<<p.shares, 64 * WAVES, 0, stream>>>(p);
            kv_attention_join<DT, 32 * WAVES, D, 1><<<dim3(p.shares, 32 * WAVES * D / 1024), 256, 0, stream>>>(p);
        } else {
            kv_attention_few<DT, D><<<p.shares, 256, 0, stream>>>(p);
            kv_attention_join<DT, FEW_ROWS, D, 256 / D><<<dim3(p.shares, (l.few_rows + 3) / 4), 256, 0, stream>>>(p);
        }
    }
    return int(hipGetLastError());
}

}  // namespace wq8

using namespace wq8;

WQ8_API void wq8_kv_attention_workspace(int tokens, int requests, int heads, int group, int head_dim, int sms, int64_t* sizes) {
    sizes[0] = sizes[1] = 0;
    if (tokens < 1 || requests < 1 || heads < 1 || group < 1) return;
    const Launches l = plan_launches(tokens, requests, heads, group, head_dim, sms);
    sizes[0] = l.bytes[0] + l.bytes[1];
}

WQ8_API int wq8_kv_attention(const void* q, void* out, const long long* strides, const int8_t* k_codes, const float* k_scales, const int8_t* v_codes,
                             const float* v_scales, const void* tables, int64_t table_stride, int width, const void* lens, const void* starts, int tokens,
                             int requests, int heads, int group, int head_dim, int block, int64_t pages, float scale, int causal, int window, int dtype,
                             int sms, void* workspace, hipStream_t stream) {
    if (dtype != DT_F16 && dtype != DT_BF16) return -1;
    if (tokens < 0 || requests < 0 || heads < 1 || heads > 65535 || group < 1 || (head_dim != 64 && head_dim != 128 && head_dim != 256) ||
        (block != 16 && block != 32 && block != 64 && block != 128) || window < 0 || pages < 0 || pages > 0x7fffffff || width < 0 || sms < 1 || int64_t(width) * block > (1 << 30))
        return -2;
    if (!tokens || !requests) return 0;
    if (int64_t(tokens) * group > 0x7fffffff - 256) return -2;  // rows are counted in 32 bits
    const Launches l = plan_launches(tokens, requests, heads, group, head_dim, sms);
    if ((l.bytes[0] + l.bytes[1] && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 16) return -2;
    AttentionArgs p = {};
    p.q = q; p.out = out;
    p.q_token = strides[0]; p.q_head = strides[1]; p.out_token = strides[2]; p.out_head = strides[3];
    p.k_codes = k_codes; p.k_scales = k_scales; p.v_codes = v_codes; p.v_scales = v_scales;
    p.tables = static_cast<const int*>(tables); p.lens = static_cast<const int*>(lens); p.starts = static_cast<const int*>(starts);
    p.table_stride = table_stride; p.pages = pages; p.width = width; p.tokens = tokens; p.requests = requests; p.heads = heads; p.group = group;
    p.group_inverse = unsigned((uint64_t(1) << 32) / unsigned(group) - (group == 1));
    p.block_log2 = __builtin_ctz(block); p.causal = causal; p.window = window; p.scale = scale;
    char* ws = static_cast<char*>(workspace);
    const auto run = [&](auto dt, auto d) { return launch_attention<decltype(dt)::value, decltype(d)::value>(p, l, ws, stream); };
    const auto of_type = [&](auto dt) {
        return head_dim == 64 ? run(dt, std::integral_constant<int, 64>()) : head_dim == 128 ? run(dt, std::integral_constant<int, 128>())
                                                                                            : run(dt, std::integral_constant<int, 256>());
    };
    return dtype == DT_F16 ? of_type(std::integral_constant<int, DT_F16>()) : of_type(std::integral_constant<int, DT_BF16>());
}

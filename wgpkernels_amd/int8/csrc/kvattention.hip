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
//   scale, rounded once to FP16 for the second product; the sum of weights takes w_j / vs, in FP32, 16 keys (of one page) at a time.
//   So weights are relative to the largest product of weight and scale, and one page of large values does not cost the others.
// - m is the running maximum, left alone until a t_j passes it by more than 8 (2^8 is far from FP16's end), so that sums are
//   rarely scaled again.
// - A value scale is taken as at least 2^-40 of the largest seen before it (and 2^-100): sums of weights stay in range over pages of zeros.
//
// Work. A tile is ROWS rows (token, query head) of one request and key/value head; its keys are cut into `splits` parts where
// tiles alone would not fill the GPU, and kv_attention_join adds the parts. Which item a workgroup takes is found on the GPU, from the
// requests' lengths: nothing is read on the host.
#include "wq8_common.h"
#include "wq8_abi.h"
#include <algorithm>
#include <type_traits>

namespace wq8 {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

struct AttentionArgs {
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int *tables, *lens, *starts;
    int64_t table_stride, pages;
    int width, tokens, requests, heads, group, block_log2, causal, window;
    int few_rows, many_rows;  // the rows of a request that this launch serves: more than few_rows, up to many_rows
    int split_items;          // items wanted of a launch that may split keys; 0: whole keys
    int max_items;
    float scale;
    // workspace of a launch that may split keys: the number of tiles, per tile {first item, parts, first row, request} and its head, partial results
    int* tile_count;
    int4* tiles;
    int* tile_heads;
    float* slots;
};

// ---- which rows and keys -------------------------------------------------------------------------------------------
struct Span { int rows, tiles, first_token, tokens; int64_t past, total; int span; };

template <int ROWS> WQ8_DEVICE Span span_of(const AttentionArgs& p, int r) {
    Span s = {};
    if (r >= p.requests) return s;
    const int begin = min(max(p.starts[r], 0), p.tokens), end = min(max(p.starts[r + 1], begin), p.tokens);
    const int64_t len = p.lens[r];
    s.first_token = begin;
    s.tokens = end - begin;
    s.past = len - s.tokens;
    s.total = p.pages ? max(int64_t(0), min(len, int64_t(p.width) << p.block_log2)) : 0;
    const int64_t rows = int64_t(s.tokens) * p.group;
    if (rows > p.few_rows && rows <= p.many_rows) {
        s.rows = int(rows);
        s.tiles = (s.rows + ROWS - 1) / ROWS;
    }
    const int64_t most = p.window ? min(s.total, int64_t(p.window) + (ROWS + p.group - 1) / p.group + 64) : s.total;
    s.span = int(min(most, int64_t(0x7fffff00)));
    return s;
}

WQ8_DEVICE int scan256(int v, int* lds4, int& total) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(v, d);
        if (int(threadIdx.x & 63) >= d) v += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds4[threadIdx.x >> 6] = v;
    __syncthreads();
    int before = 0;
    total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < int(threadIdx.x >> 6)) before += lds4[w];
        total += lds4[w];
    }
    return v + before;
}

struct Item {
    int live, request, row0, rows, first_token, head, split, splits, tile_index, item;
    int64_t past, total;
};
WQ8_DEVICE int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
WQ8_DEVICE int64_t uniform(int64_t v) { return int64_t(uint64_t(uint32_t(uniform(int(v >> 32)))) << 32 | uint32_t(uniform(int(v)))); }

// Item number -> request, head, tile, part of its keys; in this order, parts innermost. Consecutive workgroups go round the 8
// XCDs: item numbers are dealt so that each XCD takes a contiguous range, whose tiles share keys and values in its L2.
template <int ROWS> WQ8_DEVICE Item find_item(const AttentionArgs& p) {
    __shared__ int lds4[4];
    __shared__ Item found;
    const int tid = threadIdx.x;
    int chunk = 0x7fffff00;
    if (p.split_items) {
        float work = 0.0f;
        for (int base = 0; base < p.requests; base += 256) {
            const Span s = span_of<ROWS>(p, base + tid);
            work += float(s.tiles) * float(s.span);
        }
        work = wave_sum(work);
        __shared__ float sums[4];
        if ((tid & 63) == 0) sums[tid >> 6] = work;
        __syncthreads();
        work = ((sums[0] + sums[1]) + sums[2]) + sums[3];
        // keys of a part: the work over the items wanted, at least 256
        chunk = int(fminf(fmaxf(work * float(p.heads) / float(p.split_items), 256.0f), 2.0e9f)) + 63 & ~63;
    }
    const auto count_of = [&](const Span& s, int& splits) {
        splits = max(1, (s.span + chunk - 1) / chunk);
        return s.tiles * p.heads * splits;
    };
    int all = 0, all_tiles = 0;
    for (int base = 0; base < p.requests; base += 256) {
        const Span s = span_of<ROWS>(p, base + tid);
        int splits, total;
        scan256(count_of(s, splits), lds4, total);
        all += total;
        if (p.split_items && !blockIdx.x) {
            scan256(s.tiles * p.heads, lds4, total);
            all_tiles += total;
        }
    }
    if (p.split_items && !blockIdx.x && !tid) *p.tile_count = all_tiles;
    const int per = (all + 7) >> 3, item = int(blockIdx.x & 7) * per + int(blockIdx.x >> 3);
    if (!tid) found.live = 0;
    int before = 0, tiles_before = 0;
    for (int base = 0; base < p.requests; base += 256) {
        const Span s = span_of<ROWS>(p, base + tid);
        int splits, total, total_tiles;
        const int count = count_of(s, splits);
        const int end = before + scan256(count, lds4, total);
        const int tiles_end = tiles_before + scan256(s.tiles * p.heads, lds4, total_tiles);
        if (item >= end - count && item < end && int(blockIdx.x >> 3) < per) {
            const int at = item - (end - count), tile = at / splits;
            found = {item < p.max_items, base + tid, tile % s.tiles * ROWS, s.rows, s.first_token, tile / s.tiles, at % splits, splits,
                     tiles_end - s.tiles * p.heads + tile, item, s.past, s.total};
        }
        before += total;
        tiles_before += total_tiles;
        if (item < before) break;
    }
    __syncthreads();
    return {uniform(found.live), uniform(found.request), uniform(found.row0), uniform(found.rows), uniform(found.first_token), uniform(found.head),
            uniform(found.split), uniform(found.splits), uniform(found.tile_index), uniform(found.item), uniform(found.past), uniform(found.total)};
}

// Where the parts of a tile are, for kv_attention_join: written by the tile's first part.
WQ8_DEVICE void note_tile(const AttentionArgs& p, const Item& it) {
    if (!p.split_items || threadIdx.x || it.split) return;
    p.tiles[it.tile_index] = int4{it.item, it.splits, it.row0, it.request};
    p.tile_heads[it.tile_index] = it.head;
}

// Keys that the rows of tokens [first, last] see together: [low, high); and this part of them.
struct Keys { int64_t low, high; };
WQ8_DEVICE Keys keys_of(const AttentionArgs& p, const Item& it, int64_t first, int64_t last) {
    Keys k;
    k.high = p.causal ? min(it.total, it.past + last + 1) : it.total;
    k.low = p.window ? max(int64_t(0), it.past + first - p.window + 1) : 0;
    if (k.high < k.low) k.high = k.low;
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
// N vectors of 8 channels of a row in FP16; returns what a product with them is multiplied by. A lane holds part of a row: `most`
// gives the largest of its magnitudes over the row's lanes.
template <int DT, int N, typename Most> WQ8_DEVICE float load_query(const uint16_t* row, int stride, bool live, f16x8* out, Most most) {
    u32x4 raw[N];
#pragma unroll
    for (int i = 0; i < N; ++i) raw[i] = live ? *reinterpret_cast<const u32x4*>(row + i * stride) : u32x4{0, 0, 0, 0};
    if constexpr (DT == DT_F16) {
#pragma unroll
        for (int i = 0; i < N; ++i) out[i] = __builtin_bit_cast(f16x8, raw[i]);
        return 1.0f;
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
        return down;
    }
}

// A page's scales as the weights take them. `seen`: the largest value scale so far.
struct PageScales { float k, log_v, inv_v; };
WQ8_DEVICE PageScales page_scales(float ks, float vs, float seen, bool live) {
    const float v = fmaxf(fmaxf(vs, seen * 0x1p-40f), 0x1p-100f);
    return {live ? ks : 0.0f, live ? __builtin_amdgcn_logf(v) : -__builtin_inff(), 1.0f / v};
}

constexpr float LOWEST = -0x1p+120f;  // the running maximum before any key: below every t, and -inf - LOWEST = -inf
constexpr float LAG = 8.0f;

WQ8_DEVICE f16x8 weights8(const float* w) {
    f16x8 r;
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        r[j] = static_cast<_Float16>(w[j]);
        r[j + 1] = static_cast<_Float16>(w[j + 1]);
    }
    return r;
}

WQ8_DEVICE float finish(float acc, float mass) { return mass > 0.0f ? acc / mass : mass == 0.0f ? 0.0f : mass; }

// A tile's partial result: rows x D sums, then rows pairs (maximum, sum of weights).
template <int ROWS, int D> WQ8_DEVICE float* slot_of(const AttentionArgs& p, int item) { return p.slots + int64_t(item) * (ROWS * (D + 2)); }

// ---- tiles of many rows --------------------------------------------------------------------------------------------
// 128 rows, 32 a wave, over 64 keys at a time. S^T = K Q^T and O^T = V^T P^T on 32x32x16: a lane holds one row (lane % 32) and, of S^T,
// the keys 8 (i / 4) + 4 (lane / 32) + i % 4. With the second product's keys in that order a lane's weights are its operand as they
// are. The workgroup converts each 64 keys once, into LDS in the operands' order (1 KB a fragment, 16 bytes a lane,
// swizzled so that the transposing writes spread over the banks), in two buffers: while one is used, the next keys' codes are on their way
// in registers.
constexpr int TILE_ROWS = 128, TILE_KEYS = 64;

template <int DT, int D>
__global__ void __launch_bounds__(256, D == 256 ? 1 : 2) kv_attention_tiles(AttentionArgs p) {
    constexpr int KF = D / 16, CH = D / 16, KC = TILE_KEYS * CH / 256, VD = D / 4, VG = 256 / VD, VC = VG < 8 ? 8 / VG : 1;
    constexpr int SWZ = D == 64 ? 2 : 1;
    __shared__ u32x4 k_lds[2][2 * KF * 64];
    __shared__ u32x4 v_lds[2][4 * (D / 32) * 64];
    __shared__ PageScales scales[2][4];
    const Item it = find_item<TILE_ROWS>(p);
    if (!it.live) return;
    note_tile(p, it);
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, half = lane >> 5;

    // this lane's row
    const int row = it.row0 + 32 * wave + (lane & 31);
    const bool live_row = row < it.rows;
    const int token = min(row, it.rows - 1) / p.group, member = min(row, it.rows - 1) - token * p.group;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + (it.first_token + token) * p.q_token + (it.head * p.group + member) * p.q_head;
    f16x8 query[KF];
    const float query_scale = load_query<DT, KF>(q + 8 * half, 16, live_row, query, [](uint32_t t) {
        const LanePair o = swap32(__builtin_bit_cast(float, t));
        return max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
    }) * p.scale * 0x1.715476p+0f;

    // keys: of the tile, of the part, of the wave, of the row
    const int last_row = min(it.row0 + TILE_ROWS, it.rows) - 1;
    Keys tile = keys_of(p, it, it.row0 / p.group, last_row / p.group);
    tile.low &= ~int64_t(TILE_KEYS - 1);
    const int64_t part = ((tile.high - tile.low + it.splits - 1) / it.splits + TILE_KEYS - 1) & ~int64_t(TILE_KEYS - 1);
    const int64_t key0 = tile.low + it.split * part, key1 = min(tile.high, key0 + part);
    const int steps = key1 > key0 ? int((key1 - key0 + TILE_KEYS - 1) / TILE_KEYS) : 0;
    const int wave_first = it.row0 + 32 * wave, wave_last = min(wave_first + 31, it.rows - 1);
    const bool live_wave = wave_first < it.rows;
    const Keys own = keys_of(p, it, token, token);
    const Keys first = keys_of(p, it, min(wave_first, it.rows - 1) / p.group, min(wave_first, it.rows - 1) / p.group);
    const Keys last = keys_of(p, it, wave_last / p.group, wave_last / p.group);

    // loads of a step: K chunks of 16 channels of a key, V dwords (4 channels) of the 8 keys of an operand
    const int* table = p.tables + it.request * p.table_stride;
    const int block_mask = (1 << p.block_log2) - 1;
    const int64_t page_bytes = (int64_t(p.heads) << p.block_log2) * D;
    const auto page_at = [&](int64_t key) -> int { return key < key1 ? table[key >> p.block_log2] : -1; };
    int k_page[KC], v_page[VC], s_page;
    u32x4 k_raw[KC];
    uint32_t v_raw[VC][8];
    float ks_raw, vs_raw;
    const int k_key = tid / CH, k_chunk = tid % CH, v_dw = tid % VD, v_group = tid / VD;
    const auto load_pages = [&](int step) {
        const int64_t base = key0 + int64_t(step) * TILE_KEYS;
#pragma unroll
        for (int i = 0; i < KC; ++i) k_page[i] = page_at(base + k_key + i * (256 / CH));
#pragma unroll
        for (int i = 0; i < VC; ++i) v_page[i] = page_at(base + (v_group + i * VG) / 2 * 16);
        s_page = page_at(base + (tid & 3) * 16);
    };
    bool s_live;
    const auto load_codes = [&](int step) {
        const int64_t base = key0 + int64_t(step) * TILE_KEYS;
        const auto row_of = [&](int page, int64_t key) {
            const int64_t at = page >= 0 && page < p.pages ? page : 0;
            return at * page_bytes + (int64_t(it.head) << p.block_log2) * D + int(key & block_mask) * D;
        };
#pragma unroll
        for (int i = 0; i < KC; ++i)
            k_raw[i] = *reinterpret_cast<const u32x4*>(p.k_codes + row_of(k_page[i], base + k_key + i * (256 / CH)) + 16 * k_chunk);
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            const int g = v_group + i * VG;
            if (VG > 8 && g >= 8) break;
            // operand keys 16 (g / 2) + 4 (g % 2) + {0-3, 8-11}
            const int8_t* at = p.v_codes + row_of(v_page[i], base + g / 2 * 16) + (g & 1) * 4 * D + 4 * v_dw;
#pragma unroll
            for (int j = 0; j < 8; ++j) v_raw[i][j] = *reinterpret_cast<const uint32_t*>(at + (j < 4 ? j : j + 4) * D);
        }
        s_live = s_page >= 0 && s_page < p.pages;
        const int64_t at = int64_t(s_live ? s_page : 0) * p.heads + it.head;
        ks_raw = p.k_scales[at];
        vs_raw = p.v_scales[at];
    };
    float seen = 0.0f;
    const auto store_codes = [&](int buffer) {
#pragma unroll
        for (int i = 0; i < KC; ++i) {
            const int key = k_key + i * (256 / CH);
            u32x4* at = k_lds[buffer] + ((key >> 5) * KF + k_chunk) * 64;
            const u32x2 a = codes4(k_raw[i][0]), b = codes4(k_raw[i][1]), c = codes4(k_raw[i][2]), d = codes4(k_raw[i][3]);
            const int entry = (key & 31) ^ (SWZ * k_chunk & 7);
            at[entry] = u32x4{a[0], a[1], b[0], b[1]};
            at[entry + 32] = u32x4{c[0], c[1], d[0], d[1]};
        }
#pragma unroll
        for (int i = 0; i < VC; ++i) {
            const int g = v_group + i * VG;
            if (VG > 8 && g >= 8) break;
            uint32_t pairs[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j) code_pairs(v_raw[i][2 * j], v_raw[i][2 * j + 1], pairs[j]);
            u32x4* at = v_lds[buffer] + ((v_dw >> 3) * 4 + (g >> 1)) * 64;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int entry = 4 * (v_dw & 7) + c + 32 * (g & 1);
                at[entry ^ (entry >> 3 & 3)] = u32x4{pairs[0][c], pairs[1][c], pairs[2][c], pairs[3][c]};
            }
        }
        const float v = s_live ? vs_raw : 0.0f;
        float top = fmaxf(v, lane_xor<1>(v));
        top = fmaxf(top, lane_xor<2>(top));
        seen = fmaxf(seen, top);
        if (tid < 4) scales[buffer][tid] = page_scales(ks_raw, vs_raw, seen, s_live);
    };

    float top = LOWEST, mass = 0.0f;
    v16f acc[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) acc[i] = v16f{};
    const int v_entry = lane ^ (lane >> 3 & 3);

    if (steps) {
        load_pages(0);
        load_codes(0);
        load_pages(1);
        store_codes(0);
        load_codes(1);
        load_pages(2);
        __syncthreads();
    }
    for (int step = 0; step < steps; ++step) {
        const int buffer = step & 1;
        const int64_t base = key0 + int64_t(step) * TILE_KEYS;
        if (live_wave && base < last.high && base + TILE_KEYS > first.low) {
            float t[2][16];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                v16f s = {};
#pragma unroll
                for (int f = 0; f < KF; ++f) {
                    const f16x8 k = __builtin_bit_cast(f16x8, k_lds[buffer][(b * KF + f) * 64 + (lane ^ (SWZ * f & 7))]);
                    s = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, query[f], s, 0, 0, 0);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) t[b][i] = s[i];
            }
            PageScales ps[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) ps[g] = scales[buffer][g];
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float k = ps[g].k * query_scale;
#pragma unroll
                for (int i = 0; i < 8; ++i) t[g >> 1][(g & 1) * 8 + i] = __builtin_fmaf(t[g >> 1][(g & 1) * 8 + i], k, ps[g].log_v);
            }
            if (base + TILE_KEYS > first.high || base < last.low) {  // some row does not see every key of the step
                const int high = int(min(own.high - base, int64_t(64))) - 4 * half, low = int(max(own.low - base, int64_t(-64))) - 4 * half;
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = 32 * b + 8 * (i / 4) + i % 4;
                        if (key >= high || key < low) t[b][i] = -__builtin_inff();
                    }
            }
            float high = t[0][0];
#pragma unroll
            for (int i = 1; i < 32; ++i) high = fmaxf(high, t[i >> 4][i & 15]);
            if (__ballot(high > top + LAG)) {
                const LanePair o = swap32(high);
                const float next = fmaxf(top, fmaxf(o.a, o.b)), keep = __builtin_amdgcn_exp2f(top - next);
                top = next;
                mass *= keep;
#pragma unroll
                for (int i = 0; i < D / 32; ++i) acc[i] *= keep;
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float w[8], sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    w[i] = __builtin_amdgcn_exp2f(t[g >> 1][(g & 1) * 8 + i] - top);
                    sum += w[i];
                }
                mass = __builtin_fmaf(sum, ps[g].inv_v, mass);
                const f16x8 weights = weights8(w);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    const f16x8 v = __builtin_bit_cast(f16x8, v_lds[buffer][(c * 4 + g) * 64 + v_entry]);
                    acc[c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, weights, acc[c], 0, 0, 0);
                }
            }
        }
        if (step + 1 < steps) {
            store_codes(buffer ^ 1);
            load_codes(step + 2);
            load_pages(step + 3);
        }
        __syncthreads();
    }

    const LanePair both = swap32(mass);
    mass = both.a + both.b;
    if (it.splits > 1) {
        float* slot = slot_of<TILE_ROWS, D>(p, it.item);
        const int r = 32 * wave + (lane & 31);
        if (live_row) {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<v4f*>(slot + r * D + 32 * c + 8 * i + 4 * half) = v4f{acc[c][4 * i], acc[c][4 * i + 1], acc[c][4 * i + 2], acc[c][4 * i + 3]};
            if (!half) {
                slot[TILE_ROWS * D + 2 * r] = top;
                slot[TILE_ROWS * D + 2 * r + 1] = mass;
            }
        }
        return;
    }
    if (!live_row) return;
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

// ---- tiles of few rows ---------------------------------------------------------------------------------------------
// 16 rows; each of the 4 waves takes every fourth step of 32 keys by itself, straight from memory to registers, on 16x16x32: a lane
// holds one row (lane % 16). Keys: a lane loads D / 4 consecutive channels of key lane % 16 (the product's channels in that
// order for keys and queries alike). Values: a lane loads D / 16 channels of the 8 keys that the weights' layout gives it,
// 16 b + 4 (lane / 16) + i, and transposes them in registers. Pages and scales come 64 granules of 16 keys at a time, one a
// lane. The waves' sums are joined in LDS.
constexpr int FEW_ROWS = 16, FEW_KEYS = 32;

template <int DT, int D>
__global__ void __launch_bounds__(256, 2) kv_attention_few(AttentionArgs p) {
    constexpr int KF = D / 32, KV = D / 64, VF = D / 16, VW = D / 64;  // fragments; 16-byte loads of K a lane; dwords of V a key
    __shared__ float sums[4][FEW_ROWS][D + 4];
    __shared__ float tops[4][FEW_ROWS], masses[4][FEW_ROWS];
    const Item it = find_item<FEW_ROWS>(p);
    if (!it.live) return;
    note_tile(p, it);
    const int tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63, quarter = lane >> 4;
    const int row = it.row0 + (lane & 15);
    const bool live_row = row < it.rows;
    const int token = min(row, it.rows - 1) / p.group, member = min(row, it.rows - 1) - token * p.group;
    const uint16_t* q = static_cast<const uint16_t*>(p.q) + (it.first_token + token) * p.q_token + (it.head * p.group + member) * p.q_head;
    f16x8 query[KF];
    const float query_scale = load_query<DT, KF>(q + D / 4 * quarter, 8, live_row, query, [](uint32_t t) {
        LanePair o = swap16(__builtin_bit_cast(float, t));
        t = max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
        o = swap32(__builtin_bit_cast(float, t));
        return max(__builtin_bit_cast(uint32_t, o.a), __builtin_bit_cast(uint32_t, o.b));
    }) * p.scale * 0x1.715476p+0f;

    const int last_row = min(it.row0 + FEW_ROWS, it.rows) - 1;
    const int64_t first_token = it.row0 / p.group, last_token = last_row / p.group;
    Keys tile = keys_of(p, it, first_token, last_token);
    tile.low &= ~int64_t(FEW_KEYS - 1);
    const int64_t part = ((tile.high - tile.low + it.splits - 1) / it.splits + 4 * FEW_KEYS - 1) & ~int64_t(4 * FEW_KEYS - 1);
    const int64_t key0 = tile.low + it.split * part, key1 = min(tile.high, key0 + part);
    const Keys own = keys_of(p, it, token, token);
    const Keys first = keys_of(p, it, first_token, first_token), last = keys_of(p, it, last_token, last_token);

    const int* table = p.tables + it.request * p.table_stride;
    const int block_mask = (1 << p.block_log2) - 1;
    const int64_t page_bytes = (int64_t(p.heads) << p.block_log2) * D, head_bytes = (int64_t(it.head) << p.block_log2) * D;
    const int64_t wave_key0 = key0 + wave * FEW_KEYS;
    const int steps = key1 > wave_key0 ? int((key1 - wave_key0 + 4 * FEW_KEYS - 1) / (4 * FEW_KEYS)) : 0;

    // granule i of the wave: keys wave_key0 + 128 (i / 2) + 16 (i % 2); a lane holds granule 64 n + lane
    int page = 0;
    float ks = 0.0f, log_v = 0.0f, inv_v = 0.0f, seen = 0.0f;
    const auto load_granules = [&](int step) {
        const int64_t key = wave_key0 + int64_t(4 * FEW_KEYS) * (step + (lane >> 1)) + 16 * (lane & 1);
        page = key < key1 ? table[key >> p.block_log2] : -1;
        const bool live = page >= 0 && page < p.pages;
        if (!live) page = 0;
        const int64_t at = int64_t(page) * p.heads + it.head;
        const float vs = live ? p.v_scales[at] : 0.0f;
        seen = fmaxf(seen, wave_max(vs));
        const PageScales s = page_scales(p.k_scales[at], vs, seen, live);
        ks = s.k;
        log_v = s.log_v;
        inv_v = s.inv_v;
    };
    const auto from_lane = [](float v, int from) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), from)); };

    u32x4 k_raw[2][KV];
    uint32_t v_raw[8][VW];
    const auto load_codes = [&](int step) {
        const int64_t key = wave_key0 + int64_t(4 * FEW_KEYS) * step;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int64_t at = __builtin_amdgcn_readlane(page, 2 * (step & 31) + b) * page_bytes + head_bytes + (int(key + 16 * b) & block_mask) * D;
            const int8_t* k = p.k_codes + at + (lane & 15) * D + D / 4 * quarter;
#pragma unroll
            for (int i = 0; i < KV; ++i) k_raw[b][i] = reinterpret_cast<const u32x4*>(k)[i];
            const int8_t* v = p.v_codes + at + 4 * quarter * D + D / 16 * (lane & 15);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < VW; ++j) v_raw[4 * b + i][j] = reinterpret_cast<const uint32_t*>(v + i * D)[j];
        }
    };

    float top = LOWEST, mass = 0.0f;
    v4f acc[VF];
#pragma unroll
    for (int i = 0; i < VF; ++i) acc[i] = v4f{};
    if (steps) {
        load_granules(0);
        load_codes(0);
    }
    for (int step = 0; step < steps; ++step) {
        const int64_t key = wave_key0 + int64_t(4 * FEW_KEYS) * step;
        // this step's operands out of the raw registers, then the next step's loads
        f16x8 k[2][KF], v[VF];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int f = 0; f < KF; ++f) {
                const u32x2 a = codes4(k_raw[b][f >> 1][2 * (f & 1)]), c = codes4(k_raw[b][f >> 1][2 * (f & 1) + 1]);
                k[b][f] = __builtin_bit_cast(f16x8, u32x4{a[0], a[1], c[0], c[1]});
            }
#pragma unroll
        for (int j = 0; j < VW; ++j) {
            uint32_t pairs[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) code_pairs(v_raw[2 * i][j], v_raw[2 * i + 1][j], pairs[i]);
#pragma unroll
            for (int c = 0; c < 4; ++c) v[4 * j + c] = __builtin_bit_cast(f16x8, u32x4{pairs[0][c], pairs[1][c], pairs[2][c], pairs[3][c]});
        }
        float page_k[2], page_log_v[2], page_inv_v[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int from = 2 * (step & 31) + b;
            page_k[b] = from_lane(ks, from);
            page_log_v[b] = from_lane(log_v, from);
            page_inv_v[b] = from_lane(inv_v, from);
        }
        if (step + 1 < steps) {
            if (((step + 1) & 31) == 0) load_granules(step + 1);
            load_codes(step + 1);
        }
        float t[8];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            v4f s = {};
#pragma unroll
            for (int f = 0; f < KF; ++f) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[b][f], query[f], s, 0, 0, 0);
            const float m = page_k[b] * query_scale;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[4 * b + i] = __builtin_fmaf(s[i], m, page_log_v[b]);
        }
        if (key + FEW_KEYS > first.high || key + FEW_KEYS > key1 || key < last.low) {
            const int high = int(min(min(own.high, key1) - key, int64_t(64))) - 4 * quarter, low = int(max(own.low - key, int64_t(-64))) - 4 * quarter;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int at = 16 * (i >> 2) + (i & 3);
                if (at >= high || at < low) t[i] = -__builtin_inff();
            }
        }
        float high = t[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) high = fmaxf(high, t[i]);
        if (__ballot(high > top + LAG)) {
            LanePair o = swap16(high);
            o = swap32(fmaxf(o.a, o.b));
            const float next = fmaxf(top, fmaxf(o.a, o.b)), keep = __builtin_amdgcn_exp2f(top - next);
            top = next;
            mass *= keep;
#pragma unroll
            for (int i = 0; i < VF; ++i) acc[i] *= keep;
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
    }
    mass = add_xor32(add_xor16(mass));
    // a lane's sums: channels D / 4 * quarter + D / 16 * i + j of its row, i = 0-3, j = fragment
#pragma unroll
    for (int j = 0; j < VF; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sums[wave][lane & 15][D / 4 * quarter + VF * i + j] = acc[j][i];
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
        const float keep = __builtin_amdgcn_exp2f(tops[w][r] - most);
        total = __builtin_fmaf(masses[w][r], keep, total);
#pragma unroll
        for (int j = 0; j < D / 16; ++j) o[j] = __builtin_fmaf(sums[w][r][c0 + j], keep, o[j]);
    }
    const int out_row = it.row0 + r;
    if (it.splits > 1) {
        float* slot = slot_of<FEW_ROWS, D>(p, it.item);
        if (out_row < it.rows) {
#pragma unroll
            for (int j = 0; j < D / 16; j += 4) *reinterpret_cast<v4f*>(slot + r * D + c0 + j) = v4f{o[j], o[j + 1], o[j + 2], o[j + 3]};
            if (!(tid & 15)) {
                slot[FEW_ROWS * D + 2 * r] = most;
                slot[FEW_ROWS * D + 2 * r + 1] = total;
            }
        }
        return;
    }
    if (out_row >= it.rows) return;
    const int out_token = out_row / p.group, out_member = out_row - out_token * p.group;
    uint16_t* out = static_cast<uint16_t*>(p.out) + (it.first_token + out_token) * p.out_token + (it.head * p.group + out_member) * p.out_head + c0;
#pragma unroll
    for (int j = 0; j < D / 16; j += 4) {
        uint16_t e[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) e[i] = Elem<DT>::from_f(finish(o[j + i], total));
        *reinterpret_cast<u32x2*>(out + j) = u32x2{e[0] | uint32_t(e[1]) << 16, e[2] | uint32_t(e[3]) << 16};
    }
}

// ---- parts joined --------------------------------------------------------------------------------------------------
// Adds the parts of a tile in order. WAVES waves a row (few rows in many parts: each takes every WAVES-th part, their sums then added
// in order), 4 / WAVES rows at a time.
template <int DT, int ROWS, int D, int ROWS_WG>
__global__ void __launch_bounds__(256) kv_attention_join(AttentionArgs p) {
    constexpr int WAVES = ROWS_WG == 1 ? 4 : 1, C = D / 64;
    __shared__ float sums[4][D], masses[4], tops[4];
    if (int(blockIdx.x) >= *p.tile_count) return;
    const int4 tile = p.tiles[blockIdx.x];
    const Span s = span_of<ROWS>(p, tile.w);
    const int wave = uniform(int(threadIdx.x) >> 6), lane = threadIdx.x & 63;
    if (tile.y <= 1) return;
    for (int i = WAVES == 4 ? 0 : wave; i < ROWS_WG; i += WAVES == 4 ? 1 : 4) {
        const int r = blockIdx.y * ROWS_WG + i, row = tile.z + r;
        if (row >= s.rows) return;
        const int part0 = WAVES == 4 ? wave : 0;
        float top = LOWEST;
        for (int part = part0; part < tile.y; part += WAVES) top = fmaxf(top, slot_of<ROWS, D>(p, tile.x + part)[ROWS * D + 2 * r]);
        float mass = 0.0f, acc[C] = {};
#pragma unroll 4
        for (int part = part0; part < tile.y; part += WAVES) {
            const float* slot = slot_of<ROWS, D>(p, tile.x + part);
            const float keep = __builtin_amdgcn_exp2f(slot[ROWS * D + 2 * r] - top);
            mass = __builtin_fmaf(slot[ROWS * D + 2 * r + 1], keep, mass);
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = __builtin_fmaf(slot[r * D + C * lane + c], keep, acc[c]);
        }
        if constexpr (WAVES == 4) {
#pragma unroll
            for (int c = 0; c < C; ++c) sums[wave][C * lane + c] = acc[c];
            if (!lane) {
                masses[wave] = mass;
                tops[wave] = top;
            }
            __syncthreads();
            if (wave) return;
            top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
            mass = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float keep = __builtin_amdgcn_exp2f(tops[w] - top);
                mass = __builtin_fmaf(masses[w], keep, mass);
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] = __builtin_fmaf(sums[w][C * lane + c], keep, acc[c]);
            }
        }
        const int token = row / p.group, member = row - token * p.group;
        uint16_t* out = static_cast<uint16_t*>(p.out) + (s.first_token + token) * p.out_token +
                        (p.tile_heads[blockIdx.x] * p.group + member) * p.out_head + C * lane;
#pragma unroll
        for (int c = 0; c < C; ++c) out[c] = Elem<DT>::from_f(finish(acc[c], mass));
    }
}

// ---- launches ------------------------------------------------------------------------------------------------------
// Which launches serve a call, and their workspaces: few: requests of up to `limit` rows on tiles of 16; many: the others on tiles of 128.
struct Launches {
    bool few, many;
    int limit;
    int64_t tiles[2];       // most tiles (of a request and head) of each
    int split_items[2];
    int64_t items[2], bytes[2];
};

static int64_t align256(int64_t v) { return (v + 255) & ~int64_t(255); }

static Launches plan_launches(int64_t tokens, int64_t requests, int64_t heads, int64_t group, int head_dim, int sms) {
    Launches l = {};
    const int64_t rows = tokens * group, live = std::min(tokens, requests);
    // A request's rows are known on the GPU alone. On average up to 16 a request: all on the tiles of few rows (one launch)
    l.limit = 32;
    l.many = requests == 1 ? rows > l.limit : rows > FEW_ROWS * requests;
    l.few = !l.many || requests > 1;
    if (!l.many) l.limit = 0x7fffffff;
    const int64_t most[2] = {l.many ? live * ((l.limit + FEW_ROWS - 1) / FEW_ROWS) : rows / FEW_ROWS + live, rows / TILE_ROWS + live};
    const int64_t wanted[2] = {8 * int64_t(sms), 2 * int64_t(sms)};
    const int tile_rows[2] = {FEW_ROWS, TILE_ROWS};
    for (int i = 0; i < 2; ++i) {
        l.tiles[i] = most[i] * heads;
        // parts of keys where tiles alone are too few for the GPU; tiles of few rows always, requests being of many lengths
        l.split_items[i] = i == 0 || l.tiles[i] < wanted[i] ? int(wanted[i]) : 0;
        l.items[i] = l.tiles[i] + (l.split_items[i] ? l.split_items[i] + 64 : 0);
        if ((i ? l.many : l.few) && l.split_items[i])
            l.bytes[i] = 256 + align256(l.tiles[i] * 20) + align256(l.items[i] * tile_rows[i] * (head_dim + 2) * 4);
    }
    return l;
}

template <int DT, int D> static int launch_attention(AttentionArgs p, const Launches& l, char* workspace, hipStream_t stream) {
    for (int i = 0; i < 2; ++i) {
        if (!(i ? l.many : l.few)) continue;
        p.few_rows = i ? l.limit : 0;
        p.many_rows = i ? 0x7fffffff : l.limit;
        p.split_items = l.split_items[i];
        p.max_items = int(l.items[i]);
        char* at = workspace + (i ? l.bytes[0] : 0);
        p.tile_count = reinterpret_cast<int*>(at);
        p.tiles = reinterpret_cast<int4*>(at + 256);
        p.tile_heads = reinterpret_cast<int*>(p.tiles + l.tiles[i]);
        p.slots = reinterpret_cast<float*>(at + 256 + align256(l.tiles[i] * 20));
        const unsigned grid = unsigned((l.items[i] + 7) & ~int64_t(7));
        if (i) kv_attention_tiles<DT, D><<<grid, 256, 0, stream>>>(p);
        else kv_attention_few<DT, D><<<grid, 256, 0, stream>>>(p);
        if (p.split_items) {
            if (i) kv_attention_join<DT, TILE_ROWS, D, 16><<<dim3(unsigned(l.tiles[i]), TILE_ROWS / 16), 256, 0, stream>>>(p);
            else kv_attention_join<DT, FEW_ROWS, D, 1><<<dim3(unsigned(l.tiles[i]), FEW_ROWS), 256, 0, stream>>>(p);
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
    if (tokens < 0 || requests < 0 || heads < 1 || group < 1 || (head_dim != 64 && head_dim != 128 && head_dim != 256) ||
        (block != 16 && block != 32 && block != 64 && block != 128) || window < 0 || pages < 0 || pages > 0x7fffffff || width < 0 || sms < 1)
        return -2;
    if (!tokens || !requests) return 0;
    // rows and items are counted in 32 bits
    if (int64_t(tokens) * group > 0x7fffffff - TILE_ROWS || (int64_t(tokens) * group / FEW_ROWS + requests) * heads > (1 << 30)) return -2;
    const Launches l = plan_launches(tokens, requests, heads, group, head_dim, sms);
    if ((l.bytes[0] + l.bytes[1] && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 16) return -2;
    AttentionArgs p = {};
    p.q = q; p.out = out;
    p.q_token = strides[0]; p.q_head = strides[1]; p.out_token = strides[2]; p.out_head = strides[3];
    p.k_codes = k_codes; p.k_scales = k_scales; p.v_codes = v_codes; p.v_scales = v_scales;
    p.tables = static_cast<const int*>(tables); p.lens = static_cast<const int*>(lens); p.starts = static_cast<const int*>(starts);
    p.table_stride = table_stride; p.pages = pages; p.width = width; p.tokens = tokens; p.requests = requests; p.heads = heads; p.group = group;
    p.block_log2 = __builtin_ctz(block); p.causal = causal; p.window = window; p.scale = scale;
    char* ws = static_cast<char*>(workspace);
    const auto run = [&](auto dt, auto d) { return launch_attention<decltype(dt)::value, decltype(d)::value>(p, l, ws, stream); };
    const auto of_type = [&](auto dt) {
        return head_dim == 64 ? run(dt, std::integral_constant<int, 64>()) : head_dim == 128 ? run(dt, std::integral_constant<int, 128>())
                                                                                            : run(dt, std::integral_constant<int, 256>());
    };
    return dtype == DT_F16 ? of_type(std::integral_constant<int, DT_F16>()) : of_type(std::integral_constant<int, DT_BF16>());
}

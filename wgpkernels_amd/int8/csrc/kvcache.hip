// The paged 8-bit key/value cache on gfx950: block tables and slots from request lengths, writes, and reads.
//
// Codes (pages, heads, block, head_dim) int8 and one FP32 scale per (page, head): value = code * scale, scale = amax / 127
// over the page's tokens. Slot s is token s % block of page s / block.
#include "wq8_common.h"
#include "wq8_abi.h"
#include <algorithm>
#include <type_traits>

namespace wq8 {

// ---- block tables and slots ----------------------------------------------------------------------------------------
struct PlanArgs {
    const int *past, *fresh, *pages, *used;
    int* tables;
    int64_t table_stride, tokens;
    int pages_count, requests, width, block;
    int64_t* slots;
    int *positions, *starts, *lens, *used_out, *missing;
};

WQ8_DEVICE int64_t scan256(int64_t v, int64_t* lds4, int64_t& total) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(v, d);
        if (int(threadIdx.x & 63) >= d) v += o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 63) lds4[threadIdx.x >> 6] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < 4; ++w) {
        if (w < int(threadIdx.x >> 6)) before += lds4[w];
        total += lds4[w];
    }
    return v + before;
}

// Pages in order of the free list: requests in order, each taking ceil((past + new) / block) - ceil(past / block). A request
// that the tokens, its table's width, 31-bit positions or the free pages cannot hold takes none; nor then does any later one that needs pages.
// Every workgroup walks the requests, 256 at a time, and serves PLAN_TOKENS tokens: the walk is a few hundred
// nanoseconds, less than a launch of its own. A page's first token writes its table entry. Bound by the latency of its loads: 4.6 us for 256
// requests of a token each, 7.1 us for 40 prompts of 54000 tokens together.
constexpr int PLAN_TOKENS = 1024;
__global__ void __launch_bounds__(256) kv_plan_tokens(PlanArgs p) {
    __shared__ int64_t lds4[4], ends[256];
    __shared__ int64_t source[256];  // free-list index of the request's first new page
    __shared__ int pasts[256], oks[256], haves[256];
    const int64_t t0 = blockIdx.x * int64_t(PLAN_TOKENS), t1 = min(p.tokens, t0 + PLAN_TOKENS);
    const int tid = threadIdx.x;
    const int64_t used = *p.used;
    int64_t upto_ends = 0, upto_need = 0, granted = 0, refused = 0;
    for (int base = 0; base < p.requests; base += 256) {
        const int r = base + tid;
        const bool live = r < p.requests;
        const int64_t past = live ? max(0, p.past[r]) : 0, fresh = live ? max(0, p.fresh[r]) : 0;
        const int64_t have = (past + p.block - 1) / p.block, want = (past + fresh + p.block - 1) / p.block;
        int64_t total;
        const int64_t end = upto_ends + scan256(fresh, lds4, total);
        const bool fits = live && want <= p.width && end <= p.tokens && past + fresh <= 0x7fffffff;
        const int64_t need = fits ? want - have : 0;
        int64_t total_need;
        const int64_t upto = upto_need + scan256(need, lds4, total_need);
        const bool ok = fits && (!need || (used + upto <= p.pages_count && used + upto - need >= 0));
        ends[tid] = end;
        source[tid] = used + upto - need;
        pasts[tid] = int(past);
        haves[tid] = int(have);
        oks[tid] = ok;
        __syncthreads();
        if (blockIdx.x == 0 && live) {
            if (!r) p.starts[0] = 0;
            p.starts[r + 1] = int(min(end, p.tokens));
            p.lens[r] = int(ok ? past + fresh : past);
            granted += ok ? need : 0;
            refused += !ok;
        }
        const int count = min(256, p.requests - base);
        const int64_t low = max(t0, upto_ends), high = min(t1, upto_ends + total);
        for (int64_t t = low + tid; t < high; t += 256) {
            int a = 0, b = count - 1;  // the first request whose end is past t
            while (a < b) {
                const int m = (a + b) >> 1;
                if (ends[m] > t) b = m; else a = m + 1;
            }
            const int64_t begin = a ? ends[a - 1] : upto_ends;
            const int64_t position = pasts[a] + (t - begin);
            int64_t slot = -1;
            if (oks[a]) {
                const int64_t column = position / p.block;
                int* entry = p.tables + (base + a) * p.table_stride + column;
                int page;
                if (column >= haves[a]) {
                    page = p.pages[source[a] + column - haves[a]];
                    if (position % p.block == 0) *entry = page;
                } else {
                    page = *entry;
                }
                slot = int64_t(page) * p.block + position % p.block;
            }
            p.slots[t] = slot;
            p.positions[t] = int(position);
        }
        upto_ends += total;
        upto_need += total_need;
        __syncthreads();
    }
    for (int64_t t = max(t0, upto_ends) + tid; t < t1; t += 256) {  // tokens of no request
        p.slots[t] = -1;
        p.positions[t] = 0;
    }
    if (blockIdx.x == 0) {
        int64_t total_granted, total_refused;
        scan256(granted, lds4, total_granted);
        scan256(refused, lds4, total_refused);
        if (!tid) {
            if (!p.requests) p.starts[0] = 0;
            *p.used_out = int(used + total_granted);
            *p.missing = int(total_refused);
        }
    }
}

// ---- writes --------------------------------------------------------------------------------------------------------
struct CacheArgs {
    const void* x[2];          // keys, values (token, head, channel)
    void* y[2];                // reads: outputs (token, head, channel), contiguous
    int64_t token_stride[2], head_stride[2];
    int8_t* codes[2];
    float* scales[2];
    const int64_t* slots;
    int* owner;
    int64_t tokens, all_slots;
    int heads, block_log2, head_dim, group, parts;  // group: tokens a workgroup looks through, parts: workgroups that share their pages (kv_write_owned)
};

// owner[slot] = the token written there. Nothing clears it: an entry holds if it names a token of this call whose slot it is,
// which an entry of another call only does where it happens to be right.
__global__ void __launch_bounds__(256) kv_owner(CacheArgs p) {
    const int64_t t = blockIdx.x * int64_t(256) + threadIdx.x;
    if (t >= p.tokens) return;
    const int64_t slot = p.slots[t];
    if (slot >= 0 && slot < p.all_slots) p.owner[slot] = int(t);
}

// A finite value for the cache: NaN counts as zero, infinities as the largest finite number (a few steps below it: 127 times the
// rounded scale has to stay finite), so that one bad token does not turn its page's other tokens into NaN.
WQ8_DEVICE float cached_value(float v) {
    constexpr float MOST = 0x1.fffff8p+127f;
    return v != v ? 0.0f : fminf(fmaxf(v, -MOST), MOST);
}

// round(v / scale) in the low byte, inv = 1 / scale: v * inv with one correction by the remainder, so that the quotient is within an ulp
// and codes differ from those of an exact division only where v lies within that of a tie (see divisor_of). |v / scale| <= 127 (1 + 2^-24), which
// rounds to 127. TINY: scales below 2^-120, whose inverse may overflow, divide.
template <bool TINY> WQ8_DEVICE int code_of(float v, float scale, float inv) {
    float q = v * inv;
    if constexpr (TINY) q = v / scale;
    else q = __builtin_fmaf(__builtin_fmaf(-q, scale, v), inv, q);
    return rne_low_byte(q);
}

// What a page's values are divided by. Of 16-bit values over the scale of a 16-bit maximum one kind comes within an ulp of a tie without being one
// (the others are 2^-11 and more away): half of the maximum, 63.5 but for the rounding of the scale. Where the scale was rounded up its code
// is 63, not the even 64 that an FP32 quotient of 63.5 rounds to: these pages divide by the next larger number.
template <int DT> WQ8_DEVICE float divisor_of(float scale) {
    if constexpr (DT == DT_F32) return scale;
    const float middle = 63.5f * scale, off = __builtin_fmaf(-63.5f, scale, Elem<DT>::to_f(Elem<DT>::from_f(middle)));
    return off < 0.0f && off >= -0x1p-23f * middle ? __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, scale) + 1) : scale;
}

// The low bytes of four words, by three byte permutations.
WQ8_DEVICE uint32_t pack_low_bytes(int a, int b, int c, int d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(uint32_t(d), uint32_t(c), 0x0c0c0400u), __builtin_amdgcn_perm(uint32_t(b), uint32_t(a), 0x0c0c0400u), 0x05040100u);
}

// The largest of the workgroup's bit patterns of magnitudes (they order as unsigned numbers, NaN above infinity).
WQ8_DEVICE uint32_t block_max_bits(uint32_t v, uint32_t* lds4) {
    v = __builtin_bit_cast(uint32_t, row16_max(__builtin_bit_cast(float, v)));
    const auto two = [](LanePair p) { return max(__builtin_bit_cast(uint32_t, p.a), __builtin_bit_cast(uint32_t, p.b)); };
    v = two(swap16(__builtin_bit_cast(float, v)));
    v = two(swap32(__builtin_bit_cast(float, v)));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds4[threadIdx.x >> 6] = v;
    __syncthreads();
    return max(max(lds4[0], lds4[1]), max(lds4[2], lds4[3]));
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// 8 consecutive channels as they are in memory.
template <int DT> struct Raw8 {
    u32x4 v[DT == DT_F32 ? 2 : 1];
    WQ8_DEVICE void load(const typename Elem<DT>::raw* p) {
        v[0] = reinterpret_cast<const u32x4*>(p)[0];
        if constexpr (DT == DT_F32) v[1] = reinterpret_cast<const u32x4*>(p)[1];
    }
    WQ8_DEVICE void zero() {
        v[0] = u32x4{0, 0, 0, 0};
        if constexpr (DT == DT_F32) v[1] = v[0];
    }
    template <bool FINITE> WQ8_DEVICE float value(int j) const {
        float f;
        if constexpr (DT == DT_F32) f = __builtin_bit_cast(float, uint32_t(v[j >> 2][j & 3]));
        else f = Elem<DT>::to_f(uint16_t(v[0][j >> 1] >> (16 * (j & 1))));
        return FINITE ? f : cached_value(f);
    }
    // the largest magnitude's bits so far: two 16-bit patterns in a word, or one of 32
    WQ8_DEVICE uint32_t larger(uint32_t top) const {
        if constexpr (DT == DT_F32) {
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, uint32_t(v[j >> 2][j & 3]) & 0x7fffffffu);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, top), __builtin_bit_cast(u16x2, uint32_t(v[0][j]) & 0x7fff7fffu)));
        }
        return top;
    }
    static constexpr uint32_t INFINITY_BITS = DT == DT_F32 ? 0x7f800000u : DT == DT_BF16 ? 0x7f80u : 0x7c00u;
    static WQ8_DEVICE float number(uint32_t bits) {
        if constexpr (DT == DT_F32) return __builtin_bit_cast(float, bits);
        else return Elem<DT>::to_f(uint16_t(bits));
    }
};

// One page and head: rows[] names the token of each of its slots that is written, -1 for the others. The scale becomes the larger
// of the held one (none when the page's first slot is written: the page begins anew) and the new tokens' amax / 127; tokens
// that the page held are coded again where it grew. NI: vectors of 8 channels a thread, kept in registers between the maximum and the
// codes (0: any number, read twice).
template <int DT, int NI> WQ8_DEVICE void write_page(const CacheArgs& p, int which, int64_t page, int head, const int* rows, uint32_t* lds4) {
    using raw = typename Elem<DT>::raw;
    const int block = 1 << p.block_log2, per_row = p.head_dim >> 3, items = block * per_row;
    const int row_step = 256 / per_row, chunk_step = 256 - row_step * per_row;
    const int row0 = int(threadIdx.x) / per_row, chunk0 = int(threadIdx.x) - row0 * per_row;
    const raw* x = static_cast<const raw*>(p.x[which]) + head * p.head_stride[which];
    float* held = p.scales[which] + page * p.heads + head;
    const float was = *held;
    Raw8<DT> kept[NI ? NI : 1];
    // the thread's vectors: (row, chunk) from (row0, chunk0) on, 256 vectors apart
    const auto each = [&](auto body) {
        int row = row0, chunk = chunk0;
        const auto step = [&](int n) {
            if (row < block) body(n, row, chunk);
            row += row_step;
            chunk += chunk_step;
            if (chunk >= per_row) { chunk -= per_row; ++row; }
        };
        if constexpr (NI > 0) {
#pragma unroll
            for (int n = 0; n < NI; ++n) step(n);
        } else {
            for (int i = threadIdx.x; i < items; i += 256) step(0);
        }
    };
    uint32_t top = 0;
    each([&](int n, int row, int chunk) {
        const int t = rows[row];
        if (t >= 0) kept[n].load(x + t * p.token_stride[which] + 8 * chunk);
        else kept[n].zero();
        if constexpr (!NI) top = kept[0].larger(top);
    });
    if constexpr (NI > 0) each([&](int n, int, int) { top = kept[n].larger(top); });
    if constexpr (DT != DT_F32) top = max(top & 0xffffu, top >> 16);
    top = uint32_t(__builtin_amdgcn_readfirstlane(int(block_max_bits(top, lds4))));
    const bool finite = top < Raw8<DT>::INFINITY_BITS;
    const float amax = finite ? Raw8<DT>::number(top) : 0.0f;
    const float old = rows[0] >= 0 ? 0.0f : fmaxf(was, 0.0f);
    int8_t* codes = p.codes[which] + ((page * p.heads + head) << p.block_log2) * p.head_dim;
    const auto write = [&](auto plain, float amax) {
        constexpr bool PLAIN = decltype(plain)::value;  // finite values, and a scale whose inverse is finite
        const float scale = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, fmaxf(old, div127(amax)))));  // a page's one, in every lane
        const float by = scale > 0.0f ? scale : 1.0f, again = old / by, divisor = PLAIN ? divisor_of<DT>(by) : by, inv = 1.0f / divisor;
        each([&](int n, int row, int chunk) {
            const int t = rows[row];
            u32x2* at = reinterpret_cast<u32x2*>(codes + row * p.head_dim + 8 * chunk);
            int q[8];
            if (t >= 0) {
                if constexpr (!NI) kept[0].load(x + t * p.token_stride[which] + 8 * chunk);
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = code_of<!PLAIN>(kept[n].template value<PLAIN>(j), divisor, inv);
            } else {
                if (!(old < scale) || old == 0.0f) return;
                const u32x2 before = *at;
#pragma unroll
                for (int j = 0; j < 8; ++j) q[j] = rne_int(float(int8_t(before[j >> 2] >> (8 * (j & 3)))) * again);
            }
            *at = u32x2{pack_low_bytes(q[0], q[1], q[2], q[3]), pack_low_bytes(q[4], q[5], q[6], q[7])};
        });
        return scale;
    };
    float scale;
    if (finite && fmaxf(old, div127(amax)) >= 0x1p-120f) {
        scale = write(std::true_type(), amax);
    } else {
        float most = 0.0f;
        each([&](int n, int row, int chunk) {
            const int t = rows[row];
            if (t < 0) return;
            if constexpr (!NI) kept[0].load(x + t * p.token_stride[which] + 8 * chunk);
#pragma unroll
            for (int j = 0; j < 8; ++j) most = fmaxf(most, __builtin_fabsf(kept[n].template value<false>(j)));
        });
        scale = write(std::false_type(), __builtin_bit_cast(float, block_max_bits(__builtin_bit_cast(uint32_t, most), lds4)));
    }
    __syncthreads();  // every thread has read the held scale
    if (!threadIdx.x) *held = scale;
}

constexpr int KV_MAX_BLOCK = 128;
// Up to this many tokens a workgroup reads every slot by itself to find its page's tokens, and the owner pass is left out.
constexpr int KV_SCAN_TOKENS = 512;

template <int DT, int NI>
__global__ void __launch_bounds__(256) kv_write_scan(CacheArgs p) {
    __shared__ int rows[KV_MAX_BLOCK];
    __shared__ uint32_t lds4[4];
    const int token = blockIdx.x, head = blockIdx.y, which = blockIdx.z, block = 1 << p.block_log2;
    const int64_t slot = p.slots[token];
    if (slot < 0 || slot >= p.all_slots) return;
    const int64_t page = slot >> p.block_log2, page_slot = page << p.block_log2;
    const int at = int(slot - page_slot);
    if (int(threadIdx.x) < block) rows[threadIdx.x] = -1;
    __syncthreads();
    for (int t = threadIdx.x; t < p.tokens; t += 256) {
        const int64_t s = p.slots[t] - page_slot;
        if (s >= 0 && s < block) atomicMax(&rows[s], t);
    }
    __syncthreads();
    // the page is its lowest slot's token's
    if (rows[at] != token) return;
    for (int i = 0; i < at; ++i)
        if (rows[i] >= 0) return;
    write_page<DT, NI>(p, which, page, head, rows, lds4);
}

// Many tokens: a workgroup looks through p.group of them (64 at most) for those that have the lowest written slot of a page, and writes these
// pages' codes. Bound by HBM and the loads before the values' own (slots, owners, slots): 302 MB of 32760 tokens, 12 heads of 128 BF16,
// in 71 us, 4.3 TB/s. Of a page begun before, the slots ahead of the first new token are looked at one after another (1000 tokens from the
// last slot of a page of 128 on, 12 heads: 33 us; from its first: 17.4).
template <int DT, int NI>
__global__ void __launch_bounds__(256) kv_write_owned(CacheArgs p) {
    __shared__ int rows[KV_MAX_BLOCK];
    __shared__ int64_t pages[64];
    __shared__ uint32_t lds4[4];
    const int block = 1 << p.block_log2;
    const unsigned looked = blockIdx.x / unsigned(p.parts), first_part = blockIdx.x - looked * unsigned(p.parts);
    const auto writer = [&](int64_t slot) {
        const int t = p.owner[slot];
        return t >= 0 && t < p.tokens && p.slots[t] == slot ? t : -1;
    };
    if (threadIdx.x < 64) {
        const int64_t token = looked * int64_t(p.group) + threadIdx.x;
        int64_t page = -1;
        if (int(threadIdx.x) < p.group && token < p.tokens) {
            const int64_t slot = p.slots[token];
            if (slot >= 0 && slot < p.all_slots) {
                const int64_t begin = slot >> p.block_log2 << p.block_log2;
                bool lowest = p.owner[slot] == token;
                for (int64_t s = slot - 1; s >= begin && lowest; --s) lowest = writer(s) < 0;
                if (lowest) page = slot >> p.block_log2;
            }
        }
        pages[threadIdx.x] = page;
    }
    __syncthreads();
    for (int i = 0; i < p.group; ++i) {
        const int64_t page = pages[i];
        if (page < 0) continue;
        if (int(threadIdx.x) < block) rows[threadIdx.x] = writer((page << p.block_log2) + threadIdx.x);
        __syncthreads();
        for (int part = first_part; part < 2 * p.heads; part += p.parts) write_page<DT, NI>(p, part & 1, page, part >> 1, rows, lds4);
        __syncthreads();
    }
}

template <int DT, int NI> static int launch_pages(CacheArgs p, hipStream_t stream) {
    if (p.tokens <= KV_SCAN_TOKENS) {
        kv_write_scan<DT, NI><<<dim3(unsigned(p.tokens), p.heads, 2), 256, 0, stream>>>(p);
    } else {
        // Tokens a workgroup: fewer where workgroups are few (each token may have a page of its own). Finding the pages costs a workgroup about
        // as much as writing one, so it then writes several heads where there are enough workgroups.
        p.group = 64;
        while (p.group > 4 && p.tokens * p.heads * 2 < p.group * int64_t(4096)) p.group >>= 1;
        const int64_t groups = (p.tokens + p.group - 1) / p.group;
        p.parts = int(std::max<int64_t>(1, std::min<int64_t>(2 * p.heads, 4096 / groups)));
        if (groups * p.parts > MAX_BLOCKS_256) return -2;
        kv_owner<<<unsigned((p.tokens + 255) / 256), 256, 0, stream>>>(p);
        kv_write_owned<DT, NI><<<unsigned(groups * p.parts), 256, 0, stream>>>(p);
    }
    return int(hipGetLastError());
}

template <int DT> static int launch_write(const CacheArgs& p, hipStream_t stream) {
    const int vectors = (p.head_dim << p.block_log2) + 2047 >> 11;
    return vectors <= 1 ? launch_pages<DT, 1>(p, stream) : vectors <= 2 ? launch_pages<DT, 2>(p, stream) : vectors <= 4 ? launch_pages<DT, 4>(p, stream)
         : vectors <= 8 ? launch_pages<DT, 8>(p, stream) : vectors <= 16 ? launch_pages<DT, 16>(p, stream) : launch_pages<DT, 0>(p, stream);
}

// ---- reads ---------------------------------------------------------------------------------------------------------
// READ_VECTORS of 8 channels a thread: four where there are many (a 32760-token latent of 12 heads, keys and values: 61.6 us against 73 with one; 302 MB, 5 TB/s, bound by HBM).
template <int DT, int READ_VECTORS>
__global__ void __launch_bounds__(256) kv_read_rows(CacheArgs p) {
    using raw = typename Elem<DT>::raw;
    const int per_row = p.head_dim >> 3, per_token = p.heads * per_row, which = blockIdx.y;
    // vectors blockIdx.x * 256 * READ_VECTORS + 256 n + threadIdx.x of (token, head, chunk): the wide division is the workgroup's alone
    const int64_t first = blockIdx.x * int64_t(256 * READ_VECTORS), token0 = first / per_token;
    const unsigned in = unsigned(first - token0 * per_token) + threadIdx.x;
    float v[READ_VECTORS][8];
    int64_t to[READ_VECTORS];
#pragma unroll
    for (int n = 0; n < READ_VECTORS; ++n) {
        const unsigned at = in + 256 * n, rest = at % unsigned(per_token), head = rest / unsigned(per_row), c = rest % unsigned(per_row);
        const int64_t token = token0 + at / unsigned(per_token);
        to[n] = token < p.tokens ? token * per_token + rest : -1;
        const int64_t slot = token < p.tokens ? p.slots[token] : -1;
        const bool live = slot >= 0 && slot < p.all_slots;
        const int64_t row = live ? (slot >> p.block_log2) * p.heads + head : 0, in_page = live ? slot & ((1 << p.block_log2) - 1) : 0;
        u32x2 q = {0, 0};
        float scale = 0.0f;
        if (live) {
            scale = p.scales[which][row];
            q = *reinterpret_cast<const u32x2*>(p.codes[which] + ((row << p.block_log2) + in_page) * p.head_dim + 8 * c);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[n][j] = float(int8_t(q[j >> 2] >> (8 * (j & 3)))) * scale;
    }
#pragma unroll
    for (int n = 0; n < READ_VECTORS; ++n)
        if (to[n] >= 0) store8<DT>(static_cast<raw*>(p.y[which]) + to[n] * 8, v[n]);
}

static bool bad_cache(int64_t tokens, int64_t pages, int heads, int block, int head_dim) {
    return tokens < 0 || tokens > 0x7fffffff || pages < 0 || heads < 1 || heads > 65535 || head_dim < 8 || head_dim % 8 || head_dim > 1024 ||
           block < 1 || block > KV_MAX_BLOCK || (block & (block - 1)) || pages > 0x7fffffff;
}

}  // namespace wq8

using namespace wq8;

WQ8_API int wq8_kv_plan(const void* past, const void* fresh, int32_t* tables, int64_t table_stride, const void* pages, int pages_count, const void* used,
                        int requests, int width, int block, int64_t tokens, int64_t* slots, int32_t* positions, int32_t* starts, int32_t* lens,
                        int32_t* used_out, int32_t* missing, hipStream_t stream) {
    if (requests < 0 || width < 0 || block < 1 || tokens < 0 || tokens > 0x7fffffff || pages_count < 0) return -2;
    const PlanArgs p = {static_cast<const int*>(past), static_cast<const int*>(fresh), static_cast<const int*>(pages), static_cast<const int*>(used),
                        tables, table_stride, tokens, pages_count, requests, width, block, slots, positions, starts, lens, used_out, missing};
    kv_plan_tokens<<<unsigned(std::max<int64_t>(1, (tokens + PLAN_TOKENS - 1) / PLAN_TOKENS)), 256, 0, stream>>>(p);
    return int(hipGetLastError());
}

WQ8_API int wq8_kv_write(const void* k, const void* v, const long long* strides, const long long* slots, int64_t tokens, int8_t* k_codes, float* k_scales,
                         int8_t* v_codes, float* v_scales, int64_t pages, int heads, int block, int head_dim, int dtype, int32_t* owner,
                         hipStream_t stream) {
    if (dtype < 0 || dtype > 2) return -1;
    if (bad_cache(tokens, pages, heads, block, head_dim)) return -2;
    if (!tokens || !pages) return 0;
    const CacheArgs p = {{k, v}, {}, {strides[0], strides[2]}, {strides[1], strides[3]}, {k_codes, v_codes}, {k_scales, v_scales},
                         reinterpret_cast<const int64_t*>(slots), owner, tokens, pages * block, heads, __builtin_ctz(block), head_dim, 0, 0};
    return dtype == DT_F16 ? launch_write<DT_F16>(p, stream) : dtype == DT_BF16 ? launch_write<DT_BF16>(p, stream) : launch_write<DT_F32>(p, stream);
}

WQ8_API int wq8_kv_read(const int8_t* k_codes, const float* k_scales, const int8_t* v_codes, const float* v_scales, const long long* slots, int64_t tokens,
                        void* k, void* v, int64_t pages, int heads, int block, int head_dim, int dtype, hipStream_t stream) {
    if (dtype < 0 || dtype > 2) return -1;
    if (bad_cache(tokens, pages, heads, block, head_dim)) return -2;
    if (!tokens) return 0;
    const CacheArgs p = {{}, {k, v}, {}, {}, {const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes)},
                         {const_cast<float*>(k_scales), const_cast<float*>(v_scales)}, reinterpret_cast<const int64_t*>(slots), nullptr, tokens, pages * block,
                         heads, __builtin_ctz(block), head_dim, 0, 0};
    const int64_t vectors = tokens * heads * (head_dim >> 3);
    const int each = vectors >= 1 << 20 ? 4 : 1;
    const int64_t blocks = (vectors + 256 * each - 1) / (256 * each);
    if (blocks > MAX_BLOCKS_256) return -2;
    const dim3 grid(static_cast<unsigned>(blocks), 2);
    const auto run = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (each == 4) kv_read_rows<DT, 4><<<grid, 256, 0, stream>>>(p);
        else kv_read_rows<DT, 1><<<grid, 256, 0, stream>>>(p);
    };
    if (dtype == DT_F16) run(std::integral_constant<int, DT_F16>());
    else if (dtype == DT_BF16) run(std::integral_constant<int, DT_BF16>());
    else run(std::integral_constant<int, DT_F32>());
    return int(hipGetLastError());
}

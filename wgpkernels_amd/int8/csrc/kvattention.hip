// Attention over the paged 8-bit key/value cache on gfx950.
//
// Row (token t of request r, query head h) of head_dim channels, on key/value head h / group:
//     s_j = scale q . k_j,   p_j = exp(s_j - max s) over the keys j that the row sees,   out = sum p_j v_j / sum p_j.
// The row stands at position lens[r] - new[r] + t; it sees the keys up to its own position (causal) or every key of the
// request, and with a window w those after position - w alone. A row that sees no key is zero, as is one on pages outside
// the cache: their keys are hidden.
#include "wq8_common.h"
#include "wq8_abi.h"
#include <algorithm>

namespace wq8 {

struct AttentionArgs {
    const void* q;
    void* out;
    int64_t q_token, q_head, out_token, out_head;
    const int8_t *k_codes, *v_codes;
    const float *k_scales, *v_scales;
    const int *tables, *lens, *starts;
    int64_t table_stride, pages;
    int width, tokens, requests, heads, group, head_dim, block, causal, window;
    float scale;
};

// One wave a row: 64 keys at a time, a lane each for the scores, then a lane for every 64th channel of the sum.
template <int DT>
__global__ void __launch_bounds__(256) kv_attention_rows(AttentionArgs p) {
    using raw = typename Elem<DT>::raw;
    __shared__ float rows[4][256];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t index = blockIdx.x * int64_t(4) + wave;
    const int q_heads = p.heads * p.group;
    const int64_t token = index / q_heads;
    const int qh = int(index - token * q_heads), head = qh / p.group;
    int request = -1, begin = 0, end = 0;
    for (int r = 0; r < p.requests && token < p.tokens; ++r) {
        begin = p.starts[r];
        end = p.starts[r + 1];
        if (token >= begin && token < end) { request = r; break; }
    }
    if (request < 0) return;
    const raw* q = static_cast<const raw*>(p.q) + token * p.q_token + qh * p.q_head;
    for (int c = lane; c < p.head_dim; c += 64) rows[wave][c] = Elem<DT>::to_f(q[c]) * p.scale * 0x1.715476p+0f;
    const int64_t len = p.lens[request], position = len - (end - begin) + (token - begin);
    const int64_t total = min(len, int64_t(p.width) * p.block);
    const int64_t high = p.causal ? min(total, position + 1) : total, low = p.window ? max(int64_t(0), position - p.window + 1) : 0;
    const int* table = p.tables + request * p.table_stride;
    float top = -0x1p+120f, mass = 0.0f, acc[4] = {};
    for (int64_t base = low / 64 * 64; base < high; base += 64) {
        const int64_t key = base + lane;
        float s = -__builtin_inff(), vs = 0.0f;
        int64_t row = 0;
        if (key >= low && key < high) {
            const int64_t page = table[key / p.block];
            if (page >= 0 && page < p.pages) {
                row = ((page * p.heads + head) * p.block + key % p.block) * p.head_dim;
                vs = p.v_scales[page * p.heads + head];
                s = 0.0f;
                for (int c = 0; c < p.head_dim; c += 4) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(p.k_codes + row + c);
                    for (int j = 0; j < 4; ++j) s = __builtin_fmaf(rows[wave][c + j], float(int8_t(w >> (8 * j))), s);
                }
                s *= p.k_scales[page * p.heads + head];
            }
        }
        float m = s;
        for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
        m = fmaxf(m, top);
        const float keep = __builtin_amdgcn_exp2f(top - m), w = __builtin_amdgcn_exp2f(s - m);
        top = m;
        mass = __builtin_fmaf(mass, keep, w);
        for (int i = 0; i < 4; ++i) acc[i] *= keep;
        const float wv = w * vs;
        for (int j = 0; j < 64; ++j) {
            const float f = __shfl(wv, j);
            const int64_t at = __shfl(row, j);
            if (f != 0.0f)
                for (int i = 0; i < 4; ++i)
                    if (lane + 64 * i < p.head_dim) acc[i] = __builtin_fmaf(f, float(p.v_codes[at + lane + 64 * i]), acc[i]);
        }
    }
    for (int d = 1; d < 64; d <<= 1) mass += __shfl_xor(mass, d);
    raw* out = static_cast<raw*>(p.out) + token * p.out_token + qh * p.out_head;
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < p.head_dim) out[lane + 64 * i] = Elem<DT>::from_f(mass > 0.0f ? acc[i] / mass : mass == 0.0f ? 0.0f : mass);
}

}  // namespace wq8

using namespace wq8;

WQ8_API void wq8_kv_attention_workspace(int tokens, int requests, int heads, int group, int head_dim, int64_t keys, int sms, int64_t* sizes) {
    (void)tokens; (void)requests; (void)heads; (void)group; (void)head_dim; (void)keys; (void)sms;
    sizes[0] = sizes[1] = 0;
}

WQ8_API int wq8_kv_attention(const void* q, void* out, const long long* strides, const int8_t* k_codes, const float* k_scales, const int8_t* v_codes,
                             const float* v_scales, const void* tables, int64_t table_stride, int width, const void* lens, const void* starts, int tokens,
                             int requests, int heads, int group, int head_dim, int block, int64_t pages, float scale, int causal, int window, int dtype,
                             int sms, void* workspace, hipStream_t stream) {
    (void)sms; (void)workspace;
    if (dtype != DT_F16 && dtype != DT_BF16) return -1;
    if (tokens < 0 || requests < 0 || heads < 1 || group < 1 || (head_dim != 64 && head_dim != 128 && head_dim != 256) ||
        (block != 16 && block != 32 && block != 64 && block != 128) || window < 0) return -2;
    if (!tokens || !requests) return 0;
    const AttentionArgs p = {q, out, strides[0], strides[1], strides[2], strides[3], k_codes, v_codes, k_scales, v_scales, static_cast<const int*>(tables),
                             static_cast<const int*>(lens), static_cast<const int*>(starts), table_stride, pages, width, tokens, requests, heads, group,
                             head_dim, block, causal, window, scale};
    const int64_t blocks = (int64_t(tokens) * heads * group + 3) / 4;
    if (blocks > 0x7fffffff) return -2;
    if (dtype == DT_F16) kv_attention_rows<DT_F16><<<unsigned(blocks), 256, 0, stream>>>(p);
    else kv_attention_rows<DT_BF16><<<unsigned(blocks), 256, 0, stream>>>(p);
    return int(hipGetLastError());
}

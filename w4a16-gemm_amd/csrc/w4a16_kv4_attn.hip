// Attention over the 4-bit key/value cache (include/w4a16.h has the format and what is computed).
#include <math.h>

#include "w4a16_internal.h"
#include "w4a16_kv4.h"

namespace w4a16 {

// One wave per (query, query head).  Keys go by in tiles of 64: lane t takes the score of key t, the tile's
// probabilities pass through LDS, and lane d adds up values d and d + D/2.
template <int D, int G>
__global__ void __launch_bounds__(64)
kv4_attention_kernel(Kv4Attn a) {
    __shared__ float qs[D], ps[64];
    __shared__ int pages[64];
    constexpr int NG = D / G, HALF = D / 2;
    const int lane = threadIdx.x;
    const int b = blockIdx.x / a.heads, head = blockIdx.x % a.heads, h = head / a.rep;
    const Kv4Seq s = kv4_seq(a, b);
    for (int i = blockIdx.y; i < s.count; i += gridDim.y) {
        const int64_t row = s.first + i;
        const int pos = s.len - s.count + i;
        const int end = a.causal ? min(pos + 1, s.len) : s.len;
        const int begin = a.window > 0 ? max(0, pos - a.window + 1) : 0;
        __syncthreads();
        for (int d = lane; d < D; d += 64) qs[d] = load16(a.q[row * a.q_token + head * a.q_head + d], a.bf16) * a.scale2;
        __syncthreads();
        float top = -INFINITY, total = 0.f, o0 = 0.f, o1 = 0.f;
        for (int t0 = begin & ~15; t0 < end; t0 += 64) {
            const int t = t0 + lane;
            int page = t < end && t >= begin ? a.table[b * a.table_stride + t / a.c.P] : -1;
            if (page >= a.c.pages) page = -1;
            float x = -INFINITY;
            if (page >= 0) {
                const uint8_t* kv = a.c.head(page, h);
                const int at = t % a.c.P;
                x = 0.f;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float sc = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kKeyScale, g, at)));
                    const float ze = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kKeyZero, g, at)));
                    float dot = 0.f;
                    for (int j = 0; j < G; ++j) {
                        const int d = g * G + j;
                        const uint32_t byte = kv[kv4_key_row<D>(at) + d % HALF];
                        dot += qs[d] * ((float)((d < HALF ? byte : byte >> 4) & 15u) - ze);
                    }
                    x += dot * sc;
                }
            }
            float m = x;
            for (int w = 1; w < 64; w *= 2) m = fmaxf(m, __shfl_xor(m, w, 64));
            const bool nan = __any(x != x);
            const float next = nan ? NAN : fmaxf(top, m);
            const float safe = next == -INFINITY ? 0.f : next;
            const float p = page >= 0 ? exp2f(x - safe) : 0.f;
            float sum = p;
            for (int w = 1; w < 64; w *= 2) sum += __shfl_xor(sum, w, 64);
            const float keep = exp2f(top - safe);
            total = total * keep + sum;
            o0 *= keep;
            o1 *= keep;
            top = next;
            __syncthreads();
            ps[lane] = p;
            pages[lane] = page;
            __syncthreads();
            if (lane < HALF) {
                for (int r = 0; r < 64; ++r) {
                    const int pg = pages[r];
                    if (pg < 0) continue;
                    const uint8_t* kv = a.c.head(pg, h);
                    const int at = (t0 + r) % a.c.P;
                    const uint32_t byte = kv[kv4_value_tile<D>(a.c.P, at) + lane * 16 + kv4_place(at & 15)];
                    const int g0 = lane / G, g1 = (lane + HALF) / G;
                    const float s0 = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kValueScale, g0, at)));
                    const float z0 = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kValueZero, g0, at)));
                    const float s1 = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kValueScale, g1, at)));
                    const float z1 = half_bits(*(const uint16_t*)(kv + kv4_side<D, G>(a.c.P, kValueZero, g1, at)));
                    o0 += ps[r] * (((float)(byte & 15u) - z0) * s0);
                    o1 += ps[r] * (((float)(byte >> 4) - z1) * s1);
                }
            }
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;   // a row that sees nothing: zeros; NaN stays NaN
        uint16_t* dst = a.out + (row * a.heads + head) * D;
        if (lane < HALF) {
            dst[lane] = store16(o0 * inv, a.bf16);
            dst[lane + HALF] = store16(o1 * inv, a.bf16);
        }
        if (a.lse && lane == 0) a.lse[row * a.heads + head] = total == 0.f ? -INFINITY : (top + log2f(total)) * 0.69314718055994531f;
    }
}

static const char* check_attention(const w4a16_kv4_cache* c, const w4a16_kv4_attention_args* a, const w4a16_device_limits* lim) {
    if (const char* m = kv4_check(c)) return m;
    if (!a || !lim) return "null pointer";
    if (a->tokens < 0 || a->batch < 0 || a->table_width < 0 || a->heads < 1 || a->heads > 4096 || a->tokens >= (int64_t)1 << 31 ||
        a->batch >= (int64_t)1 << 20 || a->table_width * c->page_size >= (int64_t)1 << 31 || a->max_q < 1 || a->window < 0 ||
        a->tokens * a->heads >= (int64_t)1 << 31 || a->batch * a->heads >= (int64_t)1 << 31)
        return "dimensions out of range";
    if (a->heads % c->kv_heads != 0) return "the query heads must be a multiple of the KV heads";
    if (!a->q_start && a->tokens != a->batch) return "without q_start there is one query per sequence";
    if (!(a->scale > 0.f) || !isfinite(a->scale)) return "scale must be positive and finite";
    if (a->tokens == 0 || a->batch == 0) return nullptr;
    if (!a->q || !a->out || !a->seq_lens || (!a->block_table && a->table_width > 0)) return "null pointer";
    if (a->table_width > 0 && a->batch > 1 && a->table_stride < a->table_width) return "rows of the block table overlap";
    if (reinterpret_cast<uintptr_t>(a->q) % 2 != 0 || reinterpret_cast<uintptr_t>(a->out) % 16 != 0 ||
        (reinterpret_cast<uintptr_t>(a->lse) | reinterpret_cast<uintptr_t>(a->block_table) | reinterpret_cast<uintptr_t>(a->seq_lens) |
         reinterpret_cast<uintptr_t>(a->q_start)) % 4 != 0)
        return "out must be 16-byte aligned, q 2-byte, the others 4-byte aligned";
    return nullptr;
}

}  // namespace w4a16

using namespace w4a16;

extern "C" int64_t w4a16_kv4_attention_workspace(const w4a16_kv4_cache* cache, const w4a16_kv4_attention_args* args,
                                                 const w4a16_device_limits* lim) {
    if (const char* m = check_attention(cache, args, lim)) return kv4_fail(-1, "kv4_attention", m);
    return 0;
}

extern "C" int w4a16_kv4_attention(const w4a16_kv4_cache* cache, const w4a16_kv4_attention_args* args, const w4a16_device_limits* lim,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
    const int64_t need = w4a16_kv4_attention_workspace(cache, args, lim);
    if (need < 0) return W4A16_ERR_INVALID;
    if (workspace_bytes < need || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 != 0)))
        return kv4_fail(W4A16_ERR_WORKSPACE, "kv4_attention", "workspace missing, unaligned or too small");
    if (args->tokens == 0 || args->batch == 0) return W4A16_OK;
    Kv4Attn a{};
    a.c = kv4_of(cache);
    a.q = (const uint16_t*)args->q;
    a.out = (uint16_t*)args->out;
    a.lse = args->lse;
    a.q_token = args->q_token_stride;
    a.q_head = args->q_head_stride;
    a.table = args->block_table;
    a.table_stride = args->table_stride;
    a.lens = args->seq_lens;
    a.q_start = args->q_start;
    a.width = (int)args->table_width;
    a.tokens = (int)args->tokens;
    a.heads = (int)args->heads;
    a.rep = (int)(args->heads / cache->kv_heads);
    a.window = (int)(args->window < 0x7fffffff ? args->window : 0);
    a.scale2 = args->scale * 1.44269504088896341f;
    a.bf16 = args->bf16 != 0;
    a.causal = args->causal != 0;
    const dim3 grid((unsigned)(args->batch * args->heads), (unsigned)(args->max_q < 65535 ? args->max_q : 65535));
    hipStream_t st = (hipStream_t)stream;
    kv4_sizes(cache, [&](auto d, auto g) {
        hipLaunchKernelGGL((kv4_attention_kernel<d.value, g.value>), grid, dim3(64), 0, st, a);
    });
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return kv4_fail(W4A16_ERR_HIP, "kv4_attention", hipGetErrorString(e));
    return W4A16_OK;
}

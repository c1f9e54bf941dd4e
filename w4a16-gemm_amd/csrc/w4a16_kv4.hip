// Writing keys and values into the 4-bit cache and reading them back (include/w4a16.h has the format).
#include <stdio.h>

#include "w4a16_internal.h"
#include "w4a16_kv4.h"

namespace w4a16 {

// One wave per (token, KV head) of K (blockIdx.y even) or V.  Lane j holds values j and j + D/2, the two
// codes of byte j.  Every operation is an IEEE fp32 operation, so the bytes are the format's definition.
template <int D, int G>
__global__ void __launch_bounds__(256)
kv4_write_kernel(Kv4 c, const uint16_t* __restrict__ k, const uint16_t* __restrict__ v, int bf16, int tokens, int64_t k_token,
                 int64_t k_head, int64_t v_token, int64_t v_head, const int64_t* __restrict__ slots) {
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t token = unit / c.H;
    const int h = (int)(unit % c.H);
    if (token >= tokens) return;
    const int64_t slot = slots[token];
    if (slot < 0 || slot >= c.slots()) return;
    const bool value = blockIdx.y != 0;
    const uint16_t* src = value ? v + token * v_token + h * v_head : k + token * k_token + h * k_head;
    const bool live = lane < D / 2;
    const float x0 = live ? load16(src[lane], bf16) : 0.f, x1 = live ? load16(src[lane + D / 2], bf16) : 0.f;
    float x[2] = {fminf(fmaxf(x0, -65504.f), 65504.f), fminf(fmaxf(x1, -65504.f), 65504.f)};
    const bool nan[2] = {x0 != x0, x1 != x1};
    constexpr int NG = D / G;
    float lo[NG], hi[NG], s[NG], z[NG];
    bool bad[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        lo[g] = NG == 2 ? x[g] : fminf(x[0], x[1]);
        hi[g] = NG == 2 ? x[g] : fmaxf(x[0], x[1]);
        if (!live) lo[g] = INFINITY, hi[g] = -INFINITY;
#pragma unroll
        for (int m = 1; m < 64; m *= 2) {
            lo[g] = fminf(lo[g], __shfl_xor(lo[g], m, 64));
            hi[g] = fmaxf(hi[g], __shfl_xor(hi[g], m, 64));
        }
        bad[g] = __any(NG == 2 ? nan[g] : nan[0] || nan[1]);
        const float step = fmaxf(fmaxf((hi[g] - lo[g]) / 15.f, fmaxf(fabsf(lo[g]), fabsf(hi[g])) / 96.f), 0x1p-14f);
        s[g] = half_bits(to_half_bits(step));
        z[g] = rintf(-lo[g] / s[g] * 8.f) / 8.f;
    }
    uint32_t q[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int g = NG == 2 ? i : 0;
        q[i] = bad[g] ? 0u : (uint32_t)fminf(fmaxf(rintf(x[i] / s[g] + z[g]), 0.f), 15.f);
    }
    const int page = (int)(slot / c.P), t = (int)(slot % c.P);
    uint8_t* head = c.head(page, h);
    if (live) {
        const uint8_t byte = (uint8_t)(q[0] | (q[1] << 4));
        if (value) head[kv4_value_tile<D>(c.P, t) + lane * 16 + kv4_place(t & 15)] = byte;
        else head[kv4_key_row<D>(t) + lane] = byte;
    }
    if (lane < NG) {
        const int g = lane;
        const bool b = g == 0 ? bad[0] : bad[NG - 1];
        const float sg = g == 0 ? s[0] : s[NG - 1], zg = g == 0 ? z[0] : z[NG - 1];
        *reinterpret_cast<uint16_t*>(head + kv4_side<D, G>(c.P, value ? kValueScale : kKeyScale, g, t)) = b ? 0x7E00u : to_half_bits(sg);
        *reinterpret_cast<uint16_t*>(head + kv4_side<D, G>(c.P, value ? kValueZero : kKeyZero, g, t)) = b ? 0x7E00u : to_half_bits(zg);
    }
}

template <int D, int G>
__global__ void __launch_bounds__(256)
kv4_read_kernel(Kv4 c, const int64_t* __restrict__ slots, int tokens, int bf16, uint16_t* __restrict__ k, uint16_t* __restrict__ v) {
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int64_t token = unit / c.H;
    const int h = (int)(unit % c.H);
    if (token >= tokens || lane >= D / 2) return;
    const bool value = blockIdx.y != 0;
    const int64_t slot = slots[token];
    uint16_t* dst = (value ? v : k) + unit * D;
    if (slot < 0 || slot >= c.slots()) {
        dst[lane] = dst[lane + D / 2] = 0;
        return;
    }
    const int page = (int)(slot / c.P), t = (int)(slot % c.P);
    const uint8_t* head = c.head(page, h);
    const uint32_t byte = value ? head[kv4_value_tile<D>(c.P, t) + lane * 16 + kv4_place(t & 15)] : head[kv4_key_row<D>(t) + lane];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + i * (D / 2);
        const float s = half_bits(*reinterpret_cast<const uint16_t*>(head + kv4_side<D, G>(c.P, value ? kValueScale : kKeyScale, d / G, t)));
        const float z = half_bits(*reinterpret_cast<const uint16_t*>(head + kv4_side<D, G>(c.P, value ? kValueZero : kKeyZero, d / G, t)));
        float x = ((float)((byte >> (4 * i)) & 15u) - z) * s;
        asm("" : "+v"(x));      // the product, then its rounding: fused into one mixed FMA with +0, -0 would become +0
        dst[d] = store16(x, bf16);
    }
}

// Shared by the entry points: the cache's sizes and pointer.  Returns a message, or null.
const char* kv4_check(const w4a16_kv4_cache* c) {
    if (!c) return "null pointer";
    if (c->head_dim != 64 && c->head_dim != 128) return "unsupported head size, supported: 64, 128";
    if (c->group_size != 64 && c->group_size != 128) return "unsupported group size, supported: 64, 128";
    if (c->group_size > c->head_dim) return "the group size must divide the head size";
    if (c->page_size < 16 || c->page_size > 4096 || c->page_size % 16 != 0) return "the page size must be a multiple of 16, 16..4096";
    if (c->kv_heads < 1 || c->kv_heads > 1024) return "kv_heads must be 1..1024";
    if (c->pages < 0 || c->pages >= (int64_t)1 << 31) return "dimensions out of range";
    if (c->pages > 0 && !c->data) return "null pointer";
    if (reinterpret_cast<uintptr_t>(c->data) % 16 != 0) return "the cache must be 16-byte aligned";
    return nullptr;
}

Kv4 kv4_of(const w4a16_kv4_cache* c) {
    return Kv4{(uint8_t*)c->data, w4a16_kv4_page_bytes(c->page_size, c->head_dim, c->group_size), (int)c->pages, (int)c->page_size,
               (int)c->kv_heads};
}

int kv4_fail(int code, const char* who, const char* what) {
    char msg[256];
    snprintf(msg, sizeof(msg), "%s: %s", who, what);
    w4a16_set_last_error(msg);
    return code;
}

}  // namespace w4a16

using namespace w4a16;

extern "C" int64_t w4a16_kv4_page_bytes(int64_t page_size, int64_t head_dim, int64_t group_size) {
    const w4a16_kv4_cache c{nullptr, 0, page_size, 1, head_dim, group_size};
    if (kv4_check(&c)) return 0;
    return page_size * (head_dim + 8 * (head_dim / group_size));
}

extern "C" int w4a16_kv4_write(const w4a16_kv4_cache* cache, const void* k, const void* v, int bf16, int64_t tokens,
                               int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                               const int64_t* slots, void* stream) {
    if (const char* m = kv4_check(cache)) return kv4_fail(W4A16_ERR_INVALID, "kv4_write", m);
    if (tokens < 0 || tokens >= (int64_t)1 << 31 || tokens * cache->kv_heads >= (int64_t)1 << 31)
        return kv4_fail(W4A16_ERR_INVALID, "kv4_write", "dimensions out of range");
    if (tokens == 0 || cache->pages == 0) return W4A16_OK;
    if (!k || !v || !slots) return kv4_fail(W4A16_ERR_INVALID, "kv4_write", "null pointer");
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 2 != 0 || reinterpret_cast<uintptr_t>(slots) % 8 != 0)
        return kv4_fail(W4A16_ERR_INVALID, "kv4_write", "k and v must be 2-byte aligned, slots 8-byte aligned");
    const dim3 grid((unsigned)((tokens * cache->kv_heads + 3) / 4), 2);
    kv4_sizes(cache, [&](auto d, auto g) {
        hipLaunchKernelGGL((kv4_write_kernel<d.value, g.value>), grid, dim3(256), 0, (hipStream_t)stream, kv4_of(cache), (const uint16_t*)k,
                           (const uint16_t*)v, bf16, (int)tokens, k_token_stride, k_head_stride, v_token_stride, v_head_stride, slots);
    });
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return kv4_fail(W4A16_ERR_HIP, "kv4_write", hipGetErrorString(e));
    return W4A16_OK;
}

extern "C" int w4a16_kv4_read(const w4a16_kv4_cache* cache, const int64_t* slots, int64_t tokens, int bf16, void* k, void* v,
                              void* stream) {
    if (const char* m = kv4_check(cache)) return kv4_fail(W4A16_ERR_INVALID, "kv4_read", m);
    if (tokens < 0 || tokens >= (int64_t)1 << 31 || tokens * cache->kv_heads >= (int64_t)1 << 31)
        return kv4_fail(W4A16_ERR_INVALID, "kv4_read", "dimensions out of range");
    if (tokens == 0) return W4A16_OK;
    if (!k || !v || !slots) return kv4_fail(W4A16_ERR_INVALID, "kv4_read", "null pointer");
    if ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) % 16 != 0 || reinterpret_cast<uintptr_t>(slots) % 8 != 0)
        return kv4_fail(W4A16_ERR_INVALID, "kv4_read", "k and v must be 16-byte aligned, slots 8-byte aligned");
    const dim3 grid((unsigned)((tokens * cache->kv_heads + 3) / 4), 2);
    kv4_sizes(cache, [&](auto d, auto g) {
        hipLaunchKernelGGL((kv4_read_kernel<d.value, g.value>), grid, dim3(256), 0, (hipStream_t)stream, kv4_of(cache), slots, (int)tokens,
                           bf16, (uint16_t*)k, (uint16_t*)v);
    });
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return kv4_fail(W4A16_ERR_HIP, "kv4_read", hipGetErrorString(e));
    return W4A16_OK;
}

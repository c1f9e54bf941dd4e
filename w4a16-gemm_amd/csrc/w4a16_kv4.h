// The 4-bit key/value cache: layout, parameters and device building blocks shared by its kernels.
// The format is defined in include/w4a16.h.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "w4a16.h"
#include "w4a16_device.h"

namespace w4a16 {

// A cache as the kernels take it.
struct Kv4 {
    uint8_t* data;
    uint32_t head_bytes, page_bytes;         // bytes of one (page, KV head), and of one page (at most 576 MiB)
    int pages, P, H;

    __host__ __device__ int64_t slots() const { return (int64_t)pages * P; }
    __device__ uint8_t* head(int page, int h) const {
        return data + (uint64_t)(uint32_t)h * head_bytes + (uint64_t)(uint32_t)page * page_bytes;
    }
};

enum { kKeyScale = 0, kKeyZero = 1, kValueScale = 2, kValueZero = 3 };

// Offsets within the bytes of one (page, KV head).
template <int D>
__device__ __forceinline__ int kv4_key_row(int t) { return t * (D / 2); }
template <int D>
__device__ __forceinline__ int kv4_value_tile(int P, int t) { return P * (D / 2) + (t >> 4) * (D / 2 * 16); }
// Place of token t of 16 in a value tile's 16 bytes: the two middle tokens of four change places, so that
// bytes 0, 2 and 1, 3 of a dword, which one mask takes, hold neighbouring tokens.
__device__ __forceinline__ int kv4_place(int t) { return (t & 12) | ((t & 1) << 1) | ((t >> 1) & 1); }
template <int D, int G>
__device__ __forceinline__ int kv4_side(int P, int which, int group, int t) {
    return P * D + ((which * (D / G) + group) * P + t) * 2;
}

__device__ __forceinline__ float half_bits(uint16_t b) { return (float)__builtin_bit_cast(_Float16, b); }
__device__ __forceinline__ uint16_t to_half_bits(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }

// The value of another lane of the row of 16: the neighbour, the pair over, the four and the eight mirrored.
template <int CTRL>
__device__ __forceinline__ int dpp(int v) {
    return __builtin_amdgcn_mov_dpp(v, CTRL, 0xF, 0xF, true);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, dpp<CTRL>(__builtin_bit_cast(int, v)));
}
constexpr int kXor1 = 0xB1, kXor2 = 0x4E, kHalfMirror = 0x141, kMirror = 0x140;
constexpr int kShiftDown = 0x100;            // + n: lane i gets lane i + n's, 0 past the row's end
constexpr int kBroadcast = 0x150;            // + n: every lane of the row gets lane n's

// 16-bit inputs and outputs, fp16 or bf16.
__device__ __forceinline__ float load16(uint16_t b, bool bf16) {
    return bf16 ? __builtin_bit_cast(float, (uint32_t)b << 16) : half_bits(b);
}
__device__ __forceinline__ uint16_t store16(float v, bool bf16) {
    return bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : to_half_bits(v);
}

// Host side, in w4a16_kv4.hip: what is wrong with a cache's sizes or pointer (null: nothing), the cache as the
// kernels take it, and a failing entry point's message and status.
const char* kv4_check(const w4a16_kv4_cache* c);
Kv4 kv4_of(const w4a16_kv4_cache* c);
int kv4_fail(int code, const char* who, const char* what);

// Calls f with the cache's head and group size as compile-time constants.
template <class F>
inline void kv4_sizes(const w4a16_kv4_cache* c, F f) {
    using Small = std::integral_constant<int, 64>;
    using Large = std::integral_constant<int, 128>;
    if (c->head_dim == 64) f(Small{}, Small{});
    else if (c->group_size == 64) f(Large{}, Small{});
    else f(Large{}, Large{});
}

// Attention's arguments as the kernels take them.
struct Kv4Attn {
    Kv4 c;
    const uint16_t* q;
    uint16_t* out;
    float* lse;
    int64_t q_token, q_head;
    const int* table;
    int64_t table_stride;
    const int* lens;
    const int* q_start;
    int width, tokens, heads, rep;           // rep: query heads of one KV head
    int window;                              // 0: none
    float scale2;                            // scale * log2(e)
    int bf16, causal;
    int q_wide;                              // q's rows can be read 16 bytes at a time
};

// What one sequence asks: queries first .. first + count - 1, keys 0 .. len - 1.
struct Kv4Seq {
    int first, count, len;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4Attn& a, int b) {
    Kv4Seq s;
    s.first = b;
    s.count = 1;
    if (a.q_start) {
        s.first = min(max(a.q_start[b], 0), a.tokens);
        s.count = min(max(a.q_start[b + 1], s.first), a.tokens) - s.first;
    }
    const int64_t most = (int64_t)a.width * a.c.P;
    s.len = (int)min((int64_t)max(a.lens[b], 0), most);
    return s;
}

}  // namespace w4a16

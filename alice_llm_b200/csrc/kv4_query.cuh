// What both kernels of the 4-bit attention (csrc/kv4_attn.cu, csrc/kv4_prompt.cu) do with codes and queries: unpacking, rotation among the lanes that hold a row.
#pragma once
#include <cuda_fp16.h>

#include "kv4.cuh"

namespace alice {

__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t u) { return *reinterpret_cast<const __half2*>(&u); }
// The eight codes of a word less LESS, two to a register: .. [0] nibbles 0 and 4, [1] 1 and 5, [2] 2 and 6, [3] 3 and 7. Four bits put under
// the exponent of 1024 are 1024 + code, or with the next four 1024 + 16 code; both steps are exact.
struct Codes { uint32_t v[4]; };
__device__ __forceinline__ uint32_t under_exponent(uint32_t x, uint32_t mask) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(x), "r"(mask), "r"(0x64006400u));      // x & mask | 1024s, one instruction
    return r;
}
template <int LESS>
__device__ __forceinline__ Codes unpack(uint32_t x) {
    static_assert(LESS == 0 || LESS == 8, "");
    constexpr uint32_t EVEN = 0x000f000fu, ODD = 0x00f000f0u;
    const __half2 less = __half2half2(__ushort_as_half(LESS ? 0xe408 : 0xe400)), sixteenth = __half2half2(__ushort_as_half(0x2c00)),
                  less16 = __half2half2(__ushort_as_half(LESS ? 0xd480 : 0xd400));      // -1024 - LESS, 1 / 16, -64 - LESS
    const uint32_t y = x >> 8;
    Codes c;
    c.v[0] = half2_bits(__hadd2(bits_half2(under_exponent(x, EVEN)), less));
    c.v[1] = half2_bits(__hfma2(bits_half2(under_exponent(x, ODD)), sixteenth, less16));
    c.v[2] = half2_bits(__hadd2(bits_half2(under_exponent(y, EVEN)), less));
    c.v[3] = half2_bits(__hfma2(bits_half2(under_exponent(y, ODD)), sixteenth, less16));
    return c;
}

// (sin, cos) of the pairs that dims dim0 .. dim0 + 3 are in: of two pairs, or (pairs half a head apart) of four.
struct Turn { float4 a, b; };
__device__ __forceinline__ Turn turn_at(const float* turn, uint32_t dim0, const Kv4Rope& rope) {
    auto at = [](const float* p) { return *reinterpret_cast<const float4*>(p); };
    Turn w{};
    if (dim0 < rope.dims) {
        const uint32_t half = rope.dims / 2, j = rope.neox ? 2 * (dim0 < half ? dim0 : dim0 - half) : dim0;
        w.a = at(turn + j);
        if (rope.neox) w.b = at(turn + j + 4);
    }
    return w;
}
// 4 consecutive floats of a query, those of piece k (of 128 dims) from dim0 on, rotated. The lanes of a row hold it 4 dims a lane and piece.
template <int PIECES>
__device__ __forceinline__ float4 rotated4(const float4 (&row)[PIECES], int k, uint32_t dim0, const Turn& w, const Kv4Rope& rope) {
    const float4 x = row[k];
    if (rope.neox) {
        const uint32_t half = rope.dims / 2, lane = threadIdx.x & 31;
        const bool in = dim0 < rope.dims, upper = dim0 >= half;
        const uint32_t other = upper ? dim0 - half : dim0 + half, from = in ? lane + other / 4 - dim0 / 4 & 31 : lane;      // a piece is 32 lanes, or all of the row
        float4 o = make_float4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < PIECES; i++) {
            const float4 y = make_float4(__shfl_sync(0xffffffffu, row[i].x, from), __shfl_sync(0xffffffffu, row[i].y, from), __shfl_sync(0xffffffffu, row[i].z, from), __shfl_sync(0xffffffffu, row[i].w, from));
            if (PIECES == 1 || other / 128 == (uint32_t)i) o = y;
        }
        if (!in) return x;
        const float sg = upper ? 1.0f : -1.0f;
        return make_float4(x.x * w.a.y + sg * (o.x * w.a.x), x.y * w.a.w + sg * (o.y * w.a.z), x.z * w.b.y + sg * (o.z * w.b.x), x.w * w.b.w + sg * (o.w * w.b.z));
    }
    if (dim0 >= rope.dims) return x;
    return make_float4(x.x * w.a.y - x.y * w.a.x, x.x * w.a.x + x.y * w.a.y, x.z * w.a.w - x.w * w.a.z, x.z * w.a.z + x.w * w.a.w);
}

}  // namespace alice

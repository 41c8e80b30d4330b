// Arguments of the paged cache's and the readout's kernels, shared by their
// translation units and the entry points.
#pragma once
#include "zg_hip.h"
#include <type_traits>

#include "zg_device.hpp"
#include "zg_internal.hpp"

namespace zg {

// n / d for n < 2^31 and a divisor the host knows: (n * mul) >> shift with
// mul = 2^shift / d rounded up to the next integer, shift = 31 + ceil(log2 d).
// The excess of mul over 2^shift / d is at most 1, so the quotient is exact
// while n * d < 2^shift.
struct FastDiv {
    uint32_t d = 1, mul = 0x80000001u, shift = 31;
    static FastDiv of(uint32_t d) {
        FastDiv f;
        uint32_t l = 0;
        while (((uint64_t)1 << l) < d) ++l;
        f.d = d;
        f.shift = 31 + l;
        f.mul = (uint32_t)((((uint64_t)1) << f.shift) / d + 1);
        return f;
    }
    __host__ __device__ uint32_t quotient(uint32_t n) const { return (uint32_t)(((uint64_t)n * mul) >> shift); }
};

// The pool of pages on the device; a slot's offset is counted in units of 64
// elements, which 32 bits hold for any pool the entry points take.
struct PagedPool {
    void* keys;
    void* values;
    uint32_t pages;
    FastDiv page_tokens;
    uint32_t page_units;  // page_stride / 64
    uint32_t slot_units;  // kv_heads * head_dim / 64
    int kv_heads, head_dim, bf16;
};

struct AppendArgs {
    PagedPool pool;
    const int32_t* table;
    uint32_t rows, stride, prefix_tokens;
    size_t tokens;
    int q_heads;
    const void *q, *k, *v;
    size_t q_stride, q_head_stride, k_stride, v_stride;
    int io_bf16;
    const float *q_norm, *k_norm;
    float eps;
    int rotate;
    float theta_scale;
    const int32_t *positions, *token_rows;
    void* q_out;
    int32_t* status;
};

struct PagedAttnArgs {
    PagedPool pool;
    const int32_t* table;
    const int32_t* lengths;
    const int32_t* prefix;
    uint32_t rows, stride, prefix_tokens;
    int q_heads, group;
    const void* q;
    size_t q_stride;
    int io_bf16;
    float scale;
    void* workspace;
    void* out;
    size_t out_stride;
    int32_t* status;
};

struct LogitArgs {
    size_t rows, vocab;
    const void* logits;
    size_t ld;
    int bf16;
    zg_logit_rules rules;
    void* out;
    size_t out_ld;
    uint32_t* greedy;
    int record;
    void* workspace;
    int32_t* status;
};

hipError_t paged_append(const AppendArgs& a, hipStream_t st);
hipError_t paged_attn(const PagedAttnArgs& a, hipStream_t st);
size_t paged_attn_workspace(uint32_t rows, int q_heads, int kv_heads, int head_dim, int bf16, uint32_t prefix_tokens,
                            uint64_t row_tokens);
hipError_t logits_adjust(const LogitArgs& a, hipStream_t st);
size_t logits_workspace(size_t rows, size_t vocab);

// ------------------------------------------------------------ device helpers

// f32 -> bf16, nearest even; NaN stays NaN.
__device__ __forceinline__ uint16_t to_bf16(float x) {
    const uint32_t u = __float_as_uint(x);
    if ((u & 0x7fffffffu) > 0x7f800000u) return (uint16_t)((u >> 16) | 0x40u);
    return (uint16_t)((u + 0x7fffu + ((u >> 16) & 1u)) >> 16);
}
// f64 -> bf16 in one rounding, nearest even: the f32 on the way is rounded to
// odd (towards zero, its last bit set where anything was dropped), so that its
// tie is a tie of the 64 bits too.
__device__ __forceinline__ uint16_t to_bf16(double x) {
    const float y = (float)x;
    uint32_t u = __float_as_uint(y);
    if ((double)y != x) u = (fabs((double)y) > fabs(x) ? u - 1 : u) | 1u;
    return to_bf16(__uint_as_float(u));
}

// Four consecutive elements, stored as f32 or bf16.
template <bool BF16>
__device__ __forceinline__ v4f load4(const void* base, size_t at) {
    if constexpr (BF16) {
        const uint2 w = *(const uint2*)((const uint16_t*)base + at);
        return v4f{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                   __uint_as_float(w.y & 0xffff0000u)};
    } else {
        return *(const v4f*)((const float*)base + at);
    }
}
template <bool BF16>
__device__ __forceinline__ void store4(void* base, size_t at, v4f x) {
    if constexpr (BF16) {
        uint2 w;
        w.x = to_bf16(x[0]) | (uint32_t)to_bf16(x[1]) << 16;
        w.y = to_bf16(x[2]) | (uint32_t)to_bf16(x[3]) << 16;
        *(uint2*)((uint16_t*)base + at) = w;
    } else {
        *(v4f*)((float*)base + at) = x;
    }
}

// What a wave wrote to LDS, its other lanes read after this.
__device__ __forceinline__ void same_wave() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The value of the lane 16 or 32 further on (xor), without the LDS.
template <int XOR>
__device__ __forceinline__ float other_quarter(float x) {
    if constexpr (XOR == 16) {
        const auto y = __builtin_amdgcn_permlane16_swap(__float_as_int(x), __float_as_int(x), false, false);
        return __int_as_float((threadIdx.x & 16) ? y[0] : y[1]);
    } else {
        const auto y = __builtin_amdgcn_permlane32_swap(__float_as_int(x), __float_as_int(x), false, false);
        return __int_as_float((threadIdx.x & 32) ? y[0] : y[1]);
    }
}

}  // namespace zg

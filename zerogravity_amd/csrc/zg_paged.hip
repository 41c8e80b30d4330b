// Appending tokens to a paged KV cache, with the head norms and the position
// rotation on the way (include/zg_hip.h, zg_paged_append_device).
#include "zg_paged.hpp"

namespace zg {

constexpr int kMaxPairs = 128;

constexpr int kAheadHeads = 3;  // heads that a thread has loaded before it uses the first

// Sum over aligned groups of W lanes, in every lane, in a fixed order.
template <int W>
__device__ __forceinline__ float group_sum(float v) {
    v += dpp_f<kDppXor1>(v);
    v += dpp_f<kDppXor2>(v);
    v += dpp_f<kDppHalfMirror>(v);
    v += dpp_f<0x140>(v);  // row_mirror: lane i <-> 15 - i within 16
    if (W >= 32) v += other_quarter<16>(v);
    if (W >= 64) v += other_quarter<32>(v);
    return v;
}

// Sine and cosine of |x| <= pi / 4 by their series, which end below 2^-25 of
// the result there; the roundings are about one step of it.
__device__ __forceinline__ void sin_cos(float x, float& s, float& c) {
    const float y = x * x;
    s = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880.0f, -1.0f / 5040.0f), 1.0f / 120.0f), -1.0f / 6.0f), x);
    c = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f), -1.0f / 720.0f), 1.0f / 24.0f), -0.5f),
             1.0f);
}

// A head of D elements lies on D/4 neighbouring lanes, four elements a lane,
// so a norm is a sum over those lanes and a pair's other element a lane away.
// Workgroup (token, y) takes the token's heads (queries, then keys, then
// values) y * 256 / (D/4) and on, gridDim.y of them apart.  A prompt is bound
// by memory, one token by its chain of loads: so the heads are asked for
// before anything else is known of the token, and the angles, one for each
// pair, are formed under them.  8 + 2 + 2 heads of 256 elements, 32 bits to a
// bfloat16 cache: one token 3.9 us, 8192 39 us = 4.7 TB/s, 32768 140 us = 5.3.
template <bool IO, bool KV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
    constexpr int LH = D / 4, SLOTS = 256 / LH;
    __shared__ __align__(16) float cs[kMaxPairs], sn[kMaxPairs];
    const size_t t = blockIdx.x;
    const int tid = threadIdx.x, l = tid % LH, slot = tid / LH, e = 4 * l;
    const int kvs = a.pool.kv_heads, heads = a.q_heads + 2 * kvs, step = gridDim.y * SLOTS, half = a.rotate / 2;
    v4f x[kAheadHeads];
    auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < kAheadHeads; ++u) {
            if (h0 + u * step >= heads) break;
            const int h = min(h0 + u * step + slot, heads - 1);
            const bool query = h < a.q_heads, value = h >= a.q_heads + kvs;
            const int kh = query ? 0 : value ? h - a.q_heads - kvs : h - a.q_heads;
            const void* from = query ? a.q : value ? a.v : a.k;
            x[u] = load4<IO>(from, (query ? t * a.q_stride + (size_t)h * a.q_head_stride
                                          : t * (value ? a.v_stride : a.k_stride) + (size_t)kh * D) + e);
        }
    };
    load(blockIdx.y * SLOTS);
    const int p = a.positions[t];
    // theta_scale^tid by squaring, under the loads (128 of them as an argument
    // were read from the host's memory: 8192 tokens 40.4 us for 39.4, one 4.1 for 3.9)
    double frequency = 1.0, power = (double)a.theta_scale;
#pragma unroll
    for (int bit = 1; bit < kMaxPairs; bit *= 2, power *= power)
        if (tid & bit) frequency *= power;
    const uint32_t row = a.token_rows ? (uint32_t)a.token_rows[t] : (uint32_t)t;
    if (p < 0) return;
    if (tid < half) {
        // the angle in quarter turns, 64 bits until it is within half a one
        const double turns = (double)p * frequency * 0.63661977236758134308;  // 2 / pi
        const double q = rint(turns);
        float s, c;
        sin_cos((float)((turns - q) * 1.57079632679489661923), s, c);
        const int n = (int)((long long)q & 3);
        cs[tid] = n == 0 ? c : n == 1 ? -s : n == 2 ? -c : s;
        sn[tid] = n == 0 ? s : n == 1 ? c : n == 2 ? -s : -c;
    }
    const uint32_t own = (uint32_t)p - a.prefix_tokens, pg = a.pool.page_tokens.quotient(own & 0x7fffffffu);
    // where the token's key and value go; all ones: nowhere
    uint64_t at = ~0ull;
    int bad = 0;
    if ((uint32_t)p < a.prefix_tokens || row >= a.rows || pg >= a.stride) {
        bad = ZG_STATUS_POSITION;
    } else {
        const uint32_t page = (uint32_t)a.table[(size_t)row * a.stride + pg];
        if (page >= a.pool.pages) bad = ZG_STATUS_PAGE;
        else
            at = ((uint64_t)page * a.pool.page_units +
                  (uint64_t)(own - pg * a.pool.page_tokens.d) * a.pool.slot_units) * 64;
    }
    if (bad && a.status && tid == 0 && blockIdx.y == 0) atomicOr(a.status, bad);
    lds_barrier();
    // Element i < half pairs with i + half, half / 4 lanes on: for the 64
    // rotated elements of the models here 8 lanes, a step within 16.
    const bool low = e < half, turned = e < 2 * half;
    const int partner = 4 * ((tid & 63) + (low ? half / 4 : -(half / 4)));
    v4f c = {}, s = {};
    if (turned) {
        c = *(const v4f*)&cs[low ? e : e - half];
        s = *(const v4f*)&sn[low ? e : e - half];
        if (low) s = -s;
    }
    for (int h0 = blockIdx.y * SLOTS; h0 < heads; h0 += kAheadHeads * step) {
        if (h0 != (int)blockIdx.y * SLOTS) load(h0);
#pragma unroll
        for (int u = 0; u < kAheadHeads; ++u) {
            if (h0 + u * step >= heads) break;
            const int h = h0 + u * step + slot;
            const bool query = h < a.q_heads, value = h >= a.q_heads + kvs;
            const float* gamma = query ? a.q_norm : value ? nullptr : a.k_norm;
            v4f y = x[u];
            const float ss = group_sum<LH>(fmaf(y[0], y[0], fmaf(y[1], y[1], fmaf(y[2], y[2], y[3] * y[3]))));
            if (gamma) {
                const float inv = 1.0f / sqrtf(ss / D + a.eps);
                const v4f g = *(const v4f*)(gamma + e);
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = y[j] * inv * g[j];
            }
            v4f o;
            if (half == 32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) o[j] = dpp_f<0x128>(y[j]);  // row_ror:8
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    o[j] = __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(y[j])));
            }
            if (turned && !value)
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = y[j] * c[j] + o[j] * s[j];
            if (h >= heads) continue;
            if (query) store4<IO>(a.q_out, (t * a.q_heads + h) * D + e, y);
            else if (at != ~0ull)
                store4<KV>(value ? a.pool.values : a.pool.keys, at + (size_t)(value ? h - a.q_heads - kvs : h - a.q_heads) * D + e, y);
        }
    }
}

hipError_t paged_append(const AppendArgs& a, hipStream_t st) {
    const int heads = a.q_heads + 2 * a.pool.kv_heads;
    auto go = [&](auto io, auto kv, auto dim) {
        constexpr int D = decltype(dim)::value, slots = 1024 / D;
        // Few tokens: a workgroup for each set of heads (400 tokens 5.2 us, with
        // one for a token 5.7); many: one for a token (1000 tokens 8.5, 9.0).
        const int y = a.tokens < 512 ? (heads + slots - 1) / slots : 1;
        paged_append_kernel<decltype(io)::value, decltype(kv)::value, D>
            <<<dim3((unsigned)a.tokens, y), 256, 0, st>>>(a);
        return hipGetLastError();
    };
    auto by_dim = [&](auto io, auto kv) {
        switch (a.pool.head_dim) {
        case 64: return go(io, kv, std::integral_constant<int, 64>{});
        case 128: return go(io, kv, std::integral_constant<int, 128>{});
        default: return go(io, kv, std::integral_constant<int, 256>{});
        }
    };
    if (a.io_bf16) return a.pool.bf16 ? by_dim(std::true_type{}, std::true_type{}) : by_dim(std::true_type{}, std::false_type{});
    return a.pool.bf16 ? by_dim(std::false_type{}, std::true_type{}) : by_dim(std::false_type{}, std::false_type{});
}

}  // namespace zg

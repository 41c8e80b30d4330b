// Appending tokens to a paged KV cache, with the head norms and the position
// rotation on the way (include/zg_hip.h, zg_paged_append_device).
#include "zg_paged.hpp"

namespace zg {

constexpr int kMaxPairs = 128;

// theta_scale^i in 64 bits, formed on the host and passed by value: a launch
// that is captured into a graph keeps them.
struct Frequencies {
    double f[kMaxPairs];
};

// A head of D elements lies on D/4 neighbouring lanes, four elements a lane.
// Workgroup (token, y) takes the token's heads (queries, then keys, then
// values) y * 256 / (D/4) and on, gridDim.y of them apart.
template <bool IO, bool KV, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a, Frequencies fr) {
    constexpr int LH = D / 4, SLOTS = 256 / LH;
    __shared__ float cs[kMaxPairs], sn[kMaxPairs];
    const size_t t = blockIdx.x;
    const int tid = threadIdx.x, l = tid % LH, slot = tid / LH;
    const int p = a.positions[t];
    if (p < 0) return;
    const int half = a.rotate / 2;
    if (tid < half) {
        // the angle in quarter turns, 64 bits until it is within half a one
        const double turns = (double)p * fr.f[tid] * 0.63661977236758134308;  // 2 / pi
        const double q = rint(turns);
        const float x = (float)((turns - q) * 1.57079632679489661923);
        const float s = sinf(x), c = cosf(x);
        const int n = (int)((long long)q & 3);
        cs[tid] = n == 0 ? c : n == 1 ? -s : n == 2 ? -c : s;
        sn[tid] = n == 0 ? s : n == 1 ? c : n == 2 ? -s : -c;
    }
    const uint32_t row = a.token_rows ? (uint32_t)a.token_rows[t] : (uint32_t)t;
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
    __syncthreads();
    const int heads = a.q_heads + 2 * a.pool.kv_heads;
    for (int h0 = blockIdx.y * SLOTS; h0 < heads; h0 += gridDim.y * SLOTS) {
        const int h = min(h0 + slot, heads - 1);
        const bool live = h0 + slot < heads, query = h < a.q_heads, value = h >= a.q_heads + a.pool.kv_heads;
        const int kh = query ? 0 : value ? h - a.q_heads - a.pool.kv_heads : h - a.q_heads;
        v4f x = query   ? load4<IO>(a.q, t * a.q_stride + (size_t)h * a.q_head_stride + 4 * l)
                : value ? load4<IO>(a.v, t * a.v_stride + (size_t)kh * D + 4 * l)
                        : load4<IO>(a.k, t * a.k_stride + (size_t)kh * D + 4 * l);
        const float* gamma = query ? a.q_norm : value ? nullptr : a.k_norm;
        float ss = fmaf(x[0], x[0], fmaf(x[1], x[1], fmaf(x[2], x[2], x[3] * x[3])));
        ss = wave_sum_xor(ss, LH);
        if (gamma) {
            const float inv = 1.0f / sqrtf(ss / D + a.eps);
            const v4f g = *(const v4f*)(gamma + 4 * l);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = x[j] * inv * g[j];
        }
        // element i < half pairs with i + half, half / 4 lanes on
        const int e = 4 * l;
        const bool low = e < half, turned = e < 2 * half && !value;
        const int partner = (tid & 63) + (low ? half / 4 : -(half / 4));
        v4f y = x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float o = __shfl(x[j], partner, kWave);
            if (turned) {
                const float c = cs[low ? e + j : e + j - half], s = sn[low ? e + j : e + j - half];
                y[j] = low ? x[j] * c - o * s : x[j] * c + o * s;
            }
        }
        if (!live) continue;
        if (query) store4<IO>(a.q_out, (t * a.q_heads + h) * D + e, y);
        else if (at != ~0ull) store4<KV>(value ? a.pool.values : a.pool.keys, at + (size_t)kh * D + e, y);
    }
}

hipError_t paged_append(const AppendArgs& a, hipStream_t st) {
    Frequencies fr{};
    double f = 1.0;
    for (int i = 0; i < a.rotate / 2; ++i, f *= (double)a.theta_scale) fr.f[i] = f;
    const int heads = a.q_heads + 2 * a.pool.kv_heads;
    auto go = [&](auto io, auto kv, auto dim) {
        constexpr int D = decltype(dim)::value, slots = 1024 / D;
        // few tokens: a workgroup for each set of heads
        const int y = a.tokens < 512 ? (heads + slots - 1) / slots : 1;
        paged_append_kernel<decltype(io)::value, decltype(kv)::value, D>
            <<<dim3((unsigned)a.tokens, y), 256, 0, st>>>(a, fr);
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

// Attention of a batch over a shared prefix and each row's own pages
// (include/zg_hip.h, zg_paged_attn_device).
#include "zg_paged.hpp"

namespace zg {

// Workgroup (row, query head): wave w takes tokens w, w + 4, ... of the
// prefix and then of the row, with the running maximum and sum of a softmax;
// the four waves' parts are joined at the end.
template <bool IO, bool KV, int D>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedAttnArgs a) {
    constexpr int LH = D / 4;  // lanes that hold a head; the others repeat them
    __shared__ float part_m[4], part_l[4], part_o[4][D];
    const uint32_t r = blockIdx.x, h = blockIdx.y;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l = lane % LH;
    const int given = a.lengths[r];
    if (given < 0) return;
    const uint32_t room = a.stride * a.pool.page_tokens.d, own = min((uint32_t)given, room);
    int bad = (uint32_t)given > room ? ZG_STATUS_POSITION : 0;
    const uint32_t kvh = h / a.group;
    const v4f q = load4<IO>(a.q, r * a.q_stride + (size_t)h * D + 4 * l);
    float m = -INFINITY, sum = 0.0f;
    v4f o = {};
    for (uint32_t i = wv; i < a.prefix_tokens + own; i += 4) {
        const bool shared = i < a.prefix_tokens;
        const uint32_t t = shared ? i : i - a.prefix_tokens, pg = a.pool.page_tokens.quotient(t);
        const uint32_t page = (uint32_t)(shared ? a.prefix[pg] : a.table[(size_t)r * a.stride + pg]);
        if (page >= a.pool.pages) {
            bad |= ZG_STATUS_PAGE;
            continue;
        }
        const uint64_t at = ((uint64_t)page * a.pool.page_units +
                             (uint64_t)(t - pg * a.pool.page_tokens.d) * a.pool.slot_units) * 64 + kvh * D + 4 * l;
        const v4f k = load4<KV>(a.pool.keys, at), v = load4<KV>(a.pool.values, at);
        float s = fmaf(q[0], k[0], fmaf(q[1], k[1], fmaf(q[2], k[2], q[3] * k[3])));
        s = wave_sum_xor(s, LH) * a.scale;
        const float top = fmaxf(m, s), safe = top == -INFINITY ? 0.0f : top;
        const float keep = expf(m - safe), e = expf(s - safe);
        sum = sum * keep + e;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = fmaf(e, v[j], o[j] * keep);
        m = top;
    }
    if (bad && a.status && lane == 0) atomicOr(a.status, bad);
    if (lane == 0) {
        part_m[wv] = m;
        part_l[wv] = sum;
    }
    if (lane < LH) *(v4f*)&part_o[wv][4 * l] = o;
    __syncthreads();
    if (wv || lane >= LH) return;
    float top = fmaxf(fmaxf(part_m[0], part_m[1]), fmaxf(part_m[2], part_m[3]));
    if (top == -INFINITY) top = 0.0f;
    v4f y = {};
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const float e = expf(part_m[w] - top);
        total += e * part_l[w];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = fmaf(e, part_o[w][4 * l + j], y[j]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = total == 0.0f ? 0.0f : y[j] / total;
    store4<IO>(a.out, r * a.out_stride + (size_t)h * D + 4 * l, y);
}

size_t paged_attn_workspace(uint32_t, int, int, int, uint32_t) { return 256; }

hipError_t paged_attn(const PagedAttnArgs& a, hipStream_t st) {
    auto go = [&](auto io, auto kv, auto dim) {
        paged_attn_kernel<decltype(io)::value, decltype(kv)::value, decltype(dim)::value>
            <<<dim3(a.rows, a.q_heads), 256, 0, st>>>(a);
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

// Penalties, biases and masks on a batch's logits, and the highest one left
// (include/zg_hip.h, zg_logits_adjust_device).
#include "zg_paged.hpp"

namespace zg {

constexpr int kLogitSlice = 4096;  // tokens of a row per workgroup
constexpr uint32_t kSeen = 0x80000000u;

// Order of two candidates of the greedy readout: the higher value, the lower
// index of equal ones.  Index -1: none.
struct Best {
    float v;
    int i;
};
__device__ __forceinline__ Best better(Best a, Best b) {
    const bool second = b.i >= 0 && (a.i < 0 || b.v > a.v || (b.v == a.v && b.i < a.i));
    return second ? b : a;
}
__device__ __forceinline__ Best wave_best(Best b) {
    for (int off = 32; off > 0; off >>= 1) {
        Best o;
        o.v = __shfl_xor(b.v, off, kWave);
        o.i = __shfl_xor(b.i, off, kWave);
        b = better(b, o);
    }
    return b;
}

// Workgroup (slice, row).  The row's history and biases that fall into the
// slice are gathered in LDS: per token the count of its generated
// occurrences (the top bit: it is in the history at all) and the index of
// its first bias; then the slice's logits pass through registers once.
template <bool BF16>
__global__ __launch_bounds__(256) void logits_adjust_kernel(LogitArgs a, int slices) {
    __shared__ uint32_t count[kLogitSlice];
    __shared__ int bias[kLogitSlice];
    __shared__ int twice;
    __shared__ Best found[4];
    const size_t r = blockIdx.y;
    const int tid = threadIdx.x;
    const zg_logit_rules& u = a.rules;
    const int held = u.history ? u.history_lengths[r] : 0;
    if (held < 0) return;
    const size_t first = (size_t)blockIdx.x * kLogitSlice;
    const int n = (int)min((size_t)kLogitSlice, a.vocab - first);
    for (int i = tid; i < kLogitSlice; i += 256) {
        count[i] = 0;
        bias[i] = 0x7fffffff;
    }
    if (tid == 0) twice = 0;
    __syncthreads();
    if (u.history) {
        const int32_t* tokens = u.history + r * u.history_stride;
        const size_t len = min((size_t)held, u.history_stride);
        const int prompt = u.prompt_lengths ? u.prompt_lengths[r] : 0;
        for (size_t i = tid; i < len; i += 256) {
            const uint32_t at = (uint32_t)tokens[i] - (uint32_t)first;
            if ((uint32_t)tokens[i] < a.vocab && at < (uint32_t)n) {
                atomicOr(&count[at], kSeen);
                if ((long long)i >= prompt) atomicAdd(&count[at], 1u);
            }
        }
    }
    const int32_t* ids = u.bias_ids ? u.bias_ids + r * u.bias_stride : nullptr;
    const float* values = u.bias_ids ? u.bias_values + r * u.bias_stride : nullptr;
    const int nb = ids ? max(0, min(u.bias_lengths[r], (int)u.bias_stride)) : 0;
    for (int i = tid; i < nb; i += 256) {
        const uint32_t at = (uint32_t)ids[i] - (uint32_t)first;
        if ((uint32_t)ids[i] < a.vocab && at < (uint32_t)n && atomicMin(&bias[at], i) != 0x7fffffff) twice = 1;
    }
    __syncthreads();
    const double rep = u.repetition ? (double)u.repetition[r] : 1.0;
    const double freq = u.frequency ? (double)u.frequency[r] : 0.0, pres = u.presence ? (double)u.presence[r] : 0.0;
    int mask_row = -1;
    if (u.masks) mask_row = u.mask_of ? u.mask_of[r] : (int)r;
    // a mask that is not there allows nothing
    const bool none = mask_row >= 0 && (size_t)mask_row >= u.mask_rows;
    const uint32_t* mask = mask_row >= 0 && !none ? u.masks + (size_t)mask_row * u.mask_stride : nullptr;
    Best best{0.0f, -1};
    bool odd = false;
    for (int i = tid; i < n; i += 256) {
        const size_t t = first + i;
        float x;
        if constexpr (BF16) x = bf16_to_f32(((const uint16_t*)a.logits)[r * a.ld + t]);
        else x = ((const float*)a.logits)[r * a.ld + t];
        const uint32_t c = count[i];
        const int b = bias[i];
        if (c || b != 0x7fffffff) {
            double v = (double)x;
            if (c) v = v > 0.0 ? v / rep : v * rep;
            if (c & ~kSeen) v = v - freq * (double)(c & ~kSeen) - pres;
            if (b != 0x7fffffff) {
                double add = (double)values[b];
                if (twice)
                    for (int j = b + 1; j < nb; ++j)
                        if (ids[j] == (int)t) add += (double)values[j];
                v += add;
            }
            x = (float)v;
            if constexpr (BF16) x = bf16_to_f32(to_bf16(x));
        }
        const bool allowed = !none && (!mask || (mask[t >> 5] >> (t & 31) & 1u));
        if (!allowed) x = -INFINITY;
        if constexpr (BF16) ((uint16_t*)a.out)[r * a.out_ld + t] = to_bf16(x);
        else ((float*)a.out)[r * a.out_ld + t] = x;
        odd |= x != x || x == INFINITY;
        if (x > -INFINITY) best = better(best, Best{x, (int)t});
    }
    if (a.status && __any(odd) && (tid & 63) == 0) atomicOr(a.status, ZG_STATUS_NONFINITE);
    if (!a.greedy) return;
    best = wave_best(best);
    if ((tid & 63) == 0) found[tid >> 6] = best;
    __syncthreads();
    if (tid == 0) {
        best = better(better(found[0], found[1]), better(found[2], found[3]));
        ((Best*)a.workspace)[r * slices + blockIdx.x] = best;
    }
}

// Workgroup r: the row's slices joined, its id stored and recorded.
__global__ __launch_bounds__(64) void logits_greedy_kernel(LogitArgs a, int slices) {
    const size_t r = blockIdx.x;
    const zg_logit_rules& u = a.rules;
    const int held = u.history ? u.history_lengths[r] : 0;
    if (held < 0) return;
    Best best{0.0f, -1};
    for (int i = threadIdx.x; i < slices; i += 64) best = better(best, ((const Best*)a.workspace)[r * slices + i]);
    best = wave_best(best);
    if (threadIdx.x) return;
    a.greedy[r] = (uint32_t)best.i;
    if (a.record && best.i >= 0 && (size_t)held < u.history_stride) {
        u.history[r * u.history_stride + held] = best.i;
        u.history_lengths[r] = held + 1;
    }
}

static int slices_of(size_t vocab) { return (int)((vocab + kLogitSlice - 1) / kLogitSlice); }

size_t logits_workspace(size_t rows, size_t vocab) { return rows * slices_of(vocab) * sizeof(Best); }

hipError_t logits_adjust(const LogitArgs& a, hipStream_t st) {
    const int slices = slices_of(a.vocab);
    const dim3 grid(slices, (unsigned)a.rows);
    if (a.bf16) logits_adjust_kernel<true><<<grid, 256, 0, st>>>(a, slices);
    else logits_adjust_kernel<false><<<grid, 256, 0, st>>>(a, slices);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.greedy) return e;
    logits_greedy_kernel<<<(unsigned)a.rows, 64, 0, st>>>(a, slices);
    return hipGetLastError();
}

}  // namespace zg
